"""The entry points of the token rows at their edges, without a GPU: csrc/tokens.cpp against stand-ins for the CUDA runtime and for the kernels (see
test_tokens_host.py, whose helpers are used here)."""
import ctypes as C
import os
import subprocess

import pytest
import torch

import datago_b200 as dg
from datago_b200 import tokens as tk
from test_tokens_host import AT, CSRC, INVALID, OK, ROOT, SYNC_LIMIT, TOO_LARGE, launched, matrix, refused, rows8


@pytest.fixture(scope="module")
def library(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("fake") / "libtokens_edges.so")
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    sources = [os.path.join(ROOT, "tests", f) for f in ("fake_device.cpp", "fake_tokens_edges.cpp")]
    sources += [os.path.join(CSRC, f) for f in ("tokens.cpp", "api.cu", "feeder.cpp", "host_blocks.cpp", "host_logic.cpp", "jpeg_header.cpp")]
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-pthread", "-Wl,-Bsymbolic", "-I", os.path.join(cuda, "include"), "-x", "c++", *sources, "-o", out], check=True)
    return out


@pytest.fixture
def L(library, monkeypatch):
    monkeypatch.setattr(dg, "library_path", lambda: library)
    monkeypatch.setattr(dg, "_lib", None)
    monkeypatch.delenv("DATAGO_B200_REBUILD", raising=False)
    lib = tk.lib()
    lib.fake_launches()
    yield lib
    monkeypatch.setattr(tk, "_lib", None)


@pytest.fixture
def ctx(L):
    return dg.Context(0)


@pytest.mark.parametrize("rows,cols,by_column,column", [(768, 1, True, 1), (16, 1, True, 1), (768, 1, False, 0), (1, 768, True, 1), (1, 768, False, 0), (768, 2, True, 1), (1, 1, True, 0), (1, 1, False, 0)])
def test_rows8_of_a_single_row_or_column_keep_their_order(L, ctx, monkeypatch, rows, cols, by_column, column):
    monkeypatch.setattr(tk, "_on_device", lambda ctx, t, name: None)
    r = tk.Rows8.empty(rows, cols, "cpu", by_column=by_column)
    desc = tk._rows8(ctx, r, "a")
    assert int.from_bytes(desc[-4:], "little") == column  # dg_rows8.by_column
    launched(L, L.dg_product(ctx._h, None, desc, rows8(5, cols), matrix(rows, 5, data=3 * AT), None, 0))
    assert tk._rows8(ctx, r, "out", by_column) == desc or (rows == 1 and cols == 1)


@pytest.mark.parametrize("rows,cols,period", [(6144, 1152, 256), (90000, 1152, 300), (100000, 512, 500), (4, 256, 2), (7, 33, 3), (24, 16384, 24), (1, 8, 1), (55056, 1152, 2294)])
def test_a_norms_backward_pass_needs_what_was_asked_for(L, ctx, rows, cols, period):
    need = L.dg_rms_norm_backward_workspace(ctx._h, rows, cols, period)
    assert need > 0
    x, h = matrix(rows, cols), matrix(rows, cols, data=1 << 40)
    for dresidual in (AT, None):  # residual_rows is ignored without dresidual
        if dresidual and rows % period:
            continue
        launched(L, L.dg_rms_norm_backward(ctx._h, None, x, h, AT, None, None, None, dresidual, period, AT, AT, need))
    assert L.dg_rms_norm_backward_workspace(ctx._h, rows, cols, 0) <= need


def test_the_norms_two_outputs_are_apart(L, ctx):
    def call(y, y8):
        return L.dg_rms_norm(ctx._h, None, matrix(), None, None, 1e-6, None, y, y8, None)
    launched(L, call(matrix(data=2 * AT), rows8(values=3 * AT)))
    refused(L, call(matrix(data=2 * AT), rows8(values=2 * AT)))
    refused(L, call(matrix(data=2 * AT), rows8(values=2 * AT + 4 * 512 - 16)))
    launched(L, call(matrix(data=2 * AT), rows8(values=2 * AT + 4 * 512)))


def test_a_single_row_is_apart_from_rows_beside_it(L, ctx):
    # rows of 256 elements of 2 bytes, 512 elements apart; one row beside them, whatever distance it names
    def call(at, cols=256, ld=None, rows=1):
        return L.dg_rms_norm(ctx._h, None, matrix(ld=512, data=AT), matrix(rows, cols, ld, data=at), None, 1e-6, matrix(ld=512, data=AT), None, None, None)
    launched(L, call(AT + 512))
    launched(L, call(AT + 512 + 3 * 1024))
    launched(L, call(AT + 512, ld=300))
    launched(L, call(AT - 512))
    for at in (AT, AT + 2, AT + 510, AT + 514, AT + 1024, AT + 3 * 1024, AT - 510):
        refused(L, call(at))
    launched(L, call(AT + 512, ld=512, rows=2))
    refused(L, call(AT + 512, ld=600, rows=2))  # the second one is in the first columns of the rows


def test_images_are_counted_in_32_bits(L, ctx):
    one = (C.c_float * 4)(1, 1, 1, 1)

    def call(n):
        return L.dg_patch_rows(ctx._h, None, AT, n, 1, 1, 1, 1, one, one, rows8(n, 1, values=1 << 50, scales=1 << 52), None)
    launched(L, call((1 << 31) - 1024))
    for n in ((1 << 31) - 1023, 1 << 31, (1 << 32) - 1):
        refused(L, call(n), TOO_LARGE)


def test_dropout_takes_the_last_index_there_is(L, ctx):
    def call(offset, per_row, rows=4):
        return L.dg_dropout(ctx._h, None, matrix(rows), 0.1, 1, offset, per_row, matrix(rows, data=2 * AT))
    for per_row, count in ((0, 1024), (1, 4)):
        launched(L, call((1 << 64) - count, per_row))
        refused(L, call((1 << 64) - count + 1, per_row))
        refused(L, call((1 << 64) - 1, per_row))


@pytest.mark.parametrize("cols,status", [(16384, OK), (16385, TOO_LARGE), (32768, TOO_LARGE)])
def test_a_norm_has_as_many_columns_as_the_header_says(L, ctx, cols, status):
    with open(os.path.join(ROOT, "include", "datago_b200.h")) as f:
        text = f.read()
    assert "cols at most 16384" in text and "at most 32768" not in text
    x, h = matrix(4, cols), matrix(4, cols, data=2 * AT)
    need = L.dg_rms_norm_backward_workspace(ctx._h, 4, cols, 0)
    check = launched if status == OK else lambda L, rc: refused(L, rc, status)
    check(L, L.dg_rms_norm(ctx._h, None, x, None, None, 1e-6, None, h, None, None))
    check(L, L.dg_rms_norm_backward(ctx._h, None, x, h, AT, None, None, None, None, 0, AT, AT, need))


def test_every_context_learns_of_products_that_gave_up(L):
    first, second = dg.Context(0), dg.Context(0)
    for c in (first, second):
        assert L.dg_product_status(c._h, None) == OK
    L.fake_gave_up(3)
    refused(L, L.dg_product_status(first._h, None), SYNC_LIMIT)
    assert L.dg_product_status(first._h, None) == OK  # once
    later = dg.Context(0)
    assert L.dg_product_status(later._h, None) == OK  # reported before there was this one
    refused(L, L.dg_product_status(second._h, None), SYNC_LIMIT)  # its own report, which the other one's call has not taken
    assert b"3 CTAs" in L.dg_last_error()
    assert L.dg_product_status(second._h, None) == OK
    L.fake_gave_up(1)
    for c in (later, second, first):
        refused(L, L.dg_product_status(c._h, None), SYNC_LIMIT)
        assert b"1 CTAs" in L.dg_last_error()
        assert L.dg_product_status(c._h, None) == OK


@pytest.mark.parametrize("m,n,k", [(1152, 768, 1 << 20), (4096, 1152, 57600), (4096, 4096, 131072), (64, 64, 1 << 24), (1, 1, (1 << 31) - 1024), (65536, 65536, 1 << 20), (8192, 8192, 8192), (8192, 8192, 8193),
                                   (131072, 1152, 768), (200, 4801, 8320), (1152, 768, 57600)])
@pytest.mark.parametrize("b_by_column", [0, 1])
def test_no_part_of_a_contraction_is_longer_than_64_groups(L, ctx, m, n, k, b_by_column):
    v = (C.c_uint64 * 6)()
    L.fake_product_plan(C.c_uint64(m), C.c_uint64(n), C.c_uint64(k), b_by_column, v)
    splits, per_split, together, tiles, slots, a_stays = v
    groups = -(-k // 128)
    assert per_split <= 64 and (splits - 1) * per_split < groups <= splits * per_split
    assert 1 <= together <= splits and tiles * together < 1 << 31 and (splits == 1 or per_split % 4 == 0)
    part = m * -(-n // 4) * 16
    if splits == 1:
        assert together == 1
        return
    # all parts at once, or as many as half a GB holds and a place for their sum
    kept = splits if together == splits else together + 1
    assert L.dg_product_workspace(ctx._h, m, n, k) >= kept * part
    assert together == 1 or together * part <= 1 << 29
    assert together == splits or (together + 1) * part > 1 << 29
