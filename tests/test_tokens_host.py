"""The entry points of the token rows without a GPU: what they refuse, and how they deal the work out.  csrc/tokens.cpp is built against a
stand-in for the CUDA runtime and for the kernels; addresses are numbers that nobody follows."""
import ctypes as C
import os
import subprocess

import pytest
import torch

import datago_b200 as dg
from datago_b200 import tokens as tk

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "datago_b200", "csrc")
OK, INVALID, SYNC_LIMIT, TOO_LARGE = 0, 1, 10, 11
AT = 1 << 20  # an address


@pytest.fixture(scope="module")
def library(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("fake") / "libtokens.so")
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    sources = [os.path.join(ROOT, "tests", f) for f in ("fake_device.cpp", "fake_tokens.cpp")]
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


def matrix(rows=4, cols=256, ld=None, dtype=1, data=AT):
    return tk._matrix_desc(data or 0, rows, cols, cols if ld is None else ld, dtype, 0)


def rows8(rows=4, cols=256, ld=None, scale_ld=None, block=1, values=AT, scales=AT, by_column=0):
    return tk._rows8_desc(values or 0, scales or 0, rows, cols, -(-(rows if by_column else cols) // 16) * 16 if ld is None else ld, -(-cols // 512) * 4 if scale_ld is None else scale_ld, block, by_column)


BAD_MATRICES = [None, matrix(cols=0), matrix(ld=255), matrix(dtype=3), matrix(dtype=-1), matrix(data=None), matrix(data=AT + 1), matrix(dtype=0, data=AT + 2),
                matrix(rows=1 << 41), matrix(cols=1 << 31, ld=1 << 31), matrix(ld=1 << 59)]
BAD_ROWS8 = [None, rows8(cols=0), rows8(ld=255), rows8(ld=264), rows8(ld=240), rows8(scale_ld=0), rows8(cols=1024, scale_ld=4), rows8(scale_ld=6), rows8(block=0),
             rows8(block=64), rows8(values=None), rows8(scales=None), rows8(values=AT + 8), rows8(scales=AT + 2), rows8(rows=1 << 41)]


def refused(L, rc, status=INVALID):
    assert rc == status, (rc, L.dg_last_error())
    assert L.dg_last_error()
    assert L.fake_launches() == 0


def launched(L, rc, times=1):
    assert rc == OK, L.dg_last_error()
    assert L.fake_launches() == times


def test_a_planning_context_and_no_context_have_no_token_rows(L):
    planning = dg.Context(dg.DG_DEVICE_NONE)
    for ctx in (planning._h, None):
        m, r = matrix(), rows8()
        refused(L, L.dg_quantize_rows(ctx, None, (m), (r)))
        refused(L, L.dg_product(ctx, None, (r), (r), (matrix(4, 4)), None, 0))
        refused(L, L.dg_product_status(ctx, None))
        refused(L, L.dg_dropout(ctx, None, (m), 0.1, 0, 0, 0, (m)))
        refused(L, L.dg_rms_norm(ctx, None, (m), None, None, 1e-6, None, (matrix(data=2 * AT)), None, None))
        one = (C.c_float * 3)(1, 1, 1)
        refused(L, L.dg_patch_rows(ctx, None, AT, 1, 16, 16, 3, 16, one, one, (rows8(1, 768)), None))


def test_quantize_rows_refuses(L, ctx):
    call = lambda m, r: L.dg_quantize_rows(ctx._h, None, m, r)  # noqa: E731
    for m in BAD_MATRICES:
        refused(L, call(m, rows8(values=2 * AT)))
    for r in BAD_ROWS8:
        refused(L, call(matrix(data=3 * AT), r))
    refused(L, call(matrix(), rows8(by_column=1)))               # the transpose has 256 rows
    refused(L, call(matrix(), rows8(256, 4, by_column=1, ld=240)))
    refused(L, call(matrix(), rows8(256, 4, by_column=2)))
    refused(L, call(matrix(rows=0), rows8(256, 16, by_column=1)))
    far = 2 * AT
    for r in (rows8(), rows8(values=AT + 512 * 3), rows8(values=AT - 512), rows8(256, 4, by_column=1, ld=512)):
        refused(L, call(matrix(), r))                            # over the source
    launched(L, call(matrix(), rows8(values=far)))
    launched(L, call(matrix(), rows8(values=far, block=128)))
    launched(L, call(matrix(ld=1024), rows8(values=AT + 512, ld=2048)))  # other columns of the same rows
    refused(L, call(matrix(ld=1024), rows8(values=AT + 496, ld=2048)))
    launched(L, call(matrix(ld=300), rows8(256, 4, by_column=1, values=far)))
    launched(L, call(matrix(rows=0, data=None), rows8(0, values=None, scales=None)), 0)


def test_patch_rows_refuses(L, ctx):
    one, zero, nan = (C.c_float * 4)(1, 1, 1, 1), (C.c_float * 4)(1, 0, 1, 1), (C.c_float * 4)(1, float("nan"), 1, 1)

    def call(n=2, h=32, w=48, c=3, p=16, mean=one, std=one, out8=rows8(12, 768), out=None, pixels=AT):
        return L.dg_patch_rows(ctx._h, None, pixels, n, h, w, c, p, mean, std, (out8), (out))
    launched(L, call())
    launched(L, call(out8=None, out=matrix(12, 768)))
    launched(L, call(n=0, pixels=None, out8=rows8(0, 768)), 0)
    for bad in (dict(out8=None), dict(out=matrix(12, 768)), dict(mean=None), dict(std=None), dict(c=0), dict(c=5), dict(p=0), dict(p=5), dict(h=0), dict(h=40), dict(w=40),
                dict(std=zero), dict(std=nan), dict(mean=nan), dict(pixels=None), dict(out8=rows8(11, 768)), dict(out8=rows8(12, 256)), dict(out8=rows8(12, 768, block=128)), dict(out8=rows8(12, 768, by_column=1)),
                dict(out8=None, out=matrix(12, 767)), dict(n=1 << 20), dict(std=(C.c_float * 4)(1, 1e-39, 1, 1))):
        refused(L, call(**bad))
    refused(L, call(h=128, w=128, p=128, out8=rows8(2, 49152)), TOO_LARGE)
    refused(L, call(n=1, h=1 << 14, w=1 << 14, c=1, p=1, out8=rows8(1 << 28, 1)), TOO_LARGE)


def test_product_refuses(L, ctx):
    def call(a=rows8(), b=rows8(8), out=matrix(4, 8, data=3 * AT), work=None, nbytes=0):
        return L.dg_product(ctx._h, None, (a), (b), (out), work, nbytes)
    launched(L, call())
    launched(L, call(a=rows8(block=128), b=rows8(8, block=128)))
    launched(L, call(a=rows8(by_column=1), b=rows8(8, by_column=1)))
    launched(L, call(a=rows8(0, values=None, scales=None), out=matrix(0, 8, data=None)), 0)
    refused(L, call(out=matrix(4, 8)))
    refused(L, call(b=rows8(8, values=3 * AT + 16)))
    for r in BAD_ROWS8:
        refused(L, call(a=r))
        refused(L, call(b=r))
    for m in BAD_MATRICES:
        refused(L, call(out=m))
    refused(L, call(b=rows8(8, 128)))
    refused(L, call(b=rows8(0)))
    refused(L, call(out=matrix(5, 8)))
    refused(L, call(out=matrix(4, 9)))
    # a long contraction of few rows is split, and its parts need room
    a, b, out = rows8(64, 8192), rows8(64, 8192), matrix(64, 64, data=3 * AT)
    need = L.dg_product_workspace(ctx._h, 64, 64, 8192)
    assert need >= 2 * 64 * 64 * 4
    refused(L, call(a, b, out))
    refused(L, call(a, b, out, AT, need - 1))
    refused(L, call(a, b, out, AT + 4, need))
    launched(L, call(a, b, out, AT, need))


def test_product_status_reports_once(L, ctx):
    assert L.dg_product_status(ctx._h, None) == OK
    L.fake_gave_up(3)
    refused(L, L.dg_product_status(ctx._h, None), SYNC_LIMIT)
    assert L.dg_product_status(ctx._h, None) == OK


def test_rms_norm_refuses(L, ctx):
    out = matrix(data=2 * AT)

    def call(x=matrix(), residual=None, weight=None, eps=1e-6, sum=None, y=out, y8=None, rstd=None):
        return L.dg_rms_norm(ctx._h, None, (x), (residual), (weight), eps, (sum), (y), (y8), rstd)
    launched(L, call())
    launched(L, call(residual=matrix(2, data=3 * AT), weight=matrix(1, dtype=0, data=4 * AT), sum=matrix(), y=None, y8=rows8(values=5 * AT), rstd=AT))
    for bad in (dict(sum=matrix(data=AT + 512)), dict(y=matrix()), dict(y8=rows8()), dict(sum=matrix(data=3 * AT), y8=rows8(values=3 * AT)), dict(sum=matrix(), residual=matrix(2, data=AT + 512)),
                dict(y=matrix(data=3 * AT), sum=matrix(data=3 * AT))):
        refused(L, call(**bad))
    launched(L, call(x=matrix(0, data=None), y=matrix(0, data=None)), 0)
    for m in BAD_MATRICES:
        refused(L, call(x=m))
        if m is not None:
            refused(L, call(residual=m))
            refused(L, call(sum=m))
            refused(L, call(y=m))
    for r in BAD_ROWS8[1:]:
        refused(L, call(y8=r))
    for bad in (dict(residual=matrix(3)), dict(residual=matrix(0)), dict(residual=matrix(cols=128, ld=128)), dict(residual=matrix(dtype=0)), dict(weight=matrix(2)),
                dict(weight=matrix(1, 128)), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(sum=matrix(ld=512)), dict(sum=matrix(5)),
                dict(y=matrix(dtype=0)), dict(y8=rows8(block=128)), dict(y8=rows8(by_column=1)), dict(y8=rows8(5)), dict(rstd=AT + 1), dict(y=None)):
        refused(L, call(**bad))
    wide = matrix(cols=16392, ld=16392)
    refused(L, call(x=wide, y=wide), TOO_LARGE)


def test_rms_norm_backward_refuses(L, ctx):
    need = L.dg_rms_norm_backward_workspace(ctx._h, 4, 256, 2)
    assert need > 0

    def call(dy=matrix(), h=matrix(data=4 * AT), rstd=AT, weight=None, dsum=None, dx=matrix(), dr=AT, period=2, dw=AT, work=AT, nbytes=need):
        return L.dg_rms_norm_backward(ctx._h, None, (dy), (h), rstd, (weight), (dsum), (dx), dr, period, dw, work, nbytes)
    launched(L, call())
    launched(L, call(dx=None, dr=None, period=7))
    empty = matrix(0, data=None)
    launched(L, call(empty, empty, None, dx=empty, work=None, nbytes=0))  # the weight's gradient becomes zero
    for m in BAD_MATRICES:
        refused(L, call(dy=m))
        refused(L, call(h=m))
        if m is not None:
            refused(L, call(dsum=m))
            refused(L, call(dx=m))
    for bad in (dict(rstd=None), dict(rstd=AT + 2), dict(dr=AT + 2), dict(dw=AT + 2), dict(period=0), dict(period=3), dict(weight=matrix(2)), dict(h=matrix(dtype=0)),
                dict(dx=matrix(ld=512)), dict(dsum=matrix(data=3 * AT, ld=512), dx=matrix(data=3 * AT)), dict(dx=matrix(data=4 * AT)), dict(dx=matrix(data=AT + 512)), dict(dx=None, dr=None, dw=None), dict(work=None), dict(nbytes=need - 1), dict(work=AT + 4)):
        refused(L, call(**bad))
    wide = matrix(cols=16392, ld=16392)
    refused(L, call(wide, wide, dx=wide), TOO_LARGE)


def test_dropout_refuses(L, ctx):
    def call(x=matrix(), p=0.1, seed=1, offset=0, per_row=0, y=matrix(data=2 * AT)):
        return L.dg_dropout(ctx._h, None, (x), p, seed, offset, per_row, (y))
    launched(L, call())
    launched(L, call(y=matrix()))
    launched(L, call(p=0.0))
    launched(L, call(p=65535 / 65536))
    launched(L, call(offset=(1 << 64) - 1 - 4, per_row=1))
    launched(L, call(x=matrix(0, data=None), y=matrix(0, data=None)), 0)
    for m in BAD_MATRICES:
        refused(L, call(x=m))
        refused(L, call(y=m))
    for bad in (dict(p=-0.1), dict(p=1.0), dict(p=0.999999), dict(p=float("nan")), dict(offset=(1 << 64) - 4), dict(y=matrix(5)), dict(y=matrix(dtype=2)), dict(y=matrix(ld=512))):
        refused(L, call(**bad))


@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 48, 64), (7, 1024, 768), (128, 240, 128), (129, 241, 129), (200, 4801, 512), (1152, 768, 57600), (131072, 1152, 768),
                                   (37, 65, 1 << 20), (1 << 20, 16, 16), (5, 1 << 17, 640)])
@pytest.mark.parametrize("b_by_column", [0, 1])
def test_product_plans_cover_the_output_and_the_contraction(L, ctx, m, n, k, b_by_column):
    v = (C.c_uint32 * 8)()
    L.fake_product_plan(C.c_uint64(m), C.c_uint64(n), C.c_uint64(k), b_by_column, v)
    tile_n, tiles_m, tiles_n, splits, per_split, sums, slots, a_stays = v
    groups = -(-k // 128)
    assert tile_n % 32 == 0 and 32 <= tile_n <= (256 if sums == 1 else 224)
    assert (tiles_m - 1) * 256 < m <= tiles_m * 256 and (tiles_n - 1) * tile_n < n <= tiles_n * tile_n
    assert splits == 1 or k > 1920  # what the binding counts on
    assert (splits == 1 or per_split % 4 == 0) and (splits - 1) * per_split < groups <= splits * per_split
    # the rings fit what the kernel has for them, and work while something is under way
    b_bytes = (128 if b_by_column else tile_n // 2) * 128
    assert slots >= 2 and (groups * 16384 if a_stays else slots * 2 * 16384) + slots * 2 * b_bytes <= 192 * 1024
    assert not a_stays or (splits == 1 and groups <= 12)
    if splits > 1:
        assert L.dg_product_workspace(ctx._h, m, n, k) >= splits * m * -(-n // 4) * 16


@pytest.mark.parametrize("rows,cols,period,residual", [(1, 8, 1, 0), (1, 8, 1, 1), (100000, 1152, 1, 1), (55056, 1152, 2294, 1), (55056, 1152, 55056, 0), (64, 16384, 4, 1), (12, 300, 12, 1)])
def test_norm_backward_deals_out_every_row(L, rows, cols, period, residual):
    v = (C.c_uint32 * 2)()
    L.fake_backward_split(C.c_uint64(rows), C.c_uint64(cols), C.c_uint64(period), residual, v)
    workers, parts = v
    assert 1 <= workers <= 148 * 32 and 1 <= parts <= rows // period
    ctx = dg.Context(0)
    assert L.dg_rms_norm_backward_workspace(ctx._h, rows, cols, period if residual else 0) >= 4 * cols * (workers + (parts * period if parts > 1 else 0))


def test_tensors_of_the_host_and_of_other_shapes_are_refused():
    class Here:
        device, _h = 0, None
    x = torch.zeros(4, 256)
    for call in (lambda: tk.quantize_rows(Here, x), lambda: tk.rms_norm(Here, x), lambda: tk.dropout(Here, x, 0.1, 1), lambda: tk.patch_rows(Here, torch.zeros(1, 16, 16, 3, dtype=torch.uint8), 16, (0,) * 3, (1,) * 3),
                 lambda: tk.product(Here, tk.Rows8.empty(4, 256, "cpu"), tk.Rows8.empty(4, 256, "cpu")), lambda: tk.product(Here, x, x), lambda: tk.dropout(Here, [1.0], 0.1, 1),
                 lambda: tk.rms_norm_backward(Here, x, x, x[:, 0])):
        with pytest.raises(dg.DatagoB200Error):
            call()


def test_rows8_start_where_the_kernels_want_them():
    for rows, cols, block in ((1, 1, 1), (5, 588, 1), (300, 1000, 128)):
        r = tk.Rows8.empty(rows, cols, "cpu", block)
        assert r.shape == (rows, cols) and r.scales.shape == (-(-rows // block), -(-cols // 128))
        assert r.values.stride(0) % 16 == 0 and r.scales.stride(0) % 4 == 0
