"""Token rows at their edges: single rows and none, widths at the border of what a launch may have, states that change between a forward pass
and its backward pass, sums that have to come out exactly.

Products of whole numbers whose sums of magnitudes stay below 2^23 are exact in 32 bits in any order, also where additions cut off what lies below 2^-23 of
the largest addend: such tests want equality."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import datago_b200 as dg
from datago_b200 import tokens as tk

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
MEAN, STD = (0.48, 0.46, 0.41), (0.27, 0.26, 0.28)


@pytest.fixture(scope="module")
def ctx():
    return dg.Context(0)


def rand(shape, dtype, seed, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * spread).to(dtype)


def some_pixels(shape, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(0, 256, shape, generator=g, device="cuda", dtype=torch.uint8)


def stem_of(ctx, p=0.25, width=96, dtype=F32):
    return tk.PatchStem(ctx, 14, MEAN, STD, rand((width, 588), F32, 1, 0.02), rand((width,), F32, 2), p=p, seed=5, dtype=dtype)


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


# ---- states --------------------------------------------------------------------------------------------------------------
def test_a_backward_pass_goes_by_its_forward_pass(ctx):
    stem, pixels, positions, dy = stem_of(ctx), some_pixels((2, 28, 42, 3), 3), rand((6, 96), F32, 4), rand((12, 96), F32, 5)
    saved = stem.forward(pixels, positions, offset=11)[1]
    want = stem.backward(saved, dy)
    kept = stem.p, stem.seed, stem.norm_weight
    for change in (dict(p=0.0), dict(p=0.75), dict(seed=6), dict(norm_weight=None), dict(norm_weight=rand((96,), F32, 7))):
        for name, value in change.items():
            setattr(stem, name, value)
        assert same(stem.backward(saved, dy), want), change
        stem.p, stem.seed, stem.norm_weight = kept
    stem.p = 0.0  # and one without dropout stays one
    saved = stem.forward(pixels, positions)[1]
    want = stem.backward(saved, dy)
    stem.p = 0.5
    assert same(stem.backward(saved, dy), want)


def test_a_captured_stem_reads_the_weight_that_was_set(ctx):
    stem, pixels, positions = stem_of(ctx), some_pixels((2, 28, 42, 3), 13), rand((6, 96), F32, 14)
    stem.forward(pixels, positions)
    places = stem.weight8.values.data_ptr(), stem.weight8.scales.data_ptr()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = stem.forward(pixels, positions)[0]
    new = rand((96, 588), F32, 15, 0.05)
    stem.set_weight(new)
    assert (stem.weight8.values.data_ptr(), stem.weight8.scales.data_ptr()) == places
    graph.replay()
    other = tk.PatchStem(ctx, 14, MEAN, STD, new, stem.norm_weight, p=0.25, seed=5, dtype=F32)
    want = other.forward(pixels, positions)[0]
    assert torch.equal(norm.sum, want.sum) and torch.equal(norm.y.values.float(), want.y.values.float())
    stem.set_weight(rand((100, 588), F32, 16))  # of another shape: elsewhere
    assert stem.weight8.shape == (100, 588)


# ---- autograd --------------------------------------------------------------------------------------------------------------
def calls_on(ctx, t, plain):
    """Every function on `t` (64 x 256) where `plain` does as well."""
    rstd = torch.ones(64, device="cuda")
    return (lambda: tk.quantize_rows(ctx, t), lambda: tk.rms_norm(ctx, t), lambda: tk.rms_norm(ctx, plain, residual=t), lambda: tk.rms_norm(ctx, plain, weight=t[0]),
            lambda: tk.rms_norm_backward(ctx, t, plain, rstd), lambda: tk.rms_norm_backward(ctx, plain, t, rstd), lambda: tk.rms_norm_backward(ctx, plain, plain, rstd, dsum=t),
            lambda: tk.dropout(ctx, t, 0.5, 1), lambda: tk.dropout(ctx, plain, 0.5, 1, out=t))


def test_tensors_whose_gradient_would_be_lost_are_refused(ctx):
    leaf, plain = rand((64, 256), F32, 20).requires_grad_(), rand((64, 256), F32, 21)
    for t in (leaf, leaf * 2):
        for call in calls_on(ctx, t, plain):
            with pytest.raises(dg.DatagoB200Error, match="grad"):
                call()
        with torch.no_grad():
            for call in calls_on(ctx, t.detach().clone().requires_grad_(), plain):
                call()


def test_a_stem_takes_parameters(ctx):
    weight, norm_weight, positions = (torch.nn.Parameter(rand(s, F32, 22 + i, 0.1)) for i, s in enumerate(((96, 588), (96,), (6, 96))))
    pixels, dy = some_pixels((2, 28, 42, 3), 25), rand((12, 96), F32, 26)
    stem = tk.PatchStem(ctx, 14, MEAN, STD, weight, norm_weight, p=0.1, dtype=F32)
    norm, saved = stem.forward(pixels, positions)
    got = stem.backward(saved, dy)
    assert not norm.sum.requires_grad
    other = tk.PatchStem(ctx, 14, MEAN, STD, weight.detach(), norm_weight.detach(), p=0.1, dtype=F32)
    assert same(got, other.backward(other.forward(pixels, positions.detach())[1], dy))


def test_autograd_notices_results_that_are_written_into_its_tensors(ctx):
    w = torch.ones(64, 256, device="cuda", requires_grad=True)
    plain, rstd, pixels = rand((64, 256), F32, 27), torch.ones(64, device="cuda"), some_pixels((64, 8, 8, 4), 28)
    a8, b8 = tk.quantize_rows(ctx, rand((64, 100), F32, 29)), tk.quantize_rows(ctx, rand((256, 100), F32, 30))
    for write in (lambda x: tk.dropout(ctx, x, 0.5, 1, out=x), lambda x: tk.rms_norm(ctx, x, sum_out=x), lambda x: tk.rms_norm_backward(ctx, x, plain, rstd, dx_out=x),
                  lambda x: tk.product(ctx, a8, b8, F32, out=x), lambda x: tk.patch_rows(ctx, pixels, 8, MEAN + (0.5,), STD + (0.5,), F32, out=x)):
        x = rand((64, 256), F32, 31)
        loss = (x * w).sum()
        write(x)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    with torch.inference_mode():
        x = rand((64, 256), F32, 32)
        tk.dropout(ctx, x, 0.5, 1, out=x)


def test_a_stem_refuses_what_is_no_tensor(ctx):
    stem, pixels = stem_of(ctx), some_pixels((1, 14, 14, 3), 70)
    before = stem.weight8
    for call in (lambda: stem.set_weight([1.0]), lambda: stem.set_weight(None), lambda: stem.forward(pixels, [[0.0] * 96]), lambda: stem.forward(pixels, rand((1, 96), F32, 1).cpu()),
                 lambda: tk.PatchStem(ctx, 14, MEAN, STD, "weight")):
        with pytest.raises(dg.DatagoB200Error):
            call()
    assert stem.weight8 is before
    stem.norm_weight = [1.0] * 96
    with pytest.raises(dg.DatagoB200Error):
        stem.forward(pixels, rand((1, 96), F32, 1))


# ---- single rows and none --------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("block", [1, 128])
@pytest.mark.parametrize("m,n", [(768, 33), (33, 47), (16, 1), (1, 768), (1, 1), (1000, 300)])
def test_product_over_a_single_row_of_transposed_operands(ctx, m, n, block):
    a, b = tk.quantize_rows(ctx, rand((1, m), F32, 40), transpose=True, block=block), tk.quantize_rows(ctx, rand((1, n), F32, 41), transpose=True, block=block)
    want = a.to_float().double() @ b.to_float().double().t()  # one product each
    assert torch.equal(tk.product(ctx, a, b, F32).double(), want.float().double())
    by_row = tk.Rows8.empty(n, 1, "cuda", block)
    by_row.values.copy_(b.values)
    by_row.scales.view(torch.uint8).copy_(b.scales.view(torch.uint8))
    assert torch.equal(tk.product(ctx, a, by_row, F32).double(), want.float().double())


def test_stem_of_a_single_patch(ctx):
    stem, pixels, positions, dy = stem_of(ctx, p=0.0), some_pixels((1, 14, 14, 3), 42), rand((1, 96), F32, 43), rand((1, 96), F32, 44)
    norm, saved = stem.forward(pixels, positions)
    dweight, dpositions, dnorm = stem.backward(saved, dy)
    dx = tk.rms_norm_backward(ctx, dy, norm.sum, norm.rstd, stem.norm_weight)[0]
    x = tk.patch_rows(ctx, pixels, 14, MEAN, STD, F32)
    # every group is one number, which its scale brings to [224, 448]: half a step of e4m3 is 2^-4 of it, each
    want = dx.double().t() @ x.double()
    assert bool(((dweight - want).abs() <= (2 * 2.0 ** -4 + 2.0 ** -7) * want.abs()).all())
    assert torch.equal(dpositions, dx) and dnorm.shape == (96,)


def test_stem_of_no_images(ctx):
    stem = stem_of(ctx)
    norm, saved = stem.forward(some_pixels((0, 28, 42, 3), 45), rand((6, 96), F32, 46))
    assert norm.y.shape == (0, 96) and norm.sum.shape == (0, 96)
    dweight, dpositions, dnorm = stem.backward(saved, torch.empty(0, 96, device="cuda"))
    assert dweight.shape == (96, 588) and dpositions.shape == (6, 96) and dnorm.shape == (96,)
    assert not bool(dweight.any()) and not bool(dpositions.any()) and not bool(dnorm.any())


def test_a_row_beside_other_rows_is_apart_from_them(ctx):
    big = rand((12, 512), F32, 55)
    x, weight, position = big[:, 256:], big[0, :256], big[3:4, :256]
    want = tk.rms_norm(ctx, x.clone(), weight.clone(), residual=position.clone())
    got = tk.rms_norm(ctx, x, weight, residual=position, sum_out=x)
    assert torch.equal(got.y, want.y) and torch.equal(x, want.sum)
    with pytest.raises(dg.DatagoB200Error):
        tk.rms_norm(ctx, x, big[0, 128:384], sum_out=x)


def test_dropout_of_the_last_indices_there_are(ctx):
    x = torch.ones(4, 24, device="cuda")
    first = (1 << 64) - 96
    whole = tk.dropout(ctx, x, 0.5, 3, first)
    for r in range(4):  # row by row, the last one alone
        assert torch.equal(tk.dropout(ctx, x[r:r + 1], 0.5, 3, first + 24 * r), whole[r:r + 1])
    assert torch.equal(tk.dropout(ctx, x[:, :1], 0.5, 3, (1 << 64) - 4, per_row=True)[3], tk.dropout(ctx, x[:1, :1], 0.5, 3, (1 << 64) - 1)[0])
    for call in (lambda: tk.dropout(ctx, x, 0.5, 3, first + 1), lambda: tk.dropout(ctx, x, 0.5, 3, (1 << 64) - 3, per_row=True)):
        with pytest.raises(dg.DatagoB200Error):
            call()


# ---- borders ---------------------------------------------------------------------------------------------------------------
def norms_of_wide_rows():
    own = dg.Context(0)
    for dtype in (F32, BF16):
        for cols in (12288, 12280, 12273, 12264, 12289, 16384):  # the weight as floats: 48 KB and a little less or more
            x, w = rand((3, cols), dtype, cols), rand((cols,), F32, 50)
            got = tk.rms_norm(own, x, w)
            want = x.double() / torch.sqrt(x.double().square().mean(1, keepdim=True) + 1e-6) * w.double()
            # a sum of 64 + 14 additions, a handful of products, the rounding to the type
            assert bool(((got.y.double() - want).abs() <= (50 * 2.0 ** -24 + (2.0 ** -8 if dtype is BF16 else 2.0 ** -24)) * want.abs() + 1e-30).all()), (dtype, cols)


def test_norm_of_weights_that_need_more_shared_memory_than_a_launch_has_unasked():
    # in a process of its own: what a kernel has been allowed once it may have from then on
    here = os.path.dirname(os.path.abspath(__file__))
    code = "import sys; sys.path[:0] = [%r, %r]; import test_gpu_tokens_edges as t; t.norms_of_wide_rows()" % (here, os.path.dirname(here))
    subprocess.run([sys.executable, "-c", code], check=True, timeout=300)


def test_norm_has_16384_columns_at_most(ctx):
    for cols in (16384, 16385):
        x, rstd = rand((2, cols), BF16, 51), torch.ones(2, device="cuda")
        for call in (lambda: tk.rms_norm(ctx, x), lambda: tk.rms_norm_backward(ctx, x, x.clone(), rstd)):
            if cols == 16384:
                call()
            else:
                with pytest.raises(dg.DatagoB200Error, match="16384"):
                    call()


# ---- products ----------------------------------------------------------------------------------------------------------------
def whole_numbers(rows, cols, most, scales, seed, by_column=False):
    """Rows8 of whole numbers up to `most` in magnitude, whose groups have scales 2^0 .. 2^scales."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = tk.Rows8.empty(rows, cols, "cuda", by_column=by_column)
    r.values.copy_(torch.randint(-most, most + 1, (rows, cols), generator=g, device="cuda", dtype=torch.int8).float())
    r.scales.view(torch.uint8).copy_(torch.randint(127, 128 + scales, r.scales.shape, generator=g, device="cuda", dtype=torch.uint8))
    return r


def sum_of_products(a, b):
    total = torch.zeros(a.shape[0], b.shape[0], dtype=torch.float64, device="cuda")
    step = 16384
    for k in range(0, a.shape[1], step):
        part = [tk.Rows8(r.values[:, k:k + step], r.scales[:, k // 128:(k + step) // 128]).to_float().double() for r in (a, b)]
        total += part[0] @ part[1].t()
    return total


@pytest.mark.parametrize("m,n,k,most,scales", [(1, 1, 5, 7, 2), (7, 1024, 768, 7, 2), (129, 241, 513, 7, 2), (300, 96, 1500, 7, 2), (2561, 520, 300, 7, 2), (20001, 200, 640, 7, 2),
                                               (64, 64, 20000, 2, 1), (1152, 768, 5000, 3, 1), (250, 130, 9000, 3, 1)])
@pytest.mark.parametrize("a_turned,b_turned", [(False, False), (True, True)])
def test_products_of_whole_numbers_are_exact(ctx, m, n, k, most, scales, a_turned, b_turned):
    a, b = whole_numbers(m, k, most, scales, m + k, a_turned), whole_numbers(n, k, most, scales, n + k + 1, b_turned)
    assert k * (most << scales) ** 2 < 1 << 23
    assert torch.equal(tk.product(ctx, a, b, F32).double(), sum_of_products(a, b))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n", [1, 2, 3, 4, 7, 8, 9, 15, 33, 250, 685, 894])
def test_product_leaves_what_lies_behind_the_columns(ctx, dtype, n):
    # rows of the output begin at multiples of 16 bytes, and end anywhere; what lies between them belongs to the caller
    for m, k, gap in ((5, 200, 0), (300, 128, 16), (70, 9000, 8)):
        a, b = whole_numbers(m, k, 1, 0, m + k), whole_numbers(n, k, 1, 0, n + k)
        big = torch.full((m, -(-n // 8) * 8 + gap), 7.0, dtype=dtype, device="cuda")
        tk.product(ctx, a, b, dtype, out=big[:, :n])
        want = sum_of_products(a, b).float().to(dtype)
        assert torch.equal(big[:, :n], want) and bool((big[:, n:] == 7).all()), (m, k)


def one_and_ones(rows, groups):
    """2^15 in the first column, nothing in the rest of its group, ones elsewhere."""
    r = tk.Rows8.empty(rows, 128 * groups, "cuda")
    r.values.copy_(torch.ones(1, device="cuda"))
    r.values[:, 1:128].copy_(torch.zeros(1, device="cuda"))
    r.scales.view(torch.uint8).fill_(127)
    r.scales.view(torch.uint8)[:, 0] = 127 + 15
    return r


@pytest.mark.parametrize("m,n,groups", [(1152, 768, 2048), (2560, 2560, 320), (64, 64, 1 << 13), (4096, 1152, 450)])
def test_long_sums_lose_what_64_groups_lose(ctx, m, n, groups):
    # Beside 2^30 the tensor cores' sums have steps of 2^7, and all that 32 ones add is cut off, up to the end of the part.  Other parts are exact; they
    # are off by 2^6 at most each time when they are added; there are 16, or one for 60 groups.
    got = tk.product(ctx, one_and_ones(m, groups), one_and_ones(n, groups), F32).double()
    off = (got - (2.0 ** 30 + 128 * (groups - 1))).abs().max()
    assert off <= 63 * 128 + 64 * max(17, groups // 60 + 2), off


def test_parts_that_do_not_fit_their_workspace_at_once(ctx):
    m, n, k = 4096, 2048, 163840  # 20 parts of 32 MB
    assert tk.lib().dg_product_workspace(ctx._h, m, n, k) < 20 * m * n * 4
    a, b = whole_numbers(m, k, 1, 0, 60), whole_numbers(n, k, 1, 0, 61)
    want = sum_of_products(a, b)
    assert torch.equal(tk.product(ctx, a, b, F32).double(), want)
    got = tk.product(ctx, a, b, BF16)
    assert torch.equal(got, want.float().to(BF16))  # rounded once
    tk.product_status(ctx)


# ---- buckets of batches ------------------------------------------------------------------------------------------------------
CFG = dict(crop_and_resize=True, default_image_size=512, downsampling_ratio=16, min_aspect_ratio=0.5, max_aspect_ratio=2.0)


def same_image_batch(tfm, count=2, seed=9):
    image = np.random.default_rng(seed).integers(0, 256, (300, 400, 3), dtype=np.uint8)
    b = tfm.batch([image] * count, flags=dg.BATCH_COLLATE)
    b.upload()
    b.run()
    return b


def test_a_bucket_of_a_closed_batch_is_refused():
    tfm = dg.Context(0, CFG)
    stem = tk.PatchStem(tfm, 16, MEAN, STD, rand((96, 768), F32, 1, 0.02), dtype=F32)
    b = same_image_batch(tfm)
    b.sync()
    array = b.buckets()[0]["array"]
    tokens = array.shape[1] * array.shape[2] // 256
    positions, dy = rand((tokens, 96), F32, 2), rand((2 * tokens, 96), F32, 3)
    saved = stem.forward(array, positions)[1]
    got = stem.backward(saved, dy)
    pixels = torch.as_tensor(array, device="cuda")
    assert same(stem.backward(stem.forward(pixels, positions)[1], dy), got)
    del pixels
    b.close()
    for call in (lambda: tk.patch_rows(tfm, array, 16, MEAN, STD), lambda: stem.forward(array, positions), lambda: stem.backward(saved, dy)):
        with pytest.raises(dg.DatagoB200Error, match="closed"):
            call()


def test_a_buckets_array_is_read_behind_its_batch_and_before_the_batch_goes():
    tfm, other = dg.Context(0, CFG), dg.Context(0)
    want = None
    for stream in (torch.cuda.Stream(), torch.cuda.default_stream(), torch.cuda.Stream()):
        with torch.cuda.stream(stream):
            for _ in range(4):
                b = same_image_batch(tfm)
                rows = tk.patch_rows(other, b.buckets()[0]["array"], 16, MEAN, STD, F32)  # without waiting for the batch
                b.close()
                same_image_batch(tfm, seed=10).close()  # another one in its place
                want = rows if want is None else want
                stream.synchronize()
                assert torch.equal(rows, want)
    b = same_image_batch(tfm)
    b.sync()
    assert torch.equal(tk.patch_rows(tfm, torch.as_tensor(b.buckets()[0]["array"], device="cuda"), 16, MEAN, STD, F32), want)
    torch.cuda.synchronize()
    b.close()


def test_a_buckets_array_can_be_read_in_a_graph():
    tfm = dg.Context(0, CFG)
    b = same_image_batch(tfm)
    b.sync()
    want = b.patch_rows(0, 16, MEAN, STD, F32)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        first, second = b.patch_rows(0, 16, MEAN, STD, F32), tk.patch_rows(tfm, b.buckets()[0]["array"], 16, MEAN, STD, F32)
    first.zero_()
    second.zero_()
    graph.replay()
    assert torch.equal(first, want) and torch.equal(second, want)
    torch.cuda.synchronize()
    b.close()
