"""Token rows on the GPU: each operator against its definition in 64 bits, at the sizes and values where it can go wrong, and a run of
them together as a model's stem uses them.

Tolerances.  A rounding to bf16 is off by at most 2^-9 of the value's magnitude rounded up to a power of two, 2^-8 of the value; to f16 2^-11, or
half its smallest step, 2^-25; to f32 2^-24; to e4m3 2^-4, or half its smallest step, 2^-10 (of the scale).  A sum of n terms in 32 bits, in
any order, is off by at most n * 2^-24 of the sum of the magnitudes; tests of sums use that bound with the number of additions that
one value goes through."""
import math

import numpy as np
import pytest
import torch

import datago_b200 as dg
from datago_b200 import synth, tokens as tk

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HALF_STEP = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
TINY = {F32: 2.0 ** -150, BF16: 2.0 ** -134, F16: 2.0 ** -25}
CFG = dict(crop_and_resize=True, default_image_size=512, downsampling_ratio=16, min_aspect_ratio=0.5, max_aspect_ratio=2.0)
MEAN, STD = (0.48, 0.46, 0.41, 0.5), (0.27, 0.26, 0.28, 0.25)


@pytest.fixture(scope="module")
def ctx():
    return dg.Context(0)


def rand(shape, dtype, seed, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * spread).to(dtype)


def placed(x, lead, gap):
    """x's values at `lead` elements into a larger tensor, `gap` elements between rows; and that tensor, to see what lies around."""
    rows, cols = x.shape
    big = torch.full((lead + rows * (cols + gap) + 8,), 7.0, dtype=x.dtype, device="cuda")
    view = big[lead:lead + rows * (cols + gap)].view(rows, cols + gap)[:, :cols]
    view.copy_(x)
    return view, big


def untouched(view, big):
    mask = torch.ones_like(big, dtype=torch.bool)
    mask.as_strided(view.shape, view.stride(), view.storage_offset()).fill_(False)
    return bool((big[mask] == 7.0).all())


def close(got, want, bound, what=""):
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), (what, float((off - bound).max()), float(off.max()))


# ---- 8-bit rows -------------------------------------------------------------------------------------------------------
def e4m3(v):
    """The nearest e4m3 number, ties to even, of finite float64 |v| <= 448."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(v / step) * step


def rows8_of(x, block):
    """(values, scale exponents) of a float64 matrix by the definition; groups with something not finite are NaN and 255."""
    rows, cols = x.shape
    pad = torch.zeros(-(-rows // block) * block, -(-cols // 128) * 128, dtype=torch.float64, device=x.device)
    pad[:rows, :cols] = x
    groups = pad.view(-1, block, pad.shape[1] // 128, 128)
    top = groups.abs().amax((1, 3))
    bad = ~torch.isfinite(groups).all(3).all(1)
    e = (torch.ceil(torch.log2(torch.where(bad, 1.0, top) / 448)) + 127).clamp(min=0)  # 0 for a group of zeros
    q = e4m3(torch.where(bad[:, None, :, None], 0.0, groups) / torch.exp2(e - 127)[:, None, :, None])
    q = torch.where(bad[:, None, :, None], math.nan, q).view(pad.shape)[:rows, :cols]
    return q, torch.where(bad, 255.0, e)


def same_rows8(got, want, block):
    q, e = rows8_of(want, block)
    assert torch.equal(got.scales.view(torch.uint8).double(), e)
    v = got.values.double()
    assert torch.equal(torch.isnan(v), torch.isnan(q)) and torch.equal(torch.nan_to_num(v), torch.nan_to_num(q))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (3, 129), (130, 7), (257, 384), (128, 1000), (515, 72)])
@pytest.mark.parametrize("transpose,block", [(False, 1), (True, 1), (False, 128), (True, 128)])
def test_quantize_rows(ctx, dtype, rows, cols, transpose, block):
    x = rand((rows, cols), dtype, rows * cols + block)
    x[:, ::5] *= 100
    x[rows // 2] = 0
    want = x.double()
    for lead, gap in ((0, 0), (1, 3), (8, 8)):
        got = tk.quantize_rows(ctx, placed(x, lead, gap)[0], transpose=transpose, block=block)
        same_rows8(got, want.t() if transpose else want, block)


@pytest.mark.parametrize("transpose,block", [(False, 1), (True, 1), (False, 128), (True, 128)])
def test_quantize_rows_of_extremes(ctx, transpose, block):
    x = torch.zeros(300, 400, device="cuda")
    x[0, 0], x[0, 129], x[0, 300] = 448.0, 449.0, 2.0 ** -149            # the border of a scale; the smallest number there is
    x[1, 5], x[2, 6], x[3, 7], x[3, 8] = math.inf, -math.inf, math.nan, 1.0
    x[140, :] = torch.finfo(F32).max
    x[141, 128:256] = torch.linspace(-1, 1, 128, device="cuda") * 2.0 ** -120
    x[142, 256:384] = 1.0 + torch.arange(128, device="cuda") / 128.0      # every mantissa: ties too
    x[200, 399] = -2.0 ** -126
    same_rows8(tk.quantize_rows(ctx, x, transpose=transpose, block=block), x.double().t() if transpose else x.double(), block)


def test_quantize_rows_leaves_what_lies_behind_the_columns(ctx):
    x = rand((37, 200), BF16, 4)
    values = torch.full((37, 256), 3.0, device="cuda").to(torch.float8_e4m3fn)
    scales = torch.full((37, 8), 9, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)
    tk.quantize_rows(ctx, x, out=tk.Rows8(values[:, :200], scales[:, :2]))
    assert bool((values[:, 200:].float() == 3).all()) and bool((scales[:, 2:].view(torch.uint8) == 9).all())
    assert torch.equal(values[:, :200].float(), tk.quantize_rows(ctx, x).values.float())


def patches_of(pixels, p):
    """float64 rows, by the definition, one index at a time"""
    n, h, w, c = pixels.shape
    x = (pixels.double() / 255 - torch.tensor(MEAN[:c], dtype=torch.float64, device="cuda").float().double()) / torch.tensor(STD[:c], device="cuda").double()
    return torch.stack([x[i, Y:Y + p, X:X + p].reshape(-1) for i in range(n) for Y in range(0, h, p) for X in range(0, w, p)])


@pytest.mark.parametrize("channels", [1, 2, 3, 4])
@pytest.mark.parametrize("n,grid,p", [(1, (1, 1), 1), (2, (3, 5), 3), (3, (2, 7), 14), (2, (5, 4), 16), (1, (3, 3), 20), (1, (9, 2), 8), (2, (2, 90), 5), (1, (2, 1), 109)])
@pytest.mark.parametrize("lead", [0, 1, 8])
def test_patch_rows(ctx, channels, n, grid, p, lead):
    h, w = grid[0] * p, grid[1] * p
    g = torch.Generator(device="cuda").manual_seed(channels * 100 + p)
    big = torch.randint(0, 256, (lead + n * h * w * channels,), generator=g, device="cuda", dtype=torch.uint8)
    pixels = big[lead:].view(n, h, w, channels)
    want = patches_of(pixels, p)
    # pixel * gain + shift: the rounded gain and shift and the one rounding of the result
    off = 2.0 ** -24 * (1 / 0.25 + 0.5 / 0.25 + want.abs())
    got = tk.patch_rows(ctx, pixels, p, MEAN[:channels], STD[:channels], F32)
    close(got, want, off)
    for dtype in (BF16, F16):
        close(tk.patch_rows(ctx, pixels, p, MEAN[:channels], STD[:channels], dtype), want, off + HALF_STEP[dtype] * (want.abs() + off) + TINY[dtype])
    got8 = tk.patch_rows(ctx, pixels, p, MEAN[:channels], STD[:channels])
    same_rows8(got8, got.double(), 1)


def test_patch_rows_into_rows_further_apart(ctx):
    pixels = torch.randint(0, 256, (2, 28, 42, 3), device="cuda", dtype=torch.uint8)
    want = tk.patch_rows(ctx, pixels, 14, MEAN[:3], STD[:3], BF16)
    view, big = placed(torch.zeros_like(want), 3, 5)
    tk.patch_rows(ctx, pixels, 14, MEAN[:3], STD[:3], BF16, out=view)
    assert torch.equal(view, want) and untouched(view, big)


# ---- product -----------------------------------------------------------------------------------------------------------
def operand(ctx, rows, cols, block, seed, spread=1.0):
    x = rand((rows, cols), F32, seed, spread)
    x[:, ::7] *= 30
    return tk.quantize_rows(ctx, x, block=block)


def check_product(ctx, a, b, dtype, out=None):
    got = tk.product(ctx, a, b, dtype, out=out)
    wa, wb = a.to_float().double(), b.to_float().double()
    want, size = wa @ wb.t(), wa.abs() @ wb.abs().t()
    # The products are exact (4 by 4 significant bits).  32 of them are added to the sum at a time: 33 addends, each of which may lose what is
    # below 2^-23 of the largest, which is at most the sum of the magnitudes; parts of a split contraction are added once more.
    steps = -(-a.shape[1] // 32) + 148
    off = steps * 33 * 2.0 ** -23 * size
    most = torch.finfo(dtype).max * (1 + HALF_STEP[dtype] / 2)  # from here on the nearest value of the type is an infinity
    over, near = want.abs() - off >= most, want.abs() + off >= most
    assert torch.equal(torch.where(over, got.double(), 0.0), torch.where(over, want.sign() * math.inf, 0.0))
    close(torch.where(near, 0.0, got.double()), torch.where(near, 0.0, want), off + HALF_STEP[dtype] * (want.abs() + off) + TINY[dtype], (a.shape, b.shape))
    return got


@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 48, 64), (7, 1024, 768), (128, 128, 128), (129, 16, 32), (127, 17, 33), (77, 200, 300), (300, 241, 513), (200, 480, 1152), (5, 300, 4096),
                                   (1000, 96, 96), (64, 64, 20000)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_product(ctx, m, n, k, dtype):
    check_product(ctx, operand(ctx, m, k, 1, m + k), operand(ctx, n, k, 128, n + k, 0.05), dtype)


@pytest.mark.parametrize("a_block,b_block", [(1, 1), (128, 1), (128, 128)])
def test_product_of_every_kind_of_scales(ctx, a_block, b_block):
    check_product(ctx, operand(ctx, 333, 700, a_block, 1), operand(ctx, 500, 700, b_block, 2), F32)
    check_product(ctx, operand(ctx, 130, 5000, a_block, 3), operand(ctx, 140, 5000, b_block, 4), F32)


@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (33, 47, 130), (130, 200, 300), (257, 520, 1000), (1152, 768, 5000), (300, 96, 40)])
@pytest.mark.parametrize("a_turned,b_turned", [(True, True), (True, False), (False, True)])
@pytest.mark.parametrize("block", [1, 128])
def test_product_of_transposed_operands(ctx, m, n, k, a_turned, b_turned, block):
    def operand_of(rows, seed, turned):
        x = rand((k, rows) if turned else (rows, k), F32, seed)
        return tk.quantize_rows(ctx, placed(x, 3, 5)[0], transpose=turned, block=block)
    check_product(ctx, operand_of(m, 1, a_turned), operand_of(n, 2, b_turned), F32)


def test_product_of_more_tiles_than_the_chip_holds(ctx):
    check_product(ctx, operand(ctx, 20001, 200, 1, 5), operand(ctx, 1000, 200, 128, 6), BF16)


def test_product_whose_last_tiles_are_partly_outside(ctx):
    # a warp without rows in a tile follows, in the same CTA, one that has just sent its rows out
    for m, n, k in ((20001, 1000, 200), (20033, 104, 300), (19000, 1000, 128)):
        a, b = operand(ctx, m, k, 1, 15), operand(ctx, n, k, 128, 16)
        first = check_product(ctx, a, b, BF16)
        for _ in range(20):
            assert torch.equal(tk.product(ctx, a, b, BF16), first)


@pytest.mark.parametrize("dtype,lead,gap", [(BF16, 1, 3), (F32, 4, 4), (F16, 8, 16), (F32, 1, 0)])
def test_product_into_rows_of_any_distance(ctx, dtype, lead, gap):
    for m, n, k in ((200, 250, 384), (70, 33, 9000)):
        a, b = operand(ctx, m, k, 1, 7), operand(ctx, n, k, 1, 8)
        view, big = placed(torch.zeros((m, n), dtype=dtype, device="cuda"), lead, gap)
        check_product(ctx, a, b, dtype, out=view)
        assert untouched(view, big)


def test_new_matrices_have_rows_that_begin_at_16_bytes(ctx):
    a, b = operand(ctx, 50, 200, 1, 17), operand(ctx, 33, 200, 1, 18)
    for dtype in (F32, BF16, F16):
        got = tk.product(ctx, a, b, dtype)
        n = tk.rms_norm(ctx, got)
        dx = tk.rms_norm_backward(ctx, n.y, n.sum, n.rstd)[0]
        assert all(x.stride(0) * x.element_size() % 16 == 0 and x.shape == (50, 33) for x in (n.y, n.sum, dx))
        assert tk.dropout(ctx, got.contiguous(), 0.5, 1).is_contiguous()
        assert got.shape == (50, 33) and got.stride(1) == 1 and got.stride(0) * got.element_size() % 16 == 0 and got.data_ptr() % 16 == 0
        dense = tk.product(ctx, a, b, dtype, out=torch.empty(50, 33, dtype=dtype, device="cuda"))
        assert dense.is_contiguous() and torch.equal(dense, got)


def test_product_ignores_what_lies_behind_the_columns(ctx):
    x = operand(ctx, 40, 200, 1, 9)
    b = operand(ctx, 30, 200, 1, 10)
    want = check_product(ctx, x, b, F32)
    for r in (x, b):
        base = torch.full((r.shape[0], 256), math.nan, device="cuda").to(torch.float8_e4m3fn)
        scales = torch.full((r.shape[0], 8), 255, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)
        base[:, :200].copy_(r.values)
        scales.view(torch.uint8)[:, :2].copy_(r.scales.view(torch.uint8))
        r.values, r.scales = base[:, :200], scales[:, :2]
    assert torch.equal(tk.product(ctx, x, b, F32), want)


def test_product_keeps_nan_in_its_row_and_group(ctx):
    x, w = rand((150, 512), F32, 11), rand((40, 512), F32, 12)
    x[3, 200] = math.nan      # the group 1 of row 3 becomes NaN
    w[17, 5] = math.inf
    got = tk.product(ctx, tk.quantize_rows(ctx, x), tk.quantize_rows(ctx, w), F32)
    nan = torch.isnan(got)
    assert bool(nan[3].all()) and bool(nan[:, 17].all())
    nan[3], nan[:, 17] = False, False
    assert not bool(nan.any())


def test_product_over_all_scales(ctx):
    x = torch.ones(200, 128, device="cuda") * torch.exp2(torch.arange(200, device="cuda") - 100.0)[:, None]
    w = torch.ones(16, 128, device="cuda") * torch.exp2(torch.arange(16, device="cuda") * 4 - 32.0)[:, None]
    got = tk.product(ctx, tk.quantize_rows(ctx, x), tk.quantize_rows(ctx, w), F32)
    want = 128 * x[:, :1].double() * w[:, 0].double()
    assert torch.equal(got, want.float())  # a power of two, or an infinity beyond 2^128


def test_product_gives_the_same_sums_twice(ctx):
    a, b = operand(ctx, 300, 30000, 1, 13), operand(ctx, 200, 30000, 1, 14)
    assert torch.equal(tk.product(ctx, a, b, F32), tk.product(ctx, a, b, F32))
    tk.product_status(ctx)


# ---- norm --------------------------------------------------------------------------------------------------------------
def norm_of(x, residual, weight, eps):
    h = x.double()
    if residual is not None:
        h = h + residual.double().repeat(len(x) // len(residual), 1)
    rstd = 1 / torch.sqrt(h.square().mean(1) + eps)
    return h, rstd, h * rstd[:, None] * (1.0 if weight is None else weight.double())


NORM_SIZES = [(1, 1, 1), (1, 1, 1152), (3, 5, 9), (2, 7, 255), (2, 3, 520), (2, 4, 800), (1, 9, 1280), (2, 3, 1500), (1, 4, 2048), (2, 2, 3000), (2, 3, 5000), (1, 3, 8000), (1, 2, 16384)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("images,tokens,cols", NORM_SIZES)
def test_rms_norm(ctx, dtype, images, tokens, cols):
    x, r = rand((images * tokens, cols), dtype, cols), rand((tokens, cols), dtype, cols + 1, 0.1)
    for weight, residual, lead, gap in ((None, None, 0, 0), (rand((cols,), F32, 3), r, 0, 0), (rand((cols,), dtype, 4), placed(r, 3, 1)[0], 1, 5)):
        h, rstd, y = norm_of(x, residual, weight, 1e-6)
        x_at = placed(x, lead, gap)[0]
        got = tk.rms_norm(ctx, x_at, weight, residual=residual)
        close(got.sum, h, HALF_STEP[dtype] * (h.abs() + TINY[F32]) + 2.0 ** -24 * h.abs() + TINY[dtype])
        # the sum: 2 * 2^-24 per square (h and its square), at most 64 + 14 additions of positive terms, the mean, the root (halved), the reciprocal
        rel = (0.5 * (3 + 78 + 3) + 3) * 2.0 ** -24
        close(got.rstd, rstd, rel * rstd)
        off = (rel + 4 * 2.0 ** -24) * y.abs()
        close(got.y, y, off + HALF_STEP[dtype] * (y.abs() + off) + TINY[dtype])
        got8 = tk.rms_norm(ctx, x_at, weight, residual=residual, eight_bit=True)
        assert torch.equal(got8.sum, got.sum) and torch.equal(got8.rstd, got.rstd)
        s = torch.exp2(got8.y.scales.view(torch.uint8).double() - 127).repeat_interleave(128, 1)[:, :cols]
        top = torch.stack([part.abs().amax(1) for part in y.split(128, 1)], 1).repeat_interleave(128, 1)[:, :cols]
        assert bool((top <= 448 * s * (1 + 1e-5)).all()) and bool((top >= 224 * s * (1 - 1e-5))[s > 2.0 ** -127].all())
        close(got8.y.values.double() * s, y, off + 2.0 ** -4 * (y.abs() + off) + 2.0 ** -10 * s)


def test_rms_norm_in_place_and_of_a_strided_sum(ctx):
    x, r = rand((12, 300), BF16, 20), rand((4, 300), BF16, 21)
    want = tk.rms_norm(ctx, x, None, residual=r, eight_bit=True)
    view, big = placed(x, 5, 7)
    got = tk.rms_norm(ctx, view, None, residual=r, eight_bit=True, sum_out=view)
    assert torch.equal(view, want.sum) and untouched(view, big)
    assert torch.equal(got.y.values.float(), want.y.values.float())


def test_rms_norm_of_rows_that_are_not_finite_or_zero(ctx):
    x = rand((5, 200), F32, 22)
    x[1, 3], x[2, 4], x[3] = math.nan, math.inf, 0.0
    n = tk.rms_norm(ctx, x, eight_bit=True)
    s = n.y.scales.view(torch.uint8)
    assert bool((s[1] == 255).all()) and s[2, 0] == 255      # inf * 0 is NaN; the other group of that row is zeros
    assert bool((n.y.values[3].float() == 0).all()) and bool((s[3] == 0).all())
    clean = tk.rms_norm(ctx, x[[0, 4]], eight_bit=True)
    assert torch.equal(n.y.values[[0, 4]].float(), clean.y.values.float())


def backward_of(dy, h, rstd, weight, dsum, period):
    dy, h, r = dy.double(), h.double(), rstd.double()[:, None]
    g = dy if weight is None else dy * weight.double()
    hat = h * r
    dx = r * (g - hat * (g * hat).mean(1, keepdim=True))
    size = r * (g.abs() + hat.abs() * (g * hat).abs().mean(1, keepdim=True))
    if dsum is not None:
        dx, size = dx + dsum.double(), size + dsum.double().abs()
    return dx, size, dx.view(-1, period, dx.shape[1]).sum(0), size.view(-1, period, dx.shape[1]).sum(0), (dy * hat).sum(0), (dy * hat).abs().sum(0)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("images,tokens,cols", NORM_SIZES + [(5000, 1, 33), (700, 3, 1000), (2, 3000, 64), (1, 700, 1152)])
def test_rms_norm_backward(ctx, dtype, images, tokens, cols):
    rows = images * tokens
    dy, h, w = rand((rows, cols), dtype, 30), rand((rows, cols), dtype, 31), rand((cols,), dtype, 32)
    rstd = torch.rsqrt(h.double().square().mean(1) + 1e-6).float()
    for weight, dsum, lead, gap in ((None, None, 0, 0), (w, rand((rows, cols), dtype, 33), 3, 1)):
        dx, size, dr, dr_size, dw, dw_size = backward_of(dy, h, rstd, weight, dsum, tokens)
        at = [placed(t, lead, gap)[0] for t in (dy, h)]
        got = tk.rms_norm_backward(ctx, *at, rstd, weight, dsum, residual_rows=tokens)
        # the mean goes through at most 64 + 14 additions; a handful of products around it
        off = 90 * 2.0 ** -24 * size
        close(got[0], dx, off + HALF_STEP[dtype] * (dx.abs() + off) + TINY[dtype], "dx")
        close(got[1], dr, (90 + images) * 2.0 ** -24 * dr_size + TINY[F32], "dresidual")
        close(got[2], dw, (4 + rows + 300) * 2.0 ** -24 * dw_size + TINY[F32], "dweight")
        without = tk.rms_norm_backward(ctx, *at, rstd, weight, dsum)  # in the same places: rows elsewhere may be added up in another order
        assert without[1] is None and torch.equal(without[0], got[0])


def test_rms_norm_backward_is_the_slope(ctx):
    rows, tokens, cols = 6, 3, 40
    x, r, w, dy = (rand(s, F32, 40 + i) for i, s in enumerate(((rows, cols), (tokens, cols), (cols,), (rows, cols))))
    n = tk.rms_norm(ctx, x, w, residual=r)
    dx, dr, dw = tk.rms_norm_backward(ctx, dy, n.sum, n.rstd, w, residual_rows=tokens)
    loss = lambda x, r, w: float((norm_of(x, r, w, 1e-6)[2] * dy.double()).sum())  # noqa: E731
    rng = np.random.default_rng(0)
    for which, grad in ((0, dx), (1, dr), (2, dw)):
        for _ in range(8):
            at = tuple(int(rng.integers(s)) for s in grad.shape)
            ends = []
            for step in (2.0 ** -20, -2.0 ** -20):
                args = [x.double(), r.double(), w.double()]
                args[which][at] += step
                ends.append(loss(*args))
            # the third derivative's share of a step of 2^-20 and the roundings of two sums of 240 terms in 64 bits, far below 1e-5
            assert abs((ends[0] - ends[1]) * 2.0 ** 19 - float(grad[at])) < 1e-5 * (1 + abs(float(grad[at])))


def test_rms_norm_backward_in_place(ctx):
    dy, h, dsum = rand((50, 300), BF16, 50), rand((50, 300), BF16, 51), rand((50, 300), BF16, 52)
    rstd = torch.rsqrt(h.float().square().mean(1))
    want = tk.rms_norm_backward(ctx, dy, h, rstd, None, dsum, residual_rows=10)
    for target in ("dy", "dsum"):
        a, s = dy.clone(), dsum.clone()
        got = tk.rms_norm_backward(ctx, a, h, rstd, None, s, residual_rows=10, dx_out=a if target == "dy" else s)
        assert all(torch.equal(g, t) for g, t in zip(got, want))


def test_rows_that_are_none(ctx):
    empty = torch.empty(0, 256, dtype=BF16, device="cuda")
    assert tk.quantize_rows(ctx, empty).shape == (0, 256)
    assert tk.rms_norm(ctx, empty, residual=torch.ones(3, 256, dtype=BF16, device="cuda")).y.shape == (0, 256)
    assert tk.dropout(ctx, empty, 0.5, 1).shape == (0, 256)
    assert tk.product(ctx, tk.quantize_rows(ctx, empty), operand(ctx, 5, 256, 1, 1)).shape == (0, 5)
    dx, dr, dw = tk.rms_norm_backward(ctx, empty, empty, torch.empty(0, device="cuda"), residual_rows=3)
    assert dx.shape == (0, 256) and not bool(dr.any()) and not bool(dw.any()) and dr.shape == (3, 256)


# ---- dropout -----------------------------------------------------------------------------------------------------------
def philox(counter, seed):
    """One block of Philox4x32-10, in whole numbers (the paper's round function)."""
    c, k = [counter & 0xFFFFFFFF, counter >> 32, 0, 0], [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        u, v = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(v >> 32) ^ c[1] ^ k[0], v & 0xFFFFFFFF, (u >> 32) ^ c[3] ^ k[1], u & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def kept(seed, first, count, threshold):
    out = []
    for i in range(first, first + count):
        half = philox(i >> 3, seed)[(i & 7) >> 1] >> (16 * (i & 1)) & 0xFFFF
        out.append(half >= threshold)
    return torch.tensor(out, device="cuda")


def test_the_generator_is_the_published_one():
    # known answers of the paper's authors for counters and keys of zeros and of ones
    assert philox(0, 0) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,cols,lead,gap", [(1, 1, 0, 0), (3, 8, 0, 0), (5, 77, 0, 0), (5, 77, 1, 2), (9, 64, 8, 8), (2, 500, 0, 4)])
@pytest.mark.parametrize("p,seed,offset,per_row", [(0.1, 1, 0, False), (0.5, (1 << 64) - 3, (1 << 35) + 5, False), (0.75, 12345678901234, 3, True), (0.0, 0, 0, False),
                                                   (65535 / 65536, 7, (1 << 63) + 9, True)])
def test_dropout(ctx, dtype, rows, cols, lead, gap, p, seed, offset, per_row):
    x = rand((rows, cols), dtype, 60)
    x[0, 0] = math.nan
    t = int(p * 65536 + 0.5)
    mask = kept(seed, offset, rows if per_row else rows * cols, t)
    mask = mask.view(-1, 1).expand(rows, cols) if per_row else mask.view(rows, cols)
    at, big = placed(x, lead, gap)
    got = tk.dropout(ctx, at, p, seed, offset, per_row=per_row)
    want = torch.where(mask, x.double() * (65536 / (65536 - t)), 0.0)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    want = torch.nan_to_num(want)
    # the factor and the product are rounded to 32 bits, the result to its type
    off = 2 * 2.0 ** -24 * want.abs()
    close(torch.nan_to_num(got, nan=0.0), want, off + HALF_STEP[dtype] * (want.abs() + off) + TINY[dtype])
    tk.dropout(ctx, at, p, seed, offset, per_row=per_row, out=at)  # in place
    assert torch.equal(torch.nan_to_num(at), torch.nan_to_num(got)) and untouched(at, big)


def test_dropout_of_parts_is_dropout_of_the_whole(ctx):
    x = torch.ones(64, 1000, device="cuda")
    whole = tk.dropout(ctx, x, 0.3, 99, 5)
    for first in (1, 7, 40):
        assert torch.equal(tk.dropout(ctx, x[first:], 0.3, 99, 5 + first * 1000), whole[first:])
    share = float((tk.dropout(ctx, torch.ones(1 << 12, 1 << 12, device="cuda", dtype=BF16), 0.3, 4) == 0).float().mean())
    assert abs(share - 0.3) < 6 * math.sqrt(0.21 / 2 ** 24)


# ---- together ----------------------------------------------------------------------------------------------------------
def stem_of(stem, weight, pixels, positions, norm_weight, offset):
    """The stem in 64 bits from its 8-bit operands on."""
    x = tk.patch_rows(stem.ctx, pixels, stem.patch, stem.mean, stem.std).to_float().double() @ stem.weight8.to_float().double().t()
    t = int(stem.p * 65536 + 0.5)
    mask = kept(stem.seed, offset, x.numel(), t).view(x.shape) * (65536 / (65536 - t))
    h, rstd, y = norm_of(x * mask, positions, norm_weight, stem.eps)
    return mask, h, rstd, y


def make_stem(ctx, dtype=F32, width=96, channels=3, patch=14, p=0.25):
    weight = rand((width, patch * patch * channels), F32, 70, 0.02)
    norm_weight = rand((width,), F32, 71)
    return tk.PatchStem(ctx, patch, MEAN[:channels], STD[:channels], weight, norm_weight, p=p, seed=5, dtype=dtype), weight, norm_weight


def test_stem_and_its_gradients(ctx):
    stem, weight, norm_weight = make_stem(ctx)
    pixels = torch.randint(0, 256, (3, 42, 28, 3), device="cuda", dtype=torch.uint8)
    positions = rand((6, 96), F32, 72, 0.1)
    norm, saved = stem.forward(pixels, positions, offset=1000)
    mask, h, rstd, y = stem_of(stem, weight, pixels, positions, norm_weight, 1000)
    close(norm.sum, h, 1e-4 * h.abs().max())
    # 8-bit output: half a step of e4m3 on top of what 32-bit sums of 588 terms lose
    close(norm.y.to_float(), y, 2.0 ** -4 * y.abs() + 2.0 ** -9 * y.abs().amax() + 1e-4)
    dy = rand(norm.sum.shape, F32, 73, 1e-2)
    dweight, dpositions, dnorm = stem.backward(saved, dy)
    dx, _, dr, _, dw, _ = backward_of(dy, norm.sum, norm.rstd, norm_weight, None, 6)
    close(dpositions, dr, 1e-4 * dr.abs().max())
    close(dnorm, dw, 1e-4 * dw.abs().max())
    x8 = tk.quantize_rows(ctx, tk.patch_rows(ctx, pixels, 14, stem.mean, stem.std, F32), transpose=True).to_float().double()
    dx8 = tk.quantize_rows(ctx, (dx * mask).float(), transpose=True).to_float().double()
    # an element at the border of two e4m3 numbers may go the other way: a step of one of 18 rows
    close(dweight, dx8 @ x8.t(), 2.0 ** -3 * (dx8.abs().amax(1, keepdim=True) * x8.abs().amax(1)[None]))
    assert float((dweight.double() - dx8 @ x8.t()).norm() / (dx8 @ x8.t()).norm()) < 1e-2


def test_stem_reads_the_buckets_of_a_batch():
    tfm = dg.Context(0, CFG)
    rng = np.random.default_rng(8)
    jpegs = [synth.encode_jpeg(synth.natural_image(rng, w, h, 4.0, True), 90, "4:2:0", 0) for w, h in ((640, 480), (650, 470), (300, 500))]
    with tfm.batch(jpegs, flags=dg.BATCH_COLLATE) as b:
        b.upload()
        b.run()
        rows = [b.patch_rows(k, 16, MEAN[:3], STD[:3], F32) for k in range(len(b.buckets()))]  # without waiting for the batch
        outs = b.download()
        b.sync()
        buckets = b.buckets()
    assert sorted(i for k in buckets for i in k["items"]) == [0, 1, 2]
    for bucket, got in zip(buckets, rows):
        pixels = torch.from_numpy(np.stack([outs[i] for i in bucket["items"]])).cuda()
        assert torch.equal(got, tk.patch_rows(tfm, pixels, 16, MEAN[:3], STD[:3], F32))
    with pytest.raises(dg.DatagoB200Error):
        b.patch_rows(0, 16, MEAN[:3], STD[:3])


def test_a_batch_on_the_current_stream_hands_its_buckets_over():
    rng = np.random.default_rng(9)
    img = rng.integers(0, 256, (300, 400, 3), dtype=np.uint8)
    for stream in (torch.cuda.Stream(), torch.cuda.default_stream()):
        tfm = dg.Context(0, CFG, stream=stream.cuda_stream)
        with torch.cuda.stream(stream):
            with tfm.batch([img, img], flags=dg.BATCH_COLLATE) as b:
                b.upload()
                b.run()
                rows = b.patch_rows(0, 16, MEAN[:3], STD[:3])
                outs = b.download()
                b.sync()
            want = tk.patch_rows(tfm, torch.from_numpy(np.stack(outs)).cuda(), 16, MEAN[:3], STD[:3])
            assert torch.equal(rows.values.view(torch.uint8), want.values.view(torch.uint8))


def test_the_status_of_products_is_not_asked_for_inside_a_capture(ctx):
    a, b = operand(ctx, 40, 256, 1, 97), operand(ctx, 30, 256, 1, 98)
    want = tk.product(ctx, a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = tk.product(ctx, a, b)
        with pytest.raises(dg.DatagoB200Error):
            tk.product_status(ctx)
    graph.replay()
    assert torch.equal(got, want)
    tk.product_status(ctx)


def test_indices_beyond_32_bits(ctx):
    # 4.6 G elements, 9.2 GB: the last rows of a large matrix are those of the rows alone
    rows, cols, tail = 70001, 65536, 5
    x = torch.full((rows, cols), 1.5, dtype=BF16, device="cuda")
    x[-tail:] = rand((tail, cols), BF16, 99)
    whole = tk.dropout(ctx, x, 0.25, 3, 7)
    assert torch.equal(whole[-tail:], tk.dropout(ctx, x[-tail:], 0.25, 3, 7 + (rows - tail) * cols))
    q = tk.quantize_rows(ctx, x)
    same_rows8(tk.Rows8(q.values[-tail:], q.scales[-tail:]), x[-tail:].double(), 1)
    del whole, q
    narrow = x.view(-1, 1024)  # 4.48 M rows
    last = tk.rms_norm(ctx, narrow, residual=narrow[:1])
    alone = tk.rms_norm(ctx, narrow[-200:], residual=narrow[:1])
    assert torch.equal(last.y[-200:], alone.y) and torch.equal(last.sum[-200:], alone.sum) and torch.equal(last.rstd[-200:], alone.rstd)
    a = tk.quantize_rows(ctx, narrow[:, :128])
    del last, x, narrow
    b = operand(ctx, 640, 128, 128, 3)
    out = tk.product(ctx, a, b)  # 2.87 G elements
    part = tk.Rows8(a.values[-300:], a.scales[-300:])
    assert torch.equal(out[-300:], tk.product(ctx, part, b))
    tk.product_status(ctx)


def test_a_captured_stem_replays_on_new_inputs(ctx):
    stem, weight, norm_weight = make_stem(ctx, BF16, width=200)
    pixels = torch.randint(0, 256, (2, 42, 28, 3), device="cuda", dtype=torch.uint8)
    positions, dy = rand((6, 200), BF16, 80, 0.1), rand((12, 200), BF16, 81, 1e-2)
    stem.backward(stem.forward(pixels, positions, 8)[1], dy)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm, saved = stem.forward(pixels, positions, 8)
        grads = stem.backward(saved, dy)
    for seed in (1, 2):
        g = torch.Generator(device="cuda").manual_seed(seed)
        pixels.copy_(torch.randint(0, 256, pixels.shape, generator=g, device="cuda", dtype=torch.uint8))
        graph.replay()
        want, wsaved = stem.forward(pixels, positions, 8)
        wgrads = stem.backward(wsaved, dy)
        assert torch.equal(norm.y.values.float(), want.y.values.float()) and torch.equal(norm.sum, want.sum)
        assert all(torch.equal(a, b) for a, b in zip(grads, wgrads))


def test_two_streams_at_once(ctx):
    a, b = operand(ctx, 100, 20000, 1, 90), operand(ctx, 120, 20000, 1, 91)
    dy, h = rand((4000, 512), BF16, 92), rand((4000, 512), BF16, 93)
    rstd = torch.rsqrt(h.float().square().mean(1))
    want = tk.product(ctx, a, b, F32), tk.rms_norm_backward(ctx, dy, h, rstd, residual_rows=40)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append((tk.product(ctx, a, b, F32), tk.rms_norm_backward(ctx, dy, h, rstd, residual_rows=40)))
    torch.cuda.synchronize()
    for p, grads in got:
        assert torch.equal(p, want[0]) and all(torch.equal(x, y) for x, y in zip(grads, want[1]))


def test_the_stream_of_the_context_is_used_without_one():
    x = rand((300, 256), F32, 95)
    torch.cuda.synchronize()
    own = dg.Context(0)
    src = tk._matrix(own, x, "x")
    out = tk.Rows8.empty(300, 256, "cuda")
    assert tk.lib().dg_quantize_rows(own._h, None, src, tk._rows8(own, out, "out")) == 0
    torch.cuda.ExternalStream(own.stream).synchronize()
    same_rows8(out, x.double(), 1)


def test_refusals_leave_the_device_usable(ctx):
    x = rand((8, 256), BF16, 96)
    for call in (lambda: tk.dropout(ctx, x, 1.0, 1), lambda: tk.dropout(ctx, x, 0.1, -1), lambda: tk.rms_norm(ctx, x, residual=x[:3]), lambda: tk.quantize_rows(ctx, x, block=64),
                 lambda: tk.quantize_rows(ctx, x.t()), lambda: tk.product(ctx, tk.quantize_rows(ctx, x), tk.quantize_rows(ctx, x[:, :128])), lambda: tk.rms_norm(ctx, x.double()),
                 lambda: tk.product(ctx, x, x), lambda: tk.patch_rows(ctx, x, 16, MEAN, STD), lambda: tk.rms_norm(ctx, x, weight=x[0, :100])):
        with pytest.raises(dg.DatagoB200Error):
            call()
    assert torch.equal(tk.dropout(ctx, x, 0.0, 1), x)


@pytest.mark.parametrize("channels", [0, 5])
def test_pixels_of_other_channels_are_refused(ctx, channels):
    pixels = torch.zeros(1, 16, 16, channels, dtype=torch.uint8, device="cuda")
    with pytest.raises(dg.DatagoB200Error):
        tk.patch_rows(ctx, pixels, 16, (0.5,) * channels, (0.5,) * channels)
