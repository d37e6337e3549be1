"""What lies between a bucket of pixels and a transformer's first layer, as measurable cases.

A bucket is a dense uint8 [images, height, width, channels] array in device memory.  Its patches become rows in 8 bits
(e4m3 values, one power-of-two scale for each 128 features), the rows meet the patch-embedding weight in a product, and
the token rows get positions, dropout and a norm whose output is 8-bit rows again.  What a case's `op` names:

  patch     patches of a bucket, normalised per channel, as 8-bit rows
  columns   the transposed matrix as 8-bit rows: an operand whose contraction runs over the tokens
  product   8-bit rows times 8-bit rows: out[m, n] = sum over k of a[m, k] * b[n, k], scales included
  wgrad     the gradient of the product's weight: both operands as 8-bit rows along the tokens, then their product
  norm      h = x + positions; root-mean-square norm of h times a weight, as 8-bit rows
  backward  the norm's gradients: of x, of the positions (shared by all images) and of the weight
  dropout   Philox4x32-10 with the element's index as its counter; the same call on a gradient is the backward pass

Where `own` is false the operators run in their plain form, elementary torch operations in 32 bits.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
MEAN, STD = (0.48, 0.46, 0.41, 0.5), (0.27, 0.26, 0.28, 0.25)
GROUP = 128
EPS = 1e-6


def listed():
    return [
        # one photo in patches of 14 pixels: 588 features, no multiple of anything
        dict(name="patch_odd", op="patch", images=1, height=700, width=980, channels=3, patch=14),
        # a training batch of 1024-class images from one landscape bucket
        dict(name="patch_bucket", op="patch", images=48, height=896, width=1152, channels=3, patch=16),
        # token gradients of a ragged batch, for a product whose contraction runs over the tokens
        dict(name="columns_ragged", op="columns", rows=37003, cols=1000, dtype="bf16"),
        # a handful of tokens through the embedding: all latency
        dict(name="product_few", op="product", rows=7, inner=768, cols=1024, dtype="bf16"),
        # odd patches of a few images
        dict(name="product_odd", op="product", rows=9477, inner=588, cols=1000, dtype="f16"),
        # a training batch of 1024-class images: 32 images of 4096 tokens
        dict(name="product_batch", op="product", rows=131072, inner=768, cols=1152, dtype="bf16"),
        # the gradient of the embedding weight over the tokens of a batch
        dict(name="weight_gradient", op="wgrad", rows=57600, inner=768, cols=1152, dtype="bf16"),
        # the stem's norm for one token
        dict(name="norm_one", op="norm", images=1, tokens=1, cols=1152, dtype="bf16"),
        # positions added and normed for a training batch
        dict(name="norm_batch", op="norm", images=32, tokens=4096, cols=1152, dtype="bf16"),
        # its backward pass, positions shared by the images, a token grid that is no power of two
        dict(name="norm_backward", op="backward", images=24, tokens=2294, cols=1152, dtype="bf16"),
        # dropout of a training batch's token rows
        dict(name="dropout_batch", op="dropout", rows=131072, cols=1152, dtype="bf16", p=0.1, per_row=False, offset=0),
        # whole tokens dropped from a few images in 32 bits, late in a run's count
        dict(name="dropout_tokens", op="dropout", rows=1571, cols=777, dtype="f32", p=0.5, per_row=True, offset=(1 << 33) + 5),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("patch", "columns", "product", "product", "wgrad", "norm", "backward", "dropout"))
    if op == "patch":
        patch, channels = rng.choice((8, 14, 16, 20)), rng.choice((1, 3, 3, 4))
        images, height, width = _spread(rng, 1, 48), patch * _spread(rng, 4, 56), patch * _spread(rng, 4, 56)
        return dict(op=op, images=images, height=height, width=width, channels=channels, patch=patch)
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    if op == "product":
        return dict(op=op, rows=_spread(rng, 1, 131072), inner=_spread(rng, 64, 768), cols=_spread(rng, 48, 1152), dtype=dtype)
    if op == "wgrad":
        return dict(op=op, rows=_spread(rng, 100, 57600), inner=_spread(rng, 64, 768), cols=_spread(rng, 48, 1152), dtype=dtype)
    if op == "norm":
        return dict(op=op, images=_spread(rng, 1, 32), tokens=_spread(rng, 1, 2048), cols=_spread(rng, 48, 1152), dtype=dtype)
    if op == "backward":
        return dict(op=op, images=_spread(rng, 1, 24), tokens=_spread(rng, 1, 1147), cols=_spread(rng, 48, 1152), dtype=dtype)
    if op == "columns":
        return dict(op=op, rows=_spread(rng, 1, 37003), cols=_spread(rng, 48, 1152), dtype=dtype)
    return dict(op=op, rows=_spread(rng, 1, 65536), cols=_spread(rng, 48, 1152), dtype=dtype, p=rng.choice((0.0, 0.1, 0.25, 0.5, 0.9)),
                per_row=rng.random() < 0.3, offset=rng.choice((0, rng.randrange(1 << 20), rng.randrange(1 << 40))))


def work(case):
    op = case["op"]
    size = {"f32": 4, "bf16": 2, "f16": 2}.get(case.get("dtype"))
    if op == "patch":
        pixels = case["images"] * case["height"] * case["width"] * case["channels"]
        features = case["patch"] ** 2 * case["channels"]
        return {"bytes": 2 * pixels + pixels // features * -(-features // GROUP), "flops": 4 * pixels}
    if op == "columns":
        n = case["rows"] * case["cols"]
        return {"bytes": n * (size + 1) + case["cols"] * -(-case["rows"] // GROUP), "flops": 2 * n}
    if op == "product":
        m, k, n = case["rows"], case["inner"], case["cols"]
        return {"bytes": (m + n) * k + m * -(-k // GROUP) + m * n * size, "flops": 2 * m * n * k}
    if op == "wgrad":
        t, k, n = case["rows"], case["inner"], case["cols"]
        return {"bytes": t * (k + n) * size + n * k * 4, "flops": 2 * t * n * k}
    if op == "dropout":
        n = case["rows"] * case["cols"]
        return {"bytes": 2 * n * size, "flops": n}
    i, t, n = case["images"], case["tokens"], case["cols"]
    if op == "norm":
        return {"bytes": i * t * (n * (2 * size + 1) + -(-n // GROUP)) + t * n * size + n * size, "flops": 6 * i * t * n}
    return {"bytes": i * t * (n * 3 * size + 4) + t * n * 4 + n * (size + 4), "flops": 12 * i * t * n}


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _normal(shape, g, dtype, spread=1.0):
    """Activations: normal values, a few columns of them ten times as large."""
    x = torch.randn(shape, generator=g, device="cuda")
    loud = 1 + 9 * (torch.rand(shape[-1], generator=g, device="cuda") < 0.01)
    return (x * loud * spread).to(dtype)


def _pixels(case, g):
    """Images with an even background, a gradient across it, noise, and a saturated part."""
    n, h, w, c = case["images"], case["height"], case["width"], case["channels"]
    base = torch.rand((n, 1, 1, c), generator=g, device="cuda") * 200
    ramp = torch.linspace(0, 60, w, device="cuda").view(1, 1, w, 1)
    noise = torch.randn((n, h, w, c), generator=g, device="cuda") * 12
    return (base + ramp + noise).clamp_(0, 255).to(torch.uint8)


def _rows8(x, block=1):
    """A matrix as 8-bit rows: values, and scales of 128 features (of `block` rows).  Rows of values begin at multiples of
    128 bytes, rows of scales at multiples of 4."""
    rows, cols = x.shape
    padded = torch.zeros((-(-rows // block) * block, -(-cols // GROUP) * GROUP), device=x.device)
    padded[:rows, :cols] = x.float()
    groups = padded.view(-1, block, padded.shape[1] // GROUP, GROUP)
    mantissa, exponent = torch.frexp(groups.abs().amax(dim=(1, 3)))  # the mantissa is in [0.5, 1): 448 is 0.875 * 2^9
    e = exponent - 9 + 127 + (mantissa > 0.875).int()
    e = torch.where(mantissa == 0, torch.zeros_like(e), e.clamp(min=0))
    inverse = torch.ldexp(torch.ones_like(mantissa), 127 - e)
    values = (groups * inverse.view(inverse.shape[0], 1, -1, 1)).to(torch.float8_e4m3fn).view(padded.shape)[:rows, :cols]
    scales = torch.nn.functional.pad(e.to(torch.uint8), (0, -e.shape[1] % 4)).view(torch.float8_e8m0fnu)
    return values, scales[:, :e.shape[1]]


def _wide(values, scales, block=1):
    """What 8-bit rows stand for, in 32 bits."""
    factor = scales.float().repeat_interleave(block, 0)[:values.shape[0]].repeat_interleave(GROUP, 1)[:, :values.shape[1]]
    return values.float() * factor


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, dtype = case["op"], TYPES.get(case.get("dtype"))
    s = {"case": case, "ctx": _context()}
    if op == "patch":
        s["pixels"] = _pixels(case, g)
    elif op == "columns":
        s["x"] = _normal((case["rows"], case["cols"]), g, dtype, 1e-3)
    elif op == "product":
        s["a"] = _rows8(_normal((case["rows"], case["inner"]), g, dtype))
        s["b"] = _rows8(_normal((case["cols"], case["inner"]), g, torch.float32, 0.02), GROUP)
    elif op == "wgrad":
        s["x"] = _normal((case["rows"], case["inner"]), g, dtype)
        s["dy"] = _normal((case["rows"], case["cols"]), g, dtype, 1e-3)
    elif op in ("norm", "backward"):
        rows, cols = case["images"] * case["tokens"], case["cols"]
        s["weight"] = (1 + 0.1 * torch.randn(cols, generator=g, device="cuda")).to(dtype)
        if op == "norm":
            s["x"] = _normal((rows, cols), g, dtype)
            s["positions"] = _normal((case["tokens"], cols), g, dtype, 0.1)
        else:
            s["dy"] = _normal((rows, cols), g, dtype, 1e-3)
            s["h"] = _normal((rows, cols), g, dtype)
            s["rstd"] = torch.rsqrt(s["h"].double().square().mean(1) + EPS).float()
    else:
        s["x"] = _normal((case["rows"], case["cols"]), g, dtype)
        s["seed"] = int(torch.randint(0, 1 << 62, (), generator=g, device="cuda"))
    return s


def _context():
    """The handle that a program keeps for the device."""
    import datago_b200
    if not hasattr(_context, "kept"):
        _context.kept = datago_b200.Context(0)
    return _context.kept


# ---- one pass -------------------------------------------------------------------------------------------------------
def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    from datago_b200 import tokens as tk
    case, ctx, op = s["case"], s["ctx"], s["case"]["op"]
    if op == "patch":
        c = case["channels"]
        r = tk.patch_rows(ctx, s["pixels"], case["patch"], MEAN[:c], STD[:c])
        return r.values, r.scales
    if op == "columns":
        r = tk.quantize_rows(ctx, s["x"], transpose=True)
        return r.values, r.scales
    if op == "product":
        return tk.product(ctx, tk.Rows8(*s["a"]), tk.Rows8(*s["b"], block=GROUP), TYPES[case["dtype"]])
    if op == "wgrad":
        return tk.product(ctx, tk.quantize_rows(ctx, s["dy"], transpose=True), tk.quantize_rows(ctx, s["x"], transpose=True), torch.float32)
    if op == "norm":
        n = tk.rms_norm(ctx, s["x"], s["weight"], residual=s["positions"], eps=EPS, eight_bit=True)
        return n.y.values, n.y.scales, n.sum, n.rstd
    if op == "backward":
        return tk.rms_norm_backward(ctx, s["dy"], s["h"], s["rstd"], s["weight"], residual_rows=case["tokens"])
    return tk.dropout(ctx, s["x"], case["p"], s["seed"], case["offset"], per_row=case["per_row"])


def _patches(pixels, p):
    n, h, w, c = pixels.shape
    return pixels.view(n, h // p, p, w // p, p, c).permute(0, 1, 3, 2, 4, 5).reshape(-1, p * p * c)


def _plain(s):
    case, op = s["case"], s["case"]["op"]
    dtype = TYPES.get(case.get("dtype"))
    if op == "patch":
        p, c = case["patch"], case["channels"]
        mean, std = (torch.tensor(v[:c], device="cuda").repeat(p * p) for v in (MEAN, STD))
        return _rows8((_patches(s["pixels"], p).float() / 255 - mean) / std)
    if op == "columns":
        return _rows8(s["x"].t())
    if op == "product":
        return (_wide(*s["a"]) @ _wide(*s["b"], GROUP).t()).to(dtype)
    if op == "wgrad":  # in 64 bits: the sum runs over all tokens
        return (_wide(*_rows8(s["dy"].t())).double() @ _wide(*_rows8(s["x"].t())).double().t()).float()
    if op == "norm":
        h = (s["x"].float().view(case["images"], case["tokens"], -1) + s["positions"].float()).view(s["x"].shape)
        rstd = torch.rsqrt(h.square().mean(1) + EPS)
        return *_rows8(h * rstd[:, None] * s["weight"].float()), h.to(dtype), rstd
    if op == "backward":
        dy, hat = s["dy"].float(), s["h"].float() * s["rstd"][:, None]
        g = dy * s["weight"].float()
        dx = (g - hat * (g * hat).mean(1, keepdim=True)) * s["rstd"][:, None]
        return dx.to(dtype), dx.view(case["images"], case["tokens"], -1).sum(0), (dy * hat).sum(0)
    threshold = round(case["p"] * 65536)
    keep = _bits16(s["seed"], case["offset"], s["x"].shape[0] if case["per_row"] else s["x"].numel()) >= threshold
    keep = keep.view(-1, 1) if case["per_row"] else keep.view(s["x"].shape)
    return torch.where(keep, s["x"].float() * (65536 / (65536 - threshold)), 0.0).to(dtype)


def _bits16(seed, offset, count):
    """16 random bits for each index from `offset` on: eight of them from one Philox4x32-10 block (Salmon et al., 2011)."""
    first, mask = offset >> 3, 0xFFFFFFFF
    block = torch.arange(first, (offset + count + 7) >> 3, device="cuda")
    c0, c1, c2, c3 = block & mask, block >> 32, torch.zeros_like(block), torch.zeros_like(block)
    k0, k1 = seed & mask, seed >> 32
    for _ in range(10):
        u, v = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((v >> 32) & mask) ^ c1 ^ k0, v & mask, ((u >> 32) & mask) ^ c3 ^ k1, u & mask
        k0, k1 = (k0 + 0x9E3779B9) & mask, (k1 + 0xBB67AE85) & mask
    halves = torch.stack([h for c in (c0, c1, c2, c3) for h in (c & 0xFFFF, c >> 16)], 1).view(-1)
    return halves[offset - 8 * first:][:count]


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------
def _e4m3(v):
    """The nearest of e4m3's numbers (ties to the even one), for |v| <= 448."""
    exponent = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(exponent - 3)
    return torch.round(v / step) * step


def _quantised(x, rows=1):
    """Values and scales of a matrix in 64 bits, group by group of columns."""
    values, scales = [], []
    for part in x.split(GROUP, 1):
        top = part.abs().amax(1)
        if rows > 1:
            top = torch.stack([t.amax() for t in top.split(rows)])
        scale = torch.exp2(torch.ceil(torch.log2(top / 448)).clamp(min=-127))
        values.append(_e4m3(part / scale.repeat_interleave(rows)[:len(x), None]))
        scales.append(scale)
    return torch.cat(values, 1), torch.stack(scales, 1)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "patch":
        p, c = case["patch"], case["channels"]
        out = []
        for image in s["pixels"]:
            x = (image.double() / 255 - torch.tensor(MEAN[:c], device="cuda", dtype=torch.float64)) / torch.tensor(STD[:c], device="cuda", dtype=torch.float64)
            out.append(_quantised(torch.cat([band.unfold(1, p, p).permute(1, 0, 3, 2).flatten(1) for band in x.split(p)])))
        return tuple(torch.cat(v) for v in zip(*out))
    if op == "columns":
        return _quantised(s["x"].double().t())
    if op == "product":
        (a, ea), (b, eb) = s["a"], s["b"]
        out = 0.0
        for k in range(ea.shape[1]):
            part = slice(k * GROUP, (k + 1) * GROUP)
            scale = eb[:, k].double().repeat_interleave(GROUP)[:len(b)]
            out = out + (a[:, part].double() @ b[:, part].double().t()) * ea[:, k].double()[:, None] * scale
        return out
    if op == "wgrad":
        wide = [q.double() * e.double().repeat_interleave(GROUP, 1)[:, :q.shape[1]] for q, e in (_quantised(s[n].double().t()) for n in ("dy", "x"))]
        return wide[0] @ wide[1].t()
    if op == "norm":
        h = s["x"].double() + s["positions"].double().repeat(case["images"], 1)
        root = 1 / torch.sqrt((h * h).sum(1) / case["cols"] + EPS)
        return *_quantised(h * root[:, None] * s["weight"].double()), h, root
    if op == "backward":
        dy, h, w, r = s["dy"].double(), s["h"].double(), s["weight"].double(), s["rstd"].double()[:, None]
        along = (dy * w * h).sum(1, keepdim=True) / case["cols"]
        dx = r * dy * w - r ** 3 * h * along
        return dx, sum(dx.split(case["tokens"])), (dy * h * r).sum(0)
    threshold = int(case["p"] * 65536 + 0.5)
    x = s["x"].double() * (65536 / (65536 - threshold))
    index = torch.arange(len(x) if case["per_row"] else x.numel(), device="cuda") + case["offset"]
    low = _kept(s["seed"], index, threshold)
    return torch.where(low[:, None] if case["per_row"] else low.view(x.shape), x, 0.0)


def _kept(seed, index, threshold):
    """For each index, whether its 16 bits of the Philox block index >> 3 reach the threshold; the products in halves of 16 bits."""
    def mul(a, m):
        lo, hi = a * (m & 0xFFFF), a * (m >> 16)
        total = (lo >> 16) + hi
        return total >> 16, ((total & 0xFFFF) << 16) | (lo & 0xFFFF)
    word = [(index >> 3) & 0xFFFFFFFF, index >> 35, torch.zeros_like(index), torch.zeros_like(index)]
    for i in range(10):
        key = [(part + i * weyl) % (1 << 32) for part, weyl in ((seed % (1 << 32), 0x9E3779B9), (seed >> 32, 0xBB67AE85))]
        (h0, l0), (h1, l1) = mul(word[0], 0xD2511F53), mul(word[2], 0xCD9E8D57)
        word = [h1 ^ word[1] ^ key[0], l1, h0 ^ word[3] ^ key[1], l0]
    lane = index & 7
    chosen = sum(torch.where((lane >> 1) == i, w, 0) for i, w in enumerate(word))
    return ((chosen >> (16 * (lane & 1))) & 0xFFFF) >= threshold
