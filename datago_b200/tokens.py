"""Token rows: from a bucket of pixels to what a transformer's first layer reads (the dg_patch_rows ... dg_dropout part of
include/datago_b200.h), on torch tensors.

Every function takes the Context of the tensors' device first, launches on torch's current stream of that device and returns
without waiting; nothing is kept between calls, so calls can be captured into CUDA graphs.  Results are new tensors unless `out` is given; the
rows of new ones (dropout's apart) begin at multiples of 16 bytes, so those whose rows are no multiple of that long are not contiguous (a product of
124515 x 685 over 768 columns in bfloat16 takes 87 us, into contiguous rows 170).  Matrices are 2-d tensors of float32, bfloat16 or float16 whose columns
are neighbours in memory; their rows, those of `out` too, may be any distance apart.
Gradients are calls of their own (rms_norm_backward, dropout on the gradient, product on operands quantised along the contraction);
PatchStem puts them together for the stem of a model.  Autograd knows nothing of these calls: while it records, tensors that require a gradient are
refused (detach() them, or call under no_grad()), and what is written into a caller's tensor counts as a change in place.
"""
import ctypes as C
import struct

import torch

from . import Batch, DatagoB200Error, DeviceArray, _check, lib as _library

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_LEGACY_STREAM = 1  # cudaStreamLegacy: torch's default stream, which has no handle of its own
GROUP = 128         # columns that share a scale


# dg_matrix and dg_rows8 of the header as bytes, whose address ctypes passes on: a call makes up to six of them, and a Structure costs
# four times as much
_matrix_desc = struct.Struct("QQQQiI").pack  # data, rows, cols, ld, dtype
_rows8_desc = struct.Struct("QQQQQQII").pack  # values, scales, rows, cols, ld, scale_ld, block

_floats = [struct.Struct(f"{n}f").pack for n in range(1, 5)]

_lib = None


def lib():
    """The library, with the signatures of the entry points that are used here."""
    global _lib
    L = _library()
    if L is not _lib:
        i, u32, u64, vp, f32, f64 = C.c_int, C.c_uint32, C.c_uint64, C.c_void_p, C.c_float, C.c_double
        sig = {
            "dg_patch_rows": (i, [vp, vp, vp, u32, u32, u32, u32, u32, vp, vp, vp, vp]),
            "dg_quantize_rows": (i, [vp, vp, vp, vp]),
            "dg_product_workspace": (u64, [vp, u64, u64, u64]),
            "dg_product": (i, [vp, vp, vp, vp, vp, vp, u64]),
            "dg_product_status": (i, [vp, vp]),
            "dg_rms_norm": (i, [vp, vp, vp, vp, vp, f32, vp, vp, vp, vp]),
            "dg_rms_norm_backward_workspace": (u64, [vp, u64, u64, u64]),
            "dg_rms_norm_backward": (i, [vp, vp, vp, vp, vp, vp, vp, vp, vp, u64, vp, vp, u64]),
            "dg_dropout": (i, [vp, vp, vp, f64, u64, u64, i, vp]),
        }
        for name, (res, args) in sig.items():
            fn = getattr(L, name)
            fn.restype, fn.argtypes = res, args
        _lib = L
    return L


class Rows8:
    """Rows in 8 bits: values float8_e4m3fn [rows, cols], scales float8_e8m0fnu [ceil(rows / block), ceil(cols / 128)].  Rows of values, or of
    a transpose (by_column) columns of values, are neighbours in memory and begin at multiples of 16 bytes, rows of scales at multiples of 4: what
    the functions here return, and empty() makes."""
    __slots__ = ("values", "scales", "block")

    def __init__(self, values, scales, block=1):
        self.values, self.scales, self.block = values, scales, block

    @classmethod
    def empty(cls, rows, cols, device, block=1, by_column=False):
        groups = -(-cols // GROUP)
        strides = (1, -(-rows // 16) * 16) if by_column else (-(-cols // 16) * 16, 1)
        values = torch.empty_strided((rows, cols), strides, dtype=torch.float8_e4m3fn, device=device)
        scales = torch.empty_strided((-(-rows // block), groups), (-(-groups // 4) * 4, 1), dtype=torch.float8_e8m0fnu, device=device)
        return cls(values, scales, block)

    @property
    def shape(self):
        return self.values.shape

    def to_float(self):
        """What the rows stand for, as float32."""
        rows, cols = self.values.shape
        scales = self.scales.float().repeat_interleave(self.block, 0)[:rows].repeat_interleave(GROUP, 1)[:, :cols]
        return self.values.float() * scales


class Norm:
    """What rms_norm returns: y (a tensor, or Rows8), sum (h, what the backward pass and the next residual want) and rstd."""
    __slots__ = ("y", "sum", "rstd")

    def __init__(self, y, sum, rstd):
        self.y, self.sum, self.rstd = y, sum, rstd

    def __iter__(self):
        return iter((self.y, self.sum, self.rstd))


def _invalid(msg):
    return DatagoB200Error(1, msg)


def _on_device(ctx, t, name):
    if not isinstance(t, torch.Tensor):
        raise _invalid(f"{name}: a torch tensor is wanted")
    device = t.get_device()  # -1 for tensors of the host
    if device != ctx.device or device < 0:
        raise _invalid(f"{name} is on {t.device}, the context on cuda:{ctx.device}")
    if t.requires_grad and torch.is_grad_enabled():
        raise _invalid(f"{name} requires a gradient, which would be lost here: detach() it, or call under no_grad()")


def _changed(out):
    """Tells autograd that a caller's tensor, or Rows8, has been written to."""
    for t in (out.values, out.scales) if isinstance(out, Rows8) else (out,):
        if not t.is_inference():
            torch.autograd.graph.increment_version(t)


def _matrix(ctx, t, name):
    _on_device(ctx, t, name)
    dtype, shape = _DTYPES.get(t.dtype), t.shape
    if dtype is None or len(shape) != 2:
        raise _invalid(f"{name}: a 2-d tensor of float32, bfloat16 or float16 is wanted")
    (rows, cols), (step, one) = shape, t.stride()
    if (one != 1 and cols > 1) or (rows > 1 and step < cols):
        raise _invalid(f"{name}: columns have to be neighbours in memory, rows apart")
    return _matrix_desc(t.data_ptr(), rows, cols, step if rows > 1 else cols, dtype, 0)


def _vector(ctx, t, name, cols):
    """A weight as a matrix of one row."""
    if t is None:
        return None
    _on_device(ctx, t, name)
    dtype = _DTYPES.get(t.dtype)
    if dtype is None or t.dim() != 1 or t.shape[0] != cols or (cols > 1 and t.stride(0) != 1):
        raise _invalid(f"{name}: {cols} neighbouring elements of float32, bfloat16 or float16 are wanted")
    return _matrix_desc(t.data_ptr(), 1, cols, cols, dtype, 0)


def _rows8(ctx, r, name, transposed=None):
    """transposed: whether values have to be by column, where the sizes leave it open"""
    if not isinstance(r, Rows8):
        raise _invalid(f"{name}: Rows8 is wanted")
    v, s = r.values, r.scales
    _on_device(ctx, v, name)
    _on_device(ctx, s, name)
    shape, sshape, block = v.shape, s.shape, r.block
    if v.dtype != torch.float8_e4m3fn or s.dtype != torch.float8_e8m0fnu or len(shape) != 2 or len(sshape) != 2 or (block != 1 and block != GROUP):
        raise _invalid(f"{name}: values float8_e4m3fn, scales float8_e8m0fnu, both 2-d, and block 1 or 128 are wanted")
    (rows, cols), (srows, groups) = shape, sshape
    if srows != -(-rows // block) or groups != -(-cols // GROUP):
        raise _invalid(f"{name}: {rows} x {cols} values have {-(-rows // r.block)} x {-(-cols // GROUP)} scales")
    (ld, one), (scale_ld, sone) = v.stride(), s.stride()
    if sone != 1 and groups > 1:
        raise _invalid(f"{name}: scales have to be neighbours in memory")
    # A single column, or row, fits both orders.  Rows of a single column that are neighbours are its line: the transpose of one row.
    by_row, by_column = one == 1 if cols > 1 else ld != 1 or rows <= 1, ld == 1 or rows <= 1
    if transposed is not None:
        by_row, by_column = by_row and not transposed, by_column and transposed
    if by_row:
        ld, column = ld if rows > 1 else -(-cols // 16) * 16, 0
    elif by_column:
        ld, column = one if cols > 1 else -(-rows // 16) * 16, 1
    else:
        raise _invalid(f"{name}: rows{' or columns' if transposed is None else ' by column' if transposed else ''} have to be neighbours in memory")
    return _rows8_desc(v.data_ptr(), s.data_ptr(), rows, cols, ld, scale_ld if srows > 1 else -(-groups // 4) * 4, block, column)


# The current stream's handle without an object around it, where torch has that.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda device: torch.cuda.current_stream(device).cuda_stream)


def _out(ctx, out, rows, cols, dtype, like, name):
    """A result and its descriptor: a new matrix, or the caller's"""
    if out is None:
        ld = (cols + 3) // 4 * 4 if dtype is torch.float32 else (cols + 7) // 8 * 8
        out = torch.empty_strided((rows, cols), (ld, 1), dtype=dtype, device=like.device)
        return out, _matrix_desc(out.data_ptr(), rows, cols, ld, _DTYPES[dtype], 0)
    if not isinstance(out, torch.Tensor) or out.shape != (rows, cols) or out.dtype != dtype:
        raise _invalid(f"{name}: a tensor ({rows}, {cols}) of {dtype} is wanted")
    return out, _matrix(ctx, out, name)


def _new_rows8(rows, cols, like):
    """Rows8.empty and its descriptor"""
    groups = -(-cols // GROUP)
    ld, scale_ld, device = -(-cols // 16) * 16, -(-groups // 4) * 4, like.device
    values = torch.empty_strided((rows, cols), (ld, 1), dtype=torch.float8_e4m3fn, device=device)
    scales = torch.empty_strided((rows, groups), (scale_ld, 1), dtype=torch.float8_e8m0fnu, device=device)
    return Rows8(values, scales), _rows8_desc(values.data_ptr(), scales.data_ptr(), rows, cols, ld, scale_ld, 1, 0)


def _workspace(nbytes, like):
    """(the tensor that keeps it, its address)"""
    if not nbytes:
        return None, None
    work = torch.empty(nbytes, dtype=torch.uint8, device=like.device)
    return work, work.data_ptr()


def _streams_of(batch):
    """(torch's current stream, the stream of a batch) where they differ, else None.  While the current stream is being captured it cannot wait for what is
    outside: the batch then has to be complete."""
    device, handle = batch.ctx.device, batch.ctx.stream
    current = torch.cuda.current_stream(device)
    if current.cuda_stream == (handle or 0):
        return None
    with torch.cuda.device(device):
        if torch.cuda.is_current_stream_capturing():
            return None
    return current, torch.cuda.ExternalStream(handle, device) if handle else torch.cuda.default_stream(device)


def patch_rows(ctx, pixels, patch, mean, std, dtype=None, out=None):
    """Patches of a bucket (uint8 [n, height, width, channels]: a tensor, or a DeviceArray of Batch.buckets()) as rows: Rows8, or with `dtype` a
    tensor.  Row (i, Y, X), feature (y, x, c) is (pixel / 255 - mean[c]) / std[c]; height and width are multiples of `patch`.  A DeviceArray is read behind
    its batch's run(), and its batch may be closed right after the call (inside a stream capture neither is waited for)."""
    if isinstance(pixels, DeviceArray):
        batch = pixels._owner if isinstance(pixels._owner, Batch) else None
        if batch is not None and not batch._h:
            raise _invalid("pixels: the batch is closed")
        streams = None if batch is None else _streams_of(batch)
        if streams:
            streams[0].wait_stream(streams[1])
        rows = patch_rows(ctx, torch.as_tensor(pixels, device=f"cuda:{ctx.device}"), patch, mean, std, dtype, out)
        if streams:
            streams[1].wait_stream(streams[0])  # the batch's memory is handed on in the order of its own stream
        return rows
    _on_device(ctx, pixels, "pixels")
    if pixels.dtype != torch.uint8 or pixels.dim() != 4 or not pixels.is_contiguous():
        raise _invalid("pixels: a contiguous uint8 [n, height, width, channels] tensor is wanted")
    n, h, w, c = pixels.shape
    if not 1 <= c <= 4:
        raise _invalid(f"{c} channels: 1 to 4 are wanted")
    if len(mean) != c or len(std) != c:
        raise _invalid(f"mean and std: {c} numbers are wanted")
    patch = int(patch)
    if patch < 1 or h % patch or w % patch or h == 0 or w == 0:
        raise _invalid(f"{h} x {w} pixels are no whole number of {patch} x {patch} patches")
    rows, cols = n * (h // patch) * (w // patch), patch * patch * c
    desc8, desc, given = None, None, out is not None
    if dtype is None:
        if out is None:
            out, desc8 = _new_rows8(rows, cols, pixels)
        else:
            desc8 = _rows8(ctx, out, "out")
    else:
        if dtype not in _DTYPES:
            raise _invalid("dtype: float32, bfloat16 or float16 is wanted")
        out, desc = _out(ctx, out, rows, cols, dtype, pixels, "out")
    floats = _floats[c - 1]
    _check(lib().dg_patch_rows(ctx._h, _raw_stream(ctx.device) or _LEGACY_STREAM, pixels.data_ptr(), n, h, w, c, patch, floats(*mean), floats(*std),
                               desc8, desc))
    if given:
        _changed(out)
    return out


def quantize_rows(ctx, x, transpose=False, block=1, out=None):
    """A matrix, or its transpose, as Rows8, with a scale for each 128 columns of `block` (1 or 128) rows of the result (`out` has a
    block of its own).  The transpose keeps the matrix's order in memory."""
    src = _matrix(ctx, x, "x")
    rows, cols = x.shape
    given = out is not None
    if not given:
        if block not in (1, GROUP):
            raise _invalid("block is 1 or 128")
        out = Rows8.empty(cols, rows, x.device, block, True) if transpose else Rows8.empty(rows, cols, x.device, block)
    _check(lib().dg_quantize_rows(ctx._h, _raw_stream(ctx.device) or _LEGACY_STREAM, src, _rows8(ctx, out, "out", transpose)))
    if given:
        _changed(out)
    return out


def product(ctx, a, b, dtype=torch.bfloat16, out=None):
    """a @ b^T of two Rows8 with the same columns, summed in 32 bits: [rows of a, rows of b] of `dtype`."""
    da, db = _rows8(ctx, a, "a"), _rows8(ctx, b, "b")
    if dtype not in _DTYPES:
        raise _invalid("dtype: float32, bfloat16 or float16 is wanted")
    (m, k), n, given = a.values.shape, b.values.shape[0], out is not None
    out, desc = _out(ctx, out, m, n, dtype, a.values, "out")
    L = lib()
    nbytes = L.dg_product_workspace(ctx._h, m, n, k) if k > 1920 else 0
    work, at = _workspace(nbytes, out)
    _check(L.dg_product(ctx._h, _raw_stream(ctx.device) or _LEGACY_STREAM, da, db, desc, at, nbytes))
    if given:
        _changed(out)
    return out


def product_status(ctx):
    """Waits for torch's current stream of the context's device; raises when a product has given up waiting for a copy."""
    _check(lib().dg_product_status(ctx._h, _raw_stream(ctx.device) or _LEGACY_STREAM))


def rms_norm(ctx, x, weight=None, residual=None, eps=1e-6, eight_bit=False, sum_out=None):
    """h = x + residual (row r takes row r % len(residual)), y = h / sqrt(mean(h^2) + eps) * weight: Norm(y, sum=h, rstd).  y is Rows8 with
    `eight_bit`, else of x's dtype.  sum_out may be x: h in its place."""
    src = _matrix(ctx, x, "x")
    rows, cols = x.shape
    w = _vector(ctx, weight, "weight", cols)
    r = None if residual is None else _matrix(ctx, residual, "residual")
    total, total_desc = _out(ctx, sum_out, rows, cols, x.dtype, x, "sum_out")
    rstd = torch.empty_strided((rows,), (1,), dtype=torch.float32, device=x.device)
    y16 = y8 = None
    if eight_bit:
        y, y8 = _new_rows8(rows, cols, x)
    else:
        y, y16 = _out(ctx, None, rows, cols, x.dtype, x, "y")
    _check(lib().dg_rms_norm(ctx._h, _raw_stream(ctx.device) or _LEGACY_STREAM, src, r, w, eps, total_desc, y16, y8, rstd.data_ptr()))
    if sum_out is not None:
        _changed(total)
    return Norm(y, total, rstd)


def rms_norm_backward(ctx, dy, h, rstd, weight=None, dsum=None, residual_rows=None, dx_out=None):
    """Gradients of rms_norm from the gradient of y (and, in dsum, of h): (dx, dresidual, dweight).  dresidual is float32 [residual_rows, cols],
    or None without residual_rows; dweight float32 [cols].  dx_out may be dy or dsum."""
    g, hm = _matrix(ctx, dy, "dy"), _matrix(ctx, h, "h")
    rows, cols = dy.shape
    w = _vector(ctx, weight, "weight", cols)
    s = None if dsum is None else _matrix(ctx, dsum, "dsum")
    _on_device(ctx, rstd, "rstd")
    if rstd.dtype != torch.float32 or rstd.numel() != rows or not rstd.is_contiguous():
        raise _invalid(f"rstd: {rows} neighbouring float32 are wanted")
    dx, dx_desc = _out(ctx, dx_out, rows, cols, dy.dtype, dy, "dx_out")
    period = int(residual_rows or 0)
    if residual_rows is not None and (period < 1 or rows % period):
        raise _invalid(f"{residual_rows} residual rows do not divide {rows}")
    dweight = torch.empty_strided((cols,), (1,), dtype=torch.float32, device=dy.device)
    dresidual = torch.empty_strided((period, cols), (cols, 1), dtype=torch.float32, device=dy.device) if period else None
    L = lib()
    nbytes = L.dg_rms_norm_backward_workspace(ctx._h, rows, cols, period)
    work, at = _workspace(nbytes, dy)
    _check(L.dg_rms_norm_backward(ctx._h, _raw_stream(ctx.device) or _LEGACY_STREAM, g, hm, rstd.data_ptr(), w, s, dx_desc,
                                  dresidual.data_ptr() if period else None, period, dweight.data_ptr(), at, nbytes))
    if dx_out is not None:
        _changed(dx)
    return dx, dresidual, dweight


def dropout(ctx, x, p, seed, offset=0, per_row=False, out=None):
    """x with elements (or, per_row, rows) dropped with probability p and the others scaled up.  The mask is a function of (seed, offset + index):
    the same call on the gradient is the backward pass.  out may be x."""
    src = _matrix(ctx, x, "x")
    given = out is not None
    if not given:
        out = torch.empty_strided(x.shape, (x.shape[1], 1), dtype=x.dtype, device=x.device)  # one long row, if x is
    out, desc = _out(ctx, out, *x.shape, x.dtype, x, "out")
    seed, offset = int(seed), int(offset)
    if not 0 <= seed < 1 << 64 or not 0 <= offset < 1 << 64:
        raise _invalid("seed and offset are in [0, 2^64)")
    _check(lib().dg_dropout(ctx._h, _raw_stream(ctx.device) or _LEGACY_STREAM, src, p, seed, offset, per_row, desc))
    if given:
        _changed(out)
    return out


def _detached(t):
    return t.detach() if isinstance(t, torch.Tensor) else t  # (what is no tensor is refused where it is used)


class PatchStem:
    """The stem of a model that reads buckets: patches as 8-bit rows, the product with the embedding weight, dropout, positions (shared by
    the images of a bucket), norm, 8-bit rows for the first layer.

    weight: [width, patch * patch * channels]; norm_weight: [width] or None.  The weight is laid out in 8 bits (scales of 128 x 128 blocks)
    here and by set_weight, not with every call.  weight, norm_weight and positions may require gradients: backward returns them."""

    def __init__(self, ctx, patch, mean, std, weight, norm_weight=None, p=0.0, seed=0, eps=1e-6, dtype=torch.bfloat16):
        self.ctx, self.patch, self.mean, self.std = ctx, int(patch), tuple(mean), tuple(std)
        self.norm_weight, self.p, self.seed, self.eps, self.dtype = norm_weight, float(p), int(seed), float(eps), dtype
        self.weight8 = None
        self.set_weight(weight)

    def set_weight(self, weight):
        """After an optimizer step: the new weight in 8 bits, on torch's current stream.  One of the same shape takes the old one's place in memory, so that
        captured forward passes read it too."""
        weight = _detached(weight)
        kept = self.weight8 if self.weight8 is not None and self.weight8.shape == getattr(weight, "shape", None) else None
        self.weight8 = quantize_rows(self.ctx, weight, block=GROUP, out=kept)

    def forward(self, pixels, positions, offset=0):
        """(Norm with Rows8 for the first layer, what backward wants).  positions: [tokens of an image, width] of the stem's dtype (row r of all takes row
        r % len(positions)).  offset: where this batch's elements begin in the run's count (see dropout)."""
        norm_weight = _detached(self.norm_weight)
        x = product(self.ctx, patch_rows(self.ctx, pixels, self.patch, self.mean, self.std), self.weight8, self.dtype)
        if self.p:
            dropout(self.ctx, x, self.p, self.seed, offset, out=x)
        norm = rms_norm(self.ctx, x, norm_weight, residual=_detached(positions), eps=self.eps, eight_bit=True, sum_out=x)
        # what later changes of the stem's attributes must not change: the same draws and the same weight go into the gradients
        return norm, (pixels, norm.sum, norm.rstd, len(positions), offset, self.p, self.seed, norm_weight)

    def backward(self, saved, dy, dsum=None):
        """Gradients (weight, positions, norm_weight), float32, from those of the norm's output and, in dsum, of its sum, with the p, seed and
        norm_weight of that forward pass, whatever the stem has now (an evaluation between the two may set p to 0).  The pixels of the bucket still
        have to be there."""
        pixels, h, rstd, tokens, offset, p, seed, norm_weight = saved
        dx, dpositions, dnorm = rms_norm_backward(self.ctx, dy, h, rstd, norm_weight, dsum, tokens)
        if p:
            dropout(self.ctx, dx, p, seed, offset, out=dx)
        x = patch_rows(self.ctx, pixels, self.patch, self.mean, self.std, self.dtype)
        if not len(x):  # a sum over no rows; the transposes would have no columns
            return torch.zeros(dx.shape[1], x.shape[1], dtype=torch.float32, device=dx.device), dpositions, dnorm
        dweight = product(self.ctx, quantize_rows(self.ctx, dx, transpose=True), quantize_rows(self.ctx, x, transpose=True), torch.float32)
        return dweight, dpositions, dnorm
