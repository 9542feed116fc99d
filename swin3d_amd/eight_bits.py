"""Dense layers whose rows are held in eight bits.

At inference a layer's input is whole numbers with a scale a row (`Int8Rows`), its weight whole numbers with a scale an output
channel, and the product a sum of whole numbers, exact, with both scales behind it:

    sum, rows = add_norm_int8(x, branch, block.norm2)           # (x + branch, its LayerNorm or RMSNorm in eight bits)
    y = linear_int8(rows, quantize_rows(layer.weight), layer.bias)
    y = mlp_int8(rows, quantize_rows(fc1.weight), fc1.bias, quantize_rows(fc2.weight), fc2.bias)

In training a layer keeps what its backward reads of its input in eight bits, in groups of sixteen numbers with a scale each
(`keep_rows`): the forward is the layer's own in fp16, and so is the gradient of its input; the weight's gradient is that of rows half a step off at most.
That is a 254th of their group's largest number, and where a scale of four bits is above what the group needs up to an eighth of that more; in groups whose
largest number is below 127 2^-21, whose scales are whole multiples of 2^-24, up to 2^-25 more; and of numbers above 65,088, where codes end, up to 416:

    y = checkpointed_linear(x, layer.weight, layer.bias)
    y = checkpointed_mlp(x, fc1.weight, fc1.bias, fc2.weight, fc2.bias)

`swin3d_amd.encoder.eight_bit_inference` and `eight_bit_checkpoints` make the blocks of a network use them.

All take dense CUDA (HIP) tensors, enqueue on torch's current stream of their device and do not wait.  What is wrong with an argument
raises ValueError, CPU tensors included.
"""
import ctypes
import functools
from typing import NamedTuple

import torch
import torch.nn as nn
from torch.autograd.function import Function, once_differentiable

from . import _lib
from .swin_blocks import followed

_DTYPE_CODE = {torch.float32: _lib.S3D_DTYPE_F32, torch.float16: _lib.S3D_DTYPE_F16}
_MOST_CHANNELS, _MOST_SUMMED, _MOST_WIDTH, _MOST_HIDDEN = 8192, 65536, 16384, 8192


class Int8Rows(NamedTuple):
    """Rows in eight bits: codes int8 [N,C], scales float32 [N]; row i stands for codes[i] * scales[i]."""
    codes: torch.Tensor
    scales: torch.Tensor

    def values(self, dtype=torch.float16):
        """[N,C] in float16 or float32: what the rows stand for.  No autograd."""
        codes, scales = self
        if not (isinstance(codes, torch.Tensor) and codes.is_cuda and scales is not None and _ready(codes.device, codes, scales)
                and codes.dtype is torch.int8 and codes.dim() == 2 and scales.dtype is torch.float32 and scales.shape == codes.shape[:1]
                and codes.shape[0] <= 0x7fffffff):
            _check_rows("rows", self)
            codes, scales = _dense(codes), _dense(scales)
        if dtype not in _DTYPE_CODE:
            raise ValueError(f"dtype {dtype} (float16 or float32)")
        n, c = codes.shape
        if c == 0 or c % 4 or c > _MOST_CHANNELS:
            raise ValueError(f"rows of {c} channels (a multiple of 4, at most {_MOST_CHANNELS})")
        _unfollowed("Int8Rows.values", scales)
        dev = codes.device
        out = torch.empty((n, c), dtype=dtype, device=dev)
        with _lib.on(dev):
            status = _lib.lib().s3d_int8_values(codes.data_ptr(), scales.data_ptr(), out.data_ptr(), _DTYPE_CODE[dtype], n, c, _lib.stream(dev))
        _lib.check(status, "s3d_int8_values")
        return out


def _dense(t):
    """t as the kernels read it: dense and 16-byte aligned.  (A parameter whose storage has been freed has a null pointer, which of a bias, a norm's weight or
    a residual would say that there is none.)"""
    at = t.data_ptr()
    if at == 0 and t.numel() > 0:
        raise ValueError(f"a tensor {tuple(t.shape)} without memory")
    if not t.is_contiguous():
        return t.contiguous()
    return t if at % 16 == 0 else t.clone()


def _check(name, t, dtypes, shape, device=None):
    """t is a tensor on the GPU (on `device`) of one of the dtypes and of `shape`, in which None stands for any size."""
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a tensor, got {type(t).__name__}")
    sizes = t.shape
    fits = t.is_cuda and t.dtype in dtypes and len(sizes) == len(shape) and (device is None or t.device == device)
    if fits:
        for size, got in zip(shape, sizes):
            fits = fits and (size is None or size == got)
    if not fits:
        wanted = ",".join("any" if s is None else str(s) for s in shape)
        kinds = " or ".join(str(d).replace("torch.", "") for d in dtypes)
        where = "on a CUDA (HIP) device" if device is None else f"on {device}"
        raise ValueError(f"{name} must be {kinds} [{wanted}] {where}, got {t.dtype} {tuple(sizes)} on {t.device}")
    if len(shape) == 2:
        _check_row_count(name, sizes[0])


def _check_row_count(name, count):
    if count > 0x7fffffff:
        raise ValueError(f"{name} has {count} rows (at most 2^31 - 1)")


def _check_rows(name, rows, device=None):
    if not isinstance(rows, tuple) or len(rows) != 2:
        raise ValueError(f"{name} must be Int8Rows, got {type(rows).__name__}")
    codes, scales = rows
    _check(f"{name}.codes", codes, _INT8, _ANY_ROWS, device)
    _check(f"{name}.scales", scales, _FP32, (codes.shape[0],), codes.device)


_INT8, _FP32, _FP16, _EITHER = (torch.int8,), (torch.float32,), (torch.float16,), (torch.float16, torch.float32)
_ANY_ROWS = (None, None)


def _ready(dev, *tensors):
    """All of them (None aside) are plain, dense and 16-byte aligned on `dev`: nothing about them has to be looked at or copied but shapes and types."""
    return all(t is None or (type(t) in _PLAIN and t.device == dev and t.is_contiguous() and (at := t.data_ptr()) != 0 and at % 16 == 0) for t in tensors)


_PLAIN = (torch.Tensor, nn.Parameter)


def _unfollowed(what, *tensors):
    """These calls are no operations of autograd: nothing may follow them."""
    if followed():
        raise RuntimeError(f"{what} does not run under a transform, a forward-mode derivative, a dispatch mode or a tracer")
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad(), or detach what requires one")


def _empty_rows(n, c, device):
    return Int8Rows(torch.empty((n, c), dtype=torch.int8, device=device), torch.empty(n, dtype=torch.float32, device=device))


def _norm_parameters(norm, rms, c, dev):
    """(weight, bias) of a norm over c channels, either may be None.  normalized_shape is a plain attribute and says nothing of what the parameters
    are by now: the kernel reads c numbers of each."""
    weight, bias = norm.weight, None if rms else norm.bias
    for name, p in (("norm.weight", weight), ("norm.bias", bias)):
        if p is not None and not (p.dtype is torch.float32 and p.device == dev and p.dim() == 1 and p.numel() == c):
            _check(name, p, (torch.float32, torch.float16, torch.bfloat16, torch.float64), (c,), dev)
    return weight, bias


def add_norm_int8(x, residual, norm, inplace=False):
    """(x + residual, norm(x + residual) in eight bits) for x fp32 [N,C] and `norm` a torch.nn.LayerNorm or RMSNorm over C.

    residual   fp16 / fp32 [N,C] or None (then the first result is x itself)
    inplace    write the sum back into x instead of a new tensor
    C is a multiple of 4 and at most 8192.  A row with a number that is not finite stands for NaN.  No autograd.
    """
    _check("x", x, _FP32, _ANY_ROWS)
    n, c = x.shape
    dev = x.device
    if c == 0 or c % 4 or c > _MOST_CHANNELS:
        raise ValueError(f"rows of {c} channels (a multiple of 4, at most {_MOST_CHANNELS})")
    rms = isinstance(norm, nn.RMSNorm)
    kind = nn.RMSNorm if rms else nn.LayerNorm
    # (a class or an instance with a forward of its own is another norm)
    if not isinstance(norm, kind) or type(norm).forward is not kind.forward or "forward" in norm.__dict__ or tuple(norm.normalized_shape) != (c,):
        raise ValueError(f"norm must be a LayerNorm or RMSNorm over the {c} channels, got {norm}")
    weight, bias = _norm_parameters(norm, rms, c, dev)
    if residual is not None:
        _check("residual", residual, _EITHER, (n, c), dev)
    _unfollowed("add_norm_int8", x, residual, weight, bias)
    if inplace and residual is not None and not (x.is_contiguous() and x.data_ptr() % 16 == 0):
        raise ValueError("x must be contiguous and 16-byte aligned to be written in place")
    eps = norm.eps if norm.eps is not None else torch.finfo(torch.float32).eps
    rows_in = _dense(x)
    res_ptr, res_code, summed = None, 0, x
    if residual is not None:
        residual = _dense(residual)
        res_ptr, res_code = residual.data_ptr(), _DTYPE_CODE[residual.dtype]
        summed = x if inplace else torch.empty((n, c), dtype=torch.float32, device=dev)
    gamma, beta = (None if p is None else _dense(p) if p.dtype is torch.float32 else _dense(p).detach().float() for p in (weight, bias))
    rows = _empty_rows(n, c, dev)
    with _lib.on(dev):
        status = _lib.lib().s3d_add_norm_int8(
            rows_in.data_ptr(), res_ptr, res_code, None if gamma is None else gamma.data_ptr(), None if beta is None else beta.data_ptr(), float(eps),
            int(rms), None if residual is None else summed.data_ptr(), rows.codes.data_ptr(), rows.scales.data_ptr(), n, c, _lib.stream(dev))
    _lib.check(status, "s3d_add_norm_int8")
    if residual is not None and inplace:
        torch.autograd.graph.increment_version(x)      # (as torch's own changes in place: a graph that has kept x for its backward refuses it then)
    return summed, rows


def quantize_rows(x):
    """Int8Rows of fp16 or fp32 rows [N,C]: the input of a layer, or a weight [out,in].  scale = max |row| / 127, code = row / scale to the
    nearest, ties to even.  C is a multiple of 4 and at most 8192.  No autograd: x is taken as its data."""
    _check("x", x, _EITHER, _ANY_ROWS)
    n, c = x.shape
    if c == 0 or c % 4 or c > _MOST_CHANNELS:
        raise ValueError(f"rows of {c} channels (a multiple of 4, at most {_MOST_CHANNELS})")
    _unfollowed("quantize_rows")
    x = _dense(x.detach())
    rows = _empty_rows(n, c, x.device)
    with _lib.on(x.device):
        status = _lib.lib().s3d_quantize_rows(x.data_ptr(), _DTYPE_CODE[x.dtype], rows.codes.data_ptr(), rows.scales.data_ptr(), n, c,
                                              _lib.stream(x.device))
    _lib.check(status, "s3d_quantize_rows")
    return rows


def _layer_operands(name, weight, bias, k, dev):
    """(codes, scales, bias or None) of a layer of k inputs, as the kernels read them."""
    _check_rows(name, weight, dev)
    codes, scales = weight
    n = codes.shape[0]
    if codes.shape[1] != k:
        raise ValueError(f"{name} takes {codes.shape[1]} channels, the rows have {k}")
    if bias is not None:
        _check(f"the bias of {name}", bias, (torch.float32, torch.float16), (n,), dev)
        bias = _dense(bias).float()      # (where autograd follows it, the result requires a gradient and is refused)
    return _dense(codes), _dense(scales), bias


def _product_operands(rows, weight, bias):
    """(x, its scales, w, its scales, bias or None, rows, inputs, outputs, device), as the kernels read them."""
    if isinstance(rows, tuple) and isinstance(weight, tuple) and len(rows) == len(weight) == 2:
        (x, sx), (w, sw) = rows, weight
        # (the usual operands: each is looked at once)
        if isinstance(x, torch.Tensor) and x.is_cuda and sx is not None and w is not None and sw is not None \
                and _ready(x.device, x, sx, w, sw, bias) and x.dtype is w.dtype is torch.int8 \
                and sx.dtype is sw.dtype is torch.float32 and (bias is None or bias.dtype is torch.float32):
            a, b = x.shape, w.shape
            if len(a) == len(b) == 2 and a[1] == b[1] and sx.shape == a[:1] and sw.shape == b[:1] and (bias is None or bias.shape == b[:1]) \
                    and a[0] <= 0x7fffffff:
                return x, sx, w, sw, bias, a[0], a[1], b[0], x.device
    _check_rows("rows", rows)
    m, k = rows[0].shape
    dev = rows[0].device
    w, sw, bias = _layer_operands("weight", weight, bias, k, dev)
    return _dense(rows[0]), _dense(rows[1]), w, sw, bias, m, k, w.shape[0], dev


def linear_int8(rows, weight, bias=None, gelu=False):
    """fp16 [N,out]: rows @ weight.T + bias, then GELU (the exact form) where `gelu`.

    rows     Int8Rows [N,in]: of add_norm_int8 or quantize_rows
    weight   Int8Rows [out,in]: quantize_rows(layer.weight)
    bias     fp32 or fp16 [out], or None
    The sums are exact, scales, bias and GELU fp32, with one rounding at the end.  in is a multiple of 16 up to 65536, out of 8.  No autograd.
    """
    x, sx, w, sw, bias, m, k, n, dev = _product_operands(rows, weight, bias)
    if k == 0 or k % 16 or k > _MOST_SUMMED or n == 0 or n % 8:
        raise ValueError(f"a layer from {k} to {n} channels (from a multiple of 16 up to {_MOST_SUMMED}, to a multiple of 8)")
    _unfollowed("linear_int8", sx, sw, bias)
    y = torch.empty((m, n), dtype=torch.float16, device=dev)
    with _lib.on(dev):
        status = _lib.lib().s3d_linear_int8(x.data_ptr(), sx.data_ptr(), w.data_ptr(), sw.data_ptr(), None if bias is None else bias.data_ptr(),
                                            y.data_ptr(), m, n, k, int(bool(gelu)), _lib.stream(dev))
    _lib.check(status, "s3d_linear_int8")
    return y


def mlp_int8(rows, weight1, bias1, weight2, bias2):
    """linear_int8(quantize_rows(linear_int8(rows, weight1, bias1, gelu=True)), weight2, bias2) as one call.  Both widths are multiples
    of 16 up to 8192; biases as for linear_int8, either may be None.

    Not the fastest form of an MLP everywhere: from 16,384 rows and 192 C on, at 48 to 192 channels over up to 1024, both layers run as one kernel in fp16
    (s3d_mlp, which inference without eight bits takes), at that line in 0.9 to 1.25 of this call's time, with more rows in 0.6 to 1.0 of it (us, fp16 / this:
    149,993 rows of 160 101 / 144, 595,677 of 80 137 / 232, 37,499 of 192 53.3 / 54.2)."""
    x, sx, w1, s1, bias1, m, c, hidden, dev = _product_operands(rows, weight1, bias1)
    w2, s2, bias2 = _layer_operands("weight2", weight2, bias2, hidden, dev)
    if w2.shape[0] != c or any(w == 0 or w % 16 or w > _MOST_HIDDEN for w in (c, hidden)):
        raise ValueError(f"an MLP from {c} over {hidden} to {w2.shape[0]} channels (back to as many, multiples of 16 up to {_MOST_HIDDEN})")
    _unfollowed("mlp_int8", sx, s1, bias1, s2, bias2)
    y = torch.empty((m, c), dtype=torch.float16, device=dev)
    lib = _lib.lib()
    with _lib.on(dev):
        ws_bytes = lib.s3d_mlp_int8_workspace_bytes(m, c, hidden)
        workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
        status = lib.s3d_mlp_int8(x.data_ptr(), sx.data_ptr(), w1.data_ptr(), s1.data_ptr(), None if bias1 is None else bias1.data_ptr(), w2.data_ptr(),
                                  s2.data_ptr(), None if bias2 is None else bias2.data_ptr(), y.data_ptr(), m, c, hidden, workspace.data_ptr(), ws_bytes,
                                  _lib.stream(dev))
    _lib.check(status, "s3d_mlp_int8")
    return y


# ---- checkpoints -------------------------------------------------------------------------------------------------------------

def _check_width(name, width):
    if width == 0 or width % 16 or width > _MOST_WIDTH:
        raise ValueError(f"{name} of {width} channels (a multiple of 16, at most {_MOST_WIDTH})")


def keep_rows(x):
    """uint8 [17 N C / 16]: fp16 rows [N,C] in eight bits, in groups of sixteen numbers: codes int8 [N,C], then a byte with the scale of
    every group (s3d_keep_rows has the form).  C is a multiple of 16, at most 16384.  x is taken as its data."""
    _check("x", x, _FP16, _ANY_ROWS)
    m, k = x.shape
    _check_width("rows", k)
    _unfollowed("keep_rows")
    x = _dense(x.detach())
    kept = torch.empty(_kept_size(m, k), dtype=torch.uint8, device=x.device)
    with _lib.on(x.device):
        status = _lib.lib().s3d_keep_rows(x.data_ptr(), kept.data_ptr(), m, k, _lib.stream(x.device))
    _lib.check(status, "s3d_keep_rows")
    return kept


def kept_values(kept, channels):
    """fp16 [N,channels]: what kept rows stand for, exactly."""
    _check("kept", kept, (torch.uint8,), (None,))
    _check_width("rows", channels)
    m, rest = divmod(kept.numel(), channels + channels // 16)
    if rest:
        raise ValueError(f"{kept.numel()} bytes are no whole number of rows of {channels} channels")
    _check_row_count("kept", m)
    _unfollowed("kept_values")
    kept = _dense(kept)
    out = torch.empty((m, channels), dtype=torch.float16, device=kept.device)
    with _lib.on(kept.device):
        status = _lib.lib().s3d_kept_values(kept.data_ptr(), out.data_ptr(), m, channels, _lib.stream(kept.device))
    _lib.check(status, "s3d_kept_values")
    return out


def _ptr(t):
    return None if t is None else t.data_ptr()



def _rows_like(t, dtype):
    """A gradient that came in, as the kernels read it."""
    return _dense(t if t.dtype == dtype else t.to(dtype))


def _parameter_gradients(dtypes, needs, shapes, rows, device):
    """(type, gradients or None): one type for all of them, fp32 if any of those wanted is; zeros where there are no rows."""
    wanted = [d for d, need in zip(dtypes, needs) if need]
    dtype = torch.float32 if not wanted or torch.float32 in wanted else torch.float16
    make = torch.empty if rows else torch.zeros
    return dtype, [make(shape, dtype=dtype, device=device) if need else None for shape, need in zip(shapes, needs)]


def _saved_places(sizes):
    """(where blocks of as many bytes begin in one buffer, each on a multiple of 256, and its size)."""
    places, at = [], 0
    for size in sizes:
        places.append(at)
        at += size + -size % 256
    return places, at


def _kept_size(m, k):
    return m * k + m * (k // 16)


def _typed(grads, dtypes):
    return (g if g is None or g.dtype == d else g.to(d) for g, d in zip(grads, dtypes))


class _KeptLinear(Function):
    """graph: whether one is recorded; without it nothing is kept.  scaled: (rows of the parameters, what they are multiplied by)."""

    @staticmethod
    def forward(ctx, graph, x, weight, bias, scaled):
        need_x, need_weight = (graph and need for need in ctx.needs_input_grad[1:3])
        (m, k), n, dev = x.shape, weight.shape[0], x.device
        y = torch.empty((m, n), dtype=torch.float16, device=dev)
        # one buffer for what the backward reads: kept rows, and the weight transposed
        places, size = _saved_places((_kept_size(m, k) if need_weight else 0, 2 * n * k if need_x else 0))
        saved = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
        if m:
            rows, weight, bias = _dense(x), _dense(weight), None if bias is None else _dense(bias)
            at = saved.data_ptr() if size else 0
            lib = _lib.lib()
            ws_bytes = lib.s3d_kept_linear_workspace_bytes(n, k)
            workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
            with _lib.on(dev):
                status = lib.s3d_kept_linear(
                    rows.data_ptr(), weight.data_ptr(), _DTYPE_CODE[weight.dtype], _ptr(bias), 0 if bias is None else _DTYPE_CODE[bias.dtype],
                    y.data_ptr(), at + places[0] if need_weight else None, at + places[1] if need_x else None, m, n, k, *scaled,
                    workspace.data_ptr(), ws_bytes, _lib.stream(dev))
            _lib.check(status, "s3d_kept_linear")
        ctx.save_for_backward(saved)
        ctx.scaled, ctx.shapes, ctx.places, ctx.dtypes = scaled, (m, n, k), places, [weight.dtype, None if bias is None else bias.dtype]
        return y

    @staticmethod
    def backward(ctx, dy):
        return _linear_gradients_once(ctx, dy) if torch.is_grad_enabled() else _linear_gradients(ctx, dy)


def _linear_gradients(ctx, dy):
    saved, = ctx.saved_tensors
    (m, n, k), places, dev, needs = ctx.shapes, ctx.places, dy.device, ctx.needs_input_grad[1:4]
    dx = torch.empty((m, k), dtype=torch.float16, device=dev) if needs[0] else None
    dtype, grads = _parameter_gradients(ctx.dtypes, needs[1:], ((n, k), (n,)), m, dev)
    if m:
        dy, at = _rows_like(dy, torch.float16), 0 if saved is None else saved.data_ptr()
        lib = _lib.lib()
        ws_bytes = lib.s3d_kept_linear_grad_workspace_bytes(m, n, k)
        workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
        with _lib.on(dev):
            status = lib.s3d_kept_linear_grad(dy.data_ptr(), at + places[1] if needs[0] else None, at + places[0] if needs[1] else None, _ptr(dx),
                                              *(_ptr(g) for g in grads), _DTYPE_CODE[dtype], m, n, k, *ctx.scaled, workspace.data_ptr(), ws_bytes,
                                              _lib.stream(dev))
        _lib.check(status, "s3d_kept_linear_grad")
    return (None, dx, *_typed(grads, ctx.dtypes), None)


class _KeptMlp(Function):
    @staticmethod
    def forward(ctx, graph, x, weight1, bias1, weight2, bias2):
        needs = [graph and need for need in ctx.needs_input_grad[1:]]
        (m, c), hidden, dev = x.shape, weight1.shape[0], x.device
        behind = any(needs[:3])
        y = torch.empty((m, c), dtype=torch.float16, device=dev)
        wanted = needs[1], behind or needs[3], needs[0], behind
        places, size = _saved_places([size if want else 0 for size, want in zip(
            (_kept_size(m, c), _kept_size(m, hidden), 2 * c * hidden, 2 * c * hidden), wanted)])
        saved = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
        params = weight1, bias1, weight2, bias2
        if m:
            rows, params = _dense(x), [None if p is None else _dense(p) for p in params]
            at = saved.data_ptr() if size else 0
            lib = _lib.lib()
            ws_bytes = lib.s3d_kept_mlp_workspace_bytes(m, c, hidden)
            workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
            with _lib.on(dev):
                status = lib.s3d_kept_mlp(
                    rows.data_ptr(), *(_ptr(p) for p in params), _dtype_codes(*(None if p is None else p.dtype for p in params)), y.data_ptr(),
                    *(at + place if want else None for place, want in zip(places, wanted)), m, c, hidden, workspace.data_ptr(), ws_bytes,
                    _lib.stream(dev))
            _lib.check(status, "s3d_kept_mlp")
        ctx.save_for_backward(saved)
        ctx.shapes, ctx.places, ctx.wanted = (m, c, hidden), places, wanted
        ctx.dtypes = [None if p is None else p.dtype for p in params]
        return y

    @staticmethod
    def backward(ctx, dy):
        return _mlp_gradients_once(ctx, dy) if torch.is_grad_enabled() else _mlp_gradients(ctx, dy)


def _mlp_gradients(ctx, dy):
    saved, = ctx.saved_tensors
    needs, (m, c, hidden), dev = ctx.needs_input_grad[1:], ctx.shapes, dy.device
    dx = torch.empty((m, c), dtype=torch.float16, device=dev) if needs[0] else None
    dtype, grads = _parameter_gradients(ctx.dtypes, needs[1:], ((hidden, c), (hidden,), (c, hidden), (c,)), m, dev)
    if m:
        dy, at = _rows_like(dy, torch.float16), 0 if saved is None else saved.data_ptr()
        kept_x, kept_h, turned1, turned2 = (at + place if want else None for place, want in zip(ctx.places, ctx.wanted))
        lib = _lib.lib()
        ws_bytes = lib.s3d_kept_mlp_grad_workspace_bytes(m, c, hidden)
        workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
        with _lib.on(dev):
            status = lib.s3d_kept_mlp_grad(dy.data_ptr(), turned1, turned2, kept_x, kept_h, _ptr(dx), *(_ptr(g) for g in grads), _DTYPE_CODE[dtype], m, c,
                                           hidden, workspace.data_ptr(), ws_bytes, _lib.stream(dev))
        _lib.check(status, "s3d_kept_mlp_grad")
    return (None, dx, *_typed(grads, ctx.dtypes))


@functools.lru_cache(maxsize=32)
def _dtype_codes(*dtypes):
    return (ctypes.c_int32 * len(dtypes))(*(_DTYPE_CODE.get(d, 0) for d in dtypes))


# (a graph of the gradients: they are no functions of what they are made from that autograd could follow, and say so when it tries)
_linear_gradients_once, _mlp_gradients_once = once_differentiable(_linear_gradients), once_differentiable(_mlp_gradients)


def _check_layer(name, weight, bias, k, dev):
    _check(name, weight, tuple(_DTYPE_CODE), (None, k), dev)
    if bias is not None:
        _check(f"the bias of {name}", bias, tuple(_DTYPE_CODE), (weight.shape[0],), dev)
    _check_width(f"{name}: rows", k)
    _check_width(f"{name}: results", weight.shape[0])


def _no_followers(what):
    if followed():
        raise RuntimeError(f"{what} does not run under a transform, a forward-mode derivative, a dispatch mode or a tracer")


def checkpointed_linear(x, weight, bias=None, scaled=None):
    """F.linear(x, weight, bias) in fp16 for fp16 rows [N,in] and parameters in fp16 or fp32, which keeps x for its backward in eight
    bits: 1.0625 bytes a number in place of two.  y and the gradient of x are those of the layer in fp16; the gradients of the parameters come in
    their own type, weight's from what was kept.  scaled: (rows, factor), for a layer whose first `rows` outputs (a multiple of 16) are `factor` times
    those of the parameters, as q's are in an attention.  Widths are multiples of 16 up to 16384.  Gradients of gradients are refused.

    Where x has a gradient an fp16 copy of the weight, transposed, is kept too, 2 in out bytes.  So does a layer under autocast with parameters in fp32; one
    with parameters in fp16 keeps no copy, and with fewer than some 2.1 out rows less than this one."""
    _check("x", x, _FP16, _ANY_ROWS)
    _check_layer("weight", weight, bias, x.shape[1], x.device)
    _no_followers("checkpointed_linear")
    rows, factor = (0, 1.0) if scaled is None else scaled
    if not hasattr(type(rows), "__index__") or isinstance(rows, torch.Tensor) or not 0 <= rows <= weight.shape[0] or rows % 16:
        raise ValueError(f"{rows} scaled outputs of {weight.shape[0]} (a multiple of 16)")
    if isinstance(factor, torch.Tensor) and factor.requires_grad and torch.is_grad_enabled():
        raise ValueError("the factor of scaled outputs is a number, of which there is no gradient: multiply the parameters where it is trained")
    return _KeptLinear.apply(torch.is_grad_enabled(), x, weight, bias, (int(rows), float(factor)))


def checkpointed_mlp(x, weight1, bias1, weight2, bias2):
    """F.linear(F.gelu(F.linear(x, weight1, bias1)), weight2, bias2) in fp16 for fp16 rows [N,C] and parameters in fp16 or fp32, which keeps
    x and the hidden layer's rows in front of GELU in eight bits: for a hidden layer of 4 C channels 5.3 C bytes a row, where x and the hidden layer on both
    sides of GELU are 18 C.  Beside them fp16 copies of the weights, transposed, 4 C hidden bytes (see checkpointed_linear).  Widths are multiples of 16 up to
    16384, biases may be None.  Gradients of gradients are refused.

    The gradients go by what was kept.  The operands of products are fp16 numbers, as those of the layers one by one are: GELU of the hidden layer, in the
    backward also that of what was kept and, for the gradients of x and weight1, the hidden layer's gradient are rounded to fp16.  bias1's gradient is a sum
    of unrounded ones."""
    _check("x", x, _FP16, _ANY_ROWS)
    c = x.shape[1]
    _check_layer("weight1", weight1, bias1, c, x.device)
    _check_layer("weight2", weight2, bias2, weight1.shape[0], x.device)
    if weight2.shape[0] != c:
        raise ValueError(f"an MLP from {c} to {weight2.shape[0]} channels (back to as many)")
    _no_followers("checkpointed_mlp")
    return _KeptMlp.apply(torch.is_grad_enabled(), x, weight1, bias1, weight2, bias2)
