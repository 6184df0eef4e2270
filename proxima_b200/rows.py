"""Operators on embedding rows held in torch CUDA tensors.

An index searches embeddings; these are the steps around it that need the same
products: cutting rows to 8 bits (``quantize_rows`` / ``dequantize_rows``),
the whole score matrix of 8-bit rows (``int8_scores``: the searches return a
top-k only), and the loss the embeddings are trained with, a softmax over the
base, with its gradient (``softmax_cross_entropy``).

Each call runs on the current torch stream of its tensors' device and returns
without waiting. Tensors must be CUDA tensors of one device (TypeError /
ValueError otherwise); arrays whose columns are not contiguous, or whose rows
do not start on 16-byte boundaries where the tensor cores read them, are
copied first. The kernels are libproxima_b200's; there is no fallback, and the
calls cannot be traced (RuntimeError; torch.compile runs them between graphs).
"""

from __future__ import annotations

import math

import torch
from torch.autograd import forward_ad

from . import _lib

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}
_INT8_MAX_DIM = 131071
_PROXY = torch._C._TorchDispatchModeKey.PROXY
_is_tracing, _dispatch_mode, _is_grad_enabled = torch._C._is_tracing, torch._C._get_dispatch_mode, torch.is_grad_enabled


def _not_traced(name: str) -> None:
    """A trace would record the empty results, not what the kernels write to
    their memory."""
    if _is_tracing() or _dispatch_mode(_PROXY) is not None:
        raise RuntimeError(f"{name} cannot be traced: its kernels run on the tensors' memory")


def _check(a, name: str, ndim: int, dtypes) -> None:
    if not isinstance(a, torch.Tensor) or not a.is_cuda or a.dim() != ndim or a.dtype not in dtypes:
        names = ", ".join(str(t).removeprefix("torch.") for t in dtypes)
        raise TypeError(f"argument '{name}': expected a {ndim}-d CUDA tensor of {names}")


def _same_device(device, **tensors) -> None:
    for name, a in tensors.items():
        if a is not None and a.device != device:
            raise ValueError(f"argument '{name}' is on {a.device}, expected {device}")


def _dim(a, name: str) -> int:
    if a.shape[1] == 0:
        raise ValueError(f"argument '{name}': dim must be > 0")
    return a.shape[1]


def _ld(a) -> int:
    """Row stride in elements (a single row's stride says nothing)."""
    return a.stride(0) if a.shape[0] > 1 else max(a.stride(0), a.shape[1])


def _plain(a):
    """`a` with contiguous columns and rows that do not overlap."""
    if a.stride(1) != 1 and a.shape[1] > 1 or a.shape[0] > 1 and a.stride(0) < a.shape[1]:
        return a.contiguous()
    return a


def _empty_rows(n: int, dim: int, dtype, device):
    """An n x dim tensor whose rows start on 16-byte boundaries."""
    unit = 16 // dtype.itemsize
    if dim % unit == 0:
        return torch.empty((n, dim), dtype=dtype, device=device)
    return torch.empty((n, (dim + unit - 1) // unit * unit), dtype=dtype, device=device)[:, :dim]


def _tiled(a):
    """`a` as the tensor cores read it, and its row stride: a copy unless its
    rows start on 16-byte boundaries."""
    a = _plain(a)
    unit = 16 // a.dtype.itemsize
    if a.data_ptr() % 16 == 0 and (a.shape[0] <= 1 or a.stride(0) % unit == 0):
        return a, (a.stride(0) if a.shape[0] > 1 else (a.shape[1] + unit - 1) // unit * unit)
    b = _empty_rows(a.shape[0], a.shape[1], a.dtype, a.device)
    b.copy_(a)
    return b, b.stride(0)


def _aligned(a):
    """A 1-d float32 tensor, contiguous and on a 16-byte boundary."""
    if a is None:
        return None
    a = a.contiguous()
    return a if a.data_ptr() % 16 == 0 else a.clone()


def _ptr(a):
    return None if a is None else a.data_ptr()


def _stream(index: int) -> int:
    """The current stream of a device (what torch.cuda.current_stream's
    cuda_stream gives, without making a Stream object for it)."""
    return torch._C._cuda_getCurrentRawStream(index)


def _wanted(*tensors) -> bool:
    """Whether a derivative with respect to one of the tensors may be asked
    for: it requires a gradient, or carries a tangent (forward mode), of which
    requires_grad says nothing."""
    if _is_grad_enabled():
        for a in tensors:
            if a is not None and a.requires_grad:
                return True
    # The level is -1 outside forward mode, where looking for tangents costs time.
    return getattr(forward_ad, "_current_level", 0) >= 0 and any(
        a is not None and forward_ad.unpack_dual(a).tangent is not None for a in tensors)


class _NoDerivative(torch.autograd.Function):
    """An operator without a derivative: its results belong to the graph of
    its inputs, and a backward pass that reaches them raises."""

    @staticmethod
    def forward(ctx, name, call, *args):
        ctx.name = name
        out = call(*args)
        if isinstance(out, tuple):
            ctx.mark_non_differentiable(*(a for a in out if not a.is_floating_point()))
        return out

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError(f"{ctx.name} has no derivative: detach its inputs, or its results")


def quantize_rows(x):
    """Cuts each row of x (n x dim, float32, float16 or bfloat16) to signed
    8-bit codes with one scale: ``scales = max|x| / 127`` (float32) and
    ``codes = x / scales`` rounded to nearest, ties to even. Returns (codes
    int8 n x dim, scales float32 n); the rows of codes start on 16-byte
    boundaries, as ``int8_scores`` reads them. A row of zeros has scale 0; a
    row with a NaN or an infinity has scale NaN and codes 0. Codes stay within
    127 also where the scale is so small (below 1e-38) that it is itself
    rounded. Not differentiable: a backward pass that reaches the scales
    raises."""
    _not_traced("quantize_rows")
    _check(x, "x", 2, tuple(_TYPES))
    _dim(x, "x")
    return _NoDerivative.apply("quantize_rows", _quantize, x) if _wanted(x) else _quantize(x)


def _quantize(x):
    (n, dim), dev = x.shape, x.device
    x = _plain(x)
    codes = _empty_rows(n, dim, torch.int8, dev)
    scales = torch.empty(n, dtype=torch.float32, device=dev)
    if n:
        index = dev.index
        _lib.check(_lib.load().px_quantize_rows_device(
            index, x.data_ptr(), _TYPES[x.dtype], n, dim, _ld(x), codes.data_ptr(), codes.stride(0),
            scales.data_ptr(), _stream(index)))
    return codes, scales


def dequantize_rows(codes, scales, dtype=torch.float32):
    """The values 8-bit rows stand for: ``codes * scales[:, None]``, rounded
    once to ``dtype`` (float32, float16 or bfloat16). Not differentiable: a
    backward pass that reaches the result raises."""
    _not_traced("dequantize_rows")
    _check(codes, "codes", 2, (torch.int8,))
    _check(scales, "scales", 1, (torch.float32,))
    if dtype not in _TYPES:
        raise TypeError("argument 'dtype': expected float32, float16 or bfloat16")
    n, dim = codes.shape[0], _dim(codes, "codes")
    if scales.shape[0] != n:
        raise ValueError(f"scales length {scales.shape[0]} must equal the number of rows {n}")
    _same_device(codes.device, scales=scales)
    args = (codes, scales, dtype)
    return _NoDerivative.apply("dequantize_rows", _dequantize, *args) if _wanted(scales) else _dequantize(*args)


def _dequantize(codes, scales, dtype):
    n, dim = codes.shape
    codes, scales = _plain(codes), scales.contiguous()
    out = torch.empty((n, dim), dtype=dtype, device=codes.device)
    if n:
        _lib.check(_lib.load().px_dequantize_rows_device(
            codes.device.index, codes.data_ptr(), _ld(codes), scales.data_ptr(), n, dim, _TYPES[dtype],
            out.data_ptr(), dim, _stream(codes.device.index)))
    return out


def int8_scores(q_codes, q_scales, codes, scales, bias=None, dtype=torch.float32, out=None):
    """The score matrix of 8-bit queries (m x dim) and base rows (n x dim):
    ``(q_codes @ codes.T) * q_scales[:, None] * scales + bias`` as an m x n
    tensor of ``dtype`` (float32, float16 or bfloat16), the sums exact in
    32-bit integers (dim <= 131071). ``bias`` (float32, n) is added to each
    base row's scores; with ``bias = -0.5 * |row|^2`` scores order rows as L2
    distance does. ``out`` receives the result if given (its rows may be
    strided). Not differentiable: a backward pass that reaches the result
    raises, and with ``out`` no input may require a gradient."""
    _not_traced("int8_scores")
    _check(q_codes, "q_codes", 2, (torch.int8,))
    _check(q_scales, "q_scales", 1, (torch.float32,))
    _check(codes, "codes", 2, (torch.int8,))
    _check(scales, "scales", 1, (torch.float32,))
    if bias is not None:
        _check(bias, "bias", 1, (torch.float32,))
    if dtype not in _TYPES:
        raise TypeError("argument 'dtype': expected float32, float16 or bfloat16")
    (m, dim), n, dev = q_codes.shape, codes.shape[0], codes.device
    _dim(q_codes, "q_codes")
    if codes.shape[1] != dim:
        raise ValueError(f"query dim {dim} does not match row dim {codes.shape[1]}")
    if dim > _INT8_MAX_DIM:
        raise ValueError(f"dim={dim} exceeds {_INT8_MAX_DIM}: a sum of 8-bit products could pass 32 bits")
    if q_scales.shape[0] != m:
        raise ValueError(f"q_scales length {q_scales.shape[0]} must equal the number of queries {m}")
    if scales.shape[0] != n:
        raise ValueError(f"scales length {scales.shape[0]} must equal the number of rows {n}")
    if bias is not None and bias.shape[0] != n:
        raise ValueError(f"bias length {bias.shape[0]} must equal the number of rows {n}")
    _same_device(dev, q_codes=q_codes, q_scales=q_scales, scales=scales, bias=bias, out=out)
    if out is not None:
        _check(out, "out", 2, (dtype,))
        if out.shape != (m, n):
            raise ValueError(f"out has shape {tuple(out.shape)}, expected {(m, n)}")
        if out.requires_grad:
            raise ValueError("out must not require a gradient")
        if n > 1 and out.stride(1) != 1 or m > 1 and out.stride(0) < n:
            raise ValueError("out must have contiguous columns and rows that do not overlap")
    args = (q_codes, q_scales, codes, scales, bias, dtype, out)
    if not _wanted(q_scales, scales, bias):
        return _scores(*args)
    if out is not None:
        raise ValueError("out cannot be given where a derivative may be asked for: detach the scales and the bias")
    return _NoDerivative.apply("int8_scores", _scores, *args)


def _scores(q_codes, q_scales, codes, scales, bias, dtype, out):
    (m, dim), n, dev = q_codes.shape, codes.shape[0], codes.device
    if out is None:
        out = torch.empty((m, n), dtype=dtype, device=dev)
    if m and n:
        (qc, ldq), (xc, ldx) = _tiled(q_codes), _tiled(codes)
        qs, xs = q_scales.contiguous(), scales.contiguous()
        b = None if bias is None else bias.contiguous()
        _lib.check(_lib.load().px_int8_scores_device(
            dev.index, qc.data_ptr(), ldq, qs.data_ptr(), m, xc.data_ptr(), ldx, xs.data_ptr(), n, dim, _ptr(b),
            _TYPES[dtype], out.data_ptr(), _ld(out), _stream(dev.index)))
    return out


def _xent_forward(queries, rows, targets, scale, bias, ignore_index, reduction):
    """The loss, and what the backward needs: the operands as the tensor cores
    read them, and the buffer that holds each query's loss and lse and the
    reduction's divisor."""
    lib, dev = _lib.load(), queries.device
    (t, dim), v, index = queries.shape, rows.shape[0], dev.index
    q, ldq = _tiled(queries)
    r, ldr = _tiled(rows)
    targets, bias = targets.contiguous(), _aligned(bias)
    part = (4 * t + 255) // 256 * 256  # bytes of one float per query
    need = lib.px_softmax_xent_workspace_bytes(index, t, v, dim, 0)
    kept = torch.empty(2 * part + 256, dtype=torch.uint8, device=dev)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    out = torch.empty(() if reduction else t, dtype=torch.float32, device=dev)
    base = kept.data_ptr()
    loss = base if reduction else out.data_ptr()
    _lib.check(lib.px_softmax_xent_device(
        index, q.data_ptr(), ldq, t, r.data_ptr(), ldr, v, dim, _TYPES[q.dtype], targets.data_ptr(), ignore_index, scale,
        _ptr(bias), reduction, loss, base + part, out.data_ptr() if reduction else None,
        base + 2 * part if reduction else None, ws.data_ptr(), need, _stream(index)))
    return out, (q, ldq, r, ldr, targets, bias, kept, part)


class _SoftmaxCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, queries, rows, targets, scale, bias, ignore_index, reduction):
        out, (q, ldq, r, ldr, targets, bias, kept, part) = _xent_forward(queries, rows, targets, scale, bias,
                                                                         ignore_index, reduction)
        ctx.save_for_backward(q, r, targets, bias, kept, None if reduction else out)
        ctx.args = (ldq, ldr, part, scale, ignore_index, reduction)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        lib = _lib.load()
        q, r, targets, bias, kept, out = ctx.saved_tensors
        ldq, ldr, part, scale, ignore_index, reduction = ctx.args
        (t, dim), v, dev = q.shape, r.shape[0], q.device
        index = dev.index
        want_q, want_r = ctx.needs_input_grad[:2]
        dq = torch.empty((t, dim), dtype=q.dtype, device=dev) if want_q else None
        dr = torch.empty((v, dim), dtype=r.dtype, device=dev) if want_r else None
        stride = 0 if reduction or (t > 1 and grad.stride(0) == 0) else 1
        if stride:
            grad = grad.contiguous()
        base = kept.data_ptr()
        need = lib.px_softmax_xent_workspace_bytes(index, t, v, dim, 1)
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        _lib.check(lib.px_softmax_xent_backward_device(
            index, q.data_ptr(), ldq, t, r.data_ptr(), ldr, v, dim, _TYPES[q.dtype], targets.data_ptr(), ignore_index,
            scale, _ptr(bias), base if reduction else out.data_ptr(), base + part, grad.data_ptr(), stride,
            base + 2 * part if reduction else None, _ptr(dq), dim, _ptr(dr), dim, ws.data_ptr(), need, _stream(index)))
        return dq, dr, None, None, None, None, None


def softmax_cross_entropy(queries, rows, targets, scale=1.0, bias=None, ignore_index=-100, reduction="mean"):
    """Cross entropy of queries (t x dim) under a softmax over all base rows
    (v x dim), both float16 or bfloat16, without keeping the t x v logits
    ``scale * queries @ rows.T + bias``: ``log sum_j exp z_ij - z_i,target``,
    float32. Differentiable (once, backward) in queries and rows; the backward
    computes the logits again, in pieces of the base.

    targets: int64, row numbers; ``ignore_index`` gives a query loss 0 and no
    gradient, any other number outside [0, v) loss NaN and no gradient. bias
    (float32, v, no gradient): added to a row's logits, for instance the
    correction for how rows were sampled; -inf (or any value below -2e31)
    leaves a row out; above 1e31 it
    makes losses NaN. scale: a positive number (one over the temperature). reduction: "mean" (over the
    queries not ignored; NaN if there are none), "sum" or "none". Queries and
    rows must be finite even where ignored or left out. With float16 the
    gradients of one call's losses should lie within a few orders of magnitude:
    what is below 2^-39 of the largest is lost."""
    _not_traced("softmax_cross_entropy")
    _check(queries, "queries", 2, (torch.float16, torch.bfloat16))
    _check(rows, "rows", 2, (queries.dtype,))
    _check(targets, "targets", 1, (torch.int64,))
    if bias is not None:
        _check(bias, "bias", 1, (torch.float32,))
        if bias.requires_grad:
            raise ValueError("bias has no gradient: pass bias.detach()")
    scale = float(scale)
    if not scale > 0.0 or math.isinf(scale):
        raise ValueError("scale must be positive and finite")
    if scale >= 2.0 ** 127:
        raise ValueError("scale must be below 2^127")
    ignore_index = int(ignore_index)
    if not -2 ** 63 <= ignore_index < 2 ** 63:
        raise ValueError("ignore_index must be a 64-bit integer")
    if reduction not in _REDUCTIONS:
        raise ValueError("reduction must be 'none', 'sum' or 'mean'")
    if _dim(queries, "queries") != rows.shape[1]:
        raise ValueError(f"query dim {queries.shape[1]} does not match row dim {rows.shape[1]}")
    if rows.shape[0] == 0:
        raise ValueError("a softmax needs at least one base row")
    if targets.shape[0] != queries.shape[0]:
        raise ValueError(f"targets length {targets.shape[0]} must equal the number of queries {queries.shape[0]}")
    if bias is not None and bias.shape[0] != rows.shape[0]:
        raise ValueError(f"bias length {bias.shape[0]} must equal the number of rows {rows.shape[0]}")
    _same_device(queries.device, rows=rows, targets=targets, bias=bias)
    if queries.shape[0] == 0:
        # No query: an empty loss, or the sum or mean of one, with zero gradients.
        loss = queries.float().sum(1) + rows[:0].float().sum()
        return {"none": lambda: loss, "sum": loss.sum, "mean": loss.mean}[reduction]()
    args = (queries, rows, targets, scale, bias, ignore_index, _REDUCTIONS[reduction])
    if _wanted(queries, rows, bias):
        return _SoftmaxCrossEntropy.apply(*args)
    return _xent_forward(*args)[0]


def rows_status(device=None) -> None:
    """Waits for the device's current stream and raises PxError (ETIMEOUT) if
    a bounded device-side wait of one of these operators has given up since
    the last call; the results it left undone are NaN. The record is one per
    device, for all streams and threads, and the call clears it."""
    device = torch.device("cuda", torch.cuda.current_device() if device is None else torch.device(device).index)
    _lib.check(_lib.load().px_rows_status_device(device.index, _stream(device.index)))
