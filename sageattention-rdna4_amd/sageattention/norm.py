"""The root-mean-square norm around attention: with the residual's addition, 8-bit outputs, and gradients.

    y, hidden = rms_norm(x, weight, eps, residual=hidden)          # recorded by autograd
    codes, scales, hidden = rms_norm_quant(x, weight, eps, residual=hidden)
    q = rms_norm(q, q_weight, eps)                                 # heads, from a fused projection's view

Each is one launch on the current stream (gradients two) that reads every row once, works in fp32,
synchronizes nothing, and can be captured into a graph. Codes and scales follow the quantizers of this
package: one scale per row, int8 for fp16 or e4m3. A call that is not served raises `ValueError` with
the reason.
"""
import math

import torch
from torch.autograd import forward_ad

from .cache import _DTYPES, _gradient, _launch, _library, _refuse

_NONE = (0, 0, 0)


def _layout(what, tensors):
    """The row dimensions (d0, d1, d2) that the tensors, all of one shape, have in common, and each one's
    strides in them."""
    shape = tensors[0][1].shape
    together = True
    for name, t in tensors:
        if t.data_ptr() & 15:
            _refuse(what, "ptr_align: %s must be 16-byte aligned" % name)
        if not t.is_contiguous():
            together = False
            if t.stride(-1) != 1:
                _refuse(what, "stride_last: %s must have contiguous rows" % name)
    n = shape[-1]
    if together:
        return (1, 1, tensors[0][1].numel() // n), [(0, 0, n)] * len(tensors)
    names, tensors = zip(*tensors)
    dims, strides = [], [[] for _ in tensors]
    for i, size in enumerate(shape[:-1]):
        if size == 1:
            continue
        step = [t.stride(i) for t in tensors]
        if dims and all(s[-1] == st * size for s, st in zip(strides, step)):
            dims[-1] *= size               # this dimension continues the one before in every tensor
            for s, st in zip(strides, step):
                s[-1] = st
        else:
            dims.append(size)
            for s, st in zip(strides, step):
                s.append(st)
    if len(dims) > 3:
        _refuse(what, "strides: rows lie in more than three dimensions %s" % (tuple(dims),))
    for name, s in zip(names, strides):
        if any(st & 7 for st in s):
            _refuse(what, "stride_align: strides of %s must be multiples of 8 elements" % name)
    pad = 3 - len(dims)
    return tuple([1] * pad + dims), [tuple([0] * pad + s) for s in strides]


def _check(what, x, weight, others):
    """Checks the rows, the weight, and tensors of the rows' shape."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        _refuse(what, "device: x must be a tensor on the GPU")
    if x.dtype not in _DTYPES:
        _refuse(what, "dtype: x is %s (fp16 and bf16 are served)" % x.dtype)
    shape, dev = x.shape, x.device
    n = shape[-1] if shape else 0
    if n % 8 or not 8 <= n <= 16384:
        _refuse(what, "row: x is %s (rows of a multiple of 8 values up to 16384 are served)" % (
            tuple(shape),))
    if not isinstance(weight, torch.Tensor) or weight.device != dev:
        _refuse(what, "device: weight must be a tensor on %s" % dev)
    if weight.dtype not in (x.dtype, torch.float32):
        _refuse(what, "dtype: weight is %s (x's %s and float32 are served)" % (weight.dtype, x.dtype))
    if weight.shape != shape[-1:]:
        _refuse(what, "shape: weight is %s, not %s" % (tuple(weight.shape), tuple(shape[-1:])))
    if not weight.is_contiguous():
        _refuse(what, "stride_last: weight must be contiguous")
    if weight.data_ptr() & 15:
        _refuse(what, "ptr_align: weight must be 16-byte aligned")
    for name, t in others:
        if not isinstance(t, torch.Tensor) or t.device != dev:
            _refuse(what, "device: %s must be a tensor on %s" % (name, dev))
        if t.dtype != x.dtype:
            _refuse(what, "dtype: %s is %s, x %s" % (name, t.dtype, x.dtype))
        if t.shape != shape:
            _refuse(what, "shape: %s is %s, x %s" % (name, tuple(t.shape), tuple(shape)))


def _new(x, dtype, whole):
    """A new contiguous tensor of x's shape, or of a value per row."""
    if whole and x.is_contiguous() and dtype is x.dtype:
        return torch.empty_like(x)
    return torch.empty(x.shape if whole else x.shape[:-1], dtype=dtype, device=x.device)


def _norm(what, x, weight, eps, residual, out, keep_rstd):
    """The launch: (y, scales or None, sum or None, rstd or None)."""
    others = [] if residual is None else [("residual", residual)]
    _check(what, x, weight, others)
    eps = float(eps)
    if not 0.0 <= eps < math.inf:
        _refuse(what, "eps: must be finite and not negative (got %r)" % (eps,))
    dev, dtype = x.device, x.dtype
    y = _new(x, (dtype, torch.int8, torch.float8_e4m3fn)[out], True)
    scales = _new(x, torch.float32, False) if out else None
    total = None if residual is None else _new(x, dtype, True)
    rstd = _new(x, torch.float32, False) if keep_rstd else None
    lib = _library(what, dev)
    if x.numel():
        dims, strides = _layout(what, [("x", x)] + others)
        _launch(dev, lib.rms_norm, x, strides[0], residual, _NONE if residual is None else strides[1],
                weight, dims, x.shape[-1], eps, out, y, scales, total, rstd)
    return y, scales, total, rstd


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps, residual):
        y, _, total, rstd = _norm("rms_norm", x, weight, eps, residual, 0, True)
        ctx.save_for_backward(x if residual is None else total, weight, rstd)
        ctx.residual = residual is not None
        ctx.set_materialize_grads(False)
        return (y, total) if ctx.residual else y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dsum=None):
        t, weight, rstd = ctx.saved_tensors
        if dy is None:                     # only the sum was used
            return dsum, None, None, dsum
        dx, dw = rms_norm_backward(_gradient(dy), t, weight, rstd, _gradient(dsum))
        return dx, dw, None, dx if ctx.residual else None


def rms_norm(x, weight, eps=1e-6, residual=None, return_rstd=False):
    """x / sqrt(mean(x^2) + eps) * weight over the last dimension; with `residual`, of x + residual, and
    `(y, x + residual)` is returned.

    x: fp16 or bf16, any number of dimensions, rows of a multiple of 8 values up to 16384; rows may lie
    apart (a view of a fused projection), in three dimensions at most. residual: x's shape and dtype.
    weight: (n,) of x's dtype or fp32. The sum is added, normed and scaled in fp32; y and the sum (new,
    contiguous, of x's shape and dtype) are each rounded once. Autograd records the call where x, weight or
    residual need a gradient. `return_rstd` appends 1 / sqrt(...) of each row (fp32, x's shape without
    the last dimension), for `rms_norm_backward`; such a call is not recorded. Forward-mode tangents are
    refused (`NotImplementedError`).
    """
    # (a forward-mode tangent, which needs no gradient, is refused there)
    if not return_rstd and (forward_ad._current_level >= 0 or torch.is_grad_enabled() and (
            getattr(x, "requires_grad", False) or getattr(weight, "requires_grad", False)
            or getattr(residual, "requires_grad", False))):
        return _RmsNorm.apply(x, weight, eps, residual)
    y, _, total, rstd = _norm("rms_norm", x, weight, eps, residual, 0, return_rstd)
    done = (y,) if residual is None else (y, total)
    if return_rstd:
        done += (rstd,)
    return done if len(done) > 1 else y


def rms_norm_quant(x, weight, eps=1e-6, residual=None, int8=None):
    """`rms_norm` with the result as 8-bit codes: `(codes, scales)`, with `residual` `(codes, scales, sum)`.

    codes: x's shape, int8 (`int8=True`, the default for fp16) or float8_e4m3fn; scales: fp32, x's shape
    without the last dimension. codes * scale stands for the norm's fp32 result, rounded once: scale =
    max(max|y| / 127 or 448, 1e-12). A row that holds a NaN or an infinity has zero codes and a NaN scale.
    No gradients: autograd records nothing here.
    """
    if int8 is None:
        int8 = isinstance(x, torch.Tensor) and x.dtype == torch.float16
    y, scales, total, _ = _norm("rms_norm_quant", x, weight, eps, residual, 1 if int8 else 2, False)
    return (y, scales) if residual is None else (y, scales, total)


def rms_norm_backward(dy, x, weight, rstd, dsum=None):
    """The gradients `(dx, dweight)` of `rms_norm` from `dy`, that of its result.

    x: the rows that were normed, the returned sum where there was a residual (dx is then the gradient of
    both). rstd: as `return_rstd` gave it. dsum: the gradient of the returned sum, added to dx. dx has x's
    shape and dtype, contiguous; dweight weight's dtype, summed in fp32 and the same from call to call.
    """
    what = "rms_norm_backward"
    others = [("dy", dy)] + ([] if dsum is None else [("dsum", dsum)])
    _check(what, x, weight, others)
    dev = x.device
    if not isinstance(rstd, torch.Tensor) or rstd.device != dev:
        _refuse(what, "device: rstd must be a tensor on %s" % dev)
    if rstd.dtype != torch.float32 or rstd.shape != x.shape[:-1] or not rstd.is_contiguous():
        _refuse(what, "rstd: a contiguous float32 tensor of shape %s is needed" % (tuple(x.shape[:-1]),))
    lib = _library(what, dev)
    dx = _new(x, x.dtype, True)
    if not x.numel():
        return dx, torch.zeros_like(weight)
    dw = torch.empty_like(weight)
    dims, strides = _layout(what, [("x", x)] + others)
    n = x.shape[-1]
    work = torch.empty(lib.rms_norm_bwd_workspace_bytes(x.numel() // n, n), dtype=torch.uint8, device=dev)
    _launch(dev, lib.rms_norm_bwd, dy, strides[1], x, strides[0], dsum,
            _NONE if dsum is None else strides[2], weight, rstd, dims, n, dx, dw, work)
    return dx, dw
