"""Training with `sageattn`: its backward pass.

    out = sageattn_train(q, k, v, is_causal=True)      # as sageattn, recorded by autograd
    out.backward(dout)

`sageattn_backward` is the pass itself. It recomputes the probabilities in 16 bits from Q and K (the
forward call's 8-bit codes are not kept) and from their logsumexp, which it works out, too, or is
given where the keys are part of a larger set. It takes one to four launches on the current stream and
synchronizes nothing, so that it can be captured into a graph. A call that is not served raises
`ValueError` with the reason.
"""
import torch

from .cache import _DTYPES, _HEAD_DIMS, _empty, _gradient, _launch, _library, _refuse, _view
from .core import sageattn

#: what the scores' factor may be (a logsumexp is divided by it)
_LEAST_SCALE = 1e-30


def _row_floats(what, name, t, shape, device):
    """Checks a contiguous fp32 tensor of one value per row."""
    if not isinstance(t, torch.Tensor) or t.device != device:
        _refuse(what, "device: %s must be a tensor on %s" % (name, device))
    if t.dtype != torch.float32:
        _refuse(what, "dtype: %s must be float32 (got %s)" % (name, t.dtype))
    if t.shape != shape:
        _refuse(what, "shape: %s is %s, not %s" % (name, tuple(t.shape), shape))
    if not t.is_contiguous():
        _refuse(what, "stride_last: %s must be contiguous" % name)


def _scale(what, sm_scale, D):
    """The scores' factor."""
    sm = D ** -0.5 if sm_scale is None else float(sm_scale)
    if not _LEAST_SCALE <= sm <= 1 / _LEAST_SCALE:
        _refuse(what, "sm_scale: must lie between 1e-30 and 1e30 (got %r)" % (sm_scale,))
    return sm


def _plain(tensors, tensor_layout):
    """Whether all are contiguous GPU tensors of one served dtype, of one device, of a served head_dim, which
    need no closer look."""
    if tensor_layout != "HND" and tensor_layout != "NHD":
        return False
    first = tensors[0]
    if not isinstance(first, torch.Tensor) or first.dtype not in _DTYPES or not first.is_cuda:
        return False
    dtype, device = first.dtype, first.device
    for t in tensors:
        if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.device != device \
                or not t.is_contiguous() or t.data_ptr() & 15:
            return False
        shape = t.shape
        if len(shape) != 4 or shape[3] not in _HEAD_DIMS or 0 in shape:
            return False
    return True


def _strides(t, nhd):
    sb, s1, s2, _ = t.stride()
    return (sb, s2, s1) if nhd else (sb, s1, s2)


def sageattn_backward(dout, q, k, v, out=None, lse=None, tensor_layout="HND", is_causal=False, sm_scale=None,
                      dlse=None):
    """The gradients `(dq, dk, dv)` of `sageattn(q, k, v, ...)` from `dout`, that of its output.

    q, k, v, tensor_layout, is_causal, sm_scale: as the forward call had them. dlse (B, H, N) fp32: the
    gradient of the logsumexp, where the caller used it. out and dout have q's shape and dtype (any strides
    that `sageattn` takes, rows less than 2^24 elements apart), the gradients are contiguous, of q's, k's and
    v's shapes and dtype.

    out, lse: left out after `sageattn`, whose output and logsumexp are those of 8-bit scores; the pass
    works out those of the 16-bit scores that it forms, two products more to its seven. Given together they
    are attention's in 16 bits or more (a logsumexp under its scores leaves results finite: weights end at
    4 in fp16). Keys that are one part of those a query sees (attention over parts,
    merged by their logsumexp) have their gradients from calls with the merged out and lse, a call for each
    part; dq is the calls' sum. A row with a logsumexp of -infinity saw nothing and counts for nothing. Values have to be finite,
    those of a padded batch's unused rows too: 0 times a NaN or an infinity is NaN. fp16 needs a loss scale only
    where dout or the gradients themselves leave its range; dK loses bits of rows whose gradient is some 2^15 under the
    largest row's of the heads that share a key.
    """
    what = "sageattn_backward"
    anew = out is None and lse is None
    # (dout in the place of an out that is not given: checked twice)
    read = (q, k, v, dout if anew else out, dout)
    plain = _plain(read, tensor_layout)
    if not plain:
        if not anew and (out is None or lse is None):
            _refuse(what, "out: out and lse are given together or not at all")
        for name, t in zip(("q", "k", "v", "dout" if anew else "out", "dout"), read):
            _view(what, tensor_layout, name, t)
        for name, t in zip(("k", "v", "dout" if anew else "out", "dout"), read[1:]):
            if t.device != q.device:
                _refuse(what, "device: %s is on %s, q on %s" % (name, t.device, q.device))
            if t.dtype != q.dtype:
                _refuse(what, "dtype: %s is %s, q %s" % (name, t.dtype, q.dtype))
    dev, dtype, shape = q.device, q.dtype, q.shape
    if k.shape != v.shape:
        _refuse(what, "shape: k is %s, v %s" % (tuple(k.shape), tuple(v.shape)))
    for name, t in (("dout" if anew else "out", read[3]), ("dout", dout)):
        if t.shape != shape:
            _refuse(what, "shape: %s is %s, q %s" % (name, tuple(t.shape), tuple(shape)))
    if tensor_layout == "HND":
        (B, H, N, D), (B_kv, H_kv, N_kv, D_kv) = shape, k.shape
    else:
        (B, N, H, D), (B_kv, N_kv, H_kv, D_kv) = shape, k.shape
    if B_kv != B or D_kv != D:
        _refuse(what, "shape: k is %s, q %s" % (tuple(k.shape), tuple(shape)))
    if H % H_kv:
        _refuse(what, "heads: %d query heads on %d K/V heads" % (H, H_kv))
    if is_causal and N != N_kv:
        _refuse(what, "seq_len: causal attention needs as many queries as keys (%d, %d)" % (N, N_kv))
    if not anew:
        _row_floats(what, "lse", lse, (B, H, N), dev)
    if dlse is not None:
        _row_floats(what, "dlse", dlse, (B, H, N), dev)
    sm = _scale(what, sm_scale, D)
    lib = _library(what, dev)
    grads = (_empty(q), _empty(k), _empty(v))
    size = lib.attn_bwd_workspace_bytes(dtype, bool(is_causal), B, H, N, H_kv, N_kv, D, anew)
    work = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    nhd = tensor_layout == "NHD"
    # (batch, head, row) strides: of contiguous tensors by their sizes
    rows, rows_kv = ((N * H * D, D, H * D), (N_kv * H_kv * D, D, H_kv * D)) if nhd else \
        ((H * N * D, N * D, D), (H_kv * N_kv * D, N_kv * D, D))
    whole = (rows, rows_kv, rows_kv, rows, rows)
    strides = whole if plain else [_strides(t, nhd) for t in read]
    if anew:
        read = (q, k, v, None, dout)
    _launch(dev, lib.attn_bwd, dtype, is_causal, read, strides, grads, whole[:3], lse, dlse,
            (B, H, N, H_kv, N_kv, D), sm, work, size)
    return grads


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, tensor_layout, is_causal, sm_scale, options):
        out, lse = sageattn(q, k, v, tensor_layout, is_causal, sm_scale, return_lse=True, **options)
        ctx.save_for_backward(q, k, v)
        ctx.call = (tensor_layout, bool(is_causal), sm_scale)
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, dlse):
        q, k, v = ctx.saved_tensors
        if dout is None and dlse is None:
            return (None,) * 7
        dout = q.new_zeros(q.shape) if dout is None else _gradient(dout)
        return sageattn_backward(dout, q, k, v, None, None, *ctx.call, dlse=_gradient(dlse)) + (None,) * 4


def sageattn_train(q, k, v, tensor_layout="HND", is_causal=False, sm_scale=None, return_lse=False,
                   **kwargs):
    """`sageattn` as an operation that autograd records: the same arguments and results, with gradients
    to q, k and v (from the logsumexp's gradient too, with `return_lse`).

    The gradients are those of attention itself on q, k and v: the forward call's rounding to 8 bits counts as
    the identity. Of the forward call nothing but q, k and v is kept. Gradients of gradients are not served. To
    capture a training step into a graph, capture `sageattn` and `sageattn_backward`, or a forward pass with `torch.autograd.grad`:
    gradients that autograd adds up in leaves (`backward()`) belong to the stream that first used the leaf.
    """
    _scale("sageattn_train", sm_scale, 1)
    out, lse = _Attention.apply(q, k, v, tensor_layout, is_causal, sm_scale, kwargs)
    return (out, lse) if return_lse else out
