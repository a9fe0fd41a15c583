"""Serving from a quantized K/V cache: rotary positions, the paged cache, attention over it.

    table = rotary_table(32768, 128, device="cuda")
    cache = KVCache.allocate(num_pages=4096, num_heads=8, head_dim=128, dtype=torch.float16)
    # a step: rotate the queries, put the new tokens' K and V into the cache, attend to all of it
    q = apply_rotary(q, table, positions)
    cache.write(k, v, block_table, lens, table=table, positions=positions)
    o = sageattn_cached(q, cache, block_table, lens + n)

`sageattn` quantizes the K and V of each call; a program that decodes keeps them quantized instead, by
the same scheme (K int8 for fp16 or e4m3, V e4m3, a scale per token and head, no smoothing: a mean over
the sequence is not known while it grows). Every call is one or two launches on the current stream,
synchronizes nothing and reads no length on the host, so that a step can be captured into a graph and
replayed as the sequences grow. Tensors are checked as `sageattn` checks its own: a call that is not
served raises `ValueError` with the reason.

A sequence's tokens lie in pages of 64 that `block_table` (B, max_pages) int32 numbers: position p in
page `block_table[b, p // 64]`. A number outside the pool (-1, say) names no page: nothing is written
there, zeros are read from it, and nobody attends to it. A row of K or V that holds a NaN or an
infinity is held as NaN: so come out the rows that attend to it, and only they.
"""
import math

import torch

from . import sk1_backend as _sk1
from .sk1_backend.sk1_loader import SageLib, strided_view_reason, torch_stream

PAGE = 64

_HEAD_DIMS = (64, 128)
_DTYPES = (torch.float16, torch.bfloat16)

#: device index -> the library, once the device is known to be served
_LIBRARIES = {}


def _refuse(what, reason):
    raise ValueError("%s: %s" % (what, reason))


def _library(what, device):
    """The library, where it serves this device."""
    lib = _LIBRARIES.get(device.index)
    if lib is None:
        if not _sk1.arch_supported(device):
            raise RuntimeError("%s: device arch is %r; libsagemi355.so is built for %s" % (
                what, _sk1.device_arch(device) or "<unknown>", ", ".join(_sk1.SUPPORTED_ARCHS)))
        lib = _LIBRARIES[device.index] = SageLib.get()
    return lib


def _launch(device, call, *args):
    """The call on the device's current stream, with the device current."""
    if device.index == torch.cuda.current_device():
        call(*args, torch_stream(device))
    else:
        with torch.cuda.device(device):
            call(*args, torch_stream(device))


def _view(what, tensor_layout, name, t):
    """The tensor as a (B, H, N, D) view of a served dtype and head_dim."""
    if tensor_layout != "HND" and tensor_layout != "NHD":
        _refuse(what, "layout: tensor_layout must be HND or NHD (got %r)" % (tensor_layout,))
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        _refuse(what, "device: %s must be a tensor on the GPU" % name)
    if t.dim() != 4:
        _refuse(what, "rank: %s must have 4 dimensions (got %d)" % (name, t.dim()))
    if t.dtype not in _DTYPES:
        _refuse(what, "dtype: %s is %s (fp16 and bf16 are served)" % (name, t.dtype))
    if not t.numel():
        _refuse(what, "seq_len: %s is empty %s" % (name, tuple(t.shape)))
    if t.shape[3] not in _HEAD_DIMS:
        _refuse(what, "head_dim: %s has %d (64 and 128 are served)" % (name, t.shape[3]))
    if tensor_layout == "NHD":
        t = t.transpose(1, 2)
    reason = strided_view_reason(t, name)
    if reason is not None:
        _refuse(what, "%s: %s %s" % (reason, name, tuple(t.stride())))
    return t


def _empty(like):
    """A new contiguous tensor of `like`'s shape, dtype and device."""
    return torch.empty_like(like) if like.is_contiguous() else like.new_empty(like.shape)


def _ints(what, name, t, device, rows, columns=None):
    """Checks an int32 tensor (rows,), or (rows, columns) with contiguous rows (columns -1: any);
    returns the elements between two rows, 0 where there is one."""
    if not isinstance(t, torch.Tensor) or t.device != device:
        _refuse(what, "device: %s must be a tensor on %s" % (name, device))
    if t.dtype != torch.int32:
        _refuse(what, "dtype: %s must be int32 (got %s)" % (name, t.dtype))
    shape = t.shape
    if columns is None:
        if len(shape) != 1 or shape[0] != rows:
            _refuse(what, "shape: %s is %s, not (%d,)" % (name, tuple(shape), rows))
        if rows > 1 and t.stride(0) != 1:
            _refuse(what, "stride_last: %s must be contiguous" % name)
        return 0
    if len(shape) != 2 or shape[0] != rows or columns not in (-1, shape[1]) or shape[1] < 1:
        _refuse(what, "shape: %s is %s, not (%d, %s)" % (
            name, tuple(shape), rows, "..." if columns < 0 else columns))
    step, last = t.stride()
    if last != 1 and shape[1] > 1:
        _refuse(what, "stride_last: %s must have contiguous rows" % name)
    if rows == 1:
        return 0
    if step < shape[1] and step != 0:
        _refuse(what, "stride_overlap: rows of %s overlap" % name)
    return step


def _check_table(what, table, positions, device, B, N, D):
    """Checks a rotary table and positions; returns the elements between two rows of positions."""
    if not isinstance(table, torch.Tensor) or table.device != device:
        _refuse(what, "device: table must be a tensor on %s" % device)
    if table.dtype != torch.float32 or table.dim() != 2 or not table.is_contiguous() \
            or table.data_ptr() & 15:
        _refuse(what, "table: a contiguous fp32 (positions, R) tensor is needed, as rotary_table's")
    rows, R = table.shape
    if rows < 1 or R % 16 or not 16 <= R <= D:
        _refuse(what, "table: %s: R must be a multiple of 16 up to the head_dim %d" % (
            tuple(table.shape), D))
    if isinstance(positions, torch.Tensor) and positions.dim() == 1:
        return _ints(what, "positions", positions, device, N)
    return _ints(what, "positions", positions, device, B, N)


def rotary_table(length, dim, base=10000.0, *, scaling=None, factor=1.0, original_length=None,
                 device="cuda"):
    """The fp32 (length, dim) table of `apply_rotary` and `KVCache.write`: cosines of dim/2
    frequencies base^(-2i/dim) at each position, then their sines, worked out in 64 bits.

    `scaling` stretches it for contexts `factor` times as long as the trained one:
    "linear" divides positions by factor; "ntk" raises the base to base * factor^(dim/(dim-2)), which
    leaves the fastest frequency and divides the slowest by factor; "yarn" divides the frequencies that
    turn less than once over `original_length` positions, keeps those that turn 32 times or more, blends
    between (linearly in the frequency's index), and scales the rotated vectors by 0.1 ln(factor) + 1.
    """
    what = "rotary_table"
    if length < 1 or dim < 16 or dim % 16:
        _refuse(what, "length must be positive and dim a multiple of 16 (got %r, %r)" % (length, dim))
    if scaling not in (None, "linear", "ntk", "yarn"):
        _refuse(what, "scaling must be None, 'linear', 'ntk' or 'yarn' (got %r)" % (scaling,))
    if not factor >= 1.0 or not base > 1.0:
        _refuse(what, "factor must be at least 1 and base over 1 (got %r, %r)" % (factor, base))
    if scaling == "yarn" and (original_length is None or original_length < 1):
        _refuse(what, "'yarn' needs the original_length")
    position = torch.arange(length, dtype=torch.float64, device=device)
    index = torch.arange(dim // 2, dtype=torch.float64, device=device)
    if scaling == "ntk":
        base = base * factor ** (dim / (dim - 2))
    freq = base ** (-2.0 * index / dim)
    size = 1.0
    if scaling == "linear":
        position = position / factor
    elif scaling == "yarn":
        def index_of(turns):   # the (real) index of the frequency that turns so often
            return dim * math.log(original_length / (turns * 2 * math.pi)) / (2 * math.log(base))
        low = max(math.floor(index_of(32.0)), 0)
        high = min(math.ceil(index_of(1.0)), dim - 1)
        blend = ((index - low) / max(high - low, 1e-3)).clamp(0.0, 1.0)
        freq = freq * (1.0 - blend) + freq / factor * blend
        size = 0.1 * math.log(factor) + 1.0
    angle = position[:, None] * freq
    return (size * torch.cat((angle.cos(), angle.sin()), 1)).float()


def apply_rotary(x, table, positions, tensor_layout="HND", interleaved=False, inverse=False):
    """x with rotary positions applied, as a new tensor of the same layout and dtype.

    x: (B, H, N, D) for `tensor_layout="HND"` or (B, N, H, D) for "NHD", D = 64 or 128, fp16 or bf16.
    table: fp32 (rows, R), `rotary_table`'s; the first R columns of each head are rotated (R a multiple
    of 16), the others copied. positions: int32 (B, N), or (N,) for all sequences alike; where one lies
    outside the table, the rotated columns are NaN. A pair (a, b), columns (i, i + R/2) or, `interleaved`,
    (2i, 2i + 1), becomes (a c - b s, b c + a s), in fp32 with one rounding to x's dtype at the end.
    `inverse` turns by the negative angle: the gradient of x from that of the result (autograd records
    neither this call nor the others here). It gives x back from the result where the table's pairs are of
    size 1; a "yarn" table's are larger, and x comes back times their size squared.
    """
    what = "apply_rotary"
    xx = _view(what, tensor_layout, "x", x)
    B, _, N, D = xx.shape
    dev = x.device
    p_sb = _check_table(what, table, positions, dev, B, N, D)
    lib = _library(what, dev)
    out = _empty(x)
    _launch(dev, lib.rotary, xx, out if tensor_layout == "HND" else out.transpose(1, 2), table,
            positions, p_sb, interleaved, inverse)
    return out


class KVCache:
    """A pool of pages of 64 tokens' quantized K and V rows, and the calls that fill and read it.

    k8 (num_pages, num_heads, 64, head_dim) int8 or float8_e4m3fn, v8 likewise float8_e4m3fn, sk and sv
    (num_pages, num_heads, 64) fp32: the rows' codes and scales. `dtype` (fp16 or bf16) is that of the
    tensors which are written and read and of the queries; int8 keys are for fp16, as in `sageattn`.
    The tensors are the caller's to keep, copy or share; codes hold no NaN as long as `write` makes
    them. Which pages a sequence has is the caller's too: every call takes a `block_table`.
    """

    def __init__(self, k8, sk, v8, sv, dtype=torch.float16):
        what = "KVCache"
        if dtype not in (torch.float16, torch.bfloat16):
            _refuse(what, "dtype: %s is not served (fp16 and bf16 only)" % dtype)
        for name, t in (("k8", k8), ("sk", sk), ("v8", v8), ("sv", sv)):
            if not isinstance(t, torch.Tensor) or not t.is_cuda or t.device != k8.device:
                _refuse(what, "device: %s must be a tensor on the pool's GPU" % name)
            if not t.is_contiguous() or t.data_ptr() & 15:
                _refuse(what, "stride: %s must be contiguous and 16-byte aligned" % name)
        if k8.dtype not in (torch.int8, torch.float8_e4m3fn) or v8.dtype != torch.float8_e4m3fn \
                or sk.dtype != torch.float32 or sv.dtype != torch.float32:
            _refuse(what, "dtype: codes are int8 (K) or float8_e4m3fn, scales fp32")
        if k8.dtype == torch.int8 and dtype == torch.bfloat16:
            _refuse(what, "bf16_int8: int8 K is served for fp16 only")
        if k8.dim() != 4 or k8.shape[2] != PAGE or k8.shape[3] not in _HEAD_DIMS \
                or min(k8.shape) < 1 or v8.shape != k8.shape or sk.shape != k8.shape[:3] \
                or sv.shape != k8.shape[:3]:
            _refuse(what, "shape: codes are (pages, heads, 64, 64 or 128), scales (pages, heads, 64)")
        self.k8, self.sk, self.v8, self.sv, self.dtype = k8, sk, v8, sv, dtype
        self.device = k8.device
        self.int8 = k8.dtype == torch.int8
        self.num_pages, self.num_heads, _, self.head_dim = k8.shape

    @classmethod
    def allocate(cls, num_pages, num_heads, head_dim=128, dtype=torch.float16, int8=None,
                 device="cuda"):
        """A new, empty pool: 2 head_dim + 8 bytes a token and head. `int8` (default: for fp16)
        selects int8 keys, else e4m3."""
        int8 = dtype == torch.float16 if int8 is None else bool(int8)
        shape = (num_pages, num_heads, PAGE, head_dim)
        k_type = torch.int8 if int8 else torch.float8_e4m3fn

        def codes(kind):
            return torch.zeros(shape, device=device, dtype=torch.uint8).view(kind)
        return cls(codes(k_type), torch.zeros(shape[:3], device=device),
                   codes(torch.float8_e4m3fn), torch.zeros(shape[:3], device=device), dtype)

    def _check_rows(self, what, t):
        if t.device != self.device:
            _refuse(what, "device: the pool is on %s, the rows on %s" % (self.device, t.device))
        if t.dtype != self.dtype:
            _refuse(what, "dtype: the cache's is %s, the rows' %s" % (self.dtype, t.dtype))
        if t.shape[3] != self.head_dim:
            _refuse(what, "head_dim: the cache's is %d, the rows' %d" % (self.head_dim, t.shape[3]))

    def write(self, k, v, block_table, start, lens=None, tensor_layout="HND", table=None,
              positions=None, interleaved=False):
        """Quantizes new tokens' K and V into the cache: token n of sequence b to position
        `start[b] + n`, for n < lens[b] (default: all).

        k, v: (B, num_heads, N, head_dim), or (B, N, num_heads, head_dim) for "NHD"; block_table (B,
        max_pages), start and lens (B,) int32. With `table` and `positions`, K is rotated first, as by
        `apply_rotary` but without its rounding (a drafted token's position, its depth in the tree, is
        not its place in the cache). The rest of the pool is left as it was. No two tokens of a call
        may go to the same place (two sequences that share a page and both write to it).
        """
        what = "KVCache.write"
        kk, vv = _view(what, tensor_layout, "k", k), _view(what, tensor_layout, "v", v)
        self._check_rows(what, kk)
        self._check_rows(what, vv)
        dev = self.device
        B, H, N, D = kk.shape
        if vv.shape != kk.shape or H != self.num_heads:
            _refuse(what, "heads: k %s and v %s for a cache of %d heads" % (
                tuple(kk.shape), tuple(vv.shape), self.num_heads))
        t_sb = _ints(what, "block_table", block_table, dev, B, -1)
        _ints(what, "start", start, dev, B)
        if lens is not None:
            _ints(what, "lens", lens, dev, B)
        p_sb = 0
        if table is not None:
            p_sb = _check_table(what, table, positions, dev, B, N, D)
        elif positions is not None:
            _refuse(what, "table: positions are given without a rotary table")
        _launch(dev, _library(what, dev).cache_write, self, kk, vv, block_table, t_sb, start, lens,
                table, positions, p_sb, interleaved)

    def read(self, block_table, lens, n, start=None, tensor_layout="HND"):
        """(k, v), the cached rows in 16 bits: row i < lens[b] of sequence b is position `start[b] +
        i` (start None: i), code times scale rounded once; rows from lens[b] up to `n` are zeros.
        block_table (B, max_pages), lens and start (B,) int32; the results have n rows in
        `tensor_layout`."""
        what = "KVCache.read"
        if tensor_layout not in ("HND", "NHD"):
            _refuse(what, "layout: tensor_layout must be HND or NHD (got %r)" % (tensor_layout,))
        n = int(n)
        if n < 1:
            _refuse(what, "seq_len: n must be at least 1 (got %d)" % n)
        if not isinstance(block_table, torch.Tensor) or block_table.dim() != 2 \
                or block_table.shape[0] < 1:
            _refuse(what, "shape: block_table must be a (B, max_pages) tensor")
        dev, B, H, D = self.device, block_table.shape[0], self.num_heads, self.head_dim
        t_sb = _ints(what, "block_table", block_table, dev, B, -1)
        _ints(what, "lens", lens, dev, B)
        if start is not None:
            _ints(what, "start", start, dev, B)
        lib = _library(what, dev)
        hnd = tensor_layout == "HND"
        # both in one allocation: every row is a multiple of 128 bytes
        kv = torch.empty((2, B, H, n, D) if hnd else (2, B, n, H, D), device=dev, dtype=self.dtype)
        k, v = kv.unbind(0)
        _launch(dev, lib.cache_read, self, k if hnd else k.transpose(1, 2),
                v if hnd else v.transpose(1, 2), block_table, t_sb, start, lens)
        return k, v


def sageattn_cached(q, cache, block_table, kv_lens, tensor_layout="HND", q_lens=None, tree_mask=None,
                    sm_scale=None, return_lse=False):
    """Attention of each sequence's newest tokens over all of its cached tokens, theirs included.

    q: (B, H, T, D) for "HND" or (B, T, H, D) for "NHD", of the cache's dtype and head_dim; H a
    multiple of the cache's heads (query head h reads K/V head h // (H // num_heads)). kv_lens (B,)
    int32: the sequences' cached tokens, the last T of which are the new ones (`KVCache.write` comes
    first). New token i sees every token before the new ones and, among those, token j where
    `tree_mask[b, i, j]`; without a mask, where j <= i (T = 1: decoding; more: a prompt's next part).
    tree_mask: bool or uint8, (T, T) or (B, T, T). q_lens (B,) int32: sequence b's new tokens where it
    has fewer than T (its K and V rows being written for as many).

    Returns the output in q's layout and dtype; with `return_lse=True` the pair `(out, lse)`, lse (B,
    H, T) fp32 as `sageattn` defines it. A token that sees nothing, and tokens from q_lens[b] on, give
    zeros and -inf; a score of -infinity counts as not seen, one of +infinity or NaN makes the row NaN. A
    token that was never written (a scale of 0) is seen as a row of zeros. Queries are not quantized: the
    result is that of the cached values to 16 bits.
    """
    what = "sageattn_cached"
    qq = _view(what, tensor_layout, "q", q)
    if not isinstance(cache, KVCache):
        _refuse(what, "cache: a KVCache is needed (got %s)" % type(cache).__name__)
    cache._check_rows(what, qq)
    B, H, T, D = qq.shape
    if H % cache.num_heads:
        _refuse(what, "heads: %d query heads for %d K/V heads" % (H, cache.num_heads))
    dev = cache.device
    t_sb = _ints(what, "block_table", block_table, dev, B, -1)
    _ints(what, "kv_lens", kv_lens, dev, B)
    if q_lens is not None:
        _ints(what, "q_lens", q_lens, dev, B)
    m_sb = m_sr = 0
    if tree_mask is not None:
        if not isinstance(tree_mask, torch.Tensor) or tree_mask.device != dev:
            _refuse(what, "device: tree_mask must be a tensor on %s" % dev)
        if tree_mask.dtype not in (torch.bool, torch.uint8):
            _refuse(what, "dtype: tree_mask must be bool or uint8 (got %s)" % tree_mask.dtype)
        if tree_mask.shape != (T, T) and tree_mask.shape != (B, T, T):
            _refuse(what, "shape: tree_mask is %s, not (%d, %d) or (%d, %d, %d)" % (
                tuple(tree_mask.shape), T, T, B, T, T))
        m_sr = tree_mask.stride(-2) if T > 1 else 1
        m_sb = tree_mask.stride(0) if tree_mask.dim() == 3 and B > 1 else 0
        if (T > 1 and tree_mask.stride(-1) != 1) or m_sr < T or 0 < m_sb < T:
            _refuse(what, "stride_last: tree_mask must have contiguous rows that do not overlap")
    sm = D ** -0.5 if sm_scale is None else float(sm_scale)
    lib = _library(what, dev)
    need = lib.cache_attn_workspace_bytes(B, H, cache.num_heads, T, block_table.shape[1], D)
    out = _empty(q)
    lse = torch.empty((B, H, T), device=dev, dtype=torch.float32) if return_lse else None
    tmp = torch.empty(need, device=dev, dtype=torch.uint8) if need else None
    _launch(dev, lib.cache_attn, cache, qq, out if tensor_layout == "HND" else out.transpose(1, 2),
            block_table, t_sb, kv_lens, q_lens, tree_mask, m_sb, m_sr, sm, lse, tmp, need)
    return (out, lse) if return_lse else out
