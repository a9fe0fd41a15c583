"""64-bit CPU references of the cache operators, and the tolerances of their GPU tests."""
import torch

PAGE = 64
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def hnd(x, layout):
    return x if layout == "HND" else x.transpose(1, 2)


def rotate(x, table, positions, interleaved, inverse=False):
    """(B, H, N, D) float64, pairs turned one by one; positions (B, N)."""
    R = table.shape[1]
    cs = table.double()[positions.long()][:, None]
    c, s = cs[..., :R // 2], cs[..., R // 2:] * (-1 if inverse else 1)
    y = x.double().clone()
    for i in range(R // 2):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
        xa, xb = x[..., a].double(), x[..., b].double()
        y[..., a] = xa * c[..., i] - xb * s[..., i]
        y[..., b] = xb * c[..., i] + xa * s[..., i]
    return y


def rotate_fp32(x, table, positions, interleaved):
    """The rotation with one fp32 rounding for each product and sum."""
    R = table.shape[1]
    cs = table[positions.long()][:, None]
    c, s = cs[..., :R // 2], cs[..., R // 2:]
    y = x.float().clone()
    a = slice(0, R, 2) if interleaved else slice(0, R // 2)
    b = slice(1, R, 2) if interleaved else slice(R // 2, R)
    xa, xb = x[..., a].float(), x[..., b].float()
    y[..., a] = xa * c - xb * s
    y[..., b] = xb * c + xa * s
    return y


def quantize(x, int8):
    """(codes as float32, scales) of fp32 rows by the scheme; rows that are not finite: 0 and NaN."""
    top = torch.tensor(127.0 if int8 else 448.0)
    fine = torch.isfinite(x).all(-1)
    x = torch.where(fine[..., None], x, torch.zeros(()))
    scale = (x.abs().amax(-1) / top).clamp(min=1e-12)
    code = x / scale[..., None]
    code = code.round() if int8 else code.clamp(-448, 448).to(torch.float8_e4m3fn).float()
    return code, torch.where(fine, scale, torch.tensor(float("nan")))


def gather(cache, block_table, b, n):
    """Sequence b's first n positions: k, v (H, n, D) float64, and which of them have a page."""
    H, D = cache.num_heads, cache.head_dim
    k, v = torch.zeros(2, H, n, D, dtype=torch.float64)
    held = torch.zeros(n, dtype=torch.bool)
    rows = [block_table[b].tolist()[p // PAGE] if p // PAGE < block_table.shape[1] else -1
            for p in range(n)]
    at = [i for i, page in enumerate(rows) if 0 <= page < cache.num_pages]
    if at:
        page = torch.tensor([rows[i] for i in at])
        slot = torch.tensor([i % PAGE for i in at])
        for out, codes, scales in ((k, cache.k8, cache.sk), (v, cache.v8, cache.sv)):
            dev = codes.device
            c = codes.view(torch.uint8)[page.to(dev), :, slot.to(dev)].cpu().view(codes.dtype)
            s = scales[page.to(dev), :, slot.to(dev)].cpu()
            out[:, at] = (c.double() * s.double()[..., None]).transpose(0, 1)
        held[at] = True
    return k, v, held


def attention(q, cache, block_table, kv_lens, q_lens=None, mask=None, sm_scale=None):
    """(o, lse, slack) for q (B, H, T, D) on the CPU: float64 results, and how far the kernel's fp32 and
    fp16 intermediate roundings may move an output element (before its own rounding) and an lse.

    With A = max_j sum_d |q_d k_jd| sm_scale over a row's visible keys: a score is D products (exact)
    summed in fp32 and two fp32 operations, off by at most (D + 4) 2^-23 A (twice a rounding's half
    step for sums that are truncated); log2 SV, 2^x and 1/SV add at most 2^-20. A weight is then
    off by twice that (its own, and the sum's it is divided by) and by its rounding to fp16, 2^-12 (11
    bits: half a step); so an output is off by at most that times sum_j p_j |v_j|, plus the fp32
    sums of n terms, n 2^-23 of the same. A weight includes its value's scale, and one 2^28 below the
    row's largest is rounded to 2^-39 of that: per key at most 2^-39 of the largest p_j |v_jd| there is.
    """
    B, H, T, D = q.shape
    G = H // cache.num_heads
    sm = D ** -0.5 if sm_scale is None else sm_scale
    o = torch.zeros(B, H, T, D, dtype=torch.float64)
    lse = torch.full((B, H, T), -torch.inf, dtype=torch.float64)
    slack_o, slack_l = torch.zeros_like(o), torch.zeros_like(lse)
    for b in range(B):
        n = max(0, int(kv_lens[b]))
        t = T if q_lens is None else min(T, max(0, int(q_lens[b])))
        k, v, held = gather(cache, block_table, b, n)
        for i in range(t):
            seen = held.clone()
            for j in range(n):
                draft = j - (n - t)
                if draft >= 0:
                    ok = draft <= i if mask is None else \
                        bool((mask if mask.dim() == 2 else mask[b])[i, draft])
                    seen[j] &= ok
            if not seen.any():
                continue
            for h in range(H):
                kk, vv = k[h // G][seen], v[h // G][seen]
                x = q[b, h, i].double()
                s = kk @ x * sm
                a = (kk.abs() @ x.abs() * sm).max()
                p = torch.softmax(s, 0)
                o[b, h, i] = p @ vv
                lse[b, h, i] = torch.logsumexp(s, 0)
                err = (D + 4) * 2.0 ** -23 * a + 2.0 ** -20
                m = kk.shape[0]
                spread = p @ vv.abs()
                slack_o[b, h, i] = (2 * err + 2.0 ** -12 + m * 2.0 ** -23) * spread \
                    + m * 2.0 ** -39 * (p[:, None] * vv.abs()).max()
                slack_l[b, h, i] = err + (m + 8) * 2.0 ** -23 + 2.0 ** -22 * lse[b, h, i].abs()
    return o, lse, (slack_o, slack_l)


def check_attention(out, ref, slack, dtype):
    bound = slack + HALF_STEP[dtype] * (ref.abs() + slack) + 2.0 ** -24   # fp16's least half step
    nan = torch.isnan(ref)
    assert torch.equal(torch.isnan(out), nan)
    off = torch.where(nan, torch.zeros(()).double(), (out.double() - ref).abs() - bound)
    assert (off <= 0).all(), "worst %.3g over its bound at %s" % (
        off.max(), [int(x) for x in (off == off.max()).nonzero()[0]])


def check_lse(lse, ref, slack):
    empty = torch.isinf(ref)
    assert torch.equal(torch.isneginf(lse.double()), empty)
    off = (lse.double() - ref).abs()[~empty & ~torch.isnan(ref)]
    assert (off <= slack[~empty & ~torch.isnan(ref)]).all(), off.max()
    assert torch.equal(torch.isnan(lse), torch.isnan(ref))


def random_tree(T, gen):
    """(T, T) mask of a random tree of drafted tokens: each sees itself and its ancestors."""
    m = torch.zeros(T, T, dtype=torch.bool)
    for j in range(T):
        up = int(torch.randint(-1, max(j, 1), (1,), generator=gen)) if j else -1
        if up >= 0:
            m[j] = m[up]
        m[j, j] = True
    return m
