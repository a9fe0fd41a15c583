"""Attention's gradients from their definition in 64 bits, and how far the kernels' may lie from them.

A rounding to 16 bits is off by half a step, u = eps / 2 relative to the value (fp16's subnormal numbers:
2^-25 at most), a sum of n products in fp32 by n 2^-24 of the sum of their sizes. With |x| the sizes:
    P        e = (D + 3) 2^-24 sm |q||k| + 2^-22 (|lse| + 1) from the score, the logsumexp's factor and
             the exponential; rounded for its product: u
    dV_j     u |dV_j| + sum_i P |dout| (u + e + n 2^-24)
    dS       |dS| (e + u + 2^-22) + P (D + 3) 2^-24 (|dout||v| + |dout||out| + |dlse|)
    dQ_i     u |dQ_i| + sm sum_j (err dS + n 2^-24 |dS|) |k_j|, and dK likewise
fp16 holds P times 2^12 and dS times a power of two that brings its bound over 2^13: what falls under
their normal numbers is off by 2^-25 2^-12, and by 2^-25 2^-13 of the bound.
"""
import torch

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
E = 2.0 ** -24


def hnd(t, layout):
    return t if layout == "HND" else t.transpose(1, 2)


def mm(a, b):
    """a (.., n, m) b (.., p, m)^T; the transpose laid out anew."""
    return a @ b.transpose(-1, -2).contiguous()


def seen_of(N, N_kv, causal, device):
    if not causal:
        return torch.ones(N, N_kv, dtype=torch.bool, device=device)
    return torch.ones(N, N_kv, dtype=torch.bool, device=device).tril()


def forward(q, k, v, causal, sm):
    """Output and logsumexp of (B, H, N, D) tensors in 64 bits."""
    G = q.shape[1] // k.shape[1]
    k, v = (t.double().repeat_interleave(G, 1) for t in (k, v))
    s = mm(q.double() * sm, k)
    s = s.masked_fill(~seen_of(q.shape[2], k.shape[2], causal, q.device), -torch.inf)
    lse = torch.logsumexp(s, -1)
    return torch.exp(s - lse[..., None]) @ v, lse


def gradients(dout, q, k, v, out, lse, dlse, causal, sm, dtype=None):
    """{"dq": (value, tolerance), ..} for (B, H, N, D) tensors of 16 bits, or of 64 where `dtype` says what the
    tolerances count, head by head."""
    dtype = dtype or q.dtype                       # of the roundings
    u, f16 = U[dtype], dtype == torch.float16
    B, H, N, D = q.shape
    H_kv, N_kv = k.shape[1:3]
    G = H // H_kv
    want = {n: [torch.zeros(t.shape, dtype=torch.float64, device=q.device) for _ in range(2)]
            for n, t in (("dq", q), ("dk", k), ("dv", v))}
    seen = seen_of(N, N_kv, causal, q.device)
    for b in range(B):
        for h in range(H):
            hk = h // G
            qq, gg, oo = (t[b, h].double() for t in (q, dout, out))
            kk, vv = k[b, hk].double(), v[b, hk].double()
            l = lse[b, h].double()[:, None]
            dl = torch.zeros_like(l) if dlse is None else dlse[b, h].double()[:, None]
            none = torch.isneginf(l)
            l = l.masked_fill(none, 0.0)
            p = torch.exp(mm(qq, kk) * sm - l)
            p = p.masked_fill(~seen | none, 0.0)
            e = (D + 3) * E * sm * mm(qq.abs(), kk.abs()) + 4 * E * (l.abs() + 1)
            d = (gg * oo).sum(1, keepdim=True) - dl
            ds = p * (mm(gg, vv) - d)
            size = mm(gg.abs(), vv.abs()) + (gg * oo).abs().sum(1, keepdim=True) + dl.abs()
            err = ds.abs() * (e + u + 4 * E) + p * (D + 3) * E * size
            perr = p * (u + e + N * G * E)
            if f16:
                perr = perr + 2.0 ** -37 * (p > 0)
                bound = gg.norm(dim=1).max() * vv.norm(dim=1).max() + d.abs().max()
                err = err + 2.0 ** -38 * bound * (p > 0)
            want["dv"][0][b, hk] += p.t().contiguous() @ gg
            want["dv"][1][b, hk] += perr.t().contiguous() @ gg.abs()
            want["dq"][0][b, h] = sm * (ds @ kk)
            want["dq"][1][b, h] = sm * ((err + N_kv * E * ds.abs()) @ kk.abs())
            want["dk"][0][b, hk] += sm * (ds.t().contiguous() @ qq)
            want["dk"][1][b, hk] += sm * ((err + N * G * E * ds.abs()).t().contiguous() @ qq.abs())
    least = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    return {n: (x, t + u * x.abs() + least) for n, (x, t) in want.items()}


def check(got, want, note=""):
    """Every value within its tolerance; returns the largest share of it that was used."""
    worst = 0.0
    for x, name in zip(got, ("dq", "dk", "dv")):
        value, tol = want[name]
        assert torch.isfinite(x).all(), (name, note)
        share = ((x.double() - value).abs() / tol).max().item()
        worst = max(worst, share)
        assert share <= 1.0, (name, share, note)
    return worst
