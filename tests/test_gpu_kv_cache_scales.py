"""Attention over cached rows whose value scales are 0 or lie very far apart (GPU), against 64-bit
results. A weight carries its value's scale, and the sum that it is divided by does not: these are the
caches where the two drift apart.
"""
import math

import pytest
import torch

import kv_cache_ref as ref
from sage_testutil import have_gfx950

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not have_gfx950(), reason="needs a gfx950 GPU")]


def _ints(*n):
    return torch.tensor(n, dtype=torch.int32, device="cuda")


def _attend(q, k, v, seen, blank, sm):
    """(o, lse, slack_o, slack_l) in 64 bits: q (H, T, D) over rows k, v (H, n, D) where `seen` (T, n), and
    over `blank` more rows of zeros that all see.

    The slack is `kv_cache_ref.attention`'s: a score of at most a = sum |q_d k_d| sm is off by (D + 4) 2^-23
    a, its logarithm, exponential and reciprocal by 2^-20, a weight and the sum that divides it by that each;
    the fp16 rounding of a weight is 2^-11 of it, and 2^-39 of the row's largest weight below 2^-28
    of that; an fp32 sum of n terms is off by n 2^-23.
    """
    n, D = blank + k.shape[1], q.shape[2]
    q = q.double()
    s = (q @ k.transpose(1, 2) * sm).masked_fill(~seen, -torch.inf)
    a = (q.abs() @ k.abs().transpose(1, 2) * sm).amax()
    top = s.amax(-1, keepdim=True).clamp(min=0.0 if blank else -1e300)
    total = (s - top).exp().sum(-1, keepdim=True) + blank * (-top).exp()
    p = (s - top).exp() / total
    lse = (top + total.log())[..., 0]
    err = (D + 4) * 2.0 ** -23 * a + 2.0 ** -20
    slack = (2 * err + 2.0 ** -11 + n * 2.0 ** -23) * (p @ v.abs()) \
        + n * 2.0 ** -39 * (p[..., None] * v.abs()[:, None]).amax((-1, -2))[..., None]
    return p @ v, lse, slack, err + (n + 8) * 2.0 ** -23 + 2.0 ** -22 * lse.abs()


# ------------------------------------------------------------------------ tokens never written
@pytest.mark.parametrize("blank", [16384, 40000])
@pytest.mark.parametrize("T", [1, 8, 16, 40])
@pytest.mark.parametrize("B", [1, 2048])
def test_nothing_but_tokens_never_written(B, T, blank):
    # in runs (1 sequence) and by a block for each plane (2048), 4 to 160 rows of a K/V head
    from sageattention import KVCache, sageattn_cached
    cache = KVCache.allocate(1, 1, 64)
    pages = -(-blank // 64)
    table = torch.zeros(1, pages, dtype=torch.int32, device="cuda").expand(B, pages)
    lens = torch.full((B,), 64, dtype=torch.int32, device="cuda")
    lens[B // 2] = blank
    q = torch.randn(B, 4, T, 64, generator=torch.Generator().manual_seed(T)).half().cuda()
    o, lse = sageattn_cached(q, cache, table, lens, return_lse=True)
    assert not o.any()
    for b, n in ((B // 2, blank), (B - 1, blank if B == 1 else 64)):
        # token i sees all tokens but the T - 1 - i last ones
        want = torch.tensor([math.log(n - T + 1 + i) for i in range(T)], dtype=torch.float64)
        bound = 2.0 ** -20 + (n + 8) * 2.0 ** -23 + 2.0 ** -22 * want
        assert ((lse[b].double().cpu() - want).abs() <= bound).all()


@pytest.mark.parametrize("T", [1, 8, 16, 40])
@pytest.mark.parametrize("B,blank", [(1, 16384), (1, 40001), (1, 2 ** 21 + 70), (2048, 16384),
                                     (2048, 40001)])
def test_tokens_never_written_before_others(B, blank, T):
    # the first is in runs of a few pages, and of 256 or more for 2^21 tokens; 2048 a block for each plane
    from sageattention import KVCache, sageattn_cached
    gen, D, H, n = torch.Generator().manual_seed(T + blank), 64, 4, 6 + T
    pages = -(-(blank + n) // 64)
    cache = KVCache.allocate(5, 1, D)
    table = torch.zeros(1, pages, dtype=torch.int32, device="cuda")
    first = blank // 64
    table[0, first:] = torch.arange(1, 1 + pages - first)
    k, v = (torch.randn(1, 1, n, D, generator=gen).mul(x).half().cuda() for x in (3.0, 1.0))
    cache.write(k, v, table, _ints(blank))
    at = B // 2
    lens = torch.full((B,), 64, dtype=torch.int32, device="cuda")
    lens[at] = blank + n
    q = torch.randn(B, H, T, D, generator=gen).mul(3.0).half()
    o, lse = sageattn_cached(q.cuda(), cache, table.expand(B, pages), lens, return_lse=True)
    kk, vv = (x[0, 0].cpu() for x in cache.read(table, _ints(n), n, start=_ints(blank)))
    # the codes' own values: 16-bit reads of them round
    at_page, slot = table[0, (blank + torch.arange(n)) // 64].long(), (blank + torch.arange(n)).cuda() % 64
    k64 = (cache.k8[at_page, 0, slot].double() * cache.sk[at_page, 0, slot].double()[:, None]).cpu()
    v64 = (cache.v8.view(torch.uint8)[at_page, 0, slot].cpu().view(torch.float8_e4m3fn).double()
           * cache.sv[at_page, 0, slot].double().cpu()[:, None])
    assert torch.equal(k64.half(), kk) and torch.equal(v64.half(), vv)
    seen = torch.arange(n) <= n - T + torch.arange(T)[:, None]
    want, wl, slack, slack_l = _attend(q[at], k64.expand(H, n, D), v64.expand(H, n, D), seen, blank,
                                       D ** -0.5)
    assert want.abs().max() > 0.05      # the written ones weigh something
    ref.check_attention(o[at].cpu(), want, slack, torch.float16)
    ref.check_lse(lse[at].cpu(), wl, slack_l)


# ------------------------------------------------------------------------ scales far apart
def _far_apart(n, D, gen):
    """V rows (1, 1, n, D) of bf16: a third of zeros (a scale of 1e-12), a third ordinary, a third between
    1e-30 and 1e30."""
    size = 10.0 ** torch.randint(-30, 31, (n,), generator=gen).float()
    size[torch.arange(n) % 3 == 0], size[torch.arange(n) % 3 == 1] = 0, 1
    return (torch.randn(1, 1, n, D, generator=gen) * size[:, None]).bfloat16()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", [1, 8, 16, 40])
@pytest.mark.parametrize("n", [63, 300, 3000])
@pytest.mark.parametrize("where", ["first", "middle", "late", "all"])
def test_bf16_values_of_every_size(where, n, T, D):
    """Rows of up to bf16's largest value beside rows of zeros at like scores: every row counts in the sum
    that a result is divided by. In one launch (n = 63, 300 at up to 32 rows of a K/V head) and in runs.

    Beyond `_attend`'s slack: log2 of scales between 2^-40 and 2^119.2 and scores below 2^6 make numbers of
    up to 2^8, whose logarithm, sum, maximum's shift and difference are rounded at 2^-17 each: 4 of them
    move a weight by less than 2^-15 of it, and the sum by as much.
    """
    from sageattention import KVCache, sageattn_cached
    gen, H = torch.Generator().manual_seed(1000 * n + T + D), 4
    past = max(0, n - T)
    top = torch.finfo(torch.bfloat16).max
    big = {"first": [1], "middle": [past // 2], "late": [n - 1 - T // 2], "all": range(2, n, 7)}[where]
    k = torch.randn(1, 1, n, D, generator=gen).bfloat16()
    v = _far_apart(n, D, gen)
    for i, at in enumerate(big):
        v[0, 0, at] = torch.randn(D, generator=gen).clamp(-3, 3).mul(1e38 * 4.0 ** -(i % 20)).bfloat16()
    v[0, 0, list(big)[-1], D // 3] = -top
    pages = -(-n // 64)
    cache = KVCache.allocate(pages, 1, D, torch.bfloat16)
    table = torch.randperm(pages, generator=gen).int()[None].cuda()
    cache.write(k.cuda(), v.cuda(), table, _ints(0))
    q = torch.randn(1, H, T, D, generator=gen).mul(2.0).bfloat16()
    o, lse = sageattn_cached(q.cuda(), cache, table, _ints(n), return_lse=True)
    k64, v64, _ = ref.gather(cache, table.cpu(), 0, n)
    seen = torch.arange(n) <= n - T + torch.arange(T)[:, None]
    want, wl, slack, slack_l = _attend(q[0], k64.expand(H, n, D), v64.expand(H, n, D), seen, 0, D ** -0.5)
    far = 2.0 ** -15
    spread = torch.softmax((q[0].double() @ k64.transpose(1, 2) * D ** -0.5).masked_fill(~seen, -torch.inf),
                           -1) @ v64.abs()
    ref.check_attention(o[0].cpu(), want, slack + 2 * far * spread, torch.bfloat16)
    ref.check_lse(lse[0].cpu(), wl, slack_l + far)


@pytest.mark.parametrize("T", [1, 8, 16, 40])
def test_bf16_values_of_every_size_in_ragged_runs(T):
    # 70 sequences: runs that end one plane and begin another, with and without large values
    from sageattention import KVCache, sageattn_cached
    gen, B, H, D = torch.Generator().manual_seed(T), 70, 4, 64
    lens = [int(x) for x in torch.randint(T, 2400, (B,), generator=gen)]
    width = -(-max(lens) // 64)
    cache = KVCache.allocate(B * width, 1, D, torch.bfloat16)
    table = torch.randperm(B * width, generator=gen).int().view(B, width).cuda()
    k = torch.randn(B, 1, max(lens), D, generator=gen).bfloat16()
    v = torch.cat([_far_apart(max(lens), D, gen) for _ in range(B)])
    for b in range(0, B, 2):
        v[b, 0, lens[b] * (b % 5) // 6] = torch.randn(D, generator=gen).mul(2e37).bfloat16()
    cache.write(k.cuda(), v.cuda(), table, torch.zeros(B, dtype=torch.int32, device="cuda"))
    q = torch.randn(B, H, T, D, generator=gen).mul(2.0).bfloat16()
    o, lse = sageattn_cached(q.cuda(), cache, table, _ints(*lens), return_lse=True)
    for b in range(0, B, 3):
        n = lens[b]
        k64, v64, _ = ref.gather(cache, table.cpu(), b, n)
        seen = torch.arange(n) <= n - T + torch.arange(T)[:, None]
        want, wl, slack, slack_l = _attend(q[b], k64.expand(H, n, D), v64.expand(H, n, D), seen, 0, 0.125)
        p = torch.softmax((q[b].double() @ k64.transpose(1, 2) * 0.125).masked_fill(~seen, -torch.inf), -1)
        ref.check_attention(o[b].cpu(), want, slack + 2.0 ** -14 * (p @ v64.abs()), torch.bfloat16)
        ref.check_lse(lse[b].cpu(), wl, slack_l + 2.0 ** -15)


# ----------------------------------------------------------------------------- largest values
@pytest.mark.parametrize("int8", [True, False])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", [1, 8, 16, 40])
@pytest.mark.parametrize("n", [700, 5000])
def test_fp16_largest_values_stay_finite(n, T, D, int8):
    """A mean of fp16's largest value is that value, also where all weights are rounded up: one token of 32
    weighs 1 and the others exp(-2 sm) = (1 + 1.05 2^-11) / 2, which fp16 takes for (1 + 2^-10) / 2."""
    from sageattention import KVCache, sageattn_cached
    sm = -0.5 * math.log(0.5 * (1 + 1.05 * 2.0 ** -11))
    top = torch.finfo(torch.float16).max
    k, v = torch.zeros(2, 1, 1, n, D, dtype=torch.float16)
    k[..., 0], k[:, :, ::32, 0] = -1, 1
    v[..., 0], v[..., 1], v[..., 2] = top, -top, 1
    pages = -(-n // 64)
    cache = KVCache.allocate(pages, 1, D, int8=int8)
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    cache.write(k.cuda(), v.cuda(), table, _ints(0))
    q = torch.zeros(1, 4, T, D, device="cuda", dtype=torch.float16)
    q[..., 0] = 1
    o = sageattn_cached(q, cache, table, _ints(n), sm_scale=sm).cpu()
    for column, want in ((0, top), (1, -top)):
        # the weights' 2^-11 and the result's own half step
        off = (o[..., column].double() - want).abs()
        assert torch.isfinite(o[..., column]).all() and (off <= 2.0 ** -10 * top).all()


# --------------------------------------------------------------------------- infinite scores
@pytest.mark.parametrize("dtype,int8", [(torch.float16, True), (torch.float16, False),
                                        (torch.bfloat16, False)])
@pytest.mark.parametrize("T", [1, 8, 16, 40])
@pytest.mark.parametrize("n", [100, 3000])
def test_infinite_scores(n, T, dtype, int8):
    # a query's infinity meets a column of negative keys, or one that is positive in the newest token's row
    from sageattention import KVCache, sageattn_cached
    gen, pages = torch.Generator().manual_seed(n + T), -(-n // 64)
    cache = KVCache.allocate(pages, 1, 64, dtype, int8)
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    k, v = (torch.randn(1, 1, n, 64, generator=gen).to(dtype) for _ in range(2))
    k[..., 0], k[..., 1], k[0, 0, n - 1, 1] = -1, -1, 1
    cache.write(k.cuda(), v.cuda(), table, _ints(0))
    q = torch.randn(1, 4, T, 64, generator=gen).to(dtype)
    q[:, 1, :, 0] = q[:, 2, :, 1] = torch.inf
    o, lse = (x.cpu() for x in sageattn_cached(q.cuda(), cache, table, _ints(n), return_lse=True))
    assert torch.isfinite(o[:, [0, 3]]).all() and torch.isfinite(lse[:, [0, 3]]).all()
    assert not o[:, 1].any() and torch.isneginf(lse[:, 1]).all()     # as if nothing were seen
    # only the last token sees the newest
    assert not o[:, 2, :-1].any() and torch.isneginf(lse[:, 2, :-1]).all()
    assert torch.isnan(o[:, 2, -1]).all() and torch.isnan(lse[:, 2, -1]).all()
