"""Attention over a cache at the sizes that its launches allow (GPU)."""
import pytest
import torch

import kv_cache_ref as ref
from sage_testutil import have_gfx950

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not have_gfx950(), reason="needs a gfx950 GPU")]


def test_rows_of_many_prompts_parts():
    # 2^24 rows, most of them of tokens that are not there: 64 sequences x 32 heads x 8192 new tokens
    from sageattention import KVCache, sageattn_cached
    B, H, H_kv, T, D = 64, 32, 8, 8192, 64
    gen = torch.Generator().manual_seed(3)
    q_lens = [1 + b % 5 for b in range(B)]
    lens = [q + 90 + b % 40 for b, q in enumerate(q_lens)]
    cache = KVCache.allocate(3 * B, H_kv, D)
    table = torch.full((B, T // 64), -1, dtype=torch.int32)
    table[:, :3] = torch.randperm(3 * B, generator=gen).int().view(B, 3)
    k, v = (torch.randn(B, H_kv, max(lens), D, generator=gen).half().cuda() for _ in range(2))
    ints = {n: torch.tensor(x, dtype=torch.int32, device="cuda")
            for n, x in (("start", [0] * B), ("q", q_lens), ("kv", lens))}
    cache.write(k, v, table.cuda(), ints["start"], ints["kv"])
    few = torch.randn(B, H, max(q_lens), D, generator=gen).half()
    q = torch.empty(B, H, T, D, device="cuda", dtype=torch.float16).fill_(float("nan"))
    q[:, :, :max(q_lens)] = few.cuda()
    o, lse = sageattn_cached(q, cache, table.cuda(), ints["kv"], q_lens=ints["q"], return_lse=True)
    del q
    assert not o[:, :, max(q_lens):].any() and torch.isneginf(lse[:, :, max(q_lens):]).all()
    some = [0, 1, 31, 62, 63]
    want, wl, slack = ref.attention(few[some], cache, table[some], [lens[b] for b in some],
                                    [q_lens[b] for b in some])
    # with 2^-11 for the rounding of a weight to fp16
    ref.check_attention(o[some, :, :max(q_lens)].cpu(), want, 2 * slack[0], torch.float16)
    ref.check_lse(lse[some, :, :max(q_lens)].cpu(), wl, slack[1])


@pytest.mark.parametrize("B,H,H_kv,T,past,D", [
    (1, 8, 2, 2100, 300, 128),     # 66 row blocks in fewer than 8 runs
    (2, 32, 1, 1100, 200, 64),     # 275 in one run of both planes
    (1, 32, 1, 8200, 70, 64),      # 2050: a block for each, of one plane
])
def test_parts_of_more_row_blocks_than_an_xcd_holds(B, H, H_kv, T, past, D):
    from sageattention import KVCache, sageattn_cached
    gen = torch.Generator().manual_seed(T)
    q_lens = [T - 600 * b for b in range(B)]
    lens = [past * (b + 1) + t for b, t in enumerate(q_lens)]
    pages = -(-max(lens) // 64)
    cache = KVCache.allocate(B * pages, H_kv, D)
    table = torch.randperm(B * pages, generator=gen).int().view(B, pages)
    k, v, q = (torch.randn(B, h, n, D, generator=gen).mul(x).half()
               for h, n, x in ((H_kv, max(lens), 1.0), (H_kv, max(lens), 1.0), (H, T, 2.0)))
    ints = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0] * B, lens, q_lens)]
    cache.write(k.cuda(), v.cuda(), table.cuda(), ints[0], ints[1])
    o, lse = sageattn_cached(q.cuda(), cache, table.cuda(), ints[1], q_lens=ints[2], return_lse=True)
    chain = torch.ones(T, T, dtype=torch.bool, device="cuda").tril()
    again = sageattn_cached(q.cuda(), cache, table.cuda(), ints[1], q_lens=ints[2], tree_mask=chain)
    assert torch.equal(o, again)
    o, lse = o.cpu(), lse.cpu()
    for b, (n, t) in enumerate(zip(lens, q_lens)):
        assert not o[b, :, t:].any() and torch.isneginf(lse[b, :, t:]).all()
        rows = torch.unique(torch.cat((torch.tensor([0, 1, t - 2, t - 1]), torch.randint(0, t, (40,), generator=gen))))
        k64, v64, _ = ref.gather(cache, table, b, n)
        for h in range(H):
            kk, vv = k64[h // (H // H_kv)], v64[h // (H // H_kv)]
            x = q[b, h, rows].double()
            s = x @ kk.T / D ** 0.5
            a = (x.abs() @ kk.abs().T / D ** 0.5).amax()
            s[torch.arange(n) > n - t + rows[:, None]] = -torch.inf
            p = torch.softmax(s, -1)
            # the bound of kv_cache_ref.attention, with 2^-11 for a weight's rounding
            err = (D + 4) * 2.0 ** -23 * a + 2.0 ** -20
            slack = (2 * err + 2.0 ** -11 + n * 2.0 ** -23) * (p @ vv.abs()) + n * 2.0 ** -39 * vv.abs().amax()
            ref.check_attention(o[b, h, rows], p @ vv, slack, torch.float16)
            want = torch.logsumexp(s, -1)
            ref.check_lse(lse[b, h, rows], want, err + (n + 8) * 2.0 ** -23 + 2.0 ** -22 * want.abs())
