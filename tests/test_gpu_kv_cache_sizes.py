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
