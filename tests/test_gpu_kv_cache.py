"""Rotary positions, the quantized K/V cache and attention over it (GPU), against 64-bit references.

Codes and scales have to be the scheme's bit for bit; rotations are off by three fp32 roundings and the
last one; attention by what `kv_cache_ref.attention` derives.
"""
import pytest
import torch

import kv_cache_ref as ref
from sage_testutil import have_gfx950

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not have_gfx950(), reason="needs a gfx950 GPU")]

KINDS = [(torch.float16, True), (torch.float16, False), (torch.bfloat16, False)]
KIND_IDS = ["fp16-int8", "fp16-e4m3", "bf16-e4m3"]


def _randn(shape, dtype, layout, gen, scale=1.0):
    """CPU (B, H, N, D) values and the same on the GPU in the layout."""
    x = (torch.randn(shape, generator=gen) * scale).to(dtype)
    return x, ref.hnd(x, layout).contiguous().cuda()


def _lens(*n):
    return torch.tensor(n, dtype=torch.int32, device="cuda")


def _pages(lens, num_pages, gen, width=None):
    """A block table with each sequence's pages in random order, -1 behind them."""
    width = width or max(1, max(-(-n // 64) for n in lens))
    order = torch.randperm(num_pages, generator=gen).int()
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(lens):
        used = -(-n // 64)
        table[b, :used] = order[at:at + used]
        at += used
    assert at <= num_pages
    return table.cuda()


def _dirty(cache):
    """Fills a pool with what no row of it may be: NaN codes and NaN scales."""
    cache.k8.view(torch.uint8).fill_(0x7F)
    cache.v8.view(torch.uint8).fill_(0x7F)
    cache.sk.fill_(float("nan"))
    cache.sv.fill_(float("nan"))


def _filled(dtype, int8, H_kv, D, lens, gen, dirty=True, extra=2, width=None, scale=1.0):
    """A cache that holds random rows for sequences of these lengths, and their block table."""
    from sageattention import KVCache
    num = sum(-(-n // 64) for n in lens) + extra
    cache = KVCache.allocate(num, H_kv, D, dtype, int8)
    if dirty:
        _dirty(cache)
    table = _pages(lens, num, gen, width)
    n = max(max(lens), 1)
    _, k = _randn((len(lens), H_kv, n, D), dtype, "HND", gen, scale)
    _, v = _randn((len(lens), H_kv, n, D), dtype, "HND", gen, scale)
    cache.write(k, v, table, _lens(*[0] * len(lens)), _lens(*lens))
    return cache, table


# ------------------------------------------------------------------------------------- rotary
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("layout", ["HND", "NHD"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,H,N,D,R", [(1, 1, 1, 128, 128), (2, 3, 5, 64, 64), (3, 10, 65, 128, 32),
                                       (1, 4, 333, 64, 16), (2, 8, 7, 128, 96),
                                       (1, 7, 5003, 128, 128), (2, 3, 6001, 64, 48)])
def test_rotary(B, H, N, D, R, dtype, layout, interleaved):
    from sageattention import apply_rotary, rotary_table
    gen = torch.Generator().manual_seed(B * N + R)
    x, xg = _randn((B, H, N, D), dtype, layout, gen, 3.0)
    table = rotary_table(4096, R, device="cpu")
    pos = torch.randint(0, 4096, (B, N), generator=gen).int()
    for inverse in (False, True):
        y = apply_rotary(xg, table.cuda(), pos.cuda(), layout, interleaved, inverse)
        assert y.shape == xg.shape and y.dtype == dtype and y.is_contiguous()
        got = ref.hnd(y.cpu(), layout)
        want = ref.rotate(x, table, pos, interleaved, inverse)
        # two products and a sum in fp32, each term at most |a| + |b|, then the result's half step
        a, b = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, R // 2), slice(R // 2, R))
        size = torch.zeros_like(want)
        size[..., a] = size[..., b] = x[..., a].double().abs() + x[..., b].double().abs()
        bound = 3 * 2.0 ** -24 * size
        bound = bound + ref.HALF_STEP[dtype] * (want.abs() + bound) + 2.0 ** -25
        assert ((got.double() - want).abs() <= bound).all()
        assert torch.equal(got[..., R:], x[..., R:])


def test_rotary_takes_fused_views_and_shared_positions():
    from sageattention import apply_rotary, rotary_table
    gen = torch.Generator().manual_seed(3)
    fused = torch.randn(2, 37, 3, 5, 128, generator=gen).half().cuda()
    table = rotary_table(64, 64)
    pos = torch.randint(0, 64, (37,), generator=gen).int().cuda()
    for i in range(3):
        view = fused[:, :, i]
        y = apply_rotary(view, table, pos, "NHD")
        assert torch.equal(y, apply_rotary(view.contiguous(), table, pos.expand(2, 37), "NHD"))


def test_rotary_marks_positions_outside_the_table():
    from sageattention import apply_rotary, rotary_table
    x = torch.ones(1, 2, 5, 128, device="cuda", dtype=torch.float16)
    table = rotary_table(10, 64)
    y = apply_rotary(x, table, torch.tensor([[0, 9, 10, -1, 2 ** 31 - 1]], dtype=torch.int32).cuda())
    bad = torch.isnan(y)
    assert not bad[:, :, :2].any() and bad[:, :, 2:, :64].all() and not bad[..., 64:].any()
    assert (y[..., 64:] == 1).all()


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_inverse_is_the_gradient(interleaved):
    # L = sum(w * rotary(x)): its gradient by x is inverse(w), and its differences agree with that
    from sageattention import apply_rotary, rotary_table
    gen = torch.Generator().manual_seed(9)
    table = rotary_table(512, 64)
    pos = torch.randint(0, 512, (1, 6), generator=gen).int().cuda()
    x = torch.randint(-8, 9, (1, 2, 6, 128), generator=gen).half().cuda()
    w = torch.randint(-8, 9, (1, 2, 6, 128), generator=gen).half().cuda()
    grad = apply_rotary(w, table, pos, interleaved=interleaved, inverse=True).double()
    for at in ((0, 0, 0, 0), (0, 1, 3, 33), (0, 0, 5, 63), (0, 1, 2, 100)):
        up, down = x.clone(), x.clone()
        up[at] += 4
        down[at] -= 4
        d = [(w.double() * apply_rotary(t, table, pos, interleaved=interleaved).double()).sum()
             for t in (up, down)]
        # the pair's four outputs of magnitude <= 17 are off by 2^-11 of it each, weighted by <= 8
        assert abs((d[0] - d[1]) / 8 - grad[at]) <= (4 * 17 * 8 / 8 + 12) * 2.0 ** -11


# -------------------------------------------------------------------------------- write, read
@pytest.mark.parametrize("dtype,int8", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("layout", ["HND", "NHD"])
@pytest.mark.parametrize("H,N,D,start", [(1, 1, 128, 0), (2, 1, 64, 63), (3, 5, 128, 62),
                                         (8, 130, 128, 1), (2, 200, 64, 64)])
def test_write_holds_the_schemes_codes(dtype, int8, layout, H, N, D, start):
    from sageattention import KVCache
    B, gen = 3, torch.Generator().manual_seed(N + D)
    k, kg = _randn((B, H, N, D), dtype, layout, gen)
    v, vg = _randn((B, H, N, D), dtype, layout, gen, 5.0)
    k[0, 0, 0], kg = 0, ref.hnd(k, layout).contiguous().cuda()
    k, v = ref.hnd(kg.cpu(), layout), ref.hnd(vg.cpu(), layout)
    lens, starts = [N, 0, max(1, N - 3)], [start, start, start + 7]
    table = _pages([s + n for s, n in zip(starts, (N, N, N))], 3 * 8, gen)
    cache = KVCache.allocate(24, H, D, dtype, int8)
    _dirty(cache)
    before = [t.clone() for t in (cache.k8, cache.sk, cache.v8, cache.sv)]
    cache.write(kg, vg, table, _lens(*starts), _lens(*lens), tensor_layout=layout)
    kc, ks = ref.quantize(k.float(), int8)
    vc, vs = ref.quantize(v.float(), False)
    want = [t.cpu().clone() for t in before]
    want[0] = want[0].view(torch.uint8)
    want[2] = want[2].view(torch.uint8)
    kb = (kc.to(torch.int8) if int8 else kc.to(torch.float8_e4m3fn)).view(torch.uint8)
    vb = vc.to(torch.float8_e4m3fn).view(torch.uint8)
    t = table.cpu()
    for b in range(B):
        for n in range(lens[b]):
            page, slot = int(t[b, (starts[b] + n) // 64]), (starts[b] + n) % 64
            want[0][page, :, slot], want[1][page, :, slot] = kb[b, :, n], ks[b, :, n]
            want[2][page, :, slot], want[3][page, :, slot] = vb[b, :, n], vs[b, :, n]
    assert torch.equal(cache.k8.cpu().view(torch.uint8), want[0])
    assert torch.equal(cache.v8.cpu().view(torch.uint8), want[2])
    assert torch.equal(cache.sk.cpu().view(torch.int32), want[1].view(torch.int32))
    assert torch.equal(cache.sv.cpu().view(torch.int32), want[3].view(torch.int32))


@pytest.mark.parametrize("dtype,int8", KINDS, ids=KIND_IDS)
def test_write_and_the_prologue_agree(dtype, int8):
    # the cached codes and scales are those that the prologue makes without smoothing
    from sageattention import KVCache
    from sageattention.sk1_backend.hip_prologue import HipPrologue
    gen = torch.Generator().manual_seed(5)
    _, k = _randn((1, 2, 192, 128), dtype, "HND", gen)
    _, v = _randn((1, 2, 192, 128), dtype, "HND", gen)
    k8, sk, v8t, sv = HipPrologue.get().quant_kv(k, v, smooth_k=False, int8=int8)
    cache = KVCache.allocate(3, 2, 128, dtype, int8)
    cache.write(k, v, torch.arange(3, dtype=torch.int32, device="cuda")[None], _lens(0))
    def rows(t):
        return t.view(torch.uint8).transpose(0, 1).reshape(2, 192, -1)
    assert torch.equal(rows(cache.k8), k8.view(torch.uint8))
    assert torch.equal(rows(cache.v8), v8t.view(torch.uint8).transpose(1, 2))
    assert torch.equal(cache.sk.transpose(0, 1).reshape(2, 192), sk)
    assert torch.equal(cache.sv.transpose(0, 1).reshape(2, 192), sv)


@pytest.mark.parametrize("dtype,int8", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("D,R,interleaved", [(128, 128, False), (128, 32, True), (64, 64, True),
                                             (64, 48, False)])
def test_write_rotates_k(dtype, int8, D, R, interleaved):
    from sageattention import KVCache, rotary_table
    B, H, N, gen = 2, 3, 21, torch.Generator().manual_seed(R)
    k, kg = _randn((B, H, N, D), dtype, "NHD", gen)
    v, vg = _randn((B, H, N, D), dtype, "NHD", gen)
    table = rotary_table(99, R, device="cpu")
    pos = torch.randint(0, 99, (B, N), generator=gen).int()
    pages = _pages([N, N], 2, gen)
    cache = KVCache.allocate(2, H, D, dtype, int8)
    cache.write(kg, vg, pages, _lens(0, 0), tensor_layout="NHD", table=table.cuda(),
                positions=pos.cuda(), interleaved=interleaved)
    kc, ks = ref.quantize(ref.rotate_fp32(k, table, pos, interleaved), int8)
    vc, vs = ref.quantize(v.float(), False)
    for b in range(B):
        p = int(pages[b, 0])
        assert torch.equal(cache.k8.cpu()[p, :, :N].float(), kc[b])
        assert torch.equal(cache.v8.cpu()[p, :, :N].float(), vc[b])
        assert torch.equal(cache.sk.cpu()[p, :, :N], ks[b])
        assert torch.equal(cache.sv.cpu()[p, :, :N], vs[b])


@pytest.mark.parametrize("dtype,int8", KINDS, ids=KIND_IDS)
def test_rows_that_are_not_finite_are_held_as_nan(dtype, int8):
    from sageattention import KVCache, rotary_table
    gen = torch.Generator().manual_seed(8)
    k, _ = _randn((1, 2, 9, 128), dtype, "HND", gen)
    v = k.clone()
    for n, bad in ((0, float("inf")), (3, -float("inf")), (5, float("nan"))):
        k[0, 0, n, 17] = bad
        v[0, 1, n, 127] = bad
    k[0, 1, 7], v[0, 0, 7] = 0, torch.finfo(dtype).min
    cache = KVCache.allocate(1, 2, 128, dtype, int8)
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    cache.write(k.cuda(), v.cuda(), table, _lens(0))
    for x, codes, scales, i8 in ((k, cache.k8, cache.sk, int8), (v, cache.v8, cache.sv, False)):
        c, s = ref.quantize(x.float(), i8)
        assert torch.equal(codes.cpu()[0, :, :9].float(), c[0])
        assert torch.equal(torch.isnan(scales.cpu()[0, :, :9]), torch.isnan(s[0]))
        assert torch.equal(scales.cpu()[0, :, :9].nan_to_num(), s[0].nan_to_num())
    # a position outside the table: K's row is NaN, V's is not
    cache.write(v.cuda(), k.cuda(), table, _lens(20), _lens(1), table=rotary_table(4, 64),
                positions=torch.full((1, 9), 4, dtype=torch.int32, device="cuda"))
    assert torch.isnan(cache.sk[0, :, 20]).all() and torch.isfinite(cache.sv[0, 1, 20])


@pytest.mark.parametrize("dtype,int8", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("layout", ["HND", "NHD"])
@pytest.mark.parametrize("H,D,lens,start,n", [(1, 128, (1,), (0,), 1), (3, 64, (70, 0, 5), (0, 9, 60), 70),
                                              (2, 128, (200, 1, 63), (0, 64, 1), 203)])
def test_read(dtype, int8, layout, H, D, lens, start, n):
    gen = torch.Generator().manual_seed(n)
    total = [s + m for s, m in zip(start, lens)]
    cache, table = _filled(dtype, int8, H, D, total, gen)
    got = cache.read(table, _lens(*lens), n, start=_lens(*start), tensor_layout=layout)
    for x, codes, scales in zip(got, (cache.k8, cache.v8), (cache.sk, cache.sv)):
        x = ref.hnd(x.cpu(), layout)
        assert x.shape == (len(lens), H, n, D) and x.dtype == dtype
        for b in range(len(lens)):
            for i in range(n):
                if i >= lens[b]:
                    assert (x[b, :, i] == 0).all()
                    continue
                page, slot = int(table[b, (start[b] + i) // 64]), (start[b] + i) % 64
                want = (codes[page, :, slot].float() * scales[page, :, slot, None]).to(dtype).cpu()
                assert torch.equal(x[b, :, i], want)


def test_bad_pages_are_no_pages():
    # numbers outside the pool, and positions behind the table: nothing is written, zeros are read
    from sageattention import KVCache, sageattn_cached
    gen = torch.Generator().manual_seed(2)
    cache = KVCache.allocate(3, 2, 64)
    table = torch.tensor([[0, 3, 1], [-1, 2, -2 ** 31], [2 ** 31 - 1, -1, -1]], dtype=torch.int32).cuda()
    _, k = _randn((3, 2, 200, 64), torch.float16, "HND", gen)
    _, v = _randn((3, 2, 200, 64), torch.float16, "HND", gen)
    cache.write(k, v, table, _lens(0, 0, 0))
    rk, rv = (x.cpu() for x in cache.read(table, _lens(200, 200, 200), 200))
    for x, src, int8 in ((rk, k, True), (rv, v, False)):
        c, s = ref.quantize(src.float().cpu(), int8)
        want = (c * s[..., None]).half()
        held = torch.zeros(3, 200, dtype=torch.bool)
        held[0, :64] = held[0, 128:192] = held[1, 64:128] = True
        assert torch.equal(x, torch.where(held[:, None, :, None], want, torch.zeros((), dtype=torch.half)))
    q, qg = _randn((3, 2, 2, 64), torch.float16, "HND", gen)
    kv = [190, 200, 2 ** 31 - 1]
    o, lse = sageattn_cached(qg, cache, table, _lens(*kv), return_lse=True)
    want, wl, slack = ref.attention(q, cache, table.cpu(), [190, 200, 192])
    ref.check_attention(o.cpu()[:2], want[:2], slack[0][:2], torch.float16)
    ref.check_lse(lse.cpu()[:2], wl[:2], slack[1][:2])
    assert (o[2] == 0).all() and torch.isneginf(lse[2]).all()
    # a negative start: the positions before 0 are nowhere
    cache.write(k[:, :, :5], v[:, :, :5], table, _lens(-3, -2 ** 31, -5), None)
    assert torch.equal(cache.read(table, _lens(2, 0, 0), 2)[1][0].cpu(),
                       (lambda c, s: (c * s[..., None]).half())(*ref.quantize(v[0, :, 3:5].float().cpu(), False)))


# ---------------------------------------------------------------------------------- attention
@pytest.mark.parametrize("dtype,int8", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,H_kv,T,lens", [
    (1, 1, 1, (1,)), (4, 4, 1, (64, 65, 0)), (8, 1, 1, (63, 200, 1)), (6, 2, 1, (700, 33)),
    (2, 1, 5, (5, 64, 3)), (8, 2, 9, (130, 9, 70)), (3, 3, 17, (17, 100)), (16, 2, 33, (300, 90)),
    (8, 1, 70, (200, 70)), (4, 2, 130, (131, 400)),
])
def test_attention_of_the_newest_tokens(dtype, int8, D, H, H_kv, T, lens):
    # without a mask: causal among the new tokens; fewer cached tokens than new ones leave rows empty
    from sageattention import sageattn_cached
    gen = torch.Generator().manual_seed(T * H + D)
    cache, table = _filled(dtype, int8, H_kv, D, lens, gen)
    q, qg = _randn((len(lens), H, T, D), dtype, "HND", gen, 2.0)
    o, lse = sageattn_cached(qg, cache, table, _lens(*lens), return_lse=True)
    want, wl, slack = ref.attention(q, cache, table.cpu(), lens)
    ref.check_attention(o.cpu(), want, slack[0], dtype)
    ref.check_lse(lse.cpu(), wl, slack[1])
    nhd = sageattn_cached(qg.transpose(1, 2).contiguous(), cache, table, _lens(*lens), "NHD")
    assert torch.equal(nhd.transpose(1, 2), o)


@pytest.mark.parametrize("dtype,int8", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("D,H,H_kv,T,lens", [
    (128, 8, 2, 7, (7, 71, 300)), (64, 5, 5, 16, (64, 80, 17)), (128, 16, 2, 33, (100, 35)),
    (64, 4, 1, 64, (64, 190)), (128, 8, 1, 100, (100, 300)),
])
def test_attention_of_trees(dtype, int8, D, H, H_kv, T, lens):
    from sageattention import sageattn_cached
    B, gen = len(lens), torch.Generator().manual_seed(T + D)
    cache, table = _filled(dtype, int8, H_kv, D, lens, gen)
    q, qg = _randn((B, H, T, D), dtype, "NHD", gen, 2.0)
    mask = torch.stack([ref.random_tree(T, gen) for _ in range(B)])
    mask[0, T // 2] = False            # with a context of no token: a row that sees nothing
    q_lens = [T] + [max(1, T - 3 * b) for b in range(1, B)]
    for m, ql in ((mask, None), (mask[1], q_lens), (mask, q_lens)):
        o, lse = sageattn_cached(qg, cache, table, _lens(*lens), "NHD",
                                 q_lens=None if ql is None else _lens(*ql), tree_mask=m.cuda(),
                                 return_lse=True, sm_scale=0.11)
        want, wl, slack = ref.attention(q, cache, table.cpu(), lens, ql, m, 0.11)
        ref.check_attention(o.cpu().transpose(1, 2), want, slack[0], dtype)
        ref.check_lse(lse.cpu(), wl, slack[1])
    as_bytes = sageattn_cached(qg, cache, table, _lens(*lens), "NHD", q_lens=_lens(*q_lens),
                               tree_mask=mask.cuda().to(torch.uint8) * 3, sm_scale=0.11)
    assert torch.equal(as_bytes, o)
    wide = torch.zeros(B, T + 3, T + 5, dtype=torch.bool, device="cuda")
    wide[:, :T, :T] = mask.cuda()
    assert torch.equal(o, sageattn_cached(qg, cache, table, _lens(*lens), "NHD", q_lens=_lens(*q_lens),
                                          tree_mask=wide[:, :T, :T], sm_scale=0.11))


@pytest.mark.parametrize("H", [1, 4, 12])
@pytest.mark.parametrize("T", [1, 2, 3, 4, 5, 6, 9, 64, 67, 131])
def test_masks_at_every_place_of_a_page(T, H):
    # drafted tokens that begin anywhere in a page, masks of any bytes at any alignment, short drafts
    from sageattention import sageattn_cached
    gen = torch.Generator().manual_seed(1000 * H + T)
    starts = list(range(0, 67, 3)) + [126, 127, 128, 129, 190] + [-1, -T // 2]
    B, D = len(starts), 64
    q_lens = [T if b % 3 else max(1, T - b // 3) for b in range(B)]
    lens = [max(0, s + t) for s, t in zip(starts, q_lens)]
    cache, table = _filled(torch.float16, True, 1, D, lens, gen)
    q, qg = _randn((B, H, T, D), torch.float16, "HND", gen, 2.0)
    kinds = torch.tensor([0, 0, 0, 1, 1, 2, 127, 128, 129, 255], dtype=torch.uint8)
    pool = kinds[torch.randint(0, 10, (B, T, T + 5), generator=gen)].cuda()
    for at in (0, 1, 5):
        mask = pool[:, :, at:at + T]
        o, lse = sageattn_cached(qg, cache, table, _lens(*lens), q_lens=_lens(*q_lens), tree_mask=mask,
                                 return_lse=True)
        for b in range(B):
            n, t = lens[b], q_lens[b]
            k, v, _ = ref.gather(cache, table.cpu(), b, n)
            s = q[b].double() @ k[0].T / D ** 0.5
            draft = torch.arange(n) - (n - t)
            seen = (draft < 0) | (mask[b].cpu() != 0)[:, draft.clamp(min=0)]
            s[:, ~seen] = -torch.inf
            empty = ~seen.any(1) | (torch.arange(T) >= t)
            p = torch.softmax(s, -1)
            p[:, empty] = 0.0
            a = (q[b].double().abs() @ k[0].abs().T / D ** 0.5).amax() if n else 0.0
            # the bound of kv_cache_ref.attention
            err = 2 * ((D + 4) * 2.0 ** -23 * a + 2.0 ** -20) + 2.0 ** -12 + n * 2.0 ** -23
            spread = n * 2.0 ** -39 * v[0].abs().amax() if n else 0.0
            ref.check_attention(o[b].cpu(), p @ v[0], err * (p @ v[0].abs()) + spread, torch.float16)
            want = torch.logsumexp(s, -1)
            want[:, empty] = -torch.inf
            ref.check_lse(lse[b].cpu(), want, torch.full_like(want, err + 1e-5))


@pytest.mark.parametrize("dtype,int8", KINDS, ids=KIND_IDS)
def test_a_chain_mask_is_the_default(dtype, int8):
    from sageattention import sageattn_cached
    gen = torch.Generator().manual_seed(1)
    cache, table = _filled(dtype, int8, 2, 128, (200, 31), gen)
    _, q = _randn((2, 8, 31, 128), dtype, "HND", gen)
    chain = torch.ones(31, 31, dtype=torch.bool, device="cuda").tril()
    assert torch.equal(sageattn_cached(q, cache, table, _lens(200, 31), tree_mask=chain),
                       sageattn_cached(q, cache, table, _lens(200, 31)))


@pytest.mark.parametrize("dtype,int8", KINDS, ids=KIND_IDS)
def test_masked_tokens_that_are_not_finite_reach_only_who_sees_them(dtype, int8):
    from sageattention import sageattn_cached
    T, L, gen = 6, 80, torch.Generator().manual_seed(4)
    cache, table = _filled(dtype, int8, 2, 128, (L,), gen)
    bad = {2: float("nan"), 3: float("inf"), 4: torch.finfo(dtype).min}
    for which in ("k", "v", "kv"):
        rows = [(torch.randn(1, 2, 1, 128, generator=gen).to(dtype)) for _ in range(2)]
        for j, value in bad.items():
            k, v = rows[0].clone(), rows[1].clone()
            if "k" in which:
                k[..., 5] = value
            if "v" in which:
                v[..., 77] = value
            cache.write(k.cuda(), v.cuda(), table, _lens(L - T + j))
        # token i sees itself; 0 and 1 none of the bad ones; 5 sees 4, whose values are finite
        mask = torch.eye(T, dtype=torch.bool)
        mask[1, 0] = mask[5, 4] = True
        q, qg = _randn((1, 4, T, 128), dtype, "HND", gen)
        o = sageattn_cached(qg, cache, table, _lens(L), tree_mask=mask.cuda()).cpu()
        clean = [0, 1, 5] if "v" == which else [0, 1]
        assert torch.isfinite(o[:, :, [0, 1]]).all()
        assert torch.isnan(o[:, :, [2, 3]]).all()
        want, _, slack = ref.attention(q, cache, table.cpu(), [L], mask=mask)
        ref.check_attention(o[:, :, clean], want[:, :, clean], slack[0][:, :, clean], dtype)


@pytest.mark.parametrize("dtype,int8", KINDS, ids=KIND_IDS)
def test_value_scales_far_apart(dtype, int8):
    # V rows of very different sizes, the largest of them with no weight to speak of
    from sageattention import KVCache, sageattn_cached
    L, gen = 150, torch.Generator().manual_seed(6)
    cache = KVCache.allocate(4, 1, 128, dtype, int8)
    table = torch.tensor([[2, 0, 3]], dtype=torch.int32, device="cuda")
    k, v = torch.randn(2, 1, 1, L, 128, generator=gen)
    q = torch.randn(1, 2, 1, 128, generator=gen)
    size = 10.0 ** torch.randint(-6, 3, (L,), generator=gen).float()
    v = v * size[None, None, :, None]
    q, k, v = q.to(dtype), k.to(dtype), v.to(dtype)
    v[0, 0, 20] = 0
    k[0, 0, 100], v[0, 0, 100] = -4 * q[0, 0, 0], 60000
    cache.write(k.cuda(), v.cuda(), table, _lens(0))
    o, lse = sageattn_cached(q.cuda(), cache, table, _lens(L), return_lse=True)
    want, wl, slack = ref.attention(q, cache, table.cpu(), [L])
    ref.check_attention(o.cpu(), want, slack[0], dtype)
    ref.check_lse(lse.cpu(), wl, slack[1])


def test_tokens_never_written_count_as_zeros():
    from sageattention import KVCache, sageattn_cached
    cache = KVCache.allocate(1, 1, 64)
    one = torch.ones(1, 1, 1, 64, device="cuda", dtype=torch.float16)
    cache.write(one, one, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), _lens(0))
    o, lse = sageattn_cached(one * 0, cache, torch.zeros(1, 1, dtype=torch.int32, device="cuda"),
                             _lens(10), return_lse=True)
    assert (o.double() - 0.1).abs().max() <= 2.0 ** -11 * 0.1 + 1e-5
    assert (lse.double() - torch.log(torch.tensor(10.0))).abs().max() <= 1e-5


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", [3, 8, 40])
@pytest.mark.parametrize("L,B,H_kv", [(5000, 1, 2), (1100, 3, 1), (40000, 1, 1)])
def test_long_sequences_are_split_and_joined(L, B, H_kv, T, D):
    # split over many blocks, 12 to 160 rows of a K/V head
    from sageattention import sageattn_cached
    gen = torch.Generator().manual_seed(L)
    lens = [L - 97 * b for b in range(B)]
    cache, table = _filled(torch.float16, True, H_kv, D, lens, gen)
    q, qg = _randn((B, 4 * H_kv, T, D), torch.float16, "HND", gen, 2.0)
    o, lse = sageattn_cached(qg, cache, table, _lens(*lens), return_lse=True)
    again = sageattn_cached(qg, cache, table, _lens(*lens))
    assert torch.equal(o, again)       # sums have one order
    if L < 10000 and T == 3:
        want, wl, slack = ref.attention(q, cache, table.cpu(), lens)
        ref.check_attention(o.cpu(), want, slack[0], torch.float16)
        ref.check_lse(lse.cpu(), wl, slack[1])
        return
    for b in range(B):   # all rows of a sequence at once
        n = lens[b]
        k, v, _ = ref.gather(cache, table.cpu(), b, n)
        k, v = k.repeat_interleave(4, 0), v.repeat_interleave(4, 0)
        s = q[b].double() @ k.transpose(1, 2) / D ** 0.5
        a = (q[b].double().abs() @ k.abs().transpose(1, 2) / D ** 0.5).amax()
        late = torch.arange(n) > n - T + torch.arange(T)[:, None]
        s[:, late] = -torch.inf
        p = torch.softmax(s, -1)
        # the bound of kv_cache_ref.attention
        err = 2 * ((D + 4) * 2.0 ** -23 * a + 2.0 ** -20) + 2.0 ** -12 + n * 2.0 ** -23
        ref.check_attention(o[b].cpu(), p @ v, err * (p @ v.abs()), torch.float16)
        assert ((lse[b].cpu().double() - torch.logsumexp(s, -1)).abs() <= err + 1e-5).all()


@pytest.mark.parametrize("H,H_kv,D", [(8, 2, 128), (3, 3, 64)])
@pytest.mark.parametrize("T,past", [(300, 0), (257, 700), (601, 5), (128, 1500)])
def test_a_prompts_parts(T, past, H, H_kv, D):
    # many new tokens in causal order, after others or by themselves, of sequences that have fewer of them
    from sageattention import sageattn_cached
    gen = torch.Generator().manual_seed(T + past)
    q_lens = [T, T - 1, T - 130 if T > 140 else 3, 1, 0, T]
    lens = [past + t for t in q_lens[:5]] + [T // 2]
    cache, table = _filled(torch.float16, True, H_kv, D, lens, gen)
    q, qg = _randn((6, H, T, D), torch.float16, "HND", gen, 2.0)
    o, lse = sageattn_cached(qg, cache, table, _lens(*lens), q_lens=_lens(*q_lens), return_lse=True)
    for b, (n, t) in enumerate(zip(lens, q_lens)):
        k, v, _ = ref.gather(cache, table.cpu(), b, n)
        k, v = k.repeat_interleave(H // H_kv, 0), v.repeat_interleave(H // H_kv, 0)
        s = q[b].double() @ k.transpose(1, 2) / D ** 0.5
        a = (q[b].double().abs() @ k.abs().transpose(1, 2) / D ** 0.5).amax() if n else 0.0
        s[:, torch.arange(n) > n - t + torch.arange(T)[:, None]] = -torch.inf
        empty = (torch.arange(T) >= t) | (torch.arange(T) < t - n)
        p = torch.softmax(s, -1)
        p[:, empty] = 0.0
        # the bound of kv_cache_ref.attention
        err = 2 * ((D + 4) * 2.0 ** -23 * a + 2.0 ** -20) + 2.0 ** -12 + n * 2.0 ** -23
        spread = n * 2.0 ** -39 * v.abs().amax() if n else 0.0
        ref.check_attention(o[b].cpu(), p @ v, err * (p @ v.abs()) + spread, torch.float16)
        want = torch.logsumexp(s, -1) if n else torch.full((H, T), -torch.inf).double()
        want[:, empty] = -torch.inf
        ref.check_lse(lse[b].cpu(), want, torch.full_like(want, err + 1e-5))


@pytest.mark.parametrize("H,H_kv,T,D", [(16, 4, 8, 128), (16, 4, 8, 64), (8, 4, 1, 64), (4, 4, 3, 128),
                                        (4, 2, 50, 128), (8, 1, 40, 64)])
def test_many_ragged_sequences_in_runs(H, H_kv, T, D):
    # runs that end one plane, hold short ones whole and begin another; sequences without a token between
    from sageattention import sageattn_cached
    gen = torch.Generator().manual_seed(23)
    B = 68
    lens = [int(x) for x in torch.randint(0, 2600, (B,), generator=gen)]
    lens[::5] = [int(x) for x in torch.randint(0, 70, (len(lens[::5]),), generator=gen)]
    lens[0], lens[7], lens[8], lens[66], lens[67] = 2600, 0, 0, 1, 0
    cache, table = _filled(torch.bfloat16, False, H_kv, D, lens, gen)
    q, qg = _randn((B, H, T, D), torch.bfloat16, "HND", gen, 2.0)
    o, lse = sageattn_cached(qg, cache, table, _lens(*lens), return_lse=True)
    o, lse, at = o.cpu(), lse.cpu(), table.cpu()
    for b in range(B):
        n = lens[b]
        k, v, _ = ref.gather(cache, at, b, n)
        k, v = k.repeat_interleave(H // H_kv, 0), v.repeat_interleave(H // H_kv, 0)
        s = q[b].double() @ k.transpose(1, 2) / D ** 0.5
        a = (q[b].double().abs() @ k.abs().transpose(1, 2) / D ** 0.5).amax() if n else 0.0
        s[:, torch.arange(n) > n - T + torch.arange(T)[:, None]] = -torch.inf
        empty = torch.arange(T) < T - n
        p = torch.softmax(s, -1)
        p[:, empty] = 0.0
        # the bound of kv_cache_ref.attention
        err = 2 * ((D + 4) * 2.0 ** -23 * a + 2.0 ** -20) + 2.0 ** -12 + n * 2.0 ** -23
        spread = n * 2.0 ** -39 * v.abs().amax() if n else 0.0
        ref.check_attention(o[b], p @ v, err * (p @ v.abs()) + spread, torch.bfloat16)
        want = torch.logsumexp(s, -1) if n else torch.full((H, T), -torch.inf).double()
        want[:, empty] = -torch.inf
        ref.check_lse(lse[b], want, torch.full_like(want, err + 1e-5))


def test_more_planes_than_the_card_holds():
    # 2200 planes: a block for each, of any length
    from sageattention import sageattn_cached
    gen = torch.Generator().manual_seed(21)
    B, pick = 1100, [0, 1, 64, 300, 1030]
    lens = [pick[int(i)] for i in torch.randint(0, 5, (B,), generator=gen)]
    lens[B - 1] = 1030
    cache, table = _filled(torch.float16, True, 2, 64, lens, gen)
    q, qg = _randn((B, 6, 1, 64), torch.float16, "HND", gen, 2.0)
    o, lse = sageattn_cached(qg, cache, table, _lens(*lens), return_lse=True)
    some = [0, 1, 2, 3, 4, 5, 550, 800, B - 1]
    want, wl, slack = ref.attention(q[some], cache, table.cpu()[some], [lens[b] for b in some])
    ref.check_attention(o.cpu()[some], want, slack[0], torch.float16)
    ref.check_lse(lse.cpu()[some], wl, slack[1])


@pytest.mark.parametrize("T", [1, 20])
def test_sequences_that_share_pages_and_fused_queries(T):
    # a common prefix's pages in both tables, queries as a view of a fused projection
    from sageattention import KVCache, sageattn_cached
    gen = torch.Generator().manual_seed(22)
    cache = KVCache.allocate(40, 2, 128, torch.bfloat16)
    own = torch.randperm(40, generator=gen).int()
    table = torch.stack((own[:20], torch.cat((own[:12], own[20:28])))).cuda()
    _, k = _randn((2, 2, 1280, 128), torch.bfloat16, "HND", gen)
    _, v = _randn((2, 2, 1280, 128), torch.bfloat16, "HND", gen)
    lens = [1271, 1240]
    cache.write(k[:1], v[:1], table[:1], _lens(0), _lens(lens[0]))
    cache.write(k[1:, :, 768:], v[1:, :, 768:], table[1:], _lens(768), _lens(lens[1] - 768))
    fused = torch.randn(2, T, 3, 6, 128, generator=gen).bfloat16().cuda()
    for i in range(3):
        o = sageattn_cached(fused[:, :, i], cache, table, _lens(*lens), "NHD")
        want, _, slack = ref.attention(fused[:, :, i].transpose(1, 2).cpu(), cache, table.cpu(), lens)
        ref.check_attention(o.transpose(1, 2).cpu(), want, slack[0], torch.bfloat16)


@pytest.mark.parametrize("dtype,int8", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("H,H_kv,T,D", [(2, 2, 1, 128), (4, 1, 1, 64), (8, 2, 6, 128), (20, 2, 5, 64),
                                        (16, 1, 9, 128)])
@pytest.mark.parametrize("B", [5, 70, 131])
def test_ragged_batches(dtype, int8, H, H_kv, T, D, B):
    # many sequences of every length, none and fewer tokens than new ones among them: equal shares of all
    # their pages, each of which may end one sequence, hold several and begin another
    from sageattention import sageattn_cached
    gen = torch.Generator().manual_seed(B + T)
    pick = [0, 1, 63, 64, 65, 130, 200, 641, 1000]
    lens = [pick[int(i)] for i in torch.randint(0, len(pick), (B,), generator=gen)]
    lens[B // 2], lens[0], lens[B - 1] = 1500, 0, 0
    cache, table = _filled(dtype, int8, H_kv, D, lens, gen)
    q, qg = _randn((B, H, T, D), dtype, "HND", gen, 2.0)
    q_lens = torch.randint(0, T + 1, (B,), generator=gen).int() if T > 1 else None
    o, lse = sageattn_cached(qg, cache, table, _lens(*lens), return_lse=True,
                             q_lens=None if q_lens is None else q_lens.cuda())
    some = [0, 1, B // 2, B - 2, B - 1] + [int(i) for i in torch.randint(0, B, (8,), generator=gen)]
    want, wl, slack = ref.attention(q[some], cache, table.cpu()[some], [lens[b] for b in some],
                                    None if q_lens is None else q_lens[some])
    ref.check_attention(o.cpu()[some], want, slack[0], dtype)
    ref.check_lse(lse.cpu()[some], wl, slack[1])
    # and each as it comes out alone
    one = [b for b in range(B) if b % 7 == 0]
    for b in one:
        alone = sageattn_cached(qg[b:b + 1], cache, table[b:b + 1], _lens(lens[b]),
                                q_lens=None if q_lens is None else q_lens[b:b + 1].cuda())
        off = (alone[0].double() - o[b].double()).abs().cpu()
        assert (off <= 4 * ref.HALF_STEP[dtype] * o[b].double().abs().cpu()
                + 2 ** -10 * o[b].double().abs().max().cpu() + 1e-7).all()


def test_pools_beyond_32_bits():
    # codes of more than 2^32 bytes: pages at both ends, written, read and attended to
    from sageattention import KVCache, sageattn_cached
    gen = torch.Generator().manual_seed(7)
    num = 2 ** 32 // (64 * 128) + 5
    cache = KVCache.allocate(num, 1, 128, torch.bfloat16)
    table = torch.tensor([[num - 1, 0, num - 2, num // 2 + 1]], dtype=torch.int32, device="cuda")
    _, k = _randn((1, 1, 250, 128), torch.bfloat16, "HND", gen)
    _, v = _randn((1, 1, 250, 128), torch.bfloat16, "HND", gen)
    cache.write(k, v, table, _lens(0))
    for x, y in zip((k, v), cache.read(table, _lens(250), 250)):
        c, s = ref.quantize(x.float().cpu(), False)
        assert torch.equal(y.cpu(), (c * s[..., None]).bfloat16())
    q, qg = _randn((1, 2, 3, 128), torch.bfloat16, "HND", gen)
    want, _, slack = ref.attention(q, cache, table.cpu(), [250])
    ref.check_attention(sageattn_cached(qg, cache, table, _lens(250)).cpu(), want, slack[0],
                        torch.bfloat16)


# ------------------------------------------------------------------------------ used together
def test_decoding_with_drafted_trees():
    """Prompts, then rounds of drafted trees of which a path is kept: each round's attention against
    the 64-bit result over what the cache holds, and the cache against one that was never drafted into."""
    from sageattention import KVCache, apply_rotary, rotary_table, sageattn_cached
    B, H, H_kv, D, dtype, gen = 2, 8, 2, 128, torch.float16, torch.Generator().manual_seed(12)
    table = rotary_table(512, D, scaling="yarn", factor=4.0, original_length=128)
    cache, plain = (KVCache.allocate(12, H_kv, D, dtype) for _ in range(2))
    pages = _pages([190, 190], 12, gen)
    lens = torch.tensor([70, 41], dtype=torch.int32, device="cuda")
    pos = torch.arange(70, dtype=torch.int32, device="cuda").expand(B, 70)
    _, k = _randn((B, H_kv, 70, D), dtype, "HND", gen)
    _, v = _randn((B, H_kv, 70, D), dtype, "HND", gen)
    for c in (cache, plain):
        c.write(k, v, pages, _lens(0, 0), lens, table=table, positions=pos)
    T = 11
    for step in range(4):
        trees = torch.stack([ref.random_tree(T, gen) for _ in range(B)])
        depth = trees.sum(2).int() - 1
        pos = (lens.cpu()[:, None] + depth).cuda()
        q, qg = _randn((B, H, T, D), dtype, "HND", gen)
        _, k = _randn((B, H_kv, T, D), dtype, "HND", gen)
        _, v = _randn((B, H_kv, T, D), dtype, "HND", gen)
        cache.write(k, v, pages, lens, table=table, positions=pos)
        qr = apply_rotary(qg, table, pos)
        o = sageattn_cached(qr, cache, pages, lens + T, tree_mask=trees.cuda())
        want, _, slack = ref.attention(qr.cpu(), cache, pages.cpu(), (lens + T).tolist(), mask=trees)
        ref.check_attention(o.cpu(), want, slack[0], dtype)
        # the deepest token's path is kept: its rows are written again, in order
        path = [trees[b, int(depth[b].argmax())].nonzero()[:, 0] for b in range(B)]
        n = max(len(p) for p in path)
        at = torch.stack([torch.nn.functional.pad(p, (0, n - len(p))) for p in path]).cuda()
        pick = at[:, None, :, None].expand(B, H_kv, n, D)
        kept = _lens(*[len(p) for p in path])
        for c in (cache, plain):
            c.write(k.gather(2, pick), v.gather(2, pick), pages, lens, kept, table=table,
                    positions=pos.gather(1, at))
        lens = lens + kept
        for x, y in zip(cache.read(pages, lens, 190), plain.read(pages, lens, 190)):
            assert torch.equal(x, y)


def test_steps_replay_in_a_graph_as_sequences_grow():
    from sageattention import KVCache, apply_rotary, rotary_table, sageattn_cached
    B, H, H_kv, D, gen = 2, 8, 2, 128, torch.Generator().manual_seed(13)
    table, pages = rotary_table(4096, D), _pages([2000, 2000], 70, gen)
    caches = [KVCache.allocate(70, H_kv, D) for _ in range(2)]
    lens = torch.tensor([1300, 62], dtype=torch.int32, device="cuda")
    past = [torch.randn(B, H_kv, 1300, D, generator=gen).half().cuda() for _ in range(2)]
    for c in caches:
        c.write(*past, pages, _lens(0, 0), lens)
    q, k, v = (torch.empty(B, h, 1, D, device="cuda", dtype=torch.float16) for h in (H, H_kv, H_kv))

    def step(cache, lens):
        cache.write(k, v, pages, lens, table=table, positions=lens[:, None])
        return sageattn_cached(apply_rotary(q, table, lens[:, None]), cache, pages, lens + 1,
                               return_lse=True)
    grown = lens.clone()
    for t in (q, k, v):
        t.normal_()
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        step(caches[0], grown)
    torch.cuda.current_stream().wait_stream(warm)
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(caches[0], grown)
    with torch.cuda.graph(other):
        out2 = step(caches[0], grown)
    for i in range(5):
        for t, g in zip((q, k, v), (H, H_kv, H_kv)):
            t.copy_(torch.randn(B, g, 1, D, generator=gen).half())
        (graph if i % 2 else other).replay()
        got = [t.clone() for t in (out if i % 2 else out2)]
        want = step(caches[1], lens)
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        lens = lens + 1
        grown.copy_(lens)


def test_calls_run_on_the_current_stream():
    from sageattention import sageattn_cached
    gen = torch.Generator().manual_seed(14)
    cache, table = _filled(torch.float16, True, 8, 128, (4000, 100), gen)
    _, q = _randn((2, 32, 2, 128), torch.float16, "HND", gen)
    want = sageattn_cached(q, cache, table, _lens(4000, 100))
    lens = _lens(4000, 100)
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for i in range(8):
        with torch.cuda.stream(side[i % 2]):
            outs.append(sageattn_cached(q, cache, table, lens))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


# ---------------------------------------------------------------------------------- refusals
def test_refusals():
    from sageattention import KVCache, apply_rotary, rotary_table, sageattn_cached
    cache = KVCache.allocate(4, 2, 128)
    table = torch.zeros(1, 4, dtype=torch.int32, device="cuda")
    rot, pos = rotary_table(16, 128), torch.zeros(1, 3, dtype=torch.int32, device="cuda")
    q = torch.zeros(1, 4, 3, 128, device="cuda", dtype=torch.float16)
    k, lens = q[:, :2], _lens(3)

    def attn(reason, q=q, cache=cache, table=table, lens=lens, **kw):
        with pytest.raises(ValueError, match=reason):
            sageattn_cached(q, cache, table, lens, **kw)

    def write(reason, k=k, v=k, table=table, start=lens, lens=None, **kw):
        with pytest.raises(ValueError, match=reason):
            cache.write(k, v, table, start, lens, **kw)

    def rotary(reason, x=q, table=rot, positions=pos, **kw):
        with pytest.raises(ValueError, match=reason):
            apply_rotary(x, table, positions, **kw)
    attn("device", q=q.cpu())
    attn("layout", tensor_layout="NDH")
    attn("rank", q=q[0])
    attn("dtype", q=q.float())
    attn("dtype", q=q.bfloat16())
    attn("head_dim", q=q[..., :96])
    attn("head_dim", q=q[..., :64])
    attn("stride_align", q=torch.zeros(1, 4, 3, 132, device="cuda", dtype=torch.float16)[..., :128])
    attn("stride_last", q=q.transpose(2, 3).contiguous().transpose(2, 3))
    attn("heads", q=q[:, :3])
    attn("cache", cache=None)
    attn("seq_len", q=q[:, :, :0])
    attn("shape", table=table[0])
    attn("shape", table=torch.zeros(2, 4, dtype=torch.int32, device="cuda"))
    attn("dtype", table=table.long())
    attn("stride", table=torch.zeros(1, 8, dtype=torch.int32, device="cuda")[:, ::2])
    attn("device", lens=lens.cpu())
    attn("shape", lens=_lens(3, 3))
    attn("dtype", lens=lens.float())
    attn("shape", q_lens=_lens(3, 3))
    attn("sm_scale", sm_scale=0.0)
    attn("sm_scale", sm_scale=float("inf"))
    attn("shape", tree_mask=torch.ones(3, 4, dtype=torch.bool, device="cuda"))
    attn("shape", tree_mask=torch.ones(2, 3, 3, dtype=torch.bool, device="cuda"))
    attn("dtype", tree_mask=torch.ones(3, 3, device="cuda"))
    attn("device", tree_mask=torch.ones(3, 3, dtype=torch.bool))
    attn("stride", tree_mask=torch.ones(1, 3, dtype=torch.bool, device="cuda").expand(3, 3))
    attn("stride", tree_mask=torch.ones(3, 3, dtype=torch.bool, device="cuda").t())
    write("heads", k=q, v=q)
    write("heads", v=k[:, :, :2])
    write("dtype", k=k.bfloat16(), v=k.bfloat16())
    write("dtype", v=k.bfloat16())
    write("device", v=k.cpu())
    write("shape", start=_lens(1, 2))
    write("shape", lens=_lens(1, 2))
    write("table", positions=pos)
    write("device", table=table, start=lens, k=k.cpu(), v=k.cpu())
    with pytest.raises(ValueError, match="device: positions"):
        cache.write(k, k, table, lens, table=rot)
    rotary("table", table=rot.half())
    rotary("table", table=rot[:, :120])
    rotary("table", table=rotary_table(8, 144))
    rotary("shape", positions=pos[:, :2])
    rotary("dtype", positions=pos.long())
    rotary("stride_nonpos", x=q[:, :1].expand(1, 4, 3, 128))
    rotary("stride_overlap", x=torch.cat((q, q)), positions=torch.zeros(
        9, dtype=torch.int32, device="cuda").as_strided((2, 3), (1, 1)))
    for bad in (dict(dtype=torch.bfloat16, int8=True), dict(dtype=torch.float32), dict(head_dim=96),
                dict(num_pages=0)):
        with pytest.raises(ValueError, match="KVCache"):
            KVCache.allocate(**{**dict(num_pages=1, num_heads=1), **bad})
    with pytest.raises(ValueError, match="shape"):
        KVCache(cache.k8, cache.sk[:2], cache.v8, cache.sv)
    with pytest.raises(ValueError, match="seq_len"):
        cache.read(table, lens, 0)
    with pytest.raises(ValueError, match="layout"):
        cache.read(table, lens, 3, tensor_layout="DNH")
