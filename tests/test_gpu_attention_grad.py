"""`sageattn_backward` against the gradients' definition in 64 bits: types, head layouts, lengths from one
token on, odd sizes, strides, cut loops, rows that saw nothing, parts of the keys, graphs and streams."""
import pytest
import torch

from grad_ref import check, forward, gradients, hnd

pytestmark = pytest.mark.gpu


def case(B, H, H_kv, N, N_kv, D, dtype, causal, layout="HND", dlse=False, seed=0, size=2.0 ** -7,
         sm=None):
    """16-bit inputs of a backward call, and what it should give."""
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def rand(h, n, scale):
        shape = (B, h, n, D) if layout == "HND" else (B, n, h, D)
        return (scale * torch.randn(shape, generator=gen, device="cuda")).to(dtype)
    q, k, v, dout = rand(H, N, 2.0), rand(H_kv, N_kv, 1.0), rand(H_kv, N_kv, 1.0), rand(H, N, size)
    s = D ** -0.5 if sm is None else sm
    o, lse = forward(hnd(q, layout), hnd(k, layout), hnd(v, layout), causal, s)
    out = hnd(o.to(dtype), layout).contiguous()
    lse = lse.float()
    dl = size * torch.randn(B, H, N, generator=gen, device="cuda") if dlse else None
    return dict(dout=dout, q=q, k=k, v=v, out=out, lse=lse, tensor_layout=layout, is_causal=causal,
                sm_scale=sm, dlse=dl)


def wanted(c):
    l = c["tensor_layout"]
    s = c["q"].shape[-1] ** -0.5 if c["sm_scale"] is None else c["sm_scale"]
    return gradients(*(hnd(c[n], l) for n in ("dout", "q", "k", "v", "out")), c["lse"], c["dlse"],
                     c["is_causal"], s)


def verify(c, want=None, note=""):
    from sageattention import sageattn_backward
    got = sageattn_backward(**c)
    for g, n in zip(got, "qkv"):
        assert g.shape == c[n].shape and g.dtype == c[n].dtype and g.is_contiguous()
    share = check([hnd(g, c["tensor_layout"]) for g in got], want or wanted(c), note)
    print("share of the tolerance used: %.3f" % share)
    return got


F16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("N,N_kv,causal", [
    (64, 64, False), (64, 64, True), (1, 1, True), (1, 1, False), (2, 2, True), (31, 31, True),
    (33, 65, False), (63, 63, True), (65, 65, True), (127, 127, True), (128, 128, True),
    (129, 129, True), (1, 300, False), (300, 1, False), (257, 257, True), (257, 77, False),
    (40, 513, False), (640, 640, True)])
def test_lengths(dtype, D, N, N_kv, causal):
    verify(case(1, 2, 2, N, N_kv, D, dtype, causal, seed=N))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("layout", ["HND", "NHD"])
@pytest.mark.parametrize("B,H,H_kv,N,N_kv,D,causal,dlse", [
    (2, 8, 2, 200, 200, 128, True, True), (3, 6, 1, 90, 141, 64, False, False),
    (2, 5, 5, 321, 321, 64, True, False), (1, 12, 2, 130, 67, 128, False, True)])
def test_heads_and_layouts(dtype, layout, B, H, H_kv, N, N_kv, D, causal, dlse):
    verify(case(B, H, H_kv, N, N_kv, D, dtype, causal, layout, dlse))


@pytest.mark.parametrize("dtype,D", [(F16, 128), (BF16, 128), (F16, 64), (BF16, 64)])
@pytest.mark.parametrize("B,H,H_kv,N,N_kv,causal", [
    (1, 1, 1, 3000, 3000, True), (1, 4, 1, 2500, 70, False), (1, 3, 3, 50, 4100, False),
    (1, 8, 8, 1777, 1777, True), (9, 12, 4, 700, 700, True), (2, 10, 10, 1100, 1000, False)])
def test_cut_loops_and_full_grids(dtype, D, B, H, H_kv, N, N_kv, causal):
    verify(case(B, H, H_kv, N, N_kv, D, dtype, causal, dlse=causal))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("N,N_kv,causal", [
    (1, 1, True), (33, 33, True), (64, 64, True), (129, 129, True), (65, 31, False), (31, 130, False)])
@pytest.mark.parametrize("D", [64, 128])
def test_many_planes(dtype, N, N_kv, causal, D):
    """Short sequences by blocks of 128 columns (few planes take blocks of 64)."""
    verify(case(20, 16, 8, N, N_kv, D, dtype, causal, "NHD", dlse=not causal, seed=N))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_strides(dtype):
    """Views of fused projections, head slices, a gradient whose rows lie apart."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    B, N, H, D = 2, 150, 6, 64
    fused = torch.randn(B, N, 3, H, D, generator=gen, device="cuda").to(dtype)
    q, k, v = fused.unbind(2)                                        # NHD
    o, lse = forward(*(t.transpose(1, 2) for t in (q, k, v)), True, 0.2)
    wide = torch.zeros(B, N, H, 2 * D, dtype=dtype, device="cuda")
    wide[..., :D] = (2.0 ** -7 * torch.randn(B, N, H, D, generator=gen, device="cuda")).to(dtype)
    c = dict(dout=wide[..., :D], q=q, k=k, v=v, out=o.to(dtype).transpose(1, 2), lse=lse.float(),
             tensor_layout="NHD", is_causal=True, sm_scale=0.2, dlse=None)
    got = verify(c)
    same = verify(dict(c, **{n: c[n].contiguous() for n in ("dout", "q", "k", "v", "out")}))
    assert all(torch.equal(a, b) for a, b in zip(got, same))
    # heads of a larger HND tensor, physically NHD
    pool = torch.randn(B, N, 9, D, generator=gen, device="cuda").to(dtype).transpose(1, 2)
    q, k, v = pool[:, :6], pool[:, 6:8], pool[:, 7:9]
    o, lse = forward(q, k, v, False, D ** -0.5)
    verify(dict(dout=wide[..., :D].transpose(1, 2), q=q, k=k, v=v, out=o.to(dtype), lse=lse.float(),
                tensor_layout="HND", is_causal=False, sm_scale=None, dlse=None))


def test_rows_far_apart():
    """Rows as far apart as are served; one step further is refused."""
    from sageattention import sageattn_backward
    far = (1 << 24) - 8
    c = case(1, 1, 1, 65, 65, 64, BF16, True)
    store = torch.zeros(65 * far, dtype=BF16, device="cuda")
    for n in ("q", "k", "v", "dout", "out"):
        # the columns of each tensor at a place of their own
        at = 64 * ("q", "k", "v", "dout", "out").index(n)
        view = store[at:].as_strided((1, 1, 65, 64), (far, far, far, 1))
        view.copy_(c[n])
        c[n] = view
    verify(c)
    wide = store.as_strided((1, 1, 2, 64), (far + 8, far + 8, far + 8, 1))
    with pytest.raises(ValueError, match="stride_int32"):
        sageattn_backward(wide, wide, wide, wide, wide, torch.zeros(1, 1, 2, device="cuda"))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D,causal", [(64, True), (128, False)])
def test_rows_that_saw_nothing(dtype, D, causal):
    c = case(2, 4, 2, 200, 200, D, dtype, causal, dlse=True)
    empty = torch.rand(2, 4, 200, device="cuda") < 0.3
    empty[0, 0] = True                                  # a whole head
    c["lse"] = c["lse"].masked_fill(empty, -torch.inf)
    got = verify(c)
    assert (got[0][empty] == 0).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_parts_of_the_keys(dtype):
    """Two calls on parts of the keys with the whole's output and logsumexp give the whole's gradients."""
    c = case(1, 4, 2, 300, 400, 64, dtype, False, dlse=True)
    want = wanted(c)
    parts = []
    for at, to in ((0, 130), (130, 400)):
        part = dict(c, k=c["k"][:, :, at:to], v=c["v"][:, :, at:to])
        parts.append(verify(part))
    dq = parts[0][0].double() + parts[1][0].double()
    value, tol = want["dq"]
    # each part's share is rounded by itself
    u = torch.finfo(dtype).eps / 2
    assert ((dq - value).abs() <= tol + u * (parts[0][0].double().abs() + parts[1][0].double().abs())).all()
    for i, name in ((1, "dk"), (2, "dv")):
        value, tol = want[name]
        got = torch.cat((parts[0][i], parts[1][i]), 2).double()
        assert ((got - value).abs() <= tol).all(), name


@pytest.mark.parametrize("dtype,size", [(F16, 2.0 ** -20), (F16, 2.0 ** -14), (F16, 2.0 ** 6), (BF16, 2.0 ** -40),
                                        (BF16, 2.0 ** 20)])
def test_sizes_of_the_gradient(dtype, size):
    verify(case(1, 2, 1, 260, 260, 128, dtype, True, size=size))
    c = case(1, 2, 2, 200, 333, 64, dtype, False, size=size, dlse=True)
    # rows of very different sizes
    c["dout"] = c["dout"] * (2.0 ** -torch.arange(200, device="cuda").remainder(8))[:, None].to(dtype)
    verify(c)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("sm", [1e-3, 0.5, 1.0])
def test_scales_of_the_scores(dtype, sm):
    verify(case(1, 2, 2, 129, 129, 64, dtype, True, sm=sm))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D,H,H_kv,N,N_kv,causal", [
    (64, 6, 2, 100, 100, True), (64, 4, 2, 130, 384, False), (64, 3, 1, 1, 33, False), (128, 4, 4, 192, 192, True),
    (128, 6, 2, 60, 150, False), (64, 2, 2, 384, 384, True)])
def test_small_calls_in_one_launch(dtype, D, H, H_kv, N, N_kv, causal):
    """Blocks that work out their rows' constants by themselves: shared heads, ragged ends, rows that saw nothing,
    rows that lie apart."""
    from sageattention.sk1_backend.sk1_loader import SageLib
    assert SageLib.get().attn_bwd_workspace_bytes(dtype, causal, 1, H, N, H_kv, N_kv, D) == 0
    c = case(1, H, H_kv, N, N_kv, D, dtype, causal, "NHD", dlse=True, seed=D)
    empty = torch.rand(1, H, N, generator=torch.Generator("cuda").manual_seed(1), device="cuda") < 0.2
    c["lse"] = c["lse"].masked_fill(empty, -torch.inf)
    for n in ("dout", "out", "q"):
        wide = torch.zeros(1, N, H, D + 8, dtype=dtype, device="cuda")
        wide[..., :D] = c[n]
        c[n] = wide[..., :D]
    got = verify(c)
    assert (got[0].transpose(1, 2)[empty] == 0).all()
    assert all(torch.equal(a, b) for a, b in zip(got, verify(c)))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("B,H,H_kv,N,N_kv,layout", [
    (1, 2, 2, 1600, 77, "NHD"), (2, 3, 1, 1541, 128, "HND"), (1, 4, 2, 1000, 64, "NHD"), (1, 2, 1, 1777, 65, "HND"),
    (1, 4, 4, 1537, 1, "HND"), (1, 1, 1, 1999, 33, "NHD"), (40, 10, 10, 63, 96, "HND"), (3, 48, 12, 257, 97, "NHD"),
    (2, 40, 40, 1300, 17, "HND")])
def test_few_keys(dtype, B, H, H_kv, N, N_kv, layout):
    """Many queries on keys that one block holds: key counts around its tiles and its waves, ragged queries, shared
    heads, rows that saw nothing, one part and many."""
    c = case(B, H, H_kv, N, N_kv, 64, dtype, False, layout, dlse=True, seed=N_kv)
    empty = torch.rand(B, H, N, generator=torch.Generator("cuda").manual_seed(2), device="cuda") < 0.1
    c["lse"] = c["lse"].masked_fill(empty, -torch.inf)
    got = verify(c)
    dq = got[0] if layout == "HND" else got[0].transpose(1, 2)
    assert (dq[empty] == 0).all()
    assert all(torch.equal(a, b) for a, b in zip(got, verify(c)))


def test_few_keys_of_rows_of_unlike_size():
    """Each query's dS has a power of two of its own for dQ: gradients 2^-8 times their neighbours' lose nothing."""
    c = case(1, 2, 2, 1600, 77, 64, F16, False)
    small = torch.arange(1600, device="cuda") % 2 == 1
    c["dout"] = torch.where(small[:, None], c["dout"] * 2.0 ** -8, c["dout"])
    whole = verify(c)[0]
    c["dout"] = torch.where(small[:, None], c["dout"], torch.zeros_like(c["dout"]))
    alone = verify(c)[0]
    assert torch.equal(whole[:, :, small], alone[:, :, small])


@pytest.mark.parametrize("dtype,N_kv", [(F16, 131073), (BF16, 100000)])
def test_long_keys_and_long_queries(dtype, N_kv):
    """A few queries on many keys, and many queries on a few keys."""
    verify(case(1, 2, 1, 3, N_kv, 128, dtype, False))
    verify(case(1, 2, 1, N_kv, 5, 64, dtype, False))


def test_keys_past_32_bits():
    """K and V whose rows lie past 2^31 elements: heads of a long cache in 16 bits."""
    N_kv, heads = 300000, 60
    store = torch.zeros(1, N_kv, heads, 128, dtype=BF16, device="cuda")
    assert store.numel() > 1 << 31
    gen = torch.Generator(device="cuda").manual_seed(1)
    for h in (3, 59):
        store[:, :, h] = torch.randn(1, N_kv, 128, generator=gen, device="cuda").to(BF16)
    c = case(1, 1, 1, 40, 64, 128, BF16, False, "NHD")
    k, v = store[:, :, 59:], store[:, :, 3:4]
    o, lse = forward(*(t.transpose(1, 2) for t in (c["q"], k, v)), False, 128 ** -0.5)
    verify(dict(c, k=k, v=v, out=o.to(BF16).transpose(1, 2), lse=lse.float()))


def test_zero_gradient_is_zero():
    from sageattention import sageattn_backward
    for dtype in (F16, BF16):
        c = case(1, 4, 2, 200, 200, 128, dtype, True)
        c["dout"] = torch.zeros_like(c["dout"])
        assert all((g == 0).all() for g in sageattn_backward(**c))


def test_a_nan_stays_with_its_queries():
    """A row of dout that holds a NaN: its dq is NaN, the other rows' dq are as they were."""
    from sageattention import sageattn_backward
    for dtype in (F16, BF16):
        c = case(1, 2, 2, 200, 200, 64, dtype, False)
        before = sageattn_backward(**c)
        c["dout"] = c["dout"].clone()
        c["dout"][0, 1, 77, 5] = torch.nan
        dq, dk, dv = sageattn_backward(**c)
        others = torch.ones(1, 2, 200, dtype=torch.bool, device="cuda")
        others[0, 1, 77] = False
        assert torch.isnan(dq[0, 1, 77]).all() and torch.equal(dq[others], before[0][others])
        assert torch.isnan(dv[0, 1, :, 5]).all() and torch.isnan(dk[0, 1]).all()
        assert torch.isfinite(dk[0, 0]).all() and torch.isfinite(dv[0, 0]).all()


def test_the_same_bits_every_time():
    from sageattention import sageattn_backward
    for dims in ((1, 6, 1, 1541, 1541, 128, BF16, False), (1, 8, 2, 1777, 1777, 64, F16, True)):
        c = case(*dims)
        first = sageattn_backward(**c)
        for _ in range(5):
            assert all(torch.equal(a, b) for a, b in zip(first, sageattn_backward(**c)))


@pytest.mark.parametrize("dims", [(2, 8, 2, 333, 333, 128, BF16, True), (1, 6, 1, 1541, 700, 64, F16, False)])
def test_graph(dims):
    """A captured call, replayed on changed inputs with eager work between the replays."""
    from sageattention import sageattn_backward
    c = case(*dims, dlse=True)
    names = ("dout", "q", "k", "v", "out", "lse", "dlse")
    others = [case(*dims, dlse=True, seed=s) for s in (11, 12, 13)]
    sageattn_backward(**c)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = sageattn_backward(**c)
    for o in others:
        eager = sageattn_backward(**o)
        for n in names:
            c[n].copy_(o[n])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, eager))


def test_two_streams():
    from sageattention import sageattn_backward
    cases = [case(1, 6, 1, 1541, 1541, 128, BF16, True), case(2, 4, 4, 900, 900, 64, F16, False)]
    want = [sageattn_backward(**c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(4):
        got = []
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(sageattn_backward(**c))
        torch.cuda.synchronize()
        for w, g in zip(want, got):
            assert all(torch.equal(a, b) for a, b in zip(w, g))


def test_offsets_past_32_bits():
    """More than 2^31 elements in q, out, dout and dq: the last heads' rows, and sums over all heads."""
    from sageattention import sageattn_backward
    H, N, N_kv, D = 257, 65600, 33, 128
    gen = torch.Generator(device="cuda").manual_seed(5)

    def rand(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=BF16)
    q, dout = rand(1, H, N, D), rand(1, H, N, D)
    assert q.numel() > 1 << 31
    k, v = rand(1, 1, N_kv, D), rand(1, 1, N_kv, D)
    out, lse = torch.empty_like(q), torch.empty(1, H, N, device="cuda")
    for h in range(H):
        s = q[0, h].float() @ k[0, 0].float().T.contiguous() * D ** -0.5
        lse[0, h] = torch.logsumexp(s, 1)
        out[0, h] = (torch.softmax(s, 1) @ v[0, 0].float()).to(BF16)
    dq, dk, dv = sageattn_backward(dout, q, k, v, out, lse)
    value = {n: torch.zeros(N_kv, D, dtype=torch.float64, device="cuda") for n in ("dk", "dv")}
    size = {n: torch.zeros(N_kv, D, dtype=torch.float64, device="cuda") for n in ("dk", "dv")}
    kk, vv = k[0, 0].double(), v[0, 0].double()
    for h in range(H):
        qq, gg, oo = (t[0, h].double() for t in (q, dout, out))
        p = torch.exp(qq @ kk.T.contiguous() * D ** -0.5 - lse[0, h].double()[:, None])
        ds = p * (gg @ vv.T.contiguous() - (gg * oo).sum(1, keepdim=True)) * D ** -0.5
        if h in (0, 128, H - 1):
            want = ds @ kk
            # bf16's roundings of dS and of the result, and fp32's of dS's terms
            tol = 2.0 ** -7 * (ds.abs() @ kk.abs()) + 2.0 ** -8 * want.abs() + 1e-3
            assert ((dq[0, h].double() - want).abs() <= tol).all(), h
        for n, w, x in (("dv", p, gg), ("dk", ds, qq)):
            value[n] += w.T.contiguous() @ x
            size[n] += w.abs().T.contiguous() @ x.abs()
    for n, got in (("dk", dk), ("dv", dv)):
        # 1.7e7 products: roundings of 2^-8 of each, random, and the sum in fp32
        assert ((got[0, 0].double() - value[n]).abs() <= 2.0 ** -8 * value[n].abs() + 2.0 ** -11 * size[n]).all(), n


def test_refusals():
    from sageattention import sageattn_backward
    c = case(1, 4, 2, 40, 40, 64, BF16, True)

    def refused(match, **changed):
        with pytest.raises(ValueError, match=match):
            sageattn_backward(**dict(c, **changed))
    refused("layout", tensor_layout="BHND")
    refused("device", q=c["q"].cpu())
    refused("device", lse=c["lse"].cpu())
    refused("device", dlse=1.0)
    refused("rank", q=c["q"][0])
    refused("dtype", q=c["q"].float())
    refused("dtype", dout=c["dout"].half())
    refused("dtype", lse=c["lse"].double())
    refused("head_dim", **{n: c[n][..., :32] for n in ("q", "k", "v", "out", "dout")})
    refused("shape", v=c["v"][:, :, :39])
    refused("shape", out=c["out"][:, :, :39])
    refused("shape", dout=c["dout"][:, :3])
    refused("shape", k=c["k"].repeat(2, 1, 1, 1), v=c["v"].repeat(2, 1, 1, 1))
    refused("shape", lse=c["lse"][:, :, :39])
    refused("shape", dlse=c["lse"][:, :3])
    refused("heads", k=c["q"][:, :3], v=c["q"][:, :3])
    refused("seq_len", k=c["k"][:, :, :39].contiguous(), v=c["v"][:, :, :39].contiguous())
    refused("seq_len", **{n: c[n][:, :, :0] for n in ("q", "k", "v", "out", "dout")})
    refused("stride_last", dout=c["dout"].transpose(2, 3).contiguous().transpose(2, 3))
    refused("stride_last", lse=c["lse"].transpose(1, 2).contiguous().transpose(1, 2))
    refused("stride_nonpos", dout=c["dout"][:, :1].expand(1, 4, 40, 64))
    refused("sm_scale", sm_scale=0.0)
    refused("sm_scale", sm_scale=float("nan"))
    refused("sm_scale", sm_scale=1e-31)
    verify(c)
