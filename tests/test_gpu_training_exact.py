"""The gradients of `sageattn_train`, from q, k and v alone, against those of attention itself in 64 bits.

Nothing of the forward call enters the expectation: its output and logsumexp are those of 8-bit scores, which
differ from the 16-bit scores' by more than the gradients' roundings as soon as scores spread by more than one or
K has a mean.

Tolerances count roundings as `grad_ref` does, with the logsumexp and d = sum_j P_ij dP_ij as the pass forms them. With
E = 2^-24, s the score, z = sm |q||k| its terms' sizes, w = |dout||v| those of dP's, n the keys:
    score, exponent     e = (D + 8) E z + (D / 16 + 8) E (|lse| + 1)
    logsumexp           sum_j P_j e_j + 2 n E + 4 E (|lse| + 1)
    P, relative         a = e + that
    d                   sum_j P_j (a_j + (D + 3 + n) E) w_j
    dS                  |dS| (a + u + 4 E) + P ((D + 3) E (w + |d| + |dlse|) + error of d)
    P, for dV           P (u + a + N G E)
and the roundings of sums, results and fp16's subnormal numbers as there.
bf16 has fp32's exponents, and the exponential and the matrix instructions hold no numbers under 2^-126: a weight, a
dS or a sum under it is off by all of it. (Scores of spread 100 have keys whose weights are all e^-88 = 2^-127 or less:
their dV and dK are 1e-39 and come out as 0.)
"""
import pytest
import torch

from grad_ref import E, U, check, forward, hnd, mm, seen_of

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
TINY = 2.0 ** -126


def exact_gradients(dout, q, k, v, dlse, causal, sm):
    """{"dq": (value, tolerance), ..} of (B, H, N, D) tensors, head by head."""
    u, f16 = U[q.dtype], q.dtype == F16
    B, H, N, D = q.shape
    H_kv, n = k.shape[1:3]
    G = H // H_kv
    want = {x: [torch.zeros(t.shape, dtype=torch.float64, device=q.device) for _ in range(2)]
            for x, t in (("dq", q), ("dk", k), ("dv", v))}
    seen = seen_of(N, n, causal, q.device)
    for b in range(B):
        for h in range(H):
            hk = h // G
            qq, gg, kk, vv = (t.double() for t in (q[b, h], dout[b, h], k[b, hk], v[b, hk]))
            dl = torch.zeros(N, 1, dtype=torch.float64, device=q.device) if dlse is None \
                else dlse[b, h].double()[:, None]
            s = (mm(qq, kk) * sm).masked_fill(~seen, -torch.inf)
            lse = torch.logsumexp(s, 1, keepdim=True)
            p = torch.exp(s - lse)
            dp = mm(gg, vv)
            d = (p * dp).sum(1, keepdim=True)
            ds = p * (dp - d + dl)
            e = (D + 8) * E * sm * mm(qq.abs(), kk.abs()) + (D / 16 + 8) * E * (lse.abs() + 1)
            a = e + (p * e).sum(1, keepdim=True) + 2 * n * E + 4 * E * (lse.abs() + 1)
            w = mm(gg.abs(), vv.abs())
            err_d = (p * (a + (D + 3 + n) * E) * w).sum(1, keepdim=True)
            err = ds.abs() * (a + u + 4 * E) + p * ((D + 3) * E * (w + d.abs() + dl.abs()) + err_d)
            perr = p * (u + a + N * G * E)
            if f16:
                # dK's power of two is one for the group's heads
                group = dout[b, hk * G:(hk + 1) * G].double()
                bound = group.norm(dim=-1).max() * vv.norm(dim=1).max() * 2 + dl.abs().max()
                perr = perr + 2.0 ** -37 * (p > 0)
                err = err + 2.0 ** -38 * bound * (p > 0)
            else:
                perr = perr + TINY * (p > 0)
                err = err + TINY * (1 + w + d.abs() + dl.abs()) * (p > 0)
            want["dv"][0][b, hk] += p.t().contiguous() @ gg
            want["dv"][1][b, hk] += perr.t().contiguous() @ gg.abs()
            want["dq"][0][b, h] = sm * (ds @ kk)
            want["dq"][1][b, h] = sm * ((err + n * E * ds.abs()) @ kk.abs())
            want["dk"][0][b, hk] += sm * (ds.t().contiguous() @ qq)
            want["dk"][1][b, hk] += sm * ((err + N * G * E * ds.abs()).t().contiguous() @ qq.abs())
    least = torch.finfo(q.dtype).smallest_normal * torch.finfo(q.dtype).eps if f16 else TINY
    return {x: (value, tol + u * value.abs() + least) for x, (value, tol) in want.items()}


def inputs(B, H, H_kv, N, N_kv, D, dtype, layout="HND", spread=1.0, mean=0.0, seed=0):
    """q, k, v and gradients of the output and of the logsumexp: scores of a given spread, four of K's columns around
    a mean."""
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def rand(h, n, size):
        shape = (B, h, n, D) if layout == "HND" else (B, n, h, D)
        return size * torch.randn(shape, generator=gen, device="cuda")
    q, k, v, dout = (rand(H, N, spread ** 0.5), rand(H_kv, N_kv, spread ** 0.5), rand(H_kv, N_kv, 1.0),
                     rand(H, N, 2.0 ** -7))
    k[..., ::D // 4] += mean
    dlse = 2.0 ** -7 * torch.randn(B, H, N, generator=gen, device="cuda")
    return [t.to(dtype) for t in (q, k, v, dout)] + [dlse]


def verify(got, q, k, v, dout, dlse, layout, causal, sm=None):
    sm = q.shape[-1] ** -0.5 if sm is None else sm
    dout, q, k, v = (hnd(t.detach(), layout) for t in (dout, q, k, v))
    share = check([hnd(t, layout) for t in got], exact_gradients(dout, q, k, v, dlse, causal, sm))
    print("share of the tolerance used: %.3f" % share)


@pytest.mark.parametrize("mean", [0.0, 10.0])
@pytest.mark.parametrize("spread", [1.0, 4.0, 20.0, 100.0])
@pytest.mark.parametrize("dtype,int8", [(F16, None), (F16, False), (BF16, None)])
@pytest.mark.parametrize("B,H,H_kv,N,N_kv,D,causal,layout", [
    (1, 4, 2, 600, 600, 128, True, "HND"), (2, 6, 2, 257, 333, 64, False, "NHD")])
def test_gradients_are_attentions(B, H, H_kv, N, N_kv, D, causal, layout, dtype, int8, spread, mean):
    """Scores of every spread and K with a mean, both kinds of 8-bit products in the forward call."""
    from sageattention import sageattn, sageattn_train
    q, k, v, dout, dlse = inputs(B, H, H_kv, N, N_kv, D, dtype, layout, spread, mean)
    q, k, v = (t.requires_grad_() for t in (q, k, v))
    out, lse = sageattn_train(q, k, v, layout, causal, return_lse=True, sk1_int8=int8)
    with torch.no_grad():
        want = sageattn(q, k, v, layout, causal, return_lse=True, sk1_int8=int8)
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    got = torch.autograd.grad((out, lse), (q, k, v), (dout, dlse), retain_graph=True)
    verify(got, q, k, v, dout, dlse, layout, causal)
    got = torch.autograd.grad(out, (q, k, v), dout)
    verify(got, q, k, v, dout, None, layout, causal)


def test_weights_over_their_range_in_the_forward_calls_logsumexp():
    """Scores whose 8-bit forms are off by more than the 16 that fp16's weights have room for: finite gradients."""
    from sageattention import sageattn_train
    q, k, v, dout, _ = inputs(1, 4, 4, 2048, 2048, 128, F16, spread=100.0)
    q, k, v = (t.requires_grad_() for t in (q, k, v))
    got = torch.autograd.grad(sageattn_train(q, k, v, is_causal=True), (q, k, v), dout)
    verify(got, q, k, v, dout, None, "HND", True)


def test_a_causal_first_row_weighs_its_key_with_one():
    """One key alone: its weight is 1 whatever the scores, so dV is dout and dS is dlse."""
    from sageattention import sageattn_train
    for dtype in (F16, BF16):
        q, k, v, dout, dlse = inputs(3, 2, 2, 1, 1, 64, dtype, spread=30.0, mean=10.0)
        q, k, v = (t.requires_grad_() for t in (q, k, v))
        out, lse = sageattn_train(q, k, v, is_causal=True, return_lse=True)
        got = torch.autograd.grad((out, lse), (q, k, v), (dout, dlse))
        assert torch.equal(got[2], dout)
        verify(got, q, k, v, dout, dlse, "HND", True)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("B,H,H_kv,N,N_kv,D,causal,layout", [
    (1, 1, 1, 1, 1, 64, True, "HND"), (1, 2, 1, 3, 20000, 128, False, "HND"), (1, 2, 2, 300, 1, 64, False, "NHD"),
    (1, 8, 2, 257, 257, 64, True, "NHD"), (1, 2, 1, 129, 129, 128, True, "HND"), (2, 3, 1, 63, 191, 128, False, "NHD"),
    (1, 1, 1, 3000, 3000, 64, True, "HND"), (1, 6, 2, 1541, 1541, 128, True, "NHD"), (1, 4, 2, 2500, 70, 64, False, "HND"),
    (20, 16, 8, 65, 65, 64, True, "NHD"), (20, 8, 8, 40, 513, 128, False, "HND"), (1, 3, 3, 50, 4100, 64, False, "HND")])
def test_without_the_forward_calls_results(B, H, H_kv, N, N_kv, D, causal, layout, dtype):
    """sageattn_backward on its own: from one row on, tiles of both widths, cut and whole; the same bits again."""
    from sageattention import sageattn_backward
    q, k, v, dout, dlse = inputs(B, H, H_kv, N, N_kv, D, dtype, layout, 3.0, 2.0, seed=N)
    for dl in (dlse, None):
        got = sageattn_backward(dout, q, k, v, tensor_layout=layout, is_causal=causal, sm_scale=0.1, dlse=dl)
        verify(got, q, k, v, dout, dl, layout, causal, 0.1)
        again = sageattn_backward(dout, q, k, v, None, None, layout, causal, 0.1, dl)
        assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("sm", [1e-30, 1e-3, 1.0, 30.0])
def test_scales_of_the_scores(dtype, sm):
    """Weights all alike, up to one weight alone."""
    from sageattention import sageattn_backward
    q, k, v, dout, dlse = inputs(1, 4, 2, 150, 200, 64, dtype)
    verify(sageattn_backward(dout, q, k, v, sm_scale=sm, dlse=dlse), q, k, v, dout, dlse, "HND", False, sm)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_strides(dtype):
    """Views of a fused projection, and a gradient whose rows lie apart."""
    from sageattention import sageattn_backward
    fused = inputs(2, 18, 18, 150, 150, 64, dtype, "NHD")[1].unflatten(2, (3, 6))
    q, k, v = fused.unbind(2)
    wide = torch.zeros(2, 150, 6, 136, dtype=dtype, device="cuda")
    wide[..., :64] = inputs(2, 6, 6, 150, 150, 64, dtype, "NHD", seed=1)[3]
    dout = wide[..., :64]
    got = sageattn_backward(dout, q, k, v, tensor_layout="NHD", is_causal=True)
    verify(got, q, k, v, dout, None, "NHD", True)
    same = sageattn_backward(*(t.contiguous() for t in (dout, q, k, v)), tensor_layout="NHD", is_causal=True)
    assert all(torch.equal(a, b) for a, b in zip(got, same))


@pytest.mark.parametrize("dtype,causal", [(F16, True), (BF16, False)])
def test_against_differences(dtype, causal):
    """The 64-bit loss's change along a direction, with the logsumexp in it, is the gradients' product with it."""
    from sageattention import sageattn_backward
    q, k, v, dout, dlse = inputs(1, 2, 2, 130, 130, 64, dtype, spread=2.0, mean=3.0)
    got = sageattn_backward(dout, q, k, v, is_causal=causal, dlse=dlse)
    want = exact_gradients(dout, q, k, v, dlse, causal, 0.125)
    step = 1e-4
    for i, name in enumerate(("dq", "dk", "dv")):
        along = torch.randn(q.shape, dtype=torch.float64, device="cuda")

        def loss(h):
            args = [q.double(), k.double(), v.double()]
            args[i] = args[i] + h * along
            o, lse = forward(*args, causal, 0.125)
            return (o * dout.double()).sum() + (lse * dlse.double()).sum()
        change = (loss(step) - loss(-step)) / (2 * step)
        tol = (want[name][1] * along.abs()).sum()
        assert ((got[i].double() * along).sum() - change).abs() <= tol + 1e-6 * change.abs(), name


def test_graph_and_streams():
    """Captured and replayed on other inputs with eager work between; two calls on two streams at once."""
    from sageattention import sageattn_backward
    dims = (1, 6, 2, 1541, 1541, 128, BF16)

    def call(q, k, v, dout, dlse):
        return sageattn_backward(dout, q, k, v, is_causal=True, dlse=dlse)
    held = inputs(*dims)
    call(*held)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call(*held)
    for seed in (11, 12, 13):
        other = inputs(*dims, seed=seed)
        eager = call(*other)
        for a, b in zip(held, other):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, eager))
    sets = [inputs(*dims, seed=s) for s in (1, 2)]
    want = [call(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for x, stream in zip(sets, streams):
            with torch.cuda.stream(stream):
                got.append(call(*x))
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert all(torch.equal(s, t) for s, t in zip(a, b))


def test_merged_parts_by_autograd():
    """Attention over parts of the keys, merged in torch by the parts' logsumexp: autograd carries the merge's gradients
    into each part's call. Against a merge of 64-bit parts, along the path that each part's tolerance covers."""
    from sageattention import sageattn_train
    q, k, v, dout, _ = inputs(1, 4, 2, 200, 300, 64, F16, spread=2.0)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    parts = [sageattn_train(q, k[:, :, a:b], v[:, :, a:b], return_lse=True) for a, b in ((0, 130), (130, 300))]
    for p in parts:
        for t in p:
            t.retain_grad()
    weights = torch.softmax(torch.stack([p[1] for p in parts]), 0)
    merged = sum(p[0].float() * w[..., None] for p, w in zip(parts, weights))
    got = torch.autograd.grad(merged, leaves + [t for p in parts for t in p], dout.float())
    with torch.no_grad():
        ends = ((0, 130), (130, 300))
        dq, tol = 0.0, 0.0
        for i, (a, b) in enumerate(ends):
            want = exact_gradients(got[3 + 2 * i], q, k[:, :, a:b], v[:, :, a:b], got[4 + 2 * i], False, 0.125)
            for x, name in ((got[1], "dk"), (got[2], "dv")):
                assert ((x[:, :, a:b].double() - want[name][0]).abs() <= want[name][1]).all()
            dq, tol = dq + want["dq"][0], tol + want["dq"][1] + U[F16] * want["dq"][0].abs()
        assert ((got[0].double() - dq).abs() <= tol + U[F16] * dq.abs()).all()


def test_refusals():
    from sageattention import sageattn_backward
    q, k, v, dout, dlse = inputs(1, 4, 2, 40, 40, 64, BF16)
    for kept in (dict(out=dout), dict(lse=dlse)):
        with pytest.raises(ValueError, match="out and lse|lse must be"):
            sageattn_backward(dout, q, k, v, **kept)
    with pytest.raises(ValueError, match="dtype"):
        sageattn_backward(dout.half(), q, k, v)
    with pytest.raises(ValueError, match="shape: dout"):
        sageattn_backward(dout[:, :3], q, k, v)
    with pytest.raises(ValueError, match="shape: dlse"):
        sageattn_backward(dout, q, k, v, dlse=dlse[:, :3])
    with pytest.raises(ValueError, match="device"):
        sageattn_backward(dout.cpu(), q, k, v)
    verify(sageattn_backward(dout, q, k, v, dlse=dlse), q, k, v, dout, dlse, "HND", False)


class _Attention64(torch.autograd.Function):
    """Causal attention with a given result, its gradients those of attention in 64 bits on q, k and v."""
    @staticmethod
    def forward(ctx, q, k, v, out):
        ctx.save_for_backward(q, k, v)
        return out.double()

    @staticmethod
    def backward(ctx, g):
        with torch.enable_grad():
            q, k, v = (t.detach().requires_grad_() for t in ctx.saved_tensors)
            out = forward(q, k, v, True, q.shape[-1] ** -0.5)[0]
        return torch.autograd.grad(out, (q, k, v), g) + (None,)


def test_block_of_a_transformer():
    """norm with the residual -> projection -> norm of heads -> attention -> projection -> norm: the gradients of all
    parameters and of the input against the same block in 64 bits, where attention's come from its inputs alone."""
    from sageattention import rms_norm, sageattn_train
    B, N, H, H_kv, D = 2, 257, 4, 2, 64
    n, heads = H * D, H + 2 * H_kv

    def rand(*shape, seed, size=1.0):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        return (size * torch.randn(shape, generator=gen, device="cuda")).to(F16)
    params = dict(w1=rand(n, seed=1) * 0.1 + 1, wqkv=rand(heads * D, n, seed=2, size=n ** -0.5),
                  wq=rand(D, seed=3) * 0.1 + 1, wk=rand(D, seed=4) * 0.1 + 1,
                  wo=rand(n, n, seed=5, size=n ** -0.5), w2=rand(n, seed=6) * 0.1 + 1)
    x, hidden, grad = rand(B, N, n, seed=7), rand(B, N, n, seed=8), rand(B, N, n, seed=9, size=2.0 ** -6)
    seen = {}

    def block(p, x, hidden, norm, attend):
        y, total = norm(x, p["w1"], hidden)
        qkv = (y @ p["wqkv"].t()).unflatten(-1, (heads, D))
        q, k, v = qkv[:, :, :H], qkv[:, :, H:H + H_kv], qkv[:, :, H + H_kv:]
        o = attend(norm(q, p["wq"], None), norm(k, p["wk"], None), v)
        return norm(o.reshape(B, N, n) @ p["wo"].t(), p["w2"], total)[0]

    def attend16(q, k, v):
        out = sageattn_train(q, k, v, "NHD", True)
        seen["out"] = out.detach()
        return out

    def norm64(t, w, residual):
        t = t if residual is None else t + residual
        y = t / torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-6) * w
        return y if residual is None else (y, t)

    def attend64(q, k, v):
        return _Attention64.apply(*(t.transpose(1, 2) for t in (q, k, v, seen["out"]))).transpose(1, 2)
    leaves = {name: t.clone().requires_grad_() for name, t in dict(params, x=x, hidden=hidden).items()}
    block(leaves, leaves["x"], leaves["hidden"], lambda t, w, r: rms_norm(t, w, 1e-6, residual=r),
          attend16).backward(grad)
    exact = {name: t.double().requires_grad_() for name, t in dict(params, x=x, hidden=hidden).items()}
    block(exact, exact["x"], exact["hidden"], norm64, attend64).backward(grad.double())
    for name, t in leaves.items():
        want = exact[name].grad
        rel = ((t.grad.double() - want).norm() / want.norm()).item()
        # forward and backward pass through about 20 roundings of 2^-11 at most each, and the attention's
        # gradients see scores that the roundings of q and k, at 2^-11 of |score| = 8 or less, have moved
        assert rel <= 30 * 2.0 ** -11, (name, rel)
        print(name, "%.2g" % rel)


@pytest.mark.parametrize("D,N,causal", [(64, 200, False), (64, 700, True), (128, 150, True), (128, 2048, True)])
def test_a_logsumexp_under_its_scores(D, N, causal):
    """A given logsumexp that is some units under that of the scores, as one of scores of fewer bits may be: fp16's weights
    end at 2^1.99 in place of infinity, those under it are the formula's, and results stay finite."""
    from sageattention import sageattn_backward
    q, k, v, dout, _ = inputs(1, 2, 2, N, N, D, F16, spread=4.0)
    out, lse = forward(q, k, v, causal, D ** -0.5)
    for less in (2.0, 5.0, 40.0):
        got = sageattn_backward(dout, q, k, v, out.half(), (lse - less).float(), is_causal=causal)
        assert all(torch.isfinite(t).all() for t in got), less
        s = (mm(q[0].double(), k[0].double()) * D ** -0.5).masked_fill(~seen_of(N, N, causal, "cuda"), -torch.inf)
        p = torch.exp(s - (lse - less).float()[0, ..., None])
        held = p.clamp(max=2.0 ** 1.99)
        e = (D + 8) * E * D ** -0.5 * mm(q[0].double().abs(), k[0].double().abs()) + (D / 16 + 8) * E * (lse[0, ..., None].abs() + less + 1)
        want = held.transpose(1, 2).contiguous() @ dout[0].double()
        tol = (held * (U[F16] + e + N * E) + 2.0 ** -37).transpose(1, 2).contiguous() @ dout[0].double().abs() + U[F16] * want.abs()
        assert ((got[2][0].double() - want).abs() <= tol + 2.0 ** -24).all(), less


def test_the_forward_calls_own_results_stay_finite():
    from sageattention import sageattn, sageattn_backward
    q, k, v, dout, _ = inputs(1, 4, 4, 2048, 2048, 128, F16, spread=100.0)
    out, lse = sageattn(q, k, v, is_causal=True, return_lse=True)
    assert all(torch.isfinite(t).all() for t in sageattn_backward(dout, q, k, v, out, lse, is_causal=True))


def test_results_past_fp16_are_infinite():
    """A gradient over 65504 comes out as infinity, which a loss scale is lowered by, not as the largest number."""
    from sageattention import sageattn_backward
    for N in (70, 3000):
        q, k, v, _, _ = inputs(1, 2, 2, N, N, 64, F16)
        dout = torch.full_like(q, 60000.0)
        dv = sageattn_backward(dout, q, k, v, is_causal=True)[2]
        assert torch.isposinf(dv[0, :, 0]).all()        # key 0: the sum of all rows' weights on it is over 1.1


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_a_nan_stays_with_its_queries(dtype):
    """A query's or a gradient's NaN: that row's dq, and its head's dk and dv; the other rows' dq are as they were."""
    from sageattention import sageattn_backward
    q, k, v, dout, _ = inputs(1, 2, 2, 200, 200, 64, dtype)
    before = sageattn_backward(dout, q, k, v)
    others = torch.ones(1, 2, 200, dtype=torch.bool, device="cuda")
    others[0, 1, 77] = False
    for t in (q, dout):
        was = t[0, 1, 77, 5].item()
        t[0, 1, 77, 5] = torch.nan
        dq, dk, dv = sageattn_backward(dout, q, k, v)
        t[0, 1, 77, 5] = was
        assert torch.isnan(dq[0, 1, 77]).all() and torch.equal(dq[others], before[0][others])
        assert torch.isnan(dk[0, 1]).all() and torch.isnan(dv[0, 1, :, 5]).all()
        assert torch.equal(dk[0, 0], before[1][0, 0]) and torch.equal(dv[0, 0], before[2][0, 0])


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_rows_without_a_gradient_count_for_nothing(dtype):
    """A padded batch's unused rows, whose gradient is zero: their dq is 0, and dk and dv are those of the others."""
    from sageattention import sageattn_backward
    q, k, v, dout, _ = inputs(2, 4, 2, 300, 140, 64, dtype, spread=4.0)
    dout[:, :, 130:] = 0
    got = sageattn_backward(dout, q, k, v)
    assert (got[0][:, :, 130:] == 0).all()
    verify(got, q, k, v, dout, None, "HND", False)
    assert all((g == 0).all() for g in sageattn_backward(torch.zeros_like(dout), q, k, v))


def test_keys_past_32_bits_and_long_keys():
    from sageattention import sageattn_backward
    store = torch.zeros(1, 300000, 60, 128, dtype=BF16, device="cuda")
    assert store.numel() > 1 << 31
    q, k, v, dout, dlse = inputs(1, 1, 1, 40, 300000, 128, BF16, "NHD", spread=2.0)
    store[:, :, 59:], store[:, :, 3:4] = k, v
    got = sageattn_backward(dout, q, store[:, :, 59:], store[:, :, 3:4], tensor_layout="NHD", dlse=dlse)
    verify(got, q, k, v, dout, dlse, "NHD", False)
    q, k, v, dout, dlse = inputs(1, 2, 1, 1, 131073, 64, F16, spread=2.0)
    verify(sageattn_backward(dout, q, k, v, dlse=dlse), q, k, v, dout, dlse, "HND", False)
