"""The training operators together, as a transformer's block uses them, and a decoding step with the norm."""
import pytest
import torch

from grad_ref import U, check, forward, gradients, mm

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def rand(*shape, dtype=F16, seed=0, size=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (size * torch.randn(shape, generator=gen, device="cuda")).to(dtype)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("layout,H_kv,causal", [("HND", 4, True), ("NHD", 2, False)])
def test_attention_by_autograd(dtype, layout, H_kv, causal):
    """sageattn_train's results are sageattn's, its gradients the formula's on them."""
    from sageattention import sageattn, sageattn_train
    B, H, N, D = 2, 4, 300, 64

    def shape(h):
        return (B, h, N, D) if layout == "HND" else (B, N, h, D)
    q, k, v = (rand(*shape(h), dtype=dtype, seed=s).requires_grad_() for s, h in enumerate((H, H_kv, H_kv)))
    out, lse = sageattn_train(q, k, v, layout, causal, return_lse=True)
    with torch.no_grad():
        want = sageattn(q, k, v, layout, causal, return_lse=True)
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    dout, dlse = rand(*shape(H), dtype=dtype, seed=5, size=2.0 ** -7), \
        2.0 ** -7 * torch.randn(B, H, N, device="cuda")
    hnd = (lambda t: t) if layout == "HND" else (lambda t: t.transpose(1, 2))
    for grads in ((dout, dlse), (dout, None), (None, dlse)):
        got = torch.autograd.grad([r for r, g in zip((out, lse), grads) if g is not None], (q, k, v),
                                  [g for g in grads if g is not None], retain_graph=True)
        g = torch.zeros_like(dout) if grads[0] is None else grads[0]
        check([hnd(t) for t in got], gradients(*(hnd(t.detach()) for t in (g, q, k, v, out)), lse.detach(), grads[1],
                                               causal, D ** -0.5))
    # an expanded gradient, of a part of the inputs
    dq, = torch.autograd.grad(out.float().sum(), (q,), retain_graph=True)
    assert dq.shape == q.shape and torch.isfinite(dq).all()
    with torch.no_grad():
        assert not sageattn_train(q, k, v, layout, causal).requires_grad
    with pytest.raises(RuntimeError):
        first, = torch.autograd.grad(out.float().sum(), (q,), create_graph=True)
        torch.autograd.grad(first.float().sum(), (q,))


@pytest.mark.parametrize("dtype,causal", [(F16, True), (BF16, False)])
def test_gradients_against_differences(dtype, causal):
    """The 64-bit loss's change along a direction is the gradients' product with it."""
    from sageattention import sageattn_backward
    B, H, N, D = 1, 2, 130, 64
    q, k, v, dout = (rand(B, H, N, D, dtype=dtype, seed=s) for s in range(4))
    sm = D ** -0.5
    o, lse = forward(q, k, v, causal, sm)
    out = o.to(dtype)
    got = sageattn_backward(dout, q, k, v, out, lse.float(), is_causal=causal)
    want = gradients(dout, q, k, v, out, lse.float(), None, causal, sm)
    # the output's rounding, u of it, moves dS = P (dout.v - dout.out): sm P |dout||out| u |k_j|, and for dk |q_i|
    s = mm(q.double() * sm, k.double())
    if causal:
        s = s.masked_fill(~torch.ones(N, N, dtype=torch.bool, device="cuda").tril(), -torch.inf)
    p = torch.exp(s - lse[..., None])
    moved = sm * U[dtype] * p * (dout.double() * o).abs().sum(-1, keepdim=True)
    moved = {"dq": moved @ k.double().abs(), "dk": moved.transpose(2, 3).contiguous() @ q.double().abs(), "dv": 0.0}
    step = 1e-4
    for i, (name, x) in enumerate((("dq", q), ("dk", k), ("dv", v))):
        along = torch.randn(x.shape, dtype=torch.float64, device="cuda")

        def loss(h):
            args = [q.double(), k.double(), v.double()]
            args[i] = args[i] + h * along
            return (forward(*args, causal, sm)[0] * dout.double()).sum()
        change = (loss(step) - loss(-step)) / (2 * step)
        tol = ((want[name][1] + moved[name]) * along.abs()).sum()
        assert ((got[i].double() * along).sum() - change).abs() <= tol + 1e-6 * change.abs(), name


class _Exact(torch.autograd.Function):
    """Attention with given results, its gradients by the definition in 64 bits."""
    @staticmethod
    def forward(ctx, q, k, v, out, lse):
        ctx.save_for_backward(q, k, v, out, lse)
        return out.double()

    @staticmethod
    def backward(ctx, g):
        q, k, v, out, lse = ctx.saved_tensors
        got = gradients(g, q, k, v, out, lse, None, True, q.shape[-1] ** -0.5, dtype=F16)
        return got["dq"][0], got["dk"][0], got["dv"][0], None, None


def test_block_of_a_transformer():
    """norm with the residual -> projection -> norm of heads -> attention -> projection -> norm: the gradients of
    all parameters and of the input, against the same block in 64 bits around the same attention results."""
    from sageattention import rms_norm, sageattn_train
    B, N, H, H_kv, D = 2, 257, 4, 2, 64
    n, heads = H * D, H + 2 * H_kv
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

    def norm16(t, w, residual):
        return rms_norm(t, w, 1e-6, residual=residual)

    def attend16(q, k, v):
        out, lse = sageattn_train(q, k, v, "NHD", True, return_lse=True)
        seen["out"], seen["lse"] = out.detach(), lse.detach()
        return out

    def norm64(t, w, residual):
        t = t if residual is None else t + residual
        y = t / torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-6) * w
        return y if residual is None else (y, t)

    def attend64(q, k, v):
        return _Exact.apply(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2),
                            seen["out"].transpose(1, 2), seen["lse"]).transpose(1, 2)
    leaves = {name: t.clone().requires_grad_() for name, t in dict(params, x=x, hidden=hidden).items()}
    block(leaves, leaves["x"], leaves["hidden"], norm16, attend16).backward(grad)
    exact = {name: t.double().requires_grad_() for name, t in dict(params, x=x, hidden=hidden).items()}
    block(exact, exact["x"], exact["hidden"], norm64, attend64).backward(grad.double())
    for name, t in leaves.items():
        want = exact[name].grad
        rel = ((t.grad.double() - want).norm() / want.norm()).item()
        # forward and backward pass through about 20 roundings of 2^-11 at most each, and the attention's
        # gradients see scores that the roundings of q and k, at 2^-11 of |score| = 8 or less, have moved
        assert rel <= 30 * 2.0 ** -11, (name, rel)


def test_step_in_a_graph():
    """A forward pass and its gradients by torch.autograd.grad, captured and replayed on other inputs."""
    from sageattention import rms_norm, sageattn_train
    x, w = rand(2, 4, 200, 64).requires_grad_(), rand(64, seed=1).requires_grad_()
    g = rand(2, 4, 200, 64, seed=2, size=2.0 ** -7)

    def step():
        y = rms_norm(x, w)
        return torch.autograd.grad(sageattn_train(y, y, x, is_causal=True), (x, w), g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (10, 11, 12):
        with torch.no_grad():
            x.copy_(rand(2, 4, 200, 64, seed=seed))
            g.copy_(rand(2, 4, 200, 64, seed=seed + 5, size=2.0 ** -7))
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_decoding_step():
    """One token's step with the norm ahead of it and of the heads, eager and captured: the same bits; the norm of
    single tokens is that of the prompt's rows."""
    from sageattention import KVCache, apply_rotary, rms_norm, rms_norm_quant, rotary_table, sageattn_cached
    B, H, H_kv, D, n = 3, 4, 2, 64, 256
    table = rotary_table(512, D)
    cache = KVCache.allocate(num_pages=12, num_heads=H_kv, head_dim=D, dtype=F16)
    pages = torch.arange(12, dtype=torch.int32, device="cuda").view(B, 4)
    lens = torch.tensor([5, 64, 130], dtype=torch.int32, device="cuda")
    prompt = rand(B, H_kv, 130, D, seed=1)
    cache.write(prompt, prompt, pages, torch.zeros_like(lens), lens=lens)
    w, wh, wqkv = rand(n, seed=2) * 0.1 + 1, rand(D, seed=3) * 0.1 + 1, rand((H + 2 * H_kv) * D, n, seed=4, size=n ** -0.5)
    x, hidden = rand(B, 1, n, seed=5), rand(B, 1, n, seed=6)

    def step():
        y, total = rms_norm(x, w, residual=hidden)
        qkv = (y @ wqkv.t()).unflatten(-1, (-1, D))
        q, k, v = qkv[:, :, :H], qkv[:, :, H:H + H_kv], qkv[:, :, H + H_kv:]
        q = apply_rotary(rms_norm(q, wh), table, lens[:, None], tensor_layout="NHD")
        cache.write(rms_norm(k, wh), v, pages, lens, tensor_layout="NHD", table=table, positions=lens[:, None])
        o = sageattn_cached(q, cache, pages, lens + 1, tensor_layout="NHD")
        return (o, total) + rms_norm_quant(o.reshape(B, 1, n), w, residual=total)
    eager = step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, eager):
            assert torch.equal(a, b)
    many = rms_norm(x.expand(B, 700, n).contiguous(), w, residual=hidden.expand(B, 700, n))
    one = rms_norm(x, w, residual=hidden)
    # another cut of a row's sum: both within the norm's tolerance of each other
    assert (many[0][:, 77].double() - one[0][:, 0].double()).abs().max() <= 2 * U[F16] * one[0].double().abs().max()
