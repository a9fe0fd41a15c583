"""The root-mean-square norm where its squares vanish in 32 bits, and what autograd has to refuse or take."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


@pytest.mark.parametrize("n", [8, 64, 200, 1000, 2048, 4096, 16384])
@pytest.mark.parametrize("size", [1e-37, 1e-30, 1e-23, 1e-22, 1e-20, 1e-14, 1e-13, 1.0, 1e18, 1e25])
@pytest.mark.parametrize("eps", [0.0, 1e-40, 1e-30, 1e-6])
def test_rows_of_every_size(n, size, eps):
    """bf16 rows whose squares lie under fp32's normal numbers or over all of them, with an eps as small or none: the norm,
    its root, codes and gradients are the definition's."""
    from sageattention import rms_norm, rms_norm_backward, rms_norm_quant
    gen = torch.Generator(device="cuda").manual_seed(n)
    x = (size * (1 + torch.rand(3, n, generator=gen, device="cuda")) *
         (1 - 2 * (torch.rand(3, n, generator=gen, device="cuda") < 0.5).float())).to(BF16)
    r = (x * 0.5).flip(0).contiguous()
    w = 1 + 0.25 * torch.rand(n, generator=gen, device="cuda")
    for residual in (None, r):
        t = x.double() if residual is None else x.double() + residual.double()
        rstd = (t.square().mean(-1) + float(torch.tensor(eps))).rsqrt()
        want = t * rstd[..., None] * w.double()
        got = rms_norm(x, w, eps, residual=residual, return_rstd=True)
        # the sum of n squares, the mean, the root and the two products in 32 bits; t itself once rounded; where the
        # squares are scaled, those (of values a quarter of the least one at the least) are normal numbers
        u = (n / 2 + 12) * 2.0 ** -24
        assert ((got[-1].double() - rstd).abs() <= u * rstd).all()
        assert ((got[0].double() - want).abs() <= (u + 2.0 ** -8) * want.abs() + 2.0 ** -133).all()
        if size * 2.0 ** 110 > 1:
            codes = rms_norm_quant(x, w, eps, residual=residual, int8=True)
            scale = (want.abs().amax(-1) / 127).clamp(min=1e-12)
            assert ((codes[1].double() - scale).abs() <= 2 * u * scale).all()
            # within half a step, and what the quotient is off by
            off = (codes[0].double() * scale[..., None] - want).abs()
            assert (off <= scale[..., None] * (0.5 + 254 * u)).all()
    if 1e-30 <= size <= 1e18:
        dy = (torch.randn(3, n, generator=gen, device="cuda") * size).to(BF16)
        _, rstd = rms_norm(x, w, eps, return_rstd=True)
        dx, _ = rms_norm_backward(dy, x, w, rstd)
        g, xhat = dy.double() * w.double(), x.double() * rstd.double()[..., None]
        want = rstd.double()[..., None] * (g - xhat * (g * xhat).mean(-1, keepdim=True))
        tol = rstd.double()[..., None] * (g.abs() + xhat.abs() * (g * xhat).abs().mean(-1, keepdim=True)) * (n + 12) * 2.0 ** -24
        assert ((dx.double() - want).abs() <= 2.0 ** -8 * want.abs() + tol + 2.0 ** -126).all()


def test_a_row_of_zeros():
    """0 / sqrt(eps) is 0; with eps 0 it is 0 / 0."""
    from sageattention import rms_norm
    x, w = torch.zeros(2, 64, dtype=BF16, device="cuda"), torch.ones(64, dtype=BF16, device="cuda")
    assert (rms_norm(x, w) == 0).all() and (rms_norm(x, w, 1e-38) == 0).all() and torch.isnan(rms_norm(x, w, 0.0)).all()


def test_forward_mode_tangents_are_refused():
    """A tangent is not dropped without a word: the call raises, with gradients enabled or not; other tensors pass."""
    import torch.autograd.forward_ad as forward_ad
    from sageattention import rms_norm, sageattn_train
    x, w = torch.randn(3, 64, device="cuda").half(), torch.ones(64, device="cuda").half()
    want = rms_norm(x, w)
    q = torch.randn(1, 2, 40, 64, device="cuda").half()
    with forward_ad.dual_level():
        dual = [forward_ad.make_dual(t, torch.ones_like(t)) for t in (x, w, q)]
        for enabled in (True, False):
            with torch.set_grad_enabled(enabled):
                for call in (lambda: rms_norm(dual[0], w), lambda: rms_norm(x, dual[1]),
                             lambda: rms_norm(x, w, residual=dual[0]), lambda: sageattn_train(dual[2], q, q)):
                    with pytest.raises(NotImplementedError):
                        call()
                assert torch.equal(rms_norm(x, w), want)
    assert torch.equal(rms_norm(x, w), want)


def test_gradients_that_begin_off_16_bytes():
    """Results joined behind an odd number of values, as a flat buffer of parameters and activations: the gradients come
    back as contiguous views 2 bytes off, and are taken."""
    from sageattention import rms_norm, sageattn_train
    x, w = torch.randn(5, 64, device="cuda").half().requires_grad_(), torch.ones(64, device="cuda").half().requires_grad_()
    q = torch.randn(1, 2, 40, 64, device="cuda").half().requires_grad_()
    odd = torch.zeros(1, device="cuda").half()
    for make, leaves in ((lambda: rms_norm(x, w), (x, w)), (lambda: rms_norm(x, w, residual=x), (x, w)),
                         (lambda: sageattn_train(q, q, q), (q,)),
                         (lambda: sageattn_train(q, q, q, return_lse=True), (q,))):
        results = make()
        results = results if isinstance(results, tuple) else (results,)
        want = torch.autograd.grad(results, leaves, [t.detach() for t in results], retain_graph=True)
        flat = [torch.cat([odd.to(t.dtype), t.flatten()]) for t in results]
        got = torch.autograd.grad(flat, leaves, [torch.cat([odd.to(t.dtype), t.detach().flatten()]) for t in results])
        assert all(torch.equal(a, b) for a, b in zip(got, want))
