"""`rms_norm`, `rms_norm_quant` and `rms_norm_backward` against their formulas in 64 bits.

Tolerances: a rounding to 16 bits is off by half a step, u = eps / 2 of the value; a row's sum in fp32, of 32
values a lane at most and then in pairs or wave by wave, by 64 2^-24 of itself (a root halves that), and
each further operation by 2^-24. dw is a sum of `rows` products in runs, off by the longest run's length
times 2^-24 of the sum of their sizes.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
U = {F16: 2.0 ** -11, BF16: 2.0 ** -8, F32: 2.0 ** -24}
E = 2.0 ** -24
TINY = {F16: 2.0 ** -25, BF16: 2.0 ** -134, F32: 2.0 ** -150}


def rows(shape, dtype, seed=0, size=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = size * torch.randn(shape, generator=gen, device="cuda")
    return (x * (0.25 + torch.rand(x.shape[:-1] + (1,), generator=gen, device="cuda"))).to(dtype)


def weights(n, dtype, seed=7):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (1 + 0.25 * torch.randn(n, generator=gen, device="cuda")).to(dtype)


def wanted(x, w, eps, residual):
    t = x.double() if residual is None else x.double() + residual.double()
    r = 1 / torch.sqrt(t.square().mean(-1, keepdim=True) + eps)
    return t, r, t * r * w.double()


def near(got, want, rel, dtype, floor=0.0):
    tol = want.abs() * (rel + U[dtype]) + TINY[dtype] + floor
    assert torch.isfinite(got).all()
    share = ((got.double() - want).abs() / tol).max().item()
    assert share <= 1.0, share


SIZES = [8, 16, 56, 64, 72, 128, 136, 256, 264, 512, 520, 1024, 1032, 2048, 2056, 4096, 4104, 8192, 8200,
         16384]


@pytest.mark.parametrize("n", SIZES)
@pytest.mark.parametrize("dtype,wtype", [(F16, F16), (BF16, BF16), (BF16, F32), (F16, F32)])
@pytest.mark.parametrize("residual", [False, True])
def test_norm(n, dtype, wtype, residual):
    from sageattention import rms_norm
    for count in (1, 5, 67):
        x, w = rows((count, n), dtype, n), weights(n, wtype)
        res = rows((count, n), dtype, n + 1, 3.0) if residual else None
        t, r, y = wanted(x, w, 1e-6, res)
        got = rms_norm(x, w, 1e-6, residual=res, return_rstd=True)
        near(got[0], y, 80 * E, dtype)
        near(got[-1], r[:, 0], 80 * E, F32)
        if residual:
            near(got[1], t, 2 * E, dtype)
        plain = rms_norm(x, w, 1e-6, residual=res)
        assert torch.equal(plain[0] if residual else plain, got[0])


@pytest.mark.parametrize("n", SIZES)
@pytest.mark.parametrize("dtype,int8", [(F16, True), (F16, False), (BF16, False), (BF16, True)])
def test_codes(n, dtype, int8):
    from sageattention import rms_norm_quant
    for count, residual in ((1, False), (37, True)):
        x, w = rows((count, n), dtype, n), weights(n, dtype)
        res = rows((count, n), dtype, n + 1, 3.0) if residual else None
        t, _, y = wanted(x, w, 1e-6, res)
        got = rms_norm_quant(x, w, 1e-6, residual=res, int8=int8)
        assert got[0].dtype == (torch.int8 if int8 else torch.float8_e4m3fn)
        scale = y.abs().amax(-1) / (127 if int8 else 448)
        near(got[1], scale, 90 * E, F32)
        steps, held = y / scale[:, None], got[0].double()
        # half a step of the code, which y and the scale may shift by their own errors
        half = torch.full_like(steps, 0.5) if int8 else \
            (steps.abs() * 2.0 ** -4).clamp(min=2.0 ** -10)
        assert ((held - steps).abs() <= half + 200 * E * (127 if int8 else 448)).all()
        assert (held.abs().amax(-1) == (127 if int8 else 448)).all()
        if residual:
            near(got[2], t, 2 * E, dtype)


@pytest.mark.parametrize("n", SIZES)
@pytest.mark.parametrize("dtype,wtype", [(F16, F16), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("count,dsum", [(1, False), (3, True), (131, True), (5000, False)])
def test_gradients(n, dtype, wtype, count, dsum):
    from sageattention import rms_norm_backward
    if count * n > 1 << 25:
        count = (1 << 25) // n
    x, w, dy = rows((count, n), dtype, n), weights(n, wtype), rows((count, n), dtype, n + 2, 2.0 ** -7)
    ds = rows((count, n), dtype, n + 3, 2.0 ** -7) if dsum else None
    rstd = (x.float().square().mean(-1) + 1e-6).rsqrt()
    dx, dw = rms_norm_backward(dy, x, w, rstd, dsum=ds)
    t, r, g = x.double(), rstd.double()[:, None], dy.double() * w.double()
    along = (g * t * r).mean(-1, keepdim=True)
    size = r * (g.abs() + t.abs() * r * (g * t * r).abs().mean(-1, keepdim=True))
    want = r * (g - t * r * along) + (0 if ds is None else ds.double())
    size = size + (0 if ds is None else ds.double().abs())
    tol = 80 * E * size + U[dtype] * want.abs() + TINY[dtype]
    assert ((dx.double() - want).abs() <= tol).all()
    parts = dy.double() * t * r
    want = parts.sum(0)
    tol = (count + 4) * E * parts.abs().sum(0) + U[wtype] * want.abs() + TINY[wtype]
    assert ((dw.double() - want).abs() <= tol).all()
    again = rms_norm_backward(dy, x, w, rstd, dsum=ds)
    assert torch.equal(dx, again[0]) and torch.equal(dw, again[1])
