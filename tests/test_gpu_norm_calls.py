"""How the norm is called: views of fused projections, refusals, rows that hold no numbers, graphs, streams,
autograd, sizes past 32 bits."""
import pytest
import torch

from test_gpu_norm import BF16, E, F16, F32, U, near, rows, wanted, weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_views(dtype):
    """Heads of a fused projection: rows in up to three dimensions, beside tensors that lie otherwise."""
    from sageattention import rms_norm, rms_norm_backward, rms_norm_quant
    B, N, H, D = 3, 37, 5, 64
    fused = rows((B, N, 3, H, D), dtype, 1)
    w = weights(D, dtype)
    for x in (fused[:, :, 1], fused[:, 3:9, 0], fused[..., 2, :, :].transpose(1, 2), fused[0, :, 2, 1],
              fused[:, :1, 0], fused[:, :, 0, :, :].transpose(0, 1)[4], fused[:, ::2, 1, ::2],
              rows((B, D), dtype)[:, None].expand(B, 4, D)):
        t, r, y = wanted(x, w, 1e-6, None)
        got, rstd = rms_norm(x, w, 1e-6, return_rstd=True)
        assert got.is_contiguous() and rstd.shape == x.shape[:-1]
        near(got, y, 80 * E, dtype)
        same = rms_norm(x.contiguous(), w, 1e-6)
        assert torch.equal(got, same)
        codes, scales = rms_norm_quant(x, w, 1e-6)
        again = rms_norm_quant(x.contiguous(), w, 1e-6)
        assert torch.equal(codes.view(torch.uint8), again[0].view(torch.uint8)) and torch.equal(scales, again[1])
        # the gradient's tensors each with strides of their own
        dy = torch.zeros(x.shape[:-1] + (2 * D,), dtype=dtype, device="cuda")[..., :D]
        dy.copy_(rows(x.shape, dtype, 9))
        ds = rows(x.shape, dtype, 10)
        a = rms_norm_backward(dy, x, w, rstd, dsum=ds)
        b = rms_norm_backward(dy.contiguous(), x.contiguous(), w, rstd, dsum=ds)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_residual_of_other_strides():
    from sageattention import rms_norm
    x, w = rows((4, 10, 256), BF16), weights(256, BF16)
    wide = rows((4, 20, 512), BF16, 3)
    res = wide[:, ::2, 256:]
    got, total = rms_norm(x, w, residual=res)
    want = rms_norm(x, w, residual=res.contiguous())
    assert torch.equal(got, want[0]) and torch.equal(total, want[1])


def test_no_rows():
    from sageattention import rms_norm, rms_norm_backward, rms_norm_quant
    x, w = torch.empty(0, 5, 64, dtype=BF16, device="cuda"), weights(64, F32)
    assert rms_norm(x, w).shape == x.shape
    codes, scales, total = rms_norm_quant(x, w, residual=x)
    assert codes.shape == x.shape and scales.shape == (0, 5) and total.shape == x.shape
    dx, dw = rms_norm_backward(x, x, w, torch.empty(0, 5, device="cuda"))
    assert dx.shape == x.shape and (dw == 0).all() and dw.dtype == F32


def test_zero_rows_and_one_row():
    from sageattention import rms_norm, rms_norm_quant
    w = weights(128, F16)
    assert (rms_norm(torch.zeros(3, 128, dtype=F16, device="cuda"), w) == 0).all()
    codes, scales = rms_norm_quant(torch.zeros(3, 128, dtype=F16, device="cuda"), w)
    assert (codes == 0).all() and (scales == torch.tensor(1e-12, device="cuda")).all()
    x = rows((128,), F16)
    y, rstd = rms_norm(x, w, return_rstd=True)
    assert y.shape == (128,) and rstd.shape == ()
    near(y, wanted(x, w, 1e-6, None)[2], 80 * E, F16)


@pytest.mark.parametrize("n", [64, 512, 1024, 4096, 16384])
def test_values_whose_squares_pass_fp32(n):
    from sageattention import rms_norm
    w = torch.ones(n, dtype=BF16, device="cuda")
    for size in (1e20, 1e30, 1e37):
        x = rows((5, n), BF16, n)
        x[2:4] = (x[2:4].float() * size).to(BF16)
        y, rstd = rms_norm(x, w, return_rstd=True)
        t, r, want = wanted(x, w, 1e-6, None)
        near(y, want, 100 * E, BF16)
        # 1 / 1e38 is no normal number of fp32: its step is 2^-149
        near(rstd, r[:, 0], 100 * E, F32, floor=2.0 ** -149)


@pytest.mark.parametrize("n", [64, 520, 4096])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_rows_that_hold_no_numbers(n, dtype):
    from sageattention import rms_norm, rms_norm_quant
    x, w = rows((6, n), dtype), weights(n, dtype)
    clean, clean_codes = rms_norm(x, w), rms_norm_quant(x, w)
    x[1, n // 2] = torch.nan
    x[4, 0] = torch.inf
    y = rms_norm(x, w)
    codes, scales = rms_norm_quant(x, w)
    held = codes.view(torch.uint8)
    ok = torch.tensor([0, 2, 3, 5], device="cuda")
    assert torch.equal(y[ok], clean[ok]) and torch.isnan(y[1]).all()
    assert torch.equal(held[ok], clean_codes[0].view(torch.uint8)[ok])
    assert torch.equal(scales[ok], clean_codes[1][ok])
    assert torch.isnan(scales[[1, 4]]).all() and (held[[1, 4]] == 0).all()


def test_large_eps_and_none():
    from sageattention import rms_norm
    x, w = rows((3, 256), F16), weights(256, F32)
    for eps in (0.0, 1.0, 1e4):
        near(rms_norm(x, w, eps), wanted(x, w, eps, None)[2], 80 * E, F16)


def test_refusals():
    from sageattention import rms_norm, rms_norm_backward, rms_norm_quant
    x, w = rows((4, 64), BF16), weights(64, BF16)
    rstd = torch.ones(4, device="cuda")
    for f in (rms_norm, rms_norm_quant):
        for match, args in (
                ("device", (x.cpu(), w)), ("device", (x, w.cpu())), ("device", (None, w)), ("device", (x, None)),
                ("dtype", (x.float(), w)), ("dtype", (x, w.half())), ("shape", (x, w[:56])),
                ("row", (x[:, :60], w[:60])), ("row", (x[0, 0], w)), ("shape", (x, w[None])),
                ("row", (torch.zeros(1, 16392, dtype=BF16, device="cuda"), weights(16392, BF16))),
                ("stride_last", (x.t().contiguous().t(), w)),
                ("stride_last", (x, torch.ones(128, dtype=BF16, device="cuda")[::2])),
                ("ptr_align", (rows((65 * 4 + 8,), BF16)[1:257].view(4, 64), w)),
                ("ptr_align", (x, torch.ones(72, dtype=BF16, device="cuda")[1:65])),
                ("stride_align", (rows((4, 68), BF16)[:, :64], w)),
                ("strides", (rows((2, 3, 4, 5, 6, 64), BF16)[:, ::2, ::2, ::2, ::2], w))):
            with pytest.raises(ValueError, match=match):
                f(*args)
        for match, extra in (("eps", dict(eps=-1.0)), ("eps", dict(eps=float("nan"))),
                             ("eps", dict(eps=float("inf"))), ("shape", dict(residual=x[:3])),
                             ("dtype", dict(residual=x.half())), ("device", dict(residual=x.cpu()))):
            with pytest.raises(ValueError, match=match):
                f(x, w, **extra)
    for match, args, extra in (
            ("rstd", (x, x, w, rstd[:3]), {}), ("rstd", (x, x, w, rstd.double()), {}),
            ("device", (x, x, w, rstd.cpu()), {}), ("shape", (x[:3], x, w, rstd), {}),
            ("dtype", (x.half(), x, w, rstd), {}), ("shape", (x, x, w, rstd), dict(dsum=x[:3])),
            ("device", (x.cpu(), x, w, rstd), {})):
        with pytest.raises(ValueError, match=match):
            rms_norm_backward(*args, **extra)


def test_graph():
    from sageattention import rms_norm, rms_norm_backward, rms_norm_quant
    x, res, w = rows((37, 4096), BF16), rows((37, 4096), BF16, 1), weights(4096, F32)
    dy = rows((37, 4096), BF16, 2)

    def run():
        y, total, rstd = rms_norm(x, w, residual=res, return_rstd=True)
        return (y, total, *rms_norm_quant(x, w, residual=res, int8=True),
                *rms_norm_backward(dy, total, w, rstd, dsum=y))
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for seed in (5, 6, 7):
        x.copy_(rows((37, 4096), BF16, seed))
        dy.copy_(rows((37, 4096), BF16, seed + 10))
        want = run()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_two_streams():
    from sageattention import rms_norm_backward
    sets = []
    for n, count in ((128, 9000), (2048, 700)):
        x, w = rows((count, n), F16, n), weights(n, F16)
        rstd = (x.float().square().mean(-1) + 1e-6).rsqrt()
        sets.append((rows((count, n), F16, n + 1), x, w, rstd))
    want = [rms_norm_backward(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        got = []
        for s, stream in zip(sets, streams):
            with torch.cuda.stream(stream):
                got.append(rms_norm_backward(*s))
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_autograd():
    """Gradients by autograd are the backward call's, of rows, weight and residual, whichever results were
    used; leaves do not share their gradients' memory."""
    from sageattention import rms_norm, rms_norm_backward
    x, res, w = rows((9, 256), BF16), rows((9, 256), BF16, 1), weights(256, F32)
    dy, ds = rows((9, 256), BF16, 2), rows((9, 256), BF16, 3)
    _, total, rstd = rms_norm(x, w, residual=res, return_rstd=True)
    want = rms_norm_backward(dy, total, w, rstd, dsum=ds)
    leaves = [t.clone().requires_grad_() for t in (x, w, res)]
    y, s = rms_norm(leaves[0], leaves[1], residual=leaves[2])
    torch.autograd.backward((y, s), (dy, ds))
    assert torch.equal(leaves[0].grad, want[0]) and torch.equal(leaves[2].grad, want[0])
    assert torch.equal(leaves[1].grad, want[1])
    leaves[0].grad.zero_()
    assert torch.equal(leaves[2].grad, want[0])
    # the sum alone; the norm alone, its gradient in rows that lie apart
    a, b = (t.clone().requires_grad_() for t in (x, res))
    y, s = rms_norm(a, w, residual=b)
    s.backward(ds)
    assert torch.equal(a.grad, ds) and torch.equal(b.grad, ds)
    a = x.clone().requires_grad_()
    y = rms_norm(a, w)
    wide = torch.zeros(9, 512, dtype=BF16, device="cuda")
    wide[:, :256] = dy
    y.backward(wide[:, :256])
    rstd = rms_norm(x, w, return_rstd=True)[1]
    assert torch.equal(a.grad, rms_norm_backward(dy, x, w, rstd)[0])
    with torch.no_grad():
        assert not rms_norm(a, w).requires_grad


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_gradients_against_differences(dtype):
    """The 64-bit formula's change along a direction is the gradients' product with it."""
    from sageattention import rms_norm, rms_norm_backward
    x, w, dy, along = (rows((6, 128), dtype, s) for s in (0, 1, 2, 3))
    w = weights(128, F32)
    turn = torch.randn(128, device="cuda", dtype=torch.float64)
    rstd = rms_norm(x, w, return_rstd=True)[1]
    dx, dw = rms_norm_backward(dy, x, w, rstd)

    def loss(t, v):
        r = 1 / torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-6)
        return (t * r * v * dy.double()).sum()
    step, t, v = 1e-5, x.double(), w.double()
    for got, change in ((dx, lambda h: loss(t + h * along.double(), v)), (dw, lambda h: loss(t, v + h * turn))):
        with_ = along.double() if got is dx else turn
        want = (change(step) - change(-step)) / (2 * step)
        # dx and dw are off by half a step of their type each; the difference by step^2, 1e-10
        off = (U[got.dtype] + 100 * E) * (got.double() * with_).abs().sum() + 1e-6 * want.abs() + 1e-6
        assert (((got.double() * with_).sum() - want).abs() <= off), (float(want), float(off))


def test_offsets_past_32_bits():
    from sageattention import rms_norm, rms_norm_backward
    n = 4096
    count = (1 << 31) // n + 3
    x = torch.ones(count, n, dtype=BF16, device="cuda")
    x[-3:] = rows((3, n), BF16)
    w = weights(n, BF16)
    y, rstd = rms_norm(x, w, return_rstd=True)
    near(y[-3:], wanted(x[-3:], w, 1e-6, None)[2], 80 * E, BF16)
    assert torch.equal(y[0], y[count // 2])
    dx, dw = rms_norm_backward(y, x, w, rstd)
    last = rms_norm_backward(y[-3:].contiguous(), x[-3:], w, rstd[-3:].contiguous())
    assert torch.equal(dx[-3:], last[0])
    per = y[0].double() * rstd[0].double()           # a row of ones' share of dw
    want = per * (count - 3) + (y[-3:].double() * x[-3:].double() * rstd[-3:, None].double()).sum(0)
    # sums of 1024 rows and of 512 shares in fp32
    assert ((dw.double() - want).abs() <= (U[BF16] + 1600 * E) * want.abs() + 1e-2).all()
