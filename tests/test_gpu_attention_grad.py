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
