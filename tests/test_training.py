"""The training operators' host side (CPU, no GPU): refusals for tensors off the GPU, and the C ABI's
argument checks, made before any launch."""
import ctypes

import pytest
import torch


def test_entry_points_refuse_cpu_tensors():
    import sageattention as sage
    q, lse = torch.zeros(1, 2, 5, 64, dtype=torch.float16), torch.zeros(1, 2, 5)
    with pytest.raises(ValueError, match="sageattn_backward: device"):
        sage.sageattn_backward(q, q, q, q, q, lse)
    with pytest.raises(ValueError, match="layout"):
        sage.sageattn_backward(q, q, q, q, q, lse, tensor_layout="NDH")
    with pytest.raises(ValueError, match="device"):
        sage.sageattn_train(q.requires_grad_(), q, q)
    with pytest.raises(ValueError, match="sageattn_train: sm_scale"):
        sage.sageattn_train(q, q, q, sm_scale=0.0)
    with pytest.raises(NotImplementedError, match="attn_mask"):
        sage.sageattn_train(q, q, q, attn_mask=lse)
    x, w = torch.zeros(3, 64, dtype=torch.float16), torch.ones(64, dtype=torch.float16)
    for f in (sage.rms_norm, sage.rms_norm_quant):
        with pytest.raises(ValueError, match="%s: device" % f.__name__):
            f(x, w)
    with pytest.raises(ValueError, match="rms_norm: device"):
        sage.rms_norm(x.requires_grad_(), w)
    with pytest.raises(ValueError, match="rms_norm_backward: device"):
        sage.rms_norm_backward(x, x, w, torch.ones(3))


@pytest.fixture(scope="module")
def lib():
    from sageattention.sk1_backend.sk1_loader import SageLib
    return SageLib.get().lib


def _refused(lib, rc, text):
    assert rc == 1 and text in lib.sage_last_error(), (rc, lib.sage_last_error())


def test_backward_checks(lib):
    p = ctypes.c_void_p(256)

    def call(dtype=1, causal=0, B=1, H=4, N=100, H_kv=2, N_kv=80, D=64, scale=0.1, q=(p, 8192, 8192, 64), lse=p,
             work=p, size=1 << 30, dk=(p, 8192, 8192, 64), dlse=None):
        view = (p, 8192, 8192, 64)
        return lib.sage_attn_bwd(dtype, causal, *q, *view, *view, *view, *view, lse, dlse, *view, *dk, *view, B,
                                 H, N, H_kv, N_kv, D, scale, work, size, None)
    _refused(lib, call(dtype=2), b"dtype")
    _refused(lib, call(D=96), b"head_dim")
    _refused(lib, call(N=0), b"n_lt_1")
    _refused(lib, call(N_kv=0), b"n_lt_1")
    _refused(lib, call(H_kv=3), b"heads")
    _refused(lib, call(H_kv=0), b"heads")
    _refused(lib, call(causal=1), b"seq_len")
    _refused(lib, call(q=(None, 8192, 8192, 64)), b"q is NULL")
    _refused(lib, call(q=(ctypes.c_void_p(8), 8192, 8192, 64)), b"ptr_align")
    _refused(lib, call(q=(p, 8192, 8192, 60)), b"stride_align")
    _refused(lib, call(dk=(p, 8192, 0, 64)), b"dk: stride_nonpos")
    _refused(lib, call(dk=(p, 8192, 8192, 1 << 24)), b"dk: stride_int32")
    _refused(lib, call(lse=None), b"lse is NULL")
    _refused(lib, call(lse=ctypes.c_void_p(2)), b"4-byte")
    _refused(lib, call(dlse=ctypes.c_void_p(2)), b"4-byte")
    for scale in (0.0, -1.0, float("nan"), float("inf"), 1e-31, 1e31):
        _refused(lib, call(scale=scale), b"sm_scale")
    large = dict(N=1000, N_kv=800)
    _refused(lib, call(work=None, **large), b"workspace")
    _refused(lib, call(work=ctypes.c_void_p(64), **large), b"workspace")
    need = lib.sage_attn_bwd_workspace_bytes(1, 0, 1, 4, 1000, 2, 800, 64)
    assert need >= 2 * 4 * 1024 * 4
    _refused(lib, call(size=need - 1, **large), b"need %d bytes" % need)
    assert lib.sage_attn_bwd_workspace_bytes(0, 0, 1, 4, 100, 2, 80, 64) == 0      # small calls need none
    _refused(lib, call(B=1 << 14, H=1 << 10), b"grid")


def test_backward_workspace(lib):
    size = lib.sage_attn_bwd_workspace_bytes
    # the rows' two constants, padded to tiles; fp16's largest values come on top
    assert size(1, 1, 1, 32, 16384, 8, 16384, 128) == 2 * 32 * 16384 * 4
    assert size(0, 1, 1, 32, 16384, 8, 16384, 128) > 2 * 32 * 16384 * 4
    # parts of long tiles: no more than the resident blocks and their tiles hold
    for dims in ((1, 1, 16384, 1, 16384, 128), (1, 6, 11000, 1, 11000, 128), (8, 8, 16000, 8, 100, 64)):
        B, H, N, H_kv, N_kv, D = dims
        for causal in (0, 1) if N == N_kv else (0,):
            least = 2 * B * H * -(-N // 64) * 64 * 4
            assert 0 < size(1, causal, *dims) - least < 2048 * 128 * D * 4 * 3
    assert size(1, 0, 1, 3, 10, 2, 10, 64) == -1


def test_norm_checks(lib):
    p = ctypes.c_void_p(256)

    def call(dtype=1, out=0, x=(p, 0, 0, 64), res=(None, 0, 0, 0), w=p, dims=(1, 1, 5), n=64, eps=1e-6, y=p, scales=None,
             total=None, rstd=None):
        return lib.sage_rms_norm(dtype, 0, out, *x, *res, w, *dims, n, eps, y, scales, total, rstd, None)
    _refused(lib, call(dtype=3), b"dtype")
    _refused(lib, call(out=3), b"out")
    for n in (0, 4, 60, 16392):
        _refused(lib, call(n=n), b"row")
    for dims in ((0, 1, 5), (1, 1, 0), (1, 1, 1 << 31), (1 << 20, 1 << 20, 1)):
        _refused(lib, call(dims=dims), b"rows")
    _refused(lib, call(x=(None, 0, 0, 64)), b"x is NULL")
    _refused(lib, call(x=(ctypes.c_void_p(8), 0, 0, 64)), b"ptr_align")
    _refused(lib, call(x=(p, 0, 4, 64)), b"stride_align")
    _refused(lib, call(res=(ctypes.c_void_p(8), 0, 0, 64)), b"residual: ptr_align")
    _refused(lib, call(w=None), b"NULL")
    _refused(lib, call(y=None), b"NULL")
    _refused(lib, call(out=1), b"NULL")
    _refused(lib, call(y=ctypes.c_void_p(8)), b"ptr_align")
    _refused(lib, call(total=ctypes.c_void_p(8)), b"ptr_align")
    _refused(lib, call(rstd=ctypes.c_void_p(2)), b"ptr_align")
    for eps in (-1.0, float("nan"), float("inf")):
        _refused(lib, call(eps=eps), b"eps")

    def back(dy=(p, 0, 0, 64), x=(p, 0, 0, 64), ds=(None, 0, 0, 0), w=p, rstd=p, dims=(1, 1, 5), n=64, dx=p, dw=p, work=p,
             size=1 << 20):
        return lib.sage_rms_norm_bwd(1, 0, *dy, *x, *ds, w, rstd, *dims, n, dx, dw, work, size, None)
    _refused(lib, back(n=12), b"row")
    _refused(lib, back(dims=(1, 0, 5)), b"rows")
    _refused(lib, back(dy=(None, 0, 0, 64)), b"dy is NULL")
    _refused(lib, back(ds=(p, 0, 0, 63)), b"dsum: stride_align")
    for name in ("w", "rstd", "dx", "dw"):
        _refused(lib, back(**{name: None}), b"NULL")
    _refused(lib, back(dx=ctypes.c_void_p(8)), b"ptr_align")
    _refused(lib, back(work=None), b"workspace")
    need = lib.sage_rms_norm_bwd_workspace_bytes(5, 64)
    assert need == 64 * 4          # five rows: one block's share
    _refused(lib, back(size=need - 1), b"workspace")
    assert lib.sage_rms_norm_bwd_workspace_bytes(16384, 4096) == 512 * 4096 * 4
    assert lib.sage_rms_norm_bwd_workspace_bytes(5, 12) == -1
