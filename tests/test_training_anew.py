"""A backward call without output and logsumexp: the C entry's checks and workspace, made on the host."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from sageattention.sk1_backend.sk1_loader import SageLib
    return SageLib.get().lib


def test_checks(lib):
    p, none = ctypes.c_void_p(256), ctypes.c_void_p(None)
    view = (p, 8192, 8192, 64)

    def call(o=(none, 0, 0, 0), lse=none, work=p, size=1 << 30):
        return lib.sage_attn_bwd(1, 0, *view, *view, *view, *o, *view, lse, none, *view, *view, *view, 1, 4, 100, 2, 80, 64,
                                 0.1, work, size, None)
    # one of the two alone
    assert call(lse=p) == 1 and b"o is NULL" in lib.sage_last_error()
    assert call(o=view) == 1 and b"lse is NULL" in lib.sage_last_error()
    need = lib.sage_attn_bwd_anew_workspace_bytes(1, 0, 1, 4, 100, 2, 80, 64)
    assert call(size=need - 1) == 1 and b"need %d bytes" % need in lib.sage_last_error()
    assert call(work=none) == 1 and b"workspace" in lib.sage_last_error()


def test_workspace(lib):
    given, anew = lib.sage_attn_bwd_workspace_bytes, lib.sage_attn_bwd_anew_workspace_bytes
    # small calls that need none with a logsumexp: the rows' constants, and three sums for each of a block's 128
    assert given(1, 0, 1, 4, 100, 2, 80, 64) == 0
    assert anew(1, 0, 1, 4, 100, 2, 80, 64) == 2 * 4 * 128 * 4 + 4 * 2 * 3 * 128 * 4
    # whole tiles: 32 heads of 128 blocks
    assert anew(1, 1, 1, 32, 16384, 8, 16384, 128) - given(1, 1, 1, 32, 16384, 8, 16384, 128) == 32 * 128 * 3 * 128 * 4
    assert anew(1, 0, 1, 3, 10, 2, 10, 64) == -1
    assert anew(1, 1, 1, 2, 10, 2, 11, 64) == -1


def test_entry_point_refuses_cpu_tensors():
    import sageattention as sage
    q, lse = torch.zeros(1, 2, 5, 64, dtype=torch.float16), torch.zeros(1, 2, 5)
    with pytest.raises(ValueError, match="out and lse"):
        sage.sageattn_backward(q, q, q, q, lse=lse)
    with pytest.raises(ValueError, match="sageattn_backward: device"):
        sage.sageattn_backward(q, q, q, q)
