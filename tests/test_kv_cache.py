"""The cache operators' host side (CPU, no GPU): rotary tables, refusals of the Python entry points for
tensors off the GPU, and the C ABI's argument checks (made before any launch)."""
import ctypes
import math
import os
import re

import pytest
import torch

import kv_cache_ref as ref
from test_codegen import (PKG, _assembly, _kernel_resources, early_mfma_reads, masked_mfmas,
                          undefined_converts)


# ------------------------------------------------------------------------------------- tables
def _turns(table):
    """Each frequency's angle at position 1 (mod 2 pi), and the table's size."""
    c, s = table[1].double().chunk(2)
    return torch.atan2(s, c), (c * c + s * s).sqrt()


def test_rotary_table_is_cosines_then_sines():
    from sageattention import rotary_table
    t = rotary_table(70000, 32, device="cpu")
    assert t.dtype == torch.float32 and t.shape == (70000, 32)
    for p in (0, 1, 777, 69999):
        for i in range(16):
            angle = p * 10000.0 ** (-2 * i / 32)
            # the 64-bit angle is off by an ulp of 7e4, the entry by half a step of fp32
            assert abs(float(t[p, i]) - math.cos(angle)) <= 2.0 ** -25 + 2.0 ** -36
            assert abs(float(t[p, 16 + i]) - math.sin(angle)) <= 2.0 ** -25 + 2.0 ** -36


def test_rotary_table_scalings():
    from sageattention import rotary_table
    base = torch.tensor([500.0 ** (-2 * i / 64) for i in range(32)], dtype=torch.float64)
    linear, size = _turns(rotary_table(4, 64, 500.0, scaling="linear", factor=4.0, device="cpu"))
    assert torch.allclose(linear, base / 4, rtol=1e-6) and torch.allclose(size, torch.ones(32).double())
    ntk, _ = _turns(rotary_table(4, 64, 500.0, scaling="ntk", factor=4.0, device="cpu"))
    assert math.isclose(float(ntk[0]), 1.0, rel_tol=1e-6)
    assert math.isclose(float(ntk[31]), float(base[31]) / 4, rel_tol=1e-5)
    yarn, size = _turns(rotary_table(4, 64, 500.0, scaling="yarn", factor=4.0, original_length=1000,
                                     device="cpu"))
    # frequency i turns 1000 base_i / (2 pi) times over the trained length
    turns = 1000 * base / (2 * math.pi)
    for i in range(32):
        if turns[i] >= 32:
            assert math.isclose(float(yarn[i]), float(base[i]), rel_tol=1e-6)
        assert base[i] / 4 * (1 - 1e-6) <= yarn[i] <= base[i] * (1 + 1e-6)
    assert math.isclose(float(yarn[31]), float(base[31]) / 4, rel_tol=1e-6) or turns[31] > 1
    assert torch.allclose(size, torch.full((32,), 0.1 * math.log(4.0) + 1.0).double(), rtol=1e-6)
    assert (yarn[1:] < yarn[:-1]).all()


@pytest.mark.parametrize("bad", [dict(length=0), dict(dim=8), dict(dim=24), dict(scaling="no"),
                                 dict(factor=0.5), dict(base=1.0), dict(scaling="yarn", factor=2.0)])
def test_rotary_table_refusals(bad):
    from sageattention import rotary_table
    with pytest.raises(ValueError, match="rotary_table"):
        rotary_table(**{**dict(length=8, dim=64, device="cpu"), **bad})


# ----------------------------------------------------------------------------------- refusals
def test_entry_points_refuse_tensors_off_the_gpu():
    from sageattention import KVCache, apply_rotary, rotary_table, sageattn_cached
    x = torch.zeros(1, 2, 3, 64, dtype=torch.float16)
    ints = torch.zeros(1, 3, dtype=torch.int32)
    with pytest.raises(ValueError, match="apply_rotary: device"):
        apply_rotary(x, rotary_table(4, 64, device="cpu"), ints)
    with pytest.raises(ValueError, match="sageattn_cached: device"):
        sageattn_cached(x, None, ints, ints[:, 0])
    with pytest.raises(ValueError, match="KVCache: device"):
        KVCache.allocate(1, 1, device="cpu")
    with pytest.raises(ValueError, match="apply_rotary: layout"):
        apply_rotary(x, None, ints, "BHND")


def _lib():
    from sageattention.sk1_backend import sk1_loader
    if not os.path.isfile(sk1_loader.LIB_PATH):
        pytest.skip("library not built")
    return sk1_loader.SageLib.get().lib


P = ctypes.c_void_p(16)
BAD = ctypes.c_void_p(8)


def _call(name, order, good, changes):
    args = dict(good, **changes)
    lib = _lib()
    rc = getattr(lib, name)(*[args[n] for n in order])
    return rc, lib.sage_last_error()


POOL = ["k8", "sk", "v8", "sv", "num_pages", "table", "t_sb", "max_pages"]
COMMON = dict(dtype=0, int8=1, k8=P, sk=P, v8=P, sv=P, num_pages=4, table=P, t_sb=3, max_pages=3, B=2,
              H=4, N=5, D=128, stream=None)


def _view(n):
    return [n, n + "_sb", n + "_sh", n + "_sr"]


def _strides(*names):
    return {n + s: v for n in names for s, v in (("", P), ("_sb", 2560), ("_sh", 640), ("_sr", 128))}


@pytest.mark.parametrize("change,reason", [
    (dict(dtype=2), b"dtype"), (dict(x=None), b"NULL"), (dict(x=BAD), b"ptr_align"),
    (dict(x_sb=0), b"stride_nonpos"), (dict(o_sr=132), b"stride_align"), (dict(N=0), b"seq_len"),
    (dict(D=96), b"head_dim"), (dict(rot=None), b"NULL"), (dict(rot=BAD), b"ptr_align"),
    (dict(rows=0), b"no rows"), (dict(R=0), b"R must"), (dict(R=24), b"R must"),
    (dict(R=144), b"R must"), (dict(positions=None), b"NULL"), (dict(p_sb=4), b"overlap"),
    (dict(B=2 ** 20, H=2 ** 10), b"grid"), (dict(B=2 ** 40), b"grid"),
])
def test_rotary_argument_checks(change, reason):
    order = ["dtype"] + _view("x") + _view("o") + ["B", "H", "N", "D", "rot", "rows", "R", "positions",
                                                  "p_sb", "interleaved", "inverse", "stream"]
    good = dict(COMMON, **_strides("x", "o"), rot=P, rows=9, R=64, positions=P, p_sb=5, interleaved=0,
                inverse=0)
    rc, err = _call("sage_rotary", order, good, change)
    assert rc == 1 and reason in err


@pytest.mark.parametrize("change,reason", [
    (dict(dtype=3), b"dtype"), (dict(dtype=1), b"bf16_int8"), (dict(k8=None), b"NULL"),
    (dict(sv=BAD), b"ptr_align"), (dict(num_pages=0), b"num_pages"), (dict(num_pages=2 ** 31), b"num_pages"),
    (dict(max_pages=0), b"max_pages"), (dict(max_pages=2 ** 24 + 1, t_sb=2 ** 25), b"max_pages"),
    (dict(t_sb=2), b"overlap"), (dict(D=32), b"head_dim"), (dict(B=0), b"seq_len"),
    (dict(k_sr=4), b"stride_align"), (dict(v=None), b"NULL"), (dict(start=None), b"start"),
    (dict(rot=P, positions=None), b"NULL"), (dict(rot=P, positions=P, R=8), b"R must"),
])
def test_write_argument_checks(change, reason):
    order = ["dtype", "int8"] + _view("k") + _view("v") + ["B", "H", "N", "D"] + POOL + [
        "start", "lens", "rot", "rows", "R", "positions", "p_sb", "interleaved", "stream"]
    good = dict(COMMON, **_strides("k", "v"), start=P, lens=None, rot=None, rows=4, R=64, positions=None,
                p_sb=5, interleaved=0)
    rc, err = _call("sage_cache_write", order, good, change)
    assert rc == 1 and reason in err


@pytest.mark.parametrize("change,reason", [
    (dict(dtype=-1), b"dtype"), (dict(table=None), b"NULL"), (dict(lens=None), b"lens"),
    (dict(k=None), b"NULL"), (dict(v_sh=-640), b"stride_nonpos"), (dict(D=256), b"head_dim"),
])
def test_read_argument_checks(change, reason):
    order = ["dtype", "int8"] + POOL + ["start", "lens"] + _view("k") + _view("v") + [
        "B", "H", "N", "D", "stream"]
    rc, err = _call("sage_cache_read", order, dict(COMMON, **_strides("k", "v"), start=None, lens=P), change)
    assert rc == 1 and reason in err


@pytest.mark.parametrize("change,reason", [
    (dict(dtype=1), b"bf16_int8"), (dict(H_kv=3), b"heads"), (dict(H_kv=0), b"heads"),
    (dict(T=0), b"seq_len"), (dict(D=80), b"head_dim"), (dict(kv_lens=None), b"kv_lens"),
    (dict(mask=P, m_sr=4), b"tree_mask"), (dict(mask=P, m_sr=5, m_sb=3), b"tree_mask"),
    (dict(scale=0.0), b"sm_scale"), (dict(scale=float("nan")), b"sm_scale"),
    (dict(lse=ctypes.c_void_p(18)), b"ptr_align"), (dict(ws=None), b"workspace"),
    (dict(ws=BAD), b"workspace"), (dict(ws_bytes=4), b"workspace"), (dict(T=2 ** 26), b"grid"),
    (dict(max_pages=2 ** 25, t_sb=2 ** 25), b"max_pages"), (dict(q_sr=2), b"stride_align"),
])
def test_attention_argument_checks(change, reason):
    order = ["dtype", "int8"] + _view("q") + POOL + ["kv_lens", "q_lens", "mask", "m_sb", "m_sr"] + \
        _view("o") + ["B", "H", "T", "H_kv", "D", "scale", "lse", "ws", "ws_bytes", "stream"]
    good = dict(COMMON, **_strides("q", "o"), kv_lens=P, q_lens=None, mask=None, m_sb=0, m_sr=0, T=5,
                H_kv=2, scale=0.1, lse=None, ws=P, ws_bytes=2 ** 40, max_pages=999, t_sb=999)
    rc, err = _call("sage_cache_attn", order, good, change)
    assert rc == 1 and reason in err


def test_workspace_sizes():
    lib = _lib()
    assert lib.sage_cache_attn_workspace_bytes(64, 32, 8, 64, 1, 128) == 0    # nothing to split
    assert lib.sage_cache_attn_workspace_bytes(1, 32, 8, 1, 2000, 128) > 0
    assert lib.sage_cache_attn_workspace_bytes(1, 32, 5, 1, 2000, 128) == -1
    assert lib.sage_cache_attn_workspace_bytes(1, 32, 8, 1, 0, 128) == -1


@pytest.mark.parametrize("B,H,H_kv,T,max_pages,D,served", [
    # many prompts' parts, a block for each plane and 128 rows: the rows' limit, D/8 threads each
    (64, 32, 8, 8192, 128, 128, True), (512, 32, 8, 8192, 128, 128, True),
    (1024, 32, 8, 8192, 128, 128, False), (1024, 32, 8, 8192, 128, 64, True),
    # decoding of as many planes as a launch has blocks of 256 threads
    (2 ** 21 - 1, 8, 8, 1, 1, 64, True), (2 ** 21, 8, 8, 1, 1, 64, False),
    # one K/V head: eight blocks for each 128 rows
    (1, 2 ** 20, 1, 255, 1, 64, True), (1, 2 ** 20, 1, 256, 1, 64, False),
])
def test_sizes_are_refused_by_the_launch_that_they_need(B, H, H_kv, T, max_pages, D, served):
    lib = _lib()
    n = lib.sage_cache_attn_workspace_bytes(B, H, H_kv, T, max_pages, D)
    assert n == 0 if served else n == -1 and b"grid" in lib.sage_last_error()


# ------------------------------------------------------------------------------------ oracles
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", [33, 64, 66, 96, 100, 128, 144, 200, 400])
def test_runs_fill_the_card_once(T, D):
    # two blocks a CU, 32 CUs to each of the 8 XCDs that runs are dealt to with all their row blocks
    B, H, H_kv, pages = 8, 32, 8, 128
    tiles = -(-T * (H // H_kv) // 16)
    blocks = -(-tiles // 8)
    rows = 16 * -(-tiles // blocks)
    floats = _lib().sage_cache_attn_workspace_bytes(B, H, H_kv, T, pages, D) // 4
    parts = (floats - 2 * B * H_kv) // (D + 2)
    runs = parts // (blocks * 2 * rows)
    assert floats == runs * blocks * 2 * rows * (D + 2) + 2 * B * H_kv
    assert 0.8 * 64 < -(-runs // 8) * blocks <= 64


def test_the_reference_rotations_agree():
    gen = torch.Generator().manual_seed(0)
    from sageattention import rotary_table
    table, x = rotary_table(50, 32, device="cpu"), torch.randn(2, 3, 7, 64, generator=gen)
    pos = torch.randint(0, 50, (2, 7), generator=gen)
    for interleaved in (False, True):
        a = ref.rotate(x, table, pos, interleaved)
        assert torch.allclose(a, ref.rotate_fp32(x, table, pos, interleaved).double(), atol=1e-6)
        assert torch.allclose(ref.rotate(a, table, pos, interleaved, True), x.double(), atol=1e-6)


# ---------------------------------------------------------------------------- generated code
# The rules of the main loops' code hold for the cache's kernels: every MFMA runs with the whole wave
# active, no result is read before its MFMA is done, nothing spills, no flat accesses, converts into a
# half-word keep a defined other half.
def test_attention_mfmas_run_with_the_whole_wave():
    asm = _assembly(os.path.join(PKG, "csrc", "cache_attn.hip"))
    assert "v_mfma_f32_16x16x32_f16" in asm and "v_mfma_f32_16x16x32_bf16" in asm
    assert masked_mfmas(asm) == []


def test_attention_products_are_read_after_they_are_done():
    # 16 cycles a 16x16x32 MFMA of 16-bit operands, counted as for the main loops' MFMAs
    asm = _assembly(os.path.join(PKG, "csrc", "cache_attn.hip"))
    bad = early_mfma_reads(asm, min_other=16)
    assert not bad, bad[:4]


@pytest.mark.parametrize("source", ["cache_attn.hip", "kv_cache.hip"])
def test_cache_kernels_do_not_spill(source):
    res = _kernel_resources(_assembly(os.path.join(PKG, "csrc", source)))
    assert res and [r for r in res if r[2] or r[3]] == []


@pytest.mark.parametrize("source", ["cache_attn.hip", "kv_cache.hip"])
def test_cache_kernels_have_no_flat_accesses(source):
    asm = _assembly(os.path.join(PKG, "csrc", source))
    assert "global_load" in asm and re.findall(r"^\s*flat_\w+", asm, re.M) == []
    assert re.findall(r"^\s*v_pk_(?:add|mul|fma)_f32", asm, re.M) == []


def test_cache_codes_are_converted_from_defined_words():
    ir = _assembly(os.path.join(PKG, "csrc", "kv_cache.hip"), ("-emit-llvm",))
    assert "cvt.pk.fp8.f32" in ir and undefined_converts(ir) == []
