"""Code-generation invariants of the training kernels, by the checks of `test_codegen.py`: matrix instructions
with the whole wave active, results read after they are there, no spilled registers."""
import os

import pytest

import test_codegen as codegen

CSRC = os.path.join(codegen.PKG, "csrc")
BWD, NORM = os.path.join(CSRC, "attn_bwd.hip"), os.path.join(CSRC, "norm.hip")


def test_matrix_instructions_run_with_the_whole_wave():
    codegen.test_main_loop_mfmas_run_with_the_whole_wave(BWD)


def test_matrix_results_are_read_after_they_are_there():
    # the 16-bit 32x32x16 product takes 8 passes, and its result is there 12 wait states on: no read is closer
    asm = codegen._assembly(BWD)
    assert "v_mfma_f32_32x32x16" in asm and "32x32x64" not in asm
    assert not codegen.early_mfma_reads(asm, min_other=12)
    # (the check sees the reads: some lie there)
    assert codegen.early_mfma_reads(asm, min_other=13)


@pytest.mark.parametrize("source", [BWD, NORM])
def test_no_spilled_registers(source):
    codegen.test_no_kernel_spills_registers(source)


def test_no_flat_accesses():
    for source in (BWD, NORM):
        codegen.test_no_flat_accesses(source)
