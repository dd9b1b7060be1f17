"""No instruction reads a matrix instruction's result too soon in the attention kernels whose
maxima are inline assembly, before which the compiler leaves no wait states."""
import os
import subprocess

import pytest


@pytest.mark.parametrize("source", ["attn_mfma.hip", "attn_dense.hip"])
def test_no_matrix_result_is_read_too_soon(source, tmp_path, monkeypatch):
    import asm_hazards
    from vecattention_amd import build
    # Passes + 3 for 16-bit operands, of which 32x32x16 takes 8.
    monkeypatch.setattr(asm_hazards, "NEED", {**asm_hazards.NEED, "v_mfma_f32_32x32x16_bf16": 11,
                                              "v_mfma_f32_32x32x16_f16": 11})
    out = tmp_path / "kernels.s"
    subprocess.run([build.hipcc(), *build.FLAGS, "--cuda-device-only", "-S",
                    os.path.join(build.CSRC, source), "-o", str(out)], check=True,
                   capture_output=True)
    count, early = asm_hazards.early_reads(out.read_text())
    assert count > 300 and early == []
