"""The scaled 8-bit MFMAs' results, like every other's, are read only after the matrix core has
written them (CPU only): the walk of ``test_isa_mfma_waits`` over the kernel that issues them."""

from __future__ import annotations

import os
import shutil

import pytest

import test_isa_mfma_waits as isa

# Four-cycle passes: 32x32x64 runs 64 cycles on 8-bit operands, 16x16x128 runs 32.
SCALED = {"v_mfma_scale_f32_32x32x64_f8f6f4": 16, "v_mfma_scale_f32_16x16x128_f8f6f4": 8}


@pytest.mark.skipif(not shutil.which(isa.HIPCC) and not os.path.exists(isa.HIPCC), reason="hipcc not available")
def test_no_scaled_result_is_read_early(monkeypatch):
    isa.OUT.mkdir(parents=True, exist_ok=True)
    path = isa._assemble(isa.CSRC / "fm_linear_fp8.hip")
    monkeypatch.setattr(isa, "PASSES", {**isa.PASSES, **SCALED})
    found, count = [], 0
    for name, ins, labels in isa._functions(path):
        count += sum(op in SCALED for op, _ in ins)
        found += isa._early_reads(name, ins, labels)
    assert count > 100, "no scaled MFMAs found"
    assert not found, "\n".join(found[:20])
