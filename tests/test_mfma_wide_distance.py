"""The same check of the built code as test_mfma_distance.py's for the 32x32x16
forms, whose eight passes take 12 wait states instead of the 16x16x32 forms' 8."""
import os

import pytest

import test_mfma_distance as base

WIDE = {"v_mfma_f32_32x32x16_%s" % t: 12 for t in ("f16", "bf16")}


def test_wide_forms_need_more(monkeypatch):
    k = [(0, "v_mfma_f32_32x32x16_f16 v[0:15], v[20:23], v[24:27], 0"), (8, "s_nop 9"), (12, "v_add_f32_e32 v40, v41, v15")]
    assert not base.short_reads(k)
    monkeypatch.setattr(base, "NEEDED", {**base.NEEDED, **WIDE})
    assert len(base.short_reads(k)) == 1
    assert not base.short_reads([k[0], (8, "s_nop 11"), k[2]])


@pytest.mark.skipif(not (os.path.exists(base.OBJDUMP) and os.path.exists(base.LIB)),
                    reason="needs llvm-objdump and the built library")
def test_no_wide_result_is_read_early(monkeypatch, tmp_path):
    monkeypatch.setattr(base, "NEEDED", {**base.NEEDED, **WIDE})
    base.test_no_mfma_result_is_read_early(tmp_path)
