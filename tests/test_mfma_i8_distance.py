"""The same check of the built code as test_mfma_distance.py's for the 32x32x32
product of 8-bit integers: eight passes, 12 wait states."""
import os

import pytest

import test_mfma_distance as base

WIDE = {"v_mfma_i32_32x32x32_i8": 12}


def test_the_form_is_looked_at(monkeypatch):
    k = [(0, "v_mfma_i32_32x32x32_i8 v[0:15], v[20:23], v[24:27], 0"), (8, "s_nop 9"), (12, "v_add_u32_e32 v40, v41, v15")]
    monkeypatch.setattr(base, "NEEDED", {**base.NEEDED, **WIDE})
    assert len(base.short_reads(k)) == 1
    assert not base.short_reads([k[0], (8, "s_nop 11"), k[2]])


@pytest.mark.skipif(not (os.path.exists(base.OBJDUMP) and os.path.exists(base.LIB)),
                    reason="needs llvm-objdump and the built library")
def test_no_result_is_read_early(monkeypatch, tmp_path):
    monkeypatch.setattr(base, "NEEDED", {**base.NEEDED, **WIDE})
    base.test_no_mfma_result_is_read_early(tmp_path)
