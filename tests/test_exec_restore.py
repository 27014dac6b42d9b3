"""Register copies in front of the point where all lanes are back, checked on the built code.

Where a wave's lanes have taken ways of their own, they meet again at a block that begins by restoring the execution
mask (s_or_b64 exec, exec, ...).  amdclang++ of ROCm 7.2 has been seen, where registers were short, to put a copy or a reload
of a vector register in front of that: the lanes that did not come by that way keep what the register held before.  This test
disassembles the library's gfx950 code objects and looks at each such restore: from where the lanes that were off enter (the
target of an s_cbranch_execz) to the restore nothing may write a vector register or memory.
"""
import os
import re
import shutil
import subprocess

import pytest

from test_mfma_distance import LIB, OBJDUMP

# (to and from scalar registers: these do not ask the mask)
VECTOR = re.compile(r"(v_(?!readlane|writelane|readfirstlane|nop)|ds_|global_|flat_|buffer_|scratch_)")


def early_writes(lines):
    """(restores, [what is written in front of one]).  lines: a kernel's instructions as (offset, text, offset of a branch's target or None)."""
    entered = {}
    for _, text, target in lines:
        if target is not None:
            entered.setdefault(target, set()).add(text.split()[0])
    restores, bad = 0, []
    for i, (_, text, _) in enumerate(lines):
        if not text.startswith("s_or_b64 exec, exec,"):
            continue
        restores += 1
        seen = []
        for j in range(i, -1, -1):
            offset, t, _ = lines[j]
            op, _, args = t.partition(" ")
            if j < i:
                if args.startswith("exec") or "saveexec" in op or op.startswith(("s_cbranch", "s_branch", "v_cmpx")):
                    break  # the mask is another here, or this is not a way to the restore
                if VECTOR.match(op):
                    seen.append(t)
            if offset in entered:
                if "s_cbranch_execz" in entered[offset]:
                    bad += seen
                break
    return restores, bad


def test_early_writes_are_found():
    k = [(0, "s_and_saveexec_b64 s[0:1], vcc", None), (4, "s_cbranch_execz 2", 16), (8, "v_add_f32_e32 v1, v2, v3", None), (12, "s_nop 0", None),
         (16, "v_mov_b32_e32 v101, v110", None), (20, "s_or_b64 exec, exec, s[0:1]", None), (24, "s_endpgm", None)]
    assert early_writes(k) == (1, ["v_mov_b32_e32 v101, v110"])
    k[4] = (16, "scratch_load_dword v5, off, s32", None)
    assert early_writes(k)[1]
    for k[4] in ((16, "v_readlane_b32 s4, v60, 3", None), (16, "v_writelane_b32 v60, s4, 3", None)):
        assert early_writes(k) == (1, [])
    # the body of a branch that is not jumped over
    assert early_writes([(0, "s_and_saveexec_b64 s[0:1], vcc", None), (4, "v_mov_b32_e32 v1, 0", None), (8, "s_or_b64 exec, exec, s[0:1]", None)]) == (1, [])


@pytest.mark.skipif(not (os.path.exists(OBJDUMP) and os.path.exists(LIB)), reason="needs llvm-objdump and the built library")
def test_no_vector_register_is_written_before_the_lanes_are_back(tmp_path):
    lib = str(tmp_path / "lib.so")
    shutil.copy(LIB, lib)
    subprocess.run([OBJDUMP, "--offloading", lib], check=True, capture_output=True, cwd=str(tmp_path))
    restores, bad, of_sampling = 0, [], 0
    for b in tmp_path.iterdir():
        if not b.name.endswith("gfx950"):
            continue
        out = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", str(b)], check=True, capture_output=True, text=True).stdout
        for sym in re.split(r"^(?=[0-9a-f]+ <)", out, flags=re.M):
            head, *body = sym.splitlines() or [""]
            if not re.match(r"[0-9a-f]+ <", head):
                continue
            base, lines = int(head.split()[0], 16), []
            for line in body:
                m = re.match(r"\s+(\S.*?)\s*// ([0-9A-F]+):(.*)$", line)
                if m:
                    target = re.search(r"\+0x([0-9a-f]+)>", m.group(3))
                    target = int(target.group(1), 16) if target else 0
                    lines.append((int(m.group(2), 16) - base, m.group(1), target if m.group(1).startswith(("s_cbranch", "s_branch")) else None))
            n, early = early_writes(lines)
            restores += n
            of_sampling += n if "sample_" in head else 0
            bad += ["%s: %s" % (head.split()[1][:100], t) for t in early]
    assert restores > 5000 and of_sampling > 100
    assert not bad, "\n".join(bad[:20])
