"""What the compiler does not check around the loads that attention_kv4.hip issues from assembly,
straight into LDS, checked in the gfx950 assembly of that source (CPU: compiled here, nothing runs):

* M0, which the assembly sets right before each, is used by nothing else in those kernels;
* conversions to and from 6 bits, in assembly too, read nothing that a matrix instruction or one of
  the transcendental unit wrote right before."""
import os
import re
import subprocess

import pytest

from tenzo_amd import build

LOAD = re.compile(r"global_load_lds_dword(x4)? v\[\d+:\d+\], off")
CONVERT = re.compile(r"v_cvt_scalef32_(2xpk16_fp6_f32|pk32_f32_fp6) ")
SLOW = re.compile(r"v_(mfma|smfmac|exp|log|rcp|rsq|sqrt|sin|cos)_\S+ v(\[(\d+):(\d+)\]|(\d+))")


def kernels(text):
    """{name: its lines} of the functions with such loads."""
    found = {}
    for m in re.finditer(r"^(\w+):[^\n]*\n(.*?)^\.Lfunc_end", text, re.S | re.M):
        lines, app = [], False
        for line in m.group(2).split("\n"):
            app = (app or "#APP" in line or "#ASMSTART" in line) and not (
                "#NO_APP" in line or "#ASMEND" in line)
            code = line.split(";")[0].strip()
            if code and not code.startswith(".") and not code.endswith(":"):
                lines.append((code, app))
        if any(LOAD.search(c) for c, _ in lines):
            found[m.group(1)] = lines
    return found


def vectors(text):
    """Vector registers that operands name."""
    out = set()
    for m in re.finditer(r"\bv(?:\[(\d+):(\d+)\]|(\d+))", text):
        out |= {int(m[3])} if m[3] else set(range(int(m[1]), int(m[2]) + 1))
    return out


def wrong(lines):
    bad = []
    for i, (code, app) in enumerate(lines):
        if LOAD.search(code):
            before = [c for c, _ in lines[max(i - 2, 0):i]]
            if not (app and len(before) == 2 and before[0].startswith("s_mov_b32 m0,") and
                    before[1] == "s_nop 0"):
                bad.append(code)
        elif not app and re.search(r"\bm0\b", code):
            bad.append(code)
        elif CONVERT.match(code):
            sources = vectors(code.split(",", 1)[1])
            for prev, _ in lines[max(i - 20, 0):i]:  # (a matrix instruction takes 16 passes at most)
                if SLOW.match(prev) and vectors(prev.split(",")[0]) & sources:
                    bad.append((prev, code))
    return bad


def test_planted_mistakes_are_seen():
    load = [("s_mov_b32 m0, s4", True), ("s_nop 0", True),
            ("global_load_lds_dwordx4 v[2:3], off", True)]
    cvt = ("v_cvt_scalef32_2xpk16_fp6_f32 v[40:45], v[0:15], v[16:31], v32", True)
    assert not wrong(load + [cvt])
    assert wrong([load[0], load[2]]) and wrong([*load, ("v_movreld_b32_e32 v1, m0", False)])
    assert wrong([("v_exp_f32_e32 v32, v33", False), cvt])
    assert wrong([("v_mfma_f32_16x16x32_f16 v[0:3], v[50:53], v[54:57], 0", False), cvt])
    assert not wrong([("v_exp_f32_e32 v39, v32", False), cvt])


def test_assembly_of_the_kernels(tmp_path):
    if not os.path.exists(build.HIPCC):
        pytest.skip("needs hipcc")
    out = str(tmp_path / "attention_kv4.s")
    subprocess.run([build.HIPCC, *build.FLAGS, "--cuda-device-only", "-S",
                    os.path.join(build.CSRC, "attention_kv4.hip"), "-o", out], check=True,
                   capture_output=True)
    with open(out) as f:
        found = kernels(f.read())
    assert len(found) == 4  # fp32 and fp16, steps dealt evenly and a workgroup for all
    for name, lines in found.items():
        assert not wrong(lines), (name, wrong(lines)[:3])
        assert sum(bool(CONVERT.match(c)) for c, _ in lines) >= 8, name
