"""The checks of test_assembly_hazards.py for the loads that gemm_i8.hip issues from assembly (CPU:
compiled here, nothing runs)."""
import os
import re
import subprocess

import pytest

from tenzo_amd import build
from tests.test_assembly_hazards import hazards, kernels


def test_assembly_loads_are_spaced(tmp_path):
    if not os.path.exists(build.HIPCC):
        pytest.skip("needs hipcc")
    out = str(tmp_path / "gemm_i8.s")
    subprocess.run([build.HIPCC, *build.FLAGS, "--cuda-device-only", "-S",
                    os.path.join(build.CSRC, "gemm_i8.hip"), "-o", out], check=True,
                   capture_output=True)
    with open(out) as f:
        found = kernels(f.read())
    assert len(found) == 36  # every tile, type of outputs, with and without the largest values
    for name, lines in found.items():
        assert not hazards(lines), (name, hazards(lines)[:3])
        assert not [c for c, app in lines if not app and re.search(r"\bm0\b", c)], name
