"""The plan of the attention over the 4-bit cache as the tests state it (kv4_plan.py), against the
sizes of workspaces that the library computes (a host function: no GPU)."""
import random

import pytest

from tenzo_amd import _lib
from tests.kv4_plan import plan


@pytest.mark.parametrize("seed", range(6))
def test_workspaces(seed):
    rng = random.Random(seed)
    ws = _lib.load().tenzo_hip_attn_kv4_ws_bytes
    kernels = set()
    for _ in range(4000):
        Hkv = rng.choice([1, 2, 3, 5, 8])
        Hq = Hkv * rng.randint(1, 16)
        B = int(2 ** rng.uniform(0, 9))
        cu = rng.random() < 0.6
        T = int(B * 2 ** rng.uniform(0, 11)) if cu else B
        width = int(2 ** rng.uniform(0, 16)) - 1
        want = plan(T, B, Hq, Hkv, width, cu)
        for dtype in (0, 1):
            assert ws(T, B, Hq, Hkv, width, int(cu), dtype) == want[2], (T, B, Hq, Hkv, width, cu)
        kernels.add((want[0], want[1] > 1))
    assert kernels == {("4", False), ("4", True), ("16", False), ("16", True), ("32", False),
                       ("32", True), ("128", False), ("128", True), ("4 even", False),
                       ("16 even", False)}
