"""Attention over the 4-bit cache at the ends of fp32's range, by every kernel: keys far above or
below 1 with queries that bring the scores back, values whose averages fp32 holds, and values
from one end to the other along a sequence."""
import numpy as np
import pytest

from tests import kv4_sampled
from tests.kv4_plan import plan
from tests.test_gpu_kv4 import PAGE, Setup, ops, torch_dev  # noqa: F401
from tests.test_gpu_kv4_prompts import Wide

pytestmark = pytest.mark.gpu

CALLS = {
    "4": (Setup, 4, 2, [(1, 300), (1, 40)]),
    "16": (Setup, 8, 1, [(5, 300), (7, 40)]),
    "32": (Setup, 16, 4, [(300, 310), (150, 290), (100, 100)]),
    "128": (Setup, 20, 5, [(1000, 1000), (900, 950), (660, 661)]),
    "128 joined": (Wide, 4, 1, [(70, 200), (90, 700)]),
}


@pytest.mark.parametrize("kind", ["large_keys", "small_keys", "large_values", "small_values",
                                  "rising", "falling"])
@pytest.mark.parametrize("call", CALLS)
def test_ends_of_the_range(torch_dev, ops, call, kind):
    make, Hq, Hkv, seqs = CALLS[call]
    s = make(seqs, Hq, Hkv, layers=1, seed=len(call))
    ks, vs = s.pools[2], s.pools[3]
    t = np.zeros((s.nb, 1, 1, PAGE, 1), np.int64)  # a slot's position
    for b in range(len(seqs)):
        for p, page in enumerate(s.tables[b]):
            if page >= 0:
                t[page, 0, 0, :, 0] = np.arange(PAGE) + p * PAGE
    if kind == "large_keys":
        ks[:] = 127 + 112
        s.q *= 2.0 ** -110
    elif kind == "small_keys":
        ks[:] = 127 - 117
        s.q *= 2.0 ** 115
    elif kind == "large_values":
        vs[:] = 127 + 116
    elif kind == "small_values":
        vs[:] = 127 - 114
    else:
        up = 3 + 230 * (t % 200) // 200
        vs[:] = up if kind == "rising" else 236 - up
    s.dev(torch_dev)
    kernel, parts, _ = plan(s.T, len(seqs), Hq, Hkv, s.tables.shape[1], True)
    assert (kernel, parts > 1) == (call.split()[0], call in ("4", "16", "32", "128 joined"))
    print("attn range", call, kind, flush=True)
    out = ops.attn_kv4(s.d["q"], *s.args(), **s.opts()).cpu().numpy()
    kv4_sampled.check(s, out)
