"""Ranges of cu_q that lie over each other, which the calls on a paged cache do not give a meaning:
they end, nothing but the rows and pages of the call's sequences changes, and the next call is
right."""
import numpy as np
import pytest

from tests.kv4_plan import plan
from tests.test_gpu_kv4 import D, Setup, ops, torch_dev  # noqa: F401
from tests.test_gpu_kv4_prompts import Wide

pytestmark = pytest.mark.gpu

CALLS = {
    "4 even": (Setup, 4, 2, 1, [(1, 9000)] + [(1, 30 + b) for b in range(60)]),
    "16 even": (Setup, 16, 2, 1, [(7, 4000)] + [(1 + b % 5, 20 + 7 * b) for b in range(40)]),
    "16": (Setup, 8, 1, 1, [(5, 300), (7, 40), (9, 9)]),
    "32": (Setup, 16, 4, 1, [(300, 310), (150, 290), (100, 100)]),
    "128": (Wide, 4, 1, 1, [(70, 200), (90, 700), (80, 80)]),
}


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("kind", ["back", "all", "pairs", "swapped"])
def test_ranges_over_each_other(torch_dev, ops, call, kind):
    torch = torch_dev
    make, Hq, Hkv, layers, seqs = CALLS[call]
    s = make(seqs, Hq, Hkv, layers=layers, seed=4, tail=5, extra=9).dev(torch)
    B = len(seqs)
    assert plan(s.T, B, Hq, Hkv, s.tables.shape[1], True)[0] == call
    rows = int(s.cu[-1])
    cu = s.cu.copy()
    if kind == "back":      # the last sequences have the first ones' rows once more
        cu[B // 2:] = s.cu[:B + 1 - B // 2]
    elif kind == "all":     # every other one has all rows
        cu[::2], cu[1::2] = 0, rows
    elif kind == "pairs":
        cu[1:] = np.maximum(cu[1:] - 1, 0)
        cu[::3] = 0
    else:
        cu = cu[::-1].copy()
        cu[-1] = rows
    print("overlap", call, kind, flush=True)
    bad = torch.from_numpy(cu).cuda()
    start = np.full((s.T, Hq, D), 7.0, np.float32)
    out = torch.from_numpy(start).cuda()
    opts = {"rope_cs": s.d["rope"], "cu_q": bad}
    ops.attn_kv4(s.d["q"], *s.args(), **opts, out=out)
    torch.cuda.synchronize()
    assert (out[rows:] == 7).all()
    before = [a.clone() for a in s.dp]
    ops.kv4_append(s.d["k"], s.d["v"], *s.args(), **opts)
    ops.kv4_read(*s.args(), rows=s.T, cu_q=bad)
    torch.cuda.synchronize()
    held = np.unique(s.tables[s.tables >= 0])
    free = torch.from_numpy(np.setdiff1d(np.arange(s.nb), held)).cuda()
    for a, b in zip(s.dp, before):
        assert torch.equal(a[free], b[free])
        a.copy_(b)
    out.fill_(7)
    ops.attn_kv4(s.d["q"], *s.args(), **s.opts(), out=out)
    s.check_attention(out.cpu().numpy(), start)
