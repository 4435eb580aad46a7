"""Attention over the 4-bit cache checked at some of a call's rows (prompts have too many for
numpy): a row is a sequence of its own that ends at the row's position."""
import numpy as np

from tests import kv4_plain as plain


def check(s, out, count=60, seed=0):
    """s: a test_gpu_kv4.Setup. Queries and weights are held to 24 bits or to 22 (2^-21 for both)."""
    at = plain.places(s.T, s.tables, s.ctx, s.cu, plain.limit_of(s.tables, s.rope))
    rows = np.random.default_rng(seed).permutation([r for r, a in enumerate(at) if a])[:count]
    seq, pos = np.array([at[r] for r in rows]).T
    want, tol = plain.attention(s.q[rows], s.pools, s.tables[seq], pos + 1, s.layer, s.rope, None,
                                np.zeros((len(rows), s.Hq, 128)), 2.0 ** -21)
    # (2^-37 of the largest value that any row sees)
    G = s.Hq // s.Hkv
    for i, b in enumerate(seq):
        tol[i] += 2.0 ** -37 * np.repeat(
            plain._largest(s.pools, s.tables[b], int(s.ctx[b]), s.layer), G)[:, None]
    got = out.reshape(s.T, s.Hq, 128)[rows].astype(np.float64)
    step = np.finfo(s.dtype)
    tol += float(step.eps) / 2 * (np.abs(want) + tol) + float(step.smallest_subnormal) / 2
    worst = float((np.abs(got - want) / tol).max())
    assert np.isfinite(got).all() and worst <= 1, worst
