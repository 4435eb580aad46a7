"""fp16 calls of attention over trees are as exact in every kernel that the plan may choose, whatever
else is in the batch: queries are held to 2^-24 of the largest of 32 dims or better, weights to 22 bits,
and an output is rounded once."""
import numpy as np
import pytest

from tests import tree_plain as plain
from tests.test_gpu_kv4 import D, ops, torch_dev  # noqa: F401
from tests.test_gpu_tree import WIDE, Trees

pytestmark = pytest.mark.gpu


def check(s, out):
    """Every output within the rounding of the value that 64 bits give, and of what fp32 sums, queries
    and weights of 2^-21 may be off: of an interval, what its two ends round to."""
    want = np.zeros((s.T, s.Hq, D))
    want, tol = plain.attention(s.q, s.mask, s.pools, s.tables, s.ctx, s.layer, s.cu, want,
                                2.0 ** -21, 2.0 ** -21)
    # what is below fp16's smallest numbers is lost: half of 2^-24, where the row's largest weight
    # stands for 2^12 or more, of each token's values (up to 6 times the largest scale, 2)
    tol += 2.0 ** -37 * max(c for _, c in s.seqs) * 12
    got = out.cpu().numpy().reshape(want.shape)
    low, high = (want - tol).astype(np.float16), (want + tol).astype(np.float16)
    off = np.where(got < low, low.astype(np.float64) - got, got.astype(np.float64) - high)
    assert np.isfinite(got).all()
    print("outputs beyond:", int((off > 0).sum()), "of", off.size, "worst", float(off.max()))
    assert (off <= 0).all()


PLANS = [([(26, 60), (40, 45)], 20, 5, "16", None),
         ([(26, 60), (40, 45)], 20, 5, "128 even", WIDE),
         ([(130, 170), (100, 1000), (64, 64)], 16, 1, "128 even", WIDE),
         ([(50 + i % 15, 70 + 3 * i) for i in range(60)], 8, 2, "128", None)]


@pytest.mark.parametrize("seqs,Hq,Hkv,kernel,width", PLANS)
def test_weights(torch_dev, ops, seqs, Hq, Hkv, kernel, width):
    """Small queries: scores are near each other and exact, so what is off is the weights'."""
    s = Trees(seqs, Hq, Hkv, "tree", dtype=np.float16, width=width, layers=1)
    s.q = (s.q / 8).astype(np.float16)
    s.dev(torch_dev)
    print("weights", seqs[:3], s.kernel(), flush=True)
    assert s.kernel() == kernel
    check(s, s.run(ops))


@pytest.mark.parametrize("seqs,Hq,Hkv,kernel,width", PLANS)
def test_queries_with_one_large_dim(torch_dev, ops, seqs, Hq, Hkv, kernel, width):
    """One dim of each 32 is 3000 times the others, where no key has anything: the others count with
    all of their bits."""
    s = Trees(seqs, Hq, Hkv, "tree", dtype=np.float16, width=width, layers=1)
    s.q[:, :, ::32] = 3000
    s.pools[0][..., ::16] &= 0xf0  # dim 32 g: the low codes of byte 16 g
    s.dev(torch_dev)
    print("queries", seqs[:3], s.kernel(), flush=True)
    assert s.kernel() == kernel
    check(s, s.run(ops))
