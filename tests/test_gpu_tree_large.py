"""Trees' operators, rotary positions and the 8-bit product on tensors whose offsets pass 32 bits (up
to 16 GB), and rows as far apart as they may be."""
import numpy as np
import pytest

from tests import tree_plain as plain
from tests.test_gpu_gemm_i8 import make
from tests.test_gpu_kv4 import PAGE, ops, torch_dev  # noqa: F401
from tests.test_gpu_rope import check
from tests.test_gpu_tree import WIDE, Trees, drafts

pytestmark = pytest.mark.gpu


def test_rope_past_32_bits(torch_dev, ops):
    torch = torch_dev
    T, cols = 70000, 32768
    x = torch.zeros((T, cols), dtype=torch.float16, device="cuda")
    rows = [0, 65535, 65536, T - 1]
    x[rows] = torch.randn((len(rows), cols), device="cuda").half()
    was = x[rows].clone()
    at = torch.arange(T, dtype=torch.int32, device="cuda")
    f, _ = ops.rope_freqs(128)
    assert ops.rope(x, at, f.cuda(), out=x) is x
    check(x[rows], was, np.array(rows, np.int32), f.numpy(), False, 1.0, "float16", 128)
    assert not x[1:65535].any()


def test_gemm_past_32_bits(torch_dev, ops):
    torch = torch_dev
    M, N, K = 17000, 131072, 16
    args, _ = make(torch, ops, 1, N, K)
    codes = torch.randint(-128, 128, (M, K), dtype=torch.int8, device="cuda")
    q = torch.rand((M, 2), device="cuda").view(torch.int32)
    y, idx = ops.gemm_i8(codes, q, *args[2:], dtype=torch.float16, want_idx=True)
    for m in (0, 16383, 16384, M - 1):
        one, at = ops.gemm_i8(codes[m:m + 1], q[m:m + 1], *args[2:], dtype=torch.float16,
                              want_idx=True)
        assert torch.equal(one[0], y[m]) and at.item() == idx[m].item()


@pytest.mark.parametrize("M", [3, 20, 200])
def test_gemm_rows_far_apart(torch_dev, ops, M):
    """Rows of codes 2^22 bytes apart, the most that is allowed."""
    torch = torch_dev
    args, want = make(torch, ops, M, 130, 272, seed=M)
    wide = torch.zeros((M, 1 << 22), dtype=torch.int8, device="cuda")
    wide[:, :272] = args[0]
    y, idx = ops.gemm_i8(wide[:, :272], *args[1:], want_idx=True)
    assert torch.equal(y.cpu(), torch.from_numpy(want))
    np.testing.assert_array_equal(idx.cpu().numpy(), plain.first_best(want))


@pytest.mark.parametrize("width", [None, WIDE])
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_attention_and_acceptance_past_32_bits(torch_dev, ops, dtype, width):
    """Pages at the end of pools of 5.4 GB of codes: bit for bit what small pools with the same
    pages give."""
    torch = torch_dev
    s = Trees([(40, 300), (64, 100)], 8, 2, "tree", dtype=dtype, width=width, layers=3).dev(torch)
    want = s.run(ops)
    nb = s.dp[0].shape[0]
    big = 5_400_000_000 // (3 * 2 * PAGE * 64)
    pools = ops.kv4_pool(big, 3, 2)
    for a, b in zip(pools, s.dp):
        a[big - nb:] = b
    tables = s.d["tables"] + (big - nb)
    tables[s.d["tables"] < 0] = -1
    got = ops.attn_tree_kv4(s.d["q"], s.d["mask"], *pools, tables, *s.args()[5:], cu_q=s.d["cu"])
    assert torch.equal(got, want)
    parents = torch.from_numpy(s.parents).cuda()
    tokens, target = (torch.from_numpy(a // 3).cuda() for a in drafts(s.rng, s.parents, 0.95))
    one = ops.tree_accept(parents, tokens, target, *s.dp, s.d["tables"], s.d["ctx"], 64,
                          cu_q=s.d["cu"])
    two = ops.tree_accept(parents, tokens, target, *pools, tables, s.d["ctx"], 64, cu_q=s.d["cu"])
    assert one[1].max() > 1
    for a, b in zip(one, two):
        assert torch.equal(a, b)
    for a, b in zip(pools, s.dp):
        assert torch.equal(a[big - nb:], b) and not a[:big - nb].any()
