"""The cases of attention over the paged cache in 4 bits once more for the kernels of long prompts:
how rows and tokens are shared among workgroups follows from the rows and from the width of the
tables, so the same sequences are given tables of many more columns (parts of a few hundred
tokens of 128 rows), and many rows short ones (32 rows)."""
import numpy as np
import pytest

from tests import test_gpu_kv4 as base
from tests.test_gpu_kv4 import D, PAGE, ops, torch_dev  # noqa: F401

pytestmark = pytest.mark.gpu


class Wide(base.Setup):
    """Tables so wide that rows * kv heads / 128 * positions is past 3500 tiles of 64."""

    def dev(self, torch):
        rows = self.T * self.Hq
        assert rows > 64 * len(self.seqs), "an average sequence of more than 64 rows"
        columns = -(-int(1.2 * 3500 * 64 * 128 / rows) // PAGE)
        more = max(0, columns - self.tables.shape[1])
        self.tables = np.pad(self.tables, ((0, 0), (0, more)), constant_values=-1)
        return super().dev(torch)


@pytest.fixture
def wide(monkeypatch):
    monkeypatch.setattr(base, "Setup", Wide)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("Hq,Hkv,seqs", [
    (5, 1, [(33, 33), (1, 1), (64, 200)]), (4, 4, [(70, 70), (130, 131), (16, 300)]),
    (20, 5, [(40, 90), (17, 17), (3, 0)]), (2, 1, [(300, 310)]), (16, 1, [(20, 64), (4, 4)]),
    (4, 1, [(200, 230), (1, 1), (130, 100), (0, 0), (97, 2000)]), (3, 1, [(150, 150), (260, 700)]),
    (8, 2, [(64, 1000), (65, 65)]), (4, 1, [(40, 1100), (60, 900), (30, 2100)]),
    (4, 1, [(20 + b % 3, 20 + 5 * (b % 7)) for b in range(66)])])
def test_rows(torch_dev, ops, wide, Hq, Hkv, seqs, dtype):
    base.test_attention_rows(torch_dev, ops, Hq, Hkv, seqs, dtype)


@pytest.mark.parametrize("kind", ["keys", "values", "small", "large", "rising", "falling",
                                  "zeros", "one_group"])
@pytest.mark.parametrize("n,Hq", [(70, 4), (129, 1)])
def test_scale_range(torch_dev, ops, wide, kind, n, Hq):
    base.test_attention_scale_range(torch_dev, ops, kind, n, Hq)


def test_peaked_and_flat(torch_dev, ops, wide):
    base.test_attention_peaked_and_flat(torch_dev, ops, 70)


def test_bad_pages(torch_dev, ops, wide):
    base.test_attention_bad_pages(torch_dev, ops, 25)


def test_rope_shorter_than_tables(torch_dev, ops, wide, monkeypatch):
    """Also lengths past the rotation's rows: padding."""
    s = Wide([(50, 60), (50, 61)], 4, 1, seed=1)
    s.rope = s.rope[:60]
    s.dev(torch_dev)
    s.check_attention(ops.attn_kv4(s.d["q"], *s.args(), **s.opts()).cpu().numpy())


def test_strides(torch_dev, ops):
    """q and out slices of wider buffers at odd offsets."""
    torch = torch_dev
    s = Wide([(30, 700), (41, 41)], 8, 2, seed=1).dev(torch)
    rows = torch.randn((s.T, 3 + 12 * D), device="cuda")
    q = rows[:, 3:3 + 8 * D]
    s.q = q.cpu().numpy().reshape(s.T, 8, D)
    buf = torch.full((s.T, 5 + 8 * D), 3.0, device="cuda")
    ops.attn_kv4(q, *s.args(), **s.opts(), out=buf[:, 1:1 + 8 * D])
    s.check_attention(buf[:, 1:1 + 8 * D].cpu().numpy())
    assert (buf[:, 0] == 3).all() and (buf[:, 1 + 8 * D:] == 3).all()


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("Hq,Hkv,seqs", [
    (16, 2, [(300, 330), (150, 150), (120, 500)]), (32, 8, [(17, 17)] * 9 + [(120, 128)])])
def test_many_rows_of_few_tokens(torch_dev, ops, Hq, Hkv, seqs, dtype):
    base.test_attention_rows(torch_dev, ops, Hq, Hkv, seqs, dtype)


@pytest.mark.parametrize("make", [base.Setup, Wide])
@pytest.mark.parametrize("end", [1000, -1, 2 ** 31 - 1, 69])
def test_range_outside_the_rows(torch_dev, ops, make, end):
    """A range of cu_q that the rows do not hold, or that ends before it begins, is no sequence:
    its rows' outputs and its pages stay as they were."""
    torch = torch_dev
    s = make([(70, 90)], 4, 1, seed=5, tail=6).dev(torch)
    n = s.d["tables"]
    tables = torch.cat([n, n.flip(1).roll(1, 1)])
    ctx = torch.tensor([90, 90], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 70, end], dtype=torch.int32, device="cuda")
    start = np.full((s.T, 4, D), 7.0, np.float32)
    out = torch.from_numpy(start).cuda()
    ops.attn_kv4(s.d["q"], *s.dp, tables, ctx, s.layer, rope_cs=s.d["rope"], cu_q=cu, out=out)
    s.check_attention(out.cpu().numpy(), start)
    ops.kv4_append(s.d["k"], s.d["v"], *s.dp, tables, ctx, s.layer, rope_cs=s.d["rope"], cu_q=cu)
    base.plain.append(s.k, s.v, s.pools, s.tables, s.ctx, s.layer, s.rope, s.cu)
    base.pools_equal(s, s.dp)
