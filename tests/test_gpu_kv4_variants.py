"""Attention over the 4-bit cache by the kernels and joins that ordinary sizes take and the other tests
do not: prompts that fill the GPU without parts, 32 rows a workgroup in parts, batches of tokens whose
heads are joined by groups of lanes, short tables, and more pages than the prompts' kernel keeps
at a time. Each says which kernel it means (kv4_plan)."""
import numpy as np
import pytest

from tests import kv4_sampled
from tests.kv4_plan import plan
from tests.test_gpu_kv4 import PAGE, Setup, ops, torch_dev  # noqa: F401

pytestmark = pytest.mark.gpu


def attend(ops, s):
    return ops.attn_kv4(s.d["q"], *s.args(), **s.opts()).cpu().numpy()


def planned(s):
    return plan(s.T, len(s.seqs), s.Hq, s.Hkv, s.tables.shape[1], s.cu is not None)[:2]


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("Hq,Hkv,seqs", [
    (20, 5, [(1000, 1000), (900, 1711), (660, 661), (1, 1400), (0, 9)]),
    (32, 8, [(1300, 1333), (257, 2000)]), (7, 1, [(3001, 3001), (4300, 4300), (13, 4000)])])
def test_prompts_in_one_part(torch_dev, ops, Hq, Hkv, seqs, dtype):
    s = Setup(seqs, Hq, Hkv, layers=2, dtype=dtype, seed=Hq).dev(torch_dev)
    assert planned(s) == ("128", 1)
    print("attn one part", Hq, seqs, dtype.__name__, flush=True)
    kv4_sampled.check(s, attend(ops, s), 100)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("Hq,Hkv,seqs", [
    (16, 4, [(293, 352), (260, 271)]), (8, 8, [(540, 540), (510, 511), (1, 300)])])
def test_32_rows_in_parts(torch_dev, ops, Hq, Hkv, seqs, dtype):
    s = Setup(seqs, Hq, Hkv, dtype=dtype, seed=Hq).dev(torch_dev)
    kernel, parts = planned(s)
    assert kernel == "32" and parts > 1
    print("attn 32 rows", Hq, seqs, dtype.__name__, flush=True)
    kv4_sampled.check(s, attend(ops, s), 200)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("Hq,Hkv,kernel", [(32, 8, "4 even"), (64, 8, "16 even"),
                                           (30, 10, "4 even")])
def test_batch_of_tokens(torch_dev, ops, Hq, Hkv, kernel, dtype):
    """Over 1024 rows times heads: 8 heads to a workgroup of the join."""
    rng = np.random.default_rng(Hq)
    lens = [3000, 0, 2222, 1, 256, 257, -1, 64] + [int(n) for n in rng.integers(1, 2000, 36)]
    s = Setup([(1, c) for c in lens], Hq, Hkv, layers=1, cu=False, dtype=dtype, seed=Hq).dev(
        torch_dev)
    assert planned(s)[0] == kernel and s.T * Hq > 1024
    print("attn tokens", Hq, Hkv, dtype.__name__, flush=True)
    s.check_attention(attend(ops, s))


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("Hq,Hkv,kernel", [(8, 2, "4"), (4, 4, "4"), (16, 2, "16"), (15, 3, "16")])
def test_short_tables(torch_dev, ops, Hq, Hkv, kernel, dtype):
    """One step's worth of positions: nothing to join."""
    lens = [1, 0, 255, 256, 100, 16, 17, 64, 65, 200]
    s = Setup([(1, c) for c in lens], Hq, Hkv, cu=False, dtype=dtype, seed=Hq).dev(torch_dev)
    assert planned(s) == (kernel, 1)
    print("attn short", Hq, Hkv, dtype.__name__, flush=True)
    s.check_attention(attend(ops, s))


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_tokens_joined_by_16(torch_dev, ops, dtype):
    """Over 1024 rows times heads, in parts of a grid."""
    s = Setup([(20, 700), (23, 24), (19, 555)], 24, 3, layers=1, dtype=dtype, seed=2).dev(torch_dev)
    kernel, parts = planned(s)
    assert kernel == "16" and parts > 1 and s.T * s.Hq > 1024
    print("attn join", parts, flush=True)
    s.check_attention(attend(ops, s))


def test_many_pages_of_prompts(torch_dev, ops):
    """A part of more than 16384 tokens: page numbers taken anew on the way, some of them of pages
    that the pool does not hold."""
    s = Setup([(70, 33500)], 1, 1, layers=1, seed=8)
    s.tables[0, 1029] = -1
    s.tables[0, 2000] = s.nb
    # (a table so wide that a part has over 16384 tokens; the rotation's rows are the limit)
    s.tables = np.pad(s.tables, ((0, 0), (0, 700000 - s.tables.shape[1])), constant_values=-1)
    s.dev(torch_dev)
    kernel, parts = planned(s)
    assert kernel == "128" and 700000 * PAGE // parts > 17000
    print("attn many pages", parts, flush=True)
    kv4_sampled.check(s, attend(ops, s), 20)
