"""Trees of drafted tokens on the GPU against the plain forms: plans and accepted paths bit for bit,
attention within the rounding of fp32 sums, counted per output."""
import numpy as np
import pytest

from tests import tree_plain as plain
from tests.test_gpu_kv4 import D, PAGE, Setup, ops, torch_dev  # noqa: F401
from tests.tree_kernels import plan

pytestmark = pytest.mark.gpu


def random_parents(rng, n, way="tree"):
    if way == "chain":
        return np.arange(-1, n - 1)
    if way == "flat":
        return np.full(n, -1)
    p = np.floor(rng.uniform(0.2, 1, n) * np.arange(n)).astype(int)
    p = np.minimum(p, np.arange(n) - 1)
    if way == "odd":  # several roots, and numbers that are nobody's parent
        p[rng.integers(0, n, max(1, n // 4))] = -1
        i = rng.integers(0, n, max(1, n // 4))
        p[i] = rng.choice([n, 10 ** 9, -7, -2 ** 31], len(i))
        p[n // 2] = n // 2
    return p


def forest(rng, seqs, tail=0, way="tree"):
    rows = [random_parents(rng, n, way) for n, _ in seqs if n]
    return np.concatenate([*rows, np.full(tail, 5)]).astype(np.int32)


# -------------------------------------------------------------------- plan ----

PLANS = [[(1, 1)], [(5, 9), (0, 3), (64, 64), (3, 0), (17, 1000)], [(64, 70000)], [(65, 70)],
         [(130, 200), (1, 7), (64, 64), (63, 100)], [(700, 900), (128, 128)], [(9, 4), (70, 60)],
         [(i % 7, 40 + i) for i in range(150)]]


@pytest.mark.parametrize("way", ["tree", "chain", "flat", "odd"])
@pytest.mark.parametrize("seqs", PLANS, ids=lambda s: f"{len(s)}x{max(n for n, _ in s)}")
def test_plan(torch_dev, ops, seqs, way):
    torch, rng = torch_dev, np.random.default_rng(len(seqs))
    print("plan", seqs[:4], way, flush=True)
    parents = forest(rng, seqs, 3, way)
    ctx = np.array([c for _, c in seqs], np.int32)
    cu = np.concatenate([[0], np.cumsum([n for n, _ in seqs])]).astype(np.int32)
    most = max(n for n, _ in seqs)
    mask, at = ops.tree_plan(torch.from_numpy(parents).cuda(), torch.from_numpy(ctx).cuda(), most,
                             cu_q=torch.from_numpy(cu).cuda())
    mask, at = mask.cpu().numpy().view(np.uint64), at.cpu().numpy()
    want, where = mask.copy(), at.copy()  # (rows of no sequence as they are)
    plain.tree_plan(parents, ctx, cu, most, want, where)
    np.testing.assert_array_equal(mask, want)
    np.testing.assert_array_equal(at, where)


def test_plan_of_single_nodes(torch_dev, ops):
    torch = torch_dev
    ctx = torch.tensor([4, 0, 900, -3], dtype=torch.int32).cuda()
    mask, at = ops.tree_plan(torch.full((4,), -1, dtype=torch.int32).cuda(), ctx, 1)
    assert mask.cpu().tolist() == [[1], [0], [1], [0]] and at.cpu().tolist() == [3, 0, 899, 0]


# --------------------------------------------------------------- attention ----

WIDE = 20000  # pages of a table: the plan takes its width for the context


class Trees(Setup):
    def __init__(self, seqs, Hq, Hkv, way="tree", words=None, **more):
        super().__init__(seqs, Hq, Hkv, rope=False, **more)
        most = max(n for n, _ in seqs)
        words = words or max(1, -(-most // 64))
        self.mask = np.zeros((self.T, max(words, -(-most // 64))), np.uint64)
        self.parents = forest(self.rng, seqs, self.T - sum(n for n, _ in seqs),
                              "tree" if way == "bits" else way)
        if way == "bits":  # any bits, some rows without one, those of nobody's node set
            self.mask[:] = self.rng.integers(0, 2 ** 63, self.mask.shape).astype(np.uint64) * 2 + \
                self.rng.integers(0, 2, self.mask.shape).astype(np.uint64)
            self.mask[self.rng.integers(0, self.T, max(1, self.T // 5))] = 0
        else:
            plain.tree_plan(self.parents, np.full(len(seqs), 10 ** 6, np.int32), self.cu,
                            self.mask.shape[1] * 64, self.mask, np.zeros(self.T, np.int32))
        self.mask = np.ascontiguousarray(self.mask[:, :words])

    def dev(self, torch):
        super().dev(torch)
        self.d["mask"] = torch.from_numpy(self.mask.view(np.int64)).cuda()
        return self

    def run(self, ops, out=None, q=None, mask=None):
        return ops.attn_tree_kv4(self.d["q"] if q is None else q,
                                 self.d["mask"] if mask is None else mask, *self.args(),
                                 cu_q=self.d["cu"], out=out)

    def check(self, out, start=None):
        want = np.zeros((self.T, self.Hq, D)) if start is None else start.astype(np.float64)
        # queries and weights are held to 22 bits or more in fp32 calls (2^-21 for the two), in
        # fp16 calls of 128 rows weights to 11 (half a step: 2^-11), elsewhere every bit
        half = self.dtype == np.float16 and self.kernel().startswith("128")
        want, tol = plain.attention(self.q, self.mask, self.pools, self.tables, self.ctx,
                                    self.layer, self.cu, want, 2.0 ** -21,
                                    2.0 ** -11 if half else 2.0 ** -21)
        got = out.cpu().numpy().reshape(want.shape).astype(np.float64)
        step = np.finfo(self.dtype)
        tol = tol + float(step.eps) / 2 * (np.abs(want) + tol) + float(step.smallest_subnormal) / 2
        worst = float(np.max(np.abs(got - want) / np.where(tol > 0, tol, 1e-300)))
        assert np.isfinite(got).all() and worst <= 1, worst

    def kernel(self):
        return plan(self.T, len(self.seqs), self.Hq, self.Hkv, self.tables.shape[1],
                    self.cu is not None, self.dtype == np.float16)[0]


@pytest.mark.parametrize("way", ["tree", "bits"])
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("seqs,Hq,Hkv,kernel,width", [
    ([(1, 1)], 1, 1, "4", None), ([(2, 3000)], 2, 2, "4", None),
    ([(3, 3), (0, 40), (2, 0), (1, 17)], 2, 2, "4", None),
    ([(9, 9)], 10, 5, "16", None), ([(12, 777)], 20, 5, "16", None),
    ([(3, 40), (5, 5), (6, 130), (7, 0), (1, 65)], 16, 2, "16", None),
    ([(60, 600), (55, 65)], 4, 4, "16", None), ([(12, 5000)], 8, 8, "16", None),
    ([(6, 700 + 97 * i) for i in range(9)], 8, 8, "16 even", None),
    ([(1 + i % 2, 500 + 211 * i) for i in range(12)], 16, 16, "4 even", None),
    ([(2, 300)] * 5 + [(4, 4000)], 8, 8, "4 even", 400),
    ([(10, 60 + i) for i in range(48)], 32, 8, "32", None),
    ([(26, 777)], 20, 5, "128 even", WIDE), ([(130, 131)], 1, 1, "128 even", WIDE),
    ([(33, 40), (5, 5), (64, 130), (7, 0), (1, 65)], 16, 2, "128 even", WIDE),
    ([(130, 170), (100, 1000), (64, 64)], 16, 1, "128 even", WIDE),
    ([(64, 200), (61, 5000), (40, 0), (30, 30)], 16, 1, "128 even", WIDE),
    ([(40 + i, 300 + 50 * i) for i in range(9)], 8, 4, "128 even", WIDE)])
def test_attention(torch_dev, ops, seqs, Hq, Hkv, kernel, width, dtype, way):
    s = Trees(seqs, Hq, Hkv, way, dtype=dtype, width=width, tail=2, seed=len(seqs)).dev(torch_dev)
    print("tree", seqs[:4], Hq, Hkv, dtype.__name__, way, s.kernel(), flush=True)
    assert s.kernel().startswith(kernel)
    out = torch_dev.full((s.T, Hq, D), 7.0, dtype=s.d["q"].dtype, device="cuda")
    got = s.run(ops, out)
    assert got is out
    s.check(out, np.full((s.T, Hq, D), 7.0))  # (rows behind the last sequence as they were)


BOTH = pytest.mark.parametrize("width", [None, WIDE])  # 16 rows a workgroup, 128


@BOTH
@pytest.mark.parametrize("way", ["chain", "flat", "odd"])
def test_attention_shapes_of_trees(torch_dev, ops, way, width):
    s = Trees([(40, 100), (64, 64), (129, 400)], 8, 2, way, width=width).dev(torch_dev)
    assert (s.kernel() == "128 even") == (width == WIDE)
    s.check(s.run(ops))


@BOTH
@pytest.mark.parametrize("prior", list(range(0, 70, 3)))
def test_attention_where_the_tree_begins(torch_dev, ops, prior, width):
    """Trees that begin anywhere within a tile of 64 tokens and go over its end."""
    s = Trees([(67, prior + 67), (5, prior + 5)], 4, 2, "bits", seed=prior,
              width=width).dev(torch_dev)
    assert (s.kernel() == "128 even") == (width == WIDE)
    s.check(s.run(ops))


@BOTH
def test_attention_chain_is_causal(torch_dev, ops, width):
    """A tree that is a chain gives what attn_kv4 gives for the same rows."""
    torch = torch_dev
    s = Trees([(30, 333), (27, 64)], 8, 2, "chain", width=width).dev(torch)
    a = s.run(ops).cpu().numpy()
    b = ops.attn_kv4(s.d["q"], *s.args(), cu_q=s.d["cu"]).cpu().numpy()
    np.testing.assert_allclose(a, b, rtol=0, atol=2e-5 * np.abs(b).max())


def test_attention_without_cu(torch_dev, ops):
    s = Trees([(1, 5), (1, 0), (1, 700), (1, 1)], 8, 4, "bits", cu=False).dev(torch_dev)
    s.check(s.run(ops))


@BOTH
def test_attention_more_rows_than_tokens(torch_dev, ops, width):
    s = Trees([(20, 12), (70, 3), (8, 8), (90, 66)], 8, 2, "bits", width=width).dev(torch_dev)
    s.check(s.run(ops))


@BOTH
def test_attention_fewer_words_than_nodes(torch_dev, ops, width):
    s = Trees([(140, 300), (3, 10)], 4, 2, "bits", words=1, width=width).dev(torch_dev)
    s.check(s.run(ops))


@BOTH
def test_attention_absent_pages(torch_dev, ops, width):
    """Pages outside the pool, in front of the tree, within it, and all of a sequence's."""
    s = Trees([(40, 300), (33, 100), (16, 90), (66, 500)], 16, 1, "bits", width=width)
    s.tables[0, [2, 17]] = [-1, s.nb]
    s.tables[1, :4] = -1
    s.tables[2] = 10 ** 9
    s.tables[3, 20:32] = -5
    s.dev(torch_dev)
    s.check(s.run(ops))


def test_attention_strides(torch_dev, ops):
    """Queries in a wider projection, masks in wider rows, outputs in every other row."""
    torch = torch_dev
    s = Trees([(26, 90), (3, 3)], 4, 2).dev(torch)
    q = torch.randn((s.T, 4 * D + 300), device="cuda")  # (2-D, as out)
    q[:, 77:77 + 4 * D] = s.d["q"].reshape(s.T, -1)
    mask = torch.full((s.T, 5), -1, dtype=torch.int64, device="cuda")
    mask[:, 2:3] = s.d["mask"]
    out = torch.full((2 * s.T, 4 * D), 3.0, device="cuda")
    s.run(ops, out=out[::2], q=q[:, 77:77 + 4 * D], mask=mask[:, 2:3])
    s.check(out[::2])
    assert (out[1::2] == 3).all()


@BOTH
def test_attention_large_scales(torch_dev, ops, width):
    """Rows of the cache whose scales are the largest and the smallest ones stand where the mask
    does not look."""
    s = Trees([(40, 200), (64, 64)], 8, 1, "bits", width=width)
    for b, (n, c) in enumerate(s.seqs):
        rows = s.mask[s.cu[b]:s.cu[b + 1]]
        rows &= ~np.uint64(0b101000)  # nodes 3 and 5
        for j in (3, 5):
            t = c - n + j
            for a, v in zip(s.pools[2:], (252, 255)):
                a[s.tables[b, t // PAGE], :, :, t % PAGE] = v
    s.dev(torch_dev)
    s.check(s.run(ops))


@pytest.mark.parametrize("order", ["rising", "falling", "any"])
def test_attention_values_of_every_size(torch_dev, ops, order):
    """Scales of values from the smallest to the largest, fp32, 128 rows a workgroup: what fp16 does
    not hold as it is moves by a power of two."""
    s = Trees([(40, 300), (33, 100), (9, 700)], 8, 1, "bits", width=WIDE)
    assert s.kernel() == "128 even"
    for b, (n, c) in enumerate(s.seqs):
        e = s.rng.integers(1, 250, c)
        e = np.sort(e) if order == "rising" else -np.sort(-e) if order == "falling" else e
        for t in range(c):
            at = (s.tables[b, t // PAGE], slice(None), slice(None), t % PAGE)
            s.pools[3][at] = e[t] - s.rng.integers(0, 2, 4)
    s.dev(torch_dev)
    s.check(s.run(ops))


@pytest.mark.parametrize("scale", [20, 100, 150, 220])
def test_attention_keys_of_every_size(torch_dev, ops, scale):
    """Scales of keys far from 1, and queries that bring the scores back, fp32."""
    s = Trees([(40, 300), (33, 100)], 8, 1, "bits", width=WIDE)
    s.pools[2][:] = scale + s.rng.integers(-2, 3, s.pools[2].shape)
    s.q = (s.q * 2.0 ** (126 - scale)).astype(np.float32)
    s.dev(torch_dev)
    s.check(s.run(ops))


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("seqs,Hkv,shares", [([(140, 3000), (60, 2500)], 1, 36),
                                             ([(140, 3000), (60, 2500)], 8, 21),
                                             ([(100, 2000)] * 7, 2, 5)])
def test_attention_joins(torch_dev, ops, seqs, Hkv, shares, dtype):
    """128 rows a workgroup, over 1024 rows times heads: the records of a row's head come from one
    group of lanes up to 16 shares a unit, from 8 beyond."""
    Hq = 8 * Hkv if Hkv < 8 else Hkv
    s = Trees(seqs, Hq, Hkv, "tree", dtype=dtype, width=WIDE).dev(torch_dev)
    assert s.kernel() == "128 even" and s.T * Hq > 1024
    assert 512 // ((s.T * Hq // Hkv // 128 + len(seqs)) * Hkv) == shares
    s.check(s.run(ops))


@pytest.mark.parametrize("dtype,count,way", [(np.float16, 60, "tree"), (np.float16, 60, "bits"),
                                             (np.float32, 190, "bits"), (np.float32, 190, "odd")])
def test_attention_of_many_trees(torch_dev, ops, dtype, count, way):
    """128 rows a workgroup, a workgroup for all tokens: padding slots, trees without nodes, nodes in
    front of the cache, absent pages, rows behind the last sequence."""
    rng = np.random.default_rng(count)
    seqs = [(int(rng.integers(30, 65)), int(rng.integers(64, 330))) for _ in range(count)]
    seqs[:8] = [(50, 0), (0, 7), (70, 60), (1, 1), (64, 64), (33, -3), (65, 320), (2, 17)]
    s = Trees(seqs, 8, 2 if count < 100 else 1, way, dtype=dtype, tail=3, layers=1)
    s.tables[4, 1], s.tables[9, 0], s.tables[10] = -1, s.nb, -7
    s.dev(torch_dev)
    print("many trees", dtype.__name__, count, way, s.kernel(), flush=True)
    assert s.kernel() == "128"
    out = torch_dev.full((s.T, 8, D), 7.0, dtype=s.d["q"].dtype, device="cuda")
    s.check(s.run(ops, out), np.full((s.T, 8, D), 7.0))


@pytest.mark.parametrize("seqs,Hq,kernel,width", [
    ([(1 + i % 2, 200 + 40 * i) for i in range(70)], 2, "4 even", None),
    ([(6, 300 + 30 * i) for i in range(65)], 8, "16 even", None),
    ([(6, 300 + 30 * i) for i in range(64)], 8, "16 even", None),
    ([(16 + i % 5, 30 + 7 * i) for i in range(70)], 8, "128 even", WIDE)])
def test_attention_of_over_64_trees(torch_dev, ops, seqs, Hq, kernel, width):
    """Steps dealt evenly over more sequences than a wave has lanes, some of them padding."""
    seqs = list(seqs)
    seqs[3], seqs[20], seqs[-1] = (5, 0), (0, 9), (9, 4)
    s = Trees(seqs, Hq, 2, "tree", width=width, tail=2, layers=1).dev(torch_dev)
    print("trees", len(seqs), s.kernel(), flush=True)
    assert s.kernel() == kernel
    out = torch_dev.full((s.T, Hq, D), 7.0, dtype=s.d["q"].dtype, device="cuda")
    s.check(s.run(ops, out), np.full((s.T, Hq, D), 7.0))


@BOTH
def test_attention_queries_that_are_not_finite(torch_dev, ops, width):
    """A row with an infinity or NaN in its query is NaN where it sees a token, and no other row is
    touched."""
    s = Trees([(40, 300), (64, 64)], 8, 1, "tree", width=width).dev(torch_dev)
    want = s.run(ops).cpu().numpy()
    bad = [(3, 0, 5, np.inf), (17, 7, 127, np.nan), (60, 2, 64, -np.inf)]
    for r, h, d, v in bad:
        s.d["q"][r, h, d] = v
    got = s.run(ops).cpu().numpy()
    for r, h, _, _ in bad:
        assert np.isnan(got[r, h]).all(), (r, h)
        got[r, h] = want[r, h]
    np.testing.assert_array_equal(got, want)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_attention_over_many_pages(torch_dev, ops, dtype):
    """Shares of more pages than a workgroup has page numbers at a time (1024); a few rows looked
    at."""
    s = Trees([(130, 64400)], 128, 8, "tree", dtype=dtype, layers=1).dev(torch_dev)
    assert s.kernel() == "128 even"
    n, c = s.seqs[0]
    assert (n * 16 // 128 + 1) * 8 * (c // 64) // 512 > 1024 // 4
    got = s.run(ops).cpu().numpy()
    half = dtype == np.float16
    t = np.arange(c)
    at = (s.tables[0, t // PAGE], 0)
    for r, h in ((0, 0), (63, 17), (64, 127), (129, 64), (100, 90)):
        K, V = (plain.values(a[at[0], 0, h // 16, t % PAGE], b[at[0], 0, h // 16, t % PAGE])
                for a, b in ((s.pools[0], s.pools[2]), (s.pools[1], s.pools[3])))
        node = t - (c - n)
        bit = (s.mask[r, np.clip(node // 64, 0, 2)] >> (node % 64).astype(np.uint64)) & np.uint64(1)
        see = (node < 0) | (bit == 1)
        want, tol = plain.attention_row(s.q[r, h].astype(np.float64) / np.sqrt(D), K[see], V[see],
                                        np.abs(V).max(), 2.0 ** -21,
                                        2.0 ** -11 if half else 2.0 ** -21)
        tol = tol + float(np.finfo(dtype).eps) / 2 * (np.abs(want) + tol) + 2.0 ** -25 * half
        assert (np.abs(got[r, h] - want) <= tol).all(), (r, h)


# ------------------------------------------------------------------ accept ----

def drafts(rng, parents, agree=0.8):
    """Tokens of a few kinds, and targets that often are a child's."""
    T = len(parents)
    tokens, target = rng.integers(0, 5, T), rng.integers(0, 5, T)
    return tokens.astype(np.int32), np.where(rng.random(T) < agree, target, -9).astype(np.int32)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("seqs,layers,Hkv,way", [
    ([(1, 1)], 1, 1, "tree"), ([(26, 300)], 3, 5, "tree"),
    ([(5, 9), (0, 3), (64, 64), (3, 0), (17, 100), (9, 4)], 2, 2, "tree"),
    ([(40, 41), (40, 57), (33, 50)], 1, 9, "chain"), ([(130, 200), (100, 333)], 2, 17, "chain"),
    ([(60, 100), (200, 201)], 2, 3, "odd"), ([(2, 18 + i) for i in range(70)], 2, 1, "chain")])
def test_accept(torch_dev, ops, seqs, layers, Hkv, way, int8):
    torch, rng = torch_dev, np.random.default_rng(len(seqs) + layers)
    print("accept", seqs[:4], layers, Hkv, way, int8, flush=True)
    s = Setup(seqs, Hkv, Hkv, layers=layers, rope=False, tail=2)
    parents = forest(rng, seqs, 2, way)
    tokens, target = drafts(rng, parents)
    if way == "chain":  # long paths, broken somewhere
        target[:-1] = tokens[1:]
        target[rng.integers(0, len(target), 2)] = -9
    pools = s.pools
    if int8:
        shape = s.pools[0].shape[:4]
        pools = [rng.integers(-128, 128, shape + (128,)).astype(np.int8) for _ in range(2)] + \
            [rng.random(shape).astype(np.float32) for _ in range(2)]
    s.tables[0, -1] = s.nb if len(seqs) > 60 else s.tables[0, -1]
    put = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    dev = [put(a.copy()) for a in pools]
    most = max(n for n, _ in seqs)
    for m in (most, max(1, most // 3)):
        ctx = put(s.ctx)
        got = ops.tree_accept(put(parents), put(tokens), put(target), *dev, put(s.tables), ctx, m,
                              cu_q=put(s.cu))
        want = plain.tree_accept(parents, tokens, target, pools, s.tables, s.ctx, s.cu, m)
        for a, b in zip(got, want):
            np.testing.assert_array_equal(a.cpu().numpy(), b)
        for a, b in zip(dev, pools):
            np.testing.assert_array_equal(a.cpu().numpy(), b)
        np.testing.assert_array_equal(ctx.cpu().numpy(), s.ctx)


def test_accept_without_cu(torch_dev, ops):
    torch = torch_dev
    s = Setup([(1, 5), (1, 0), (1, 700)], 2, 2, rope=False, cu=False).dev(torch)
    z = torch.arange(3, dtype=torch.int32).cuda()
    got = ops.tree_accept(z - 1, z, z + 40, *s.dp, s.d["tables"], s.d["ctx"], 2)
    assert [a.cpu().tolist() for a in got] == [[[0, -1], [-1, -1], [0, -1]], [1, 0, 1],
                                               [40, -1, 42], [5, 0, 700]]
    for a, b in zip(s.pools, s.dp):
        np.testing.assert_array_equal(a, b.cpu().numpy())


# ------------------------------------------------------- streams and graphs ----

def test_captured_steps(torch_dev, ops):
    """Plan, attention and acceptance captured on a side stream, replayed with other trees,
    lengths and pages in between and eager work beside them: each replay as the eager calls."""
    torch = torch_dev
    s = Trees([(26, 200), (64, 300), (5, 0), (30, 64)], 8, 2).dev(torch)
    d, rng = s.d, np.random.default_rng(3)
    parents = torch.from_numpy(s.parents).cuda()
    tokens = torch.zeros_like(parents)
    target = torch.zeros_like(parents)
    start = [a.clone() for a in s.dp]

    def step():
        mask, at = ops.tree_plan(parents, d["ctx"], 64, cu_q=d["cu"])
        o = ops.attn_tree_kv4(d["q"], mask, *s.args(), cu_q=d["cu"])
        got = ops.tree_accept(parents, tokens, target, *s.dp, d["tables"], d["ctx"], 64,
                              cu_q=d["cu"])
        return [mask, at, o, *got]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step()
    for i in range(4):
        parents.copy_(torch.from_numpy(forest(rng, s.seqs)))
        a, b = drafts(rng, s.parents, 0.9)
        tokens.copy_(torch.from_numpy(a // 3))
        target.copy_(torch.from_numpy(b // 3))
        d["ctx"].copy_(torch.tensor([200 - i, 300 - 7 * i, 0, 64], dtype=torch.int32))
        for x, y in zip(s.dp, start):
            x.copy_(y)
        want = [t.clone() for t in step()]
        pools = [t.clone() for t in s.dp]
        for x, y in zip(s.dp, start):
            x.copy_(y)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(out + s.dp, want + pools):
            assert torch.equal(x, y), i


def test_two_captured_calls_share_nothing(torch_dev, ops):
    """Two captured calls with workspaces, replayed on two streams at once."""
    torch = torch_dev
    sets = [Trees([(26, 3000 + i)], 20, 5, seed=i).dev(torch) for i in range(2)]
    want = [s.run(ops).clone() for s in sets]
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for s, st in zip(sets, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            outs.append(s.run(ops))
        graphs.append(g)
    for _ in range(5):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b)
