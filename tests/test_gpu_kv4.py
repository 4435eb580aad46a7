"""The paged cache in 4 bits on the GPU: append, read and attention against the plain forms in
64 bits. Pools bit for bit (a value next to the border of two codes goes where its exact value
lies); attention within the rounding of fp32 sums, counted per output in kv4_plain.attention,
and half a step of the output's type."""
import numpy as np
import pytest

from tests import kv4_plain as plain

pytestmark = pytest.mark.gpu
D, PAGE = 128, 16


@pytest.fixture(scope="module")
def torch_dev():
    import torch
    assert torch.cuda.is_available(), "GPU test needs a visible GPU"
    from tenzo_amd import _lib
    _lib.load()
    return torch


@pytest.fixture(scope="module")
def ops(torch_dev):
    from tenzo_amd import ops
    return ops


class Setup:
    """Sequences of (rows, length) over a pool whose slots that no sequence holds have scales of
    2^125 and of no meaning."""

    def __init__(self, seqs, Hq, Hkv, layers=2, seed=0, extra=3, width=None, cu=True, rope=True,
                 dtype=np.float32, tail=0, fill=True):
        rng = self.rng = np.random.default_rng(seed)
        self.seqs, self.Hq, self.Hkv, self.layer = seqs, Hq, Hkv, layers - 1
        pages = [max(0, -(-c // PAGE)) for _, c in seqs]
        self.nb = sum(pages) + extra
        width = width or max(pages + [1])
        self.tables = np.full((len(seqs), width), -1, np.int32)
        perm = rng.permutation(self.nb).astype(np.int32)
        at = 0
        for b, n in enumerate(pages):
            self.tables[b, :n] = perm[at:at + n][:width]
            at += n
        self.ctx = np.array([c for _, c in seqs], np.int32)
        self.cu = np.concatenate([[0], np.cumsum([n for n, _ in seqs])]).astype(np.int32) \
            if cu else None
        self.T = sum(n for n, _ in seqs) + tail
        shape = (self.nb, layers, Hkv, PAGE)
        codes = [rng.integers(0, 256, shape + (64,), dtype=np.uint8) for _ in range(2)]
        scales = [rng.choice(np.array([252, 252, 255], np.uint8), shape + (4,)) for _ in range(2)]
        if fill:
            for b, (_, c) in enumerate(seqs):
                for t0 in range(0, min(max(c, 0), width * PAGE), PAGE):
                    n = min(PAGE, c - t0)
                    for s in scales:
                        s[self.tables[b, t0 // PAGE], :, :, :n] = rng.integers(
                            124, 129, (layers, Hkv, n, 4))
        self.pools = [*codes, *scales]
        self.rope = rng.standard_normal((width * PAGE, 64)) if rope else None
        if rope:
            self.rope = np.concatenate([np.cos(self.rope), np.sin(self.rope)], 1).astype(
                np.float32)
        self.dtype = dtype
        self.q = (1.5 * rng.standard_normal((self.T, Hq, D))).astype(dtype)
        self.k = (2 * rng.standard_normal((self.T, Hkv, D))).astype(dtype)
        self.v = rng.standard_normal((self.T, Hkv, D)).astype(dtype)

    def dev(self, torch):
        put = lambda a: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
        self.d = {n: put(getattr(self, n)) for n in ("tables", "ctx", "cu", "rope", "q", "k", "v")}
        self.dp = [put(a) for a in self.pools]
        return self

    def args(self):
        return (*self.dp, self.d["tables"], self.d["ctx"], self.layer)

    def opts(self):
        return {"rope_cs": self.d["rope"], "cu_q": self.d["cu"]}

    def check_attention(self, out, start=None):
        want = np.zeros((self.T, self.Hq, D)) if start is None else start.astype(np.float64)
        # (queries and weights are held to 16 bits in fp16 calls, to 22 in fp32 ones: 2^-15 and
        # 2^-21 for the two of them)
        half = self.dtype == np.float16
        want, tol = plain.attention(self.q, self.pools, self.tables, self.ctx, self.layer,
                                    self.rope, self.cu, want, 2.0 ** -15 if half else 2.0 ** -21)
        got = out.reshape(want.shape).astype(np.float64)
        # half a step of the type: relative, and below its smallest normal number 2^-14 (fp16)
        # half of the constant step 2^-24 that its numbers have there
        step = np.finfo(self.dtype)
        tol = tol + float(step.eps) / 2 * (np.abs(want) + tol) + float(step.smallest_subnormal) / 2
        finite = bool(np.isfinite(got).all())
        worst = float(np.max(np.abs(got - want) / np.where(tol > 0, tol, 1e-300)))
        assert finite and worst <= 1, worst


def pools_equal(s, got):
    for a, b in zip(s.pools, got):
        np.testing.assert_array_equal(a, b.cpu().numpy())


# ------------------------------------------------------------------ append ----

@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("seqs,cu,Hkv", [
    ([(1, 1)], False, 1), ([(1, 16)], False, 5), ([(1, 17), (1, 0), (1, 300)], False, 8),
    ([(3, 3), (1, 40), (0, 9), (17, 33), (50, 50)], True, 5), ([(5, 3), (2, 0)], True, 2),
    ([(1, i % 37) for i in range(100)], False, 3), ([(1, i % 37) for i in range(70)], True, 1)])
def test_append_and_read(torch_dev, ops, seqs, cu, Hkv, dtype):
    """Pools bit for bit, rows of other layers, of padding and behind the last sequence left as
    they were; read back as the values that they stand for."""
    s = Setup(seqs, Hkv, Hkv, cu=cu, dtype=dtype, tail=2 if cu else 0, fill=False).dev(torch_dev)
    print("append", seqs[:4], Hkv, dtype.__name__, flush=True)
    ops.kv4_append(s.d["k"], s.d["v"], *s.args(), **s.opts())
    k, v = ops.kv4_read(*s.args(), rows=s.T, cu_q=s.d["cu"], dtype=s.d["k"].dtype)
    plain.append(s.k, s.v, s.pools, s.tables, s.ctx, s.layer, s.rope, s.cu)
    pools_equal(s, s.dp)
    at = plain.places(s.T, s.tables, s.ctx, s.cu, s.tables.shape[1] * PAGE)
    for got, codes, scales in ((k, s.pools[0], s.pools[2]), (v, s.pools[1], s.pools[3])):
        want = np.zeros((s.T, Hkv, D))
        for r, w in enumerate(at):
            if w:
                p = (s.tables[w[0], w[1] // PAGE], s.layer, slice(None), w[1] % PAGE)
                want[r] = plain.values(codes[p], scales[p])
        np.testing.assert_array_equal(got.cpu().numpy(), want.astype(dtype))


def test_append_borders(torch_dev, ops):
    """Values on and beside the borders of two codes and of two scales, signed zeros, groups of
    zeros, of the smallest and the largest numbers, NaN and infinities."""
    torch = torch_dev
    rows = []
    near = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0]
    for e in (-40, 0, 60):
        for top in (4.0, 6.0, 7.0, np.nextafter(np.float32(7), np.float32(8)), 7.5):
            x = []
            for b in near:
                b = np.float32(b)
                x += [b, np.nextafter(b, np.float32(0)), np.nextafter(b, np.float32(9))]
            x = np.array([-v if i % 2 else v for i, v in enumerate(x)] + [0.0, -0.0], np.float32)
            x = np.clip(x, -np.float32(top), np.float32(top))
            rows.append(np.ldexp(np.concatenate([x, [top], np.zeros(32 - len(x) - 1)]), e))
    rows += [np.zeros(32), -np.zeros(32), np.full(32, 1e-45), np.full(32, 2.0 ** -126),
             np.r_[np.full(31, 2.0 ** -130), 3e-38], np.full(32, 3.4e38), np.full(32, 1.75 * 2.0 ** 127),
             np.r_[np.nan, np.ones(31)], np.r_[np.inf, -np.inf, np.nan, np.ones(29)],
             np.full(32, np.nan)]
    while len(rows) % 4:
        rows.append(np.ones(32))
    x = np.stack(rows).astype(np.float32).reshape(-1, 1, D)
    s = Setup([(len(x), len(x))], 1, 1, rope=False).dev(torch)
    s.k, s.v = x, x[::-1].copy()
    ops.kv4_append(torch.from_numpy(s.k).cuda(), torch.from_numpy(s.v).cuda(), *s.args(),
                   cu_q=s.d["cu"])
    plain.append(s.k, s.v, s.pools, s.tables, s.ctx, s.layer, None, s.cu)
    pools_equal(s, s.dp)


def test_append_rotated_borders(torch_dev, ops):
    """Rotations whose exact result lies within a 64-bit step of a border: an fp32 rounding of
    the rotated value would meet it from the wrong side."""
    torch = torch_dev
    rng = np.random.default_rng(4)
    T = 400
    s = Setup([(T, T)], 1, 1, seed=9)
    ang = rng.uniform(0.1, 1.4, (s.tables.shape[1] * PAGE, 64))
    s.rope = np.concatenate([np.cos(ang), np.sin(ang)], 1).astype(np.float32)
    # x0 c - x1 s next to a border b: x0 = fp32((b + x1 s) / c), many x1 tried for the nearest
    for r in range(T):
        c, sn = s.rope[r, :64].astype(np.float64), s.rope[r, 64:].astype(np.float64)
        b = rng.choice([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], 64)
        x1 = rng.uniform(0.5, 1, (200, 64)).astype(np.float32).astype(np.float64)
        x0 = ((b + x1 * sn) / c).astype(np.float32).astype(np.float64)
        off = np.abs(x0 * c - x1 * sn - b)
        best = np.where(off == 0, 1, off).argmin(0)
        s.k[r, 0, :64] = x0[best, np.arange(64)]
        s.k[r, 0, 64:] = x1[best, np.arange(64)]
        s.k[r, 0, [0, 32]] = 6.0 / c[[0, 32]]
        s.k[r, 0, [64, 96]] = 0.0
    s.dev(torch)
    ops.kv4_append(s.d["k"], s.d["v"], *s.args(), **s.opts())
    plain.append(s.k, s.v, s.pools, s.tables, s.ctx, s.layer, s.rope, s.cu)
    pools_equal(s, s.dp)


def test_append_rotated_range(torch_dev, ops):
    """Rotated keys of every magnitude that fp32 has, its subnormal numbers among them, alone and
    beside zeros."""
    torch = torch_dev
    T = 270
    s = Setup([(T, T)], 1, 1, seed=11)
    s.k = np.ldexp(s.rng.uniform(-2, 2, (T, 1, D)), np.arange(-148, T - 148)[:, None, None]).astype(
        np.float32)
    s.k[::3, 0, 5::9] = 0
    s.dev(torch)
    ops.kv4_append(s.d["k"], s.d["v"], *s.args(), **s.opts())
    plain.append(s.k, s.v, s.pools, s.tables, s.ctx, s.layer, s.rope, s.cu)
    pools_equal(s, s.dp)


def test_append_strides_and_bad_pages(torch_dev, ops):
    """Keys and values as slices of a fused projection at an odd stride and offset; pages out of
    the pool, lengths above the tables' and the rotation's rows: nothing is written there."""
    torch = torch_dev
    s = Setup([(6, 20), (2, 40), (3, 200), (2, 33), (1, 75)], 2, 2, width=5, seed=3, fill=False)
    s.tables[0, 1] = s.nb
    s.tables[1, 2] = -7
    s.tables[3, 2] = 2 ** 31 - 1
    s.rope = s.rope[:70]
    s.dev(torch)
    wide = torch.randn((s.T, 1 + 7 * D + 3), device="cuda")
    k, v = wide[:, 1:1 + 2 * D], wide[:, 1 + 3 * D:1 + 5 * D]
    ops.kv4_append(k, v, *s.args(), **s.opts())
    plain.append(k.cpu().numpy().reshape(-1, 2, D), v.cpu().numpy().reshape(-1, 2, D), s.pools,
                 s.tables, s.ctx, s.layer, s.rope, s.cu)
    pools_equal(s, s.dp)
    got, _ = ops.kv4_read(*s.args(), rows=s.T, cu_q=s.d["cu"])
    assert got[[0, 1, 11]].any(-1).all() and not got[2:11].any() and not got[12].any()


# --------------------------------------------------------------- attention ----

HEADS = [(4, 4), (4, 2), (20, 5), (6, 2), (5, 1), (7, 1), (8, 1), (32, 2)]


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("Hq,Hkv", HEADS)
def test_attention_token(torch_dev, ops, Hq, Hkv, dtype):
    """One token a sequence: lengths 1, around pages and tiles, padding slots."""
    lens = [1, 2, 15, 16, 17, 0, 31, 33, 63, 64, 65, 100, -3, 127, 128, 129, 255, 256, 257, 300]
    s = Setup([(1, c) for c in lens], Hq, Hkv, cu=False, dtype=dtype, seed=Hq).dev(torch_dev)
    print("attn token", Hq, Hkv, dtype.__name__, flush=True)
    s.check_attention(ops.attn_kv4(s.d["q"], *s.args(), **s.opts()).cpu().numpy())


@pytest.mark.parametrize("ctx", [1000, 4097, 9001, 30000])
@pytest.mark.parametrize("Hq,Hkv,dtype", [(4, 1, np.float32), (8, 1, np.float16),
                                          (3, 1, np.float32)])
def test_attention_long(torch_dev, ops, ctx, Hq, Hkv, dtype):
    """The long axis split over workgroups, with a short sequence beside."""
    s = Setup([(1, ctx), (1, 5)], Hq, Hkv, layers=1, cu=False, dtype=dtype, seed=ctx).dev(
        torch_dev)
    print("attn long", ctx, Hq, flush=True)
    s.check_attention(ops.attn_kv4(s.d["q"], *s.args(), **s.opts()).cpu().numpy())


@pytest.mark.parametrize("Hq,Hkv,dtype", [(4, 1, np.float32), (8, 1, np.float16),
                                          (12, 1, np.float32), (8, 2, np.float16)])
def test_attention_ragged_batch(torch_dev, ops, Hq, Hkv, dtype):
    """Lengths from 0 to 9000 side by side: workgroups that end a sequence, take others whole
    and begin the next; several rows a sequence, more of them than their length holds."""
    rng = np.random.default_rng(Hq)
    lens = [9000, 0, 256, 257, 1, 512, 0, 700, 5000, 255, 3000, 0] + list(rng.integers(1, 400, 20))
    s = Setup([(1, int(c)) for c in lens], Hq, Hkv, layers=1, cu=False, dtype=dtype,
              seed=Hq).dev(torch_dev)
    print("attn ragged", Hq, Hkv, flush=True)
    s.check_attention(ops.attn_kv4(s.d["q"], *s.args(), **s.opts()).cpu().numpy())
    rows = [int(n) for n in rng.integers(0, 4, len(lens))]
    s = Setup(list(zip(rows, map(int, lens))), Hq, Hkv, layers=1, dtype=dtype, seed=Hq + 1,
              tail=2).dev(torch_dev)
    start = np.full((s.T, Hq, D), 7.0, dtype)
    out = torch_dev.from_numpy(start).cuda()
    ops.attn_kv4(s.d["q"], *s.args(), **s.opts(), out=out)
    s.check_attention(out.cpu().numpy(), start)


def test_attention_many_pages(torch_dev, ops):
    """More page numbers than a workgroup keeps at a time: one sequence of 17000 tokens among
    slots that are empty but fill the GPU."""
    lens = [0] * 450
    lens[77], lens[300] = 17000, 16500
    s = Setup([(1, c) for c in lens], 16, 4, layers=1, cu=False, seed=5).dev(torch_dev)
    print("attn many pages", flush=True)
    s.check_attention(ops.attn_kv4(s.d["q"], *s.args(), **s.opts()).cpu().numpy())


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("Hq,Hkv,seqs", [
    (4, 1, [(2, 2), (3, 40), (1, 65)]), (8, 1, [(7, 100), (5, 5), (0, 30), (9, 2)]),
    (5, 1, [(33, 33), (1, 1), (64, 200)]), (4, 4, [(70, 70), (130, 131), (16, 300)]),
    (20, 5, [(40, 90), (17, 17), (3, 0)]), (2, 1, [(300, 310)]), (16, 1, [(20, 64), (4, 4)]),
    (4, 1, [(200, 230), (1, 1), (130, 100), (0, 0), (97, 2000)]), (3, 1, [(150, 150), (260, 700)]),
    (8, 2, [(64, 1000), (65, 65)])])
def test_attention_rows(torch_dev, ops, Hq, Hkv, seqs, dtype):
    """Several rows a sequence, each up to its own position; rows before position 0, empty
    sequences, and rows behind the last sequence that stay as they were."""
    torch = torch_dev
    s = Setup(seqs, Hq, Hkv, dtype=dtype, seed=len(seqs) + Hq, tail=3).dev(torch)
    print("attn rows", Hq, Hkv, seqs, dtype.__name__, flush=True)
    start = np.full((s.T, Hq, D), 7.0, dtype)
    out = torch.from_numpy(start).cuda().reshape(s.T, Hq * D)
    got = ops.attn_kv4(s.d["q"].reshape(s.T, -1), *s.args(), **s.opts(), out=out)
    assert got is out
    s.check_attention(out.cpu().numpy(), start)


@pytest.mark.parametrize("n", [1, 3, 40])
def test_attention_peaked_and_flat(torch_dev, ops, n):
    """Scores far apart (weights that underflow, the largest first, last or in the middle),
    all equal (a zero query), and a channel hundreds of times the others."""
    torch = torch_dev
    s = Setup([(n, 333)] * 4, 4, 2, seed=n)
    c = np.array([0, n, 2 * n, 3 * n, 4 * n])
    s.q[c[0]:c[1]] *= 60
    s.q[c[1]:c[2]] = 0
    s.q[c[2]:c[3], :, 7] *= 400
    s.q[c[3]:c[4]] *= 1e-20
    s.dev(torch)
    s.check_attention(ops.attn_kv4(s.d["q"], *s.args(), **s.opts()).cpu().numpy())


@pytest.mark.parametrize("kind", ["keys", "values", "small", "large", "rising", "falling",
                                  "zeros", "one_group"])
@pytest.mark.parametrize("n,Hq", [(1, 4), (1, 12), (5, 8), (70, 4)])
def test_attention_scale_range(torch_dev, ops, kind, n, Hq):
    """Scales that fp16 does not span: tokens and groups 2^60 apart, everything tiny or large,
    growing and shrinking along the sequence, groups and tokens of zeros with any scale."""
    s = Setup([(n, 200), (n, 70)], Hq, 1, layers=1, seed=n)
    rng = np.random.default_rng(n + Hq)
    ks, vs = s.pools[2], s.pools[3]
    t = np.empty(s.nb * PAGE, np.int64)  # a slot's position
    for b in range(2):
        for p in range(s.tables.shape[1]):
            if s.tables[b, p] >= 0:
                t[s.tables[b, p] * PAGE:][:PAGE] = np.arange(PAGE) + p * PAGE
    t = t.reshape(s.nb, 1, 1, PAGE, 1)
    some = np.broadcast_to(rng.random(ks.shape[:-1] + (1,)) < 0.1, ks.shape)
    if kind == "keys":
        s.q *= 1e-8
        ks[some] = rng.integers(60, 160, some.sum())
    elif kind == "values":
        vs[some] = rng.integers(60, 190, some.sum())
    elif kind == "small":
        vs[:], ks[:] = 127 - 90, 127 - 60
    elif kind == "large":
        vs[:], ks[:] = 127 + 80, 127 + 60
        s.q *= 2.0 ** -60
    elif kind == "rising":
        vs[:] = 100 + t // 4
    elif kind == "falling":
        vs[:] = 160 - t // 4
        ks[:] = 127 - t % 30
    elif kind == "zeros":
        for c, e in ((s.pools[0], ks), (s.pools[1], vs)):
            c[rng.random(c.shape[:-1]) < 0.3] = 0x80  # zeros and negative zeros
            e[(c.reshape(*c.shape[:-1], 4, 16) & 0x77 == 0).all(-1)] = rng.choice([0, 1, 200, 255])
    else:
        ks[..., 2], vs[..., 1] = 127 - 35, 127 - 33
    for e in (ks, vs):
        for b, (_, c) in enumerate(s.seqs):
            if c % PAGE:
                e[s.tables[b, c // PAGE], :, :, c % PAGE:] = 252
    s.dev(torch_dev)
    print("attn scales", kind, n, Hq, flush=True)
    s.check_attention(ops.attn_kv4(s.d["q"], *s.args(), **s.opts()).cpu().numpy())


@pytest.mark.parametrize("n", [1, 2, 25])
def test_attention_bad_pages(torch_dev, ops, n):
    """Pages that the pool does not hold are absent: their tokens are left out, in the middle,
    at the end, and all of a sequence's (zeros); lengths that the tables do not hold: padding."""
    torch = torch_dev
    s = Setup([(n, 100), (n, 77), (n, 40), (n, 1000), (n, 64)], 8, 2, seed=n, width=8)
    s.tables[0, 3] = -1
    s.tables[1, 4] = s.nb
    s.tables[2, :] = [-5, 2 ** 31 - 1, -2 ** 31, 0, 0, 0, 0, 0]
    s.dev(torch)
    s.check_attention(ops.attn_kv4(s.d["q"], *s.args(), **s.opts()).cpu().numpy())


@pytest.mark.parametrize("rope", [True, False])
def test_attention_strides(torch_dev, ops, rope):
    """q a slice of a fused projection at an odd offset, out a slice of a wider buffer, the
    table a slice of a wider one."""
    torch = torch_dev
    s = Setup([(3, 50), (1, 20), (6, 6)], 8, 2, seed=1, rope=rope, width=4).dev(torch)
    wide = torch.randn((s.T, 3 + 12 * D), device="cuda")
    q = wide[:, 3:3 + 8 * D]
    s.q = q.cpu().numpy().reshape(s.T, 8, D)
    tables = torch.full((3, 11), -1, dtype=torch.int32, device="cuda")
    tables[:, 5:9] = s.d["tables"]
    s.d["tables"] = tables[:, 5:9]
    buf = torch.full((s.T, 5 + 8 * D), 3.0, device="cuda")
    ops.attn_kv4(q, *s.args(), **s.opts(), out=buf[:, 1:1 + 8 * D])
    s.check_attention(buf[:, 1:1 + 8 * D].cpu().numpy())
    assert (buf[:, 0] == 3).all() and (buf[:, 1 + 8 * D:] == 3).all()


def test_attention_rope_shorter_than_tables(torch_dev, ops):
    torch = torch_dev
    s = Setup([(2, 60), (2, 61)], 4, 1, seed=1)
    s.rope = s.rope[:60]
    s.dev(torch)
    s.check_attention(ops.attn_kv4(s.d["q"], *s.args(), **s.opts()).cpu().numpy())


def test_offsets_past_32_bits(torch_dev, ops):
    """Pools of more than 4 GiB of codes each, the sequence in their last pages."""
    torch = torch_dev
    layers, Hkv = 30, 8
    nb = (1 << 32) // (layers * Hkv * 1024) + 40
    s = Setup([(5, 300)], 16, Hkv, layers=1, seed=2).dev(torch)
    s.layer = layers - 1
    dp = ops.kv4_pool(nb, layers, Hkv)
    assert dp[0].numel() > 1 << 32
    at = torch.from_numpy(s.tables[0].astype(np.int64)).cuda()
    shift = nb - s.nb
    for big, small in zip(dp, s.dp):
        big[at + shift, s.layer] = small[at, 0]
    tables = s.d["tables"] + shift
    args = (*dp, tables, s.d["ctx"], s.layer)
    out = ops.attn_kv4(s.d["q"], *args, **s.opts()).cpu().numpy()
    ops.kv4_append(s.d["k"], s.d["v"], *args, **s.opts())
    s.layer = 0
    s.check_attention(out)
    plain.append(s.k, s.v, s.pools, s.tables, s.ctx, 0, s.rope, s.cu)
    for big, want in zip(dp, s.pools):
        np.testing.assert_array_equal(big[at + shift, layers - 1].cpu().numpy(),
                                      want[s.tables[0], 0])


def test_empty_calls(torch_dev, ops):
    torch = torch_dev
    s = Setup([(1, 5)], 4, 2).dev(torch)
    none = torch.empty((0, 4 * D), device="cuda")
    i = lambda *n: torch.zeros(n, dtype=torch.int32, device="cuda")  # noqa: E731
    pools = s.dp
    assert ops.attn_kv4(none, *pools, i(0, 3), i(0), 0).shape == (0, 4 * D)
    ops.kv4_append(none[:, :2 * D], none[:, :2 * D], *pools, i(0, 3), i(0), 0)
    out = torch.full((2, 4 * D), 5.0, device="cuda")
    ops.attn_kv4(torch.ones((2, 4 * D), device="cuda"), *pools, i(0, 3), i(0), 0, cu_q=i(1),
                 out=out)
    assert (out == 5).all()
    k, v = ops.kv4_read(*pools, i(0, 3), i(0), 0, rows=2, cu_q=i(1))
    assert k.shape == (2, 2, D) and not k.any() and not v.any()
    # a table without columns: every sequence is padding
    out = ops.attn_kv4(torch.ones((2, 4 * D), device="cuda"), *pools, i(2, 0), i(2) + 1, 0)
    assert not out.any()


def test_other_stream_and_graph(torch_dev, ops):
    """On a stream of the caller's, and captured into a graph (two of them alive at once) that
    is replayed on new contents of the same buffers, against eager calls between the replays."""
    torch = torch_dev
    sets = [Setup([(1, 3000), (1, 40), (1, 0)], 8, 2, cu=False, seed=1).dev(torch),
            Setup([(3, 500), (20, 64)], 4, 1, seed=2).dev(torch)]
    st = torch.cuda.Stream()
    graphs = []

    def step(s):
        ops.kv4_append(s.d["k"], s.d["v"], *s.args(), **s.opts())
        return ops.attn_kv4(s.d["q"], *s.args(), **s.opts())

    for s in sets:
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            first = step(s)
        st.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            out = step(s)
        graphs.append((g, out, first))
    for i in range(3):
        for s, (g, out, _) in zip(sets, graphs):
            gen = torch.Generator(device="cuda").manual_seed(i)
            for n in ("q", "k", "v"):
                s.d[n].copy_(torch.randn(s.d[n].shape, device="cuda", generator=gen))
            want = step(s)
            out.fill_(9)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
