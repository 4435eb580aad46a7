"""Beam search on the GPU: selection and reordering against the plain forms in 64 bits.
Beams and tokens equal, scores within an fp32 rounding (2^-24 relative) of the 64-bit ones plus
that of the sum of exponentials (1e-8 absolute: each exponential is off by at most 2 steps of
2^-24 with either sign, the log of the sum by the mean of those)."""
import numpy as np
import pytest

from tests import kv4_plain as plain

pytestmark = pytest.mark.gpu
PAGE = 16


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


def check(got, logits, scores, k):
    want = plain.beam_select(logits, scores, k)
    s, b, t = (a.cpu().numpy() for a in got)
    np.testing.assert_array_equal(b, want[1])
    np.testing.assert_array_equal(t, want[2])
    fin = np.isfinite(want[0])
    np.testing.assert_array_equal(s[~fin], want[0][~fin])
    assert (np.abs(s[fin] - want[0][fin]) <= 2.0 ** -24 * np.abs(want[0][fin]) + 3e-7).all()


def run(torch, ops, logits, scores, k):
    return ops.beam_select(torch.from_numpy(logits).cuda(), torch.from_numpy(scores).cuda(), k)


@pytest.mark.parametrize("B,W,V,k", [
    (1, 1, 1, 1), (1, 1, 7, 7), (2, 3, 5, 15), (1, 4, 1000, 8), (3, 2, 4095, 4), (2, 2, 4097, 5),
    (5, 8, 8192, 16), (1, 64, 257, 64), (2, 1, 32000, 64), (1, 5, 128256, 10), (4, 3, 50257, 6),
    (1, 16, 200003, 32), (70, 4, 1003, 8), (1, 1, 600000, 3)])
@pytest.mark.parametrize("scale", [0.1, 3.0, 40.0])
def test_select(torch_dev, ops, B, W, V, k, scale):
    print("beam", B, W, V, k, scale, flush=True)
    rng = np.random.default_rng(V + k)
    logits = (scale * rng.standard_normal((B, W, V))).astype(np.float32)
    scores = (-10 * rng.random((B, W))).astype(np.float32)
    check(run(torch_dev, ops, logits, scores, k), logits, scores, k)


@pytest.mark.parametrize("V", [33, 5000, 20000])
@pytest.mark.parametrize("kind", ["equal", "few", "rising", "falling", "steps", "same_beams",
                                  "first_step", "masked", "masked_row", "all_masked", "strange",
                                  "tiny", "block"])
def test_select_orders(torch_dev, ops, kind, V):
    """Equal logits (the lowest index first), orders of the vocabulary that put all of the best
    in one place, beams that do not count, masked tokens and beams, NaN and infinities."""
    rng = np.random.default_rng(V)
    B, W, k = 3, 4, 8
    x = rng.standard_normal((B, W, V)).astype(np.float32)
    s = (-5 * rng.random((B, W))).astype(np.float32)
    if kind == "equal":
        x[:], s[:] = 0.5, -1.0
    elif kind == "few":
        x = rng.integers(0, 3, x.shape).astype(np.float32)
        s = np.round(s)
    elif kind == "rising":
        x = np.sort(x, -1)
    elif kind == "falling":
        x = -np.sort(-x, -1)
    elif kind == "steps":
        x = np.floor(4 * x) / 4
    elif kind == "same_beams":
        x[:] = x[:, :1]
        s[:] = s[:, :1]
    elif kind == "first_step":
        x[:] = x[:, :1]
        s[:] = [0, -np.inf, -np.inf, -np.inf]
    elif kind == "masked":
        x[:] = -np.inf
        x[:, :, [3, 7, 20]] = [1.0, 0.5, 2.0]
        x[1] = -np.inf
        x[1, 2, 30] = 4.0
    elif kind == "masked_row":
        x[:, 1] = -np.inf
        x[:, 2, : V // 2] = np.finfo(np.float32).min
    elif kind == "all_masked":
        x[:] = -np.inf
        s[2] = -np.inf
    elif kind == "strange":
        x[:, :, 5] = np.nan
        x[:, 1, 9] = np.inf
        x[0, 0] = np.nan
        s[1, 2] = np.nan
        s[2, 3] = np.inf
    elif kind == "tiny":
        x *= 1e-30
    elif kind == "block":
        x[:, :, V // 3:V // 3 + 30] += 50
    check(run(torch_dev, ops, x, s, k), x, s, k)


@pytest.mark.parametrize("B,W,V,k", [(1, 16, 2723, 32), (3, 16, 70000, 32), (2, 32, 20000, 64),
                                     (2, 1, 50000, 64), (1, 64, 40000, 64), (2, 5, 90001, 64)])
@pytest.mark.parametrize("kind", ["alike", "one_beam", "first_step", "one_place"])
def test_select_many(torch_dev, ops, B, W, V, k, kind):
    """Many candidates from many lists: of beams alike, of one beam far above the others, of one
    beam alone, and all side by side in the vocabulary."""
    print("beam", B, W, V, k, kind, flush=True)
    rng = np.random.default_rng(V + k)
    x = (2 * rng.standard_normal((B, W, V))).astype(np.float32)
    s = (-3 * rng.random((B, W))).astype(np.float32)
    if kind == "one_beam":
        s[:, 1:] -= 30
    elif kind == "first_step":
        s[:, 1:] = -np.inf
    elif kind == "one_place":
        x[:, :, V // 2:V // 2 + k] += 20
    check(run(torch_dev, ops, x, s, k), x, s, k)


@pytest.mark.parametrize("V,k", [(2049, 1), (2069, 20), (2048 + 255, 64), (4096 + 300, 64),
                                 (20000, 16), (20000, 64)])
@pytest.mark.parametrize("allowed", [None, 3, 200, 300])
def test_select_few(torch_dev, ops, V, k, allowed):
    """A last slice of few logits, and vocabularies of which all but a few are masked."""
    print("beam few", V, k, allowed, flush=True)
    rng = np.random.default_rng(V + k)
    x = rng.standard_normal((2, 3, V)).astype(np.float32)
    if allowed:
        keep = np.zeros(V, bool)
        keep[rng.permutation(V)[:allowed // 2]] = True
        keep[100:100 + allowed // 2] = True
        x[..., ~keep] = -np.inf
    s = (-rng.random((2, 3))).astype(np.float32)
    check(run(torch_dev, ops, x, s, k), x, s, k)


def test_select_strides(torch_dev, ops):
    """Rows of a padded vocabulary, at an odd stride and offset."""
    torch = torch_dev
    wide = torch.randn((2 * 3, 1003), device="cuda")
    x = wide[:, 1:1001].unflatten(0, (2, 3))
    s = torch.zeros((2, 3), device="cuda")
    check(ops.beam_select(x, s, 6), x.cpu().numpy(), s.cpu().numpy(), 6)


def test_select_graph(torch_dev, ops):
    torch = torch_dev
    x = torch.randn((2, 4, 30000), device="cuda")
    s = torch.zeros((2, 4), device="cuda")
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        ops.beam_select(x, s, 8)
    st.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        out = ops.beam_select(x, s, 8)
    for i in range(3):
        x.copy_(torch.randn(x.shape, device="cuda"))
        want = ops.beam_select(x, s, 8)
        for a in out:
            a.fill_(-9)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


# ----------------------------------------------------------------- reorder ----

def caches(rng, B, W, pages, layers, Hkv, kv4=True):
    nb = B * W * pages + 2
    tables = rng.permutation(nb)[:B * W * pages].reshape(B * W, pages).astype(np.int32)
    shape = (nb, layers, Hkv, PAGE)
    if kv4:
        return tables, [rng.integers(0, 256, shape + (w,), dtype=np.uint8) for w in (64, 64, 4, 4)]
    return tables, [rng.integers(-128, 128, shape + (128,), dtype=np.int8) for _ in range(2)] + \
        [rng.standard_normal(shape).astype(np.float32) for _ in range(2)]


@pytest.mark.parametrize("B,W,ctx,layers,Hkv,kv4", [
    (1, 1, 5, 1, 1, True), (1, 2, 16, 2, 1, True), (2, 4, 37, 3, 5, True),
    (3, 8, 1, 1, 8, True), (1, 9, 63, 2, 2, True), (2, 16, 95, 1, 3, False),
    (1, 33, 20, 2, 1, True), (1, 64, 47, 1, 2, False), (4, 3, 300, 2, 2, True)])
def test_reorder(torch_dev, ops, B, W, ctx, layers, Hkv, kv4):
    """Several rounds of parents: any, a rotation (every slot is overwritten and read), all of
    one, none moved; pools and tables whole, so nothing else changes."""
    torch = torch_dev
    rng = np.random.default_rng(ctx)
    pages = ctx // PAGE + 2
    tables, pools = caches(rng, B, W, pages, layers, Hkv, kv4)
    lens = np.full(B * W, ctx, np.int32)
    d = [torch.from_numpy(a.copy()).cuda() for a in (tables, lens, *pools)]
    rounds = [rng.integers(0, W, (B, W)), np.tile(np.roll(np.arange(W), 1), (B, 1)),
              np.full((B, W), W - 1), np.tile(np.arange(W), (B, 1)), rng.integers(-2, W + 2, (B, W))]
    for parents in rounds:
        parents = parents.astype(np.int32)
        wide = torch.from_numpy(np.concatenate([parents, parents], 1)).cuda()
        ops.beam_reorder_paged(wide[:, :W], *d)
        plain.reorder(parents, tables, lens, pools)
        np.testing.assert_array_equal(d[0].cpu().numpy(), tables)
        for a, b in zip(d[2:], pools):
            np.testing.assert_array_equal(a.cpu().numpy(), b)


def test_reorder_out_of_range(torch_dev, ops):
    """Lengths of 0, below 0 and above the tables, page numbers outside the pool: nothing moves
    there."""
    torch = torch_dev
    rng = np.random.default_rng(0)
    B, W = 5, 3
    tables, pools = caches(rng, B, W, 4, 2, 2)
    lens = np.repeat(np.array([0, -5, 65, 64, 30], np.int32), W)
    tables[12, 1] = -1
    tables[13, 1] = len(pools[0])
    parents = np.tile(np.array([1, 2, 0], np.int32), (B, 1))
    d = [torch.from_numpy(a.copy()).cuda() for a in (tables, lens, *pools)]
    ops.beam_reorder_paged(torch.from_numpy(parents).cuda(), *d)
    plain.reorder(parents, tables, lens, pools)
    np.testing.assert_array_equal(d[0].cpu().numpy(), tables)
    for a, b in zip(d[2:], pools):
        np.testing.assert_array_equal(a.cpu().numpy(), b)
