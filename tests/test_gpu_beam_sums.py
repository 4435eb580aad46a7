"""Beam selection where the sums of exponentials decide: vocabularies whose tokens lie at one distance
below the best, so that what an fp32 exponential is off by adds up instead of averaging out, and
beams whose candidates are nearer to each other than that. Beams and tokens as in 64 bits; scores
within 2^-24 of themselves (fp32) and 1.25e-6, which csrc/beam.hip counts for a log-sum."""
import numpy as np
import pytest

from tests import kv4_plain as plain
from tests.test_gpu_beam import ops, torch_dev  # noqa: F401

pytestmark = pytest.mark.gpu


def log_sums(x):
    top = x.astype(np.float64).max(-1, keepdims=True)
    return (top + np.log(np.exp(x - top).sum(-1, keepdims=True)))[..., 0]


def level(rng, B, W, V, best=1):
    """Logits [B][W][V]: `best` tokens at some logit (the same ones in all beams), the others 3 to
    13 below it, at one distance or at a few."""
    top = rng.uniform(-4, 4, (B, W, 1)).astype(np.float32)
    x = np.broadcast_to(top - rng.uniform(3, 13, (B, W, 1)).astype(np.float32), (B, W, V)).copy()
    some = rng.random((B, W)) < 0.3
    x[some] -= rng.integers(0, 3, (int(some.sum()), V)).astype(np.float32)
    x[..., rng.permutation(V)[:best]] = top
    return x


def even(x, at):
    """The scores with which all beams' best candidates come to `at`, as near as fp32 has them."""
    return (at + log_sums(x) - x.max(-1)).astype(np.float32)


def check(torch, ops, x, s, k):
    """Beams and tokens as in 64 bits. Candidates that are mathematically equal may lie 2^-46 from
    each other there, in any order: sums of exponentials are rounded to some 20 * 2^-53 of
    themselves (in pairs), the log, its sum with the largest logit and the two differences to
    2^-53 of numbers up to 20 each, in numpy and in the kernel."""
    got = ops.beam_select(torch.from_numpy(x).cuda(), torch.from_numpy(s).cuda(), k)
    score, beam, token = (a.cpu().numpy() for a in got)
    want = plain.beam_select(x, s, k)
    if (beam != want[1]).any() or (token != want[2]).any():
        at = (np.arange(len(x))[:, None], beam, token)
        mine = x[at] - log_sums(x)[at[:2]] + s[at[:2]]
        real = np.isfinite(want[0])
        assert (np.abs(mine - want[0])[real] <= 2.0 ** -46).all()
        np.testing.assert_array_equal(mine[~real], want[0][~real])
        assert all(len(set(zip(*c))) == k for c in zip(beam, token))
    real = np.isfinite(want[0])
    np.testing.assert_array_equal(score[~real], want[0][~real])
    off = np.abs(score[real] - want[0][real])
    assert (off <= 2.0 ** -24 * np.abs(want[0][real]) + 1.25e-6).all(), off.max()


@pytest.mark.parametrize("B,W,V,k", [(40, 2, 128256, 2), (60, 4, 5000, 8), (25, 8, 32000, 16),
                                     (200, 3, 2000, 2), (4, 40, 9001, 64), (3, 64, 3000, 64)])
def test_near_beams(torch_dev, ops, B, W, V, k):
    """The best candidates of all beams within some 1e-7 of each other."""
    print("beam near", B, W, V, k, flush=True)
    rng = np.random.default_rng(V + W)
    x = level(rng, B, W, V)
    check(torch_dev, ops, x, even(x, 0.0), k)


@pytest.mark.parametrize("W,V,best,k", [(64, 2000, 64, 64), (64, 5000, 64, 64), (30, 3000, 40, 20),
                                        (5, 20000, 2000, 40)])
def test_many_near_candidates(torch_dev, ops, W, V, best, k):
    """More of them than are ranked at once."""
    print("beam many near", W, V, best, k, flush=True)
    rng = np.random.default_rng(V + W)
    x = level(rng, 3, W, V, best)
    s = even(x, -1.0)
    s[1, ::3] = -np.inf
    check(torch_dev, ops, x, s, k)


def test_near_to_the_last(torch_dev, ops):
    """Near candidates at the border of the k best, the others far above them; beams that are alike
    (equal sums: the lower beam first) and beams of masked tokens beside them."""
    rng = np.random.default_rng(3)
    B, W, V, k = 50, 6, 4000, 3
    x = level(rng, B, W, V)
    s = even(x, -2.0)
    s[:, :2] += 3
    x[:10, 4] = x[:10, 3]
    s[:10, 4] = s[:10, 3]
    x[20:30, 5] = -np.inf
    x[20:30, 4, 7:] = np.finfo(np.float32).min
    check(torch_dev, ops, x, s, k)


@pytest.mark.parametrize("gap", [0.5, 3.0, 6.3, 8.48, 9.7, 11.1, 30.0])
@pytest.mark.parametrize("V", [2048, 4096, 128256])
def test_level_sums(torch_dev, ops, V, gap):
    """One beam, the others of its tokens `gap` below: its scores alone."""
    x = np.full((3, 1, V), -gap, np.float32) + np.float32([0, 1.3, -70.1])[:, None, None]
    x[..., V // 2] += np.float32(gap)
    check(torch_dev, ops, x, even(x, 0.0), 4)


@pytest.mark.parametrize("allowed", [1, 3, 12])
@pytest.mark.parametrize("V", [3000, 40000])
def test_near_beams_of_few_tokens(torch_dev, ops, V, allowed):
    """All but a few tokens masked, so that -inf is among the k best, and beams as near as fp32 puts
    their scores."""
    rng = np.random.default_rng(V + allowed)
    x = level(rng, 30, 8, V, 1)
    keep = rng.permutation(V)[:allowed]
    y = np.full_like(x, -np.inf)
    y[..., keep] = np.sort(x[..., rng.permutation(V)[:allowed]], -1)
    y[..., keep[0]] += np.float32(7)
    check(torch_dev, ops, y, even(y, -3.0), 16)
