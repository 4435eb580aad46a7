"""Beam selection for batches of so many rows that a slice has 4096 logits (16 a thread; the other
tests' have 2048): from 1024 slices of that size on."""
import numpy as np
import pytest

from tests.test_gpu_beam import check, ops, run, torch_dev  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("k", [5, 40])
@pytest.mark.parametrize("kind", ["normal", "equal", "few", "rising", "first_step", "masked",
                                  "all_masked", "strange", "block", "last_slice"])
def test_slices_of_4096(torch_dev, ops, kind, k):
    B, W, V = 57, 6, 8192 + 101
    assert B * W * -(-V // 4096) >= 1024
    print("beam batch", kind, k, flush=True)
    rng = np.random.default_rng(k)
    x = rng.standard_normal((B, W, V)).astype(np.float32)
    s = (-5 * rng.random((B, W))).astype(np.float32)
    if kind == "equal":
        x[:], s[:] = 0.5, -1.0
    elif kind == "few":
        x = rng.integers(0, 3, x.shape).astype(np.float32)
        s = np.round(s)
    elif kind == "rising":
        x = np.sort(x, -1)
    elif kind == "first_step":
        s[:, 1:] = -np.inf
    elif kind == "masked":
        keep = rng.permutation(V)[:300]
        y = np.full_like(x, -np.inf)
        y[..., keep] = x[..., keep]
        x = y
        x[5] = -np.inf
        x[5, 2, 30] = 4.0
    elif kind == "all_masked":
        x[:, 1:] = -np.inf
        x[3] = -np.inf
        x[:, 0, : V // 2] = np.finfo(np.float32).min
        s[4] = -np.inf
    elif kind == "strange":
        x[:, :, 5] = np.nan
        x[:, 1, 9] = np.inf
        x[0, 0] = np.nan
        s[1, 2] = np.nan
        s[2, 3] = np.inf
    elif kind == "block":
        x[:, :, V // 3:V // 3 + 30] += 50
    elif kind == "last_slice":
        x[:, :, 8192:] += 20
    check(run(torch_dev, ops, x, s, k), x, s, k)
