"""The 8-bit product in each of its kernels (gemm_plan in csrc/gemm_i8.hip, stated once more so that a
test says which kernel it runs), at channels that end inside a tile: every value bit for bit, the first of
equal columns, NaN and infinities."""
import numpy as np
import pytest

from tenzo_amd import _lib
from tests import tree_plain as plain
from tests.test_gpu_kv4 import ops, torch_dev  # noqa: F401

# channels and tokens of a workgroup, channels of a part of a row's largest value
SHAPES = {"1: 16x16": (16, 16, 16), "16x16": (16, 16, 16), "32x16": (32, 16, 32),
          "32x32": (32, 32, 32), "64x32": (64, 32, 64), "tile 64x32": (64, 32, 32),
          "tile 64x64": (64, 64, 32), "tile 128x64": (128, 64, 64), "tile 128x128": (128, 128, 32),
          "tile 256x128": (256, 128, 64), "tile 256x256": (256, 256, 128)}


def _up(a, b):
    return -(-a // b)


def shape(M, N):
    def count(s):
        return _up(N, SHAPES[s][0]) * _up(M, SHAPES[s][1])

    def fits(s):
        return count(s) <= 256

    if fits("16x16"):
        return "1: 16x16" if M <= 4 else "16x16"
    if fits("32x16") or (M <= 16 and count("64x32") < 900):
        return "32x16"
    if fits("32x32") and M > 16:
        return "32x32"
    if fits("tile 64x32") and M > 32:
        return "tile 64x32"
    if M <= 32 and (fits("64x32") or count("64x32") >= 900):
        return "64x32"
    if fits("tile 64x64"):
        return "tile 64x64"
    if fits("tile 128x64") or (M <= 64 and count("tile 256x128") < 300):
        return "tile 128x64"
    if count("tile 128x128") <= 400:
        return "tile 128x128"
    if 150 <= count("tile 256x256") <= 192 and 2 * _up(M, 256) == _up(M, 128):
        return "tile 256x256"
    return "tile 256x128" if count("tile 256x128") >= 300 else "tile 128x128"


def test_plan():
    """The parts that a row's largest value comes in are those of the shape stated here."""
    rng = np.random.default_rng(0)
    seen = set()
    for _ in range(20000):
        M, N = (int(np.exp(rng.uniform(0, np.log(top)))) for top in (6000, 200000))
        s = shape(M, N)
        seen.add(s)
        parts = _up(N, SHAPES[s][0]) * (SHAPES[s][0] // SHAPES[s][2])
        assert _lib.load().tenzo_hip_gemm_i8_ws_bytes(M, N, 64, 1) == 8 * M * parts, (M, N, s)
    assert seen == set(SHAPES)


# of every shape a last tile of few channels or rows, and one that is nearly whole
CASES = [("1: 16x16", 3, 4001, 272), ("16x16", 15, 3999, 144), ("32x16", 20, 3901, 272),
         ("32x32", 30, 6901, 112), ("64x32", 20, 13801, 272), ("64x32", 31, 60031, 80),
         ("tile 64x32", 45, 4501, 272), ("tile 64x64", 200, 3897, 272),
         ("tile 128x64", 290, 6145, 144), ("tile 128x64", 40, 40001, 64),
         ("tile 128x128", 700, 3801, 272), ("tile 128x128", 641, 6275, 80),
         ("tile 256x128", 1100, 14701, 112), ("tile 256x256", 1500, 6909, 272),
         ("tile 256x256", 1409, 6657, 80)]


def device(torch, ops, codes, inv, w, scales):
    put = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    (M, K), N = codes.shape, len(w)
    q = np.stack([inv.view(np.int32), np.zeros(M, np.int32)], 1)
    return put(codes), put(q), ops.i8_rows_repack(put(w), N, K), put(scales), N, K


def product(codes, inv, w, scales):
    """y [M][N] fp32: sums exact (in fp64, below 2^53), the two products of fp32 rounded one by one."""
    acc = codes.astype(np.float64) @ w.astype(np.float64).T
    with np.errstate(invalid="ignore"):  # (0 times an infinity)
        return acc.astype(np.float32) * (inv[:, None] * scales)


@pytest.mark.gpu
@pytest.mark.parametrize("kernel,M,N,K", CASES)
def test_every_value(torch_dev, ops, kernel, M, N, K):
    torch, rng = torch_dev, np.random.default_rng(M + N)
    print("gemm", M, N, K, shape(M, N), flush=True)
    assert shape(M, N) == kernel
    codes, w = (rng.integers(-128, 128, (n, K)).astype(np.int8) for n in (M, N))
    inv = rng.uniform(0.001, 0.1, M).astype(np.float32)
    scales = rng.uniform(-0.01, 0.02, N).astype(np.float32)
    args, want = device(torch, ops, codes, inv, w, scales), product(codes, inv, w, scales)
    first = plain.first_best(want)
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        y = torch.full((M + 1, N + 3), 3.0, dtype=dtype, device="cuda")
        _, idx = ops.gemm_i8(*args, out=y[:M, 1:1 + N], want_idx=True)
        assert torch.equal(y[:M, 1:1 + N].cpu(), torch.from_numpy(want).to(dtype))
        np.testing.assert_array_equal(idx.cpu().numpy(), first)
        assert (y[M] == 3).all() and (y[:, 0] == 3).all() and (y[:, 1 + N:] == 3).all()
        assert torch.equal(ops.gemm_i8(*args, dtype=dtype), y[:M, 1:1 + N])


@pytest.mark.gpu
@pytest.mark.parametrize("kernel,M,N,K", CASES)
def test_first_of_equal_columns(torch_dev, ops, kernel, M, N, K):
    """Columns of one sum, their scales apart: the largest of them, and for rows of the other sign the
    smallest, stand in several columns, of a tile or of many, the last one among them."""
    torch, rng = torch_dev, np.random.default_rng(M + N + 1)
    print("gemm", M, N, K, shape(M, N), flush=True)
    assert shape(M, N) == kernel
    codes = np.where(rng.random((M, 1)) < 0.5, -1, 1).astype(np.int8).repeat(K, 1)
    w, inv = np.ones((N, K), np.int8), np.ones(M, np.float32)
    for spread in (1, 40, N):
        scales = rng.uniform(-1, 1, N).astype(np.float32)
        for value in (2, -2):
            start = rng.integers(0, N)
            at = np.unique((start + rng.integers(0, spread, 5)) % N)
            scales[at] = value
        if spread == N:
            scales[N - 1] = 2
        args, want = device(torch, ops, codes, inv, w, scales), product(codes, inv, w, scales)
        for dtype in (torch.float32, torch.float16, torch.bfloat16):
            y, idx = ops.gemm_i8(*args, dtype=dtype, want_idx=True)
            assert torch.equal(y.cpu(), torch.from_numpy(want).to(dtype))
            np.testing.assert_array_equal(idx.cpu().numpy(), plain.first_best(want))


@pytest.mark.gpu
@pytest.mark.parametrize("kernel,M,N", [(k, m, n) for k, m, n, _ in CASES] + [
    ("tile 64x32", 250, 1999), ("64x32", 32, 16001), ("tile 64x64", 250, 3999)])
def test_first_of_equal_columns_of_a_part(torch_dev, ops, kernel, M, N):
    """Sums of a few small numbers, whose largest one in a window of 64 columns is often there several
    times, in other columns for each row: of any two lanes the one with the lower column has to win."""
    torch, rng = torch_dev, np.random.default_rng(M + N + 3)
    K = 16
    print("gemm", M, N, K, shape(M, N), flush=True)
    assert shape(M, N) == kernel
    codes, w = (rng.integers(-1, 2, (n, K)).astype(np.int8) for n in (M, N))
    inv, rows = np.ones(M, np.float32), 0
    sums = product(codes, inv, w, np.ones(N, np.float32))
    for start in [0, N - 64, *(64 * rng.integers(0, N // 64, 10))]:
        scales = np.full(N, 0.0625, np.float32)
        scales[start:start + 64] = 1
        args, want = device(torch, ops, codes, inv, w, scales), sums * scales
        rows += ((want == want.max(1)[:, None]).sum(1) > 1).sum()
        for dtype in (torch.float32, torch.float16, torch.bfloat16):
            y, idx = ops.gemm_i8(*args, dtype=dtype, want_idx=True)
            assert torch.equal(y.cpu(), torch.from_numpy(want).to(dtype))
            np.testing.assert_array_equal(idx.cpu().numpy(), plain.first_best(want))
    print("rows with equal columns:", int(rows))
    assert rows > 3 * M


@pytest.mark.gpu
@pytest.mark.parametrize("kernel,M,N,K", CASES)
def test_nan_and_infinities(torch_dev, ops, kernel, M, N, K):
    """NaN counts as -inf; a row of nothing else, or of zeros, gives column 0."""
    torch, rng = torch_dev, np.random.default_rng(M + N + 2)
    print("gemm", M, N, K, shape(M, N), flush=True)
    assert shape(M, N) == kernel
    codes, w = (rng.integers(-128, 128, (n, K)).astype(np.int8) for n in (M, N))
    inv = np.ones(M, np.float32)
    scales = [np.zeros(N, np.float32), np.full(N, np.nan, np.float32),
              rng.uniform(-1, 1, N).astype(np.float32), rng.uniform(-1, 1, N).astype(np.float32)]
    scales[2][rng.integers(0, N, N // 3)] = np.nan
    scales[2][rng.integers(0, N, 3)] = np.inf
    scales[3][:] = np.where(np.arange(N) < N - 2, np.nan, scales[3])  # (the last tile alone counts)
    for s in scales:
        args, want = device(torch, ops, codes, inv, w, s), product(codes, inv, w, s)
        for dtype in (torch.float32, torch.float16):
            y, idx = ops.gemm_i8(*args, dtype=dtype, want_idx=True)
            np.testing.assert_array_equal(y.float().cpu().numpy(),
                                          torch.from_numpy(want).to(dtype).float().numpy())
            np.testing.assert_array_equal(idx.cpu().numpy(), plain.first_best(want))
