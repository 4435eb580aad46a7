"""The product of 8-bit integers with scales for tokens and channels on the GPU, bit for bit: the
sums are whole numbers and the two fp32 products are rounded one by one."""
import numpy as np
import pytest

from tests import tree_plain as plain
from tests.test_gpu_kv4 import ops, torch_dev  # noqa: F401

pytestmark = pytest.mark.gpu


def make(torch, ops, M, N, K, seed=0, wide=0):
    rng = np.random.default_rng(seed)
    codes = rng.integers(-128, 128, (M, K + wide)).astype(np.int8)
    w = rng.integers(-128, 128, (N, K)).astype(np.int8)
    inv = rng.uniform(0.001, 0.1, M).astype(np.float32)
    scales = rng.uniform(-0.01, 0.02, N).astype(np.float32)
    q = np.stack([inv.view(np.int32), rng.integers(-9, 9, M).astype(np.int32)], 1)
    put = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    dev = (put(codes)[:, :K], put(np.ascontiguousarray(q)), ops.i8_rows_repack(put(w), N, K),
           put(scales), N, K)
    return dev, plain.gemm_i8(codes[:, :K], inv, w, scales)


SIZES = [(1, 1, 16), (1, 64, 64), (2, 65, 80), (3, 1000, 48), (16, 130, 2560), (17, 63, 112),
         (26, 2560, 6912), (32, 200, 1040), (33, 70, 256), (64, 4100, 512), (65, 129, 272),
         (100, 640, 2560), (128, 512, 640), (130, 257, 6912), (200, 2560, 2560), (257, 1023, 400),
         (300, 515, 272), (513, 1300, 96), (700, 3840, 2560), (1024, 1024, 1024), (2049, 300, 128),
         (26, 40000, 320), (5, 33000, 160), (1, 128256, 64), (61, 20000, 1616), (1500, 6912, 528)]


@pytest.mark.parametrize("kind", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_gemm(torch_dev, ops, M, N, K, kind):
    torch = torch_dev
    print("gemm", M, N, K, kind, flush=True)
    dtype = getattr(torch, kind)
    args, want = make(torch, ops, M, N, K, seed=M + N, wide=0 if M % 2 else 32)
    y, idx = ops.gemm_i8(*args, dtype=dtype, want_idx=True)
    assert y.dtype == dtype and y.shape == (M, N)
    assert torch.equal(y.cpu(), torch.from_numpy(want).to(dtype))
    np.testing.assert_array_equal(idx.cpu().numpy(), plain.first_best(want))
    # into rows of a wider buffer, without the index
    out = torch.full((M, N + 5), 3.0, dtype=dtype, device="cuda")
    assert torch.equal(ops.gemm_i8(*args, out=out[:, 2:2 + N]), y)
    assert (out[:, :2] == 3).all() and (out[:, 2 + N:] == 3).all()


@pytest.mark.parametrize("M,N,K", [(4, 3999, 1104), (16, 6913, 80), (20, 6901, 144),
                                   (30, 13801, 272), (19, 70001, 112), (48, 40001, 96),
                                   (47, 3900, 16), (300, 60001, 64), (90, 1000, 4112)])
def test_gemm_of_every_shape(torch_dev, ops, M, N, K):
    torch = torch_dev
    print("gemm", M, N, K, flush=True)
    args, want = make(torch, ops, M, N, K, seed=M + N, wide=16 * (M % 3))
    for kind in (torch.float32, torch.float16):
        y, idx = ops.gemm_i8(*args, dtype=kind, want_idx=True)
        assert torch.equal(y.cpu(), torch.from_numpy(want).to(kind))
        np.testing.assert_array_equal(idx.cpu().numpy(), plain.first_best(want))


@pytest.mark.parametrize("M,N,K", [(1100, 14701, 48), (1100, 14800, 176), (2000, 9985, 32)])
def test_tiles_in_halves(torch_dev, ops, M, N, K):
    """Tiles of 256 x 128 past a multiple of 256, which come as halves (the last half of the first
    case has no channel), against the call with the largest values, whose tiles stay whole."""
    torch = torch_dev
    tiles = -(-N // 256) * -(-M // 128)
    assert tiles > 512 and 0 < tiles % 256 <= 128
    args, want = make(torch, ops, M, N, K, seed=N)
    for kind in (torch.float32, torch.bfloat16):
        y = torch.full((M + 1, N), 3.0, dtype=kind, device="cuda")
        ops.gemm_i8(*args, out=y[:M])
        assert torch.equal(y[:M].cpu(), torch.from_numpy(want).to(kind)) and (y[M] == 3).all()
        assert torch.equal(y[:M], ops.gemm_i8(*args, dtype=kind, want_idx=True)[0])


@pytest.mark.parametrize("M,N,K", [(1, 500, 320), (40, 300, 208), (300, 257, 512)])
def test_rows_of_the_lm_head(torch_dev, ops, M, N, K):
    """Each row bit for bit what the LM head's product and its argmax give."""
    torch = torch_dev
    rng = np.random.default_rng(1)
    x = torch.from_numpy(rng.standard_normal((M, K)).astype(np.float32)).cuda()
    codes, q = ops.actquant127(x)
    w = torch.from_numpy(rng.integers(-127, 128, (N, K)).astype(np.int8)).cuda()
    packed, scales = ops.i8_rows_repack(w, N, K), torch.rand(N, device="cuda") * 0.01
    y, idx = ops.gemm_i8(codes, q, packed, scales, N, K, want_idx=True)
    one = torch.zeros(1, dtype=torch.int32, device="cuda")
    for m in range(0, M, 7):
        logits = torch.empty(N, device="cuda")
        ops.lm_head_i8_codes_into(codes[m:m + 1], q[m:m + 1], packed, scales, N, K, logits, one)
        assert torch.equal(logits, y[m]) and one.item() == idx[m].item()


@pytest.mark.parametrize("M", [1, 20, 90, 400])
def test_ties_nan_and_infinities(torch_dev, ops, M):
    """The first of equal columns; NaN counts as -inf; a row of NaN gives column 0."""
    torch = torch_dev
    N, K = 700, 64
    args, _ = make(torch, ops, M, N, K, seed=2)
    scales = torch.zeros(N, device="cuda")
    y, idx = ops.gemm_i8(args[0], args[1], args[2], scales, N, K, want_idx=True)
    assert (y == 0).all() and (idx == 0).all()
    scales[:] = float("nan")
    y, idx = ops.gemm_i8(args[0], args[1], args[2], scales, N, K, want_idx=True)
    assert y.isnan().all() and (idx == 0).all()
    scales[:] = 1.0
    scales[13] = float("inf")
    scales[600:] = float("nan")
    y, idx = ops.gemm_i8(args[0], args[1], args[2], scales, N, K, want_idx=True)
    np.testing.assert_array_equal(idx.cpu().numpy(), plain.first_best(y.cpu().numpy()))


def test_largest_sums(torch_dev, ops):
    """Sums up to the range of int32: K 131056 of -128 times -128."""
    torch = torch_dev
    for M in (1, 70):
        N, K = 65, 131056
        codes = torch.full((M, K), -128, dtype=torch.int8, device="cuda")
        w = torch.full((N, K), -128, dtype=torch.int8, device="cuda")
        q = torch.ones((M, 2), device="cuda").view(torch.int32)
        y = ops.gemm_i8(codes, q, ops.i8_rows_repack(w, N, K), torch.ones(N, device="cuda"), N, K)
        assert (y == float(np.float32(K * 16384))).all()


def test_empty(torch_dev, ops):
    args, _ = make(torch_dev, ops, 1, 10, 32)
    y, idx = ops.gemm_i8(args[0][:0], args[1][:0], *args[2:], want_idx=True)
    assert y.shape == (0, 10) and idx.shape == (0,)


def test_captured(torch_dev, ops):
    """Two captured products with workspaces of their own, replayed at once on two streams."""
    torch = torch_dev
    sets = [make(torch, ops, m, 3000, 640, seed=m)[0] for m in (26, 150)]
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for a, st in zip(sets, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            outs.append(ops.gemm_i8(*a, want_idx=True))
        graphs.append(g)
    for i in range(4):
        for a in sets:
            a[0].copy_(torch.roll(a[0], i + 1, 0))
        want = [[t.clone() for t in ops.gemm_i8(*a, want_idx=True)] for a in sets]
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
