"""Rotary positions on the GPU against the definition in 64 bits; tolerances are the counted
roundings (tree_plain.rope) and half a step of the type."""
import numpy as np
import pytest

from tests import tree_plain as plain
from tests.test_gpu_kv4 import ops, torch_dev  # noqa: F401

pytestmark = pytest.mark.gpu
HALF = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
SMALL = {"float32": 2.0 ** -149, "float16": 2.0 ** -24, "bfloat16": 2.0 ** -133}


def check(got, x, positions, freqs, interleaved, mscale, kind, dim):
    x = x.double().cpu().numpy().reshape(len(positions), -1, dim)
    want, tol = plain.rope(x, positions, freqs, interleaved, mscale)
    got = got.double().cpu().numpy().reshape(want.shape)
    tol = tol + HALF[kind] * (np.abs(want) + tol) + SMALL[kind] / 2
    kept = slice(2 * len(freqs), None)
    np.testing.assert_array_equal(got[..., kept], x[..., kept])
    worst = float(np.max(np.abs(got - want) / tol))
    assert np.isfinite(got).all() and worst <= 1, worst


@pytest.mark.parametrize("kind", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,H,dim,rot", [
    (1, 1, 2, 2), (1, 25, 128, 128), (3, 5, 128, 32), (26, 40, 128, 128), (7, 3, 96, 24),
    (5, 2, 80, 80), (130, 6, 64, 64), (33, 2, 256, 128), (2, 1, 1024, 1024), (9, 3, 10, 6),
    (601, 25, 128, 128), (300, 7, 96, 96), (2, 256, 128, 64), (257, 1, 128, 128)])
def test_rope(torch_dev, ops, T, H, dim, rot, interleaved, kind):
    torch = torch_dev
    print("rope", T, H, dim, rot, interleaved, kind, flush=True)
    rng = np.random.default_rng(T * dim)
    dtype = getattr(torch, kind)
    wide = torch.from_numpy(rng.standard_normal((T, H * dim + 3))).to(dtype).cuda()
    x = wide[:, 2:2 + H * dim]  # (rows that begin anywhere)
    positions = rng.integers(-5, 100000, T).astype(np.int32)
    positions[0] = 0
    f, _ = ops.rope_freqs(rot, 10000.0)
    got = ops.rope(x, torch.from_numpy(positions).cuda(), f.cuda(), head_dim=dim,
                   interleaved=interleaved, mscale=1.25)
    assert got.is_contiguous() and got.shape == x.shape and got.dtype == dtype
    check(got, x, positions, f.numpy(), interleaved, 1.25, kind, dim)


@pytest.mark.parametrize("interleaved", [False, True])
def test_far_positions(torch_dev, ops, interleaved):
    """The largest positions, the smallest ones, quarters of a turn and their neighbours."""
    torch, rng = torch_dev, np.random.default_rng(0)
    positions = np.concatenate([[2 ** 31 - 1, -2 ** 31, 2 ** 24, 2 ** 24 + 1, 10 ** 6, -1, 1, 0],
                                rng.integers(-2 ** 31, 2 ** 31, 500)]).astype(np.int32)
    f = np.concatenate([[1.0, np.pi / 2, np.pi / 4, np.pi, 1e-9, 0.0, 2 * np.pi, 0.1],
                        rng.uniform(0, 1, 56)])
    x = torch.from_numpy(rng.standard_normal((len(positions), 2, 128))).float().cuda()
    got = ops.rope(x, torch.from_numpy(positions).cuda(), torch.from_numpy(f).cuda(),
                   interleaved=interleaved)
    check(got, x, positions, f, interleaved, 1.0, "float32", 128)


def test_every_angle(torch_dev, ops):
    """Two million angles of a turn: cosines and sines within 2^-23."""
    torch = torch_dev
    T = 1 << 15
    f = np.linspace(0, 2 * np.pi / T, 64, endpoint=False) + 1e-12
    x = torch.zeros((T, 1, 128), device="cuda")
    x[..., :64] = 1
    p = np.arange(T, dtype=np.int32)
    got = ops.rope(x, torch.from_numpy(p).cuda(), torch.from_numpy(f).cuda()).cpu().numpy()
    a = p[:, None] * f
    assert np.abs(got[:, 0, :64] - np.cos(a)).max() <= 2.0 ** -23
    assert np.abs(got[:, 0, 64:] - np.sin(a)).max() <= 2.0 ** -23


def test_in_place_and_strides(torch_dev, ops):
    """The q | k part of a fused projection in place: v stays; turned back by the negative
    positions."""
    torch = torch_dev
    qkv = torch.randn((41, 30 * 128), device="cuda")
    old = qkv.clone()
    f, m = ops.rope_freqs(128, 500000.0, "parts", 16.0, 4096)
    assert m == pytest.approx(0.1 * np.log(16) + 1)
    at = torch.arange(9000, 9041, dtype=torch.int32, device="cuda")
    qk = qkv[:, :25 * 128]
    assert ops.rope(qk, at, f.cuda(), out=qk) is qk
    check(qk, old[:, :25 * 128], at.cpu().numpy(), f.numpy(), False, 1.0, "float32", 128)
    assert torch.equal(qkv[:, 25 * 128:], old[:, 25 * 128:])
    ops.rope(qk, -at, f.cuda(), out=qk)
    assert (qkv - old).abs().max() < 1e-5  # two turns of values below 6: 2 (3 2^-23) 6 sqrt 2
    other = torch.full((41, 26 * 128), 9.0, device="cuda")
    ops.rope(qk, at, f.cuda(), out=other[:, 128:])
    assert torch.equal(other[:, 128:], ops.rope(qk, at, f.cuda())) and (other[:, :128] == 9).all()


def test_agrees_with_the_cache_rotation(torch_dev, ops):
    """rope and kv4_append without a table store the codes that kv4_append stores with one, where
    both rotations are exact (quarters of a turn)."""
    torch, rng = torch_dev, np.random.default_rng(1)
    T = 32
    f = torch.full((64,), np.pi / 2, dtype=torch.float64, device="cuda")
    at = np.arange(T)
    cs = np.concatenate([np.repeat(np.array([1, 0, -1, 0])[at % 4][:, None], 64, 1),
                         np.repeat(np.array([0, 1, 0, -1])[at % 4][:, None], 64, 1)], 1)
    k = torch.from_numpy(rng.standard_normal((T, 256)).astype(np.float32)).cuda()
    tables = torch.arange(2, dtype=torch.int32, device="cuda")[None]
    ctx = torch.tensor([T], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, T], dtype=torch.int32, device="cuda")
    one, two = ops.kv4_pool(2, 1, 2), ops.kv4_pool(2, 1, 2)
    ops.kv4_append(k, k, *one, tables, ctx, 0, cu_q=cu,
                   rope_cs=torch.from_numpy(cs.astype(np.float32)).cuda())
    turned = ops.rope(k, torch.arange(T, dtype=torch.int32, device="cuda"), f)
    ops.kv4_append(turned, k, *two, tables, ctx, 0, cu_q=cu)
    for a, b in zip(one, two):
        assert torch.equal(a, b)


def test_empty(torch_dev, ops):
    torch = torch_dev
    got = ops.rope(torch.zeros((0, 256), device="cuda"),
                   torch.zeros(0, dtype=torch.int32, device="cuda"),
                   torch.zeros(64, dtype=torch.float64, device="cuda"))
    assert got.shape == (0, 256)


def test_captured(torch_dev, ops):
    torch = torch_dev
    x = torch.randn((50, 25 * 128), device="cuda")
    at = torch.arange(50, dtype=torch.int32, device="cuda")
    f = ops.rope_freqs(128)[0].cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = ops.rope(x, at, f)
    for i in range(3):
        x.normal_()
        at.add_(1000)
        want = ops.rope(x, at, f)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
