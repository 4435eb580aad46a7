"""What the entry points of trees of drafted tokens, rotary positions and the 8-bit product refuse,
at the C ABI and in tenzo_amd.ops (nothing is launched, so no GPU is needed), and the frequencies
against their formulas."""
import ctypes

import numpy as np
import pytest
import torch

from tenzo_amd import _lib, ops
from tests import tree_kernels
from tests.test_kv4_refusals import A, POOLS, SEQS, _cache, _swap, cpu  # noqa: F401

CALLS = {
    "plan": ("tenzo_hip_tree_plan", dict(parents=A, ctx=A, cu=A, B=3, T=9, most=5, mask=A, at=A,
                                         stream=None)),
    "attn": ("tenzo_hip_attn_tree_kv4", dict(q=A, dtype=0, qs=1024, mask=A, ms=2, words=2, **POOLS,
                                             Hq=8, Hkv=2, **SEQS, out=A, os=1024, ws=A,
                                             ws_bytes=1 << 40, stream=None)),
    "accept": ("tenzo_hip_tree_accept", dict(
        parents=A, tokens=A, target=A, pk=A, pv=A, pks=A, pvs=A, n_blocks=4, n_layers=2, Hkv=2,
        row_bytes=64, tables=A, stride=8, width=8, ctx=A, cu=A, B=3, T=9, most=5, path=A + 4096,
        count=A + 4160, next=A + 4176, lens=A + 4192, stream=None)),
    "rope": ("tenzo_hip_rope", dict(x=A, dtype=0, xs=1024, at=A, f=A, T=3, H=8, dim=128, rot=128,
                                    inter=0, m=1.0, out=A + 8192, os=1024, stream=None)),
    "gemm": ("tenzo_hip_gemm_i8", dict(codes=A, cs=64, q=A, w=A, s=A, M=3, N=70, K=64, y=A, dtype=0,
                                       ys=70, idx=A, ws=A, ws_bytes=1 << 20, stream=None)),
}
CACHE_BAD = [dict(pk=None), dict(pvs=None), dict(pk=A + 4), dict(pks=A + 2), dict(n_layers=0),
             dict(n_blocks=-1), dict(n_blocks=1 << 31), dict(Hkv=0), dict(tables=None),
             dict(stride=7), dict(width=-1), dict(ctx=None), dict(B=-1), dict(T=-1),
             dict(width=1 << 28)]
BAD = {
    "plan": [dict(parents=None), dict(ctx=None), dict(mask=None), dict(at=None), dict(mask=A + 4),
             dict(B=-1), dict(T=-1), dict(T=1 << 31), dict(most=0), dict(most=4097),
             dict(cu=None)],
    "attn": CACHE_BAD + [dict(layer=2), dict(layer=-1), dict(T=4), dict(q=None), dict(out=None),
                         dict(qs=1023), dict(os=1000), dict(Hq=7), dict(Hq=34), dict(Hq=0),
                         dict(dtype=2), dict(mask=None), dict(mask=A + 4), dict(words=0),
                         dict(words=1025), dict(ms=1)],
    "accept": CACHE_BAD + [dict(parents=None), dict(tokens=None), dict(target=None),
                           dict(path=None), dict(count=None), dict(next=None), dict(lens=None),
                           dict(row_bytes=32), dict(most=0), dict(most=4097), dict(cu=None),
                           dict(n_layers=65536), dict(lens=A), dict(count=A), dict(next=A),
                           dict(path=A)],
    "rope": [dict(T=1 << 24), dict(x=None), dict(at=None), dict(f=None), dict(out=None), dict(dtype=3),
             dict(dtype=-1), dict(T=-1), dict(H=0), dict(dim=1), dict(dim=1026), dict(rot=0),
             dict(rot=3), dict(rot=130), dict(xs=1023), dict(os=1000), dict(H=257), dict(x=A + 2),
             dict(f=A + 4), dict(at=A + 2), dict(out=A, os=2048)],
    "gemm": [dict(codes=None), dict(q=None), dict(w=None), dict(s=None), dict(y=None),
             dict(ws=None), dict(ws_bytes=8), dict(ws=A + 4), dict(dtype=3), dict(M=-1),
             dict(M=(1 << 20) + 1), dict(N=0), dict(N=(1 << 29) + 1), dict(K=0), dict(K=40),
             dict(K=131072, cs=131072), dict(cs=48), dict(cs=72), dict(ys=69), dict(codes=A + 8),
             dict(w=A + 4), dict(s=A + 2), dict(y=A + 2)],
}


@pytest.mark.parametrize("name,bad", [(n, b) for n in BAD for b in BAD[n]],
                         ids=lambda v: v if isinstance(v, str) else "_".join(v))
def test_c_refusals(name, bad):
    fn, good = CALLS[name]
    L = _lib.load()
    rc = getattr(L, fn)(*{**good, **bad}.values())
    assert rc in (-1, -2, -3, -4, -5, -6) and L.tenzo_hip_last_error()


@pytest.mark.parametrize("name", list(CALLS))
def test_c_empty_calls(name):
    """No rows: nothing to do, whatever the pointers."""
    fn, good = CALLS[name]
    none = {k: None for k, v in good.items() if v in (A, A + 8192)}
    empty = {"rope": dict(T=0), "gemm": dict(M=0)}.get(name, dict(B=0, T=0))
    assert getattr(_lib.load(), fn)(*{**good, **none, **empty}.values()) == 0


def test_workspaces():
    L = _lib.load()
    assert L.tenzo_hip_gemm_i8_ws_bytes(5, 128256, 2560, 0) == 0
    assert L.tenzo_hip_gemm_i8_ws_bytes(0, 100, 64, 1) == 0
    assert L.tenzo_hip_gemm_i8_ws_bytes(5, 128256, 2560, 1) >= 5 * 8
    assert L.tenzo_hip_attn_tree_kv4_ws_bytes(0, 3, 8, 2, 9, 1, 0) == 0
    assert L.tenzo_hip_attn_tree_kv4_ws_bytes(30, 1, 8, 3, 9, 1, 0) == 0


def test_plan_of_trees():
    L, rng = _lib.load(), np.random.default_rng(0)
    for _ in range(3000):
        Hkv = int(rng.choice([1, 2, 5, 8]))
        Hq, B = Hkv * int(rng.choice([1, 2, 4, 8, 16])), int(rng.integers(1, 65))
        T, width = int(rng.integers(B, 130 * B)), int(rng.integers(0, 4000) * rng.integers(0, 2))
        cu = bool(rng.integers(0, 5))
        T = T if cu else B
        for half in (0, 1):
            want = tree_kernels.plan(T, B, Hq, Hkv, width, cu, half)[2]
            assert L.tenzo_hip_attn_tree_kv4_ws_bytes(T, B, Hq, Hkv, width, cu, half) == want


def _i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


@pytest.mark.parametrize("i,make", [
    (0, lambda t: t[..., :32]), (0, lambda t: t.to(torch.int8)), (1, lambda t: t[:4]),
    (2, lambda t: t[..., 0]), (3, lambda t: t.float()), (0, lambda t: t.transpose(1, 2)),
    (4, lambda t: t.long()), (4, lambda t: t[0]), (4, lambda t: t.T.contiguous().T),
    (5, lambda t: t[:2]), (5, lambda t: t.long()), (4, lambda t: t[:2])])
def test_ops_refuse_caches(cpu, i, make):  # noqa: F811
    args = _cache()
    args = _swap(args, i, make(args[i]))
    mask = torch.zeros((3, 1), dtype=torch.int64)
    with pytest.raises(ValueError):
        ops.attn_tree_kv4(torch.zeros((3, 256)), mask, *args)
    with pytest.raises(ValueError):
        ops.tree_accept(_i32(3), _i32(3), _i32(3), *args[:6], 2)


def test_ops_refuse_rows(cpu):  # noqa: F811
    args = _cache()
    x, mask, cu = torch.zeros((3, 256)), torch.zeros((3, 1), dtype=torch.int64), _i32(4)
    f = torch.zeros(64, dtype=torch.float64)
    q, w, s = _i32(3, 2), torch.zeros(4096, dtype=torch.uint8), torch.zeros(50)
    c = torch.zeros((3, 64), dtype=torch.int8)
    bad = [lambda: ops.attn_tree_kv4(x[:2], mask[:2], *args),
           lambda: ops.attn_tree_kv4(x, mask[:2], *args),
           lambda: ops.attn_tree_kv4(x, mask[:, :0], *args),
           lambda: ops.attn_tree_kv4(x, mask.int(), *args),
           lambda: ops.attn_tree_kv4(x, mask[:, 0], *args),
           lambda: ops.attn_tree_kv4(x, mask.expand(3, 2), *args),
           lambda: ops.attn_tree_kv4(x.bfloat16(), mask, *args),
           lambda: ops.attn_tree_kv4(x[:, :200], mask, *args),
           lambda: ops.attn_tree_kv4(x, mask, *args, cu_q=cu[:3]),
           lambda: ops.attn_tree_kv4(x, mask, *args, out=x[:, :128]),
           lambda: ops.tree_plan(_i32(3), _i32(2), 4), lambda: ops.tree_plan(_i32(3, 1), _i32(3), 4),
           lambda: ops.tree_plan(_i32(3).long(), _i32(3), 4),
           lambda: ops.tree_plan(_i32(3), _i32(3).long(), 4),
           lambda: ops.tree_plan(_i32(9), _i32(3), 4, cu_q=_i32(3)),
           lambda: ops.tree_plan(_i32(9), _i32(3), 4, cu_q=_i32(4).long()),
           lambda: ops.tree_plan(_i32(6)[::2], _i32(3), 4),
           lambda: ops.tree_accept(_i32(3), _i32(2), _i32(3), *args[:6], 2),
           lambda: ops.tree_accept(_i32(3), _i32(3), _i32(3).long(), *args[:6], 2),
           lambda: ops.tree_accept(_i32(4), _i32(4), _i32(4), *args[:6], 2),
           lambda: ops.rope(x.double(), _i32(3), f), lambda: ops.rope(x[0], _i32(256), f),
           lambda: ops.rope(x, _i32(2), f), lambda: ops.rope(x, _i32(3).long(), f),
           lambda: ops.rope(x, _i32(3), f.float()), lambda: ops.rope(x, _i32(3), f[None]),
           lambda: ops.rope(x, _i32(3), f, head_dim=100),
           lambda: ops.rope(x, _i32(3), f, head_dim=0),
           lambda: ops.rope(x.T.contiguous().T, _i32(3), f),
           lambda: ops.rope(x, _i32(3), f, out=x.half()),
           lambda: ops.rope(x, _i32(3), f, out=x[:2]),
           lambda: ops.gemm_i8(c, q, w, s, 50, 48), lambda: ops.gemm_i8(c, q[:2], w, s, 50, 64),
           lambda: ops.gemm_i8(c, q, w[:4095], s, 50, 64),
           lambda: ops.gemm_i8(c, q, w, s[:49], 50, 64),
           lambda: ops.gemm_i8(c.int(), q, w, s, 50, 64),
           lambda: ops.gemm_i8(c, q.float(), w, s, 50, 64),
           lambda: ops.gemm_i8(c, q, w.int(), s, 50, 64),
           lambda: ops.gemm_i8(c, q, w, s.half(), 50, 64),
           lambda: ops.gemm_i8(c, q, w, s, 50, 64, dtype=torch.float64),
           lambda: ops.gemm_i8(c.T.contiguous().T, q, w, s, 50, 64),
           lambda: ops.gemm_i8(c, q, w, s, 50, 64, out=torch.zeros((3, 51))),
           lambda: ops.gemm_i8(c, q, w, s, 50, 64, out=torch.zeros((50, 3)).T)]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            print(i)
            call()


def test_ops_refuse_other_devices(cpu, monkeypatch):  # noqa: F811
    monkeypatch.setattr(ops, "_dev", lambda: 0)
    args = _cache()
    x = torch.zeros((3, 256))
    for call in (lambda: ops.attn_tree_kv4(x, torch.zeros((3, 1), dtype=torch.int64), *args),
                 lambda: ops.tree_plan(_i32(3), _i32(3), 1),
                 lambda: ops.tree_accept(_i32(3), _i32(3), _i32(3), *args[:6], 2),
                 lambda: ops.rope(x, _i32(3), torch.zeros(64, dtype=torch.float64)),
                 lambda: ops.gemm_i8(torch.zeros((3, 64), dtype=torch.int8), _i32(3, 2),
                                     torch.zeros(4096, dtype=torch.uint8), torch.zeros(50), 50,
                                     64)):
        with pytest.raises(ValueError):
            call()


# ------------------------------------------------------------- frequencies ----

def test_frequencies():
    i = np.arange(0, 64, 2)
    for theta in (10000.0, 500000.0):
        f = theta ** (-i / 64)
        got, m = ops.rope_freqs(64, theta)
        np.testing.assert_allclose(got.numpy(), f, rtol=1e-14)
        assert m == 1
        np.testing.assert_allclose(ops.rope_freqs(64, theta, "linear", 8.0)[0].numpy(), f / 8,
                                   rtol=1e-14)
        got, m = ops.rope_freqs(64, theta, "base", 8.0)
        np.testing.assert_allclose(got.numpy(), (theta * 8 ** (64 / 62)) ** (-i / 64), rtol=1e-13)
        # (the slowest pair is slowed down by just the factor)
        np.testing.assert_allclose(got[-1].item(), f[-1] / 8, rtol=1e-12)
        got, m = ops.rope_freqs(64, theta, "parts", 16.0, trained=4096, fast=32, slow=1)
        turns = 4096 * f / (2 * np.pi)
        keep = np.clip((turns - 1) / 31, 0, 1)
        np.testing.assert_allclose(got.numpy(), f * keep + f / 16 * (1 - keep), rtol=1e-13)
        assert m == pytest.approx(0.1 * np.log(16) + 1, rel=1e-6)
        assert got[0] == 1 and got[-1] == pytest.approx(f[-1] / 16)


@pytest.mark.parametrize("bad", [
    dict(rot_dim=0), dict(rot_dim=3), dict(theta=0.0), dict(theta=float("inf")),
    dict(theta=float("nan")), dict(scaling="linear", factor=0.5),
    dict(scaling="linear", factor=float("nan")), dict(scaling="base", rot_dim=2, factor=2.0),
    dict(scaling="parts", factor=2.0, trained=0.0), dict(scaling="parts", factor=2.0, fast=1.0),
    dict(scaling="parts", factor=2.0, slow=-1.0)], ids=lambda b: "_".join(b))
def test_frequencies_refused(bad):
    with pytest.raises(RuntimeError):
        ops.rope_freqs(**{"rot_dim": 64, **bad})


def test_unknown_scaling_refused():
    with pytest.raises(ValueError):
        ops.rope_freqs(64, scaling="other")
