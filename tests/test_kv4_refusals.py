"""What the 4-bit paged cache's and beam search's entry points refuse, at the C ABI and in
tenzo_amd.ops (nothing is launched, so no GPU is needed), and their plain forms against direct
statements."""
import ctypes

import numpy as np
import pytest
import torch

from tenzo_amd import _lib, ops
from tests import kv4_plain as plain

BUF = ctypes.create_string_buffer(1 << 16)
A = (ctypes.addressof(BUF) + 255) & ~255  # an address that is never followed

POOLS = dict(pk=A, pv=A, pks=A, pvs=A, n_blocks=4, n_layers=2, layer=1)
SEQS = dict(tables=A, stride=8, width=8, ctx=A, cu=None, B=3, T=3)
ROPE = dict(rope=A, n_pos=128)
CALLS = {
    "append": ("tenzo_hip_kv4_append", dict(k=A, v=A, dtype=0, ks=256, vs=256, **POOLS, Hkv=2,
                                            **SEQS, **ROPE, stream=None)),
    "read": ("tenzo_hip_kv4_read", dict(**POOLS, Hkv=2, **SEQS, k=A, v=A, dtype=0, stream=None)),
    "attn": ("tenzo_hip_attn_kv4", dict(q=A, dtype=0, qs=1024, **POOLS, Hq=8, Hkv=2, **SEQS,
                                        **ROPE, out=A, os=1024, ws=A, ws_bytes=1 << 40,
                                        stream=None)),
    "beam": ("tenzo_hip_beam_select", dict(x=A, stride=100, s=A, B=2, W=4, V=100, k=8, os=A, ob=A,
                                           ot=A, ws=A, ws_bytes=1 << 40, stream=None)),
    "reorder": ("tenzo_hip_beam_reorder_paged", dict(
        parents=A, ps=4, tables=A, ts=8, width=8, ctx=A, B=2, W=4, pk=A, pv=A, pks=A, pvs=A,
        n_blocks=4, n_layers=2, Hkv=2, row_bytes=64, stream=None)),
}
CACHE_BAD = [dict(pk=None), dict(pvs=None), dict(pk=A + 4), dict(pks=A + 2), dict(layer=2),
             dict(layer=-1), dict(n_layers=0), dict(n_blocks=-1), dict(n_blocks=1 << 31),
             dict(Hkv=0), dict(tables=None), dict(stride=7), dict(width=-1), dict(ctx=None),
             dict(T=4), dict(B=-1), dict(T=-1), dict(dtype=2), dict(width=1 << 28)]
BAD = {
    "append": CACHE_BAD + [dict(k=None), dict(v=None), dict(ks=255), dict(vs=0), dict(n_pos=-1)],
    "read": CACHE_BAD + [dict(k=None), dict(v=None), dict(k=A + 4)],
    "attn": CACHE_BAD + [dict(q=None), dict(out=None), dict(qs=1023), dict(os=1000), dict(Hq=7),
                         dict(Hq=34), dict(Hq=0), dict(n_pos=-1)],
    "beam": [dict(x=None), dict(s=None), dict(os=None), dict(ob=None), dict(ot=None),
             dict(ws=None), dict(ws_bytes=8), dict(ws=A + 4), dict(stride=99), dict(B=-1),
             dict(W=0), dict(W=65), dict(k=0), dict(k=65), dict(V=0), dict(V=1), dict(V=1 << 29)],
    "reorder": [dict(parents=None), dict(tables=None), dict(ctx=None), dict(pk=None),
                dict(pv=A + 8), dict(pks=A + 1), dict(ps=3), dict(ts=7), dict(width=-1),
                dict(B=-1), dict(B=65536), dict(W=0), dict(W=65), dict(n_layers=0), dict(Hkv=0),
                dict(n_blocks=-1), dict(row_bytes=32)],
}


@pytest.mark.parametrize("name,bad", [(n, b) for n in BAD for b in BAD[n]],
                         ids=lambda v: v if isinstance(v, str) else "_".join(v))
def test_c_refusals(name, bad):
    fn, good = CALLS[name]
    L = _lib.load()
    if name == "read" and "n_pos" in bad:
        pytest.skip("no rotation")
    rc = getattr(L, fn)(*{**good, **bad}.values())
    assert rc in (-1, -2, -3, -4, -5, -6) and L.tenzo_hip_last_error()


@pytest.mark.parametrize("name", ["append", "read", "attn"])
def test_c_empty_calls(name):
    """No rows: nothing to do, whatever the pointers."""
    fn, good = CALLS[name]
    none = {k: None for k, v in good.items() if v == A}
    assert getattr(_lib.load(), fn)(*{**good, **none, "B": 0, "T": 0}.values()) == 0


@pytest.fixture
def cpu(monkeypatch):
    """CPU tensors pass for tensors of the current device (their device number is -1); what is
    refused is refused before the library is called."""
    monkeypatch.setattr(ops, "_dev", lambda: -1)
    monkeypatch.setattr(ops, "_stream", lambda: 0)

    def no_call(*a):
        raise AssertionError("the library was called")

    class Lib:
        def __getattr__(self, name):
            return no_call

    monkeypatch.setattr(ops._lib, "load", lambda: Lib())


def _cache(Hkv=2, B=3, width=4):
    return [*ops.kv4_pool(5, 2, Hkv, device="cpu"), torch.zeros((B, width), dtype=torch.int32),
            torch.ones(B, dtype=torch.int32), 0]


def _swap(args, i, v):
    return [*args[:i], v, *args[i + 1:]]


@pytest.mark.parametrize("i,make", [
    (0, lambda t: t[..., :32]), (0, lambda t: t.to(torch.int8)), (1, lambda t: t[:4]),
    (2, lambda t: t[..., 0]), (3, lambda t: t.float()), (0, lambda t: t.transpose(1, 2)),
    (4, lambda t: t.long()), (4, lambda t: t[0]), (4, lambda t: t.T.contiguous().T),
    (5, lambda t: t[:2]), (5, lambda t: t.long()), (4, lambda t: t[:2])])
def test_ops_refuse_caches(cpu, i, make):
    args = _cache()
    args = _swap(args, i, make(args[i]))
    x = torch.zeros((3, 256))
    for call in (lambda: ops.kv4_append(x, x, *args), lambda: ops.attn_kv4(x, *args),
                 lambda: ops.kv4_read(*args, rows=3)):
        with pytest.raises(ValueError):
            call()


def test_ops_refuse_rows(cpu):
    args = _cache()
    x = torch.zeros((3, 256))
    cu = torch.zeros(4, dtype=torch.int32)
    bad = [lambda: ops.kv4_append(x[:2], x[:2], *args), lambda: ops.kv4_append(x, x[:, :128], *args),
           lambda: ops.kv4_append(x.double(), x, *args), lambda: ops.kv4_append(x, x.half(), *args),
           lambda: ops.kv4_append(x.T.contiguous().T, x, *args),
           lambda: ops.kv4_append(x, x, *args, cu_q=cu[:3]),
           lambda: ops.kv4_append(x, x, *args, cu_q=cu.long()),
           lambda: ops.kv4_append(x, x, *args, rope_cs=torch.zeros((9, 64))),
           lambda: ops.kv4_append(x, x, *args, rope_cs=torch.zeros((9, 128)).double()),
           lambda: ops.kv4_read(*args, cu_q=cu), lambda: ops.kv4_read(*args, rows=4),
           lambda: ops.kv4_append(torch.zeros((7, 256)), torch.zeros((6, 256)), *args, cu_q=cu),
           lambda: ops.attn_kv4(torch.zeros((3, 200)), *args),
           lambda: ops.attn_kv4(torch.zeros((3, 384)), *args),
           lambda: ops.attn_kv4(x, *args, out=torch.zeros((3, 128))),
           lambda: ops.attn_kv4(x.bfloat16(), *args)]
    for call in bad:
        with pytest.raises(ValueError):
            call()


def test_ops_refuse_other_devices(cpu, monkeypatch):
    monkeypatch.setattr(ops, "_dev", lambda: 0)
    args = _cache()
    x = torch.zeros((3, 256))
    for call in (lambda: ops.kv4_append(x, x, *args), lambda: ops.attn_kv4(x, *args),
                 lambda: ops.kv4_read(*args),
                 lambda: ops.beam_select(torch.zeros((1, 2, 9)), torch.zeros((1, 2)), 2),
                 lambda: ops.beam_reorder_paged(torch.zeros((1, 3), dtype=torch.int32), *args[4:6],
                                                *args[:4])):
        with pytest.raises(ValueError):
            call()


def test_ops_refuse_beams(cpu):
    x, s = torch.zeros((2, 3, 50)), torch.zeros((2, 3))
    for call in (lambda: ops.beam_select(x[0], s, 2), lambda: ops.beam_select(x, s[:1], 2),
                 lambda: ops.beam_select(x.double(), s, 2), lambda: ops.beam_select(x, s.half(), 2),
                 lambda: ops.beam_select(x.transpose(0, 1), s.T, 2),
                 lambda: ops.beam_select(x.transpose(1, 2), torch.zeros((2, 50)), 2)):
        with pytest.raises(ValueError):
            call()
    pools = ops.kv4_pool(5, 2, 2, device="cpu")
    p = torch.zeros((2, 3), dtype=torch.int32)
    t, c = torch.zeros((6, 4), dtype=torch.int32), torch.ones(6, dtype=torch.int32)
    for a in ((p.long(), t, c, *pools), (p[0], t, c, *pools), (p, t[:5], c, *pools),
              (p, t, c[:2], *pools), (p, t.long(), c, *pools), (p, t, c, pools[2], *pools[1:]),
              (p, t, c, pools[0].float(), *pools[1:]), (p, t, c, *pools[:3], pools[3][..., 0]),
              (p, t.T.contiguous().T, c, *pools)):
        with pytest.raises(ValueError):
            ops.beam_reorder_paged(*a)


# ------------------------------------------------------------ plain forms ----

def test_plain_quantizer():
    """Against the distance to every representable value."""
    rng = np.random.default_rng(0)
    x = rng.standard_normal((200, 128)) * np.exp(rng.standard_normal((200, 1)) * 5)
    c, e = plain.quantize(x)
    v = plain.values(c, e).reshape(200, 4, 32)
    g = x.reshape(200, 4, 32)
    scale = np.ldexp(1.0, e.astype(int) - 127)[..., None]
    assert (np.abs(g).max(-1) <= 7 * scale[..., 0]).all()
    assert (np.abs(g).max(-1) > 3.5 * scale[..., 0]).all()
    lv = np.concatenate([plain.LEVELS, -plain.LEVELS])
    best = np.abs(g[..., None] - lv * scale[..., None]).min(-1)
    np.testing.assert_allclose(np.abs(v - g), best, rtol=1e-12)


def test_plain_attention_is_softmax():
    rng = np.random.default_rng(1)
    pools = [rng.integers(0, 256, (3, 1, 1, 16, w), dtype=np.uint8) for w in (64, 64)]
    pools += [np.full((3, 1, 1, 16, 4), 127, np.uint8)] * 2
    tables, ctx = np.array([[2, 0]]), np.array([20])
    q = rng.standard_normal((1, 2, 128))
    out, tol = plain.attention(q, pools, tables, ctx, 0, None, None, np.zeros((1, 2, 128)))
    K = plain.values(pools[0][[2, 0], 0, 0], pools[2][[2, 0], 0, 0]).reshape(-1, 128)[:20]
    V = plain.values(pools[1][[2, 0], 0, 0], pools[3][[2, 0], 0, 0]).reshape(-1, 128)[:20]
    t = torch.softmax(torch.from_numpy(q[0] @ K.T / np.sqrt(128)), -1) @ torch.from_numpy(V)
    np.testing.assert_allclose(out[0], t.numpy(), rtol=1e-12, atol=1e-13)
    assert (tol > 0).all()
