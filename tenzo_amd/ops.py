"""Operator-level interface of the decode hot path on torch device tensors.

Mirrors the reference operator surface - ``ROCmRuntime::executeBitLinearTL1``
/ ``executeRMSNorm`` (reference ``src/runtime/ROCmRuntime.h:19-37``), the
free GEMV functions ``compute_linear_gguf_q4_0`` / ``_gptq`` / ``_awq``
(``TenzoEngine.cpp:1022-1175``), ``FusedKVCache::forward_attention_raw``
(``TenzoEngine.cpp:447-919``) and ``compute_logits`` (``:1634-1720``) - with
the same argument meaning; and, without a counterpart there, the operators of
batched beam decoding over a paged cache in 4 bits. Every call goes through
libtenzo_hip.so on the current torch stream; tensors must live on the GPU.
"""
from __future__ import annotations

import ctypes
import functools
import math

import torch

from . import _lib

F32, F16 = 0, 1


def _ptr(t: torch.Tensor | None):
    if t is None:
        return None
    if not t.is_cuda:
        raise ValueError("tenzo_amd ops take GPU tensors")
    if not t.is_contiguous():
        raise ValueError("tenzo_amd ops take contiguous tensors")
    return t.data_ptr()  # (the declared argument types convert it)


# The small calls' kernels take 5 to 10 us, so their Python side shows: no Stream object, pointer
# object or view where a number or the tensor itself will do. Per call, us, with them | without:
# gemv_q4_0 10.3 | 7.3, attn_int8_decode 14.6 | 11.4, rmsnorm_quant31 + bitlinear_tl1 22.2 | 16.5.
def _stream() -> int:
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def _rows(x: torch.Tensor, K: int) -> torch.Tensor:
    """x as contiguous rows of K: x.reshape(-1, K).contiguous()."""
    if x.dim() == 2 and x.shape[1] == K and x.is_contiguous():
        return x
    return x.reshape(-1, K).contiguous()


def _dtype_code(t: torch.Tensor) -> int:
    if t.dtype == torch.float32:
        return F32
    if t.dtype == torch.float16:
        return F16
    raise ValueError(f"unsupported dtype {t.dtype}")


# ------------------------------------------------------------------ TL1 ----

def tl1_packed_bytes(N: int, K: int) -> int:
    return int(_lib.load().tenzo_hip_tl1_packed_bytes(N, K))


def tl1_repack(w_tl1: torch.Tensor, N: int, K: int) -> torch.Tensor:
    """TL1 bytes [N/64][K/2][32] -> device GEMV layout (uint8 tensor)."""
    out = torch.empty(tl1_packed_bytes(N, K), dtype=torch.uint8, device=w_tl1.device)
    _lib.check(_lib.load().tenzo_hip_tl1_repack(_ptr(w_tl1), _ptr(out), N, K, _stream()),
               "tl1_repack")
    return out


def padded(K: int) -> int:
    return (K + 63) // 64 * 64


def rmsnorm_quant31(x: torch.Tensor, norm_w: torch.Tensor | None = None, eps: float = 1e-5,
                    do_norm: bool | None = None, want_y: bool = False):
    """build_lut's activation quantization of each row of x ([M][K] or [K]),
    optionally after rms_norm_raw. Returns (codes int8 [M][Kp], actq int32
    [M][2] viewed as {inv_scale(float bits), code_sum}, y or None)."""
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    M, K = x2.shape
    codes = torch.empty((M, padded(K)), dtype=torch.int8, device=x.device)
    q = torch.empty((M, 2), dtype=torch.int32, device=x.device)
    norm = bool(do_norm) if do_norm is not None else norm_w is not None
    y = torch.empty_like(x2) if (want_y and norm) else None
    _lib.check(_lib.load().tenzo_hip_rmsnorm_quant31(
        _ptr(x2), _ptr(norm_w), int(norm), eps, M, K, _ptr(codes), _ptr(q), _ptr(y), _stream()),
        "rmsnorm_quant31")
    return codes, q, y


def actq_inv_scale(q: torch.Tensor) -> torch.Tensor:
    return q[:, 0].contiguous().view(torch.float32)


def bitlinear_tl1(codes: torch.Tensor, q: torch.Tensor, w_packed: torch.Tensor, w_scale: float,
                  N: int, K: int, want_acc: bool = False):
    M = codes.shape[0]
    y = torch.empty((M, N), dtype=torch.float32, device=codes.device)
    acc = torch.empty((M, N), dtype=torch.int32, device=codes.device) if want_acc else None
    _lib.check(_lib.load().tenzo_hip_bitlinear_tl1(
        _ptr(codes), _ptr(q), _ptr(w_packed), w_scale, M, N, K, _ptr(y), _ptr(acc), _stream()),
        "bitlinear_tl1")
    return y, acc


def bitlinear_tl1_lut(codes: torch.Tensor, q: torch.Tensor, w_packed: torch.Tensor,
                      w_scale: float, N: int, K: int, want_acc: bool = False,
                      y: torch.Tensor | None = None):
    """bitlinear_tl1 by the reference's table method (a 16-entry table per
    activation pair in LDS, looked up per 4-bit weight pair): the same bits;
    kept to measure the two methods against each other."""
    M = codes.shape[0]
    if y is None:
        y = torch.empty((M, N), dtype=torch.float32, device=codes.device)
    acc = torch.empty((M, N), dtype=torch.int32, device=codes.device) if want_acc else None
    _lib.check(_lib.load().tenzo_hip_bitlinear_tl1_lut(
        _ptr(codes), _ptr(q), _ptr(w_packed), w_scale, M, N, K, _ptr(y), _ptr(acc), _stream()),
        "bitlinear_tl1_lut")
    return y, acc


def bitlinear_tl1_into(codes: torch.Tensor, q: torch.Tensor, w_packed: torch.Tensor,
                       w_scale: float, N: int, K: int, y: torch.Tensor) -> torch.Tensor:
    """bitlinear_tl1 writing into a caller-owned y (no allocation per call)."""
    M = codes.shape[0]
    _lib.check(_lib.load().tenzo_hip_bitlinear_tl1(
        _ptr(codes), _ptr(q), _ptr(w_packed), w_scale, M, N, K, _ptr(y), None, _stream()),
        "bitlinear_tl1")
    return y


def bitlinear_tl1_batch(codes: torch.Tensor, q: torch.Tensor, w_packed: torch.Tensor,
                        w_scale: float, N: int, K: int, want_acc: bool = False,
                        tile: int = 0, y: torch.Tensor | None = None):
    """The TL1 contraction of all M token rows of codes at once on int8 MFMA
    (prefill): the results of bitlinear_tl1, bit for bit."""
    M = codes.shape[0]
    if y is None:
        y = torch.empty((M, N), dtype=torch.float32, device=codes.device)
    acc = torch.empty((M, N), dtype=torch.int32, device=codes.device) if want_acc else None
    _lib.check(_lib.load().tenzo_hip_bitlinear_tl1_batch(
        _ptr(codes), _ptr(q), _ptr(w_packed), w_scale, M, N, K, _ptr(y), _ptr(acc), tile,
        _stream()), "bitlinear_tl1_batch")
    return y, acc


def bitlinear_tl1_f32(x: torch.Tensor, w_packed: torch.Tensor, w_scale: float, N: int,
                      K: int) -> torch.Tensor:
    """executeBitLinearTL1(act, w, out, M, K, N, scale) on device tensors."""
    x2 = _rows(x, K)
    M = x2.shape[0]
    y = torch.empty((M, N), dtype=torch.float32, device=x.device)
    _lib.check(_lib.load().tenzo_hip_bitlinear_tl1_f32(
        _ptr(x2), _ptr(w_packed), w_scale, M, N, K, _ptr(y), _stream()), "bitlinear_tl1_f32")
    return y


def rmsnorm(x: torch.Tensor, w: torch.Tensor | None, eps: float = 1e-5) -> torch.Tensor:
    """executeRMSNorm(in, w, out, dim, eps)."""
    y = torch.empty_like(x)
    _lib.check(_lib.load().tenzo_hip_rmsnorm(_ptr(x), _ptr(w), _ptr(y), x.numel(), eps,
                                             _stream()), "rmsnorm")
    return y


# ------------------------------------------------------------ attention ----

def rope_table(theta: float, pos0: int, n_pos: int, head_dim: int = 128) -> torch.Tensor:
    """Host-side cos/sin rows (reference RoPE angles) as a CPU float tensor."""
    cs = torch.empty((n_pos, head_dim), dtype=torch.float32)
    _lib.load().tenzo_hip_rope_table(theta, head_dim, pos0, n_pos,
                                     ctypes.c_void_p(cs.data_ptr()))
    return cs


def attn_int8_decode(q, k_new, v_new, kc, vc, ks, vs, rope_cs, pos: int, want_rot=False):
    """forward_attention_raw for B sequences at position pos.

    q [B][Hq*128], k_new/v_new [B][Hkv*128] fp32; kc/vc [B][Hkv][max_seq][128]
    int8 and ks/vs [B][Hkv][max_seq] fp16 (updated in place at pos);
    rope_cs [128] fp32 on the device. Returns out [B][Hq*128] (and rotated
    q, k when want_rot)."""
    B, Hkv, max_seq, D = kc.shape
    Hq = q.numel() // (B * D)
    out = torch.empty((B, Hq * D), dtype=torch.float32, device=q.device)
    q_rot = torch.empty_like(out) if want_rot else None
    k_rot = torch.empty((B, Hkv * D), dtype=torch.float32, device=q.device) if want_rot else None
    _lib.check(_lib.load().tenzo_hip_attn_int8_decode(
        _ptr(q), _ptr(k_new), _ptr(v_new), _ptr(kc), _ptr(vc), _ptr(ks), _ptr(vs), _ptr(rope_cs),
        B, Hq, Hkv, max_seq, pos, _ptr(out), _ptr(q_rot), _ptr(k_rot), _stream()),
        "attn_int8_decode")
    return (out, q_rot, k_rot) if want_rot else out


KV_TERN_MODES = {"tl1_fused": 1, "popcount_fused": 2}


def attn_tern_decode(mode, q, k_new, v_new, kb, vb, ks, vs, rope_cs, pos: int, want_rot=False):
    """forward_attention_raw in a ternary KV mode ("tl1_fused" / "popcount_fused",
    or 1 / 2) for B sequences at position pos.

    kb/vb [B][Hkv][max_seq][32] uint8 rows and ks/vs [B][Hkv][max_seq] fp32
    (updated in place at pos); the rest as attn_int8_decode."""
    mode = KV_TERN_MODES.get(mode, mode)
    B, Hkv, max_seq, R = kb.shape
    assert R == 32 and kb.dtype == torch.uint8 and ks.dtype == torch.float32
    D = 128
    Hq = q.numel() // (B * D)
    out = torch.empty((B, Hq * D), dtype=torch.float32, device=q.device)
    q_rot = torch.empty_like(out) if want_rot else None
    k_rot = torch.empty((B, Hkv * D), dtype=torch.float32, device=q.device) if want_rot else None
    _lib.check(_lib.load().tenzo_hip_attn_tern_decode(
        int(mode), _ptr(q), _ptr(k_new), _ptr(v_new), _ptr(kb), _ptr(vb), _ptr(ks), _ptr(vs),
        _ptr(rope_cs), B, Hq, Hkv, max_seq, pos, _ptr(out), _ptr(q_rot), _ptr(k_rot), _stream()),
        "attn_tern_decode")
    return (out, q_rot, k_rot) if want_rot else out


def attn_paged_int8_decode(q, k_new, v_new, pk, pv, pks, pvs, block_table, layer: int, rope_cs,
                           pos: int):
    """PagedKVCache::forward_attention_raw for one layer at position pos (batch 1).

    pk/pv [blocks][n_layers][Hkv][16][128] int8 and pks/pvs [blocks][n_layers][Hkv][16]
    fp32 (updated in place at pos); block_table int32 covering position pos."""
    nb, n_layers, Hkv, page, D = pk.shape
    assert page == 16 and pk.dtype == torch.int8 and pks.dtype == torch.float32
    assert block_table.dtype == torch.int32 and block_table.numel() * 16 > pos
    Hq = q.numel() // D
    out = torch.empty((1, Hq * D), dtype=torch.float32, device=q.device)
    _lib.check(_lib.load().tenzo_hip_attn_paged_int8_decode(
        _ptr(q), _ptr(k_new), _ptr(v_new), _ptr(pk), _ptr(pv), _ptr(pks), _ptr(pvs),
        _ptr(block_table), n_layers, layer, _ptr(rope_cs), Hq, Hkv, pos, _ptr(out), _stream()),
        "attn_paged_int8_decode")
    return out


# ------------------------------------------------- paged cache in 4 bits ----

KV4_PAGE = 16


_dev = torch._C._cuda_getDevice


@functools.lru_cache(4096)
def _attn_kv4_ws(*args: int) -> int:
    return _lib.load().tenzo_hip_attn_kv4_ws_bytes(*args)


@functools.lru_cache(4096)
def _beam_select_ws(*args: int) -> int:
    return _lib.load().tenzo_hip_beam_select_ws_bytes(*args)


def _on(t: torch.Tensor, dev: int, dtype: torch.dtype, name: str) -> int:
    """The address of a tensor of the current device (the kernels run on its stream)."""
    if t.get_device() != dev:
        raise ValueError(f"{name}: on {t.device}, the current device is cuda:{dev}")
    if t.dtype is not dtype:
        raise ValueError(f"{name}: {t.dtype}, not {dtype}")
    return t.data_ptr()


def _whole(t: torch.Tensor, dev: int, dtype: torch.dtype, name: str) -> int:
    if not t.is_contiguous():
        raise ValueError(f"{name}: not contiguous")
    return _on(t, dev, dtype, name)


def _row_stride(t: torch.Tensor, cols: int, name: str) -> int:
    """Elements between the rows of t, [rows][cols] or more dims that fold to it."""
    shape, st = t.shape, t.stride()
    if len(shape) == 2 and shape[1] == cols and st[1] == 1:
        return st[0] if shape[0] > 1 else cols
    if math.prod(shape[1:]) == cols and (not t.numel() or t[0].is_contiguous()):
        return st[0] if shape[0] > 1 else cols
    raise ValueError(f"{name}: {tuple(shape)} with strides {st}, not rows of {cols}")


def _row_args(t: torch.Tensor, cols: int, dev: int, dtype: torch.dtype, name: str):
    """The address of t and the elements between its rows, checked."""
    shape = t.shape
    if len(shape) == 2 and shape[1] == cols and t.dtype is dtype and t.get_device() == dev:
        between, step = t.stride()
        if step == 1:
            return t.data_ptr(), between if shape[0] > 1 else cols
    return _on(t, dev, dtype, name), _row_stride(t, cols, name)


def kv4_pool(n_blocks: int, n_layers: int, n_kv_heads: int, device="cuda"):
    """Empty pools (pk, pv, pks, pvs) of n_blocks 16-token pages of a cache in 4 bits: codes
    [blocks][layers][kv heads][16][64] and scales [blocks][layers][kv heads][16][4], uint8."""
    shape = (n_blocks, n_layers, n_kv_heads, KV4_PAGE)
    return tuple(torch.zeros((*shape, w), dtype=torch.uint8, device=device)
                 for w in (64, 64, 4, 4))


# (The calls on a cache check a dozen tensors, and the smallest run for 4 us on the GPU: each
# property is asked for once and the words for what is wrong are looked for afterwards. Host side
# of a call: append 9 us, attn 15, select 13 (two launches each), reorder 8; the sizes of
# workspaces, a function of the arguments, are asked for once.)
_U8, _I32, _F32 = torch.uint8, torch.int32, torch.float32


def _kv4_cache(pk, pv, pks, pvs, block_tables, ctx_lens, cu_q, layer, rows, dev):
    """The arguments that the calls on a cache share, checked: (pool addresses), (n_blocks,
    n_layers, layer, Hkv), (tables, stride, width, lengths, cu_q, B, rows)."""
    shape, tshape, tstride = pk.shape, block_tables.shape, block_tables.stride()
    if (len(shape) == 5 and len(tshape) == 2 and shape[4] == 64 and shape[3] == KV4_PAGE
            and pv.shape == shape and pks.shape == (*shape[:4], 4) and pvs.shape == pks.shape
            and pk.dtype is _U8 and pv.dtype is _U8 and pks.dtype is _U8 and pvs.dtype is _U8
            and pk.is_contiguous() and pv.is_contiguous() and pks.is_contiguous()
            and pvs.is_contiguous() and block_tables.dtype is _I32 and ctx_lens.dtype is _I32
            and (tstride[1] == 1 or tshape[1] < 2) and ctx_lens.is_contiguous()
            and ctx_lens.shape == tshape[:1] and pk.get_device() == dev
            and pv.get_device() == dev and pks.get_device() == dev and pvs.get_device() == dev
            and block_tables.get_device() == dev and ctx_lens.get_device() == dev):
        B, width = tshape
        if cu_q is None:
            if rows == B:
                return ((pk.data_ptr(), pv.data_ptr(), pks.data_ptr(), pvs.data_ptr()),
                        (shape[0], shape[1], layer, shape[2]),
                        (block_tables.data_ptr(), tstride[0] if B > 1 else width, width,
                         ctx_lens.data_ptr(), None, B, rows))
            raise ValueError(f"{rows} rows for {B} sequences of one token: pass cu_q")
        if cu_q.shape == (B + 1,):
            return ((pk.data_ptr(), pv.data_ptr(), pks.data_ptr(), pvs.data_ptr()),
                    (shape[0], shape[1], layer, shape[2]),
                    (block_tables.data_ptr(), tstride[0] if B > 1 else width, width,
                     ctx_lens.data_ptr(), _whole(cu_q, dev, _I32, "cu_q"), B, rows))
        raise ValueError(f"cu_q: {tuple(cu_q.shape)}, not ({B + 1},)")
    if len(shape) != 5 or shape[3:] != (KV4_PAGE, 64) or pv.shape != shape:
        raise ValueError(f"pk, pv: {tuple(shape)}, {tuple(pv.shape)}, not "
                         "[blocks][layers][kv heads][16][64]")
    if pks.shape != (*shape[:4], 4) or pvs.shape != pks.shape:
        raise ValueError(f"pks, pvs: {tuple(pks.shape)}, {tuple(pvs.shape)}, not "
                         "[blocks][layers][kv heads][16][4] of the codes")
    for t, name in ((pk, "pk"), (pv, "pv"), (pks, "pks"), (pvs, "pvs")):
        _whole(t, dev, _U8, name)
    if len(tshape) != 2 or (tshape[1] > 1 and tstride[1] != 1):
        raise ValueError("block_tables: a row of page numbers per sequence")
    _on(block_tables, dev, _I32, "block_tables")
    _whole(ctx_lens, dev, _I32, "ctx_lens")
    raise ValueError(f"ctx_lens: {tuple(ctx_lens.shape)}, not a length for each of {tshape[0]} "
                     "sequences")


def _rope_rows(rope_cs, dev):
    if rope_cs is None:
        return None, 0
    shape = rope_cs.shape
    if len(shape) != 2 or shape[1] != 128 or not shape[0]:  # (none at all would mean no rotation)
        raise ValueError(f"rope_cs: {tuple(shape)}, not [positions][128]")
    if rope_cs.dtype is _F32 and rope_cs.get_device() == dev and rope_cs.is_contiguous():
        return rope_cs.data_ptr(), shape[0]
    return _whole(rope_cs, dev, _F32, "rope_cs"), shape[0]


def kv4_append(k, v, pk, pv, pks, pvs, block_tables, ctx_lens, layer: int, rope_cs=None,
               cu_q=None) -> None:
    """Rotates the keys of new tokens, rounds keys and values to 4 bits and writes them into
    the paged cache (pools of kv4_pool, updated in place).

    k, v [T][Hkv*128] (or [T][Hkv][128]) fp32 or fp16, rows any stride apart (slices of a
    fused q | k | v do); block_tables int32 [B][pages], ctx_lens int32 [B], the new tokens
    included. cu_q int32 [B+1]: sequence b's rows are cu_q[b] .. cu_q[b+1]-1, at its last
    positions; None: row b is sequence b's one new token. rope_cs: rows cos | sin of
    positions 0, 1, ... (rope_table; None: no rotation). Lengths of 0 or less, or above what
    the tables or rope_cs hold, are padding slots; pages outside the pool are skipped."""
    dev = _dev()
    T = k.shape[0]
    pools, where, seqs = _kv4_cache(pk, pv, pks, pvs, block_tables, ctx_lens, cu_q, layer, T, dev)
    dt, dtype, cols = _dtype_code(k), k.dtype, where[3] * 128
    kp, ks = _row_args(k, cols, dev, dtype, "k")
    vp, vs = _row_args(v, cols, dev, dtype, "v")
    if v.shape[0] != T:
        raise ValueError(f"{T} rows of k, {v.shape[0]} of v")
    rc = _lib.load().tenzo_hip_kv4_append(kp, vp, dt, ks, vs, *pools, *where, *seqs,
                                          *_rope_rows(rope_cs, dev), _stream())
    if rc:
        _lib.check(rc, "kv4_append")


def kv4_read(pk, pv, pks, pvs, block_tables, ctx_lens, layer: int, rows: int | None = None,
             cu_q=None, dtype=torch.float32):
    """The cached keys (rotated) and values at the positions of a call's rows, as kv4_append
    places them: (k, v) [rows][Hkv][128]. rows: as many as the call has (with cu_q; without,
    one a sequence). Rows that stand nowhere are zeros."""
    dev = _dev()
    if rows is None:
        if cu_q is not None:
            raise ValueError("kv4_read: rows is needed with cu_q")
        rows = block_tables.shape[0]
    pools, where, seqs = _kv4_cache(pk, pv, pks, pvs, block_tables, ctx_lens, cu_q, layer, rows,
                                    dev)
    k = pk.new_empty((rows, where[3], 128), dtype=dtype)
    v = torch.empty_like(k)
    _lib.check(_lib.load().tenzo_hip_kv4_read(*pools, *where, *seqs, k.data_ptr(), v.data_ptr(),
                                              _dtype_code(k), _stream()), "kv4_read")
    return k, v


def attn_kv4(q, pk, pv, pks, pvs, block_tables, ctx_lens, layer: int, rope_cs=None, cu_q=None,
             out=None):
    """Attention over a paged cache in 4 bits: q [T][Hq*128] (or [T][Hq][128]) fp32 or fp16,
    rotated at its rows' positions (rope_cs, None: not), each row attending to the positions
    up to its own; the other arguments as kv4_append, which comes first. Returns out like q
    (into `out` when given, which must not overlap q: rows behind the last sequence stay as they
    are; they are not initialised otherwise). Rows that see no token are zeros."""
    dev = _dev()
    T = q.shape[0]
    pools, where, seqs = _kv4_cache(pk, pv, pks, pvs, block_tables, ctx_lens, cu_q, layer, T, dev)
    cols = q.shape[1] if q.dim() == 2 else math.prod(q.shape[1:])
    Hkv = where[3]
    if Hkv < 1 or cols % 128 or (cols // 128) % Hkv:
        raise ValueError(f"q: {tuple(q.shape)}, not rows of heads of 128 over {Hkv} kv heads")
    dt, dtype = _dtype_code(q), q.dtype
    qp, qs = _row_args(q, cols, dev, dtype, "q")
    if out is None:
        out = q.new_empty(q.shape)
        op, os = out.data_ptr(), cols
    elif out.shape == q.shape:
        op, os = _row_args(out, cols, dev, dtype, "out")
    else:
        raise ValueError(f"out: {tuple(out.shape)}, q: {tuple(q.shape)}")
    rope = _rope_rows(rope_cs, dev)
    if not T:
        return out
    Hq = cols // 128
    nbytes = _attn_kv4_ws(T, seqs[5], Hq, Hkv, seqs[2], cu_q is not None, dt)
    ws = pk.new_empty(nbytes) if nbytes else None  # (held until the launch)
    rc = _lib.load().tenzo_hip_attn_kv4(qp, dt, qs, *pools, *where[:3], Hq, Hkv, *seqs, *rope,
                                        op, os, ws.data_ptr() if nbytes else None, nbytes, _stream())
    if rc:
        _lib.check(rc, "attn_kv4")
    return out


# -------------------------------------------------------- quantized GEMV ---

def gemv_q4_0(act: torch.Tensor, w: torch.Tensor, K: int, N: int) -> torch.Tensor:
    a = _rows(act, K)
    B = a.shape[0]
    y = torch.empty((B, N), dtype=torch.float32, device=act.device)
    _lib.check(_lib.load().tenzo_hip_gemv_q4_0(_ptr(a), _dtype_code(a), _ptr(w), _ptr(y), K, N,
                                               B, _stream()), "gemv_q4_0")
    return y


def gemv_q8_0(act: torch.Tensor, w: torch.Tensor, K: int, N: int) -> torch.Tensor:
    """compute_linear_gguf_q8_0 for B activation rows (fp32 or fp16) of K:
    w = N rows of K/32 blocks of 34 bytes. Returns [B][N] fp32."""
    a = _rows(act, K)
    B = a.shape[0]
    y = torch.empty((B, N), dtype=torch.float32, device=act.device)
    _lib.check(_lib.load().tenzo_hip_gemv_q8_0(_ptr(a), _dtype_code(a), _ptr(w), _ptr(y), K, N,
                                               B, _stream()), "gemv_q8_0")
    return y


def gemv_q4_0_q8_0(qa: torch.Tensor, w: torch.Tensor, K: int, N: int) -> torch.Tensor:
    B = qa.numel() // (K // 32 * 34)
    y = torch.empty((B, N), dtype=torch.float32, device=qa.device)
    _lib.check(_lib.load().tenzo_hip_gemv_q4_0_q8_0(_ptr(qa), _ptr(w), _ptr(y), K, N, B,
                                                    _stream()), "gemv_q4_0_q8_0")
    return y


def _gemv_gq(fn_name, act, qweight, scales, qzeros, K, N, group):
    a = _rows(act, K)
    B = a.shape[0]
    y = torch.empty((B, N), dtype=torch.float32, device=act.device)
    fn = getattr(_lib.load(), fn_name)
    _lib.check(fn(_ptr(a), _dtype_code(a), _ptr(qweight), _ptr(scales), _dtype_code(scales),
                  _ptr(qzeros), _ptr(y), K, N, group, B, _stream()), fn_name)
    return y


def gemv_gptq(act, qweight, scales, qzeros, K: int, N: int, group: int = 128):
    return _gemv_gq("tenzo_hip_gemv_gptq", act, qweight, scales, qzeros, K, N, group)


def gemv_awq(act, qweight, scales, qzeros, K: int, N: int, group: int = 128):
    return _gemv_gq("tenzo_hip_gemv_awq", act, qweight, scales, qzeros, K, N, group)


# -------------------------------------------------------------- LM head ----

def i8_packed_bytes(V: int, H: int) -> int:
    return int(_lib.load().tenzo_hip_i8_packed_bytes(V, H))


def i8_rows_repack(w: torch.Tensor, V: int, H: int) -> torch.Tensor:
    out = torch.empty(i8_packed_bytes(V, H), dtype=torch.uint8, device=w.device)
    _lib.check(_lib.load().tenzo_hip_i8_rows_repack(_ptr(w), _ptr(out), V, H, _stream()),
               "i8_rows_repack")
    return out


def lm_head_i8(x, norm_w, w_packed, scales, V: int, H: int, eps: float = 1e-5):
    logits = torch.empty(V, dtype=torch.float32, device=x.device)
    _lib.check(_lib.load().tenzo_hip_lm_head_i8(_ptr(x), _ptr(norm_w), eps, _ptr(w_packed),
                                                _ptr(scales), _ptr(logits), V, H, _stream()),
               "lm_head_i8")
    return logits


def actquant127(x: torch.Tensor, norm_w: torch.Tensor | None = None, eps: float = 1e-5):
    """compute_logits' activation quantization of each row of x ([M][K] or
    [K]), after rms_norm_raw when norm_w is given. Returns (codes int8 [M][K],
    actq int32 [M][2])."""
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    M, K = x2.shape
    codes = torch.empty((M, K), dtype=torch.int8, device=x.device)
    q = torch.empty((M, 2), dtype=torch.int32, device=x.device)
    _lib.check(_lib.load().tenzo_hip_rmsnorm_quant127(
        _ptr(x2), _ptr(norm_w), int(norm_w is not None), eps, M, K, _ptr(codes), _ptr(q),
        _stream()), "rmsnorm_quant127")
    return codes, q


def lm_head_i8_codes_into(codes, q, w_packed, scales, V: int, H: int, logits,
                          idx=None):
    """The LM-head GEMV on precomputed codes into caller-owned logits (and the
    fused greedy argmax into idx when given)."""
    _lib.check(_lib.load().tenzo_hip_lm_head_i8_codes(
        _ptr(codes), _ptr(q), _ptr(w_packed), _ptr(scales), _ptr(logits), V, H, _ptr(idx),
        _stream()), "lm_head_i8_codes")
    return logits


def argmax(logits: torch.Tensor) -> torch.Tensor:
    out = torch.empty(1, dtype=torch.int32, device=logits.device)
    _lib.check(_lib.load().tenzo_hip_argmax(_ptr(logits), logits.numel(), _ptr(out), _stream()),
               "argmax")
    return out


def sample_top_k_top_p(logits: torch.Tensor, top_k: int, top_p: float, temperature: float,
                       r: float) -> int:
    """sample_top_k_top_p's sampling branch on device logits with the draw r."""
    out = torch.empty(1, dtype=torch.int32, device=logits.device)
    _lib.check(_lib.load().tenzo_hip_sample_top_k_top_p(
        _ptr(logits), logits.numel(), int(top_k), float(top_p), float(temperature), float(r),
        _ptr(out), _stream()), "sample_top_k_top_p")
    return int(out.item())


def beam_select(logits: torch.Tensor, scores: torch.Tensor, k: int):
    """The best k continuations of each request: logits [B][W][V] fp32 (beams any stride
    apart), scores [B][W] fp32, the beams' running log-probabilities. Returns (scores [B][k]
    fp32, beams [B][k] int32, tokens [B][k] int32) of the candidates scores + log_softmax(
    logits), in the falling order that they have in 64 bits; among equal ones the lower beam,
    then the larger logit, then the lower token comes first. Scores are within 1.25e-6 and half
    a step of fp32. NaN and +inf count as -inf, which comes last."""
    dev = _dev()
    shape = logits.shape
    if len(shape) != 3 or scores.shape != shape[:2]:
        raise ValueError(f"logits [B][W][V] and scores [B][W]: {tuple(shape)}, "
                         f"{tuple(scores.shape)}")
    (B, W, V), (between, ld, step) = shape, logits.stride()
    ld = ld if W > 1 else between if B > 1 else V
    if (V > 1 and step != 1) or (B > 1 and between != W * ld):
        raise ValueError(f"logits: strides {logits.stride()}")
    lp = _on(logits, dev, torch.float32, "logits")
    sp = _whole(scores, dev, torch.float32, "scores")
    L = _lib.load()
    nbytes = _beam_select_ws(B, W, V, k)
    ws = logits.new_empty(nbytes // 4)  # (whole numbers of 8 bytes; held until the launch)
    out = scores.new_empty((B, k))
    beams = torch.empty_like(out, dtype=torch.int32)
    tokens = torch.empty_like(beams)
    _lib.check(L.tenzo_hip_beam_select(lp, ld, sp, B, W, V, k, out.data_ptr(), beams.data_ptr(),
                                       tokens.data_ptr(), ws.data_ptr(), nbytes, _stream()),
               "beam_select")
    return out, beams, tokens


def beam_reorder_paged(parents, block_tables, ctx_lens, pk, pv, pks, pvs) -> None:
    """Reorders the paged caches of B requests with W beams in place: slot i of request b goes
    on from slot parents[b][i] (int32 [B][W], for instance beams[:, :W] of beam_select).

    block_tables int32 [B*W][pages] and ctx_lens int32 [B*W] (the beams of a request have one
    length c): table entries of full pages (below c // 16) are taken from the parent, the c %
    16 rows of the page in progress are copied into the slot's own page c // 16, in all layers
    and heads. A slot's pages from c // 16 on have to be its own. Pools of kv4_pool or of the
    int8 paged cache (codes [blocks][layers][kv heads][16][128] int8, scales [..][16] fp32)."""
    dev = _dev()
    if parents.dim() != 2 or (parents.shape[1] > 1 and parents.stride(1) != 1):
        raise ValueError("parents: a row of W slots per request")
    B, W = parents.shape
    if block_tables.dim() != 2 or block_tables.shape[0] != B * W or (
            block_tables.shape[1] > 1 and block_tables.stride(1) != 1):
        raise ValueError(f"block_tables: {tuple(block_tables.shape)}, not a row of page numbers "
                         f"for each of {B} x {W} beams")
    if ctx_lens.shape != (B * W,):
        raise ValueError(f"ctx_lens: {tuple(ctx_lens.shape)}, not ({B * W},)")
    shape = tuple(pk.shape)
    kv4 = pk.dtype == torch.uint8
    code, scale = (torch.uint8, torch.uint8) if kv4 else (torch.int8, torch.float32)
    if len(shape) != 5 or shape[3:] != (KV4_PAGE, 64 if kv4 else 128) or pv.shape != shape:
        raise ValueError(f"pk, pv: {shape}, {tuple(pv.shape)}")
    want = shape[:4] + ((4,) if kv4 else ())
    if pks.shape != want or pvs.shape != want:
        raise ValueError(f"pks, pvs: {tuple(pks.shape)}, {tuple(pvs.shape)}, not {want}")
    width = block_tables.shape[1]
    _lib.check(_lib.load().tenzo_hip_beam_reorder_paged(
        _on(parents, dev, torch.int32, "parents"), parents.stride(0) if B > 1 else W,
        _on(block_tables, dev, torch.int32, "block_tables"),
        block_tables.stride(0) if B * W > 1 else width, width,
        _whole(ctx_lens, dev, torch.int32, "ctx_lens"), B, W, _whole(pk, dev, code, "pk"),
        _whole(pv, dev, code, "pv"), _whole(pks, dev, scale, "pks"),
        _whole(pvs, dev, scale, "pvs"), shape[0], shape[1], shape[2], 64 if kv4 else 128,
        _stream()), "beam_reorder_paged")


def embed_i8(w_packed, scales, token: torch.Tensor, V: int, H: int) -> torch.Tensor:
    x = torch.empty(H, dtype=torch.float32, device=w_packed.device)
    _lib.check(_lib.load().tenzo_hip_embed_i8(_ptr(w_packed), _ptr(scales), _ptr(token), V, H,
                                              _ptr(x), _stream()), "embed_i8")
    return x
