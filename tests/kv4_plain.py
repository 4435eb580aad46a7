"""Plain numpy forms, in 64 bits, of the operators on a paged cache in 4 bits and of beam
search, written from their definitions (include/tenzo_hip.h)."""
import numpy as np

D, PAGE = 128, 16
LEVELS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
TOP = 1.75 * 2.0 ** 127


def quantize(x):
    """Rows [..., 128] (fp64) -> codes [..., 64], scales [..., 4]."""
    x = np.where(np.isnan(x), 0.0, np.clip(x, -TOP, TOP))
    g = x.reshape(*x.shape[:-1], 4, 32)
    mant, e = np.frexp(np.abs(g).max(-1))
    e = np.where(mant > 0.875, e - 2, e - 3)  # max <= 7 * 2^e
    e = np.where(np.abs(g).max(-1) == 0, -126, np.maximum(e, -126))
    a = np.ldexp(np.abs(g), -e[..., None])
    m = sum((a >= t if even else a > t).astype(np.uint8) for t, even in
            ((0.25, 0), (0.75, 1), (1.25, 0), (1.75, 1), (2.5, 0), (3.5, 1), (5, 0)))
    c = (m | (np.signbit(g).astype(np.uint8) << 3)).reshape(*x.shape[:-1], 64, 2)
    return c[..., 0] | (c[..., 1] << 4), (e + 127).astype(np.uint8)


def values(codes, scales):
    c = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], 4, 32)
    v = np.where(c & 8, -1.0, 1.0) * LEVELS[c & 7]
    s = np.ldexp(1.0, np.where(scales > 252, 0, scales.astype(int)) - 127)
    return (v * s[..., None]).reshape(*codes.shape[:-1], D)


def rotate(x, cs):
    x = np.asarray(x, np.float64)
    if cs is None:
        return x
    c, s = cs[:64].astype(np.float64), cs[64:].astype(np.float64)
    a, b = x[..., :64], x[..., 64:]
    return np.concatenate([a * c - b * s, a * s + b * c], -1)


def places(T, tables, ctx, cu, limit):
    """(sequence, position) of every row, None where it stands nowhere but in a sequence, and
    False behind the last one."""
    B = len(ctx)
    out = []
    for r in range(T):
        if cu is None:
            b, n, i = r, 1, 0
        else:
            b = int(np.searchsorted(cu[1:], r, side="right"))
            if b >= B:
                out.append(False)
                continue
            n, i = int(cu[b + 1] - cu[b]), r - int(cu[b])
        c = int(ctx[b])
        c = c if 0 < c <= limit else 0
        pos = c - n + i
        out.append((b, pos) if 0 <= pos < c else None)
    return out


def limit_of(tables, rope):
    n = tables.shape[1] * PAGE
    return n if rope is None else min(n, len(rope))


def append(k, v, pools, tables, ctx, layer, rope, cu):
    """Updates pools = (pk, pv, pks, pvs) in place; k, v [T][Hkv][128]."""
    pk, pv, pks, pvs = pools
    for r, at in enumerate(places(len(k), tables, ctx, cu, limit_of(tables, rope))):
        if not at:
            continue
        b, pos = at
        page = tables[b, pos // PAGE]
        if not 0 <= page < len(pk):
            continue
        where = (page, layer, slice(None), pos % PAGE)
        pk[where], pks[where] = quantize(rotate(k[r], None if rope is None else rope[pos]))
        pv[where], pvs[where] = quantize(np.asarray(v[r], np.float64))


def _largest(pools, table, c, layer):
    t = np.arange(c)
    page = table[t // PAGE]
    t, page = t[(page >= 0) & (page < len(pools[1]))], page[(page >= 0) & (page < len(pools[1]))]
    v = values(pools[1][page, layer, :, t % PAGE], pools[3][page, layer, :, t % PAGE])
    return np.abs(v).max((0, 2))


def attention(q, pools, tables, ctx, layer, rope, cu, out, parts_eps=0.0):
    """out [T][Hq][128] and how far fp32 sums may be from it, both updated for the rows of
    sequences. q [T][Hq][128]; parts_eps: what queries and weights are rounded to."""
    pk, pv, pks, pvs = pools
    Hq, Hkv = q.shape[1], pk.shape[2]
    G = Hq // Hkv
    u = 2.0 ** -24
    tol = np.zeros_like(out)
    for r, at in enumerate(places(len(q), tables, ctx, cu, limit_of(tables, rope))):
        if at is False:
            continue
        out[r] = 0.0
        if at is None:
            continue
        b, pos = at
        t = np.arange(pos + 1)
        page = tables[b, t // PAGE]
        ok = (page >= 0) & (page < len(pk))
        t, page = t[ok], page[ok]
        if not len(t):
            continue
        K = values(pk[page, layer, :, t % PAGE], pks[page, layer, :, t % PAGE])  # [n][Hkv][128]
        V = values(pv[page, layer, :, t % PAGE], pvs[page, layer, :, t % PAGE])
        vmax = _largest(pools, tables[b], int(ctx[b]), layer)
        x = rotate(q[r], None if rope is None else rope[pos]) / np.sqrt(D)
        mag = np.abs(np.asarray(q[r], np.float64)).reshape(Hq, 2, 64).sum(1) / np.sqrt(D)
        mag = np.concatenate([mag, mag], -1)  # bounds a rotated element's rounding
        for h in range(Hq):
            kk, vv = K[:, h // G], V[:, h // G]
            s = kk @ x[h]
            p = np.exp(s - s.max())
            p /= p.sum()
            out[r, h] = p @ vv
            # a score: the query's roundings (rotation 3, scale 2, parts), 128 products summed;
            # a weight: its score's error twice (it and the sum's), the difference's and the
            # exponential's rounding; the sums of n weights and n products
            # (and 2^-37 of a token's largest key element, times the query)
            ds = ((6 * u + parts_eps) * (np.abs(kk) @ mag[h]) +
                  128 * u * (np.abs(kk) @ np.abs(x[h])) +
                  2.0 ** -37 * np.abs(kk).max(-1) * np.abs(x[h]).sum()).max()
            dp = 2 * ds + (8 + 2 * (s.max() - s).max()) * u + parts_eps
            tol[r, h] = (dp + 2 * (len(t) + 32) * u) * (p @ np.abs(vv))
            # weights and products below 2^-126 have no relative precision (or count as 0)
            tol[r, h] += 2.0 ** -126 * (1 + np.abs(vv)).sum(0)
            # weights are held times 2^15 in fp16 parts, whose smallest step is 2^-24: half of it
            tol[r, h] += 2.0 ** -40 * p.max() * np.abs(vv).sum(0)
            tol[r, h] += 2.0 ** -37 * vmax[h // G]  # of the largest value that any row sees
    return out, tol


def beam_select(logits, scores, k):
    """(scores [B][k], beams, tokens); among equal scores the lower beam, then the larger logit
    (64 bits do not tell 1e-30 from 2e-30 in a score), then the lower token first."""
    x = np.where(logits < np.inf, logits, -np.inf).astype(np.float64)
    s = np.where(scores < np.inf, scores, -np.inf).astype(np.float64)
    B, W, V = x.shape
    top = x.max(-1, keepdims=True)
    top = np.where(np.isinf(top), 0, top)
    with np.errstate(divide="ignore", invalid="ignore"):
        lp = x - (top + np.log(np.exp(x - top).sum(-1, keepdims=True)))
    lp = np.where(x == -np.inf, -np.inf, lp) + s[..., None]
    flat = np.arange(W * V)
    order = np.stack([np.lexsort((flat, -x[b].ravel(), flat // V, -lp[b].ravel()))[:k]
                      for b in range(B)])
    return np.take_along_axis(lp.reshape(B, W * V), order, 1), order // V, order % V


def reorder(parents, tables, ctx, pools):
    B, W = parents.shape
    old, oldp = tables.copy(), [a.copy() for a in pools]
    for b in range(B):
        c = int(ctx[b * W])
        if not 0 < c <= tables.shape[1] * PAGE:
            continue
        full, fill = c // PAGE, c % PAGE
        for i in range(W):
            p = int(parents[b, i])
            if not 0 <= p < W:
                continue
            tables[b * W + i, :full] = old[b * W + p, :full]
            if fill:
                src, dst = old[b * W + p, full], old[b * W + i, full]
                if 0 <= src < len(pools[0]) and 0 <= dst < len(pools[0]):
                    for a, o in zip(pools, oldp):
                        a[dst, :, :, :fill] = o[src, :, :, :fill]
