"""Plain numpy forms, in 64 bits, of the operators on trees of drafted tokens, of rotary positions
and of the 8-bit product, written from their definitions (include/tenzo_hip.h)."""
import numpy as np

from tests.kv4_plain import D, PAGE, values


def sequences(T, ctx, cu, limit):
    """(first row, rows, length) of each sequence; length 0 for padding slots."""
    out = []
    for b in range(len(ctx)):
        first, end = (b, b + 1) if cu is None else (int(cu[b]), int(cu[b + 1]))
        n = end - first if 0 <= first < end <= T else 0
        c = int(ctx[b])
        out.append((first, n, c if 0 < c <= limit else 0))
    return out


def ancestors(parents):
    """For each node the set of its ancestors and itself."""
    out = []
    for i, p in enumerate(parents):
        out.append({i} | (out[p] if 0 <= p < i else set()))
    return out


def tree_plan(parents, ctx, cu, most, mask, positions):
    """Updates mask [T][words] and positions [T] for the rows of sequences."""
    for first, n, c in sequences(len(parents), ctx, cu, 2 ** 31 - 1):
        for i, seen in enumerate(ancestors(parents[first:first + n])):
            if i >= most:
                break
            there = c > 0 and c - n + i >= 0
            mask[first + i] = 0
            positions[first + i] = c - n + len(seen) - 1 if there else 0
            for j in seen if there else ():
                mask[first + i, j // 64] |= np.uint64(1) << np.uint64(j % 64)


def tree_accept(parents, tokens, target, pools, tables, ctx, cu, most):
    """(path, count, next, lens); pools updated in place."""
    B = len(ctx)
    path = np.full((B, most), -1, np.int32)
    count, last, lens = np.zeros(B, np.int32), np.full(B, -1, np.int32), ctx.copy()
    for b, (first, n, c) in enumerate(sequences(len(parents), ctx, cu, tables.shape[1] * PAGE)):
        if n == 0 or c < max(n, 1):
            continue
        prior, at, nodes = c - n, 0, []
        while at is not None and len(nodes) < most:
            nodes.append(at)
            at = next((v for v in range(at + 1, n) if parents[first + v] == at and
                       tokens[first + v] == target[first + at]), None)
        path[b, :len(nodes)] = nodes
        count[b], last[b], lens[b] = len(nodes), target[first + nodes[-1]], prior + len(nodes)
        for k, at in enumerate(nodes):
            src, dst = prior + at, prior + k
            sp, dp = tables[b, src // PAGE], tables[b, dst // PAGE]
            if src != dst and 0 <= sp < len(pools[0]) and 0 <= dp < len(pools[0]):
                for a in pools:
                    a[dp, :, :, dst % PAGE] = a[sp, :, :, src % PAGE]
    return path, count, last, lens


def attention_row(x, kk, vv, vmax, q_eps, w_eps):
    """softmax(kk x) vv of one row and head (x over sqrt(128) already) over the tokens that it sees,
    and how far fp32 sums may be from it; vmax: the largest value that any row sees."""
    u = 2.0 ** -24
    s = kk @ x
    p = np.exp(s - s.max())
    p /= p.sum()
    out = p @ vv
    # (of a query's dim also 2^-19 of the largest of its 32 dims in fp16 calls of 128 rows, which
    # hold it in 4 parts of 6 bits, and 2^-24 in fp32 ones: 5 parts)
    half = w_eps > 2.0 ** -12
    big = np.abs(x).reshape(4, 32).max(1).repeat(32)
    ds = ((3 * u + q_eps + 128 * u) * (np.abs(kk) @ np.abs(x)) +
          (2.0 ** -19 if half else 2.0 ** -24) * (np.abs(kk) @ big) +
          2.0 ** -37 * np.abs(kk).max(-1) * np.abs(x).sum()).max()
    # (weights p (1 + e), |e| <= w_eps, over their own sum: sum p (1 + e) v / sum p (1 + e) - sum p v
    # = sum p e (v - o) to first order, o the output, and sum p |e| |v - o| <= w_eps (sum p |v| + |o|)
    # <= 2 w_eps sum p |v|)
    dp = 2 * ds + (8 + 2 * (s.max() - s).max()) * u + 2 * w_eps
    tol = (dp + 2 * (len(s) + 32) * u) * (p @ np.abs(vv))
    tol += 2.0 ** -126 * (1 + np.abs(vv)).sum(0)
    # weights below fp16's normal numbers have a constant step, 2^-24 of what 1 stands for: 2^-15 of
    # the largest weight, in fp16 calls of 128 rows 2^-8; half of it
    tol += (2.0 ** -33 if half else 2.0 ** -40) * p.max() * np.abs(vv).sum(0)
    return out, tol + 2.0 ** -37 * vmax


def attention(q, mask, pools, tables, ctx, layer, cu, out, q_eps, w_eps):
    """out [T][Hq][128] and how far fp32 sums may be from it (the roundings that
    kv4_plain.attention counts, without those of a rotation), both updated for the rows of
    sequences. q [T][Hq][128]; q_eps, w_eps: what queries and weights are rounded to."""
    pk, pv, pks, pvs = pools
    Hq, Hkv = q.shape[1], pk.shape[2]
    G = Hq // Hkv
    tol = np.zeros_like(out)
    for b, (first, n, c) in enumerate(sequences(len(q), ctx, cu, tables.shape[1] * PAGE)):
        t = np.arange(c)
        page = tables[b, t // PAGE]
        held = (page >= 0) & (page < len(pk))
        at = np.where(held, page, 0)
        K = values(pk[at, layer, :, t % PAGE], pks[at, layer, :, t % PAGE])  # [c][Hkv][128]
        V = values(pv[at, layer, :, t % PAGE], pvs[at, layer, :, t % PAGE])
        vmax = np.abs(V[held]).max((0, 2)) if held.any() else np.zeros(Hkv)
        for i in range(n):
            r = first + i
            out[r] = 0.0
            node = t - (c - n)
            word = np.clip(node // 64, 0, mask.shape[1] - 1)
            bit = (mask[r, word] >> (node % 64).astype(np.uint64)) & np.uint64(1)
            see = held & ((node < 0) | ((bit == 1) & (node // 64 < mask.shape[1])))
            if c - n + i < 0 or not see.any():
                continue
            x = np.asarray(q[r], np.float64) / np.sqrt(D)
            for h in range(Hq):
                out[r, h], tol[r, h] = attention_row(x[h], K[see, h // G], V[see, h // G],
                                                     vmax[h // G], q_eps, w_eps)
    return out, tol


def rope(x, positions, freqs, interleaved, mscale):
    """x [T][H][dim] (64 bits) turned, and how far fp32 may be from it: cosines and sines within
    2^-23 and 2^-51 of the angle (and what this form's own product loses, 2^-52), times mscale
    (rounded), a product and a sum rounded."""
    half = len(freqs)
    out, tol = x.copy(), np.zeros_like(x)
    angle = positions.astype(np.float64)[:, None] * freqs
    c, s = np.cos(angle)[:, None] * mscale, np.sin(angle)[:, None] * mscale
    one = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    two = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    a, b = x[..., one], x[..., two]
    out[..., one], out[..., two] = a * c - b * s, a * s + b * c
    off = 2.0 ** -23 + 2 * 2.0 ** -24 + 2.0 ** -50 * np.abs(angle)[:, None]
    tol[..., one] = tol[..., two] = mscale * (np.abs(a) + np.abs(b)) * off
    return out, tol + 2.0 ** -24 * np.abs(out)


def gemm_i8(codes, inv, w, scales):
    """y [M][N] fp32: sums exact, the two products of fp32 rounded one by one."""
    acc = codes.astype(np.int64) @ w.astype(np.int64).T
    return acc.astype(np.float32) * (inv[:, None] * scales)


def first_best(y):
    y = np.where(np.isnan(y), -np.inf, y)
    return y.argmax(1).astype(np.int32)  # (the first of equal ones)
