"""Whole steps of decoding with trees in the kernels and types that small fp32 batches do not reach: 128
rows a workgroup with steps dealt evenly and with all tokens of a tree, fp16 and fp32. The text is given, so
nothing hangs on near choices: each step's tree has some of it, and the model's logits after the nodes
that agree, and the cache's rows at the end, are held against those of decoding one by one.

Layer 0's rows are bit for bit the same: they come from embedding, norm, quantization, an exact product,
rope and append, row by row. In layer 1 attention has summed up in another order and, in fp16, rounded
outputs another way (2^-11), which moves a few of the next quantizer's codes by one of 127, and with them
about one of 50 of a cached row's 4-bit codes by a step (a quarter of its value) or one of its four scales
(a group rounded anew: a tenth): below 0.1 of a row's norm, where a row of another token differs by
about 1.4 of it. Logits see less than that."""
import numpy as np
import pytest

from tests import kv4_plain, tree_kernels
from tests import test_gpu_tree_decode as decode
from tests.test_gpu_kv4 import D, PAGE, ops, torch_dev  # noqa: F401

pytestmark = pytest.mark.gpu
V = decode.V
NEAR = 0.3  # of a row's norm


class Model(decode.Model):
    """decode.Model with projections, rotary positions, cache and attention in fp16 where asked."""
    dtype = None

    def forward(self, tokens, positions, lens, cu, mask):
        ops, Hq, Hkv = self.ops, decode.HQ, decode.HKV
        x = self.embedding[tokens.long()]
        for i in range(decode.LAYERS):
            qkv = self.product(x, self.norms[i], self.qkv[i], dtype=self.dtype)
            qk = qkv[:, :(Hq + Hkv) * D]
            ops.rope(qk, positions, self.f, mscale=self.mscale, out=qk)
            where = (*self.pools, self.tables, lens, i)
            ops.kv4_append(qkv[:, Hq * D:(Hq + Hkv) * D], qkv[:, (Hq + Hkv) * D:], *where, cu_q=cu)
            if mask is None:
                att = ops.attn_kv4(qkv[:, :Hq * D], *where, cu_q=cu)
            else:
                att = ops.attn_tree_kv4(qkv[:, :Hq * D], mask, *where, cu_q=cu)
            assert att.dtype == self.dtype
            x = x + self.product(att.float(), None, self.o[i])
        return self.product(x, self.norms[-1], self.head, want_idx=True)


def tree(rng, text, at, n):
    """(tokens, parents, targets) of a tree below token `at` of a text: some of its nodes go on as it
    does, and those have the text's next token for a target."""
    tokens, parents, depth, real = [text[at]], [-1], [0], [True]
    for i in range(1, n):
        p = int(rng.integers(max(0, i - 6), i))
        parents.append(p)
        depth.append(depth[p] + 1)
        goes_on = rng.random() < 0.6
        tokens.append(text[at + depth[i]] if goes_on else int(rng.integers(0, V)))
        real.append(real[p] and tokens[i] == text[at + depth[i]])
    return tokens, parents, [text[at + d + 1] if r else int(rng.integers(0, V))
                             for d, r in zip(depth, real)]


@pytest.mark.parametrize("kernel,dtype,B,N,Hq,Hkv,pages", [
    ("16", "float16", 2, 9, 4, 2, 10), ("128 even", "float16", 3, 40, 16, 2, 1100),
    ("128 even", "float32", 2, 40, 16, 2, 1100), ("128", "float16", 30, 40, 16, 2, 10),
    ("128", "float32", 78, 40, 16, 2, 10)])
def test_steps(torch_dev, ops, monkeypatch, kernel, dtype, B, N, Hq, Hkv, pages):
    torch = torch_dev
    print("decode", kernel, dtype, B, N, flush=True)
    assert tree_kernels.plan(B * N, B, Hq, Hkv, pages, True, dtype == "float16")[0] == kernel
    for name, value in dict(B=B, HQ=Hq, HKV=Hkv, PAGES=pages, COLS=(Hq + 2 * Hkv) * D).items():
        monkeypatch.setattr(decode, name, value)
    rng = np.random.default_rng(B)
    m = Model(torch, ops)
    m.dtype = getattr(torch, dtype)
    L, steps = 120, 9
    text = rng.integers(0, V, (B, L + N + 1))
    i32 = lambda a: torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")  # noqa: E731
    # one by one: logits after each token, and the cache
    logits = [m.forward(i32(text[:, t]), i32([t] * B), i32([t + 1] * B), None, None)[0]
              for t in range(L)]
    want = m.cache([L] * B)
    # the first tokens of each text as chains, the rest by trees
    for a in m.pools:
        a.zero_()
    first = rng.integers(3, 16, B)
    cu = np.concatenate([[0], np.cumsum(first)])
    m.forward(i32(np.concatenate([text[b, :n] for b, n in enumerate(first)])),
              i32(np.concatenate([np.arange(n) for n in first])), i32(first), i32(cu), None)
    tokens, parents, target = (i32(np.zeros(B * N)) for _ in range(3))
    cu, state = i32(N * np.arange(B + 1)), i32(first)

    def step():
        now = state + N
        mask, at = ops.tree_plan(parents, now, N, cu_q=cu)
        y, _ = m.forward(tokens, at, now, cu, mask)
        path, count, last, after = ops.tree_accept(parents, tokens, target, *m.pools, m.tables, now,
                                                   N, cu_q=cu)
        state.copy_(after)
        return y, path, count, last

    graph, worst, moved = None, 0.0, 0
    have = first.copy()
    for k in range(steps):
        trees = [tree(rng, text[b], have[b], N) for b in range(B)]
        for dst, i in ((tokens, 0), (parents, 1), (target, 2)):
            dst.copy_(i32(np.concatenate([t[i] for t in trees])))
        if k == 4:  # from here on replayed
            keep = [a.clone() for a in (*m.pools, state)]
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                step()
            side.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                out = step()
            for a, b in zip((*m.pools, state), keep):
                a.copy_(b)
            torch.cuda.synchronize()
        if graph is None:
            out = step()
        else:
            graph.replay()
        torch.cuda.synchronize()
        y, (path, count, last) = out[0], (a.cpu().numpy() for a in out[1:])
        for b in range(B):
            n, at = count[b], have[b]
            nodes = path[b, :n]
            assert n >= 1 and nodes[0] == 0 and (path[b, n:] == -1).all()
            np.testing.assert_array_equal(np.asarray(trees[b][0])[nodes], text[b, at:at + n])
            assert last[b] == text[b, at + n] and state[b].item() == at + n
            for i, node in enumerate(nodes):
                if at + i < L:
                    a = logits[at + i][b]
                    worst = max(worst, float((y[b * N + node] - a).norm() / a.norm()))
            moved += int((nodes != np.arange(n)).sum())
            have[b] += n
        if have.max() > L:
            break
    print("steps", k + 1, "tokens", int((have - first).sum()), "moved", moved, "logits", worst)
    assert moved > 2 * B and k >= 5 and worst < NEAR
    far = 0.0
    for b, (rows, was) in enumerate(zip(m.cache(np.minimum(have, L)), want)):
        n = len(rows[0])
        for x, y in zip(rows, was):
            np.testing.assert_array_equal(x[:, 0], y[:n, 0])
        for p in (0, 1):  # keys, values
            x, y = (kv4_plain.values(a[p][:n], a[p + 2][:n]) for a in (rows, was))
            off = np.linalg.norm(x - y, axis=-1) / np.linalg.norm(y, axis=-1)
            far = max(far, float(off.max()))
    print("rows of the cache", far)
    assert far < NEAR
