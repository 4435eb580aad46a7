"""Decoding with trees of drafted tokens, all of it as a program would call it: two sequences and a
small model of random weights in 8 bits. A step plans its trees, and in each layer normalises and
quantizes, projects to q | k | v, turns q and k to the nodes' positions, appends to the paged cache
in 4 bits, attends to context and ancestors and projects back; then the LM head gives the model's
token after each node and the trees' accepted paths stay in the cache. The tokens have to be those
of decoding one by one, whatever was drafted, and the cache's rows theirs but for codes that another
order of sums moves by a step; then the same steps run from a captured graph."""
import numpy as np
import pytest

from tests.test_gpu_kv4 import D, PAGE, ops, torch_dev  # noqa: F401

pytestmark = pytest.mark.gpu
LAYERS, HQ, HKV, H, V = 2, 4, 2, 256, 700
COLS = (HQ + 2 * HKV) * D
B, PAGES, LONG, N = 2, 12, 150, 9  # tokens to decode, nodes of a tree
PROMPT = (5, 40)


class Model:
    def __init__(self, torch, ops, seed=0):
        rng = np.random.default_rng(seed)
        put = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
        self.torch, self.ops = torch, ops

        def weights(n, k):
            w = put(rng.integers(-127, 128, (n, k)).astype(np.int8))
            scales = put(rng.uniform(0.5, 1.5, n).astype(np.float32) / (73 * k ** 0.5))
            return ops.i8_rows_repack(w, n, k), scales, n, k

        self.qkv = [weights(COLS, H) for _ in range(LAYERS)]
        self.o = [weights(H, HQ * D) for _ in range(LAYERS)]
        self.head = weights(V, H)
        self.norms = [put((1 + 0.1 * rng.standard_normal(H)).astype(np.float32))
                      for _ in range(LAYERS + 1)]
        self.embedding = put(rng.standard_normal((V, H)).astype(np.float32))
        f, self.mscale = ops.rope_freqs(D, 10000.0, "parts", 4.0, 64, 8.0, 1.0)
        self.f = f.cuda()
        self.pools = ops.kv4_pool(B * PAGES + 1, LAYERS, HKV)
        self.tables = put(rng.permutation(B * PAGES + 1)[:B * PAGES].reshape(B, PAGES).astype(
            np.int32))

    def product(self, x, norm, w, **more):
        codes, q = self.ops.actquant127(x, norm)
        return self.ops.gemm_i8(codes, q, *w, **more)

    def forward(self, tokens, positions, lens, cu, mask):
        """The model's token after each row; the rows are the last of their sequences."""
        ops = self.ops
        x = self.embedding[tokens.long()]
        for i in range(LAYERS):
            qkv = self.product(x, self.norms[i], self.qkv[i])
            qk = qkv[:, :(HQ + HKV) * D]
            ops.rope(qk, positions, self.f, mscale=self.mscale, out=qk)
            where = (*self.pools, self.tables, lens, i)
            ops.kv4_append(qkv[:, HQ * D:(HQ + HKV) * D], qkv[:, (HQ + HKV) * D:], *where, cu_q=cu)
            if mask is None:
                att = ops.attn_kv4(qkv[:, :HQ * D], *where, cu_q=cu)
            else:
                att = ops.attn_tree_kv4(qkv[:, :HQ * D], mask, *where, cu_q=cu)
            x = x + self.product(att, None, self.o[i])
        return self.product(x, self.norms[-1], self.head, want_idx=True)

    def cache(self, lens):
        """The cached rows of each sequence, in order."""
        out = []
        for b in range(B):
            t = np.arange(int(lens[b]))
            page = self.tables[b].cpu().numpy()[t // PAGE]
            out.append([a.cpu().numpy()[page, :, :, t % PAGE] for a in self.pools])
        return out


def one_by_one(torch, m, prompts):
    """Greedy decoding, a token a sequence and step: tokens after the prompts, their logits' margin
    over the second best, and the caches."""
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    tokens = [list(p) for p in prompts]
    margin = []
    for step in range(max(PROMPT) + LONG):
        now = [min(step, len(t) - 1) for t in tokens]
        lens = i32(*[n + 1 for n in now])
        y, idx = m.forward(i32(*[t[n] for t, n in zip(tokens, now)]), i32(*now), lens, None, None)
        top = y.topk(2, dim=1).values
        for b in range(B):
            if step == len(tokens[b]) - 1 and len(tokens[b]) < PROMPT[b] + LONG:
                tokens[b].append(int(idx[b]))
                margin.append(float(top[b, 0] - top[b, 1]))
    return tokens, min(margin)


def drafted(rng, truth, at, wrong):
    """A tree of N nodes below token `at` of a sequence: some of its nodes go on as it does."""
    tokens, parents = [truth[at]], [-1]
    depth = [0]
    for i in range(1, N):
        p = int(rng.integers(max(0, i - 4), i))
        parents.append(p)
        depth.append(depth[p] + 1)
        real = truth[at + depth[i]] if at + depth[i] < len(truth) else 0
        tokens.append(real if rng.random() > wrong else int(rng.integers(0, V)))
    return tokens, parents


def test_trees_give_the_tokens_of_one_by_one(torch_dev, ops):
    torch = torch_dev
    rng = np.random.default_rng(5)
    prompts = [rng.integers(0, V, n).tolist() for n in PROMPT]
    m = Model(torch, ops)
    truth, margin = one_by_one(torch, m, prompts)
    print("smallest margin of a choice", margin)
    lens = [len(t) - 1 for t in truth]
    want = m.cache(lens)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    # the prompts but for their last token, as chains
    for a in m.pools:
        a.zero_()
    flat = [t for p in prompts for t in p[:-1]]
    m.forward(i32(flat), i32([i for p in prompts for i in range(len(p) - 1)]),
              i32([len(p) - 1 for p in prompts]),
              i32([0, len(prompts[0]) - 1, len(flat)]), None)
    tokens, parents = i32([0] * (B * N)), i32([0] * (B * N))
    cu, state = i32([0, N, 2 * N]), i32([len(p) - 1 for p in prompts])

    def step():
        now = state + N
        mask, at = ops.tree_plan(parents, now, N, cu_q=cu)
        _, target = m.forward(tokens, at, now, cu, mask)
        path, count, last, after = ops.tree_accept(parents, tokens, target, *m.pools, m.tables, now,
                                                   N, cu_q=cu)
        state.copy_(after)
        return path, count, last

    graph = None
    got = [list(p) for p in prompts]
    taken, steps = 0, 0
    while min(len(g) - p for g, p in zip(got, PROMPT)) < LONG - N:
        trees = [drafted(rng, truth[b], len(got[b]) - 1, 0.3 if steps % 3 else 0.0)
                 for b in range(B)]
        tokens.copy_(i32([t for x, _ in trees for t in x]))
        parents.copy_(i32([p for _, x in trees for p in x]))
        if steps == 6:  # from here on replayed
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
        path, count, last = (a.cpu().tolist() for a in out)
        for b in range(B):
            assert path[b][0] == 0 and 1 <= count[b] <= N
            got[b] += [trees[b][0][k] for k in path[b][1:count[b]]] + [last[b]]
            assert state[b].item() == len(got[b]) - 1
            # (the batch decides how a product or an attention sums up; no choice here is so near)
            assert got[b] == truth[b][:len(got[b])], (steps, b)
            taken += count[b]
        steps += 1
    print("tokens a step and sequence:", taken / steps / B)
    assert steps > 12 and taken > 1.5 * steps * B
    # The keys and values of the tokens that are there now, from one by one: the projections see
    # attention that was summed up in another order, so codes may differ by a step here and there.
    for b, (have, was) in enumerate(zip(m.cache(state.tolist()), want)):
        for x, y in zip(have, was):
            assert (x != y[:len(x)]).mean() < 0.02, b
