"""Batched beam decoding with everything that a step takes, as a program would call it: two
requests of four beams and a small model of random ternary weights. After a prompt each step
normalises and quantizes, projects to q | k | v, appends to the paged cache in 4 bits, attends,
projects back, takes the logits, selects and reorders. Every operator's result is checked
against its plain 64-bit form on the operands of that step; then the same steps are replayed from
a captured graph and give the same bits."""
import numpy as np
import pytest

from tests import kv4_plain as plain
from tests.test_gpu_kv4 import D, PAGE, ops, torch_dev  # noqa: F401
from tenzo_amd import formats, synth

pytestmark = pytest.mark.gpu
B, W, LAYERS, HQ, HKV, H, V = 2, 4, 2, 4, 2, 256, 500
ROWS, PAGES, N = B * W, 4, 14  # N tokens of prompt; the cache goes over two pages' borders


class Model:
    def __init__(self, torch, ops, seed=0):
        rng = np.random.default_rng(seed)
        put = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
        self.torch, self.ops = torch, ops
        self.cols = (HQ + 2 * HKV) * D
        self.wqkv = [ops.tl1_repack(put(formats.tl1_random(self.cols, H, rng)), self.cols, H)
                     for _ in range(LAYERS)]
        self.wo = [ops.tl1_repack(put(formats.tl1_random(H, HQ * D, rng)), H, HQ * D)
                   for _ in range(LAYERS)]
        self.norms = [put((1 + 0.1 * rng.standard_normal(H)).astype(np.float32))
                      for _ in range(LAYERS + 1)]
        head, scale = synth.head_quantize(rng.normal(0, 0.08, (V, H)).astype(np.float32))
        self.head, self.head_scale = ops.i8_rows_repack(put(head), V, H), put(scale)
        self.embedding = put(rng.standard_normal((V, H)).astype(np.float32))
        self.rope = ops.rope_table(10000.0, 0, PAGES * PAGE).cuda()
        self.pools = ops.kv4_pool(ROWS * PAGES + 1, LAYERS, HKV)
        # the prompt's full pages would be shared; here it ends in the first one, each slot's own
        self.tables = put(rng.permutation(ROWS * PAGES + 1)[:ROWS * PAGES].reshape(
            ROWS, PAGES).astype(np.int32))
        self.ctx = torch.zeros(ROWS, dtype=torch.int32, device="cuda")
        self.prompt = put(np.repeat(rng.integers(0, V, (B, 1, N)), W, 1))
        self.tokens = torch.zeros(ROWS, dtype=torch.int32, device="cuda")
        self.scores = torch.zeros((B, W), device="cuda")
        self.state = [*self.pools, self.tables, self.ctx, self.tokens, self.scores]

    def layers(self, x, cu, look):
        ops = self.ops
        for i in range(LAYERS):
            codes, q, _ = ops.rmsnorm_quant31(x, self.norms[i])
            qkv, _ = ops.bitlinear_tl1_batch(codes, q, self.wqkv[i], 0.02, self.cols, H)
            qs, ks, vs = qkv.split([HQ * D, HKV * D, HKV * D], 1)
            where = (*self.pools, self.tables, self.ctx, i)
            before = look and [a.cpu().numpy() for a in self.pools]
            ops.kv4_append(ks, vs, *where, rope_cs=self.rope, cu_q=cu)
            att = ops.attn_kv4(qs, *where, rope_cs=self.rope, cu_q=cu)
            if look:
                self.check_layer(i, qs, ks, vs, before, att, cu)
            codes, q, _ = ops.rmsnorm_quant31(att)
            x = x + ops.bitlinear_tl1_batch(codes, q, self.wo[i], 0.02, H, HQ * D)[0]
        return x

    def check_layer(self, i, qs, ks, vs, pools, att, cu):
        host = lambda t: t.cpu().numpy()  # noqa: E731
        tables, ctx, rope = host(self.tables), host(self.ctx), host(self.rope)
        cu = None if cu is None else host(cu)
        heads = lambda t, n: host(t).reshape(-1, n, D)  # noqa: E731
        plain.append(heads(ks, HKV), heads(vs, HKV), pools, tables, ctx, i, rope, cu)
        for a, b in zip(pools, self.pools):
            np.testing.assert_array_equal(host(b), a)
        want, tol = plain.attention(heads(qs, HQ), pools, tables, ctx, i, rope, cu,
                                    np.zeros((len(qs), HQ, D)), 2.0 ** -21)
        tol = tol + 2.0 ** -24 * (np.abs(want) + tol)  # (half a step of fp32)
        assert (np.abs(heads(att, HQ) - want) <= tol).all()

    def choose(self, x, look):
        """From the last rows' hidden states to the next tokens, the caches reordered."""
        ops, torch = self.ops, self.torch
        logits = torch.stack([ops.lm_head_i8(r, self.norms[-1], self.head, self.head_scale, V, H)
                              for r in x]).view(B, W, V)
        best, beams, tokens = ops.beam_select(logits, self.scores, 2 * W)
        parents = beams[:, :W]
        state = look and [a.cpu().numpy() for a in (self.tables, self.ctx, *self.pools)]
        ops.beam_reorder_paged(parents, self.tables, self.ctx, *self.pools)
        if look:
            want = plain.beam_select(logits.cpu().numpy(), self.scores.cpu().numpy(), 2 * W)
            np.testing.assert_array_equal(beams.cpu().numpy(), want[1])
            np.testing.assert_array_equal(tokens.cpu().numpy(), want[2])
            plain.reorder(want[1][:, :W].astype(np.int32), state[0], state[1], state[2:])
            np.testing.assert_array_equal(self.tables.cpu().numpy(), state[0])
            for a, b in zip(state[2:], self.pools):
                np.testing.assert_array_equal(b.cpu().numpy(), a)
        self.scores.copy_(best[:, :W])
        self.tokens.copy_(tokens[:, :W].reshape(-1))

    def start(self, look=False):
        torch = self.torch
        self.ctx.fill_(N)
        cu = torch.arange(0, ROWS * N + 1, N, dtype=torch.int32, device="cuda")
        x = self.layers(self.embedding[self.prompt.reshape(-1)], cu, look)
        # (one beam of each request counts before the first choice)
        self.scores.fill_(-np.inf)
        self.scores[:, 0] = 0
        self.choose(x[N - 1::N].contiguous(), look)

    def step(self, look=False):
        self.ctx.add_(1)
        self.choose(self.layers(self.embedding[self.tokens.long()], None, look), look)


def test_beam_decode(torch_dev, ops):
    torch = torch_dev
    m = Model(torch, ops)
    m.start(look=True)
    first = [a.clone() for a in m.state]
    moved, trace = 0, []
    for i in range(20):
        print("step", i, flush=True)
        old = m.tables.clone()
        m.step(look=True)
        moved += int((m.tables != old).any())
        trace.append([a.clone() for a in m.state])
    assert moved, "full pages changed hands"
    # the same from a graph, twice, with eager work between the replays
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m.step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        m.step()
    for _ in range(2):
        for a, b in zip(m.state, first):
            a.copy_(b)
        for want in trace:
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(m.state, want):
                assert torch.equal(a, b)
            assert ops.beam_select(torch.zeros((1, 1, 9), device="cuda"),
                                   torch.zeros((1, 1), device="cuda"), 1)[2].item() == 0
