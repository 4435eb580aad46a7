"""How many bits of the queries the attention over the 4-bit cache keeps, seen where it matters most:
one token at a high score, whose values are zeros, and one at score 0 whose values are larger by
about what its weight is smaller, so that an output is a value times exp(-score). A score has one
product that is not zero, so nothing but the query's own roundings enters it."""
import numpy as np
import pytest

from tests.kv4_plan import plan
from tests.test_gpu_kv4 import D, PAGE, ops, torch_dev  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("kernel,B,Hq,Hkv,rows,width", [
    ("4", 1, 4, 1, 1, 1), ("4", 2, 8, 4, 1, 300), ("4 even", 48, 8, 2, 1, 300),
    ("16", 1, 8, 1, 1, 1), ("16", 2, 12, 1, 1, 300), ("16 even", 48, 16, 2, 1, 300),
    ("16 even", 16, 16, 2, 7, 257), ("32", 5, 16, 4, 300, 40), ("128", 1, 16, 2, 200, 4000),
    ("128", 5, 20, 5, 600, 60)])
def test_queries_keep_their_bits(torch_dev, ops, kernel, B, Hq, Hkv, rows, width, dtype):
    torch = torch_dev
    assert plan(B * rows, B, Hq, Hkv, width, rows > 1)[0] == kernel
    print("attn parts", kernel, B, Hq, Hkv, rows, width, dtype.__name__, flush=True)
    rng = np.random.default_rng(Hq + rows + width)
    c = rows + 1  # every row sees the first two tokens
    pages = -(-c // PAGE)
    # queries of 100 (scores of 50 to 55, base 2: 80) or, in the prompts' kernel, whose weights are
    # held in steps of 2^-40 of the largest, of 24 (12 to 13, base 2: 19)
    big, up = (24, 18) if kernel == "128" else (100, 74)
    pools = [a.numpy() for a in ops.kv4_pool(B * pages, 1, Hkv, device="cpu")]
    pools[2][:], pools[3][:] = 127, 127
    tables = np.full((B, width), -1, np.int32)
    tables[:, :pages] = np.arange(B * pages).reshape(B, pages)
    first = tables[:, 0]
    pools[0][first, 0, :, 1, 0] = 7        # token 1: its key's dim 0 is 6
    pools[1][first, 0, :, 0] = 0x53        # token 0: values 1.5 and 3, times 2^up
    pools[3][first, 0, :, 0] = 127 + up
    q = rng.standard_normal((B * rows, Hq, D)).astype(dtype)  # (dims 1 and on: times zeros)
    q[..., 0] = rng.uniform(0.96 * big, 1.04 * big, q.shape[:2])
    cu = None if rows == 1 else torch.arange(0, B * rows + 1, rows, dtype=torch.int32).cuda()
    ctx = torch.full((B,), c, dtype=torch.int32).cuda()
    out = ops.attn_kv4(torch.from_numpy(q).cuda(), *(torch.from_numpy(a).cuda() for a in pools),
                       torch.from_numpy(tables).cuda(), ctx, 0, cu_q=cu).cpu().numpy()
    n = np.tile(np.arange(rows), B) + 2.0  # tokens that a row sees, all but token 1 at score 0
    s = q[..., 0].astype(np.float64) * 6 / np.sqrt(D)
    low = np.exp(-s) / (1 + (n[:, None] - 1) * np.exp(-s))
    want = (low * 2.0 ** up)[..., None] * np.tile([1.5, 3.0], D // 2)
    # a score of s: the constant's and the product's rounding, in the prompts' kernel 2^-22 for the
    # query's parts, the difference's rounding (and the base's there); the exponential's step, and
    # one or two each for the weights' sum, the product, the joins and the division; 2^-41 of the
    # largest weight there
    u = 2.0 ** -24
    rel = (5 * u + (2.0 ** -22 if kernel == "128" else 0)) * s + 16 * u
    if kernel == "128":
        rel += (2.0 ** -41 + 2.0 ** -22 * low) / low
    tol = want * rel[..., None]
    # half a step of the type, of the number as it may be
    tol += np.spacing((want + tol).astype(dtype)).astype(np.float64) / 2
    worst = float((np.abs(out - want) / tol).max())
    assert worst <= 1, worst
