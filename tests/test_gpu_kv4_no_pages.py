"""Pools without a page: every table entry is outside them, so all tokens are absent."""
import numpy as np
import pytest

from tests.kv4_plan import plan
from tests.test_gpu_kv4 import D, ops, torch_dev  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kernel,B,Hq,Hkv,rows,width", [
    ("4", 2, 4, 2, 1, 300), ("4 even", 48, 8, 2, 1, 300), ("16", 1, 8, 1, 5, 9),
    ("32", 5, 16, 4, 300, 40), ("128", 1, 16, 2, 200, 4000)])
def test_no_pages(torch_dev, ops, kernel, B, Hq, Hkv, rows, width):
    torch = torch_dev
    T = B * rows
    assert plan(T, B, Hq, Hkv, width, True)[0] == kernel
    print("no pages", kernel, flush=True)
    pools = ops.kv4_pool(0, 2, Hkv)
    tables = torch.zeros((B, width), dtype=torch.int32, device="cuda")
    ctx = torch.full((B,), width * 16, dtype=torch.int32, device="cuda")
    cu = torch.arange(0, T + 1, rows, dtype=torch.int32, device="cuda")
    x = torch.ones((T, Hkv * D), device="cuda")
    ops.kv4_append(x, x, *pools, tables, ctx, 1, cu_q=cu)
    k, v = ops.kv4_read(*pools, tables, ctx, 1, rows=T, cu_q=cu)
    out = torch.full((T, Hq * D), 7.0, device="cuda")
    ops.attn_kv4(torch.ones((T, Hq * D), device="cuda"), *pools, tables, ctx, 1, cu_q=cu, out=out)
    assert not k.any() and not v.any() and not out.any()


def test_reorder_without_pages(torch_dev, ops):
    torch = torch_dev
    tables = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    ctx = torch.full((2,), 35, dtype=torch.int32, device="cuda")
    parents = torch.tensor([[1, 1]], dtype=torch.int32, device="cuda")
    ops.beam_reorder_paged(parents, tables, ctx, *ops.kv4_pool(0, 2, 3))
    np.testing.assert_array_equal(tables.cpu().numpy(), [[4, 5, 2, 3], [4, 5, 6, 7]])
