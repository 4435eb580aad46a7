"""A table of rotations without a row: refused, not taken for no rotation (its address is null)."""
import pytest
import torch

from tenzo_amd import ops
from tests.test_kv4_refusals import _cache, cpu  # noqa: F401


def test_no_rotation_rows(cpu):
    x, none = torch.zeros((3, 256)), torch.zeros((0, 128))
    with pytest.raises(ValueError, match="rope_cs"):
        ops.kv4_append(x, x, *_cache(), rope_cs=none)
    with pytest.raises(ValueError, match="rope_cs"):
        ops.attn_kv4(x, *_cache(), rope_cs=none)
