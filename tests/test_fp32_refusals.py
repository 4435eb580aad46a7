"""What the entry points of tenzo_amd.ops that read fp32 do with other types: rows of gemm_i8, rope or
attention over the 4-bit cache in fp16 or bf16 would be read as floats, past their end. Nothing is
launched, so no GPU is needed."""
import pytest
import torch

from tenzo_amd import ops
from tests.test_kv4_refusals import cpu  # noqa: F401

M, K, N = 3, 64, 50
X, W, LOGITS = torch.zeros((M, K)), torch.ones(K), torch.zeros(N)
CODES, ACTQ = torch.zeros((M, K), dtype=torch.int8), torch.zeros((M, 2), dtype=torch.int32)
PACKED, SCALES = torch.zeros(4096, dtype=torch.uint8), torch.ones(N)
Q, KV, CS = torch.zeros((1, 512)), torch.zeros((1, 256)), torch.zeros(128)
INT8 = [torch.zeros((1, 2, 32, 128), dtype=torch.int8)] * 2 + [torch.zeros((1, 2, 32)).half()] * 2
TERN = [torch.zeros((1, 2, 32, 32), dtype=torch.uint8)] * 2 + [torch.zeros((1, 2, 32))] * 2
PAGED = [torch.zeros((4, 1, 2, 16, 128), dtype=torch.int8)] * 2 + [torch.zeros((4, 1, 2, 16))] * 2
TABLE = torch.zeros(4, dtype=torch.int32)

CALLS = {
    "actquant127": (ops.actquant127, [X, W], [0, 1]),
    "rmsnorm_quant31": (ops.rmsnorm_quant31, [X, W], [0, 1]),
    "rmsnorm": (ops.rmsnorm, [W, W], [0, 1]),
    "bitlinear_tl1_f32": (ops.bitlinear_tl1_f32, [X, PACKED, 1.0, N, K], [0]),
    "lm_head_i8": (ops.lm_head_i8, [W, W, PACKED, SCALES, N, K], [0, 1, 3]),
    "lm_head_i8_codes_into": (ops.lm_head_i8_codes_into,
                              [CODES[:1], ACTQ[:1], PACKED, SCALES, N, K, LOGITS], [3, 6]),
    "argmax": (ops.argmax, [LOGITS], [0]),
    "sample_top_k_top_p": (ops.sample_top_k_top_p, [LOGITS, 4, 0.9, 1.0, 0.5], [0]),
    "attn_int8_decode": (ops.attn_int8_decode, [Q, KV, KV, *INT8, CS, 3], [0, 1, 2, 7]),
    "attn_tern_decode": (ops.attn_tern_decode, ["tl1_fused", Q, KV, KV, *TERN, CS, 3],
                         [1, 2, 3, 8]),
    "attn_paged_int8_decode": (ops.attn_paged_int8_decode,
                               [Q, KV, KV, *PAGED, TABLE, 0, CS, 3], [0, 1, 2, 9]),
}


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float64, torch.int32])
@pytest.mark.parametrize("fn,i", [(n, i) for n, c in CALLS.items() for i in c[2]])
def test_other_types_refused(cpu, monkeypatch, fn, i, dtype):  # noqa: F811
    monkeypatch.setattr(ops, "_ptr", lambda t: None if t is None else t.data_ptr())
    call, args, _ = CALLS[fn]
    args = list(args)
    args[i] = args[i].to(dtype)
    with pytest.raises(ValueError, match="not torch.float32"):
        call(*args)


@pytest.mark.parametrize("fn,i", [("actquant127", 1), ("rmsnorm_quant31", 1), ("rmsnorm", 1),
                                  ("lm_head_i8", 0), ("lm_head_i8", 1)])
def test_other_lengths_refused(cpu, monkeypatch, fn, i):  # noqa: F811
    monkeypatch.setattr(ops, "_ptr", lambda t: None if t is None else t.data_ptr())
    call, args, _ = CALLS[fn]
    args = list(args)
    args[i] = args[i][..., :48].contiguous()
    with pytest.raises(ValueError, match="not 64 values"):
        call(*args)


@pytest.mark.parametrize("fn", CALLS)
def test_fp32_reaches_the_library(cpu, monkeypatch, fn):  # noqa: F811
    monkeypatch.setattr(ops, "_ptr", lambda t: None if t is None else t.data_ptr())
    call, args, _ = CALLS[fn]
    with pytest.raises(AssertionError, match="the library was called"):
        call(*args)
