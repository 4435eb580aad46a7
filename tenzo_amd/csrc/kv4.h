// The paged cache held in 4 bits: its layout, the sequences of a call and the conversions that
// its kernels share (kv4_cache.hip, attention_kv4.hip).
//
// A row of 128 values is four groups of 32, each E2M1 codes (0 .5 1 1.5 2 3 4 6 and their
// negatives) times a power of two of its own (E8M0: 2^(s - 127)): 64 + 4 bytes in place of the
// 128 + 4 of an int8 row. Every value is exact in bf16, and the codes are what gfx950 converts
// two at a time with the scale applied, so a row costs 64 conversions and no multiplication.
// Byte i of a row holds dim 2i in its low nibble and dim 2i + 1 in its high one. Pools as the
// int8 paged cache has them: codes [blocks][n_layers][Hkv][16][64], scales
// [blocks][n_layers][Hkv][16][4].
#pragma once

#include "common.h"

namespace tz {

constexpr int kKv4Dim = 128;
constexpr int kKv4Page = 16;
constexpr int kKv4Row = 64;    // code bytes of a row
constexpr int kKv4Scales = 4;  // scale bytes of a row

// The sequences of a call. Row r of the T rows belongs to sequence s with cu[s] <= r < cu[s + 1]
// (cu null: row r is sequence r's only one) and stands at position ctx[s] - n + (r - cu[s]), n
// the sequence's rows. What the device finds in these arrays is checked before it is used: a
// length above `limit` (the table's width, the rotation's rows) counts as 0, a range outside the T
// rows as empty, a page outside the pool as absent. Ranges that lie over each other (cu decreasing
// somewhere) give rows no meaning, but nothing else is read or written for them.
struct Kv4Seqs {
    const int32_t* tables;
    const int32_t* ctx;
    const int32_t* cu;
    int64_t table_stride;
    int64_t n_blocks;
    int B, limit, T;
    int n_layers, layer, Hkv;

    __device__ __forceinline__ int length(int s) const {
        const int c = ctx[s];
        return c > 0 && c <= limit ? c : 0;
    }
    // Rows of sequence s (none where cu has no range of the T rows there), and its first.
    __device__ __forceinline__ int rows(int s, int& first) const {
        if (!cu) {
            first = s;
            return 1;
        }
        const int begin = cu[s], end = cu[s + 1];
        first = begin;
        return begin >= 0 && end > begin && end <= T ? end - begin : 0;
    }
    // Row (of 16-token pages) of head 0 in logical page `p` of sequence s, or -1.
    __device__ __forceinline__ int64_t page_base(int s, int p) const {
        const int64_t blk = tables[(int64_t)s * table_stride + p];
        return blk >= 0 && blk < n_blocks ? (blk * n_layers + layer) * Hkv * kKv4Page : -1;
    }
};

__device__ __forceinline__ int max_row16(int v) {  // over the 16 lanes of a DPP row
    v = max(v, dpp_i<kDppXor1>(v));
    v = max(v, dpp_i<kDppXor2>(v));
    v = max(v, dpp_i<kDppHalfMirror>(v));
    return max(v, dpp_i<kDppMirror>(v));
}

// Position of row r and its sequence; false where it stands nowhere (padding). The sequence is
// looked for by the 16 lanes of a DPP row, all of them active and with the same r.
__device__ __forceinline__ bool kv4_place(const Kv4Seqs& q, int r, int lane16, int& seq,
                                          int& pos) {
    if (!q.cu) {
        seq = r;
        pos = q.length(r) - 1;
        return pos >= 0;
    }
    seq = pos = -1;
    for (int b = lane16; b < q.B; b += 16) {
        int first;
        const int n = q.rows(b, first), c = q.length(b);
        if (r >= first && r < first + n) {
            seq = b;
            pos = c - n + (r - first);
        }
    }
    const int mine = seq;  // (of two sequences with ranges over each other the later one)
    seq = max_row16(seq);
    pos = max_row16(mine == seq ? pos : -1);
    return pos >= 0;
}

// 2^(s - 127) as fp32. Bytes above 252, which no append writes, count as 0: whatever a pool holds
// is finite, so that a token with weight 0 adds nothing.
__device__ __forceinline__ float e8m0_to_float(uint32_t s) {
    return __uint_as_float(s == 0 || s > 252 ? 0x00400000u : s << 23);
}

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// Eight codes of two groups, the low four times `lo`, the upper four times `hi`.
__device__ __forceinline__ void fp4_to_float8(uint32_t w, float lo, float hi, float (&v)[8]) {
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, lo, 0);
    const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, lo, 1);
    const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, hi, 2);
    const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, hi, 3);
    v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
    v[4] = c.x, v[5] = c.y, v[6] = d.x, v[7] = d.y;
}

template <bool HALF>
__device__ __forceinline__ float ld_act(const void* p, int64_t i) {
    return HALF ? __half2float(reinterpret_cast<const __half*>(p)[i])
                : reinterpret_cast<const float*>(p)[i];
}
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef _Float16 f16x4_any __attribute__((ext_vector_type(4), aligned(2)));
// Four values in a row, at any element's address (one load: the GPU takes unaligned ones).
template <bool HALF>
__device__ __forceinline__ void ld_act4(const void* p, int64_t i, float (&v)[4]) {
    if (HALF) {
        const f16x4_any x =
            *reinterpret_cast<const f16x4_any*>(reinterpret_cast<const uint16_t*>(p) + i);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = (float)x[k];
    } else {
        const f32x4_any x =
            *reinterpret_cast<const f32x4_any*>(reinterpret_cast<const float*>(p) + i);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = x[k];
    }
}
template <bool HALF>
__device__ __forceinline__ void st_act(void* p, int64_t i, float v) {
    if (HALF)
        reinterpret_cast<uint16_t*>(p)[i] = float_to_half_bits(v);
    else
        reinterpret_cast<float*>(p)[i] = v;
}

// Argument checks that the entry points share. Fills `q`.
int kv4_check(const char* what, const void* pk, const void* pv, const void* pks, const void* pvs,
              int64_t n_blocks, int n_layers, int layer, int Hkv, const int32_t* block_tables,
              int64_t table_stride, int table_width, const int32_t* ctx_lens,
              const int32_t* cu_q, int B, int64_t T, const float* rope_cs, int n_pos, Kv4Seqs& q);

}  // namespace tz
