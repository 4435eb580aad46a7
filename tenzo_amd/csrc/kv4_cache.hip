// Writing to and reading from the paged cache held in 4 bits (layout: kv4.h).
#include "kv4.h"

namespace tz {
namespace {

struct Kv4Append {
    const void* k;
    const void* v;
    int64_t k_stride, v_stride;
    uint8_t* pk;
    uint8_t* pv;
    uint8_t* pks;
    uint8_t* pvs;
    const float* rope;
    int items;  // T * Hkv
};

constexpr float kKv4Max = 0x1.cp127f;  // the largest magnitude whose codes stay finite: 7 * 2^125

// r rounded to fp32 so that it never meets the border of two codes unless it lies on it: towards
// zero, with the last bit set when anything was cut off. The borders are fp32 numbers of a few
// bits, so a code taken from this value is the one that r itself rounds to.
__device__ __forceinline__ float round_sticky(double r) {
    const float t = (float)r;
    const double back = (double)t;
    uint32_t b = __float_as_uint(t);
    if (fabs(back) > fabs(r)) b -= 1;
    if (back != r) b |= 1;
    return __uint_as_float(b);
}

// The same where r lies within fp32's normal numbers (`high`, its upper word without the sign, in
// kHighLow .. kHighTop): its upper 23 bits of fraction, with the exponent of fp32.
constexpr uint32_t kHighLow = 897u << 20, kHighTop = (1151u << 20) - 1;
__device__ __forceinline__ uint32_t high_word(double r) {
    return (uint32_t)__double2hiint(r) & 0x7fffffffu;
}
__device__ __forceinline__ float cut_sticky(double r) {
    const uint32_t hi = (uint32_t)__double2hiint(r), lo = (uint32_t)__double2loint(r);
    const uint32_t b = __builtin_amdgcn_alignbit(hi, lo, 29) - (896u << 23);
    return __uint_as_float((b & 0x7fffffffu) | (hi & 0x80000000u) | min(lo & 0x1fffffffu, 1u));
}

__device__ __forceinline__ float tame(float x) {  // NaN counts as 0, what is beyond is held there
    return x == x ? fminf(fmaxf(x, -kKv4Max), kKv4Max) : 0.0f;
}

// The scale byte of a group whose largest magnitude has the bits `top`: the smallest e with top <=
// 7 * 2^(e - 127) (codes up to 7 go to 6, the last one), at least 1: the exponent field less 2, one
// more above 1.75.
__device__ __forceinline__ int group_scale(uint32_t top) {
    return max((int)((top + 0x1FFFFFu) >> 23) - 2, 1);
}

// Four values of one group as codes, the first in the low nibble.
__device__ __forceinline__ uint32_t codes4(const float (&x)[4], int e) {
    const float s = __uint_as_float((uint32_t)e << 23);
    uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, x[0], x[1], s, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], s, 1);
    return w & 0xffffu;
}

__device__ __forceinline__ uint32_t max8(uint32_t m) {  // over the 8 lanes of a half DPP row
    m = max(m, (uint32_t)dpp_i<kDppXor1>((int)m));
    m = max(m, (uint32_t)dpp_i<kDppXor2>((int)m));
    return max(m, (uint32_t)dpp_i<kDppHalfMirror>((int)m));
}
// Of four values, the bits of the largest magnitude (a NaN's are above all numbers').
__device__ __forceinline__ uint32_t top4(const float (&x)[4]) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) m = max(m, __float_as_uint(x[j]) & 0x7fffffffu);
    return m;
}

// A row's codes and scales to its place: lane l of 16 has dims 4l .. 4l + 3 and 64 + 4l .. + 3.
__device__ __forceinline__ void write_row(float (&lo)[4], float (&hi)[4], int l, uint8_t* codes,
                                          uint8_t* scales) {
    uint32_t ml = top4(lo), mh = top4(hi);
    if (__ballot(max(ml, mh) > __float_as_uint(kKv4Max))) {  // (rare)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            lo[j] = tame(lo[j]);
            hi[j] = tame(hi[j]);
        }
        ml = top4(lo);
        mh = top4(hi);
    }
    const int el = group_scale(max8(ml)), eh = group_scale(max8(mh));
    reinterpret_cast<uint16_t*>(codes)[l] = (uint16_t)codes4(lo, el);
    reinterpret_cast<uint16_t*>(codes)[16 + l] = (uint16_t)codes4(hi, eh);
    if ((l & 7) == 0) {
        scales[l >> 3] = (uint8_t)el;
        scales[2 + (l >> 3)] = (uint8_t)eh;
    }
}

// 16 lanes to a head of a row, its key and its value: lane l has dims 4l .. 4l + 3 and 64 + 4l
// .. 64 + 4l + 3, so that a dim and its partner of the rotation meet in one lane and a group of
// 32 lies in 8 lanes. Bound by the vector work beside the bytes: 9245 rows of 5 kv heads, fp32, 14.4
// us, 3.7 TB/s (15.5 where fp64 is converted rather than cut to fp32 by its bits, and NaN and
// infinities are looked at one by one); one row 2.4 us, a chain of four loads.
template <bool HALF>
__global__ void __launch_bounds__(256) kv4_append_kernel(Kv4Append a, Kv4Seqs sq) {
    const int l = threadIdx.x & 15;
    const int item = (int)blockIdx.x * 16 + (threadIdx.x >> 4);
    if (item >= a.items) return;
    const int row = item / sq.Hkv, h = item - row * sq.Hkv;
    float klo[4], khi[4], vlo[4], vhi[4];
    const int64_t ka = row * a.k_stride + h * kKv4Dim + 4 * l;
    const int64_t va = row * a.v_stride + h * kKv4Dim + 4 * l;
    ld_act4<HALF>(a.k, ka, klo);
    ld_act4<HALF>(a.k, ka + 64, khi);
    ld_act4<HALF>(a.v, va, vlo);
    ld_act4<HALF>(a.v, va + 64, vhi);
    int seq, pos;
    if (!kv4_place(sq, row, l, seq, pos)) return;
    const int64_t base = sq.page_base(seq, pos / kKv4Page);
    if (base < 0) return;
    const int64_t dst = base + h * kKv4Page + pos % kKv4Page;
    write_row(vlo, vhi, l, a.pv + dst * kKv4Row, a.pvs + dst * kKv4Scales);
    if (a.rope) {
        // in 64 bits, where both products are exact: a key is rounded once, to its code
        float c4[4], s4[4];
        ld_act4<false>(a.rope, (int64_t)pos * kKv4Dim + 4 * l, c4);
        ld_act4<false>(a.rope, (int64_t)pos * kKv4Dim + 64 + 4 * l, s4);
        double a0[4], a1[4];
        uint32_t low = 0xffffffffu, top = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const double c = c4[j], s = s4[j], x0 = klo[j], x1 = khi[j];
            a0[j] = __builtin_fma(-x1, s, x0 * c);
            a1[j] = __builtin_fma(x1, c, x0 * s);
            low = min(low, min(high_word(a0[j]), high_word(a1[j])));
            top = max(top, max(high_word(a0[j]), high_word(a1[j])));
        }
        if (__ballot(low < kHighLow || top > kHighTop)) {  // (zeros, mostly)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                klo[j] = round_sticky(a0[j]);
                khi[j] = round_sticky(a1[j]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                klo[j] = cut_sticky(a0[j]);
                khi[j] = cut_sticky(a1[j]);
            }
        }
    }
    write_row(klo, khi, l, a.pk + dst * kKv4Row, a.pks + dst * kKv4Scales);
}

struct Kv4Read {
    const uint8_t* pk;
    const uint8_t* pv;
    const uint8_t* pks;
    const uint8_t* pvs;
    void* k;
    void* v;
    int items;
};

// 16 lanes to a head of a row, its key and its value: lane l has dims 8l .. 8l + 7 (fp16) or 4l ..
// 4l + 3 and 64 + 4l .. 64 + 4l + 3 (fp32), so that a store writes 256 bytes in a row. Bound by the
// bytes written: 9245 rows of 5 kv heads, fp32, 11.6 us, 4.6 TB/s (with 8l .. 8l + 7 14).
template <bool HALF>
__global__ void __launch_bounds__(256) kv4_read_kernel(Kv4Read a, Kv4Seqs sq) {
    const int l = threadIdx.x & 15;
    const int item = (int)blockIdx.x * 16 + (threadIdx.x >> 4);
    if (item >= a.items) return;
    const int row = item / sq.Hkv, h = item - row * sq.Hkv;
    const int lo = HALF ? l >> 2 : l >> 3, hi = HALF ? lo : 2 + lo;  // the codes' scales
    auto codes8 = [&](const uint8_t* row) -> uint32_t {
        if (HALF) return reinterpret_cast<const uint32_t*>(row)[l];
        const uint16_t* c = reinterpret_cast<const uint16_t*>(row);
        return c[l] | (uint32_t)c[16 + l] << 16;
    };
    float v[2][8] = {};
    int seq, pos;
    if (kv4_place(sq, row, l, seq, pos)) {
        const int64_t base = sq.page_base(seq, pos / kKv4Page);
        if (base >= 0) {
            const int64_t src = base + h * kKv4Page + pos % kKv4Page;
            const uint32_t wk = codes8(a.pk + src * kKv4Row);
            const uint32_t wv = codes8(a.pv + src * kKv4Row);
            const uint8_t* sk = a.pks + src * kKv4Scales;
            const uint8_t* sv = a.pvs + src * kKv4Scales;
            fp4_to_float8(wk, e8m0_to_float(sk[lo]), e8m0_to_float(sk[hi]), v[0]);
            fp4_to_float8(wv, e8m0_to_float(sv[lo]), e8m0_to_float(sv[hi]), v[1]);
        }
    }
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        void* out = w ? a.v : a.k;
        const int64_t at = (int64_t)item * kKv4Dim + (HALF ? 8 : 4) * l;
        if (HALF) {
            uint32_t p[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
                p[k] = float_to_half_bits(v[w][2 * k]) |
                       (uint32_t)float_to_half_bits(v[w][2 * k + 1]) << 16;
            *reinterpret_cast<uint4*>((uint16_t*)out + at) = uint4{p[0], p[1], p[2], p[3]};
        } else {
            float4* o = reinterpret_cast<float4*>((float*)out + at);
            o[0] = make_float4(v[w][0], v[w][1], v[w][2], v[w][3]);
            o[16] = make_float4(v[w][4], v[w][5], v[w][6], v[w][7]);
        }
    }
}

}  // namespace

int kv4_check(const char* what, const void* pk, const void* pv, const void* pks, const void* pvs,
              int64_t n_blocks, int n_layers, int layer, int Hkv, const int32_t* block_tables,
              int64_t table_stride, int table_width, const int32_t* ctx_lens,
              const int32_t* cu_q, int B, int64_t T, const float* rope_cs, int n_pos,
              Kv4Seqs& q) {
    TZ_CHECK(B >= 0 && T >= 0 && T <= INT32_MAX, "%s: B=%d T=%lld", what, B, (long long)T);
    TZ_CHECK(Hkv > 0 && Hkv <= 65535, "%s: bad head count (Hkv=%d)", what, Hkv);
    TZ_CHECK(n_layers > 0 && layer >= 0 && layer < n_layers, "%s: layer %d of %d", what, layer,
             n_layers);
    TZ_CHECK(n_blocks >= 0 && n_blocks <= INT32_MAX, "%s: %lld blocks", what,
             (long long)n_blocks);
    TZ_CHECK(table_width >= 0 && table_width <= (1 << 26) &&
                 (table_stride >= table_width || B <= 1),
             "%s: block tables of %d pages, %lld apart", what, table_width,
             (long long)table_stride);
    TZ_CHECK(cu_q || T == B, "%s: %lld rows for %d sequences of one token", what, (long long)T, B);
    TZ_CHECK(!rope_cs || n_pos >= 0, "%s: %d rotation rows", what, n_pos);
    q.tables = block_tables;
    q.ctx = ctx_lens;
    q.cu = cu_q;
    q.table_stride = table_stride;
    q.n_blocks = n_blocks;
    q.B = B;
    q.T = (int)T;
    q.limit = table_width * kKv4Page;
    if (rope_cs && n_pos < q.limit) q.limit = n_pos;
    q.n_layers = n_layers;
    q.layer = layer;
    q.Hkv = Hkv;
    if (T == 0 || B == 0) return TENZO_SUCCESS;
    TZ_CHECK(ctx_lens, "%s: null pointer", what);
    TZ_CHECK((pk && pv && pks && pvs) || n_blocks == 0, "%s: null pointer", what);
    TZ_CHECK(block_tables || table_width == 0, "%s: null pointer", what);
    TZ_CHECK((((uintptr_t)pk | (uintptr_t)pv) & 15) == 0 &&
                 (((uintptr_t)pks | (uintptr_t)pvs) & 3) == 0,
             "%s: code pools must be 16-byte aligned, scale pools 4-byte", what);
    return TENZO_SUCCESS;
}

}  // namespace tz

using namespace tz;

extern "C" {

TENZO_HIP_API int tenzo_hip_kv4_append(const void* k, const void* v, int dtype, int64_t k_stride,
                                       int64_t v_stride, uint8_t* pk, uint8_t* pv, uint8_t* pks,
                                       uint8_t* pvs, int64_t n_blocks, int n_layers, int layer,
                                       int Hkv, const int32_t* block_tables,
                                       int64_t table_stride, int table_width,
                                       const int32_t* ctx_lens, const int32_t* cu_q, int B,
                                       int64_t T, const float* rope_cs, int n_pos, void* stream) {
    Kv4Seqs q{};
    const int rc = kv4_check("kv4_append", pk, pv, pks, pvs, n_blocks, n_layers, layer, Hkv,
                             block_tables, table_stride, table_width, ctx_lens, cu_q, B, T,
                             rope_cs, n_pos, q);
    if (rc) return rc;
    TZ_CHECK(dtype == 0 || dtype == 1, "kv4_append: dtype %d", dtype);
    if (T == 0 || B == 0) return TENZO_SUCCESS;
    TZ_CHECK(k && v, "kv4_append: null pointer");
    TZ_CHECK(T == 1 || (k_stride >= (int64_t)Hkv * kKv4Dim && v_stride >= (int64_t)Hkv * kKv4Dim),
             "kv4_append: row strides %lld, %lld below %d heads", (long long)k_stride,
             (long long)v_stride, Hkv);
    Kv4Append a{k, v, k_stride, v_stride, pk, pv, pks, pvs, rope_cs, 0};
    const int64_t blocks = ceil_div(T * Hkv, 16);
    TZ_CHECK(blocks <= 0xffffff, "kv4_append: %lld rows of %d heads", (long long)T, Hkv);
    a.items = (int)(T * Hkv);
    const dim3 grid((unsigned)blocks);
    if (dtype)
        hipLaunchKernelGGL(kv4_append_kernel<true>, grid, dim3(256), 0, (hipStream_t)stream, a, q);
    else
        hipLaunchKernelGGL(kv4_append_kernel<false>, grid, dim3(256), 0, (hipStream_t)stream, a,
                           q);
    return launch_status("kv4_append_kernel");
}

TENZO_HIP_API int tenzo_hip_kv4_read(const uint8_t* pk, const uint8_t* pv, const uint8_t* pks,
                                     const uint8_t* pvs, int64_t n_blocks, int n_layers,
                                     int layer, int Hkv, const int32_t* block_tables,
                                     int64_t table_stride, int table_width,
                                     const int32_t* ctx_lens, const int32_t* cu_q, int B,
                                     int64_t T, void* k_out, void* v_out, int dtype,
                                     void* stream) {
    Kv4Seqs q{};
    const int rc = kv4_check("kv4_read", pk, pv, pks, pvs, n_blocks, n_layers, layer, Hkv,
                             block_tables, table_stride, table_width, ctx_lens, cu_q, B, T,
                             nullptr, 0, q);
    if (rc) return rc;
    TZ_CHECK(dtype == 0 || dtype == 1, "kv4_read: dtype %d", dtype);
    if (T == 0) return TENZO_SUCCESS;
    TZ_CHECK(k_out && v_out, "kv4_read: null pointer");
    TZ_CHECK((((uintptr_t)k_out | (uintptr_t)v_out) & 15) == 0,
             "kv4_read: outputs must be 16-byte aligned");
    Kv4Read a{pk, pv, pks, pvs, k_out, v_out, 0};
    const int64_t blocks = ceil_div(T * Hkv, 16);
    TZ_CHECK(blocks <= 0xffffff, "kv4_read: %lld rows of %d heads", (long long)T, Hkv);
    a.items = (int)(T * Hkv);
    const dim3 grid((unsigned)blocks);
    if (dtype)
        hipLaunchKernelGGL(kv4_read_kernel<true>, grid, dim3(256), 0, (hipStream_t)stream, a, q);
    else
        hipLaunchKernelGGL(kv4_read_kernel<false>, grid, dim3(256), 0, (hipStream_t)stream, a, q);
    return launch_status("kv4_read_kernel");
}

}  // extern "C"
