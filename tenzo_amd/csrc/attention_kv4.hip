// Attention over the paged cache held in 4 bits (layout: kv4.h): every row of queries at its own
// position of its own sequence, o = sum_t softmax_t(q.k_t / sqrt(128)) v_t over the positions up
// to its own; a row that sees no position is zero.
#include "kv4.h"

namespace tz {
namespace {

constexpr float kQkScale = 0.08838834764831845f;  // 1/sqrt(128)

struct Kv4Attn {
    const void* q;
    void* out;
    int64_t q_stride, out_stride;
    const uint8_t* pk;
    const uint8_t* pv;
    const uint8_t* pks;
    const uint8_t* pvs;
    const float* rope;
    int G;
};

// The plain form: a workgroup per (row, query head), a token to a thread, 256 at a time with the
// running maximum and sum of the softmax.
template <bool HALF>
__global__ void __launch_bounds__(256) kv4_attn_plain_kernel(Kv4Attn a, Kv4Seqs sq) {
    __shared__ float qs[kKv4Dim], ps[256], red[4];
    __shared__ int64_t rows[256];
    const int tid = threadIdx.x, row = blockIdx.x, qh = blockIdx.y, h = qh / a.G;
    int seq, pos;
    const bool there = kv4_place(sq, row, tid & 15, seq, pos);
    if (!there) {
        if (seq < sq.B && (!sq.cu || row >= sq.cu[0]) && tid < kKv4Dim)
            st_act<HALF>(a.out, row * a.out_stride + (int64_t)qh * kKv4Dim + tid, 0.0f);
        return;
    }
    if (tid < 64) {
        const int64_t at = row * a.q_stride + (int64_t)qh * kKv4Dim + tid;
        float x0 = ld_act<HALF>(a.q, at), x1 = ld_act<HALF>(a.q, at + 64);
        if (a.rope) {
            const float* cs = a.rope + (int64_t)pos * kKv4Dim + tid;
            const float c = cs[0], s = cs[64], y0 = x0;
            x0 = __builtin_fmaf(x0, c, -__fmul_rn(x1, s));
            x1 = __builtin_fmaf(y0, s, __fmul_rn(x1, c));
        }
        qs[tid] = __fmul_rn(x0, kQkScale);
        qs[tid + 64] = __fmul_rn(x1, kQkScale);
    }
    __syncthreads();
    float m = -INFINITY, l = 0.0f, o = 0.0f;
    for (int t0 = 0; t0 <= pos; t0 += 256) {
        const int t = t0 + tid;
        float s = -INFINITY;
        int64_t r = -1;
        if (t <= pos) {
            const int64_t base = sq.page_base(seq, t / kKv4Page);
            if (base >= 0) {
                r = base + h * kKv4Page + t % kKv4Page;
                s = 0.0f;
                for (int w = 0; w < 16; ++w) {
                    float v[8];
                    fp4_to_float8(reinterpret_cast<const uint32_t*>(a.pk + r * kKv4Row)[w],
                                  e8m0_to_float(a.pks[r * kKv4Scales + w / 4]), v);
                    for (int j = 0; j < 8; ++j) s = __builtin_fmaf(qs[8 * w + j], v[j], s);
                }
            }
        }
        const float mc = fmaxf(m, block256_max(s, red));
        const float scale = m == -INFINITY ? 0.0f : expf(m - mc);
        ps[tid] = r < 0 ? 0.0f : expf(s - mc);
        rows[tid] = r;
        m = mc;
        __syncthreads();
        l *= scale;
        o *= scale;
        for (int i = 0; i < 256; ++i) {
            if (rows[i] < 0) continue;
            l += ps[i];
            if (tid < kKv4Dim) {
                const uint32_t c = (a.pv[rows[i] * kKv4Row + tid / 2] >> (4 * (tid & 1))) & 15;
                const f32x2 v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(
                    c, e8m0_to_float(a.pvs[rows[i] * kKv4Scales + tid / 32]), 0);
                o = __builtin_fmaf(ps[i], v.x, o);
            }
        }
        __syncthreads();
    }
    if (tid < kKv4Dim)
        st_act<HALF>(a.out, row * a.out_stride + (int64_t)qh * kKv4Dim + tid,
                     l > 0.0f || l != l ? o / l : 0.0f);
}

}  // namespace
}  // namespace tz

using namespace tz;

extern "C" {

TENZO_HIP_API size_t tenzo_hip_attn_kv4_ws_bytes(int64_t T, int B, int Hq, int Hkv,
                                                 int table_width) {
    return 0;
}

TENZO_HIP_API int tenzo_hip_attn_kv4(const void* q, int dtype, int64_t q_stride,
                                     const uint8_t* pk, const uint8_t* pv, const uint8_t* pks,
                                     const uint8_t* pvs, int64_t n_blocks, int n_layers,
                                     int layer, int Hq, int Hkv, const int32_t* block_tables,
                                     int64_t table_stride, int table_width,
                                     const int32_t* ctx_lens, const int32_t* cu_q, int B,
                                     int64_t T, const float* rope_cs, int n_pos, void* out,
                                     int64_t out_stride, void* ws, size_t ws_bytes,
                                     void* stream) {
    Kv4Seqs s{};
    const int rc = kv4_check("attn_kv4", pk, pv, pks, pvs, n_blocks, n_layers, layer, Hkv,
                             block_tables, table_stride, table_width, ctx_lens, cu_q, B, T,
                             rope_cs, n_pos, s);
    if (rc) return rc;
    TZ_CHECK(dtype == 0 || dtype == 1, "attn_kv4: dtype %d", dtype);
    TZ_CHECK(Hq > 0 && Hq % Hkv == 0 && Hq / Hkv <= 16,
             "attn_kv4: 1 to 16 query heads a kv head (Hq=%d Hkv=%d)", Hq, Hkv);
    if (T == 0 || B == 0) return TENZO_SUCCESS;
    TZ_CHECK(q && out, "attn_kv4: null pointer");
    TZ_CHECK(T == 1 || (q_stride >= (int64_t)Hq * kKv4Dim && out_stride >= (int64_t)Hq * kKv4Dim),
             "attn_kv4: row strides %lld, %lld below %d heads", (long long)q_stride,
             (long long)out_stride, Hq);
    const size_t need = tenzo_hip_attn_kv4_ws_bytes(T, B, Hq, Hkv, table_width);
    TZ_CHECK(need == 0 || (ws && ws_bytes >= need), "attn_kv4: %zu bytes of workspace needed, %zu given",
             need, ws ? ws_bytes : 0);
    Kv4Attn a{q, out, q_stride, out_stride, pk, pv, pks, pvs, rope_cs, Hq / Hkv};
    const dim3 grid((unsigned)T, (unsigned)Hq);
    if (dtype)
        hipLaunchKernelGGL(kv4_attn_plain_kernel<true>, grid, dim3(256), 0, (hipStream_t)stream,
                           a, s);
    else
        hipLaunchKernelGGL(kv4_attn_plain_kernel<false>, grid, dim3(256), 0, (hipStream_t)stream,
                           a, s);
    return launch_status("kv4_attn_plain_kernel");
}

}  // extern "C"
