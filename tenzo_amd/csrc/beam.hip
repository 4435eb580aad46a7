// Beam search on the device: the best k continuations of a request's W beams over the
// vocabulary, and the reordering of the beams' paged caches.
//
// Selection: candidate (w, t) has the score s_w + x_wt - log sum_u exp(x_wu), in 64 bits (two
// beams' candidates can lie closer than fp32 tells apart); the k largest are taken, among equal
// ones the lower beam, then the larger logit, then the lower token. So a beam's candidates come
// in the order of (logit, token) and the first k of each beam hold the answer. A logit that is not below +inf (NaN, +inf) counts as -inf.
#include <climits>

#include "common.h"

namespace tz {
namespace {

constexpr int kBeamMax = 64;  // beams and candidates, upper bounds

struct BeamSelect {
    const float* logits;
    const float* scores;
    int64_t stride;
    int W, k;
    int V;
    double* lse;   // [B * W]
    float2* cand;  // [B * W][k] value, index
    float* out_scores;
    int32_t* out_beams;
    int32_t* out_tokens;
};

__device__ __forceinline__ float beam_logit(float x) { return x < INFINITY ? x : -INFINITY; }

// Order "a before b" of (value, index).
__device__ __forceinline__ bool before(double a, int ia, double b, int ib) {
    return a > b || (a == b && ia < ib);
}

// The first of a workgroup's (value, index) pairs, in every thread.
__device__ __forceinline__ void block_first(double& v, int& i, double* rv, int* ri) {
    for (int d = 32; d > 0; d >>= 1) {
        const double ov = __shfl_xor(v, d);
        const int oi = __shfl_xor(i, d);
        if (before(ov, oi, v, i)) v = ov, i = oi;
    }
    if ((threadIdx.x & 63) == 0) rv[threadIdx.x >> 6] = v, ri[threadIdx.x >> 6] = i;
    __syncthreads();
    for (int w = 0; w < 4; ++w)
        if (before(rv[w], ri[w], v, i)) v = rv[w], i = ri[w];
    __syncthreads();
}

// The plain form: a workgroup per beam, one pass for the sum of exponentials and k for the best
// k logits, each the first after the one before.
__global__ void __launch_bounds__(256) beam_rows_kernel(BeamSelect a) {
    __shared__ double rv[4];
    __shared__ int ri[4];
    const int row = blockIdx.x, tid = threadIdx.x;
    const float* x = a.logits + row * a.stride;
    double last = INFINITY;
    int last_i = -1;
    double m = 0.0, sum = 0.0;
    for (int j = 0; j < a.k; ++j) {
        double v = -INFINITY;
        int i = INT_MAX;
        for (int t = tid; t < a.V; t += 256) {
            const double xv = beam_logit(x[t]);
            if (before(last, last_i, xv, t) && before(xv, t, v, i)) v = xv, i = t;
        }
        block_first(v, i, rv, ri);
        last = v;
        last_i = i;
        if (tid == 0) a.cand[(int64_t)row * a.k + j] = make_float2((float)v, __int_as_float(i));
        if (j == 0) {
            m = v == -INFINITY ? 0.0 : v;
            for (int t = tid; t < a.V; t += 256) sum += exp((double)beam_logit(x[t]) - m);
            for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
            if ((tid & 63) == 0) rv[tid >> 6] = sum;
            __syncthreads();
            if (tid == 0) a.lse[row] = m + log((rv[0] + rv[1]) + (rv[2] + rv[3]));
            __syncthreads();
        }
    }
}

__global__ void __launch_bounds__(256) beam_pick_kernel(BeamSelect a) {
    __shared__ double rv[4];
    __shared__ int ri[4];
    const int b = blockIdx.x, tid = threadIdx.x, n = a.W * a.k;
    double last = INFINITY;
    int last_i = -1;
    for (int j = 0; j < a.k; ++j) {
        double v = -INFINITY;
        int i = INT_MAX;
        for (int c = tid; c < n; c += 256) {
            const int w = c / a.k;
            const float2 e = a.cand[(int64_t)b * n + c];
            const int t = __float_as_int(e.y);
            if (t == INT_MAX) continue;  // a vocabulary smaller than k
            const double lse = a.lse[b * a.W + w], s = beam_logit(a.scores[b * a.W + w]);
            double xv = -INFINITY;
            if (e.x > -INFINITY) xv = s + ((double)e.x - lse);
            if (before(last, last_i, xv, c) && before(xv, c, v, i)) v = xv, i = c;
        }
        block_first(v, i, rv, ri);
        last = v;
        last_i = i;
        if (tid == 0) {
            a.out_scores[b * a.k + j] = (float)v;
            a.out_beams[b * a.k + j] = i / a.k;
            a.out_tokens[b * a.k + j] = __float_as_int(a.cand[(int64_t)b * n + i].y);
        }
    }
}

// ------------------------------------------------------------- reordering --

struct BeamReorder {
    const int32_t* parents;
    int32_t* tables;
    const int32_t* ctx;
    int64_t parent_stride, table_stride, n_blocks, planes;
    uint8_t* codes[2];
    uint8_t* scales[2];
    int B, W, width, row_bytes;
    int piece_blocks;
};

constexpr int kPageTokens = 16;

// In place: slot i of a request takes the cached tokens of slot parents[i]. The pages that are
// full change hands through the table; the rows of the page in progress are copied into the
// slot's own page. One thread moves one piece (16 bytes of codes, a row's scale or a column of
// the table) for all W slots: it has read every parent's piece before it writes the first, so
// no slot's piece is lost whatever the permutation, and no two threads touch the same piece.
template <int WMAX>
__global__ void __launch_bounds__(256) beam_reorder_kernel(BeamReorder a) {
    const int b = blockIdx.y;
    const int c = a.ctx[(int64_t)b * a.W];
    if (c <= 0 || c > a.width * kPageTokens) return;
    const int full = c / kPageTokens, fill = c % kPageTokens;
    const int32_t* parents = a.parents + b * a.parent_stride;
    int32_t* table = a.tables + (int64_t)b * a.W * a.table_stride;
    if ((int)blockIdx.x >= a.piece_blocks) {
        const int col = ((int)blockIdx.x - a.piece_blocks) * 256 + threadIdx.x;
        if (col >= full) return;
        int32_t v[WMAX];
#pragma unroll
        for (int i = 0; i < WMAX; ++i)
            if (i < a.W) {
                const int p = parents[i];
                v[i] = table[(p >= 0 && p < a.W ? p : i) * a.table_stride + col];
            }
#pragma unroll
        for (int i = 0; i < WMAX; ++i)
            if (i < a.W) {
                const int p = parents[i];
                if (p >= 0 && p < a.W && p != i) table[i * a.table_stride + col] = v[i];
            }
        return;
    }
    if (fill == 0) return;
    const int per_plane = 2 * a.row_bytes + 2 * kPageTokens;
    const int64_t item = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t plane = item / per_plane;
    int p = (int)(item - plane * per_plane);
    if (plane >= a.planes) return;
    const bool code = p < 2 * a.row_bytes;
    int which, token, off, page_bytes;
    uint8_t* pool;
    if (code) {
        which = p >= a.row_bytes;
        off = (p - which * a.row_bytes) * 16;
        token = off / a.row_bytes;
        page_bytes = a.row_bytes * kPageTokens;
        pool = a.codes[which];
    } else {
        p -= 2 * a.row_bytes;
        which = p >= kPageTokens;
        token = p - which * kPageTokens;
        off = token * 4;
        page_bytes = 4 * kPageTokens;
        pool = a.scales[which];
    }
    if (token >= fill) return;
    uint4 v[WMAX];
    int64_t dst[WMAX];
#pragma unroll
    for (int i = 0; i < WMAX; ++i) {
        dst[i] = -1;
        if (i >= a.W) continue;
        const int par = parents[i];
        if (par < 0 || par >= a.W || par == i) continue;
        const int64_t from = table[par * a.table_stride + full];
        const int64_t to = table[i * a.table_stride + full];
        if (from < 0 || from >= a.n_blocks || to < 0 || to >= a.n_blocks) continue;
        const uint8_t* src = pool + (from * a.planes + plane) * page_bytes + off;
        dst[i] = (to * a.planes + plane) * page_bytes + off;
        if (code)
            v[i] = *reinterpret_cast<const uint4*>(src);
        else
            v[i].x = *reinterpret_cast<const uint32_t*>(src);
    }
#pragma unroll
    for (int i = 0; i < WMAX; ++i) {
        if (i >= a.W || dst[i] < 0) continue;
        if (code)
            *reinterpret_cast<uint4*>(pool + dst[i]) = v[i];
        else
            *reinterpret_cast<uint32_t*>(pool + dst[i]) = v[i].x;
    }
}

}  // namespace
}  // namespace tz

using namespace tz;

extern "C" {

TENZO_HIP_API size_t tenzo_hip_beam_select_ws_bytes(int B, int W, int64_t V, int k) {
    (void)V;
    if (B <= 0 || W <= 0 || k <= 0) return 0;
    return (size_t)B * W * (8 + (size_t)k * 8);
}

TENZO_HIP_API int tenzo_hip_beam_select(const float* logits, int64_t row_stride,
                                        const float* scores, int B, int W, int64_t V, int k,
                                        float* out_scores, int32_t* out_beams,
                                        int32_t* out_tokens, void* ws, size_t ws_bytes,
                                        void* stream) {
    TZ_CHECK(B >= 0 && W > 0 && W <= kBeamMax && k > 0 && k <= kBeamMax,
             "beam_select: B=%d, 1 to %d beams (%d) and candidates (%d)", B, kBeamMax, W, k);
    TZ_CHECK(V > 0 && V * W < INT32_MAX && k <= V * W,
             "beam_select: %d of %lld candidates (V=%lld)", k, (long long)(V * W), (long long)V);
    TZ_CHECK((int64_t)B * W <= INT32_MAX / kBeamMax, "beam_select: %d x %d beams", B, W);
    if (B == 0) return TENZO_SUCCESS;
    TZ_CHECK(logits && scores && out_scores && out_beams && out_tokens,
             "beam_select: null pointer");
    TZ_CHECK(row_stride >= V || B * W == 1, "beam_select: rows %lld apart, V=%lld",
             (long long)row_stride, (long long)V);
    const size_t need = tenzo_hip_beam_select_ws_bytes(B, W, V, k);
    TZ_CHECK(ws && ws_bytes >= need && ((uintptr_t)ws & 7) == 0,
             "beam_select: %zu bytes of workspace needed, %zu given", need, ws ? ws_bytes : 0);
    BeamSelect a{};
    a.logits = logits;
    a.scores = scores;
    a.stride = row_stride;
    a.W = W;
    a.k = k;
    a.V = (int)V;
    a.lse = (double*)ws;
    a.cand = (float2*)((char*)ws + (size_t)B * W * 8);
    a.out_scores = out_scores;
    a.out_beams = out_beams;
    a.out_tokens = out_tokens;
    hipLaunchKernelGGL(beam_rows_kernel, dim3((unsigned)(B * W)), dim3(256), 0,
                       (hipStream_t)stream, a);
    const int rc = launch_status("beam_rows_kernel");
    if (rc) return rc;
    hipLaunchKernelGGL(beam_pick_kernel, dim3((unsigned)B), dim3(256), 0, (hipStream_t)stream, a);
    return launch_status("beam_pick_kernel");
}

TENZO_HIP_API int tenzo_hip_beam_reorder_paged(const int32_t* parents, int64_t parent_stride,
                                               int32_t* block_tables, int64_t table_stride,
                                               int table_width, const int32_t* ctx_lens, int B,
                                               int W, void* pk, void* pv, void* pks, void* pvs,
                                               int64_t n_blocks, int n_layers, int Hkv,
                                               int row_bytes, void* stream) {
    TZ_CHECK(B >= 0 && B <= 65535 && W > 0 && W <= kBeamMax,
             "beam_reorder_paged: B=%d, 1 to %d beams (%d)", B, kBeamMax, W);
    TZ_CHECK(n_layers > 0 && Hkv > 0 && n_blocks >= 0 && n_blocks <= INT32_MAX &&
                 (int64_t)n_layers * Hkv <= (1 << 20),
             "beam_reorder_paged: pools of %lld blocks, %d layers, %d heads", (long long)n_blocks,
             n_layers, Hkv);
    TZ_CHECK(row_bytes == 64 || row_bytes == 128,
             "beam_reorder_paged: rows of 64 or 128 code bytes (%d)", row_bytes);
    TZ_CHECK(table_width >= 0 && table_width <= INT32_MAX / kPageTokens &&
                 (table_stride >= table_width || (int64_t)B * W <= 1) &&
                 (parent_stride >= W || B <= 1),
             "beam_reorder_paged: tables of %d pages, %lld apart, parents %lld apart", table_width,
             (long long)table_stride, (long long)parent_stride);
    if (B == 0 || table_width == 0) return TENZO_SUCCESS;
    TZ_CHECK(parents && block_tables && ctx_lens, "beam_reorder_paged: null pointer");
    TZ_CHECK((pk && pv && pks && pvs) || n_blocks == 0, "beam_reorder_paged: null pointer");
    TZ_CHECK((((uintptr_t)pk | (uintptr_t)pv) & 15) == 0 &&
                 (((uintptr_t)pks | (uintptr_t)pvs) & 3) == 0,
             "beam_reorder_paged: code pools must be 16-byte aligned, scale pools 4-byte");
    BeamReorder a{};
    a.parents = parents;
    a.tables = block_tables;
    a.ctx = ctx_lens;
    a.parent_stride = parent_stride;
    a.table_stride = table_stride;
    a.n_blocks = n_blocks;
    a.planes = (int64_t)n_layers * Hkv;
    a.codes[0] = (uint8_t*)pk;
    a.codes[1] = (uint8_t*)pv;
    a.scales[0] = (uint8_t*)pks;
    a.scales[1] = (uint8_t*)pvs;
    a.B = B;
    a.W = W;
    a.width = table_width;
    a.row_bytes = row_bytes;
    a.piece_blocks = (int)ceil_div(a.planes * (2 * row_bytes + 2 * kPageTokens), 256);
    const dim3 grid((unsigned)(a.piece_blocks + ceil_div(table_width, 256)), (unsigned)B);
    if (W <= 8)
        hipLaunchKernelGGL(beam_reorder_kernel<8>, grid, dim3(256), 0, (hipStream_t)stream, a);
    else if (W <= 16)
        hipLaunchKernelGGL(beam_reorder_kernel<16>, grid, dim3(256), 0, (hipStream_t)stream, a);
    else
        hipLaunchKernelGGL(beam_reorder_kernel<kBeamMax>, grid, dim3(256), 0, (hipStream_t)stream,
                           a);
    return launch_status("beam_reorder_kernel");
}

}  // extern "C"
