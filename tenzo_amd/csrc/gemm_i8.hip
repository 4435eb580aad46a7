// The product of 8-bit integers with a scale for each token and each channel:
// y[m][n] = float(sum_k codes[m][k] W[n][k]) * (q[m].inv_scale * scales[n]), sums exact in int32,
// over weights in the LM head's layout (blocks of 64 rows x 16 k, 1 KiB each, a row's blocks side
// by side).
#include "common.h"

namespace tz {
namespace {

typedef int i4v __attribute__((ext_vector_type(4)));

struct GemmI8 {
    const int8_t* codes;
    int64_t ldc;
    const tenzo_hip_actq_t* q;
    const uint8_t* w;
    const float* scales;
    void* y;
    int64_t ldy;
    float2* best;  // [M][parts]: a row's largest value of some columns and its column (null: not asked)
    int64_t N;
    int M, KB;  // KB: K / 16
    int parts;
    int dtype;
};

__device__ __forceinline__ void store_y(const GemmI8& a, int64_t at, float v) {
    if (a.dtype == 0)
        reinterpret_cast<float*>(a.y)[at] = v;
    else if (a.dtype == 1)
        reinterpret_cast<uint16_t*>(a.y)[at] = float_to_half_bits(v);
    else
        reinterpret_cast<__bf16*>(a.y)[at] = (__bf16)v;
}

// The larger value, of equal ones the lower column; NaN counts as -inf.
__device__ __forceinline__ void take_best(float& v, int& n, float ov, int on) {
    if (ov > v || (ov == v && on < n)) {
        v = ov;
        n = on;
    }
}

// Few tokens: 16 NT rows of weights to a workgroup, whose KW waves share K: a wave has every KW-th
// 64 of it, straight from memory to the matrix cores' operands, DEPTH steps ahead. The codes of the
// 16 MT tokens come the same way, out of the L2. At the end the waves' sums meet in LDS.
template <int MT, int NT, int KW, int DEPTH>
__global__ void __launch_bounds__(64 * KW) gemm_i8_few_kernel(GemmI8 a) {
    __shared__ i4v red[KW][NT * MT][64];
    const int lane = threadIdx.x & 63, col = lane & 15, j = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t n0 = (int64_t)blockIdx.x * (16 * NT);
    const int m0 = blockIdx.y * (16 * MT);
    const int steps = (a.KB + 3) >> 2, mine = steps > wave ? (steps - wave + KW - 1) / KW : 0;
    const uint8_t* wb = a.w + (n0 >> 6) * ((int64_t)a.KB << 10) + ((n0 & 63) + col) * 16;
    const int8_t* ab[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) ab[t] = a.codes + (int64_t)min(m0 + 16 * t + col, a.M - 1) * a.ldc;
    i4v wv[DEPTH][NT], av[DEPTH][MT];
    auto load = [&](int u, int i) {  // (past the last: that one again)
        const int st = min(wave + KW * max(min(i, mine - 1), 0), steps - 1);
        const int kb = min(4 * st + j, a.KB - 1);
#pragma unroll
        for (int t = 0; t < NT; ++t)
            wv[u][t] = __builtin_nontemporal_load(
                reinterpret_cast<const i4v*>(wb + ((int64_t)kb << 10) + t * 256));
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            av[u][t] = *reinterpret_cast<const i4v*>(ab[t] + kb * 16);
            if (4 * st + j >= a.KB) av[u][t] = i4v{0, 0, 0, 0};
        }
    };
    i4v acc[NT][MT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int s = 0; s < MT; ++s) acc[t][s] = i4v{0, 0, 0, 0};
#pragma unroll
    for (int u = 0; u < DEPTH; ++u) load(u, u);
    for (int i = 0; i < mine; i += DEPTH) {
#pragma unroll
        for (int u = 0; u < DEPTH; ++u) {
            if (i + u < mine) {
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int s = 0; s < MT; ++s)
                        acc[t][s] = __builtin_amdgcn_mfma_i32_16x16x64_i8(av[u][s], wv[u][t],
                                                                         acc[t][s], 0, 0, 0);
            }
            load(u, i + u + DEPTH);
        }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int s = 0; s < MT; ++s) red[wave][t * MT + s][lane] = acc[t][s];
    __syncthreads();
    // thread: a row of the tile and a column, the columns side by side
    for (int it = threadIdx.x; it < 16 * MT * 16 * NT; it += 64 * KW) {
        const int nn = it % (16 * NT), mm = it / (16 * NT), m = m0 + mm;
        const int64_t n = n0 + nn;
        const int tile = nn / 16 * MT + mm / 16, from = nn % 16 + 16 * (mm % 16 / 4);
        int sum = 0;
#pragma unroll
        for (int w = 0; w < KW; ++w) sum += red[w][tile][from][mm % 4];
        float v = -INFINITY;
        if (m < a.M && n < a.N) {
            const float y = (float)sum * __fmul_rn(a.q[m].inv_scale, a.scales[n]);
            store_y(a, m * a.ldy + n, y);
            if (y > v) v = y;
        }
        if (a.best) {
            int at = (int)n;
#pragma unroll
            for (int d = 1; d < 16 * NT; d <<= 1)
                take_best(v, at, __shfl_xor(v, d), __shfl_xor(at, d));
            if (nn == 0 && m < a.M)
                a.best[(int64_t)m * a.parts + blockIdx.x] = make_float2(v, __int_as_float(at));
        }
    }
}

__global__ void __launch_bounds__(256) gemm_i8_best_kernel(const float2* best, int parts,
                                                           int32_t* out) {
    __shared__ float rv[4];
    __shared__ int ri[4];
    const float2* row = best + (int64_t)blockIdx.x * parts;
    float v = -INFINITY;
    int n = INT32_MAX;
    for (int i = threadIdx.x; i < parts; i += 256) {
        const float2 e = row[i];
        take_best(v, n, e.x, __float_as_int(e.y));
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) take_best(v, n, __shfl_xor(v, d), __shfl_xor(n, d));
    if ((threadIdx.x & 63) == 0) {
        rv[threadIdx.x >> 6] = v;
        ri[threadIdx.x >> 6] = n;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 4; ++w) take_best(v, n, rv[w], ri[w]);
        out[blockIdx.x] = n;
    }
}

// Tokens and weight rows of a workgroup.
struct GemmPlan {
    int bm, bn;
};
GemmPlan gemm_plan(int64_t M, int64_t N, int64_t K) {
    GemmPlan p;
    p.bm = M <= 16 ? 16 : M <= 32 ? 32 : 64;
    p.bn = ceil_div(N, 64) * ceil_div(M, p.bm) >= 512 ? 64 : 16;
    return p;
}

template <int MT>
void launch_few(const GemmPlan& p, const GemmI8& a, hipStream_t st) {
    const dim3 grid((unsigned)ceil_div(a.N, p.bn), (unsigned)ceil_div(a.M, p.bm));
    if (p.bn == 64)
        hipLaunchKernelGGL((gemm_i8_few_kernel<MT, 4, 4, 4>), grid, dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((gemm_i8_few_kernel<MT, 1, 8, 4>), grid, dim3(512), 0, st, a);
}

}  // namespace
}  // namespace tz

using namespace tz;

extern "C" {

TENZO_HIP_API size_t tenzo_hip_gemm_i8_ws_bytes(int64_t M, int64_t N, int64_t K, int want_idx) {
    if (M <= 0 || N <= 0 || K <= 0 || !want_idx) return 0;
    return (size_t)(M * ceil_div(N, gemm_plan(M, N, K).bn)) * sizeof(float2);
}

TENZO_HIP_API int tenzo_hip_gemm_i8(const int8_t* codes, int64_t codes_stride,
                                    const tenzo_hip_actq_t* q, const void* w_packed,
                                    const float* scales, int64_t M, int64_t N, int64_t K, void* y,
                                    int dtype, int64_t y_stride, int32_t* out_idx, void* ws,
                                    size_t ws_bytes, void* stream) {
    TZ_CHECK(dtype >= 0 && dtype <= 2, "gemm_i8: dtype %d", dtype);
    TZ_CHECK(M >= 0 && M <= (1 << 20) && N > 0 && N <= (1 << 30), "gemm_i8: M=%lld N=%lld",
             (long long)M, (long long)N);
    // (sums of K products of at most 2^14 stay within int32)
    TZ_CHECK(K > 0 && K % 16 == 0 && K <= 131056, "gemm_i8: K=%lld, not a multiple of 16 up to "
             "131056", (long long)K);
    if (M == 0) return TENZO_SUCCESS;
    TZ_CHECK(codes && q && w_packed && scales && y, "gemm_i8: null pointer");
    TZ_CHECK(M == 1 || (codes_stride >= K && codes_stride % 16 == 0 && y_stride >= N),
             "gemm_i8: row strides %lld, %lld of %lld codes, %lld outputs",
             (long long)codes_stride, (long long)y_stride, (long long)K, (long long)N);
    TZ_CHECK((((uintptr_t)codes | (uintptr_t)w_packed) & 15) == 0 &&
                 (((uintptr_t)q | (uintptr_t)scales) & 3) == 0 &&
                 ((uintptr_t)y & (dtype ? 1 : 3)) == 0,
             "gemm_i8: codes and weights must be 16-byte aligned, the others to their elements");
    const size_t need = tenzo_hip_gemm_i8_ws_bytes(M, N, K, out_idx != nullptr);
    TZ_CHECK(need == 0 || (ws && ws_bytes >= need && ((uintptr_t)ws & 7) == 0),
             "gemm_i8: %zu bytes of workspace needed, 8-byte aligned, %zu given", need,
             ws ? ws_bytes : 0);
    const GemmPlan p = gemm_plan(M, N, K);
    const hipStream_t st = (hipStream_t)stream;
    GemmI8 a{codes, codes_stride, q, (const uint8_t*)w_packed, scales, y, y_stride,
             out_idx ? (float2*)ws : nullptr, N, (int)M, (int)(K / 16), (int)ceil_div(N, p.bn),
             dtype};
    if (p.bm == 16)
        launch_few<1>(p, a, st);
    else if (p.bm == 32)
        launch_few<2>(p, a, st);
    else
        launch_few<4>(p, a, st);
    const int rc = launch_status("gemm_i8_few_kernel");
    if (rc || !out_idx) return rc;
    hipLaunchKernelGGL(gemm_i8_best_kernel, dim3((unsigned)M), dim3(256), 0, st, a.best, a.parts,
                       out_idx);
    return launch_status("gemm_i8_best_kernel");
}

}  // extern "C"
