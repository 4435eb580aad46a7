// The product of 8-bit integers with a scale for each token and each channel:
// y[m][n] = float(sum_k codes[m][k] W[n][k]) * (q[m].inv_scale * scales[n]), sums exact in int32,
// over weights in the LM head's layout (blocks of 64 rows x 16 k, 1 KiB each, a row's blocks side
// by side).
#include "lds_ring.h"

namespace tz {
namespace {

typedef int i4v __attribute__((ext_vector_type(4)));
typedef int i16v __attribute__((ext_vector_type(16)));

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

// Two outputs of 16 bits, each rounded from its fp32 value.
template <int TYPE>
__device__ __forceinline__ uint32_t pack_y(float a, float b) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    if (TYPE == 1) return float_to_half_bits(a) | (uint32_t)float_to_half_bits(b) << 16;
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
}
// 16 bytes of outputs, and as they are stored: at any element's address.
template <int TYPE>
struct Out {
    typedef float type;
    struct __attribute__((packed, aligned(4))) any {
        float v __attribute__((ext_vector_type(4)));
    };
    any v;
};
template <>
struct Out<1> {
    typedef uint16_t type;
    struct __attribute__((packed, aligned(2))) any {
        uint16_t v __attribute__((ext_vector_type(8)));
    };
    any v;
};
template <>
struct Out<2> : Out<1> {};

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

// Many tokens: a workgroup of WR x WT x KW waves has 32 RT WR weight rows x 32 CT WT tokens, a wave
// 32 RT x 32 CT of them, and its KW groups of waves take turns of 64 k; their sums meet in LDS at
// the end. A step is a turn of every group. Its slot of the ring in LDS holds for each group
//   weights: blocks of 64 rows x 16 k as they are in memory (row r's 16 bytes at 16 r);
//   codes:   rows of 64 bytes, the 16-byte piece p of row r at place p ^ (r / 4 % 4) of it.
// Both are filled by loads straight into LDS, S - 1 steps ahead; a fragment of either is read
// with the 16 lanes that LDS serves together in different banks. The codes are the first operand,
// so that a register of the result holds 32 neighbouring channels of a token in 32 lanes.
// Each half of a step's fragments (32 k) is read while the half before it is multiplied.
template <int TYPE, int WR, int WT, int KW, int RT, int CT, int S>
__global__ void __launch_bounds__(64 * WR * WT * KW, WR * WT * KW >= 8 ? 1 : 2)
gemm_i8_tile_kernel(GemmI8 a) {
    constexpr int W = WR * WT * KW, BN = 32 * RT * WR, BM = 32 * CT * WT;
    static_assert(BN % 64 == 0, "whole blocks of rows");
    constexpr int kWLoads = BN / 16, kGroup = kWLoads + BM / 16;  // loads of 1 KiB per group
    constexpr int kSlot = KW * kGroup * 1024, X = KW * kGroup / W;
    static_assert(X * W == KW * kGroup, "as many loads a step for each wave");
    static_assert(S >= 3 && (S - 1) * X <= 63, "vmcnt counts at most 63 loads");
    constexpr int kRed = (KW - 1) * WR * WT * RT * CT * 4096, kRing = S * kSlot;
    static_assert(kRed + WR * WT * RT * 4096 <= kRing, "sums and outputs go out by way of the ring");
    __shared__ __attribute__((aligned(16))) char ring[kRing];
    __shared__ float inv[BM];

    const int lane = threadIdx.x & 63, i = lane & 31, g = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wr = wave % WR, wt = wave / WR % WT, kg = wave / (WR * WT);
    // Consecutive tiles to one XCD, as bands of 4 tiles of weight rows, so that what its
    // workgroups read at a time is few tiles of either operand.
    const int G = gridDim.x, id = blockIdx.x;
    const int tid = (G & 7) == 0 ? (id & 7) * (G >> 3) + (id >> 3) : id;
    const int nt = (int)((a.N + BN - 1) / BN), mt = (a.M + BM - 1) / BM;
    if (tid >= nt * mt) return;
    const int band = tid / (4 * mt), wide = min(4, nt - 4 * band), in_band = tid - band * 4 * mt;
    const int bn = 4 * band + in_band % wide, m0 = in_band / wide * BM;
    const int64_t n0 = (int64_t)bn * BN;
    const int rows = min(BM, a.M - m0), blocks = min(BN / 64, (int)((a.N + 63) / 64 - n0 / 64));
    const int K = a.KB * 16, steps = (a.KB + 4 * KW - 1) / (4 * KW);
    for (int m = threadIdx.x; m < BM; m += 64 * W) inv[m] = a.q[m0 + min(m, rows - 1)].inv_scale;

    const u4v rw = buf_words(a.w + (n0 >> 6) * ((int64_t)K * 64), (uint32_t)blocks * (uint32_t)K * 64u);
    const u4v rc = buf_words(a.codes + (int64_t)m0 * a.ldc, (uint32_t)((rows - 1) * a.ldc + K));
    // This wave's loads of a step: byte offsets, advanced from step to step. What lies past a row's
    // K (which the next row's codes may follow) is taken from past the resource, as zeros; weights
    // there count nothing then.
    uint32_t off[X];
    int left[X];  // K still in front of a lane's piece
#pragma unroll
    for (int x = 0; x < X; ++x) {
        const int l = (wave + W * x) % kGroup, k = (wave + W * x) / kGroup;
        const int row = 16 * (l - kWLoads) + (lane >> 2);
        const int piece = (lane & 3) ^ (row >> 2 & 3);
        off[x] = l < kWLoads ? (uint32_t)(l >> 2) * (uint32_t)K * 64u +
                                   (uint32_t)(4 * k + (l & 3)) * 1024u + (uint32_t)lane * 16u
                             : (uint32_t)(row * a.ldc) + (uint32_t)(64 * k + piece * 16);
        left[x] = l < kWLoads ? INT32_MAX : K - 64 * k - piece * 16;
    }
    auto load = [&](uint32_t slot, int x) {
        const int l = wave + W * x;
        const bool isw = l % kGroup < kWLoads;
        to_lds16_asm(isw ? rw : rc, slot + (uint32_t)l * 1024u, left[x] > 0 ? off[x] : 0x80000000u);
        off[x] += isw ? 4096u * KW : 64u * KW;
        left[x] -= isw ? 0 : 64 * KW;
    };

    i16v acc[RT][CT];
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int u = 0; u < CT; ++u) acc[t][u] = i16v{};
    struct Frag {
        i4v a[RT], b[CT];
    };
    const uint32_t wrow = (uint32_t)(kg * kGroup * 1024 + g * 1024 + i * 16);
    const uint32_t crow = (uint32_t)((kg * kGroup + kWLoads) * 1024 + (wt * CT * 32 + i) * 64);
    const uint32_t swz = (uint32_t)((g ^ (i >> 2 & 3)) * 16);
    auto read = [&](const char* slot, int h, Frag& f) {
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            const int rt = wr * RT + t;
            f.a[t] = *reinterpret_cast<const i4v*>(slot + wrow + (rt >> 1) * 4096 + h * 2048 +
                                                   (rt & 1) * 512);
        }
#pragma unroll
        for (int u = 0; u < CT; ++u)
            f.b[u] = *reinterpret_cast<const i4v*>(slot + crow + u * 2048 +
                                                   (swz ^ (uint32_t)(h * 32)));
    };
    auto mma = [&](const Frag& f, uint32_t slot, bool loads) {
#pragma unroll
        for (int t = 0; t < RT; ++t) {
#pragma unroll
            for (int u = 0; u < CT; ++u)
                acc[t][u] =
                    __builtin_amdgcn_mfma_i32_32x32x32_i8(f.b[u], f.a[t], acc[t][u], 0, 0, 0);
            if (loads)  // (a later step's go out between the products)
#pragma unroll
                for (int x = 0; x < X; ++x)
                    if (x * RT / X == t) load(slot, x);
        }
    };

    const uint32_t ring0 = lds_addr(ring);
    uint32_t in = ring0;  // the slot to load into next
#pragma unroll
    for (int j = 0; j < S - 1; ++j) {
#pragma unroll
        for (int x = 0; x < X; ++x) load(in, x);
        in += kSlot;
    }
    const char* cur = ring;
    const char* nxt = ring + kSlot;
    Frag f0, f1;
    wait_vm_asm<(S - 2) * X>();
    block_barrier();
    read(cur, 0, f0);
    for (int s = 0; s < steps; ++s) {
        wait_vm_asm<(S - 3) * X>();  // the next step's loads have landed
        __builtin_amdgcn_s_waitcnt(15 | (3 << 14) | (7 << 4));  // lgkmcnt(0)
        block_barrier();  // everyone's, and everyone has read the step before
        read(cur, 1, f1);
        issue_point();
        mma(f0, in, true);
        issue_point();
        in = in == ring0 + (S - 1) * kSlot ? ring0 : in + kSlot;
        read(nxt, 0, f0);
        issue_point();
        mma(f1, 0, false);
        cur = nxt;
        nxt = nxt == ring + (S - 1) * kSlot ? ring : nxt + kSlot;
        __builtin_amdgcn_sched_barrier(0);  // the step's products stay ahead of the next barrier
    }
    wait_vm_asm<0>();  // the loads past the end still write the ring
    __syncthreads();

    if (KW > 1) {  // groups 1 .. hand their sums to group 0
        i16v* red = reinterpret_cast<i16v*>(ring);
        const int wv = wave % (WR * WT);
        if (kg > 0) {
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int u = 0; u < CT; ++u)
                    red[((((kg - 1) * WR * WT + wv) * RT + t) * CT + u) * 64 + lane] = acc[t][u];
        }
        __syncthreads();
        if (kg > 0) return;
#pragma unroll
        for (int k = 0; k < KW - 1; ++k)
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int u = 0; u < CT; ++u)
                    acc[t][u] += red[(((k * WR * WT + wv) * RT + t) * CT + u) * 64 + lane];
    }

    // Register 4 q + e of acc[t][u]: channel 32 t + i, token 32 u + 8 q + 4 g + e. 32 tokens at a
    // time go through the wave's part of the ring, so that a lane stores 16 bytes of a token:
    // pieces of 16 bytes, in an order of the token's own that brings what is written at a time
    // into all banks. Two bytes of one or four to a store: 14 us of 256 x 256 outputs, 3 so.
    constexpr int E = TYPE ? 8 : 4, P = 32 * RT / E;  // outputs of a piece, pieces of a token
    auto place = [](int row) { return ((TYPE ? (row & 1) * 4 : 0) ^ (row >> 2 & 1) * 8) & (P - 1); };
    char* out = ring + kRed + wave % (WR * WT) * (RT * 4096);
    const int64_t nw = n0 + wr * RT * 32;
    float sc[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) sc[t] = nw + i + 32 * t < a.N ? a.scales[nw + i + 32 * t] : 0.0f;
#pragma unroll
    for (int u = 0; u < CT; ++u) {
        const int mu = (wt * CT + u) * 32;
        float bv[16];
        int bi[16];
#pragma unroll
        for (int r = 0; r < 16; r += 2) {
            const int row = 8 * (r >> 2) + 4 * g + (r & 3);
            const float iv[2] = {inv[mu + row], inv[mu + row + 1]};
            bv[r] = bv[r + 1] = -INFINITY;
            bi[r] = bi[r + 1] = (int)nw + i;
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                float y[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    y[k] = (float)acc[t][u][r + k] * __fmul_rn(iv[k], sc[t]);
                    if (a.best && nw + i + 32 * t < a.N && y[k] > bv[r + k]) {
                        bv[r + k] = y[k];
                        bi[r + k] = (int)nw + i + 32 * t;
                    }
                }
                const int n = 32 * t + i;
                if (TYPE == 0) {
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        *reinterpret_cast<float*>(out + (row + k) * (P * 16) +
                                                  (n / 4 ^ place(row + k)) * 16 + n % 4 * 4) = y[k];
                } else {
                    // (lanes of two neighbouring channels: one has both of a token, one of the next)
                    const int odd = i & 1;
                    const float other = dpp_f<kDppXor1>(odd ? y[0] : y[1]);
                    const uint32_t w = pack_y<TYPE>(odd ? other : y[0], odd ? y[1] : other);
                    *reinterpret_cast<uint32_t*>(out + (row + odd) * (P * 16) +
                                                 (n / 8 ^ place(row + odd)) * 16 + n % 8 / 2 * 4) =
                        w;
                }
            }
        }
        asm volatile("" ::: "memory");  // (a wave's accesses to LDS are made in order)
#pragma unroll
        for (int k = 0; k < P / 2; ++k) {
            const int at = lane + 64 * k, row = at / P, m = m0 + mu + row;
            const int64_t n = nw + (at % P ^ place(row)) * E;
            const Out<TYPE> v = *reinterpret_cast<const Out<TYPE>*>(out + at * 16);
            if (m >= a.M) continue;
            typename Out<TYPE>::type* y =
                reinterpret_cast<typename Out<TYPE>::type*>(a.y) + m * a.ldy + n;
            if (n + E <= a.N) {
                *reinterpret_cast<typename Out<TYPE>::any*>(y) = v.v;
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (n + e < a.N) y[e] = v.v.v[e];
            }
        }
        asm volatile("" ::: "memory");
        if (a.best) {
            // 16 tokens' best of 32 lanes: half of the tokens go to the other half of the lanes
            // each time, and the last of the five has one token in two lanes
#pragma unroll
            for (int d = 8; d >= 1; d >>= 1)
#pragma unroll
                for (int k = 0; k < d; ++k) {
                    const bool up = i & (d << 1);
                    float v = up ? bv[k + d] : bv[k];
                    int n = up ? bi[k + d] : bi[k];
                    take_best(v, n, __shfl_xor(up ? bv[k] : bv[k + d], d << 1),
                              __shfl_xor(up ? bi[k] : bi[k + d], d << 1));
                    bv[k] = v;
                    bi[k] = n;
                }
            take_best(bv[0], bi[0], __shfl_xor(bv[0], 1), __shfl_xor(bi[0], 1));
            const int r = i >> 1;  // (bits 4 .. 1 of the lane are bits 3 .. 0 of the token)
            const int m = m0 + mu + 8 * (r >> 2) + 4 * g + (r & 3);
            if ((i & 1) == 0 && m < a.M)
                a.best[(int64_t)m * a.parts + bn * WR + wr] = make_float2(bv[0], __int_as_float(bi[0]));
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

// The kernel for M tokens and N channels, and the parts that a row's largest value comes in.
enum GemmShape { kFewNarrow, kFewWide, kTile64, kTile128, kTile256 };
struct GemmPlan {
    GemmShape shape;
    int bm;     // tokens of a workgroup, few tokens
    int parts;  // columns: as many as the rows' bests
};
GemmPlan gemm_plan(int64_t M, int64_t N, int64_t K) {
    GemmPlan p;
    p.bm = M <= 16 ? 16 : M <= 32 ? 32 : 64;
    if (M <= 64) {
        p.shape = ceil_div(N, 64) >= 512 ? kFewWide : kFewNarrow;
        p.parts = (int)ceil_div(N, p.shape == kFewWide ? 64 : 16);
        return p;
    }
    if (ceil_div(M, 256) * ceil_div(N, 256) >= 160)
        p.shape = kTile256;
    else if (ceil_div(M, 128) * ceil_div(N, 128) >= 160)
        p.shape = kTile128;
    else
        p.shape = kTile64;
    p.parts = (int)(p.shape == kTile256 ? 2 * ceil_div(N, 256)
                    : p.shape == kTile128 ? 2 * ceil_div(N, 128) : 2 * ceil_div(N, 64));
    return p;
}

template <int MT>
void launch_few(const GemmPlan& p, const GemmI8& a, hipStream_t st) {
    const dim3 grid((unsigned)a.parts, (unsigned)ceil_div(a.M, p.bm));
    if (p.shape == kFewWide)
        hipLaunchKernelGGL((gemm_i8_few_kernel<MT, 4, 4, 4>), grid, dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((gemm_i8_few_kernel<MT, 1, 8, 4>), grid, dim3(512), 0, st, a);
}
template <int TYPE, int WR, int WT, int KW, int RT, int CT, int S>
void launch_tile(const GemmI8& a, hipStream_t st) {
    // (a number of workgroups that is shared out among the XCDs evenly: the last have no tile)
    const int64_t nt = ceil_div(a.N, 32 * RT * WR), mt = ceil_div(a.M, 32 * CT * WT);
    hipLaunchKernelGGL((gemm_i8_tile_kernel<TYPE, WR, WT, KW, RT, CT, S>),
                       dim3((unsigned)(ceil_div(nt * mt, 8) * 8)), dim3(64 * WR * WT * KW), 0, st, a);
}

template <int TYPE>
void launch_shape(GemmShape shape, const GemmI8& a, hipStream_t st) {
    if (shape == kTile256)
        launch_tile<TYPE, 2, 4, 1, 4, 2, 4>(a, st);
    else if (shape == kTile128)
        launch_tile<TYPE, 2, 2, 1, 2, 2, 4>(a, st);
    else
        launch_tile<TYPE, 2, 2, 2, 1, 1, 4>(a, st);
}

}  // namespace
}  // namespace tz

using namespace tz;

extern "C" {

TENZO_HIP_API size_t tenzo_hip_gemm_i8_ws_bytes(int64_t M, int64_t N, int64_t K, int want_idx) {
    if (M <= 0 || N <= 0 || K <= 0 || !want_idx) return 0;
    return (size_t)(M * gemm_plan(M, N, K).parts) * sizeof(float2);
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
    TZ_CHECK(M == 1 || (codes_stride >= K && codes_stride % 16 == 0 && codes_stride <= 1 << 22 &&
                        y_stride >= N),
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
    GemmI8 a{codes, M == 1 ? K : codes_stride, q, (const uint8_t*)w_packed, scales, y, y_stride,
             out_idx ? (float2*)ws : nullptr, N, (int)M, (int)(K / 16), p.parts, dtype};
    if (p.shape >= kTile64) {
        if (dtype == 0)
            launch_shape<0>(p.shape, a, st);
        else if (dtype == 1)
            launch_shape<1>(p.shape, a, st);
        else
            launch_shape<2>(p.shape, a, st);
    } else if (p.bm == 16)
        launch_few<1>(p, a, st);
    else if (p.bm == 32)
        launch_few<2>(p, a, st);
    else
        launch_few<4>(p, a, st);
    const int rc = launch_status("gemm_i8 kernel");
    if (rc || !out_idx) return rc;
    hipLaunchKernelGGL(gemm_i8_best_kernel, dim3((unsigned)M), dim3(256), 0, st, a.best, a.parts,
                       out_idx);
    return launch_status("gemm_i8_best_kernel");
}

}  // extern "C"
