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
    int full;  // (tiles: the first that comes as halves)
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

// The larger value, of equal ones the lower column; NaN counts as -inf. (Without a branch: of ||, &&
// and if, the compiler lost the assignment for equal values where v and n are of an array of 16 - the
// body of the branch was empty -, so that the higher of two equal columns could be the answer.)
__device__ __forceinline__ void take_best(float& v, int& n, float ov, int on) {
    const bool take = (ov > v) | ((ov == v) & (on < n));
    v = take ? ov : v;
    n = take ? on : n;
}

// A token of 2 D from either half of a wave's rows of 16 lanes: lanes with bit 4 keep the upper D.
template <int D, int N>
__device__ __forceinline__ void best_swap16(float (&v)[N], int (&n)[N]) {
#pragma unroll
    for (int k = 0; k < D; ++k) {
        const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[k]),
                                                        __float_as_uint(v[k + D]), false, false);
        const auto b = __builtin_amdgcn_permlane16_swap((uint32_t)n[k], (uint32_t)n[k + D], false,
                                                        false);
        v[k] = __uint_as_float(a[0]);
        n[k] = (int)b[0];
        take_best(v[k], n[k], __uint_as_float(a[1]), (int)b[1]);
    }
}
// From either half of the wave: the upper 32 lanes keep the upper D.
template <int D, int N>
__device__ __forceinline__ void best_swap32(float (&v)[N], int (&n)[N]) {
#pragma unroll
    for (int k = 0; k < D; ++k) {
        const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[k]),
                                                        __float_as_uint(v[k + D]), false, false);
        const auto b = __builtin_amdgcn_permlane32_swap((uint32_t)n[k], (uint32_t)n[k + D], false,
                                                        false);
        v[k] = __uint_as_float(a[0]);
        n[k] = (int)b[0];
        take_best(v[k], n[k], __uint_as_float(a[1]), (int)b[1]);
    }
}
// And of 2 D tokens: lanes that are `up` keep the upper D, their partners by CTRL the others.
template <int D, int CTRL, int N>
__device__ __forceinline__ void best_halve(float (&v)[N], int (&n)[N], bool up) {
#pragma unroll
    for (int k = 0; k < D; ++k) {
        const float give = up ? v[k] : v[k + D];
        const int give_n = up ? n[k] : n[k + D];
        v[k] = up ? v[k + D] : v[k];
        n[k] = up ? n[k + D] : n[k];
        take_best(v[k], n[k], dpp_f<CTRL>(give), dpp_i<CTRL>(give_n));
    }
}

// Few tokens: 16 NT rows of weights to a workgroup, whose KW waves share K: a wave has every KW-th
// 128 of it, straight from memory to the matrix cores' operands, both halves loaded a turn ahead
// (loads three to seven steps ahead, or 16 waves where there are tokens, take longer; a line of codes,
// 128 bytes of a row, belongs to one wave's turn). The codes of the 16 MT tokens come the same way,
// out of the L2. At the end the waves' sums meet in LDS. 1 x 2560 x 6912: 5.7 us, 24 x 2560 x 6912:
// 8.4, where the weights take 3.5: a launch, 7 dependent rounds of loads, and the meeting;
// 26 x 128256 x 2560: 64 to 66 us, 5.1 TB/s, bound by the weights.
constexpr uint32_t kNone = 0x80000000u;  // an offset past every resource
constexpr int kNt = 2;                   // a load that leaves nothing in the caches
template <int MT, int NT, int KW>
__global__ void __launch_bounds__(64 * KW) gemm_i8_few_kernel(GemmI8 a) {
    __shared__ i4v red[KW][NT * MT][64];
    const int lane = threadIdx.x & 63, col = lane & 15, j = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t n0 = (int64_t)blockIdx.x * (16 * NT);
    const int m0 = blockIdx.y * (16 * MT);
    const int turns = ((a.KB + 7) / 8 - wave + KW - 1) / KW;
    // (what lies past K, or past the last turn, is taken from past the resources: zeros, and nothing
    // is read)
    const int rows = min(16 * MT, a.M - m0);
    const auto rw = buf(a.w + (n0 >> 6) * ((int64_t)a.KB << 10), (uint32_t)a.KB << 10);
    const auto rc = buf(a.codes + (int64_t)m0 * a.ldc, (uint32_t)((rows - 1) * a.ldc + a.KB * 16));
    const uint32_t w0 = (uint32_t)((n0 & 63) + col) * 16, c0 = (uint32_t)(col * a.ldc);
    i4v wv[2][NT], av[2][MT];
    auto load = [&](int u, int turn) {
        const uint32_t kb = (uint32_t)(8 * (wave + KW * turn) + 4 * u + j);
#pragma unroll
        for (int t = 0; t < NT; ++t)
            wv[u][t] = __builtin_bit_cast(
                i4v, __builtin_amdgcn_raw_buffer_load_b128(rw, w0 + (kb << 10) + t * 256, 0, kNt));
#pragma unroll
        for (int t = 0; t < MT; ++t)
            av[u][t] = __builtin_bit_cast(
                i4v, __builtin_amdgcn_raw_buffer_load_b128(
                         rc, kb < (uint32_t)a.KB ? c0 + (uint32_t)(16 * t * a.ldc) + kb * 16 : kNone,
                         0, 0));
    };
    i4v acc[NT][MT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int s = 0; s < MT; ++s) acc[t][s] = i4v{0, 0, 0, 0};
#pragma unroll
    for (int u = 0; u < 2; ++u) load(u, 0);
    for (int i = 0; i < turns; ++i) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int s = 0; s < MT; ++s)
                    acc[t][s] = __builtin_amdgcn_mfma_i32_16x16x64_i8(av[u][s], wv[u][t], acc[t][s],
                                                                     0, 0, 0);
            load(u, i + 1);
        }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int s = 0; s < MT; ++s) red[wave][t * MT + s][lane] = acc[t][s];
    __syncthreads();
    // thread: a row of the tile and a column, the columns side by side
    constexpr int kOutputs = 16 * MT * 16 * NT, PER = (kOutputs + 64 * KW - 1) / (64 * KW);
    float best[PER];
    int at[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int it = threadIdx.x + 64 * KW * k;
        if (it >= kOutputs) return;
        const int nn = it % (16 * NT), mm = it / (16 * NT), m = m0 + mm;
        const int64_t n = n0 + nn;
        const int tile = nn / 16 * MT + mm / 16, from = nn % 16 + 16 * (mm % 16 / 4);
        int sum = 0;
#pragma unroll
        for (int w = 0; w < KW; ++w) sum += red[w][tile][from][mm % 4];
        best[k] = -INFINITY;
        at[k] = (int)n;
        if (m < a.M && n < a.N) {
            const float y = (float)sum * __fmul_rn(a.q[m].inv_scale, a.scales[n]);
            store_y(a, m * a.ldy + n, y);
            if (y > best[k]) best[k] = y;
        }
    }
    if (!a.best) return;
    if constexpr (PER == 8 && NT == 4) {
        // 8 tokens' best of 64 lanes: half of them go to the other half of the lanes each time (lane
        // bits 5, 4, 3 become bits 2, 1, 0 of the token's number), then each has 8 lanes
        best_swap32<4>(best, at);
        best_swap16<2>(best, at);
        best_halve<1, kDppMirror>(best, at, lane & 8);
        take_best(best[0], at[0], dpp_f<kDppHalfMirror>(best[0]), dpp_i<kDppHalfMirror>(at[0]));
        take_best(best[0], at[0], dpp_f<kDppXor2>(best[0]), dpp_i<kDppXor2>(at[0]));
        take_best(best[0], at[0], dpp_f<kDppXor1>(best[0]), dpp_i<kDppXor1>(at[0]));
        const int k = (lane >> 5) * 4 + (lane >> 4 & 1) * 2 + (lane >> 3 & 1), m = m0 + wave + KW * k;
        if ((lane & 7) == 0 && m < a.M)
            a.best[(int64_t)m * a.parts + blockIdx.x] = make_float2(best[0], __int_as_float(at[0]));
    } else {
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            float v = best[k];
            int n = at[k];
            take_best(v, n, dpp_f<kDppXor1>(v), dpp_i<kDppXor1>(n));
            take_best(v, n, dpp_f<kDppXor2>(v), dpp_i<kDppXor2>(n));
            take_best(v, n, dpp_f<kDppHalfMirror>(v), dpp_i<kDppHalfMirror>(n));
            take_best(v, n, dpp_f<kDppMirror>(v), dpp_i<kDppMirror>(n));
#pragma unroll
            for (int d = 16; d < 16 * NT; d <<= 1)
                take_best(v, n, __shfl_xor(v, d), __shfl_xor(n, d));
            const int it = threadIdx.x + 64 * KW * k, m = m0 + it / (16 * NT);
            if (it % (16 * NT) == 0 && m < a.M)
                a.best[(int64_t)m * a.parts + blockIdx.x] = make_float2(v, __int_as_float(n));
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
// 4001 x 6912 x 2560, fp16: 78 us, 1.8 POP/s. The matrix units are busy in 46% of the cycles (58% of
// those in which a CU has a tile: 864 of them leave CUs without one a fifth of the time), at the 1.87 GHz
// that the power of random data leaves: zeros take the same cycles at 2.4 GHz, 64 us. 300 x 128256 x
// 2560, fp16, with the largest: 159 us.
template <int WR, int WT, int KW, int RT, int CT, int S>
struct GemmTile {
    static constexpr int W = WR * WT * KW, BN = 32 * RT * WR, BM = 32 * CT * WT;
    static_assert(BN % 64 == 0, "whole blocks of rows");
    static constexpr int kWLoads = BN / 16, kGroup = kWLoads + BM / 16;  // loads of 1 KiB per group
    static constexpr int kSlot = KW * kGroup * 1024, X = KW * kGroup / W;
    static_assert(X * W == KW * kGroup, "as many loads a step for each wave");
    static_assert(S >= 3 && (S - 1) * X <= 63, "vmcnt counts at most 63 loads");
    static constexpr int kRed = (KW - 1) * WR * WT * RT * CT * 4096, kRing = S * kSlot;
    static_assert(kRed + WR * WT * RT * 4096 <= kRing, "sums and outputs go out by way of the ring");

    // The tile of channels from n0 (its number among those: bn) and tokens from m0.
    template <int TYPE, bool BEST>
    static __device__ __forceinline__ void run(const GemmI8& a, int64_t n0, int bn, int m0,
                                               char* ring, float* inv);
};

template <int WR, int WT, int KW, int RT, int CT, int S>
template <int TYPE, bool BEST>
__device__ __forceinline__ void GemmTile<WR, WT, KW, RT, CT, S>::run(const GemmI8& a, int64_t n0,
                                                                     int bn, int m0, char* ring,
                                                                     float* inv) {
    const int lane = threadIdx.x & 63, i = lane & 31, g = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wr = wave % WR, wt = wave / WR % WT, kg = wave / (WR * WT);
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
        if (m0 + mu >= a.M) break;
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
                    if (BEST && nw + i + 32 * t < a.N && y[k] > bv[r + k]) {
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
        if (BEST) {
            // 16 tokens' best of 32 lanes: half of the tokens go to the other half of the lanes
            // each time (lane bits 4 .. 1 become token bits 3 .. 0), the last time a token has two
            best_swap16<8>(bv, bi);
            best_halve<4, kDppMirror>(bv, bi, i & 8);
            best_halve<2, kDppHalfMirror>(bv, bi, i & 4);
            best_halve<1, kDppXor2>(bv, bi, i & 2);
            take_best(bv[0], bi[0], dpp_f<kDppXor1>(bv[0]), dpp_i<kDppXor1>(bi[0]));
            const int r = i >> 1, m = m0 + mu + 8 * (r >> 2) + 4 * g + (r & 3);
            if ((i & 1) == 0 && m < a.M)
                a.best[(int64_t)m * a.parts + bn * WR + wr] =
                    make_float2(bv[0], __int_as_float(bi[0]));
        }
    }
}

// HALVES: tiles from a.full on come as two halves of their channels, where up to 128 tiles are left
// over from a multiple of 256: a CU with one tile more than the others makes all wait for it, a half
// takes less. us, whole | halves: 1024 x 20480 x 2560 (640 tiles) 70 | 62, 2500 x 6912 x 2560 (540) 68 |
// 60, 8000 x 2560 x 2560 (630) 69 | 65; no change where the multiple is odd (864 tiles: 81), since
// two tiles of a CU take little longer than one.
template <int TYPE, bool BEST, int WR, int WT, int KW, int RT, int CT, int S, bool HALVES>
__global__ void __launch_bounds__(64 * WR * WT * KW, RT * CT > 4 || KW > 1 ? 2 : WR * WT / 2)
gemm_i8_tile_kernel(GemmI8 a) {
    typedef GemmTile<WR, WT, KW, RT, CT, S> Tile;
    typedef GemmTile<WR, WT, KW, HALVES ? RT / 2 : RT, CT, HALVES ? S + 1 : S> Half;
    __shared__ __attribute__((aligned(16))) char ring[Tile::kRing > Half::kRing ? Tile::kRing
                                                                                : Half::kRing];
    __shared__ float inv[Tile::BM];
    const int nt = (int)((a.N + Tile::BN - 1) / Tile::BN), mt = (a.M + Tile::BM - 1) / Tile::BM;
    // Consecutive tiles to one XCD, as bands of 4 tiles of weight rows, so that what its
    // workgroups read at a time is few tiles of either operand.
    const int G = HALVES ? a.full : gridDim.x, id = blockIdx.x, past = id - G;
    const int tid = past >= 0 ? G + (past >> 1) : (id & 7) * (G >> 3) + (id >> 3);
    if (tid >= nt * mt) return;
    const int band = tid / (4 * mt), wide = min(4, nt - 4 * band), in_band = tid - band * 4 * mt;
    const int bn = 4 * band + in_band % wide, m0 = in_band / wide * Tile::BM;
    const int64_t n0 = (int64_t)bn * Tile::BN;
    if (HALVES && past >= 0) {
        const int64_t h0 = n0 + (past & 1) * Half::BN;
        if (h0 < a.N) Half::template run<TYPE, BEST>(a, h0, 2 * bn + (past & 1), m0, ring, inv);
    } else {
        Tile::template run<TYPE, BEST>(a, n0, bn, m0, ring, inv);
    }
}

// Joins the parts of a row's largest value, W waves to a row.
template <int W>
__global__ void __launch_bounds__(W > 1 ? 64 * W : 256)
gemm_i8_best_kernel(const float2* best, int parts, int M, int32_t* out) {
    __shared__ float rv[W];
    __shared__ int ri[W];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int m = W > 1 ? blockIdx.x : blockIdx.x * 4 + wave;
    if (m >= M) return;
    const float2* row = best + (int64_t)m * parts;
    float v = -INFINITY;
    int n = INT32_MAX;
#pragma unroll 4
    for (int i = W > 1 ? threadIdx.x : lane; i < parts; i += 64 * W) {
        const float2 e = row[i];
        take_best(v, n, e.x, __float_as_int(e.y));
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) take_best(v, n, __shfl_xor(v, d), __shfl_xor(n, d));
    if (W > 1) {
        if (lane == 0) {
            rv[wave] = v;
            ri[wave] = n;
        }
        __syncthreads();
        if (wave > 0) return;
#pragma unroll
        for (int w = 1; w < W; ++w) take_best(v, n, rv[w], ri[w]);
    }
    if (lane == 0) out[m] = n;
}

// The kernel of a call, and the parts that a row's largest value comes in.
enum GemmShape { kOne16x16, kFew16x16, kFew32x16, kFew32x32, kFew64x32, kTile64x32, kTile64x64,
                 kTile128x64, kTile128x128, kTile256x128, kTile256x256 };  // channels x tokens
struct GemmPlan {
    GemmShape shape;
    int parts;
};
// Larger workgroups read less for a product, smaller ones are more and each takes less time: the
// smallest shape whose workgroups have a CU each is nearly always the fastest, and beyond that the
// largest, but for few tokens, whose weights the GPU can do no more than stream. Measured, us (fp16
// outputs, weights not in the caches), by the columns of kShapes below:
//                       1:16x16 16x16 32x16 32x32 64x32 | 64x32 64x64 128x64 128x128 256x128 256x256
//     1 x   2560 x 2560    3.7   3.9   4.3   4.7   6.9 |   6.6   8.2     10      12      23      27
//    24 x   2560 x 2560    5.8   5.5   4.9   6.4   8.7 |   7.4   8.5     11      13      26      28
//     1 x   2560 x 6912    5.7   6.5   7.2   8.0    14 |    15    17     23      41      84      65
//    16 x   2560 x 6912    8.2   7.5   9.4    10    15 |    16    17     24      41      84      66
//    24 x   2560 x 6912     12    12   8.4    12    16 |    16    18     24      40      85      65
//   100 x   2560 x 6912     26    27    21    18  15.8 |  15.5    18     26      42      86      68
//   300 x   2560 x 6912     63    66    46    41    31 |    25  19.1     28      41      86      69
//    16 x   6912 x 2560    7.0   6.9   5.8   6.3   8.4 |   9.2   9.1     12      17      33      28
//    32 x   6912 x 2560     12    11   8.8   8.2    10 |    10   9.4     13      18      34      29
//   100 x   6912 x 2560     30    27    20    20    17 |    15   9.8     13      20      36      31
//   200 x   6912 x 2560     51    45    35    30    25 |    21    14    12.8      19      36      37
//   512 x   6912 x 2560    131   114    77    64    53 |    44    27    22.5    21.0      36      40
//  1024 x   6912 x 2560                                |    84    44     37    29.9    37.0      41
//  2048 x   6912 x 2560                                |          77     61      53    42.3    42.8
//  4001 x   2560 x 6912                                |                        101      91      80
//     1 x 128256 x 2560     66    53    52    55    53 |    74    63     62      64      64      83
//    32 x 128256 x 2560    177   163   123    91    65 |    87    74     69      79      71      89
//   300 x 128256 x 2560                           680 |   486   243    195     182     148     197
// (Over 180 sizes this rule takes 1% longer than the fastest shape of each. From 33 to some 600 tokens
// the fastest takes 2 to 4 times what its bytes do: a workgroup a CU walks the whole of K, one barrier
// for each 64, two products of a wave between them; of the tiles only the smallest shares K.)
// (channels and tokens of a workgroup, channels of a part)
constexpr int kShapes[][3] = {{16, 16, 16},   {16, 16, 16},   {32, 16, 32},    {32, 32, 32},
                              {64, 32, 64},   {64, 32, 32},   {64, 64, 32},    {128, 64, 64},
                              {128, 128, 32}, {256, 128, 64}, {256, 256, 128}};
GemmPlan gemm_plan(int64_t M, int64_t N) {
    const auto count = [&](GemmShape s) {
        return ceil_div(N, kShapes[s][0]) * ceil_div(M, kShapes[s][1]);
    };
    const auto fits = [&](GemmShape s) { return count(s) <= 256; };
    GemmShape s = kTile128x128;
    if (fits(kFew16x16))
        s = M <= 4 ? kOne16x16 : kFew16x16;  // (16 waves to a workgroup, 8)
    else if (fits(kFew32x16) || (M <= 16 && count(kFew64x32) < 900))
        s = kFew32x16;
    else if (fits(kFew32x32) && M > 16)
        s = kFew32x32;
    else if (fits(kTile64x32) && M > 32)
        s = kTile64x32;
    else if (M <= 32 && (fits(kFew64x32) || count(kFew64x32) >= 900))
        s = kFew64x32;
    else if (fits(kTile64x64))
        s = kTile64x64;
    else if (fits(kTile128x64) || (M <= 64 && count(kTile256x128) < 300))
        s = kTile128x64;
    else if (count(kTile128x128) <= 400)
        s = kTile128x128;
    else if (count(kTile256x256) >= 150 && count(kTile256x256) <= 192 &&
             2 * ceil_div(M, 256) == ceil_div(M, 128))
        s = kTile256x256;  // (one to a CU: of 256 x 128 some CUs would have two)
    else if (count(kTile256x128) >= 300)
        s = kTile256x128;
    return {s, (int)(ceil_div(N, kShapes[s][0]) * (kShapes[s][0] / kShapes[s][2]))};
}

template <int MT, int NT, int KW>
void launch_few(const GemmI8& a, hipStream_t st) {
    hipLaunchKernelGGL((gemm_i8_few_kernel<MT, NT, KW>),
                       dim3((unsigned)ceil_div(a.N, 16 * NT), (unsigned)ceil_div(a.M, 16 * MT)),
                       dim3(64 * KW), 0, st, a);
}
template <int TYPE, bool BEST, int WR, int WT, int KW, int RT, int CT, int S, bool HALVES = false>
void launch_tile(GemmI8 a, hipStream_t st) {
    // (a number of workgroups that is shared out among the XCDs evenly: the last have no tile)
    const int64_t tiles = ceil_div(a.N, 32 * RT * WR) * ceil_div(a.M, 32 * CT * WT);
    int64_t wgs = ceil_div(tiles, 8) * 8;
    a.full = (int)wgs;
    if (HALVES && tiles > 256 && tiles % 256 > 0 && tiles % 256 <= 128) {
        a.full = (int)(tiles / 256 * 256);
        wgs = a.full + 2 * (tiles % 256);
    }
    hipLaunchKernelGGL((gemm_i8_tile_kernel<TYPE, BEST, WR, WT, KW, RT, CT, S, HALVES>),
                       dim3((unsigned)wgs), dim3(64 * WR * WT * KW), 0, st, a);
}
template <int TYPE, bool BEST>
void launch_shape(GemmShape shape, const GemmI8& a, hipStream_t st) {
    switch (shape) {
        case kOne16x16: return launch_few<1, 1, 16>(a, st);
        case kFew16x16: return launch_few<1, 1, 8>(a, st);
        case kFew32x16: return launch_few<1, 2, 8>(a, st);
        case kFew32x32: return launch_few<2, 2, 8>(a, st);
        case kFew64x32: return launch_few<2, 4, 4>(a, st);
        case kTile64x32: return launch_tile<TYPE, BEST, 2, 1, 4, 1, 1, 4>(a, st);
        case kTile64x64: return launch_tile<TYPE, BEST, 2, 2, 1, 1, 1, 9>(a, st);
        case kTile128x64: return launch_tile<TYPE, BEST, 2, 2, 1, 2, 1, 6>(a, st);
        case kTile128x128: return launch_tile<TYPE, BEST, 4, 2, 1, 1, 2, 4>(a, st);
        case kTile256x128: return launch_tile<TYPE, BEST, 4, 2, 1, 2, 2, 3, !BEST>(a, st);
        case kTile256x256: return launch_tile<TYPE, BEST, 2, 4, 1, 4, 2, 4>(a, st);
    }
}

}  // namespace
}  // namespace tz

using namespace tz;

extern "C" {

TENZO_HIP_API size_t tenzo_hip_gemm_i8_ws_bytes(int64_t M, int64_t N, int64_t K, int want_idx) {
    if (M <= 0 || N <= 0 || K <= 0 || !want_idx) return 0;
    return (size_t)(M * gemm_plan(M, N).parts) * sizeof(float2);
}

TENZO_HIP_API int tenzo_hip_gemm_i8(const int8_t* codes, int64_t codes_stride,
                                    const tenzo_hip_actq_t* q, const void* w_packed,
                                    const float* scales, int64_t M, int64_t N, int64_t K, void* y,
                                    int dtype, int64_t y_stride, int32_t* out_idx, void* ws,
                                    size_t ws_bytes, void* stream) {
    TZ_CHECK(dtype >= 0 && dtype <= 2, "gemm_i8: dtype %d", dtype);
    TZ_CHECK(M >= 0 && M <= (1 << 20) && N > 0 && N <= (1 << 29), "gemm_i8: M=%lld N=%lld",
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
    const GemmPlan p = gemm_plan(M, N);
    const hipStream_t st = (hipStream_t)stream;
    GemmI8 a{codes, M == 1 ? K : codes_stride, q, (const uint8_t*)w_packed, scales, y, y_stride,
             out_idx ? (float2*)ws : nullptr, N, (int)M, (int)(K / 16), p.parts, dtype, 0};
    if (dtype == 0)
        out_idx ? launch_shape<0, true>(p.shape, a, st) : launch_shape<0, false>(p.shape, a, st);
    else if (dtype == 1)
        out_idx ? launch_shape<1, true>(p.shape, a, st) : launch_shape<1, false>(p.shape, a, st);
    else
        out_idx ? launch_shape<2, true>(p.shape, a, st) : launch_shape<2, false>(p.shape, a, st);
    const int rc = launch_status("gemm_i8 kernel");
    if (rc || !out_idx) return rc;
    if (a.parts > 256)
        hipLaunchKernelGGL(gemm_i8_best_kernel<8>, dim3((unsigned)M), dim3(512), 0, st, a.best,
                           a.parts, a.M, out_idx);
    else
        hipLaunchKernelGGL(gemm_i8_best_kernel<1>, dim3((unsigned)ceil_div(M, 4)), dim3(256), 0,
                           st, a.best, a.parts, a.M, out_idx);
    return launch_status("gemm_i8_best_kernel");
}

}  // extern "C"
