// Attention over the paged cache held in 4 bits (layout: kv4.h): every row of queries at its own
// position of its own sequence, o = sum_t softmax_t(q.k_t / sqrt(128)) v_t over the positions up
// to its own; a row that sees no position is zero.
#include "kv4.h"

namespace tz {
namespace {

constexpr float kQkScale = 0.08838834764831845f;  // 1/sqrt(128)
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kSub = 4;             // 16-token pages of a wave's step
constexpr int kTile = 16 * kSub;    // tokens of a wave's step
constexpr int kMaxPages = 1024;     // pages of a workgroup's part of the context
constexpr int kQStride = 132;       // floats of a query in LDS
constexpr int kParts = 3;           // parts of 8 bits of an fp32 value: every bit

// The prompts' kernel holds keys and values in fp16. Scale bytes whose values are exact there as
// they are: 0.5 * 2^(s - 127) to 6 * 2^(s - 127), down to its smallest subnormal, which the matrix
// cores take.
constexpr int kLowScale = 104, kTopScale = 140;
constexpr float kWeightBits = 15.0f;  // weights, at most 1, are held times 2^15

struct Kv4Attn {
    const void* q;
    void* out;
    int64_t q_stride, out_stride;
    const uint8_t* pk;
    const uint8_t* pv;
    const uint8_t* pks;
    const uint8_t* pvs;
    const float* rope;
    float* part_o;    // records of rows' unfinished sums: 128 sums,
    float2* part_ml;  // maximum (base 2) and sum of weights
    int G, Hq, T;
    uint32_t g_mul;  // 2^32 / G, rounded up (0: G is 1)
    int chunk, splits;  // tokens of a split
    int wgs;            // workgroups of a call whose steps are dealt evenly
    int most;           // and the steps that it can have, where no two sequences share rows
    int vec_out;        // out allows accesses of 4 elements

    // r / G, exact for r < 2^28 and G up to 16 (a division is some 40 instructions).
    __device__ __forceinline__ int token(int r) const {
        return g_mul ? (int)__umulhi((uint32_t)r, g_mul) : r;
    }
};

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

union Frag {
    uint32_t w[4];
    bf16x8 v;
};
union Frag16 {
    uint32_t w[4];
    uint4 q;
    f16x8 v;
};

template <int CTRL>
__device__ __forceinline__ float ror16(float v) {  // rotation within 16 lanes
    return dpp_f<CTRL>(v);
}
constexpr int kDppRor4 = 0x124, kDppRor8 = 0x128;

__device__ __forceinline__ float max_quarters(float x) {
    float a, b;
    lane_halves(x, a, b);
    lane_pairs16(fmaxf(a, b), a, b);
    return fmaxf(a, b);
}
__device__ __forceinline__ float sum_quarters(float x) {
    float a, b;
    lane_halves(x, a, b);
    lane_pairs16(a + b, a, b);
    return a + b;
}

// The upper halves of two floats (bf16 towards zero), a in the low half.
__device__ __forceinline__ uint32_t pack_hi(float a, float b) {
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}
__device__ __forceinline__ float masked(float v, uint32_t m) {
    return __uint_as_float(__float_as_uint(v) & m);
}

// Two floats as fp16, the first in the low half, and what that leaves of them.
__device__ __forceinline__ uint32_t pack16(float a, float b) {
    const f32x2 v = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
}
__device__ __forceinline__ float rest_lo(float x, uint32_t h) {
    float r;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(x));
    return r;
}
__device__ __forceinline__ float rest_hi(float x, uint32_t h) {
    float r;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]"
        : "=v"(r)
        : "v"(h), "v"(x));
    return r;
}

// Eight codes as fp16, times their scale (which the conversion takes the exponent of).
__device__ __forceinline__ uint4 fp4_to_half8(uint32_t w, float scale) {
    union {
        f16x2 h[4];
        uint4 q;
    } f;
    f.h[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 0);
    f.h[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 1);
    f.h[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 2);
    f.h[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 3);
    return f.q;
}
// The scale 2^(s - 127) of a byte of kLowScale .. kTopScale, or of less (about 0).
__device__ __forceinline__ float byte_scale(int s) {
    return __uint_as_float((uint32_t)max(s, 1) << 23);
}
__device__ __forceinline__ float pow2(int e) {  // 2^e, 0 or the largest power where that is beyond
    return e < -126 ? 0.0f : __uint_as_float((uint32_t)(min(e, 127) + 127) << 23);
}
__device__ __forceinline__ bool in_range(int s) {
    return (uint32_t)(s - kLowScale) <= (uint32_t)(kTopScale - kLowScale);
}
__device__ __forceinline__ bool no_codes(uint4 c) {
    return ((c.x | c.y | c.z | c.w) & 0x77777777u) == 0;
}

// A query row's power of two: the one that brings its largest element to 2^13 .. 2^14, so that the
// second parts of its elements stay normal in fp16 too (2^-38 of the largest is still seen).
__device__ __forceinline__ int row_shift(float amax) {
    const int e = (int)(__float_as_uint(amax) >> 23);
    return 140 - min(max(e, 14), 254);
}

// Where pieces of 8 fp16 of a row of 128 stand in LDS: rows of 256 bytes, the pieces in an order
// of the row's own, so that eight lanes' writes or reads (8 rows, one piece) and 16 lanes'
// transposing reads (4 rows, two pieces) meet all banks once. Only the low three bits of the
// piece and of the row take part: 16 rows on, or 8 pieces on, is a constant away.
__device__ __forceinline__ int piece_at(int row, int p) {
    return row * kKv4Dim + ((p ^ (2 * (row & 3) + (row >> 2 & 1))) << 3);
}

// Four outputs, the weighted sum over the sum of weights (0 where no token was seen).
template <bool HALF>
__device__ __forceinline__ void store4(const Kv4Attn& a, int64_t at, f32x4 v, float l) {
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;  // (2^-24 of the output; a division each: 1 us)
    float o[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = v[k] * inv;
    if (!a.vec_out) {
#pragma unroll
        for (int k = 0; k < 4; ++k) st_act<HALF>(a.out, at + k, o[k]);
    } else if (HALF) {
        uint2 w;
        w.x = float_to_half_bits(o[0]) | (uint32_t)float_to_half_bits(o[1]) << 16;
        w.y = float_to_half_bits(o[2]) | (uint32_t)float_to_half_bits(o[3]) << 16;
        *reinterpret_cast<uint2*>((uint16_t*)a.out + at) = w;
    } else {
        *reinterpret_cast<float4*>((float*)a.out + at) = make_float4(o[0], o[1], o[2], o[3]);
    }
}

// Sequence and row tile of a work unit: the unit-th tile when every sequence has
// ceil(rows * G / RT) of them. False past the last.
__device__ __forceinline__ bool find_unit(const Kv4Seqs& sq, int unit, int G, int RT, int& seq,
                                          int& tile) {
    if (!sq.cu) {
        const int per = (G + RT - 1) / RT;
        seq = unit / per;
        tile = unit - seq * per;
        return seq < sq.B;
    }
    const int lane = threadIdx.x & 63;
    for (int base = 0; base < sq.B; base += 64) {
        const int b = base + lane;
        int n = 0, first;
        if (b < sq.B) n = sq.rows(b, first);
        const int nt = (int)(((int64_t)n * G + RT - 1) / RT);
        int incl = nt;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(incl, d);
            if (lane >= d) incl += o;
        }
        const uint64_t past = __ballot(incl > unit);
        if (past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            seq = base + l;
            tile = unit - __builtin_amdgcn_readlane(incl - nt, l);
            return true;
        }
        unit -= __builtin_amdgcn_readlane(incl, 63);
    }
    return false;
}

// Work of a sequence where steps are dealt evenly: each of its (kv head, row tile) units takes
// ceil(length / 256) steps, whatever of them a row sees, and counts one more for what a unit costs
// besides (its queries, the first tokens' way, the sums' meeting: about 4 us, a step 3 to 5).
constexpr int kStep = 4 * kTile;
struct SeqWork {
    int first, n, c, steps, tiles;
    __device__ __forceinline__ SeqWork(const Kv4Seqs& sq, int b, int G, int RT) {
        n = sq.rows(b, first);
        c = sq.length(b);
        steps = (c + kStep - 1) / kStep;
        tiles = (n * G + RT - 1) / RT;
    }
    __device__ __forceinline__ int slots() const { return steps + 1; }  // of a unit
    __device__ __forceinline__ int total(int Hkv) const {
        return c > 0 ? slots() * tiles * Hkv : 0;
    }
};

// Sums that stay at the largest number once they reach it: where ranges of cu_q lie over each other
// the sequences' work adds up to anything.
__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) {
    return __builtin_elementwise_add_sat(a, b);
}

// The work of this thread's sequences, b0 up to b1, that of the threads before (the return value)
// and of all of them; no work at all where it is more than `most`.
template <int ROWS>
__device__ __forceinline__ int scan_work(const Kv4Attn& a, const Kv4Seqs& sq, int b0, int b1,
                                         uint32_t* wsum, int& mine, int& all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t v = 0;
    for (int b = b0; b < b1; ++b) v = add_sat(v, SeqWork(sq, b, a.G, ROWS).total(sq.Hkv));
    uint32_t incl = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t o = __shfl_up(incl, d);
        if (lane >= d) incl = add_sat(incl, o);
    }
    if (lane == 63) wsum[wave] = incl;
    __syncthreads();
    uint32_t before = incl - v, sum = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        before += w < wave ? wsum[w] : 0;
        sum = add_sat(sum, wsum[w]);
    }
    mine = (int)v;
    all = sum <= (uint32_t)a.most ? (int)sum : 0;
    return (int)before;
}

// A value that all lanes of the wave hold, for scalar registers.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Workgroup w of N has the slots [w q + min(w, r), + q + (w < r)), q and r of total / N.
__device__ __forceinline__ int wg_start(int w, int total, int N) {
    const int q = total / N, r = total - q * N;
    return w * q + min(w, r);
}
__device__ __forceinline__ int wg_of(int g, int total, int N) {
    const int q = total / N, r = total - q * N;
    return g < r * (q + 1) ? g / (q + 1) : r + (g - r * (q + 1)) / q;
}

// A piece of work: the rows of a tile against the tokens [t0, t0 + len) of their sequence.
struct Segment {
    int seq, first, n, c, tile, h;
    int t0, len;
    bool whole;   // no other piece has these rows (steps dealt evenly)
    int64_t rec;  // else the record of the first row
    int split;    // (a grid of splits)
};

// One workgroup: RT = ROWS * RW rows (token, query head of one kv head) of a sequence against a
// part of its tokens. Wave w has the rows group w % RW and every (4 / RW)-th step of 64 tokens.
//
// Scores come transposed, S^T = K Q^T, so that a lane keeps one row: K is the A operand (16
// tokens x 32 dims: the lane's 16 code bytes are a token's group of 32 dims, one scale, four
// steps of 8 dims), Q the B operand. In S^T's layout a lane holds 4 tokens of its row per 16,
// which is what the B operand of O^T = V^T P^T wants when the value rows are taken in the same
// order: no weight changes lanes. V^T comes from value rows in LDS (bf16, private to the wave)
// by transposing reads. Codes times scale are exact in bf16; queries and weights are split into
// three parts of 8 bits, every bit that fp32 holds, whatever the type of the call (with two in fp16
// calls, a part in 2^15 at worst, scores of 50 were wrong by 2^-10 of an output; the two save 1%
// of a batch of tokens with 4 query heads a kv head, 12% with 8 and 4% of drafts). With 4 rows the
// parts stand in columns side by side (column = part * ROWS + row) and one MFMA serves all of them.
//
// A step loads 136 bytes a token straight to registers, the next step's during the products.
// 130000 tokens of one sequence, 20 / 5 heads: 23 us, 3.8 TB/s (and 3 for the join), bound by
// the vector work on codes and weights beside the loads; up to 256 tokens 6 us, a chain of loads
// (length, page number, codes), the products' latency and the waves' meeting.
template <int ROWS, int RW>
struct Kv4Smem {
    static constexpr int RT = ROWS * RW;
    // the queries first, then 32 value rows (bf16) a wave, at last the rows' sums
    static constexpr int kMain =
        4 * 32 * kKv4Dim > 2 * RT * kQStride ? 4 * 32 * kKv4Dim : 2 * RT * kQStride;
    __align__(16) uint16_t main[kMain];
    float2 ml[4][16];
    int pg[kMaxPages];
};

template <int ROWS, int RW, bool HALF, bool EVEN>
__device__ __forceinline__ void kv4_segment(const Kv4Attn& a, const Kv4Seqs& sq, const Segment& g,
                                            Kv4Smem<ROWS, RW>& sm) {
    constexpr int SLOTS = 16 / ROWS, NM = SLOTS == 1 ? kParts : 1, TW = 4 / RW, RT = ROWS * RW;
    static_assert(SLOTS == 1 || SLOTS > kParts, "a column for each part");
    static_assert(TW > 1, "a row's sums meet from several waves");
    static_assert(32 * kKv4Dim * 2 >= 16 * kKv4Dim * 4, "the rows' sums fit a wave's values");
    uint16_t* smem = sm.main;
    int* pg = sm.pg;
    int tid = threadIdx.x;
    // (opaque, so that what follows from it is not kept in registers from piece to piece)
    if (EVEN) asm volatile("" : "+v"(tid));
    const int lane = tid & 63, col = lane & 15, j = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rw = wave % RW, tw = wave / RW;
    const int n = g.n, first = g.first, c = g.c, h = g.h, t0 = g.t0;
    const int row0 = g.tile * RT;  // of the sequence's n * G
    const int last_i = min(n - 1, a.token(row0 + RT - 1));
    const int t1 = min(min(t0 + g.len, c - n + last_i + 1), c);  // tokens that some row sees

    // the lane's row
    const int slot = col / ROWS, qi = a.token(row0 + rw * ROWS + col % ROWS);
    const int pos = qi < n && c > 0 ? c - n + qi : -1;

    // the page numbers of the first kMaxPages pages and the rows' queries, rotated and scaled, by
    // way of LDS (each wave needs all of a row)
    const int32_t* table = sq.tables + (int64_t)g.seq * sq.table_stride + t0 / kKv4Page;
    const int pages = t1 > t0 ? (t1 - t0 + kKv4Page - 1) / kKv4Page : 0;
    auto stage_pages = [&](int from) {
        for (int p = from + tid; p < min(pages, from + kMaxPages); p += 256) {
            const int id = table[p];
            pg[p - from] = id >= 0 && id < sq.n_blocks ? id : -1;
        }
    };
    float* qs = reinterpret_cast<float*>(smem);
    // (no load under a condition, where it would be waited for: rows and positions that are not
    // there read others, whose results nobody writes)
    constexpr int QT = RT / 4;
    float x0[QT], x1[QT], cv[QT], sv[QT];
    const int last_row = n * a.G - 1;
#pragma unroll
    for (int k = 0; k < QT; ++k) {
        const int r2 = min(row0 + wave + 4 * k, last_row), i2 = a.token(r2);
        const int64_t at = (int64_t)(first + i2) * a.q_stride +
                           (int64_t)(h * a.G + (r2 - i2 * a.G)) * kKv4Dim + lane;
        x0[k] = ld_act<HALF>(a.q, at);
        x1[k] = ld_act<HALF>(a.q, at + 64);
        cv[k] = 1.0f;
        sv[k] = 0.0f;
    }
    if (a.rope && c > 0)
#pragma unroll
        for (int k = 0; k < QT; ++k) {
            const int p2 = c - n + a.token(min(row0 + wave + 4 * k, last_row));
            const float* cs = a.rope + (int64_t)min(max(p2, 0), c - 1) * kKv4Dim + lane;
            cv[k] = cs[0];
            sv[k] = cs[64];
        }
    stage_pages(0);
#pragma unroll
    for (int k = 0; k < QT; ++k) {
        const int rr = wave + 4 * k;
        const float y0 = x0[k];
        x0[k] = __builtin_fmaf(y0, cv[k], -__fmul_rn(x1[k], sv[k]));
        x1[k] = __builtin_fmaf(y0, sv[k], __fmul_rn(x1[k], cv[k]));
        qs[rr * kQStride + lane] = __fmul_rn(x0[k], kQkScale * kLog2e);
        qs[rr * kQStride + lane + 64] = __fmul_rn(x1[k], kQkScale * kLog2e);
    }
    __syncthreads();

    uint4 kr[kSub], vr[kSub];
    uint32_t ksc[kSub], vsc[kSub];
    const uint32_t lane_code = (uint32_t)(col * kKv4Row + j * 16);
    const uint32_t lane_scale = (uint32_t)(col * kKv4Scales + j);
    // (a page that the pool does not hold: another one is read in its place and masked)
    auto page_row = [&](int id) -> int64_t {
        return (((int64_t)max(id, 0) * sq.n_layers + sq.layer) * sq.Hkv + h) * kKv4Page;
    };
    auto load_k = [&](int tt, int id) {
        const int64_t row = page_row(id);
        kr[tt] = *reinterpret_cast<const uint4*>(a.pk + row * kKv4Row + lane_code);
        ksc[tt] = (a.pks + row * kKv4Scales)[lane_scale];
    };
    auto load_v = [&](int tt, int id) {
        const int64_t row = page_row(id);
        vr[tt] = *reinterpret_cast<const uint4*>(a.pv + row * kKv4Row + lane_code);
        vsc[tt] = (a.pvs + row * kKv4Scales)[lane_scale];
    };
    int id_next[kSub];
    // page numbers of the step at t out of the kMaxPages from token w0 on
    auto next_ids = [&](int t, int w0) {
#pragma unroll
        for (int tt = 0; tt < kSub; ++tt) {
            const int p = min(((t - w0) >> 4) + tt, pages - 1 - ((w0 - t0) >> 4));
            id_next[tt] = __builtin_amdgcn_readfirstlane(pg[p]);
        }
    };

    f32x4 acc[8];
#pragma unroll
    for (int d = 0; d < 8; ++d) acc[d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;

    uint16_t* vb = smem + wave * (32 * kKv4Dim);
    int wr[4], rd[4];  // the lane's pieces of its token's row, and of the transposing reads
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        wr[k] = piece_at(col, 4 * j + k);
        rd[k] = piece_at(4 * j + (col >> 2), 2 * k + (col >> 1 & 1)) + (col & 1) * 4;
    }

    int t = t0 + kTile * tw;
    const bool any = sq.n_blocks > 0;
    if (t < t1 && any) {
        next_ids(t, t0);
#pragma unroll
        for (int tt = 0; tt < kSub; ++tt) load_k(tt, id_next[tt]);
#pragma unroll
        for (int tt = 0; tt < kSub; ++tt) load_v(tt, id_next[tt]);
    }
    // Q as B operands: the lane's 32 dims 32j .. 32j + 31 of its row, in parts (part p of a value:
    // what its parts before leave, cut to 8 bits)
    Frag qf[NM][4];
    {
        const uint32_t m1 = slot >= 1 ? 0xffff0000u : 0, m2 = slot >= 2 ? 0xffff0000u : 0;
        const float* src = qs + (rw * ROWS + col % ROWS) * kQStride + 32 * j;
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
            f32x4 x = *reinterpret_cast<const f32x4*>(src + e);
            if (SLOTS > 1)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    x[k] -= masked(x[k], m1);
                    x[k] -= masked(x[k], m2);
                    if (slot >= kParts) x[k] = 0.0f;
                }
#pragma unroll
            for (int p = 0; p < NM; ++p) {
                qf[p][e >> 3].w[(e >> 1) & 3] = pack_hi(x[0], x[1]);
                qf[p][e >> 3].w[((e >> 1) & 3) + 1] = pack_hi(x[2], x[3]);
#pragma unroll
                for (int k = 0; k < 4; ++k) x[k] -= masked(x[k], 0xffff0000u);
            }
        }
    }
    __syncthreads();
    // (kMaxPages pages at a time: page numbers in LDS)
    for (int w0 = t0;;) {
        const int w1 = min(t1, w0 + kMaxPages * kKv4Page);
        for (; t < w1 && any; t += kTile * TW) {
            const int next = t + kTile * TW;
            f32x4 s[kSub];
            // (the steps outermost: an MFMA waits some 60 cycles for the sum that it adds to, so
            // neighbours have different ones)
            float sc[kSub];
#pragma unroll
            for (int tt = 0; tt < kSub; ++tt) {
                sc[tt] = e8m0_to_float(ksc[tt]);
                s[tt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            }
#pragma unroll
            for (int st = 0; st < 4; ++st) {
                union {
                    bf16x2 p[4];
                    bf16x8 v;
                } kf[kSub];
#pragma unroll
                for (int tt = 0; tt < kSub; ++tt) {
                    const uint32_t w = st == 0 ? kr[tt].x : st == 1 ? kr[tt].y : st == 2 ? kr[tt].z
                                                                                       : kr[tt].w;
                    kf[tt].p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc[tt], 0);
                    kf[tt].p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc[tt], 1);
                    kf[tt].p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc[tt], 2);
                    kf[tt].p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc[tt], 3);
                }
#pragma unroll
                for (int p = 0; p < NM; ++p)
#pragma unroll
                    for (int tt = 0; tt < kSub; ++tt)
                        s[tt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                            kf[tt].v, qf[p][st].v, s[tt], 0, 0, 0);
            }
            bool bad = false;
            int id_now[kSub];
#pragma unroll
            for (int tt = 0; tt < kSub; ++tt) {
                id_now[tt] = ((t - t0) >> 4) + tt < pages ? id_next[tt] : -1;
                bad = bad || id_now[tt] < 0;
            }
            if (next < w1) {
                next_ids(next, w0);
#pragma unroll
                for (int tt = 0; tt < kSub; ++tt) load_k(tt, id_next[tt]);
            }
            float top = -INFINITY;
#pragma unroll
            for (int tt = 0; tt < kSub; ++tt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float v = s[tt][i];
                    if (SLOTS > 1) v += ror16<kDppRor8>(v);
                    if (SLOTS > 1) v += ror16<kDppRor4>(v);
                    s[tt][i] = v;
                }
            // a step that a row may not see whole: past its position, or absent pages
            if (bad || t + kTile - 1 > c - n + a.token(row0)) {
#pragma unroll
                for (int tt = 0; tt < kSub; ++tt)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (id_now[tt] < 0 || t + 16 * tt + 4 * j + i > pos) s[tt][i] = -INFINITY;
            }
#pragma unroll
            for (int tt = 0; tt < kSub; ++tt)
                top = fmaxf(top, fmaxf(fmaxf(s[tt][0], s[tt][1]), fmaxf(s[tt][2], s[tt][3])));
            const float mn = fmaxf(m, max_quarters(top));
            const float base = mn == -INFINITY ? 0.0f : mn;
            const float alpha = __builtin_amdgcn_exp2f(m - base);
            m = mn;
            if (__ballot(alpha != 1.0f)) {
#pragma unroll
                for (int d = 0; d < 8; ++d) acc[d] *= alpha;
                l *= alpha;
            }
#pragma unroll
            for (int tt = 0; tt < kSub; ++tt) {
#pragma unroll
                for (int i = 0; i < 4; ++i) s[tt][i] = __builtin_amdgcn_exp2f(s[tt][i] - base);
                l += (s[tt][0] + s[tt][1]) + (s[tt][2] + s[tt][3]);
            }
            const uint32_t m1 = slot >= 1 ? 0xffff0000u : 0, m2 = slot >= 2 ? 0xffff0000u : 0;
#pragma unroll
            for (int u = 0; u < kSub / 2; ++u) {
                // 32 value rows, by two 16-token pages
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int tt = 2 * u + k;
                    const float sc = e8m0_to_float(vsc[tt]);
                    const uint32_t w[4] = {vr[tt].x, vr[tt].y, vr[tt].z, vr[tt].w};
#pragma unroll
                    for (int st = 0; st < 4; ++st) {
                        union {
                            bf16x2 p[4];
                            uint4 v;
                        } f;
                        f.p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[st], sc, 0);
                        f.p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[st], sc, 1);
                        f.p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[st], sc, 2);
                        f.p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[st], sc, 3);
                        *reinterpret_cast<uint4*>(vb + wr[st] + k * 16 * kKv4Dim) = f.v;
                    }
                }
                if (u == kSub / 2 - 1 && next < w1)
#pragma unroll
                    for (int tt = 0; tt < kSub; ++tt) load_v(tt, id_next[tt]);
                Frag pf[NM];
                float p8[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    p8[e] = s[2 * u + (e >> 2)][e & 3];
                    if (SLOTS > 1) {
                        p8[e] -= masked(p8[e], m1);
                        p8[e] -= masked(p8[e], m2);
                    }
                }
#pragma unroll
                for (int p = 0; p < NM; ++p)
#pragma unroll
                    for (int e = 0; e < 8; e += 2) {
                        pf[p].w[e >> 1] = pack_hi(p8[e], p8[e + 1]);
                        p8[e] -= masked(p8[e], 0xffff0000u);
                        p8[e + 1] -= masked(p8[e + 1], 0xffff0000u);
                    }
#pragma unroll
                for (int d0 = 0; d0 < 8; d0 += 4) {
                    typedef __attribute__((address_space(3))) s16x4* lds4;
                    union {
                        s16x4 h[2];
                        bf16x8 v;
                    } vf[4];
#pragma unroll
                    for (int d = 0; d < 4; ++d) {
                        // (lane 4r + i of 16: half a piece of row r, in return for column 4r + i)
                        uint16_t* src = vb + rd[d] + (d0 >> 2) * 64;
                        vf[d].h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)src);
                        vf[d].h[1] =
                            __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(src + 16 * kKv4Dim));
                    }
#pragma unroll
                    for (int p = 0; p < NM; ++p)
#pragma unroll
                        for (int d = 0; d < 4; ++d)
                            acc[d0 + d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                                vf[d].v, pf[p].v, acc[d0 + d], 0, 0, 0);
                }
            }
        }
        w0 += kMaxPages * kKv4Page;
        if (w0 >= t1 || !any) break;
        __syncthreads();
        stage_pages((w0 - t0) / kKv4Page);
        __syncthreads();
        if (t < t1) {
            next_ids(t, w0);
#pragma unroll
            for (int tt = 0; tt < kSub; ++tt) load_k(tt, id_next[tt]);
#pragma unroll
            for (int tt = 0; tt < kSub; ++tt) load_v(tt, id_next[tt]);
        }
    }

    l = sum_quarters(l);
    if (SLOTS > 1) {
#pragma unroll
        for (int d = 0; d < 8; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float v = slot < kParts ? acc[d][i] : 0.0f;
                v += ror16<kDppRor8>(v);
                v += ror16<kDppRor4>(v);
                acc[d][i] = v;
            }
    }
    // the waves' sums meet: every wave's rows in its own part of the value buffer
    float* o = reinterpret_cast<float*>(vb);
    if (slot == 0) {
#pragma unroll
        for (int d = 0; d < 8; ++d)
            *reinterpret_cast<f32x4*>(o + col * kKv4Dim + 16 * d + 4 * j) = acc[d];
        if (j == 0) sm.ml[wave][col] = make_float2(m, l);
    }
    __syncthreads();
    for (int it = tid; it < RT * 32; it += 256) {
        const int rr = it >> 5, d4 = it & 31, grp = rr / ROWS, cc = rr % ROWS;
        const int r2 = row0 + rr, i2 = a.token(r2);
        if (i2 >= n) continue;
        float M = -INFINITY, L = 0.0f;
        f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < TW; ++w) M = fmaxf(M, sm.ml[w * RW + grp][cc].x);
        const float base = M == -INFINITY ? 0.0f : M;
#pragma unroll
        for (int w = 0; w < TW; ++w) {
            const float2 e = sm.ml[w * RW + grp][cc];
            const float f = __builtin_amdgcn_exp2f(e.x - base);
            L += e.y * f;
            const float* from =
                reinterpret_cast<const float*>(smem + (w * RW + grp) * (32 * kKv4Dim));
            v += f * *reinterpret_cast<const f32x4*>(from + cc * kKv4Dim + 4 * d4);
        }
        const int64_t g2 = (int64_t)first + i2, hd = h * a.G + (r2 - i2 * a.G);
        // to `out` where no other piece has any of the row's tokens, else a record
        if (EVEN ? g.whole : c - n + i2 < a.chunk || a.splits == 1) {
            if (EVEN || g.split == 0)
                store4<HALF>(a, g2 * a.out_stride + hd * kKv4Dim + 4 * d4, v, L);
        } else {
            const int64_t at = EVEN ? g.rec + rr : (g2 * a.Hq + hd) * a.splits + g.split;
            *reinterpret_cast<f32x4*>(a.part_o + at * kKv4Dim + 4 * d4) = v;
            if (d4 == 0) a.part_ml[at] = make_float2(M, L);
        }
    }
    if (EVEN) __syncthreads();
}

// A grid of (unit, split, kv head): every workgroup one piece.
template <int ROWS, int RW, bool HALF>
__global__ void __launch_bounds__(256, ROWS == 16 ? 2 : 3)
kv4_attn_kernel(Kv4Attn a, Kv4Seqs sq) {
    __shared__ Kv4Smem<ROWS, RW> sm;
    const int per_unit = sq.Hkv * a.splits;
    // (from the last unit on: the latest rows of a prompt see the most tokens)
    const int back = blockIdx.x / per_unit, rest = blockIdx.x - back * per_unit;
    const int unit = a.wgs / per_unit - 1 - back;
    Segment g;
    g.split = rest / sq.Hkv;
    g.h = rest - g.split * sq.Hkv;
    if (!find_unit(sq, unit, a.G, ROWS * RW, g.seq, g.tile)) return;
    g.n = sq.rows(g.seq, g.first);
    g.c = sq.length(g.seq);
    g.t0 = g.split * a.chunk;
    g.len = a.chunk;
    const int last_i = min(g.n - 1, a.token(g.tile * ROWS * RW + ROWS * RW - 1));
    if (g.split > 0 && g.t0 >= min(g.c - g.n + last_i + 1, g.c)) return;
    kv4_segment<ROWS, RW, HALF, false>(a, sq, g, sm);
}

constexpr int kRowsRT = 128;

// Sequence and row tile of a work unit of the prompts' kernel, those that see the most tokens first
// whatever their sequence: tile k of a sequence starts at position length - rows + 128 k / G, and
// the unit-th largest start, in 64 tokens, is found by bisection (a lane a sequence; one sequence,
// or over 64 in their order, from the last unit on). 3 prompts of 633 to 2000 tokens, 20 / 5 heads:
// 103 us, in the order of the rows 119.
__device__ __forceinline__ bool find_unit_latest(const Kv4Seqs& sq, int unit, int units, int G,
                                                 int& seq, int& tile) {
    if (!sq.cu || sq.B == 1 || sq.B > 64)
        return find_unit(sq, units - 1 - unit, G, kRowsRT, seq, tile);
    const int lane = threadIdx.x & 63;
    int n = 0, c = 0, first;
    if (lane < sq.B) {
        n = sq.rows(lane, first);
        c = sq.length(lane);
    }
    const int tiles = (int)(((int64_t)n * G + kRowsRT - 1) / kRowsRT), prior = max(c - n, 0);
    // tiles of the lane's sequence that start past 64 x
    auto past = [&](int x) {
        const int64_t ahead = ((int64_t)x * 64 - prior) * G / kRowsRT;
        return (int64_t)x * 64 < prior ? tiles : (int)max((int64_t)tiles - 1 - ahead, (int64_t)0);
    };
    if (unit >= wave_sum_i32(tiles)) return false;
    int lo = 0, hi = max(c, n) / 64 + 1;  // (no tile starts past the largest)
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) hi = max(hi, __shfl_xor(hi, d));
    while (lo < hi) {  // the smallest start that at most `unit` tiles lie past
        const int x = lo + (hi - lo) / 2;
        if (wave_sum_i32(past(x)) <= unit)
            hi = x;
        else
            lo = x + 1;
    }
    const int later = past(lo), here = past(lo - 1) - later;
    int rank = unit - wave_sum_i32(later), incl = here;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(incl, d);
        if (lane >= d) incl += o;
    }
    const uint64_t mine = __ballot(incl > rank);
    if (!mine) return false;
    const int l = __ffsll((unsigned long long)mine) - 1;
    seq = l;
    rank -= __builtin_amdgcn_readlane(incl - here, l);
    tile = __builtin_amdgcn_readlane(tiles - 1 - later, l) - rank;
    return true;
}

// Prompts: 128 rows to a workgroup, 32 (two column tiles) to a wave, all against the same 64 tokens
// at a time. The waves convert a quarter of the tile's keys and values each, into LDS as fp16,
// and every fragment of 1 KB read from there serves both column tiles and both parts, 4 MFMAs. The
// codes of the next tile are loaded during the products and go into the other half of LDS after
// them: one barrier a tile.
//
// fp16 parts take two thirds of the MFMAs that bf16's would, and half of the vector work of
// splitting the weights. Codes times scale are exact in fp16 (a token whose scales are out of its
// range is moved by a power of two of its own: scores are multiplied back, values share one for
// all tokens; what lies 2^37 below the largest is then lost). Queries, scaled by a power of two,
// and weights are split into two parts, 22 bits: 2^-22 of a value is lost, little beside what fp32
// sums lose (and of a weight 2^-40 of the largest, fp16's smallest step).
//
// Prompts of 2000, 1456 and 633 tokens, 20 / 5 heads: 103 us, 324 TFLOP/s of the formula's (twice
// that with the parts). The matrix units are busy for a third of it and the vector units nearly as
// long, and two waves a SIMD, all that the registers allow, overlap them only in part; 16 us go
// into a workgroup's queries and outputs.
template <bool HALF>
__global__ void __launch_bounds__(256, 2) kv4_attn_rows_kernel(Kv4Attn a, Kv4Seqs sq) {
    // two tiles' keys and values (the first is the queries' on their way to registers before)
    __shared__ __align__(16) uint16_t tiles[2][2][kTile * kKv4Dim];
    __shared__ __align__(16) int moved[2][kTile];  // the power of two that tokens' keys are moved by
    __shared__ int flags[2][4], tops[4];
    __shared__ int pg[kMaxPages];
    const int per_unit = sq.Hkv * a.splits;
    const int nth = blockIdx.x / per_unit, rest = blockIdx.x - nth * per_unit;
    const int split = rest / sq.Hkv, h = rest - split * sq.Hkv;
    int seq, tile;
    if (!find_unit_latest(sq, nth, a.wgs / per_unit, a.G, seq, tile)) return;
    int first;
    const int n = sq.rows(seq, first);
    const int c = sq.length(seq);
    const int t0 = split * a.chunk, row0 = tile * kRowsRT;
    const int last_i = min(n - 1, a.token(row0 + kRowsRT - 1));
    const int t1 = min(min(t0 + a.chunk, c - n + last_i + 1), c);  // tokens that some row sees
    if (split > 0 && t0 >= t1) return;

    const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, j = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wrow = row0 + 32 * wave;  // the wave's first row
    const int32_t* table = sq.tables + (int64_t)seq * sq.table_stride + t0 / kKv4Page;
    const int pages = t1 > t0 ? (t1 - t0 + kKv4Page - 1) / kKv4Page : 0;
    auto stage_pages = [&](int from) {
        for (int p = from + tid; p < min(pages, from + kMaxPages); p += 256) {
            const int id = table[p];
            pg[p - from] = id >= 0 && id < sq.n_blocks ? id : -1;
        }
    };
    stage_pages(0);

    // the lane's rows, and their queries as B operands (dims 32j .. 32j + 31; no load under a
    // condition, as above)
    const int last_row = n * a.G - 1;
    int pos[2];
    int64_t grow[2];
    int head[2];
    bool row_ok[2];
    int up[2];  // the power of two that a row's query is moved by
    Frag16 qf[2][2][4];
#pragma unroll
    for (int ct = 0; ct < 2; ++ct) {
        const int r = wrow + 16 * ct + col, i = a.token(r);
        head[ct] = h * a.G + (r - i * a.G);
        row_ok[ct] = i < n;
        pos[ct] = row_ok[ct] && c > 0 ? c - n + i : -1;
        grow[ct] = (int64_t)first + i;
        // 16 rows by way of the wave's own 8 KB: rows of 512 bytes in, a lane's 32 dims out
        float* qs = reinterpret_cast<float*>(tiles[0][0]) + wave * (16 * kKv4Dim);
        auto place = [](int row, int d) { return row * kKv4Dim + (d ^ ((row & 7) << 2)); };
        float x0[16], x1[16], cv[16], sv[16];
#pragma unroll
        for (int rr = 0; rr < 16; ++rr) {
            const int r2 = min(wrow + 16 * ct + rr, last_row), i2 = a.token(r2);
            const int64_t at = (int64_t)(first + i2) * a.q_stride +
                               (int64_t)(h * a.G + (r2 - i2 * a.G)) * kKv4Dim + lane;
            x0[rr] = ld_act<HALF>(a.q, at);
            x1[rr] = ld_act<HALF>(a.q, at + 64);
            cv[rr] = 1.0f;
            sv[rr] = 0.0f;
        }
        if (a.rope && c > 0)
#pragma unroll
            for (int rr = 0; rr < 16; ++rr) {
                const int p2 = c - n + a.token(min(wrow + 16 * ct + rr, last_row));
                const float* cs = a.rope + (int64_t)min(max(p2, 0), c - 1) * kKv4Dim + lane;
                cv[rr] = cs[0];
                sv[rr] = cs[64];
            }
#pragma unroll
        for (int rr = 0; rr < 16; ++rr) {
            const float y0 = x0[rr];
            x0[rr] = __builtin_fmaf(y0, cv[rr], -__fmul_rn(x1[rr], sv[rr]));
            x1[rr] = __builtin_fmaf(y0, sv[rr], __fmul_rn(x1[rr], cv[rr]));
            qs[place(rr, lane)] = __fmul_rn(x0[rr], kQkScale * kLog2e);
            qs[place(rr, lane + 64)] = __fmul_rn(x1[rr], kQkScale * kLog2e);
        }
        f32x4 x[8];
        float amax = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[e] = *reinterpret_cast<const f32x4*>(qs + place(col, 32 * j + 4 * e));
#pragma unroll
            for (int k = 0; k < 4; ++k) amax = fmaxf(amax, fabsf(x[e][k]));
        }
        up[ct] = row_shift(max_quarters(amax));
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[e] *= pow2(up[ct]);
#pragma unroll
            for (int k = 0; k < 4; k += 2) {
                const uint32_t hi = pack16(x[e][k], x[e][k + 1]);
                qf[ct][0][e >> 1].w[2 * (e & 1) + k / 2] = hi;
                qf[ct][1][e >> 1].w[2 * (e & 1) + k / 2] =
                    pack16(rest_lo(x[e][k], hi), rest_hi(x[e][k + 1], hi));
            }
        }
    }
    __syncthreads();

    f32x4 acc[2][8];
    float m[2], l[2];
#pragma unroll
    for (int ct = 0; ct < 2; ++ct) {
        m[ct] = -INFINITY;
        l[ct] = 0.0f;
#pragma unroll
        for (int d = 0; d < 8; ++d) acc[ct][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    int vshift = 0, vtop = 1;
    int wr[4], rd[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        wr[k] = piece_at(col, 4 * j + k);
        rd[k] = piece_at(4 * j + (col >> 2), 2 * k + (col >> 1 & 1)) + (col & 1) * 4;
    }
    // a lane's share of a tile: 32 dims of token 16 wave + col
    uint4 kr = {}, vr = {};
    int ks = 0, vs = 0;
    bool none = false;  // no one's token
    auto load = [&](int t, int w0) {
        const int p = min(((t - w0) >> 4) + wave, pages - 1 - ((w0 - t0) >> 4));
        const int id = __builtin_amdgcn_readfirstlane(pg[p]);
        const int64_t row =
            (((int64_t)max(id, 0) * sq.n_layers + sq.layer) * sq.Hkv + h) * kKv4Page;
        const uint32_t code = (uint32_t)(col * kKv4Row + j * 16), sc = col * kKv4Scales + j;
        kr = *reinterpret_cast<const uint4*>(a.pk + row * kKv4Row + code);
        vr = *reinterpret_cast<const uint4*>(a.pv + row * kKv4Row + code);
        ks = (a.pks + row * kKv4Scales)[sc];
        vs = (a.pvs + row * kKv4Scales)[sc];
        none = id < 0 || t + 16 * wave + col >= t1;  // (looked at with the scales, when they come)
    };
    auto store = [&](uint16_t* dst, uint4 codes, int byte) {
        const float sc = byte_scale(byte);
        const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
#pragma unroll
        for (int st = 0; st < 4; ++st)
            *reinterpret_cast<uint4*>(dst + wave * 16 * kKv4Dim + wr[st]) =
                fp4_to_half8(w[st], sc);
    };
    const int low = c - n + a.token(wrow);                      // the wave's first position
    const int high = c - n + min(n - 1, a.token(wrow + 31));  // and its last
    // A tile into its half of LDS. What fp16 does not hold as it is: keys are moved token by token;
    // values all together, which waits for the tile's turn (the values then go in again).
    int vby = 0;
    bool skip = false;
    auto convert = [&](int half) {
        skip = none;
        int kb = skip ? 127 : ks, by = 0, flag = 0;
        vby = skip ? 127 + vshift : vs;
        if (__ballot(!in_range(kb) || !in_range(vby - vshift))) {
            if (kb > 252 || no_codes(kr)) kb = 0;
            if (vby > 252 || no_codes(vr)) vby = 0;
            by = (int)max_quarters((float)kb) - kTopScale;
            kb -= by;
            flag = __ballot(vby > 0 && vby - vshift < kLowScale) ? 3 : 1;
        }
        if (!skip) vtop = max(vtop, vby);
        store(tiles[half][0], kr, kb);
        store(tiles[half][1], vr, vby - vshift);
        if (j == 0) moved[half][16 * wave + col] = by;
        if (lane == 0) flags[half][wave] = flag;
    };
    int w0 = t0;
    const bool any = t0 < t1 && sq.n_blocks > 0;
    __syncthreads();
    if (any) {
        load(t0, w0);
        convert(0);
    }
    for (int t = t0, half = 0; t < t1 && any; t += kTile, half ^= 1) {
        int ids[4];
        bool bad = false;
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) {
            const int p = ((t - w0) >> 4) + tt;
            ids[tt] = p < pages - ((w0 - t0) >> 4) ? __builtin_amdgcn_readfirstlane(pg[p]) : -1;
            bad = bad || ids[tt] < 0;
        }
        __syncthreads();
        const uint16_t* kt = tiles[half][0];
        uint16_t* vt = tiles[half][1];
        const int* fl = flags[half];
        const int flag = __builtin_amdgcn_readfirstlane(fl[0] | fl[1] | fl[2] | fl[3]);
        const bool scaled = flag != 0;
        if (scaled) {
            // the values' power of two for the largest scale so far, and the tile once more
            const int mine = (int)wave_max((float)vtop);
            if (lane == 0) tops[wave] = mine;
            __syncthreads();
            vtop = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
            const int shift = vtop - kTopScale;
            if (vtop - vshift > kTopScale || (flag > 1 && vtop - vshift < kTopScale)) {
                const float f = pow2(vshift - shift);
#pragma unroll
                for (int ct = 0; ct < 2; ++ct)
#pragma unroll
                    for (int d = 0; d < 8; ++d) acc[ct][d] *= f;
                if (skip) vby += shift - vshift;
                vshift = shift;
                store(vt, vr, vby - vshift);
            }
            __syncthreads();
        }
        const int next = t + kTile;
        if (next < t1) {
            if (next >= w0 + kMaxPages * kKv4Page) {  // (page numbers kMaxPages at a time)
                w0 = next;
                stage_pages((w0 - t0) / kKv4Page);
                __syncthreads();
            }
            load(next, w0);
        }
        if (t <= high && a.token(wrow) < n) {
            f32x4 s[2][4];
            // (neighbouring MFMAs add to different sums, as above)
#pragma unroll
            for (int tt = 0; tt < 4; ++tt) s[0][tt] = s[1][tt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int st = 0; st < 4; ++st) {
                f16x8 kf[4];
#pragma unroll
                for (int tt = 0; tt < 4; ++tt)
                    kf[tt] = *reinterpret_cast<const f16x8*>(kt + wr[st] + tt * 16 * kKv4Dim);
#pragma unroll
                for (int p = 0; p < 2; ++p)
#pragma unroll
                    for (int tt = 0; tt < 4; ++tt)
#pragma unroll
                        for (int ct = 0; ct < 2; ++ct)
                            s[ct][tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                                kf[tt], qf[ct][p][st].v, s[ct][tt], 0, 0, 0);
            }
            // (by both powers at once: a large key's and a small query's may be beyond fp32 alone)
            if (scaled)
#pragma unroll
                for (int tt = 0; tt < 4; ++tt) {
                    const i32x4 by = *reinterpret_cast<const i32x4*>(moved[half] + 16 * tt + 4 * j);
#pragma unroll
                    for (int ct = 0; ct < 2; ++ct)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            s[ct][tt][i] = __builtin_ldexpf(s[ct][tt][i], by[i] - up[ct]);
                }
            const float unit[2] = {scaled ? 1.0f : pow2(-up[0]), scaled ? 1.0f : pow2(-up[1])};
            const bool mask = bad || t + kTile - 1 > low;
            float shift[2];
#pragma unroll
            for (int ct = 0; ct < 2; ++ct) {
                if (mask)
#pragma unroll
                    for (int tt = 0; tt < 4; ++tt)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (ids[tt] < 0 || t + 16 * tt + 4 * j + i > pos[ct])
                                s[ct][tt][i] = -INFINITY;
                float top[4];
#pragma unroll
                for (int tt = 0; tt < 4; ++tt)
                    top[tt] = fmaxf(fmaxf(s[ct][tt][0], s[ct][tt][1]),
                                    fmaxf(s[ct][tt][2], s[ct][tt][3]));
                const float mn = fmaxf(
                    m[ct],
                    unit[ct] * max_quarters(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]))));
                const float base = mn == -INFINITY ? 0.0f : mn;
                const float alpha = __builtin_amdgcn_exp2f(m[ct] - base);
                m[ct] = mn;
                shift[ct] = kWeightBits - base;
                if (__ballot(alpha != 1.0f)) {
#pragma unroll
                    for (int d = 0; d < 8; ++d) acc[ct][d] *= alpha;
                    l[ct] *= alpha;
                }
            }
            // (parts of tokens are alike: a wave at its products goes first, and the two of a SIMD
            // take turns. 512 rows after 8000 tokens 95 us, 104 without; whole prompts of up to
            // 2000 tokens, which are not alike, 103.4 and 101.9.)
            if (a.splits > 1) __builtin_amdgcn_s_setprio(1);
            // (the weights of the second 32 tokens between the products of the first)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                Frag16 pf[2][2];  // [column tile][part]
#pragma unroll
                for (int ct = 0; ct < 2; ++ct) {
                    float sum[2];
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        f32x4& w = s[ct][2 * u + k];
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            w[i] = __builtin_amdgcn_exp2f(
                                __builtin_fmaf(w[i], unit[ct], shift[ct]));
                        sum[k] = (w[0] + w[1]) + (w[2] + w[3]);
                    }
                    l[ct] += sum[0] + sum[1];
#pragma unroll
                    for (int e = 0; e < 8; e += 2) {
                        const float p0 = s[ct][2 * u + (e >> 2)][e & 3];
                        const float p1 = s[ct][2 * u + (e >> 2)][(e & 3) + 1];
                        const uint32_t hi = pack16(p0, p1);
                        pf[ct][0].w[e >> 1] = hi;
                        pf[ct][1].w[e >> 1] = pack16(rest_lo(p0, hi), rest_hi(p1, hi));
                    }
                }
#pragma unroll
                for (int d0 = 0; d0 < 8; d0 += 4) {
                    typedef __attribute__((address_space(3))) s16x4* lds4;
                    union {
                        s16x4 h[2];
                        f16x8 v;
                    } vf[4];
#pragma unroll
                    for (int d = 0; d < 4; ++d) {
                        uint16_t* src = vt + rd[d] + (d0 >> 2) * 64 + u * 32 * kKv4Dim;
                        vf[d].h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)src);
                        vf[d].h[1] =
                            __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(src + 16 * kKv4Dim));
                    }
#pragma unroll
                    for (int p = 0; p < 2; ++p)
#pragma unroll
                        for (int d = 0; d < 4; ++d)
#pragma unroll
                            for (int ct = 0; ct < 2; ++ct)
                                acc[ct][d0 + d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                                    vf[d].v, pf[ct][p].v, acc[ct][d0 + d], 0, 0, 0);
                }
            }
            if (a.splits > 1) __builtin_amdgcn_s_setprio(0);
        }
        if (next < t1) convert(half ^ 1);
    }
#pragma unroll
    for (int ct = 0; ct < 2; ++ct) {
        float L = sum_quarters(l[ct]);
        if (!row_ok[ct]) continue;
        // (by the sum of weights, and the 2^15 in both, before the values' power of two)
        const auto times = [](f32x4 v, int e) {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = __builtin_ldexpf(v[i], e);
            return v;
        };
        if (pos[ct] < a.chunk || a.splits == 1) {
            if (split > 0) continue;
            if (vshift != 0 && L != 0.0f) {
#pragma unroll
                for (int d = 0; d < 8; ++d) acc[ct][d] = times(acc[ct][d] * (1.0f / L), vshift);
                L = 1.0f;
            }
#pragma unroll
            for (int d = 0; d < 8; ++d)
                store4<HALF>(a, grow[ct] * a.out_stride + (int64_t)head[ct] * kKv4Dim + 16 * d +
                                    4 * j,
                             acc[ct][d], L);
        } else {
            const int64_t at = (grow[ct] * a.Hq + head[ct]) * a.splits + split;
            const int e = vshift - (int)kWeightBits;
#pragma unroll
            for (int d = 0; d < 8; ++d)
                *reinterpret_cast<f32x4*>(a.part_o + at * kKv4Dim + 16 * d + 4 * j) =
                    times(acc[ct][d], e);
            if (j == 0)
                a.part_ml[at] = make_float2(m[ct], __builtin_ldexpf(L, -(int)kWeightBits));
        }
    }
}

// Several sequences of a few rows: all their steps in a row (sequence by sequence, unit by unit)
// and an equal share of them to each of as many workgroups as the GPU holds at once, so that
// lengths, which only the device knows, need not be alike. A share holds the end of a unit that
// an earlier workgroup began, whole units and the beginning of one: two records at most. 48
// sequences of up to 8190 tokens (223127 in all), 32 / 8 heads, fp16: 54 us, 4.5 TB/s.
template <int ROWS, bool HALF>
__global__ void __launch_bounds__(256, ROWS == 16 ? 2 : 3)
kv4_attn_even_kernel(Kv4Attn a, Kv4Seqs sq) {
    __shared__ Kv4Smem<ROWS, 1> sm;
    __shared__ uint32_t wsum[4];
    __shared__ int at_base, at_seq;
    const int per = (sq.B + 255) / 256, b0 = threadIdx.x * per;
    if (threadIdx.x == 0) at_seq = sq.B;
    int mine, total;
    int base = scan_work<ROWS>(a, sq, b0, min(sq.B, b0 + per), wsum, mine, total);
    total = uniform(total);
    const int begin = wg_start(blockIdx.x, total, a.wgs);
    const int end = wg_start(blockIdx.x + 1, total, a.wgs);
    if (begin >= end) return;
    if (begin >= base && begin < base + mine) {
        int b = b0;
        for (;; ++b) {
            const int w = SeqWork(sq, b, a.G, ROWS).total(sq.Hkv);
            if (begin < base + w) break;
            base += w;
        }
        at_seq = b;
        at_base = base;
    }
    __syncthreads();
    int b = uniform(at_seq);
    base = uniform(at_base);
    for (int at = begin; at < end && b < sq.B;) {
        const SeqWork w(sq, b, a.G, ROWS);
        const int past = at - base;
        if (past >= w.total(sq.Hkv)) {
            base += w.total(sq.Hkv);
            ++b;
            continue;
        }
        const int unit = past / w.slots(), s0 = past - unit * w.slots();
        const int len = min(w.slots() - s0, end - at);
        at += len;
        // (slot 0 is the one without tokens)
        const int from = max(s0 - 1, 0), to = s0 + len - 1;
        if (to == from) continue;
        Segment g;
        g.seq = b;
        g.first = w.first;
        g.n = w.n;
        g.c = w.c;
        g.h = unit / w.tiles;
        g.tile = unit - g.h * w.tiles;
        g.t0 = from * kStep;
        g.len = (to - from) * kStep;
        g.whole = to - from == w.steps;
        g.rec = ((int64_t)blockIdx.x * 2 + (from == 0 ? 1 : 0)) * ROWS;
        g.split = 0;
        kv4_segment<ROWS, 1, HALF, true>(a, sq, g, sm);
    }
}

// The records of a row's head, GROUPS lanes groups of 32 x 4 dims sharing them: record k of ns
// is first + k * step, of k >= 1 `skip` less.
struct Records {
    int64_t first, step, skip;
    int ns;
    __device__ __forceinline__ int64_t at(int k) const {
        return first + k * step - (k > 0 ? skip : 0);
    }
};
template <bool HALF, int GROUPS>
__device__ __forceinline__ void kv4_join(const Kv4Attn& a, const Records& rc, int64_t out_at, int g,
                                         f32x4 (*ov)[32], float* lv) {
    const int lane = threadIdx.x & 63, d4 = threadIdx.x & 31;
    // a group's first sums are on their way while the maximum is found
    constexpr int kAhead = GROUPS > 1 ? 1 : 6;
    f32x4 pv[kAhead];
    float2 pe[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
        const int s = g + GROUPS * k;
        const int64_t at = rc.at(min(s, rc.ns - 1));  // (no load under a condition)
        pv[k] = *reinterpret_cast<const f32x4*>(a.part_o + at * kKv4Dim + 4 * d4);
        pe[k] = a.part_ml[at];
        if (s >= rc.ns) pe[k] = make_float2(-INFINITY, 0.0f);
    }
    float M = -INFINITY;
    if (GROUPS > 1) {
        for (int s = lane; s < rc.ns; s += 64) M = fmaxf(M, a.part_ml[rc.at(s)].x);
        M = wave_max(M);
    } else {
        for (int s = kAhead; s < rc.ns; ++s) M = fmaxf(M, a.part_ml[rc.at(s)].x);
#pragma unroll
        for (int k = 0; k < kAhead; ++k) M = fmaxf(M, pe[k].x);
    }
    const float base = M == -INFINITY ? 0.0f : M;
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    float L = 0.0f;
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
        const float f = __builtin_amdgcn_exp2f(pe[k].x - base);
        L += pe[k].y * f;
        v += f * pv[k];
    }
#pragma unroll 4
    for (int s = g + GROUPS * kAhead; s < rc.ns; s += GROUPS) {
        const float2 e = a.part_ml[rc.at(s)];
        const float f = __builtin_amdgcn_exp2f(e.x - base);
        L += e.y * f;
        v += f * *reinterpret_cast<const f32x4*>(a.part_o + rc.at(s) * kKv4Dim + 4 * d4);
    }
    if (GROUPS > 1) {
        ov[g][d4] = v;
        if (d4 == 0) lv[g] = L;
        __syncthreads();
        if (g > 0) return;
        for (int k = 1; k < GROUPS; ++k) v += ov[k][d4], L += lv[k];
    }
    store4<HALF>(a, out_at + 4 * d4, v, L);
}

// Rows times heads up to which each gets a workgroup for its records: 20 of up to 127 records 2.6 to
// 3.8 us; 1536 of about three 61 us in all, 59 with a group of lanes each; 30000, 107 and 59.
constexpr int kWideJoin = 1024;

// Joins the splits of a grid: a workgroup has a row's head (WIDE: few rows, many records a head,
// shared by 16 groups of lanes) or 16 of its heads.
template <bool HALF, bool WIDE>
__global__ void __launch_bounds__(512) kv4_join_kernel(Kv4Attn a, Kv4Seqs sq) {
    __shared__ f32x4 ov[WIDE ? 16 : 1][32];
    __shared__ float lv[16];
    const int row = blockIdx.x, tid = threadIdx.x, grp = tid >> 5;
    int seq, pos;
    if (!kv4_place(sq, row, tid & 15, seq, pos) || pos < a.chunk) return;
    const int head = WIDE ? (int)blockIdx.y : (int)blockIdx.y * 16 + grp;
    if (head >= a.Hq) return;
    const Records rc{((int64_t)row * a.Hq + head) * a.splits, 1, 0, pos / a.chunk + 1};
    kv4_join<HALF, WIDE ? 16 : 1>(a, rc, row * a.out_stride + (int64_t)head * kKv4Dim,
                                  WIDE ? grp : 0, ov, lv);
}

// Joins the shares of steps dealt evenly: a workgroup has a row's head (WIDE: few rows, many
// records a head, shared by 8 groups of lanes) or 8 of its heads. Rows of sequences without tokens,
// which no workgroup has had, are written as zeros.
template <int ROWS, bool HALF, bool WIDE>
__global__ void __launch_bounds__(256) kv4_join_even_kernel(Kv4Attn a, Kv4Seqs sq) {
    __shared__ f32x4 ov[WIDE ? 8 : 1][32];
    __shared__ float lv[8];
    __shared__ uint32_t wsum[4];
    __shared__ unsigned long long at;  // the row's sequence, plus 1, and the work before it
    const int row = blockIdx.x, tid = threadIdx.x, grp = tid >> 5;
    const int per = (sq.B + 255) / 256, b0 = tid * per, b1 = min(sq.B, b0 + per);
    if (tid == 0) at = 0;
    int mine, total;
    int base = scan_work<ROWS>(a, sq, b0, b1, wsum, mine, total);
    for (int b = b0; b < b1; ++b) {
        const SeqWork w(sq, b, a.G, ROWS);
        if (row >= w.first && row < w.first + w.n)
            atomicMax(&at, (unsigned long long)(b + 1) << 32 | (uint32_t)base);
        base += w.total(sq.Hkv);
    }
    __syncthreads();
    const int seq = uniform((int)(at >> 32)) - 1;
    const int head = WIDE ? (int)blockIdx.y : (int)blockIdx.y * 8 + grp;
    if (seq < 0 || head >= a.Hq) return;
    base = uniform((int)at);
    total = uniform(total);
    const SeqWork w(sq, seq, a.G, ROWS);
    const int64_t out_at = row * a.out_stride + (int64_t)head * kKv4Dim;
    if (w.c == 0) {
        if (!WIDE || grp == 0)
            store4<HALF>(a, out_at + 4 * (tid & 31), f32x4{0.0f, 0.0f, 0.0f, 0.0f}, 0.0f);
        return;
    }
    if (total == 0) return;
    const int h = head / a.G, r = (row - w.first) * a.G + head - h * a.G;
    const int start = base + (h * w.tiles + r / ROWS) * w.slots() + 1;
    const int w0 = wg_of(start, total, a.wgs), w1 = wg_of(start + w.steps - 1, total, a.wgs);
    if (w0 == w1) return;
    // workgroup w0 has the unit's beginning (its second record), those after it continue it
    const Records rc{((int64_t)w0 * 2 + 1) * ROWS + r % ROWS, 2 * ROWS, ROWS, w1 - w0 + 1};
    kv4_join<HALF, WIDE ? 8 : 1>(a, rc, out_at, WIDE ? grp : 0, ov, lv);
}

// Rows of a workgroup and how the tokens are dealt out, from what the host knows.
struct Kv4Plan {
    int rows, rw, splits, chunk;  // rw 8: the prompts' kernel
    bool even;
    int most;  // steps dealt evenly, at most
    int64_t wgs;
    size_t records;
};
Kv4Plan kv4_plan(int64_t T, int B, int G, int Hkv, int table_width, bool cu) {
    Kv4Plan p{};
    const int64_t per = cu ? ceil_div(T * G, B) : G;  // rows of an average sequence
    p.rows = per <= 4 ? 4 : 16;
    const int64_t ctx = (int64_t)table_width * kKv4Page;
    // Rows of a workgroup: 16 against 256 tokens at a time spread few rows over the GPU; the
    // prompts' kernel, once it has work for a while (16 us go into its queries and outputs), reads
    // and converts a token once for 128; between, many rows of few tokens, 32. Measured in us, 20 /
    // 5 heads, 16 rows | 32 | 128: a prompt of 100 tokens 7.5 | 8.9 | 21, one of 1000 38 | 34 | 44,
    // 32 of up to 128 44 | 32 | 21; 128 tokens after 4000 33 | 37 | 38, 200 after 7800 63 | 66 |
    // 56, 512 after 8000 160 | 200 | 102.
    const double units128 = (double)T * G * Hkv / kRowsRT;
    p.rw = 1;
    if (per > 64 && (units128 > 320 || units128 * ctx > 3500 * kTile))
        p.rw = 8;
    else if (per > 16 && T * G / 16 * Hkv > 512 && ctx <= 1024)
        p.rw = 2;
    const int rt = p.rows * p.rw;
    const int64_t units = cu ? T * G / rt + B : (int64_t)B * ceil_div(G, rt);
    const int64_t step = p.rw > 4 ? kTile : kTile * (4 / p.rw);
    const int64_t steps = ctx > 0 ? ceil_div(ctx, step) : 1;
    const int room = p.rows == 16 ? 512 : 768;  // workgroups that the GPU holds at once
    const int64_t most = units * Hkv * (steps + 1);
    // Units that fill the GPU twice over are balanced by its own scheduling, and where every
    // workgroup has a step at most there is nothing to balance. Between: 48 sequences of up to 8190
    // tokens, 32 / 8 heads, 59 us (a grid of splits 69).
    p.even = p.rw == 1 && B > 1 && units * Hkv < 2 * room && units * Hkv * steps > room &&
             most <= INT32_MAX;
    if (p.even) {
        p.most = (int)most;
        p.wgs = most < room ? most : room;
        p.splits = 1;
        p.records = (size_t)p.wgs * 2 * p.rows;
        return p;
    }
    const int64_t likely = cu ? (ceil_div(T * G, rt) > B ? ceil_div(T * G, rt) : B) : units;
    // (of a prompt's splits, those past its earlier rows have nothing to do)
    const double own = ctx > 0 ? (double)T / B / ctx : 0.0;  // of a sequence's tokens, its rows'
    const double some = 1.0 - 0.5 * (own < 1.0 ? own : 1.0);
    const double fits = (double)room / (likely * Hkv);
    int64_t s = fits > 1.0 ? 1 + (int64_t)((fits - 1.0) / some) : 1;
    s = s > steps ? steps : s;
    p.chunk = (int)(ceil_div(steps, s) * step);
    p.splits = ctx > 0 ? (int)ceil_div(ctx, p.chunk) : 1;
    p.wgs = units * p.splits * Hkv;
    p.records = p.splits > 1 ? (size_t)T * G * Hkv * p.splits : 0;
    return p;
}

template <int ROWS, int RW, bool HALF>
void launch_kv4(const Kv4Attn& a, const Kv4Seqs& s, hipStream_t st) {
    hipLaunchKernelGGL((kv4_attn_kernel<ROWS, RW, HALF>), dim3(a.wgs), dim3(256), 0, st, a, s);
}
template <int ROWS, bool HALF>
int launch_kv4_even(const Kv4Attn& a, const Kv4Seqs& s, hipStream_t st) {
    hipLaunchKernelGGL((kv4_attn_even_kernel<ROWS, HALF>), dim3(a.wgs), dim3(256), 0, st, a, s);
    const int rc = launch_status("kv4_attn_even_kernel");
    if (rc) return rc;
    // few rows: a head to a workgroup, its records to 8 groups of lanes
    if ((int64_t)a.T * a.Hq <= kWideJoin)
        hipLaunchKernelGGL((kv4_join_even_kernel<ROWS, HALF, true>), dim3(a.T, a.Hq), dim3(256), 0,
                           st, a, s);
    else
        hipLaunchKernelGGL((kv4_join_even_kernel<ROWS, HALF, false>),
                           dim3(a.T, (a.Hq + 7) / 8), dim3(256), 0, st, a, s);
    return launch_status("kv4_join_even_kernel");
}
template <bool HALF>
int launch_kv4_plan(const Kv4Plan& p, const Kv4Attn& a, const Kv4Seqs& s, hipStream_t st) {
    if (p.even)
        return p.rows == 4 ? launch_kv4_even<4, HALF>(a, s, st)
                           : launch_kv4_even<16, HALF>(a, s, st);
    if (p.rows == 4)
        launch_kv4<4, 1, HALF>(a, s, st);
    else if (p.rw == 1)
        launch_kv4<16, 1, HALF>(a, s, st);
    else if (p.rw == 2)
        launch_kv4<16, 2, HALF>(a, s, st);
    else
        hipLaunchKernelGGL(kv4_attn_rows_kernel<HALF>, dim3(a.wgs), dim3(256), 0, st, a, s);
    const int rc = launch_status("kv4_attn_kernel");
    if (rc || p.splits == 1) return rc;
    if ((int64_t)a.T * a.Hq <= kWideJoin)
        hipLaunchKernelGGL((kv4_join_kernel<HALF, true>), dim3(a.T, a.Hq), dim3(512), 0, st, a, s);
    else
        hipLaunchKernelGGL((kv4_join_kernel<HALF, false>), dim3(a.T, (a.Hq + 15) / 16), dim3(512),
                           0, st, a, s);
    return launch_status("kv4_join_kernel");
}

}  // namespace
}  // namespace tz

using namespace tz;

extern "C" {

TENZO_HIP_API size_t tenzo_hip_attn_kv4_ws_bytes(int64_t T, int B, int Hq, int Hkv,
                                                 int table_width, int has_cu, int /*dtype*/) {
    if (T <= 0 || B <= 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv || table_width < 0) return 0;
    const Kv4Plan p = kv4_plan(T, B, Hq / Hkv, Hkv, table_width, has_cu != 0);
    return p.records * (kKv4Dim * 4 + 8);
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
    const size_t need = tenzo_hip_attn_kv4_ws_bytes(T, B, Hq, Hkv, table_width, cu_q != nullptr,
                                                    dtype);
    TZ_CHECK(need == 0 || (ws && ws_bytes >= need && ((uintptr_t)ws & 15) == 0),
             "attn_kv4: %zu bytes of workspace needed, 16-byte aligned, %zu given", need,
             ws ? ws_bytes : 0);
    const int G = Hq / Hkv;
    const Kv4Plan p = kv4_plan(T, B, G, Hkv, table_width, cu_q != nullptr);
    TZ_CHECK(p.wgs <= 0xffffff && T <= 0x7fffff && Hq <= 65535, "attn_kv4: %lld rows of %d heads",
             (long long)T, Hq);
    Kv4Attn a{};
    a.q = q;
    a.out = out;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.pk = pk;
    a.pv = pv;
    a.pks = pks;
    a.pvs = pvs;
    a.rope = rope_cs;
    a.part_o = (float*)ws;
    a.part_ml = (float2*)((char*)ws + p.records * kKv4Dim * 4);
    a.wgs = (int)p.wgs;
    a.G = G;
    a.g_mul = G == 1 ? 0 : (uint32_t)((0x100000000ull + G - 1) / G);
    a.Hq = Hq;
    a.T = (int)T;
    a.most = p.most;
    a.chunk = p.chunk;
    a.splits = p.splits;
    a.vec_out = (((uintptr_t)out | (uintptr_t)(out_stride * (dtype ? 2 : 4))) & 15) == 0;
    return dtype ? launch_kv4_plan<true>(p, a, s, (hipStream_t)stream)
                 : launch_kv4_plan<false>(p, a, s, (hipStream_t)stream);
}

}  // extern "C"
