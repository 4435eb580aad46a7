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
constexpr int kVStride = 144;       // bf16 of a value row in LDS: 288 bytes, 8 rows over all banks

struct Kv4Attn {
    const void* q;
    void* out;
    int64_t q_stride, out_stride;
    const uint8_t* pk;
    const uint8_t* pv;
    const uint8_t* pks;
    const uint8_t* pvs;
    const float* rope;
    float* part_o;   // [T * Hq][splits][128]
    float2* part_ml; // [T * Hq][splits]: maximum (base 2) and sum
    int G, Hq, T;
    int chunk, splits;  // tokens of a split
    int vec_out;        // out allows accesses of 4 elements
};

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

union Frag {
    uint32_t w[4];
    bf16x8 v;
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

// Four outputs, the weighted sum over the sum of weights (0 where no token was seen).
template <bool HALF>
__device__ __forceinline__ void store4(const Kv4Attn& a, int64_t at, f32x4 v, float l) {
    float o[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = l != 0.0f ? v[k] / l : 0.0f;
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
        int n = 0;
        if (b < sq.B) n = max(0, sq.cu[b + 1] - sq.cu[b]);
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

// One workgroup: RT = ROWS * RW rows (token, query head of one kv head) of a sequence against a
// part of its tokens. Wave w has the rows group w % RW and every (4 / RW)-th step of 64 tokens.
//
// Scores come transposed, S^T = K Q^T, so that a lane keeps one row: K is the A operand (16
// tokens x 32 dims: the lane's 16 code bytes are a token's group of 32 dims, one scale, four
// steps of 8 dims), Q the B operand. In S^T's layout a lane holds 4 tokens of its row per 16,
// which is what the B operand of O^T = V^T P^T wants when the value rows are taken in the same
// order: no weight changes lanes. V^T comes from value rows in LDS (bf16, private to the wave)
// by transposing reads. Codes times scale are exact in bf16; queries and weights are split into
// NP parts of 8 bits (fp32: 3, every bit; fp16: 2). With ROWS < 16 the parts stand in columns
// side by side (column = part * ROWS + row) and one MFMA serves all of them.
template <int ROWS, int NP, int RW, int NW, bool HALF>
__global__ void __launch_bounds__(64 * NW, NW == 4 ? 3 : 2) kv4_attn_kernel(Kv4Attn a, Kv4Seqs sq) {
    constexpr int SLOTS = 16 / ROWS, NM = SLOTS == 1 ? NP : 1, TW = NW / RW, RT = ROWS * RW;
    static_assert(SLOTS == 1 || SLOTS >= NP, "a column for each part");
    __shared__ __align__(16) uint16_t vbuf[NW][32 * kVStride];
    __shared__ float2 ml[NW][16];
    __shared__ int pg[kMaxPages];
    static_assert(sizeof(vbuf[0]) >= 16 * kKv4Dim * 4, "the rows' sums fit a wave's part");
    static_assert(sizeof(vbuf) >= RT * kQStride * 4, "the queries fit the value buffer");

    const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, j = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rw = wave % RW, tw = wave / RW;
    const int per_unit = sq.Hkv * a.splits;
    const int unit = blockIdx.x / per_unit, rest = blockIdx.x - unit * per_unit;
    const int split = rest / sq.Hkv, h = rest - split * sq.Hkv;
    int seq, tile;
    if (!find_unit(sq, unit, a.G, RT, seq, tile)) return;
    int n = 1, first = seq;
    if (sq.cu) {
        first = sq.cu[seq];
        n = sq.cu[seq + 1] - first;
    }
    const int c = sq.length(seq);
    const int row0 = tile * RT;                       // of the sequence's n * G
    const int last_i = min(n - 1, (row0 + RT - 1) / a.G);
    const int t0 = split * a.chunk;
    const int t1 = min(min(t0 + a.chunk, c - n + last_i + 1), c);  // tokens that some row sees
    if (split > 0 && t0 >= t1) return;

    // the lane's row
    const int slot = col / ROWS, r = row0 + rw * ROWS + col % ROWS;
    const int qi = r / a.G, head = h * a.G + (r - qi * a.G);
    const bool row_ok = qi < n && first >= 0 && first + qi < a.T;
    const int pos = row_ok && c > 0 ? c - n + qi : -1;
    const int64_t grow = (int64_t)first + qi;

    const int npg = t1 > t0 ? (t1 - t0 + kKv4Page - 1) / kKv4Page : 0;
    for (int p = tid; p < npg; p += 64 * NW) {
        const int blk = sq.tables[(int64_t)seq * sq.table_stride + t0 / kKv4Page + p];
        pg[p] = blk >= 0 && blk < sq.n_blocks ? blk : -1;
    }

    // the rows' queries, rotated and scaled, by way of LDS (each wave needs all of a row)
    float* qs = reinterpret_cast<float*>(vbuf);
    for (int it = tid; it < RT * 64; it += 64 * NW) {
        const int rr = it >> 6, d = it & 63, r2 = row0 + rr, i2 = r2 / a.G;
        const int p2 = i2 < n && first >= 0 && first + i2 < a.T && c > 0 ? c - n + i2 : -1;
        float x0 = 0.0f, x1 = 0.0f;
        if (p2 >= 0) {
            const int64_t at = ((int64_t)first + i2) * a.q_stride +
                               (int64_t)(h * a.G + (r2 - i2 * a.G)) * kKv4Dim + d;
            x0 = ld_act<HALF>(a.q, at);
            x1 = ld_act<HALF>(a.q, at + 64);
            if (a.rope) {
                const float* cs = a.rope + (int64_t)p2 * kKv4Dim + d;
                const float cv = cs[0], sv = cs[64], y0 = x0;
                x0 = __builtin_fmaf(x0, cv, -__fmul_rn(x1, sv));
                x1 = __builtin_fmaf(y0, sv, __fmul_rn(x1, cv));
            }
        }
        qs[rr * kQStride + d] = __fmul_rn(x0, kQkScale * kLog2e);
        qs[rr * kQStride + d + 64] = __fmul_rn(x1, kQkScale * kLog2e);
    }
    __syncthreads();

    f32x4 acc[8];
#pragma unroll
    for (int d = 0; d < 8; ++d) acc[d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;

    uint4 kr[kSub], vr[kSub];
    uint32_t ksc[kSub], vsc[kSub];
    const uint32_t lane_code = (uint32_t)(col * kKv4Row + j * 16);
    const uint32_t lane_scale = (uint32_t)(col * kKv4Scales + j);
    auto page_row = [&](int t, int tt) -> int64_t {
        const int p = min(((t - t0) >> 4) + tt, npg - 1);
        const int id = __builtin_amdgcn_readfirstlane(pg[p]);
        return (((int64_t)max(id, 0) * sq.n_layers + sq.layer) * sq.Hkv + h) * kKv4Page;
    };
    auto load_k = [&](int t) {
#pragma unroll
        for (int tt = 0; tt < kSub; ++tt) {
            const int64_t row = page_row(t, tt);
            kr[tt] = *reinterpret_cast<const uint4*>(a.pk + row * kKv4Row + lane_code);
            ksc[tt] = (a.pks + row * kKv4Scales)[lane_scale];
        }
    };
    auto load_v = [&](int t) {
#pragma unroll
        for (int tt = 0; tt < kSub; ++tt) {
            const int64_t row = page_row(t, tt);
            vr[tt] = *reinterpret_cast<const uint4*>(a.pv + row * kKv4Row + lane_code);
            vsc[tt] = (a.pvs + row * kKv4Scales)[lane_scale];
        }
    };
    uint16_t* vb = vbuf[wave];
    const uint32_t vw = (uint32_t)(col * kVStride + j * 32);
    const uint32_t vrd = (uint32_t)((4 * j + (col >> 2)) * kVStride + (col & 3) * 4);

    int t = t0 + kTile * tw;
    const bool any = sq.n_blocks > 0;
    if (t < t1 && any) {
        load_k(t);
        load_v(t);
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
                    if (NP == 3) x[k] -= masked(x[k], m2);
                    if (SLOTS > NP && slot >= NP) x[k] = 0.0f;
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
    for (; t < t1 && any; t += kTile * TW) {
        const int next = t + kTile * TW;
        f32x4 s[kSub];
#pragma unroll
        for (int tt = 0; tt < kSub; ++tt) {
            const float sc = e8m0_to_float(ksc[tt]);
            const uint32_t w[4] = {kr[tt].x, kr[tt].y, kr[tt].z, kr[tt].w};
            s[tt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int st = 0; st < 4; ++st) {
                union {
                    bf16x2 p[4];
                    bf16x8 v;
                } kf;
                kf.p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[st], sc, 0);
                kf.p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[st], sc, 1);
                kf.p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[st], sc, 2);
                kf.p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[st], sc, 3);
#pragma unroll
                for (int p = 0; p < NM; ++p)
                    s[tt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf.v, qf[p][st].v, s[tt], 0, 0,
                                                                    0);
            }
        }
        bool bad = false;
        int id_now[kSub];
#pragma unroll
        for (int tt = 0; tt < kSub; ++tt) {
            const int p = ((t - t0) >> 4) + tt;
            id_now[tt] = p < npg ? __builtin_amdgcn_readfirstlane(pg[p]) : -1;
            bad = bad || id_now[tt] < 0;
        }
        if (next < t1) load_k(next);
        float top = -INFINITY;
#pragma unroll
        for (int tt = 0; tt < kSub; ++tt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float v = s[tt][i];
                if (ROWS == 4) v += ror16<kDppRor8>(v);
                if (ROWS == 4) v += ror16<kDppRor4>(v);
                if (ROWS == 8) v += ror16<kDppRor8>(v);
                s[tt][i] = v;
            }
        // a step that a row may not see whole: past its position, or absent pages
        if (bad || t + kTile - 1 > c - n + row0 / a.G) {
#pragma unroll
            for (int tt = 0; tt < kSub; ++tt)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (id_now[tt] < 0 || t + 16 * tt + 4 * j + i > pos) s[tt][i] = -INFINITY;
        }
#pragma unroll
        for (int tt = 0; tt < kSub; ++tt)
#pragma unroll
            for (int i = 0; i < 4; ++i) top = fmaxf(top, s[tt][i]);
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
        for (int tt = 0; tt < kSub; ++tt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[tt][i] = __builtin_amdgcn_exp2f(s[tt][i] - base);
                l += s[tt][i];
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
                    *reinterpret_cast<uint4*>(vb + vw + k * 16 * kVStride + st * 8) = f.v;
                }
            }
            if (u == kSub / 2 - 1 && next < t1) load_v(next);
            Frag pf[NM];
            float p8[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                p8[e] = s[2 * u + (e >> 2)][e & 3];
                if (SLOTS > 1) {
                    p8[e] -= masked(p8[e], m1);
                    if (NP == 3) p8[e] -= masked(p8[e], m2);
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
            for (int d = 0; d < 8; ++d) {
                typedef __attribute__((address_space(3))) s16x4* lds4;
                union {
                    s16x4 h[2];
                    bf16x8 v;
                } vf;
                vf.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(vb + vrd + d * 16));
                vf.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (lds4)(vb + vrd + 16 * kVStride + d * 16));
#pragma unroll
                for (int p = 0; p < NM; ++p)
                    acc[d] =
                        __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf.v, pf[p].v, acc[d], 0, 0, 0);
            }
        }
    }

    l = sum_quarters(l);
    if (SLOTS > 1) {
#pragma unroll
        for (int d = 0; d < 8; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float v = slot < NP ? acc[d][i] : 0.0f;
                v += ror16<kDppRor8>(v);
                if (ROWS == 4) v += ror16<kDppRor4>(v);
                acc[d][i] = v;
            }
    }
    if (TW > 1) {
        // the waves' sums meet: every wave's rows in its own part of the value buffer
        float* o = reinterpret_cast<float*>(vb);
        if (slot == 0) {
#pragma unroll
            for (int d = 0; d < 8; ++d)
                *reinterpret_cast<f32x4*>(o + col * kKv4Dim + 16 * d + 4 * j) = acc[d];
            if (j == 0) ml[wave][col] = make_float2(m, l);
        }
        __syncthreads();
        for (int it = tid; it < RT * 32; it += 64 * NW) {
            const int rr = it >> 5, d4 = it & 31, grp = rr / ROWS, cc = rr % ROWS;
            const int r2 = row0 + rr, i2 = r2 / a.G;
            if (i2 >= n || first < 0 || first + i2 >= a.T) continue;
            float M = -INFINITY, L = 0.0f;
            f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < TW; ++w) M = fmaxf(M, ml[w * RW + grp][cc].x);
            const float base = M == -INFINITY ? 0.0f : M;
#pragma unroll
            for (int w = 0; w < TW; ++w) {
                const float2 e = ml[w * RW + grp][cc];
                const float f = __builtin_amdgcn_exp2f(e.x - base);
                L += e.y * f;
                v += f * *reinterpret_cast<const f32x4*>(
                             reinterpret_cast<const float*>(vbuf[w * RW + grp]) + cc * kKv4Dim +
                             4 * d4);
            }
            const int p2 = c > 0 ? c - n + i2 : -1;
            const int64_t g2 = (int64_t)first + i2, hd = h * a.G + (r2 - i2 * a.G);
            if (p2 < a.chunk || a.splits == 1) {
                if (split == 0)
                    store4<HALF>(a, g2 * a.out_stride + hd * kKv4Dim + 4 * d4, v, L);
            } else {
                const int64_t at = (g2 * a.Hq + hd) * a.splits + split;
                *reinterpret_cast<f32x4*>(a.part_o + at * kKv4Dim + 4 * d4) = v;
                if (d4 == 0) a.part_ml[at] = make_float2(M, L);
            }
        }
    } else if (row_ok && slot == 0) {
        if (pos < a.chunk || a.splits == 1) {
            if (split == 0)
#pragma unroll
                for (int d = 0; d < 8; ++d)
                    store4<HALF>(a, grow * a.out_stride + (int64_t)head * kKv4Dim + 16 * d + 4 * j,
                                 acc[d], l);
        } else {
            const int64_t at = (grow * a.Hq + head) * a.splits + split;
#pragma unroll
            for (int d = 0; d < 8; ++d)
                *reinterpret_cast<f32x4*>(a.part_o + at * kKv4Dim + 16 * d + 4 * j) = acc[d];
            if (j == 0) a.part_ml[at] = make_float2(m, l);
        }
    }
}

// Joins the splits of a row and head: 32 lanes x 4 dims, 16 groups of splits.
template <bool HALF>
__global__ void __launch_bounds__(512) kv4_join_kernel(Kv4Attn a, Kv4Seqs sq) {
    __shared__ f32x4 ov[16][32];
    __shared__ float lv[16];
    const int row = blockIdx.x, head = blockIdx.y, tid = threadIdx.x;
    int seq, pos;
    if (!kv4_place(sq, row, tid & 15, seq, pos) || pos < a.chunk) return;
    const int ns = pos / a.chunk + 1;
    const int64_t at = ((int64_t)row * a.Hq + head) * a.splits;
    const float2* ml = a.part_ml + at;
    float M = -INFINITY;
    for (int s = tid & 63; s < ns; s += 64) M = fmaxf(M, ml[s].x);
    M = wave_max(M);
    const float base = M == -INFINITY ? 0.0f : M;
    const int d4 = tid & 31, g = tid >> 5;
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    float L = 0.0f;
#pragma unroll 4
    for (int s = g; s < ns; s += 16) {
        const float2 e = ml[s];
        const float f = __builtin_amdgcn_exp2f(e.x - base);
        L += e.y * f;
        v += f * *reinterpret_cast<const f32x4*>(a.part_o + (at + s) * kKv4Dim + 4 * d4);
    }
    ov[g][d4] = v;
    if (d4 == 0) lv[g] = L;
    __syncthreads();
    if (g == 0) {
        for (int k = 1; k < 16; ++k) v += ov[k][d4], L += lv[k];
        store4<HALF>(a, row * a.out_stride + (int64_t)head * kKv4Dim + 4 * d4, v, L);
    }
}

// Rows and waves of a workgroup, tokens of a split and how many splits, from what the host knows.
struct Kv4Plan {
    int rows, rw, nw, splits, chunk;
    int64_t units;
};
Kv4Plan kv4_plan(int64_t T, int B, int G, int Hkv, int table_width, bool cu, bool half) {
    Kv4Plan p{};
    const int64_t per = cu ? ceil_div(T * G, B) : G;  // rows of an average sequence
    const int packed = half ? 8 : 4;
    p.rows = per <= packed ? packed : 16;
    p.rw = per <= 16 ? 1 : per <= 32 ? 2 : 4;
    const int rt = p.rows * p.rw;
    p.units = cu ? T * G / rt + B : (int64_t)B * ceil_div(G, rt);
    const int64_t ctx = (int64_t)table_width * kKv4Page;
    const int64_t wgs = p.units * Hkv;
    // few sequences that three steps of 8 waves get through: the second launch costs more
    p.nw = p.rw == 1 && wgs <= 256 && ctx <= 3 * 8 * kTile ? 8 : 4;
    const int64_t step = kTile * (p.nw / p.rw);
    // else enough workgroups for every CU to have four, each wave a step of tokens at least
    int64_t s = p.nw == 8 ? 1 : ceil_div(1024, wgs);
    s = s < ceil_div(ctx, step) ? s : ceil_div(ctx, step);
    if (s < 1) s = 1;
    int64_t chunk = ceil_div(ceil_div(ctx, s), step) * step;
    if (chunk > kMaxPages * kKv4Page) chunk = kMaxPages * kKv4Page;
    if (chunk < step) chunk = step;
    p.chunk = (int)chunk;
    p.splits = ctx > 0 ? (int)ceil_div(ctx, chunk) : 1;
    return p;
}

template <int ROWS, int NP, int RW, int NW, bool HALF>
void launch_kv4(const Kv4Attn& a, const Kv4Seqs& s, unsigned wgs, hipStream_t st) {
    hipLaunchKernelGGL((kv4_attn_kernel<ROWS, NP, RW, NW, HALF>), dim3(wgs), dim3(64 * NW), 0, st,
                       a, s);
}
template <int PACKED, int NP, bool HALF>
void launch_kv4_plan(const Kv4Plan& p, const Kv4Attn& a, const Kv4Seqs& s, unsigned wgs,
                     hipStream_t st) {
    if (p.rows == PACKED && p.nw == 8)
        launch_kv4<PACKED, NP, 1, 8, HALF>(a, s, wgs, st);
    else if (p.rows == PACKED)
        launch_kv4<PACKED, NP, 1, 4, HALF>(a, s, wgs, st);
    else if (p.nw == 8)
        launch_kv4<16, NP, 1, 8, HALF>(a, s, wgs, st);
    else if (p.rw == 1)
        launch_kv4<16, NP, 1, 4, HALF>(a, s, wgs, st);
    else if (p.rw == 2)
        launch_kv4<16, NP, 2, 4, HALF>(a, s, wgs, st);
    else
        launch_kv4<16, NP, 4, 4, HALF>(a, s, wgs, st);
}

}  // namespace
}  // namespace tz

using namespace tz;

extern "C" {

TENZO_HIP_API size_t tenzo_hip_attn_kv4_ws_bytes(int64_t T, int B, int Hq, int Hkv,
                                                 int table_width, int has_cu, int dtype) {
    if (T <= 0 || B <= 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv || table_width < 0) return 0;
    const Kv4Plan p = kv4_plan(T, B, Hq / Hkv, Hkv, table_width, has_cu != 0, dtype != 0);
    return p.splits > 1 ? (size_t)T * Hq * p.splits * (kKv4Dim * 4 + 8) : 0;
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
    const Kv4Plan p = kv4_plan(T, B, G, Hkv, table_width, cu_q != nullptr, dtype != 0);
    const int64_t wgs = p.units * p.splits * Hkv;
    TZ_CHECK(wgs <= 0xffffff && T <= 0x7fffff && Hq <= 65535, "attn_kv4: %lld rows of %d heads",
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
    a.part_ml = (float2*)((char*)ws + (size_t)T * Hq * p.splits * kKv4Dim * 4);
    a.G = G;
    a.Hq = Hq;
    a.T = (int)T;
    a.chunk = p.chunk;
    a.splits = p.splits;
    a.vec_out = (((uintptr_t)out | (uintptr_t)(out_stride * (dtype ? 2 : 4))) & 15) == 0;
    hipStream_t st = (hipStream_t)stream;
    if (dtype)
        launch_kv4_plan<8, 2, true>(p, a, s, (unsigned)wgs, st);
    else
        launch_kv4_plan<4, 3, false>(p, a, s, (unsigned)wgs, st);
    const int rc2 = launch_status("kv4_attn_kernel");
    if (rc2 || p.splits == 1) return rc2;
    const dim3 jgrid((unsigned)T, (unsigned)Hq);
    if (dtype)
        hipLaunchKernelGGL(kv4_join_kernel<true>, jgrid, dim3(512), 0, st, a, s);
    else
        hipLaunchKernelGGL(kv4_join_kernel<false>, jgrid, dim3(512), 0, st, a, s);
    return launch_status("kv4_join_kernel");
}

}  // extern "C"
