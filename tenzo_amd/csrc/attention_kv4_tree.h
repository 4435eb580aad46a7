// A piece of work of attention over trees of drafted tokens (part of attention_kv4.hip): 128 rows
// of a sequence's nodes and query heads, 32 (two column tiles) to a wave, against a part of its
// tokens, 64 at a time.
//
// Scores come from the matrix cores' own 4-bit products: a lane's 16 code bytes are a token's group
// of 32 dims and its scale byte the group's, just what v_mfma_scale_f32_16x16x128_f8f6f4 takes, so
// keys go from memory to the products as they are, 128 dims at once. Queries are split into parts
// of 6 bits (E2M3) with a scale for each 32 dims of a row and each part: with 2^E <= the largest
// element, a part in units of 2^(E - 1 - 5 p) leaves at most 2^(E - 4 - 5 p) of any. Five parts leave
// 2^-24 of the largest of a query's 32 dims; the products cost 5/8 of what they do with fp16 operands in
// two parts. (fp16 queries take five too: beside a dim 100 times as large as the others, four would
// leave 2^-19 of it, 2^-12 of the others, less than their own 11 bits.)
//
// Codes and scales are loaded straight into a ring in LDS, kAhead steps before they are used (a step
// takes little longer than its codes' way from memory: with one step ahead, in registers, each took
// 4 us, whatever its products). Values go on as in the prompts' kernel: each wave converts 16
// tokens' to fp16 (moved by a power of two common to all where scales are out of its range), for the
// next step, and every fragment read from there serves both column tiles.
//
// A row's scores come out of the products as logarithms of its weights: queries carry 1/sqrt(128)
// and log2 e, and the sums begin at kBits less the row's maximum so far. Only where a score goes
// beyond what the weights' type holds (fp16 calls: 2^3 above the maximum; fp32 calls: at all) are
// maximum, weights and sums moved. Weights are held in two parts of fp16, 22 bits, whatever the call's
// type, so that a tree is answered as exactly here as in the kernels of fewer rows (what is below
// fp16's numbers is lost: 2^-37 of a row's largest weight in fp16 calls, 2^-40 in fp32 ones). Their sum
// comes from the products too, from the same parts against ones.
//
// With one part of weights and four of queries fp16 calls take 16 to 20% less, at 1.27 times the error
// of their outputs' rounding (2.64e-4 against 2.08e-4): a tree's answer would depend on what else is in
// the batch. us, one and four | two and five: 16 trees of up to 64 nodes after up to 4036 tokens, 32 / 8
// heads, fp16, with the join 67 | 84; 2 of up to 60 after up to 31941, 16 / 2, 51.5 | 61.6.
//
// Without the join 76 and 55 us (fp32 rows take as long). A step takes two workgroups a CU 2.5 us, of
// which a SIMD's two waves spend 1.5 on products and 0.9 on exponentials and other vector work, little of
// it side by side. (With one part of weights, where it was 2.1: one workgroup alone 1.5, eight waves of
// 16 rows 2.2, fragments of values read into two buffers 2.1.) All 256 registers are taken; 11 more
// (2 or 3 where a workgroup has all tokens) wait in scratch memory for the steps with masks and the end.
#pragma once

constexpr int kHardScale = 252;  // scale bytes above it count as 0

constexpr int kRing = 5, kAhead = kRing - 1;

struct Kv4TreeSmem {
    struct Slot {
        __align__(16) uint8_t k[4][kKv4Page * kKv4Row];  // a step's pages
        uint8_t v[4][kKv4Page * kKv4Row];
        uint8_t scales[4][2][kKv4Page * kKv4Scales];  // of keys and values
    } ring[kRing];
    __align__(16) uint16_t values[2][kTile * kKv4Dim];
    __align__(16) int held[kRing][4];  // is the page there (looked at where some are not)
    __align__(16) int flags[2][4];
    int tops[4];
    int pg[kMaxPages];
};
static_assert(sizeof(Kv4TreeSmem) <= 80 * 1024, "two workgroups to a CU");

// 16 bytes a lane, or 4, straight into LDS: lane l's to dst + 16 l, or + 4 l. Issued from assembly
// for the reasons that lds_ring.h gives.
__device__ __forceinline__ void global_to_lds16(const void* p, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
                 :
                 : "s"(lds), "v"(p)
                 : "memory");
}
__device__ __forceinline__ void global_to_lds4(const void* p, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off"
                 :
                 : "s"(lds), "v"(p)
                 : "memory");
}

typedef uint32_t u32x6 __attribute__((ext_vector_type(6)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x32 __attribute__((ext_vector_type(32)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

// 32 values over a power of two as E2M3, and back. Element 2 i of the codes is a[i], 2 i + 1 b[i].
// (The instructions write their results while they still read: the compiler does not keep the
// registers apart by itself.)
__device__ __forceinline__ u32x6 to_fp6(f32x16 a, f32x16 b, float scale) {
    u32x6 r;
    asm("v_cvt_scalef32_2xpk16_fp6_f32 %0, %1, %2, %3\n\ts_nop 4"
        : "=&v"(r)
        : "v"(a), "v"(b), "v"(scale));
    return r;
}
__device__ __forceinline__ f32x32 from_fp6(u32x6 c, float scale) {
    f32x32 r;
    asm("v_cvt_scalef32_pk32_f32_fp6 %0, %1, %2\n\ts_nop 4" : "=&v"(r) : "v"(c), "v"(scale));
    return r;
}

// acc += keys (codes and their scale byte) times part P of the queries.
template <int P>
__device__ __forceinline__ f32x4 mfma_fp4_fp6(uint4 k, int kscale, const u32x6& q, int qscales,
                                              f32x4 acc) {
    const i32x8 a = {(int)k.x, (int)k.y, (int)k.z, (int)k.w, 0, 0, 0, 0};
    const i32x8 b = {(int)q[0], (int)q[1], (int)q[2], (int)q[3], (int)q[4], (int)q[5], 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 4, 2, 0, kscale, P & 3,
                                                            qscales);
}

// The largest of 16 (fmaxf takes a second instruction for each, to quiet NaN that are not there).
__device__ __forceinline__ float max16(const f32x4 (&s)[4]) {
    float v = -INFINITY;
#pragma unroll
    for (int tt = 0; tt < 4; ++tt)
#pragma unroll
        for (int i = 0; i < 4; ++i) v = __builtin_amdgcn_fmed3f(v, s[tt][i], INFINITY);
    return v;
}

// Waits for the wave's accesses to LDS, not for its loads, and for the others.
__device__ __forceinline__ void lds_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

template <bool HALF>
__device__ __forceinline__ void kv4_tree_segment(const Kv4Attn& a, const Kv4Seqs& sq,
                                                 const Segment& g, Kv4TreeSmem& sm) {
    constexpr int QP = 5, PP = 2;  // parts of queries and of weights
    constexpr float kUnit = kQkScale * kLog2e;
    constexpr float kBits = HALF ? 12.0f : 15.0f, kMost = 15.0f;  // log2 of the weights: usual, most
    const int n = g.n, c = g.c, h = g.h, first = g.first, t0 = g.t0;
    const int row0 = g.tile * kRowsRT, t1 = min(t0 + g.len, c);
    int tid = threadIdx.x;
    // (opaque, so that what follows from it is not kept in registers from piece to piece)
    asm volatile("" : "+v"(tid));
    const int lane = tid & 63, col = lane & 15, j = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wrow = row0 + 32 * wave;  // the wave's first row
    const bool rows_here = a.token(wrow) < n;
    int* pg = sm.pg;
    const int32_t* table = sq.tables + (int64_t)g.seq * sq.table_stride + t0 / kKv4Page;
    const int pages = (t1 - t0 + kKv4Page - 1) / kKv4Page;
    // (whether there is one that the pool does not hold)
    auto stage_pages = [&](int from) {
        bool gone = false;
        for (int p = from + tid; p < min(pages, from + kMaxPages); p += 256) {
            const int id = table[p];
            gone = gone || id < 0 || id >= sq.n_blocks;
            pg[p - from] = id >= 0 && id < sq.n_blocks ? id : -1;
        }
        return __syncthreads_or(gone) != 0;
    };
    // the lane's rows and their queries' dims 32 j .. 32 j + 31 (rows that are not there read
    // another one's, whose results nobody writes), on their way with the page numbers
    float x[2][32];
#pragma unroll
    for (int ct = 0; ct < 2; ++ct) {
        const int r = min(wrow + 16 * ct + col, n * a.G - 1), i = a.token(r);
        const int64_t at = (int64_t)(first + i) * a.q_stride +
                           (int64_t)(h * a.G + (r - i * a.G)) * kKv4Dim + 32 * j;
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
            float v[4];
            ld_act4<HALF>(a.q, at + e, v);
#pragma unroll
            for (int k = 0; k < 4; ++k) x[ct][e + k] = v[k];
        }
    }
    if (tid < kRing * 4) sm.held[0][tid] = 1;
    bool gone = stage_pages(0);
    // Loads of the step at t: a wave has its page's codes and scales. Steps past the end load the last
    // page again, in place of a page that the pool does not hold another one is read, and masked.
    const bool any = sq.n_blocks > 0 && t1 > t0;
    const uint32_t ring0 = lds_addr(&sm.ring[0]);
    int w0 = t0;  // the first token of the page numbers in LDS
    auto load = [&](int page, int slot) {
        const int id = uniform(page);
        const int64_t row =
            (((int64_t)max(id, 0) * sq.n_layers + sq.layer) * sq.Hkv + h) * kKv4Page;
        const uint32_t dst = ring0 + slot * (uint32_t)sizeof(sm.ring[0]);
        global_to_lds16(a.pk + row * kKv4Row + lane * 16, dst + wave * 1024);
        global_to_lds16(a.pv + row * kKv4Row + lane * 16, dst + 4096 + wave * 1024);
        if (lane < 32)
            global_to_lds4((lane < 16 ? a.pks : a.pvs) + (row + col) * kKv4Scales,
                           dst + 8192 + wave * 128);
        if (gone && lane == 0) sm.held[slot][wave] = id >= 0;
    };
    if (any)
#pragma unroll
        for (int k = 0; k < kAhead; ++k) load(pg[min(4 * k + wave, pages - 1)], k);

    u32x6 qf[2][QP];
    int qs[2][(QP + 3) / 4];  // four parts' scale bytes
    float poison[2];  // NaN for a row with an infinity or NaN, which 6 bits do not hold, or 0
#pragma unroll
    for (int ct = 0; ct < 2; ++ct) {
        f32x16 even, odd;
        float amax = 0.0f, bad = 0.0f;
#pragma unroll
        for (int e = 0; e < 32; ++e) {
            bad += x[ct][e] * 0.0f;
            const float v = x[ct][e] * kUnit;
            amax = fmaxf(amax, fabsf(v));
            if (e & 1)
                odd[e >> 1] = v;
            else
                even[e >> 1] = v;
        }
        poison[ct] = sum_quarters(bad);
        const int e0 = (int)(__float_as_uint(amax) >> 23) - 1;  // of 2^(E - 1)
#pragma unroll
        for (int p = 0; p < QP; ++p) {
            const int e = max(e0 - 5 * p, 1);
            const float scale = __uint_as_float((uint32_t)e << 23);
            qf[ct][p] = to_fp6(even, odd, scale);
            if (p % 4 == 0) qs[ct][p / 4] = 0;
            qs[ct][p / 4] |= e << (8 * (p % 4));
            if (p + 1 < QP) {
                const f32x32 got = from_fp6(qf[ct][p], scale);
#pragma unroll
                for (int k = 0; k < 16; ++k) even[k] -= got[2 * k], odd[k] -= got[2 * k + 1];
            }
        }
    }

    f32x4 acc[2][8], sum[2];  // of weighted values, of weights (every element the same)
    float m[2];
#pragma unroll
    for (int ct = 0; ct < 2; ++ct) {
        m[ct] = -INFINITY;
        sum[ct] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
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
    // the wave's share of the values: a lane's 32 dims of token 16 wave + col
    uint4 vr = {};
    auto store = [&](uint16_t* dst, int byte) {
        const float sc = byte_scale(byte);
        const uint32_t w[4] = {vr.x, vr.y, vr.z, vr.w};
#pragma unroll
        for (int st = 0; st < 4; ++st)
            *reinterpret_cast<uint4*>(dst + wave * 16 * kKv4Dim + wr[st]) =
                fp4_to_half8(w[st], sc);
    };
    // The values of the step at t into their half of LDS. What fp16 does not hold as it is waits for the
    // step's turn (the values then go in again).
    int vby = 0;
    bool skip = false;
    auto convert = [&](int t, int slot, int half) {
        const auto& from = sm.ring[slot];
        vr = *reinterpret_cast<const uint4*>(from.v[wave] + col * kKv4Row + j * 16);
        const int vs = from.scales[wave][1][col * kKv4Scales + j];
        int flag = 0;
        vby = vs;
        skip = false;
        if (gone || t + kTile > t1) {
            skip = (gone && !sm.held[slot][wave]) || t + 16 * wave + col >= t1;  // no one's token
            if (skip) vby = 127 + vshift;
        }
        if (__ballot(!in_range(vby - vshift))) {
            if (vby > kHardScale || no_codes(vr)) vby = 0;
            flag = __ballot(vby > 0 && vby - vshift < kLowScale) ? 3 : 1;
        }
        if (!skip) vtop = max(vtop, vby);
        store(sm.values[half], vby - vshift);
        if (lane == 0) sm.flags[half][wave] = flag;
    };
    constexpr int kOut = 3 * (kAhead - 1);  // loads of a wave that stay under way
    if (any) {
        wait_vm_asm<kOut>();
        convert(t0, 0, 0);
    }
    int slot = 0;
    for (int t = t0, half = 0; t < t1 && any; t += kTile, half ^= 1) {
        wait_vm_asm<kOut>();
        lds_barrier();  // everyone's keys of this step are there, and values as fp16
        const int* fl = sm.flags[half];
        const int flag = __builtin_amdgcn_readfirstlane(fl[0] | fl[1] | fl[2] | fl[3]);
        uint16_t* vt = sm.values[half];
        if (flag) {
            // the values' power of two for the largest scale so far, and the step once more
            const int mine = (int)wave_max((float)vtop);
            if (lane == 0) sm.tops[wave] = mine;
            __syncthreads();
            vtop = max(max(sm.tops[0], sm.tops[1]), max(sm.tops[2], sm.tops[3]));
            const int shift = vtop - kTopScale;
            if (vtop - vshift > kTopScale || (flag > 1 && vtop - vshift < kTopScale)) {
                const float f = pow2(vshift - shift);
#pragma unroll
                for (int ct = 0; ct < 2; ++ct)
#pragma unroll
                    for (int d = 0; d < 8; ++d) acc[ct][d] *= f;
                if (skip) vby += shift - vshift;
                vshift = shift;
                store(vt, vby - vshift);
            }
            __syncthreads();
        }
        // the loads of kAhead steps later, into the slot of the step before
        const int later = t + kAhead * kTile;
        if (later < t1 && later >= w0 + kMaxPages * kKv4Page) {  // (kMaxPages numbers at a time)
            w0 = later;
            gone = stage_pages((w0 - t0) / kKv4Page) || gone;
        }
        const int page = pg[min(((later - w0) >> 4) + wave, pages - 1 - ((w0 - t0) >> 4))];
        const int before = slot == 0 ? kRing - 1 : slot - 1;
        const int after = slot == kRing - 1 ? 0 : slot + 1;
        if (rows_here) {
            f32x4 s[2][4];
            const auto& from = sm.ring[slot];
            uint4 kr[4];  // a token of each page a lane
            int ks[4];
#pragma unroll
            for (int tt = 0; tt < 4; ++tt) {
                kr[tt] = *reinterpret_cast<const uint4*>(from.k[tt] + col * kKv4Row + j * 16);
                ks[tt] = from.scales[tt][0][col * kKv4Scales + j];
                if (ks[tt] > kHardScale) ks[tt] = 0;
            }
#pragma unroll
            for (int ct = 0; ct < 2; ++ct) {
                const float b = m[ct] == -INFINITY ? kBits : kBits - m[ct];
#pragma unroll
                for (int tt = 0; tt < 4; ++tt) s[ct][tt] = f32x4{b, b, b, b};
            }
            // (neighbouring products add to different sums)
            auto part = [&](auto number) {
                constexpr int P = decltype(number)::value;
#pragma unroll
                for (int tt = 0; tt < 4; ++tt)
#pragma unroll
                    for (int ct = 0; ct < 2; ++ct)
                        s[ct][tt] = mfma_fp4_fp6<P>(kr[tt], ks[tt], qf[ct][P], qs[ct][P / 4],
                                                    s[ct][tt]);
            };
            // (the small parts first)
            part(std::integral_constant<int, 4>{});
            part(std::integral_constant<int, 3>{});
            part(std::integral_constant<int, 2>{});
            load(page, before);
            part(std::integral_constant<int, 1>{});
            part(std::integral_constant<int, 0>{});
            // the tree's own tokens, and pages that are not there
            if (gone || t + kTile > c - n) {
                const int* hd = sm.held[slot];
#pragma unroll
                for (int ct = 0; ct < 2; ++ct) {
                    const int i = a.token(wrow + 16 * ct + col);
                    const uint64_t bits =
                        i < n && c - n + i >= 0
                            ? seen64(a, (int64_t)first + i, t, c - n, c) >> (4 * j)
                            : 0;
#pragma unroll
                    for (int tt = 0; tt < 4; ++tt)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (!hd[tt] || !(bits >> (16 * tt + i) & 1))
                                s[ct][tt][i] = -INFINITY;
                }
            }
            float top[2];
            bool over = false;
#pragma unroll
            for (int ct = 0; ct < 2; ++ct) {
                top[ct] = max_quarters(max16(s[ct]));
                over = over || top[ct] > (m[ct] == -INFINITY ? -INFINITY : kMost);
            }
            if (__ballot(over)) {
#pragma unroll
                for (int ct = 0; ct < 2; ++ct) {
                    // rows beyond the limit have their maximum there again
                    const bool up = top[ct] > (m[ct] == -INFINITY ? -INFINITY : kMost);
                    const float by = up ? top[ct] - kBits : 0.0f;
                    const float f = m[ct] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(-by);
                    if (up) m[ct] = (m[ct] == -INFINITY ? 0.0f : m[ct]) + by;
#pragma unroll
                    for (int d = 0; d < 8; ++d) acc[ct][d] *= f;
                    sum[ct] *= f;
#pragma unroll
                    for (int tt = 0; tt < 4; ++tt) s[ct][tt] -= by;
                }
            }
            __builtin_amdgcn_s_setprio(1);
            // (the weights of the second 32 tokens between the products of the first)
            Frag16 ones;
#pragma unroll
            for (int k = 0; k < 4; ++k) ones.w[k] = 0x3c003c00u;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                Frag16 pf[2][PP];  // [column tile][part]
#pragma unroll
                for (int ct = 0; ct < 2; ++ct)
#pragma unroll
                    for (int e = 0; e < 8; e += 2) {
                        const f32x4& w = s[ct][2 * u + (e >> 2)];
                        const float p0 = __builtin_amdgcn_exp2f(w[e & 3]);
                        const float p1 = __builtin_amdgcn_exp2f(w[(e & 3) + 1]);
                        const uint32_t hi = pack16(p0, p1);
                        pf[ct][0].w[e >> 1] = hi;
                        pf[ct][1].w[e >> 1] = pack16(rest_lo(p0, hi), rest_hi(p1, hi));
                    }
#pragma unroll
                for (int p = 0; p < PP; ++p)
#pragma unroll
                    for (int ct = 0; ct < 2; ++ct)
                        sum[ct] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones.v, pf[ct][p].v,
                                                                         sum[ct], 0, 0, 0);
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
                    for (int p = 0; p < PP; ++p)
#pragma unroll
                        for (int d = 0; d < 4; ++d)
#pragma unroll
                            for (int ct = 0; ct < 2; ++ct)
                                acc[ct][d0 + d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                                    vf[d].v, pf[ct][p].v, acc[ct][d0 + d], 0, 0, 0);
                }
            }
            __builtin_amdgcn_s_setprio(0);
        } else {
            load(page, before);
        }
        wait_vm_asm<kOut>();
        if (t + kTile < t1) convert(t + kTile, after, half ^ 1);
        slot = after;
    }
    wait_vm_asm<0>();  // the loads past the end still write the ring
#pragma unroll
    for (int ct = 0; ct < 2; ++ct) {
        float L = sum[ct][0];
        const int r = wrow + 16 * ct + col, i = a.token(r);
        if (i >= n) continue;
        if (m[ct] != -INFINITY) L += poison[ct];
        // (by the sum of weights, and the 2^kBits in both, before the values' power of two)
        const auto times = [](f32x4 v, int e) {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = __builtin_ldexpf(v[i], e);
            return v;
        };
        if (g.whole) {
            if (vshift != 0 && L != 0.0f) {
#pragma unroll
                for (int d = 0; d < 8; ++d) acc[ct][d] = times(acc[ct][d] * (1.0f / L), vshift);
                L = 1.0f;
            }
#pragma unroll
            for (int d = 0; d < 8; ++d)
                store4<HALF>(a, ((int64_t)first + i) * a.out_stride +
                                    (int64_t)(h * a.G + (r - i * a.G)) * kKv4Dim + 16 * d + 4 * j,
                             acc[ct][d], L);
        } else {
            const int64_t at = g.rec + 32 * wave + 16 * ct + col;
            const int e = vshift - (int)kBits;
#pragma unroll
            for (int d = 0; d < 8; ++d)
                *reinterpret_cast<f32x4*>(a.part_o + at * kKv4Dim + 16 * d + 4 * j) =
                    times(acc[ct][d], e);
            if (j == 0)
                a.part_ml[at] = make_float2(m[ct], __builtin_ldexpf(L, -(int)kBits));
        }
    }
    lds_barrier();
}
