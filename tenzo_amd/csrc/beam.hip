// Beam search on the device: the best k continuations of a request's W beams over the
// vocabulary, and the reordering of the beams' paged caches.
//
// Selection: candidate (w, t) has the score s_w + x_wt - log sum_u exp(x_wu); the k largest are
// taken, among equal ones the lower beam, then the larger logit, then the lower token. So a beam's
// candidates come in the order of (logit, token) and the first k of each beam hold the answer. A
// logit that is not below +inf (NaN, +inf) counts as -inf. Two beams' candidates can lie closer
// than exponentials in fp32 tell apart; where they do, the log-sums are taken anew in 64 bits.
#include <climits>

#include "common.h"

namespace tz {
namespace {

constexpr int kBeamMax = 64;      // beams and candidates, upper bounds
constexpr int kSliceCand = 1024;  // a slice's candidates in LDS
constexpr int kSliceFew = 256;    // logits above -inf that are put in order as they are
constexpr int kPickCand = 512;    // the candidates that the last step ranks

// A row's log-sum from fp32 exponentials is nearer than this to the true one. x - max and its
// product with log2 e are rounded to 2^-24 of themselves each, in base 2 at most 8.1 of them on a
// slice's average (5 of 6 parts of the weight at 4095 logits 9.7 below one), 6.7e-7; log2 e
// itself 7e-8, the exponential's step 1.2e-7, eight of them added in fp32 1.8e-7. (Seen: 2.8e-7.)
constexpr double kLogSumError = 1.25e-6;

// Up to here a slice's bound is the best of its waves' own, above it that of their merged order:
// 19 x 16 beams over 154773 logits, 32 candidates, 58 us merged and 70 not, 8 beams over 128256,
// 64 candidates, 15 and 67; 48 x 8 beams over 128256, 16 candidates, 55.6 and 54.2.
constexpr int kWaveBound = 16;

struct BeamSelect {
    const float* logits;
    const float* scores;
    int64_t stride;
    int W, k, V;
    int ns;         // slices of a row
    double2* sums;  // [B * W][ns]: a slice's maximum and its sum of exponentials below it
    float2* cand;   // [B * W][ns][k]: its best logits, in order: value, token (INT_MAX: none)
    float* out_scores;
    int32_t* out_beams;
    int32_t* out_tokens;
};

// NaN and +inf count as -inf; -0 as 0.
__device__ __forceinline__ float beam_logit(float x) {
    return (x < INFINITY ? x : -INFINITY) + 0.0f;
}

// Bits in the order of the values.
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t b = __float_as_uint(x);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float from_ordered(uint32_t o) {
    return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}

// The value of lane l ^ M.
template <int M>
__device__ __forceinline__ float lane_xor(float v) {
    if constexpr (M >= 32) {
        float lo, hi;
        lane_halves(lane_xor<M - 32>(v), lo, hi);
        return threadIdx.x & 32 ? lo : hi;
    } else if constexpr (M >= 16) {
        float lo, hi;
        lane_pairs16(lane_xor<M - 16>(v), lo, hi);
        return threadIdx.x & 16 ? lo : hi;
    } else if constexpr (M == 15) {
        return dpp_f<kDppMirror>(v);
    } else if constexpr (M == 8) {
        return dpp_f<0x128>(v);  // row_ror:8
    } else if constexpr (M == 7) {
        return dpp_f<kDppHalfMirror>(v);
    } else if constexpr (M == 4) {
        return dpp_f<0x1B>(dpp_f<kDppHalfMirror>(v));
    } else if constexpr (M == 3) {
        return dpp_f<0x1B>(v);  // quad_perm [3,2,1,0]
    } else if constexpr (M == 2) {
        return dpp_f<kDppXor2>(v);
    } else if constexpr (M == 1) {
        return dpp_f<kDppXor1>(v);
    } else {
        static_assert(M == 0, "no such exchange");
        return v;
    }
}

template <int M>
__device__ __forceinline__ double lane_xor(double v) {
    const uint64_t b = __double_as_longlong(v);
    const uint32_t lo = __float_as_uint(lane_xor<M>(__uint_as_float((uint32_t)b)));
    const uint32_t hi = __float_as_uint(lane_xor<M>(__uint_as_float((uint32_t)(b >> 32))));
    return __longlong_as_double((uint64_t)hi << 32 | lo);
}
// Over the 64 lanes, in all of them.
__device__ __forceinline__ double lanes_sum(double v) {
    v += lane_xor<32>(v);
    v += lane_xor<16>(v);
    v += lane_xor<8>(v);
    v += lane_xor<4>(v);
    v += lane_xor<2>(v);
    return v + lane_xor<1>(v);
}
__device__ __forceinline__ double lanes_max(double v) {
    v = fmax(v, lane_xor<32>(v));
    v = fmax(v, lane_xor<16>(v));
    v = fmax(v, lane_xor<8>(v));
    v = fmax(v, lane_xor<4>(v));
    v = fmax(v, lane_xor<2>(v));
    return fmax(v, lane_xor<1>(v));
}

// exp(x) of x up to 0, within 2^-50: x log2 e = n + f, and 2^f by the polynomial of degree 10
// through its values at the Chebyshev nodes of [-1/2, 1/2] (4.5e-16 of it). 128256 of them by a
// workgroup take 8 us less than the library's, which takes any x.
__device__ __forceinline__ double exp64(double x) {
    constexpr double kC[] = {
        0x1.e6063f7217bc6p-28, 0x1.b675bca4eeebbp-24, 0x1.62bfd47773353p-20, 0x1.ffcb54062e698p-17,
        0x1.430913096fd9fp-13, 0x1.5d87fe9d7a584p-10, 0x1.3b2ab6fba1ddap-7, 0x1.c6b08d703ce49p-5,
        0x1.ebfbdff82c598p-3, 0x1.62e42fefa3a19p-1, 0x1.0000000000000p+0};
    constexpr double kLog2e = 0x1.71547652b82fep0, kRound = 0x1.8p52;  // (a sum's low word is n)
    x = fmax(x, -1000.0);  // (0 from there on)
    const double t = __builtin_fma(x, kLog2e, kRound);
    const double f = __builtin_fma(x, kLog2e, kRound - t);
    double p = kC[0];
#pragma unroll
    for (int i = 1; i <= 10; ++i) p = __builtin_fma(p, f, kC[i]);
    return __builtin_ldexp(p, __double2loint(t));
}

// One step of a descending bitonic sort over the 64 lanes: lane l and l ^ M, the one without
// the mask's top bit keeps the larger.
template <int M>
__device__ __forceinline__ float sort_step(float v) {
    constexpr int top = M >= 32 ? 32 : M >= 16 ? 16 : M >= 8 ? 8 : M >= 4 ? 4 : M >= 2 ? 2 : 1;
    const float o = lane_xor<M>(v);
    return threadIdx.x & top ? fminf(v, o) : fmaxf(v, o);
}
__device__ __forceinline__ float sort64_desc(float v) {
    v = sort_step<1>(v);
    v = sort_step<1>(sort_step<3>(v));
    v = sort_step<1>(sort_step<2>(sort_step<7>(v)));
    v = sort_step<1>(sort_step<2>(sort_step<4>(sort_step<15>(v))));
    v = sort_step<1>(sort_step<2>(sort_step<4>(sort_step<8>(sort_step<31>(v)))));
    return sort_step<1>(
        sort_step<2>(sort_step<4>(sort_step<8>(sort_step<16>(sort_step<63>(v))))));
}

// The 64 largest of two descending lists, a value a lane, in order.
__device__ __forceinline__ float merge64(float v, float reversed) {
    v = sort_step<32>(fmaxf(v, reversed));
    return sort_step<1>(sort_step<2>(sort_step<4>(sort_step<8>(sort_step<16>(v)))));
}

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

// Stage 1, a workgroup per slice of 256 * E logits of a row, held in registers: the slice's
// maximum and sum of exponentials, and its k best logits in order. The k-th largest of 64 lanes'
// maxima (a wave's, or of the waves' merged order) is a bound that at least k of the slice reach;
// the list of those that do is short (about 2k of 4096 ordinary logits) and put in order by
// counting. Where too many reach it (equal logits, masked vocabularies: -inf is no bound) and
// more than 256 are above -inf the k-th largest is found bit by bit instead, and among its equals
// the lowest tokens. Bound by reading the logits, 8 waves a SIMD (64 registers) keep the loads
// coming: 48 x 8 beams over 128256 logits 45 us, 4.4 TB/s.
template <int E>
__global__ void __launch_bounds__(256, 8) beam_slice_kernel(BeamSelect a) {
    __shared__ uint64_t list[kSliceCand];
    __shared__ float tops[4][64];
    __shared__ double part[4];
    __shared__ int cnt, red[4];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int row = blockIdx.x / a.ns, slice = blockIdx.x - row * a.ns;
    const int base = slice * (256 * E) + tid * 4;  // element i, c: token base + 1024 i + c
    const float* x = a.logits + row * a.stride;
    float v[E];
    if (slice * (256 * E) + 256 * E <= a.V) {
#pragma unroll
        for (int i = 0; i < E / 4; ++i) {
            const f32x4u q = __builtin_nontemporal_load(
                reinterpret_cast<const f32x4u*>(x + base + 1024 * i));
#pragma unroll
            for (int c = 0; c < 4; ++c) v[4 * i + c] = q[c];
        }
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const int t = base + 1024 * (i / 4) + i % 4;
            v[i] = t < a.V ? x[t] : -INFINITY;
        }
    }
    if (tid == 0) cnt = 0;
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        v[i] = beam_logit(v[i]);
        top = fmaxf(top, v[i]);
    }
    tops[wave][lane] = sort64_desc(top);
    __syncthreads();
    const float M = fmaxf(fmaxf(tops[0][0], tops[1][0]), fmaxf(tops[2][0], tops[3][0]));
    float tau;
    if (a.k > kWaveBound) {
        const float lo = merge64(tops[0][lane], tops[1][63 - lane]);
        const float hi = merge64(tops[2][lane], tops[3][63 - lane]);
        tau = lane_f(merge64(lo, lane_xor<63>(hi)), a.k - 1);
    } else {
        tau = fmaxf(fmaxf(tops[0][a.k - 1], tops[1][a.k - 1]),
                    fmaxf(tops[2][a.k - 1], tops[3][a.k - 1]));
    }
    const float ref = M == -INFINITY ? 0.0f : M;

    // few terms are added in 32 bits, their sums in 64 (with exponentials in 64 bits, to 2e-9, the
    // selection of 48 x 8 beams takes 66 us in place of 53)
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < E; i += 8) {
        float e[8];
#pragma unroll
        for (int c = 0; c < 8; ++c)
            e[c] = __builtin_amdgcn_exp2f((v[i + c] - ref) * 1.4426950408889634f);
        sum += (double)(((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7])));
    }
    sum = lanes_sum(sum);
    if (lane == 0) part[wave] = sum;

    const auto token = [&](int i) { return base + 1024 * (i / 4) + i % 4; };
    const auto key = [&](int i) {
        return (uint64_t)ordered(v[i]) << 32 | (uint32_t)(INT_MAX - token(i));
    };
    if (tau > -INFINITY && top >= tau) {
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (v[i] >= tau) {
                const int at = atomicAdd(&cnt, 1);
                if (at < kSliceCand) list[at] = key(i);
            }
    }
    __syncthreads();
    int n = cnt;
    if (tau == -INFINITY || n > kSliceCand) {
        // sum of a count over the workgroup
        const auto total = [&](int c) {
            c = wave_sum_i32(c);
            __syncthreads();
            if (lane == 0) red[wave] = c;
            __syncthreads();
            return (red[0] + red[1]) + (red[2] + red[3]);
        };
        int mine = 0, real = 0;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            mine += token(i) < a.V ? 1 : 0;
            real += v[i] > -INFINITY ? 1 : 0;
        }
        const int want = min(a.k, total(mine));
        uint32_t bar = ordered(-INFINITY);
        real = total(real);
        // the want-th largest value, from its highest bit on; a few are listed all
        if (real >= want && real > kSliceFew) {
            bar = 0;
            for (int bit = 31; bit >= 0; --bit) {
                const uint32_t up = bar | 1u << bit;
                int c = 0;
#pragma unroll
                for (int i = 0; i < E; ++i) c += ordered(v[i]) >= up && token(i) < a.V ? 1 : 0;
                if (total(c) >= want) bar = up;
            }
        }
        const float least = from_ordered(bar);
        int c = 0;
#pragma unroll
        for (int i = 0; i < E; ++i) c += v[i] > least ? 1 : 0;
        const int need = want - total(c);
        // its equals below token `until` are the ones needed
        const int from = slice * (256 * E);
        int until = from;
        if (need > 0) {
            int below = 0;
            for (int step = 256 * E; step > 0; step >>= 1) {
                c = 0;
#pragma unroll
                for (int i = 0; i < E; ++i)
                    c += v[i] == least && token(i) < a.V && token(i) < from + below + step ? 1 : 0;
                if (total(c) < need) below += step;
            }
            until = from + below + 1;
        }
        __syncthreads();
        if (tid == 0) cnt = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (v[i] > least || (v[i] == least && token(i) < a.V && token(i) < until))
                list[atomicAdd(&cnt, 1) & (kSliceCand - 1)] = key(i);
        __syncthreads();
        n = cnt;
    }
    const int64_t at = (int64_t)row * a.ns + slice;
    if (tid == 0) a.sums[at] = make_double2(M, (part[0] + part[1]) + (part[2] + part[3]));
    for (int i = tid; i < n; i += 256) {
        const uint64_t me = list[i];
        int rank = 0;
        for (int o = 0; o < n; ++o) rank += list[o] > me ? 1 : 0;
        if (rank < a.k)
            a.cand[at * a.k + rank] = make_float2(
                from_ordered((uint32_t)(me >> 32)), __int_as_float(INT_MAX - (int)(uint32_t)me));
    }
    if (tid >= n && tid < a.k)
        a.cand[at * a.k + tid] = make_float2(-INFINITY, __int_as_float(INT_MAX));
}

struct BeamCand {
    double s;
    float x;
    int w, t;
};
__device__ __forceinline__ bool before(const BeamCand& a, const BeamCand& b) {
    if (a.s != b.s) return a.s > b.s;
    if (a.w != b.w) return a.w < b.w;
    if (a.x != b.x) return a.x > b.x;
    return a.t < b.t;
}

// Stage 2, a workgroup per request: the rows' log-sums, then the best k of the slices' lists. The
// first few of every list (2k of a beam's or more, up to 1024 in all) are put in order (sorted by
// waves, merged in pairs), and their k-th (in fp32, rounded down), less what the log-sums may be
// off by, is a bound that the k best reach. Those that do are ranked by counting; where they are
// many (equal scores, masked beams or tokens) the k best are taken one after the other. Where one
// of the k best has another beam's candidate so near that the log-sums leave their order open, the
// beams' are summed in 64 bits from the logits (27 us a beam of 128256) and all are ranked once
// more. 48 x 8 beams, 32 slices, 16 candidates: 8.5 us, latency from end to end.
__global__ void __launch_bounds__(1024) beam_pick_kernel(BeamSelect a) {
    __shared__ double lse[kBeamMax], own[kBeamMax], peak[kBeamMax], part[16];
    __shared__ double ls[kPickCand];
    __shared__ uint32_t near[2];  // beams whose log-sums are needed in 64 bits
    __shared__ float lx[kPickCand], tops[16][64];
    __shared__ int lw[kPickCand], lt[kPickCand], lr[kPickCand], open[kPickCand], cnt, opened;
    __shared__ BeamCand best[16];
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int per = a.ns * a.k, total = a.W * per, lists = a.W * a.ns;
    const float2* cand = a.cand + (int64_t)b * total;
    const int depth = max(1, min(min(a.k, 1024 / lists), (2 * a.k + a.ns - 1) / a.ns));
    const int heads = lists * depth, first = min(tid, heads - 1) / depth * a.k + tid % depth;
    // (loads whose places are clamped, none under a condition, where it would be waited for)
    const float2 head = cand[first];
    constexpr int kOwn = 4;  // a thread's candidates where they are few, loaded during the log-sums
    const bool few = total <= 1024 * kOwn;
    float2 mine[kOwn];
#pragma unroll
    for (int i = 0; i < kOwn; ++i) mine[i] = cand[min(tid + 1024 * i, total - 1)];
    for (int w = wave; w < a.W; w += 16) {
        const double2* sums = a.sums + ((int64_t)b * a.W + w) * a.ns;
        const float score = a.scores[b * a.W + w];
        double2 e = sums[min(lane, a.ns - 1)];
        if (lane >= a.ns) e.x = -INFINITY;
        double m = e.x;
        for (int i = lane + 64; i < a.ns; i += 64) m = fmax(m, sums[i].x);
        m = lanes_max(m);
        double s = e.x > -INFINITY ? e.y * exp(e.x - m) : 0.0;
        for (int i = lane + 64; i < a.ns; i += 64)
            if (sums[i].x > -INFINITY) s += sums[i].y * exp(sums[i].x - m);
        s = lanes_sum(s);
        if (lane == 0) {
            lse[w] = m > -INFINITY ? m + log(s) : 0.0;
            peak[w] = m;
            own[w] = beam_logit(score);
        }
    }
    if (tid == 0) cnt = opened = near[0] = near[1] = 0;
    __syncthreads();
    const auto get = [&](int c, float2 e) {
        BeamCand r;
        r.w = c / per;
        r.x = e.x;
        r.t = __float_as_int(e.y);
        r.s = e.x > -INFINITY ? ((double)e.x - lse[r.w]) + own[r.w] : -INFINITY;
        return r;
    };
    float top = -INFINITY;
    if (tid < heads) top = __double2float_rd(get(first, head).s);
    for (int i = tid + 1024; i < lists; i += 1024)
        top = fmaxf(top, __double2float_rd(get(i * a.k, cand[i * a.k]).s));
    float sorted = sort64_desc(top);
    tops[wave][lane] = sorted;
    __syncthreads();
    for (int half = heads > 512 ? 8 : heads > 128 ? 4 : 1; half > 0; half >>= 1) {
        if (wave < half) {
            sorted = merge64(sorted, tops[wave + half][63 - lane]);
            tops[wave][lane] = sorted;
        }
        __syncthreads();
    }
    const double bound = (double)tops[0][a.k - 1] - 2 * kLogSumError;
    const auto keep = [&](const BeamCand& c) {
        if (c.t == INT_MAX || c.s < bound) return;
        const int at = atomicAdd(&cnt, 1);
        if (at < kPickCand) ls[at] = c.s, lx[at] = c.x, lw[at] = c.w, lt[at] = c.t;
    };
#pragma unroll
    for (int i = 0; i < kOwn; ++i)
        if (few && tid + 1024 * i < total) keep(get(tid + 1024 * i, mine[i]));
    if (!few) {  // only the lists whose first candidate reaches the bound
        for (int i = tid; i < lists; i += 1024)
            if (get(i * a.k, cand[i * a.k]).s >= bound) {
                const int at = atomicAdd(&opened, 1);
                if (at < kPickCand) open[at] = i * a.k;
            }
        __syncthreads();
        for (int e = tid; e < min(opened, kPickCand) * a.k; e += 1024) {
            const int c = open[e / a.k] + e % a.k;
            keep(get(c, cand[c]));
        }
    }
    __syncthreads();
    // a beam's log-sum in 64 bits (a beam without candidates: nothing to do)
    const auto sum_exactly = [&](int w) {
        const double m = peak[w];
        if (m == -INFINITY || own[w] == -INFINITY) return;
        const float* x = a.logits + ((int64_t)b * a.W + w) * a.stride;
        double s = 0.0;
        float v[8], next[8];  // (the next ones are loaded during the sums)
        const auto load = [&](int t0) {
#pragma unroll
            for (int i = 0; i < 8; ++i) next[i] = x[min(t0 + 1024 * i, a.V - 1)];
        };
        load(tid);
        for (int t0 = tid; t0 < a.V; t0 += 8 * 1024) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = t0 + 1024 * i < a.V ? next[i] : -INFINITY;
            load(t0 + 8 * 1024);
#pragma unroll
            for (int i = 0; i < 8; ++i) s += exp64((double)beam_logit(v[i]) - m);
        }
        s = lanes_sum(s);
        if (lane == 0) part[wave] = s;
        __syncthreads();
        if (tid == 0) {
            s = 0.0;
            for (int i = 0; i < 16; ++i) s += part[i];
            lse[w] = m + log(s);
        }
        __syncthreads();
    };
    const auto sum_near = [&]() {
        for (int w = 0; w < a.W; ++w)
            if (near[w >> 5] >> (w & 31) & 1) sum_exactly(w);
    };
    const int n = cnt;
    if (n <= kPickCand && opened <= kPickCand) {
        for (bool first = a.W > 1;; first = false) {
            // four lanes to a candidate; equal scores are rare and looked at in full
            const int q = tid & 3;
            for (int i0 = 0; i0 < n; i0 += 256) {
                const int i = i0 + (tid >> 2);
                const double me = ls[min(i, n - 1)];
                int rank = 0;
                uint64_t beams = 0;  // that have a candidate next to this one
                for (int o = q; o < n; o += 4) {
                    rank += ls[o] > me ? 1 : 0;
                    if (fabs(ls[o] - me) <= 2 * kLogSumError && i < n) {
                        if (lw[o] != lw[i]) beams |= 1ull << lw[o] | 1ull << lw[i];
                    }
                    if (ls[o] == me && i < n &&
                        before(BeamCand{me, lx[o], lw[o], lt[o]},
                               BeamCand{me, lx[i], lw[i], lt[i]}))
                        ++rank;
                }
                rank += dpp_i<kDppXor1>(rank);
                rank += dpp_i<kDppXor2>(rank);
                if (i < n && q == 0) lr[i] = rank;
                if (first && beams && rank < a.k) {
                    atomicOr(&near[0], (uint32_t)beams);
                    atomicOr(&near[1], (uint32_t)(beams >> 32));
                }
            }
            __syncthreads();
            if (!first || !(near[0] | near[1])) break;
            sum_near();
            for (int i = tid; i < n; i += 1024)
                if (ls[i] > -INFINITY) ls[i] = ((double)lx[i] - lse[lw[i]]) + own[lw[i]];
            __syncthreads();
        }
        for (int i = tid; i < n; i += 1024)
            if (lr[i] < a.k) {
                a.out_scores[b * a.k + lr[i]] = (float)ls[i];
                a.out_beams[b * a.k + lr[i]] = lw[i];
                a.out_tokens[b * a.k + lr[i]] = lt[i];
            }
        return;
    }
    const BeamCand none{-INFINITY, -INFINITY, INT_MAX, INT_MAX};
    for (bool first = a.W > 1;; first = false) {
        BeamCand last{INFINITY, INFINITY, -1, -1};
        uint64_t beams = 0;
        // (once more than k times where the last one's neighbours are looked for)
        for (int j = 0; j < a.k + (first ? 1 : 0); ++j) {
            BeamCand m = none;
            for (int c = tid; c < total; c += 1024) {
                const BeamCand e = get(c, cand[c]);
                if (e.t == INT_MAX) continue;
                if (first && j > 0 && e.w != last.w && fabs(e.s - last.s) <= 2 * kLogSumError)
                    beams |= 1ull << e.w | 1ull << last.w;
                if (before(last, e) && before(e, m)) m = e;
            }
            if (j == a.k) break;
            for (int d = 32; d > 0; d >>= 1) {
                const BeamCand o{__shfl_xor(m.s, d), __shfl_xor(m.x, d), __shfl_xor(m.w, d),
                                 __shfl_xor(m.t, d)};
                if (before(o, m)) m = o;
            }
            if (lane == 0) best[wave] = m;
            __syncthreads();
            m = best[0];
            for (int w = 1; w < 16; ++w)
                if (before(best[w], m)) m = best[w];
            __syncthreads();
            last = m;
            if (tid == 0) {
                a.out_scores[b * a.k + j] = (float)m.s;
                a.out_beams[b * a.k + j] = m.w;
                a.out_tokens[b * a.k + j] = m.t;
            }
        }
        if (!first) return;
        if (beams) {
            atomicOr(&near[0], (uint32_t)beams);
            atomicOr(&near[1], (uint32_t)(beams >> 32));
        }
        __syncthreads();
        if (!(near[0] | near[1])) return;
        sum_near();
    }
}

// Logits a thread of stage 1 holds: 8 where 16 would leave fewer than four workgroups a CU. 8 x
// 128256 logits 13.2 us with 8 and 14.7 with 16, 192 x 32089 23.3 and 20.8, 384 x 128256 74 and 54.
int beam_elems(int64_t rows, int64_t V) {
    return rows * ceil_div(V, 256 * 16) >= 1024 ? 16 : 8;
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
    int copiers;  // workgroups that copy a request's pieces
};

constexpr int kPageTokens = 16;

// One piece of the page in progress (bytes `at` of pages of `size`), for all slots of a request:
// every parent's is read before the first is written, so no slot's is lost whatever the
// permutation, and no two threads touch the same piece. Lane i of `from` and `to` has slot i's
// pages, from -1 where it stays.
template <int WMAX, typename P>
__device__ __forceinline__ void move_piece(int from, int to, uint8_t* pool, int64_t size,
                                           int64_t at) {
    P v[WMAX];
#pragma unroll
    for (int i = 0; i < WMAX; ++i) {
        const int page = __builtin_amdgcn_readlane(from, i);
        v[i] = P{};
        if (page >= 0) v[i] = *reinterpret_cast<const P*>(pool + page * size + at);
    }
#pragma unroll
    for (int i = 0; i < WMAX; ++i)
        if (__builtin_amdgcn_readlane(from, i) >= 0)
            *reinterpret_cast<P*>(pool + __builtin_amdgcn_readlane(to, i) * size + at) = v[i];
}

// In place: slot i of a request takes the cached tokens of slot parents[i]. The pages that are
// full change hands through the table (a thread a column, all slots read before one is written);
// the rows of the page in progress are copied into the slot's own page, in pieces of 16 bytes of
// codes and 4 of scales. A page's planes lie side by side, so a request's moves are a few long
// copies; each of its a.copiers workgroups takes pieces in turn (the page numbers, a chain of
// three loads, are found once for all of them). 48 x 8 beams, 150 planes, 14 rows: 43 us, 4.1 TB/s
// read and written (a workgroup for every 256 pieces, each finding its pages: 86).
template <int WMAX>
__global__ void __launch_bounds__(256) beam_reorder_kernel(BeamReorder a) {
    const int b = blockIdx.y;
    const int c = a.ctx[(int64_t)b * a.W];
    if (c <= 0 || c > a.width * kPageTokens) return;
    const int full = c / kPageTokens, fill = c % kPageTokens;
    const int32_t* parents = a.parents + b * a.parent_stride;
    int32_t* table = a.tables + (int64_t)b * a.W * a.table_stride;
    if ((int)blockIdx.x >= a.copiers) {
        const int col = ((int)blockIdx.x - a.copiers) * 256 + threadIdx.x;
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
    const int slot = threadIdx.x & 63;
    int from = -1, to = -1;
    if (slot < a.W) {
        const int par = parents[slot];
        const bool other = par >= 0 && par < a.W && par != slot;
        from = table[(other ? par : slot) * a.table_stride + full];
        to = table[slot * a.table_stride + full];
        if (!other || from >= a.n_blocks || to < 0 || to >= a.n_blocks) from = -1;
    }
    const int step = a.copiers * 256, first = blockIdx.x * 256 + threadIdx.x;
    // codes: row_bytes pieces a plane, token by token
    const int pieces = (int)a.planes * a.row_bytes, shift = a.row_bytes == 64 ? 6 : 7;
#pragma unroll
    for (int w = 0; w < 2; ++w)
        for (int p = first; p < pieces; p += step)
            if ((p & (a.row_bytes - 1)) >> (shift - 4) < fill)
                move_piece<WMAX, uint4>(from, to, w ? a.codes[1] : a.codes[0],
                                        a.planes * a.row_bytes * kPageTokens, (int64_t)p * 16);
    const int rows = (int)a.planes * kPageTokens;
#pragma unroll
    for (int w = 0; w < 2; ++w)
        for (int p = first; p < rows; p += step)
            if ((p & (kPageTokens - 1)) < fill)
                move_piece<WMAX, uint32_t>(from, to, w ? a.scales[1] : a.scales[0],
                                           a.planes * 4 * kPageTokens, (int64_t)p * 4);
}

}  // namespace
}  // namespace tz

using namespace tz;

extern "C" {

TENZO_HIP_API size_t tenzo_hip_beam_select_ws_bytes(int B, int W, int64_t V, int k) {
    if (B <= 0 || W <= 0 || k <= 0 || V <= 0) return 0;
    const int64_t rows = (int64_t)B * W;
    return (size_t)(rows * ceil_div(V, 256 * beam_elems(rows, V))) * (16 + (size_t)k * 8);
}

TENZO_HIP_API int tenzo_hip_beam_select(const float* logits, int64_t row_stride,
                                        const float* scores, int B, int W, int64_t V, int k,
                                        float* out_scores, int32_t* out_beams,
                                        int32_t* out_tokens, void* ws, size_t ws_bytes,
                                        void* stream) {
    TZ_CHECK(B >= 0 && W > 0 && W <= kBeamMax && k > 0 && k <= kBeamMax,
             "beam_select: B=%d, 1 to %d beams (%d) and candidates (%d)", B, kBeamMax, W, k);
    TZ_CHECK(V > 0 && V <= (1 << 30) && V * W < INT32_MAX && k <= V * W,
             "beam_select: %d of %lld candidates (V=%lld)", k, (long long)(V * W), (long long)V);
    const int64_t rows = (int64_t)B * W;
    const int elems = beam_elems(rows, V);
    const int64_t ns = ceil_div(V, 256 * elems);
    TZ_CHECK(rows * ns <= 0xffffff && B <= 0x3fffff, "beam_select: %d x %d beams", B, W);
    if (B == 0) return TENZO_SUCCESS;
    TZ_CHECK(logits && scores && out_scores && out_beams && out_tokens,
             "beam_select: null pointer");
    TZ_CHECK(row_stride >= V || B * W == 1, "beam_select: rows %lld apart, V=%lld",
             (long long)row_stride, (long long)V);
    const size_t need = tenzo_hip_beam_select_ws_bytes(B, W, V, k);
    TZ_CHECK(ws && ws_bytes >= need && ((uintptr_t)ws & 15) == 0,
             "beam_select: %zu bytes of workspace needed, %zu given", need, ws ? ws_bytes : 0);
    BeamSelect a{};
    a.logits = logits;
    a.scores = scores;
    a.stride = row_stride;
    a.W = W;
    a.k = k;
    a.V = (int)V;
    a.ns = (int)ns;
    a.sums = (double2*)ws;
    a.cand = (float2*)((char*)ws + (size_t)(rows * ns) * 16);
    a.out_scores = out_scores;
    a.out_beams = out_beams;
    a.out_tokens = out_tokens;
    const dim3 grid((unsigned)(rows * ns));
    if (elems == 16)
        hipLaunchKernelGGL(beam_slice_kernel<16>, grid, dim3(256), 0, (hipStream_t)stream, a);
    else
        hipLaunchKernelGGL(beam_slice_kernel<8>, grid, dim3(256), 0, (hipStream_t)stream, a);
    const int rc = launch_status("beam_slice_kernel");
    if (rc) return rc;
    hipLaunchKernelGGL(beam_pick_kernel, dim3((unsigned)B), dim3(1024), 0, (hipStream_t)stream, a);
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
    const int64_t most = ceil_div(a.planes * row_bytes, 256), share = ceil_div(2048, B);
    a.copiers = (int)(most < share ? most : share);
    const dim3 grid((unsigned)(a.copiers + ceil_div(table_width, 256)), (unsigned)B);
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
