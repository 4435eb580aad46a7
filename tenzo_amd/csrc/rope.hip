// Rotary positions: every row of heads turned at a position of its own.
#include <cmath>

#include "common.h"

namespace tz {
namespace {

struct Rope {
    const void* x;
    void* out;
    int64_t x_stride, out_stride;
    const int32_t* pos;
    const double* freqs;
    float mscale;
    int H, D, half;  // half: pairs of a head
    uint32_t p_mul;  // 2^32 / groups of pairs, rounded up (0: one group)
    uint32_t c_mul;  // and of a head's chunks that are only copied
    int chunks;      // those (0: nothing to copy)
};

constexpr int kPairs = 512;  // of a head, at most

// n / d for n < 2^16 and mul = 2^32 / d, rounded up.
__device__ __forceinline__ int div_by(int n, uint32_t mul) {
    return mul ? (int)__umulhi((uint32_t)n, mul) : n;
}

// Cosine and sine of pos * freq, within 2^-23 and the 2^-51 of the angle that 64 bits lose: it is
// taken in turns, of which whole ones leave exactly, and the rest, an eighth of a turn to either
// side of a quarter, by their series in fp32 (the first terms left out are below 2^-29 and 2^-33).
__device__ __forceinline__ float2 turn(int pos, double freq) {
    const double t = (double)pos * (freq * 0.15915494309189533577);
    const double r = t - rint(t);
    const float q = rintf((float)r * 4.0f);
    const float x = (float)((r - 0.25 * (double)q) * 6.283185307179586477);
    const float z = x * x;
    float s = __builtin_fmaf(z, 2.7557319224e-6f, -1.9841269841e-4f);
    s = __builtin_fmaf(z, s, 8.3333333333e-3f);
    s = __builtin_fmaf(z, s, -1.6666666667e-1f);
    s = __builtin_fmaf(x * z, s, x);
    float c = __builtin_fmaf(z, -2.7557319224e-7f, 2.4801587302e-5f);
    c = __builtin_fmaf(z, c, -1.3888888889e-3f);
    c = __builtin_fmaf(z, c, 4.1666666667e-2f);
    c = __builtin_fmaf(z, c, -0.5f);
    c = __builtin_fmaf(z, c, 1.0f);
    const int k = (int)q & 3;
    const float cs = k & 1 ? s : c, sn = k & 1 ? c : s;
    return make_float2(k == 1 || k == 2 ? -cs : cs, k >= 2 ? -sn : sn);
}

// E elements of TYPE (0 fp32, 1 fp16, 2 bf16) at any element's address.
template <int TYPE>
struct Element {
    typedef float type;
};
template <>
struct Element<1> {
    typedef _Float16 type;
};
template <>
struct Element<2> {
    typedef __bf16 type;
};
template <int TYPE, int E>
struct Chunk {
    typedef typename Element<TYPE>::type T;
    typedef T vec __attribute__((ext_vector_type(E)));
    struct __attribute__((packed, aligned(sizeof(T)))) any {
        vec v;
    };
    vec v;
    __device__ __forceinline__ void load(const void* p, int64_t i) {
        v = reinterpret_cast<const any*>(reinterpret_cast<const T*>(p) + i)->v;
    }
    __device__ __forceinline__ void store(void* p, int64_t i) const {
        reinterpret_cast<any*>(reinterpret_cast<T*>(p) + i)->v = v;
    }
};
template <int TYPE>
struct Chunk<TYPE, 1> {
    typedef typename Element<TYPE>::type T;
    T v[1];
    __device__ __forceinline__ void load(const void* p, int64_t i) {
        v[0] = reinterpret_cast<const T*>(p)[i];
    }
    __device__ __forceinline__ void store(void* p, int64_t i) const {
        reinterpret_cast<T*>(p)[i] = v[0];
    }
};

// (a, b) -> (a c - b s, a s + b c) for the pairs of every head, in fp32 and rounded once. An item
// is E pairs of a head: two chunks of E elements, `half` apart or side by side. Each is read and
// written by one thread, so `out` may be `x`.
//
// A workgroup has a row, whose angles, the 64-bit work in them, its threads take once for all heads.
// 8001 rows of 40 heads of 128, fp16: 26 us, 6.3 TB/s read and written
// (a part stays in the last cache), bound by that; 26 rows of 25 heads, fp32: 3 us, a launch and
// the chain of position, angle, LDS and row; 8000 rows of one head, fp16: 5.4 us, workgroups of which 8
// threads have a part of the row.
template <int TYPE, int E, bool INTER>
__global__ void __launch_bounds__(256) rope_kernel(Rope a) {
    __shared__ float cs[kPairs], sn[kPairs];
    const int row = blockIdx.x;
    for (int i = threadIdx.x; i < a.half; i += 256) {
        const float2 v = turn(a.pos[row], a.freqs[i]);
        cs[i] = v.x * a.mscale;
        sn[i] = v.y * a.mscale;
    }
    __syncthreads();
    const int64_t x0 = row * a.x_stride, o0 = row * a.out_stride;
    const int groups = a.half / E, items = a.H * groups;
    for (int it = threadIdx.x; it < items; it += 256) {
        const int h = div_by(it, a.p_mul), p = (it - h * groups) * E;
        const int64_t xa = x0 + h * a.D, oa = o0 + h * a.D;
        const int at[2] = {INTER ? 2 * p : p, INTER ? 2 * p + E : a.half + p};
        Chunk<TYPE, E> v[2];
        v[0].load(a.x, xa + at[0]);
        v[1].load(a.x, xa + at[1]);
        float x[2 * E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            x[e] = (float)v[0].v[e];
            x[E + e] = (float)v[1].v[e];
        }
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int i0 = INTER ? 2 * e : e, i1 = INTER ? 2 * e + 1 : E + e;
            const float c = cs[p + e], s = sn[p + e];
            const float y0 = __builtin_fmaf(x[i0], c, -__fmul_rn(x[i1], s));
            x[i1] = __builtin_fmaf(x[i0], s, __fmul_rn(x[i1], c));
            x[i0] = y0;
        }
#pragma unroll
        for (int e = 0; e < E; ++e) {
            v[0].v[e] = (typename Element<TYPE>::type)x[e];
            v[1].v[e] = (typename Element<TYPE>::type)x[E + e];
        }
        v[0].store(a.out, oa + at[0]);
        v[1].store(a.out, oa + at[1]);
    }
    const int copies = a.H * a.chunks;
    for (int it = threadIdx.x; it < copies; it += 256) {
        const int h = div_by(it, a.c_mul), p = 2 * a.half + (it - h * a.chunks) * E;
        Chunk<TYPE, E> v;
        v.load(a.x, x0 + h * a.D + p);
        v.store(a.out, o0 + h * a.D + p);
    }
}

template <int TYPE, int E>
int launch_rope(const Rope& a0, int T, bool inter, hipStream_t st) {
    Rope a = a0;
    const int groups = a.half / E;
    const auto mul = [](int d) {
        return d <= 1 ? 0u : (uint32_t)((0x100000000ull + (unsigned)d - 1) / (unsigned)d);
    };
    a.p_mul = mul(groups);
    a.chunks = a.out == a.x ? 0 : (a.D - 2 * a.half) / E;
    a.c_mul = mul(a.chunks);
    if (inter)
        hipLaunchKernelGGL((rope_kernel<TYPE, E, true>), dim3(T), dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((rope_kernel<TYPE, E, false>), dim3(T), dim3(256), 0, st, a);
    return launch_status("rope_kernel");
}

}  // namespace
}  // namespace tz

using namespace tz;

extern "C" {

TENZO_HIP_API int tenzo_hip_rope(const void* x, int dtype, int64_t x_stride,
                                 const int32_t* positions, const double* freqs, int64_t T, int H,
                                 int head_dim, int rot_dim, int interleaved, float mscale,
                                 void* out, int64_t out_stride, void* stream) {
    TZ_CHECK(dtype >= 0 && dtype <= 2, "rope: dtype %d", dtype);
    TZ_CHECK(T >= 0 && T < 1 << 24, "rope: %lld rows", (long long)T);
    TZ_CHECK(head_dim >= 2 && head_dim <= 1024 && H >= 1 && (int64_t)H * head_dim <= 32768,
             "rope: %d heads of %d", H, head_dim);
    TZ_CHECK(rot_dim >= 2 && rot_dim % 2 == 0 && rot_dim <= head_dim,
             "rope: %d of %d dims to turn", rot_dim, head_dim);
    if (T == 0) return TENZO_SUCCESS;
    TZ_CHECK(x && out && positions && freqs, "rope: null pointer");
    const int64_t cols = (int64_t)H * head_dim;
    TZ_CHECK(T == 1 || (x_stride >= cols && out_stride >= cols),
             "rope: row strides %lld, %lld below %d heads", (long long)x_stride,
             (long long)out_stride, H);
    TZ_CHECK(x != out || T == 1 || x_stride == out_stride,
             "rope: in place with strides %lld, %lld", (long long)x_stride, (long long)out_stride);
    const uintptr_t size = dtype ? 2 : 4;
    TZ_CHECK((((uintptr_t)x | (uintptr_t)out) & (size - 1)) == 0 && ((uintptr_t)freqs & 7) == 0 &&
                 ((uintptr_t)positions & 3) == 0,
             "rope: addresses that are not aligned to their elements");
    Rope a{x, out, x_stride, out_stride, positions, freqs, mscale, H, head_dim, rot_dim / 2, 0, 0,
           0};
    const int rest = head_dim - rot_dim;
    const auto fits = [&](int e) { return a.half % e == 0 && rest % e == 0; };
    const hipStream_t st = (hipStream_t)stream;
    const bool in = interleaved != 0;
    const int n = (int)T;
    if (dtype == 0)
        return fits(4) ? launch_rope<0, 4>(a, n, in, st) : launch_rope<0, 1>(a, n, in, st);
    if (dtype == 1)
        return fits(8)   ? launch_rope<1, 8>(a, n, in, st)
               : fits(4) ? launch_rope<1, 4>(a, n, in, st)
                         : launch_rope<1, 1>(a, n, in, st);
    return fits(8)   ? launch_rope<2, 8>(a, n, in, st)
           : fits(4) ? launch_rope<2, 4>(a, n, in, st)
                     : launch_rope<2, 1>(a, n, in, st);
}

TENZO_HIP_API int tenzo_hip_rope_freqs(int rot_dim, double theta, int scaling, double factor,
                                       double trained, double fast, double slow,
                                       double* freqs_host, float* mscale) {
    TZ_CHECK(rot_dim >= 2 && rot_dim % 2 == 0, "rope_freqs: %d dims", rot_dim);
    TZ_CHECK(theta > 0 && std::isfinite(theta), "rope_freqs: theta %g", theta);
    TZ_CHECK(scaling >= 0 && scaling <= 3, "rope_freqs: scaling %d", scaling);
    TZ_CHECK(scaling == 0 || (factor >= 1 && std::isfinite(factor)), "rope_freqs: factor %g",
             factor);
    TZ_CHECK(scaling != 2 || rot_dim > 2, "rope_freqs: %d dims", rot_dim);
    TZ_CHECK(scaling != 3 || (trained > 0 && std::isfinite(trained) && fast > slow && slow >= 0),
             "rope_freqs: %g positions, ramp from %g to %g turns", trained, slow, fast);
    TZ_CHECK(freqs_host && mscale, "rope_freqs: null pointer");
    const double base =
        scaling == 2 ? theta * std::pow(factor, (double)rot_dim / (rot_dim - 2)) : theta;
    for (int i = 0; i < rot_dim / 2; ++i) {
        double f = std::pow(base, -2.0 * i / rot_dim);
        if (scaling == 1) f /= factor;
        if (scaling == 3) {
            const double turns = trained * f / 6.283185307179586477;
            double keep = (turns - slow) / (fast - slow);
            keep = keep < 0 ? 0 : keep > 1 ? 1 : keep;
            f = f * keep + f / factor * (1 - keep);
        }
        freqs_host[i] = f;
    }
    *mscale = scaling == 3 ? (float)(0.1 * std::log(factor) + 1.0) : 1.0f;
    return TENZO_SUCCESS;
}

}  // extern "C"
