// Trees of drafted tokens over a paged cache: what their nodes see and where they stand, and which
// of them the model agrees with. A sequence's nodes are its rows of the call, in its last slots
// (kv4.h: Kv4Seqs); parents[row] is the parent's place among them, a negative one or one that does
// not come before its child is none.
#include "kv4.h"

namespace tz {
namespace {

constexpr int kMostNodes = 4096;  // of a sequence

struct TreePlan {
    const int32_t* parents;
    uint64_t* mask;
    int32_t* positions;
    int words, most;
};

// A wave to 64 nodes of a sequence. Up to 64 nodes in all a node's ancestors are gathered by
// doubling: after k rounds a lane knows 2^k of them and the one after those. More nodes walk up
// one by one, over parents in LDS; each is smaller than the one before, so the words of a mask
// come from its last to its first. 64 trees of up to 64 nodes: 2.5 us, a launch and two loads in a
// row; 8 of up to 130: 3.4.
__global__ void __launch_bounds__(64) tree_plan_kernel(TreePlan a, Kv4Seqs sq) {
    __shared__ int par[kMostNodes];
    const int b = blockIdx.x, lane = threadIdx.x, i = blockIdx.y * 64 + lane;
    int first;
    const int n = min(sq.rows(b, first), a.most), c = sq.length(b);
    if (blockIdx.y * 64 >= n) return;
    const int prior = c - sq.rows(b, first);
    const bool there = i < n && c > 0 && prior + i >= 0;
    uint64_t* m = a.mask + (int64_t)(first + i) * a.words;
    if (n <= 64) {
        int up = i < n ? a.parents[first + i] : -1;
        if (up >= i) up = -1;
        uint64_t bits = 1ull << lane;
        while (__ballot(up >= 0)) {
            const int from = max(up, 0);
            const uint64_t other = __shfl(bits, from);
            const int next = __shfl(up, from);
            if (up >= 0) {
                bits |= other;
                up = next;
            }
        }
        if (i < n) {
            m[0] = there ? bits : 0;
            for (int w = 1; w < a.words; ++w) m[w] = 0;
            a.positions[first + i] = there ? prior + (int)__popcll(bits) - 1 : 0;
        }
        return;
    }
    for (int k = lane; k < n; k += 64) par[k] = a.parents[first + k];
    __syncthreads();
    if (i >= n) return;
    int w = a.words - 1, depth = -1;
    uint64_t bits = 0;
    for (int j = there ? i : -1; j >= 0;) {
        for (; w > j >> 6; --w) {
            m[w] = bits;
            bits = 0;
        }
        bits |= 1ull << (j & 63);
        ++depth;
        const int p = par[j];
        j = p < j ? p : -1;
    }
    for (; w >= 0; --w) {
        m[w] = bits;
        bits = 0;
    }
    a.positions[first + i] = there ? prior + depth : 0;
}

struct TreeAccept {
    const int32_t* parents;
    const int32_t* tokens;
    const int32_t* target;
    int32_t* path;
    int32_t* count;
    int32_t* next;
    int32_t* lens;
    uint8_t* pk;
    uint8_t* pv;
    uint8_t* pks;
    uint8_t* pvs;
    int most;
};

// The lowest child of node `at` with the token that the model says there, or -1. A whole wave.
__device__ __forceinline__ int agreed_child(const TreeAccept& a, int first, int n, int at,
                                            int lane) {
    const int said = a.target[first + at];
    for (int base = (at + 1) & ~63; base < n; base += 64) {
        const int v = base + lane;
        const bool hit = v > at && v < n && a.parents[first + v] == at &&
                         a.tokens[first + v] == said;
        const uint64_t hits = __ballot(hit);
        if (hits) return base + __ffsll((unsigned long long)hits) - 1;
    }
    return -1;
}

constexpr int kMoveRows = 16, kMoveHeads = 8;

// A workgroup to a sequence, layer and 8 heads. Each walks the tree by itself (a second launch
// would cost more); those of the first layer and heads write what came out. Rows are moved 16 at a
// time, all read before one is written: a row's new slot is never above its old one, so slots that
// are still to be read lie behind those that are written. 64 trees of up to 64 nodes, 30 layers of 5
// heads: 8.6 us, the walk's chain of loads (a target, then 64 parents and tokens, for each node of the
// path), and rows that go by way of scratch memory between load and store (80 bytes a thread, int8
// pools 144: the compiler does not hold `v` and `to` in registers); one tree of 26, 3.4.
template <int PIECES>  // of 16 bytes, of a row's codes
__global__ void __launch_bounds__(256) tree_accept_kernel(TreeAccept a, Kv4Seqs sq) {
    __shared__ int path[kMostNodes];
    __shared__ int total;
    const int b = blockIdx.x, layer = blockIdx.y, h0 = blockIdx.z * kMoveHeads;
    const int tid = threadIdx.x, lane = tid & 63;
    int first;
    const int n = sq.rows(b, first), c = sq.length(b), prior = c - n;
    const bool alive = n > 0 && prior >= 0 && c > 0;
    if (tid < 64) {
        int k = 0, last = -1;
        for (int at = alive ? 0 : -1; at >= 0 && k < a.most; ++k) {
            if (lane == 0) path[k] = at;
            last = at;
            at = agreed_child(a, first, n, at, lane);
        }
        if (lane == 0) total = k;
        if (layer == 0 && blockIdx.z == 0 && lane == 0) {
            a.count[b] = k;
            a.next[b] = last >= 0 ? a.target[first + last] : -1;
            a.lens[b] = k > 0 ? prior + k : sq.ctx[b];
        }
    }
    __syncthreads();
    const int count = total;
    if (layer == 0 && blockIdx.z == 0)
        for (int k = tid; k < a.most; k += 256)
            a.path[(int64_t)b * a.most + k] = k < count ? path[k] : -1;
    const int heads = min(kMoveHeads, sq.Hkv - h0);
    const auto row_of = [&](int slot) -> int64_t {  // of head 0 of this layer, or -1
        const int64_t blk = sq.tables[(int64_t)b * sq.table_stride + slot / kKv4Page];
        return blk >= 0 && blk < sq.n_blocks
                   ? ((blk * sq.n_layers + layer) * sq.Hkv + h0) * kKv4Page + slot % kKv4Page
                   : -1;
    };
    constexpr int PER = kMoveRows * kMoveHeads * 2 * PIECES / 256;
    for (int k0 = 0; k0 < count; k0 += kMoveRows) {
        const int k1 = min(count, k0 + kMoveRows);
        if (path[k1 - 1] == k1 - 1) continue;  // (nothing moves before the first gap)
        uint4 v[PER];
        uint8_t* to[PER];
#pragma unroll
        for (int u = 0; u < PER; ++u) {
            const int it = tid + 256 * u, piece = it % PIECES, kv = it / PIECES % 2;
            const int h = it / (2 * PIECES) % kMoveHeads, k = k0 + it / (2 * PIECES * kMoveHeads);
            to[u] = nullptr;
            if (k >= k1 || h >= heads || path[k] == k) continue;
            const int64_t src = row_of(prior + path[k]), dst = row_of(prior + k);
            if (src < 0 || dst < 0) continue;
            uint8_t* p = kv ? a.pv : a.pk;
            v[u] = *reinterpret_cast<const uint4*>(p + (src + h * kKv4Page) * (PIECES * 16) +
                                                   piece * 16);
            to[u] = p + (dst + h * kKv4Page) * (PIECES * 16) + piece * 16;
        }
        const int kv = tid & 1, h = tid / 2 % kMoveHeads, k = k0 + tid / (2 * kMoveHeads);
        uint32_t sv = 0;
        uint8_t* sto = nullptr;
        if (k < k1 && h < heads && path[k] != k) {
            const int64_t src = row_of(prior + path[k]), dst = row_of(prior + k);
            if (src >= 0 && dst >= 0) {
                uint8_t* p = kv ? a.pvs : a.pks;
                sv = *reinterpret_cast<const uint32_t*>(p + (src + h * kKv4Page) * 4);
                sto = p + (dst + h * kKv4Page) * 4;
            }
        }
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
#pragma unroll
        for (int u = 0; u < PER; ++u)
            if (to[u]) *reinterpret_cast<uint4*>(to[u]) = v[u];
        if (sto) *reinterpret_cast<uint32_t*>(sto) = sv;
        __syncthreads();
    }
}

}  // namespace
}  // namespace tz

using namespace tz;

extern "C" {

TENZO_HIP_API int tenzo_hip_tree_plan(const int32_t* parents, const int32_t* ctx_lens,
                                      const int32_t* cu_q, int B, int64_t T, int most,
                                      uint64_t* mask, int32_t* positions, void* stream) {
    TZ_CHECK(B >= 0 && T >= 0 && T <= INT32_MAX, "tree_plan: B=%d T=%lld", B, (long long)T);
    TZ_CHECK(most >= 1 && most <= kMostNodes, "tree_plan: up to %d nodes, not %d", kMostNodes,
             most);
    TZ_CHECK(cu_q || T == B, "tree_plan: %lld rows for %d sequences of one token", (long long)T,
             B);
    if (T == 0 || B == 0) return TENZO_SUCCESS;
    TZ_CHECK(parents && ctx_lens && mask && positions, "tree_plan: null pointer");
    TZ_CHECK(((uintptr_t)mask & 7) == 0, "tree_plan: masks must be 8-byte aligned");
    Kv4Seqs q{};
    q.ctx = ctx_lens;
    q.cu = cu_q;
    q.B = B;
    q.T = (int)T;
    q.limit = INT32_MAX;
    const TreePlan a{parents, mask, positions, (int)ceil_div(most, 64), most};
    hipLaunchKernelGGL(tree_plan_kernel, dim3(B, a.words), dim3(64), 0, (hipStream_t)stream, a, q);
    return launch_status("tree_plan_kernel");
}

TENZO_HIP_API int tenzo_hip_tree_accept(const int32_t* parents, const int32_t* tokens,
                                        const int32_t* target, void* pk, void* pv, void* pks,
                                        void* pvs, int64_t n_blocks, int n_layers, int Hkv,
                                        int row_bytes, const int32_t* block_tables,
                                        int64_t table_stride, int table_width,
                                        const int32_t* ctx_lens, const int32_t* cu_q, int B,
                                        int64_t T, int most, int32_t* path, int32_t* count,
                                        int32_t* next, int32_t* lens, void* stream) {
    Kv4Seqs q{};
    const int rc = kv4_check("tree_accept", pk, pv, pks, pvs, n_blocks, n_layers, 0, Hkv,
                             block_tables, table_stride, table_width, ctx_lens, cu_q, B, T,
                             nullptr, 0, q);
    if (rc) return rc;
    TZ_CHECK(most >= 1 && most <= kMostNodes, "tree_accept: up to %d nodes, not %d", kMostNodes,
             most);
    TZ_CHECK(row_bytes == 64 || row_bytes == 128, "tree_accept: rows of %d bytes", row_bytes);
    TZ_CHECK(n_layers <= 65535 && Hkv <= 65535 * kMoveHeads, "tree_accept: %d layers", n_layers);
    if (B == 0) return TENZO_SUCCESS;
    TZ_CHECK(ctx_lens && path && count && next && lens, "tree_accept: null pointer");
    TZ_CHECK(lens != ctx_lens && count != ctx_lens && next != ctx_lens && path != ctx_lens,
             "tree_accept: the lengths are read while outputs are written");
    TZ_CHECK(T == 0 || (parents && tokens && target), "tree_accept: null pointer");
    const TreeAccept a{parents, tokens, target, path, count, next, lens, (uint8_t*)pk,
                       (uint8_t*)pv, (uint8_t*)pks, (uint8_t*)pvs, most};
    const dim3 grid(B, n_layers, (unsigned)ceil_div(Hkv, kMoveHeads));
    if (row_bytes == 64)
        hipLaunchKernelGGL(tree_accept_kernel<4>, grid, dim3(256), 0, (hipStream_t)stream, a, q);
    else
        hipLaunchKernelGGL(tree_accept_kernel<8>, grid, dim3(256), 0, (hipStream_t)stream, a, q);
    return launch_status("tree_accept_kernel");
}

}  // extern "C"
