// kvq_evict: shrink every (batch row, kv head) of a contiguous cache to a budget of tokens.
//
// Selection.  A token's key is an unsigned order of (protected, weight): protected tokens (sinks, recent ones) have the
// largest key, then fp32 weights in their order (NaN as -inf, -0 as +0).  The budget-th largest key K* is found digit by
// digit from the top (radix selection, 8 bits a pass over the row's keys); all larger keys are kept, and of the keys equal
// to K* the lowest slots until the budget is full.  No sort, no rounding, no dependence on the order of atomics (they only
// count).
//
// Moves.  A kept token in a slot below the budget stays.  The kept ones behind the budget fill the freed slots, both in
// ascending order: sources (>= budget) and destinations (< budget) are disjoint, so the moves run in place and in parallel,
// and there are no more of them than tokens that are evicted.  Shrinking by one token per decode step moves one token per
// head, whatever the budget, where a compaction that keeps the order would move half of the cache.
//
// One CTA per (batch row, kv head).
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "kvq_internal.h"

namespace kvq {

constexpr int kEvictThreads = 1024;
constexpr int kEvictWarps = kEvictThreads / 32;

struct EvictParams {
    KvqEvictArgs a;
    int* moves;              // [B * Hkv][2][max_moves]: destinations, sources
    long long max_moves;
};

constexpr uint32_t kKeyProtected = 0xffffffffu;

// unsigned order of fp32 weights: larger weight, larger key; below kKeyProtected for every weight
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) w = -INFINITY;
    const uint32_t u = __float_as_uint(w + 0.f);           // -0 + 0 = +0
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// exclusive prefix sum over the CTA of two counters packed in 64 bits; returns the total in `total`
__device__ __forceinline__ unsigned long long block_scan(unsigned long long v, unsigned long long* sh, unsigned long long& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned long long incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long x = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += x;
    }
    __syncthreads();
    if (lane == 31) sh[warp] = incl;
    __syncthreads();
    unsigned long long w = sh[lane];                       // kEvictWarps == 32
    unsigned long long wi = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long x = __shfl_up_sync(0xffffffffu, wi, o);
        if (lane >= o) wi += x;
    }
    total = __shfl_sync(0xffffffffu, wi, 31);
    const unsigned long long base = __shfl_sync(0xffffffffu, wi - w, warp);
    return base + incl - v;
}

__global__ void __launch_bounds__(kEvictThreads) evict_kernel(const EvictParams p) {
    static_assert(kEvictWarps == 32, "the block scan reads one warp total per lane");
    pdl_launch_dependents();
    pdl_wait();
    const KvqEvictArgs& a = p.a;
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    __shared__ unsigned hist[256];
    __shared__ unsigned long long sh[32];
    __shared__ uint32_t sel[2];
    const int n = max(0, min(a.lengths[b], a.cap)), m = a.budget;
    const int seen = a.seen[b];
    if (n <= m) return;
    float* w = a.weights + b * a.w_stride_b + h * a.w_stride_h;
    int* pos = a.positions + b * a.p_stride_b + h * a.p_stride_h;
    auto position = [&](int s) -> int {
        const int q = pos[s];
        return q >= 0 ? q : seen - n + s;
    };
    auto key_of = [&](int s) -> uint32_t {
        const int q = position(s);
        return (q < a.sinks || q >= seen - a.recent) ? kKeyProtected : weight_key(w[s]);
    };
    // ---- the budget-th largest key
    uint32_t prefix = 0, mask = 0;
    unsigned need = (unsigned)m;                           // of the keys that match the prefix so far, the largest `need`
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        for (int s = tid; s < n; s += kEvictThreads) {
            const uint32_t k = key_of(s);
            if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255u], 1u);
        }
        __syncthreads();
        if (warp == 0) {
            // lane l owns digits 255 - 8 l ... 248 - 8 l (largest first)
            unsigned c[8], sum = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) { c[j] = hist[255 - 8 * lane - j]; sum += c[j]; }
            unsigned incl = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned x = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += x;
            }
            unsigned before = incl - sum;                  // keys with a larger digit than this lane's
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (need > before && need <= before + c[j]) {
                    sel[0] = (uint32_t)(255 - 8 * lane - j);
                    sel[1] = need - before;
                }
                before += c[j];
            }
        }
        __syncthreads();
        prefix |= sel[0] << shift;
        mask |= 255u << shift;
        need = sel[1];
        __syncthreads();
    }
    // ---- kept slots, in ascending order: ties, freed slots and moving tokens are counted by prefix sums
    const long long row = (long long)b * a.Hkv + h;
    int* dst = p.moves + row * 2 * p.max_moves;
    int* src = dst + p.max_moves;
    unsigned eq_before = 0, freed = 0, moved = 0;
    for (int s0 = 0; s0 < n; s0 += kEvictThreads) {
        const int s = s0 + tid;
        uint32_t k = 0;
        bool eq = false;
        int q = 0;
        if (s < n) {
            q = position(s);
            k = (q < a.sinks || q >= seen - a.recent) ? kKeyProtected : weight_key(w[s]);
            eq = k == prefix;
        }
        unsigned long long total;
        const unsigned rank = eq_before + (unsigned)block_scan(eq ? 1ull : 0ull, sh, total);
        eq_before += (unsigned)total;
        const bool keep = s < n && (k > prefix || (eq && rank < need));
        const bool hole = s < m && s < n && !keep, mover = s >= m && keep;
        const unsigned long long ex = block_scan((hole ? 1ull : 0ull) | (mover ? 1ull << 32 : 0ull), sh, total);
        if (hole) dst[freed + (unsigned)ex] = s;
        if (mover) src[moved + (unsigned)(ex >> 32)] = s;
        freed += (unsigned)total;
        moved += (unsigned)(total >> 32);
        if (keep && s < m) pos[s] = q;
    }
    __syncthreads();                                       // the lists are complete (written and read by this CTA)
    // ---- move: one warp per token and buffer row, 16, 4 or 1 bytes at a time
    for (unsigned i = warp; i < moved; i += kEvictWarps) {
        const int d = dst[i], s = src[i];
        for (int j = 0; j < a.n_bufs; ++j) {
            const KvqEvictBuf& f = a.bufs[j];
            char* base = (char*)f.base + b * f.stride_b + h * f.stride_h;
            char* to = base + d * f.stride_s;
            const char* from = base + s * f.stride_s;
            const unsigned long long al = (unsigned long long)to | (unsigned long long)from | (unsigned long long)f.row_bytes;
            if ((al & 15) == 0)
                for (long long x = lane; x < (f.row_bytes >> 4); x += 32) ((uint4*)to)[x] = ((const uint4*)from)[x];
            else if ((al & 3) == 0)
                for (long long x = lane; x < (f.row_bytes >> 2); x += 32) ((uint32_t*)to)[x] = ((const uint32_t*)from)[x];
            else
                for (long long x = lane; x < f.row_bytes; x += 32) to[x] = from[x];
        }
        if (lane == 0) {
            pos[d] = position(s);
            w[d] = w[s];
        }
    }
    __syncthreads();
    for (int s = m + tid; s < n; s += kEvictThreads) {
        w[s] = 0.f;
        pos[s] = -1;
    }
}

// After every row has read its length: lengths and new_lengths may be one array.
__global__ void evict_lengths_kernel(const EvictParams p) {
    pdl_launch_dependents();
    pdl_wait();
    const int b = blockIdx.x * blockDim.x + threadIdx.x;
    if (b < p.a.B) p.a.new_lengths[b] = min(max(0, min(p.a.lengths[b], p.a.cap)), p.a.budget);
}

}  // namespace kvq

extern "C" size_t kvq_evict_workspace_bytes(int32_t B, int32_t Hkv, int32_t cap, int32_t budget) {
    if (B <= 0 || Hkv <= 0 || cap <= 0 || budget <= 0) return 256;
    const long long moves = cap - budget < budget ? cap - budget : budget;
    const size_t n = (size_t)B * Hkv * 2 * (moves > 0 ? moves : 0) * sizeof(int);
    return ((n + 255) & ~(size_t)255) + 256;
}

extern "C" int kvq_evict(const KvqEvictArgs* args, kvq_stream_t stream) {
    using namespace kvq;
    if (!args) return KVQ_EINVAL;
    const KvqEvictArgs& a = *args;
    if (a.B < 0 || a.Hkv <= 0 || a.cap < 0 || a.budget <= 0 || a.sinks < 0 || a.recent < 0) return KVQ_EINVAL;
    if ((long long)a.sinks + a.recent > a.budget) return KVQ_EINVAL;
    if (a.n_bufs < 0 || a.n_bufs > KVQ_EVICT_MAX_BUFS) return KVQ_EINVAL;
    if (a.B == 0) return KVQ_OK;
    if (!a.lengths || !a.seen || !a.new_lengths || !a.weights || !a.positions) return KVQ_EINVAL;
    for (int j = 0; j < a.n_bufs; ++j)
        if (!a.bufs[j].base || a.bufs[j].row_bytes <= 0) return KVQ_EINVAL;
    if (a.Hkv > 65535 || a.B > 65535) return KVQ_ELIMIT;
    if (!a.workspace || (((uintptr_t)a.workspace) & 15) || a.workspace_bytes < kvq_evict_workspace_bytes(a.B, a.Hkv, a.cap, a.budget))
        return KVQ_EWORKSPACE;
    EvictParams p;
    p.a = a;
    p.moves = (int*)a.workspace;
    p.max_moves = a.cap - a.budget < a.budget ? a.cap - a.budget : a.budget;
    if (p.max_moves < 0) p.max_moves = 0;
    cudaStream_t st = (cudaStream_t)stream;
    int rc = KVQ_OK;
    if (a.cap > a.budget) rc = launch_pdl(evict_kernel, dim3(a.Hkv, a.B), dim3(kEvictThreads), 0, st, p);
    if (rc) return rc;
    return launch_pdl(evict_lengths_kernel, dim3((a.B + 127) / 128), dim3(128), 0, st, p);
}
