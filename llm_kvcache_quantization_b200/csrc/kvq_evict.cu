// kvq_evict: shrink every (batch row, kv head) of a contiguous cache to a budget of tokens.
//
// Selection.  A token's key is an unsigned order of (protected, weight): protected tokens (sinks, recent ones) have the
// largest key, then fp32 weights in their order (NaN as -inf, -0 as +0).  The budget-th largest key K* is found digit by
// digit: keys minus the row's smallest one, 8 bits a time from the highest bit that the row's range has, so that already
// the first digit tells binades apart (the top bits of the keys themselves are the same for almost all weights of a row).
// The search ends as soon as all keys of the digit reached are kept - on distinct weights after two or three digits.  Larger
// keys are kept, and of the keys equal to K* the lowest slots until the budget is full.  No sort, no rounding, no
// dependence on the order of atomics (they only count).
//
// Moves.  A kept token in a slot below the budget stays.  The kept ones behind the budget fill the freed slots, both in
// ascending order: sources (>= budget) and destinations (< budget) are disjoint, so the moves run in place and in parallel,
// and there are no more of them than tokens that are evicted.  Shrinking by one token per decode step moves one token per
// head, whatever the budget, where a compaction that keeps the order would move half of the cache.
//
// Split.  A cluster of 1 to 8 CTAs per (batch row, kv head): each takes a run of at most 4096 slots, 8 per thread, whose
// weights and positions it reads once and keeps in registers (beyond 32 768 slots a CTA's run is longer and read again, from
// L2, by every pass).  Histograms and counts are read across the cluster through distributed shared memory, the lists of
// moves go through global memory (L2); a warp moves 32 tokens of one buffer at a time, 8 loads in flight per lane.
// What bounds it: latency, of some ten barriers and as many dependent reads, and for large evictions the moved rows.  Measured,
// fp16 K and V of 128 channels: 2049 -> 2048 tokens, 64 rows, 8.5 us a call; 32 001 -> 4096 tokens, 32 rows, 54 us when all
// kept tokens have to move (118 MB read and written, 27 us of it in the moves), 15 us when few have.
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "kvq_internal.h"

namespace kvq {

constexpr int kEvictThreads = 512;
constexpr int kEvictWarps = kEvictThreads / 32;
constexpr int kEvictDigit = 8;                             // bits of a digit
constexpr int kEvictBins = 1 << kEvictDigit;
constexpr int kEvictPasses = 4;
constexpr int kEvictItems = 8;                             // slots of a thread that registers hold
constexpr int kEvictRun = kEvictThreads * kEvictItems;
constexpr int kEvictMaxCluster = 8;

struct EvictParams {
    KvqEvictArgs a;
    int* moves;              // [B * Hkv][4][max_moves]: destinations, sources, and the sources' positions and weights
    long long max_moves;
    int per_cta;             // slots of a CTA, a multiple of kEvictRun
};

constexpr uint32_t kKeyProtected = 0xffffffffu;

// unsigned order of fp32 weights: larger weight, larger key; below kKeyProtected for every weight
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) w = -INFINITY;
    const uint32_t u = __float_as_uint(w + 0.f);           // -0 + 0 = +0
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ void cluster_sync(int ranks) {  // release and acquire: shared and global memory of the cluster
    if (ranks == 1) __syncthreads();
    else asm volatile("barrier.cluster.arrive;\n\tbarrier.cluster.wait;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_addr(const void* p, int rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    return r;
}
__device__ __forceinline__ unsigned cluster_ld(uint32_t addr) {
    unsigned v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint4 cluster_ld4(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}

__device__ __forceinline__ unsigned warp_prefix(unsigned v) {       // inclusive
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned x = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += x;
    }
    return v;
}
// Sum of sh[0 .. warp) for the calling warp, sh being one count per warp (complete behind a barrier); all in `total`.
__device__ __forceinline__ unsigned warps_before(const unsigned* sh, unsigned& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned c = lane < kEvictWarps ? sh[lane] : 0u, incl = warp_prefix(c);
    total = __shfl_sync(0xffffffffu, incl, 31);
    return __shfl_sync(0xffffffffu, incl - c, warp);
}

// Moves first .. first + 31 of one buffer, in units of V, by one warp; lane l holds source and destination of move first + l.
template <typename V>
__device__ __forceinline__ void move_rows(const KvqEvictBuf& f, char* base, int src, int dst, int count) {
    constexpr int U = 8;
    const int lane = threadIdx.x & 31;
    const int units = (int)(f.row_bytes / (int)sizeof(V));
    // Unit u of move i; 32 units further for the next step.  (Divisions per step would be most of the kernel's instructions.)
    const int di = 32 / units, du = 32 - di * units;
    int i = lane / units, u = lane - i * units;
    auto next = [&](int& i_, int& u_) {
        i_ += di, u_ += du;
        if (u_ >= units) u_ -= units, ++i_;
    };
    while (__any_sync(0xffffffffu, i < count)) {
        V v[U];
        int li = i, lu = u;
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int s = __shfl_sync(0xffffffffu, src, li & 31);
            if (li < count) v[j] = ((const V*)(base + s * f.stride_s))[lu];
            next(li, lu);
        }
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int d = __shfl_sync(0xffffffffu, dst, i & 31);
            if (i < count) ((V*)(base + d * f.stride_s))[u] = v[j];
            next(i, u);
        }
    }
}

// REGS: a thread's slots are kept in registers (per_cta == kEvictRun).
template <bool REGS>
__global__ void __launch_bounds__(kEvictThreads, 2) evict_kernel(const EvictParams p) {
    pdl_launch_dependents();
    constexpr int G = REGS ? kEvictItems : 4;              // slots of a thread that are read at a time
    const KvqEvictArgs& a = p.a;
    const int h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = blockIdx.x, ranks = gridDim.x;        // the cluster spans x
    __shared__ alignas(16) unsigned hist[kEvictPasses][kEvictBins];
    __shared__ uint4 part[kEvictMaxCluster][kEvictBins / 4];
    __shared__ unsigned sums[kEvictWarps], sums2[kEvictWarps], sums3[kEvictWarps], sel[3], range[3], totals[2], lowest;
    for (int i = tid; i < kEvictPasses * kEvictBins; i += kEvictThreads) (&hist[0][0])[i] = 0;
    pdl_wait();
    const int n = max(0, min(a.lengths[b], a.cap)), m = a.budget;
    const int seen = a.seen[b];
    if (h == 0 && rank == 0 && tid == 0) a.new_lengths[b] = min(n, m);
    if (n <= m) return;                                    // the whole cluster
    float* w = a.weights + b * a.w_stride_b + h * a.w_stride_h;
    int* pos = a.positions + b * a.p_stride_b + h * a.p_stride_h;
    // This warp's slots: s0 + 32 i + lane, below s1.
    const int per_warp = REGS ? 32 * kEvictItems : p.per_cta / kEvictWarps;
    const long long first = (long long)rank * p.per_cta + warp * per_warp;
    const int s0 = (int)min((long long)n, first), s1 = (int)min((long long)n, first + per_warp);
    const int groups = REGS ? 1 : (s1 - s0 + 32 * G - 1) / (32 * G);
    uint32_t key[G];                                       // of a group of slots; 0 behind the row
    int q[G];
    float wt[G];
    auto slot = [&](int g, int j) -> int { return s0 + (g * G + j) * 32 + lane; };
    auto load = [&](int g) {
#pragma unroll
        for (int j = 0; j < G; ++j) {
            const int s = slot(g, j);
            q[j] = s < s1 ? pos[s] : 0;
            wt[j] = s < s1 ? w[s] : 0.f;
        }
#pragma unroll
        for (int j = 0; j < G; ++j) {
            const int s = slot(g, j);
            if (q[j] < 0) q[j] = seen - n + s;
            key[j] = s >= s1 ? 0u : (q[j] < a.sinks || q[j] >= seen - a.recent) ? kKeyProtected : weight_key(wt[j]);
        }
    };
    if (REGS) load(0);
    // ---- range of the weights' keys, and the protected tokens (0 is below every key)
    unsigned lo = kKeyProtected, hi = 0, prot = 0;
    for (int g = 0; g < groups; ++g) {
        if (!REGS) load(g);
#pragma unroll
        for (int j = 0; j < G; ++j) {
            const bool pr = key[j] == kKeyProtected;
            prot += pr;
            if (!pr) hi = max(hi, key[j]);
            if (key[j] != 0) lo = min(lo, key[j]);
        }
    }
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);
    prot = __reduce_add_sync(0xffffffffu, prot);
    if (lane == 0) sums[warp] = lo, sums2[warp] = hi, sums3[warp] = prot;
    __syncthreads();
    if (warp == 0) {
        const bool in = lane < kEvictWarps;
        lo = __reduce_min_sync(0xffffffffu, in ? sums[lane] : kKeyProtected);
        hi = __reduce_max_sync(0xffffffffu, in ? sums2[lane] : 0u);
        prot = __reduce_add_sync(0xffffffffu, in ? sums3[lane] : 0u);
        if (lane == 0) range[0] = lo, range[1] = hi, range[2] = prot;
    }
    cluster_sync(ranks);
    {
        const bool in = lane < ranks;
        lo = __reduce_min_sync(0xffffffffu, in ? cluster_ld(cluster_addr(&range[0], lane)) : kKeyProtected);
        hi = __reduce_max_sync(0xffffffffu, in ? cluster_ld(cluster_addr(&range[1], lane)) : 0u);
        prot = __reduce_add_sync(0xffffffffu, in ? cluster_ld(cluster_addr(&range[2], lane)) : 0u);
    }
    // Keys minus lo from here on; protected ones stay the largest, slots behind the row are told by s >= s1.
    auto rel = [&](uint32_t k) -> uint32_t { return k == kKeyProtected ? k : k - lo; };
    // ---- the budget-th largest key, as `prefix` of what is left of a key shifted by `shift`
    uint32_t prefix = kKeyProtected;
    int shift = 0;
    unsigned need = (unsigned)m, same = prot;              // of the keys that match the prefix, the largest `need` are kept
    const unsigned* counts = nullptr;                      // where this CTA's share of `same` stands
    bool found = prot >= need;
    if (!found && n - m <= n / 16) {
        // Few tokens go (a decode step): mostly they are among those of the smallest weight, tokens that nobody looked at.
        unsigned cnt = 0;
        for (int g = 0; g < groups; ++g) {
            if (!REGS) load(g);
#pragma unroll
            for (int j = 0; j < G; ++j) cnt += key[j] == lo;
        }
        cnt = __reduce_add_sync(0xffffffffu, cnt);
        if (lane == 0) sums[warp] = cnt;
        __syncthreads();
        if (warp == 0) {
            cnt = __reduce_add_sync(0xffffffffu, lane < kEvictWarps ? sums[lane] : 0u);
            if (lane == 0) lowest = cnt;
        }
        cluster_sync(ranks);
        const unsigned all = __reduce_add_sync(0xffffffffu, lane < ranks ? cluster_ld(cluster_addr(&lowest, lane)) : 0u);
        if (all >= (unsigned)(n - m)) {
            found = true;
            prefix = 0;                                    // rel(lo)
            same = all;
            need = all - (unsigned)(n - m);
            counts = &lowest;
        }
    }
    if (!found) {
        need -= prot;
        prefix = 0;
        shift = 32 - __clz(hi - lo);
        for (int pass = 0;; ++pass) {                      // at most 4: 32 bits
            const int bits = min(shift, kEvictDigit), up = shift;
            shift -= bits;
            const uint32_t digits = (1u << bits) - 1;
            for (int g = 0; g < groups; ++g) {
                if (!REGS) load(g);
#pragma unroll
                for (int j = 0; j < G; ++j) {
                    const uint32_t k = rel(key[j]);
                    // shifts of 32 are taken in two steps
                    if (slot(g, j) < s1 && key[j] != kKeyProtected && (k >> (up >> 1) >> (up - (up >> 1))) == prefix)
                        atomicAdd(&hist[pass][(k >> shift) & digits], 1u);
                }
            }
            cluster_sync(ranks);
            // The cluster's sums.  Distributed shared memory is read once, 16 bytes a thread: 2100 cycles with 8 CTAs (one
            // thread per digit with 8 scalar reads 2900, digits of 10 bits 4100, of 11 bits 7000).
            constexpr int QUADS = kEvictBins / 4;
            static_assert(kEvictThreads == kEvictMaxCluster * QUADS, "one thread per CTA and four digits");
            const int quad = QUADS - 1 - tid % QUADS, r = tid / QUADS;      // threads in descending order of digits
            if (r < ranks) part[r][tid % QUADS] = cluster_ld4(cluster_addr(&hist[pass][4 * quad], r));
            __syncthreads();
            unsigned c[4] = {0u, 0u, 0u, 0u}, sum = 0;
            if (tid < QUADS) {
                for (int k = 0; k < ranks; ++k) {
                    const uint4 v = part[k][tid];
                    c[0] += v.w, c[1] += v.z, c[2] += v.y, c[3] += v.x;
                }
                sum = c[0] + c[1] + c[2] + c[3];
            }
            const unsigned incl = warp_prefix(sum);
            if (lane == 31) sums[warp] = incl;
            __syncthreads();
            unsigned total, before = warps_before(sums, total) + incl - sum;
            if (tid < QUADS) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (need > before && need <= before + c[j]) {
                        sel[0] = (uint32_t)(4 * quad + 3 - j);
                        sel[1] = need - before;
                        sel[2] = c[j];
                    }
                    before += c[j];
                }
            }
            __syncthreads();
            prefix = prefix << bits | sel[0];
            need = sel[1];
            same = sel[2];
            counts = &hist[pass][sel[0]];
            if (need == same || shift == 0) break;
            // sel and sums are written again behind the next cluster barrier
        }
    }
    // ---- keep: a larger key, or an equal one among the first `need` of the row (all of them, mostly)
    unsigned rank0 = 0;                                    // equal keys in front of this warp's slots
    const bool ties = need != same;
    if (ties) {                                            // shift == 0: equal means equal
        unsigned cnt = 0;
        for (int g = 0; g < groups; ++g) {
            if (!REGS) load(g);
#pragma unroll
            for (int j = 0; j < G; ++j) cnt += slot(g, j) < s1 && rel(key[j]) == prefix;
        }
        cnt = __reduce_add_sync(0xffffffffu, cnt);
        if (lane == 0) sums3[warp] = cnt;
        if (!counts) counts = &range[2];
        const unsigned in_front = __reduce_add_sync(0xffffffffu, lane < rank ? cluster_ld(cluster_addr(counts, lane)) : 0u);
        __syncthreads();
        unsigned total;
        rank0 = in_front + warps_before(sums3, total);
    }
    // bits of the kept slots among the group that is loaded; `e`: equal keys in front of the group
    auto keeps = [&](int g, unsigned& e) -> uint32_t {
        uint32_t kept = 0;
#pragma unroll
        for (int j = 0; j < G; ++j) {
            const bool in = slot(g, j) < s1;
            const uint32_t k = rel(key[j]) >> shift;
            bool keep = in && k >= prefix;
            if (ties) {
                const unsigned eq = __ballot_sync(0xffffffffu, in && k == prefix);
                keep = in && (k > prefix || (k == prefix && e + __popc(eq & ((1u << lane) - 1)) < need));
                e += __popc(eq);
            }
            kept |= (uint32_t)keep << j;
        }
        return kept;
    };
    // freed slots and moving tokens of this warp, then of those in front of it
    unsigned freed = 0, moved = 0, e = rank0;
    uint32_t kept = 0;
    for (int g = 0; g < groups; ++g) {
        if (!REGS) load(g);
        kept = keeps(g, e);
#pragma unroll
        for (int j = 0; j < G; ++j) {
            const int s = slot(g, j);
            const bool keep = kept >> j & 1;
            freed += s < m && s < s1 && !keep;
            moved += s >= m && keep;
        }
    }
    freed = __reduce_add_sync(0xffffffffu, freed);
    moved = __reduce_add_sync(0xffffffffu, moved);
    if (lane == 0) sums[warp] = freed, sums2[warp] = moved;
    __syncthreads();
    unsigned all_freed, all_moved;
    unsigned at_freed = warps_before(sums, all_freed), at_moved = warps_before(sums2, all_moved);
    if (tid == 0) totals[0] = all_freed, totals[1] = all_moved;
    cluster_sync(ranks);
    const unsigned tf = lane < ranks ? cluster_ld(cluster_addr(&totals[0], lane)) : 0u,
                   tm = lane < ranks ? cluster_ld(cluster_addr(&totals[1], lane)) : 0u;
    at_freed += __reduce_add_sync(0xffffffffu, lane < rank ? tf : 0u);
    at_moved += __reduce_add_sync(0xffffffffu, lane < rank ? tm : 0u);
    const unsigned row_moved = __reduce_add_sync(0xffffffffu, tm);
    const long long row = (long long)b * a.Hkv + h;
    int* dst = p.moves + row * 4 * p.max_moves;
    int* src = dst + p.max_moves;
    int* src_pos = src + p.max_moves;
    int* src_w = src_pos + p.max_moves;
    e = rank0;
    for (int g = 0; g < groups; ++g) {
        if (!REGS) {
            load(g);
            kept = keeps(g, e);
        }
#pragma unroll
        for (int j = 0; j < G; ++j) {
            const int s = slot(g, j);
            const bool keep = kept >> j & 1, hole = s < m && s < s1 && !keep, mover = s >= m && keep;
            const unsigned holes = __ballot_sync(0xffffffffu, hole), movers = __ballot_sync(0xffffffffu, mover);
            const unsigned front = (1u << lane) - 1;
            if (hole) dst[at_freed + __popc(holes & front)] = s;
            if (mover) {
                const unsigned i = at_moved + __popc(movers & front);
                src[i] = s;
                src_pos[i] = q[j];
                src_w[i] = __float_as_int(wt[j]);
            }
            if (s < m) {
                if (keep) pos[s] = q[j];
            } else if (s < s1) {
                w[s] = 0.f;
                pos[s] = -1;
            }
            at_freed += __popc(holes);
            at_moved += __popc(movers);
        }
    }
    cluster_sync(ranks);                                        // the lists are complete
    // ---- moves: 32 tokens of a buffer, or of the weights and positions, per warp
    const long long batches = (row_moved + 31) / 32;
    for (long long x = rank * kEvictWarps + warp; x < batches * (a.n_bufs + 1); x += ranks * kEvictWarps) {
        const int i0 = (int)(x / (a.n_bufs + 1)) * 32, j = (int)(x % (a.n_bufs + 1)) - 1, i = i0 + lane;
        const int count = min(32, (int)row_moved - i0);
        const int d = lane < count ? __ldcg(dst + i) : 0;
        if (j < 0) {
            if (lane < count) {
                pos[d] = __ldcg(src_pos + i);
                w[d] = __int_as_float(__ldcg(src_w + i));
            }
            continue;
        }
        const int s = lane < count ? __ldcg(src + i) : 0;
        const KvqEvictBuf& f = a.bufs[j];
        char* base = (char*)f.base + b * f.stride_b + h * f.stride_h;
        const unsigned long long al = (unsigned long long)f.base | (unsigned long long)f.stride_b | (unsigned long long)f.stride_h |
                                      (unsigned long long)f.stride_s | (unsigned long long)f.row_bytes;
        if ((al & 15) == 0) move_rows<uint4>(f, base, s, d, count);
        else if ((al & 7) == 0) move_rows<uint2>(f, base, s, d, count);
        else if ((al & 3) == 0) move_rows<uint32_t>(f, base, s, d, count);
        else if ((al & 1) == 0) move_rows<uint16_t>(f, base, s, d, count);
        else move_rows<uint8_t>(f, base, s, d, count);
    }
}

static int launch_evict(const EvictParams& p, int ranks, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ranks, p.a.Hkv, p.a.B);
    cfg.blockDim = dim3(kEvictThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ranks;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    return check_cuda(cudaLaunchKernelEx(&cfg, p.per_cta == kEvictRun ? evict_kernel<true> : evict_kernel<false>, p));
}

}  // namespace kvq

extern "C" size_t kvq_evict_workspace_bytes(int32_t B, int32_t Hkv, int32_t cap, int32_t budget) {
    if (B <= 0 || Hkv <= 0 || cap <= 0 || budget <= 0) return 256;
    const long long moves = cap - budget < budget ? cap - budget : budget;
    const size_t n = (size_t)B * Hkv * 4 * (moves > 0 ? moves : 0) * sizeof(int);
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
    for (int j = 0; j < a.n_bufs; ++j) {
        if (!a.bufs[j].base || a.bufs[j].row_bytes <= 0) return KVQ_EINVAL;
        if (a.bufs[j].row_bytes > (1 << 30)) return KVQ_ELIMIT;
    }
    if (a.Hkv > 65535 || a.B > 65535) return KVQ_ELIMIT;
    if (!a.workspace || (((uintptr_t)a.workspace) & 15) || a.workspace_bytes < kvq_evict_workspace_bytes(a.B, a.Hkv, a.cap, a.budget))
        return KVQ_EWORKSPACE;
    // every head of a row reads its length
    if (a.new_lengths < a.lengths + a.B && a.lengths < a.new_lengths + a.B) return KVQ_EINVAL;
    EvictParams p;
    p.a = a;
    p.moves = (int*)a.workspace;
    p.max_moves = a.cap - a.budget < a.budget ? a.cap - a.budget : a.budget;
    if (p.max_moves < 0) p.max_moves = 0;
    int ranks = 1;
    while (ranks < kEvictMaxCluster && a.cap > kEvictRun * ranks) ranks *= 2;
    const long long per = ((long long)a.cap + ranks - 1) / ranks, runs = per > 0 ? (per + kEvictRun - 1) / kEvictRun : 1;
    p.per_cta = (int)(runs * kEvictRun);                   // fits: cap / 8 + 4095
    return launch_evict(p, ranks, (cudaStream_t)stream);
}
