// Host side of kvq_span_attn: validation, choice of the kernel and of the cut, launches.
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <math.h>
#include <stdlib.h>

#include <atomic>

#include "kvq_internal.h"
#include "kvq_span.cuh"
#include "kvq_span_mma.cuh"

namespace kvq {

struct SpanPlan {
    SpanParams p;
    bool asym;
    int kind;               // 1 tensor-core kernel, 0 generic
    int ts;                 // tokens per tile
    long long rows;
    size_t o_bytes, ml_bytes, fin_bytes, logit_bytes;
    size_t total() const { return o_bytes + ml_bytes + fin_bytes + logit_bytes; }
};

static size_t pad256(size_t n) { return (n + 255) & ~(size_t)255; }

static bool span_side_ok(const KvqCacheSide& s, const KvqAttnArgs& a, bool asym) {
    if (!s.payload || (((uintptr_t)s.payload | (uintptr_t)s.pay_stride_b | (uintptr_t)s.pay_stride_h | (uintptr_t)s.pay_stride_s) & 15))
        return false;
    if (a.format != KVQ_FMT_FP16 && (!s.scale || (((uintptr_t)s.scale | (uintptr_t)s.zp) & 1))) return false;
    return !asym || s.zp;
}

static int max_visible_tiles(const SpanParams& p, int ts) {
    const long long ctx = p.a.max_ctx;
    if (p.window <= 0) return (int)((ctx + ts - 1) / ts);
    const long long win = p.window < ctx ? p.window : ctx;
    const long long snk = p.sinks < ctx - win ? p.sinks : ctx - win;
    const long long t = (snk + ts - 1) / ts + (win + ts - 1) / ts + 1;       // a window may start inside a tile
    const long long all = (ctx + ts - 1) / ts;
    return (int)(t < all ? t : all);
}

// ---- tensor-core kernel: eligibility, launch configuration, tensor maps
template <int FMT, bool ASYM, int GS, int D>
struct SpanTag {};

// Calls f(SpanTag<...>{}) for the instantiation of these arguments; KVQ_EUNSUPPORTED if there is none.
template <class F>
static int span_dispatch(const SpanParams& p, bool asym, F&& f) {
    const int fmt = p.a.format, gs = p.a.group_size, d = p.a.D;
#define KVQ_SPAN_CASE(FMT_, ASYM_, GS_, D_) \
    if (fmt == FMT_ && asym == ASYM_ && gs == GS_ && d == D_) return f(SpanTag<FMT_, ASYM_, GS_, D_>{});
#define KVQ_SPAN_GS(FMT_, ASYM_)                                                                                         \
    KVQ_SPAN_CASE(FMT_, ASYM_, 32, 128) KVQ_SPAN_CASE(FMT_, ASYM_, 64, 128) KVQ_SPAN_CASE(FMT_, ASYM_, 128, 128)         \
    KVQ_SPAN_CASE(FMT_, ASYM_, 32, 64) KVQ_SPAN_CASE(FMT_, ASYM_, 64, 64)
    KVQ_SPAN_CASE(KVQ_FMT_FP16, false, 128, 128)
    KVQ_SPAN_CASE(KVQ_FMT_FP16, false, 64, 64)
    KVQ_SPAN_GS(KVQ_FMT_INT8, false)
    KVQ_SPAN_GS(KVQ_FMT_INT8, true)
    KVQ_SPAN_GS(KVQ_FMT_INT4, false)
    KVQ_SPAN_GS(KVQ_FMT_INT4, true)
#undef KVQ_SPAN_GS
#undef KVQ_SPAN_CASE
    return KVQ_EUNSUPPORTED;
}

template <int FMT, bool ASYM, int GS, int D>
static int span_ctas_per_sm(SpanTag<FMT, ASYM, GS, D>, int& out) {
    // once per device: the shared-memory limit is an attribute of the function on that device
    static std::atomic<int> cached[64];
    int dev = 0;
    int rc = check_cuda(cudaGetDevice(&dev));
    if (rc) return rc;
    if (dev < 0 || dev >= 64) return KVQ_EUNSUPPORTED;
    int n = cached[dev].load(std::memory_order_relaxed);
    if (n == 0) {
        const size_t smem = SpanShape<FMT, ASYM, GS, D>::smem();
        rc = check_cuda(cudaFuncSetAttribute(span_mma_kernel<FMT, ASYM, GS, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        if (rc) return rc;
        rc = check_cuda(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, span_mma_kernel<FMT, ASYM, GS, D>, kSpanWarps * 32, smem));
        if (rc) return rc;
        if (n < 1) n = 1;
        cached[dev].store(n, std::memory_order_relaxed);
    }
    out = n;
    return KVQ_OK;
}

// Payload as (row bytes in 128-byte rows of `tpr` tokens, token rows, kv heads, batch rows or pages); box = 128 bytes x
// box_rows.  Rows at or beyond the extent are zero-filled by the copy engine.
static int span_map(CUtensorMap* map, const KvqCacheSide& sd, const KvqAttnArgs& a, const KvqPageTable& pg, int rb, int tpr, int box_rows) {
    EncodeTiledFn enc = encode_tiled_fn();
    if (!enc) return KVQ_EUNSUPPORTED;
    const int tokens = pg.table ? pg.page_size : a.max_ctx, major = pg.table ? pg.num_pages : a.B;
    const cuuint64_t rs = (cuuint64_t)tpr * sd.pay_stride_s;
    cuuint64_t dims[4] = {(cuuint64_t)(rb < 128 ? 128 : rb), (cuuint64_t)(tokens / tpr), (cuuint64_t)a.Hkv, (cuuint64_t)major};
    // a dimension of extent 1 never advances: any legal stride
    cuuint64_t strides[3] = {rs, a.Hkv > 1 ? (cuuint64_t)sd.pay_stride_h : rs, major > 1 ? (cuuint64_t)sd.pay_stride_b : rs};
    cuuint32_t box[4] = {128, (cuuint32_t)box_rows, 1, 1};
    cuuint32_t estr[4] = {1, 1, 1, 1};
    const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(sd.payload), dims, strides, box, estr,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? KVQ_OK : KVQ_EUNSUPPORTED;
}

// Tokens of one payload copy, 0 if the kernel cannot take the layout.  A copy must not cross a page, and must be at least
// 1024 bytes (the period of the swizzle).
template <int FMT, bool ASYM, int GS, int D>
static int span_box(SpanTag<FMT, ASYM, GS, D>, const SpanParams& p) {
    using S = SpanShape<FMT, ASYM, GS, D>;
    int box = S::TS;
    if (p.pg.table)
        while (box >= 16 && p.pg.page_size % box) box /= 2;
    return box >= 16 && box * (S::RB < 128 ? S::RB : 128) >= 1024 ? box : 0;
}

template <int FMT, bool ASYM, int GS, int D>
static int span_tile(SpanTag<FMT, ASYM, GS, D>) { return SpanShape<FMT, ASYM, GS, D>::TS; }

static bool span_mma_side(const KvqCacheSide& s, const SpanParams& p, int rb, int tpr, int ng) {
    const KvqAttnArgs& a = p.a;
    const int major = p.pg.table ? p.pg.num_pages : a.B;
    if (s.pay_stride_s < rb || (tpr > 1 && s.pay_stride_s != rb)) return false;
    if ((a.Hkv > 1 && s.pay_stride_h <= 0) || (major > 1 && s.pay_stride_b <= 0)) return false;
    if (s.pay_stride_s >= (1LL << 36) || s.pay_stride_h >= (1LL << 40) || s.pay_stride_b >= (1LL << 40)) return false;
    if (ng == 0) return true;
    return s.sc_stride_s == ng;
}

// Bytes, 16 at most, that all scale and zero-point rows are aligned to.
static int span_unit(const SpanParams& p) {
    const KvqAttnArgs& a = p.a;
    const int major = p.pg.table ? p.pg.num_pages : a.B;
    uintptr_t bits = 16;
    for (const KvqCacheSide* s : {&a.k, &a.v}) {
        bits |= (uintptr_t)s->scale | (uintptr_t)s->zp;
        if (a.Hkv > 1) bits |= (uintptr_t)(2 * s->sc_stride_h);
        if (major > 1) bits |= (uintptr_t)(2 * s->sc_stride_b);
    }
    return (int)(bits & (~bits + 1));
}

template <int FMT, bool ASYM, int GS, int D>
static bool span_mma_ok(SpanTag<FMT, ASYM, GS, D> tag, const SpanParams& p) {
    using S = SpanShape<FMT, ASYM, GS, D>;
    const KvqAttnArgs& a = p.a;
    if (getenv("KVQ_FORCE_GENERIC") || a.max_ctx < S::TPR || a.max_ctx > (1 << 28)) return false;    // slots x groups in 32 bits
    if (!(fabsf(a.sm_scale) > 0.f && fabsf(a.sm_scale) <= 1e30f)) return false;      // masked logits are -inf before the scale
    const int ng = S::F16 ? 0 : S::NG;
    return span_box(tag, p) && span_mma_side(a.k, p, S::RB, S::TPR, ng) && span_mma_side(a.v, p, S::RB, S::TPR, ng);
}

template <int FMT, bool ASYM, int GS, int D>
static int launch_span_mma(SpanTag<FMT, ASYM, GS, D> tag, const SpanParams& p, cudaStream_t st) {
    using S = SpanShape<FMT, ASYM, GS, D>;
    SpanMmaParams mp;
    mp.p = p;
    mp.box_tokens = span_box(tag, p);
    mp.unit = FMT == KVQ_FMT_FP16 ? 16 : span_unit(p);
    CUtensorMap kmap, vmap;
    int rc, n;
    if ((rc = span_ctas_per_sm(tag, n))) return rc;
    if ((rc = span_map(&kmap, p.a.k, p.a, p.pg, S::RB, S::TPR, mp.box_tokens / S::TPR))) return rc;
    if ((rc = span_map(&vmap, p.a.v, p.a, p.pg, S::RB, S::TPR, mp.box_tokens / S::TPR))) return rc;
    return launch_pdl(span_mma_kernel<FMT, ASYM, GS, D>, dim3(p.ctas), dim3(kSpanWarps * 32), S::smem(), st, mp, kmap, vmap);
}

static int span_plan(const KvqSpanAttnArgs& s, SpanPlan& pl) {
    const KvqAttnArgs& a = s.attn;
    if (a.B < 0 || a.Hq <= 0 || a.Hkv <= 0 || a.D <= 0 || a.max_ctx < 0) return KVQ_EINVAL;
    if (a.Hq % a.Hkv != 0) return KVQ_EINVAL;
    if (a.format != KVQ_FMT_FP16 && a.format != KVQ_FMT_INT8 && a.format != KVQ_FMT_INT4) return KVQ_EINVAL;
    if (a.D != 64 && a.D != 128 && a.D != 256) return KVQ_EUNSUPPORTED;
    int gs = a.group_size == -1 || a.format == KVQ_FMT_FP16 ? a.D : a.group_size;
    if (gs <= 0 || a.D % gs != 0 || gs % 8 != 0) return KVQ_EINVAL;
    pl.asym = a.k.zp != nullptr || a.v.zp != nullptr;
    if (pl.asym && a.format == KVQ_FMT_FP16) return KVQ_EINVAL;
    if (a.splits || a.stages || a.tail_tokens) return KVQ_EINVAL;
    if (a.n_out || a.q_chan_scale || a.part_o || a.part_m || a.part_l) return KVQ_EUNSUPPORTED;
    if (s.window < 0 || s.sinks < 0 || (s.sinks > 0 && s.window == 0)) return KVQ_EINVAL;
    if (s.weights && (s.pages.table || s.window > 0)) return KVQ_EUNSUPPORTED;
    if (s.pages.table) {
        if (s.pages.page_size <= 0 || s.pages.cols <= 0 || s.pages.num_pages <= 0) return KVQ_EINVAL;
        if ((long long)s.pages.cols * s.pages.page_size < a.max_ctx) return KVQ_EINVAL;
    }
    SpanParams& p = pl.p;
    p = SpanParams();
    p.a = a;
    p.a.group_size = gs;
    p.pg = s.pages;
    p.window = s.window;
    p.sinks = s.sinks;
    p.n_rep = a.Hq / a.Hkv;
    p.rep_chunks = (p.n_rep + kHeadsPerCta - 1) / kHeadsPerCta;
    p.hr = a.Hkv * p.rep_chunks;
    p.weights = s.weights;
    p.w_stride_b = s.w_stride_b;
    p.w_stride_h = s.w_stride_h;
    pl.kind = 0;
    pl.ts = kSpanGenericTS;
    int slots = device_sm_count() * 4;
    span_dispatch(p, pl.asym, [&](auto tag) {
        if (!span_mma_ok(tag, p)) return KVQ_OK;
        int n = 1;
        if (span_ctas_per_sm(tag, n)) n = 1;               // no device: the launch will say so
        pl.kind = 1;
        pl.ts = span_tile(tag);
        slots = device_sm_count() * n;
        return KVQ_OK;
    });
    pl.rows = (long long)a.B * p.hr;
    const long long per_row = max_visible_tiles(p, pl.ts);
    if (pl.rows * (per_row + 64) >= (1LL << 31) || pl.rows >= (1LL << 30) || a.B > 65535) return KVQ_ELIMIT;
    // Rows that are not cut need no join, and the next row's CTA starts while one ends.  That pays for rows of at most 256
    // tokens, and for longer ones when there are enough to fill the chip: INT8 256 rows of 1024 tokens 26 -> 21 us, 1024 rows of
    // 2048 106 -> 100 (of 1 to 2048: 75 -> 61); against it, 64 rows of 1024 tokens 11.6 -> 15.9, 256 of 4096 56 -> 63.
    const long long tokens = per_row * pl.ts;
    p.row_mode = tokens <= 256 || (2 * pl.rows >= slots && tokens <= 1024) || (pl.rows >= 2 * slots && tokens <= 2048);
    // Otherwise a CTA has at least one tile (the generic kernel: one for each warp), and the cut counts the work of starting
    // a row (q, lookups, writing the part) as one more tile, on long rows only: of short ones it would leave CTAs idle.
    // INT8 32 x 8 K, 148 x 3 CTAs: 60.4 us without it, 57.8 with; INT4 with zero-points 1 x 1.2 K tokens 11.4 without, 13.4.
    p.row_cost = p.row_mode ? 0 : pl.kind ? (per_row >= 16 ? 1 : 0) : 4;
    p.min_tiles = (pl.kind ? 1 : 4) + p.row_cost;
    long long ctas = (pl.rows * (per_row + p.row_cost) + p.min_tiles - 1) / p.min_tiles;
    p.ctas = p.row_mode ? (int)pl.rows : (int)(ctas < slots ? ctas : slots);
    const size_t parts = p.row_mode ? 0 : (size_t)p.ctas + pl.rows;
    pl.o_bytes = pad256(parts * kHeadsPerCta * a.D * sizeof(float));
    pl.ml_bytes = pad256(parts * kHeadsPerCta * 2 * sizeof(float));
    pl.fin_bytes = s.weights ? pad256((size_t)a.B * a.Hq * 2 * sizeof(float)) : 0;
    pl.logit_bytes = s.weights ? pad256((size_t)pl.rows * a.max_ctx * kHeadsPerCta * sizeof(float)) : 0;
    return KVQ_OK;
}

template <int FMT, bool ASYM, int D>
static int launch_span_generic(const SpanParams& p, cudaStream_t st) {
    const size_t dyn = (size_t)4 * kHeadsPerCta * D * sizeof(float);
    return launch_pdl(span_generic_kernel<FMT, ASYM, D>, dim3(p.ctas), dim3(128), dyn, st, p);
}
template <int FMT, bool ASYM>
static int span_generic_d(const SpanParams& p, cudaStream_t st) {
    switch (p.a.D) {
        case 64: return launch_span_generic<FMT, ASYM, 64>(p, st);
        case 128: return launch_span_generic<FMT, ASYM, 128>(p, st);
        default: return launch_span_generic<FMT, ASYM, 256>(p, st);
    }
}
static int span_generic(const SpanPlan& pl, cudaStream_t st) {
    const SpanParams& p = pl.p;
    if (p.a.format == KVQ_FMT_FP16) return span_generic_d<KVQ_FMT_FP16, false>(p, st);
    if (p.a.format == KVQ_FMT_INT8)
        return pl.asym ? span_generic_d<KVQ_FMT_INT8, true>(p, st) : span_generic_d<KVQ_FMT_INT8, false>(p, st);
    return pl.asym ? span_generic_d<KVQ_FMT_INT4, true>(p, st) : span_generic_d<KVQ_FMT_INT4, false>(p, st);
}

template <int TS>
static int span_join(const SpanParams& p, cudaStream_t st) {
    const dim3 grid(p.a.Hq, p.a.B);
    switch (p.a.D) {
        case 64: return launch_pdl(span_join_kernel<2, TS>, grid, dim3(kJoinThreads), 0, st, p);
        case 128: return launch_pdl(span_join_kernel<4, TS>, grid, dim3(kJoinThreads), 0, st, p);
        default: return launch_pdl(span_join_kernel<8, TS>, grid, dim3(kJoinThreads), 0, st, p);
    }
}

int span_error_flag(int reset) {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_span_error_flag, sizeof(int)) != cudaSuccess) return KVQ_ECUDA;
    if (reset && v) {
        const int z = 0;
        if (cudaMemcpyToSymbol(g_span_error_flag, &z, sizeof(int)) != cudaSuccess) return KVQ_ECUDA;
    }
    return v;
}

}  // namespace kvq

extern "C" size_t kvq_span_attn_workspace_bytes(const KvqSpanAttnArgs* args) {
    kvq::SpanPlan pl;
    if (!args || kvq::span_plan(*args, pl) != KVQ_OK) return 0;
    return pl.total() ? pl.total() : 256;
}

extern "C" int kvq_span_attn_kernel_kind(const KvqSpanAttnArgs* args) {
    kvq::SpanPlan pl;
    if (!args) return KVQ_EINVAL;
    const int rc = kvq::span_plan(*args, pl);
    return rc ? rc : pl.kind;
}

extern "C" int kvq_span_attn(const KvqSpanAttnArgs* args, kvq_stream_t stream) {
    using namespace kvq;
    if (!args) return KVQ_EINVAL;
    SpanPlan pl;
    int rc = span_plan(*args, pl);
    if (rc) return rc;
    SpanParams& p = pl.p;
    const KvqAttnArgs& a = p.a;
    if (a.B == 0) return KVQ_OK;
    if (!a.q || !a.out || (a.q_stride_b & 1) || (a.q_stride_h & 1) || (((uintptr_t)a.q) & 3)) return KVQ_EINVAL;
    if (a.max_ctx > 0 && (!span_side_ok(a.k, a, pl.asym) || !span_side_ok(a.v, a, pl.asym))) return KVQ_EINVAL;
    if (pl.total() && (!a.workspace || a.workspace_bytes < pl.total() || (((uintptr_t)a.workspace) & 15))) return KVQ_EWORKSPACE;
    char* ws = (char*)a.workspace;
    p.ws_o = (float*)ws;
    p.ws_ml = (float*)(ws + pl.o_bytes);
    p.fin = p.weights ? (float*)(ws + pl.o_bytes + pl.ml_bytes) : nullptr;
    p.logits = p.weights ? (float*)(ws + pl.o_bytes + pl.ml_bytes + pl.fin_bytes) : nullptr;
    cudaStream_t st = (cudaStream_t)stream;
    rc = pl.kind ? span_dispatch(p, pl.asym, [&](auto tag) { return launch_span_mma(tag, p, st); }) : span_generic(pl, st);
    if (rc) return rc;
    if (!p.row_mode) {
        switch (pl.ts) {
            case 32: rc = span_join<32>(p, st); break;
            case 64: rc = span_join<64>(p, st); break;
            case 128: rc = span_join<128>(p, st); break;
            default: rc = span_join<256>(p, st); break;
        }
        if (rc) return rc;
    }
    if (p.weights && a.max_ctx > 0)
        rc = launch_pdl(span_weights_kernel, dim3((a.max_ctx + 255) / 256, a.Hkv, a.B), dim3(256), 0, st, p);
    return rc;
}
