// Host side of kvq_span_attn: validation, choice of the kernel and of the cut, launches.
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <stdlib.h>

#include "kvq_internal.h"
#include "kvq_span.cuh"

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
    if (a.format != KVQ_FMT_FP16 && !s.scale) return false;
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
    pl.rows = (long long)a.B * p.hr;
    const long long per_row = max_visible_tiles(p, pl.ts);
    if (pl.rows * per_row >= (1LL << 31) || pl.rows >= (1LL << 30) || a.B > 65535) return KVQ_ELIMIT;
    int slots = device_sm_count() * 4;
    // A run of fewer than 4 tiles leaves warps of the CTA without work; a row of at most 8 tiles (two per warp) is
    // not worth cutting: it takes one CTA, and the join is saved.
    p.min_tiles = 4;
    p.row_mode = per_row <= 8;
    long long ctas = (pl.rows * per_row + p.min_tiles - 1) / p.min_tiles;
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
    if ((rc = span_generic(pl, st))) return rc;
    if (!p.row_mode && (rc = span_join<kSpanGenericTS>(p, st))) return rc;
    if (p.weights && a.max_ctx > 0)
        rc = launch_pdl(span_weights_kernel, dim3((a.max_ctx + 255) / 256, a.Hkv, a.B), dim3(256), 0, st, p);
    return rc;
}
