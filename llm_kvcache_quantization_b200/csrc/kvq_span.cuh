// Attention of one new token over the visible span of a paged or contiguous cache (kvq_span_attn): how the work is cut,
// the shape-agnostic kernel, the join and the accumulation of attention weights.
//
//   out[b,h] = sum_{s visible} e^(x_s - M) V^_s / sum_{s visible} e^(x_s - M),   x_s = sm_scale q.K^_s,  M = max x_s
//   visible  = { s < n : s >= n - window or s < sinks }
//
// Cut.  A row (batch row b, kv head, chunk of 8 query heads) is a list of token tiles of TS tokens: the tiles that the
// sinks touch, then the tiles from the window's first token to the last token.  The tiles of all rows, laid end to end,
// with a few imaginary ones in front of each row for what it costs to start and to end it, are divided into runs whose lengths
// differ by at most one, one per CTA of a single resident wave; a CTA walks the tiles of its run and leaves one unnormalised
// partial (o, m, l) per row that it met.  The partial of (CTA c, row r) has slot c + r: along the runs either c or r grows
// from one partial to the next, so slots are distinct and at most ctas + rows of them exist.  The join recomputes the cut
// and finds the CTAs of its row.  With one run per row (`row_mode`, short spans) the kernel writes the output itself and
// there is no join.  (Measured and not kept: the CTA that arrives last at a row joins it - atomics on one word by up to 74
// CTAs and one CTA reading all partials cost more than a second launch, 33 us against 19 for a window of 4 K tokens x 32 rows.)
#pragma once

#include <cuda_fp16.h>
#include <stdint.h>

#include "kvq_decode_generic.cuh"
#include "kvq_internal.h"

namespace kvq {

struct SpanParams {
    KvqAttnArgs a;
    KvqPageTable pg;
    int window, sinks;
    int n_rep, rep_chunks;
    int hr;                 // rows per batch row: Hkv * rep_chunks
    int ctas;               // runs the tiles are cut into
    int min_tiles;          // a run has at least this many units
    int row_cost;           // imaginary tiles in front of a row
    int row_mode;           // one run per row, direct output
    float* ws_o;            // [ctas + rows][8][D]
    float* ws_ml;           // [ctas + rows][8][2]   (m in log2 units, l)
    float* fin;             // [B * Hq][2]           (m in log2 units, 1 / l); weights only
    float* logits;          // [rows][max_ctx][8]    log2 units; weights only
    float* weights;
    long long w_stride_b, w_stride_h;
};

__device__ int g_span_error_flag = 0;    // bit 0: a bounded wait expired, bit 1: a page table entry outside the pool was met

struct RowView {
    int n;                  // cached tokens
    int wstart;             // first token of the window
    int sinks;              // tokens below this stay visible
    int sa;                 // tiles in front of the gap
    int wt0;                // first tile of the window
    int tiles;
};

template <int TS>
__device__ __forceinline__ RowView row_view(const SpanParams& p, int b) {
    RowView v;
    int n = p.a.context_lens ? p.a.context_lens[b] : p.a.max_ctx;
    n = max(0, min(n, p.a.max_ctx));
    v.n = n;
    v.wstart = p.window > 0 ? max(0, n - p.window) : 0;
    v.sinks = min(p.sinks, v.wstart);
    v.wt0 = v.wstart / TS;
    v.sa = min((v.sinks + TS - 1) / TS, v.wt0);
    v.tiles = n > 0 ? v.sa + (n + TS - 1) / TS - v.wt0 : 0;
    return v;
}
template <int TS>
__device__ __forceinline__ int tile_token(const RowView& v, int i) { return (i < v.sa ? i : v.wt0 + i - v.sa) * TS; }
__device__ __forceinline__ bool token_visible(const RowView& v, int tok) {
    return tok < v.n && (tok >= v.wstart || tok < v.sinks);
}
// every token of the tile is visible
template <int TS>
__device__ __forceinline__ bool tile_full(const RowView& v, int tok0) {
    return tok0 + TS <= v.n && (tok0 >= v.wstart || tok0 + TS <= v.sinks);
}

// The cut: runs 0 .. longer-1 have q + 1 tiles, the others q.
struct SpanCut {
    int runs, q, longer;
};
__device__ __forceinline__ SpanCut span_cut(const SpanParams& p, int total) {
    SpanCut k;
    k.runs = max(1, min(p.ctas, (int)((unsigned)total / (unsigned)p.min_tiles)));
    k.q = (unsigned)total / (unsigned)k.runs;
    k.longer = total - k.q * k.runs;
    return k;
}
__device__ __forceinline__ int span_first(const SpanCut& k, int c) { return c * k.q + min(c, k.longer); }
__device__ __forceinline__ int span_run_of(const SpanCut& k, int u) {          // the run of tile u
    const int edge = k.longer * (k.q + 1);
    return u < edge ? (unsigned)u / (unsigned)(k.q + 1) : k.longer + (int)((unsigned)(u - edge) / (unsigned)k.q);
}

// The run of CTA `cta`: `left` units (imaginary and real tiles) from unit `i` of row (b, hr); unit row_cost is the row's
// first tile.  Every warp finds it by itself: no barrier.
struct SpanCursor {
    int b, hr, i, left;
    int u;                  // the run's next unit in the count over all rows
    SpanCut cut;
};
template <int TS>
__device__ __forceinline__ int row_units(const SpanParams& p, int b) {
    const int t = row_view<TS>(p, b).tiles;
    return t > 0 ? t + p.row_cost : 0;
}
template <int TS>
__device__ __forceinline__ SpanCursor span_locate(const SpanParams& p, int cta) {
    SpanCursor c;
    c.b = c.hr = c.i = c.left = c.u = 0;
    c.cut.runs = c.cut.q = c.cut.longer = 0;
    if (p.row_mode) {
        c.b = cta / p.hr;
        c.hr = cta - c.b * p.hr;
        c.left = row_units<TS>(p, c.b);
        return c;
    }
    const int lane = threadIdx.x & 31;
    int sum = 0;
#pragma unroll 1
    for (int b = lane; b < p.a.B; b += 32) sum += row_units<TS>(p, b);
    sum = __reduce_add_sync(0xffffffffu, sum);
    const int total = sum * p.hr;
    if (total == 0) return c;
    c.cut = span_cut(p, total);
    if (cta >= c.cut.runs) return c;
    c.u = span_first(c.cut, cta);
    c.left = span_first(c.cut, cta + 1) - c.u;
    int before = 0;                                        // units of the batch rows in front of this group of 32
#pragma unroll 1
    for (int b0 = 0;; b0 += 32) {
        const int t = b0 + lane < p.a.B ? row_units<TS>(p, b0 + lane) * p.hr : 0;
        int incl = t;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += x;
        }
        const unsigned past = __ballot_sync(0xffffffffu, c.u < before + incl);
        if (past) {                                        // the first lane whose rows reach beyond unit u
            const int l = __ffs(past) - 1;
            const int off = c.u - before - __shfl_sync(0xffffffffu, incl - t, l);
            const int units = __shfl_sync(0xffffffffu, t, l) / p.hr;
            c.b = b0 + l;
            c.hr = off / units;
            c.i = off - c.hr * units;
            return c;
        }
        before += __shfl_sync(0xffffffffu, incl, 31);
    }
}
// Tiles [i0, i1) of the row of a cursor that belong to the run, and the units that it takes
struct SpanPiece {
    int i0, i1, units;
};
__device__ __forceinline__ SpanPiece span_piece(const SpanParams& p, const SpanCursor& c, const RowView& v) {
    SpanPiece s;
    const int end = min(v.tiles > 0 ? v.tiles + p.row_cost : 0, c.i + c.left);
    s.units = end - c.i;
    s.i0 = max(c.i - p.row_cost, 0);
    s.i1 = max(end - p.row_cost, 0);
    return s;
}
// Next row of a run (a row's tiles are used up): skips rows without tiles.
template <int TS>
__device__ __forceinline__ void span_next_row(const SpanParams& p, SpanCursor& c, RowView& v) {
    c.i = 0;
    if (++c.hr < p.hr) return;
    c.hr = 0;
    do {
        ++c.b;
        v = row_view<TS>(p, c.b);
    } while (v.tiles == 0);                                // only called with tiles left, so a row follows
}

// ---------------------------------------------------------------------------------------------------------------------
// Shape-agnostic kernel: any head size of 64 / 128 / 256, group size, page size and strides.  CUDA-core products; lane =
// token for q.K, lane = channel slice for P.V.  It is bound by its instructions (a few percent of the memory rate); the
// tensor-core kernel takes every layout that the package's caches and pools produce.
// ---------------------------------------------------------------------------------------------------------------------
constexpr int kSpanGenericTS = 32;

// N channels from d0 of one token row as fp32 values code * scale + zp (exact product, one rounding of the sum)
template <int FMT, bool ASYM, int N>
__device__ __forceinline__ void load_value(const char* row, int d0, float sc, float zp, float* out) {
    if (FMT == KVQ_FMT_FP16) {
        const __half* p = (const __half*)row + d0;
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float2 f = __half22float2(*(const __half2*)(p + i));
            out[i] = f.x;
            out[i + 1] = f.y;
        }
    } else if (FMT == KVQ_FMT_INT8) {
        const int8_t* p = (const int8_t*)row + d0;
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const char2 c = *(const char2*)(p + i);
            out[i] = ASYM ? fmaf((float)c.x, sc, zp) : (float)c.x * sc;
            out[i + 1] = ASYM ? fmaf((float)c.y, sc, zp) : (float)c.y * sc;
        }
    } else {
        const uint8_t* p = (const uint8_t*)row + d0 / 2;
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            const float x = (float)((int)(p[i] >> 4) - 8), y = (float)((int)(p[i] & 15) - 8);
            out[2 * i] = ASYM ? fmaf(x, sc, zp) : x * sc;
            out[2 * i + 1] = ASYM ? fmaf(y, sc, zp) : y * sc;
        }
    }
}

// Byte / element offset of token `tok` of batch row b inside a side's buffers: the batch row or page part, and the row in it.
__device__ __forceinline__ void token_place(const SpanParams& p, int b, int tok, long long& major, long long& minor) {
    if (!p.pg.table) {
        major = b;
        minor = tok;
        return;
    }
    const int blk = tok / p.pg.page_size;
    int page = p.pg.table[b * p.pg.stride_b + blk];
    if (page < 0 || page >= p.pg.num_pages) {
        atomicOr(&g_span_error_flag, 2);
        page = 0;
    }
    major = page;
    minor = tok - blk * p.pg.page_size;
}

template <int FMT, bool ASYM, int D>
__global__ void __launch_bounds__(128) span_generic_kernel(const SpanParams p) {
    constexpr int EPL = D / 32, NW = 4, H = kHeadsPerCta, TS = kSpanGenericTS;
    const KvqAttnArgs& a = p.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int gs = a.group_size;
    __shared__ float q_s[H][D];
    __shared__ float red_ml[NW][H][2];
    extern __shared__ float red_acc[];                     // [NW][H][D]
    pdl_wait();
    SpanCursor c = span_locate<TS>(p, blockIdx.x);
    if (c.left == 0 && !p.row_mode) return;
    const float qk_scale = a.sm_scale * kLog2e;
    RowView v = row_view<TS>(p, c.b);
    for (;;) {
        const int b = c.b, kvh = c.hr / p.rep_chunks, rc = c.hr - kvh * p.rep_chunks;
        const int h0 = kvh * p.n_rep + rc * H, nh = min(H, p.n_rep - rc * H);
        const int row = b * p.hr + c.hr;
        const SpanPiece pc = span_piece(p, c, v);
        if (pc.i0 < pc.i1 || p.row_mode) {                 // not only imaginary ones; uniform over the CTA
        __syncthreads();
        for (int i = tid; i < H * D; i += 128) {
            const int h = i / D, d = i % D;
            float x = 0.f;
            if (h < nh) {
                __half qv = ((const __half*)a.q)[b * a.q_stride_b + (h0 + h) * a.q_stride_h + d];
                if (a.inv_tau) qv = __hmul(qv, __float2half_rn(a.inv_tau[h0 + h]));
                x = __half2float(qv) * qk_scale;
            }
            q_s[h][d] = x;
        }
        __syncthreads();
        float m[H], l[H], acc[H][EPL];
#pragma unroll
        for (int h = 0; h < H; ++h) {
            m[h] = -INFINITY;
            l[h] = 0.f;
#pragma unroll
            for (int e = 0; e < EPL; ++e) acc[h][e] = 0.f;
        }
        for (int i = pc.i0 + warp; i < pc.i1; i += NW) {
            const int tok0 = tile_token<TS>(v, i), tok = tok0 + lane;
            const bool valid = token_visible(v, tok);
            float s[H];
#pragma unroll
            for (int h = 0; h < H; ++h) s[h] = 0.f;
            long long mj = 0, mn = 0;
            if (valid) {
                token_place(p, b, tok, mj, mn);
                const char* krow = (const char*)a.k.payload + mj * a.k.pay_stride_b + kvh * a.k.pay_stride_h + mn * a.k.pay_stride_s;
                const long long so = mj * a.k.sc_stride_b + kvh * a.k.sc_stride_h + mn * a.k.sc_stride_s;
                for (int d0 = 0; d0 < D; d0 += 8) {
                    float sc = 1.f, zp = 0.f, kf[8];
                    if (FMT != KVQ_FMT_FP16) sc = __half2float(((const __half*)a.k.scale)[so + d0 / gs]);
                    if (ASYM) zp = __half2float(((const __half*)a.k.zp)[so + d0 / gs]);
                    load_value<FMT, ASYM, 8>(krow, d0, sc, zp, kf);
#pragma unroll
                    for (int h = 0; h < H; ++h)
                        if (h < nh) {
#pragma unroll
                            for (int j = 0; j < 8; ++j) s[h] = fmaf(q_s[h][d0 + j], kf[j], s[h]);
                        }
                }
                if (p.logits) {
                    float* lg = p.logits + ((long long)row * a.max_ctx + tok) * H;
#pragma unroll
                    for (int h = 0; h < H; ++h)
                        if (h < nh) lg[h] = s[h];
                }
            }
#pragma unroll
            for (int h = 0; h < H; ++h) {
                if (h < nh) {
                    const float sv = valid ? s[h] : -INFINITY;
                    const float m_new = fmaxf(m[h], warp_max(sv));
                    const float m_ref = m_new == -INFINITY ? 0.f : m_new;    // nothing but -inf so far: e^-inf, not NaN
                    const float corr = exp2f(m[h] - m_ref);
                    const float pj = valid ? exp2f(sv - m_ref) : 0.f;
                    l[h] = l[h] * corr + warp_sum(pj);
#pragma unroll
                    for (int e = 0; e < EPL; ++e) acc[h][e] *= corr;
                    m[h] = m_new;
                    s[h] = pj;
                }
            }
            const unsigned vmask = __ballot_sync(0xffffffffu, valid);
            for (int j = 0; j < TS; ++j) {
                const long long jm = __shfl_sync(0xffffffffu, mj, j), jn = __shfl_sync(0xffffffffu, mn, j);
                float pj[H];
#pragma unroll
                for (int h = 0; h < H; ++h) pj[h] = __shfl_sync(0xffffffffu, s[h], j);
                if (!((vmask >> j) & 1)) continue;
                const char* vrow = (const char*)a.v.payload + jm * a.v.pay_stride_b + kvh * a.v.pay_stride_h + jn * a.v.pay_stride_s;
                const long long so = jm * a.v.sc_stride_b + kvh * a.v.sc_stride_h + jn * a.v.sc_stride_s + (lane * EPL) / gs;
                float sc = 1.f, zp = 0.f, vf[EPL];
                if (FMT != KVQ_FMT_FP16) sc = __half2float(((const __half*)a.v.scale)[so]);
                if (ASYM) zp = __half2float(((const __half*)a.v.zp)[so]);
                load_value<FMT, ASYM, EPL>(vrow, lane * EPL, sc, zp, vf);
#pragma unroll
                for (int h = 0; h < H; ++h)
                    if (h < nh) {
#pragma unroll
                        for (int e = 0; e < EPL; ++e) acc[h][e] = fmaf(pj[h], vf[e], acc[h][e]);
                    }
            }
        }
        // merge the warps, leave the partial or the output
#pragma unroll
        for (int h = 0; h < H; ++h) {
            if (lane == 0) { red_ml[warp][h][0] = m[h]; red_ml[warp][h][1] = l[h]; }
#pragma unroll
            for (int e = 0; e < EPL; ++e) red_acc[(warp * H + h) * D + lane * EPL + e] = acc[h][e];
        }
        __syncthreads();
        for (int i = tid; i < nh * D; i += 128) {
            const int h = i / D, d = i % D;
            float M = -INFINITY;
#pragma unroll
            for (int w = 0; w < NW; ++w) M = fmaxf(M, red_ml[w][h][0]);
            const float ref = M == -INFINITY ? 0.f : M;
            float o = 0.f, L = 0.f;
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                const float lw = red_ml[w][h][1];
                if (lw != 0.f) {                           // 0: no token, or nothing but -inf logits
                    const float wgt = exp2f(red_ml[w][h][0] - ref);
                    o += red_acc[(w * H + h) * D + d] * wgt;
                    L += lw * wgt;
                }
            }
            if (p.row_mode) {
                const float r = L != 0.f ? o / L : 0.f;
                ((__half*)a.out)[b * a.out_stride_b + (h0 + h) * a.out_stride_h + d] = __float2half_rn(r);
                if (d == 0 && p.fin) {
                    float* f = p.fin + 2 * ((long long)b * a.Hq + h0 + h);
                    f[0] = ref;
                    f[1] = L != 0.f ? 1.f / L : 0.f;
                }
            } else {
                const long long slot = (long long)blockIdx.x + row;
                p.ws_o[(slot * H + h) * D + d] = o;
                if (d == 0) { p.ws_ml[(slot * H + h) * 2] = M; p.ws_ml[(slot * H + h) * 2 + 1] = L; }
            }
        }
        }
        c.left -= pc.units;
        c.u += pc.units;
        if (c.left <= 0) break;                            // uniform
        span_next_row<TS>(p, c, v);
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// Join: CTA = (query head, batch row), 8 warps; warp w takes the row's partials w, w + 8, ..., a lane EPL channels, four
// partials in flight.  Latency bound: the cut (one round trip for the context lengths), then one or two for the partials.
// ---------------------------------------------------------------------------------------------------------------------
constexpr int kJoinThreads = 256;

template <int EPL, int TS>
__global__ void __launch_bounds__(kJoinThreads) span_join_kernel(const SpanParams p) {
    constexpr int D = EPL * 32, H = kHeadsPerCta, NW = kJoinThreads / 32, U = 4;
    pdl_launch_dependents();
    const KvqAttnArgs& a = p.a;
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    __shared__ float red[NW][D + 1];
    __shared__ float red_m[NW];
    // The cut, before the wait for the partials: this kernel starts only when every CTA of the one before is past its own
    // wait, so the lengths are there.
    const int tiles = row_view<TS>(p, b).tiles;
    int sum = 0, before = 0;
#pragma unroll 1
    for (int i = lane; i < a.B; i += 32) {
        const int t = row_units<TS>(p, i);
        sum += t;
        if (i < b) before += t;
    }
    sum = __reduce_add_sync(0xffffffffu, sum);
    before = __reduce_add_sync(0xffffffffu, before);
    const int kvh = h / p.n_rep, hk = h - kvh * p.n_rep, rc = hk / H, hl = hk - rc * H;
    const int hr = kvh * p.rep_chunks + rc, row = b * p.hr + hr;
    int c0 = 0, c1 = -1;
    if (tiles > 0) {
        const SpanCut cut = span_cut(p, sum * p.hr);
        const int first = before * p.hr + hr * (tiles + p.row_cost) + p.row_cost;
        c0 = span_run_of(cut, first);
        c1 = span_run_of(cut, first + tiles - 1);
    }
    pdl_wait();

    float M = -INFINITY, L = 0.f, acc[EPL];
#pragma unroll
    for (int e = 0; e < EPL; ++e) acc[e] = 0.f;
    for (int s0 = c0 + warp; s0 <= c1; s0 += U * NW) {
        float2 ml[U];
        float ov[U][EPL];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int s = s0 + u * NW;
            ml[u] = make_float2(-INFINITY, 0.f);
            if (s <= c1) {
                const long long slot = ((long long)s + row) * H + hl;
                ml[u] = *reinterpret_cast<const float2*>(p.ws_ml + slot * 2);
                const float* o = p.ws_o + slot * D + lane * EPL;
#pragma unroll
                for (int e = 0; e < EPL; e += 2) *reinterpret_cast<float2*>(&ov[u][e]) = *reinterpret_cast<const float2*>(o + e);
            }
        }
        float Mn = M;
#pragma unroll
        for (int u = 0; u < U; ++u) Mn = fmaxf(Mn, ml[u].x);
        const float ref = Mn == -INFINITY ? 0.f : Mn;
        const float c = exp2f(M - ref);
        L *= c;
#pragma unroll
        for (int e = 0; e < EPL; ++e) acc[e] *= c;
        M = Mn;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (s0 + u * NW <= c1 && ml[u].y != 0.f) {     // l = 0: nothing but -inf logits in that run
                const float w = exp2f(ml[u].x - ref);
                L += ml[u].y * w;
#pragma unroll
                for (int e = 0; e < EPL; ++e) acc[e] += ov[u][e] * w;
            }
        }
    }
    if (lane == 0) red_m[warp] = M;
    __syncthreads();
    float Mt = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) Mt = fmaxf(Mt, red_m[w]);
    const float ref = Mt == -INFINITY ? 0.f : Mt;
    const float c = exp2f(M - ref);
#pragma unroll
    for (int e = 0; e < EPL; ++e) red[warp][lane * EPL + e] = acc[e] * c;
    if (lane == 0) red[warp][D] = L * c;
    __syncthreads();
    float Lt = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) Lt += red[w][D];
    if (tid < D) {
        float o = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) o += red[w][tid];
        const float r = Lt != 0.f ? o / Lt : 0.f;
        ((__half*)a.out)[b * a.out_stride_b + h * a.out_stride_h + tid] = __float2half_rn(r);
    }
    if (tid == 0 && p.fin) {
        float* f = p.fin + 2 * ((long long)b * a.Hq + h);
        f[0] = ref;
        f[1] = Lt != 0.f ? 1.f / Lt : 0.f;
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// weights[b,k,s] += sum over the heads of kv head k of 2^(x_s - M_h) / l_h, one thread per token, heads in a fixed order.
// ---------------------------------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(256) span_weights_kernel(const SpanParams p) {
    constexpr int H = kHeadsPerCta;
    pdl_launch_dependents();
    pdl_wait();
    const KvqAttnArgs& a = p.a;
    const int kvh = blockIdx.y, b = blockIdx.z;
    const int n = a.context_lens ? max(0, min(a.context_lens[b], a.max_ctx)) : a.max_ctx;
    const int s = blockIdx.x * 256 + threadIdx.x;
    if (s >= n) return;
    const float* f = p.fin + 2 * ((long long)b * a.Hq + kvh * p.n_rep);
    float w = 0.f;
    for (int rc = 0; rc < p.rep_chunks; ++rc) {
        const int nh = min(H, p.n_rep - rc * H);
        const float* lg = p.logits + ((long long)(b * p.hr + kvh * p.rep_chunks + rc) * a.max_ctx + s) * H;
        float x[H];
        *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(lg);
        *reinterpret_cast<float4*>(x + 4) = *reinterpret_cast<const float4*>(lg + 4);
#pragma unroll
        for (int h = 0; h < H; ++h)
            if (h < nh) w = fmaf(exp2f(x[h] - f[2 * (rc * H + h)]), f[2 * (rc * H + h) + 1], w);
    }
    float* dst = p.weights + b * p.w_stride_b + kvh * p.w_stride_h + s;
    *dst += w;
}

}  // namespace kvq
