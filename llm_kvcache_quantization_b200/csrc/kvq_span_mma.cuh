// Tensor-core kernel of kvq_span_attn (head_dim 64 / 128; fp16, INT8 and packed INT4 caches, groups of 32 / 64 / 128
// channels, with or without zero-points; contiguous or paged).
//
// What bounds it: the cache is read once (every query head of a kv head shares the CTA), so HBM; the arithmetic per byte is
// what has to be kept small.  Per tile of TS tokens a warp issues
//   q.K   mma.sync m16n8k16, tokens on M, the <= 8 query heads on N.  A code enters as the fp16 SUBNORMAL code + offset
//         (offset 128 or 8, value (code + offset) 2^-24: one prmt / and, no conversion); the products stay per group, start
//         from -offset sum_group q (the C operand of the group's first mma) and are multiplied by the token's fp32 scale
//         afterwards.  Codes, q and products are exact; the offset costs one more bit of the fp32 sums.
//         Zero-points add z_group sum_group q.
//   P.V   channels on M, heads on N, tokens on K.  The V scale goes into P: for one group per token in fp32 before P is
//         rounded to fp16 (one rounding, 2^-11 of p), for several groups as an fma of fp16 pairs per group, with P in two
//         fp16 parts (rounded once too: with P in one part, rounded again by the product, INT4 outputs were off by 3.4e-4 rms, now 2.9e-4).  V codes enter with their offset as well; offset x sum P scale_v (one mma with a matrix of ones) is
//         taken out after every tile, so that a sum over 10^5 tokens does not carry it along.  V zero-points are one more
//         mma, with the groups on M.
// The sums of products with subnormal codes are exact to about 2^-14 of the largest p scale_v of 16 tokens in units of 2^-24:
// the tensor core aligns a product by the exponents of its operands, which for a subnormal one is that of 2^-14.  That is
// 2^-14 of an INT8 step; INT4 codes enter the product with V as 16 n, 2^-18 of a step (as n 2^-24 a channel whose heaviest
// tokens have code 0 was off by more than the rounding of P allows).
// The rounding of P is relative as long as P scale_v stays in fp16's normal range, whatever the scales: probabilities are
// 2^(x - r) with r = (a maximum of the logits x so far) - e, where e keeps 2^(e+3) scale_v <= 2^15 for the largest scale met
// so far, and r moves only when a logit exceeds it by e + 3: no maximum over the warp in most tiles.
// Copies.  A CTA walks tiles of 4 x TSW tokens, TSW per warp, through a ring of slots that each hold the K, the V and the
// scales of a tile.  One warp fetches a tile for all: payload by cp.async.bulk.tensor (128-byte rows, 128-byte swizzle; rows
// shorter than that hold 2 or 4 tokens, longer ones come as 2 halves), one copy per page piece that has a visible token or one
// for the tile; scales by cp.async.bulk, or 16 bytes a lane where pieces are of fewer than 64 tokens (copies of 32 to 256 bytes
// each keep the copy engine busy: INT8 32 x 8 K in pages of 16 65 us with them, 61 without; in pages of 64 54 and 55) or of
// contiguous rows that do not start on 16 bytes; all on the slot's mbarrier.  The warp that finishes a slot last refills it, so
// there is no producer warp and no barrier inside a row; every warp has looked up the pages of the tile that the slot takes
// next by then.  Waits are bounded; an expired one raises bit 0 of the error flag.
// Measured: INT8 32 x 8 K 52 us (5.2 TB/s), pages of 64 55, of 16 61; INT4 16 x 8 K 24.4 (2.8 TB/s); INT4 with zero-points and
// 32-channel groups 4 x 32 K 48.8 (3.4 TB/s), pages of 32 62; fp16 16 x 4 K 28.4 (4.7 TB/s).  INT8 and fp16 are bound by HBM with
// two slots per CTA in flight, INT4 by instructions (some 500 of 32 tokens and a warp, a third of them unpacking).
// (Measured and not kept, INT8 32 x 8 K / INT4 16 x 8 K, 60 / 28 us before: K and V parts in slots of their own 60 / 28, with
// 8 KB slots 64 / 36; a ring per warp 62 / 35.)
#pragma once

#include "kvq_ptx.cuh"
#include "kvq_span.cuh"

namespace kvq {

constexpr int kSpanWarps = 4;
constexpr int kSpanMaxSlots = 4;

template <int FMT, bool ASYM, int GS, int D>
struct SpanShape {
    static constexpr bool F16 = FMT == KVQ_FMT_FP16;
    static constexpr int RB = F16 ? 2 * D : FMT == KVQ_FMT_INT8 ? D : D / 2;   // payload bytes of a token
    static constexpr int TPR = RB < 128 ? 128 / RB : 1;                        // tokens per 128-byte row
    static constexpr int TSW = RB >= 256 ? 16 : RB >= 128 ? 32 : 64;           // tokens of a warp
    static constexpr int TS = kSpanWarps * TSW;                                // tokens of a tile
    static constexpr int NG = F16 ? 1 : D / GS;
    static constexpr int TILE = TS * RB;                                       // bytes of K (or V) of a tile
    static constexpr int SCB = F16 ? 0 : TS * NG * 2;                          // bytes of one scale table of a tile
    static constexpr int SCT = (ASYM ? 2 : 1) * SCB;                           // scales (and zero-points) of K, or of V
    static constexpr int SLOT = 2 * TILE;                                      // payload of a slot; the scales of all slots follow
    static constexpr int SLOTS = 2;
    // CTAs that registers have to allow on an SM: as many as shared memory has room for.
    // (INT4 4 x 32 K with zero-points / 16 x 8 K: 32 tokens a warp and 3 or 4 CTAs 54 / 26.6 us, 64 tokens 47 / 24.4; a window of
    // 16 K in 32-channel groups, one sequence: 3 CTAs 14.8 us, 2 12.4.  INT8 of 64 channels, 16 x 8 K: 39 -> 31.6.)
    static constexpr int CTAS = RB == 32 ? 4 : RB == 64 && NG == 4 ? 2 : 3;
    static constexpr size_t smem() {
        const size_t ring = (size_t)SLOTS * (SLOT + 2 * SCT);
        const size_t red = (size_t)kSpanWarps * kHeadsPerCta * (D + 8) * 4;
        return (ring > red ? ring : red) + 1024;
    }
};

struct SpanMmaParams {
    SpanParams p;
    int box_tokens;          // tokens of one payload copy: divides the tile and the page
    int unit;                // bytes that all scale rows are aligned to: 16, 8, 4 or 2
};

__device__ __forceinline__ void sts128(uint32_t addr, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void sts16(uint32_t addr, unsigned short v) {
    asm volatile("st.shared.u16 [%0], %1;" ::"r"(addr), "h"(v) : "memory");
}
// `bytes` (a multiple of 16) from 16-byte aligned global memory, counted on the barrier
__device__ __forceinline__ void span_bulk(uint32_t dst, const void* src, int bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

// by the calling thread; 2 bytes are waited for
__device__ __forceinline__ void span_cp_small(uint32_t dst, const void* src, int unit) {
    if (unit == 8) asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
    else if (unit == 4) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
    else sts16(dst, __ldg((const unsigned short*)src));
}
__device__ __forceinline__ void span_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ uint32_t span_lds32(uint32_t addr) {
    uint32_t w;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(addr));
    return w;
}
__device__ __forceinline__ uint32_t span_lds16(uint32_t addr) {
    unsigned short u;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(u) : "r"(addr));
    return u;
}
// c = a * b + (c0, c1, c0, c1): the first product of a group starts from the offset of its column (query head)
__device__ __forceinline__ void mma16816_from(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1, float c0, float c1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%10,%11};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
}

__device__ __forceinline__ uint32_t span_atom_add(uint32_t addr) {
    uint32_t old;
    asm volatile("atom.acq_rel.cta.shared.add.u32 %0, [%1], 1;" : "=r"(old) : "r"(addr) : "memory");
    return old;
}

template <int FMT, bool ASYM, int GS, int D>
__global__ void __launch_bounds__(kSpanWarps * 32, SpanShape<FMT, ASYM, GS, D>::CTAS)
span_mma_kernel(const SpanMmaParams mp, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
    using S = SpanShape<FMT, ASYM, GS, D>;
    constexpr bool F16 = S::F16, I8 = FMT == KVQ_FMT_INT8;
    constexpr int RB = S::RB, TPR = S::TPR, TS = S::TS, TSW = S::TSW, NG = S::NG, TILE = S::TILE, SCB = S::SCB, SCT = S::SCT;
    constexpr int SUB = TSW / 16, H = kHeadsPerCta, SLOT = S::SLOT, SLOTS = S::SLOTS;
    constexpr int NQ = D / 8;                                  // fragment registers of q
    constexpr int SUBSTEP = 16 * (RB < 128 ? RB : 128);        // bytes between 16-token pieces of a tile
    constexpr float OFFSET = I8 ? 128.f : 8.f;
    constexpr float U24 = 1.f / 16777216.f;
    const SpanParams& p = mp.p;
    const KvqAttnArgs& a = p.a;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, t = lane & 3;

    extern __shared__ unsigned char smem_dyn[];
    unsigned char* smem = smem_dyn + ((1024u - (smem_u32(smem_dyn) & 1023u)) & 1023u);
    const uint32_t ring_u = smem_u32(smem), scale_u = ring_u + SLOTS * SLOT;
    __shared__ __align__(8) unsigned long long bars[SLOTS];
    __shared__ uint32_t done[SLOTS];                      // warps that have finished with a slot
    __shared__ float red_ml[kSpanWarps][H][2];
    __shared__ float red_w[kSpanWarps][H];
    __shared__ float red_tot[H][2];

    const int box = mp.box_tokens, nbox = TS / box;
    const int unit = mp.unit;
    const bool lanes = box < 64 || unit < 16;                  // scales come `unit` bytes a lane
    const uint32_t bar0 = smem_u32(&bars[0]), done0 = smem_u32(&done[0]);
    if (threadIdx.x == 0) {
        for (int s = 0; s < SLOTS; ++s) {
            mbar_init(bar0 + 8 * s, F16 || !lanes ? 1 : 33);   // the copies' bytes, and 32 lanes' scales
            done[s] = 0;
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&kmap) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&vmap) : "memory");
    }
    __syncthreads();
    pdl_wait();                                                // q, the cache, the lengths and the table

    SpanCursor cur = span_locate<TS>(p, blockIdx.x);
    if (cur.left == 0 && !p.row_mode) return;                  // uniform over the CTA
    RowView v = row_view<TS>(p, cur.b);
    const float scale2 = fabsf(a.sm_scale) * kLog2e * (F16 ? 1.f : 1.f / U24);       // q carries the sign; subnormal codes
    // ldmatrix addresses of this lane inside a slot; 16-byte chunk c of token piece `sub`: (slot + base) ^ (c << 4), plus
    // sub * SUBSTEP, plus TS * 128 for the second half of a 256-byte row
    uint32_t lk, lv;
    {
        auto base = [&](int r, int hi) -> uint32_t {           // token r of the warp's share, odd chunk or not
            if (RB >= 128) return (uint32_t)((warp * TSW + r) * 128 + ((hi ^ (r & 7)) << 4));
            const int row = r / TPR;
            return (uint32_t)((warp * TSW / TPR + row) * 128 + ((((r % TPR) * (RB / 16)) | hi) ^ (row & 7)) * 16);
        };
        lk = base(((lane >> 3) & 1) * 8 + (lane & 7), lane >> 4);
        lv = F16 ? base((lane >> 4) * 8 + (lane & 7), (lane >> 3) & 1) : lk;
    }
    auto chunk_addr = [&](uint32_t lane_slot, int sub, int c) -> uint32_t {
        uint32_t x = lane_slot ^ ((uint32_t)(c & 6) << 4);
        if (RB == 32 && (sub & 1)) x ^= 64u;                   // four tokens a row: the swizzle's row number moves by 4
        return x + sub * SUBSTEP + (RB > 128 ? (c >> 3) * (TS * 128) : 0);
    };
    // where the cache view ends, if the copies leave something of its last tokens out
    const int tail = !F16 && !p.pg.table && (a.max_ctx % TPR || (a.max_ctx * NG & ((unit >> 1) - 1))) ? a.max_ctx : -1;
    int slot = 0;
    uint32_t phase = 0;
    bool failed = false;

    for (;;) {
        const int b = cur.b, kvh = cur.hr / p.rep_chunks, rc = cur.hr - kvh * p.rep_chunks;
        const int h0 = kvh * p.n_rep + rc * H, nh = min(H, p.n_rep - rc * H);
        const long long row = (long long)b * p.hr + cur.hr;
        const SpanPiece pc = span_piece(p, cur, v);            // tiles i0 .. i1 - 1 of the row are this run's
        if (pc.i0 < pc.i1 || p.row_mode) {                     // not only imaginary ones
        const int ntile = pc.i1 - pc.i0;
        const int slot0 = slot;                                // slot of the row's first tile

        // Where piece `lane` (of `box` tokens) of tile k is: batch row or page, and the row in it
        int major, minor;
        bool vis;                                              // it has a visible token
        auto place = [&](int k) {
            const int tok = tile_token<TS>(v, pc.i0 + k) + lane * box;
            vis = k < ntile && lane < nbox && tok < v.n && (tok + box > v.wstart || tok < v.sinks);
            major = b;
            minor = tok;
            if (p.pg.table && vis) {
                const int blk = tok / p.pg.page_size;
                major = __ldg(p.pg.table + b * p.pg.stride_b + blk);
                minor = tok - blk * p.pg.page_size;
            }
        };
        // ---- request the tile that place() looked up into slot s; called by one whole warp
        auto issue = [&](int s) {
            const uint32_t dst = ring_u + s * SLOT, sb = scale_u + s * 2 * SCT, bar = bar0 + 8 * s;
            // scales of the piece; the last token row of a contiguous cache may end inside 16 bytes, see patch()
            int sbytes = 0, all = 0;
            if (vis) {
                if (p.pg.table && (major < 0 || major >= p.pg.num_pages)) {
                    atomicOr(&g_span_error_flag, 2);
                    major = 0;
                }
                if (!F16 && !lanes) sbytes = min(box, p.pg.table ? box : a.max_ctx - minor) * (2 * NG) & ~15;
                all = 2 * box * RB + (ASYM ? 4 : 2) * sbytes;
            }
            all = __reduce_add_sync(0xffffffffu, all);
            if (lane == 0) mbar_expect_tx(bar, all);
            __syncwarp();
            if (vis) {
                const uint32_t d = dst + lane * box * (RB < 128 ? RB : 128);
                tma_load_4d(d, &kmap, bar, 0, minor / TPR, kvh, major);
                if (RB > 128) tma_load_4d(d + TS * 128, &kmap, bar, 128, minor / TPR, kvh, major);
                tma_load_4d(d + TILE, &vmap, bar, 0, minor / TPR, kvh, major);
                if (RB > 128) tma_load_4d(d + TILE + TS * 128, &vmap, bar, 128, minor / TPR, kvh, major);
                if (!F16 && sbytes) {
                    const uint32_t ds = sb + lane * box * (2 * NG);
                    const long long ok_ = (long long)major * a.k.sc_stride_b + (long long)kvh * a.k.sc_stride_h + minor * NG;
                    const long long ov_ = (long long)major * a.v.sc_stride_b + (long long)kvh * a.v.sc_stride_h + minor * NG;
                    span_bulk(ds, (const __half*)a.k.scale + ok_, sbytes, bar);
                    span_bulk(ds + SCT, (const __half*)a.v.scale + ov_, sbytes, bar);
                    if (ASYM) {
                        span_bulk(ds + SCB, (const __half*)a.k.zp + ok_, sbytes, bar);
                        span_bulk(ds + SCT + SCB, (const __half*)a.v.zp + ov_, sbytes, bar);
                    }
                }
            }
            if (!F16 && lanes && unit < 16) {
                // rows of a contiguous cache whose slots do not fill 16 bytes of scales (what is left at its end: see patch())
                const int n = a.max_ctx * NG;
#pragma unroll 4
                for (int c0 = 0; c0 < SCB / unit; c0 += 32) {
                    const int el = (c0 + lane) * (unit >> 1), pi = el / NG / box & 31;
                    const bool on = __shfl_sync(0xffffffffu, (int)vis, pi) && c0 + lane < SCB / unit;
                    const int mj = __shfl_sync(0xffffffffu, major, pi), mn = __shfl_sync(0xffffffffu, minor, pi) * NG + el - pi * box * NG;
                    if (on && (p.pg.table || mn + (unit >> 1) <= n)) {
                        const uint32_t ds = sb + 2 * el;
                        const long long ok_ = (long long)mj * a.k.sc_stride_b + (long long)kvh * a.k.sc_stride_h + mn;
                        const long long ov_ = (long long)mj * a.v.sc_stride_b + (long long)kvh * a.v.sc_stride_h + mn;
                        span_cp_small(ds, (const __half*)a.k.scale + ok_, unit);
                        span_cp_small(ds + SCT, (const __half*)a.v.scale + ov_, unit);
                        if (ASYM) {
                            span_cp_small(ds + SCB, (const __half*)a.k.zp + ok_, unit);
                            span_cp_small(ds + SCT + SCB, (const __half*)a.v.zp + ov_, unit);
                        }
                    }
                }
                if (unit == 2) span_arrive(bar);
                else cp_async_mbar_arrive(bar);
            } else if (!F16 && lanes) {
                constexpr int CH = SCB / 16, TPC = 8 / NG; // chunks of a table, tokens of a chunk
#pragma unroll
                for (int c0 = 0; c0 < CH; c0 += 32) {
                    const int tok = (c0 + lane) * TPC, pi = tok / box & 31;
                    const bool on = __shfl_sync(0xffffffffu, (int)vis, pi) && c0 + lane < CH;
                    const int mj = __shfl_sync(0xffffffffu, major, pi), mn = __shfl_sync(0xffffffffu, minor, pi) + tok % box;
                    if (on) {
                        const uint32_t ds = sb + 16 * (c0 + lane);
                        const long long ok_ = (long long)mj * a.k.sc_stride_b + (long long)kvh * a.k.sc_stride_h + mn * NG;
                        const long long ov_ = (long long)mj * a.v.sc_stride_b + (long long)kvh * a.v.sc_stride_h + mn * NG;
                        cp_async16(ds, (const __half*)a.k.scale + ok_, 16);
                        cp_async16(ds + SCT, (const __half*)a.v.scale + ov_, 16);
                        if (ASYM) {
                            cp_async16(ds + SCB, (const __half*)a.k.zp + ok_, 16);
                            cp_async16(ds + SCT + SCB, (const __half*)a.v.zp + ov_, 16);
                        }
                    }
                }
                cp_async_mbar_arrive(bar);
            }
        };
        // What the copies leave out at the end of a contiguous cache, fetched with plain loads by the warp that owns the tokens:
        // a last 128-byte row that the cache does not fill (it lies outside the tensor map) and scales that do not fill a unit.
        auto patch = [&](const KvqCacheSide& cs, uint32_t dst, uint32_t sdst, int tok0) {
            const int whole = a.max_ctx / TPR * TPR, rest = a.max_ctx - whole;
            constexpr int CPT = RB / 16;
            if (lane < rest * CPT) {
                const int tk = whole + lane / CPT, c = lane % CPT, row_ = (tk - tok0) / TPR, cc = (tk % TPR) * CPT + c;
                const uint4 w = *reinterpret_cast<const uint4*>((const char*)cs.payload + (long long)b * cs.pay_stride_b +
                                                                (long long)kvh * cs.pay_stride_h + (long long)tk * RB + 16 * c);
                sts128(dst + row_ * 128 + ((cc ^ (row_ & 7)) << 4), w);
            }
            const int swhole = a.max_ctx * NG & -(unit >> 1), srest = a.max_ctx * NG - swhole;          // fp16 values
            if (lane < srest) {
                const long long off = (long long)b * cs.sc_stride_b + (long long)kvh * cs.sc_stride_h + swhole + lane;
                const uint32_t d = sdst + (swhole - tok0 * NG + lane) * 2;
                sts16(d, ((const unsigned short*)cs.scale)[off]);
                if (ASYM) sts16(d + SCB, ((const unsigned short*)cs.zp)[off]);
            }
        };
        // Tokens of the warp's share that are not visible may hold anything, NaN included.  Their logits become -inf, so P is
        // 0; what P is multiplied with is overwritten with zeros here (fp16: the V rows, else the V scales and zero-points).
        auto blank = [&](uint32_t vb, uint32_t vsb, int wtok) {
#pragma unroll 1
            for (int r = lane; r < TSW; r += 32) {
                if (token_visible(v, wtok + r)) continue;
                if (F16) {
                    const int rr = warp * TSW + r;
#pragma unroll 1
                    for (int c = 0; c < RB / 16; ++c)
                        sts128(vb + (c >> 3) * (TS * 128) + rr * 128 + (((c & 7) ^ (rr & 7)) << 4), make_uint4(0u, 0u, 0u, 0u));
                } else {
#pragma unroll 1
                    for (int j = 0; j < NG; ++j) {
                        sts16(vsb + (r * NG + j) * 2, 0);
                        if (ASYM) sts16(vsb + SCB + (r * NG + j) * 2, 0);
                    }
                }
            }
        };
        auto wait = [&]() {
            // after a wait that expired the results are void; the slot protocol goes on to the end, with a short limit, so that
            // no copy of this CTA is still in flight when it leaves
            bool ok = false;
            for (int i = failed ? kWaitLimit - 4096 : 0; i < kWaitLimit && !ok; ++i) ok = mbar_try_wait(bar0 + 8 * slot, phase);
            if (!__all_sync(0xffffffffu, ok) && !failed) {
                failed = true;
                if (lane == 0) atomicOr(&g_span_error_flag, 1);
            }
        };
        if (warp == 0) {
#pragma unroll 1
            for (int k = 0; k < min(SLOTS, ntile); ++k) {
                place(k);
                issue((slot0 + k) % SLOTS);
            }
        }

        // ---- q fragments: lane (g, t) holds channels of head g in the channel order of the K fragments
        uint32_t qf[NQ];
        float qb[F16 ? 1 : NG][2];                             // -offset 2^-24 sum of the group's q, heads 2t and 2t+1
        uint32_t qz[2] = {0u, 0u};                             // B fragment of the groups' sums of q: fp16 parts hi, lo
        {
            const bool hv = g < nh;
            const uint32_t* q32 = reinterpret_cast<const uint32_t*>((const __half*)a.q + (long long)b * a.q_stride_b +
                                                                    (long long)(h0 + (hv ? g : 0)) * a.q_stride_h);
            const uint32_t sign = a.sm_scale < 0.f ? 0x80008000u : 0u;
            const uint32_t tau2 = a.inv_tau ? h2_as_u32(__half2half2(__float2half_rn(a.inv_tau[h0 + (hv ? g : 0)]))) : 0u;
            auto ld = [&](int ch) -> uint32_t {                // channels ch, ch + 1 (ch even)
                uint32_t w = hv ? q32[ch >> 1] : 0u;
                if (a.inv_tau) w = hmul2_u(w, tau2);
                return w ^ sign;
            };
            float qs[NG];
#pragma unroll
            for (int G = 0; G < NG; ++G) qs[G] = 0.f;
            auto add = [&](float& s, uint32_t w, float f) {
                const float2 x = __half22float2(u32_as_h2(w));
                s += (x.x + x.y) * f;
            };
            if (F16) {
#pragma unroll
                for (int j = 0; j < D / 16; ++j) {
                    qf[2 * j] = ld(16 * j + 2 * t);
                    qf[2 * j + 1] = ld(16 * j + 8 + 2 * t);
                }
            } else if (I8) {
#pragma unroll
                for (int j = 0; j < D / 16; ++j) {
                    qf[2 * j] = ld(16 * j + 4 * t);
                    qf[2 * j + 1] = ld(16 * j + 4 * t + 2);
                    add(qs[16 * j / GS], qf[2 * j], 1.f);
                    add(qs[16 * j / GS], qf[2 * j + 1], 1.f);
                }
            } else {
#pragma unroll
                for (int j = 0; j < D / 32; ++j) {
                    const uint32_t w0 = ld(32 * j + 8 * t), w1 = ld(32 * j + 8 * t + 2), w2 = ld(32 * j + 8 * t + 4),
                                   w3 = ld(32 * j + 8 * t + 6);
                    qf[4 * j] = prmt(w0, w2, 0x7632u);          // odd channels: low nibbles
                    qf[4 * j + 1] = prmt(w1, w3, 0x7632u);
                    // even channels: high nibbles enter as 16 n, so q / 16 (exact down to q = 2^-10, off by 2^-25 below)
                    qf[4 * j + 2] = hmul2_u(prmt(w0, w2, 0x5410u), kHsixteenth);
                    qf[4 * j + 3] = hmul2_u(prmt(w1, w3, 0x5410u), kHsixteenth);
                    add(qs[32 * j / GS], qf[4 * j], 1.f);
                    add(qs[32 * j / GS], qf[4 * j + 1], 1.f);
                    add(qs[32 * j / GS], qf[4 * j + 2], 16.f);
                    add(qs[32 * j / GS], qf[4 * j + 3], 16.f);
                }
            }
            if (!F16) {
#pragma unroll
                for (int G = 0; G < NG; ++G) {
                    float s = qs[G];
                    s += __shfl_xor_sync(0xffffffffu, s, 1);
                    s += __shfl_xor_sync(0xffffffffu, s, 2);   // sum of q over group G, head g
                    qb[G][0] = __shfl_sync(0xffffffffu, s, 8 * t) * (-OFFSET * U24);
                    qb[G][1] = __shfl_sync(0xffffffffu, s, 8 * t + 4) * (-OFFSET * U24);
                    if (ASYM && (G >> 1) == t) {               // rows 2t, 2t+1 of the B fragment are groups 2t, 2t+1
                        const __half hi = __float2half_rn(s), lo = __float2half_rn(s - __half2float(hi));
                        qz[0] |= (uint32_t)__half_as_ushort(hi) << (16 * (G & 1));
                        qz[1] |= (uint32_t)__half_as_ushort(lo) << (16 * (G & 1));
                    }
                }
            }
        }

        float r_run[2] = {-INFINITY, -INFINITY};               // reference of the probabilities, log2 units, heads 2t, 2t+1
        float l_run[2] = {0.f, 0.f};
        float vlim = F16 ? INFINITY : 0.f;                     // largest |scale_v| that the present e allows
        float e_lift = 12.f;
        float o[D / 16][4];
        float oz[4] = {0.f, 0.f, 0.f, 0.f};                    // rows = groups: sum of P z
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[i][j] = 0.f;

        for (int k = 0; k < ntile; ++k) {
            if (p.pg.table) place(k + SLOTS);                  // the tile that takes this slot next
            const int tok0 = tile_token<TS>(v, pc.i0 + k), wtok = tok0 + warp * TSW;
            const bool partial = !tile_full<TSW>(v, wtok) || (tail > wtok && tail <= wtok + TSW);
            const bool active = wtok < v.n && (wtok + TSW > v.wstart || wtok < v.sinks);       // uniform over the warp

            // ================= q.K
            float x[SUB][4];
            wait();
            if (active) {
                const uint32_t kb = ring_u + slot * SLOT, ksb = scale_u + slot * 2 * SCT + warp * TSW * NG * 2, kzb = ksb + SCB;
                if (partial) {
                    if (tail > wtok && tail <= wtok + TSW) {
                        patch(a.k, kb, scale_u + slot * 2 * SCT, tok0);
                        patch(a.v, kb + TILE, scale_u + slot * 2 * SCT + SCT, tok0);
                        __syncwarp();
                    }
                    blank(kb + TILE, ksb + SCT, wtok);
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // before the copy that refills the slot
                    __syncwarp();
                }
                const uint32_t kl = kb + lk;
#pragma unroll
                for (int sub = 0; sub < SUB; ++sub) {
                    if (F16) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) x[sub][j] = 0.f;
#pragma unroll
                        for (int j = 0; j < D / 16; ++j) {
                            uint32_t r[4];
                            ldmatrix_x4(chunk_addr(kl, sub, 2 * j), r);
                            mma16816(x[sub], r[0], r[1], r[2], r[3], qf[2 * j], qf[2 * j + 1]);
                        }
                    } else {
                        float s0[NG], s1[NG];                  // scales of token rows g and g + 8
                        load_row_floats<NG>(ksb + (16 * sub + g) * NG * 2, s0);
                        load_row_floats<NG>(ksb + (16 * sub + 8 + g) * NG * 2, s1);
                        float xz[4];
                        if (ASYM) {
                            // z (16 tokens x groups) times the groups' sums of q: one mma over both fp16 parts of the sums
                            uint32_t za = 0u, zb = 0u;
                            if (NG == 1) {
                                if (t == 0) { za = span_lds16(kzb + (16 * sub + g) * 2); zb = span_lds16(kzb + (16 * sub + 8 + g) * 2); }
                            } else if (t < NG / 2) {
                                za = span_lds32(kzb + (16 * sub + g) * NG * 2 + 4 * t);
                                zb = span_lds32(kzb + (16 * sub + 8 + g) * NG * 2 + 4 * t);
                            }
                            mma16816_from(xz, za, zb, za, zb, qz[0], qz[1], 0.f, 0.f);
                        }
                        float acc[4];
#pragma unroll
                        for (int c = 0; c < RB / 16; c += 2) {
                            uint32_t r[4];
                            ldmatrix_x4(chunk_addr(kl, sub, c), r);
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                constexpr int CPG = I8 ? GS / 16 : GS / 32;    // 16-byte chunks per group
                                const int cc = c + e, G = cc / CPG;
                                const uint32_t wa = r[2 * e], wb = r[2 * e + 1];
                                if (I8) {
                                    const uint32_t ua = wa ^ 0x80808080u, ub = wb ^ 0x80808080u;
                                    const uint32_t a0 = prmt(ua, 0u, 0x4140u), a1 = prmt(ub, 0u, 0x4140u), a2 = prmt(ua, 0u, 0x4342u),
                                                   a3 = prmt(ub, 0u, 0x4342u);
                                    if (cc % CPG == 0) mma16816_from(acc, a0, a1, a2, a3, qf[2 * cc], qf[2 * cc + 1], qb[G][0], qb[G][1]);
                                    else mma16816(acc, a0, a1, a2, a3, qf[2 * cc], qf[2 * cc + 1]);
                                } else {
                                    const uint32_t wa8 = wa >> 8, wb8 = wb >> 8;
                                    const uint32_t a0 = wa & 0x000F000Fu, a1 = wb & 0x000F000Fu, a2 = wa8 & 0x000F000Fu,
                                                   a3 = wb8 & 0x000F000Fu;
                                    if (cc % CPG == 0) mma16816_from(acc, a0, a1, a2, a3, qf[4 * cc], qf[4 * cc + 1], qb[G][0], qb[G][1]);
                                    else mma16816(acc, a0, a1, a2, a3, qf[4 * cc], qf[4 * cc + 1]);
                                    mma16816(acc, wa & 0x00F000F0u, wb & 0x00F000F0u, wa8 & 0x00F000F0u, wb8 & 0x00F000F0u,
                                             qf[4 * cc + 2], qf[4 * cc + 3]);
                                }
                                if (cc % CPG == CPG - 1) {
                                    if (G == 0 && !ASYM) {
                                        x[sub][0] = acc[0] * s0[G]; x[sub][1] = acc[1] * s0[G];
                                        x[sub][2] = acc[2] * s1[G]; x[sub][3] = acc[3] * s1[G];
                                    } else if (G == 0) {
                                        x[sub][0] = fmaf(acc[0], s0[G], xz[0] * U24); x[sub][1] = fmaf(acc[1], s0[G], xz[1] * U24);
                                        x[sub][2] = fmaf(acc[2], s1[G], xz[2] * U24); x[sub][3] = fmaf(acc[3], s1[G], xz[3] * U24);
                                    } else {
                                        x[sub][0] = fmaf(acc[0], s0[G], x[sub][0]); x[sub][1] = fmaf(acc[1], s0[G], x[sub][1]);
                                        x[sub][2] = fmaf(acc[2], s1[G], x[sub][2]); x[sub][3] = fmaf(acc[3], s1[G], x[sub][3]);
                                    }
                                }
                            }
                        }
                    }
                }
            }
            // ================= online softmax
            uint32_t pb[SUB][2];                               // P^T fragments; for NG == 1 with the V scale inside
            uint32_t pl[!F16 && NG > 1 ? SUB : 1][2];          // what rounding to fp16 left of P; for several groups
            uint32_t pz[ASYM && NG == 1 ? SUB : 1][2];         // P^T without the scale, for the zero-points
            const uint32_t vb = ring_u + slot * SLOT + TILE, vsb = scale_u + slot * 2 * SCT + SCT + warp * TSW * NG * 2, vzb = vsb + SCB;
            if (active) {
                if (p.logits) {
#pragma unroll
                    for (int sub = 0; sub < SUB; ++sub)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int tok = wtok + 16 * sub + 8 * e + g;
                            if (tok < v.n)
                                *reinterpret_cast<float2*>(p.logits + (row * a.max_ctx + tok) * H + 2 * t) =
                                    make_float2(x[sub][2 * e] * scale2, x[sub][2 * e + 1] * scale2);
                        }
                }
                if (partial) {
#pragma unroll
                    for (int sub = 0; sub < SUB; ++sub) {
                        const int ta = wtok + 16 * sub + g;
                        if (!token_visible(v, ta)) x[sub][0] = x[sub][1] = -INFINITY;
                        if (!token_visible(v, ta + 8)) x[sub][2] = x[sub][3] = -INFINITY;
                    }
                }
                float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int sub = 0; sub < SUB; ++sub) {
                    mx[0] = fmaxf(mx[0], fmaxf(x[sub][0], x[sub][2]));
                    mx[1] = fmaxf(mx[1], fmaxf(x[sub][1], x[sub][3]));
                }
                float r_new[2] = {r_run[0], r_run[1]};
                bool moved = false;
                if (!F16) {
                    // the largest V scale of the share: TSW * NG / 32 consecutive values per lane
                    constexpr int VPL = TSW * NG / 32;         // 1, 2, 4 or 8
                    float vm = 0.f;
                    if (VPL >= 2) {
                        __half2 m2 = u32_as_h2(span_lds32(vsb + lane * VPL * 2) & 0x7fff7fffu);
#pragma unroll
                        for (int i = 1; i < VPL / 2; ++i) m2 = __hmax2(m2, u32_as_h2(span_lds32(vsb + lane * VPL * 2 + 4 * i) & 0x7fff7fffu));
                        const float2 f = __half22float2(m2);
                        vm = fmaxf(f.x, f.y);
                    } else {
#pragma unroll
                        for (int i = 0; i < VPL; ++i) {
                            const float s = fabsf(__half2float(__ushort_as_half((unsigned short)span_lds16(vsb + (lane * VPL + i) * 2))));
                            vm = fmaxf(vm, s);
                        }
                    }
                    if (__any_sync(0xffffffffu, vm > vlim)) {
#pragma unroll
                        for (int off = 1; off <= 16; off <<= 1) vm = fmaxf(vm, __shfl_xor_sync(0xffffffffu, vm, off));
                        // exponent of the power of two above vm; at least 0: 2^(e + 3) <= 2^15
                        const int ex = max((int)(__float_as_uint(fminf(vm, 65504.f)) >> 23) - 126, 0);
                        vlim = vm > 65504.f ? INFINITY : __uint_as_float((uint32_t)(ex + 127) << 23);
                        const float e_new = 12.f - (float)ex;
                        r_new[0] += e_lift - e_new;            // e only falls: P shrinks with it
                        r_new[1] += e_lift - e_new;
                        e_lift = e_new;
                        moved = true;
                    }
                }
                // P stays below 2^(e + 3): the reference moves only when a logit rises that far above the maximum that set it
                // (-inf - -inf = NaN compares false: nothing but -inf so far)
                const float over = fmaxf(mx[0] * scale2 - r_new[0], mx[1] * scale2 - r_new[1]);
                if (__any_sync(0xffffffffu, over > e_lift + 3.f)) {
#pragma unroll
                    for (int off = 4; off <= 16; off <<= 1) {
                        mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], off));
                        mx[1] = fmaxf(mx[1], __shfl_xor_sync(0xffffffffu, mx[1], off));
                    }
                    r_new[0] = fmaxf(r_new[0], mx[0] * scale2 - e_lift);
                    r_new[1] = fmaxf(r_new[1], mx[1] * scale2 - e_lift);
                    moved = true;
                }
                if (moved) {                                   // uniform over the warp
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        // exp2(-inf) = 0 the first time; a reference that stays -inf has nothing to scale
                        const float c = r_new[e] == r_run[e] ? 1.f : fast_exp2(r_run[e] - r_new[e]);
                        l_run[e] *= c;
#pragma unroll
                        for (int i = 0; i < D / 16; ++i) {
                            o[i][e] *= c;
                            o[i][2 + e] *= c;
                        }
                        if (ASYM) oz[e] *= c;
                        r_run[e] = r_new[e];
                    }
                }
                const float rneg[2] = {r_run[0] == -INFINITY ? 0.f : -r_run[0], r_run[1] == -INFINITY ? 0.f : -r_run[1]};
                float ps[2] = {0.f, 0.f};
#pragma unroll
                for (int sub = 0; sub < SUB; ++sub) {
                    float p0 = fast_exp2(fmaf(x[sub][0], scale2, rneg[0])), p1 = fast_exp2(fmaf(x[sub][1], scale2, rneg[1]));
                    float p2 = fast_exp2(fmaf(x[sub][2], scale2, rneg[0])), p3 = fast_exp2(fmaf(x[sub][3], scale2, rneg[1]));
                    ps[0] += p0 + p2;
                    ps[1] += p1 + p3;
                    if (!F16 && NG == 1) {
                        if (ASYM) {
                            pz[sub][0] = movmatrix_trans(pack_h2(p0, p1));
                            pz[sub][1] = movmatrix_trans(pack_h2(p2, p3));
                        }
                        float va[1], vc[1];
                        load_row_floats<1>(vsb + (16 * sub + g) * 2, va);
                        load_row_floats<1>(vsb + (16 * sub + 8 + g) * 2, vc);
                        p0 *= va[0]; p1 *= va[0]; p2 *= vc[0]; p3 *= vc[0];
                    }
                    const uint32_t h0 = pack_h2(p0, p1), h1 = pack_h2(p2, p3);
                    pb[sub][0] = movmatrix_trans(h0);          // tokens 2t, 2t+1 of head g
                    pb[sub][1] = movmatrix_trans(h1);          // tokens 2t+8, 2t+9
                    if (!F16 && NG > 1) {
                        const float2 f0 = __half22float2(u32_as_h2(h0)), f1 = __half22float2(u32_as_h2(h1));
                        pl[sub][0] = movmatrix_trans(pack_h2(p0 - f0.x, p1 - f0.y));
                        pl[sub][1] = movmatrix_trans(pack_h2(p2 - f1.x, p3 - f1.y));
                    }
                }
                l_run[0] += ps[0];
                l_run[1] += ps[1];

                // ================= P.V
                const uint32_t vl = vb + lv;
                float sp[NG][4];                               // sum of P scale_v over the tile, per group: heads 2t, 2t+1
#pragma unroll
                for (int sub = 0; sub < SUB; ++sub) {
                    if (F16) {
#pragma unroll
                        for (int i = 0; i < D / 16; ++i) {
                            uint32_t r[4];
                            ldmatrix_x4_trans(chunk_addr(vl, sub, 2 * i), r);
                            mma16816(o[i], r[0], r[1], r[2], r[3], pb[sub][0], pb[sub][1]);
                        }
                        continue;
                    }
                    uint32_t pg[NG][2];
                    if (NG == 1) {
                        pg[0][0] = pb[sub][0];
                        pg[0][1] = pb[sub][1];
                    } else {
                        uint32_t sx[NG], sy[NG];
                        load_scale_pairs<NG>(vsb + (16 * sub + 2 * t) * 2 * NG, sx, 0xffffffffu);
                        load_scale_pairs<NG>(vsb + (16 * sub + 2 * t + 8) * 2 * NG, sy, 0xffffffffu);
#pragma unroll
                        for (int G = 0; G < NG; ++G) {
                            pg[G][0] = hfma2_u(pb[sub][0], sx[G], hmul2_u(pl[sub][0], sx[G]));
                            pg[G][1] = hfma2_u(pb[sub][1], sy[G], hmul2_u(pl[sub][1], sy[G]));
                        }
                    }
                    constexpr uint32_t kOnes = 0x3c003c00u;
#pragma unroll
                    for (int G = 0; G < NG; ++G) {
                        if (sub == 0) mma16816_from(sp[G], kOnes, kOnes, kOnes, kOnes, pg[G][0], pg[G][1], 0.f, 0.f);
                        else mma16816(sp[G], kOnes, kOnes, kOnes, kOnes, pg[G][0], pg[G][1]);
                    }
                    if (ASYM) {
                        uint32_t zlo = 0u, zhi = 0u;           // row g = group g: (z[2t], z[2t+1]), (z[2t+8], z[2t+9])
                        if (g < NG) {
                            const uint32_t za = vzb + ((16 * sub + 2 * t) * NG + g) * 2;
                            zlo = span_lds16(za) | (span_lds16(za + 2 * NG) << 16);
                            zhi = span_lds16(za + 16 * NG) | (span_lds16(za + 18 * NG) << 16);
                        }
                        const int zs = ASYM && NG == 1 ? sub : 0;
                        mma16816(oz, zlo, 0u, zhi, 0u, NG == 1 ? pz[zs][0] : pb[sub][0], NG == 1 ? pz[zs][1] : pb[sub][1]);
                        if (NG > 1) mma16816(oz, zlo, 0u, zhi, 0u, pl[sub][0], pl[sub][1]);
                    }
#pragma unroll
                    for (int c = 0; c < RB / 16; c += 2) {
                        uint32_t r[4];
                        ldmatrix_x4_trans(chunk_addr(vl, sub, c), r);
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int cc = c + e;
                            if (I8) {
                                const uint32_t X = r[2 * e] ^ 0x80808080u, Y = r[2 * e + 1] ^ 0x80808080u;
                                const int G = 16 * cc / GS;
                                mma16816(o[cc], prmt(X, 0u, 0x4240u), prmt(X, 0u, 0x4341u), prmt(Y, 0u, 0x4240u), prmt(Y, 0u, 0x4341u),
                                         pg[G][0], pg[G][1]);
                            } else {
                                // both nibbles as 16 n: the sums of n 2^-24 keep 4 bits less
                                constexpr uint32_t M = 0x00F000F0u;
                                const uint32_t X = r[2 * e], Y = r[2 * e + 1];
                                const int G = 32 * cc / GS;
                                mma16816(o[2 * cc], X & M, (X << 4) & M, Y & M, (Y << 4) & M, pg[G][0], pg[G][1]);
                                mma16816(o[2 * cc + 1], (X >> 8) & M, (X >> 4) & M, (Y >> 8) & M, (Y >> 4) & M, pg[G][0], pg[G][1]);
                            }
                        }
                    }
                }
                if (!F16) {
                    // take the codes' offset out again, tile by tile: what is cancelled is never more than one tile's worth
#pragma unroll
                    for (int i = 0; i < D / 16; ++i) {
                        const int G = 16 * i / GS;
                        const float c = I8 ? OFFSET * U24 : 16.f * OFFSET * U24;
                        o[i][0] = fmaf(sp[G][0], -c, o[i][0]); o[i][1] = fmaf(sp[G][1], -c, o[i][1]);
                        o[i][2] = fmaf(sp[G][0], -c, o[i][2]); o[i][3] = fmaf(sp[G][1], -c, o[i][3]);
                    }
                }
            }
            // through with the slot: the last warp to say so fetches the tile that takes it next
            __syncwarp();
            uint32_t old = 0;
            if (lane == 0) old = span_atom_add(done0 + 4 * slot);
            old = __shfl_sync(0xffffffffu, old, 0);
            if (old == kSpanWarps - 1) {
                if (lane == 0) done[slot] = 0;
                __syncwarp();
                if (k + SLOTS < ntile) {
                    if (!p.pg.table) place(k + SLOTS);
                    issue(slot);
                }
            }
            if (++slot == SLOTS) { slot = 0; phase ^= 1u; }
        }

        if (cur.left <= pc.units) pdl_launch_dependents();     // the join may be set up; it waits for this kernel's end
        // ---- merge the warps through the ring's memory (every copy of this row has landed), leave the partial or the output
#pragma unroll
        for (int off = 4; off <= 16; off <<= 1) {
            l_run[0] += __shfl_xor_sync(0xffffffffu, l_run[0], off);
            l_run[1] += __shfl_xor_sync(0xffffffffu, l_run[1], off);
        }
        __syncthreads();
        constexpr int DR = D + 8;                              // row pitch: the 8-byte stores below spread over the banks
        float* red = reinterpret_cast<float*>(smem);           // [warp][head][DR]
        float* ra = red + warp * H * DR;
        if (g == 0) {
            red_ml[warp][2 * t][0] = r_run[0]; red_ml[warp][2 * t][1] = l_run[0];
            red_ml[warp][2 * t + 1][0] = r_run[1]; red_ml[warp][2 * t + 1][1] = l_run[1];
        }
        if (ASYM && g < NG) {
            ra[(2 * t) * DR + D + g] = oz[0];
            ra[(2 * t + 1) * DR + D + g] = oz[1];
        }
        constexpr float f0 = F16 ? 1.f : I8 ? 1.f / U24 : 1.f / (16.f * U24);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            int d0, d1;                                        // channels of fragment rows g and g + 8
            if (F16) { d0 = 16 * i + g; d1 = d0 + 8; }
            else if (I8) { d0 = 16 * i + 2 * g; d1 = d0 + 1; }
            else { d0 = 32 * (i >> 1) + 4 * g + 2 * (i & 1); d1 = d0 + 1; }
            ra[(2 * t) * DR + d0] = o[i][0] * f0;
            ra[(2 * t + 1) * DR + d0] = o[i][1] * f0;
            ra[(2 * t) * DR + d1] = o[i][2] * f0;
            ra[(2 * t + 1) * DR + d1] = o[i][3] * f0;
        }
        __syncthreads();
        if (threadIdx.x < H) {
            const int h = threadIdx.x;
            float M = -INFINITY, L = 0.f;
#pragma unroll
            for (int w = 0; w < kSpanWarps; ++w)
                if (red_ml[w][h][1] != 0.f) M = fmaxf(M, red_ml[w][h][0]);
#pragma unroll
            for (int w = 0; w < kSpanWarps; ++w) {
                const float lw = red_ml[w][h][1];
                const float wgt = lw != 0.f ? exp2f(red_ml[w][h][0] - (M == -INFINITY ? 0.f : M)) : 0.f;
                red_w[w][h] = wgt;
                if (lw != 0.f) L += lw * wgt;
            }
            red_tot[h][0] = M;
            red_tot[h][1] = L;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < nh * D; i += kSpanWarps * 32) {
            const int h = i / D, d = i % D;
            float ov = 0.f;
#pragma unroll
            for (int w = 0; w < kSpanWarps; ++w) {
                const float wgt = red_w[w][h];
                if (wgt != 0.f) {
                    float val = red[(w * H + h) * DR + d];
                    if (ASYM) val += red[(w * H + h) * DR + D + d / GS];
                    ov = fmaf(val, wgt, ov);
                }
            }
            const float M = red_tot[h][0], L = red_tot[h][1];
            if (p.row_mode) {
                ((__half*)a.out)[(long long)b * a.out_stride_b + (long long)(h0 + h) * a.out_stride_h + d] =
                    __float2half_rn(L != 0.f ? ov / L : 0.f);
                if (d == 0 && p.fin) {
                    float* f = p.fin + 2 * ((long long)b * a.Hq + h0 + h);
                    f[0] = M == -INFINITY ? 0.f : M;
                    f[1] = L != 0.f ? 1.f / L : 0.f;
                }
            } else {
                const long long slot = (long long)blockIdx.x + row;
                p.ws_o[(slot * H + h) * D + d] = ov;
                if (d == 0) { p.ws_ml[(slot * H + h) * 2] = M; p.ws_ml[(slot * H + h) * 2 + 1] = L; }
            }
        }
        }
        cur.left -= pc.units;
        cur.u += pc.units;
        if (cur.left <= 0) break;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();                                       // the ring may be written again
        span_next_row<TS>(p, cur, v);
    }
}

}  // namespace kvq
