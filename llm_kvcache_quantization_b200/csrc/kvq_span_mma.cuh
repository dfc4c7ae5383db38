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
//   P.V   channels on M, heads on N, tokens on K.  V codes become exact signed fp16 (a sum over 10^5 tokens would feel an
//         offset), the V scale goes into P: for one group per token in fp32 before P is rounded to fp16 (one rounding,
//         2^-11 of p), for several groups as a product of fp16 pairs per group (a second rounding).  V zero-points are one
//         more mma, with the groups on M.
// Both roundings of P are relative as long as P scale_v stays in fp16's normal range, whatever the scales: probabilities are
// kept relative to r = max logit - e, with e such that 2^e scale_v <= 2^14 (2^e <= 2^15) for the largest scale met so far.  r
// only grows, so it takes the place of the running maximum in the online softmax and costs nothing per element.
//
// Copies.  Each of the 4 warps owns a ring of tiles and walks every fourth tile of the CTA's run: payload by
// cp.async.bulk.tensor (128-byte rows, 128-byte swizzle; rows shorter than that hold 2 or 4 tokens, longer ones are fetched
// as 2 halves), one copy per page piece of 16 / 32 / TS tokens, scales by 16-byte cp.async, all on the slot's mbarrier.  No
// producer warp and no CTA barrier inside a row.  Waits are bounded; an expired one raises bit 0 of the error flag.
#pragma once

#include "kvq_ptx.cuh"
#include "kvq_span.cuh"

namespace kvq {

constexpr int kSpanWarps = 4;
constexpr int kSpanMaxStages = 4;

template <int FMT, bool ASYM, int GS, int D>
struct SpanShape {
    static constexpr bool F16 = FMT == KVQ_FMT_FP16;
    static constexpr int RB = F16 ? 2 * D : FMT == KVQ_FMT_INT8 ? D : D / 2;   // payload bytes of a token
    static constexpr int TPR = RB < 128 ? 128 / RB : 1;                        // tokens per 128-byte row
    static constexpr int TS = RB < 128 ? 64 : 32;                              // tokens per tile
    static constexpr int NG = F16 ? 1 : D / GS;
    static constexpr int TILE = TS * RB;                                       // bytes of K (or V) of a tile
    static constexpr int SCB = F16 ? 0 : TS * NG * 2;                          // bytes of one scale tile
    static constexpr int SCT = (ASYM ? 4 : 2) * SCB;
    static constexpr size_t smem(int nstage) {
        const size_t ring = (size_t)kSpanWarps * nstage * (2 * TILE + SCT);
        const size_t red = (size_t)kSpanWarps * kHeadsPerCta * (D + 8) * 4;
        return (ring > red ? ring : red) + 1024;
    }
};

struct SpanMmaParams {
    SpanParams p;
    int nstage;
    int box_tokens;          // tokens of one payload copy: divides TS and the page
};

// shared-memory offset of 16-byte chunk c of token r inside a payload tile
template <int RB, int TS>
__device__ __forceinline__ uint32_t span_off(int r, int c) {
    if (RB >= 128) return (uint32_t)((c >> 3) * (TS * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4));
    constexpr int TPR = RB < 128 ? 128 / RB : 1;
    const int row = r / TPR, cc = (r % TPR) * (RB / 16) + c;
    return (uint32_t)(row * 128 + ((cc ^ (row & 7)) << 4));
}
__device__ __forceinline__ void sts128(uint32_t addr, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
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

template <int FMT, bool ASYM, int GS, int D>
__global__ void __launch_bounds__(kSpanWarps * 32, 4)
span_mma_kernel(const SpanMmaParams mp, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
    using S = SpanShape<FMT, ASYM, GS, D>;
    constexpr bool F16 = S::F16, I8 = FMT == KVQ_FMT_INT8;
    constexpr int RB = S::RB, TPR = S::TPR, TS = S::TS, NG = S::NG, TILE = S::TILE, SCB = S::SCB, SCT = S::SCT;
    constexpr int SUB = TS / 16, H = kHeadsPerCta;
    constexpr int NQ = D / 8;                                  // fragment registers of q
    constexpr float OFFSET = I8 ? 128.f : 8.f;
    const SpanParams& p = mp.p;
    const KvqAttnArgs& a = p.a;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, t = lane & 3;
    const int nstage = mp.nstage;

    extern __shared__ unsigned char smem_dyn[];
    unsigned char* smem = smem_dyn + ((1024u - (smem_u32(smem_dyn) & 1023u)) & 1023u);
    const uint32_t pay_u = smem_u32(smem) + (uint32_t)(warp * nstage * 2 * TILE);
    const uint32_t sc_u = smem_u32(smem) + (uint32_t)(kSpanWarps * nstage * 2 * TILE + warp * nstage * SCT);
    __shared__ __align__(8) unsigned long long bars[kSpanWarps][kSpanMaxStages];
    __shared__ float red_ml[kSpanWarps][H][2];
    __shared__ float red_w[kSpanWarps][H];
    __shared__ float red_tot[H][2];
    __shared__ int sh[kSpanWarps + 4];

    const uint32_t bar0 = smem_u32(&bars[warp][0]);
    if (lane == 0) {
        for (int s = 0; s < nstage; ++s) mbar_init(bar0 + 8 * s, F16 ? 1 : 33);      // expect_tx (+ 32 cp.async arrivals)
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&kmap) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&vmap) : "memory");
    }
    __syncwarp();
    pdl_wait();                                                // q, the cache, the lengths and the table

    SpanCursor cur = span_locate<TS, kSpanWarps * 32>(p, blockIdx.x, sh);
    if (cur.left == 0 && !p.row_mode) return;                  // uniform over the CTA
    RowView v = row_view<TS>(p, cur.b);
    const float scale2 = fabsf(a.sm_scale) * kLog2e * (F16 ? 1.f : 16777216.f);      // q carries the sign; 2^24: subnormals
    const int box = mp.box_tokens, nbox = TS / box;
    int issued = 0, taken = 0;                                 // tiles of this warp over the whole run: slot = count % nstage
    int islot = 0, tslot = 0;
    uint32_t tphase = 0;
    bool failed = false;

    for (;;) {
        const int b = cur.b, kvh = cur.hr / p.rep_chunks, rc = cur.hr - kvh * p.rep_chunks;
        const int h0 = kvh * p.n_rep + rc * H, nh = min(H, p.n_rep - rc * H);
        const long long row = (long long)b * p.hr + cur.hr;
        const int i0 = cur.i + warp, i1 = min(v.tiles, cur.i + cur.left);
        const int n_my = i0 < i1 && !failed ? (i1 - i0 + kSpanWarps - 1) / kSpanWarps : 0;

        // ---- request tile k of this warp's list
        auto issue = [&](int k) {
            const int tok0 = tile_token<TS>(v, i0 + k * kSpanWarps);
            const uint32_t pb = pay_u + islot * 2 * TILE, sb = sc_u + islot * SCT, bar = bar0 + 8 * islot;
            if (++islot == nstage) islot = 0;
            ++issued;
            // batch row or page, and the row in it, of the piece of `box` tokens that this lane's number names
            int page = b, prow = tok0 + lane * box;
            if (p.pg.table) {
                // pieces without a visible token hold nothing that is used (their pages may be gone): page 0 serves
                const int tok = prow;
                page = prow = 0;
                if (lane < nbox && tok < v.n && (tok + box > v.wstart || tok < v.sinks)) {
                    const int blk = tok / p.pg.page_size;
                    page = __ldg(p.pg.table + b * p.pg.stride_b + blk);
                    prow = tok - blk * p.pg.page_size;
                    if (page < 0 || page >= p.pg.num_pages) {
                        atomicOr(&g_span_error_flag, 2);
                        page = 0;
                    }
                }
            }
            if (lane == 0) mbar_expect_tx(bar, 2 * TILE);
            __syncwarp();
            if (lane < nbox) {
                const uint32_t off = lane * box * (RB < 128 ? RB : 128);
                const int y = prow / TPR;
                tma_load_4d(pb + off, &kmap, bar, 0, y, kvh, page);
                if (RB > 128) tma_load_4d(pb + TS * 128 + off, &kmap, bar, 128, y, kvh, page);
                tma_load_4d(pb + TILE + off, &vmap, bar, 0, y, kvh, page);
                if (RB > 128) tma_load_4d(pb + TILE + TS * 128 + off, &vmap, bar, 128, y, kvh, page);
            }
            if (!F16) {
                constexpr int CH = TS * NG / 8;                // 16-byte chunks of one scale tile
#pragma unroll
                for (int c0 = 0; c0 < CH; c0 += 32) {
                    const int c = c0 + lane;
                    const int ct = c * 8 / NG;                 // first token of the chunk, relative to the tile
                    int mj = b, mn = tok0 + ct, nbytes = 16;   // batch row or page, row, bytes inside the buffers
                    if (p.pg.table) {
                        const int bx = min(ct / box, nbox - 1);
                        mj = __shfl_sync(0xffffffffu, page, bx);
                        mn = __shfl_sync(0xffffffffu, prow, bx) + ct - bx * box;
                    } else {
                        nbytes = max(0, min(16, (a.max_ctx - mn) * 2 * NG));
                        if (nbytes == 0) mn = 0;
                    }
                    if (CH >= 32 || c < CH) {
                        const uint32_t dst = sb + 16 * c;
                        const long long ok_ = (long long)mj * a.k.sc_stride_b + (long long)kvh * a.k.sc_stride_h + (long long)mn * NG;
                        const long long ov_ = (long long)mj * a.v.sc_stride_b + (long long)kvh * a.v.sc_stride_h + (long long)mn * NG;
                        cp_async16(dst, (const __half*)a.k.scale + ok_, nbytes);
                        cp_async16(dst + SCB, (const __half*)a.v.scale + ov_, nbytes);
                        if (ASYM) {
                            cp_async16(dst + 2 * SCB, (const __half*)a.k.zp + ok_, nbytes);
                            cp_async16(dst + 3 * SCB, (const __half*)a.v.zp + ov_, nbytes);
                        }
                    }
                }
                cp_async_mbar_arrive(bar);
            }
        };
        __syncwarp();
        const int prolog = min(nstage - 1, n_my);
        for (int k = 0; k < prolog; ++k) issue(k);

        // ---- q fragments: lane (g, t) holds channels of head g in the channel order of the K fragments
        uint32_t qf[NQ];
        float qb[NG][2];                                       // -offset 2^-24 sum of the group's q, heads 2t and 2t+1
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
                    float s = qs[G] * (-OFFSET / 16777216.f);
                    s += __shfl_xor_sync(0xffffffffu, s, 1);
                    s += __shfl_xor_sync(0xffffffffu, s, 2);
                    qb[G][0] = __shfl_sync(0xffffffffu, s, 8 * t);
                    qb[G][1] = __shfl_sync(0xffffffffu, s, 8 * t + 4);
                }
            }
        }

        float r_run[2] = {-INFINITY, -INFINITY};               // max logit - e, log2 units, heads 2t and 2t+1
        float m_run[2] = {-INFINITY, -INFINITY};               // max logit
        float l_run[2] = {0.f, 0.f};
        float vlim = F16 ? INFINITY : 0.f;                     // largest |scale_v| that the present e allows
        float e_lift = F16 ? 14.f : 0.f;
        float o[D / 16][4];
        float oz[4] = {0.f, 0.f, 0.f, 0.f};                    // rows = groups: sum of P z
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[i][j] = 0.f;

        for (int k = 0; k < n_my; ++k) {
            __syncwarp();                                      // every lane has finished with the slot that is refilled next
            if (k + nstage - 1 < n_my) issue(k + nstage - 1);
            const bool ok = mbar_wait_bounded(bar0 + 8 * tslot, tphase);
            const uint32_t kb = pay_u + tslot * 2 * TILE, vb = kb + TILE;
            const uint32_t ksb = sc_u + tslot * SCT, vsb = ksb + SCB, kzb = ksb + 2 * SCB, vzb = ksb + 3 * SCB;
            if (++tslot == nstage) { tslot = 0; tphase ^= 1u; }
            ++taken;
            if (!__all_sync(0xffffffffu, ok)) {
                failed = true;
                break;
            }
            const int tok0 = tile_token<TS>(v, i0 + k * kSpanWarps);
            const bool partial = !tile_full<TS>(v, tok0);
            if (TPR > 1 && !p.pg.table) {
                // a last 128-byte row that the cache does not fill is outside the tensor map: fetch its tokens here
                const int whole = a.max_ctx / TPR * TPR, rest = a.max_ctx - whole;
                if (rest && tok0 + TS > whole) {               // uniform over the warp
                    constexpr int CPT = RB / 16;
                    if (lane < 2 * rest * CPT) {
                        const int side = lane >= rest * CPT, x = lane - side * rest * CPT, tk = whole + x / CPT, c = x % CPT;
                        const KvqCacheSide& cs = side ? a.v : a.k;
                        const uint4 w = *reinterpret_cast<const uint4*>((const char*)cs.payload + (long long)b * cs.pay_stride_b +
                                                                        (long long)kvh * cs.pay_stride_h + (long long)tk * RB + 16 * c);
                        sts128((side ? vb : kb) + span_off<RB, TS>(tk - tok0, c), w);
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // before the copy that refills the slot
                    }
                    __syncwarp();
                }
            }

            // ================= q.K
            float x[SUB][4];
#pragma unroll
            for (int sub = 0; sub < SUB; ++sub) {
                const int lrow = 16 * sub + ((lane >> 3) & 1) * 8 + (lane & 7);      // ldmatrix row of this lane
                if (F16) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) x[sub][j] = 0.f;
#pragma unroll
                    for (int j = 0; j < D / 16; ++j) {
                        uint32_t r[4];
                        ldmatrix_x4(kb + span_off<RB, TS>(lrow, 2 * j + (lane >> 4)), r);
                        mma16816(x[sub], r[0], r[1], r[2], r[3], qf[2 * j], qf[2 * j + 1]);
                    }
                } else {
                    float s0[NG], s1[NG];                      // scales of token rows g and g + 8
                    load_row_floats<NG>(ksb + (16 * sub + g) * NG * 2, s0);
                    load_row_floats<NG>(ksb + (16 * sub + 8 + g) * NG * 2, s1);
                    float acc[4];
#pragma unroll
                    for (int c = 0; c < RB / 16; c += 2) {
                        uint32_t r[4];
                        ldmatrix_x4(kb + span_off<RB, TS>(lrow, c + (lane >> 4)), r);
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            constexpr int CPG = I8 ? GS / 16 : GS / 32;        // 16-byte chunks per group
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
                                const uint32_t a0 = wa & 0x000F000Fu, a1 = wb & 0x000F000Fu, a2 = wa8 & 0x000F000Fu, a3 = wb8 & 0x000F000Fu;
                                if (cc % CPG == 0) mma16816_from(acc, a0, a1, a2, a3, qf[4 * cc], qf[4 * cc + 1], qb[G][0], qb[G][1]);
                                else mma16816(acc, a0, a1, a2, a3, qf[4 * cc], qf[4 * cc + 1]);
                                mma16816(acc, wa & 0x00F000F0u, wb & 0x00F000F0u, wa8 & 0x00F000F0u, wb8 & 0x00F000F0u, qf[4 * cc + 2],
                                         qf[4 * cc + 3]);
                            }
                            if (cc % CPG == CPG - 1) {
                                if (G == 0) {
                                    x[sub][0] = acc[0] * s0[G]; x[sub][1] = acc[1] * s0[G];
                                    x[sub][2] = acc[2] * s1[G]; x[sub][3] = acc[3] * s1[G];
                                } else {
                                    x[sub][0] = fmaf(acc[0], s0[G], x[sub][0]); x[sub][1] = fmaf(acc[1], s0[G], x[sub][1]);
                                    x[sub][2] = fmaf(acc[2], s1[G], x[sub][2]); x[sub][3] = fmaf(acc[3], s1[G], x[sub][3]);
                                }
                            }
                        }
                    }
                    if (ASYM) {
                        load_row_floats<NG>(kzb + (16 * sub + g) * NG * 2, s0);
                        load_row_floats<NG>(kzb + (16 * sub + 8 + g) * NG * 2, s1);
#pragma unroll
                        for (int G = 0; G < NG; ++G) {
                            const float z0 = s0[G] * (-1.f / OFFSET), z1 = s1[G] * (-1.f / OFFSET);
                            x[sub][0] = fmaf(z0, qb[G][0], x[sub][0]); x[sub][1] = fmaf(z0, qb[G][1], x[sub][1]);
                            x[sub][2] = fmaf(z1, qb[G][0], x[sub][2]); x[sub][3] = fmaf(z1, qb[G][1], x[sub][3]);
                        }
                    }
                }
            }
            if (p.logits) {
#pragma unroll
                for (int sub = 0; sub < SUB; ++sub)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int tok = tok0 + 16 * sub + 8 * e + g;
                        if (tok < v.n)
                            *reinterpret_cast<float2*>(p.logits + (row * a.max_ctx + tok) * H + 2 * t) =
                                make_float2(x[sub][2 * e] * scale2, x[sub][2 * e + 1] * scale2);
                    }
            }
            if (partial) {
#pragma unroll
                for (int sub = 0; sub < SUB; ++sub) {
                    const int ta = tok0 + 16 * sub + g;
                    if (!token_visible(v, ta)) x[sub][0] = x[sub][1] = -INFINITY;
                    if (!token_visible(v, ta + 8)) x[sub][2] = x[sub][3] = -INFINITY;
                }
            }

            // ================= online softmax
            float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int sub = 0; sub < SUB; ++sub) {
                mx[0] = fmaxf(mx[0], fmaxf(x[sub][0], x[sub][2]));
                mx[1] = fmaxf(mx[1], fmaxf(x[sub][1], x[sub][3]));
            }
#pragma unroll
            for (int off = 4; off <= 16; off <<= 1) {
                mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], off));
                mx[1] = fmaxf(mx[1], __shfl_xor_sync(0xffffffffu, mx[1], off));
            }
            if (!F16) {
                // the largest V scale of the tile: lane = TS * NG / 32 consecutive values
                constexpr int VPL = TS * NG / 32;              // 1, 2, 4 or 8 fp16 values per lane
                float vm = 0.f;
#pragma unroll
                for (int i = 0; i < VPL; ++i) {
                    const float s = fabsf(__half2float(__ushort_as_half((unsigned short)span_lds16(vsb + (lane * VPL + i) * 2))));
                    if (!partial || token_visible(v, tok0 + (lane * VPL + i) / NG)) vm = fmaxf(vm, s);
                }
                if (__any_sync(0xffffffffu, vm > vlim)) {
#pragma unroll
                    for (int off = 1; off <= 16; off <<= 1) vm = fmaxf(vm, __shfl_xor_sync(0xffffffffu, vm, off));
                    // smallest power of two >= vm (frexp: vm = f 2^ex, f in [0.5, 1)); at least 2^-1: 2^e <= 2^15
                    int ex;
                    frexpf(fminf(vm, 65504.f), &ex);
                    ex = max(ex, -1);
                    vlim = vm > 65504.f ? INFINITY : exp2f((float)ex);
                    e_lift = 14.f - (float)ex;
                }
            }
            float corr[2], rneg[2];
            bool changed = false;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                m_run[e] = fmaxf(m_run[e], mx[e] * scale2);
                const float r_new = m_run[e] == -INFINITY ? -INFINITY : m_run[e] - e_lift;
                const float ref = r_new == -INFINITY ? 0.f : r_new;      // nothing but -inf so far: p = 0, not NaN
                changed |= r_new != r_run[e];
                corr[e] = fast_exp2(r_run[e] - ref);           // exp2(-inf) = 0 on the first tile
                r_run[e] = r_new;
                rneg[e] = -ref;
            }
            float ps[2] = {0.f, 0.f};
            uint32_t pb[SUB][2];                               // P^T fragments; for NG == 1 with the V scale inside
            uint32_t pz[ASYM && NG == 1 ? SUB : 1][2];         // P^T without the scale, for the zero-points
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
                    if (partial) {                             // slots that are not visible may hold NaN scales
                        if (!token_visible(v, tok0 + 16 * sub + g)) va[0] = 0.f;
                        if (!token_visible(v, tok0 + 16 * sub + 8 + g)) vc[0] = 0.f;
                    }
                    p0 *= va[0]; p1 *= va[0]; p2 *= vc[0]; p3 *= vc[0];
                }
                pb[sub][0] = movmatrix_trans(pack_h2(p0, p1));     // tokens 2t, 2t+1 of head g
                pb[sub][1] = movmatrix_trans(pack_h2(p2, p3));     // tokens 2t+8, 2t+9
            }
            l_run[0] = fmaf(l_run[0], corr[0], ps[0]);
            l_run[1] = fmaf(l_run[1], corr[1], ps[1]);
            if (__any_sync(0xffffffffu, changed)) {
#pragma unroll
                for (int i = 0; i < D / 16; ++i) {
                    o[i][0] *= corr[0]; o[i][1] *= corr[1]; o[i][2] *= corr[0]; o[i][3] *= corr[1];
                }
                if (ASYM) { oz[0] *= corr[0]; oz[1] *= corr[1]; }
            }

            // ================= P.V
#pragma unroll
            for (int sub = 0; sub < SUB; ++sub) {
                uint32_t mlo = 0xffffffffu, mhi = 0xffffffffu;     // tokens (2t, 2t+1) and (2t+8, 2t+9) that are visible
                if (partial) {
                    const int tg = tok0 + 16 * sub + 2 * t;
                    mlo = (token_visible(v, tg) ? 0x0000ffffu : 0u) | (token_visible(v, tg + 1) ? 0xffff0000u : 0u);
                    mhi = (token_visible(v, tg + 8) ? 0x0000ffffu : 0u) | (token_visible(v, tg + 9) ? 0xffff0000u : 0u);
                }
                if (F16) {
                    const int vrow = 16 * sub + (lane >> 4) * 8 + (lane & 7);
#pragma unroll
                    for (int i = 0; i < D / 16; ++i) {
                        uint32_t r[4];
                        ldmatrix_x4_trans(vb + span_off<RB, TS>(vrow, 2 * i + ((lane >> 3) & 1)), r);
                        mma16816(o[i], r[0] & mlo, r[1] & mlo, r[2] & mhi, r[3] & mhi, pb[sub][0], pb[sub][1]);
                    }
                } else {
                    uint32_t pg[NG][2];
                    if (NG == 1) {
                        pg[0][0] = pb[sub][0];
                        pg[0][1] = pb[sub][1];
                    } else {
                        uint32_t sx[NG], sy[NG];
                        load_scale_pairs<NG>(vsb + (16 * sub + 2 * t) * 2 * NG, sx, mlo);
                        load_scale_pairs<NG>(vsb + (16 * sub + 2 * t + 8) * 2 * NG, sy, mhi);
#pragma unroll
                        for (int G = 0; G < NG; ++G) {
                            pg[G][0] = hmul2_u(pb[sub][0], sx[G]);
                            pg[G][1] = hmul2_u(pb[sub][1], sy[G]);
                        }
                    }
                    if (ASYM) {
                        uint32_t zlo = 0u, zhi = 0u;           // row g = group g: (z[2t], z[2t+1]), (z[2t+8], z[2t+9])
                        if (g < NG) {
                            const uint32_t za = vzb + ((16 * sub + 2 * t) * NG + g) * 2;
                            zlo = (span_lds16(za) | (span_lds16(za + 2 * NG) << 16)) & mlo;
                            zhi = (span_lds16(za + 16 * NG) | (span_lds16(za + 18 * NG) << 16)) & mhi;
                        }
                        mma16816(oz, zlo, 0u, zhi, 0u, NG == 1 ? pz[ASYM && NG == 1 ? sub : 0][0] : pb[sub][0],
                                 NG == 1 ? pz[ASYM && NG == 1 ? sub : 0][1] : pb[sub][1]);
                    }
                    const int lrow = 16 * sub + ((lane >> 3) & 1) * 8 + (lane & 7);
#pragma unroll
                    for (int c = 0; c < RB / 16; c += 2) {
                        uint32_t r[4];
                        ldmatrix_x4_trans(vb + span_off<RB, TS>(lrow, c + (lane >> 4)), r);
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int cc = c + e;
                            if (I8) {
                                const uint32_t X = r[2 * e] ^ 0x80808080u, Y = r[2 * e + 1] ^ 0x80808080u;
                                const int G = 16 * cc / GS;
                                mma16816(o[cc], i8pair_to_h2(X, 0x5240u), i8pair_to_h2(X, 0x5341u), i8pair_to_h2(Y, 0x5240u),
                                         i8pair_to_h2(Y, 0x5341u), pg[G][0], pg[G][1]);
                            } else {
                                const uint32_t X = r[2 * e], Y = r[2 * e + 1], X8 = X >> 8, Y8 = Y >> 8;
                                const int G = 32 * cc / GS;
                                mma16816(o[2 * cc], nib_hi_to_h2(X), nib_lo_to_h2(X), nib_hi_to_h2(Y), nib_lo_to_h2(Y), pg[G][0], pg[G][1]);
                                mma16816(o[2 * cc + 1], nib_hi_to_h2(X8), nib_lo_to_h2(X8), nib_hi_to_h2(Y8), nib_lo_to_h2(Y8), pg[G][0],
                                         pg[G][1]);
                            }
                        }
                    }
                }
            }
        }
        if (failed) {                                          // give the other copies in flight a chance to land
            if (lane == 0) atomicOr(&g_span_error_flag, 1);
            for (; taken < issued; ++taken) {
                mbar_wait_bounded(bar0 + 8 * tslot, tphase);
                if (++tslot == nstage) { tslot = 0; tphase ^= 1u; }
            }
        }

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
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            int d0, d1;                                        // channels of fragment rows g and g + 8
            if (F16) { d0 = 16 * i + g; d1 = d0 + 8; }
            else if (I8) { d0 = 16 * i + 2 * g; d1 = d0 + 1; }
            else { d0 = 32 * (i >> 1) + 4 * g + 2 * (i & 1); d1 = d0 + 1; }
            ra[(2 * t) * DR + d0] = o[i][0];
            ra[(2 * t + 1) * DR + d0] = o[i][1];
            ra[(2 * t) * DR + d1] = o[i][2];
            ra[(2 * t + 1) * DR + d1] = o[i][3];
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
        cur.left -= i1 - cur.i;
        if (cur.left <= 0) break;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();                                       // the ring may be written again
        span_next_row<TS>(p, cur, v);
    }
}

}  // namespace kvq
