// Inline-PTX helpers shared by the tensor-core attention kernels: mbarriers, TMA, ldmatrix / movmatrix, mma, packed fp16.
#pragma once

#include <cuda.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace kvq {

// cuTensorMapEncodeTiled, resolved at run time (the library links against the runtime only); nullptr if there is none
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_tiled_fn();

constexpr int kWaitLimit = 1 << 22;  // bounded mbarrier polling

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void mbar_init(uint32_t bar, int count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
        : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// try_wait that lets the hardware park the thread for up to `hint_ns` before it reports "not yet"
__device__ __forceinline__ bool mbar_try_wait_hint(uint32_t bar, uint32_t parity, uint32_t hint_ns) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}"
        : "=r"(ok) : "r"(bar), "r"(parity), "r"(hint_ns) : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool mbar_wait_bounded(uint32_t bar, uint32_t parity) {
    for (int i = 0; i < kWaitLimit; ++i)
        if (mbar_try_wait(bar, parity)) return true;
    return false;
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1,
                                            int c2, int c3) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
        ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int src_bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(src_bytes) : "memory");
}
__device__ __forceinline__ void cp_async_mbar_arrive(uint32_t bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void lds128(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void lds64(uint32_t addr, uint32_t (&r)[2]) {
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(addr));
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
    uint32_t d;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(sel));
    return d;
}
template <int LUT>
__device__ __forceinline__ uint32_t lop3(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, %4;" : "=r"(d) : "r"(a), "r"(b), "r"(c), "n"(LUT));
    return d;
}
__device__ __forceinline__ uint32_t h2_as_u32(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 u32_as_h2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }
__device__ __forceinline__ uint32_t hmul2_u(uint32_t a, uint32_t b) { return h2_as_u32(__hmul2_rn(u32_as_h2(a), u32_as_h2(b))); }
__device__ __forceinline__ uint32_t hadd2_u(uint32_t a, uint32_t b) { return h2_as_u32(__hadd2_rn(u32_as_h2(a), u32_as_h2(b))); }
__device__ __forceinline__ uint32_t hsub2_u(uint32_t a, uint32_t b) { return h2_as_u32(__hsub2_rn(u32_as_h2(a), u32_as_h2(b))); }
__device__ __forceinline__ uint32_t hfma2_u(uint32_t a, uint32_t b, uint32_t c) {
    return h2_as_u32(__hfma2(u32_as_h2(a), u32_as_h2(b), u32_as_h2(c)));
}
// exp2 on the special-function unit; ex2.approx(-inf) = +0
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
    return h2_as_u32(__floats2half2_rn(lo, hi));
}

// fp16 scales of the token pair (tok, tok+1), `NG` groups each, re-paired per group:
// out[G] = half2(s[tok][G], s[tok+1][G]); `addr` = shared address of s[tok][0]
template <int NG>
__device__ __forceinline__ void load_scale_pairs(uint32_t addr, uint32_t (&out)[NG], uint32_t mask) {
    if (NG == 1) {
        uint32_t w;
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(addr));
        out[0] = w & mask;
    } else if (NG == 2) {
        uint32_t r[2];
        lds64(addr, r);
        out[0] = prmt(r[0], r[1], 0x5410u) & mask;
        out[NG - 1] = prmt(r[0], r[1], 0x7632u) & mask;
    } else if (NG == 4) {
        uint32_t r[4];
        lds128(addr, r);
        out[0] = prmt(r[0], r[2], 0x5410u) & mask; out[1 % NG] = prmt(r[0], r[2], 0x7632u) & mask;
        out[2 % NG] = prmt(r[1], r[3], 0x5410u) & mask; out[3 % NG] = prmt(r[1], r[3], 0x7632u) & mask;
    } else {
        uint32_t ra[4], rb[4];
        lds128(addr, ra);
        lds128(addr + 16, rb);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            out[(2 * w) % NG] = prmt(ra[w], rb[w], 0x5410u) & mask;
            out[(2 * w + 1) % NG] = prmt(ra[w], rb[w], 0x7632u) & mask;
        }
    }
}
// the NG fp16 values of one token row as floats; `addr` = shared address of s[row][0]
template <int NG>
__device__ __forceinline__ void load_row_floats(uint32_t addr, float (&f)[NG]) {
    if (NG == 1) {
        unsigned short u;
        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(u) : "r"(addr));
        f[0] = __half2float(__ushort_as_half(u));
    } else if (NG == 2) {
        uint32_t w;
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(addr));
        const float2 v = __half22float2(u32_as_h2(w));
        f[0] = v.x; f[NG - 1] = v.y;
    } else {
        uint32_t r[2];
        lds64(addr, r);
        const float2 a = __half22float2(u32_as_h2(r[0])), b = __half22float2(u32_as_h2(r[1]));
        f[0] = a.x; f[1 % NG] = a.y; f[2 % NG] = b.x; f[3 % NG] = b.y;
    }
}

constexpr uint32_t kMagic = 0x64006400u;     // half2(1024, 1024)
constexpr uint32_t kH1152 = 0x64806480u;     // half2(1152, 1152)
constexpr uint32_t kH1032 = 0x64086408u;     // half2(1032, 1032)
constexpr uint32_t kHsixteenth = 0x2c002c00u;  // half2(1/16, 1/16)
constexpr uint32_t kHm72 = 0xd480d480u;      // half2(-72, -72)

// int8 pair -> exact fp16 pair.  `w` already has its sign bits flipped (w ^ 0x80808080), so
// a byte b holds code + 128 and 0x6400 | b is the fp16 number 1152 + code.
__device__ __forceinline__ uint32_t i8pair_to_h2(uint32_t w, uint32_t sel) {
    return hsub2_u(prmt(w, 0x64646464u, sel), kH1152);
}
// two nibbles (bits 0-3 of each 16-bit half) -> exact fp16 (nibble - 8)
__device__ __forceinline__ uint32_t nib_lo_to_h2(uint32_t w) {
    return hsub2_u(lop3<0xEA>(w, 0x000F000Fu, kMagic), kH1032);            // (w & m) | magic
}
// two nibbles in bits 4-7 of each half: (1024 + 16 n) / 16 - 72 = n - 8, exact in one fma
__device__ __forceinline__ uint32_t nib_hi_to_h2(uint32_t w) {
    return hfma2_u(lop3<0xEA>(w, 0x00F000F0u, kMagic), kHsixteenth, kHm72);
}

}  // namespace kvq
