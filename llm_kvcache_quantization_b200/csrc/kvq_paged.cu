// kvq_paged_read: tokens of a paged cache -> fp16 [B, Hkv, T, D] (a chunk that was just appended, a prefix that a prompt
// shares, the whole of a sequence).
//
//   value = RN16(code * scale + zero_point): one fp16 product or fma of the exact code, which rounds once.  A code becomes
//   fp16 as 1024 + offset + code (its bits under the exponent byte 0x64) minus 1024 + offset, both exact.
//
// One thread = 8 consecutive channels of kReadUnroll tokens: 16 bytes written per token and 4 (INT4) to 16 (fp16) read,
// all loads issued before the first use.  Grid = (token tiles, head, side x batch row), so no thread divides by a head or
// batch count; the page of a token is one table entry, the same for all threads of a token.  A memory stream: bound by
// HBM for long reads, by the launch and two dependent loads (table, page) for short ones.  INT4, 8 x 8 heads x 2048 tokens (83
// MB): 22 us, 3.8 TB/s; with fp32 arithmetic and a division per token it was bound by instructions, at 27.5 us.
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "kvq_internal.h"

namespace kvq {

__device__ int g_paged_read_error_flag = 0;     // 1: a page table entry outside the table or the pool was met

constexpr int kReadThreads = 256;
constexpr int kReadUnroll = 4;

struct ReadParams {
    KvqPagedReadArgs a;
    uint32_t div_mul;        // x / page_size = (umulhi(x, div_mul) + x) >> div_shift for x < 2^31
    int div_shift;
};

// Eight codes as fp16: two packed words for INT8, one for INT4 (code + 8, channel 2i in the high nibble of byte i).
template <int FMT>
__device__ __forceinline__ void codes_to_half(const uint4& w, __half2 (&y)[4]) {
    constexpr uint32_t kExp = 0x64646464u;                               // 1024 in each fp16
    uint32_t lo, hi;                                                     // codes + offset of channels 0..3 and 4..7
    if (FMT == KVQ_FMT_INT8) {
        lo = w.x ^ 0x80808080u;
        hi = w.y ^ 0x80808080u;
    } else {
        const uint32_t even = (w.x >> 4) & 0x0f0f0f0fu, odd = w.x & 0x0f0f0f0fu;
        lo = __byte_perm(even, odd, 0x5140);
        hi = __byte_perm(even, odd, 0x7362);
    }
    uint32_t x[4] = {__byte_perm(lo, kExp, 0x4140), __byte_perm(lo, kExp, 0x4342), __byte_perm(hi, kExp, 0x4140),
                     __byte_perm(hi, kExp, 0x4342)};
    const __half2 off = __float2half2_rn(FMT == KVQ_FMT_INT8 ? 1152.f : 1032.f);
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = __hsub2(*reinterpret_cast<__half2*>(&x[j]), off);
}

template <int FMT, bool ASYM>
__global__ void __launch_bounds__(kReadThreads) paged_read_kernel(const ReadParams p) {
    const KvqPagedReadArgs& a = p.a;
    pdl_launch_dependents();
    pdl_wait();
    const int chunks = a.D >> 3, rows = kReadThreads / chunks;           // D = 64 / 128 / 256: powers of two
    const int c = threadIdx.x & (chunks - 1), r = threadIdx.x / chunks;
    const int h = blockIdx.y;
    const int side = blockIdx.z >= (unsigned)a.B, b = blockIdx.z - (side ? a.B : 0);
    const KvqCacheSide& cs = side ? a.v : a.k;
    __half* out = (__half*)(side ? a.v_out : a.k_out) + b * a.out_stride_b + h * a.out_stride_h + 8 * c;
    const int len = a.lens ? max(0, min(a.T, a.lens[b])) : a.T;
    const int start = a.start_pos ? a.start_pos[b] : 0;
    const int t0 = blockIdx.x * rows * kReadUnroll + r;
    const int g = (8 * c) / a.group_size;
    uint4 w[kReadUnroll];
    __half sc[kReadUnroll], zp[kReadUnroll];
#pragma unroll
    for (int u = 0; u < kReadUnroll; ++u) {
        const int t = t0 + u * rows;
        w[u] = make_uint4(0u, 0u, 0u, 0u);
        if (FMT == KVQ_FMT_INT4) w[u].x = 0x88888888u;                   // code 0
        sc[u] = zp[u] = __ushort_as_half(0);
        if (t < len) {
            const long long pos = (long long)start + t;
            int page = -1, row = 0;
            if (pos >= 0 && pos <= 0x7fffffffLL) {
                const uint32_t x = (uint32_t)pos;
                const int blk = (int)((__umulhi(x, p.div_mul) + x) >> p.div_shift);
                if (blk < a.pages.cols) page = a.pages.table[b * a.pages.stride_b + blk];
                row = (int)x - blk * a.pages.page_size;
            }
            if (page < 0 || page >= a.pages.num_pages) {
                g_paged_read_error_flag = 1;
                page = row = 0;
            }
            const char* src = (const char*)cs.payload + page * cs.pay_stride_b + h * cs.pay_stride_h + row * cs.pay_stride_s;
            if (FMT == KVQ_FMT_FP16) w[u] = *reinterpret_cast<const uint4*>(src + 16 * c);
            else if (FMT == KVQ_FMT_INT8) {
                const uint2 x = *reinterpret_cast<const uint2*>(src + 8 * c);
                w[u].x = x.x;
                w[u].y = x.y;
            } else w[u].x = *reinterpret_cast<const uint32_t*>(src + 4 * c);
            if (FMT != KVQ_FMT_FP16) {
                const long long so = page * cs.sc_stride_b + h * cs.sc_stride_h + row * cs.sc_stride_s + g;
                sc[u] = ((const __half*)cs.scale)[so];
                if (ASYM) zp[u] = ((const __half*)cs.zp)[so];
            }
        }
    }
#pragma unroll
    for (int u = 0; u < kReadUnroll; ++u) {
        const int t = t0 + u * rows;
        if (t >= a.T) continue;
        uint4 o = w[u];
        if (FMT != KVQ_FMT_FP16) {
            __half2 y[4];
            codes_to_half<FMT>(w[u], y);
            const __half2 s2 = __half2half2(sc[u]), z2 = __half2half2(zp[u]);
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = ASYM ? __hfma2(y[j], s2, z2) : __hmul2(y[j], s2);
            o = *reinterpret_cast<uint4*>(y);
        }
        *reinterpret_cast<uint4*>(out + t * a.out_stride_t) = o;
    }
}

static bool read_side_ok(const KvqCacheSide& s, const KvqPagedReadArgs& a, bool asym) {
    if (!s.payload || (((uintptr_t)s.payload | (uintptr_t)s.pay_stride_b | (uintptr_t)s.pay_stride_h | (uintptr_t)s.pay_stride_s) & 15))
        return false;
    if (a.format != KVQ_FMT_FP16 && !s.scale) return false;
    return !asym || s.zp;
}

int paged_read_error_flag(int reset) {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_paged_read_error_flag, sizeof(int)) != cudaSuccess) return KVQ_ECUDA;
    if (reset && v) {
        const int z = 0;
        if (cudaMemcpyToSymbol(g_paged_read_error_flag, &z, sizeof(int)) != cudaSuccess) return KVQ_ECUDA;
    }
    return v;
}

}  // namespace kvq

extern "C" int kvq_paged_read(const KvqPagedReadArgs* args, kvq_stream_t stream) {
    using namespace kvq;
    if (!args) return KVQ_EINVAL;
    KvqPagedReadArgs a = *args;
    if (a.B < 0 || a.Hkv <= 0 || a.T < 0 || a.D <= 0) return KVQ_EINVAL;
    if (a.format != KVQ_FMT_FP16 && a.format != KVQ_FMT_INT8 && a.format != KVQ_FMT_INT4) return KVQ_EINVAL;
    if (a.D != 64 && a.D != 128 && a.D != 256) return KVQ_EUNSUPPORTED;
    if (a.group_size == -1 || a.format == KVQ_FMT_FP16) a.group_size = a.D;
    if (a.group_size <= 0 || a.D % a.group_size != 0 || a.group_size % 8 != 0) return KVQ_EINVAL;
    if (a.B == 0 || a.T == 0) return KVQ_OK;
    if (!a.pages.table || a.pages.page_size <= 0 || a.pages.cols <= 0 || a.pages.num_pages <= 0) return KVQ_EINVAL;
    if (!a.k_out || !a.v_out || (((uintptr_t)a.k_out | (uintptr_t)a.v_out) & 15)) return KVQ_EINVAL;
    if ((a.out_stride_b | a.out_stride_h | a.out_stride_t) & 7) return KVQ_EINVAL;
    const bool asym = a.k.zp || a.v.zp;
    if (asym && a.format == KVQ_FMT_FP16) return KVQ_EINVAL;
    if (!read_side_ok(a.k, a, asym) || !read_side_ok(a.v, a, asym)) return KVQ_EINVAL;
    const int rows = kReadThreads / (a.D / 8) * kReadUnroll;
    if (a.Hkv > 65535 || a.B > 32767) return KVQ_ELIMIT;
    const dim3 grid((a.T + rows - 1) / rows, a.Hkv, 2 * a.B);
    ReadParams p;
    p.a = a;
    p.div_shift = 0;
    while ((1LL << p.div_shift) < a.pages.page_size) ++p.div_shift;
    p.div_mul = (uint32_t)((((1ULL << p.div_shift) - a.pages.page_size) << 32) / a.pages.page_size + 1);
    cudaStream_t st = (cudaStream_t)stream;
    if (a.format == KVQ_FMT_FP16) return launch_pdl(paged_read_kernel<KVQ_FMT_FP16, false>, grid, dim3(kReadThreads), 0, st, p);
    if (a.format == KVQ_FMT_INT8)
        return asym ? launch_pdl(paged_read_kernel<KVQ_FMT_INT8, true>, grid, dim3(kReadThreads), 0, st, p)
                    : launch_pdl(paged_read_kernel<KVQ_FMT_INT8, false>, grid, dim3(kReadThreads), 0, st, p);
    return asym ? launch_pdl(paged_read_kernel<KVQ_FMT_INT4, true>, grid, dim3(kReadThreads), 0, st, p)
                : launch_pdl(paged_read_kernel<KVQ_FMT_INT4, false>, grid, dim3(kReadThreads), 0, st, p);
}
