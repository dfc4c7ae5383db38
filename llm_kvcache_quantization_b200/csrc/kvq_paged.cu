// kvq_paged_read: tokens of a paged cache -> fp16 [B, Hkv, T, D] (a chunk that was just appended, a prefix that a prompt
// shares, the whole of a sequence).
//
//   value = RN16(code * scale + zero_point): the product is exact in fp32, the sum is one fma.
//
// One thread = 8 consecutive channels of kReadUnroll tokens: 16 bytes written per token and 4 (INT4) to 16 (fp16) read,
// all loads issued before the first use.  Grid = (token tiles, head, side x batch row), so no thread divides by a head or
// batch count; the page of a token is one table entry, the same for all threads of a token.  A memory stream: bound by
// HBM for long reads, by the launch and two dependent loads (table, page) for short ones.
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "kvq_internal.h"

namespace kvq {

__device__ int g_paged_read_error_flag = 0;     // 1: a page table entry outside the table or the pool was met

constexpr int kReadThreads = 256;
constexpr int kReadUnroll = 4;

template <int FMT, bool ASYM>
__global__ void __launch_bounds__(kReadThreads) paged_read_kernel(const KvqPagedReadArgs a) {
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
    float sc[kReadUnroll], zp[kReadUnroll];
#pragma unroll
    for (int u = 0; u < kReadUnroll; ++u) {
        const int t = t0 + u * rows;
        w[u] = make_uint4(0u, 0u, 0u, 0u);
        if (FMT == KVQ_FMT_INT4) w[u].x = 0x88888888u;                   // code 0
        sc[u] = zp[u] = 0.f;
        if (t < len) {
            const long long pos = (long long)start + t;
            const int blk = pos >= 0 && pos <= 0x7fffffffLL ? (int)pos / a.pages.page_size : -1;
            int page = -1;
            if (blk >= 0 && blk < a.pages.cols) page = a.pages.table[b * a.pages.stride_b + blk];
            int row = (int)pos - blk * a.pages.page_size;
            if (page < 0 || page >= a.pages.num_pages) {
                g_paged_read_error_flag = 1;
                page = row = 0;
            }
            const char* p = (const char*)cs.payload + page * cs.pay_stride_b + h * cs.pay_stride_h + row * cs.pay_stride_s;
            if (FMT == KVQ_FMT_FP16) w[u] = *reinterpret_cast<const uint4*>(p + 16 * c);
            else if (FMT == KVQ_FMT_INT8) {
                const uint2 x = *reinterpret_cast<const uint2*>(p + 8 * c);
                w[u].x = x.x;
                w[u].y = x.y;
            } else w[u].x = *reinterpret_cast<const uint32_t*>(p + 4 * c);
            if (FMT != KVQ_FMT_FP16) {
                const long long so = page * cs.sc_stride_b + h * cs.sc_stride_h + row * cs.sc_stride_s + g;
                sc[u] = __half2float(((const __half*)cs.scale)[so]);
                if (ASYM) zp[u] = __half2float(((const __half*)cs.zp)[so]);
            }
        }
    }
#pragma unroll
    for (int u = 0; u < kReadUnroll; ++u) {
        const int t = t0 + u * rows;
        if (t >= a.T) continue;
        uint4 o = w[u];
        if (FMT != KVQ_FMT_FP16) {
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                int code;
                if (FMT == KVQ_FMT_INT8) code = (int)(int8_t)((j < 4 ? w[u].x : w[u].y) >> (8 * (j & 3)));
                else code = (int)((w[u].x >> (8 * (j >> 1) + ((j & 1) ? 0 : 4))) & 15u) - 8;     // channel 2i in the high nibble
                x[j] = ASYM ? fmaf((float)code, sc[u], zp[u]) : (float)code * sc[u];
            }
            __half2 y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = __floats2half2_rn(x[2 * j], x[2 * j + 1]);
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
    cudaStream_t st = (cudaStream_t)stream;
    if (a.format == KVQ_FMT_FP16) return launch_pdl(paged_read_kernel<KVQ_FMT_FP16, false>, grid, dim3(kReadThreads), 0, st, a);
    if (a.format == KVQ_FMT_INT8)
        return asym ? launch_pdl(paged_read_kernel<KVQ_FMT_INT8, true>, grid, dim3(kReadThreads), 0, st, a)
                    : launch_pdl(paged_read_kernel<KVQ_FMT_INT8, false>, grid, dim3(kReadThreads), 0, st, a);
    return asym ? launch_pdl(paged_read_kernel<KVQ_FMT_INT4, true>, grid, dim3(kReadThreads), 0, st, a)
                : launch_pdl(paged_read_kernel<KVQ_FMT_INT4, false>, grid, dim3(kReadThreads), 0, st, a);
}
