// Writing token rows into the pages of a cache, quantised where the format asks for it, and
// reading them back.
//
// A group of a row (the whole row in 8 bits, 32 dimensions in 4) has one scale, stored in BF16:
//     s = bf16(max|x| / top),  c = clamp(round(x / s), -top, top),  x' = c s,   top = 127 or 7,
// c = 0 where s = 0.  The scale keeps BF16's 8 bits because its exponent range is FP32's (no
// input of any source type overflows it), and because the codes are computed against the
// rounded scale, so that its rounding moves the step by 0.4 % at most and adds no error of its
// own.  A group with an infinity or a NaN in it has no step: its scale is stored as NaN and the
// whole group reads back as NaN.  All of it is FP32 arithmetic with IEEE divisions.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "serving.h"

namespace bgtq {
namespace {

__device__ __forceinline__ float load_as_float(const void *p, int64_t i, bgtq_dtype t) {
    if (t == BGTQ_F32) return static_cast<const float *>(p)[i];
    if (t == BGTQ_F16) return __half2float(static_cast<const __half *>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
}
__device__ __forceinline__ void store_float(void *p, uint64_t i, float x, bgtq_dtype t) {
    if (t == BGTQ_F32) static_cast<float *>(p)[i] = x;
    else if (t == BGTQ_F16) static_cast<__half *>(p)[i] = __float2half_rn(x);
    else static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(x);
}

constexpr uint32_t kWarps = 4;

// One warp per (token, KV head) row, K rows in blockIdx.y = 0 and V rows in 1; lane l holds
// dimensions l, l + 32, ..., so register i of the warp is 4-bit group i.
template <int D>
__global__ void __launch_bounds__(32 * kWarps) write_rows_kernel(const PagedWriteArgs a) {
    constexpr int N = D / 32;
    const uint64_t row = (uint64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
    const uint32_t lane = threadIdx.x & 31u, H = a.c.heads;
    if (row >= a.tokens * H) return;
    const uint64_t t = row / H;
    const uint32_t h = (uint32_t)(row % H);
    const int64_t slot = a.slots[t];
    if (slot < 0) return;
    if ((uint64_t)(slot >> a.c.page_shift) >= a.c.pages) {
        if (lane == 0) atomicOr(a.status, kStatusBadSlot);
        return;
    }
    const bool is_v = blockIdx.y != 0;
    const void *src = is_v ? a.v : a.k;
    const int64_t at = (int64_t)t * (is_v ? a.v_token : a.k_token) + (int64_t)h * (is_v ? a.v_head : a.k_head);
    const uint64_t r = ((uint64_t)(slot >> a.c.page_shift) * H + h) * a.c.page_size + (slot & (a.c.page_size - 1));
    unsigned char *dst = (is_v ? a.c.v : a.c.k) + r * a.c.row_bytes;
    uint16_t *sc = (is_v ? a.c.vs : a.c.ks) + r * a.c.groups;
    float x[N], m[N];
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = load_as_float(src, at + 32 * i + lane, a.dtype);
    if (a.c.format == BGTQ_PAGES_F16 || a.c.format == BGTQ_PAGES_BF16) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            store_float(dst, 32 * i + lane, x[i], a.c.format == BGTQ_PAGES_F16 ? BGTQ_F16 : BGTQ_BF16);
        return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        // as bits, |x| orders like an integer with NaN above infinity, so the maximum keeps both
        uint32_t b = __float_as_uint(x[i]) & 0x7fffffffu;
        b = __reduce_max_sync(0xffffffffu, b);
        m[i] = __uint_as_float(b);
    }
    const bool four = a.c.format == BGTQ_PAGES_INT4;
    if (!four) {
        uint32_t b = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) b = max(b, __float_as_uint(m[i]));
#pragma unroll
        for (int i = 0; i < N; ++i) m[i] = __uint_as_float(b);
    }
    const float top = four ? 7.0f : 127.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const bool fine = m[i] <= 3.402823466e38f;
        const __nv_bfloat16 sb = __float2bfloat16_rn(__fdiv_rn(m[i], top));
        const float s = __bfloat162float(sb);
        int c = 0;
        if (fine && s > 0.0f) c = (int)fminf(fmaxf(rintf(__fdiv_rn(x[i], s)), -top), top);
        if (four) {
            const int hi = __shfl_down_sync(0xffffffffu, c, 1);
            if (!(lane & 1u)) dst[16 * i + lane / 2] = (unsigned char)((c + 8) | (hi + 8) << 4);
            if (lane == 0) sc[i] = fine ? __bfloat16_as_ushort(sb) : 0x7fffu;
        } else {
            dst[32 * i + lane] = (unsigned char)(signed char)c;
            if (i == 0 && lane == 0) sc[0] = fine ? __bfloat16_as_ushort(sb) : 0x7fffu;
        }
    }
}

template <int D>
__global__ void __launch_bounds__(32 * kWarps) read_rows_kernel(const PagedReadArgs a) {
    constexpr int N = D / 32;
    const uint64_t row = (uint64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
    const uint32_t lane = threadIdx.x & 31u, H = a.c.heads;
    if (row >= a.tokens * H) return;
    const uint64_t t = row / H;
    const uint32_t h = (uint32_t)(row % H);
    const int64_t slot = a.slots[t];
    const bool is_v = blockIdx.y != 0;
    void *out = is_v ? a.v : a.k;
    const bool past = slot >= 0 && (uint64_t)(slot >> a.c.page_shift) >= a.c.pages;
    if (past && lane == 0) atomicOr(a.status, kStatusBadSlot);
    if (slot < 0 || past) {
#pragma unroll
        for (int i = 0; i < N; ++i) store_float(out, row * D + 32 * i + lane, 0.0f, a.dtype);
        return;
    }
    const uint64_t r = ((uint64_t)(slot >> a.c.page_shift) * H + h) * a.c.page_size + (slot & (a.c.page_size - 1));
    const unsigned char *src = (is_v ? a.c.v : a.c.k) + r * a.c.row_bytes;
    const uint16_t *sc = (is_v ? a.c.vs : a.c.ks) + r * a.c.groups;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float x;
        const uint32_t d = 32 * i + lane;
        switch (a.c.format) {
            case BGTQ_PAGES_F16: x = load_as_float(src, d, BGTQ_F16); break;
            case BGTQ_PAGES_BF16: x = load_as_float(src, d, BGTQ_BF16); break;
            case BGTQ_PAGES_INT8:
                x = (float)(signed char)src[d] * __bfloat162float(__ushort_as_bfloat16(sc[0]));
                break;
            default:
                x = (float)((int)(src[d / 2] >> (4 * (d & 1u)) & 15u) - 8) *
                    __bfloat162float(__ushort_as_bfloat16(sc[i]));
        }
        store_float(out, row * D + d, x, a.dtype);
    }
}

}  // namespace

cudaError_t launch_paged_write(const PagedWriteArgs &a, cudaStream_t s) {
    const uint64_t blocks = (a.tokens * a.c.heads + kWarps - 1) / kWarps;
    if (blocks > 0x7fffffffull) return cudaErrorInvalidConfiguration;
    const dim3 grid((uint32_t)blocks, 2);
    if (a.c.dim == 64) write_rows_kernel<64><<<grid, 32 * kWarps, 0, s>>>(a);
    else write_rows_kernel<128><<<grid, 32 * kWarps, 0, s>>>(a);
    return cudaGetLastError();
}

cudaError_t launch_paged_read(const PagedReadArgs &a, cudaStream_t s) {
    const uint64_t blocks = (a.tokens * a.c.heads + kWarps - 1) / kWarps;
    if (blocks > 0x7fffffffull) return cudaErrorInvalidConfiguration;
    const dim3 grid((uint32_t)blocks, 2);
    if (a.c.dim == 64) read_rows_kernel<64><<<grid, 32 * kWarps, 0, s>>>(a);
    else read_rows_kernel<128><<<grid, 32 * kWarps, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace bgtq
