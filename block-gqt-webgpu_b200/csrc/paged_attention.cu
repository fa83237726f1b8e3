// Attention of one new token per request over the pages of a cache:
//     out = sum_t softmax_t(scale q.k_t) v_t  over the request's first `length` tokens,
// with a running maximum and sum (FP32).  A request of length 0 gives zeros and a log sum of
// minus infinity.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "serving.h"

namespace bgtq {
namespace {

constexpr float kLn2 = 0.6931471805599453f;

template <int D>
__device__ __forceinline__ void load_row(const unsigned char *p, const uint16_t *sc, bgtq_page_format f, uint32_t lane,
                                         float (&x)[D / 32]) {
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
        const uint32_t d = 32 * i + lane;
        switch (f) {
            case BGTQ_PAGES_F16: x[i] = __half2float(reinterpret_cast<const __half *>(p)[d]); break;
            case BGTQ_PAGES_BF16: x[i] = __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(p)[d]); break;
            case BGTQ_PAGES_INT8:
                x[i] = (float)(signed char)p[d] * __bfloat162float(__ushort_as_bfloat16(sc[0]));
                break;
            default:
                x[i] = (float)((int)(p[d / 2] >> (4 * (d & 1u)) & 15u) - 8) *
                       __bfloat162float(__ushort_as_bfloat16(sc[i]));
        }
    }
}

// One warp per (request, query head), its lanes over the head's dimensions.
template <int D>
__global__ void __launch_bounds__(32) attend_kernel(const PagedAttendArgs a) {
    constexpr int N = D / 32;
    const uint32_t h = blockIdx.x, b = blockIdx.y, lane = threadIdx.x, kh = h / a.group;
    int32_t len = a.lengths[b];
    if (len < 0 || (uint64_t)len > (uint64_t)a.width << a.c.page_shift) {
        if (lane == 0) atomicOr(a.status, kStatusBadExtent);
        len = len < 0 ? 0 : (int32_t)(a.width << a.c.page_shift);
    }
    float q[N], o[N] = {}, m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int64_t at = (int64_t)b * a.q_batch + (int64_t)h * a.q_head + 32 * i + lane;
        q[i] = a.dtype == BGTQ_F16 ? __half2float(static_cast<const __half *>(a.q)[at])
                                   : __bfloat162float(static_cast<const __nv_bfloat16 *>(a.q)[at]);
    }
    for (int32_t t = 0; t < len; ++t) {
        const int32_t page = a.table[(int64_t)b * a.table_stride + (t >> a.c.page_shift)];
        if ((uint32_t)page >= a.c.pages) {
            if (lane == 0) atomicOr(a.status, kStatusBadSlot);
            continue;
        }
        const uint64_t r = ((uint64_t)page * a.c.heads + kh) * a.c.page_size + (t & (a.c.page_size - 1));
        float k[N], v[N], s = 0.0f;
        load_row<D>(a.c.k + r * a.c.row_bytes, a.c.ks + r * a.c.groups, a.c.format, lane, k);
        load_row<D>(a.c.v + r * a.c.row_bytes, a.c.vs + r * a.c.groups, a.c.format, lane, v);
#pragma unroll
        for (int i = 0; i < N; ++i) s = fmaf(q[i], k[i], s);
#pragma unroll
        for (int w = 16; w; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
        s *= a.scale;
        const float mn = fmaxf(m, s), ref = mn == -INFINITY ? 0.0f : mn;
        const float old = exp2f(m - ref), p = exp2f(s - ref);
        m = mn;
        l = fmaf(l, old, p);
#pragma unroll
        for (int i = 0; i < N; ++i) o[i] = fmaf(p, v[i], o[i] * old);
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const uint64_t row = (uint64_t)b * a.q_heads + h;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint64_t at = row * D + 32 * i + lane;
        if (a.dtype == BGTQ_F16) static_cast<__half *>(a.out)[at] = __float2half_rn(o[i] * inv);
        else static_cast<__nv_bfloat16 *>(a.out)[at] = __float2bfloat16_rn(o[i] * inv);
    }
    if (a.lse && lane == 0) a.lse[row] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
}

}  // namespace

size_t paged_attend_workspace(uint32_t, uint32_t, uint32_t, uint32_t) { return 0; }

cudaError_t launch_paged_attend(const PagedAttendArgs &a, cudaStream_t s) {
    const dim3 grid(a.q_heads, a.batch);
    if (a.c.dim == 64) attend_kernel<64><<<grid, 32, 0, s>>>(a);
    else attend_kernel<128><<<grid, 32, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace bgtq
