// Penalties for tokens that a request's text holds already, biases and a grammar's mask, on its logits.
// A CTA takes a slice of the vocabulary of one row: it counts the history's tokens that fall into the slice and adds up
// the biases of its ids in shared memory, then passes over the logits once.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>

#include "serving.h"

namespace bgtq {
namespace {

constexpr uint32_t kThreads = 256;

template <int T>
__device__ __forceinline__ float load(const void *p, int64_t i) {
    if constexpr (T == BGTQ_F32) return static_cast<const float *>(p)[i];
    else if constexpr (T == BGTQ_F16) return __half2float(static_cast<const __half *>(p)[i]);
    else return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
}
template <int T>
__device__ __forceinline__ void store(void *p, int64_t i, float x) {
    if constexpr (T == BGTQ_F32) static_cast<float *>(p)[i] = x;
    else if constexpr (T == BGTQ_F16) static_cast<__half *>(p)[i] = __float2half_rn(x);
    else static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(x);
}

template <int T>
__global__ void __launch_bounds__(kThreads) logits_kernel(const LogitsArgs a) {
    extern __shared__ uint32_t smem[];
    uint32_t *counts = smem;
    float *added = reinterpret_cast<float *>(smem + a.slice);
    const uint32_t b = blockIdx.y, first = blockIdx.x * a.slice, n = min(a.slice, a.vocab - first);
    const bool history = a.tokens != nullptr, biased = a.bias != nullptr;
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) counts[i] = 0, added[i] = 0.0f;
    __syncthreads();
    if (history) {
        int32_t len = a.lengths ? __ldg(a.lengths + b) : (int32_t)a.width;
        if (len < 0 || (uint32_t)len > a.width) {
            if (threadIdx.x == 0 && blockIdx.x == 0) atomicOr(a.status, kStatusBadExtent);
            len = len < 0 ? 0 : (int32_t)a.width;
        }
        for (int32_t i = threadIdx.x; i < len; i += kThreads) {
            const int64_t at = (int64_t)b * a.tokens_stride + i;
            const int64_t id = a.id_bytes == 8 ? __ldg(static_cast<const int64_t *>(a.tokens) + at)
                                               : (int64_t)__ldg(static_cast<const int32_t *>(a.tokens) + at);
            if (id >= (int64_t)a.vocab && blockIdx.x == 0) atomicOr(a.status, kStatusBadSlot);
            const uint64_t in = (uint64_t)(id - (int64_t)first);
            if (in < n) atomicAdd(counts + in, 1u);
        }
    }
    if (biased && threadIdx.x < 32) {  // one warp, so that the entries of an id are added in their order
        for (uint32_t j = 0; j < a.entries; j += 32) {
            const uint32_t e = j + threadIdx.x;
            const int64_t at = (int64_t)b * a.bias_stride + e;
            const int32_t id = e < a.entries ? __ldg(a.bias_ids + at) : -1;
            if (id >= 0 && (uint32_t)id >= a.vocab && blockIdx.x == 0) atomicOr(a.status, kStatusBadSlot);
            const uint32_t in = id < 0 ? ~0u : (uint32_t)id - first;
            const float x = in < n ? __ldg(a.bias + at) : 0.0f;
            const uint32_t same = __match_any_sync(0xffffffffu, in < n ? in : ~0u);
            float sum = 0.0f;
            if (in < n) sum = added[in];
            for (uint32_t l = 0; l < 32; ++l) {
                const float y = __shfl_sync(0xffffffffu, x, l);
                if (same >> l & 1u) sum += y;
            }
            if (in < n) added[in] = sum;
            __syncwarp();
        }
    }
    __syncthreads();
    const float r = a.repetition ? __ldg(a.repetition + b) : 1.0f, p = a.presence ? __ldg(a.presence + b) : 0.0f;
    const float f = a.frequency ? __ldg(a.frequency + b) : 0.0f;
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
        const uint32_t v = first + i, c = counts[i];
        float x = load<T>(a.logits, (int64_t)b * a.logits_stride + v);
        if (c) {
            x = x > 0.0f ? __fdiv_rn(x, r) : __fmul_rn(x, r);
            x = __fsub_rn(__fsub_rn(x, p), __fmul_rn(f, (float)c));
        }
        if (biased) x += added[i];
        if (a.mask && !(__ldg(a.mask + (int64_t)b * a.mask_stride + v / 32) >> v % 32 & 1u)) x = -INFINITY;
        store<T>(a.out, (int64_t)b * a.out_stride + v, x);
    }
}

}  // namespace

cudaError_t launch_logits(const LogitsArgs &args, cudaStream_t s) {
    LogitsArgs a = args;
    a.slice = 4096;
    const dim3 grid((a.vocab + a.slice - 1) / a.slice, a.batch);
    const size_t smem = a.slice * 8;
    if (a.dtype == BGTQ_F32) logits_kernel<BGTQ_F32><<<grid, kThreads, smem, s>>>(a);
    else if (a.dtype == BGTQ_F16) logits_kernel<BGTQ_F16><<<grid, kThreads, smem, s>>>(a);
    else logits_kernel<BGTQ_BF16><<<grid, kThreads, smem, s>>>(a);
    return cudaGetLastError();
}

}  // namespace bgtq
