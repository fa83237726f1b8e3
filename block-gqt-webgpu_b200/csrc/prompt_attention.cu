// Attention of a packed batch of prompts of different lengths: row i of sequence s attends
// keys j of the same sequence, with the causal mask j <= i + (keys - queries), softmax with a
// running maximum and sum (FP32).  A row that sees no key gives zeros and a log sum of minus
// infinity.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "serving.h"

namespace bgtq {
namespace {

constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float as_float(const void *p, int64_t i, bgtq_dtype t) {
    return t == BGTQ_F16 ? __half2float(static_cast<const __half *>(p)[i])
                         : __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
}

// One warp per (token, query head), its lanes over the head's dimensions.
template <int D>
__global__ void __launch_bounds__(128) prompt_kernel(const PromptArgs a) {
    constexpr int N = D / 32;
    const uint32_t lane = threadIdx.x & 31u;
    const uint64_t row = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (row >= a.q_tokens * a.q_heads) return;
    const int64_t t = (int64_t)(row / a.q_heads);
    const uint32_t h = (uint32_t)(row % a.q_heads), kh = h / a.group;
    // the sequence that holds token t; one whose starts fall or pass the token counts holds none
    int64_t q0 = 0, k0 = 0, nq = 0, nk = 0, seen = 0;
    for (uint32_t i = 0; i < a.sequences; ++i) {
        const int64_t q_at = a.starts[i], k_at = a.key_starts[i];
        const int64_t n = (int64_t)a.starts[i + 1] - q_at, m = (int64_t)a.key_starts[i + 1] - k_at;
        if (q_at < 0 || k_at < 0 || n < 0 || m < 0 || q_at + n > (int64_t)a.q_tokens || k_at + m > (int64_t)a.k_tokens) {
            if (row == 0 && lane == 0) atomicOr(a.status, kStatusBadExtent);
        } else if (t >= q_at && t < q_at + n) {
            q0 = q_at, k0 = k_at, nq = n, nk = m, seen = m;
        }
    }
    if (nq == 0) return;
    if (a.causal) seen = min(seen, max((int64_t)0, t - q0 + 1 + nk - nq));
    float q[N], o[N] = {}, m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) q[i] = as_float(a.q, t * a.q_token + (int64_t)h * a.q_head + 32 * i + lane, a.dtype);
    for (int64_t j = k0; j < k0 + seen; ++j) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i)
            s = fmaf(q[i], as_float(a.k, j * a.k_token + (int64_t)kh * a.k_head + 32 * i + lane, a.dtype), s);
#pragma unroll
        for (int w = 16; w; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
        s *= a.scale;
        const float mn = fmaxf(m, s), ref = mn == -INFINITY ? 0.0f : mn;
        const float old = exp2f(m - ref), p = exp2f(s - ref);
        m = mn;
        l = fmaf(l, old, p);
#pragma unroll
        for (int i = 0; i < N; ++i)
            o[i] = fmaf(p, as_float(a.v, j * a.v_token + (int64_t)kh * a.v_head + 32 * i + lane, a.dtype), o[i] * old);
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint64_t at = row * D + 32 * i + lane;
        if (a.dtype == BGTQ_F16) static_cast<__half *>(a.out)[at] = __float2half_rn(o[i] * inv);
        else static_cast<__nv_bfloat16 *>(a.out)[at] = __float2bfloat16_rn(o[i] * inv);
    }
    if (a.lse && lane == 0) a.lse[row] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
}

}  // namespace

cudaError_t launch_prompt(const PromptArgs &a, cudaStream_t s) {
    const uint64_t blocks = (a.q_tokens * a.q_heads + 3) / 4;
    if (blocks > 0x7fffffffull) return cudaErrorInvalidConfiguration;
    if (a.dim == 64) prompt_kernel<64><<<(uint32_t)blocks, 128, 0, s>>>(a);
    else prompt_kernel<128><<<(uint32_t)blocks, 128, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace bgtq
