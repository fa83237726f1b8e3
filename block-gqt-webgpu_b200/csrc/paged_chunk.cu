// Attention of a chunk of new tokens of every request over the pages of a cache, all of them or a window and the first
// few.  A warp takes one query row of one head and passes over the tokens that it sees, 32 at a time.
#include "paged_rows.cuh"

namespace bgtq {
namespace {

constexpr uint32_t kWarps = 4;

template <int F, int D>
__device__ __forceinline__ float element(const unsigned char *rows, const uint16_t *scales, uint64_t r, uint32_t d) {
    if constexpr (F == BGTQ_PAGES_F16) return __half2float(__ushort_as_half(reinterpret_cast<const uint16_t *>(rows)[r * D + d]));
    else if constexpr (F == BGTQ_PAGES_BF16) return __uint_as_float((uint32_t)reinterpret_cast<const uint16_t *>(rows)[r * D + d] << 16);
    else if constexpr (F == BGTQ_PAGES_INT8) return (float)reinterpret_cast<const int8_t *>(rows)[r * D + d] * __uint_as_float((uint32_t)scales[r] << 16);
    else return (float)((int)(rows[(r * D + d) / 2] >> 4 * (d & 1) & 15) - 8) * __uint_as_float((uint32_t)scales[(r * D + d) / kInt4Group] << 16);
}

template <int F, int D>
__global__ void __launch_bounds__(32 * kWarps) chunk_kernel(const ChunkArgs a) {
    __shared__ float qs[kWarps][D];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    const uint64_t item = (uint64_t)blockIdx.x * kWarps + warp;
    if (item >= a.q_tokens * a.q_heads) return;
    const uint64_t row = item / a.q_heads;
    const uint32_t h = (uint32_t)(item % a.q_heads), kh = h / a.group, H = a.c.heads;
    // the request that holds the row
    uint32_t b = a.batch;
    int32_t n = 0, i = 0;
    if (!a.starts) b = (uint32_t)row, n = 1;
    else
        for (uint32_t s = 0; s < a.batch && b == a.batch; ++s) {
            const int32_t s0 = __ldg(a.starts + s), s1 = __ldg(a.starts + s + 1);
            if (s0 < 0 || s1 < s0 || (uint64_t)s1 > a.q_tokens) {
                if (lane == 0) atomicOr(a.status, kStatusBadExtent);
                continue;
            }
            if ((int64_t)row >= s0 && (int64_t)row < s1) b = s, n = s1 - s0, i = (int32_t)row - s0;
        }
    if (b == a.batch) return;
    const int32_t given = __ldg(a.lengths + b);
    const int32_t len = given < 0 ? 0 : (int32_t)min((uint64_t)given, (uint64_t)a.width << a.c.page_shift);
    if (len != given && lane == 0) atomicOr(a.status, kStatusBadExtent);
    for (uint32_t d = lane; d < (uint32_t)D; d += 32) {
        const uint16_t x = static_cast<const uint16_t *>(a.q)[(int64_t)row * a.q_token + (int64_t)h * a.q_head + d];
        qs[warp][d] = a.dtype == BGTQ_F16 ? __half2float(__ushort_as_half(x)) : __uint_as_float((uint32_t)x << 16);
    }
    __syncwarp();
    const int32_t p = len - n + i, from = a.window ? max(0, p - (int32_t)a.window + 1) : 0;
    const int32_t sinks = min((int32_t)a.sinks, from);
    float m = -INFINITY, l = 0.0f, o[D / 32] = {};
    auto pass = [&](int32_t t0, int32_t t1) {
        for (int32_t t = t0; t < t1; t += 32) {
            const int32_t mine = t + (int32_t)lane;
            uint64_t r = 0;
            bool in = mine < t1;
            if (in) {
                const int32_t page = __ldg(a.table + (int64_t)b * a.table_stride + (mine >> a.c.page_shift));
                in = (uint32_t)page < a.c.pages;
                if (!in) atomicOr(a.status, kStatusBadSlot);
                r = ((uint64_t)(uint32_t)page * H + kh << a.c.page_shift) + (mine & (a.c.page_size - 1));
            }
            float s = 0.0f;
            if (in)
                for (uint32_t d = 0; d < (uint32_t)D; ++d) s = fmaf(qs[warp][d], element<F, D>(a.c.k, a.c.ks, r, d), s);
            s = in ? s * a.scale : -INFINITY;
            float top = s;
            for (int w = 16; w; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
            top = fmaxf(top, m);
            const float ref = top == -INFINITY ? 0.0f : top, f = exp2f(m - ref), e = exp2f(s - ref);
            m = top;
            l = l * f + e;
            for (int k = 0; k < D / 32; ++k) o[k] *= f;
            for (int u = 0; u < 32; ++u) {
                const float w = __shfl_sync(0xffffffffu, e, u);
                const uint64_t ru = __shfl_sync(0xffffffffu, r, u);
                if (!__shfl_sync(0xffffffffu, (int)in, u)) continue;
                for (int k = 0; k < D / 32; ++k) o[k] = fmaf(w, element<F, D>(a.c.v, a.c.vs, ru, lane + 32 * k), o[k]);
            }
        }
    };
    pass(0, sinks);
    pass(from, p + 1);
    for (int w = 16; w; w >>= 1) l += __shfl_xor_sync(0xffffffffu, l, w);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    for (int k = 0; k < D / 32; ++k) {
        const uint64_t at = item * D + lane + 32 * k;
        if (a.dtype == BGTQ_F16) static_cast<__half *>(a.out)[at] = __float2half_rn(o[k] * inv);
        else static_cast<__nv_bfloat16 *>(a.out)[at] = __float2bfloat16_rn(o[k] * inv);
    }
    if (a.lse && lane == 0) a.lse[item] = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

template <int F>
void by_dim(const ChunkArgs &a, cudaStream_t s) {
    const uint32_t blocks = (uint32_t)((a.q_tokens * a.q_heads + kWarps - 1) / kWarps);
    if (a.c.dim == 64) chunk_kernel<F, 64><<<blocks, 32 * kWarps, 0, s>>>(a);
    else chunk_kernel<F, 128><<<blocks, 32 * kWarps, 0, s>>>(a);
}

}  // namespace

size_t chunk_workspace(const PageView &, uint32_t) { return 128; }

cudaError_t launch_chunk(const ChunkArgs &a, cudaStream_t s) {
    switch (a.c.format) {
        case BGTQ_PAGES_F16: by_dim<BGTQ_PAGES_F16>(a, s); break;
        case BGTQ_PAGES_BF16: by_dim<BGTQ_PAGES_BF16>(a, s); break;
        case BGTQ_PAGES_INT8: by_dim<BGTQ_PAGES_INT8>(a, s); break;
        default: by_dim<BGTQ_PAGES_INT4>(a, s);
    }
    return cudaGetLastError();
}

}  // namespace bgtq
