// Attention of one new token per request over the pages of a cache: the kernel is paged_attention_impl.cuh's.
#include "paged_attention_impl.cuh"

namespace bgtq {
namespace {

// More than eight query heads a KV head fill two blocks of columns, so that each page is read once for 16 heads.  (128
// requests of 16K tokens, 16 / 1 heads of 128 in 16 bits: 174 us, 323 with a block of eight at a time.)  Up to eight
// take one block: a second one, empty, costs 15 to 17 % (14 / 2 heads of 64, 32 requests of 4096: 16.8 us for 19.2).
template <int F>
cudaError_t by_shape(const PagedAttendArgs &a, cudaStream_t s) {
    if (a.c.dim == 64) return a.group <= 8 ? run<F, 64, 1, false>(a, s) : run<F, 64, 2, false>(a, s);
    return a.group <= 8 ? run<F, 128, 1, false>(a, s) : run<F, 128, 2, false>(a, s);
}

}  // namespace

// (The counters of any device with less than 4096 SMs are within the bytes that start from zero.)
size_t paged_attend_workspace(uint32_t q_heads, uint32_t kv_heads, uint32_t dim) {
    return counter_bytes() + 2ull * most_ctas() * (q_heads / kv_heads <= 8 ? 8u : 16u) * (dim + 2) * 4;
}

cudaError_t launch_paged_attend(const PagedAttendArgs &a, cudaStream_t s) {
    switch (a.c.format) {
        case BGTQ_PAGES_F16: return by_shape<F_F16>(a, s);
        case BGTQ_PAGES_BF16: return by_shape<F_BF16>(a, s);
        case BGTQ_PAGES_INT8: return by_shape<F_INT8>(a, s);
        default: return by_shape<F_INT4>(a, s);
    }
}

}  // namespace bgtq
