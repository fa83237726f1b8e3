// Attention of a chunk of new tokens of every request over the pages of a cache, all of them or a window and the first
// few: which kernel takes a call.
#include "paged_attention_impl.cuh"

namespace bgtq {
namespace {

template <int F>
cudaError_t by_shape(const ChunkArgs &a, cudaStream_t s) {
    const bool one = a.q_tokens * a.group <= 8ull * a.batch;
    if (a.c.dim == 64) return one ? run<F, 64, 1, true>(a, s) : run<F, 64, 2, true>(a, s);
    return one ? run<F, 128, 1, true>(a, s) : run<F, 128, 2, true>(a, s);
}

}  // namespace

size_t chunk_workspace(const PageView &c, uint32_t) {
    const size_t few = BGTQ_WORKSPACE_ZEROED + 2ull * most_ctas() * 16u * (c.dim + 2) * 4, many = paged_prompt_workspace(c.dim);
    return !many ? 0 : few > many ? few : many;
}

cudaError_t launch_chunk(const ChunkArgs &args, cudaStream_t s) {
    ChunkArgs a = args;
    if (a.window >= (uint64_t)a.width << a.c.page_shift) a.window = 0;  // all tokens that the table holds
    if (a.q_tokens * a.group > 16ull * a.batch) return launch_paged_prompt(a, s);
    switch (a.c.format) {
        case BGTQ_PAGES_F16: return by_shape<F_F16>(a, s);
        case BGTQ_PAGES_BF16: return by_shape<F_BF16>(a, s);
        case BGTQ_PAGES_INT8: return by_shape<F_INT8>(a, s);
        default: return by_shape<F_INT4>(a, s);
    }
}

}  // namespace bgtq
