// Attention of a chunk of new tokens of every request over the pages of a cache, all of them or a window and the first
// few: which kernel takes a call, by the columns - rows x query heads of a KV head - that its requests have on average.
//
// Few columns: the kernel of one token per request with 8 or 16 columns, a request's rows in blocks of as many.  It
// reads a request's pages once for each block.  Many: the one on the fifth-generation tensor cores, which reads them once for up
// to 256 columns (512 at head dim 64), at the price of starting and joining larger pieces.  Measured, in us (few, many):
//     32 requests of 500 to 16000 tokens, 32 / 8 heads of 128, 16 columns: 16 bits 156, 116; 8 bits 153, 181; 4 bits 157, 218
//                                                             20 columns: 16 bits 310, 116; 8 bits 272, 182; 4 bits 310, 220
//     the same, 14 / 2 heads of 64, 28 columns: 41, 44; 8 bits 41, 61; 4 bits 47, 62; 35 columns: 72, 46; 70, 63; 73, 63
//     the same, 9 / 3 heads of 64, 24 columns: 80, 58
//     one request of 30000 tokens, 20 columns of 128: 59, 41; 28 of 64: 28, 33; eight of 200 to 2000, 20 of 128: 27, 22; 28 of
//     64: 15, 21
// At head dim 64 a page is half as long, and a second block finds it in L2; hence 32 columns there and 16 at 128.
// (16-bit pages of many long requests would be better off with the other kernel from 4 columns on, those of few worse: 8
// requests of 200 to 2000, 4 columns of 128, 16 us and 22.)
// The rule knows the mean alone, and what is above was measured with equal requests.  Of 255 single tokens and one chunk of 512
// rows, each after 8000 tokens, 32 / 8 heads of 128 in 16 bits, 12 columns on average, few takes all: 2127 us, and the two kernels one
// after the other 92 for the chunk and 1273 for the rest; after 1000 tokens 404 for 42 and 174.
// 8 columns or 16: 32 requests as above, heads of 128, 8 columns 139 and 153 us (8 bits 109 and 143), 12 columns 263 and 158 (194
// and 147).
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
    if (a.q_tokens * a.group > (a.c.dim == 64 ? 32ull : 16ull) * a.batch) return launch_paged_prompt(a, s);
    switch (a.c.format) {
        case BGTQ_PAGES_F16: return by_shape<F_F16>(a, s);
        case BGTQ_PAGES_BF16: return by_shape<F_BF16>(a, s);
        case BGTQ_PAGES_INT8: return by_shape<F_INT8>(a, s);
        default: return by_shape<F_INT4>(a, s);
    }
}

}  // namespace bgtq
