// Kernel arguments and launchers of the serving operators: the paged cache's write and read, new
// tokens rotated into it, one-token and chunk attention over its pages, packed prompt attention,
// and what is put on logits.
#pragma once

#include <cstddef>
#include <cstdint>

#include <cuda_runtime.h>

#include "../../include/bgtq.h"

namespace bgtq {

constexpr uint32_t kInt4Group = 32;  // dimensions per scale of a 4-bit row
// Device status word bits of these operators (beside those of bgtq_internal.h).
constexpr uint32_t kStatusBadSlot = 4u;    // a slot or page index past the cache's pages
constexpr uint32_t kStatusBadExtent = 8u;  // a length past its table row, or packed starts out of order

// The pages as the kernels see them: row (page, head, token) of K is at
// k + ((page * heads + head) * page_size + token) * row_bytes, its scales at the same row
// index times `groups`.
struct PageView {
    unsigned char *k, *v;
    uint16_t *ks, *vs;  // BF16 scales; null for 16-bit formats
    uint32_t heads, dim, page_size, page_shift, pages, row_bytes, groups;
    bgtq_page_format format;
};

struct PagedWriteArgs {
    PageView c;
    const void *k, *v;
    int64_t k_token, k_head, v_token, v_head;  // element strides of the source
    const int64_t *slots;
    uint64_t tokens;
    bgtq_dtype dtype;
    uint32_t *status;
    uint32_t head_mul, head_shift;  // row / heads = row * head_mul >> (32 + head_shift), for the kernels
};

struct PagedReadArgs {
    PageView c;
    void *k, *v;  // dense [tokens][heads][dim]
    const int64_t *slots;
    uint64_t tokens;
    bgtq_dtype dtype;
    uint32_t *status;
    uint32_t head_mul, head_shift;
};

struct PagedAttendArgs {
    PageView c;
    const void *q;
    int64_t q_batch, q_head;  // element strides
    const int32_t *table;
    int64_t table_stride;
    const int32_t *lengths;
    void *out;
    float *lse;  // nullable
    void *workspace;
    uint32_t batch, q_heads, group, width;
    uint32_t counters;  // the launcher's: bytes of the workspace's counters
    uint32_t q_even;    // the launcher's: query rows are 16-byte aligned
    float scale;  // of the logits, times log2(e)
    bgtq_dtype dtype;
    uint32_t *status;
};

struct PromptArgs {
    const void *q, *k, *v;
    int64_t q_token, q_head, k_token, k_head, v_token, v_head;  // element strides
    const int32_t *starts, *key_starts;  // [sequences + 1]
    void *out;                            // [q_tokens][q_heads][dim]
    float *lse;                           // [q_tokens][q_heads], nullable
    uint64_t q_tokens, k_tokens;
    uint32_t sequences, q_heads, kv_heads, group, dim;
    void *workspace;
    uint32_t tiles;     // the launcher's: row tiles of a work item
    uint32_t counters;  // the launcher's: bytes of the workspace's counters
    float scale;  // of the logits, times log2(e)
    int causal;
    bgtq_dtype dtype;
    uint32_t *status;
};

struct AppendArgs {
    PageView c;
    const void *q, *k, *v;
    int64_t q_token, q_head, k_token, k_head, v_token, v_head;  // element strides
    const int64_t *slots, *positions;                            // positions nullable
    const float *rotary, *q_norm, *k_norm;                       // norms nullable
    uint64_t rotary_rows, tokens;
    void *q_out, *k_out;  // dense; k_out nullable
    float eps;
    uint32_t q_heads;
    bgtq_dtype dtype, out_dtype;
    uint32_t *status;
    uint32_t rows_mul, rows_shift;  // the launcher's: row / (q_heads + 2 heads), for the kernels
};

struct ChunkArgs {
    PageView c;
    const void *q;
    int64_t q_token, q_head;  // element strides
    const int32_t *starts;    // [batch + 1]; null: one row each
    const int32_t *table;
    int64_t table_stride;
    const int32_t *lengths;
    void *out;
    float *lse;  // nullable
    void *workspace;
    uint64_t q_tokens;
    uint32_t batch, q_heads, group, width;
    uint32_t window, sinks;  // window 0: none
    uint32_t counters;       // the launcher's: bytes of the workspace's counters
    uint32_t tiles;          // the launcher's: row tiles of a work item (many rows)
    float scale;             // of the logits, times log2(e)
    bgtq_dtype dtype;
    uint32_t *status;
};

struct LogitsArgs {
    const void *logits, *tokens;
    const int32_t *lengths, *bias_ids;
    const float *repetition, *presence, *frequency, *bias;
    const uint32_t *mask;
    void *out;
    int64_t logits_stride, tokens_stride, bias_stride, mask_stride, out_stride;
    uint32_t batch, vocab, width, id_bytes, entries;
    uint32_t tokens_even;  // the launcher's: histories are 16-byte aligned
    bgtq_dtype dtype;
    uint32_t *status;
};

cudaError_t launch_paged_write(const PagedWriteArgs &a, cudaStream_t s);
cudaError_t launch_paged_read(const PagedReadArgs &a, cudaStream_t s);
// Bytes of the workspace that launch_paged_attend needs (counters first, zero between calls).
size_t paged_attend_workspace(uint32_t q_heads, uint32_t kv_heads, uint32_t dim);
cudaError_t launch_paged_attend(const PagedAttendArgs &a, cudaStream_t s);
// Bytes of the workspace that launch_prompt needs (counters first, zero between calls).
size_t prompt_workspace(uint32_t dim);
cudaError_t launch_prompt(const PromptArgs &a, cudaStream_t s);

cudaError_t launch_append(const AppendArgs &a, cudaStream_t s);
// Bytes of the workspace that launch_chunk needs (counters first, zero between calls).
size_t chunk_workspace(const PageView &c, uint32_t q_heads);
cudaError_t launch_chunk(const ChunkArgs &a, cudaStream_t s);
// The kernel of many rows (paged_prompt.cu), which launch_chunk calls, and the bytes of its workspace.
size_t paged_prompt_workspace(uint32_t dim);
cudaError_t launch_paged_prompt(const ChunkArgs &a, cudaStream_t s);
cudaError_t launch_logits(const LogitsArgs &a, cudaStream_t s);

// SMs of a device (0: no such device), asked for once.
inline int sm_count(int device) {
    static int known[64] = {};  // (threads that race here write the same value)
    if (device < 0 || device >= 64) return 0;
    if (!known[device] && cudaDeviceGetAttribute(&known[device], cudaDevAttrMultiProcessorCount, device) != cudaSuccess) {
        known[device] = 0;
        cudaGetLastError();
    }
    return known[device];
}

}  // namespace bgtq
