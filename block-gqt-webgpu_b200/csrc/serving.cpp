// C ABI of the serving operators (paged cache, one-token and chunk attention over its pages, packed
// prompt attention, what is put on logits): argument checks before anything is launched, then one launcher each.
#include <cmath>
#include <string>

#include "bgtq_internal.h"
#include "serving.h"

using namespace bgtq;

namespace {

constexpr float kLog2e = 1.4426950408889634f;

bgtq_status refuse(const std::string &msg) {
    set_last_error(msg);
    return BGTQ_EINVAL;
}
bgtq_status launched(cudaError_t e, const char *what) {
    if (e == cudaSuccess) return BGTQ_OK;
    cudaGetLastError();  // (what the runtime still holds would be taken for the next launch's)
    set_last_error(std::string(what) + ": " + cudaGetErrorString(e));
    return BGTQ_ECUDA;
}

struct OnDevice {
    int prev = -1;
    bool ok;
    explicit OnDevice(int dev) {
        ok = cudaGetDevice(&prev) == cudaSuccess;
        if (ok && prev != dev) ok = cudaSetDevice(dev) == cudaSuccess;
        else if (ok) prev = -1;
    }
    ~OnDevice() {
        if (prev >= 0) cudaSetDevice(prev);
    }
};

bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// The kernels' view of a cache, or a refusal.
bgtq_status view(const bgtq_paged_cache *c, PageView &v) {
    if (!c) return refuse("Paged cache: null");
    if (c->dim != 64 && c->dim != 128) return refuse("Paged cache: head dim must be 64 or 128");
    if (c->format < BGTQ_PAGES_F16 || c->format > BGTQ_PAGES_INT4) return refuse("Paged cache: unknown format");
    if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1)))
        return refuse("Paged cache: page size must be a power of two from 16 to 256");
    if (c->kv_heads < 1 || c->kv_heads > 1024 || c->pages < 1 || c->pages > 0x7fffffffu)
        return refuse("Paged cache: invalid head or page count");
    const bool scaled = c->format == BGTQ_PAGES_INT8 || c->format == BGTQ_PAGES_INT4;
    if (!c->k || !c->v || !aligned(c->k, 16) || !aligned(c->v, 16))
        return refuse("Paged cache: pages must be 16-byte aligned device memory");
    if (scaled && (!c->k_scales || !c->v_scales || !aligned(c->k_scales, 16) || !aligned(c->v_scales, 16)))
        return refuse("Paged cache: scales must be 16-byte aligned device memory");
    v.k = static_cast<unsigned char *>(c->k);
    v.v = static_cast<unsigned char *>(c->v);
    v.ks = scaled ? c->k_scales : nullptr;
    v.vs = scaled ? c->v_scales : nullptr;
    v.heads = c->kv_heads;
    v.dim = c->dim;
    v.page_size = c->page_size;
    v.page_shift = (uint32_t)__builtin_ctz(c->page_size);
    v.pages = c->pages;
    v.format = c->format;
    v.groups = c->format == BGTQ_PAGES_INT4 ? c->dim / kInt4Group : c->format == BGTQ_PAGES_INT8 ? 1u : 0u;
    v.row_bytes = c->format == BGTQ_PAGES_INT4 ? c->dim / 2 : c->format == BGTQ_PAGES_INT8 ? c->dim : 2 * c->dim;
    return BGTQ_OK;
}

// scale of the logits in log2 units; 0 stands for 1 / sqrt(dim)
bool logit_scale(float scale, uint32_t dim, float &out) {
    if (!(scale >= 0.0f)) return false;
    out = (scale == 0.0f ? 1.0f / std::sqrt((float)dim) : scale) * kLog2e;
    return std::isfinite(out);
}

size_t width_of(bgtq_dtype t) { return t == BGTQ_F32 ? 4 : 2; }

}  // namespace

extern "C" {

bgtq_status bgtq_paged_write(const bgtq_paged_cache *c, const void *k, const void *v, bgtq_dtype dtype,
                             uint64_t tokens, int64_t k_token_stride, int64_t k_head_stride, int64_t v_token_stride,
                             int64_t v_head_stride, const int64_t *slots, void *stream) {
    PagedWriteArgs a{};
    if (bgtq_status s = view(c, a.c)) return s;
    if (dtype < BGTQ_F16 || dtype > BGTQ_BF16) return refuse("Paged write: source must be FP16, BF16 or FP32");
    if (tokens == 0) return BGTQ_OK;
    if (!k || !v || !slots) return refuse("Paged write: null argument");
    if (!aligned(k, width_of(dtype)) || !aligned(v, width_of(dtype)) || !aligned(slots, 8))
        return refuse("Paged write: misaligned argument");
    if (tokens > 0x7fffffffull / c->kv_heads) return refuse("Paged write: too many rows in one call");
    OnDevice on(c->device);
    a.status = on.ok ? device_status_word(c->device) : nullptr;
    if (!a.status) return launched(cudaErrorInvalidDevice, "Paged write");
    a.k = k;
    a.v = v;
    a.k_token = k_token_stride;
    a.k_head = k_head_stride;
    a.v_token = v_token_stride;
    a.v_head = v_head_stride;
    a.slots = slots;
    a.tokens = tokens;
    a.dtype = dtype;
    return launched(launch_paged_write(a, static_cast<cudaStream_t>(stream)), "Paged write");
}

bgtq_status bgtq_paged_read(const bgtq_paged_cache *c, const int64_t *slots, uint64_t tokens, void *k_out,
                            void *v_out, bgtq_dtype dtype, void *stream) {
    PagedReadArgs a{};
    if (bgtq_status s = view(c, a.c)) return s;
    if (dtype < BGTQ_F16 || dtype > BGTQ_BF16) return refuse("Paged read: output must be FP16, BF16 or FP32");
    if (tokens == 0) return BGTQ_OK;
    if (!slots || !k_out || !v_out) return refuse("Paged read: null argument");
    if (!aligned(k_out, 16) || !aligned(v_out, 16) || !aligned(slots, 8)) return refuse("Paged read: misaligned argument");
    if (tokens > 0x7fffffffull / c->kv_heads) return refuse("Paged read: too many rows in one call");
    OnDevice on(c->device);
    a.status = on.ok ? device_status_word(c->device) : nullptr;
    if (!a.status) return launched(cudaErrorInvalidDevice, "Paged read");
    a.k = k_out;
    a.v = v_out;
    a.slots = slots;
    a.tokens = tokens;
    a.dtype = dtype;
    return launched(launch_paged_read(a, static_cast<cudaStream_t>(stream)), "Paged read");
}

bgtq_status bgtq_paged_attend_workspace(const bgtq_paged_cache *c, uint32_t q_heads, size_t *bytes) {
    PageView v{};
    if (bgtq_status s = view(c, v)) return s;
    if (!bytes || !q_heads || q_heads % c->kv_heads) return refuse("Paged attention: invalid head count");
    OnDevice on(c->device);
    if (!on.ok) return launched(cudaErrorInvalidDevice, "Paged attention");
    *bytes = paged_attend_workspace(q_heads, c->kv_heads, c->dim);
    return BGTQ_OK;
}

bgtq_status bgtq_paged_attend(const bgtq_paged_cache *c, const void *q, bgtq_dtype dtype, uint32_t batch,
                              uint32_t q_heads, int64_t q_batch_stride, int64_t q_head_stride, const int32_t *table,
                              int64_t table_stride, uint32_t table_width, const int32_t *lengths, float scale,
                              void *out, float *lse, void *workspace, size_t workspace_bytes, void *stream) {
    PagedAttendArgs a{};
    if (bgtq_status s = view(c, a.c)) return s;
    if (dtype != BGTQ_F16 && dtype != BGTQ_BF16) return refuse("Paged attention: queries must be FP16 or BF16");
    if ((c->format == BGTQ_PAGES_F16 && dtype != BGTQ_F16) || (c->format == BGTQ_PAGES_BF16 && dtype != BGTQ_BF16))
        return refuse("Paged attention: queries must have the type of 16-bit pages");
    if (!q_heads || q_heads % c->kv_heads) return refuse("Paged attention: invalid head count");
    if (!logit_scale(scale, c->dim, a.scale)) return refuse("Paged attention: scale must be positive and finite");
    if (batch == 0) return BGTQ_OK;
    if (!q || !lengths || !out || (!table && table_width)) return refuse("Paged attention: null argument");
    if (batch > 65535u || q_heads > 65535u) return refuse("Paged attention: too many requests in one call");
    if ((uint64_t)table_width * c->page_size > 0x7fffffffull)
        return refuse("Paged attention: a table row must cover fewer than 2^31 tokens");
    if (!aligned(q, 2) || !aligned(out, 16) || !aligned(table, 4) || !aligned(lengths, 4) || !aligned(lse, 4))
        return refuse("Paged attention: misaligned argument");
    OnDevice on(c->device);
    a.status = on.ok ? device_status_word(c->device) : nullptr;
    if (!a.status) return launched(cudaErrorInvalidDevice, "Paged attention");
    const size_t need = paged_attend_workspace(q_heads, c->kv_heads, c->dim);
    if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
        return refuse("Paged attention: the workspace is too small or misaligned");
    a.q = q;
    a.q_batch = q_batch_stride;
    a.q_head = q_head_stride;
    a.table = table;
    a.table_stride = table_stride;
    a.lengths = lengths;
    a.out = out;
    a.lse = lse;
    a.workspace = workspace;
    a.batch = batch;
    a.q_heads = q_heads;
    a.group = q_heads / c->kv_heads;
    a.width = table_width;
    a.dtype = dtype;
    return launched(launch_paged_attend(a, static_cast<cudaStream_t>(stream)), "Paged attention");
}

bgtq_status bgtq_paged_append(const bgtq_paged_cache *c, const bgtq_append *p, void *stream) {
    AppendArgs a{};
    if (bgtq_status s = view(c, a.c)) return s;
    if (!p) return refuse("Paged append: null");
    if (p->dtype < BGTQ_F16 || p->dtype > BGTQ_BF16) return refuse("Paged append: source must be FP16, BF16 or FP32");
    if (p->out_dtype < BGTQ_F16 || p->out_dtype > BGTQ_BF16) return refuse("Paged append: output must be FP16, BF16 or FP32");
    if (p->q_heads < 1 || p->q_heads > 65535u) return refuse("Paged append: invalid head count");
    if (!(p->eps >= 0.0f) || !std::isfinite(p->eps)) return refuse("Paged append: eps must be nonnegative and finite");
    if (p->tokens == 0) return BGTQ_OK;
    if (!p->q || !p->k || !p->v || !p->slots || !p->rotary || !p->q_out) return refuse("Paged append: null argument");
    const size_t w = width_of(p->dtype);
    if (!aligned(p->q, w) || !aligned(p->k, w) || !aligned(p->v, w) || !aligned(p->slots, 8) || !aligned(p->positions, 8) ||
        !aligned(p->rotary, 16) || !aligned(p->q_norm, 16) || !aligned(p->k_norm, 16) || !aligned(p->q_out, 16) ||
        !aligned(p->k_out, 16))
        return refuse("Paged append: misaligned argument");
    if (p->tokens > 0x7fffffffull / (p->q_heads + 2 * c->kv_heads)) return refuse("Paged append: too many rows in one call");
    if (p->rotary_rows > 0x7fffffffull || (!p->positions && p->rotary_rows < p->tokens))
        return refuse("Paged append: a row of cosines and sines for every token, 2^31 - 1 at most");
    OnDevice on(c->device);
    a.status = on.ok ? device_status_word(c->device) : nullptr;
    if (!a.status) return launched(cudaErrorInvalidDevice, "Paged append");
    a.q = p->q;
    a.k = p->k;
    a.v = p->v;
    a.q_token = p->q_token_stride;
    a.q_head = p->q_head_stride;
    a.k_token = p->k_token_stride;
    a.k_head = p->k_head_stride;
    a.v_token = p->v_token_stride;
    a.v_head = p->v_head_stride;
    a.slots = p->slots;
    a.positions = p->positions;
    a.rotary = p->rotary;
    a.rotary_rows = p->rotary_rows;
    a.q_norm = p->q_norm;
    a.k_norm = p->k_norm;
    a.tokens = p->tokens;
    a.q_out = p->q_out;
    a.k_out = p->k_out;
    a.eps = p->eps;
    a.q_heads = p->q_heads;
    a.dtype = p->dtype;
    a.out_dtype = p->out_dtype;
    return launched(launch_append(a, static_cast<cudaStream_t>(stream)), "Paged append");
}

bgtq_status bgtq_paged_chunk_workspace(const bgtq_paged_cache *c, uint32_t q_heads, size_t *bytes) {
    PageView v{};
    if (bgtq_status s = view(c, v)) return s;
    if (!bytes || !q_heads || q_heads % c->kv_heads || q_heads / c->kv_heads > 128)
        return refuse("Chunk attention: invalid head count");
    OnDevice on(c->device);
    const size_t need = on.ok ? chunk_workspace(v, q_heads) : 0;
    if (!need) return launched(cudaErrorInvalidDevice, "Chunk attention");
    *bytes = need;
    return BGTQ_OK;
}

bgtq_status bgtq_paged_attend_chunk(const bgtq_paged_cache *c, const bgtq_chunk *p, void *stream) {
    ChunkArgs a{};
    if (bgtq_status s = view(c, a.c)) return s;
    if (!p) return refuse("Chunk attention: null");
    if (p->dtype != BGTQ_F16 && p->dtype != BGTQ_BF16) return refuse("Chunk attention: queries must be FP16 or BF16");
    if ((c->format == BGTQ_PAGES_F16 && p->dtype != BGTQ_F16) || (c->format == BGTQ_PAGES_BF16 && p->dtype != BGTQ_BF16))
        return refuse("Chunk attention: queries must have the type of 16-bit pages");
    if (!p->q_heads || p->q_heads % c->kv_heads || p->q_heads / c->kv_heads > 128)
        return refuse("Chunk attention: invalid head count");
    if (!logit_scale(p->scale, c->dim, a.scale)) return refuse("Chunk attention: scale must be positive and finite");
    if (p->window > 0x7fffffffu || p->sinks > 0x7fffffffu) return refuse("Chunk attention: window and sinks must be below 2^31");
    if (p->batch > 65535u || p->q_tokens > 0x7fffffffull / p->q_heads)
        return refuse("Chunk attention: too many requests or tokens in one call");
    if (!p->starts && p->q_tokens != p->batch) return refuse("Chunk attention: one query row for every request without starts");
    if (p->batch == 0 || p->q_tokens == 0) return BGTQ_OK;
    if (!p->q || !p->lengths || !p->out || (!p->table && p->table_width)) return refuse("Chunk attention: null argument");
    if ((uint64_t)p->table_width * c->page_size > 0x7fffffffull)
        return refuse("Chunk attention: a table row must cover fewer than 2^31 tokens");
    if (!aligned(p->q, 16) || !aligned(p->out, 16) || !aligned(p->starts, 4) || !aligned(p->table, 4) ||
        !aligned(p->lengths, 4) || !aligned(p->lse, 4))
        return refuse("Chunk attention: misaligned argument");
    for (int64_t s : {p->q_token_stride, p->q_head_stride})
        if (s <= 0 || s % 8 || s >= (int64_t)1 << 39)
            return refuse("Chunk attention: strides must be positive multiples of 16 bytes");
    OnDevice on(c->device);
    a.status = on.ok ? device_status_word(c->device) : nullptr;
    if (!a.status) return launched(cudaErrorInvalidDevice, "Chunk attention");
    const size_t need = chunk_workspace(a.c, p->q_heads);
    if (!need) return launched(cudaErrorInvalidDevice, "Chunk attention");
    if (!p->workspace || p->workspace_bytes < need || !aligned(p->workspace, 128))
        return refuse("Chunk attention: the workspace is too small or misaligned");
    a.q = p->q;
    a.q_token = p->q_token_stride;
    a.q_head = p->q_head_stride;
    a.starts = p->starts;
    a.table = p->table;
    a.table_stride = p->table_stride;
    a.lengths = p->lengths;
    a.out = p->out;
    a.lse = p->lse;
    a.workspace = p->workspace;
    a.q_tokens = p->q_tokens;
    a.batch = p->batch;
    a.q_heads = p->q_heads;
    a.group = p->q_heads / c->kv_heads;
    a.width = p->table_width;
    a.window = p->window;
    a.sinks = p->sinks;
    a.dtype = p->dtype;
    return launched(launch_chunk(a, static_cast<cudaStream_t>(stream)), "Chunk attention");
}

bgtq_status bgtq_adjust_logits(const bgtq_logits *p, void *stream) {
    if (!p) return refuse("Logits: null");
    if (p->dtype < BGTQ_F16 || p->dtype > BGTQ_BF16) return refuse("Logits: logits must be FP16, BF16 or FP32");
    if (p->vocab < 1 || p->vocab > 0x7ffeffffu) return refuse("Logits: invalid vocabulary");
    if (p->batch > 65535u) return refuse("Logits: too many rows in one call");
    if (p->width > 0x7fffffffu || p->entries > 0x7fffffffu) return refuse("Logits: too many tokens or biases in a row");
    if (p->tokens && p->id_bytes != 4 && p->id_bytes != 8) return refuse("Logits: token ids must have 4 or 8 bytes");
    if (p->batch == 0) return BGTQ_OK;
    if (!p->logits || !p->out || (!p->bias) != (!p->bias_ids)) return refuse("Logits: null argument");
    const size_t w = width_of(p->dtype);
    if (!aligned(p->logits, w) || !aligned(p->out, w) || !aligned(p->tokens, p->tokens ? p->id_bytes : 1) ||
        !aligned(p->lengths, 4) || !aligned(p->repetition, 4) || !aligned(p->presence, 4) || !aligned(p->frequency, 4) ||
        !aligned(p->bias_ids, 4) || !aligned(p->bias, 4) || !aligned(p->mask, 4))
        return refuse("Logits: misaligned argument");
    OnDevice on(p->device);
    LogitsArgs a{};
    a.status = on.ok ? device_status_word(p->device) : nullptr;
    if (!a.status) return launched(cudaErrorInvalidDevice, "Logits");
    a.logits = p->logits;
    a.logits_stride = p->logits_stride;
    a.tokens = p->width ? p->tokens : nullptr;
    a.tokens_stride = p->tokens_stride;
    a.width = p->width;
    a.id_bytes = p->id_bytes;
    a.lengths = p->tokens || !p->width ? p->lengths : nullptr;  // (of an empty history they are looked over)
    a.repetition = p->repetition;
    a.presence = p->presence;
    a.frequency = p->frequency;
    a.bias_ids = p->entries ? p->bias_ids : nullptr;
    a.bias = p->entries ? p->bias : nullptr;
    a.bias_stride = p->bias_stride;
    a.entries = p->bias ? p->entries : 0;  // (without biases their number says nothing)
    a.mask = p->mask;
    a.mask_stride = p->mask_stride;
    a.out = p->out;
    a.out_stride = p->out_stride;
    a.batch = p->batch;
    a.vocab = p->vocab;
    a.dtype = p->dtype;
    return launched(launch_logits(a, static_cast<cudaStream_t>(stream)), "Logits");
}

bgtq_status bgtq_prompt_workspace(int device, uint32_t dim, size_t *bytes) {
    if (dim != 64 && dim != 128) return refuse("Prompt attention: head dim must be 64 or 128");
    if (!bytes) return refuse("Prompt attention: null argument");
    OnDevice on(device);
    const size_t need = on.ok ? prompt_workspace(dim) : 0;
    if (!need) return launched(cudaErrorInvalidDevice, "Prompt attention");
    *bytes = need;
    return BGTQ_OK;
}

bgtq_status bgtq_prompt_attend(const bgtq_prompt *p, void *stream) {
    if (!p) return refuse("Prompt attention: null");
    PromptArgs a{};
    if (p->dim != 64 && p->dim != 128) return refuse("Prompt attention: head dim must be 64 or 128");
    if (p->dtype != BGTQ_F16 && p->dtype != BGTQ_BF16) return refuse("Prompt attention: Q, K, V must be FP16 or BF16");
    if (!p->q_heads || !p->kv_heads || p->q_heads % p->kv_heads || p->q_heads / p->kv_heads > 128 ||
        p->kv_heads > 65535u)
        return refuse("Prompt attention: invalid head count");
    if (!logit_scale(p->scale, p->dim, a.scale)) return refuse("Prompt attention: scale must be positive and finite");
    if (p->q_tokens > 0x7fffffffull || p->k_tokens > 0x7fffffffull || p->sequences > 0x7fffffffu)
        return refuse("Prompt attention: too many tokens in one call");
    if (p->sequences == 0 || p->q_tokens == 0) return BGTQ_OK;
    if (!p->q || !p->out || !p->starts || (p->k_tokens && (!p->k || !p->v)))
        return refuse("Prompt attention: null argument");
    if (!aligned(p->q, 16) || !aligned(p->k, 16) || !aligned(p->v, 16) || !aligned(p->out, 16) ||
        !aligned(p->starts, 4) || !aligned(p->key_starts, 4) || !aligned(p->lse, 4))
        return refuse("Prompt attention: misaligned argument");
    for (int64_t s : {p->q_token_stride, p->q_head_stride, p->k_token_stride, p->k_head_stride, p->v_token_stride,
                      p->v_head_stride})
        if (s <= 0 || s % 8 || s >= (int64_t)1 << 39)
            return refuse("Prompt attention: strides must be positive multiples of 16 bytes");
    OnDevice on(p->device);
    a.status = on.ok ? device_status_word(p->device) : nullptr;
    if (!a.status) return launched(cudaErrorInvalidDevice, "Prompt attention");
    const size_t need = prompt_workspace(p->dim);
    if (!need) return launched(cudaErrorInvalidDevice, "Prompt attention");
    if (!p->workspace || p->workspace_bytes < need || !aligned(p->workspace, 128))
        return refuse("Prompt attention: the workspace is too small or misaligned");
    a.workspace = p->workspace;
    a.q = p->q;
    a.k = p->k;
    a.v = p->v;
    a.q_token = p->q_token_stride;
    a.q_head = p->q_head_stride;
    a.k_token = p->k_token_stride;
    a.k_head = p->k_head_stride;
    a.v_token = p->v_token_stride;
    a.v_head = p->v_head_stride;
    a.starts = p->starts;
    a.key_starts = p->key_starts ? p->key_starts : p->starts;
    a.out = p->out;
    a.lse = p->lse;
    a.q_tokens = p->q_tokens;
    a.k_tokens = p->k_tokens;
    a.sequences = p->sequences;
    a.q_heads = p->q_heads;
    a.kv_heads = p->kv_heads;
    a.group = p->q_heads / p->kv_heads;
    a.dim = p->dim;
    a.causal = p->causal != 0;
    a.dtype = p->dtype;
    return launched(launch_prompt(a, static_cast<cudaStream_t>(stream)), "Prompt attention");
}

}  // extern "C"
