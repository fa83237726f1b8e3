// C ABI of the serving operators (paged cache, one-token attention over its pages, packed
// prompt attention): argument checks before anything is launched, then one launcher each.
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
