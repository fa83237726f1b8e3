// Penalties for tokens that a request's text holds already, biases and a grammar's mask, on its logits:
//     x -> x / r or x r where the token is in the text, by the sign of x;  x - presence - frequency count;  x + biases;
//     -infinity where the mask has no bit
//
// One pass over the logits, which are what there is to move.  A CTA takes a slice of the vocabulary of one row; its first
// loads - logits, mask words, the history's first tokens, biases - are all under way before it waits for one.  Counts of the
// history's tokens that fall into the slice are gathered in shared memory beside them, by integer atomics, whose order
// does not show; biases that fall into it are lined up there in the order of their entries, and each thread adds those
// of its own ids.
//
// What bounds it: 256 rows of 151936 FP32 logits take 48 us with short histories, 6.5 TB/s, the rate of a plain copy; histories
// of up to 8192 tokens, which every slice of a row reads anew, add 11, 50 biases a row 10 and a mask 3.  One row is 3 us of
// latency.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>

#include "serving.h"

namespace bgtq {
namespace {

// 256 rows of 151936 FP32 logits, histories of 16 to 8192 tokens, 50 biases a row: registers for 4 of them an SM 79 us, for 5 72,
// for 6 69.
constexpr uint32_t kThreads = 256, kResident = 6;
// Times four tokens of the history that a thread loads before it knows the length.  (With a mask too: 1 74 us, 2 75, 4 80; a row of
// 49152 with 300 tokens 3.1, 3.1 and 3.5.)
constexpr uint32_t kAhead = 1;
// CTAs that are enough to take the longer slices.  (8 rows of 151936: 296 of them in 5.5 us, more and shorter ones in 6.5; a row of
// 49152: always the longer ones 4.4 us for 3.1; the 256 rows: never 163 for 72.)
constexpr uint64_t kEnough = 296;

template <int T> struct Element {
    static constexpr uint32_t kBytes = T == BGTQ_F32 ? 4 : 2, kEach = 16 / kBytes;  // logits in 16 bytes
};
template <int T>
__device__ __forceinline__ float to_float(uint32_t bits) {
    if constexpr (T == BGTQ_F32) return __uint_as_float(bits);
    else if constexpr (T == BGTQ_F16) return __half2float(__ushort_as_half((unsigned short)bits));
    else return __uint_as_float(bits << 16);
}
template <int T>
__device__ __forceinline__ uint32_t from_float(float x) {
    if constexpr (T == BGTQ_F32) return __float_as_uint(x);
    else if constexpr (T == BGTQ_F16) return __half_as_ushort(__float2half_rn(x));
    else return __bfloat16_as_ushort(__float2bfloat16_rn(x));
}
template <int T>
__device__ __forceinline__ uint32_t load(const void *p, int64_t i) {
    if constexpr (T == BGTQ_F32) return static_cast<const uint32_t *>(p)[i];
    else return static_cast<const uint16_t *>(p)[i];
}
template <int T>
__device__ __forceinline__ void store(void *p, int64_t i, uint32_t x) {
    if constexpr (T == BGTQ_F32) static_cast<uint32_t *>(p)[i] = x;
    else static_cast<uint16_t *>(p)[i] = (uint16_t)x;
}

// U: 16 bytes of logits a thread; V: rows of logits and of results lie alike to 16 bytes.  Then a row's first 16 bytes may
// begin before it.
template <int T, int U, bool V>
__global__ void __launch_bounds__(kThreads, kResident) logits_kernel(const LogitsArgs a) {
    constexpr uint32_t E = Element<T>::kEach, kSlice = kThreads * U * E;
    extern __shared__ __align__(16) uint32_t counts[];  // [kSlice], with a history
    __shared__ uint32_t line_id[kThreads];
    __shared__ float line_x[kThreads];
    __shared__ uint32_t line[kThreads / 32];
    __shared__ uint32_t words[kSlice / 32 + 1];
    const uint32_t b = blockIdx.y, lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const char *row = static_cast<const char *>(a.logits) + (int64_t)b * a.logits_stride * Element<T>::kBytes;
    char *to = static_cast<char *>(a.out) + (int64_t)b * a.out_stride * Element<T>::kBytes;
    const int32_t vocab = (int32_t)a.vocab;
    // the slice's first id; its ids are counted from there
    const int32_t first = (int32_t)(blockIdx.x * kSlice) - (V ? (int32_t)(reinterpret_cast<uintptr_t>(row) % 16 / Element<T>::kBytes) : 0);
    auto inside = [&](int32_t id) { return id >= 0 && id < vocab && (uint32_t)(id - first) < kSlice; };
    // ---- loads ----
    uint4 x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int32_t i = first + (int32_t)((u * kThreads + threadIdx.x) * E);
        x[u] = make_uint4(0, 0, 0, 0);
        if (i >= vocab) continue;
        if (V && i >= 0 && i + (int32_t)E <= vocab) x[u] = *reinterpret_cast<const uint4 *>(row + (int64_t)i * Element<T>::kBytes);
        else {
            uint32_t *w = reinterpret_cast<uint32_t *>(&x[u]);
#pragma unroll
            for (int32_t k = 0; k < (int32_t)E; ++k) {
                const uint32_t y = i + k >= 0 && i + k < vocab ? load<T>(row, i + k) : 0u;
                if constexpr (T == BGTQ_F32) w[k] = y;
                else w[k / 2] |= y << 16 * (k & 1);
            }
        }
    }
    // the slice's words of the mask, one a thread (each thread its own ids' words: 84 us for 66 of 256 rows of 151936)
    const uint32_t word0 = (uint32_t)max(first, 0) >> 5;
    uint32_t word = ~0u;
    if (a.mask && threadIdx.x <= kSlice / 32 && word0 + threadIdx.x < (a.vocab + 31) / 32)
        word = __ldg(a.mask + (int64_t)b * a.mask_stride + word0 + threadIdx.x);
    // four tokens of the history from 4 v on; -1 past its width, and what no vocabulary holds for ids past 32 bits
    auto tokens = [&](uint32_t v) -> int4 {
        if (4 * v >= a.width) return make_int4(-1, -1, -1, -1);
        const int64_t at = (int64_t)b * a.tokens_stride + 4 * v;
        const bool whole = a.tokens_even && 4 * v + 4 <= a.width;
        if (a.id_bytes == 4) {
            const int32_t *from = static_cast<const int32_t *>(a.tokens) + at;
            if (whole) return __ldg(reinterpret_cast<const int4 *>(from));
            auto one = [&](uint32_t k) { return 4 * v + k < a.width ? __ldg(from + k) : -1; };
            return make_int4(one(0), one(1), one(2), one(3));
        }
        const int64_t *from = static_cast<const int64_t *>(a.tokens) + at;
        auto narrow = [](int64_t id) { return id < 0 ? -1 : (int32_t)min(id, (int64_t)0x7fffffff); };
        if (whole) {
            const longlong2 y = __ldg(reinterpret_cast<const longlong2 *>(from)), z = __ldg(reinterpret_cast<const longlong2 *>(from) + 1);
            return make_int4(narrow(y.x), narrow(y.y), narrow(z.x), narrow(z.y));
        }
        auto one = [&](uint32_t k) { return 4 * v + k < a.width ? narrow(__ldg(from + k)) : -1; };
        return make_int4(one(0), one(1), one(2), one(3));
    };
    int4 ids[kAhead];
    int32_t length = 0;
    float r = 1.0f, p = 0.0f, f = 0.0f;
    if (a.tokens) {
#pragma unroll
        for (uint32_t k = 0; k < kAhead; ++k) ids[k] = tokens(threadIdx.x + k * kThreads);
        length = a.lengths ? __ldg(a.lengths + b) : (int32_t)a.width;
        if (a.repetition) r = __ldg(a.repetition + b);
        if (a.presence) p = __ldg(a.presence + b);
        if (a.frequency) f = __ldg(a.frequency + b);
    }
    if (a.lengths && !a.tokens && blockIdx.x == 0 && threadIdx.x == 0 && __ldg(a.lengths + b)) atomicOr(a.status, kStatusBadExtent);
    int32_t bias_id = -1;
    float bias = 0.0f;
    auto entry = [&](uint32_t j) {
        bias_id = j < a.entries ? __ldg(a.bias_ids + (int64_t)b * a.bias_stride + j) : -1;
        bias = j < a.entries ? __ldg(a.bias + (int64_t)b * a.bias_stride + j) : 0.0f;
    };
    if (a.bias) entry(threadIdx.x);
    // the slice's biases of kThreads entries, in their order, in two steps with a wait between them and one after
    uint32_t here = 0, all = 0;
    auto line_up = [&]() {
        if (bias_id >= vocab && blockIdx.x == 0) atomicOr(a.status, kStatusBadSlot);
        here = __ballot_sync(0xffffffffu, inside(bias_id));
        if (lane == 0) line[warp] = __popc(here);
    };
    auto write_line = [&]() {
        uint32_t at = __popc(here & ((1u << lane) - 1));
        all = 0;
#pragma unroll
        for (uint32_t w = 0; w < kThreads / 32; ++w) {
            at += w < warp ? line[w] : 0;
            all += line[w];
        }
        if (here >> lane & 1u) line_id[at] = (uint32_t)(bias_id - first), line_x[at] = bias;
    };
    // ---- counts ----
    if (a.mask && threadIdx.x <= kSlice / 32) words[threadIdx.x] = word;
    if (a.bias) line_up();
    if (a.tokens)
#pragma unroll
        for (uint32_t i = 0; i < kSlice / 4 / kThreads; ++i) reinterpret_cast<uint4 *>(counts)[i * kThreads + threadIdx.x] = make_uint4(0, 0, 0, 0);
    if (a.tokens || a.bias || a.mask) __syncthreads();
    if (a.bias) write_line();
    if (a.tokens) {
        if (length < 0 || (uint32_t)length > a.width) {
            if (threadIdx.x == 0 && blockIdx.x == 0) atomicOr(a.status, kStatusBadExtent);
            length = length < 0 ? 0 : (int32_t)a.width;
        }
        auto count = [&](const int4 &four, uint32_t v) {
            const int32_t of[4] = {four.x, four.y, four.z, four.w};
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) {
                if (4 * v + k >= (uint32_t)length) break;
                if (of[k] >= vocab && blockIdx.x == 0) atomicOr(a.status, kStatusBadSlot);
                if (inside(of[k])) atomicAdd(counts + (of[k] - first), 1u);
            }
        };
#pragma unroll
        for (uint32_t k = 0; k < kAhead; ++k) count(ids[k], threadIdx.x + k * kThreads);
        for (uint32_t v = threadIdx.x + kAhead * kThreads; 4 * v < (uint32_t)length; v += 4 * kThreads) {
            int4 more[4];
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) more[k] = tokens(v + k * kThreads);
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) count(more[k], v + k * kThreads);
        }
    }
    if (a.tokens || a.bias) __syncthreads();
    // ---- the slice ----
    float y[U][E];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t *w = reinterpret_cast<const uint32_t *>(&x[u]);
#pragma unroll
        for (uint32_t k = 0; k < E; ++k) y[u][k] = to_float<T>(T == BGTQ_F32 ? w[k] : w[k / 2] >> 16 * (k & 1) & 0xffffu);
        if (!a.tokens) continue;
#pragma unroll
        for (uint32_t q = 0; q < E / 4; ++q) {
            const uint4 c = reinterpret_cast<const uint4 *>(counts + (u * kThreads + threadIdx.x) * E)[q];
            if (!(c.x | c.y | c.z | c.w)) continue;
            const uint32_t of[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k)
                if (of[k]) {
                    float &z = y[u][4 * q + k];
                    z = z > 0.0f ? __fdiv_rn(z, r) : __fmul_rn(z, r);
                    z = __fsub_rn(__fsub_rn(z, p), __fmul_rn(f, (float)of[k]));
                }
        }
    }
    for (uint32_t j = 0; j < a.entries; j += kThreads) {
        if (j) {
            entry(j + threadIdx.x);
            __syncthreads();  // (the line before this one has been read)
            line_up();
            __syncthreads();
            write_line();
            __syncthreads();
        }
        for (uint32_t k = 0; k < all; ++k) {
            const uint32_t id = line_id[k];
            if (id / E % kThreads != threadIdx.x) continue;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (uint32_t e = 0; e < E; ++e)
                    if (id == (u * kThreads + threadIdx.x) * E + e) y[u][e] += line_x[k];
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int32_t i = first + (int32_t)((u * kThreads + threadIdx.x) * E);
        if (i >= vocab) continue;
        uint32_t w[4] = {}, bits = ~0u;
        if (a.mask) {
            const uint32_t at = ((uint32_t)max(i, 0) >> 5) - word0;
            bits = i < 0 ? words[0] << -i : words[at] >> (i & 31);
            if ((i & 31) + E > 32 && i >= 0) bits |= words[at + 1] << (32 - (i & 31));  // where a row does not begin at 16 bytes
        }
#pragma unroll
        for (uint32_t k = 0; k < E; ++k) {
            const uint32_t z = from_float<T>(bits >> k & 1u ? y[u][k] : -INFINITY);
            if constexpr (T == BGTQ_F32) w[k] = z;
            else w[k / 2] |= z << 16 * (k & 1);
        }
        if (V && i >= 0 && i + (int32_t)E <= vocab) *reinterpret_cast<uint4 *>(to + (int64_t)i * Element<T>::kBytes) = make_uint4(w[0], w[1], w[2], w[3]);
        else {
#pragma unroll
            for (int32_t k = 0; k < (int32_t)E; ++k)
                if (i + k >= 0 && i + k < vocab) store<T>(to, i + k, T == BGTQ_F32 ? w[k] : w[k / 2] >> 16 * (k & 1) & 0xffffu);
        }
    }
}

template <int T, int U, bool V>
cudaError_t run(const LogitsArgs &a, cudaStream_t s) {
    constexpr uint32_t kSlice = kThreads * U * Element<T>::kEach;
    const uint32_t smem = a.tokens ? kSlice * 4 : 0, ids = a.vocab + (V ? Element<T>::kEach - 1 : 0);
    logits_kernel<T, U, V><<<dim3((ids + kSlice - 1) / kSlice, a.batch), kThreads, smem, s>>>(a);
    return cudaGetLastError();
}
template <int T, int U>
cudaError_t by_alignment(const LogitsArgs &a, cudaStream_t s) {
    const bool v = (reinterpret_cast<uintptr_t>(a.logits) - reinterpret_cast<uintptr_t>(a.out)) % 16 == 0 &&
                   (a.batch == 1 || (a.logits_stride - a.out_stride) * (int64_t)Element<T>::kBytes % 16 == 0);
    return v ? run<T, U, true>(a, s) : run<T, U, false>(a, s);
}
// Slices of 16 KB of FP32 logits (16 bits: 8 KB) where that makes enough CTAs, else of 4 KB.
template <int T>
cudaError_t by_size(const LogitsArgs &a, cudaStream_t s) {
    constexpr uint32_t kOne = kThreads * Element<T>::kEach;
    constexpr int kMost = T == BGTQ_F32 ? 4 : 2;
    if ((uint64_t)a.batch * ((a.vocab + kMost * kOne - 1) / (kMost * kOne)) >= kEnough) return by_alignment<T, kMost>(a, s);
    return by_alignment<T, 1>(a, s);
}

}  // namespace

cudaError_t launch_logits(const LogitsArgs &args, cudaStream_t s) {
    LogitsArgs a = args;
    a.tokens_even = reinterpret_cast<uintptr_t>(a.tokens) % 16 == 0 && a.tokens_stride * a.id_bytes % 16 == 0;
    if (a.dtype == BGTQ_F32) return by_size<BGTQ_F32>(a, s);
    if (a.dtype == BGTQ_F16) return by_size<BGTQ_F16>(a, s);
    return by_size<BGTQ_BF16>(a, s);
}

}  // namespace bgtq
