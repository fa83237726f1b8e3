// Writing token rows into the pages of a cache, quantised where the format asks for it, and
// reading them back.
//
// A group of a row (the whole row in 8 bits, 32 dimensions in 4) has one scale, stored in BF16:
//     s = bf16(max|x| (1 / top)),  c = clamp(round(x / s), -top, top),  x' = c s,   top = 127 or 7,
// c = 0 where s = 0.  The scale keeps BF16's 8 bits because its exponent range is FP32's (no
// input of any source type overflows it), and because the codes are computed against the
// rounded scale, so that its rounding moves the step by 0.4 % at most and adds no error of its
// own.  A group with an infinity or a NaN in it has no step: its scale is stored as NaN and the
// whole group reads back as NaN.  All of it is FP32 arithmetic with IEEE rounding.
//
// Both directions move each row once.  A thread takes eight dimensions of a row (16-byte loads and
// stores of 16-bit elements); the lanes of a row, or of a 4-bit group, agree on the maximum by
// shuffles.  16K tokens of 8 heads of 128 in 4 bits, written (21 us) and read back (16 us): 42 us
// with the second launch, 172 MB, 4.1 TB/s of a copy's 6.5.  Loads' latency bounds both first (5 and 9 warps wait
// for one at each issue), then issue (2 of 3 cycles; about twelve instructions an element, half of them the
// quotient and its code).
// 16 tokens of 3 heads: 3.3 us, two launches' latency.
#include "paged_rows.cuh"

namespace bgtq {
namespace {

constexpr uint32_t kThreads = 256;

// Eight dimensions of a row into the pages.  All lanes of a row come here together.
template <int F, int D, int T>
__device__ __forceinline__ void put(unsigned char *rows, uint16_t *scales, uint64_t r, uint32_t part, const Eight<T> &e,
                                    uint32_t lanes) {
    unsigned char *dst = rows + (r * (D / 8) + part) * Format<F>::kBytes;
    float x[8];
    e.floats(x);
    if constexpr (!Format<F>::kCodes) {
        store8<F == BGTQ_PAGES_F16 ? BGTQ_F16 : BGTQ_BF16>(dst, x);
    } else {
        constexpr uint32_t kLanes = F == BGTQ_PAGES_INT4 ? kInt4Group / 8 : D / 8;  // that share a scale
        // as bits, |x| orders like a whole number with NaN above infinity, so the maximum keeps both; elements of 16
        // bits go two at a time
        uint32_t m = 0;
        if constexpr (T == BGTQ_F32) {
#pragma unroll
            for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
#pragma unroll
            for (uint32_t w = 1; w < kLanes; w <<= 1) m = max(m, __shfl_xor_sync(lanes, m, w));
        } else {
            constexpr uint32_t kAbs = 0x7fff7fffu;
            const uint4 u = e.w[0];
            m = __vmaxs2(__vimax3_s16x2(u.x & kAbs, u.y & kAbs, u.z & kAbs), u.w & kAbs);
#pragma unroll
            for (uint32_t w = 1; w < kLanes; w <<= 1) m = __vmaxs2(m, __shfl_xor_sync(lanes, m, w));
            m = __float_as_uint(to_float<T>(max(m & 0xffffu, m >> 16)));
        }
        const uint32_t sb = encode<F>(dst, x, m);
        if (part % kLanes == 0) scales[(r * (D / 8) + part) / kLanes] = (uint16_t)sb;
    }
}
// Eight dimensions of a stored row as the values that they stand for (2^23 + u is 0x4b000000 | u).
template <int F, int D>
__device__ __forceinline__ void get(const unsigned char *rows, const uint16_t *scales, uint64_t r, uint32_t part, float (&x)[8]) {
    const unsigned char *src = rows + (r * (D / 8) + part) * Format<F>::kBytes;
    if constexpr (!Format<F>::kCodes) {
        Eight<F == BGTQ_PAGES_F16 ? BGTQ_F16 : BGTQ_BF16> e;
        e.template load<true>(src);
        e.floats(x);
    } else {
        constexpr uint32_t kLanes = F == BGTQ_PAGES_INT4 ? kInt4Group / 8 : D / 8;
        const float s = __uint_as_float((uint32_t)__ldg(scales + (r * (D / 8) + part) / kLanes) << 16);
        if constexpr (F == BGTQ_PAGES_INT4) {
            const uint32_t u = __ldg(reinterpret_cast<const uint32_t *>(src));
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const float2 v = __fmul2_rn(__fadd2_rn(make_float2(__uint_as_float(0x4b000000u | (u >> 4 * i & 15u)),
                                                                   __uint_as_float(0x4b000000u | (u >> 4 * i + 4 & 15u))),
                                                       make_float2(-8388616.0f, -8388616.0f)), make_float2(s, s));
                x[i] = v.x, x[i + 1] = v.y;
            }
        } else {
            const uint2 u = __ldg(reinterpret_cast<const uint2 *>(src));
#pragma unroll
            for (int i = 0; i < 8; ++i)
                x[i] = (__uint_as_float(0x4b000000u | (((i < 4 ? u.x : u.y) ^ 0x80808080u) >> 8 * (i & 3) & 255u)) - 8388736.0f) * s;
        }
    }
}

// kBoth: a thread takes its chunk of the K row and of the V row; else K rows are in blockIdx.y = 0, V rows in 1.
template <int F, int T, int D, bool V, bool kBoth>
__global__ void __launch_bounds__(kThreads) write_rows_kernel(const PagedWriteArgs a) {
    constexpr uint32_t kLanes = D / 8;  // of a row
    const uint64_t i = (uint64_t)blockIdx.x * kThreads + threadIdx.x;
    const uint32_t H = a.c.heads, row = (uint32_t)(i / kLanes), part = (uint32_t)(i % kLanes);
    if (row >= (uint32_t)a.tokens * H) return;
    const uint32_t t = a.head_mul ? __umulhi(row, a.head_mul) >> a.head_shift : row, h = row - t * H;
    const bool only_v = !kBoth && blockIdx.y != 0;
    const int64_t slot = __ldg(a.slots + t);
    const int64_t k_at = (int64_t)t * a.k_token + (int64_t)h * a.k_head, v_at = (int64_t)t * a.v_token + (int64_t)h * a.v_head;
    constexpr int B = Element<T>::kBytes;
    Eight<T> e, v;  // loaded beside the slot, for padding too
    e.template load<V>(static_cast<const char *>(only_v ? a.v : a.k) + ((only_v ? v_at : k_at) + 8 * part) * B);
    if constexpr (kBoth) v.template load<V>(static_cast<const char *>(a.v) + (v_at + 8 * part) * B);
    if (slot < 0) return;
    if ((uint64_t)(slot >> a.c.page_shift) >= a.c.pages) {
        if (part == 0) atomicOr(a.status, kStatusBadSlot);
        return;
    }
    const uint32_t lanes = (uint32_t)((1ull << kLanes) - 1) << (threadIdx.x & 31u & ~(kLanes - 1));
    const uint64_t r = ((uint64_t)(slot >> a.c.page_shift) * H + h << a.c.page_shift) + (slot & (a.c.page_size - 1));
    put<F, D, T>(only_v ? a.c.v : a.c.k, only_v ? a.c.vs : a.c.ks, r, part, e, lanes);
    if constexpr (kBoth) put<F, D, T>(a.c.v, a.c.vs, r, part, v, lanes);
}

template <int F, int T, int D, bool kBoth>
__global__ void __launch_bounds__(kThreads) read_rows_kernel(const PagedReadArgs a) {
    constexpr uint32_t kLanes = D / 8;
    const uint64_t i = (uint64_t)blockIdx.x * kThreads + threadIdx.x;
    const uint32_t H = a.c.heads, row = (uint32_t)(i / kLanes), part = (uint32_t)(i % kLanes);
    if (row >= (uint32_t)a.tokens * H) return;
    const uint32_t t = a.head_mul ? __umulhi(row, a.head_mul) >> a.head_shift : row, h = row - t * H;
    const bool only_v = !kBoth && blockIdx.y != 0;
    const int64_t slot = __ldg(a.slots + t);
    float x[8] = {}, v[8] = {};
    if (slot >= 0 && (uint64_t)(slot >> a.c.page_shift) < a.c.pages) {
        const uint64_t r = ((uint64_t)(slot >> a.c.page_shift) * H + h << a.c.page_shift) + (slot & (a.c.page_size - 1));
        get<F, D>(only_v ? a.c.v : a.c.k, only_v ? a.c.vs : a.c.ks, r, part, x);
        if constexpr (kBoth) get<F, D>(a.c.v, a.c.vs, r, part, v);
    } else if (slot >= 0 && part == 0) {
        atomicOr(a.status, kStatusBadSlot);
    }
    constexpr int B = Element<T>::kBytes;
    store8<T>(static_cast<char *>(only_v ? a.v : a.k) + i * 8 * B, x);
    if constexpr (kBoth) store8<T>(static_cast<char *>(a.v) + i * 8 * B, v);
}

// From about a wave of threads on, a thread takes K and V, and shares the slot and the address between them (16K
// tokens of 8 heads of 128 in 4 bits, written and read: 42.3 us, 50.4 with threads of their own); below it, threads
// of their own end sooner (4999 tokens of 2 heads of 64 in 8 bits from FP32: 5.8 us, 6.2 with both).
constexpr uint64_t kMany = 1u << 18;

template <typename Args>
Args divided(Args a) {
    const Divisor d = divisor(a.c.heads);
    a.head_mul = d.mul;
    a.head_shift = d.shift;
    return a;
}

template <int F, int T, int D, bool V>
void write_rows(const PagedWriteArgs &a, cudaStream_t s) {
    const uint64_t chunks = a.tokens * a.c.heads * (D / 8);
    const uint32_t blocks = (uint32_t)((chunks + kThreads - 1) / kThreads);
    if (chunks >= kMany) write_rows_kernel<F, T, D, V, true><<<blocks, kThreads, 0, s>>>(a);
    else write_rows_kernel<F, T, D, V, false><<<dim3(blocks, 2), kThreads, 0, s>>>(a);
}
template <int F, int T>
void write_as(const PagedWriteArgs &a, cudaStream_t s) {
    // by 16 bytes where addresses and strides allow it, else by elements (16K tokens as above: 42.3 us, 45.0)
    constexpr int B = Element<T>::kBytes;
    const bool v = even(a.k, a.k_token, a.k_head, B) && even(a.v, a.v_token, a.v_head, B);
    if (a.c.dim == 64) v ? write_rows<F, T, 64, true>(a, s) : write_rows<F, T, 64, false>(a, s);
    else v ? write_rows<F, T, 128, true>(a, s) : write_rows<F, T, 128, false>(a, s);
}
template <int F, int T, int D>
void read_rows(const PagedReadArgs &a, cudaStream_t s) {
    const uint64_t chunks = a.tokens * a.c.heads * (D / 8);
    const uint32_t blocks = (uint32_t)((chunks + kThreads - 1) / kThreads);
    if (chunks >= kMany) read_rows_kernel<F, T, D, true><<<blocks, kThreads, 0, s>>>(a);
    else read_rows_kernel<F, T, D, false><<<dim3(blocks, 2), kThreads, 0, s>>>(a);
}
template <int F, int T>
void read_as(const PagedReadArgs &a, cudaStream_t s) {
    a.c.dim == 64 ? read_rows<F, T, 64>(a, s) : read_rows<F, T, 128>(a, s);
}
template <int F>
void write_from(const PagedWriteArgs &a, cudaStream_t s) {
    if (a.dtype == BGTQ_F16) write_as<F, BGTQ_F16>(a, s);
    else if (a.dtype == BGTQ_BF16) write_as<F, BGTQ_BF16>(a, s);
    else write_as<F, BGTQ_F32>(a, s);
}
template <int F>
void read_into(const PagedReadArgs &a, cudaStream_t s) {
    if (a.dtype == BGTQ_F16) read_as<F, BGTQ_F16>(a, s);
    else if (a.dtype == BGTQ_BF16) read_as<F, BGTQ_BF16>(a, s);
    else read_as<F, BGTQ_F32>(a, s);
}

}  // namespace

cudaError_t launch_paged_write(const PagedWriteArgs &args, cudaStream_t s) {
    const PagedWriteArgs a = divided(args);
    switch (a.c.format) {
        case BGTQ_PAGES_F16: write_from<BGTQ_PAGES_F16>(a, s); break;
        case BGTQ_PAGES_BF16: write_from<BGTQ_PAGES_BF16>(a, s); break;
        case BGTQ_PAGES_INT8: write_from<BGTQ_PAGES_INT8>(a, s); break;
        default: write_from<BGTQ_PAGES_INT4>(a, s);
    }
    return cudaGetLastError();
}

cudaError_t launch_paged_read(const PagedReadArgs &args, cudaStream_t s) {
    const PagedReadArgs a = divided(args);
    switch (a.c.format) {
        case BGTQ_PAGES_F16: read_into<BGTQ_PAGES_F16>(a, s); break;
        case BGTQ_PAGES_BF16: read_into<BGTQ_PAGES_BF16>(a, s); break;
        case BGTQ_PAGES_INT8: read_into<BGTQ_PAGES_INT8>(a, s); break;
        default: read_into<BGTQ_PAGES_INT4>(a, s);
    }
    return cudaGetLastError();
}

}  // namespace bgtq
