// Rows of the paged cache in registers, eight dimensions to a thread: elements of the source types, the codes of
// a group and its scale (the formula is in paged_cache.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "serving.h"

namespace bgtq {
namespace {

template <int F> struct Format {  // a stored row
    static constexpr bool kCodes = F == BGTQ_PAGES_INT8 || F == BGTQ_PAGES_INT4;
    static constexpr int kBytes = F == BGTQ_PAGES_INT4 ? 4 : F == BGTQ_PAGES_INT8 ? 8 : 16;  // of eight dimensions
};
template <int T> struct Element {
    static constexpr int kBytes = T == BGTQ_F32 ? 4 : 2;
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

// Eight elements of type T as they lie in memory; V: loaded by 16 bytes.
template <int T> struct Eight {
    static constexpr int kWords = Element<T>::kBytes / 2;
    uint4 w[kWords];
    template <bool V>
    __device__ __forceinline__ void load(const void *p) {
        if constexpr (V) {
#pragma unroll
            for (int i = 0; i < kWords; ++i) w[i] = __ldg(static_cast<const uint4 *>(p) + i);
        } else {
            uint32_t *u = reinterpret_cast<uint32_t *>(w);
#pragma unroll
            for (int i = 0; i < 4 * kWords; ++i) {
                if constexpr (T == BGTQ_F32) u[i] = static_cast<const uint32_t *>(p)[i];
                else u[i] = static_cast<const uint16_t *>(p)[2 * i] | (uint32_t)static_cast<const uint16_t *>(p)[2 * i + 1] << 16;
            }
        }
    }
    __device__ __forceinline__ void floats(float (&x)[8]) const {
        const uint32_t *u = reinterpret_cast<const uint32_t *>(w);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_float<T>(T == BGTQ_F32 ? u[i] : u[i / 2] >> 16 * (i & 1) & 0xffffu);
    }
};
template <int T>
__device__ __forceinline__ void store8(void *p, const float (&x)[8]) {
    constexpr int N = Element<T>::kBytes / 2;
    uint32_t u[4 * N];
#pragma unroll
    for (int i = 0; i < 4 * N; ++i) {
        if constexpr (T == BGTQ_F32) u[i] = from_float<T>(x[i]);
        else u[i] = from_float<T>(x[2 * i]) | from_float<T>(x[2 * i + 1]) << 16;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) static_cast<uint4 *>(p)[i] = make_uint4(u[4 * i], u[4 * i + 1], u[4 * i + 2], u[4 * i + 3]);
}

// The codes of eight dimensions of a group whose largest |x| has the bits m, to dst; returns the group's scale.
template <int F>
__device__ __forceinline__ uint32_t encode(unsigned char *dst, const float (&x)[8], uint32_t m) {
    constexpr float kTop = F == BGTQ_PAGES_INT4 ? 7.0f : 127.0f;
    const bool fine = m < 0x7f800000u;
    // one product with the rounded 1 / top: at most an ulp of FP32 from the quotient, and the scale keeps 8 bits
    // of it (about one scale in 2^17 lands on the other side of a BF16 tie; every code and value goes by the
    // scale that is stored)
    const __nv_bfloat16 sb = __float2bfloat16_rn(__fmul_rn(__uint_as_float(m), 1.0f / kTop));
    const float s = __bfloat162float(sb);
    // Codes in the low bits of q + 1.5 * 2^23, which rounds q to the nearest whole number, ties to even (the
    // conversion instructions run at a quarter of the rate).
    constexpr uint32_t kRound = 0x4b400000u;
    uint32_t c[8];
    if (fine && s > 1e-30f && s < 1e30f) {
        // x / s, correctly rounded: one correctly rounded reciprocal y, then q = q0 + (x - s q0) y with q0 = x y
        // (Markstein, IBM J. Res. Dev. 34(1), 1990: q is the IEEE quotient where nothing over- or underflows;
        // quotients are below 128 here).  |q| <= top (1 + 2^-8) rounds to top at most: no clamp.
        const float2 y = make_float2(__frcp_rn(s), __frcp_rn(s)), minus = make_float2(-s, -s);
        const float2 round = make_float2(__uint_as_float(kRound), __uint_as_float(kRound));
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const float2 v = make_float2(x[i], x[i + 1]), q = __fmul2_rn(v, y);
            const float2 z = __fadd2_rn(__ffma2_rn(__ffma2_rn(minus, q, v), y, q), round);
            c[i] = __float_as_uint(z.x), c[i + 1] = __float_as_uint(z.y);
        }
    } else {  // scales near the ends of the exponent range, zero and NaN
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float q = fine && s > 0.0f ? fminf(fmaxf(__fdiv_rn(x[i], s), -kTop), kTop) : 0.0f;
            c[i] = __float_as_uint(__fadd_rn(q, __uint_as_float(kRound)));
        }
    }
    // The codes' places are added up: a word starts with the codes' offset (8 or 128, which makes them
    // nonnegative) in every place, less what kRound adds up to.
    constexpr uint32_t kBits = F == BGTQ_PAGES_INT4 ? 4 : 8, kEach = 32 / kBits;
    constexpr uint32_t kOffsets = F == BGTQ_PAGES_INT4 ? 0x88888888u : 0x80808080u;
    constexpr uint32_t kStart = kOffsets - kRound * (1u + (1u << kBits) + (1u << 2 * kBits));  // further places shift it out
    uint32_t u[8 / kEach];
#pragma unroll
    for (uint32_t w = 0; w < 8 / kEach; ++w) {
        u[w] = kStart;
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) u[w] += c[kEach * w + i] << kBits * i;
    }
    if constexpr (F == BGTQ_PAGES_INT4) *reinterpret_cast<uint32_t *>(dst) = u[0];
    else *reinterpret_cast<uint2 *>(dst) = make_uint2(u[0] ^ kOffsets, u[1] ^ kOffsets);
    return fine ? __bfloat16_as_ushort(sb) : 0x7fffu;
}

// row / n by one product: m = ceil(2^(31 + l) / n), 2^l >= n, is exact for rows below 2^31, which the
// entry points see to.  n = 1 needs none.
struct Divisor {
    uint32_t mul, shift;
};
inline Divisor divisor(uint32_t n) {
    uint32_t l = 0;
    while (1u << l < n) ++l;
    return {l ? (uint32_t)(((1ull << (31 + l)) + n - 1) / n) : 0, l ? l - 1 : 0};
}

inline bool even(const void *p, int64_t token, int64_t head, int bytes) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && token * bytes % 16 == 0 && head * bytes % 16 == 0;
}

}  // namespace
}  // namespace bgtq
