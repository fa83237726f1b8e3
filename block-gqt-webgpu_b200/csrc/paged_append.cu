// New tokens into the pages of a cache: heads of queries and keys normed (where the model does), rotated by their
// position, keys and values quantised and stored, queries written out, in one pass over the projections' output.
//     y = x w / sqrt(mean(x^2) + eps),   (y_i, y_{i + D/2}) -> (y_i c_i - y_{i + D/2} s_i, y_{i + D/2} c_i + y_i s_i)
// Rows that become codes are computed in pairs of FP32 numbers (a norm's factor in 64 bits) and rounded to FP32 once: a code is
// a step function of its row, and so is the same whatever order sums and products are taken in.  All else is FP32.
//
// A row is D / 16 threads, each with two runs of eight dimensions that are rotated into each other: no shared memory, a norm's
// sum and a row's largest by shuffles.  16384 tokens, 32 / 8 heads of 128 from BF16: into 16 bits 76 us, 5.3 TB/s, with norms 90;
// into 8 bits 80, with norms 109; into 4 bits 80, with norms 103, where the pairs of numbers issue as long as the loads take.  A
// step of 16 requests, 9 / 3 heads of 64, takes 2.5 us, next to nothing of which is work.
#include <type_traits>

#include "paged_rows.cuh"

namespace bgtq {
namespace {

// Small CTAs, and registers for ten of them an SM: what is slow here is waiting for loads.  (16384 tokens of 32 / 8 heads of 128
// from BF16 into 8 bits: 256 threads and 58 registers 94 us, 128 and 48 79 us; into 4 bits with norms 116 and 102 us.)
constexpr uint32_t kThreads = 128, kResident = 10;

// Pairs of FP32 numbers and what their rounding left (Dekker's product by one fused multiply-add, Knuth's two-sum), two
// at a time.
struct Two {
    float2 h, l;
};
__device__ __forceinline__ float2 minus(float2 x) { return make_float2(-x.x, -x.y); }
__device__ __forceinline__ Two times(float2 a, float2 b) {
    const float2 p = __fmul2_rn(a, b);
    return {p, __ffma2_rn(a, b, minus(p))};
}
__device__ __forceinline__ Two times(const Two &a, float2 b) {
    const Two p = times(a.h, b);
    return {p.h, __ffma2_rn(a.l, b, p.l)};
}
// p - q, rounded once (but for 2^-24 of an ulp where nothing cancels); infinities and NaN as they come
__device__ __forceinline__ float2 difference(const Two &p, const Two &q) {
    const float2 h = __fadd2_rn(p.h, minus(q.h)), z = __fadd2_rn(h, minus(p.h));
    const float2 e = __fadd2_rn(__fadd2_rn(p.h, minus(__fadd2_rn(h, minus(z)))), minus(__fadd2_rn(q.h, z)));
    const float2 r = __fadd2_rn(h, __fadd2_rn(e, __fadd2_rn(p.l, minus(q.l))));
    return make_float2(r.x == r.x ? r.x : h.x, r.y == r.y ? r.y : h.y);
}

// A thread takes eight dimensions of a row's first half and the eight of the second that they are rotated with.
template <int F, int T, int D, bool V, bool N>
__global__ void __launch_bounds__(kThreads, kResident) append_kernel(const AppendArgs a) {
    constexpr uint32_t kLanes = D / 16;  // of a row
    constexpr bool kCodes = Format<F>::kCodes;
    const uint64_t i = (uint64_t)blockIdx.x * kThreads + threadIdx.x;
    const uint32_t row = (uint32_t)(i / kLanes), part = (uint32_t)(i % kLanes);
    const uint32_t H = a.c.heads, heads = a.q_heads + 2 * H;
    if (row >= (uint32_t)a.tokens * heads) return;
    const uint32_t t = a.rows_mul ? __umulhi(row, a.rows_mul) >> a.rows_shift : row;
    uint32_t h = row - t * heads;
    const int kind = h < a.q_heads ? 0 : h < a.q_heads + H ? 1 : 2;  // Q, K, V
    h -= kind == 0 ? 0 : kind == 1 ? a.q_heads : a.q_heads + H;
    constexpr int B = Element<T>::kBytes;
    const int64_t at = (int64_t)t * (kind == 0 ? a.q_token : kind == 1 ? a.k_token : a.v_token) +
                       (int64_t)h * (kind == 0 ? a.q_head : kind == 1 ? a.k_head : a.v_head) + 8 * part;
    const char *src = static_cast<const char *>(kind == 0 ? a.q : kind == 1 ? a.k : a.v) + at * B;
    Eight<T> lo, hi;
    lo.template load<V>(src);
    hi.template load<V>(src + D / 2 * B);
    const int64_t slot = kind ? __ldg(a.slots + t) : -1;
    const int64_t pos = a.positions ? __ldg(a.positions + t) : (int64_t)t;
    const bool placed = (uint64_t)pos < a.rotary_rows;
    const uint32_t lanes = (uint32_t)((1ull << kLanes) - 1) << (threadIdx.x & 31u & ~(kLanes - 1));
    float x[8], y[8];
    lo.floats(x);
    hi.floats(y);
    if (!placed) {
        if (part == 0 && kind == 0 && h == 0) atomicOr(a.status, kStatusBadExtent);
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = y[k] = 0.0f;
    } else if (kind != 2) {
        const float4 *rotary = reinterpret_cast<const float4 *>(a.rotary + pos * D + 8 * part);
        const float *norm = N ? kind == 0 ? a.q_norm : a.k_norm : nullptr;
        // Whether FP32 holds a row's squares, its factor and what it is multiplied by on the way.  Another row is multiplied by a
        // power of two that brings its largest value, or the root of eps where that is larger, near one.  (2047 tokens of 32 / 8
        // heads of 128 with norms 16.7 us, 16.4 without the look.)
        auto ordinary = [](auto mean) { return mean > 1e-24f && mean < 1e36f; };
        auto near_one = [&]() {
            uint32_t big = 0;
#pragma unroll
            for (int k = 0; k < 8; ++k) big = max(big, max(__float_as_uint(x[k]) & 0x7fffffffu, __float_as_uint(y[k]) & 0x7fffffffu));
#pragma unroll
            for (uint32_t w = 1; w < kLanes; w <<= 1) big = max(big, __shfl_xor_sync(lanes, big, w));
            const int root = a.eps > 0.0f ? (int)(__float_as_uint(a.eps) >> 23) / 2 - 64 : -126;
            const int e = min(max(max((int)(big >> 23) - 127, root), -126), 126);
            const float g = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] *= g, y[k] *= g;
            return g;
        };
        if (kCodes && kind == 1) {
            float2 fh = make_float2(1.0f, 1.0f), fl = make_float2(0.0f, 0.0f);
            if (norm) {
                double sum = 0.0;
#pragma unroll
                for (int k = 0; k < 8; ++k) sum = fma((double)x[k], (double)x[k], fma((double)y[k], (double)y[k], sum));
#pragma unroll
                for (uint32_t w = 1; w < kLanes; w <<= 1) sum += __shfl_xor_sync(lanes, sum, w);
                double mean = sum / D + (double)a.eps;
                if (!ordinary(mean)) {
                    const double g = near_one();
                    mean *= g * g;
                }
                const double f = 1.0 / sqrt(mean);
                fh.x = fh.y = (float)f;
                fl.x = fl.y = (float)(f - (double)fh.x);
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const float4 cs = __ldg(rotary + k), ss = __ldg(rotary + D / 8 + k);
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    const int e = 4 * k + 2 * m;
                    const float2 c = m ? make_float2(cs.z, cs.w) : make_float2(cs.x, cs.y), s = m ? make_float2(ss.z, ss.w) : make_float2(ss.x, ss.y);
                    Two u{make_float2(x[e], x[e + 1]), {}}, v{make_float2(y[e], y[e + 1]), {}};
                    if (norm) {
                        auto normed = [&](float2 z, const float *w) {
                            const Two p = times(z, *reinterpret_cast<const float2 *>(w));
                            Two r = times(p, fh);
                            r.l = __ffma2_rn(p.h, fl, r.l);
                            return r;
                        };
                        u = normed(u.h, norm + 8 * part + e);
                        v = normed(v.h, norm + D / 2 + 8 * part + e);
                    }
                    const float2 p = difference(times(u, c), times(v, s)), q = difference(times(v, c), times(u, minus(s)));
                    x[e] = p.x, x[e + 1] = p.y, y[e] = q.x, y[e + 1] = q.y;
                }
            }
        } else {
            if (norm) {
                auto mean_of = [&]() {
                    float sum = 0.0f;
#pragma unroll
                    for (int k = 0; k < 8; ++k) sum = fmaf(x[k], x[k], fmaf(y[k], y[k], sum));
#pragma unroll
                    for (uint32_t w = 1; w < kLanes; w <<= 1) sum += __shfl_xor_sync(lanes, sum, w);
                    return sum / D;
                };
                float mean = mean_of() + a.eps;
                if (!ordinary(mean)) {
                    const float g = near_one();
                    mean = mean_of() + a.eps * g * g;
                }
                const float f = 1.0f / sqrtf(mean);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    x[k] *= f * __ldg(norm + 8 * part + k);
                    y[k] *= f * __ldg(norm + D / 2 + 8 * part + k);
                }
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const float4 cs = __ldg(rotary + k), ss = __ldg(rotary + D / 8 + k);
                const float c[4] = {cs.x, cs.y, cs.z, cs.w}, s[4] = {ss.x, ss.y, ss.z, ss.w};
#pragma unroll
                for (int m = 0; m < 4; ++m) {
                    const float u = x[4 * k + m], v = y[4 * k + m];
                    x[4 * k + m] = fmaf(u, c[m], -(v * s[m]));
                    y[4 * k + m] = fmaf(v, c[m], u * s[m]);
                }
            }
        }
    }
    auto write = [&](void *out, uint64_t r) {
        auto as = [&](auto type) {
            constexpr int O = decltype(type)::value, S = Element<O>::kBytes;
            char *dst = static_cast<char *>(out) + (r * D + 8 * part) * S;
            store8<O>(dst, x);
            store8<O>(dst + D / 2 * S, y);
        };
        if (a.out_dtype == BGTQ_F16) as(std::integral_constant<int, BGTQ_F16>());
        else if (a.out_dtype == BGTQ_BF16) as(std::integral_constant<int, BGTQ_BF16>());
        else as(std::integral_constant<int, BGTQ_F32>());
    };
    if (kind == 0) {
        write(a.q_out, (uint64_t)t * a.q_heads + h);
        return;
    }
    if (kind == 1 && a.k_out) write(a.k_out, (uint64_t)t * H + h);
    if (slot < 0 || !placed) return;
    if ((uint64_t)(slot >> a.c.page_shift) >= a.c.pages) {
        if (part == 0) atomicOr(a.status, kStatusBadSlot);
        return;
    }
    const uint64_t r = ((uint64_t)(slot >> a.c.page_shift) * H + h << a.c.page_shift) + (slot & (a.c.page_size - 1));
    unsigned char *dst = (kind == 1 ? a.c.k : a.c.v) + (r * (D / 8) + part) * Format<F>::kBytes;
    unsigned char *dst2 = dst + kLanes * Format<F>::kBytes;
    if constexpr (!kCodes) {
        store8<F == BGTQ_PAGES_F16 ? BGTQ_F16 : BGTQ_BF16>(dst, x);
        store8<F == BGTQ_PAGES_F16 ? BGTQ_F16 : BGTQ_BF16>(dst2, y);
    } else {
        // as bits, |x| orders like a whole number with NaN above infinity, so the maximum keeps both
        uint32_t m = 0, n = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) m = max(m, __float_as_uint(x[k]) & 0x7fffffffu), n = max(n, __float_as_uint(y[k]) & 0x7fffffffu);
        uint16_t *scales = kind == 1 ? a.c.ks : a.c.vs;
        if constexpr (F == BGTQ_PAGES_INT8) {
            m = max(m, n);
#pragma unroll
            for (uint32_t w = 1; w < kLanes; w <<= 1) m = max(m, __shfl_xor_sync(lanes, m, w));
            const uint32_t s = encode<F>(dst, x, m);
            encode<F>(dst2, y, m);
            if (part == 0) scales[r] = (uint16_t)s;
        } else {
            constexpr uint32_t kShare = kInt4Group / 8;  // lanes that share a scale
#pragma unroll
            for (uint32_t w = 1; w < kShare; w <<= 1) m = max(m, __shfl_xor_sync(lanes, m, w)), n = max(n, __shfl_xor_sync(lanes, n, w));
            const uint32_t s = encode<F>(dst, x, m), u = encode<F>(dst2, y, n);
            if (part % kShare == 0) {
                scales[(r * (D / 8) + part) / kShare] = (uint16_t)s;
                scales[(r * (D / 8) + kLanes + part) / kShare] = (uint16_t)u;
            }
        }
    }
}

template <int F, int T, int D, bool V>
void append_rows(const AppendArgs &a, cudaStream_t s) {
    const uint64_t threads = a.tokens * (a.q_heads + 2 * a.c.heads) * (D / 16);
    const uint32_t blocks = (uint32_t)((threads + kThreads - 1) / kThreads);
    if (a.q_norm || a.k_norm) append_kernel<F, T, D, V, true><<<blocks, kThreads, 0, s>>>(a);
    else append_kernel<F, T, D, V, false><<<blocks, kThreads, 0, s>>>(a);
}
template <int F, int T>
void append_as(const AppendArgs &a, cudaStream_t s) {
    constexpr int B = Element<T>::kBytes;
    const bool v = even(a.q, a.q_token, a.q_head, B) && even(a.k, a.k_token, a.k_head, B) && even(a.v, a.v_token, a.v_head, B);
    if (a.c.dim == 64) v ? append_rows<F, T, 64, true>(a, s) : append_rows<F, T, 64, false>(a, s);
    else v ? append_rows<F, T, 128, true>(a, s) : append_rows<F, T, 128, false>(a, s);
}
template <int F>
void append_from(const AppendArgs &a, cudaStream_t s) {
    if (a.dtype == BGTQ_F16) append_as<F, BGTQ_F16>(a, s);
    else if (a.dtype == BGTQ_BF16) append_as<F, BGTQ_BF16>(a, s);
    else append_as<F, BGTQ_F32>(a, s);
}

}  // namespace

cudaError_t launch_append(const AppendArgs &args, cudaStream_t s) {
    AppendArgs a = args;
    const Divisor d = divisor(a.q_heads + 2 * a.c.heads);
    a.rows_mul = d.mul;
    a.rows_shift = d.shift;
    switch (a.c.format) {
        case BGTQ_PAGES_F16: append_from<BGTQ_PAGES_F16>(a, s); break;
        case BGTQ_PAGES_BF16: append_from<BGTQ_PAGES_BF16>(a, s); break;
        case BGTQ_PAGES_INT8: append_from<BGTQ_PAGES_INT8>(a, s); break;
        default: append_from<BGTQ_PAGES_INT4>(a, s);
    }
    return cudaGetLastError();
}

}  // namespace bgtq
