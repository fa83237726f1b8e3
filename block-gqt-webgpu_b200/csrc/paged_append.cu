// New tokens into the pages of a cache: heads of queries and keys normed (where the model does), rotated by their
// position, keys and values quantised and stored, queries written out, in one pass over the projections' output.
//     y = x w / sqrt(mean(x^2) + eps),   (y_i, y_{i + D/2}) -> (y_i c_i - y_{i + D/2} s_i, y_{i + D/2} c_i + y_i s_i)
// Rows that become codes are computed in 64 bits and rounded to FP32 once: a code is a step function of its row, and
// so is the same whatever order the sums and products are taken in.  All else is FP32.
#include <type_traits>

#include "paged_rows.cuh"

namespace bgtq {
namespace {

constexpr uint32_t kThreads = 256;

// A thread takes eight dimensions of a row's first half and the eight of the second that they are rotated with.
template <int F, int T, int D, bool V>
__global__ void __launch_bounds__(kThreads) append_kernel(const AppendArgs a) {
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
        const float *norm = kind == 0 ? a.q_norm : a.k_norm;
        auto turn = [&](auto zero) {
            using R = decltype(zero);
            R u[8], v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) u[k] = x[k], v[k] = y[k];
            if (norm) {
                R sum = 0;
#pragma unroll
                for (int k = 0; k < 8; ++k) sum += u[k] * u[k] + v[k] * v[k];
#pragma unroll
                for (uint32_t w = 1; w < kLanes; w <<= 1) sum += __shfl_xor_sync(lanes, sum, w);
                const R f = R(1) / sqrt(sum / R(D) + R(a.eps));
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    u[k] *= f * R(__ldg(norm + 8 * part + k));
                    v[k] *= f * R(__ldg(norm + D / 2 + 8 * part + k));
                }
            }
            const float *rotary = a.rotary + pos * D + 8 * part;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const R c = __ldg(rotary + k), s = __ldg(rotary + D / 2 + k);
                x[k] = (float)(u[k] * c - v[k] * s);
                y[k] = (float)(v[k] * c + u[k] * s);
            }
        };
        if (kCodes && kind == 1) turn(0.0);
        else turn(0.0f);
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

template <int F, int T, int D>
void append_rows(const AppendArgs &a, cudaStream_t s) {
    const uint64_t threads = a.tokens * (a.q_heads + 2 * a.c.heads) * (D / 16);
    const uint32_t blocks = (uint32_t)((threads + kThreads - 1) / kThreads);
    constexpr int B = Element<T>::kBytes;
    if (even(a.q, a.q_token, a.q_head, B) && even(a.k, a.k_token, a.k_head, B) && even(a.v, a.v_token, a.v_head, B))
        append_kernel<F, T, D, true><<<blocks, kThreads, 0, s>>>(a);
    else append_kernel<F, T, D, false><<<blocks, kThreads, 0, s>>>(a);
}
template <int F, int T>
void append_as(const AppendArgs &a, cudaStream_t s) {
    a.c.dim == 64 ? append_rows<F, T, 64>(a, s) : append_rows<F, T, 128>(a, s);
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
