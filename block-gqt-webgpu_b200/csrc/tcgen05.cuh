// What kernels on the fifth-generation tensor cores are made of: bounded waits on barriers, TMA loads, tensor memory,
// products, exponentials on two pipes; and the encoder of tensor maps for their launches.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "serving.h"

namespace bgtq {
namespace {

constexpr float kLn2 = 0.6931471805599453f;
constexpr uint32_t kRows = 128;          // of a product's tile
constexpr uint32_t kStatusTimeout = 1u;  // a bounded wait ran out (bgtq_internal.h's kStatusWaitTimeout)

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t n) {
    asm volatile("mbarrier.init.shared.b64 [%0], %1;" ::"r"(bar), "r"(n) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok;
}
// Waits for the phase of `parity`, for a bounded number of polls.  False: it ran out, or another
// role's did (`stop`).
__device__ __forceinline__ bool bar_wait_slow(uint32_t bar, uint32_t parity, volatile uint32_t *stop) {
    for (uint32_t i = 0; i < 1u << 22; ++i) {
        if (bar_try(bar, parity)) return true;
        if ((i & 63u) == 63u && *stop) return false;
    }
    *stop = 1;
    return false;
}
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile uint32_t *stop) {
    if (bar_try(bar, parity)) return true;
    return bar_wait_slow(bar, parity, stop);
}
__device__ __forceinline__ void tma3(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y, int z) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], "
                 "[%2];" ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
}
// One lane of a converged warp.
__device__ __forceinline__ bool elect() {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok));
    return ok != 0;
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// A shared-memory operand, low word: address, and the distance between 64-element column blocks of an
// operand whose rows run along the contraction.  High word: 8-row groups 1024 bytes apart, 128-byte swizzle.
__device__ __forceinline__ uint32_t operand(uint32_t addr, uint32_t lbo) { return addr >> 4 | (lbo >> 4) << 16; }
constexpr uint32_t kOperandHigh = 1024u >> 4 | 1u << 14 | 2u << 29;
// kind::f16, FP32 accumulators, M = 128: the operands' type, whether B's rows run along the contraction, N.
__host__ __device__ constexpr uint32_t product(bool bf16, uint32_t b_rows, uint32_t n) {
    return (1u << 4) | (bf16 ? 1u << 7 | 1u << 10 : 0u) | b_rows << 16 | (n >> 3) << 17 | (kRows >> 4) << 24;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t id, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 x, y;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 x, {%1, %5};\n\t"
                 "mov.b64 y, {%2, %5};\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}" ::"r"(d), "r"(a),
                 "r"(b), "r"(id), "r"(acc), "n"(kOperandHigh) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t id, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 y;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 y, {%2, %5};\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "r"(id),
                 "r"(acc), "n"(kOperandHigh) : "memory");
}
#define BGTQ_R8(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), "=r"(r[i + 6]), "=r"(r[i + 7])
#define BGTQ_V8(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3]), "r"(r[i + 4]), "r"(r[i + 5]), "r"(r[i + 6]), "r"(r[i + 7])
// 32 columns of this thread's lane of tensor memory.
__device__ __forceinline__ void tm_load(uint32_t at, uint32_t *r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
                 "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : BGTQ_R8(r, 0), BGTQ_R8(r, 8), BGTQ_R8(r, 16), BGTQ_R8(r, 24) : "r"(at));
}
__device__ __forceinline__ void tm_store(uint32_t at, const uint32_t *r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, "
                 "%13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};"
                 ::BGTQ_V8(r, 0), BGTQ_V8(r, 8), BGTQ_V8(r, 16), BGTQ_V8(r, 24), "r"(at) : "memory");
}
__device__ __forceinline__ void tm_load16(uint32_t at, uint32_t *r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
                 "%15}, [%16];" : BGTQ_R8(r, 0), BGTQ_R8(r, 8) : "r"(at));
}
__device__ __forceinline__ void tm_store16(uint32_t at, const uint32_t *r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, "
                 "%13, %14, %15};" ::BGTQ_V8(r, 0), BGTQ_V8(r, 8), "r"(at) : "memory");
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max3(float x, float y, float z) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
    return r;
}
__device__ __forceinline__ float max_nan(float x, float y) {  // NaN if one of them is
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
    return r;
}
// 2^y of two values on the FMA pipe, y below 2^20: adding 1.5 * 2^23 rounds y to a whole number n in the low
// mantissa bits, and 2^f of the rest, -1/2 <= f <= 1/2, is the polynomial of degree 4 with the least
// largest relative error on that interval (Remez exchange): 2.7e-6 in FP32, 4e-8 on average.  From
// -126.5 down, -infinity with it, it is zero: -127 is the n whose 2^n has the bits of zero, and in
// BF16 any floor above that is a weight that a large value shows.  NaN: NaN.
__device__ __forceinline__ float2 ex2_fma(float2 y) {
    constexpr float kRound = 12582912.0f;
    y = make_float2(max_nan(y.x, -127.0f), max_nan(y.y, -127.0f));
    const float2 t = __fadd2_rn(y, make_float2(kRound, kRound));
    const float2 f = __ffma2_rn(__fadd2_rn(t, make_float2(-kRound, -kRound)), make_float2(-1.0f, -1.0f), y);
    float2 p = __ffma2_rn(f, make_float2(0.0095701022f, 0.0095701022f), make_float2(0.055917859f, 0.055917859f));
    p = __ffma2_rn(p, f, make_float2(0.24024744f, 0.24024744f));
    p = __ffma2_rn(p, f, make_float2(0.69312179f, 0.69312179f));
    p = __ffma2_rn(p, f, make_float2(0.99999928f, 0.99999928f));
    return __fmul2_rn(p, make_float2(__uint_as_float((__float_as_uint(t.x) << 23) + 0x3f800000u),
                                     __uint_as_float((__float_as_uint(t.y) << 23) + 0x3f800000u)));
}
template <bool BF>
__device__ __forceinline__ uint32_t pack(float x, float y) {
    if constexpr (BF) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
        return *reinterpret_cast<const uint32_t *>(&v);
    } else {
        const __half2 v = __floats2half2_rn(x, y);
        return *reinterpret_cast<const uint32_t *>(&v);
    }
}

// Quotients of nonnegative numbers: 32-bit division where it will do, which is nearly always.
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
    return (uint64_t)(a | b) >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b);
}

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                 const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encoder() {
    static const EncodeTiled f = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult r;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &r) != cudaSuccess ||
            r != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeTiled>(p);
    }();
    return f;
}

}  // namespace
}  // namespace bgtq
