// Attention of a packed batch of prompts of different lengths on the fifth-generation tensor
// cores: row i of sequence s attends keys j of the same sequence, with the causal mask
// j <= i + (keys - queries), softmax with a running maximum and sum (FP32).  A row that sees
// no key gives zeros and a log sum of minus infinity.
//
// A work item is a block of consecutive positions of one sequence with all query heads of one
// KV head: 128 rows a tile, floor(128 / group) positions x group heads, two tiles an item (one
// where there are few items), which share every K and V tile.  A CTA takes items until none is
// left.  Its sixteen warps have roles:
//   warps 0-3, 4-7  softmax of tile 0 and of tile 1, a thread a row: logits out of tensor memory,
//                   mask, running maximum, probabilities back into tensor memory (as 16-bit
//                   pairs in the columns where the logits were), and the output at the end
//   warp 8          TMA loads of Q, K and V (128-byte swizzle) into a ring of K / V tiles
//   warps 9, 10     the products of tile 0 and of tile 1: S = Q K^T (operands in shared memory), two
//                   K tiles ahead of softmax, and O += P V (P in tensor memory, V as it lies), FP32
//                   accumulators in tensor memory.  A warp of its own for each row tile keeps the waits
//                   of one chain under the products of the other
//   warp 11         the deal: items in order of falling length, dealt back and forth over the CTAs
//   warps 12-15     V tiles at a sequence's end or on the diagonal, before they are multiplied:
//                   rows past the end (another sequence's, or nothing) are zeroed, and an
//                   infinity or a NaN, which the zero probability of a row that does not see
//                   it would turn into a NaN, is taken out and given to the rows that do see it
// The accumulator is rescaled only when a row's maximum has grown by more than 2^8 since the
// last time: until then probabilities are taken relative to the older maximum, so they stay
// below 2^8, and P is FP16 or BF16 (the inputs' type) with the same relative error.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "serving.h"

namespace bgtq {
namespace {

constexpr float kLn2 = 0.6931471805599453f;
constexpr uint32_t kThreads = 512, kRows = 128;
constexpr uint32_t kStatusTimeout = 1u;  // a bounded wait ran out (bgtq_internal.h's kStatusWaitTimeout)
constexpr float kLazy = 8.0f;            // log2 of the growth of a maximum that is left standing

// ---- device helpers -----------------------------------------------------------------------

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
__device__ __forceinline__ void tm_store16(uint32_t at, const uint32_t *r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, "
                 "%13, %14, %15};" ::BGTQ_V8(r, 0), BGTQ_V8(r, 8), "r"(at) : "memory");
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max3_nan(float x, float y, float z) {  // NaN if one of them is
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
    return r;
}
__device__ __forceinline__ float max_nan(float x, float y) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
    return r;
}
// 2^(x c - from) of two values on the FMA pipe, for a whole `from` (below 2^20 in magnitude) and x c - from >= -126:
// adding 1.5 * 2^23 - from rounds x c to a whole number n in the low mantissa bits, and 2^f of the
// rest, -1/2 <= f <= 1/2, is the polynomial of degree 4 with the least largest relative error on
// that interval (Remez exchange): 2.7e-6 in FP32, 4e-8 on average.  n goes into the exponent.
constexpr float kRound = 12582912.0f;
__device__ __forceinline__ float2 ex2_fma(float2 x, float2 c, float2 shift) {
    const float2 t = __ffma2_rn(x, c, shift);                                   // shift = kRound - from
    const float2 f = __ffma2_rn(x, c, __fadd2_rn(shift, make_float2(-t.x, -t.y)));
    float2 p = __ffma2_rn(f, make_float2(0.0095701022f, 0.0095701022f), make_float2(0.055917859f, 0.055917859f));
    p = __ffma2_rn(p, f, make_float2(0.24024744f, 0.24024744f));
    p = __ffma2_rn(p, f, make_float2(0.69312179f, 0.69312179f));
    p = __ffma2_rn(p, f, make_float2(0.99999928f, 0.99999928f));
    p.x = __uint_as_float(__float_as_uint(p.x) + (__float_as_uint(t.x) << 23));
    p.y = __uint_as_float(__float_as_uint(p.y) + (__float_as_uint(t.y) << 23));
    return p;
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

// ---- shared memory ---------------------------------------------------------------------------

template <int D>
struct Plan {
    // Keys of a tile: as many as leave room for two tiles of logits and the outputs of both row
    // tiles in the 512 columns of tensor memory.
    static constexpr uint32_t kKeys = D == 128 ? 64 : 96;
    static constexpr uint32_t kColO = 4 * kKeys;                   // the first column of the outputs
    static constexpr uint32_t kChunks = D / 64;                    // 64-dimension columns of a tile
    static constexpr uint32_t kQChunk = kRows * 128, kQTile = kChunks * kQChunk;  // bytes: rows of 64 elements
    static constexpr uint32_t kChunk = kKeys * 128, kTile = kChunks * kChunk;
    static constexpr uint32_t kSlots = D == 128 ? 8 : 10;          // K and V tiles in the ring
    static constexpr int kFma = 6;                                 // exponentials of 16 on the FMA pipe
    static constexpr uint32_t kQ = 0, kRing = 2 * kQTile, kAfter = kRing + kSlots * kTile;
    static constexpr uint32_t kBad = kAfter;                       // [2 items][3 kinds][D] first keys
    static constexpr uint32_t kItems = kBad + 2 * 3 * D * 2;       // [2] Item
    static constexpr uint32_t kBars = kItems + 2 * 32;
    static constexpr uint32_t kBarCount = 3 * kSlots + 22;
    static constexpr uint32_t kWords = kBars + 8 * kBarCount;      // tensor memory base, stop, bad-value flags
    static constexpr uint32_t kTotal = kWords + 32 + 1024;         // and the slack to align the base
};

struct Item {
    int32_t token, count;  // first query row, positions (0: no more items)
    int32_t pos, head;     // first position in the sequence, KV head
    int32_t key, keys;     // first key row, the sequence's keys
    int32_t shift;         // keys - queries
    int32_t pad;
};

struct TileSpan {
    int32_t count, tiles, first;  // positions, key tiles, keys that the first row sees
};

template <int D, bool BF>
__global__ void __launch_bounds__(kThreads, 1) prompt_kernel(const __grid_constant__ PromptArgs a,
                                                             const __grid_constant__ CUtensorMap mq,
                                                             const __grid_constant__ CUtensorMap mk,
                                                             const __grid_constant__ CUtensorMap mv) {
    using P = Plan<D>;
    constexpr int32_t kKeys = (int32_t)P::kKeys;
    extern __shared__ unsigned char raw[];
    unsigned char *sm = raw + ((1024u - (smem_addr(raw) & 1023u)) & 1023u);
    const uint32_t base = smem_addr(sm), warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
    const uint32_t lane = threadIdx.x & 31u;
    uint16_t *bad = reinterpret_cast<uint16_t *>(sm + P::kBad);
    volatile Item *items = reinterpret_cast<volatile Item *>(sm + P::kItems);
    volatile uint32_t *words = reinterpret_cast<volatile uint32_t *>(sm + P::kWords);
    volatile uint32_t *stop = words + 1, *bad_flag = words + 2;  // bad_flag[2]
    const uint32_t bars = base + P::kBars;
    auto bar = [&](uint32_t i) { return bars + 8u * i; };
    constexpr uint32_t B_FULL = 0, B_FREE = P::kSlots, B_QFULL = 2 * P::kSlots, B_QFREE = B_QFULL + 2, B_S = B_QFREE + 2,
                       B_P = B_S + 4, B_O = B_P + 4, B_RAW = B_O + 4, B_ITEM = B_RAW + P::kSlots, B_TAKEN = B_ITEM + 2, B_END = B_TAKEN + 2;
    const uint32_t per = kRows / a.group;  // positions of a tile
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(base + P::kWords) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < P::kSlots; ++i) {
            bar_init(bar(B_FULL + i), 4);
            bar_init(bar(B_FREE + i), 2);
            bar_init(bar(B_RAW + i), 1);
        }
        for (uint32_t i = 0; i < 2; ++i) {
            bar_init(bar(B_QFULL + i), 1);
            bar_init(bar(B_QFREE + i), 1);
            bar_init(bar(B_S + 2 * i), 1);
            bar_init(bar(B_S + 2 * i + 1), 1);
            bar_init(bar(B_P + 2 * i), 4);
            bar_init(bar(B_P + 2 * i + 1), 4);
            bar_init(bar(B_O + 2 * i), 1);
            bar_init(bar(B_O + 2 * i + 1), 1);
            bar_init(bar(B_ITEM + i), 1);
            bar_init(bar(B_TAKEN + i), 15);
        }
        bar_init(bar(B_END), 1);
        bar_init(bar(B_END + 1), 1);
        words[1] = words[2] = words[3] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async();
    }
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = words[0];

    // a whole warp's wait: all of its lanes see the same answer
    auto all_wait = [&](uint32_t b, uint32_t parity) { return (bool)__all_sync(0xffffffffu, bar_wait(b, parity, stop)); };
    // The item in slot n & 1 of the deal, when it is there; a role gives it back with `taken`.
    auto next = [&](uint32_t n, Item &it) {
        if (!all_wait(bar(B_ITEM + (n & 1)), (n >> 1) & 1)) return false;
        const volatile Item &s = items[n & 1];
        // from one lane: uniform over the warp, for the compiler too
        it.token = __shfl_sync(0xffffffffu, s.token, 0), it.count = __shfl_sync(0xffffffffu, s.count, 0);
        it.pos = __shfl_sync(0xffffffffu, s.pos, 0), it.head = __shfl_sync(0xffffffffu, s.head, 0);
        it.key = __shfl_sync(0xffffffffu, s.key, 0), it.keys = __shfl_sync(0xffffffffu, s.keys, 0);
        it.shift = __shfl_sync(0xffffffffu, s.shift, 0);
        return it.count != 0;
    };
    auto taken = [&](uint32_t n) {
        __syncwarp();
        if (lane == 0) bar_arrive(bar(B_TAKEN + (n & 1)));
    };
    auto span = [&](const Item &it, int t) {
        TileSpan s;
        const int32_t at = t * (int32_t)per;
        s.count = max(0, min((int32_t)per, it.count - at));
        const int32_t from = it.pos + at + it.shift + 1;  // keys that the first row sees, if causal
        const int32_t upto = a.causal ? max(0, min(it.keys, from + s.count - 1)) : it.keys;
        s.tiles = s.count ? (upto + kKeys - 1) / kKeys : 0;
        s.first = a.causal ? max(0, min(it.keys, from)) : it.keys;
        return s;
    };

    if (warp < 8) {
        // ---- softmax: thread = row of tile t ----
        asm volatile("setmaxnreg.inc.sync.aligned.u32 184;");
        const int t = warp >> 2;
        const uint32_t row = threadIdx.x & 127u, p = row / a.group, g = row % a.group;
        const uint32_t lanes = (warp & 3u) * 32u << 16;
        const uint32_t to = tmem + lanes + P::kColO + t * D;
        // A bit for each of the two buffers of logits: the phase that its logits come in, and that of
        // the last product O += P V asked for from it.
        uint32_t phase_s = 0, phase_o = 3;
        const float inv_scale = 1.0f / a.scale;
        Item it;
        for (uint32_t n = 0; next(n, it); ++n) {
            const TileSpan sp = span(it, t);
            const bool live = p < (uint32_t)sp.count;
            int32_t sees = it.keys;
            if (a.causal) sees = max(0, min(it.keys, it.pos + t * (int32_t)per + (int32_t)p + it.shift + 1));
            float ref = -INFINITY, sum = 0.0f;  // the maximum that probabilities are relative to (log2 units)
            bool fine = true;
            for (int32_t j = 0; j < sp.tiles; ++j) {
                const uint32_t buf = j & 1, ts = tmem + lanes + (2 * t + buf) * kKeys;
                if (!(fine = all_wait(bar(B_S + 2 * t + buf), phase_s >> buf & 1u))) break;
                phase_s ^= 1u << buf;
                tc_after();
                uint32_t x[kKeys];
#pragma unroll
                for (int c = 0; c < kKeys / 32; ++c) tm_load(ts + 32 * c, x + 32 * c);
                tc_wait_ld();
                float *s = reinterpret_cast<float *>(x);
                const bool masked = (j + 1) * kKeys > sp.first;
                if (masked) {
                    const int32_t left = sees - j * kKeys;
#pragma unroll
                    for (int i = 0; i < kKeys; ++i)
                        if (i >= left) s[i] = -INFINITY;
                }
                float m0 = s[0], m1 = s[1], m2 = s[2], m3 = s[3];
#pragma unroll
                for (int i = 4; i + 7 < kKeys; i += 8) {
                    m0 = max3_nan(m0, s[i], s[i + 1]);
                    m1 = max3_nan(m1, s[i + 2], s[i + 3]);
                    m2 = max3_nan(m2, s[i + 4], s[i + 5]);
                    m3 = max3_nan(m3, s[i + 6], s[i + 7]);
                }
                m0 = max3_nan(m0, s[kKeys - 4], s[kKeys - 3]);
                m1 = max3_nan(m1, s[kKeys - 2], s[kKeys - 1]);
                // whole numbers (ex2_fma); a row that is no query stands at 0 and asks for nothing
                const float top = live ? ceilf(max_nan(max3_nan(m0, m1, m2), m3) * a.scale) : 0.0f;
                const bool grown = !(top <= ref + kLazy);  // each row for itself: no result depends on a neighbour
                if (j == 0) ref = top;
                else if (__any_sync(0xffffffffu, grown)) {
                    // not under a product that is still adding to the outputs
                    if (!(fine = all_wait(bar(B_O + 2 * t + (buf ^ 1u)), phase_o >> (buf ^ 1u) & 1u))) break;
                    tc_after();
                    const float f = grown ? ex2(ref - max_nan(ref, top)) : 1.0f;
                    if (grown) ref = max_nan(ref, top);
                    sum *= f;
#pragma unroll
                    for (int c = 0; c < D / 32; ++c) {
                        uint32_t o[32];
                        tm_load(to + 32 * c, o);
                        tc_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                        tm_store(to + 32 * c, o);
                    }
                }
                const float from = ref == -INFINITY ? 0.0f : ref;
                const float2 scale2 = make_float2(a.scale, a.scale), from2 = make_float2(-from, -from);
                float2 total = make_float2(0.0f, 0.0f);
                // Of 16 logits kFma take the FMA pipe: ex2 alone has 16 lanes an SM and clock.  Tiles with a
                // mask, and rows with an infinity, a NaN or a maximum past 2^20 in them, do without.
                const bool careful = masked || !(fabsf(from) <= 1048576.0f);
                if (careful) {
#pragma unroll
                    for (int i = 0; i < kKeys; i += 2) {
                        const float2 y = __ffma2_rn(make_float2(s[i], s[i + 1]), scale2, from2);
                        const float2 e = make_float2(ex2(y.x), ex2(y.y));
                        total = __fadd2_rn(total, e);
                        x[i / 2] = pack<BF>(e.x, e.y);
                    }
                } else {
                    const float least = (from - 126.0f) * inv_scale;
                    const float2 shift = make_float2(kRound - from, kRound - from);
#pragma unroll
                    for (int i = 0; i < kKeys; i += 2) {
                        float2 e;
                        if (i % 16 < P::kFma) e = ex2_fma(make_float2(fmaxf(s[i], least), fmaxf(s[i + 1], least)), scale2, shift);
                        else {
                            const float2 y = __ffma2_rn(make_float2(s[i], s[i + 1]), scale2, from2);
                            e = make_float2(ex2(y.x), ex2(y.y));
                        }
                        total = __fadd2_rn(total, e);
                        x[i / 2] = pack<BF>(e.x, e.y);
                    }
                }
                sum += total.x + total.y;
                tm_store(ts, x);
                if constexpr (kKeys == 96) tm_store16(ts + 32, x + 32);
                tc_wait_st();
                tc_before();
                __syncwarp();
                if (lane == 0) bar_arrive(bar(B_P + 2 * t + buf));
                phase_o ^= 1u << buf;
            }
            if (fine && sp.count) {
                if (sp.tiles) {
                    const uint32_t buf = (sp.tiles - 1) & 1;
                    if (!(fine = all_wait(bar(B_O + 2 * t + buf), phase_o >> buf & 1u))) break;
                    tc_after();
                }
                const bool none = sees == 0 || sum == 0.0f;
                const float inv = none ? 0.0f : 1.0f / sum;
                const uint32_t flagged = bad_flag[n & 1];
                const uint64_t at = (uint64_t)(it.token + t * (int32_t)per + (int32_t)p) * a.q_heads + it.head * a.group + g;
                uint16_t *out = static_cast<uint16_t *>(a.out) + at * D;
#pragma unroll
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t o[32];
                    if (sp.tiles) {
                        tm_load(to + 32 * c, o);
                        tc_wait_ld();
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = 0;
                    }
                    if (sees == 0) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = 0;
                    }
                    if (flagged) {
                        // infinities and NaN that this row sees: keys from `key0` on were looked through
                        const int32_t key0 = max(0, (span(it, 0).first / kKeys)) * kKeys;
                        const uint16_t *first = bad + (n & 1) * 3 * D + 32 * c;
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            const bool up = key0 + first[i] < sees, down = key0 + first[D + i] < sees;
                            if (key0 + first[2 * D + i] < sees || (up && down)) o[i] = 0x7fc00000u;
                            else if (up || down) o[i] = up ? 0x7f800000u : 0xff800000u;
                        }
                    }
                    if (live) {
#pragma unroll
                        for (int i = 0; i < 32; i += 8) {
                            uint4 v;
                            v.x = pack<BF>(__uint_as_float(o[i]) * inv, __uint_as_float(o[i + 1]) * inv);
                            v.y = pack<BF>(__uint_as_float(o[i + 2]) * inv, __uint_as_float(o[i + 3]) * inv);
                            v.z = pack<BF>(__uint_as_float(o[i + 4]) * inv, __uint_as_float(o[i + 5]) * inv);
                            v.w = pack<BF>(__uint_as_float(o[i + 6]) * inv, __uint_as_float(o[i + 7]) * inv);
                            *reinterpret_cast<uint4 *>(out + 32 * c + i) = v;
                        }
                    }
                }
                if (live && a.lse) a.lse[at] = none ? -INFINITY : (ref + __log2f(sum)) * kLn2;
                tc_before();
            }
            if (!fine) break;
            taken(n);
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (warp == 8) {
            // ---- loads ----
            // A tile that warps 12-15 look through lands on its slot's raw barrier, and they arrive on the
            // full one when they are done with it.
            uint32_t slot = 0, free_phase = 1, q_phase[2] = {1, 1}, issued = 0, full_phase = 0, raw = 0, raw_phase = 0;
            Item it;
            bool fine = true;
            for (uint32_t n = 0; fine && next(n, it); ++n) {
                const TileSpan s0 = span(it, 0), s1 = span(it, 1);
                const int32_t tiles = max(s0.tiles, s1.tiles);
                if (lane == 0) {
                    auto load_q = [&](int t) {
                        if (!(fine = fine && bar_wait(bar(B_QFREE + t), q_phase[t], stop))) return;
                        q_phase[t] ^= 1;
                        bar_expect(bar(B_QFULL + t), P::kChunks * per * a.group * 128u);
                        for (uint32_t c = 0; c < P::kChunks; ++c)
                            tma3(base + P::kQ + t * P::kQTile + c * P::kQChunk, &mq, bar(B_QFULL + t), 64 * c,
                                 it.head * (int32_t)a.group, it.token + t * (int32_t)per);
                    };
                    auto load_kv = [&](const CUtensorMap *map, int32_t j, bool look) {
                        if (!(fine = fine && bar_wait(bar(B_FREE + slot), free_phase, stop))) return;
                        const uint32_t on = bar((look ? B_RAW : B_FULL) + slot), bit = 1u << slot;
                        bar_expect(on, P::kTile);
                        if (!look)
                            for (int i = 0; i < 3; ++i) bar_arrive(on);
                        for (uint32_t c = 0; c < P::kChunks; ++c)
                            tma3(base + P::kRing + slot * P::kTile + c * P::kChunk, map, on, 64 * c, it.head,
                                 it.key + j * kKeys);
                        issued |= bit;
                        raw = look ? raw | bit : raw & ~bit;
                        full_phase = (full_phase & ~bit) | (free_phase ^ 1u) << slot;
                        raw_phase ^= look ? bit : 0;
                        if (++slot == P::kSlots) slot = 0, free_phase ^= 1;
                    };
                    if (s0.tiles) load_q(0);
                    if (tiles) load_kv(&mk, 0, false);
                    if (s1.tiles) load_q(1);
                    if (tiles > 1) load_kv(&mk, 1, false);
                    for (int32_t j = 0; j < tiles && fine; ++j) {
                        load_kv(&mv, j, (j + 1) * kKeys > s0.first);
                        if (j + 2 < tiles) load_kv(&mk, j + 2, false);
                    }
                }
                fine = __shfl_sync(0xffffffffu, fine, 0);
                taken(n);
            }
            // copies in flight land before the CTA ends (they have, unless a wait ran out)
            if (lane == 0 && *stop) {
                uint32_t none = 0;
                for (uint32_t i = 0; i < P::kSlots; ++i)
                    if (issued >> i & 1u)
                        bar_wait(bar((raw >> i & 1u ? B_RAW : B_FULL) + i), raw >> i & 1u ? ~raw_phase >> i & 1u : full_phase >> i & 1u,
                                 &none);
                for (int t = 0; t < 2; ++t) bar_wait(bar(B_QFULL + t), q_phase[t] ^ 1u, &none);
            }
        } else if (warp <= 10) {
            // ---- products of tile t: the warp stays together, one lane issues ----
            const int t = (int)warp - 9;
            uint32_t slot = 0, full_phase = 0, q_phase = 0, p_phase = 0;
            constexpr uint32_t ID_S = product(BF, 0, P::kKeys), ID_O = product(BF, 1, D);
            const uint32_t q_at = base + P::kQ + t * P::kQTile, s_at = tmem + 2 * t * kKeys, o_at = tmem + P::kColO + t * D;
            Item it;
            bool fine = true;
            for (uint32_t n = 0; fine && next(n, it); ++n) {
                const TileSpan sp = span(it, t), other = span(it, t ^ 1);
                const int32_t tiles = max(sp.tiles, other.tiles);
                auto advance = [&]() {
                    if (++slot == P::kSlots) slot = 0, full_phase ^= 1;
                };
                // the logits of K tile j (in slot k), and the slot's release
                auto logits = [&](uint32_t k, int32_t j) {
                    if (!elect()) return;
                    if (j >= sp.tiles) {
                        bar_arrive(bar(B_FREE + k));
                        return;
                    }
                    const uint32_t q = operand(q_at, 0), key = operand(base + P::kRing + k * P::kTile, 0), d = s_at + (j & 1) * kKeys;
#pragma unroll
                    for (uint32_t c = 0; c < P::kChunks; ++c)
#pragma unroll
                        for (uint32_t s = 0; s < 4; ++s)
                            mma_ss(d, q + (c * P::kQChunk + 32 * s) / 16, key + (c * P::kChunk + 32 * s) / 16, ID_S, c | s);
                    tc_commit(bar(B_S + 2 * t + (j & 1)));
                    tc_commit(bar(B_FREE + k));
                    if (j + 1 == sp.tiles) tc_commit(bar(B_QFREE + t));
                };
                if (sp.tiles) {
                    if (!(fine = all_wait(bar(B_QFULL + t), q_phase))) break;
                    q_phase ^= 1;
                }
                // the logits run two tiles ahead of the outputs
                for (int32_t j = 0; j < 2 && j < tiles; ++j) {
                    if (!(fine = all_wait(bar(B_FULL + slot), full_phase))) break;
                    tc_after();
                    logits(slot, j);
                    __syncwarp();
                    advance();
                }
                for (int32_t j = 0; j < tiles && fine; ++j) {
                    const uint32_t v = slot;
                    if (!(fine = all_wait(bar(B_FULL + v), full_phase))) break;
                    advance();
                    const uint32_t k = slot;
                    const bool more = j + 2 < tiles;
                    if (more) {
                        if (!(fine = all_wait(bar(B_FULL + k), full_phase))) break;
                        advance();
                    }
                    const uint32_t buf = j & 1;
                    if (j < sp.tiles) {
                        if (!(fine = all_wait(bar(B_P + 2 * t + buf), p_phase >> buf & 1u))) break;
                        p_phase ^= 1u << buf;
                    }
                    tc_after();
                    if (elect()) {
                        if (j < sp.tiles) {
                            const uint32_t val = operand(base + P::kRing + v * P::kTile, P::kChunk), pr = s_at + buf * kKeys;
#pragma unroll
                            for (uint32_t s = 0; s < P::kKeys / 16; ++s)
                                mma_ts(o_at, pr + 8 * s, val + s * 128, ID_O, j | (int32_t)s);
                            tc_commit(bar(B_O + 2 * t + buf));
                            tc_commit(bar(B_FREE + v));
                        } else bar_arrive(bar(B_FREE + v));
                    }
                    __syncwarp();
                    if (more) logits(k, j + 2);
                    __syncwarp();
                }
                if (fine) taken(n);
            }
            // products in flight end before the tensor memory is given back
            __syncwarp();
            if (*stop && elect()) {
                uint32_t none = 0;
                tc_commit(bar(B_END + t));
                bar_wait(bar(B_END + t), 0, &none);
            }
        } else if (warp == 11) {
            // ---- the deal ----
            // Sequence s has ceil(queries / (tiles per item)) blocks; block b of every sequence that
            // has it is level b.  Items go by falling level (the last blocks see the most keys), a level's
            // sequences in order, KV heads innermost; item r goes to CTA r of a round, rounds back and forth.
            const int32_t block = (int32_t)(a.tiles * per);
            auto blocks_of = [&](uint32_t s) -> int32_t {
                if (s >= a.sequences) return 0;
                const int32_t q0 = __ldg(a.starts + s), q1 = __ldg(a.starts + s + 1);
                const int32_t k0 = __ldg(a.key_starts + s), k1 = __ldg(a.key_starts + s + 1);
                if (q0 < 0 || k0 < 0 || q1 < q0 || k1 < k0 || (uint64_t)q1 > a.q_tokens || (uint64_t)k1 > a.k_tokens) {
                    if (blockIdx.x == 0) atomicOr(a.status, kStatusBadExtent);
                    return 0;
                }
                return (q1 - q0 + block - 1) / block;
            };
            int32_t level = 0;
            for (uint32_t s = lane; s < a.sequences; s += 32) level = max(level, blocks_of(s));
            level = __reduce_max_sync(0xffffffffu, level);
            uint64_t before = 0, upto = 0;  // items of levels above this one, and with it
            uint64_t r = blockIdx.x;
            for (uint32_t n = 0;; ++n) {
                r = (uint64_t)n * gridDim.x + (n & 1u ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
                while (upto <= r && level > 0) {
                    --level;
                    before = upto;
                    uint32_t c = 0;
                    for (uint32_t s = lane; s < a.sequences; s += 32) c += blocks_of(s) > level;
                    upto += (uint64_t)__reduce_add_sync(0xffffffffu, c) * a.kv_heads;
                }
                Item it{};
                if (r < upto) {
                    uint32_t nth = (uint32_t)((r - before) / a.kv_heads);
                    it.head = (int32_t)((r - before) % a.kv_heads);
                    for (uint32_t s0 = 0; s0 < a.sequences; s0 += 32) {
                        const uint32_t has = __ballot_sync(0xffffffffu, blocks_of(s0 + lane) > level);
                        const uint32_t c = __popc(has);
                        if (nth >= c) {
                            nth -= c;
                            continue;
                        }
                        const uint32_t s = s0 + __fns(has, 0, nth + 1);
                        const int32_t q0 = __ldg(a.starts + s), nq = __ldg(a.starts + s + 1) - q0;
                        it.pos = level * block;
                        it.token = q0 + it.pos;
                        it.count = min(block, nq - it.pos);
                        it.key = __ldg(a.key_starts + s);
                        it.keys = __ldg(a.key_starts + s + 1) - it.key;
                        it.shift = it.keys - nq;
                        break;
                    }
                }
                if (n >= 2 && !all_wait(bar(B_TAKEN + (n & 1)), ((n >> 1) & 1) ^ 1)) break;
                if (lane == 0) {
                    volatile Item &d = items[n & 1];
                    d.token = it.token, d.count = it.count, d.pos = it.pos, d.head = it.head;
                    d.key = it.key, d.keys = it.keys, d.shift = it.shift;
                    bad_flag[n & 1] = 0;
                    bar_arrive(bar(B_ITEM + (n & 1)));
                }
                __syncwarp();
                if (it.count == 0) break;
            }
        } else {
            // ---- V tiles that not every row sees: each of four warps its share of the dimensions ----
            constexpr uint32_t kUnits = D / 8 / 4;  // 16-byte units of a row in a warp's share
            const uint32_t share = warp - 12;
            uint32_t slot = 0, raw_phase = 0;
            Item it;
            bool fine = true;
            for (uint32_t n = 0; fine && next(n, it); ++n) {
                const TileSpan s0 = span(it, 0), s1 = span(it, 1);
                const int32_t tiles = max(s0.tiles, s1.tiles), begin = max(0, s0.first / kKeys);
                uint16_t *first = bad + (n & 1) * 3 * D;
                for (uint32_t i = lane; i < 3 * D / 4; i += 32) first[i / (D / 4) * D + share * (D / 4) + i % (D / 4)] = 0xffff;
                for (int32_t j = begin; j < tiles; ++j) {
                    if ((j + 1) * kKeys <= s0.first) continue;
                    // in the order K 0, K 1, V 0, K 2, V 1, .. of the item's loads
                    const uint32_t v = (slot + (uint32_t)min(2 * j + 2, 2 * tiles - 1)) % P::kSlots;
                    if (!(fine = all_wait(bar(B_RAW + v), raw_phase >> v & 1u))) break;
                    raw_phase ^= 1u << v;
                    unsigned char *tile = sm + P::kRing + v * P::kTile;
                    const int32_t rows = min(kKeys, it.keys - j * kKeys);
                    uint32_t found = 0;
                    constexpr uint32_t E = BF ? 0x7f80u : 0x7c00u;
#pragma unroll 4
                    for (uint32_t i = lane; i < P::kKeys * kUnits; i += 32) {
                        const uint32_t r = i / kUnits, u = share * kUnits + i % kUnits;
                        uint4 *w = reinterpret_cast<uint4 *>(tile + u / 8 * P::kChunk + r * 128 + ((u % 8 ^ (r & 7)) << 4));
                        if ((int32_t)r >= rows) *w = make_uint4(0, 0, 0, 0);
                        else {
                            const uint4 x = *w;
                            const uint32_t y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                            for (int k = 0; k < 4; ++k) found |= (y[k] & E) == E || (y[k] >> 16 & E) == E;
                        }
                    }
                    if (__any_sync(0xffffffffu, found)) {
                        __syncwarp();
                        for (uint32_t i = lane; i < (uint32_t)D / 4; i += 32) {
                            const uint32_t d = share * (D / 4) + i;
                            for (int32_t k = 0; k < rows; ++k) {
                                uint16_t *w = reinterpret_cast<uint16_t *>(tile + d / 64 * P::kChunk + k * 128 +
                                                                           (((d % 64 / 8) ^ (k & 7)) << 4)) + d % 8;
                                const uint32_t x = *w;
                                if ((x & E) != E) continue;
                                *w = 0;
                                const uint32_t kind = (x & 0x7fffu) != E ? 2 : x >> 15;  // 0 inf, 1 -inf, 2 NaN
                                const uint32_t at = (uint32_t)((j - begin) * kKeys + k);
                                if (at < first[kind * D + d]) first[kind * D + d] = (uint16_t)at;
                            }
                        }
                        if (lane == 0) bad_flag[n & 1] = 1;
                    }
                    fence_async();
                    __syncwarp();
                    if (lane == 0) bar_arrive(bar(B_FULL + v));
                }
                slot = (slot + 2 * (uint32_t)tiles) % P::kSlots;
                if (fine) taken(n);
            }
        }
    }
    // every role has left its loop; on a timeout the waits above were cut short
    __syncwarp();
    tc_before();
    __syncthreads();
    if (threadIdx.x == 0 && *stop) atomicOr(a.status, kStatusTimeout);
    if (warp == 8) {
        tc_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    }
}

// ---- launch ------------------------------------------------------------------------------------

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

// [tokens][heads][dim] as boxes of `rows` tokens x `heads_box` heads x 64 dimensions.
bool make_map(CUtensorMap *m, bool bf16, const void *p, uint32_t dim, uint32_t heads, uint64_t tokens, int64_t head,
              int64_t token, uint32_t heads_box, uint32_t rows) {
    const cuuint64_t size[3] = {dim, heads, tokens};
    const cuuint64_t stride[2] = {(cuuint64_t)head * 2, (cuuint64_t)token * 2};
    const cuuint32_t box[3] = {64, heads_box, rows}, step[3] = {1, 1, 1};
    return encoder()(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void *>(p),
                     size, stride, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                     CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, bool BF>
cudaError_t run(const PromptArgs &args, cudaStream_t s) {
    using P = Plan<D>;
    if (!encoder()) return cudaErrorNotSupported;
    auto kernel = prompt_kernel<D, BF>;
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess || dev >= 64) return e != cudaSuccess ? e : cudaErrorInvalidDevice;
    static bool ready[64] = {};
    if (!ready[dev]) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)P::kTotal);
        if (e != cudaSuccess) return e;
        ready[dev] = true;
    }
    PromptArgs a = args;
    const uint32_t per = kRows / a.group;
    CUtensorMap mq, mk, mv;
    // without any key nothing is loaded; the maps only have to be valid
    const bool keys = a.k_tokens != 0;
    if (!make_map(&mq, BF, a.q, D, a.q_heads, a.q_tokens, a.q_head, a.q_token, a.group, per) ||
        !make_map(&mk, BF, keys ? a.k : a.q, D, a.kv_heads, keys ? a.k_tokens : 1, a.k_head, a.k_token, 1, P::kKeys) ||
        !make_map(&mv, BF, keys ? a.v : a.q, D, a.kv_heads, keys ? a.k_tokens : 1, a.v_head, a.v_token, 1, P::kKeys))
        return cudaErrorInvalidValue;
    // two tiles an item share K and V loads; where that leaves SMs without work, one
    const uint64_t items2 = a.kv_heads * ((a.q_tokens + 2 * per - 1) / (2 * per));
    a.tiles = items2 >= (uint64_t)sms ? 2 : 1;
    const uint64_t most = a.kv_heads * ((a.q_tokens + a.tiles * per - 1) / (a.tiles * per) + a.sequences);
    kernel<<<(uint32_t)(most < (uint64_t)sms ? most : sms), kThreads, P::kTotal, s>>>(a, mq, mk, mv);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_prompt(const PromptArgs &a, cudaStream_t s) {
    if (a.dtype == BGTQ_BF16) return a.dim == 64 ? run<64, true>(a, s) : run<128, true>(a, s);
    return a.dim == 64 ? run<64, false>(a, s) : run<128, false>(a, s);
}

}  // namespace bgtq
