// Attention of a packed batch of prompts of different lengths on the fifth-generation tensor
// cores: row i of sequence s attends keys j of the same sequence, with the causal mask
// j <= i + (keys - queries), softmax with a running maximum and sum (FP32).  A row that sees
// no key gives zeros and a log sum of minus infinity.
//
// A work item is a block of consecutive positions of one sequence with all query heads of one
// KV head: 128 rows a tile, floor(128 / group) positions x group heads, up to four tiles (head
// dim 64) or two (128), which share every K and V tile of 64 keys.  Tensor memory sets these
// numbers: logits and outputs of all row tiles fill its 512 columns, 4 x (64 + 64) at head dim
// 64, 2 x (2 x 64 + 128) at 128, where the logits are double-buffered instead.  One CTA an SM
// takes an equal range of the items' keys, computed on the device from the lengths; an item
// across two ranges is done in parts, which its last CTA joins.  The warps have roles:
//   softmax     four warps a row tile, a thread a row: logits out of tensor memory, mask, running
//               maximum, probabilities back into tensor memory (as 16-bit pairs in the columns
//               where the logits were), and the outputs at the end
//   deal, loads one warp: this CTA's share of the items, and the TMA loads of Q, K and V (128-byte
//               swizzle) into a ring of stages
//   products    two warps, each for half of the row tiles: S = Q K^T (operands in shared memory)
//               ahead of softmax and O += P V (P in tensor memory, V as it lies), FP32
//               accumulators in tensor memory.  The warp stays together and one lane issues, so
//               that the operands sit in uniform registers; a stage holds V j and the next K
//               tile to come, so that a step has two waits and two commits
//   ends        one warp: V tiles at a sequence's end or on the diagonal, before they are
//               multiplied: rows past the end (another sequence's, or nothing) are zeroed, and an
//               infinity or a NaN, which the zero probability of a row that does not see it would
//               turn into a NaN, is taken out and added to the rows that do see it.  (In
//               a tile that every row sees an infinity is multiplied like any value: by zero, which
//               makes a NaN, where its probability is below what P's type holds)
//
// What bounds it.  A K tile of 64 keys costs a row tile 512 (head dim 128) or 256 clocks of
// tensor arithmetic; the logits' products, which read both operands from shared memory, take 48
// clocks an instruction for 32 of arithmetic, so products alone come to 640 or 320.  Its 8192
// exponentials take 512 clocks at 16 a clock, so some go to the FMA pipe (kFma).  At head dim 128
// products are the longer: four prompts of 3500 to 4096 tokens, 32 / 8 heads, causal, run at 1.03
// to 1.12 PFLOP/s (425 to 460 us, with the power limit's clock).  At 64 it is softmax: two prompts
// of 8192 tokens, 14 / 2 heads, 279 to 290 us, 830 to 860 TFLOP/s, with the exponential pipe 57 % full and
// the tensor pipe 32 %, so neither is the limit by itself; most waits are for tensor memory, in each row's
// chain of logits, maximum, exponentials and probabilities.  Short prompts are bound by their chain
// of latencies: 37 tokens take 8.3 us.  The tails (outputs,
// joining) are short loops on purpose: unrolled, their instruction fetches cost 10 us a call.
// The accumulator is rescaled only when a row's maximum has grown by more than 2^8 since the
// last time: until then probabilities are taken relative to the older maximum, so they stay
// below 2^8.  P is FP16 or BF16, the inputs' type, and its rounding is the formula's one beside the outputs'
// own; sums take probabilities before it.  In FP16 they are multiplied by 2^7, and the sums with them:
// what is above 2^-21 of a row's largest keeps 11 bits, what is below is held to 2^-32 of it.  (Rescaling at every
// growth: three prompts of 300 to 512 tokens after 3500, 32 / 8 heads of 128, 120 us for 83.)
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "serving.h"

namespace bgtq {
namespace {

constexpr float kLn2 = 0.6931471805599453f;
constexpr uint32_t kRows = 128;
constexpr uint32_t kStatusTimeout = 1u;  // a bounded wait ran out (bgtq_internal.h's kStatusWaitTimeout)
constexpr uint32_t kDeal = 4;            // items dealt ahead
// What an item costs beside its keys, in keys: queries, outputs, joining.  (None: 12 prompts of 1 to 2047 tokens,
// 14 / 2 heads of 64, 51 us for 42, two of 8192 tokens 345 us for 293; 200 and 600 are within 5 % of 384.)
constexpr int64_t kItemCost = 384;
// Items of no more keys are not split: joining costs as much as they do.  (512: 700 tokens of 32 heads of 64, 28.5 us
// for 20.9; 2048: 64 tokens after 2000, 32 / 8 heads of 128, 42 us for 25.)
constexpr int32_t kWhole = 1024;
// Keys that make a CTA worth its while where items are few and long.  (16 tokens after 8000, 14 / 2 heads of 64:
// 28.2 us with 512, 29.0 with 1024, 38.5 with 2048; 64 tokens after 2000 as above: 25.0, 26.4, 49.)
constexpr int64_t kPiece = 512;
constexpr int kJoin = 2;                 // parts of an item that are joined at a time (1: 2 % slower, 4: 5 %)
constexpr float kLazy = 8.0f;            // log2 of the growth of a maximum that is left standing
// log2 of what probabilities are multiplied by: with kLazy, what FP16 holds.  (Less growth and more of this, in FP16:
// 2^4 and 2^11 take 3 % more for three prompts of 300 to 512 tokens after 3500, 8 % for four of 3500 to 4096.)
template <bool BF> constexpr float kUp = BF ? 0.0f : 15.0f - kLazy;

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

// ---- shared memory ---------------------------------------------------------------------------

template <int D>
struct Plan {
    static constexpr uint32_t kTiles = D == 64 ? 4 : 2;            // row tiles of an item, at most
    static constexpr uint32_t kBufs = D == 64 ? 1 : 2;             // of logits, for each row tile
    static constexpr uint32_t kKeys = 64;                          // of a K or V tile
    static constexpr uint32_t kColO = kTiles * kBufs * kKeys;      // the first column of the outputs
    static constexpr uint32_t kThreads = 128 * kTiles + 128;
    // Registers: kThreads x 96 (head dim 64) or 168 at launch, 128 kTiles x kSoft + 128 x kRest afterwards: 61440
    // or 64512 in all.  More does not fit beside the tiles; the softmax threads hold 64 logits and little else.
    static constexpr uint32_t kSoft = D == 64 ? 104 : 216, kRest = D == 64 ? 64 : 72;
    // Exponentials of 16 on the FMA pipe.  Head dim 64, two prompts of 8192 tokens: none 319 us, 2 293, 4 297;
    // 128, three of 300 to 512 after 3500: none 88.6 us, 2 88.5, 4 86.9, 6 83.6, 10 90.6.
    static constexpr int kFma = D == 64 ? 2 : 6;
    static constexpr uint32_t kChunks = D / 64;                    // 64-dimension columns of a tile
    static constexpr uint32_t kQChunk = kRows * 128, kQTile = kChunks * kQChunk;  // bytes: rows of 64 elements
    static constexpr uint32_t kChunk = kKeys * 128, kTile = kChunks * kChunk;
    static constexpr uint32_t kStages = D == 128 ? 4 : 7;          // of two K or V tiles in the ring
    static constexpr uint32_t kQ = 0, kRing = kTiles * kQTile, kAfter = kRing + kStages * 2 * kTile;
    static constexpr int kTurn = D == 64 ? 16 : 32;                // dimensions of an output row stored at a time: what registers hold
    static constexpr uint32_t kOut = kAfter;                       // [softmax warps][32 rows][kTurn] outputs
    static constexpr uint32_t kBad = kOut + 4 * kTiles * 64 * kTurn;                    // [kDeal items][3 kinds][D] first keys
    static constexpr uint32_t kItems = kBad + kDeal * 3 * D * 2;   // [kDeal] Item
    static constexpr uint32_t kBars = kItems + kDeal * 48;
    static constexpr uint32_t kBarCount = 3 * kStages + 2 * kTiles + 3 * kTiles * kBufs + 2 * kDeal + 2;
    static constexpr uint32_t kWords = kBars + 8 * kBarCount;      // tensor memory base, stop, bad-value flags
    static constexpr uint32_t kTotal = kWords + 32 + 1024;         // and the slack to align the base
};

// A work item, or the K tiles [from, upto) of one.
struct Item {
    int32_t token, count;  // first query row, positions (0: no more items)
    int32_t pos, head;     // first position in the sequence, KV head
    int32_t key, keys;     // first key row, the sequence's keys
    int32_t shift;         // keys - queries
    int32_t from, upto;
    int32_t part, parts;   // the CTA that has the item's first K tile, how many CTAs have one (1: this is all of it)
    int32_t pad;
};

// Quotients of nonnegative numbers: 32-bit division where it will do, which is nearly always.
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
    return (uint64_t)(a | b) >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b);
}

struct TileSpan {
    int32_t count, tiles, first;  // positions, K tiles of this piece, keys that the first row sees
};

template <int D, bool BF>
__global__ void __launch_bounds__(Plan<D>::kThreads, 1) prompt_kernel(const __grid_constant__ PromptArgs a,
                                                             const __grid_constant__ CUtensorMap mq,
                                                             const __grid_constant__ CUtensorMap mk,
                                                             const __grid_constant__ CUtensorMap mv) {
    using P = Plan<D>;
    constexpr int32_t kKeys = (int32_t)P::kKeys;
    constexpr uint32_t NT = P::kTiles, NB = P::kBufs;
    extern __shared__ unsigned char raw[];
    unsigned char *sm = raw + ((1024u - (smem_addr(raw) & 1023u)) & 1023u);
    const uint32_t base = smem_addr(sm), warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
    const uint32_t lane = threadIdx.x & 31u;
    uint16_t *bad = reinterpret_cast<uint16_t *>(sm + P::kBad);
    volatile Item *items = reinterpret_cast<volatile Item *>(sm + P::kItems);
    volatile uint32_t *words = reinterpret_cast<volatile uint32_t *>(sm + P::kWords);
    volatile uint32_t *stop = words + 1, *bad_flag = words + 2;  // bad_flag[kDeal]
    const uint32_t bars = base + P::kBars;
    auto bar = [&](uint32_t i) { return bars + 8u * i; };
    // a stage is full, free, or (raw) to be looked through first; of each row tile: its queries are there, its
    // queries are read; of each buffer of logits: they are there (and what was asked of the tensor cores before
    // them is done), the probabilities are, the last product from it is done (a barrier of its own: the next
    // item's logits may come before softmax has looked); of each item: it is dealt, it is given back
    constexpr uint32_t B_FULL = 0, B_FREE = P::kStages, B_RAW = 2 * P::kStages, B_QFULL = 3 * P::kStages,
                       B_QFREE = B_QFULL + NT, B_S = B_QFREE + NT, B_P = B_S + NT * NB, B_O = B_P + NT * NB, B_ITEM = B_O + NT * NB,
                       B_TAKEN = B_ITEM + kDeal, B_END = B_TAKEN + kDeal;
    constexpr uint32_t W_LOAD = 4 * NT, W_MMA = W_LOAD + 1, W_ENDS = W_LOAD + 3;  // the warps past softmax
    const uint32_t per = kRows / a.group;  // positions of a tile
    if (warp == W_LOAD) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(base + P::kWords) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < P::kStages; ++i) {
            bar_init(bar(B_FULL + i), 1);
            bar_init(bar(B_FREE + i), 2);
            bar_init(bar(B_RAW + i), 1);
        }
        for (uint32_t i = 0; i < NT; ++i) {
            bar_init(bar(B_QFULL + i), 1);
            bar_init(bar(B_QFREE + i), 1);
        }
        for (uint32_t i = 0; i < NT * NB; ++i) {
            bar_init(bar(B_S + i), 1);
            bar_init(bar(B_P + i), 4);
            bar_init(bar(B_O + i), 1);
        }
        for (uint32_t i = 0; i < kDeal; ++i) {
            bar_init(bar(B_ITEM + i), 1);
            bar_init(bar(B_TAKEN + i), 4 * NT + 3);  // all warps but the dealer
        }
        bar_init(bar(B_END), 1);
        bar_init(bar(B_END + 1), 1);
        for (uint32_t i = 1; i < 2 + kDeal; ++i) words[i] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async();
    }
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = words[0];

    // a whole warp's wait: all of its lanes see the same answer
    auto all_wait = [&](uint32_t b, uint32_t parity) {
        if (__all_sync(0xffffffffu, bar_try(b, parity))) return true;
        return (bool)__all_sync(0xffffffffu, bar_wait_slow(b, parity, stop));
    };
    auto read = [&](uint32_t n, Item &it) {
        const volatile Item &s = items[n % kDeal];
        // from one lane: uniform over the warp, for the compiler too
        it.token = __shfl_sync(0xffffffffu, s.token, 0), it.count = __shfl_sync(0xffffffffu, s.count, 0);
        it.pos = __shfl_sync(0xffffffffu, s.pos, 0), it.head = __shfl_sync(0xffffffffu, s.head, 0);
        it.key = __shfl_sync(0xffffffffu, s.key, 0), it.keys = __shfl_sync(0xffffffffu, s.keys, 0);
        it.shift = __shfl_sync(0xffffffffu, s.shift, 0), it.from = __shfl_sync(0xffffffffu, s.from, 0);
        it.upto = __shfl_sync(0xffffffffu, s.upto, 0), it.part = __shfl_sync(0xffffffffu, s.part, 0);
        it.parts = __shfl_sync(0xffffffffu, s.parts, 0);
    };
    // Item n of the deal, when it is there; a role gives its slot back with `taken`.
    auto next = [&](uint32_t n, Item &it) {
        if (!all_wait(bar(B_ITEM + n % kDeal), n / kDeal & 1)) return false;
        read(n, it);
        return it.count != 0;
    };
    auto taken = [&](uint32_t n) {
        __syncwarp();
        if (lane == 0) bar_arrive(bar(B_TAKEN + n % kDeal));
    };
    auto span = [&](const Item &it, int t) {
        TileSpan s;
        const int32_t at = t * (int32_t)per;
        s.count = max(0, min((int32_t)per, it.count - at));
        const int32_t from = it.pos + at + it.shift + 1;  // keys that the first row sees, if causal
        const int32_t upto = a.causal ? max(0, min(it.keys, from + s.count - 1)) : it.keys;
        s.tiles = s.count ? max(0, min(it.upto, (upto + kKeys - 1) / kKeys) - it.from) : 0;
        s.first = a.causal ? max(0, min(it.keys, from)) : it.keys;
        return s;
    };
    auto tiles_of = [&](const Item &it) {  // K tiles that any of its row tiles takes
        int32_t n = 0;
        for (uint32_t t = 0; t < NT; ++t) n = max(n, span(it, (int)t).tiles);
        return n;
    };

    if (warp < 4 * NT) {
        // ---- softmax: thread = row of tile t ----
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(P::kSoft));
        const int t = (int)warp >> 2;
        const uint32_t row = threadIdx.x & 127u, p = row / a.group, g = row % a.group;
        const uint32_t lanes = (warp & 3u) * 32u << 16;
        const uint32_t to = tmem + lanes + P::kColO + t * D;
        uint32_t phase = 0, phase_o = 0;  // a bit for each buffer of logits
        // keys that this thread's row sees
        auto sees_of = [&](const Item &it) {
            return a.causal ? max(0, min(it.keys, it.pos + t * (int32_t)per + (int32_t)p + it.shift + 1)) : it.keys;
        };
        // (of an item only what the loop needs stays in registers; the rest is read again at its end)
        for (uint32_t n = 0;; ++n) {
            int32_t tiles, unmasked, left;  // K tiles; keys that all rows see and that this row sees, from this piece's first on
            {
                Item it;
                if (!next(n, it)) break;
                const TileSpan sp = span(it, t);
                tiles = sp.tiles;
                unmasked = sp.first - it.from * kKeys;
                left = sees_of(it) - it.from * kKeys;
            }
            float ref = -INFINITY, sum = 0.0f;  // the maximum that probabilities are relative to (log2 units)
            bool fine = true;
            for (int32_t j = 0; j < tiles; ++j) {
                const uint32_t buf = j % NB, ts = tmem + lanes + (NB * t + buf) * kKeys;
                if (!(fine = all_wait(bar(B_S + NB * t + buf), phase >> buf & 1u))) break;
                phase ^= 1u << buf;
                tc_after();
                uint32_t x[kKeys];
                tm_load(ts, x);
                tm_load(ts + 32, x + 32);
                tc_wait_ld();
                float *s = reinterpret_cast<float *>(x);
                if ((j + 1) * kKeys > unmasked) {
#pragma unroll
                    for (int i = 0; i < kKeys; ++i)
                        if (i >= left - j * kKeys) s[i] = -INFINITY;
                }
                float m0 = max3(s[0], s[1], s[2]), m1 = max3(s[3], s[4], s[5]), m2 = max3(s[6], s[7], s[8]);
                float m3 = max3(s[9], s[10], s[11]);
#pragma unroll
                for (int i = 12; i + 7 < kKeys; i += 8) {
                    m0 = max3(m0, s[i], s[i + 1]);
                    m1 = max3(m1, s[i + 2], s[i + 3]);
                    m2 = max3(m2, s[i + 4], s[i + 5]);
                    m3 = max3(m3, s[i + 6], s[i + 7]);
                }
                m0 = max3(m0, s[kKeys - 4], s[kKeys - 3]);
                m1 = max3(m1, s[kKeys - 2], s[kKeys - 1]);
                const float top = fmaxf(max3(m0, m1, m2), m3) * a.scale;
                const bool grown = top > ref + kLazy;  // each row for itself, not by the others of the warp
                if (j == 0) ref = top;
                else if (__any_sync(0xffffffffu, grown)) {
                    // not under a product that is still adding to the outputs: the other buffer's next logits
                    // come after it, or nothing does (with one buffer, these logits did)
                    if (NB == 2) {
                        const uint32_t other = buf ^ 1u, on = NB * t + other;
                        fine = j + 1 < tiles ? all_wait(bar(B_S + on), phase >> other & 1u) : all_wait(bar(B_O + on), phase_o >> other & 1u);
                        if (!fine) break;
                        tc_after();
                    }
                    const float f = grown ? ex2(ref - top) : 1.0f;
                    if (grown) ref = top;
                    sum *= f;
#pragma unroll 1
                    for (int c = 0; c < D / 16; ++c) {
                        uint32_t o[16];
                        tm_load16(to + 16 * c, o);
                        tc_wait_ld();
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                        tm_store16(to + 16 * c, o);
                    }
                }
                const float from = (ref == -INFINITY ? 0.0f : ref) - kUp<BF>;
                const float2 scale2 = make_float2(a.scale, a.scale), from2 = make_float2(-from, -from);
                float2 total = make_float2(0.0f, 0.0f);
#pragma unroll
                for (int i = 0; i < kKeys; i += 2) {
                    const float2 v = __ffma2_rn(make_float2(s[i], s[i + 1]), scale2, from2);
                    const float2 e = i % 16 < P::kFma ? ex2_fma(v) : make_float2(ex2(v.x), ex2(v.y));
                    total = __fadd2_rn(total, e);
                    x[i / 2] = pack<BF>(e.x, e.y);
                }
                sum += total.x + total.y;
                tm_store(ts, x);
                tc_wait_st();
                tc_before();
                __syncwarp();
                if (lane == 0) bar_arrive(bar(B_P + NB * t + buf));
            }
            Item it;
            read(n, it);
            const TileSpan sp = span(it, t);
            if (fine && sp.count) {
                const bool live = p < (uint32_t)sp.count;
                const int32_t sees = sees_of(it);
                // the last products of every buffer
                for (uint32_t buf = 0; buf < NB && (int32_t)buf < sp.tiles && fine; ++buf) {
                    fine = all_wait(bar(B_O + NB * t + buf), phase_o >> buf & 1u);
                    phase_o ^= 1u << buf;
                }
                if (!fine) break;
                tc_after();
                const uint32_t flagged = bad_flag[n % kDeal];
                // infinities and NaN among the values of the dimensions from d0 on that this row sees, added to
                // what the other keys came to, which may be an infinity or a NaN of their own
                auto overlay = [&](uint32_t *o, int d0, auto width) {
                    // keys from `key0` on were looked through
                    const int32_t key0 = max(0, span(it, 0).first / kKeys) * kKeys;
                    const uint16_t *first = bad + n % kDeal * 3 * D + d0;
#pragma unroll
                    for (int i = 0; i < decltype(width)::value; ++i) {
                        const bool up = key0 + first[i] < sees, down = key0 + first[D + i] < sees;
                        const bool nan = key0 + first[2 * D + i] < sees;
                        const float x = nan || up == down ? __uint_as_float(0x7fc00000u) : up ? INFINITY : -INFINITY;
                        if (nan || up || down) o[i] = __float_as_uint(__uint_as_float(o[i]) + x);
                    }
                };
                // Parts of an item go to the workspace, [warp][dimension, maximum, sum][lane], and the warp that
                // is the last of its kind to finish joins them, in the order of the CTAs.
                const bool whole = it.parts == 1;
                float *parts = reinterpret_cast<float *>(static_cast<unsigned char *>(a.workspace) + a.counters) +
                               (uint64_t)warp * (D + 2) * 32 + lane;
                constexpr uint64_t kSlot = (uint64_t)4 * NT * (D + 2) * 32;
                auto part_of = [&](int32_t c) { return parts + (2ull * c + (c == it.part ? 1 : 0)) * kSlot; };
                if (!whole) {
                    float *mine = part_of((int32_t)blockIdx.x);
                    __stcg(mine + D * 32, sp.tiles ? ref : -INFINITY);
                    __stcg(mine + (D + 1) * 32, sp.tiles ? sum : 0.0f);
#pragma unroll 1
                    for (int c = 0; c < D / 16; ++c) {
                        uint32_t o[16] = {};
                        if (sp.tiles) {
                            tm_load16(to + 16 * c, o);
                            tc_wait_ld();
                            if (flagged) overlay(o, 16 * c, std::integral_constant<int, 16>());
                        }
#pragma unroll
                        for (int i = 0; i < 16; ++i) __stcg(mine + (16 * c + i) * 32, __uint_as_float(o[i]));
                    }
                    tc_before();
                    __threadfence();
                    __syncwarp();
                    uint32_t *counter = static_cast<uint32_t *>(a.workspace) + (uint64_t)it.part * 4 * NT + warp;
                    uint32_t before = 0;
                    if (lane == 0) {
                        before = atomicAdd(counter, 1u);
                        if (before + 1 == (uint32_t)it.parts) *counter = 0;
                    }
                    if (__shfl_sync(0xffffffffu, before, 0) + 1 != (uint32_t)it.parts) {
                        taken(n);
                        continue;
                    }
                    __threadfence();
                    ref = -INFINITY, sum = 0.0f;
                    const int32_t after = it.part + it.parts;
                    for (int32_t c = it.part; c < after; c += kJoin) {
                        float m[kJoin], l[kJoin];
#pragma unroll
                        for (int b = 0; b < kJoin; ++b) {
                            m[b] = c + b < after ? __ldcg(part_of(c + b) + D * 32) : -INFINITY;
                            l[b] = c + b < after ? __ldcg(part_of(c + b) + (D + 1) * 32) : 0.0f;
                        }
                        float top = ref;
#pragma unroll
                        for (int b = 0; b < kJoin; ++b) top = max_nan(top, m[b]);
                        const float from = top == -INFINITY ? 0.0f : top;
                        sum *= ex2(ref - from);
#pragma unroll
                        for (int b = 0; b < kJoin; ++b) sum = fmaf(ex2(m[b] - from), l[b], sum);
                        ref = top;
                    }
                }
                const bool none = sees == 0;
                const float ref0 = ref == -INFINITY ? 0.0f : ref;
                const float inv = none || sum == 0.0f ? 0.0f : 1.0f / sum;  // (0: every logit is -infinity)
                // kW dimensions at a time, turned through shared memory so that kL lanes write 16 kL bytes of a row
                constexpr int kW = P::kTurn, kL = kW / 8;
                unsigned char *turn = sm + P::kOut + warp * 64 * kW;
                const int64_t first_row = (int64_t)(it.token + t * (int32_t)per) * a.q_heads + it.head * a.group;
                int32_t to_row[kL];  // of the rows that this lane writes for, from first_row on; -1 for none
#pragma unroll
                for (int i = 0; i < kL; ++i) {
                    const uint32_t tr = (warp & 3u) * 32 + (32 / kL) * i + lane / kL, rp = tr / a.group;
                    to_row[i] = rp < (uint32_t)sp.count ? (int32_t)(rp * a.q_heads + tr % a.group) : -1;
                }
                // 16-byte chunk c of row r: a phase of eight lanes meets 128 different bytes, writing and reading
                auto chunk = [&](uint32_t r, uint32_t c) { return turn + r * 2 * kW + ((c ^ r / (8 / kL) % kL) << 4); };
#pragma unroll 1
                for (int c = 0; c < D / kW; ++c) {
                    uint32_t o[kW];
                    if (!whole) {
#pragma unroll
                        for (int i = 0; i < kW; ++i) o[i] = 0;
                        const int32_t after = it.part + it.parts;
                        for (int32_t q = it.part; q < after; q += kJoin) {  // their loads in flight together
                            float f[kJoin], x[kJoin][kW];
#pragma unroll
                            for (int b = 0; b < kJoin; ++b) {
                                const float *from = part_of(q + b);
                                f[b] = q + b < after ? __ldcg(from + D * 32) : -INFINITY;
#pragma unroll
                                for (int i = 0; i < kW; ++i) x[b][i] = q + b < after ? __ldcg(from + (kW * c + i) * 32) : 0.0f;
                            }
#pragma unroll
                            for (int b = 0; b < kJoin; ++b) {
                                const float e = ex2(f[b] - ref0);  // 0 for a part of no K tile that this row sees
#pragma unroll
                                for (int i = 0; i < kW; ++i) o[i] = __float_as_uint(fmaf(e, x[b][i], __uint_as_float(o[i])));
                            }
                        }
                    } else if (sp.tiles) {
                        if constexpr (kW == 32) tm_load(to + kW * c, o);
                        else tm_load16(to + kW * c, o);
                        tc_wait_ld();
                    }
                    if (none) {
#pragma unroll
                        for (int i = 0; i < kW; ++i) o[i] = 0;
                    }
                    if (whole && flagged) overlay(o, kW * c, std::integral_constant<int, kW>());
#pragma unroll
                    for (int i = 0; i < kL; ++i) {
                        uint4 v;
                        v.x = pack<BF>(__uint_as_float(o[8 * i]) * inv, __uint_as_float(o[8 * i + 1]) * inv);
                        v.y = pack<BF>(__uint_as_float(o[8 * i + 2]) * inv, __uint_as_float(o[8 * i + 3]) * inv);
                        v.z = pack<BF>(__uint_as_float(o[8 * i + 4]) * inv, __uint_as_float(o[8 * i + 5]) * inv);
                        v.w = pack<BF>(__uint_as_float(o[8 * i + 6]) * inv, __uint_as_float(o[8 * i + 7]) * inv);
                        *reinterpret_cast<uint4 *>(chunk(lane, i)) = v;
                    }
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < kL; ++i) {
                        const uint4 v = *reinterpret_cast<uint4 *>(chunk((32 / kL) * i + lane / kL, lane % kL));
                        if (to_row[i] >= 0)
                            *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(a.out) + (first_row + to_row[i]) * D + kW * c +
                                                       8 * (lane % kL)) = v;
                    }
                    __syncwarp();
                }
                if (live && a.lse) a.lse[first_row + (int64_t)p * a.q_heads + g] = none ? -INFINITY : (ref - kUp<BF> + __log2f(sum)) * kLn2;
                tc_before();
            }
            if (!fine) break;
            taken(n);
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(P::kRest));
        if (warp == W_LOAD) {
            // ---- the deal ----
            // An item's price is its keys, as its last row sees them, and kItemCost.  Items stand in order - sequences,
            // KV heads, blocks - on a line as long as their prices, K tile j of one at kItemCost + 64 j of its stretch,
            // and the line is cut into equal ranges, one a CTA, none shorter than a tile: whatever the
            // lengths are, all CTAs end together, and where items are few, their keys are split.  An item of up to kWhole
            // keys is the CTA's in whose range it begins.
            const int32_t block = (int32_t)(a.tiles * per);
            struct Seq {
                int32_t q0, k0, nq, nk, blocks, shift;
            } sq;
            auto load_seq = [&](uint32_t s) {
                Seq q{};
                if (s >= a.sequences) return q;
                const int32_t q0 = __ldg(a.starts + s), q1 = __ldg(a.starts + s + 1);
                const int32_t k0 = __ldg(a.key_starts + s), k1 = __ldg(a.key_starts + s + 1);
                if (q0 < 0 || k0 < 0 || q1 < q0 || k1 < k0 || (uint64_t)q1 > a.q_tokens || (uint64_t)k1 > a.k_tokens) {
                    if (blockIdx.x == 0) atomicOr(a.status, kStatusBadExtent);
                    return q;
                }
                q.q0 = q0, q.k0 = k0, q.nq = q1 - q0, q.nk = k1 - k0, q.shift = q.nk - q.nq;
                q.blocks = (int32_t)(((uint32_t)q.nq + block - 1) / (uint32_t)block);
                return q;
            };
            // keys of block b, one at least
            auto keys_of = [&](const Seq &q, int32_t b) {
                if (!a.causal || b + 1 >= q.blocks) return max(1, q.nk);
                return max(1, (b + 1) * block + q.shift);
            };
            // price of the blocks before b of one head
            auto price = [&](const Seq &q, int32_t b) -> int64_t {
                if (b == 0) return 0;
                int64_t n = b * kItemCost;
                if (!a.causal) return n + (int64_t)b * max(1, q.nk);
                const int32_t m = min(b, q.blocks - 1);  // all but the last block: (b + 1) block + shift keys, or 1
                const int32_t z = q.shift < 0 ? min(m, (int32_t)((uint32_t)(1 - q.shift) / (uint32_t)block)) : 0;
                n += z + (int64_t)block * (((int64_t)m * (m + 1) - (int64_t)z * (z + 1)) / 2) + (int64_t)q.shift * (m - z);
                return b == q.blocks ? n + max(1, q.nk) : n;
            };
            // the first 32 sequences stay in the lanes, with the price of all before each of them and its own
            const Seq mine = load_seq(lane);
            const int64_t own = a.kv_heads * price(mine, mine.blocks);
            auto scan = [&](int64_t x) {
#pragma unroll
                for (int w = 1; w < 32; w <<= 1) {
                    const int64_t o = __shfl_up_sync(0xffffffffu, x, w);
                    if (lane >= (uint32_t)w) x += o;
                }
                return x;
            };
            const int64_t own_upto = scan(own);
            auto get_seq = [&](uint32_t s) {
                if (s >= 32) return load_seq(s);
                Seq q;
                q.q0 = __shfl_sync(0xffffffffu, mine.q0, s), q.k0 = __shfl_sync(0xffffffffu, mine.k0, s);
                q.nq = __shfl_sync(0xffffffffu, mine.nq, s), q.nk = __shfl_sync(0xffffffffu, mine.nk, s);
                q.blocks = __shfl_sync(0xffffffffu, mine.blocks, s), q.shift = q.nk - q.nq;
                return q;
            };
            int64_t total = __shfl_sync(0xffffffffu, own_upto, 31);
            uint32_t blocks = (uint32_t)mine.blocks;
            int32_t longest = mine.blocks ? mine.nk : 0;
            if (a.sequences > 32) {
                int64_t rest = 0;
                for (uint32_t s = lane + 32; s < a.sequences; s += 32) {
                    const Seq q = load_seq(s);
                    rest += a.kv_heads * price(q, q.blocks);
                    blocks += (uint32_t)q.blocks;
                    longest = max(longest, q.blocks ? q.nk : 0);
                }
                total += __shfl_sync(0xffffffffu, scan(rest), 31);
            }
            const int64_t all = (int64_t)__reduce_add_sync(0xffffffffu, blocks) * a.kv_heads;
            int64_t ctas = min((int64_t)gridDim.x, max((int64_t)1, total / kKeys));
            if (__reduce_max_sync(0xffffffffu, longest) > kWhole) ctas = min(ctas, max(all, total / kPiece));
            bool some = ctas > 0 && (int64_t)blockIdx.x < ctas;
            const int64_t each = some ? quotient(total, ctas) : 1, over = some ? total - each * ctas : 0;
            const int64_t start = blockIdx.x * each + min((int64_t)blockIdx.x, over);
            const int64_t end = start + each + ((int64_t)blockIdx.x < over ? 1 : 0);
            auto owner = [&](int64_t place) {
                const int64_t head = over * (each + 1);
                return (int32_t)(place < head ? quotient(place, each + 1) : over + quotient(place - head, each));
            };
            uint32_t seq = 0;
            int32_t head = 0, blk = 0;
            int64_t at = 0;  // the item at hand begins there on the line
            if (some) {
                for (uint32_t s0 = 0;; s0 += 32) {  // ends: start < total
                    int64_t price_of = own, upto = own_upto;
                    if (s0) {
                        const Seq q = load_seq(s0 + lane);
                        price_of = a.kv_heads * price(q, q.blocks);
                        upto = scan(price_of);
                    }
                    const uint32_t past = __ballot_sync(0xffffffffu, at + upto > start);
                    if (past) {
                        const uint32_t l = __ffs(past) - 1;
                        at += __shfl_sync(0xffffffffu, upto - price_of, l);
                        seq = s0 + l;
                        break;
                    }
                    if (s0 + 32 >= a.sequences) {
                        some = false;
                        break;
                    }
                    at += __shfl_sync(0xffffffffu, upto, 31);
                }
                if (some) {
                    sq = get_seq(seq);
                    const int64_t of_head = price(sq, sq.blocks);
                    head = (int32_t)quotient(start - at, of_head);
                    at += head * of_head;
                    int32_t top = sq.blocks;  // the last block that begins at or before the start
                    while (top - blk > 1) {
                        const int32_t mid = (blk + top) / 2;
                        if (at + price(sq, mid) <= start) blk = mid;
                        else top = mid;
                    }
                    at += price(sq, blk);
                }
            }
            auto deal = [&](uint32_t n) {
                Item it{};
                while (some && it.count == 0) {
                    const int32_t keys = keys_of(sq, blk), units = (keys + kKeys - 1) / kKeys;
                    const int64_t from = at + kItemCost;
                    int32_t one, two;
                    if (keys <= kWhole) {  // where it begins
                        one = 0;
                        two = at >= start ? units : 0;
                    } else {
                        one = start <= from ? 0 : (int32_t)min((int64_t)units, (start - from + kKeys - 1) / kKeys);
                        two = end <= from ? 0 : (int32_t)min((int64_t)units, (end - from + kKeys - 1) / kKeys);
                    }
                    if (one < two) {
                        it.pos = blk * block;
                        it.token = sq.q0 + it.pos;
                        it.count = min(block, sq.nq - blk * block);
                        it.head = head;
                        it.key = sq.k0;
                        it.keys = sq.nk;
                        it.shift = sq.shift;
                        it.from = one;
                        it.upto = two;
                        it.parts = 1;
                        if (one > 0 || two < units) {
                            it.part = owner(from);
                            it.parts = owner(from + (int64_t)(units - 1) * kKeys) - it.part + 1;
                        }
                    }
                    at += kItemCost + keys;
                    some = at < end;
                    if (some && ++blk == sq.blocks) {
                        blk = 0;
                        if (++head == (int32_t)a.kv_heads) {
                            head = 0;
                            do {
                                if (++seq >= a.sequences) {
                                    some = false;
                                    break;
                                }
                                sq = get_seq(seq);
                            } while (sq.blocks == 0);
                        }
                    }
                }
                if (n >= kDeal && !all_wait(bar(B_TAKEN + n % kDeal), (n / kDeal & 1) ^ 1)) return;
                if (lane == 0) {
                    volatile Item &d = items[n % kDeal];
                    d.token = it.token, d.count = it.count, d.pos = it.pos, d.head = it.head;
                    d.key = it.key, d.keys = it.keys, d.shift = it.shift, d.from = it.from, d.upto = it.upto;
                    d.part = it.part, d.parts = it.parts;
                    bad_flag[n % kDeal] = 0;
                    bar_arrive(bar(B_ITEM + n % kDeal));
                }
                __syncwarp();
            };
            // ---- loads ----
            // A stage that the last warp looks through lands on its raw barrier, and that warp arrives on the full
            // one when it is done with it.
            uint32_t slot = 0, free_phase = 1, q_phase = (1u << NT) - 1, issued = 0, full_phase = 0, raw = 0, raw_phase = 0;
            uint32_t q_issued = 0;
            Item it;
            bool fine = true;
            deal(0);
            for (uint32_t n = 0; fine && next(n, it); ++n) {
                const int32_t tiles = tiles_of(it), first = span(it, 0).first;
                auto load_q = [&](int t) {
                    if (!(fine = fine && bar_wait(bar(B_QFREE + t), q_phase >> t & 1u, stop))) return;
                    q_phase ^= 1u << t;
                    q_issued |= 1u << t;
                    bar_expect(bar(B_QFULL + t), P::kChunks * per * a.group * 128u);
                    for (uint32_t c = 0; c < P::kChunks; ++c)
                        tma3(base + P::kQ + t * P::kQTile + c * P::kQChunk, &mq, bar(B_QFULL + t), 64 * c,
                             it.head * (int32_t)a.group, it.token + t * (int32_t)per);
                };
                // first the K tiles that logits run ahead by, then V j and K j + NB: rows of tiles, -1 for none
                auto load = [&](const CUtensorMap *map, int32_t one, int32_t two, bool look) {
                    if (!(fine = fine && bar_wait(bar(B_FREE + slot), free_phase, stop))) return;
                    const uint32_t on = bar((look ? B_RAW : B_FULL) + slot), bit = 1u << slot;
                    bar_expect(on, P::kTile * (two < 0 ? 1u : 2u));
                    const uint32_t dst = base + P::kRing + slot * 2 * P::kTile;
                    for (uint32_t c = 0; c < P::kChunks; ++c)
                        tma3(dst + c * P::kChunk, map, on, 64 * c, it.head, it.key + (it.from + one) * kKeys);
                    if (two >= 0)
                        for (uint32_t c = 0; c < P::kChunks; ++c)
                            tma3(dst + P::kTile + c * P::kChunk, &mk, on, 64 * c, it.head,
                                 it.key + (it.from + two) * kKeys);
                    issued |= bit;
                    raw = look ? raw | bit : raw & ~bit;
                    full_phase = (full_phase & ~bit) | (free_phase ^ 1u) << slot;
                    raw_phase ^= look ? bit : 0;
                    if (++slot == P::kStages) slot = 0, free_phase ^= 1;
                };
                auto load_v = [&](int32_t j) {
                    load(&mv, j, j + (int32_t)NB < tiles ? j + (int32_t)NB : -1, (it.from + j + 1) * kKeys > first);
                };
                if (lane == 0) {
                    if (span(it, 0).tiles) load_q(0);
                    if (tiles) load(&mk, 0, NB == 2 && tiles > 1 ? 1 : -1, false);
                    for (uint32_t t = 1; t < NT; ++t)
                        if (span(it, (int)t).tiles) load_q((int)t);
                    if (tiles) load_v(0);
                }
                __syncwarp();
                deal(n + 1);
                if (lane == 0)
                    for (int32_t j = 1; j < tiles && fine; ++j) load_v(j);
                fine = __shfl_sync(0xffffffffu, fine, 0);
            }
            // copies in flight land before the CTA ends (they have, unless a wait ran out)
            if (lane == 0 && *stop) {
                uint32_t none = 0;
                for (uint32_t i = 0; i < P::kStages; ++i)
                    if (issued >> i & 1u)
                        bar_wait(bar((raw >> i & 1u ? B_RAW : B_FULL) + i), raw >> i & 1u ? ~raw_phase >> i & 1u : full_phase >> i & 1u,
                                 &none);
                for (uint32_t t = 0; t < NT; ++t)
                    if (q_issued >> t & 1u) bar_wait(bar(B_QFULL + t), q_phase >> t & 1u, &none);
            }
        } else if (warp < W_ENDS) {
            // ---- products of every second row tile: the warp stays together, one lane issues ----
            const uint32_t half = warp - W_MMA;
            uint32_t slot = 0, full_phase = 0, q_phase = 0, p_phase = 0;  // p_phase: a bit for each buffer of every tile
            constexpr uint32_t ID_S = product(BF, 0, P::kKeys), ID_O = product(BF, 1, D), MINE = NT / 2;
            Item it;
            bool fine = true;
            for (uint32_t n = 0; fine && next(n, it); ++n) {
                const int32_t tiles = tiles_of(it);
                if (!tiles) {
                    taken(n);
                    continue;
                }
                int32_t mine[MINE];
#pragma unroll
                for (uint32_t i = 0; i < MINE; ++i) mine[i] = span(it, (int)(half + 2 * i)).tiles;
                auto advance = [&]() {
                    if (++slot == P::kStages) slot = 0, full_phase ^= 1;
                };
                // the logits of row tile t and K tile j, which lies at `k_at`
                auto logits = [&](uint32_t t, uint32_t k_at, int32_t j) {
                    const uint32_t q = operand(base + P::kQ + t * P::kQTile, 0), key = operand(k_at, 0);
                    const uint32_t d = tmem + (NB * t + j % NB) * kKeys;
#pragma unroll
                    for (uint32_t c = 0; c < P::kChunks; ++c)
#pragma unroll
                        for (uint32_t s = 0; s < 4; ++s)
                            mma_ss(d, q + (c * P::kQChunk + 32 * s) / 16, key + (c * P::kChunk + 32 * s) / 16, ID_S, c | s);
                };
                // logits run NB tiles ahead of the outputs
                if (!(fine = all_wait(bar(B_FULL + slot), full_phase))) break;
#pragma unroll
                for (uint32_t i = 0; i < MINE; ++i) {
                    if (!mine[i]) continue;
                    const uint32_t t = half + 2 * i;
                    if (!(fine = all_wait(bar(B_QFULL + t), q_phase >> t & 1u))) break;
                    q_phase ^= 1u << t;
                    tc_after();
                    if (elect()) {
                        const uint32_t at = base + P::kRing + slot * 2 * P::kTile;
                        logits(t, at, 0);
                        tc_commit(bar(B_S + NB * t));
                        if (NB == 2 && mine[i] > 1) {
                            logits(t, at + P::kTile, 1);
                            tc_commit(bar(B_S + NB * t + 1));
                        }
                        if (mine[i] <= (int32_t)NB) tc_commit(bar(B_QFREE + t));
                    }
                    __syncwarp();
                }
                if (!fine) break;
                if (elect()) tc_commit(bar(B_FREE + slot));
                __syncwarp();
                advance();
                for (int32_t j = 0; j < tiles; ++j) {
                    const uint32_t v = slot, at = base + P::kRing + v * 2 * P::kTile;
                    if (!(fine = all_wait(bar(B_FULL + v), full_phase))) break;
                    advance();
#pragma unroll
                    for (uint32_t i = 0; i < MINE; ++i) {
                        if (j >= mine[i]) continue;
                        const uint32_t t = half + 2 * i, tb = NB * t + j % NB;
                        if (!(fine = all_wait(bar(B_P + tb), p_phase >> tb & 1u))) break;
                        p_phase ^= 1u << tb;
                        tc_after();
                        if (elect()) {
                            const uint32_t val = operand(at, P::kChunk), pr = tmem + tb * kKeys, o = tmem + P::kColO + t * D;
#pragma unroll
                            for (uint32_t s = 0; s < P::kKeys / 16; ++s) mma_ts(o, pr + 8 * s, val + s * 128, ID_O, j | (int32_t)s);
                            const bool more = j + (int32_t)NB < mine[i];
                            if (more) logits(t, at + P::kTile, j + (int32_t)NB);
                            tc_commit(bar((more ? B_S : B_O) + tb));
                            if (j + (int32_t)NB + 1 == mine[i]) tc_commit(bar(B_QFREE + t));
                        }
                        __syncwarp();
                    }
                    if (!fine) break;
                    if (elect()) tc_commit(bar(B_FREE + v));
                    __syncwarp();
                }
                if (fine) taken(n);
            }
            // products in flight end before the tensor memory is given back
            __syncwarp();
            if (*stop && elect()) {
                uint32_t none = 0;
                tc_commit(bar(B_END + half));
                bar_wait(bar(B_END + half), 0, &none);
            }
        } else {
            // ---- V tiles that not every row sees ----
            uint32_t slot = 0, raw_phase = 0;
            Item it;
            bool fine = true;
            for (uint32_t n = 0; fine && next(n, it); ++n) {
                const TileSpan s0 = span(it, 0);
                const int32_t tiles = tiles_of(it), begin = max(0, s0.first / kKeys);
                uint16_t *first = bad + n % kDeal * 3 * D;
                if (begin < it.from + tiles)
                    for (uint32_t i = lane; i < 3 * D; i += 32) first[i] = 0xffff;
                for (int32_t j = max(0, begin - it.from); j < tiles; ++j) {
                    if ((it.from + j + 1) * kKeys <= s0.first) continue;
                    const uint32_t v = (slot + 1 + (uint32_t)j) % P::kStages;  // past the stage of the first K tiles
                    if (!(fine = all_wait(bar(B_RAW + v), raw_phase >> v & 1u))) break;
                    raw_phase ^= 1u << v;
                    unsigned char *tile = sm + P::kRing + v * 2 * P::kTile;
                    const int32_t rows = min(kKeys, it.keys - (it.from + j) * kKeys);
                    uint32_t found = 0;
                    constexpr uint32_t E = BF ? 0x7f80u : 0x7c00u;
#pragma unroll 4
                    for (uint32_t i = lane; i < P::kKeys * D / 8; i += 32) {
                        const uint32_t r = i / (D / 8), u = i % (D / 8);
                        uint4 *w = reinterpret_cast<uint4 *>(tile + u / 8 * P::kChunk + r * 128 + ((u % 8 ^ (r & 7)) << 4));
                        if ((int32_t)r >= rows) *w = make_uint4(0, 0, 0, 0);
                        else {
                            const uint4 x = *w;
                            const uint32_t y[4] = {x.x, x.y, x.z, x.w};
                            // an exponent of ones carries into the sign's place
                            constexpr uint32_t kCarry = (0x8000u - E) | (0x8000u - E) << 16;
#pragma unroll
                            for (int k = 0; k < 4; ++k) found |= (y[k] & 0x7fff7fffu) + kCarry;
                        }
                    }
                    if (__any_sync(0xffffffffu, found & 0x80008000u)) {
                        __syncwarp();
                        for (uint32_t d = lane; d < (uint32_t)D; d += 32) {
                            for (int32_t k = 0; k < rows; ++k) {
                                uint16_t *w = reinterpret_cast<uint16_t *>(tile + d / 64 * P::kChunk + k * 128 +
                                                                           (((d % 64 / 8) ^ (k & 7)) << 4)) + d % 8;
                                const uint32_t x = *w;
                                if ((x & E) != E) continue;
                                *w = 0;
                                const uint32_t kind = (x & 0x7fffu) != E ? 2 : x >> 15;  // 0 inf, 1 -inf, 2 NaN
                                const uint32_t at = (uint32_t)((it.from + j - begin) * kKeys + k);
                                if (at < first[kind * D + d]) first[kind * D + d] = (uint16_t)at;
                            }
                        }
                        if (lane == 0) bad_flag[n % kDeal] = 1;
                    }
                    fence_async();
                    __syncwarp();
                    if (lane == 0) bar_arrive(bar(B_FULL + v));
                }
                slot = (slot + (uint32_t)(tiles ? tiles + 1 : 0)) % P::kStages;
                if (fine) taken(n);
            }
        }
    }
    // every role has left its loop; on a timeout the waits above were cut short
    __syncwarp();
    tc_before();
    __syncthreads();
    if (threadIdx.x == 0 && *stop) atomicOr(a.status, kStatusTimeout);
    if (warp == W_LOAD) {
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

// Bytes of the workspace's counters: one for every softmax warp of every CTA.  (Those of any device with up to 1024 SMs
// are within BGTQ_WORKSPACE_ZEROED.)
uint32_t prompt_counters(int sms, uint32_t tiles) { return ((uint32_t)sms * tiles * 16 + 127) / 128 * 128; }

template <int D, bool BF>
cudaError_t run(const PromptArgs &args, cudaStream_t s) {
    using P = Plan<D>;
    if (!encoder()) return cudaErrorNotSupported;
    auto kernel = prompt_kernel<D, BF>;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const int sms = sm_count(dev);
    if (!sms) return cudaErrorInvalidDevice;
    static bool ready[64] = {};
    if (!ready[dev]) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)P::kTotal);
        if (e != cudaSuccess) return e;
        // the warps hand registers to each other: more than the launch has would be waited for
        cudaFuncAttributes f;
        e = cudaFuncGetAttributes(&f, kernel);
        if (e != cudaSuccess) return e;
        if ((uint32_t)f.numRegs * P::kThreads < 128 * P::kTiles * P::kSoft + 128 * P::kRest) return cudaErrorNotSupported;
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
    // The row tiles of an item share its K and V loads and keep the softmax warps busy: as many as possible, while
    // that makes half as many items as there are SMs.  (512 tokens, 14 / 2 heads of 64: one tile 15.4 us, four 20.0;
    // 700 tokens of 32 heads: one 32.9 us, two 30.5, four 35.3; two prompts of 8192: one 717 us, four 293.)
    auto items = [&](uint32_t tiles) { return a.kv_heads * ((a.q_tokens + tiles * per - 1) / (tiles * per) + a.sequences - 1); };
    a.tiles = P::kTiles;
    while (a.tiles > 1 && 2 * items(a.tiles) <= (uint64_t)sms) a.tiles /= 2;
    const uint64_t ctas = items(a.tiles) * (a.k_tokens + kItemCost) / P::kKeys + 1;
    a.counters = prompt_counters(sms, P::kTiles);
    kernel<<<(uint32_t)(ctas < (uint64_t)sms ? ctas : sms), P::kThreads, P::kTotal, s>>>(a, mq, mk, mv);
    return cudaGetLastError();
}

}  // namespace

size_t prompt_workspace(uint32_t dim) {
    int dev = 0;
    const int sms = cudaGetDevice(&dev) == cudaSuccess ? sm_count(dev) : 0;
    if (!sms) return 0;
    const uint32_t tiles = dim == 64 ? Plan<64>::kTiles : Plan<128>::kTiles;
    return prompt_counters(sms, tiles) + 2ull * sms * tiles * kRows * (dim + 2) * 4;
}

cudaError_t launch_prompt(const PromptArgs &a, cudaStream_t s) {
    if (a.dtype == BGTQ_BF16) return a.dim == 64 ? run<64, true>(a, s) : run<128, true>(a, s);
    return a.dim == 64 ? run<64, false>(a, s) : run<128, false>(a, s);
}

}  // namespace bgtq
