// Attention of chunks of many new tokens over the pages of a cache on the fifth-generation tensor cores: query row i of
// request b, at position p = length - rows + i, attends the tokens t <= p of its pages, with a window only those of
// p - window < t and t < sinks; softmax with a running maximum and sum (FP32).
//
// The work is laid out as prompt_attention.cu lays it out for packed keys: an item is a block of consecutive rows of one
// request with all query heads of one KV head, 128 rows a tile, which share every K and V tile of 64 tokens; CTAs take
// equal ranges of the items' tokens, an item across two ranges is done in parts and joined by its last CTA; and the
// warps have roles (softmax, deal and loads, products, ends).  What is different:
//   units       the tiles of an item are those of the first tokens (sinks) and, after a gap, those from the first row's
//               window to the last row; a unit's tile is found by adding the gap
//   loads       a tile is 64 / page pieces or a part of a page, each a TMA box of its own: 16 lanes have one each, and
//               look up their page one stage ahead.  A page index past the cache reads as zeros and is masked
//   masks       a tile that not every row of the item sees (a sequence's end, the diagonal, a window's edges, the last
//               sinks) has a mask of 64 bits for each row
//   ends        in such tiles values past the end are zeroed, and an infinity or a NaN, which the zero probability of a
//               row that does not see it would turn into a NaN, is taken out; the rows that see it look the tile
//               through once more, in the pages, when they are written
//   codes       (8- and 4-bit pages) codes and scales are loaded as they are, and warps of their own turn a tile into
//               FP16 operands ahead of the products.  A key stays exact, so that logits are FP32's: 4-bit codes x scales
//               over a power of two of the tile's largest scale have 11 bits; 8-bit ones have 15, of which at head dim 64 a
//               second operand holds the last four, multiplied by the same queries into the same logits; at 128, where
//               tensor time is what there is least of, 8-bit codes stay plain and softmax multiplies each key's logits
//               by its scale.  The tile's power multiplies its logits as the scale of all logits does, and its
//               probabilities as an addend of their exponents, so that softmax does no more than over 16-bit pages.
//               (BF16 queries go to FP16 over a power of two of their row, which loses what is below 2^-38 of the row's
//               largest.)  A value in 8 bits is exact as well: its code by the power of two of its scale is an operand, and
//               the scale's mantissa multiplies the probability before that is rounded (an FP16 output's error 2.8e-4 of
//               its norm, 2.1e-4 in FP32 throughout; products of code and scale rounded to FP16 3.5e-4, and 4 % less time:
//               600 us for 624 and 630 for 655 of the cases below, 168 for 183 of few rows).  Where the scales of a tile are
//               more than 2^16 apart, as next to rows of 1e30, powers of two of each
//               token take their place and multiply each logit, or each probability.  Probabilities x value scales are
//               taken relative to the row's largest so far, in steps of at least 2^kRoom, so that values of any size
//               whose weight is next to nothing leave the others as they are; what is rounded away is 2^-34 of the
//               largest
//
// What bounds it.  Many rows: the tensor cores and, at head dim 64, the exponentials of softmax: four chunks of 1024 rows after
// 6000 to 8192 tokens, 32 / 8 heads of 128 in 16 bits, 445 us, 1140 TFLOP/s; two of 2048 after 24000 to 30000, 14 / 2 heads of
// 64, 470 us, 876 TFLOP/s.  Over codes the warps that turn them and the code they share the instruction caches with:
// the first in 8 bits 624 us, in 4 bits 668; the second in 8 bits 655 (96 registers of softmax's warps and the keys' second
// operand).  Few rows: 32 requests of 5 rows after 500 to 16000 tokens, 32 / 8 heads of 128, 117 us, 5.2 TB/s; in 8
// bits 183 us, 1.7 TB/s, in 4 bits 219: the time is that of turning one stage of 64 tokens, 1.3 to 1.5 us with few rows and
// with many, which is mostly latency, since all turning warps work on one stage at a time.  Few tokens: 20 to 45 us of the
// deal, the first pages' way through the table, and the join.
#include <type_traits>

#include "tcgen05.cuh"

namespace bgtq {
namespace {

constexpr uint32_t kDeal = 4;            // items dealt ahead
// What an item costs beside its keys, in keys: queries, outputs, joining.  (None: 20 requests of 1 to 700 rows after up to
// 9000, 32 / 8 heads of 128, 271 us for 146, one of 500 rows after 4000, 14 / 2 heads of 64 in 8 bits, 76 for 58; 192: 167 and
// 58, 640: 156 and 60.)
constexpr int64_t kItemCost = 384;
// Items of no more keys are not split: joining costs as much as they do, less where rows are few.  kWholeFew is for
// requests of up to 64 columns - rows x query heads of a KV head.  (700 rows of one request, 32 / 8 heads of 128, 25 us, with
// 512 for all 34; 12 prompts of 1 to 2047 rows 86 us, with 1536 92.  Few: 32 x 5 rows after 500 to 16000 in 8 bits 167 us
// with 256, 180 with 1024; 8 x 8 rows after 200 to 2000, 14 / 2 heads of 64, 21.6 and 29.8, 32 / 8 of 128 22.6 and 32.4; 128 does
// what 256 does.)
constexpr int32_t kWhole = 1024, kWholeFew = 256;
// Keys that make a CTA worth its while where items are few and long.  (8 x 8 rows after 200 to 2000 in 8 bits of 64
// dimensions: 35 us with 256, 39 with 512, 48 with 1024; 8 after 30000, 14 / 2 heads of 64: 51, 44, 38.)
constexpr int64_t kPiece = 512;
constexpr int kJoin = 2;                 // parts of an item that are joined at a time (1: 8 rows after 30000 as above 58 us for 44)
constexpr float kLazy = 8.0f;            // log2 of the growth of a maximum that is left standing
template <bool BF> constexpr float kUp = BF ? 0.0f : 15.0f - kLazy;  // log2 of what probabilities are multiplied by
// Over 8- and 4-bit pages (powers of two, as logarithms): how far a tile's largest probability x value scale may pass the
// largest before it; what such products are multiplied by; how far they may be below their probability; how far apart
// the scales of a tile may be that has one power of two.
constexpr float kRoom = 4.0f, kUpCodes = 10.0f, kApart = 100.0f;
constexpr uint32_t kNear = 16;

enum { F_F16, F_BF16, F_INT8, F_INT4 };

template <int D, int NT, int F>
struct Plan {
    static constexpr bool kCodes = F >= F_INT8;
    static constexpr uint32_t kTiles = NT;                         // row tiles of an item, at most
    static constexpr uint32_t kBufs = NT == 4 ? 1 : 2;             // of logits, for each row tile
    static constexpr uint32_t kKeys = 64;                          // of a K or V tile
    static constexpr uint32_t kColO = kTiles * kBufs * kKeys;      // the first column of the outputs
    // Warps that look at, or turn, tiles; over codes the first sees to their scales.  (Two chunks of 2048 after 24000 to 30000, 14 / 2
    // heads of 64 in 8 bits, one that turns 1189 us, four 630.)
    static constexpr uint32_t kEnds = kCodes ? (NT == 4 ? 5 : 9) : 1;
    static constexpr uint32_t kThreads = 128 * NT + 32 * (3 + kEnds);
    // Registers after the hand-over, of softmax's warps and of the others: what the launch has, in all.
    static constexpr uint32_t kSoft = NT == 4 ? (kCodes ? 96 : 104) : kCodes ? 128 : 216, kRest = NT == 4 ? (kCodes ? 48 : 64) : 72;
    // Exponentials of 16 on the FMA pipe.  (Their code is long, and beside the code that turns codes the caches of
    // instructions do not hold it: four chunks of 1024 after 8192, 32 / 8 heads of 128, with none 4 % less time in 8 bits and
    // 7 % less in 4 than with 6 of 16.)
    static constexpr int kFma = D == 64 ? 2 : kCodes ? 0 : 6;
    static constexpr uint32_t kChunks = D / 64;                    // 64-dimension columns of a tile
    static constexpr uint32_t kQChunk = kRows * 128, kQTile = kChunks * kQChunk;  // bytes: rows of 64 elements
    static constexpr uint32_t kChunk = kKeys * 128, kTile = kChunks * kChunk;
    static constexpr bool kOwn = F == F_INT8 && D == 128;          // every key's logits are multiplied by its own scale
    static constexpr bool kLow = F == F_INT8 && D == 64;           // keys have a second operand
    static constexpr uint32_t kStageBytes = (kLow ? 3 : 2) * kTile;  // a V tile and a K tile
    static constexpr uint32_t kStages = D == 128 ? (kLow ? 2 : kCodes ? 3 : 4) : (kLow ? 4 : kCodes ? 5 : 7);
    // 8- and 4-bit pages: tiles as they lie in the pages, and their scales
    static constexpr uint32_t kRow = F == F_INT8 ? D : D / 2, kGroups = F == F_INT8 ? 1 : D / 32;
    static constexpr uint32_t kRawTile = kKeys * kRow, kRawScale = kKeys * kGroups * 2;
    // (the two tiles, the scales of both, and those of the K tile's tokens' values)
    static constexpr uint32_t kRawStage = 2 * kRawTile + 3 * kRawScale, kRawStages = kCodes ? (D == 128 ? 2 : 4) : 0;
    static constexpr int kUpTile = F == F_INT8 ? 7 : 10;  // log2 of what a tile's largest scale goes to
    // What softmax has to know of the K tile in a stage is kept until that tile's logits are done with, which is sure
    // when the load warp has gone all stages and the logits' lead further.
    static constexpr uint32_t kMeta = kRawStages + kStages + kBufs <= 8 ? 8 : 16;
    static constexpr uint32_t kQ = 0, kRing = kTiles * kQTile, kRaw = kRing + kStages * kStageBytes;
    static constexpr int kTurn = NT == 4 ? 16 : 32;                // dimensions of an output row stored at a time
    static constexpr uint32_t kOut = kRaw + kRawStages * kRawStage;                     // [softmax warps][32 rows][kTurn] outputs
    // [kMeta][kBy][kKeys] what logits, and, as logarithms, probabilities are multiplied by; in 8 bits what probabilities are
    // multiplied by besides, the scales' mantissas
    static constexpr uint32_t kScales = kOut + 4 * kTiles * 64 * kTurn, kBy = F == F_INT8 ? 3 : 2;
    static constexpr uint32_t kAbout = kScales + (kCodes ? kMeta * kBy * kKeys * 4 : 0);   // [kMeta] About
    static constexpr uint32_t kBadPages = kAbout + (kCodes ? kMeta * 16 : 0);              // [kMeta] pieces without a page: K, V
    static constexpr uint32_t kItems = kBadPages + kMeta * 4;      // [kDeal] Item
    static constexpr uint32_t kBars = kItems + kDeal * 64;
    static constexpr uint32_t kBarCount = 3 * kStages + 2 * kRawStages + 4 * kTiles + 3 * kTiles * kBufs + 2 * kDeal + 2;
    static constexpr uint32_t kWords = kBars + 8 * kBarCount;      // tensor memory base, stop, bad-value flags
    static constexpr uint32_t kTotal = kWords + 32 + 1024;         // and the slack to align the base
    static_assert(kTotal <= 232448, "shared memory of a CTA");
};

// A work item, or the units [from, upto) of one.
struct Item {
    int32_t token, count;  // first query row, rows (0: no more items)
    int32_t place, head;   // the first row's position, KV head
    int32_t seq, keys;     // the request, its tokens
    int32_t sunk, gap;     // units of the first tokens, tiles between them and the window
    int32_t from, upto;
    int32_t part, parts;   // the CTA that has the item's first unit, how many CTAs have one (1: this is all of it)
};

struct TileSpan {
    int32_t count, tiles;  // rows, units of this piece
};

// Of a K tile of codes: what its logits are multiplied by, the exponent of the largest scale among its tokens' values,
// and whether (bits 0, 1) logits, and probabilities, have a factor for each token instead.
struct About {
    float mul, top;
    uint32_t each, pad;
};

__device__ __forceinline__ void tma4(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y, int z, int w) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], "
                 "[%2];" ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ void bulk(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ float from_bf16(uint32_t bits) { return __uint_as_float(bits << 16); }
__device__ __forceinline__ uint32_t sub_h(uint32_t a, uint32_t b) {
    const __half2 r = __hsub2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&r);
}
__device__ __forceinline__ uint32_t mul_h(uint32_t a, uint32_t b) {
    const __half2 r = __hmul2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&r);
}
__device__ __forceinline__ uint32_t rest_h(uint32_t a, uint32_t b, uint32_t c) {  // a b - c, rounded once
    const __half2 r = __hfma2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b),
                              __hneg2(*reinterpret_cast<const __half2 *>(&c)));
    return *reinterpret_cast<const uint32_t *>(&r);
}

template <int D, int NT, int F, bool QBF>
__global__ void __launch_bounds__(Plan<D, NT, F>::kThreads, 1) chunk_kernel(const __grid_constant__ ChunkArgs a,
                                                                    const __grid_constant__ CUtensorMap mq,
                                                                    const __grid_constant__ CUtensorMap mk,
                                                                    const __grid_constant__ CUtensorMap mv) {
    using P = Plan<D, NT, F>;
    constexpr bool kCodes = P::kCodes;
    constexpr bool kQTurn = kCodes && QBF;          // queries go from BF16 to FP16
    constexpr bool BF = kCodes ? false : QBF;       // the operands
    constexpr int32_t kKeys = (int32_t)P::kKeys;
    constexpr uint32_t NB = P::kBufs;
    extern __shared__ unsigned char raw_smem[];
    unsigned char *sm = raw_smem + ((1024u - (smem_addr(raw_smem) & 1023u)) & 1023u);
    const uint32_t base = smem_addr(sm), warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
    const uint32_t lane = threadIdx.x & 31u;
    volatile Item *items = reinterpret_cast<volatile Item *>(sm + P::kItems);
    volatile uint32_t *words = reinterpret_cast<volatile uint32_t *>(sm + P::kWords);
    volatile uint32_t *stop = words + 1, *bad_flag = words + 2;  // bad_flag[kDeal]
    volatile uint32_t *bad_pages = reinterpret_cast<volatile uint32_t *>(sm + P::kBadPages);
    const uint32_t bars = base + P::kBars;
    auto bar = [&](uint32_t i) { return bars + 8u * i; };
    // a stage is full, free, or (raw) to be looked through first; a raw stage is full, free; of each row tile: its queries
    // are there, are turned, are read, its part of an item's outputs is written; of each buffer of logits: they are there (and
    // what was asked of the tensor cores before them is done), the probabilities are, the last product from it is done; of
    // each item: it is dealt, it is given back
    constexpr uint32_t B_FULL = 0, B_FREE = P::kStages, B_RAW = 2 * P::kStages, B_CODES = 3 * P::kStages,
                       B_TURNED = B_CODES + P::kRawStages, B_QFULL = B_TURNED + P::kRawStages, B_QREADY = B_QFULL + NT,
                       B_QFREE = B_QREADY + NT, B_PART = B_QFREE + NT, B_S = B_PART + NT, B_P = B_S + NT * NB, B_O = B_P + NT * NB,
                       B_ITEM = B_O + NT * NB, B_TAKEN = B_ITEM + kDeal, B_END = B_TAKEN + kDeal;
    constexpr uint32_t W_LOAD = 4 * NT, W_MMA = W_LOAD + 1, W_ENDS = W_LOAD + 3;  // the warps past softmax
    const uint32_t per = kRows / a.group;  // rows of the request in a tile
    const uint32_t piece_rows = min(a.c.page_size, P::kKeys), piece_shift = 31 - __clz(piece_rows), pieces = P::kKeys >> piece_shift;
    if (warp == W_LOAD) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(base + P::kWords) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < P::kStages; ++i) {
            bar_init(bar(B_FULL + i), kCodes ? P::kEnds : 1);
            bar_init(bar(B_FREE + i), 2);
            bar_init(bar(B_RAW + i), 1);
        }
        for (int i = 0; i < (int)P::kRawStages; ++i) {
            bar_init(bar(B_CODES + i), 1);
            bar_init(bar(B_TURNED + i), P::kEnds);
        }
        for (uint32_t i = 0; i < NT; ++i) {
            bar_init(bar(B_QFULL + i), 1);
            bar_init(bar(B_QREADY + i), 4);
            bar_init(bar(B_QFREE + i), 1);
            bar_init(bar(B_PART + i), 4);
        }
        for (uint32_t i = 0; i < NT * NB; ++i) {
            bar_init(bar(B_S + i), 1);
            bar_init(bar(B_P + i), 4);
            bar_init(bar(B_O + i), 1);
        }
        for (uint32_t i = 0; i < kDeal; ++i) {
            bar_init(bar(B_ITEM + i), 1);
            bar_init(bar(B_TAKEN + i), 4 * NT + 2 + P::kEnds);  // all warps but the dealer
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
        it.place = __shfl_sync(0xffffffffu, s.place, 0), it.head = __shfl_sync(0xffffffffu, s.head, 0);
        it.seq = __shfl_sync(0xffffffffu, s.seq, 0), it.keys = __shfl_sync(0xffffffffu, s.keys, 0);
        it.sunk = __shfl_sync(0xffffffffu, s.sunk, 0), it.gap = __shfl_sync(0xffffffffu, s.gap, 0);
        it.from = __shfl_sync(0xffffffffu, s.from, 0), it.upto = __shfl_sync(0xffffffffu, s.upto, 0);
        it.part = __shfl_sync(0xffffffffu, s.part, 0), it.parts = __shfl_sync(0xffffffffu, s.parts, 0);
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
        const int32_t hi = max(0, min(it.keys, it.place + at + s.count));  // tokens up to the last row
        s.tiles = s.count ? max(0, min(it.upto, (hi + kKeys - 1) / kKeys - it.gap) - it.from) : 0;
        return s;
    };
    auto tiles_of = [&](const Item &it) {  // units that any of its row tiles takes
        int32_t n = 0;
        for (uint32_t t = 0; t < NT; ++t) n = max(n, span(it, (int)t).tiles);
        return n;
    };
    // the first token of unit j of the piece
    auto first_of = [&](const Item &it, int32_t j) {
        const int32_t u = it.from + j;
        return (u < it.sunk ? u : u + it.gap) * kKeys;
    };
    // whether every row of the item sees all tokens of the tile that begins with token k0
    auto plain = [&](const Item &it, int32_t k0) {
        return k0 + kKeys <= min(it.keys, it.place + 1) &&
               (!a.window || it.place + it.count - 1 - k0 < (int32_t)a.window || (uint32_t)(k0 + kKeys) <= a.sinks);
    };
    // stages that an item takes: K tiles that logits run ahead by, then V j with K j + NB
    auto lead_of = [](int32_t tiles) { return min(tiles, (int32_t)NB); };
    auto stages_of = [&](int32_t tiles) { return (uint32_t)(tiles + lead_of(tiles)); };

    if (warp < 4 * NT) {
        // ---- softmax: thread = row of tile t ----
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(P::kSoft));
        const int t = (int)warp >> 2;
        const uint32_t row = threadIdx.x & 127u, p = row / a.group;
        const uint32_t lanes = (warp & 3u) * 32u << 16;
        const uint32_t to = tmem + lanes + P::kColO + t * D;
        uint32_t phase = 0, phase_o = 0;  // a bit for each buffer of logits, and one for parts
        uint32_t q_phase = 0, stage_no = 0;
        // the tokens k0 .. k0 + 63 that a row at position `at` sees, a bit each
        auto mask_of = [&](int32_t at, int32_t keys, int32_t k0) -> uint64_t {
            const int32_t hi = min(keys, at + 1) - k0;
            uint64_t m = hi <= 0 ? 0 : hi >= 64 ? ~0ull : (1ull << hi) - 1;
            if (a.window) {
                const int64_t lo = (int64_t)at - a.window + 1 - k0, sk = (int64_t)a.sinks - k0;
                const uint64_t in = lo <= 0 ? ~0ull : lo >= 64 ? 0 : ~0ull << lo;
                m &= in | (sk <= 0 ? 0 : sk >= 64 ? ~0ull : (1ull << sk) - 1);
            }
            return m;
        };
        // (of an item only what the loop needs stays in registers; the rest is read again at its end)
        for (uint32_t n = 0;; ++n) {
            int32_t tiles, all_tiles;
            int32_t full_from, full_upto;  // units of the piece that every row sees all of (but sinks)
            float q_mul = 1.0f;  // the power of two that this row's queries were divided by
            {
                Item it;
                if (!next(n, it)) break;
                tiles = span(it, t).tiles;
                all_tiles = tiles_of(it);
                const int32_t last = it.place + it.count - 1;
                full_from = a.window ? (max(0, last - (int32_t)a.window + 1) + kKeys - 1) / kKeys : 0;
                full_upto = max(0, min(it.keys, it.place + 1)) / kKeys - it.gap - it.from;
                full_from = max(full_from - it.gap, it.sunk) - it.from;
            }
            bool fine = true;
            if constexpr (kQTurn) {
                if (tiles) {
                    if (!(fine = all_wait(bar(B_QFULL + t), q_phase))) break;
                    q_phase ^= 1;
                    unsigned char *q = sm + P::kQ + t * P::kQTile + row * 128;
                    auto chunk = [&](uint32_t u) { return reinterpret_cast<uint4 *>(q + u / 8 * P::kQChunk + ((u % 8 ^ (row & 7u)) << 4)); };
                    uint32_t big = 0;
#pragma unroll 4
                    for (uint32_t u = 0; u < D / 8; ++u) {
                        const uint4 x = *chunk(u);
                        const uint32_t y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                        for (int k = 0; k < 4; ++k) big = max(big, max(y[k] & 0x7fffu, y[k] >> 16 & 0x7fffu));
                    }
                    // the row's largest value to [2^13, 2^14): what FP16 then drops is 2^-38 of it
                    const int e = (int)(big >> 7) - 127, up = min(max(13 - e, -126), 126);
                    q_mul = __uint_as_float((uint32_t)(127 - up) << 23);
                    const float f = __uint_as_float((uint32_t)(127 + up) << 23);
#pragma unroll 4
                    for (uint32_t u = 0; u < D / 8; ++u) {
                        const uint4 x = *chunk(u);
                        const uint32_t y[4] = {x.x, x.y, x.z, x.w};
                        uint32_t z[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) z[k] = pack<false>(from_bf16(y[k] & 0xffffu) * f, __uint_as_float(y[k] & 0xffff0000u) * f);
                        *chunk(u) = make_uint4(z[0], z[1], z[2], z[3]);
                    }
                    fence_async();
                    __syncwarp();
                    if (lane == 0) bar_arrive(bar(B_QREADY + t));
                }
            }
            float ref = -INFINITY, sum = 0.0f;  // the maximum that probabilities are relative to (log2 units)
            float unit = -INFINITY;             // codes: what their products with value scales are relative to
            for (int32_t j = 0; j < tiles; ++j) {
                const uint32_t buf = j % NB, ts = tmem + lanes + (NB * t + buf) * kKeys;
                if (!(fine = all_wait(bar(B_S + NB * t + buf), phase >> buf & 1u))) break;
                phase ^= 1u << buf;
                tc_after();
                uint32_t x[kKeys];
                tm_load(ts, x);
                tm_load(ts + 32, x + 32);
                // where the K tile lay
                const uint32_t meta = (stage_no + (uint32_t)j) % P::kMeta;
                const uint32_t bad = bad_pages[meta] & 15u;
                float mul = a.scale, largest = 0.0f;
                uint32_t each = 0;
                if constexpr (kCodes) {
                    const float4 about = *reinterpret_cast<const float4 *>(sm + P::kAbout + meta * sizeof(About));
                    // (not 0, which minus infinity is not multiplied by: such logits are next to nothing)
                    mul = fmaxf(about.x * q_mul, 1.2e-38f), largest = about.y, each = __float_as_uint(about.z);
                }
                tc_wait_ld();
                float *s = reinterpret_cast<float *>(x);
                if (kCodes && (P::kOwn || each & 1u)) {
                    const float4 *by = reinterpret_cast<const float4 *>(sm + P::kScales) + meta * (P::kBy * kKeys / 4);
#pragma unroll
                    for (int i = 0; i < kKeys; i += 4) {
                        const float4 f = by[i / 4];
                        const float2 f0 = __fmul2_rn(make_float2(s[i], s[i + 1]), make_float2(f.x, f.y));
                        const float2 f1 = __fmul2_rn(make_float2(s[i + 2], s[i + 3]), make_float2(f.z, f.w));
                        s[i] = f0.x, s[i + 1] = f0.y, s[i + 2] = f1.x, s[i + 3] = f1.y;
                    }
                }
                if (j < full_from || j >= full_upto || bad) {
                    const volatile Item &it = items[n % kDeal];
                    const int32_t u = it.from + j, k0 = (u < it.sunk ? u : u + it.gap) * kKeys;
                    uint64_t m = mask_of(it.place + t * (int32_t)per + (int32_t)p, it.keys, k0);
                    for (uint32_t c = 0; c < pieces; ++c)
                        if (bad >> c & 1u) m &= ~((piece_rows == 64 ? ~0ull : (1ull << piece_rows) - 1) << (c << piece_shift));
                    const uint32_t m0 = (uint32_t)m, m1 = (uint32_t)(m >> 32);
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        if (!(m0 >> i & 1u)) s[i] = -INFINITY;
                        if (!(m1 >> i & 1u)) s[i + 32] = -INFINITY;
                    }
                }
                float c0 = max3(s[0], s[1], s[2]), c1 = max3(s[3], s[4], s[5]), c2 = max3(s[6], s[7], s[8]);
                float c3 = max3(s[9], s[10], s[11]);
#pragma unroll
                for (int i = 12; i + 7 < kKeys; i += 8) {
                    c0 = max3(c0, s[i], s[i + 1]);
                    c1 = max3(c1, s[i + 2], s[i + 3]);
                    c2 = max3(c2, s[i + 4], s[i + 5]);
                    c3 = max3(c3, s[i + 6], s[i + 7]);
                }
                c0 = max3(c0, s[kKeys - 4], s[kKeys - 3]);
                c1 = max3(c1, s[kKeys - 2], s[kKeys - 1]);
                const float top = fmaxf(max3(c0, c1, c2), c3) * mul;
                const bool grown = top > ref + kLazy;  // each row for itself, not by the others of the warp
                float beta = 0.0f;                     // 2^beta: what outputs are multiplied by
                float give = 1.0f;                     // codes: what the sum of the tile's probabilities is multiplied by
                bool moved = j != 0 && grown;
                if constexpr (kCodes) {
                    // no product is larger than the largest probability x the largest scale; where scales are far apart, look
                    const float most = unit - largest - (kApart + kUpCodes);
                    bool slow = grown || top + largest > unit + kRoom || most > ref || each & 2u;
                    moved = false;
                    if (__any_sync(0xffffffffu, slow)) {
                        if (j == 0 || grown) {
                            sum *= j == 0 ? 1.0f : ex2(ref - top);
                            ref = top;
                        }
                        const float *logs = reinterpret_cast<const float *>(sm + P::kScales) + (meta * P::kBy + 1) * kKeys;
                        float peak = top + largest;
                        // (seldom, and so short loops over tensor memory: unrolled over registers, their code costs what kFma says)
                        if (each & 2u) {
                            peak = -INFINITY;
                            tm_store(ts, x);
                            tm_store(ts + 32, x + 32);
                            tc_wait_st();
#pragma unroll 1
                            for (int c = 0; c < kKeys; c += 16) {
                                uint32_t y[16];
                                tm_load16(ts + c, y);
                                tc_wait_ld();
#pragma unroll
                                for (int i = 0; i < 16; ++i) peak = fmaxf(peak, fmaf(__uint_as_float(y[i]), mul, logs[c + i]));
                            }
                        }
                        const float now = fmaxf(peak > unit + kRoom ? peak : unit, ref - kApart);
                        if (j != 0 && now > unit) beta = unit - now, moved = true;
                        unit = now;
                        if (__any_sync(0xffffffffu, (each & 2u) || unit - largest - (kApart + kUpCodes) > ref)) {
                            // the sum for itself, and logits of the products
                            const float from = ref == -INFINITY ? 0.0f : ref;
                            tm_store(ts, x);
                            tm_store(ts + 32, x + 32);
                            tc_wait_st();
#pragma unroll 1
                            for (int c = 0; c < kKeys; c += 16) {
                                uint32_t y[16];
                                tm_load16(ts + c, y);
                                tc_wait_ld();
#pragma unroll
                                for (int i = 0; i < 16; ++i) {
                                    const float v = __uint_as_float(y[i]) * mul;
                                    sum += ex2(v - from);
                                    y[i] = __float_as_uint(each & 2u ? v + (logs[c + i] - largest) : v);
                                }
                                tm_store16(ts + c, y);
                            }
                            tc_wait_st();
                            tm_load(ts, x);
                            tm_load(ts + 32, x + 32);
                            tc_wait_ld();
                            mul = 1.0f, give = 0.0f;
                        }
                    }
                    give *= ex2(unit - largest - kUpCodes - ref);
                    if (give != give) give = 0.0f;
                } else {
                    if (j == 0) ref = top;
                    else if (grown) {
                        beta = ref - top;
                        ref = top;
                    }
                }
                if (__any_sync(0xffffffffu, moved)) {
                    // not under a product that is still adding to the outputs: the other buffer's next logits
                    // come after it, or nothing does (with one buffer, these logits did)
                    if (NB == 2) {
                        const uint32_t other = buf ^ 1u, on = NB * t + other;
                        fine = j + 1 < tiles ? all_wait(bar(B_S + on), phase >> other & 1u) : all_wait(bar(B_O + on), phase_o >> other & 1u);
                        if (!fine) break;
                        tc_after();
                    }
                    const float f = ex2(beta);
                    if (!kCodes) sum *= f;
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
                // probabilities; over codes, times the largest scale of the tile's values, relative to 2^unit
                const float from = ref == -INFINITY ? 0.0f : kCodes ? unit - largest - kUpCodes : ref - kUp<BF>;
                float2 total = make_float2(0.0f, 0.0f);
                const float2 mul2 = make_float2(mul, mul), from2 = make_float2(-from, -from);
                const float4 *mantissas = reinterpret_cast<const float4 *>(sm + P::kScales) + (meta * P::kBy + 2) * (kKeys / 4);
                float4 four = make_float4(1.0f, 1.0f, 1.0f, 1.0f);
#pragma unroll
                for (int i = 0; i < kKeys; i += 2) {
                    const float2 v = __ffma2_rn(make_float2(s[i], s[i + 1]), mul2, from2);
                    float2 e = i % 16 < P::kFma ? ex2_fma(v) : make_float2(ex2(v.x), ex2(v.y));
                    total = __fadd2_rn(total, e);
                    if constexpr (F == F_INT8) {
                        if (i % 4 == 0) four = mantissas[i / 4];
                        e = __fmul2_rn(e, i % 4 ? make_float2(four.z, four.w) : make_float2(four.x, four.y));
                    }
                    x[i / 2] = pack<BF>(e.x, e.y);
                }
                sum = kCodes ? fmaf(total.x + total.y, give, sum) : sum + (total.x + total.y);
                tm_store(ts, x);
                tc_wait_st();
                tc_before();
                __syncwarp();
                if (lane == 0) bar_arrive(bar(B_P + NB * t + buf));
            }
            stage_no += stages_of(all_tiles);
            Item it;
            read(n, it);
            const TileSpan sp = span(it, t);
            if (fine && sp.count) {
                const bool live = p < (uint32_t)sp.count;
                const int32_t at = it.place + t * (int32_t)per + (int32_t)p;  // this row's position
                // the last products of every buffer
                for (uint32_t buf = 0; buf < NB && (int32_t)buf < sp.tiles && fine; ++buf) {
                    fine = all_wait(bar(B_O + NB * t + buf), phase_o >> buf & 1u);
                    phase_o ^= 1u << buf;
                }
                if (!fine) break;
                tc_after();
                const uint32_t flagged = __shfl_sync(0xffffffffu, bad_flag[n % kDeal], 0);
                // what outputs are multiplied by to be relative to the probabilities' maximum
                const float back = !kCodes ? 1.0f : unit == -INFINITY ? 0.0f : ex2(unit - ref - kUpCodes - P::kUpTile);
                // infinities and NaN among the values that this row sees in tiles that were looked through, added to
                // what the other tokens came to, which may be an infinity or a NaN of their own
                if (flagged) {
#pragma unroll 1
                    for (int d0 = 0; d0 < D && sp.tiles; d0 += 16) {
                        uint32_t o[16];
                        tm_load16(to + d0, o);
                        tc_wait_ld();
#pragma unroll 1
                        for (int32_t j = 0; j < sp.tiles; ++j) {
                            const int32_t k0 = first_of(it, j);
                            if (plain(it, k0)) continue;
                            uint64_t m = live ? mask_of(at, it.keys, k0) : 0;
#pragma unroll 1
                            for (; m; m &= m - 1) {
                                const uint32_t k = (uint32_t)k0 + __ffsll((long long)m) - 1;
                                const int32_t page = __ldg(a.table + (int64_t)it.seq * a.table_stride + (k >> a.c.page_shift));
                                if ((uint32_t)page >= a.c.pages) continue;
                                const uint64_t r = ((uint64_t)page * a.c.heads + it.head << a.c.page_shift) + (k & (a.c.page_size - 1));
                                if constexpr (kCodes) {
                                    const uint32_t sc = __ldg(a.c.vs + r * P::kGroups + (P::kGroups == 1 ? 0 : d0 / 32));
                                    if ((sc & 0x7f80u) == 0x7f80u)
#pragma unroll
                                        for (int i = 0; i < 16; ++i) o[i] = 0x7fc00000u;
                                } else {
                                    constexpr uint32_t E = QBF ? 0x7f80u : 0x7c00u;
                                    const uint16_t *v = reinterpret_cast<const uint16_t *>(a.c.v) + r * D + d0;
#pragma unroll
                                    for (int i = 0; i < 16; ++i) {
                                        const uint32_t y = __ldg(v + i);
                                        if ((y & E) != E) continue;
                                        const float z = QBF ? from_bf16(y) : __half2float(__ushort_as_half((unsigned short)y));
                                        o[i] = __float_as_uint(__uint_as_float(o[i]) + z);
                                    }
                                }
                            }
                        }
                        __syncwarp();
                        tm_store16(to + d0, o);
                        tc_wait_st();
                    }
                }
                // Parts of an item go to the workspace, [32 rows][dimension, maximum, sum][row].  The CTA that is the last
                // to finish its part joins them, in the order of the CTAs, each warp of a row tile a quarter of the
                // dimensions of all its rows: however few rows there are, four warps have loads under way.
                const bool whole = it.parts == 1;
                constexpr uint64_t kBlock = (uint64_t)(D + 2) * 32, kSlot = 4 * NT * kBlock;
                float *parts = reinterpret_cast<float *>(static_cast<unsigned char *>(a.workspace) + a.counters) + (uint64_t)(4 * t) * kBlock + lane;
                auto part_of = [&](int32_t c, uint32_t block) { return parts + (2ull * c + (c == it.part ? 1 : 0)) * kSlot + block * kBlock; };
                // blocks of 32 rows that are this warp's to write, and its runs of kW dimensions
                constexpr int kW = P::kTurn, kL = kW / 8;
                static_assert(D == 4 * kW);
                uint32_t block = warp & 3u, block_end = block + 1;
                int run = 0, run_end = D / kW;
                if (!whole) {
                    const uint32_t blocks = ((uint32_t)sp.count * a.group + 31) / 32;
                    if (block < blocks) {
                        float *mine = part_of((int32_t)blockIdx.x, block);
                        __stcg(mine + D * 32, sp.tiles ? ref : -INFINITY);
                        __stcg(mine + (D + 1) * 32, sp.tiles ? sum : 0.0f);
#pragma unroll 1
                        for (int c = 0; c < D / 16; ++c) {
                            uint32_t o[16] = {};
                            if (sp.tiles) {
                                tm_load16(to + 16 * c, o);
                                tc_wait_ld();
                            }
#pragma unroll
                            for (int i = 0; i < 16; ++i) __stcg(mine + (16 * c + i) * 32, __uint_as_float(o[i]) * back);
                        }
                        tc_before();
                        __threadfence();
                    }
                    __syncwarp();
                    if (lane == 0) bar_arrive(bar(B_PART + t));
                    if (!(fine = all_wait(bar(B_PART + t), phase >> 8 & 1u))) break;
                    phase ^= 1u << 8;
                    __threadfence();
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
                    run = (int)block, run_end = run + 1;
                    block = 0, block_end = blocks;
                }
                const int64_t first_row = (int64_t)(it.token + t * (int32_t)per) * a.q_heads + it.head * a.group;
                unsigned char *turn = sm + P::kOut + warp * 64 * kW;
                // 16-byte chunk c of row r: a phase of eight lanes meets 128 different bytes, writing and reading
                auto chunk = [&](uint32_t r, uint32_t c) { return turn + r * 2 * kW + ((c ^ r / (8 / kL) % kL) << 4); };
#pragma unroll 1
                for (; block < block_end; ++block) {
                    const uint32_t own = 32 * block + lane, own_p = own / a.group;  // this thread's row
                    const bool none = it.place + t * (int32_t)per + (int32_t)own_p < 0 || it.keys == 0;
                    // kW dimensions at a time, turned through shared memory so that kL lanes write 16 kL bytes of a row
                    int32_t to_row[kL];  // of the rows that this lane writes for, from first_row on; -1 for none
#pragma unroll
                    for (int i = 0; i < kL; ++i) {
                        const uint32_t tr = 32 * block + (32 / kL) * i + lane / kL, rp = tr / a.group;
                        to_row[i] = rp < (uint32_t)sp.count ? (int32_t)(rp * a.q_heads + tr % a.group) : -1;
                    }
#pragma unroll 1
                    for (int c = run; c < run_end; ++c) {
                        uint32_t o[kW];
#pragma unroll
                        for (int i = 0; i < kW; ++i) o[i] = 0;
                        if (!whole) {
                            ref = -INFINITY, sum = 0.0f;
                            const int32_t after = it.part + it.parts;
#pragma unroll 1
                            for (int32_t q = it.part; q < after; q += kJoin) {  // their loads in flight together
                                float m[kJoin], l[kJoin], y[kJoin][kW];
#pragma unroll
                                for (int b = 0; b < kJoin; ++b) {
                                    const float *from = part_of(q + b, block);
                                    m[b] = q + b < after ? __ldcg(from + D * 32) : -INFINITY;
                                    l[b] = q + b < after ? __ldcg(from + (D + 1) * 32) : 0.0f;
#pragma unroll
                                    for (int i = 0; i < kW; ++i) y[b][i] = q + b < after ? __ldcg(from + (kW * c + i) * 32) : 0.0f;
                                }
                                float top = ref;
#pragma unroll
                                for (int b = 0; b < kJoin; ++b) top = max_nan(top, m[b]);
                                const float to_top = top == -INFINITY ? 0.0f : top, f = ex2(ref - to_top);
                                sum *= f;
#pragma unroll
                                for (int i = 0; i < kW; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
#pragma unroll
                                for (int b = 0; b < kJoin; ++b) {
                                    const float e = ex2(m[b] - to_top);  // 0 for a part of no tile that this row sees
                                    sum = fmaf(e, l[b], sum);
#pragma unroll
                                    for (int i = 0; i < kW; ++i) o[i] = __float_as_uint(fmaf(e, y[b][i], __uint_as_float(o[i])));
                                }
                                ref = top;
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
                        const float inv = none || sum == 0.0f ? 0.0f : whole ? back / sum : 1.0f / sum;  // (0: every logit is -infinity)
#pragma unroll
                        for (int i = 0; i < kL; ++i) {
                            auto two = [&](int k) { return pack<QBF>(__uint_as_float(o[8 * i + k]) * inv, __uint_as_float(o[8 * i + k + 1]) * inv); };
                            *reinterpret_cast<uint4 *>(chunk(lane, i)) = make_uint4(two(0), two(2), two(4), two(6));
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
                    if (run == 0 && own_p < (uint32_t)sp.count && a.lse)
                        a.lse[first_row + (int64_t)own_p * a.q_heads + own % a.group] = none ? -INFINITY : (ref - (kCodes ? 0.0f : kUp<BF>) + __log2f(sum)) * kLn2;
                }
                tc_before();
            }
            if (!fine) break;
            taken(n);
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(P::kRest));
        if (warp == W_LOAD) {
            // ---- the deal ----
            // An item's price is its tokens, as its last row sees them, and kItemCost; items stand in order - requests, KV
            // heads, blocks - on a line as long as their prices, unit j of one at kItemCost + 64 j of its stretch, and the
            // line is cut into equal ranges, one a CTA, none shorter than a tile.  An item of up to kWhole (or kWholeFew) tokens is the
            // CTA's in whose range it begins.  With a window no item is priced above `most`, which holds its units.
            const int32_t block = (int32_t)(a.tiles * per);
            const int64_t most = a.window ? (int64_t)a.window + block + ((int64_t)(a.sinks + 63u) & ~63ll) + 2 * kKeys : (int64_t)1 << 40;
            struct Seq {
                int32_t q0, nq, nk, blocks, shift;
            } sq;
            auto load_seq = [&](uint32_t s) {
                Seq q{};
                if (s >= a.batch) return q;
                const int32_t q0 = a.starts ? __ldg(a.starts + s) : (int32_t)s, q1 = a.starts ? __ldg(a.starts + s + 1) : (int32_t)s + 1;
                const int32_t given = __ldg(a.lengths + s);
                const int32_t nk = given < 0 ? 0 : (int32_t)min((uint32_t)given, a.width << a.c.page_shift);
                const bool none = q0 < 0 || q1 < q0 || (uint64_t)(uint32_t)q1 > a.q_tokens;
                if ((none || nk != given) && blockIdx.x == 0) atomicOr(a.status, kStatusBadExtent);
                if (none) return q;
                q.q0 = q0, q.nq = q1 - q0, q.nk = nk, q.shift = nk - q.nq;
                q.blocks = (int32_t)(((uint32_t)q.nq + block - 1) / (uint32_t)block);
                return q;
            };
            // tokens of block b, one at least
            auto keys_of = [&](const Seq &q, int32_t b) -> int64_t {
                const int64_t hi = b + 1 >= q.blocks ? q.nk : (int64_t)(b + 1) * block + q.shift;
                return max((int64_t)1, min(hi, most));
            };
            // price of the blocks before b of one head
            auto price = [&](const Seq &q, int32_t b) -> int64_t {
                if (b == 0) return 0;
                int64_t n = b * kItemCost;
                const int32_t m = min(b, q.blocks - 1);  // all but the last block: (b + 1) block + shift tokens, at most `most`, or 1
                const int32_t z = q.shift < 0 ? min(m, (int32_t)((uint32_t)(1 - q.shift) / (uint32_t)block)) : 0;
                int32_t y = m;
                if (a.window) y = most <= q.shift ? z : max(z, (int32_t)min((int64_t)m, quotient(most - q.shift, block)));
                n += z + (int64_t)block * (((int64_t)y * (y + 1) - (int64_t)z * (z + 1)) / 2) + (int64_t)q.shift * (y - z);
                n += (m - y) * most;
                return b == q.blocks ? n + max((int64_t)1, min((int64_t)q.nk, most)) : n;
            };
            // the first 32 requests stay in the lanes, with the price of all before each of them and its own
            const Seq mine = load_seq(lane);
            const int64_t own = a.c.heads * price(mine, mine.blocks);
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
                q.q0 = __shfl_sync(0xffffffffu, mine.q0, s), q.nq = __shfl_sync(0xffffffffu, mine.nq, s);
                q.nk = __shfl_sync(0xffffffffu, mine.nk, s), q.blocks = __shfl_sync(0xffffffffu, mine.blocks, s);
                q.shift = q.nk - q.nq;
                return q;
            };
            int64_t total = __shfl_sync(0xffffffffu, own_upto, 31);
            uint32_t blocks = (uint32_t)mine.blocks;
            auto whole_of = [&](const Seq &q) { return (int64_t)q.nq * a.group <= 64 ? kWholeFew : kWhole; };
            auto splits = [&](const Seq &q) { return q.blocks && min((int64_t)q.nk, most) > whole_of(q); };
            bool split = splits(mine);
            if (a.batch > 32) {
                int64_t rest = 0;
                for (uint32_t s = lane + 32; s < a.batch; s += 32) {
                    const Seq q = load_seq(s);
                    rest += a.c.heads * price(q, q.blocks);
                    blocks += (uint32_t)q.blocks;
                    split |= splits(q);
                }
                total += __shfl_sync(0xffffffffu, scan(rest), 31);
            }
            const int64_t all = (int64_t)__reduce_add_sync(0xffffffffu, blocks) * a.c.heads;
            int64_t ctas = min((int64_t)gridDim.x, max((int64_t)1, total / kKeys));
            if (__any_sync(0xffffffffu, split)) ctas = min(ctas, max(all, total / kPiece));
            bool some = total > 0 && ctas > 0 && (int64_t)blockIdx.x < ctas;
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
                        price_of = a.c.heads * price(q, q.blocks);
                        upto = scan(price_of);
                    }
                    const uint32_t past = __ballot_sync(0xffffffffu, at + upto > start);
                    if (past) {
                        const uint32_t l = __ffs(past) - 1;
                        at += __shfl_sync(0xffffffffu, upto - price_of, l);
                        seq = s0 + l;
                        break;
                    }
                    if (s0 + 32 >= a.batch) {
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
                    const int64_t keys = keys_of(sq, blk);
                    const int32_t pos = blk * block, count = min(block, sq.nq - pos), place = sq.shift + pos;
                    const int32_t hi = max(0, min(sq.nk, place + count));
                    const int32_t lo = a.window ? (int32_t)max((int64_t)0, (int64_t)place - a.window + 1) : 0;
                    const int32_t sunk = min((int32_t)((min(a.sinks, (uint32_t)lo) + kKeys - 1) / kKeys), lo / kKeys);
                    const int32_t gap = lo / kKeys - sunk, units = max(1, (hi + kKeys - 1) / kKeys - gap);
                    const int64_t from = at + kItemCost;
                    int32_t one, two;
                    if (keys <= whole_of(sq)) {  // where it begins
                        one = 0;
                        two = at >= start ? units : 0;
                    } else {
                        one = start <= from ? 0 : (int32_t)min((int64_t)units, (start - from + kKeys - 1) / kKeys);
                        two = end <= from ? 0 : (int32_t)min((int64_t)units, (end - from + kKeys - 1) / kKeys);
                    }
                    if (one < two) {
                        it.token = sq.q0 + pos;
                        it.count = count;
                        it.place = place;
                        it.head = head;
                        it.seq = (int32_t)seq;
                        it.keys = sq.nk;
                        it.sunk = sunk;
                        it.gap = gap;
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
                        if (++head == (int32_t)a.c.heads) {
                            head = 0;
                            do {
                                if (++seq >= a.batch) {
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
                    d.token = it.token, d.count = it.count, d.place = it.place, d.head = it.head, d.seq = it.seq;
                    d.keys = it.keys, d.sunk = it.sunk, d.gap = it.gap, d.from = it.from, d.upto = it.upto;
                    d.part = it.part, d.parts = it.parts;
                    bad_flag[n % kDeal] = 0;
                    bar_arrive(bar(B_ITEM + n % kDeal));
                }
                __syncwarp();
            };
            // ---- loads ----
            // The first stages of an item are the K tiles that logits run ahead by, then come V j and K j + NB.  Lanes in
            // fours, one for each piece of a tile: two columns of 64 dimensions of V, and of K; over codes V's codes and
            // scales, K's codes and scales, and the scales of the values of K's tokens.  A stage that the last warp looks
            // through (16 bits) lands on its raw barrier, and that warp arrives on the full one when it is done with it;
            // codes land in stages of their own.
            constexpr uint32_t kRing = kCodes ? P::kRawStages : P::kStages;
            uint32_t slot = 0, free_phase = 1, q_phase = (1u << NT) - 1, issued = 0, full_phase = 0, raw = 0, raw_phase = 0;
            uint32_t q_issued = 0, stage_no = 0;
            const uint32_t what = lane >> 2, half = what & 1u, piece = lane & 3u;
            Item it;
            bool fine = true;
            deal(0);
            for (uint32_t n = 0; fine && next(n, it); ++n) {
                const int32_t tiles = tiles_of(it);
                auto load_q = [&](int t) {
                    if (!(fine = fine && all_wait(bar(B_QFREE + t), q_phase >> t & 1u))) return;
                    q_phase ^= 1u << t;
                    q_issued |= 1u << t;
                    if (lane == 0) {
                        bar_expect(bar(B_QFULL + t), P::kChunks * per * a.group * 128u);
                        for (uint32_t c = 0; c < P::kChunks; ++c)
                            tma3(base + P::kQ + t * P::kQTile + c * P::kQChunk, &mq, bar(B_QFULL + t), 64 * c,
                                 it.head * (int32_t)a.group, it.token + t * (int32_t)per);
                    }
                    __syncwarp();
                };
                // the tile of stage k that this lane has a piece of; -1: none
                const int32_t lead = lead_of(tiles);
                auto unit_of = [&](int32_t k) -> int32_t {
                    const int32_t j = what < 2 ? k - lead : k;
                    return what < (kCodes ? 5u : 4u) && piece < pieces && j >= 0 && j < tiles ? j : -1;
                };
                auto token_of = [&](int32_t k) {
                    const int32_t j = unit_of(k);
                    return j < 0 ? 0x7fffffff : first_of(it, j) + (int32_t)(piece << piece_shift);
                };
                auto page_of = [&](int32_t k) {  // -1 past the request's tokens
                    const int32_t token = token_of(k);
                    return token < it.keys ? __ldg(a.table + (int64_t)it.seq * a.table_stride + (token >> a.c.page_shift)) : -1;
                };
                // A piece between the first tokens and the window of the item's first row is absent, whatever the table says of it.
                const int32_t shown = a.window ? (int32_t)max((int64_t)-1, (int64_t)it.place - a.window + 1 - piece_rows) : -1;
                int32_t page = tiles ? page_of(0) : 0;
                auto load = [&](int32_t k) {
                    const int32_t ahead = k + 1 < tiles + lead ? page_of(k + 1) : 0;
                    const int32_t token = token_of(k);
                    const bool hidden = token <= shown && (uint32_t)token >= a.sinks;
                    const bool there = (uint32_t)page < a.c.pages && !hidden;
                    const uint32_t bad = __ballot_sync(0xffffffffu, token < it.keys && !there);
                    const bool wrong = __any_sync(0xffffffffu, token < it.keys && !there && !hidden);
                    if (!(fine = fine && all_wait(bar((kCodes ? B_TURNED : B_FREE) + slot), free_phase))) return;
                    const bool values = k >= lead, keys = k < tiles;
                    const bool look = !kCodes && values && !plain(it, first_of(it, k - lead));
                    const uint32_t on = bar((kCodes ? B_CODES : look ? B_RAW : B_FULL) + slot), bit = 1u << slot;
                    if (lane == 0) {
                        if (wrong) atomicOr(a.status, kStatusBadSlot);
                        bad_pages[stage_no % P::kMeta] = (bad >> 8 & 15u) | (bad & 15u) << 4;
                        bar_expect(on, kCodes ? (values ? P::kRawTile + P::kRawScale : 0u) + (keys ? P::kRawTile + 2 * P::kRawScale : 0u)
                                              : (values ? P::kTile : 0u) + (keys ? P::kTile : 0u));
                    }
                    __syncwarp();
                    if (unit_of(k) >= 0) {
                        const int32_t in_page = token & (int32_t)(a.c.page_size - 1);
                        // (past the cache's last page: zeros)
                        const int32_t z = there ? page : (int32_t)a.c.pages;
                        if constexpr (!kCodes) {
                            if (half < P::kChunks)
                                tma4(base + P::kRing + slot * P::kStageBytes + (what >> 1) * P::kTile + half * P::kChunk + (piece << piece_shift) * 128,
                                     what < 2 ? &mv : &mk, on, 64 * half, in_page, it.head, z);
                        } else {
                            const uint32_t dst = base + P::kRaw + slot * P::kRawStage;
                            if (what == 0 || what == 2)
                                tma4(dst + (what >> 1) * P::kRawTile + (piece << piece_shift) * P::kRow, what == 0 ? &mv : &mk, on, 0, in_page, it.head, z);
                            else {
                                const uint64_t r = there ? ((uint64_t)page * a.c.heads + it.head << a.c.page_shift) + in_page : 0;
                                bulk(dst + 2 * P::kRawTile + (what >> 1) * P::kRawScale + (piece << piece_shift) * P::kGroups * 2,
                                     (what == 3 ? a.c.ks : a.c.vs) + r * P::kGroups, piece_rows * P::kGroups * 2, on);
                            }
                        }
                    }
                    __syncwarp();
                    issued |= bit;
                    raw = look ? raw | bit : raw & ~bit;
                    full_phase = (full_phase & ~bit) | (free_phase ^ 1u) << slot;
                    raw_phase ^= look ? bit : 0;
                    if (++slot == kRing) slot = 0, free_phase ^= 1;
                    ++stage_no;
                    page = ahead;
                };
                if (span(it, 0).tiles) load_q(0);
                if (tiles && fine) load(0);
                for (uint32_t t = 1; t < NT; ++t)
                    if (span(it, (int)t).tiles && fine) load_q((int)t);
                if (tiles && fine) load(1);
                deal(n + 1);
                for (int32_t k = 2; k < tiles + lead && fine; ++k) load(k);
            }
            // copies in flight land before the CTA ends (they have, unless a wait ran out)
            if (lane == 0 && *stop) {
                uint32_t none = 0;
                for (uint32_t i = 0; i < kRing; ++i)
                    if (issued >> i & 1u) {
                        if (kCodes) bar_wait(bar(B_CODES + i), full_phase >> i & 1u, &none);
                        else
                            bar_wait(bar((raw >> i & 1u ? B_RAW : B_FULL) + i), raw >> i & 1u ? ~raw_phase >> i & 1u : full_phase >> i & 1u,
                                     &none);
                    }
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
                    for (uint32_t l = 0; l < (P::kLow ? 2u : 1u); ++l)
#pragma unroll
                        for (uint32_t c = 0; c < P::kChunks; ++c)
#pragma unroll
                            for (uint32_t s = 0; s < 4; ++s)
                                mma_ss(d, q + (c * P::kQChunk + 32 * s) / 16, key + (l * P::kTile + c * P::kChunk + 32 * s) / 16, ID_S, l | c | s);
                };
                // logits run NB tiles ahead of the outputs
                for (int32_t j = 0; j < lead_of(tiles); ++j) {
                    const uint32_t at = base + P::kRing + slot * P::kStageBytes + P::kTile;
                    if (!(fine = all_wait(bar(B_FULL + slot), full_phase))) break;
#pragma unroll
                    for (uint32_t i = 0; i < MINE; ++i) {
                        if (j >= mine[i]) continue;
                        const uint32_t t = half + 2 * i;
                        if (j == 0) {
                            if (!(fine = all_wait(bar((kQTurn ? B_QREADY : B_QFULL) + t), q_phase >> t & 1u))) break;
                            q_phase ^= 1u << t;
                        }
                        tc_after();
                        if (elect()) {
                            logits(t, at, j);
                            tc_commit(bar(B_S + NB * t + j));
                            if (j + 1 == mine[i]) tc_commit(bar(B_QFREE + t));
                        }
                        __syncwarp();
                    }
                    if (!fine) break;
                    if (elect()) tc_commit(bar(B_FREE + slot));
                    __syncwarp();
                    advance();
                }
                if (!fine) break;
                for (int32_t j = 0; j < tiles; ++j) {
                    const uint32_t v = slot, at = base + P::kRing + v * P::kStageBytes;
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
        } else if constexpr (!kCodes) {
            // ---- V tiles that not every row sees ----
            uint32_t slot = 0, raw_phase = 0;
            Item it;
            bool fine = true;
            for (uint32_t n = 0; fine && next(n, it); ++n) {
                const int32_t tiles = tiles_of(it);
                for (int32_t j = 0; j < tiles; ++j) {
                    const int32_t k0 = first_of(it, j);
                    if (plain(it, k0)) continue;
                    const uint32_t v = (slot + (uint32_t)(lead_of(tiles) + j)) % P::kStages;
                    if (!(fine = all_wait(bar(B_RAW + v), raw_phase >> v & 1u))) break;
                    raw_phase ^= 1u << v;
                    unsigned char *tile = sm + P::kRing + v * P::kStageBytes;
                    const int32_t rows = min(kKeys, it.keys - k0);
                    uint32_t found = 0;
                    constexpr uint32_t E = QBF ? 0x7f80u : 0x7c00u;
                    // an exponent of ones carries into the sign's place
                    constexpr uint32_t kCarry = (0x8000u - E) | (0x8000u - E) << 16;
                    auto carry = [&](const uint4 &x) {
                        return ((x.x & 0x7fff7fffu) + kCarry | (x.y & 0x7fff7fffu) + kCarry | (x.z & 0x7fff7fffu) + kCarry |
                                (x.w & 0x7fff7fffu) + kCarry) & 0x80008000u;
                    };
#pragma unroll 4
                    for (uint32_t i = lane; i < P::kKeys * D / 8; i += 32) {
                        const uint32_t r = i / (D / 8), u = i % (D / 8);
                        uint4 *w = reinterpret_cast<uint4 *>(tile + u / 8 * P::kChunk + r * 128 + ((u % 8 ^ (r & 7)) << 4));
                        if ((int32_t)r >= rows) *w = make_uint4(0, 0, 0, 0);
                        else found |= carry(*w);
                    }
                    if (__any_sync(0xffffffffu, found)) {
                        __syncwarp();
                        for (uint32_t i = lane; i < P::kKeys * D; i += 32) {
                            const uint32_t r = i / D, d = i % D;
                            uint16_t *w = reinterpret_cast<uint16_t *>(tile + d / 64 * P::kChunk + r * 128 + (((d % 64 / 8) ^ (r & 7)) << 4)) + d % 8;
                            if ((*w & E) == E) *w = 0;
                        }
                        if (lane == 0) bad_flag[n % kDeal] = 1;
                    }
                    fence_async();
                    __syncwarp();
                    if (lane == 0) bar_arrive(bar(B_FULL + v));
                }
                slot = (slot + stages_of(tiles)) % P::kStages;
                if (fine) taken(n);
            }
        } else {
            // ---- codes into operands ----
            // The first of these warps sees to what softmax has to know, the others turn.
            constexpr uint32_t G = P::kGroups, kTurners = 32 * (P::kEnds - 1);
            const uint32_t me = threadIdx.x - 32 * (W_ENDS + 1);  // (the first warp has none)
            const bool weighs = warp == W_ENDS, turns = !weighs;
            // 16 bytes of a row: in 8 bits 16 dimensions, two chunks of the operand; in 4 bits 32, four chunks.  A thread has
            // kEach of them of one row, the q-th at q ^ twist(row): a phase of eight lanes then meets 128 different
            // bytes, reading and writing (of 32-byte rows, every second one twice).
            constexpr uint32_t kPer = P::kRow / 16, kOut = F == F_INT8 ? 2 : 4;
            constexpr uint32_t kEach = P::kKeys * kPer / kTurners;
            auto twist = [](uint32_t r) {
                if constexpr (kPer == 8) return r & 7u;
                else if constexpr (kPer == 2) return r >> 2 & 1u;
                else if constexpr (F == F_INT4) return r >> 1 & 3u;
                else return (r >> 2 & 1u) | ((r >> 1 ^ r >> 2) & 1u) << 1;
            };
            const uint32_t row = me & 63u;
            auto place_of = [&](uint32_t q) { return ((me >> 6) * kEach + q) ^ twist(row); };
            uint32_t slot = 0, free_phase = 1, from = 0, from_phase = 0, stage_no = 0;
            Item it;
            bool fine = true;
            auto put = [&](unsigned char *tile, uint32_t r, uint32_t u, uint4 v) {
                *reinterpret_cast<uint4 *>(tile + u / 8 * P::kChunk + r * 128 + ((u % 8 ^ (r & 7u)) << 4)) = v;
            };
            // Exponents (biased, at least that of 2^-100) of the largest and the smallest scale of a tile's tokens that are
            // there; finite ones, and the smallest of those that are not zero.
            struct Sizes {
                uint32_t top, least;
                __device__ bool apart() const { return least + kNear < top; }
            };
            auto sizes = [&](const uint16_t *scales, uint32_t rows, uint32_t bad) {
                const uint32_t *words = reinterpret_cast<const uint32_t *>(scales);
                uint32_t w[G], big = 0, small = ~0u;
#pragma unroll
                for (uint32_t i = 0; i < G; ++i) {
                    w[i] = words[lane + 32 * i];
                    big = i ? __vmaxu2(big, w[i]) : w[i];
                    small = i ? __vminu2(small, w[i]) : w[i];
                }
                big = __reduce_max_sync(0xffffffffu, max(big & 0xffffu, big >> 16));
                small = __reduce_min_sync(0xffffffffu, min(small & 0xffffu, small >> 16));
                // (all tokens there, no scale zero, negative or NaN: nearly always)
                if (rows == P::kKeys && !bad && big < 0x7f80u && small >= 0x80u) return Sizes{max(big >> 7, 27u), small >> 7};
                uint32_t top = 27, least = 255;
#pragma unroll
                for (uint32_t i = 0; i < G; ++i)
#pragma unroll
                    for (uint32_t k = 0; k < 2; ++k) {
                        const uint32_t token = (2 * (lane + 32 * i) + k) / G, e = w[i] >> 16 * k >> 7 & 255u;
                        const bool counts = e != 255u && token < rows && !(bad >> (token >> piece_shift) & 1u);
                        top = max(top, counts ? e : 0u);
                        least = min(least, counts && e ? e : 255u);
                    }
                return Sizes{__reduce_max_sync(0xffffffffu, top), __reduce_min_sync(0xffffffffu, least)};
            };
            // exponent of the largest finite scale of a token, at least that of 2^-100
            auto largest = [](const uint16_t *scales) {
                uint32_t big = 0;
#pragma unroll
                for (uint32_t g = 0; g < G; ++g) {
                    const uint32_t s = scales[g] & 0x7fffu;
                    big = max(big, s < 0x7f80u ? s : 0u);
                }
                return max(big >> 7, 27u);
            };
            // 8-bit values: probabilities take the mantissa of a scale that has one (not zero, infinity, NaN or below 2^-126),
            // values the rest, so that no bit of a value is rounded away
            auto mantissa = [](uint32_t scale) {
                const uint32_t e = scale >> 7 & 255u;
                return e - 1u < 254u ? from_bf16(0x3f80u | (scale & 0x7fu)) : 1.0f;
            };
            // what codes are multiplied by, twice: their scale over the power of two of the tile or the token, times 2^kUpTile
            auto factor = [&](const uint16_t *scales, uint32_t r, uint32_t c, const Sizes &z, bool there, auto of_values) {
                uint32_t scale = scales[r * G + (G == 1 ? 0 : c)];
                if (F == F_INT8 && decltype(of_values)::value && (scale >> 7 & 255u) - 1u < 254u) scale &= 0xff80u;
                uint32_t e = z.top;
                float f = from_bf16(scale);
                if (z.apart()) {
                    if constexpr (F == F_INT8) f = (scale & 0x7f80u) == 0x7f80u ? f : 1.0f, e = 127;
                    else e = largest(scales + r * G);
                }
                f = there ? f * __uint_as_float((254 + P::kUpTile - e) << 23) : 0.0f;
                return pack<false>(f, f);
            };
            // 16 bytes of codes times their factor, into the operand; what FP16 leaves of a product, into the second one
            auto turn = [&](const uint4 &codes, unsigned char *tile, auto plain_codes, auto low, uint32_t r, uint32_t c, uint32_t s2) {
                const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
#pragma unroll
                for (uint32_t k = 0; k < kOut; ++k) {
                    uint32_t h[4], l[4];
#pragma unroll
                    for (uint32_t b = 0; b < 4; ++b) {
                        uint32_t code;
                        if constexpr (F == F_INT8)  // 1024 + code + 128
                            code = sub_h(__byte_perm(w[2 * k + b / 2] ^ 0x80808080u, 0x64646464u, b % 2 ? 0x4342 : 0x4140), 0x64806480u);
                        else  // 1024 + code + 8 in the low half, 64 + code + 8 in the high one
                            code = sub_h((__byte_perm(w[k], 0, b | b << 8 | 0x4040u) & 0x00f0000fu) | 0x54006400u, 0x54806408u);
                        h[b] = decltype(plain_codes)::value ? code : mul_h(code, s2);
                        if constexpr (decltype(low)::value) l[b] = rest_h(code, s2, h[b]);
                    }
                    put(tile, r, c * kOut + k, make_uint4(h[0], h[1], h[2], h[3]));
                    if constexpr (decltype(low)::value) put(tile + P::kTile, r, c * kOut + k, make_uint4(l[0], l[1], l[2], l[3]));
                }
            };
            // what softmax has to know of a K tile: the first of these warps writes it
            auto weigh = [&](const uint16_t *keys, const uint16_t *values, const Sizes &zk, const Sizes &zv, uint32_t meta, uint32_t rows) {
                if (lane == 0) {
                    About &about = reinterpret_cast<About *>(sm + P::kAbout)[meta];
                    about.mul = __uint_as_float((zk.top - (P::kOwn ? 0 : P::kUpTile)) << 23) * a.scale;
                    about.top = (float)zv.top - 127.0f;
                    about.each = (zk.apart() ? 1u : 0u) | (zv.apart() ? 2u : 0u);
                }
                float *by = reinterpret_cast<float *>(sm + P::kScales) + meta * P::kBy * kKeys;
                if constexpr (F == F_INT8) {
                    const uint32_t two = reinterpret_cast<const uint32_t *>(values)[lane];
                    reinterpret_cast<float2 *>(by + 2 * kKeys)[lane] = make_float2(mantissa(two & 0xffffu), mantissa(two >> 16));
                }
                if (P::kOwn || zk.apart()) {  // over the tile's largest
                    if constexpr (F == F_INT8) {
                        const uint32_t two = reinterpret_cast<const uint32_t *>(keys)[lane];
                        reinterpret_cast<float2 *>(by)[lane] = __fmul2_rn(make_float2(from_bf16(two & 0xffffu), __uint_as_float(two & 0xffff0000u)),
                                                                          make_float2(__uint_as_float((254 - zk.top) << 23), __uint_as_float((254 - zk.top) << 23)));
                    } else {
                        for (uint32_t r = lane; r < P::kKeys; r += 32) by[r] = ex2((float)largest(keys + r * G) - (float)zk.top);
                    }
                }
                if (zv.apart())  // (logarithms; what has no scale has no weight, or no values)
                    for (uint32_t r = lane; r < P::kKeys; r += 32) {
                        if constexpr (F == F_INT8) {
                            const uint32_t s = values[r], e = s >> 7 & 255u;
                            by[kKeys + r] = r >= rows || e == 255u || !s ? -150.0f : e ? (float)e - 127.0f : __log2f(from_bf16(s));
                        }
                        else by[kKeys + r] = r < rows ? (float)largest(values + r * G) - 127.0f : -150.0f;
                    }
            };
            // A tile's codes, and what they are multiplied by, in registers
            struct Batch {
                uint4 codes[kEach];
                uint32_t s2[kEach];
            };
            // (of values in a tile that is looked through, what has a NaN for a scale is zero)
            auto fetch = [&](Batch &b, const uint4 *codes, const uint16_t *scales, uint32_t rows, uint32_t bad, bool look, auto of_values) {
#pragma unroll
                for (uint32_t q = 0; q < kEach; ++q) b.codes[q] = codes[row * kPer + place_of(q)];
                const Sizes z = sizes(scales, rows, bad);
                uint32_t found = 0;
                const bool there = row < rows && !(bad >> (row >> piece_shift) & 1u);
#pragma unroll
                for (uint32_t q = 0; q < kEach; ++q) {
                    if (G == 1 && q) {
                        b.s2[q] = b.s2[0];
                        continue;
                    }
                    const uint32_t c = place_of(q);
                    const bool nan = look && there && (scales[row * G + (G == 1 ? 0 : c)] & 0x7f80u) == 0x7f80u;
                    found |= nan;
                    b.s2[q] = factor(scales, row, c, z, there && !nan, of_values);
                }
                return found;
            };
            auto write = [&](const Batch &b, unsigned char *tile, auto plain_codes, auto low) {
#pragma unroll
                for (uint32_t q = 0; q < kEach; ++q) turn(b.codes[q], tile, plain_codes, low, row, place_of(q), b.s2[q]);
            };
            for (uint32_t n = 0; fine && next(n, it); ++n) {
                const int32_t tiles = tiles_of(it), lead = lead_of(tiles);
                for (int32_t k = 0; k < tiles + lead; ++k) {
                    if (!(fine = all_wait(bar(B_CODES + from), from_phase))) break;
                    const uint4 *codes = reinterpret_cast<const uint4 *>(sm + P::kRaw + from * P::kRawStage);
                    const uint16_t *scales = reinterpret_cast<const uint16_t *>(codes + 2 * P::kRawTile / 16);
                    constexpr uint32_t kNext = P::kRawScale / 2;
                    unsigned char *tile = sm + P::kRing + slot * P::kStageBytes;
                    const uint32_t meta = stage_no % P::kMeta, bad = bad_pages[meta];
                    const bool values = k >= lead, keys = k < tiles;
                    const uint32_t key_rows = keys ? (uint32_t)min(kKeys, it.keys - first_of(it, k)) : 0;
                    Batch of_keys, of_values;
                    if (turns && values) {
                        const int32_t k0 = first_of(it, k - lead);
                        if (fetch(of_values, codes, scales, (uint32_t)min(kKeys, it.keys - k0), bad >> 4, !plain(it, k0), std::true_type())) bad_flag[n % kDeal] = 1;
                    }
                    if (turns && keys) {
                        if constexpr (P::kOwn) {  // (codes as they are)
#pragma unroll
                            for (uint32_t q = 0; q < kEach; ++q) of_keys.codes[q] = codes[P::kRawTile / 16 + row * kPer + place_of(q)], of_keys.s2[q] = 0;
                        } else fetch(of_keys, codes + P::kRawTile / 16, scales + kNext, key_rows, bad & 15u, false, std::false_type());
                    }
                    if (weighs && keys)
                        weigh(scales + kNext, scales + 2 * kNext, sizes(scales + kNext, key_rows, bad & 15u), sizes(scales + 2 * kNext, key_rows, bad & 15u),
                              meta, key_rows);
                    __syncwarp();
                    if (lane == 0) bar_arrive(bar(B_TURNED + from));
                    if (!(fine = all_wait(bar(B_FREE + slot), free_phase))) break;
                    if (turns && values) write(of_values, tile, std::false_type(), std::false_type());
                    if (turns && keys) write(of_keys, tile + P::kTile, std::bool_constant<P::kOwn>(), std::bool_constant<P::kLow>());
                    fence_async();
                    __syncwarp();
                    if (lane == 0) bar_arrive(bar(B_FULL + slot));
                    if (++slot == P::kStages) slot = 0, free_phase ^= 1;
                    if (++from == P::kRawStages) from = 0, from_phase ^= 1;
                    ++stage_no;
                }
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

// Queries [tokens][heads][dim] as boxes of `rows` tokens x `heads_box` heads x 64 dimensions.
bool make_query_map(CUtensorMap *m, const ChunkArgs &a, uint32_t rows) {
    const cuuint64_t size[3] = {a.c.dim, a.q_heads, a.q_tokens};
    const cuuint64_t stride[2] = {(cuuint64_t)a.q_head * 2, (cuuint64_t)a.q_token * 2};
    const cuuint32_t box[3] = {64, a.group, rows}, step[3] = {1, 1, 1};
    return encoder()(m, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<void *>(a.q), size, stride, box, step,
                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// Pages [pages][heads][page][row] as boxes of up to 64 rows of one page and head: 64 dimensions of them in 16 bits, as
// products read them, or all of their codes.
bool make_page_map(CUtensorMap *m, const PageView &c, const void *rows) {
    const bool codes = c.groups != 0;
    const uint32_t wide = codes ? 1 : 2;
    const cuuint64_t size[4] = {c.row_bytes / wide, c.page_size, c.heads, c.pages};
    const cuuint64_t stride[3] = {c.row_bytes, (cuuint64_t)c.row_bytes * c.page_size, (cuuint64_t)c.row_bytes * c.page_size * c.heads};
    const cuuint32_t box[4] = {codes ? c.row_bytes : 64, c.page_size < 64 ? c.page_size : 64, 1, 1}, step[4] = {1, 1, 1, 1};
    return encoder()(m, codes ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 4, const_cast<void *>(rows), size, stride,
                     box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, codes ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B,
                     CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, int NT, int F, bool QBF>
cudaError_t run(const ChunkArgs &args, int sms, uint32_t tiles, cudaStream_t s) {
    using P = Plan<D, NT, F>;
    auto kernel = chunk_kernel<D, NT, F, QBF>;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    static bool ready[64] = {};
    if (!ready[dev]) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)P::kTotal);
        if (e != cudaSuccess) return e;
        // the warps hand registers to each other: more than the launch has would be waited for
        cudaFuncAttributes f;
        e = cudaFuncGetAttributes(&f, kernel);
        if (e != cudaSuccess) return e;
        if ((uint32_t)f.numRegs * P::kThreads < 128 * NT * P::kSoft + (P::kThreads - 128 * NT) * P::kRest) return cudaErrorNotSupported;
        ready[dev] = true;
    }
    ChunkArgs a = args;
    a.tiles = tiles;
    a.counters = BGTQ_WORKSPACE_ZEROED;
    CUtensorMap mq, mk, mv;
    if (!make_query_map(&mq, a, kRows / a.group) || !make_page_map(&mk, a.c, a.c.k) || !make_page_map(&mv, a.c, a.c.v))
        return cudaErrorInvalidValue;
    kernel<<<(uint32_t)sms, P::kThreads, P::kTotal, s>>>(a, mq, mk, mv);
    return cudaGetLastError();
}

template <int F, bool QBF>
cudaError_t by_shape(const ChunkArgs &a, int sms, cudaStream_t s) {
    // The row tiles of an item share its K and V loads and keep the softmax warps busy: as many as possible, while
    // that makes a sixth as many items as there are SMs.  (Splitting keys is no dearer than splitting rows: 500 rows
    // after 8000, 32 / 8 heads of 128, 79 us, and 102 with half as many items as SMs; two of 1000 after 4000 to 8000, 14 / 2 heads
    // of 64 in 8 bits, 104 and 149.  An eighth, or a sixteenth: 700 rows of 64 dimensions without earlier tokens 28.6 us for 23.8.)
    const uint32_t per = kRows / a.group;
    auto items = [&](uint32_t tiles) { return a.c.heads * ((a.q_tokens + tiles * per - 1) / (tiles * per) + a.batch - 1); };
    uint32_t tiles = a.c.dim == 64 ? 4 : 2;
    while (tiles > 1 && 6 * items(tiles) <= (uint64_t)sms) tiles /= 2;
    if (a.c.dim == 128) return run<128, 2, F, QBF>(a, sms, tiles, s);
    return run<64, 4, F, QBF>(a, sms, tiles, s);
}

}  // namespace

// (The counters, one for every softmax warp of every CTA, of any device with up to 1024 SMs are within the bytes that
// start from zero.)
size_t paged_prompt_workspace(uint32_t dim) {
    int dev = 0;
    const int sms = cudaGetDevice(&dev) == cudaSuccess ? sm_count(dev) : 0;
    if (!sms) return 0;
    const uint32_t tiles = dim == 64 ? 4 : 2;
    return BGTQ_WORKSPACE_ZEROED + 2ull * sms * tiles * kRows * (dim + 2) * 4;
}

cudaError_t launch_paged_prompt(const ChunkArgs &a, cudaStream_t s) {
    if (!encoder()) return cudaErrorNotSupported;
    int dev = 0;
    const cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const int sms = sm_count(dev);
    if (!sms) return cudaErrorInvalidDevice;
    const bool bf = a.dtype == BGTQ_BF16;
    switch (a.c.format) {
        case BGTQ_PAGES_F16: return by_shape<F_F16, false>(a, sms, s);
        case BGTQ_PAGES_BF16: return by_shape<F_BF16, true>(a, sms, s);
        case BGTQ_PAGES_INT8: return bf ? by_shape<F_INT8, true>(a, sms, s) : by_shape<F_INT8, false>(a, sms, s);
        default: return bf ? by_shape<F_INT4, true>(a, sms, s) : by_shape<F_INT4, false>(a, sms, s);
    }
}

}  // namespace bgtq
