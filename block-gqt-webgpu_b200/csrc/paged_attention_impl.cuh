// Attention of one new token per request, or of a few, over the pages of a cache:
//     out = sum_t softmax_t(scale q.k_t) v_t  over the request's first `length` tokens;
// of chunks (C) row i of n sees those up to its position, length - n + i, with a window the last and the first few of them.
// Chunks are the same with (row, query head) pairs for query heads: a block of 8 or 16 of them shares its units, which have
// a gap where no row's window reaches, and what a unit's edge hides from some of its columns is masked, a value that is
// not finite there taken out of the product and added for the columns that see it.  (64 requests of one row, a window of 2048, 14 / 2
// heads of 64: 25 us; the same tokens without a window 24, with the code for one token alone 22.  All of 4000 tokens, 8 requests take 13
// us, 32 17, 64 23, 128 36, 256 58: 11 us of start, pages' way and join, and then 0.18 a request, 0.16 of which is memory.)
//
// What bounds it is the one pass over K and V: 2 row_bytes a token and KV head, against 2 D
// multiply-adds for each query head, so the work is laid out for the memory system.  128 requests
// of 16K to 32K tokens, 9 / 3 heads of 64 in 16 bits: 345 us, 6.7 TB/s, a little above a plain
// copy's rate; in 8 bits 232 us, 5.1 TB/s, in 4 bits 248 us, 2.6 TB/s, where turning codes into
// operands costs as many instructions for half the bytes (they issue in 57 and 63 % of all cycles, the
// integer pipe is busy in 51 and 55 %).  Few tokens are bound by latencies instead (the deal, the first pages' way through
// the table, the join), about 10 us: one request of 4096 tokens 10.3 us, 48 of 1 to 8191, 32 / 8
// heads of 128, 32 us (3.1 TB/s), eight of 20K to 32K, 14 / 2 heads of 64 in 4 bits, 21 us.
//   * The (request, KV head, block of query heads) pairs are cut into units of kTokens tokens,
//     and the units, in order, are dealt to the CTAs in equal ranges, whatever the lengths
//     are: a range covers the end of one pair, whole pairs, and the start of another.  The
//     deal is computed on the device from the lengths, so a recorded launch stays balanced
//     while the requests grow.  A pair that lies in one range is written at once; parts of a
//     pair go to the workspace and the CTA that finishes last joins them, in order.  Of short
//     requests a warp takes a whole pair, and the four warps' pairs are dealt as one.
//   * A warp takes every fourth unit of its CTA's range, through a ring of its own in shared
//     memory filled by cp.async (rows past the length arrive as zeros), which runs ahead
//     across pair boundaries.  Nothing but the join of four warps at the end of a pair
//     synchronises the CTA.
//   * Products run on the tensor cores with the tokens as the long side: S^T = K Q^T (16
//     tokens x 8 heads), O^T = V^T P^T (16 dimensions x 8 heads), so the 8 columns hold the
//     query heads of a KV head and no row is padding.  8- and 4-bit codes become FP16
//     integers in registers (exactly); the dimensions and tokens inside a product are taken
//     in the order in which the loaded words hold them.
//   * Softmax statistics and outputs are FP32.  The probabilities are rounded to 16 bits for
//     the second product: FP16 (times 2^12, which keeps 2^-26 of the largest normal) or, over
//     BF16 pages, BF16.
//   * 8-bit pages: a key's scale multiplies its logit, a value's scale its probability before
//     the rounding.  4-bit pages: the logit is the sum of scale x partial product over groups
//     of 32 dimensions; the values are multiplied in registers by their scales over their
//     token's power of two (code x scale has 11 bits, so FP16 holds it exactly), and that
//     power multiplies the probability.  FP16's exponent range does not hold such products
//     of any scale: they are taken relative to the largest of each head, so that a value of
//     any size whose weight is next to nothing leaves the others as they are.  What is
//     rounded away is 2^-35 of the largest.  Queries are taken relative to a power of two
//     of their row's largest; FP16 drops 2^-38 of it.  (128 requests of 16K to 32K
//     tokens, 9 / 3 heads of 64 in 8 bits, 232 us for 225 with one power for all heads.)
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "serving.h"

namespace bgtq {
namespace {

constexpr float kLn2 = 0.6931471805599453f;
constexpr uint32_t kWarps = 4, kThreads = 32 * kWarps;
enum { F_F16, F_BF16, F_INT8, F_INT4 };
// Over 8- and 4-bit pages (powers of two, as logarithms): value scales below kLeast count as that; how far a unit's largest
// contribution may pass the largest before it, 10 + kRoom + 1 being what FP16 holds; how far apart the heads of a
// KV head may be in contribution over probability.
constexpr float kLeast = -100.0f, kRoom = 4.0f, kApart = 100.0f;
constexpr float kSmall = 1.0f / 65536.0f;  // of 4-bit pages' key scales, given back with the query's power

template <int F, int D, int NT>
struct Shape {
    static constexpr int kRow = F == F_INT4 ? D / 2 : F == F_INT8 ? D : 2 * D;  // bytes
    static constexpr int kGroups = F == F_INT4 ? D / 32 : F == F_INT8 ? 1 : 0;
    // Tokens of a unit: what three stages for each of eight warps of an SM hold, 64 at most.  (128 requests of 16K to 32K
    // tokens, 9 / 3 heads of 64: in 8 bits 32 tokens 299 us, 64 240; in 4 bits 32 tokens 311 us, 64 253, 128 289.)
    static constexpr int kTokens = kRow >= 256 ? 16 : kRow >= 128 ? 32 : 64;
    static constexpr int kStages = 3;
    static constexpr int kPart = kTokens * kRow;                 // K or V rows of a unit
    static constexpr int kScale = kTokens * kGroups * 2;         // K or V scales of a unit
    static constexpr int kStage = 2 * (kPart + kScale);
    static constexpr int kRing = kStages * kStage;
    static constexpr int kHeads = 8 * NT;
    static constexpr int kPartFloats = kHeads * (D + 2);         // a part in the workspace: O, m, l
    static constexpr int kSmem = kWarps * kRing + kWarps * kHeads * 8 + 128;
    static_assert(kStage >= kHeads * D * 4, "a warp's outputs are joined in the ring slot that it read last");
};

// 16-byte chunk `c` of row r in a ring slot.  Rows share 128-byte lines; the chunks of a line
// are permuted so that ldmatrix (8 rows, one chunk), the key loads (8 rows x 4 threads) and
// the value loads (4 rows two apart x 8 threads) all spread over the 32 banks.
template <int R>
__device__ __forceinline__ uint32_t place(uint32_t r, uint32_t c) {
    if constexpr (R >= 128) {
        const uint32_t x = ((r ^ (r >> 1)) & 1u) << 2 | (r >> 2 & 1u) << 1 | (r >> 1 & 1u);
        return r * R + ((c ^ x) << 4);
    } else {
        constexpr uint32_t per = 128 / R, chunks = R / 16;
        const uint32_t line = r / per, u = (r % per) * chunks + c;
        const uint32_t x = R == 64 ? ((line & 3u) ^ (line & 3u) << 1) : (line & 1u) * 3u;
        return line * 128 + ((u ^ (x & 7u)) << 4);
    }
}

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}
__device__ __forceinline__ uint32_t turn(uint32_t x) {  // an 8 x 8 matrix of 16-bit values, transposed
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
template <bool BF>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (BF)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};" : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};" : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float least(float x) {  // of x and 2^127, NaN if x is
    float y;
    asm("min.NaN.f32 %0, %1, 0f7F000000;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float from_bf16(uint32_t bits) { return __uint_as_float(bits << 16); }
__device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b) {
    const __half2 r = __hsub2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&r);
}
__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
    const __half2 r = __hmul2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&r);
}
// Bytes as FP16: 1024 + byte is 0x6400 | byte.  Signed codes come in with their sign bit
// flipped, so 1024 + 128 goes off again.
__device__ __forceinline__ uint32_t bytes_to_half(uint32_t w, uint32_t sel) {
    return sub2(__byte_perm(w, 0x64646464u, sel), 0x64806480u);
}
// Nibbles 0 of both halves (1024 + code + 8), and nibbles 1 of both halves (64 + code + 8).
__device__ __forceinline__ uint32_t nibble0(uint32_t w) { return sub2((w & 0x000f000fu) | 0x64006400u, 0x64086408u); }
__device__ __forceinline__ uint32_t nibble1(uint32_t w) { return sub2((w & 0x00f000f0u) | 0x54005400u, 0x54805480u); }

// One item of the deal: a pair (request, KV head, block of query heads), which may be cut between
// CTAs, or, of a short request, four pairs side by side, a whole one for each warp.
struct Cursor {
    uint32_t b, item, items, units, weight;
    int32_t len;
    // chunks: the request's first query row and rows, its blocks of columns and its pairs, the units of its first tokens
    // and of the gap between them and its window
    int32_t row0, n;
    uint32_t blocks, pairs, sunk, gap;
    bool quad;
    uint64_t base;     // where the item begins in the deal
    uint32_t at, end;  // the units of it that are this CTA's (quads: all or none)
};
// What an item costs beside its units, in units: its queries, the join of the warps, its output.
// (None: 48 requests of 1 to 8191 tokens, 32 / 8 heads of 128, 44 us for 33.)
constexpr uint32_t kItemCost = 10;

// (Two CTAs an SM for their registers; three of 168, with units of 32 tokens, take 269 us for 240 in 8 bits and 296 for
// 257 in 4, of the requests above.)
template <int F, int D, int NT, bool C>
__global__ void __launch_bounds__(kThreads, 2) attend_kernel(const std::conditional_t<C, ChunkArgs, PagedAttendArgs> a) {
    using S = Shape<F, D, NT>;
    constexpr bool BF = F == F_BF16;
    constexpr int T = S::kTokens, C16 = T / 16, KS = D / 16;
    extern __shared__ __align__(128) unsigned char smem[];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, row4 = lane >> 2, col4 = lane & 3u;
    unsigned char *ring = smem + warp * S::kRing;
    const uint32_t ring_at = smem_addr(ring);
    float2 *sums = reinterpret_cast<float2 *>(smem + kWarps * S::kRing);  // [warp][head]: maximum, sum
    uint32_t *flags = reinterpret_cast<uint32_t *>(sums + kWarps * S::kHeads);
    const uint32_t one_blocks = (a.group + S::kHeads - 1) / S::kHeads, one_pairs = a.c.heads * one_blocks;
    auto by_16 = [&]() {  // query rows are 16-byte aligned
        if constexpr (C) return true;
        else return a.q_even != 0;
    };
    auto blocks_of = [&](const Cursor &c) { return C ? c.blocks : one_blocks; };
    auto pairs_of = [&](const Cursor &c) { return C ? c.pairs : one_pairs; };
    const uint32_t shift = a.c.page_shift, H = a.c.heads;

    auto length = [&](uint32_t b) -> int32_t {
        const int32_t n = __ldg(a.lengths + b);
        return n < 0 ? 0 : (int32_t)min((uint32_t)n, a.width << shift);
    };
    // ---- the deal ----
    // (every warp for itself: lanes over the requests, sums by shuffles, no barrier)
    auto warp_sum = [](uint64_t x) {
#pragma unroll
        for (int w = 16; w; w >>= 1) x += __shfl_xor_sync(0xffffffffu, x, w);
        return x;
    };
    // request b of the deal, as far as the number of its units
    auto request = [&](Cursor &c, uint32_t b) {
        c.len = length(b);
        if constexpr (C) {
            c.row0 = a.starts ? __ldg(a.starts + b) : (int32_t)b;
            c.n = a.starts ? __ldg(a.starts + b + 1) - c.row0 : 1;
            if (c.row0 < 0 || c.n < 0 || (uint64_t)((int64_t)c.row0 + c.n) > a.q_tokens) c.n = -1;
            c.blocks = (uint32_t)(max(c.n, 0) * (int32_t)a.group + S::kHeads - 1) / S::kHeads;
            c.pairs = a.c.heads * c.blocks;
            // tokens from `lo` on are in the window of the first row, and so of none before it
            const int32_t lo = a.window ? (int32_t)max((int64_t)0, (int64_t)c.len - c.n - a.window + 1) : 0;
            c.sunk = min((min(a.sinks, (uint32_t)lo) + T - 1) / T, (uint32_t)lo / T);
            c.gap = lo / T - c.sunk;
            c.units = (uint32_t)(c.len + T - 1) / T - c.gap;
        } else {
            c.units = (uint32_t)(c.len + T - 1) / T;
        }
    };
    // the unit's place among the units of all of the request's tokens
    auto place_of = [](const Cursor &c, uint32_t unit) { return C && unit >= c.sunk ? unit + c.gap : unit; };
    uint64_t all_units = 0;
    bool past_table = false;
#pragma unroll 4
    for (uint32_t b = lane; b < a.batch; b += 32) {
        Cursor c;
        request(c, b);
        past_table |= c.len != __ldg(a.lengths + b) || (C && c.n < 0);
        all_units += C ? (uint64_t)c.units * c.pairs : (uint64_t)c.units;
    }
    if (past_table && blockIdx.x == 0 && warp == 0) atomicOr(a.status, kStatusBadExtent);
    all_units = warp_sum(all_units) * (C ? 1u : one_pairs);
    // A request goes by quads if a quad of its pairs is within a CTA's share of the units, or if
    // it has two units or less, where a pair spread over four warps gains nothing.  (256 requests, 32 / 8 heads of
    // 128 in 8 bits: 30 to 60 tokens 18 us, 34 without quads; 100 to 400 tokens 48 us, 55 with those of two units only.)
    const uint32_t quad_units = (uint32_t)max((uint64_t)2, min(all_units / gridDim.x / 4, (uint64_t)1 << 30));
    auto plan = [&](Cursor &c) {  // of what `request` found
        const uint32_t pairs = pairs_of(c);
        c.quad = pairs > 1 && c.units <= quad_units;
        c.items = c.len == 0 ? 0 : c.quad ? (pairs + 3) / 4 : pairs;
        c.weight = (c.quad ? 4 * c.units : c.units) + kItemCost;
    };
    uint64_t total = 0, all_items = 0;
#pragma unroll 4
    for (uint32_t b = lane; b < a.batch; b += 32) {
        Cursor c;
        request(c, b);
        plan(c);
        all_items += c.items;
        total += (uint64_t)c.items * c.weight;
    }
    total = warp_sum(total);
    all_items = warp_sum(all_items);
    // a request without tokens: zeros
    for (uint32_t b = blockIdx.x; b < a.batch; b += gridDim.x) {
        if (length(b) != 0) continue;
        uint64_t row = b;
        uint32_t heads = a.q_heads;
        if constexpr (C) {
            Cursor c;
            request(c, b);
            row = (uint64_t)max(c.row0, 0);
            heads *= (uint32_t)max(c.n, 0);
        }
        uint16_t *o = static_cast<uint16_t *>(a.out) + row * a.q_heads * D;
        for (uint64_t i = threadIdx.x; i < (uint64_t)heads * D; i += kThreads) o[i] = 0;
        if (a.lse)
            for (uint32_t i = threadIdx.x; i < heads; i += kThreads) a.lse[row * a.q_heads + i] = -INFINITY;
    }
    // as many CTAs as there are items, or rounds of four units
    const uint64_t most = max(all_items, all_units / kWarps);
    const uint32_t ctas = (uint32_t)min(most, (uint64_t)gridDim.x);
    if (blockIdx.x >= ctas) return;
    // equal ranges: the first `over` CTAs have one place more
    const uint64_t each = total / ctas, over = total - each * ctas;
    const uint64_t first = blockIdx.x * each + min((uint64_t)blockIdx.x, over);
    const uint64_t last = first + each + (blockIdx.x < over ? 1 : 0);
    auto owner = [&](uint64_t place) {
        const uint64_t head = over * (each + 1);
        return (uint32_t)(place < head ? place / (each + 1) : over + (place - head) / each);
    };
    // this CTA's share of the item: a unit, or a quad, belongs to the CTA whose range holds its place
    auto take = [&](Cursor &c) {
        if (c.quad) {
            c.at = 0;
            c.end = c.base >= first && c.base < last ? c.units : 0;
        } else {
            const uint64_t from = c.base + kItemCost;
            c.at = first <= from ? 0u : (uint32_t)min((uint64_t)c.units, first - from);
            c.end = last <= from ? 0u : (uint32_t)min((uint64_t)c.units, last - from);
        }
    };
    // the next item with units of this CTA's; false past the range's end
    auto next_item = [&](Cursor &c) {
        do {
            c.base += c.weight;
            if (c.base >= last) return false;
            if (++c.item == c.items) {
                c.item = 0;
                do {
                    if (++c.b >= a.batch) return false;
                    request(c, c.b);
                } while (c.len == 0 || (C && c.n <= 0));
                plan(c);
            }
            take(c);
        } while (c.at >= c.end);
        return true;
    };
    Cursor cur;
    {
        uint64_t base = 0;
        for (uint32_t b0 = 0;; b0 += 32) {  // ends: first < total
            if (b0 + lane < a.batch) {
                request(cur, b0 + lane);
                plan(cur);
            } else {
                cur.items = 0;
                cur.weight = 0;
            }
            const uint64_t own = (uint64_t)cur.items * cur.weight;
            uint64_t sum = own;
#pragma unroll
            for (int w = 1; w < 32; w <<= 1) {
                const uint64_t o = __shfl_up_sync(0xffffffffu, sum, w);
                if (lane >= (uint32_t)w) sum += o;
            }
            const uint32_t past = __ballot_sync(0xffffffffu, base + sum > first);
            if (past) {
                const uint32_t l = __ffs(past) - 1;
                base += __shfl_sync(0xffffffffu, sum - own, l);
                cur.b = b0 + l;
                break;
            }
            if (b0 + 32 >= a.batch) return;
            base += __shfl_sync(0xffffffffu, sum, 31);
        }
        request(cur, cur.b);
        plan(cur);
        cur.item = (uint32_t)((first - base) / cur.weight);
        cur.base = base + (uint64_t)cur.item * cur.weight;
        take(cur);
        if (cur.at >= cur.end && !next_item(cur)) return;
    }
    // a warp's first unit of an item, its step, and its pair
    auto unit0 = [&](const Cursor &c) { return c.quad ? (c.item * 4 + warp < pairs_of(c) ? 0u : c.end) : c.at + warp; };
    auto step_of = [](const Cursor &c) { return c.quad ? 1u : kWarps; };
    auto pair_of = [&](const Cursor &c) { return c.quad ? c.item * 4 + warp : c.item; };

    // ---- filling the ring ----
    Cursor pre = cur;
    uint32_t pre_unit = unit0(pre);
    bool more = true;
    // Page indices of the warp's next units of the item, `span` to a unit: one load brings a window of them, a
    // second one the window after it while this one is used.
    const uint32_t span_shift = (uint32_t)T > (1u << shift) ? 31 - __clz(T) - shift : 0, span = 1u << span_shift;
    const uint32_t window = 32 >> span_shift;
    int32_t pages_now = -1, pages_next = -1;
    uint32_t used = 0;  // units of this window that are done with
    auto fetch_pages = [&](uint32_t unit) {  // for the units from `unit` on, in the warp's step
        const uint32_t u = unit + (lane >> span_shift) * step_of(pre);
        const uint32_t t = place_of(pre, u) * T + ((lane & (span - 1)) << shift);
        return u < pre.end && t < (uint32_t)pre.len ? __ldg(a.table + (int64_t)pre.b * a.table_stride + (t >> shift)) : -1;
    };
    auto settle = [&](bool fresh) {  // moves `pre` to the warp's next unit, if there is one, and sees to its page indices
        while (more && pre_unit >= pre.end) {
            more = next_item(pre);
            if (!more) break;
            pre_unit = unit0(pre);
            fresh = true;
            // its queries, which are loaded when the ring gets there
            const uint32_t p = pair_of(pre), blocks = blocks_of(pre), h = p % blocks * S::kHeads + lane / 2;
            const bool some = p < pairs_of(pre) && lane / 2 < (uint32_t)S::kHeads && h < (C ? (uint32_t)pre.n : 1u) * a.group;
            if (some) {
                const uint16_t *at = static_cast<const uint16_t *>(a.q) + (lane & 1u) * (D / 2);
                if constexpr (C)
                    at += (int64_t)(pre.row0 + h / a.group) * a.q_token + (int64_t)(p / blocks * a.group + h % a.group) * a.q_head;
                else at += (int64_t)pre.b * a.q_batch + (int64_t)(p / blocks * a.group + h) * a.q_head;
                asm volatile("prefetch.global.L1 [%0];" ::"l"(at));
            }
        }
        if (!more) return;
        if (fresh) {
            used = 0;
            pages_now = fetch_pages(pre_unit);
            pages_next = fetch_pages(pre_unit + window * step_of(pre));
        } else if (++used == window) {
            used = 0;
            pages_now = pages_next;
            pages_next = fetch_pages(pre_unit + window * step_of(pre));
        }
    };
    settle(true);
    auto fill = [&](uint32_t stage) {
        if (more) {
            const uint32_t t0 = place_of(pre, pre_unit) * T, kh = pair_of(pre) / blocks_of(pre);
            const int32_t page = __shfl_sync(0xffffffffu, pages_now, (used << span_shift) + (lane & (span - 1)));
            const bool asked = lane < span && t0 + (lane << shift) < (uint32_t)pre.len;
            // chunks: a page of a unit between the first tokens and the window is absent, whatever the table says of it
            bool hidden = false;
            if constexpr (C) {
                const uint32_t from = t0 + (lane << shift);
                hidden = a.window && from >= a.sinks && (int64_t)from + (1 << shift) <= (int64_t)pre.len - pre.n - a.window + 1;
            }
            const bool missing = asked && (uint32_t)page >= a.c.pages;
            if (__any_sync(0xffffffffu, missing && !hidden) && lane == 0) atomicOr(a.status, kStatusBadSlot);
            const uint32_t bad = __ballot_sync(0xffffffffu, missing || (asked && hidden));
            if (lane == 0) flags[warp * 4 + stage] = bad;
            const uint32_t dst = ring_at + stage * S::kStage;
            const int32_t left = pre.len - (int32_t)t0;
            // the cache row of this KV head with which the lane's page begins (span > 1: rows are counted from there),
            // or of the unit's first token; page 0 stands for one that is not there, of which nothing is copied
            const uint32_t in_page = (1u << shift) - 1;
            const uint64_t begin = ((uint64_t)((uint32_t)page < a.c.pages ? (uint32_t)page : 0u) * H + kh << shift) + (t0 & in_page);
            constexpr uint32_t CH = S::kRow / 16;
#pragma unroll
            for (uint32_t i = 0; i < T * CH / 32; ++i) {
                const uint32_t idx = i * 32 + lane, r = idx / CH, c = idx % CH;
                const uint32_t pi = r >> shift;
                const bool ok = (int32_t)r < left && !(bad >> pi & 1u);
                const uint64_t off = (__shfl_sync(0xffffffffu, begin, pi) + (r & in_page)) * S::kRow + c * 16;
                const uint32_t to = place<S::kRow>(r, c);
                copy16(dst + to, a.c.k + off, ok ? 16u : 0u);
                copy16(dst + S::kPart + to, a.c.v + off, ok ? 16u : 0u);
            }
            if constexpr (S::kGroups != 0) {
                constexpr uint32_t N = S::kScale / 16, PER = 8 / S::kGroups;  // 16-byte chunks, tokens in one
#pragma unroll
                for (uint32_t i = 0; i < (N + 31) / 32; ++i) {
                    const uint32_t idx = i * 32 + lane, r = idx * PER, pi = min(r >> shift, 31u);
                    const bool ok = (int32_t)r < left && !(bad >> pi & 1u);
                    const uint64_t off = (__shfl_sync(0xffffffffu, begin, pi) + (r & in_page)) * S::kGroups;
                    const uint32_t bytes = ok ? min(16u, (uint32_t)(left - (int32_t)r) * S::kGroups * 2u) : 0u;
                    if (N % 32 == 0 || idx < N) {
                        copy16(dst + 2 * S::kPart + idx * 16, a.c.ks + off, bytes);
                        copy16(dst + 2 * S::kPart + S::kScale + idx * 16, a.c.vs + off, bytes);
                    }
                }
            }
            pre_unit += step_of(pre);
            settle(false);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (uint32_t s = 0; s < (uint32_t)S::kStages - 1; ++s) fill(s);

    uint32_t stage = 0;
    for (;;) {
        // ---- an item: this warp's units of its pair ----
        const uint32_t blocks = blocks_of(cur), pairs = pairs_of(cur);
        const uint32_t pair = min(pair_of(cur), pairs - 1), kh = pair / blocks, block = pair % blocks;
        const uint32_t head0 = kh * a.group + (C ? 0 : block * S::kHeads);
        // columns of the block: query heads, of chunks the (row, query head) pairs in this order
        const uint32_t col0 = block * S::kHeads;
        const uint32_t heads = min((uint32_t)S::kHeads, (C ? (uint32_t)cur.n : 1u) * a.group - col0);
        int32_t pos[NT][2];  // chunks: the positions of this thread's columns
        int32_t pos_first = 0, pos_last = 0;
        if constexpr (C) {
            const int32_t start = cur.len - cur.n;
            pos_first = start + (int32_t)(col0 / a.group);
            pos_last = start + (int32_t)((col0 + heads - 1) / a.group);
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t col = n * 8 + 2 * col4 + h;
                    pos[n][h] = col < heads ? start + (int32_t)((col0 + col) / a.group) : cur.len - 1;
                }
        }
        auto sees = [&](int32_t t, int32_t p) {
            if constexpr (C) return t <= p && (!a.window || (uint32_t)(p - t) < a.window || (uint32_t)t < a.sinks);
            else return true;
        };
        uint32_t q[KS][NT][2];
        float qs[NT][2];  // what a logit of this thread's heads is multiplied by
        {
            float x[NT][KS][4];
            float big[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const uint32_t h = n * 8 + row4;
                int64_t at;
                if constexpr (C)
                    at = (int64_t)(cur.row0 + (col0 + h) / a.group) * a.q_token + (int64_t)(head0 + (col0 + h) % a.group) * a.q_head;
                else at = (int64_t)cur.b * a.q_batch + (int64_t)(head0 + h) * a.q_head;
                big[n] = 0.0f;
                uint16_t raw[KS][4];  // slot (s, e): in the order in which the key words hold the dimensions
                if (h >= heads) {
#pragma unroll
                    for (int s = 0; s < KS; ++s) raw[s][0] = raw[s][1] = raw[s][2] = raw[s][3] = 0;
                } else if (by_16()) {
                    const uint16_t *src = static_cast<const uint16_t *>(a.q) + at;
                    if constexpr (F >= F_INT8) {
#pragma unroll
                        for (int j = 0; j < D / 32; ++j) {  // eight dimensions a load
                            const uint4 x = __ldg(reinterpret_cast<const uint4 *>(
                                src + (F == F_INT8 ? 64 * (j / 2) + 16 * col4 + 8 * (j % 2) : 32 * j + 8 * col4)));
                            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                            for (int k = 0; k < 8; ++k) {
                                const uint16_t v = (uint16_t)(w[k / 2] >> 16 * (k & 1));
                                if constexpr (F == F_INT8) raw[2 * j + k / 4][k % 4] = v;
                                else raw[2 * j + k % 4 / 2][k / 4 + 2 * (k & 1)] = v;
                            }
                        }
                    } else {
#pragma unroll
                        for (int s = 0; s < KS; ++s)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const uint32_t x = __ldg(reinterpret_cast<const uint32_t *>(src + 16 * s + 2 * col4 + 8 * e));
                                raw[s][2 * e] = (uint16_t)x;
                                raw[s][2 * e + 1] = (uint16_t)(x >> 16);
                            }
                    }
                } else {
#pragma unroll
                    for (int s = 0; s < KS; ++s)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            int d;
                            if constexpr (F == F_INT8) d = 64 * (s / 4) + 16 * col4 + 4 * (s % 4) + e;
                            else if constexpr (F == F_INT4)
                                d = 32 * (s / 2) + 8 * col4 + 2 * (s % 2) + (e & 1) * 4 + (e >> 1);
                            else d = 16 * s + 2 * col4 + (e & 1) + 8 * (e >> 1);
                            raw[s][e] = static_cast<const uint16_t *>(a.q)[at + d];
                        }
                }
#pragma unroll
                for (int s = 0; s < KS; ++s)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        x[n][s][e] = a.dtype == BGTQ_F16 ? __half2float(__ushort_as_half(raw[s][e])) : from_bf16(raw[s][e]);
                        big[n] = fmaxf(big[n], fabsf(x[n][s][e]));
                    }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float f = 1.0f;
                if constexpr (F >= F_INT8) {
                    // the row's largest value to [2^13, 2^14): what FP16 then drops is 2^-38 of it
                    float m = big[n];
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
                    const int e = (int)(__float_as_uint(m) >> 23) - 127;  // m = 0, tiny: -127; inf, NaN: 128
                    const int up = min(max(13 - e, -126), 126);
                    f = __uint_as_float((uint32_t)(127 - up) << 23);
                    const float g = __uint_as_float((uint32_t)(127 + up) << 23);
#pragma unroll
                    for (int s = 0; s < KS; ++s)
#pragma unroll
                        for (int k = 0; k < 4; ++k) x[n][s][k] *= g;
                }
                f *= F == F_INT4 ? a.scale * (1.0f / kSmall) : a.scale;
                qs[n][0] = __shfl_sync(0xffffffffu, f, col4 * 8);
                qs[n][1] = __shfl_sync(0xffffffffu, f, col4 * 8 + 4);
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    q[s][n][0] = pack<BF>(x[n][s][0], x[n][s][1]);
                    q[s][n][1] = pack<BF>(x[n][s][2], x[n][s][3]);
                }
            }
        }
        float o[KS][NT][4] = {};
        float m[NT][2], l[NT][2] = {};
#pragma unroll
        for (int n = 0; n < NT; ++n) m[n][0] = m[n][1] = -INFINITY;
        // Over 8- and 4-bit pages exponentials and sums are taken relative to 2^ref, outputs to 2^(ref + common); that is
        // each head's largest contribution (exp(logit) x value scale) up to the last unit that passed it by kRoom.
        float ref[NT][2], peak[NT][2], common = kLeast;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) ref[n][h] = F >= F_INT8 ? -3.4e38f : 0.0f, peak[n][h] = -INFINITY;

        for (uint32_t unit = unit0(cur); unit < cur.end; unit += step_of(cur)) {
            asm volatile("cp.async.wait_group %0;" ::"n"(S::kStages - 2) : "memory");
            __syncwarp();
            const unsigned char *buf = ring + stage * S::kStage;
            const uint32_t buf_at = ring_at + stage * S::kStage;
            uint16_t *ksc = reinterpret_cast<uint16_t *>(ring + stage * S::kStage + 2 * S::kPart);
            uint16_t *vsc = ksc + S::kScale / 2;
            const uint32_t bad = flags[warp * 4 + stage];
            const int32_t t0 = (int32_t)(place_of(cur, unit) * T), left = cur.len - t0;  // left: tokens of the unit that exist
            // chunks: whether there are tokens that some columns of the block see and others do not
            bool edge = false;
            if constexpr (C)
                edge = t0 + T - 1 > pos_first || (a.window && pos_last - t0 >= (int32_t)a.window && (uint32_t)(t0 + T) > a.sinks);
            // ---- S^T = K Q^T ----
            float s[C16][NT][4];
#pragma unroll
            for (int c = 0; c < C16; ++c) {
#pragma unroll
                for (int n = 0; n < NT; ++n) s[c][n][0] = s[c][n][1] = s[c][n][2] = s[c][n][3] = 0.0f;
                const uint32_t r0 = 16 * c + row4;
                if constexpr (F <= F_BF16) {
#pragma unroll
                    for (int k = 0; k < KS; ++k) {
                        uint32_t f[4];
                        ldsm4(f, buf_at + place<S::kRow>(16 * c + (lane & 15u), 2 * k + (lane >> 4)));
#pragma unroll
                        for (int n = 0; n < NT; ++n) mma<BF>(s[c][n], f, q[k][n][0], q[k][n][1]);
                    }
                } else if constexpr (F == F_INT8) {
#pragma unroll
                    for (int j = 0; j < D / 64; ++j) {
                        uint4 lo = *reinterpret_cast<const uint4 *>(buf + place<S::kRow>(r0, 4 * j + col4));
                        uint4 hi = *reinterpret_cast<const uint4 *>(buf + place<S::kRow>(r0 + 8, 4 * j + col4));
                        const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint32_t x = wl[i] ^ 0x80808080u, y = wh[i] ^ 0x80808080u;
                            const uint32_t f[4] = {bytes_to_half(x, 0x4140), bytes_to_half(y, 0x4140),
                                                   bytes_to_half(x, 0x4342), bytes_to_half(y, 0x4342)};
#pragma unroll
                            for (int n = 0; n < NT; ++n) mma<false>(s[c][n], f, q[4 * j + i][n][0], q[4 * j + i][n][1]);
                        }
                    }
                    const float k0 = from_bf16(ksc[r0]), k1 = from_bf16(ksc[r0 + 8]);
                    // (by the query's power first: a product of up to 2^28 with a large key scale may pass FP32)
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        s[c][n][0] *= k0 * qs[n][0];
                        s[c][n][1] *= k0 * qs[n][1];
                        s[c][n][2] *= k1 * qs[n][0];
                        s[c][n][3] *= k1 * qs[n][1];
                    }
                } else {
#pragma unroll
                    for (int g = 0; g < D / 32; ++g) {
                        uint32_t x = *reinterpret_cast<const uint32_t *>(buf + place<S::kRow>(r0, g) + 4 * col4);
                        uint32_t y = *reinterpret_cast<const uint32_t *>(buf + place<S::kRow>(r0 + 8, g) + 4 * col4);
                        float p[NT][4] = {};
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const uint32_t f[4] = {nibble0(x), nibble0(y), nibble1(x), nibble1(y)};
#pragma unroll
                            for (int n = 0; n < NT; ++n) mma<false>(p[n], f, q[2 * g + i][n][0], q[2 * g + i][n][1]);
                            x >>= 8;
                            y >>= 8;
                        }
                        // (products of up to 2^22 with a large key scale may pass FP32)
                        float k0, k1;
                        if constexpr (D == 64) {  // both groups' scales of a token by one load (252 us for 257; at 128 it costs 1 %)
                            const uint32_t kx = reinterpret_cast<const uint32_t *>(ksc)[r0];
                            const uint32_t ky = reinterpret_cast<const uint32_t *>(ksc)[r0 + 8];
                            k0 = g ? __uint_as_float(kx & 0xffff0000u) : from_bf16(kx);
                            k1 = g ? __uint_as_float(ky & 0xffff0000u) : from_bf16(ky);
                        } else {
                            k0 = from_bf16(ksc[r0 * S::kGroups + g]);
                            k1 = from_bf16(ksc[(r0 + 8) * S::kGroups + g]);
                        }
                        k0 *= kSmall;
                        k1 *= kSmall;
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            s[c][n][0] = fmaf(p[n][0], k0, s[c][n][0]);
                            s[c][n][1] = fmaf(p[n][1], k0, s[c][n][1]);
                            s[c][n][2] = fmaf(p[n][2], k1, s[c][n][2]);
                            s[c][n][3] = fmaf(p[n][3], k1, s[c][n][3]);
                        }
                    }
                }
            }
            // ---- logits in log2 units, masked; the running maximum ----
            float top[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) top[n][0] = top[n][1] = -INFINITY;
#pragma unroll
            for (int c = 0; c < C16; ++c)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int32_t t = 16 * c + row4 + 8 * e;
                    const bool in = t < left && !(bad && bad >> (t >> shift) & 1u);
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            float &x = s[c][n][2 * e + h];
                            x = in && (!edge || sees(t0 + t, pos[n][h])) ? (F == F_INT8 ? x : x * qs[n][h]) : -INFINITY;
                            top[n][h] = fmaxf(top[n][h], x);
                        }
                }
            // ---- chunks: values that are infinite or NaN and that not every column sees ----
            // (times the zero probability of a column that does not see one they would be a NaN.  Taken out of the unit, and
            // added to the columns that see them.)  Over 8- and 4-bit pages that is a row, or a group, of a NaN scale.
            uint64_t broken = 0;  // tokens with a NaN scale over this thread's dimensions
            bool some_broken = false;
            if constexpr (C) {
                if (edge) {
                    uint32_t found = 0;
                    if constexpr (F >= F_INT8) {
                        for (uint32_t i = lane; i < (uint32_t)T * S::kGroups; i += 32) found |= (vsc[i] & 0x7f80u) == 0x7f80u;
                    } else {
                        constexpr uint32_t E = BF ? 0x7f80u : 0x7c00u, kCarry = (0x8000u - E) | (0x8000u - E) << 16;
                        const uint4 *v = reinterpret_cast<const uint4 *>(buf + S::kPart);
                        for (uint32_t i = lane; i < (uint32_t)S::kPart / 16; i += 32) {  // an exponent of ones carries into the sign's place
                            const uint4 x = v[i];
                            found |= ((x.x & 0x7fff7fffu) + kCarry | (x.y & 0x7fff7fffu) + kCarry | (x.z & 0x7fff7fffu) + kCarry |
                                      (x.w & 0x7fff7fffu) + kCarry) & 0x80008000u;
                        }
                    }
                    some_broken = __any_sync(0xffffffffu, found);
                    if constexpr (F >= F_INT8) {
                        if (some_broken) {
                            const uint32_t g = S::kGroups == 1 ? 0 : row4 * (D / 8) / 32;
                            for (uint32_t t = 0; t < (uint32_t)T; ++t)
                                if ((vsc[t * S::kGroups + g] & 0x7f80u) == 0x7f80u) broken |= 1ull << t;
                            __syncwarp();
                            for (uint32_t i = lane; i < (uint32_t)T * S::kGroups; i += 32)
                                if ((vsc[i] & 0x7f80u) == 0x7f80u) vsc[i] = 0;
                            __syncwarp();
                        }
                    }
                }
            }
            // ---- value scales: the exponent of the unit's largest; in 4 bits, of each token's largest ----
            float *tok = reinterpret_cast<float *>(ksc);  // 4 bits: powers of two of the tokens
            float e_unit = kLeast;
            if constexpr (F == F_INT8) {
                uint32_t big = 0;
#pragma unroll
                for (uint32_t i = 0; i < (T + 31) / 32; ++i) {
                    const uint32_t x = T % 32 == 0 || lane < T ? vsc[i * 32 + lane] : 0;
                    big = max(big, x < 0x7f80u ? x : 0u);
                }
                e_unit = (float)((int)(__reduce_max_sync(0xffffffffu, big) >> 7) - 127);
            }
            if constexpr (F == F_INT4) {
                // a token's scales become FP16 over its power of two (times 2^10: code x scale has 11 bits, so FP16 holds
                // it exactly, of any scale down to 2^-24 of the token's largest), which goes to its probability
                static_assert(T % 32 == 0 && T * 4 <= S::kScale, "the powers lie where the key scales were");
                constexpr int W = S::kGroups / 2;
                __syncwarp();
                uint32_t all = 0;
#pragma unroll
                for (uint32_t i = 0; i < T / 32; ++i) {
                    uint32_t *at = reinterpret_cast<uint32_t *>(vsc) + (i * 32 + lane) * W, w[W], big = 0;
#pragma unroll
                    for (int k = 0; k < W; ++k) {
                        w[k] = at[k];
                        const uint32_t a0 = w[k] & 0xffffu, a1 = w[k] >> 16;
                        big = max(big, max(a0 < 0x7f80u ? a0 : 0u, a1 < 0x7f80u ? a1 : 0u));
                    }
                    const uint32_t e = max(big >> 7, (uint32_t)(127 + (int)kLeast));
                    const float f = __uint_as_float((264 - e) << 23);  // 2^(10 - exponent)
#pragma unroll
                    for (int k = 0; k < W; ++k) at[k] = pack<false>(from_bf16(w[k] & 0xffffu) * f, from_bf16(w[k] >> 16) * f);
                    tok[i * 32 + lane] = __uint_as_float(e << 23);
                    all = max(all, e);
                }
                e_unit = (float)((int)__reduce_max_sync(0xffffffffu, all) - 127);
                __syncwarp();
            }
            bool moved = false;
            float alpha[NT][2], beta[NT][2];  // 2^alpha: what sums are multiplied by, 2^beta: outputs
            const float above = fmaxf(e_unit, common - (kApart + 5.0f)) - kRoom - common;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float x = top[n][h];
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                    const float now = fmaxf(m[n][h], x);
                    if constexpr (F >= F_INT8) moved |= x + above > ref[n][h];
                    else {
                        moved |= now > m[n][h];
                        alpha[n][h] = beta[n][h] = now == -INFINITY ? 0.0f : m[n][h] - now;
                        ref[n][h] = now == -INFINITY ? 0.0f : now;
                    }
                    m[n][h] = now;
                }
            if (__any_sync(0xffffffffu, moved)) {
                if constexpr (F >= F_INT8) {
                    // the largest contributions, by every token's logit and exponent
#pragma unroll
                    for (int c = 0; c < C16; ++c)
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const uint32_t t = 16 * c + row4 + 8 * k;
                            uint32_t b;
                            if constexpr (F == F_INT8) b = vsc[t] < 0x7f80u ? vsc[t] >> 7 : 0u;
                            else b = __float_as_uint(tok[t]) >> 23;
#pragma unroll
                            for (int n = 0; n < NT; ++n)
#pragma unroll
                                for (int h = 0; h < 2; ++h) peak[n][h] = fmaxf(peak[n][h], s[c][n][2 * k + h] + fmaxf((float)((int)b - 127), kLeast));
                        }
                    const float before = common;
                    common = kLeast;
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            peak[n][h] = fmaxf(peak[n][h], __shfl_xor_sync(0xffffffffu, peak[n][h], 4));
                            peak[n][h] = fmaxf(peak[n][h], __shfl_xor_sync(0xffffffffu, peak[n][h], 8));
                            peak[n][h] = fmaxf(peak[n][h], __shfl_xor_sync(0xffffffffu, peak[n][h], 16));
                            // (no token yet: NaN, passed over; a column without a head has equal weights for all tokens)
                            if (n * 8 + 2 * col4 + h < heads) common = fmaxf(common, ceilf(peak[n][h] - m[n][h]));
                        }
                    common = fmaxf(common, __shfl_xor_sync(0xffffffffu, common, 1));
                    common = fmaxf(common, __shfl_xor_sync(0xffffffffu, common, 2));
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float now = fmaxf(fmaxf(peak[n][h] - common, m[n][h] - kApart), -3.4e38f);
                            alpha[n][h] = ref[n][h] - now;
                            beta[n][h] = alpha[n][h] + (before - common);
                            ref[n][h] = now;
                        }
                }
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float f = ex2(alpha[n][h]), g = F >= F_INT8 ? ex2(beta[n][h]) : f;
                        l[n][h] *= f;
#pragma unroll
                        for (int i = 0; i < KS; ++i) {
                            o[i][n][h] *= g;
                            o[i][n][2 + h] *= g;
                        }
                    }
            }
            if constexpr (C) {
                if (some_broken) {
                    auto add = [&](int i, int e, uint32_t t, float x) {
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int h = 0; h < 2; ++h)
                                if ((int32_t)t < left && sees(t0 + (int32_t)t, pos[n][h])) o[i][n][2 * e + h] += x;
                    };
                    if constexpr (F >= F_INT8) {
                        for (; broken; broken &= broken - 1) {
                            const uint32_t t = __ffsll((long long)broken) - 1;
#pragma unroll
                            for (int i = 0; i < KS; ++i)
#pragma unroll
                                for (int e = 0; e < 2; ++e) add(i, e, t, __uint_as_float(0x7fc00000u));
                        }
                    } else {
                        constexpr uint32_t E = BF ? 0x7f80u : 0x7c00u;
                        auto value = [&](uint32_t t, uint32_t d) {
                            return reinterpret_cast<uint16_t *>(ring + stage * S::kStage + S::kPart + place<S::kRow>(t, d / 8)) + d % 8;
                        };
#pragma unroll 1
                        for (uint32_t t = 0; t < (uint32_t)T; ++t)
#pragma unroll
                            for (int i = 0; i < KS; ++i)
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    const uint16_t x = *value(t, 16 * i + row4 + 8 * e);
                                    if ((x & E) == E) add(i, e, t, BF ? from_bf16(x) : __half2float(__ushort_as_half(x)));
                                }
                        __syncwarp();
                        for (uint32_t i = lane; i < (uint32_t)(T * D); i += 32) {
                            uint16_t *x = value(i / D, i % D);
                            if ((*x & E) == E) *x = 0;
                        }
                        __syncwarp();
                    }
                }
            }
            const float vmul = F == F_BF16 ? 1.0f : F == F_F16 ? 4096.0f : __uint_as_float((uint32_t)(137 - (int)common) << 23);
            // ---- probabilities, O^T += V^T P^T ----
#pragma unroll
            for (int c = 0; c < C16; ++c) {
                uint32_t p[NT][2];
                float w0 = vmul, w1 = vmul;
                // (at most 2^127: what a token of more weighs is below 2^-111, and zero times infinity is not zero)
                if constexpr (F == F_INT8) w0 = least(from_bf16(vsc[16 * c + row4]) * vmul), w1 = least(from_bf16(vsc[16 * c + row4 + 8]) * vmul);
                if constexpr (F == F_INT4) w0 = least(tok[16 * c + row4] * vmul), w1 = least(tok[16 * c + row4 + 8] * vmul);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const float e0 = ex2(s[c][n][0] - ref[n][0]), e1 = ex2(s[c][n][1] - ref[n][1]);
                    const float e2 = ex2(s[c][n][2] - ref[n][0]), e3 = ex2(s[c][n][3] - ref[n][1]);
                    l[n][0] += e0 + e2;
                    l[n][1] += e1 + e3;
                    p[n][0] = turn(pack<BF>(e0 * w0, e1 * w0));
                    p[n][1] = turn(pack<BF>(e2 * w1, e3 * w1));
                }
                if constexpr (F <= F_BF16) {
#pragma unroll
                    for (int i = 0; i < KS; ++i) {
                        uint32_t f[4];
                        ldsm4_t(f, buf_at + S::kPart + place<S::kRow>(16 * c + (lane & 7u) + (lane >> 4) * 8, 2 * i + (lane >> 3 & 1u)));
#pragma unroll
                        for (int n = 0; n < NT; ++n) mma<BF>(o[i][n], f, p[n][0], p[n][1]);
                    }
                } else {
                    // this thread's words: tokens 2c, 2c + 1, 2c + 8, 2c + 9, dimensions D/8 * row4 ..
                    constexpr int W = F == F_INT8 ? D / 32 : D / 64;  // 32-bit words of D / 8 dimensions
                    uint32_t w[4][W];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t r = 16 * c + 2 * col4 + (e & 1) + 8 * (e >> 1), byte = row4 * W * 4;
                        const unsigned char *at = buf + S::kPart + place<S::kRow>(r, byte >> 4) + (byte & 15u);
                        if constexpr (W == 4) {
                            const uint4 x = *reinterpret_cast<const uint4 *>(at);
                            w[e][0] = x.x, w[e][1] = x.y, w[e][2] = x.z, w[e][3] = x.w;
                        } else if constexpr (W == 2) {
                            const uint2 x = *reinterpret_cast<const uint2 *>(at);
                            w[e][0] = x.x, w[e][1] = x.y;
                        } else w[e][0] = *reinterpret_cast<const uint32_t *>(at);
                    }
                    if constexpr (F == F_INT8) {
#pragma unroll
                        for (int i = 0; i < W; ++i) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) w[e][i] ^= 0x80808080u;
#pragma unroll
                            for (int k = 0; k < 2; ++k) {  // two dimensions of both token pairs
                                const uint32_t y = __byte_perm(w[0][i], w[1][i], k ? 0x7362 : 0x5140);
                                const uint32_t z = __byte_perm(w[2][i], w[3][i], k ? 0x7362 : 0x5140);
                                const uint32_t f[4] = {bytes_to_half(y, 0x4140), bytes_to_half(y, 0x4342),
                                                       bytes_to_half(z, 0x4140), bytes_to_half(z, 0x4342)};
#pragma unroll
                                for (int n = 0; n < NT; ++n) mma<false>(o[2 * i + k][n], f, p[n][0], p[n][1]);
                            }
                        }
                    } else {
                        // D / 8 dimensions lie in one group: scales of the four tokens as two FP16 pairs
                        const uint32_t g = row4 * (D / 8) / 32, t = 16 * c + 2 * col4;
                        const uint32_t sa = vsc[t * S::kGroups + g] | (uint32_t)vsc[(t + 1) * S::kGroups + g] << 16;
                        const uint32_t sb = vsc[(t + 8) * S::kGroups + g] | (uint32_t)vsc[(t + 9) * S::kGroups + g] << 16;
#pragma unroll
                        for (int i = 0; i < W; ++i)
#pragma unroll
                            for (int half = 0; half < 2; ++half) {
                                uint32_t y = __byte_perm(w[0][i], w[1][i], half ? 0x7632 : 0x5410);
                                uint32_t z = __byte_perm(w[2][i], w[3][i], half ? 0x7632 : 0x5410);
#pragma unroll
                                for (int k = 0; k < 2; ++k) {
                                    const uint32_t f[4] = {mul2(nibble0(y), sa), mul2(nibble1(y), sa),
                                                           mul2(nibble0(z), sb), mul2(nibble1(z), sb)};
#pragma unroll
                                    for (int n = 0; n < NT; ++n)
                                        mma<false>(o[4 * i + 2 * half + k][n], f, p[n][0], p[n][1]);
                                    y >>= 8;
                                    z >>= 8;
                                }
                            }
                    }
                }
            }
            __syncwarp();  // the slot that the next fill takes was read in the round before this one
            fill(stage == 0 ? S::kStages - 1 : stage - 1);
            stage = stage + 1 == (uint32_t)S::kStages ? 0 : stage + 1;
        }

        // ---- the warp's part, in the ring slot that it read last (the next fill comes after a unit more) ----
        float *mine_o = reinterpret_cast<float *>(ring + (stage == 0 ? S::kStages - 1 : stage - 1) * S::kStage);
        {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float unit_out = 1.0f, x = l[n][h];
                    if constexpr (F == F_F16) unit_out = 1.0f / 4096.0f;
                    if constexpr (F >= F_INT8) unit_out = 1.0f / 1024.0f;
                    if constexpr (F == F_INT4) unit_out *= 1.0f / 1024.0f;
                    if constexpr (F >= F_INT8) {  // relative to the maximum, like the other formats'
                        const float past = m[n][h] == -INFINITY ? 0.0f : ref[n][h] - m[n][h];
                        x *= ex2(past);
                        unit_out *= ex2(past + common);
                    }
                    x += __shfl_xor_sync(0xffffffffu, x, 4);
                    x += __shfl_xor_sync(0xffffffffu, x, 8);
                    x += __shfl_xor_sync(0xffffffffu, x, 16);
                    const uint32_t head = n * 8 + 2 * col4 + h;
                    if (row4 == 0) sums[warp * S::kHeads + head] = make_float2(m[n][h], x);
#pragma unroll
                    for (int i = 0; i < KS; ++i)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const uint32_t d = F <= F_BF16 ? 16 * i + row4 + 8 * e : (D / 8) * row4 + 2 * i + e;
                            mine_o[head * D + d] = o[i][n][2 * e + h] * unit_out;
                        }
                }
        }
        auto write_out = [&](uint32_t head, uint32_t d, float x, float y, float big, float sum) {
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            uint64_t row;
            if constexpr (C) row = (uint64_t)(cur.row0 + (col0 + head) / a.group) * a.q_heads + head0 + (col0 + head) % a.group;
            else row = (uint64_t)cur.b * a.q_heads + head0 + head;
            uint32_t *out = static_cast<uint32_t *>(a.out) + (row * D + d) / 2;
            *out = a.dtype == BGTQ_F16 ? pack<false>(x * inv, y * inv) : pack<true>(x * inv, y * inv);
            if (a.lse && d == 0) a.lse[row] = sum == 0.0f ? -INFINITY : (big + __log2f(sum)) * kLn2;
        };
        if (cur.quad) {
            __syncwarp();
            if (pair_of(cur) < pairs)
                for (uint32_t i = lane; i < heads * (D / 2); i += 32) {
                    const uint32_t head = i / (D / 2), d = 2 * (i % (D / 2));
                    const float2 ml = sums[warp * S::kHeads + head], v = *reinterpret_cast<float2 *>(mine_o + head * D + d);
                    write_out(head, d, v.x, v.y, ml.x, ml.y);
                }
            __syncwarp();
            if (!next_item(cur)) break;
            if (!cur.quad) __syncthreads();
            continue;
        }
        if (lane == 0) flags[kWarps * 4 + 1 + warp] = (uint32_t)(reinterpret_cast<unsigned char *>(mine_o) - smem);
        __syncthreads();
        const bool whole = cur.at == 0 && cur.end == cur.units;
        // the CTAs that hold its first and its last unit
        const uint64_t from = cur.base + kItemCost;
        const uint32_t c_first = whole ? 0 : owner(from), c_last = whole ? 0 : owner(from + cur.units - 1);
        // at most one pair that is not whole begins in a CTA's range: its counter is that CTA's
        uint32_t *counter = static_cast<uint32_t *>(a.workspace) + c_first;
        float *parts = reinterpret_cast<float *>(static_cast<unsigned char *>(a.workspace) + a.counters);
        // this CTA's slot for the part: the pair begins before its range (first slot) or in it (second)
        float *slot = parts + (2ull * blockIdx.x + (cur.at == 0 ? 1 : 0)) * S::kPartFloats;
        const float *parts_o[kWarps];
#pragma unroll
        for (uint32_t w = 0; w < kWarps; ++w) parts_o[w] = reinterpret_cast<float *>(smem + flags[kWarps * 4 + 1 + w]);
        for (uint32_t i = threadIdx.x; i < heads * (D / 2); i += kThreads) {
            const uint32_t head = i / (D / 2), d = 2 * (i % (D / 2));
            float big = -INFINITY, sum = 0.0f, x = 0.0f, y = 0.0f;
#pragma unroll
            for (uint32_t w = 0; w < kWarps; ++w) big = fmaxf(big, sums[w * S::kHeads + head].x);
            const float ref = big == -INFINITY ? 0.0f : big;
#pragma unroll
            for (uint32_t w = 0; w < kWarps; ++w) {
                const float2 ml = sums[w * S::kHeads + head], v = *reinterpret_cast<const float2 *>(parts_o[w] + head * D + d);
                const float f = ex2(ml.x - ref);
                sum = fmaf(f, ml.y, sum);
                x = fmaf(f, v.x, x);
                y = fmaf(f, v.y, y);
            }
            if (whole) write_out(head, d, x, y, big, sum);
            else {
                *reinterpret_cast<float2 *>(slot + head * D + d) = make_float2(x, y);
                if (d == 0) *reinterpret_cast<float2 *>(slot + S::kHeads * D + 2 * head) = make_float2(big, sum);
            }
        }
        if (!whole) {
            __threadfence();
            __syncthreads();
            if (threadIdx.x == 0) {
                const uint32_t n = atomicAdd(counter, 1u);
                flags[kWarps * 4] = n == c_last - c_first;
                if (n == c_last - c_first) *counter = 0;
            }
            __syncthreads();
            if (flags[kWarps * 4]) {
                __threadfence();
                for (uint32_t i = threadIdx.x; i < heads * (D / 4); i += kThreads) {
                    const uint32_t head = i / (D / 4), d = 4 * (i % (D / 4));
                    float big = -INFINITY, sum = 0.0f, x[4] = {};
                    // kBatch parts at a time, so that their loads are in flight together
                    constexpr uint32_t kBatch = 8;
                    for (uint32_t c0 = c_first; c0 <= c_last; c0 += kBatch) {
                        float2 ml[kBatch];
                        float4 v[kBatch];
#pragma unroll
                        for (uint32_t k = 0; k < kBatch; ++k) {
                            const uint32_t c = min(c0 + k, c_last);
                            const float *p = parts + (2ull * c + (c == c_first ? 1 : 0)) * S::kPartFloats;
                            ml[k] = __ldcg(reinterpret_cast<const float2 *>(p + S::kHeads * D + 2 * head));
                            v[k] = __ldcg(reinterpret_cast<const float4 *>(p + head * D + d));
                        }
                        float now = big;
#pragma unroll
                        for (uint32_t k = 0; k < kBatch; ++k) now = fmaxf(now, ml[k].x);
                        const float ref = now == -INFINITY ? 0.0f : now, f = ex2(big - ref);
                        big = now;
                        sum *= f, x[0] *= f, x[1] *= f, x[2] *= f, x[3] *= f;
#pragma unroll
                        for (uint32_t k = 0; k < kBatch; ++k) {
                            const float g = c0 + k <= c_last ? ex2(ml[k].x - ref) : 0.0f;
                            sum = fmaf(ml[k].y, g, sum);
                            x[0] = fmaf(v[k].x, g, x[0]), x[1] = fmaf(v[k].y, g, x[1]);
                            x[2] = fmaf(v[k].z, g, x[2]), x[3] = fmaf(v[k].w, g, x[3]);
                        }
                    }
                    write_out(head, d, x[0], x[1], big, sum);
                    write_out(head, d + 2, x[2], x[3], big, sum);
                }
            }
        }
        if (!next_item(cur)) break;
        __syncthreads();
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

// CTAs of a launch at most: the workspace holds two parts of each.
uint32_t most_ctas() {
    int dev = 0;
    return cudaGetDevice(&dev) == cudaSuccess ? (uint32_t)sm_count(dev) * 4 : 0;
}
uint32_t counter_bytes() { return (most_ctas() * 4 + 15) / 16 * 16; }

template <int F, int D, int NT, bool C>
cudaError_t run(const std::conditional_t<C, ChunkArgs, PagedAttendArgs> &a, cudaStream_t s) {
    using S = Shape<F, D, NT>;
    auto kernel = attend_kernel<F, D, NT, C>;
    static int resident[64] = {};  // CTAs an SM holds, by device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || dev < 0 || dev >= 64) return e != cudaSuccess ? e : cudaErrorInvalidDevice;
    if (!resident[dev]) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
        if (e != cudaSuccess) return e;
        int n = 0;
        e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, kThreads, S::kSmem);
        if (e != cudaSuccess) return e;
        resident[dev] = n < 1 ? 1 : n > 4 ? 4 : n;
    }
    const int sms = sm_count(dev);
    if (!sms) return cudaErrorInvalidDevice;
    auto b = a;
    // (chunks share their workspace with the kernel of many rows: both keep their counters in the bytes that start from zero)
    b.counters = C ? BGTQ_WORKSPACE_ZEROED : counter_bytes();
    // queries by 16 bytes where they lie so, else by elements (32 requests of 4096 tokens, 16 / 1 heads: 29.5, 30.7 us)
    if constexpr (!C) b.q_even = reinterpret_cast<uintptr_t>(a.q) % 16 == 0 && a.q_batch % 8 == 0 && a.q_head % 8 == 0;
    kernel<<<(uint32_t)(sms * resident[dev]), kThreads, S::kSmem, s>>>(b);
    return cudaGetLastError();
}

}  // namespace
}  // namespace bgtq
