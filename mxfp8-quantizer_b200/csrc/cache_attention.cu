// cache_attention.cu -- one query token per sequence against the paged MXFP8
// cache: o = sum_j p_j v_j / sum_j p_j, p_j = exp(scale q . k_j).
//
// A cached byte is used by the G query heads that share a KV head: 4 G
// operations for 1 + 1/32 bytes, so HBM bandwidth bounds it as long as the
// arithmetic keeps up.  It is fetched once by each pass over up to 8 or 16 of
// those heads (row_tiles).  Tensor cores do both products (mma m16n8k16,
// f16 operands, f32 sums): an E4M3 value is exact in f16, so the payload needs
// one conversion and the scales stay outside the products:
//   q . k_j = sum over blocks of 32 of  2^(sk - 127) (q . payload), a sum per
//     block scaled in f32.  q is brought to f16 with one power of two a head
//     (largest element in [2^14, 2^15)): a bf16 value is exact there down to
//     2^-31 of the head's largest, an fp16 value down to 2^-28, and a smaller
//     one is off by 2^-39 of the largest at most.
//   sum_j p_j v_j: the operand is p_j 2^(sv - R + 15), for the V scale bytes sv
//     in the window R - 11 .. R.  It is two f16, p_j 2^15 and what that leaves,
//     each times the power of two: 2^-22 of relative error at most, or 2^-28 of
//     the largest weight where f16 has no more bits.  (One f16, 2^-11, was 3 %
//     faster and showed in fp16 outputs and in one bf16 output of thirty.)
//     A tile whose scales span more takes several windows from its largest byte
//     down, each a pass over V in shared memory (zero rows among small ones do:
//     their byte is 127); the accumulator is kept in units of the latest R.
//     With one R for all, columns and rows 2^29 below the largest were lost.
// The m16n8k16 shapes are used because a decode step has at most 16 rows of
// queries: a 128-row tcgen05 tile would be empty to 7/8 and would want K and V
// converted into shared memory first.
//
// Work: the tiles (POS positions) of all sequences and KV heads in a row are
// split evenly over the warps, whatever the lengths are; a change of sequence
// or head counts as kSegmentCost tiles.  A warp is on its own: it fetches its
// tiles (cp.async into a ring of its own, no block-wide barrier on the way),
// computes the scores with heads as rows and positions as columns, which is
// the layout the second product takes its operand in, and keeps its running
// maximum and sums.  A (sequence, KV head) that one warp holds whole is
// written at once; pieces of the others go to the workspace, one for the warps
// of a CTA that end inside the same segment, and a second launch joins them in
// order, so the result does not depend on timing.
//
// Measured, both launches: 64 ragged sequences of up to 4096, 32 heads over 8,
// D = 128: 50.3 us = 4.8 TB/s of cache; 8 of up to 65536, 16 heads over 2,
// D = 256: 61.3 us = 4.9 TB/s; 1 of 1000: 7.9 us.  With weights of one f16 the
// first took 49.1, of which 43 us were left without the arithmetic, 46 without
// the fetches, 45.5 without the join: a
// warp's tile takes about 1.7 us either way, and eight warps an SM are what the
// registers allow (12 or 16 with fewer registers, tiles of 16 positions for
// D <= 128, a third stage for D = 256: all slower).  Half of the issue slots are
// used (ncu), no pipe above 41 %.  K as E4M3 operands (m16n8k32), the query split
// into E4M3 pieces of 4 bits, saves the conversions of K and half of the products
// but was no faster with two pieces (49.7 us), which do not hold every query, and
// slower with the four that do (57.7 us; 8 of 65536: 75 us).
// Many short sequences pay for the change from one to the next and for tiles
// that end inside: 4096 of up to 128 positions 210 us, floor 95; 12 of them are
// the second f16 and the scales of absent positions.  Before those, 182 if the
// queries cost nothing (a prefetch of them to L2 or L1 with a segment's first
// tile gained nothing), 192 without the stores.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "../../include/mxfp8_cache.h"
#include "cache.cuh"
#include "launch.h"
#include "ptx.cuh"

namespace mxfp8 {

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kJoinWarps = 4;
constexpr int kJoinThreads = 32 * kJoinWarps;
constexpr int kSegmentCost = 2;
// With a length a lane the join finds a segment's warps from the lengths, while the first launch still runs; above it
// the first launch leaves a note (meta).  1 sequence of 1000: 7.6 us, 8.0 with notes; 32 of 4096, D = 64: 24.6 and
// 27.3; 128 of 512: 28.5 with four lengths a lane, 23.7 with notes.
constexpr int64_t kScanBatch = 32;
// V's scale bytes that one window takes: 2^(sv - R) is an f16 with three binades to spare, and p_j 2^15 keeps its bits
// down to p_j = 2^-18.  A tile's windows are a loop around the second product that is left after one turn; a copy of the
// product for tiles with several was as fast where it fitted the registers and 2 to 6 % slower where it did not.
constexpr int kWindow = 12;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr uint32_t kNoRow32 = 0xFFFFFFFFu;

// Heads in groups of 8 * NT rows: 16 where that saves a second pass over K and
// V and the accumulators fit the registers.  Each pass is work of its own, so
// the cache is fetched once a pass, in part from L2.  8 sequences of up to 16384,
// one KV head: D = 256, 8 heads 20.8 us, 16 (two passes) 25.4; D = 128, 16 heads
// 17.0 (two passes of 8: 16.5), 24 heads 19.7 (three: 19.2), 64 heads 27.3
// (eight: 32.4).  16 of up to 65536, 16 heads 41.4 (two of 8: 56.7), 32 heads 69.4 (100).
inline int row_tiles(int dim, int group) { return group > 8 && dim <= 128 ? 2 : 1; }

template <int D, int NT>
struct Config {
    static constexpr int rows = 8 * NT;
    static constexpr int pos = D <= 128 ? 32 : 16;            // positions of a tile
    static constexpr int kv_bytes = pos * D;                  // K (or V) payload of a tile
    static constexpr int sc_bytes = pos * D / 32;
    static constexpr int stage_bytes = 2 * kv_bytes + 2 * sc_bytes;
    static constexpr int stages = D <= 64 ? 3 : 2;
    // Long queries are kept in shared memory: in registers they took what the compiler needs to overlap a tile's
    // steps (8 sequences of 65536, D = 256: 61.1 us, 69.2 in registers).  16 rows of D = 128 are better off there
    // (16 sequences of 8192: 20.6 us, 21.4 in shared memory).
    static constexpr int query_bytes = D > 128 ? D * 16 * NT : 0;
    static constexpr int warp_bytes = stages * stage_bytes + query_bytes;
    static constexpr int smem = kWarps * warp_bytes;
    static constexpr int ctas_per_sm = 2;
};

struct Params {
    CacheAttentionArgs a;
    int group;        // query heads of a KV head
    int row_groups;   // ceil(group / rows)
    int64_t parts;    // warps
    int join_segments;  // that a CTA of the join looks at
    float* part_o;    // (2 * parts, rows, D): unscaled sums of the pieces
    float2* part_ml;  // (2 * parts, rows): running maximum (log2) and sum
    int2* meta;       // (batch * heads * row_groups): first and last warp of a split segment, if batch > kScanBatch
};

__device__ __forceinline__ int length_of(const CacheAttentionArgs& a, int64_t b) {
    return (int)visible_length(a.lengths[b], a.max_pages, a.c.page_shift);
}
// The same from L2: the join's look at the lengths before its own wait, when an older line may still be in L1.
__device__ __forceinline__ int early_length_of(const CacheAttentionArgs& a, int64_t b) {
    return (int)visible_length(__ldcg(a.lengths + b), a.max_pages, a.c.page_shift);
}

// Cost of a sequence's segment: its tiles and the change to it, 0 if empty.
template <int POS>
__device__ __forceinline__ int cost_of(int len) {
    return len == 0 ? 0 : (len + POS - 1) / POS + kSegmentCost;
}

// A lane's share of the sequences' costs: neighbouring sequences b0 .. b1 - 1;
// the sums (over one head group) fit 32 bits, the entry checks it.
struct Costs {
    int64_t b0, b1, total;
    uint32_t mine, upto;  // of these sequences, and of all up to them
    int len;              // of the last of them
};

template <int POS, bool kEarly = false>
__device__ __forceinline__ Costs costs_of(const CacheAttentionArgs& a, int lane) {
    Costs c;
    const int64_t per = (a.batch + 31) / 32;
    c.b0 = min(a.batch, per * lane);
    c.b1 = min(a.batch, c.b0 + per);
    c.mine = 0;
    c.len = 0;
    for (int64_t b = c.b0; b < c.b1; ++b) {
        c.len = kEarly ? early_length_of(a, b) : length_of(a, b);
        c.mine += cost_of<POS>(c.len);
    }
    c.upto = c.mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint32_t o = __shfl_up_sync(0xFFFFFFFFu, c.upto, d);
        if (lane >= d) c.upto += o;
    }
    c.total = (int64_t)__shfl_sync(0xFFFFFFFFu, c.upto, 31);
    return c;
}

// A warp's place: sequence b, head group g (KV head and row group), tile t of
// its tiles t0 .. t1 - 1 of that segment's nt; `base` is the segment's place
// in the sum of all costs, `end` the end of the warp's share of it.
struct Cursor {
    int64_t base, end, b;
    const int32_t* pages;
    int g, t, t0, t1, nt, len;
    uint32_t head;  // KV head of g
    bool done;
};

// The warp's tiles of the cursor's segment; true if there are any.
__device__ __forceinline__ bool enter(Cursor& c, int64_t begin) {
    const int64_t first = c.base + kSegmentCost;
    c.t0 = begin > first ? (int)(begin - first) : 0;
    c.t1 = c.end - first < c.nt ? (int)(c.end - first) : c.nt;
    c.t = c.t0;
    return c.t0 < c.t1;
}

__device__ __forceinline__ void set_group(const Params& p, Cursor& c, int g) {
    c.g = g;
    c.head = (uint32_t)(p.row_groups == 1 ? g : g / p.row_groups);
}

template <int POS>
__device__ __forceinline__ void enter_sequence(const Params& p, Cursor& c, int len) {
    c.len = len;
    c.nt = (c.len + POS - 1) / POS;
    c.pages = p.a.table + c.b * p.a.table_stride;
}

// To the next segment in which the warp has tiles.
template <int POS>
__device__ __forceinline__ void next_segment(const Params& p, Cursor& c, int groups) {
    do {
        c.base += c.nt + kSegmentCost;
        if (c.base + kSegmentCost >= c.end) {
            c.done = true;
            return;
        }
        if (c.g + 1 < groups) {
            set_group(p, c, c.g + 1);
        } else {
            set_group(p, c, 0);
            do {  // total cost is not exhausted: there is another sequence with tiles
                ++c.b;
                enter_sequence<POS>(p, c, length_of(p.a, c.b));
            } while (c.nt == 0);
        }
    } while (!enter(c, c.base));
}

template <int POS>
__device__ __forceinline__ void advance(const Params& p, Cursor& c, int groups) {
    if (++c.t == c.t1) next_segment<POS>(p, c, groups);
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool on) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool on) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(on ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two E4M3 bytes (the low or the high half of w) as an f16 pair.
__device__ __forceinline__ void e4m3x4_to_half2(uint32_t w, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
}

// Four UE8M0 bytes as bf16 pairs: 2^(byte - 127), NaN for 255; exact.
__device__ __forceinline__ void ue8m0x4_to_bf162(uint32_t w, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
        "cvt.rn.bf16x2.ue8m0x2 %0, a;\n\tcvt.rn.bf16x2.ue8m0x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
}

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same with nothing in d before.
__device__ __forceinline__ void mma_f16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
    const __half2 t = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&t);
}
__device__ __forceinline__ uint32_t mul_half2(uint32_t a, uint32_t b) {
    const __half2 t = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&t);
}
__device__ __forceinline__ uint32_t pack_out(bool bf16, float lo, float hi) {
    if (!bf16) return pack_half2(lo, hi);
    const __nv_bfloat162 t = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&t);
}

// Shared memory of a tile's rows of D bytes: 32-byte groups of a row are
// permuted (xor with a key of the row) so that the four rows that one access
// phase reads (K: rows r .. r + 3, V: the same after v_place) fall on different
// banks.
template <int D>
__device__ __forceinline__ constexpr int key_of(int row) {
    return D % 128 == 0 ? (row & 3) : ((row >> 1) & 1);
}
template <int D>
__device__ __forceinline__ constexpr uint32_t group_at(int row, int group) {
    return (uint32_t)(row * D + ((group ^ key_of<D>(row)) << 5));
}
// The same place as `at` (in group 0 of its row), in group blk: the key's bits
// are exchanged, the others added; a row's start has none of the key's bits.
template <int D>
__device__ __forceinline__ constexpr uint32_t in_block(uint32_t at, int blk) {
    constexpr int kKey = D % 128 == 0 ? 3 : 1;
    return (at ^ (uint32_t)((blk & kKey) << 5)) + (uint32_t)((blk & ~kKey) << 5);
}
// Row that position j of V is kept in: of each 16, the positions 2c + i, c = 0
// .. 3, that a phase of the second product reads are neighbours.
__device__ __forceinline__ constexpr int v_place(int j) { return (j & ~15) | ((j & 15) >> 1) | ((j & 1) << 3); }

// Page of position `lane` of the cursor's tile, as the table has it.  The load
// is consumed a tile later (row_of_lane): waiting for it here would cost a
// memory latency a tile.
template <int POS>
__device__ __forceinline__ int page_of_lane(const Params& p, const Cursor& c, int lane) {
    const int at = c.t * POS + lane;
    return c.done || lane >= POS || at >= c.len ? -1 : c.pages[at >> p.a.c.page_shift];  // at is within the table
}

// Cache row of position `lane` of the cursor's tile, kNoRow32 where there is none.
template <int POS>
__device__ __forceinline__ uint32_t row_of_lane(const Params& p, const Cursor& c, int page, int lane) {
    const int at = c.t * POS + lane;
    if (lane >= POS || at >= c.len) return kNoRow32;
    if ((uint32_t)page >= (uint32_t)p.a.c.num_pages) {
        if (p.a.status) atomicOr(p.a.status, kErrCacheIndex);
        return kNoRow32;
    }
    // cache_row in 32 bits: a cache has fewer rows
    return ((((uint32_t)page * (uint32_t)p.a.c.heads + c.head) << p.a.c.page_shift) |
            ((uint32_t)at & ((1u << p.a.c.page_shift) - 1u)));
}

// Fetch the rows of a whole tile whose pages hold 16 positions or more: each 16
// of them are one run of memory.
template <int D, int POS>
__device__ __forceinline__ void fetch_runs(const Params& p, uint32_t stage, uint32_t my_row, int lane) {
    constexpr int kChunks = D / 16, kRows = 32 / kChunks, kKv = POS * D;
    const int j0 = lane / kChunks, ch = lane % kChunks;
    const uint32_t k_at = stage + group_at<D>(j0, ch >> 1) + (ch & 1) * 16;
    const uint32_t v_at = stage + kKv + group_at<D>(v_place(j0), ch >> 1) + (ch & 1) * 16;
#pragma unroll
    for (int run = 0; run < POS / 16; ++run) {
        const uint64_t off = (uint64_t)__shfl_sync(0xFFFFFFFFu, my_row, run * 16) * D + lane * 16;
        const uint8_t* k = p.a.k + off;
        const uint8_t* v = p.a.v + off;
#pragma unroll
        for (int i = run * 16 / kRows; i < (run + 1) * 16 / kRows; ++i) {
            const int from = (i - run * 16 / kRows) * 512;
            cp_async16(i * kRows * D + (k_at ^ (key_of<D>(i * kRows) << 5)), k + from, true);
            cp_async16(v_place(i * kRows) * D + (v_at ^ (key_of<D>(v_place(i * kRows)) << 5)), v + from, true);
        }
    }
    // a run's scale bytes: 16 * D / 32 of them, 4 a lane
    constexpr int kWords = D / 8;
#pragma unroll
    for (int i = 0; i < (POS / 16 * kWords + 31) / 32; ++i) {
        const int idx = i * 32 + lane, run = idx / kWords, in = idx - run * kWords;
        const uint32_t row = __shfl_sync(0xFFFFFFFFu, my_row, (run * 16) & (POS - 1));
        if (POS / 16 * kWords % 32 == 0 || idx < POS / 16 * kWords) {
            const uint64_t off = (uint64_t)row * (D / 32) + in * 4;
            cp_async4(stage + 2 * kKv + idx * 4, p.a.k_scales + off, true);
            cp_async4(stage + 2 * kKv + POS * D / 32 + idx * 4, p.a.v_scales + off, true);
        }
    }
}

// Fetch those rows into a stage: payloads 16 bytes a lane, scales four bytes a
// lane (two positions' scale bytes are 4, 8, 12 or 16 contiguous ones: pages
// hold an even number of positions).  Absent positions are zeros.
template <int D, int POS>
__device__ __forceinline__ void fetch(const Params& p, uint32_t stage, uint32_t my_row, int lane) {
    constexpr int kChunks = D / 16;  // of a row
    constexpr int kKv = POS * D;
    if constexpr ((kChunks & (kChunks - 1)) == 0) {
        // A lane keeps its chunk; step i takes row i * kRows + j0.  Both the row of V and the keys split into a
        // part of i and a part of j0 that share no bits, so a step's address is the lane's own, xor a constant, plus
        // a constant.
        constexpr int kRows = 32 / kChunks;
        const int j0 = lane / kChunks, ch = lane % kChunks;
        const uint32_t k_at = group_at<D>(j0, ch >> 1) + (ch & 1) * 16;
        const uint32_t v_at = group_at<D>(v_place(j0), ch >> 1) + (ch & 1) * 16;
        const uint8_t* k = p.a.k + ch * 16;
        const uint8_t* v = p.a.v + ch * 16;
#pragma unroll
        for (int i = 0; i < POS / kRows; ++i) {
            const uint32_t row = __shfl_sync(0xFFFFFFFFu, my_row, i * kRows + j0);
            const bool on = row != kNoRow32;
            const uint64_t off = (uint64_t)(on ? row : 0u) * D;
            cp_async16(stage + i * kRows * D + (k_at ^ (key_of<D>(i * kRows) << 5)), k + off, on);
            cp_async16(stage + kKv + v_place(i * kRows) * D + (v_at ^ (key_of<D>(v_place(i * kRows)) << 5)), v + off, on);
        }
    } else {
#pragma unroll
        for (int i = 0; i < kKv / 512; ++i) {
            const int idx = i * 32 + lane;
            const int j = idx / kChunks, ch = idx - j * kChunks;
            const uint32_t row = __shfl_sync(0xFFFFFFFFu, my_row, j);
            const bool on = row != kNoRow32;
            const uint64_t off = (uint64_t)(on ? row : 0u) * D + ch * 16;
            cp_async16(stage + group_at<D>(j, ch >> 1) + (ch & 1) * 16, p.a.k + off, on);
            cp_async16(stage + kKv + group_at<D>(v_place(j), ch >> 1) + (ch & 1) * 16, p.a.v + off, on);
        }
    }
    constexpr int kPair = D / 64;    // 4-byte pieces of two positions' scales
    constexpr int kPieces = POS / 2 * kPair;
#pragma unroll
    for (int i = 0; i < (kPieces + 31) / 32; ++i) {
        const int idx = i * 32 + lane;
        const int pair = idx / kPair, in = idx - pair * kPair;
        const uint32_t even = __shfl_sync(0xFFFFFFFFu, my_row, (2 * pair) & (POS - 1));
        if (kPieces % 32 == 0 || idx < kPieces) {
            const bool on = even != kNoRow32;
            const uint64_t off = (uint64_t)(on ? even : 0u) * (D / 32) + in * 4;
            cp_async4(stage + 2 * kKv + idx * 4, p.a.k_scales + off, on);
            cp_async4(stage + 2 * kKv + POS * D / 32 + idx * 4, p.a.v_scales + off, on);
        }
    }
}

// This lane's elements of the cursor's query rows, as they are in memory.
template <int D, int NT>
__device__ __forceinline__ void load_query(const Params& p, const Cursor& c, int lane, uint32_t (&raw)[NT][D / 8]) {
    const int kv_head = (int)c.head, sub = c.g - kv_head * p.row_groups;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int in = sub * Config<D, NT>::rows + n * 8 + (lane >> 2);
        const bool on = in < p.group;
        const uint16_t* src = p.a.q + c.b * p.a.q_batch + (int64_t)(kv_head * p.group + (on ? in : 0)) * p.a.q_head;
        const bool vec = (reinterpret_cast<uintptr_t>(src) & 15) == 0;
#pragma unroll
        for (int blk = 0; blk < D / 32; ++blk) {
            const uint4 t = load8(src + blk * 32 + (lane & 3) * 8, vec);
            raw[n][4 * blk] = on ? t.x : 0u;
            raw[n][4 * blk + 1] = on ? t.y : 0u;
            raw[n][4 * blk + 2] = on ? t.z : 0u;
            raw[n][4 * blk + 3] = on ? t.w : 0u;
        }
    }
}

// The rows as MMA operands, and what a score is multiplied by: |scale| *
// log2(e) * the power of two taken out of the row.
template <int D, int NT>
__device__ __forceinline__ void settle_query(const Params& p, const uint32_t (&raw)[NT][D / 8],
                                             uint32_t (&qf)[D / 32][4 * NT], float (&mul)[NT]) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        float v[D / 32][8];
        float amax = 0.0f;
#pragma unroll
        for (int blk = 0; blk < D / 32; ++blk) {
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const uint32_t pair = raw[n][4 * blk + e / 2];
                if (p.a.q_bf16) {
                    v[blk][e] = __uint_as_float(pair << 16);
                    v[blk][e + 1] = __uint_as_float(pair & 0xFFFF0000u);
                } else {
                    const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&pair));
                    v[blk][e] = t.x;
                    v[blk][e + 1] = t.y;
                }
                amax = fmaxf(amax, fmaxf(fabsf(v[blk][e]), fabsf(v[blk][e + 1])));
            }
        }
        amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 2));
        // exponent of the largest element; subnormal and infinite ones are held at the ends of the range
        const int e = min(max((int)(__float_as_uint(amax) >> 23), 15), 254) - 127;
        // 2^(14 - e), with the sign of the scale; a product of 0 is kept as a query of 0, so that mul is above 0
        float down = copysignf(__uint_as_float((uint32_t)(127 + 14 - e) << 23), p.a.scale);
        mul[n] = fabsf(p.a.scale) * kLog2e * __uint_as_float((uint32_t)(127 - 14 + e) << 23);
        if (mul[n] == 0.0f || amax == 0.0f) {
            mul[n] = 1.0f;
            down = 0.0f;
        }
#pragma unroll
        for (int blk = 0; blk < D / 32; ++blk)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int r = 0; r < 2; ++r)
                    qf[blk][h * 2 * NT + n * 2 + r] =
                        pack_half2(v[blk][4 * h + 2 * r] * down, v[blk][4 * h + 2 * r + 1] * down);
    }
}

// Scale bytes of positions 2 q and 2 q + 1 of eight (those of the quad's
// columns), as halves of two blocks each: w[0 .. NB/2 - 1] the first's.
template <int NB>
__device__ __forceinline__ void load_scale_pair(const uint8_t* src, uint32_t (&w)[NB / 2]) {
#pragma unroll
    for (int i = 0; i < NB / 2; ++i) w[i] = reinterpret_cast<const uint32_t*>(src)[i];
}

// The next window of a tile's V scales, from the largest byte up to `left` down, but not below `floor`: the tile's scales
// in shared memory are replaced by the window's own, the others by a byte whose factor is a zero; NaN blocks (in the
// first window, left = 254) by payloads of NaN.  The scales as they were are kept in the place of K's, which are used
// up.  Returns R; `left` becomes the largest byte that the next window may take, or -1.  `least` is the tile's smallest.
template <int D, int POS>
__device__ __forceinline__ int take_window(uint8_t* st, int lane, int floor, int least, int& left) {
    constexpr int kKv = POS * D, kWords = D / 64;
    uint16_t* const kept = reinterpret_cast<uint16_t*>(st + 2 * kKv) + lane * kWords;
    uint16_t* const used = kept + kKv / 64;
    const bool first = left == 254;
    int upper = floor;
    __syncwarp();  // everyone has read what is replaced here
    if (lane < POS) {
        for (int i = 0; i < 2 * kWords; ++i) {
            if (first && (i & 1) == 0) kept[i / 2] = used[i / 2];
            const int byte = (kept[i / 2] >> (8 * (i & 1))) & 0xFF;
            if (byte <= left) upper = max(upper, byte);
        }
    }
    upper = __reduce_max_sync(0xFFFFFFFFu, upper);
    const bool last = least > upper - kWindow || upper == floor;  // the lowest window has no lower end
    const int zero = upper < 15 ? upper + 17 : upper - 15;        // (byte + 15 - R) << 10 is an f16 zero, of either sign
    if (lane < POS) {
        for (int i = 0; i < kWords; ++i) {
            int two = 0;
            for (int h = 0; h < 2; ++h) {
                const int byte = (kept[i] >> (8 * h)) & 0xFF;
                const bool in = byte <= left && byte + 15 >= upper && (last || byte > upper - kWindow);
                two |= (in ? byte : zero) << (8 * h);
                if (first && byte == 255) {
                    uint4* const row = reinterpret_cast<uint4*>(st + kKv + group_at<D>(v_place(lane), 2 * i + h));
                    row[0] = row[1] = make_uint4(0x7F7F7F7Fu, 0x7F7F7F7Fu, 0x7F7F7F7Fu, 0x7F7F7F7Fu);
                }
            }
            used[i] = (uint16_t)two;
        }
    }
    __syncwarp();
    left = last ? -1 : upper - kWindow;
    return upper;
}

// A warp's piece of a segment to a slot of the workspace: rows as in the
// scores (8 n + row) for m and l, as in acc (8 n + 2 quad + {0, 1}) for the sums.
template <int D, int NT>
__device__ __forceinline__ void put_piece(const Params& p, int64_t slot, int rows, int lane, const float (&m)[NT],
                                          const float (&l)[NT], const float (&acc)[NT][D / 16][4]) {
    const int row = lane >> 2, quad = lane & 3;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        if (quad == 0 && n * 8 + row < rows)
            gstore_plain(p.part_ml + slot * Config<D, NT>::rows + n * 8 + row, make_float2(m[n], l[n]), p.a.ww,
                         p.a.status);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int r = n * 8 + 2 * quad + j;
            if (r >= rows) continue;
#pragma unroll
            for (int blk = 0; blk < D / 32; ++blk)
                gstore_plain(reinterpret_cast<float4*>(p.part_o + (slot * Config<D, NT>::rows + r) * D + blk * 32 + 4 * row),
                             make_float4(acc[n][2 * blk][j], acc[n][2 * blk][2 + j], acc[n][2 * blk + 1][j],
                                         acc[n][2 * blk + 1][2 + j]),
                             p.a.ww, p.a.status);
        }
    }
}

template <int D, int NT>
__global__ void __launch_bounds__(kThreads, Config<D, NT>::ctas_per_sm) cache_attention_kernel(const Params p) {
    using C = Config<D, NT>;
    constexpr int POS = C::pos, kCols = POS / 8;   // positions in columns of eight
    constexpr int kBlocks = D / 32, kWords = kBlocks / 2;
    constexpr uint32_t kFull = POS == 32 ? 0xFFFFFFFFu : (1u << POS) - 1u;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int64_t ends_in[kWarps], lead_slot[kWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = lane >> 2, quad = lane & 3;
    const int groups = p.a.c.heads * p.row_groups;

    grid_wait_prerequisites();
    grid_launch_dependents();  // the second launch may take its place, with what ran before this one complete
    // ---- the warps' shares of all costs, and where this one's begins: every warp for itself ----
    const Costs costs = costs_of<POS>(p.a, lane);
    if (blockIdx.x == 0 && warp == 0 && p.a.status) {
        for (int64_t b = costs.b0; b < costs.b1; ++b)
            if ((int64_t)p.a.lengths[b] > (p.a.max_pages << p.a.c.page_shift)) atomicOr(p.a.status, kErrCacheIndex);
    }
    const int64_t total = costs.total * groups;
    const int64_t parts = min(p.parts, total);
    const int64_t first_part = (int64_t)blockIdx.x * kWarps;
    if (first_part >= parts) return;
    const Split split = make_split(parts, total);
    const int64_t part = first_part + warp;
    Cursor cur{};  // the tile that is computed
    cur.done = part >= parts;  // a warp without a share is there for the barriers
    if (!cur.done) {
        const int64_t begin = split_begin(split, part);
        cur.end = split_begin(split, part + 1);
        // the lane whose sequences hold the first unit, and the one of them
        const int at_lane = __ffs(__ballot_sync(0xFFFFFFFFu, begin < (int64_t)costs.upto * groups)) - 1;
        cur.b = __shfl_sync(0xFFFFFFFFu, costs.b0, at_lane);
        cur.base = (int64_t)(__shfl_sync(0xFFFFFFFFu, costs.upto - costs.mine, at_lane)) * groups;
        cur.len = __shfl_sync(0xFFFFFFFFu, costs.len, at_lane);
        if (p.a.batch > 32) {
            for (;; ++cur.b) {
                cur.len = length_of(p.a, cur.b);
                const int64_t n = (int64_t)cost_of<POS>(cur.len) * groups;
                if (begin < cur.base + n) break;
                cur.base += n;
            }
        }
        enter_sequence<POS>(p, cur, cur.len);
        const int g = groups == 1 ? 0 : (int)((begin - cur.base) / (cur.nt + kSegmentCost));
        set_group(p, cur, g);
        cur.base += (int64_t)g * (cur.nt + kSegmentCost);
        if (!enter(cur, begin)) next_segment<POS>(p, cur, groups);
    }

    // this lane's part of K (row `row` of eight) and V (place `quad` of four); the keys of the rows that it reads are
    // those of these two
    const uint32_t k_at = group_at<D>(row, 0) + quad * 8, v_at = group_at<D>(quad, 0) + 4 * row;
    uint8_t* const ring = smem + warp * C::warp_bytes;
    const uint32_t ring_u = smem_u32(ring);

    // ---- fetch ahead: `next` is the tile whose pages are being looked up ----
    Cursor next = cur;
    int my_page = page_of_lane<POS>(p, next, lane);
    uint32_t first_query[NT][D / 8] = {};
    if (!cur.done) load_query<D, NT>(p, cur, lane, first_query);  // on its way while the pages are
    uint32_t present = 0;  // lane s: which positions of stage s are there
    auto issue = [&](int stage) {
        if (!next.done) {
            const uint32_t my_row = row_of_lane<POS>(p, next, my_page, lane);
            const uint32_t mask = __ballot_sync(0xFFFFFFFFu, my_row != kNoRow32);
            if constexpr (D != 192) {
                if (mask == kFull && p.a.c.page_shift >= 4)
                    fetch_runs<D, POS>(p, ring_u + stage * C::stage_bytes, my_row, lane);
                else if (mask != 0)
                    fetch<D, POS>(p, ring_u + stage * C::stage_bytes, my_row, lane);
            } else {
                if (mask != 0) fetch<D, POS>(p, ring_u + stage * C::stage_bytes, my_row, lane);
            }
            if (lane == stage) present = mask;
            advance<POS>(p, next, groups);
            my_page = page_of_lane<POS>(p, next, lane);
        }
        cp_async_commit();
    };
#pragma unroll
    for (int s = 0; s < C::stages - 1; ++s) issue(s);

    uint4* const queries = reinterpret_cast<uint4*>(ring + C::stages * C::stage_bytes);  // where they are kept there
    uint32_t qf[C::query_bytes > 0 ? 1 : kBlocks][4 * NT];
    float mul[NT], m[NT], l[NT];
    float acc[NT][D / 16][4];
    int ref = 0;  // R of the latest window of V's scales
    auto start_segment = [&](const uint32_t (&raw)[NT][D / 8]) {
        if constexpr (C::query_bytes > 0) {
            uint32_t own[kBlocks][4 * NT];
            settle_query<D, NT>(p, raw, own, mul);
#pragma unroll
            for (int i = 0; i < kBlocks * NT; ++i)  // read back by the lane that wrote them
                queries[i * 32 + lane] = make_uint4(own[i / NT][4 * (i % NT)], own[i / NT][4 * (i % NT) + 1],
                                                    own[i / NT][4 * (i % NT) + 2], own[i / NT][4 * (i % NT) + 3]);
        } else {
            settle_query<D, NT>(p, raw, qf, mul);
        }
        ref = 0;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            m[n] = -INFINITY;
            l[n] = 0.0f;
#pragma unroll
            for (int i = 0; i < D / 16; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[n][i][j] = 0.0f;
        }
    };
    start_segment(first_query);

    int stage = 0;
    while (!cur.done) {
        cp_async_wait<C::stages - 2>();
        __syncwarp();  // also: the stage before this one is read, it can be filled again
        const uint32_t mask = __shfl_sync(0xFFFFFFFFu, present, stage);
        issue(stage == 0 ? C::stages - 1 : stage - 1);
        uint8_t* const st = ring + stage * C::stage_bytes;
        if (mask != 0) {
            if (mask != kFull) {  // an absent position (its weights are 0) gets the V scales of one that is there
                uint16_t* const scales = reinterpret_cast<uint16_t*>(st + 2 * C::kv_bytes + C::sc_bytes);
                if (lane < POS && !((mask >> lane) & 1)) {
#pragma unroll
                    for (int i = 0; i < kWords; ++i) scales[lane * kWords + i] = scales[(__ffs(mask) - 1) * kWords + i];
                }
                __syncwarp();
            }
            const uint8_t* ks = st + 2 * C::kv_bytes + quad * (2 * kBlocks);
            const uint8_t* vs = ks + C::sc_bytes;
            // ---- scores: rows are heads, columns positions 8 nt + 2 quad + {0, 1} ----
            float s[kCols][2 * NT];
            auto factors = [&](int nt, uint32_t (&f)[kBlocks]) {  // bf16, blocks in pairs, both positions
                uint32_t w[kWords];
                load_scale_pair<kBlocks>(ks + nt * 8 * kBlocks, w);
#pragma unroll
                for (int i = 0; i < kWords; ++i) ue8m0x4_to_bf162(w[i], f[2 * i], f[2 * i + 1]);
            };
            auto add_block = [&](int nt, int blk, const uint32_t (&q)[4 * NT], const uint32_t (&f)[kBlocks]) {
                const uint2 b = *reinterpret_cast<const uint2*>(st + in_block<D>(k_at, blk) + nt * 8 * D);
                uint32_t b0, b1, b2, b3;
                e4m3x4_to_half2(b.x, b0, b1);
                e4m3x4_to_half2(b.y, b2, b3);
                float d[4];
                if constexpr (NT == 1) {
                    mma_f16_first(d, q[0], 0u, q[1], 0u, b0, b1);
                    mma_f16(d, q[2], 0u, q[3], 0u, b2, b3);
                } else {
                    mma_f16_first(d, q[0], q[2], q[1], q[3], b0, b1);
                    mma_f16(d, q[4], q[6], q[5], q[7], b2, b3);
                }
                const uint32_t f0 = f[blk / 2], f1 = f[kWords + blk / 2];
                const float fx = __uint_as_float(blk & 1 ? f0 & 0xFFFF0000u : f0 << 16);
                const float fy = __uint_as_float(blk & 1 ? f1 & 0xFFFF0000u : f1 << 16);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    s[nt][2 * n] = blk == 0 ? d[2 * n] * fx : fmaf(d[2 * n], fx, s[nt][2 * n]);
                    s[nt][2 * n + 1] = blk == 0 ? d[2 * n + 1] * fy : fmaf(d[2 * n + 1], fy, s[nt][2 * n + 1]);
                }
            };
            if constexpr (C::query_bytes > 0) {
                uint32_t f[kCols][kBlocks];
#pragma unroll
                for (int nt = 0; nt < kCols; ++nt) factors(nt, f[nt]);
#pragma unroll
                for (int blk = 0; blk < kBlocks; ++blk) {
                    uint32_t q[4 * NT];
#pragma unroll
                    for (int i = 0; i < NT; ++i) {
                        const uint4 t = queries[(blk * NT + i) * 32 + lane];
                        q[4 * i] = t.x; q[4 * i + 1] = t.y; q[4 * i + 2] = t.z; q[4 * i + 3] = t.w;
                    }
#pragma unroll
                    for (int nt = 0; nt < kCols; ++nt) add_block(nt, blk, q, f[nt]);
                }
            } else {
#pragma unroll
                for (int nt = 0; nt < kCols; ++nt) {
                    uint32_t f[kBlocks];
                    factors(nt, f);
#pragma unroll
                    for (int blk = 0; blk < kBlocks; ++blk) add_block(nt, blk, qf[blk], f);
                }
            }
            if (mask != kFull) {
#pragma unroll
                for (int nt = 0; nt < kCols; ++nt)
#pragma unroll
                    for (int j = 0; j < 2 * NT; ++j)
                        if (!((mask >> (nt * 8 + 2 * quad + (j & 1))) & 1)) s[nt][j] = -INFINITY;
            }
            // ---- softmax, in log2 ----
            float corr[NT];
            bool moved = false;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float top = -INFINITY;
#pragma unroll
                for (int nt = 0; nt < kCols; ++nt) top = fmaxf(top, fmaxf(s[nt][2 * n], s[nt][2 * n + 1]));
                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
                const float m_new = fmaxf(m[n], top * mul[n]);
                corr[n] = m_new > m[n] ? exp2_fast(m[n] - m_new) : 1.0f;
                moved |= m_new > m[n];
                m[n] = m_new;
                float sum = 0.0f;
#pragma unroll
                for (int nt = 0; nt < kCols; ++nt)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float& v = s[nt][2 * n + j];
                        v = exp2_fast(fmaf(v, mul[n], -m_new));
                        sum += v;
                    }
                l[n] = fmaf(l[n], corr[n], sum);
            }
            // ---- the weights times 2^15 as two f16 each, neighbouring positions in a pair: the value, and what it leaves ----
            uint32_t ph[kCols][NT], pl[kCols][NT];
#pragma unroll
            for (int nt = 0; nt < kCols; ++nt)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const float x = s[nt][2 * n] * 32768.0f, y = s[nt][2 * n + 1] * 32768.0f;
                    ph[nt][n] = pack_half2(x, y);
                    const float2 held = __half22float2(*reinterpret_cast<const __half2*>(&ph[nt][n]));
                    pl[nt][n] = pack_half2(x - held.x, y - held.y);
                }
            // ---- V's scale bytes, the largest and the smallest of them ----
            uint32_t vw[kCols][kWords];
            uint32_t high = 0, low = 0xFFFFFFFFu;  // in the upper byte of each half
#pragma unroll
            for (int nt = 0; nt < kCols; ++nt) {
                load_scale_pair<kBlocks>(vs + nt * 8 * kBlocks, vw[nt]);
#pragma unroll
                for (int i = 0; i < kWords; ++i) {
                    high = __vmaxu2(__vmaxu2(high, vw[nt][i]), vw[nt][i] << 8);
                    low = __vminu2(__vminu2(low, vw[nt][i]), vw[nt][i] << 8);
                }
            }
            uint32_t ends = max((high >> 8) & 0xFFu, high >> 24) << 16 | (255u - min((low >> 8) & 0xFFu, low >> 24));
            ends = __vmaxu2(ends, __shfl_xor_sync(0xFFFFFFFFu, ends, 1));
            ends = __vmaxu2(ends, __shfl_xor_sync(0xFFFFFFFFu, ends, 2));
            const int most = (int)(ends >> 16), least = 255 - (int)(ends & 0xFFFFu);
            // ---- second product, a window of V's scales at a time; nearly always one takes all of them ----
            int upper = max(ref, most);  // R
            int left = most < 255 && least > upper - kWindow ? -1 : 254;  // the largest byte that is still to be taken
            for (;;) {
                if (left >= 0) {
                    // acc, where it is not 0 yet, stays below 2^126 in the units of the lowest R
                    float size = 0.0f;
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int i = 0; i < D / 16; ++i)
#pragma unroll
                            for (int j = 0; j < 4; ++j) size = fmaxf(size, fabsf(acc[n][i][j]));
                    const uint32_t bits = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(size));
                    const int room = bits == 0 ? ref : min(max(252 - (int)(bits >> 23), 0), 126);
                    upper = take_window<D, POS>(st, lane, max(ref - room, 0), least, left);
#pragma unroll
                    for (int nt = 0; nt < kCols; ++nt) load_scale_pair<kBlocks>(vs + nt * 8 * kBlocks, vw[nt]);
                }
                if (__any_sync(0xFFFFFFFFu, moved || upper != ref)) {  // acc is in units of 2^(ref - 142)
                    const float down = exp2_fast((float)min(ref - upper, 126));
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const float c0 = __shfl_sync(0xFFFFFFFFu, corr[n], 8 * quad) * down;
                        const float c1 = __shfl_sync(0xFFFFFFFFu, corr[n], 8 * quad + 4) * down;
#pragma unroll
                        for (int i = 0; i < D / 16; ++i) {
                            acc[n][i][0] *= c0;
                            acc[n][i][1] *= c1;
                            acc[n][i][2] *= c0;
                            acc[n][i][3] *= c1;
                        }
                    }
                }
                ref = upper;
                const uint32_t shift = (uint32_t)(15 - ref) * 0x04000400u;
                // rows are elements of V, columns heads
                const uint8_t* vsm = st + C::kv_bytes;
#pragma unroll
                for (int half = 0; half < POS / 16; ++half) {
                    uint32_t f[2][kBlocks];
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int i = 0; i < kBlocks; ++i) {  // two bytes of a word to the exponents of two f16
                            const uint32_t two = __byte_perm(vw[2 * half + t][i / 2], 0u, i & 1 ? 0x4342 : 0x4140);
                            f[t][i] = two * 1024u + shift;
                        }
#pragma unroll
                    for (int blk = 0; blk < kBlocks; ++blk) {
                        uint32_t pb[NT][2], rest[NT][2];
#pragma unroll
                        for (int t = 0; t < 2; ++t) {
                            const uint32_t by = __byte_perm(f[t][blk / 2], f[t][kWords + blk / 2], blk & 1 ? 0x7632 : 0x5410);
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                pb[n][t] = mul_half2(ph[2 * half + t][n], by);
                                rest[n][t] = mul_half2(pl[2 * half + t][n], by);
                            }
                        }
                        // positions 2 quad, 2 quad + 1, 8 + 2 quad, 9 + 2 quad; elements 4 row .. 4 row + 3 of the block
                        uint32_t w[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            w[i] = *reinterpret_cast<const uint32_t*>(
                                vsm + in_block<D>(v_at, blk) + (16 * half + 4 * (i >> 1) + 8 * (i & 1)) * D);
                        uint32_t h[2][4];  // [positions low or high][element]: pairs of neighbouring positions
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            e4m3x4_to_half2(__byte_perm(w[2 * i], w[2 * i + 1], 0x5140), h[i][0], h[i][1]);
                            e4m3x4_to_half2(__byte_perm(w[2 * i], w[2 * i + 1], 0x7362), h[i][2], h[i][3]);
                        }
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            mma_f16(acc[n][2 * blk], h[0][0], h[0][1], h[1][0], h[1][1], pb[n][0], pb[n][1]);
                            mma_f16(acc[n][2 * blk + 1], h[0][2], h[0][3], h[1][2], h[1][3], pb[n][0], pb[n][1]);
                            mma_f16(acc[n][2 * blk], h[0][0], h[0][1], h[1][0], h[1][1], rest[n][0], rest[n][1]);
                            mma_f16(acc[n][2 * blk + 1], h[0][2], h[0][3], h[1][2], h[1][3], rest[n][0], rest[n][1]);
                        }
                    }
                }
                if (left < 0) break;
                moved = false;
#pragma unroll
                for (int n = 0; n < NT; ++n) corr[n] = 1.0f;
            }
        }
        stage = stage + 1 == C::stages ? 0 : stage + 1;

        if (cur.t + 1 == cur.t1) {  // the warp's last tile of this segment
            const bool begins = cur.t0 == 0, ends = cur.t1 == cur.nt;
            const int64_t seg = cur.b * groups + cur.g;
            const int sub = cur.g - (int)cur.head * p.row_groups;
            const int64_t head0 = cur.b * p.a.q_heads + (int64_t)cur.head * p.group + sub * C::rows;
            const int rows = min(C::rows, p.group - sub * C::rows);
            if (begins && lane == 0 && p.a.batch > kScanBatch) {
                const int64_t last = split_part(split, cur.base + kSegmentCost + cur.nt - 1);
                gstore_plain(p.meta + seg, ends ? make_int2(1, 0) : make_int2((int)part, (int)last), p.a.ww,
                             p.a.status);
            }
            const float unit = exp2f((float)(ref - 142));
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                l[n] += __shfl_xor_sync(0xFFFFFFFFu, l[n], 1);
                l[n] += __shfl_xor_sync(0xFFFFFFFFu, l[n], 2);
#pragma unroll
                for (int i = 0; i < D / 16; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[n][i][j] *= unit;
            }
            if (!ends) break;  // the warp's share ends inside: kept for the join with its neighbours
            if (begins) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const float inv = l[n] == 0.0f ? 0.0f : 1.0f / l[n];
                    if (p.a.lse && quad == 0 && n * 8 + row < rows)
                        gstore_plain(p.a.lse + head0 + n * 8 + row, (m[n] + log2f(l[n])) * kLn2, p.a.lw, p.a.status);
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        // rows as in acc: 8 n + 2 quad + {0, 1}; per block the elements 4 row .. 4 row + 3
                        const float inv_j = __shfl_sync(0xFFFFFFFFu, inv, 8 * quad + 4 * j);
                        const int r = n * 8 + 2 * quad + j;
                        if (r >= rows) continue;
#pragma unroll
                        for (int blk = 0; blk < kBlocks; ++blk)
                            gstore_plain(
                                reinterpret_cast<uint2*>(p.a.out + (head0 + r) * D + blk * 32 + 4 * row),
                                make_uint2(pack_out(p.a.q_bf16, acc[n][2 * blk][j] * inv_j, acc[n][2 * blk][2 + j] * inv_j),
                                           pack_out(p.a.q_bf16, acc[n][2 * blk + 1][j] * inv_j,
                                                    acc[n][2 * blk + 1][2 + j] * inv_j)),
                                p.a.ow, p.a.status);
                    }
                }
            } else {  // the rest of a segment that began before: slot 0
                put_piece<D, NT>(p, 2 * part, rows, lane, m, l, acc);
            }
            advance<POS>(p, cur, groups);
            if (!cur.done) {
                uint32_t raw[NT][D / 8];
                load_query<D, NT>(p, cur, lane, raw);
                start_segment(raw);
            }
        } else {
            ++cur.t;
        }
    }

    // ---- warps of this CTA that end inside the same segment: one piece of theirs ----
    cp_async_wait<0>();
    const bool open = !cur.done;
    const int sub = cur.g - (int)cur.head * p.row_groups, rows = min(C::rows, p.group - sub * C::rows);
    const int64_t open_seg = cur.b * groups + cur.g, open_slot = 2 * part + (cur.t0 == 0 ? 1 : 0);
    if (lane == 0) ends_in[warp] = open ? open_seg : -1;
    __syncthreads();
    int first = warp, run = 0;  // the warps first .. first + run - 1 share this warp's segment
    if (open) {
        while (first > 0 && ends_in[first - 1] == open_seg) --first;
        while (first + run < kWarps && ends_in[first + run] == open_seg) ++run;
        if (run == 1) {
            put_piece<D, NT>(p, open_slot, rows, lane, m, l, acc);
        } else {  // into the warp's own ring: the sums, then maxima and sums of p
            float* sums = reinterpret_cast<float*>(ring);
            float2* ml = reinterpret_cast<float2*>(ring + C::rows * D * 4);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                if (quad == 0) ml[n * 8 + row] = make_float2(m[n], l[n]);
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int blk = 0; blk < kBlocks; ++blk)
                        *reinterpret_cast<float4*>(sums + (n * 8 + 2 * quad + j) * D + blk * 32 + 4 * row) =
                            make_float4(acc[n][2 * blk][j], acc[n][2 * blk][2 + j], acc[n][2 * blk + 1][j],
                                        acc[n][2 * blk + 1][2 + j]);
            }
            if (warp == first && lane == 0) lead_slot[warp] = open_slot;
        }
    }
    __syncthreads();
    if (run > 1) {
        const uint8_t* rings = smem + first * C::warp_bytes;
        auto ml_of = [&](int w, int r) {
            return reinterpret_cast<const float2*>(rings + w * C::warp_bytes + C::rows * D * 4)[r];
        };
        // a warp's rows of the joint piece, which goes to the first warp's slot
        for (int r = warp - first; r < rows; r += run) {
            float top = -INFINITY, sum = 0.0f;
            for (int w = 0; w < run; ++w) top = fmaxf(top, ml_of(w, r).x);
            float2 o[D / 64];
#pragma unroll
            for (int k = 0; k < D / 64; ++k) o[k] = make_float2(0.0f, 0.0f);
            for (int w = 0; w < run; ++w) {
                const float2 ml = ml_of(w, r);
                const float f = ml.y != 0.0f ? exp2_fast(ml.x - top) : 0.0f;
                sum += ml.y * f;
                const float* src = reinterpret_cast<const float*>(rings + w * C::warp_bytes) + r * D + 2 * lane;
#pragma unroll
                for (int k = 0; k < D / 64; ++k) {
                    o[k].x += src[64 * k] * f;
                    o[k].y += src[64 * k + 1] * f;
                }
            }
            const int64_t at = lead_slot[first] * C::rows + r;
#pragma unroll
            for (int k = 0; k < D / 64; ++k)
                gstore_plain(reinterpret_cast<float2*>(p.part_o + at * D + 2 * lane + 64 * k), o[k], p.a.ww, p.a.status);
            if (lane == 0) gstore_plain(p.part_ml + at, make_float2(top, sum), p.a.ww, p.a.status);
        }
    }
}

// Second launch: zeros for the segments of empty sequences, and the pieces of
// those that more than one warp held (one for the warps first .. last - 1 of
// each CTA, one of warp last) joined in order.  W = 4: a CTA a (sequence, query
// head), every fourth piece by one warp.  W = 1: a CTA looks at p.join_segments
// segments, a lane each, and its warps (with those of the other blockIdx.y)
// take the query heads of those with work in turn.  Latency is all there is to it, so where the pieces are follows from
// (first, last) alone, and a warp has its maxima, sums and elements of kEach
// pieces on their way at once.
template <int D, int NT, int W>
__global__ void __launch_bounds__(kJoinThreads) cache_attention_join_kernel(const Params p) {
    using C = Config<D, NT>;
    constexpr int kVecs = D / 64, kEach = 4;
    __shared__ float2 ml_of[W];
    __shared__ float2 sums[W][W > 1 ? D / 2 : 1];
    grid_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int groups = p.a.c.heads * p.row_groups;
    const int64_t segments = p.a.batch * groups;
    int64_t seg, seg0 = 0;
    int only_row = 0;  // W = 4: the one row of the segment
    if constexpr (W > 1) {
        const uint32_t b = blockIdx.x / (uint32_t)p.a.q_heads, head = blockIdx.x - b * (uint32_t)p.a.q_heads;
        const uint32_t kv_head = head / (uint32_t)p.group, in = head - kv_head * (uint32_t)p.group;
        const uint32_t sub = in / C::rows;
        seg = (int64_t)b * groups + kv_head * (uint32_t)p.row_groups + sub;
        only_row = (int)(in - sub * C::rows);
    } else {
        seg0 = (int64_t)blockIdx.x * p.join_segments;
        seg = seg0 + lane;
    }
    const bool own = W > 1 || (lane < p.join_segments && seg < segments);
    const int64_t b = own ? (uint32_t)seg / (uint32_t)groups : 0u;  // there are fewer than 2^31 of them
    int2 parts = make_int2(1, 0);  // first and last warp: (0, -1) of an empty sequence, first > last >= 0 nothing to do
    if (p.a.batch <= kScanBatch) {
        // The lengths are complete in L2: this launch began after every CTA of the first one had passed its own wait
        // for what ran before.
        const Costs costs = costs_of<C::pos, true>(p.a, lane);
        const uint32_t before = __shfl_sync(0xFFFFFFFFu, costs.upto - costs.mine, (int)b);
        const int len = __shfl_sync(0xFFFFFFFFu, costs.len, (int)b), nt = (len + C::pos - 1) / C::pos;
        const int64_t total = costs.total * groups;
        if (own && len == 0) parts = make_int2(0, -1);
        if (own && len > 0) {
            const Split split = make_split(min(p.parts, total), total);
            const int64_t tiles = (int64_t)before * groups + (seg - b * groups) * (nt + kSegmentCost) + kSegmentCost;
            const int2 held = make_int2((int)split_part(split, tiles), (int)split_part(split, tiles + nt - 1));
            if (held.x < held.y) parts = held;
        }
    }
    grid_wait_prerequisites();
    if (p.a.batch > kScanBatch && own) parts = length_of(p.a, b) == 0 ? make_int2(0, -1) : p.meta[seg];

    // one query head, row r of its segment
    auto join = [&](const int2 held, int64_t unit, int r) {
        const int first_cta = held.x / kWarps;
        const int pieces = held.y < 0 ? 0 : (held.y - 1) / kWarps - first_cta + 2;
        auto slot_of = [&](int i) {
            const int64_t slot =
                i == 0 ? 2 * (int64_t)held.x + 1 : 2 * (int64_t)(i + 1 < pieces ? (first_cta + i) * kWarps : held.y);
            return slot * C::rows + r;
        };
        float top = -INFINITY, sum = 0.0f;
        float2 o[kVecs];
#pragma unroll
        for (int k = 0; k < kVecs; ++k) o[k] = make_float2(0.0f, 0.0f);
        for (int i0 = W == 1 ? 0 : warp; i0 < pieces; i0 += kEach * W) {
            float2 ml[kEach], v[kEach][kVecs];
#pragma unroll
            for (int j = 0; j < kEach; ++j) {
                const bool on = i0 + j * W < pieces;
                const int64_t at = slot_of(on ? i0 + j * W : i0);
                ml[j] = on ? p.part_ml[at] : make_float2(-INFINITY, 0.0f);
#pragma unroll
                for (int k = 0; k < kVecs; ++k)
                    v[j][k] = on ? *reinterpret_cast<const float2*>(p.part_o + at * D + 2 * lane + 64 * k)
                                 : make_float2(0.0f, 0.0f);
            }
            float most = top;
#pragma unroll
            for (int j = 0; j < kEach; ++j) most = fmaxf(most, ml[j].x);
            const float keep = sum != 0.0f ? exp2_fast(top - most) : 0.0f;
            top = most;
            sum *= keep;
#pragma unroll
            for (int k = 0; k < kVecs; ++k) {
                o[k].x *= keep;
                o[k].y *= keep;
            }
#pragma unroll
            for (int j = 0; j < kEach; ++j) {
                const float weight = ml[j].y != 0.0f ? exp2_fast(ml[j].x - top) : 0.0f;
                sum += ml[j].y * weight;
#pragma unroll
                for (int k = 0; k < kVecs; ++k) {
                    o[k].x += v[j][k].x * weight;
                    o[k].y += v[j][k].y * weight;
                }
            }
        }
        uint16_t* const out = p.a.out + unit * D;
        if constexpr (W > 1) {
            if (lane == 0) ml_of[warp] = make_float2(top, sum);
#pragma unroll
            for (int k = 0; k < kVecs; ++k) sums[warp][lane + 32 * k] = o[k];
            __syncthreads();
            float weight[W];
#pragma unroll
            for (int w = 0; w < W; ++w) top = fmaxf(top, ml_of[w].x);
            sum = 0.0f;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                weight[w] = ml_of[w].y != 0.0f ? exp2_fast(ml_of[w].x - top) : 0.0f;
                sum += ml_of[w].y * weight[w];
            }
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            for (int d = threadIdx.x; d < D / 2; d += kJoinThreads) {
                float2 v = make_float2(0.0f, 0.0f);
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    v.x += sums[w][d].x * weight[w];
                    v.y += sums[w][d].y * weight[w];
                }
                gstore_plain(reinterpret_cast<uint32_t*>(out + 2 * d), pack_out(p.a.q_bf16, v.x * inv, v.y * inv),
                             p.a.ow, p.a.status);
            }
        } else {
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
            for (int k = 0; k < kVecs; ++k)
                gstore_plain(reinterpret_cast<uint32_t*>(out + 2 * lane + 64 * k),
                             pack_out(p.a.q_bf16, o[k].x * inv, o[k].y * inv), p.a.ow, p.a.status);
        }
        if (p.a.lse && lane == 0 && (W == 1 || warp == 0))
            gstore_plain(p.a.lse + unit, (top + log2f(sum)) * kLn2, p.a.lw, p.a.status);
    };

    const bool work = parts.y < 0 || parts.x <= parts.y;
    if constexpr (W > 1) {
        if (work) join(parts, blockIdx.x, only_row);
    } else {
        int turn = 0;  // of the warps
        for (uint32_t left = __ballot_sync(0xFFFFFFFFu, work); left != 0; left &= left - 1) {
            const int from = __ffs(left) - 1;
            const int2 held = make_int2(__shfl_sync(0xFFFFFFFFu, parts.x, from), __shfl_sync(0xFFFFFFFFu, parts.y, from));
            const int64_t at = __shfl_sync(0xFFFFFFFFu, b, from);
            const int g = (int)(seg0 + from - at * groups);
            const int kv_head = p.row_groups == 1 ? g : g / p.row_groups, sub = g - kv_head * p.row_groups;
            const int rows = min(C::rows, p.group - sub * C::rows);
            const int64_t unit = at * p.a.q_heads + (int64_t)kv_head * p.group + sub * C::rows;
            for (int r = ((warp - turn) & (kJoinWarps - 1)) + kJoinWarps * blockIdx.y; r < rows; r += kJoinWarps * gridDim.y)
                join(held, unit + r, r);
            turn = (turn + rows) & (kJoinWarps - 1);
        }
    }
}

template <int D, int NT>
int64_t ctas_of(int sm_count) {
    return (int64_t)sm_count * Config<D, NT>::ctas_per_sm;
}

template <int D, int NT>
int64_t workspace_of(int64_t segments, int sm_count) {
    const int64_t slots = 2 * kWarps * ctas_of<D, NT>(sm_count) * Config<D, NT>::rows;
    return slots * (D * 4 + 8) + segments * 8;
}

template <int D, int NT>
int launch_typed(const CacheAttentionArgs& a, int sm_count, cudaStream_t stream) {
    using C = Config<D, NT>;
    auto kernel = cache_attention_kernel<D, NT>;
    static OptIn done;
    if (int rc = opt_in(reinterpret_cast<const void*>(kernel), C::smem, true, done)) return rc;
    Params p;
    p.a = a;
    p.group = a.q_heads / a.c.heads;
    p.row_groups = (p.group + C::rows - 1) / C::rows;
    p.join_segments = 1;
    const int64_t segments = a.batch * a.c.heads * p.row_groups;
    // no more warps than the longest lengths that the table allows would use
    const int64_t most = segments * (((a.max_pages << a.c.page_shift) + C::pos - 1) / C::pos + kSegmentCost);
    const int64_t ctas = ctas_of<D, NT>(sm_count), slots = 2 * kWarps * ctas * C::rows;
    const int64_t grid = most < ctas * kWarps ? (most + kWarps - 1) / kWarps : ctas;
    p.parts = grid * kWarps;
    p.part_o = static_cast<float*>(a.workspace);
    p.part_ml = reinterpret_cast<float2*>(p.part_o + slots * D);
    p.meta = reinterpret_cast<int2*>(p.part_ml + slots);

    cudaLaunchConfig_t cfg = {};
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = C::smem;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
    if (e == cudaSuccess) {
        // Few heads are in many pieces each and get a CTA, many in few pieces a warp.  64 ragged sequences, 2048 heads:
        // 48.7 us in all with a warp, 8 long ones, 128 heads: 60 with a CTA (80 and 72 us the other way round with an
        // earlier join).  At most one segment a warp of the first launch is split: where there are more segments than
        // those, a CTA looks at several.
        const int64_t units = a.batch * a.q_heads;
        const bool single = units >= 8 * (int64_t)sm_count;
        const int64_t each = std::max(segments / p.parts, (int64_t)(kJoinWarps - 1) / p.group + 1);
        p.join_segments = (int)std::min(each, (int64_t)32);
        cfg.gridDim = dim3((unsigned)(single ? (segments + p.join_segments - 1) / p.join_segments : units));
        if (single && each == 1) cfg.gridDim.y = (unsigned)((std::min(p.group, (int)C::rows) + kJoinWarps - 1) / kJoinWarps);
        cfg.blockDim = dim3(kJoinThreads);
        cfg.dynamicSmemBytes = 0;
        e = single ? cudaLaunchKernelEx(&cfg, cache_attention_join_kernel<D, NT, 1>, p)
                   : cudaLaunchKernelEx(&cfg, cache_attention_join_kernel<D, NT, kJoinWarps>, p);
    }
    if (e == cudaSuccess) e = cudaGetLastError();
    if (e != cudaSuccess) {
        set_last_error("cache_attention_kernel launch", (int)e);
        return MXFP8_ERR_CUDA;
    }
    return MXFP8_OK;
}

}  // namespace

int64_t cache_attention_workspace(const CacheShape& c, int64_t batch, int q_heads, int sm_count) {
    const int group = q_heads / c.heads;
    const int nt = row_tiles(c.dim, group);
    const int64_t segments = batch * c.heads * ((group + 8 * nt - 1) / (8 * nt));
    switch (c.dim) {
        case 64: return nt == 1 ? workspace_of<64, 1>(segments, sm_count) : workspace_of<64, 2>(segments, sm_count);
        case 128: return nt == 1 ? workspace_of<128, 1>(segments, sm_count) : workspace_of<128, 2>(segments, sm_count);
        case 192: return workspace_of<192, 1>(segments, sm_count);
        default: return workspace_of<256, 1>(segments, sm_count);
    }
}

int launch_cache_attention(const CacheAttentionArgs& a, int sm_count, cudaStream_t stream) {
    const int nt = row_tiles(a.c.dim, a.q_heads / a.c.heads);
    switch (a.c.dim) {
        case 64: return nt == 1 ? launch_typed<64, 1>(a, sm_count, stream) : launch_typed<64, 2>(a, sm_count, stream);
        case 128: return nt == 1 ? launch_typed<128, 1>(a, sm_count, stream) : launch_typed<128, 2>(a, sm_count, stream);
        case 192: return launch_typed<192, 1>(a, sm_count, stream);
        default: return launch_typed<256, 1>(a, sm_count, stream);
    }
}

}  // namespace mxfp8
