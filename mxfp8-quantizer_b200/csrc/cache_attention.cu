// cache_attention.cu -- one query token per sequence against the paged MXFP8
// cache: o = sum_j p_j v_j / sum_j p_j, p_j = exp(scale q . k_j).
//
// Every cached byte is read once and used by the G query heads that share a KV
// head: 4 G operations for 1 + 1/32 bytes, so HBM bandwidth bounds it as long
// as the arithmetic keeps up.  Tensor cores do both products (mma m16n8k16,
// f16 operands, f32 sums): an E4M3 value is exact in f16, so the payload needs
// one conversion and the scales stay outside the products:
//   q . k_j = sum over blocks of 32 of  2^(sk - 127) (q . payload), a sum per
//     block scaled in f32.  q is brought to f16 with one power of two a head
//     (largest element in [2^14, 2^15)): a bf16 or fp16 value is exact there
//     down to 2^-38 of the head's largest.
//   sum_j p_j v_j: p_j 2^(sv - 127) is the operand, as p_j 2^(sv - R + 15) in
//     f16 with R the largest V scale byte met so far: 2^-12 of relative error
//     for every term within 29 binades of the largest possible one, terms below
//     lose bits gradually; the accumulator is rescaled when R grows.
// The m16n8k16 shapes are used because a decode step has at most 16 rows of
// queries: a 128-row tcgen05 tile would be empty to 7/8 and would want K and V
// converted into shared memory first.
//
// Work: tiles of 64 positions, of all sequences and KV heads in a row, are
// split evenly over the CTAs whatever the lengths are.  A warp owns 16
// positions of every tile: it fetches them (cp.async into a ring of its own,
// no block-wide barriers), computes the scores with heads as rows and positions
// as columns, which is the layout the second product takes its operand in, and
// keeps its own running maximum and sums.  Where a CTA leaves a (sequence, KV
// head) its warps join; if it did not hold all of its tiles, the unscaled sums go
// to the workspace, and a second launch joins those.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>

#include "../../include/mxfp8_cache.h"
#include "cache.cuh"
#include "launch.h"
#include "ptx.cuh"

namespace mxfp8 {

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kWarpPos = 16;                  // positions of a warp in a tile
constexpr int kTilePos = kWarps * kWarpPos;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// Heads in groups of 8 * NT rows: 16 where that saves a second pass over K and
// V and the accumulators fit the registers.
inline int row_tiles(int dim, int group) { return group > 8 && dim <= 128 ? 2 : 1; }

template <int D, int NT>
struct Config {
    static constexpr int rows = 8 * NT;
    static constexpr int kv_bytes = kWarpPos * D;             // K (or V) payload of a warp's positions
    static constexpr int sc_bytes = kWarpPos * D / 32;
    static constexpr int stage_bytes = 2 * kv_bytes + 2 * sc_bytes;
    static constexpr int stages = D <= 64 ? 6 : D <= 128 ? 4 : 3;
    static constexpr int f_floats = D / 32 * kWarpPos;        // scale factors of a warp's positions
    static constexpr int warp_bytes = stages * stage_bytes + 2 * f_floats * 4;
    static constexpr int join_off = kWarps * warp_bytes;
    static constexpr int ml_off = join_off + rows * D * 4;    // then m and l of every warp and row
    static constexpr int smem = ml_off + kWarps * rows * 8;
    static constexpr int ctas_per_sm = smem * 3 <= 225 * 1024 ? 3 : 2;
};

struct Params {
    CacheAttentionArgs a;
    int group;        // query heads of a KV head
    int row_groups;   // ceil(group / rows)
    int64_t grid;     // CTAs
    float* part_o;    // (2 * grid, rows, D): unscaled sums of the pieces
    float2* part_ml;  // (2 * grid, rows): running maximum (log2) and sum
    int2* meta;       // (batch * heads * row_groups): first and last CTA of a split segment
};

// A place in the sequence of all tiles: sequence b, head group g (KV head and
// row group), tile t of nt.
struct Cursor {
    int64_t b;
    int g, t, nt, len;
};

__device__ __forceinline__ int tiles_of(int len) { return (len + kTilePos - 1) / kTilePos; }

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, d));
    return v;
}

__device__ __forceinline__ int length_of(const CacheAttentionArgs& a, int64_t b) {
    return (int)visible_length(a.lengths[b], a.max_pages, a.c.page_shift);
}

// To the next tile; sequences without tiles are passed over.
__device__ __forceinline__ void advance(const Params& p, Cursor& c, int groups) {
    if (++c.t < c.nt) return;
    c.t = 0;
    if (++c.g < groups) return;
    c.g = 0;
    do {
        if (++c.b >= p.a.batch) {
            c.nt = 0;
            return;
        }
        c.len = length_of(p.a, c.b);
        c.nt = tiles_of(c.len);
    } while (c.nt == 0);
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

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
    const __half2 t = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&t);
}

// Shared memory of a warp's 16 rows of D bytes: 32-byte groups of a row are
// permuted so that the four rows that one access phase reads (K: rows r .. r +
// 3, V: the same after v_place) fall on different banks.
template <int D>
__device__ __forceinline__ uint32_t group_at(int row, int group) {
    const int key = D % 128 == 0 ? (row & 3) : ((row >> 1) & 1);
    return (uint32_t)(row * D + ((group ^ key) << 5));
}
// Row that position j of V is kept in: the positions 2c + i, c = 0 .. 3, that
// a phase of the second product reads are neighbours.
__device__ __forceinline__ int v_place(int j) { return (j >> 1) | ((j & 1) << 3); }

// Positions 16 w .. 16 w + 15 of the cursor's tile: the cache row of position
// lane (kNoRow where there is none), for lanes below 16.
__device__ __forceinline__ int64_t row_of_lane(const Params& p, const Cursor& c, int warp, int lane) {
    if (c.nt == 0 || lane >= kWarpPos) return kNoRow;
    const int at = c.t * kTilePos + warp * kWarpPos + lane;
    if (at >= c.len) return kNoRow;
    const int64_t page = table_page(p.a.table, p.a.table_stride, p.a.max_pages, c.b, at, p.a.c.page_shift);
    const int64_t row = cache_row(p.a.c, page, c.g / p.row_groups, at & ((1 << p.a.c.page_shift) - 1));
    if (row == kNoRow && p.a.status) atomicOr(p.a.status, kErrCacheIndex);
    return row;
}

// Fetch those positions into a stage: payloads 16 bytes a lane, scales four
// bytes a lane (two positions' scale bytes are 4, 8, 12 or 16 contiguous ones:
// pages hold an even number of positions).  Absent positions are zeros.
template <int D>
__device__ __forceinline__ void fetch(const Params& p, uint32_t stage, int64_t my_row, int lane) {
    constexpr int kChunks = D / 16;  // of a row
    constexpr int kKv = kWarpPos * D;
#pragma unroll
    for (int i = 0; i < kKv / 512; ++i) {
        const int idx = i * 32 + lane;
        const int j = idx / kChunks, ch = idx - j * kChunks;
        const int64_t row = __shfl_sync(0xFFFFFFFFu, my_row, j);
        const bool on = row != kNoRow;
        const int64_t off = on ? row * D + ch * 16 : 0;
        cp_async16(stage + group_at<D>(j, ch >> 1) + (ch & 1) * 16, p.a.k + off, on);
        cp_async16(stage + kKv + group_at<D>(v_place(j), ch >> 1) + (ch & 1) * 16, p.a.v + off, on);
    }
    constexpr int kPair = D / 64;    // 4-byte pieces of two positions' scales
    const int pair = lane / kPair, in = lane - pair * kPair;
    const int64_t even = __shfl_sync(0xFFFFFFFFu, my_row, (2 * pair) & 15);
    if (lane < kWarpPos / 2 * kPair) {
        const bool on = even != kNoRow;
        const int64_t off = on ? even * (D / 32) + in * 4 : 0;
        cp_async4(stage + 2 * kKv + lane * 4, p.a.k_scales + off, on);
        cp_async4(stage + 2 * kKv + kWarpPos * D / 32 + lane * 4, p.a.v_scales + off, on);
    }
}

// Query rows of a head group as MMA operands, and what a score is multiplied
// by: scale * log2(e) * the power of two taken out of the row.
template <int D, int NT>
__device__ __forceinline__ void load_query(const Params& p, const Cursor& c, int lane, uint32_t (&qf)[D / 16][2 * NT],
                                           float (&mul)[NT]) {
    const int sub = c.g % p.row_groups, kv_head = c.g / p.row_groups;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int in = sub * Config<D, NT>::rows + n * 8 + (lane >> 2);
        const bool on = in < p.group;
        const uint16_t* src = p.a.q + c.b * p.a.q_batch + (int64_t)(kv_head * p.group + (on ? in : 0)) * p.a.q_head;
        const bool vec = (reinterpret_cast<uintptr_t>(src) & 15) == 0;
        uint32_t w[D / 32][4];
#pragma unroll
        for (int blk = 0; blk < D / 32; ++blk) {
            const uint4 t = load8(src + blk * 32 + (lane & 3) * 8, vec);
            w[blk][0] = t.x; w[blk][1] = t.y; w[blk][2] = t.z; w[blk][3] = t.w;
        }
        float v[D / 32][8];
        float amax = 0.0f;
#pragma unroll
        for (int blk = 0; blk < D / 32; ++blk) {
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const uint32_t pair = on ? w[blk][e / 2] : 0u;
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
        const float down = __uint_as_float((uint32_t)(127 + 14 - e) << 23);  // 2^(14 - e)
        mul[n] = amax == 0.0f ? 0.0f : p.a.scale * kLog2e * __uint_as_float((uint32_t)(127 - 14 + e) << 23);
#pragma unroll
        for (int blk = 0; blk < D / 32; ++blk)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int r = 0; r < 2; ++r)
                    qf[blk * 2 + h][n * 2 + r] =
                        pack_half2(v[blk][4 * h + 2 * r] * down, v[blk][4 * h + 2 * r + 1] * down);
    }
}

template <int D, int NT>
__global__ void __launch_bounds__(kThreads, Config<D, NT>::ctas_per_sm) cache_attention_kernel(const Params p) {
    using C = Config<D, NT>;
    constexpr int kBlocks = D / 32;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int64_t scan_s[kWarps];
    __shared__ int64_t found_b, found_base;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = lane >> 2, quad = lane & 3;
    const int groups = p.a.c.heads * p.row_groups;

    grid_wait_prerequisites();
    // ---- this CTA's share of all tiles, and where it begins ----
    const int64_t per = (p.a.batch + kThreads - 1) / kThreads;
    const int64_t b0 = min(p.a.batch, per * threadIdx.x), b1 = min(p.a.batch, b0 + per);
    int64_t mine = 0;
    for (int64_t b = b0; b < b1; ++b) {
        mine += tiles_of(length_of(p.a, b));
        if (blockIdx.x == 0 && p.a.status && (int64_t)p.a.lengths[b] > (p.a.max_pages << p.a.c.page_shift))
            atomicOr(p.a.status, kErrCacheIndex);
    }
    int64_t upto = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int64_t o = __shfl_up_sync(0xFFFFFFFFu, upto, d);
        if (lane >= d) upto += o;
    }
    if (lane == 31) scan_s[warp] = upto;
    __syncthreads();
    int64_t before = 0, tiles = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += scan_s[w];
        tiles += scan_s[w];
    }
    const int64_t total = tiles * groups;
    const int64_t parts = min(p.grid, total);
    const int64_t cta = blockIdx.x;
    if (cta >= parts) return;
    const int64_t x0 = split_begin(cta, parts, total), x1 = split_begin(cta + 1, parts, total);
    int64_t at = (before + upto - mine) * groups;  // first tile of this thread's first sequence
    if (at <= x0 && x0 < at + mine * groups) {
        int64_t b = b0;
        for (;; ++b) {
            const int64_t n = (int64_t)tiles_of(length_of(p.a, b)) * groups;
            if (x0 < at + n) break;
            at += n;
        }
        found_b = b;
        found_base = at;
    }
    __syncthreads();
    Cursor cur;  // the tile that is computed
    cur.b = found_b;
    cur.len = length_of(p.a, cur.b);
    cur.nt = tiles_of(cur.len);
    int64_t seg0 = found_base + (x0 - found_base) / cur.nt * cur.nt;  // first tile of the segment
    cur.g = (int)((x0 - found_base) / cur.nt);
    cur.t = (int)(x0 - seg0);

    uint8_t* const ring = smem + warp * C::warp_bytes;
    const uint32_t ring_u = smem_u32(ring);
    float* const kf = reinterpret_cast<float*>(ring + C::stages * C::stage_bytes);  // [block][position]
    float* const vf = kf + C::f_floats;

    // ---- fetch ahead: `next` is the tile whose rows are looked up in my_row ----
    Cursor next = cur;
    int64_t next_x = x0;
    int64_t my_row = row_of_lane(p, next, warp, lane);
    uint32_t present = 0;  // lane s: which positions of stage s are there
    auto issue = [&](int stage) {
        if (next_x < x1) {
            fetch<D>(p, ring_u + stage * C::stage_bytes, my_row, lane);
            const uint32_t mask = __ballot_sync(0xFFFFFFFFu, my_row != kNoRow);
            if (lane == stage) present = mask;
            ++next_x;
            if (next_x < x1) {
                advance(p, next, groups);
                my_row = row_of_lane(p, next, warp, lane);
            }
        }
        cp_async_commit();
    };
#pragma unroll
    for (int s = 0; s < C::stages - 1; ++s) issue(s);

    uint32_t qf[D / 16][2 * NT];
    float mul[NT], m[NT], l[NT];
    float acc[NT][D / 16][4];
    uint32_t ref = 0;  // R: the largest V scale byte so far
    bool fresh = true;

    int stage = 0;
    for (int64_t x = x0; x < x1; ++x) {
        if (fresh) {
            load_query<D, NT>(p, cur, lane, qf, mul);
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
            fresh = false;
        }
        cp_async_wait<C::stages - 2>();
        __syncwarp();  // also: the stage before this one is read, it can be filled again
        const uint32_t mask = __shfl_sync(0xFFFFFFFFu, present, stage) & 0xFFFFu;
        issue(stage == 0 ? C::stages - 1 : stage - 1);
        const uint8_t* st = ring + stage * C::stage_bytes;
        if (mask != 0) {
            // ---- scale factors: f32 of K's, and the largest byte of V's ----
            constexpr int kPer = kWarpPos * kBlocks / 32;  // bytes a lane
            const uint8_t* ks = st + 2 * C::kv_bytes;
            const uint8_t* vs = ks + C::sc_bytes;
            uint32_t vb[kPer], top = 0;
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const int idx = i * 32 + lane, j = idx / kBlocks, blk = idx - j * kBlocks;
                kf[blk * kWarpPos + j] = ue8m0_value(ks[idx]);
                vb[i] = (mask >> j) & 1 ? vs[idx] : 0u;
                if (vb[i] != 255u) top = max(top, vb[i]);
            }
            top = __reduce_max_sync(0xFFFFFFFFu, top);
            if (top > ref) {
                const float down = exp2_fast(-(float)(top - ref));  // acc is in units of 2^(ref - 142)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < D / 16; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j) acc[n][i][j] *= down;
                ref = top;
            }
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const int idx = i * 32 + lane, j = idx / kBlocks, blk = idx - j * kBlocks;
                const int e = (int)vb[i] - (int)ref + 15 + 127;
                const float f = __uint_as_float(vb[i] == 255u ? 0x7FC00000u : (uint32_t)max(e, 0) << 23);
                vf[blk * kWarpPos + j] = f;
            }
            __syncwarp();

            // ---- scores: rows are heads, columns positions 8 nt + 2 quad + {0, 1} ----
            float s[2][4];
#pragma unroll
            for (int nt = 0; nt < 2; ++nt) {
#pragma unroll
                for (int j = 0; j < 4; ++j) s[nt][j] = 0.0f;
#pragma unroll
                for (int blk = 0; blk < kBlocks; ++blk) {
                    const uint2 w = *reinterpret_cast<const uint2*>(st + group_at<D>(nt * 8 + row, blk) + quad * 8);
                    uint32_t b0, b1, b2, b3;
                    e4m3x4_to_half2(w.x, b0, b1);
                    e4m3x4_to_half2(w.y, b2, b3);
                    float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    if constexpr (NT == 1) {
                        mma_f16(d, qf[2 * blk][0], 0u, qf[2 * blk][1], 0u, b0, b1);
                        mma_f16(d, qf[2 * blk + 1][0], 0u, qf[2 * blk + 1][1], 0u, b2, b3);
                    } else {
                        mma_f16(d, qf[2 * blk][0], qf[2 * blk][2], qf[2 * blk][1], qf[2 * blk][3], b0, b1);
                        mma_f16(d, qf[2 * blk + 1][0], qf[2 * blk + 1][2], qf[2 * blk + 1][1], qf[2 * blk + 1][3], b2,
                                b3);
                    }
                    const float2 f = *reinterpret_cast<const float2*>(kf + blk * kWarpPos + nt * 8 + 2 * quad);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        s[nt][2 * n] = fmaf(d[2 * n], f.x, s[nt][2 * n]);
                        s[nt][2 * n + 1] = fmaf(d[2 * n + 1], f.y, s[nt][2 * n + 1]);
                    }
                }
            }
            // ---- softmax, in log2 ----
            float corr[NT];
            bool moved = false;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float top_s = -INFINITY;
#pragma unroll
                for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float& v = s[nt][2 * n + j];
                        v = (mask >> (nt * 8 + 2 * quad + j)) & 1 ? v * mul[n] : -INFINITY;
                        top_s = fmaxf(top_s, v);
                    }
                top_s = fmaxf(top_s, __shfl_xor_sync(0xFFFFFFFFu, top_s, 1));
                top_s = fmaxf(top_s, __shfl_xor_sync(0xFFFFFFFFu, top_s, 2));
                const float m_new = fmaxf(m[n], top_s);
                corr[n] = exp2_fast(m[n] - m_new);
                moved |= m_new > m[n];
                m[n] = m_new;
                l[n] *= m_new > -INFINITY ? corr[n] : 1.0f;
#pragma unroll
                for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float& v = s[nt][2 * n + j];
                        v = exp2_fast(v - m_new);
                        l[n] += v;
                    }
            }
            if (__any_sync(0xFFFFFFFFu, moved)) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const float c0 = __shfl_sync(0xFFFFFFFFu, corr[n], 8 * quad);
                    const float c1 = __shfl_sync(0xFFFFFFFFu, corr[n], 8 * quad + 4);
#pragma unroll
                    for (int i = 0; i < D / 16; ++i) {
                        acc[n][i][0] *= c0;
                        acc[n][i][1] *= c1;
                        acc[n][i][2] *= c0;
                        acc[n][i][3] *= c1;
                    }
                }
            }
            // ---- second product: rows are elements of V, columns heads ----
            const uint8_t* vsm = st + C::kv_bytes;
#pragma unroll
            for (int blk = 0; blk < kBlocks; ++blk) {
                const float2 f0 = *reinterpret_cast<const float2*>(vf + blk * kWarpPos + 2 * quad);
                const float2 f1 = *reinterpret_cast<const float2*>(vf + blk * kWarpPos + 8 + 2 * quad);
                uint32_t pb[NT][2];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    pb[n][0] = pack_half2(s[0][2 * n] * f0.x, s[0][2 * n + 1] * f0.y);
                    pb[n][1] = pack_half2(s[1][2 * n] * f1.x, s[1][2 * n + 1] * f1.y);
                }
                // positions 2 quad, 2 quad + 1, 8 + 2 quad, 9 + 2 quad; elements 4 row .. 4 row + 3 of the block
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    w[i] = *reinterpret_cast<const uint32_t*>(vsm + group_at<D>(quad + 4 * (i >> 1) + 8 * (i & 1), blk) +
                                                              4 * row);
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
                }
            }
        }
        stage = stage + 1 == C::stages ? 0 : stage + 1;

        // ---- the last tile of a segment, or of this CTA: join the warps ----
        const bool ends = cur.t + 1 == cur.nt;
        if (ends || x + 1 == x1) {
            float* join = reinterpret_cast<float*>(smem + C::join_off);           // [row][D]
            float2* ml = reinterpret_cast<float2*>(smem + C::ml_off);             // [warp][row]
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                l[n] += __shfl_xor_sync(0xFFFFFFFFu, l[n], 1);
                l[n] += __shfl_xor_sync(0xFFFFFFFFu, l[n], 2);
                if (quad == 0) ml[warp * C::rows + n * 8 + row] = make_float2(m[n], l[n]);
            }
            __syncthreads();
            // acc holds rows (heads) 2 quad, 2 quad + 1: their joint maxima and this warp's factors
            float fac[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int r = n * 8 + 2 * quad + j;
                    float all = -INFINITY;
#pragma unroll
                    for (int w = 0; w < kWarps; ++w) all = fmaxf(all, ml[w * C::rows + r].x);
                    const float2 own = ml[warp * C::rows + r];
                    fac[n][j] = own.y == 0.0f ? 0.0f : exp2_fast(own.x - all) * exp2f((float)((int)ref - 142));
                }
            for (int w = 0; w < kWarps; ++w) {
                if (warp == w) {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int i = 0; i < D / 16; ++i)
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                // tile i of block i / 2: elements 4 row + 2 (i % 2) + (j / 2)
                                const int d = (i >> 1) * 32 + 4 * row + 2 * (i & 1) + (j >> 1);
                                float* dst = join + (n * 8 + 2 * quad + (j & 1)) * D + d;
                                const float v = acc[n][i][j] * fac[n][j & 1];
                                *dst = w == 0 ? v : *dst + v;
                            }
                }
                __syncthreads();
            }
            const bool whole = ends && x0 <= seg0;
            // slot 1: the segment begins in this CTA; slot 0: it began before
            const int64_t slot = 2 * cta + (x0 <= seg0 ? 1 : 0);
            const int64_t seg = cur.b * groups + cur.g;
            if (threadIdx.x == 0 && x0 <= seg0)
                gstore_plain(p.meta + seg,
                             whole ? make_int2(0, -1)
                                   : make_int2((int)cta, (int)split_part(seg0 + cur.nt - 1, parts, total)),
                             p.a.ww, p.a.status);
            const int sub = cur.g % p.row_groups;
            const int64_t head0 = (int64_t)(cur.g / p.row_groups) * p.group + sub * C::rows;
            const int rows = min(C::rows, p.group - sub * C::rows);
            for (int r = warp; r < rows; r += kWarps) {
                float all = -INFINITY, sum = 0.0f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) all = fmaxf(all, ml[w * C::rows + r].x);
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    const float2 v = ml[w * C::rows + r];
                    if (v.y != 0.0f) sum += v.y * exp2_fast(v.x - all);
                }
                if (whole) {
                    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                    const int64_t o = (cur.b * p.a.q_heads + head0 + r) * D;
                    for (int d = 2 * lane; d < D; d += 64) {
                        const float v0 = join[r * D + d] * inv, v1 = join[r * D + d + 1] * inv;
                        uint32_t h;
                        if (p.a.q_bf16) {
                            const __nv_bfloat162 t = __floats2bfloat162_rn(v0, v1);
                            h = *reinterpret_cast<const uint32_t*>(&t);
                        } else {
                            h = pack_half2(v0, v1);
                        }
                        gstore_plain(reinterpret_cast<uint32_t*>(p.a.out + o + d), h, p.a.ow, p.a.status);
                    }
                    if (p.a.lse && lane == 0)
                        gstore_plain(p.a.lse + cur.b * p.a.q_heads + head0 + r, (all + log2f(sum)) * kLn2, p.a.lw,
                                     p.a.status);
                } else {
                    float* o = p.part_o + (slot * C::rows + r) * D;
                    for (int d = 2 * lane; d < D; d += 64)
                        gstore_plain(reinterpret_cast<float2*>(o + d),
                                     make_float2(join[r * D + d], join[r * D + d + 1]), p.a.ww, p.a.status);
                    if (lane == 0)
                        gstore_plain(p.part_ml + slot * C::rows + r, make_float2(all, sum), p.a.ww, p.a.status);
                }
            }
            __syncthreads();
            seg0 += cur.nt;
            fresh = true;
        }
        if (x + 1 < x1) advance(p, cur, groups);
    }
    cp_async_wait<0>();
    grid_launch_dependents();
}

// Second launch: one CTA per (sequence, head group).  Empty sequences get
// their zeros here; segments that one CTA held are done; the pieces of the others are
// joined in the order of the CTAs.
template <int D, int NT>
__global__ void __launch_bounds__(128) cache_attention_join_kernel(const Params p) {
    using C = Config<D, NT>;
    grid_wait_prerequisites();
    const int groups = p.a.c.heads * p.row_groups;
    const int64_t seg = blockIdx.x;
    const int64_t b = seg / groups;
    const int g = (int)(seg - b * groups), sub = g % p.row_groups;
    const int rows = min(C::rows, p.group - sub * C::rows);
    const int64_t head0 = b * p.a.q_heads + (int64_t)(g / p.row_groups) * p.group + sub * C::rows;
    const bool empty = length_of(p.a, b) == 0;
    int2 ctas = make_int2(0, -1);
    if (!empty) {
        ctas = p.meta[seg];
        if (ctas.y < ctas.x) return;
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int r = warp; r < rows; r += 4) {
        float all = -INFINITY;
        for (int i = ctas.x + lane; i <= ctas.y; i += 32)
            all = fmaxf(all, p.part_ml[(2 * (int64_t)i + (i == ctas.x)) * C::rows + r].x);
        all = warp_max(all);
        float sum = 0.0f;
        float2 o[D / 64];
#pragma unroll
        for (int k = 0; k < D / 64; ++k) o[k] = make_float2(0.0f, 0.0f);
        for (int i = ctas.x; i <= ctas.y; ++i) {
            const int64_t at = (2 * (int64_t)i + (i == ctas.x)) * C::rows + r;
            const float2 ml = p.part_ml[at];
            if (ml.y == 0.0f) continue;  // no position of the piece was there
            const float f = exp2_fast(ml.x - all);
            sum += ml.y * f;
#pragma unroll
            for (int k = 0; k < D / 64; ++k) {
                const float2 v = *reinterpret_cast<const float2*>(p.part_o + at * D + 2 * lane + 64 * k);
                o[k].x += v.x * f;
                o[k].y += v.y * f;
            }
        }
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
        for (int k = 0; k < D / 64; ++k) {
            uint32_t h;
            if (p.a.q_bf16) {
                const __nv_bfloat162 t = __floats2bfloat162_rn(o[k].x * inv, o[k].y * inv);
                h = *reinterpret_cast<const uint32_t*>(&t);
            } else {
                h = pack_half2(o[k].x * inv, o[k].y * inv);
            }
            gstore_plain(reinterpret_cast<uint32_t*>(p.a.out + (head0 + r) * D + 2 * lane + 64 * k), h, p.a.ow,
                         p.a.status);
        }
        if (p.a.lse && lane == 0)
            gstore_plain(p.a.lse + head0 + r, (all + log2f(sum)) * kLn2, p.a.lw, p.a.status);
    }
}

template <int D, int NT>
int64_t grid_of(int sm_count) {
    return (int64_t)sm_count * Config<D, NT>::ctas_per_sm;
}

template <int D, int NT>
int64_t workspace_of(int64_t segments, int sm_count) {
    const int64_t slots = 2 * grid_of<D, NT>(sm_count) * Config<D, NT>::rows;
    return slots * (D * 4 + 8) + segments * 8;
}

template <int D, int NT>
int launch_typed(const CacheAttentionArgs& a, int sm_count, cudaStream_t stream) {
    using C = Config<D, NT>;
    auto kernel = cache_attention_kernel<D, NT>;
    // once per device: later launches, captured ones among them, make no such call
    static std::atomic<uint64_t> attr_set{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    const uint64_t bit = 1ull << (dev & 63);
    if (e == cudaSuccess && !(attr_set.load(std::memory_order_acquire) & bit)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::smem);
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout,
                                     (int)cudaSharedmemCarveoutMaxShared);
        if (e == cudaSuccess) attr_set.fetch_or(bit, std::memory_order_acq_rel);
    }
    if (e != cudaSuccess) {
        set_last_error("cudaFuncSetAttribute", (int)e);
        return MXFP8_ERR_CUDA;
    }
    Params p;
    p.a = a;
    p.group = a.q_heads / a.c.heads;
    p.row_groups = (p.group + C::rows - 1) / C::rows;
    const int64_t segments = a.batch * a.c.heads * p.row_groups;
    const int64_t most = segments * (((a.max_pages << a.c.page_shift) + kTilePos - 1) / kTilePos);
    const int64_t ctas = grid_of<D, NT>(sm_count);
    p.grid = ctas < most ? ctas : most;
    p.part_o = static_cast<float*>(a.workspace);
    p.part_ml = reinterpret_cast<float2*>(p.part_o + 2 * ctas * C::rows * D);
    p.meta = reinterpret_cast<int2*>(p.part_ml + 2 * ctas * C::rows);

    cudaLaunchConfig_t cfg = {};
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (p.grid > 0) {
        cfg.gridDim = dim3((unsigned)p.grid);
        cfg.blockDim = dim3(kThreads);
        cfg.dynamicSmemBytes = C::smem;
        e = cudaLaunchKernelEx(&cfg, kernel, p);
    }
    if (e == cudaSuccess) {
        cfg.gridDim = dim3((unsigned)segments);
        cfg.blockDim = dim3(128);
        cfg.dynamicSmemBytes = 0;
        e = cudaLaunchKernelEx(&cfg, cache_attention_join_kernel<D, NT>, p);
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
