// mxfp4_gemm.cu -- C (m, n) = A (m, k) B (n, k)^T for MXFP4 A and B, on the
// block-scaled tensor cores (tcgen05.mma kind::mxf4): 64 products of E2M1
// values a step, each block of 32 scaled by 2^(sa + sb - 254), summed in f32.
//
// One matrix supplies the rows of a tile (P, the lanes of tensor memory), the
// other its columns (Q).  A CTA has one warp that streams 256-column stages of
// both (TMA tiles with the 128-byte swizzle, scale chunks as untiled copies: a
// 128-row block's chunks are contiguous along K), one that copies the scales to
// tensor memory and issues the MMAs, and four or eight that read the
// accumulators back.  Two forms:
//
// wide: P is A, Q is B.  The two CTAs of a cluster pair compute one 256 x 256
//   tile (cta_group::2): each loads its 128 rows of A and half of the 256 rows
//   of B, 35 KB a stage for 4 MMAs where a CTA on its own would load 51.  A lane
//   is a row of C, its columns are contiguous in memory: 32-byte stores.  Where
//   rows of C do not start on 32 bytes, P is B and Q is A, as in the narrow form.
// narrow: P is B, Q is A.  A lane is a column of C, so a warp's stores are
//   contiguous for any alignment, and few rows of A make a narrow tile: the
//   form for single tokens, where streaming B is the whole cost.  If there are
//   fewer tiles than SMs, a cluster of CTAs shares a tile: each takes a part of
//   K, and their sums meet in shared memory over the cluster in rank order, so
//   the result does not depend on timing.
//
// Measured, bf16 out: 8192x8192x8192 187 us = 5.9 PFLOP/s for a burst, 216 us
// under the power cap; 4096x4096x4096 29.1 us = 4.7.  One pair a tile leaves the
// tensor cores waiting while its accumulators are read (256 + 48 of 512 columns
// of tensor memory: no second set fits): 8192x4096x1024 22.8 us = 3.0 PFLOP/s.
// One token through 16384x8192 16.1 us = 4.4 TB/s (matrices in turn, from HBM),
// through 4096x4096 5.7 us = 1.6 TB/s: there the launch, the first loads and the join of the split take
// longer than the stream.  Loops of a whole warp with one elected lane issue a
// stage's instructions in about a tenth of the cycles that a one-lane branch
// takes: 8192x8192x8192 was 348 us with those.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstring>

#include "../../include/mxfp4.h"
#include "gemm_barriers.h"
#include "launch.h"
#include "ptx.cuh"
#include "tcgen05.cuh"

namespace mxfp8 {

namespace {

constexpr int kTileP = 128;        // rows of P in a tile: the MMA's M
constexpr int kStageK = 256;       // elements of K in a stage: 128 bytes a row
constexpr int kStepK = 64;         // elements of K in one MMA
constexpr int kPBytes = kTileP * 128;
constexpr int kChunk = 512;        // bytes of one 128-row x 4-block scale chunk
constexpr uint64_t kWaitNs = 1000000000ull;
constexpr unsigned kErrGemmWait = 32u;   // bit of the device status word

template <int BN>
struct Narrow {
    static constexpr int q_bytes = BN * 128;
    static constexpr int sp_off = kPBytes + q_bytes;
    static constexpr int sq_off = sp_off + 2 * kChunk;
    static constexpr int stage_bytes = sq_off + 2 * kChunk;
    static constexpr int stages = BN == 128 ? 6 : 8;
    static constexpr int acc = 2;                               // accumulators in tensor memory
    static constexpr int epi_warps = 4;
    static constexpr int threads = 32 * (epi_warps + 2);
    // tensor memory: accumulators, then two sets of scales (P's and Q's of one stage)
    static constexpr int sf_cols = 16;
    static constexpr int cols_used = acc * BN + 2 * sf_cols;
    static constexpr int tmem_cols = cols_used <= 64 ? 64 : cols_used <= 128 ? 128 : cols_used <= 256 ? 256 : 512;
    using Bars = GemmBarriers<stages, acc>;
    static constexpr int bar_off = stages * stage_bytes;
    static constexpr int ctl_off = bar_off + Bars::bytes;
    static constexpr int smem = ctl_off + 16 + 1024;            // and room to align the base to 1024
    static_assert(BN <= 128 && cols_used <= 512 && stage_bytes % 1024 == 0);
    static_assert(BN * 512 <= stages * stage_bytes, "the join of a split K holds a BN x 128 f32 tile in the stages");
};

struct Wide {
    static constexpr int bn = 256;
    static constexpr int q_bytes = bn / 2 * 128;                // this CTA's half of Q
    static constexpr int sp_off = kPBytes + q_bytes;
    static constexpr int sq_off = sp_off + 2 * kChunk;          // scales of all 256 rows of Q
    static constexpr int stage_bytes = sq_off + 4 * kChunk;
    static constexpr int stages = 6;
    static constexpr int epi_warps = 8;
    static constexpr int threads = 32 * (epi_warps + 2);
    static constexpr int sf_cols = 8 + 16;
    static constexpr int tmem_cols = 512;                       // 256 + 2 * 24 of them used
    using Bars = GemmBarriers<stages, 1>;
    static constexpr int bar_off = stages * stage_bytes;
    static constexpr int ctl_off = bar_off + Bars::bytes;
    static constexpr int smem = ctl_off + 16 + 1024;
    static_assert(stage_bytes % 1024 == 0 && smem <= 227 * 1024);
};

struct GemmParams {
    const uint8_t* sp;          // scales of P and Q
    const uint8_t* sq;
    int col_chunks;             // scale chunks along K, the same for both
    int rows_p, rows_q;
    int k;
    int n_stages;               // ceil(k / 256)
    int tiles_p, n_tiles;
    int split;                  // narrow: CTAs of a cluster that share a tile
    void* out;
    int64_t ld_out;
    StoreWindow ow;
    unsigned int* status;
};

// Wait for a barrier's phase, at most kWaitNs, or until another role gave up.
// Called by whole warps; the answer is the warp's.
__device__ __forceinline__ bool wait_phase(uint32_t bar, uint32_t parity, volatile int* abort, unsigned int* status) {
    uint64_t t0 = 0;
    for (uint32_t i = 1;; ++i) {
        if (__all_sync(0xFFFFFFFFu, mbar_try_wait(bar, parity))) return true;
        if ((i & 255u) == 0) {
            const uint64_t now = global_timer_ns();
            if (t0 == 0) t0 = now;
            const bool late = now - t0 > kWaitNs;
            if (late && !*abort) {
                if (status) atomicOr(status, kErrGemmWait);
                *abort = 1;
            }
            if (__any_sync(0xFFFFFFFFu, *abort != 0)) return false;
        }
    }
}

// The load warp's end: wait until the last use of every stage is over, so that
// nothing arrives on its barriers later.  After an abort nobody may release
// the stages: then the copies themselves are waited for, as they still target this CTA.
template <int STAGES>
__device__ __forceinline__ void drain_stages(uint32_t full0, uint32_t empty0, int issued, volatile int* ctl,
                                             unsigned int* status) {
    for (int i = max(0, issued - STAGES); i < issued; ++i) {
        const int s = i % STAGES;
        const uint32_t parity = (i / STAGES) & 1;
        if (!wait_phase(empty0 + 8 * s, parity, ctl, status)) mbar_wait_bounded(full0 + 8 * s, parity, kWaitNs);
    }
}

// Tile t: groups of 16 tiles of P by all tiles of Q, so that the tiles in
// flight share operands in L2.
__device__ __forceinline__ void tile_of(const GemmParams& p, int t, int& tp, int& tq) {
    const int tiles_q = p.n_tiles / p.tiles_p;
    const int group = t / (16 * tiles_q);
    const int in = t - group * 16 * tiles_q;
    const int wide = min(16, p.tiles_p - group * 16);
    tq = in / wide;
    tp = group * 16 + in - tq * wide;
}

// The MMAs of one stage, K = 64 each; sfp and sfq hold the scales of its (at
// most two) chunks, `q_cols` columns of tensor memory a chunk of Q's.
template <int GROUP, int N>
__device__ __forceinline__ void issue_stage(uint32_t d, uint32_t rows_p, uint32_t rows_q, uint32_t sfp, uint32_t sfq,
                                            int q_cols, int steps, bool accumulate) {
    const uint64_t a = desc_sw128(rows_p), b = desc_sw128(rows_q);
#pragma unroll
    for (int j = 0; j < kStageK / kStepK; ++j) {
        if (j < steps)
            mma_mxf4<GROUP>(d, a + 2 * j, b + 2 * j, mxf4_idesc(GROUP * kTileP, N, 2 * (j & 1)), sfp + 4 * (j >> 1),
                            sfq + q_cols * (j >> 1), accumulate || j > 0);
    }
}

template <int OUT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if constexpr (OUT == MXFP8_BF16) {
        const __nv_bfloat162 t = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&t);
    } else {
        const __half2 t = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&t);
    }
}

template <int OUT>
__device__ __forceinline__ void store1(void* out, int64_t at, float v, const StoreWindow& w, unsigned int* status) {
    if constexpr (OUT == MXFP8_F32) {
        gstore_plain(static_cast<float*>(out) + at, v, w, status);
    } else {
        gstore_plain(static_cast<unsigned short*>(out) + at, (unsigned short)(pack2<OUT>(v, 0.0f) & 0xFFFFu), w, status);
    }
}

// Four f32 of one row of C, columns col .. col + 3 (those below n = rows_p).
template <int OUT>
__device__ __forceinline__ void store_quad(const GemmParams& p, int64_t row, int col, const float4& v) {
    constexpr int kEs = OUT == MXFP8_F32 ? 4 : 2;
    const int64_t at = row * p.ld_out + col;
    if (((reinterpret_cast<uintptr_t>(p.out) + (uint64_t)at * kEs) & (4 * kEs - 1)) == 0 && col + 4 <= p.rows_p) {
        if constexpr (OUT == MXFP8_F32)
            gstore_plain(reinterpret_cast<float4*>(static_cast<float*>(p.out) + at), v, p.ow, p.status);
        else
            gstore_plain(reinterpret_cast<uint2*>(static_cast<unsigned short*>(p.out) + at),
                         make_uint2(pack2<OUT>(v.x, v.y), pack2<OUT>(v.z, v.w)), p.ow, p.status);
        return;
    }
    const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (col + i < p.rows_p) store1<OUT>(p.out, at + i, f[i], p.ow, p.status);
}

// NC f32 of one row of C, columns col .. col + NC - 1 (those below n), to out, whose rows start on 32 bytes.
template <int OUT, int NC>
__device__ __forceinline__ void store_row(const GemmParams& p, int64_t row, int col, int n, const uint32_t* acc) {
    constexpr int kEs = OUT == MXFP8_F32 ? 4 : 2;
    constexpr int kPer = 32 / kEs;  // elements of one 32-byte store
    const int64_t at = row * p.ld_out + col;
    if (col + NC <= n) {
#pragma unroll
        for (int i = 0; i < NC; i += kPer) {
            if constexpr (OUT == MXFP8_F32) {
                gstore32(static_cast<float*>(p.out) + at + i, acc + i, p.ow, p.status);
            } else {
                uint32_t h[8];
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    h[j] = pack2<OUT>(__uint_as_float(acc[i + 2 * j]), __uint_as_float(acc[i + 2 * j + 1]));
                gstore32(static_cast<unsigned short*>(p.out) + at + i, h, p.ow, p.status);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < NC; ++i)
            if (col + i < n) store1<OUT>(p.out, at + i, __uint_as_float(acc[i]), p.ow, p.status);
    }
}

template <int BN, int OUT>
__global__ void __launch_bounds__(Narrow<BN>::threads, 1)
    mxfp4_gemm_narrow_kernel(const __grid_constant__ CUtensorMap map_p, const __grid_constant__ CUtensorMap map_q,
                      const GemmParams p) {
    using C = Narrow<BN>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t base = smem_u32(smem);
    using B = typename C::Bars;
    const uint32_t bars = base + C::bar_off, full0 = bars + B::full(0), empty0 = bars + B::empty(0);
    const uint32_t acc_full0 = bars + B::acc_full(0), acc_empty0 = bars + B::acc_empty(0), drained = bars + B::drained();
    volatile int* ctl = reinterpret_cast<volatile int*>(smem + C::ctl_off);  // abort, -, TMEM address
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int kLoadWarp = C::epi_warps, kMmaWarp = C::epi_warps + 1;

    if (threadIdx.x == 0) {
        for (int i = 0; i < C::stages; ++i) {
            mbar_init(full0 + 8 * i, 1);
            mbar_init(empty0 + 8 * i, 1);
        }
        for (int i = 0; i < C::acc; ++i) {
            mbar_init(acc_full0 + 8 * i, 1);
            mbar_init(acc_empty0 + 8 * i, C::epi_warps);
        }
        mbar_init(drained, 1);
        ctl[0] = 0;
        fence_mbar_init();
    }
    if (warp == kMmaWarp) tmem_alloc<1>(base + C::ctl_off + 8, C::tmem_cols);
    if (warp == kLoadWarp && lane == 0) {
        prefetch_tensormap(&map_p);
        prefetch_tensormap(&map_q);
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem = (uint32_t)ctl[2];
    const uint32_t tmem_sf = tmem + C::acc * BN;
    grid_launch_dependents();
    grid_wait_prerequisites();

    const int rank = p.split > 1 ? (int)(blockIdx.x % p.split) : 0;
    const int first_tile = blockIdx.x / p.split, tile_step = gridDim.x / p.split;
    const int ks0 = (int)((int64_t)rank * p.n_stages / p.split);
    const int ks1 = (int)((int64_t)(rank + 1) * p.n_stages / p.split);
    int issued = 0;  // stages loaded by the load thread

    if (warp == kLoadWarp) {
        bool ok = true;
        for (int t = first_tile; ok && t < p.n_tiles; t += tile_step) {
            int tp, tq;
            tile_of(p, t, tp, tq);
            for (int ks = ks0; ks < ks1; ++ks, ++issued) {
                const int s = issued % C::stages;
                if (issued >= C::stages &&
                    !wait_phase(empty0 + 8 * s, ((issued / C::stages) - 1) & 1, ctl, p.status)) {
                    ok = false;
                    break;
                }
                if (elect_one()) {
                    const uint32_t dst = base + s * C::stage_bytes, bar = full0 + 8 * s;
                    const uint32_t scales = min(2, p.col_chunks - 2 * ks) * kChunk;
                    mbar_arrive_expect_tx(bar, kPBytes + C::q_bytes + 2 * scales);
                    tma_load_2d(dst, &map_p, ks * (kStageK / 2), tp * kTileP, bar);
                    tma_load_2d(dst + kPBytes, &map_q, ks * (kStageK / 2), tq * BN, bar);
                    bulk_load(dst + C::sp_off, p.sp + ((int64_t)tp * p.col_chunks + 2 * ks) * kChunk, scales, bar);
                    bulk_load(dst + C::sq_off, p.sq + ((int64_t)tq * p.col_chunks + 2 * ks) * kChunk, scales, bar);
                }
                __syncwarp();
            }
        }
    } else if (warp == kMmaWarp) {
        int it = 0, a = 0;
        bool ok = true;
        for (int t = first_tile; ok && t < p.n_tiles; t += tile_step, ++a) {
            const int slot = a % C::acc;
            if (a >= C::acc && !wait_phase(acc_empty0 + 8 * slot, ((a / C::acc) - 1) & 1, ctl, p.status)) break;
            tcgen05_fence_after();
            for (int ks = ks0; ks < ks1; ++ks, ++it) {
                const int s = it % C::stages;
                if (!wait_phase(full0 + 8 * s, (it / C::stages) & 1, ctl, p.status)) {
                    ok = false;
                    break;
                }
                tcgen05_fence_after();
                if (elect_one()) {
                    const uint32_t src = base + s * C::stage_bytes;
                    const uint32_t sfp = tmem_sf + (it & 1) * C::sf_cols, sfq = sfp + 8;
                    const int chunks = min(2, p.col_chunks - 2 * ks);
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        if (c < chunks) {
                            tmem_copy_scales<1>(sfp + 4 * c, desc_scale_chunk(src + C::sp_off + c * kChunk));
                            tmem_copy_scales<1>(sfq + 4 * c, desc_scale_chunk(src + C::sq_off + c * kChunk));
                        }
                    }
                    issue_stage<1, BN>(tmem + slot * BN, src, src + kPBytes, sfp, sfq, 4,
                                       (p.k - ks * kStageK + kStepK - 1) / kStepK, ks > ks0);
                    tcgen05_commit<1>(empty0 + 8 * s);
                    if (ks + 1 == ks1) tcgen05_commit<1>(acc_full0 + 8 * slot);
                }
                __syncwarp();
            }
        }
        // the readers have waited for every tile's MMAs, unless one of them gave up: then some are still in flight,
        // and they end before the tensor memory goes
        if (elect_one()) tcgen05_commit<1>(drained);
        __syncwarp();
        mbar_wait_bounded(drained, 0, kWaitNs);
    } else {
        const int q4 = warp & 3;
        const uint32_t lane_off = (uint32_t)(q4 * 32) << 16;
        int a = 0;
        for (int t = first_tile; t < p.n_tiles; t += tile_step, ++a) {
            const int slot = a % C::acc;
            if (!wait_phase(acc_full0 + 8 * slot, (a / C::acc) & 1, ctl, p.status)) break;
            tcgen05_fence_after();
            int tp, tq;
            tile_of(p, t, tp, tq);
            const uint32_t d = tmem + slot * BN + lane_off;
            {
                const int64_t n = (int64_t)tp * kTileP + q4 * 32 + lane;
                const int left = min(BN, p.rows_q - tq * BN);
                float* red = reinterpret_cast<float*>(smem);
                for (int c0 = 0; c0 < left; c0 += 16) {
                    uint32_t v[16];
                    tmem_load_16(d + c0, v);
                    tmem_wait_loads();
                    tmem_loaded(v);
                    if (p.split > 1) {
#pragma unroll
                        for (int j = 0; j < 16; ++j) red[(c0 + j) * 128 + q4 * 32 + lane] = __uint_as_float(v[j]);
                    } else if (n < p.rows_p) {
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            if (c0 + j < left)
                                store1<OUT>(p.out, ((int64_t)tq * BN + c0 + j) * p.ld_out + n, __uint_as_float(v[j]),
                                            p.ow, p.status);
                    }
                }
                tcgen05_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(acc_empty0 + 8 * slot);
            }
        }
    }
    if (warp == kLoadWarp) drain_stages<C::stages>(full0, empty0, issued, ctl, p.status);
    __syncwarp();
    if (p.split > 1) {  // one tile a cluster: add the parts up, each CTA its share of the columns
        cluster_sync();
        if (warp < C::epi_warps && !ctl[0]) {
            int tp, tq;
            tile_of(p, first_tile, tp, tq);
            const int left = min(BN, p.rows_q - tq * BN);
            // a warp takes a column, a lane four of its rows; four columns at a time keep the remote loads in flight
            for (int c0 = rank + p.split * warp; c0 < left; c0 += 4 * C::epi_warps * p.split) {
                float4 sum[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                for (int r = 0; r < p.split; ++r) {
                    const uint32_t at = cluster_map(base, r) + (uint32_t)lane * 16u;
                    float4 v[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i)  // columns past `left` read what the tile left there, below BN
                        v[i] = cluster_load_f32x4(at + (uint32_t)min(c0 + i * C::epi_warps * p.split, left - 1) * 512u);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        sum[i].x += v[i].x;
                        sum[i].y += v[i].y;
                        sum[i].z += v[i].z;
                        sum[i].w += v[i].w;
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int c = c0 + i * C::epi_warps * p.split;
                    if (c < left) store_quad<OUT>(p, (int64_t)tq * BN + c, tp * kTileP + 4 * lane, sum[i]);
                }
            }
        }
        cluster_sync();  // nobody leaves while its part is still read
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    if (warp == kMmaWarp) tmem_dealloc<1>(tmem, C::tmem_cols);
}


// The wide form: a cluster pair a tile.  Each CTA loads its share, all of it
// signalled on the even CTA's barriers; that one issues for both, and each
// reads its half of the rows back: rows of C, or columns if ACROSS.
template <int OUT, bool ACROSS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Wide::threads, 1)
    mxfp4_gemm_wide_kernel(const __grid_constant__ CUtensorMap map_p, const __grid_constant__ CUtensorMap map_q,
                           const __grid_constant__ CUtensorMap map_sp, const __grid_constant__ CUtensorMap map_sq,
                           const GemmParams p) {
    using C = Wide;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t base = smem_u32(smem);
    using B = C::Bars;
    const uint32_t bars = base + C::bar_off, full0 = bars + B::full(0), empty0 = bars + B::empty(0);
    const uint32_t acc_full = bars + B::acc_full(0), acc_empty = bars + B::acc_empty(0), drained = bars + B::drained();
    volatile int* ctl = reinterpret_cast<volatile int*>(smem + C::ctl_off);  // abort, -, TMEM address
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int kLoadWarp = C::epi_warps, kMmaWarp = C::epi_warps + 1;
    const int rank = blockIdx.x & 1;

    if (threadIdx.x == 0) {
        for (int i = 0; i < C::stages; ++i) {
            mbar_init(full0 + 8 * i, 1);                  // used in the even CTA: both CTAs' copies
            mbar_init(empty0 + 8 * i, 1);
        }
        mbar_init(acc_full, 1);
        mbar_init(acc_empty, 2 * C::epi_warps);           // used in the even CTA: both CTAs' readers
        mbar_init(drained, 1);                            // committed by the even CTA in both
        ctl[0] = 0;
        fence_mbar_init();
    }
    if (warp == kMmaWarp) tmem_alloc<2>(base + C::ctl_off + 8, C::tmem_cols);
    if (warp == kLoadWarp && lane == 0) {
        prefetch_tensormap(&map_p);
        prefetch_tensormap(&map_q);
        prefetch_tensormap(&map_sp);
        prefetch_tensormap(&map_sq);
    }
    tcgen05_fence_before();
    __syncthreads();
    cluster_sync();  // the other CTA's barriers are ready, too
    tcgen05_fence_after();
    const uint32_t tmem = (uint32_t)ctl[2];
    const uint32_t tmem_sf = tmem + C::bn;
    grid_launch_dependents();
    grid_wait_prerequisites();

    const int first_tile = blockIdx.x >> 1, tile_step = gridDim.x >> 1;
    int issued = 0;  // stages loaded by the load warp

    if (warp == kLoadWarp) {
        const uint32_t even_full0 = cluster_map(full0, 0);
        bool ok = true;
        for (int t = first_tile; ok && t < p.n_tiles; t += tile_step) {
            int tp, tq;
            tile_of(p, t, tp, tq);
            for (int ks = 0; ks < p.n_stages; ++ks, ++issued) {
                const int s = issued % C::stages;
                if (issued >= C::stages &&
                    !wait_phase(empty0 + 8 * s, ((issued / C::stages) - 1) & 1, ctl, p.status)) {
                    ok = false;
                    break;
                }
                if (elect_one()) {
                    const uint32_t dst = base + s * C::stage_bytes, bar = even_full0 + 8 * s;
                    // whole boxes count, zero-filled where the matrices end
                    if (rank == 0) mbar_arrive_expect_tx(full0 + 8 * s, 2 * C::stage_bytes);
                    tma_load_2d_pair(dst, &map_p, ks * (kStageK / 2), (2 * tp + rank) * kTileP, bar);
                    tma_load_2d_pair(dst + kPBytes, &map_q, ks * (kStageK / 2), tq * C::bn + rank * (C::bn / 2), bar);
                    tma_load_2d_pair(dst + C::sp_off, &map_sp, ks * 2 * (kChunk / 4), 2 * tp + rank, bar);
                    tma_load_2d_pair(dst + C::sq_off, &map_sq, ks * 2 * (kChunk / 4), 2 * tq, bar);
                }
                __syncwarp();
            }
        }
    } else if (warp == kMmaWarp) {
        int it = 0, a = 0;
        bool ok = rank == 0;
        for (int t = first_tile; ok && t < p.n_tiles; t += tile_step, ++a) {
            if (a > 0 && !wait_phase(acc_empty, (a - 1) & 1, ctl, p.status)) break;
            tcgen05_fence_after();
            for (int ks = 0; ks < p.n_stages; ++ks, ++it) {
                const int s = it % C::stages;
                if (!wait_phase(full0 + 8 * s, (it / C::stages) & 1, ctl, p.status)) {
                    ok = false;
                    break;
                }
                tcgen05_fence_after();
                if (elect_one()) {
                    const uint32_t src = base + s * C::stage_bytes;
                    const uint32_t sfp = tmem_sf + (it & 1) * C::sf_cols, sfq = sfp + 8;
                    const int chunks = min(2, p.col_chunks - 2 * ks);
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        if (c < chunks) {
                            tmem_copy_scales<2>(sfp + 4 * c, desc_scale_chunk(src + C::sp_off + c * kChunk));
                            tmem_copy_scales<2>(sfq + 8 * c, desc_scale_chunk(src + C::sq_off + c * kChunk));
                            tmem_copy_scales<2>(sfq + 8 * c + 4, desc_scale_chunk(src + C::sq_off + (2 + c) * kChunk));
                        }
                    }
                    issue_stage<2, C::bn>(tmem, src, src + kPBytes, sfp, sfq, 8,
                                          (p.k - ks * kStageK + kStepK - 1) / kStepK, ks > 0);
                    tcgen05_commit<2>(empty0 + 8 * s);
                    if (ks + 1 == p.n_stages) tcgen05_commit<2>(acc_full);
                }
                __syncwarp();
            }
        }
        // as in the narrow form; it arrives in both CTAs, and each waits for its own below
        if (rank == 0 && elect_one()) tcgen05_commit<2>(drained);
        __syncwarp();
    } else {
        // two warps for each quarter of the lanes, 128 columns each
        const int q4 = warp & 3, col0 = (warp >> 2) * 128;
        const uint32_t d = tmem + col0 + ((uint32_t)(q4 * 32) << 16);
        const uint32_t peer_acc_empty = cluster_map(acc_empty, 0);
        int a = 0;
        for (int t = first_tile; t < p.n_tiles; t += tile_step, ++a) {
            if (!wait_phase(acc_full, a & 1, ctl, p.status)) break;
            tcgen05_fence_after();
            int tp, tq;
            tile_of(p, t, tp, tq);
            uint32_t v[4][32];
#pragma unroll
            for (int i = 0; i < 4; ++i) tmem_load_32(d + 32 * i, v[i]);
            tmem_wait_loads();
#pragma unroll
            for (int i = 0; i < 4; ++i) tmem_loaded(v[i]);
            // the accumulator is in registers: the next tile's MMAs may overwrite it
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) cluster_arrive(peer_acc_empty);
            const int64_t row = (int64_t)(2 * tp + rank) * kTileP + q4 * 32 + lane;
            if (row < p.rows_p) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int col = tq * C::bn + col0 + 32 * i;
                    if constexpr (ACROSS) {
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (col + j < p.rows_q)
                                store1<OUT>(p.out, (int64_t)(col + j) * p.ld_out + row, __uint_as_float(v[i][j]), p.ow,
                                            p.status);
                    } else {
                        store_row<OUT, 32>(p, row, col, p.rows_q, v[i]);
                    }
                }
            }
        }
    }
    if (warp == kLoadWarp) {
        drain_stages<C::stages>(full0, empty0, issued, ctl, p.status);
        mbar_wait_bounded(drained, 0, kWaitNs);  // the last arrival from the even CTA: none comes after this one has gone
    }
    __syncwarp();
    tcgen05_fence_before();
    __syncthreads();
    cluster_sync();  // the other CTA's barriers and tensor memory are no longer in use
    tcgen05_fence_after();
    if (warp == kMmaWarp) tmem_dealloc<2>(tmem, C::tmem_cols);
}

// A 2-D tensor map with zeros outside.
int encode_map(CUtensorMap* map, CUtensorMapDataType type, const void* base, uint64_t cols, uint64_t rows,
               uint64_t stride_bytes, uint32_t box_cols, uint32_t box_rows, CUtensorMapSwizzle swizzle) {
    auto encode = get_encode_fn();
    if (!encode) {
        set_last_error("cuTensorMapEncodeTiled entry point unavailable", 0);
        return MXFP8_ERR_TENSOR_MAP;
    }
    cuuint64_t dims[2] = {cols, rows};
    cuuint64_t strides[1] = {stride_bytes};
    cuuint32_t box[2] = {box_cols, box_rows};
    cuuint32_t step[2] = {1, 1};
    CUresult r = encode(map, type, 2, const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        set_last_error("cuTensorMapEncodeTiled failed", (int)r);
        return MXFP8_ERR_TENSOR_MAP;
    }
    return MXFP8_OK;
}

// A payload: boxes of 128 bytes (256 elements of K) by box_rows, 128-byte swizzle.
int encode_payload(CUtensorMap* map, const Fp4Operand& m, int64_t k, int box_rows) {
    return encode_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, m.q, (uint64_t)(k / 2), (uint64_t)m.rows, (uint64_t)m.ld, 128,
                      (uint32_t)box_rows, CU_TENSOR_MAP_SWIZZLE_128B);
}

// Its scales: a row of words per 128-row block, boxes of two chunks by box_blocks.
int encode_scales(CUtensorMap* map, const Fp4Operand& m, int64_t k, int box_blocks) {
    const uint64_t words = (uint64_t)((k + 127) / 128) * (kChunk / 4);
    return encode_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, m.s, words, (uint64_t)((m.rows + 127) / 128), words * 4,
                      2 * (kChunk / 4), (uint32_t)box_blocks, CU_TENSOR_MAP_SWIZZLE_NONE);
}

int launch_failed(const char* what, cudaError_t e) {
    set_last_error(what, (int)e);
    return MXFP8_ERR_CUDA;
}

GemmParams params_of(const Fp4GemmArgs& g, const Fp4Operand& P, const Fp4Operand& Q, int tile_p, int tile_q) {
    GemmParams p;
    p.sp = P.s;
    p.sq = Q.s;
    p.col_chunks = (int)((g.k + 127) / 128);
    p.rows_p = (int)P.rows;
    p.rows_q = (int)Q.rows;
    p.k = (int)g.k;
    p.n_stages = (int)((g.k + kStageK - 1) / kStageK);
    p.tiles_p = (int)((P.rows + tile_p - 1) / tile_p);
    p.n_tiles = p.tiles_p * (int)((Q.rows + tile_q - 1) / tile_q);
    p.split = 1;
    p.out = g.out;
    p.ld_out = g.ld_out;
    p.ow = g.ow;
    p.status = g.status;
    return p;
}

template <int OUT, bool ACROSS>
int launch_wide(const Fp4GemmArgs& g, int sm_count, cudaStream_t stream) {
    using C = Wide;
    static OptIn done;
    auto kernel = mxfp4_gemm_wide_kernel<OUT, ACROSS>;
    const Fp4Operand& P = ACROSS ? g.b : g.a;
    const Fp4Operand& Q = ACROSS ? g.a : g.b;
    if (int rc = opt_in(reinterpret_cast<const void*>(kernel), C::smem, false, done)) return rc;
    CUtensorMap map_p, map_q, map_sp, map_sq;
    if (int rc = encode_payload(&map_p, P, g.k, kTileP)) return rc;
    if (int rc = encode_payload(&map_q, Q, g.k, C::bn / 2)) return rc;
    if (int rc = encode_scales(&map_sp, P, g.k, 1)) return rc;
    if (int rc = encode_scales(&map_sq, Q, g.k, 2)) return rc;
    const GemmParams p = params_of(g, P, Q, 2 * kTileP, C::bn);
    cudaLaunchConfig_t cfg = {};
    const int pairs = sm_count / 2;
    cfg.gridDim = dim3(2u * (unsigned)(p.n_tiles < pairs ? p.n_tiles : pairs));
    cfg.blockDim = dim3(C::threads);
    cfg.dynamicSmemBytes = C::smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, map_p, map_q, map_sp, map_sq, p);
    if (e == cudaSuccess) e = cudaGetLastError();
    return e == cudaSuccess ? MXFP8_OK : launch_failed("mxfp4_gemm_wide_kernel launch", e);
}

// CTAs of a narrow tile's cluster: doubled while they fit the SMs and each
// keeps two stages.  With one stage a CTA the join costs more than the stage
// saves: 77x1000x2080 7.6 us with 4 CTAs, 8.3 with 8; 64x512x2048 5.7 and 7.5,
// 16x1000x2048 5.2 and 5.9; only 1x1024x1024 gains, 4.5 and 4.3.
int narrow_split(int64_t tiles, int n_stages, int sm_count) {
    int split = 1;
    while (split < 8 && tiles * split * 2 <= sm_count && n_stages >= 4 * split) split *= 2;
    return split;
}

template <int BN, int OUT>
int launch_narrow(const Fp4GemmArgs& g, int sm_count, cudaStream_t stream) {
    using C = Narrow<BN>;
    static OptIn done;
    auto kernel = mxfp4_gemm_narrow_kernel<BN, OUT>;
    if (int rc = opt_in(reinterpret_cast<const void*>(kernel), C::smem, false, done)) return rc;
    CUtensorMap map_p, map_q;
    if (int rc = encode_payload(&map_p, g.b, g.k, kTileP)) return rc;
    if (int rc = encode_payload(&map_q, g.a, g.k, BN)) return rc;
    GemmParams p = params_of(g, g.b, g.a, kTileP, BN);
    p.split = narrow_split(p.n_tiles, p.n_stages, sm_count);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(p.split > 1 ? p.n_tiles * p.split : p.n_tiles < sm_count ? p.n_tiles : sm_count));
    cfg.blockDim = dim3(C::threads);
    cfg.dynamicSmemBytes = C::smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)p.split;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = p.split > 1 ? 2 : 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, map_p, map_q, p);
    if (e == cudaSuccess) e = cudaGetLastError();
    return e == cudaSuccess ? MXFP8_OK : launch_failed("mxfp4_gemm_narrow_kernel launch", e);
}

template <int OUT>
int launch_out(const Fp4GemmArgs& g, int sm_count, cudaStream_t stream) {
    if (g.a.rows <= 16) return launch_narrow<16, OUT>(g, sm_count, stream);
    if (g.a.rows <= 32) return launch_narrow<32, OUT>(g, sm_count, stream);
    if (g.a.rows <= 64) return launch_narrow<64, OUT>(g, sm_count, stream);
    // More than 64 rows: both forms take a time that grows with the stages a CTA
    // walks one after another, about 5.1 + 0.32 us a stage (wide) and 7.2 + 0.36
    // (narrow).  Measured, us wide / narrow: 512x2048x2048 7.7 / 8.3,
    // 384x4096x4096 10.4 / 12.7, 256x8192x8192 16.7 / 18.8; with K long and
    // split the narrow one wins: 256x4096x4096 10.2 / 9.7, 512x1024x8192 15.3 / 10.0.
    // Rows of C that are not all on 32 bytes are stored an element a lane, which
    // costs the wide form more: 4096x4097x4096 36.4 / 54.5, 2000x2001x7168 19.1 /
    // 27.2, 1024x4097x512 9.7 / 12.8, but as many stages in both 512x4097x4096
    // 13.8 / 13.0, 1500x1501x256 8.7 / 7.6.
    const int es = OUT == MXFP8_F32 ? 4 : 2;
    const bool vec = ((reinterpret_cast<uintptr_t>(g.out) | (uint64_t)(g.ld_out * es)) & 31) == 0;
    const int64_t stages = (g.k + kStageK - 1) / kStageK;
    const int64_t narrow_tiles = ((g.a.rows + 127) / 128) * ((g.b.rows + 127) / 128);
    const int64_t wide_tiles = ((g.a.rows + 255) / 256) * ((g.b.rows + 255) / 256);
    const int split = narrow_split(narrow_tiles, (int)stages, sm_count);
    const int64_t narrow_row = (stages + split - 1) / split * ((narrow_tiles * split + sm_count - 1) / sm_count);
    const int64_t wide_row = stages * ((wide_tiles + sm_count / 2 - 1) / (sm_count / 2));
    if (vec && wide_row <= narrow_row + 6) return launch_wide<OUT, false>(g, sm_count, stream);
    if (!vec && wide_row < narrow_row) return launch_wide<OUT, true>(g, sm_count, stream);
    return launch_narrow<128, OUT>(g, sm_count, stream);
}

}  // namespace

int launch_mxfp4_gemm(const Fp4GemmArgs& g, int sm_count, cudaStream_t stream) {
    // tiles are counted in 32 bits
    if (((g.a.rows + 127) / 128) * ((g.b.rows + 127) / 128) > (1 << 24)) return MXFP8_ERR_SHAPE;
    switch (g.out_dtype) {
        case MXFP8_F32: return launch_out<MXFP8_F32>(g, sm_count, stream);
        case MXFP8_BF16: return launch_out<MXFP8_BF16>(g, sm_count, stream);
        default: return launch_out<MXFP8_FP16>(g, sm_count, stream);
    }
}

}  // namespace mxfp8
