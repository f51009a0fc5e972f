// mxfp4_convert.cu -- bf16/fp16 -> MXFP4 and MXFP4 -> bf16/fp16/f32.
//
// Both are byte streams: 2 + 1/2 + 1/32 bytes an element to quantize, 1/2 +
// 1/32 + the output's to invert; HBM bandwidth bounds them.  A warp takes some
// columns of the four rows r, r + 32, r + 64, r + 96 of one 128-row block:
// every access of a warp is contiguous, and the four rows' scale words of one
// chunk are its 16 bytes at (r % 32) * 16, one vector access.  The eight warps
// of a CTA take eight neighbouring r of the same columns.
//
// Quantizing is also near the ALUs' limit, so a lane holds 16 elements of a
// row, half a block: one shuffle for the block's amax, one scale for 16 codes.
// Measured, 8192x8192 bf16: 26.7 us = 6.36 TB/s (49.3 with 8 elements a lane and
// 64-bit index divisions); inverted to bf16 27.1 us, to f32 47.6 us (68.5 with
// 16-byte stores).  Rows off a 32-byte boundary (4096x8191): 20.2 us = 4.2 TB/s.
#include <cuda_runtime.h>

#include "../../include/mxfp4.h"
#include "launch.h"
#include "mxfp4.cuh"
#include "ptx.cuh"

namespace mxfp8 {

namespace {

constexpr int kConvertThreads = 256;
constexpr int kRowsPerWarp = 4;   // r + 32 i
constexpr int kQuantCols = 512;   // columns of a warp that quantizes: 16 a lane
constexpr int kDequantCols = 256;  // and of one that inverts: 8 a lane

// The first row of this warp (rb * 128 + r) and its first column.  CTA c takes
// columns c % segs and rows r = 8 (c / segs % 4) .. + 7 of row block c / segs / 4.
struct WarpUnit {
    int64_t row0, c0;
};

__device__ __forceinline__ WarpUnit warp_unit(uint32_t segs, int cols) {
    const uint32_t line = blockIdx.x / segs;
    return WarpUnit{(int64_t)(line >> 2) * 128 + (line & 3) * 8 + (threadIdx.x >> 5),
                    (int64_t)(blockIdx.x - line * segs) * cols};
}

__device__ __forceinline__ void load32(const uint8_t* p, uint32_t* w) {
    asm volatile("ld.global.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                 : "l"(p));
}

__device__ __forceinline__ void load16(const uint8_t* p, uint32_t* w) {
    asm volatile("ld.global.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                 : "l"(p));
}

// Elements col .. col + 15 of an X row, in two steps so that the loads of all of a
// warp's rows are in flight before the first is touched.
// load: ALIGNED rows start on 32 bytes, and a lane loads its 32.  Otherwise it
// loads the two aligned 16-byte chunks from the one that holds its first
// element on, and the last lane the one after them; only chunks that hold one of
// the row's own elements are read.
template <bool ALIGNED>
__device__ __forceinline__ void load_row16(const uint8_t* row, int64_t col, int64_t k, uint32_t (&w)[8],
                                           uint32_t (&next)[ALIGNED ? 1 : 4]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = 0u;
    if constexpr (ALIGNED) {
        if (col < k) load32(row + 2 * col, w);
    } else {
        const uint32_t h = (uint32_t)(reinterpret_cast<uintptr_t>(row) & 15);
        const int64_t end = k > 0 ? h + 2 * k : 0;  // bytes of the row from row - h
        const uint8_t* at = row - h + 2 * col;
        if (2 * col < end) load16(at, w);
        if (2 * col + 16 < end) load16(at + 16, w + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) next[i] = 0u;
        if ((threadIdx.x & 31) == 31 && 2 * col + 32 < end) load16(at + 32, next);
    }
}

// settle: the lane's elements as eight words, zeros from column k on.  The
// shift is the same for the whole warp; called by whole warps.
template <bool ALIGNED>
__device__ __forceinline__ void settle_row16(const uint8_t* row, int64_t col, int64_t k, uint32_t (&w)[8],
                                             uint32_t (&next)[ALIGNED ? 1 : 4]) {
    if constexpr (!ALIGNED) {
        const uint32_t h = (uint32_t)(reinterpret_cast<uintptr_t>(row) & 15);
        if (h != 0) {
            uint32_t t[12];
            const bool last = (threadIdx.x & 31) == 31;
#pragma unroll
            for (int i = 0; i < 8; ++i) t[i] = w[i];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                t[8 + i] = __shfl_down_sync(0xFFFFFFFFu, w[i], 1);
                if (last) t[8 + i] = next[i];
            }
#pragma unroll
            for (int step = 2; step >= 1; step >>= 1) {  // whole words: 2, 1
                if (h & (4 * step)) {
#pragma unroll
                    for (int i = 0; i + step < 12; ++i) t[i] = t[i + step];
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = __funnelshift_r(t[i], t[i + 1], 8u * (h & 3u));
        }
    }
    if (col + 16 > k) {  // the row ends inside: clear what lies behind it
        const int64_t left = k - col;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (left <= 2 * i) w[i] = 0u;
            else if (left == 2 * i + 1) w[i] &= 0xFFFFu;
        }
    }
}

// Two words of two 16-bit values each, times inv, as four f32.
template <int DT>
__device__ __forceinline__ void scale4(uint32_t w0, uint32_t w1, float inv, float* f) {
    float a, b, c, d;
    if constexpr (DT == kBF16) {
        a = __uint_as_float(w0 << 16);
        b = __uint_as_float(w0 & 0xFFFF0000u);
        c = __uint_as_float(w1 << 16);
        d = __uint_as_float(w1 & 0xFFFF0000u);
    } else {
        const float2 t0 = __half22float2(*reinterpret_cast<const __half2*>(&w0));
        const float2 t1 = __half22float2(*reinterpret_cast<const __half2*>(&w1));
        a = t0.x; b = t0.y; c = t1.x; d = t1.y;
    }
    mul2(a, b, inv, f[0], f[1]);
    mul2(c, d, inv, f[2], f[3]);
}

template <int DT, bool ALIGNED>
__global__ void __launch_bounds__(kConvertThreads) mxfp4_quantize_kernel(
    const uint8_t* __restrict__ x, int64_t m, int64_t k, int64_t row_bytes, uint8_t* __restrict__ q, int64_t q_cols,
    int64_t ld_q, uint8_t* __restrict__ s, int64_t col_chunks, uint32_t segs, StoreWindow qw, StoreWindow sw,
    unsigned int* status) {
    grid_launch_dependents();
    grid_wait_prerequisites();
    const WarpUnit u = warp_unit(segs, kQuantCols);
    const int lane = threadIdx.x & 31;
    const int64_t col = u.c0 + lane * 16;
    uint32_t w[kRowsPerWarp][8], next[kRowsPerWarp][ALIGNED ? 1 : 4];
#pragma unroll
    for (int i = 0; i < kRowsPerWarp; ++i) {
        const int64_t row = u.row0 + 32 * i;
        load_row16<ALIGNED>(x + row * row_bytes, col, row < m ? k : 0, w[i], next[i]);
    }
    uint32_t words[kRowsPerWarp];
#pragma unroll
    for (int i = 0; i < kRowsPerWarp; ++i) {
        const int64_t row = u.row0 + 32 * i;
        settle_row16<ALIGNED>(x + row * row_bytes, col, row < m ? k : 0, w[i], next[i]);
        uint32_t a = w[i][0] & 0x7FFF7FFFu;
#pragma unroll
        for (int j = 1; j < 8; ++j) a = __vmaxu2(a, w[i][j] & 0x7FFF7FFFu);
        a = max(a & 0xFFFFu, a >> 16);
        a = max(a, __shfl_xor_sync(0xFFFFFFFFu, a, 1));
        uint32_t byte;
        float inv;
        fp4_scale_from_amax<DT>(a, byte, inv);
        uint2 codes;
        float f[8];
        scale4<DT>(w[i][0], w[i][1], inv, f);
        scale4<DT>(w[i][2], w[i][3], inv, f + 4);
        codes.x = cvt_e2m1x8(f);
        scale4<DT>(w[i][4], w[i][5], inv, f);
        scale4<DT>(w[i][6], w[i][7], inv, f + 4);
        codes.y = cvt_e2m1x8(f);
        if (byte == 255u) codes = make_uint2(0u, 0u);
        if (row < m && col < q_cols)
            gstore(reinterpret_cast<uint2*>(q + row * ld_q + col / 2), codes, qw, status);
        // padding rows and columns hold 0; the word of a chunk row is its four blocks' bytes
        byte = row < m && col < q_cols ? byte : 0u;
        byte <<= 8 * ((lane >> 1) & 3);
        byte |= __shfl_xor_sync(0xFFFFFFFFu, byte, 2);
        byte |= __shfl_xor_sync(0xFFFFFFFFu, byte, 4);
        words[i] = byte;
    }
    const int64_t chunk = u.c0 / 128 + (lane >> 3);
    if ((lane & 7) == 0 && chunk < col_chunks)
        gstore(reinterpret_cast<uint4*>(s + ((u.row0 >> 7) * col_chunks + chunk) * 512 + (u.row0 & 31) * 16),
               make_uint4(words[0], words[1], words[2], words[3]), sw, status);
}

// Eight values to out + o (element index); `vec`: the place is aligned to
// their bytes (32 for f32: one whole sector a lane).
template <int OUT>
__device__ __forceinline__ void store8(void* out, int64_t o, const float (&v)[8], bool vec, const StoreWindow& w,
                                       unsigned int* status) {
    if constexpr (OUT == MXFP8_F32) {
        float* p = static_cast<float*>(out) + o;
        if (vec) {
            const uint32_t* bits = reinterpret_cast<const uint32_t*>(v);
            gstore32(p, bits, w, status);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) gstore_plain(p + i, v[i], w, status);
        }
    } else {
        uint32_t h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (OUT == MXFP8_BF16) {
                const __nv_bfloat162 t = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                h[i] = *reinterpret_cast<const uint32_t*>(&t);
            } else {
                const __half2 t = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
                h[i] = *reinterpret_cast<const uint32_t*>(&t);
            }
        }
        unsigned short* p = static_cast<unsigned short*>(out) + o;
        if (vec) {
            gstore(reinterpret_cast<uint4*>(p), make_uint4(h[0], h[1], h[2], h[3]), w, status);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                gstore_plain(p + 2 * i, (unsigned short)(h[i] & 0xFFFFu), w, status);
                gstore_plain(p + 2 * i + 1, (unsigned short)(h[i] >> 16), w, status);
            }
        }
    }
}

template <int OUT>
__global__ void __launch_bounds__(kConvertThreads) mxfp4_dequantize_kernel(
    const uint8_t* q, int64_t rows, int64_t cols, int64_t ld_q, const uint8_t* s, int64_t col_chunks, uint32_t segs,
    void* out, int64_t ld_out, StoreWindow ow, unsigned int* status) {
    grid_launch_dependents();
    grid_wait_prerequisites();
    const WarpUnit u = warp_unit(segs, kDequantCols);
    const int lane = threadIdx.x & 31;
    const int64_t col = u.c0 + lane * 8;
    if (col >= cols) return;
    uint32_t codes[kRowsPerWarp];
#pragma unroll
    for (int i = 0; i < kRowsPerWarp; ++i) {
        const int64_t row = u.row0 + 32 * i;
        codes[i] = row < rows ? __ldcs(reinterpret_cast<const uint32_t*>(q + row * ld_q + col / 2)) : 0u;
    }
    // not through the read-only path: the launch may begin while what writes the scales still runs
    const uint4 sv = *reinterpret_cast<const uint4*>(s + ((u.row0 >> 7) * col_chunks + col / 128) * 512 +
                                                     (u.row0 & 31) * 16);
    const uint32_t sw[4] = {sv.x, sv.y, sv.z, sv.w};
    constexpr int kOutBytes = OUT == MXFP8_F32 ? 4 : 2;
#pragma unroll
    for (int i = 0; i < kRowsPerWarp; ++i) {
        const int64_t row = u.row0 + 32 * i;
        if (row >= rows) return;
        const float scale = ue8m0_value((sw[i] >> (8 * ((lane >> 2) & 3))) & 0xFFu);
        uint32_t h[4];
        e2m1x8_to_half2(codes[i], h);
        float v[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&h[j]));
            v[2 * j] = __fmul_rn(t.x, scale);
            v[2 * j + 1] = __fmul_rn(t.y, scale);
        }
        const int64_t o = row * ld_out + col;
        const bool vec = ((reinterpret_cast<uintptr_t>(out) + (uint64_t)o * kOutBytes) & (8 * kOutBytes - 1)) == 0;
        store8<OUT>(out, o, v, vec, ow, status);
    }
}

// Eight rows r of each row block a CTA; -1 if the grid does not fit a launch.
int64_t convert_blocks(int64_t row_blocks, int64_t segs) {
    const int64_t blocks = row_blocks * 4 * segs;
    return blocks > 2147483647 ? -1 : blocks;
}

template <typename... P, typename... A>
int launch_convert(void (*kernel)(P...), int64_t blocks, cudaStream_t stream, const char* what, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(kConvertThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
    if (e == cudaSuccess) e = cudaGetLastError();
    if (e != cudaSuccess) {
        set_last_error(what, (int)e);
        return MXFP8_ERR_CUDA;
    }
    return MXFP8_OK;
}

}  // namespace

int launch_mxfp4_quantize(const Fp4QuantizeArgs& a, cudaStream_t stream) {
    const int64_t row_blocks = (a.m + 127) / 128, segs = (a.q_cols + kQuantCols - 1) / kQuantCols;
    const int64_t col_chunks = (a.q_cols + 127) / 128;
    const int64_t blocks = convert_blocks(row_blocks, segs);
    if (blocks < 0) return MXFP8_ERR_SHAPE;
    const bool aligned = ((reinterpret_cast<uintptr_t>(a.x) | (uint64_t)(a.m > 1 ? a.ld_x * 2 : 0)) & 31) == 0;
    auto kernel = a.dtype == MXFP8_BF16
                      ? (aligned ? mxfp4_quantize_kernel<kBF16, true> : mxfp4_quantize_kernel<kBF16, false>)
                      : (aligned ? mxfp4_quantize_kernel<kFP16, true> : mxfp4_quantize_kernel<kFP16, false>);
    return launch_convert(kernel, blocks, stream, "mxfp4_quantize_kernel launch", static_cast<const uint8_t*>(a.x), a.m,
                          a.k, a.ld_x * 2, a.q, a.q_cols, a.ld_q, a.s, col_chunks, (uint32_t)segs, a.qw, a.sw,
                          a.status);
}

int launch_mxfp4_dequantize(const uint8_t* q, int64_t rows, int64_t cols, int64_t ld_q, const uint8_t* s, void* out,
                            int out_dtype, int64_t ld_out, StoreWindow ow, unsigned int* status, cudaStream_t stream) {
    const int64_t row_blocks = (rows + 127) / 128, segs = (cols + kDequantCols - 1) / kDequantCols;
    const int64_t col_chunks = (cols + 127) / 128;
    const int64_t blocks = convert_blocks(row_blocks, segs);
    if (blocks < 0) return MXFP8_ERR_SHAPE;
    auto kernel = out_dtype == MXFP8_F32    ? mxfp4_dequantize_kernel<MXFP8_F32>
                  : out_dtype == MXFP8_BF16 ? mxfp4_dequantize_kernel<MXFP8_BF16>
                                            : mxfp4_dequantize_kernel<MXFP8_FP16>;
    return launch_convert(kernel, blocks, stream, "mxfp4_dequantize_kernel launch", q, rows, cols, ld_q, s, col_chunks,
                          (uint32_t)segs, out, ld_out, ow, status);
}

}  // namespace mxfp8
