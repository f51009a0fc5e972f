// mxfp4_convert.cu -- bf16/fp16 -> MXFP4 and MXFP4 -> bf16/fp16/f32.
//
// Both are byte streams: 2 + 1/2 + 1/32 bytes an element to quantize, 1/2 +
// 1/32 + the output's to invert; HBM bandwidth bounds them.  One warp takes
// 256 columns (8 blocks, two S chunk columns) of the four rows r, r + 32,
// r + 64, r + 96 of one 128-row block.  A lane holds 8 elements of each row
// (16 bytes of X), so every access of a warp is contiguous: 512 bytes of X and
// 128 of payload per row, and the four rows' scale words of one chunk are its
// 16 bytes at (r % 32) * 16, one vector access.  Four lanes share a block:
// its amax takes two shuffles.
#include <cuda_runtime.h>

#include "../../include/mxfp4.h"
#include "launch.h"
#include "mxfp4.cuh"
#include "ptx.cuh"
#include "stores.cuh"

namespace mxfp8 {

namespace {

constexpr int kConvertThreads = 256;
constexpr int kWarpCols = 256;    // columns of one warp
constexpr int kRowsPerWarp = 4;   // r + 32 i

// Work of this warp: row r of row block rb, columns from c0.
struct WarpUnit {
    int64_t row0;  // rb * 128 + r
    int64_t c0;
    bool any;
};

__device__ __forceinline__ WarpUnit warp_unit(int64_t row_blocks, int64_t segs) {
    const int64_t u = ((int64_t)blockIdx.x * kConvertThreads + threadIdx.x) >> 5;
    const int64_t line = u / segs;  // rb * 32 + r
    return WarpUnit{(line >> 5) * 128 + (line & 31), (u - line * segs) * kWarpCols, line < row_blocks * 32};
}

// Elements col .. col + 7 of an X row as four words, zeros from column k on.
// ALIGNED: the row starts on a 16-byte boundary.  Otherwise every lane loads
// the 16-byte chunk that holds its first element and takes the rest from the
// next lane's chunk; only chunks that hold one of the row's own elements are
// read.  Called by whole warps.
template <bool ALIGNED>
__device__ __forceinline__ uint4 load_row8(const uint8_t* row, int64_t col, int64_t k) {
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if constexpr (ALIGNED) {
        if (col < k) v = __ldcs(reinterpret_cast<const uint4*>(row + 2 * col));
    } else {
        const uint32_t h = (uint32_t)(reinterpret_cast<uintptr_t>(row) & 15);
        const uint8_t* base = row - h;                     // 16-byte aligned
        const int64_t end = h + 2 * k;                     // bytes of the row from base
        const int64_t at = 2 * col;
        uint4 next = v;
        if (at < end) v = __ldcs(reinterpret_cast<const uint4*>(base + at));
        if ((threadIdx.x & 31) == 31 && at + 16 < end) next = __ldcs(reinterpret_cast<const uint4*>(base + at + 16));
        if (h != 0) {
            uint4 nb;
            nb.x = __shfl_down_sync(0xFFFFFFFFu, v.x, 1);
            nb.y = __shfl_down_sync(0xFFFFFFFFu, v.y, 1);
            nb.z = __shfl_down_sync(0xFFFFFFFFu, v.z, 1);
            nb.w = __shfl_down_sync(0xFFFFFFFFu, v.w, 1);
            if ((threadIdx.x & 31) == 31) nb = next;
            v = bytes_from<-1>(v, nb, h);
        }
    }
    if (col + 8 > k) {  // the row ends inside: clear what lies behind it
        const int64_t left = k - col;
        uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (left <= 2 * i) w[i] = 0u;
            else if (left == 2 * i + 1) w[i] &= 0xFFFFu;
        }
    }
    return v;
}

template <int DT, bool ALIGNED>
__global__ void __launch_bounds__(kConvertThreads) mxfp4_quantize_kernel(
    const uint8_t* __restrict__ x, int64_t m, int64_t k, int64_t row_bytes, uint8_t* __restrict__ q, int64_t q_cols,
    int64_t ld_q, uint8_t* __restrict__ s, int64_t row_blocks, int64_t col_chunks, int64_t segs, StoreWindow qw,
    StoreWindow sw, unsigned int* status) {
    grid_launch_dependents();
    grid_wait_prerequisites();
    const WarpUnit u = warp_unit(row_blocks, segs);
    if (!u.any) return;
    const int lane = threadIdx.x & 31;
    const int64_t col = u.c0 + lane * 8;
    uint4 v[kRowsPerWarp];
#pragma unroll
    for (int i = 0; i < kRowsPerWarp; ++i) {
        const int64_t row = u.row0 + 32 * i;
        v[i] = row < m ? load_row8<ALIGNED>(x + row * row_bytes, col, k) : make_uint4(0u, 0u, 0u, 0u);
    }
    uint32_t words[kRowsPerWarp];
#pragma unroll
    for (int i = 0; i < kRowsPerWarp; ++i) {
        const int64_t row = u.row0 + 32 * i;
        const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
        uint32_t a = __vmaxu2(__vmaxu2(w[0] & 0x7FFF7FFFu, w[1] & 0x7FFF7FFFu),
                              __vmaxu2(w[2] & 0x7FFF7FFFu, w[3] & 0x7FFF7FFFu));
        a = max(a & 0xFFFFu, a >> 16);
        a = max(a, __shfl_xor_sync(0xFFFFFFFFu, a, 1));
        a = max(a, __shfl_xor_sync(0xFFFFFFFFu, a, 2));
        uint32_t byte;
        float inv;
        fp4_scale_from_amax<DT>(a, byte, inv);
        float f[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float lo, hi;
            if constexpr (DT == kBF16) {
                lo = __uint_as_float(w[j] << 16);
                hi = __uint_as_float(w[j] & 0xFFFF0000u);
            } else {
                const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
                lo = t.x;
                hi = t.y;
            }
            mul2(lo, hi, inv, f[2 * j], f[2 * j + 1]);
        }
        const uint32_t codes = byte == 255u ? 0u : cvt_e2m1x8(f);
        if (row < m && col < q_cols)
            gstore(reinterpret_cast<uint32_t*>(q + row * ld_q + col / 2), codes, qw, status);
        // padding rows and columns hold 0; the word of a chunk row is its four blocks' bytes
        byte = row < m && col < q_cols ? byte : 0u;
        byte <<= 8 * ((lane >> 2) & 3);
        byte |= __shfl_xor_sync(0xFFFFFFFFu, byte, 4);
        byte |= __shfl_xor_sync(0xFFFFFFFFu, byte, 8);
        words[i] = byte;
    }
    const int64_t chunk = u.c0 / 128 + (lane >> 4);
    if ((lane & 15) == 0 && chunk < col_chunks)
        gstore(reinterpret_cast<uint4*>(s + ((u.row0 >> 7) * col_chunks + chunk) * 512 + (u.row0 & 31) * 16),
               make_uint4(words[0], words[1], words[2], words[3]), sw, status);
}

// Eight values to out + o (element index), as wide as `vec` says.
template <int OUT>
__device__ __forceinline__ void store8(void* out, int64_t o, const float (&v)[8], bool vec, const StoreWindow& w,
                                       unsigned int* status) {
    if constexpr (OUT == MXFP8_F32) {
        float* p = static_cast<float*>(out) + o;
        if (vec) {
            gstore(reinterpret_cast<float4*>(p), make_float4(v[0], v[1], v[2], v[3]), w, status);
            gstore(reinterpret_cast<float4*>(p) + 1, make_float4(v[4], v[5], v[6], v[7]), w, status);
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
    const uint8_t* __restrict__ q, int64_t rows, int64_t cols, int64_t ld_q, const uint8_t* __restrict__ s,
    int64_t row_blocks, int64_t col_chunks, int64_t segs, void* out, int64_t ld_out, StoreWindow ow,
    unsigned int* status) {
    grid_launch_dependents();
    grid_wait_prerequisites();
    const WarpUnit u = warp_unit(row_blocks, segs);
    if (!u.any) return;
    const int lane = threadIdx.x & 31;
    const int64_t col = u.c0 + lane * 8;
    if (col >= cols) return;
    uint32_t codes[kRowsPerWarp];
#pragma unroll
    for (int i = 0; i < kRowsPerWarp; ++i) {
        const int64_t row = u.row0 + 32 * i;
        codes[i] = row < rows ? __ldcs(reinterpret_cast<const uint32_t*>(q + row * ld_q + col / 2)) : 0u;
    }
    const uint4 sv = __ldg(reinterpret_cast<const uint4*>(s + ((u.row0 >> 7) * col_chunks + col / 128) * 512 +
                                                          (u.row0 & 31) * 16));
    const uint32_t sw[4] = {sv.x, sv.y, sv.z, sv.w};
    constexpr int kOutBytes = OUT == MXFP8_F32 ? 4 : 2;
#pragma unroll
    for (int i = 0; i < kRowsPerWarp; ++i) {
        const int64_t row = u.row0 + 32 * i;
        if (row >= rows) return;
        const float scale = fp4_scale_value((sw[i] >> (8 * ((lane >> 2) & 3))) & 0xFFu);
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
        const bool vec = ((reinterpret_cast<uintptr_t>(out) + (uint64_t)o * kOutBytes) & 15) == 0;
        store8<OUT>(out, o, v, vec, ow, status);
    }
}

// Grid of one warp per (row of 32, 256 columns) of each row block; -1 if it
// does not fit a launch.
int64_t convert_blocks(int64_t row_blocks, int64_t segs) {
    const int64_t warps = row_blocks * 32 * segs;
    const int64_t blocks = (warps + kConvertThreads / 32 - 1) / (kConvertThreads / 32);
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
    const int64_t row_blocks = (a.m + 127) / 128, segs = (a.q_cols + kWarpCols - 1) / kWarpCols;
    const int64_t col_chunks = (a.q_cols + 127) / 128;
    const int64_t blocks = convert_blocks(row_blocks, segs);
    if (blocks < 0) return MXFP8_ERR_SHAPE;
    const bool aligned = (reinterpret_cast<uintptr_t>(a.x) & 15) == 0 && a.ld_x % 8 == 0;
    auto kernel = a.dtype == MXFP8_BF16
                      ? (aligned ? mxfp4_quantize_kernel<kBF16, true> : mxfp4_quantize_kernel<kBF16, false>)
                      : (aligned ? mxfp4_quantize_kernel<kFP16, true> : mxfp4_quantize_kernel<kFP16, false>);
    return launch_convert(kernel, blocks, stream, "mxfp4_quantize_kernel launch", static_cast<const uint8_t*>(a.x), a.m,
                          a.k, a.ld_x * 2, a.q, a.q_cols, a.ld_q, a.s, row_blocks, col_chunks, segs, a.qw, a.sw,
                          a.status);
}

int launch_mxfp4_dequantize(const uint8_t* q, int64_t rows, int64_t cols, int64_t ld_q, const uint8_t* s, void* out,
                            int out_dtype, int64_t ld_out, StoreWindow ow, unsigned int* status, cudaStream_t stream) {
    const int64_t row_blocks = (rows + 127) / 128, segs = (cols + kWarpCols - 1) / kWarpCols;
    const int64_t col_chunks = (cols + 127) / 128;
    const int64_t blocks = convert_blocks(row_blocks, segs);
    if (blocks < 0) return MXFP8_ERR_SHAPE;
    auto kernel = out_dtype == MXFP8_F32    ? mxfp4_dequantize_kernel<MXFP8_F32>
                  : out_dtype == MXFP8_BF16 ? mxfp4_dequantize_kernel<MXFP8_BF16>
                                            : mxfp4_dequantize_kernel<MXFP8_FP16>;
    return launch_convert(kernel, blocks, stream, "mxfp4_dequantize_kernel launch", q, rows, cols, ld_q, s, row_blocks,
                          col_chunks, segs, out, ld_out, ow, status);
}

}  // namespace mxfp8
