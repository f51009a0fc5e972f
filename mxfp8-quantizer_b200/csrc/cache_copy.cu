// cache_copy.cu -- rows into and out of the paged MXFP8 cache.
//
// Both are byte streams bound by HBM (3 + 1/32 bytes an element to write, 1 +
// 1/32 + the output's to read back), and by latency for a decode step's few
// rows, so K and V go in one launch and every thread has both in flight.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "../../include/mxfp8_cache.h"
#include "cache.cuh"
#include "launch.h"
#include "ptx.cuh"
#include "recipe.cuh"

namespace mxfp8 {

namespace {

constexpr int kCopyThreads = 256;

// The recipe of mxfp8_quantize on a block of 32 held by four lanes, eight
// values each: this lane's payload bytes and the block's scale byte.
template <int DT>
__device__ __forceinline__ uint32_t quantize_quarter(const uint4& v, uint2& q) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t a = __vmaxu2(__vmaxu2(w[0] & 0x7FFF7FFFu, w[1] & 0x7FFF7FFFu),
                          __vmaxu2(w[2] & 0x7FFF7FFFu, w[3] & 0x7FFF7FFFu));
    a = max(a & 0xFFFFu, a >> 16);
    a = max(a, __shfl_xor_sync(0xFFFFFFFFu, a, 1));
    a = max(a, __shfl_xor_sync(0xFFFFFFFFu, a, 2));
    uint32_t byte;
    float inv;
    scale_from_amax<DT>(a, byte, inv);
    q.x = quantize_pair<DT>(w[0], inv) | (quantize_pair<DT>(w[1], inv) << 16);
    q.y = quantize_pair<DT>(w[2], inv) | (quantize_pair<DT>(w[3], inv) << 16);
    return byte;
}

// One thread per eight elements of a token's (heads, dim) rows, of K and of V.
template <int DT>
__global__ void __launch_bounds__(kCopyThreads) cache_write_kernel(const CacheWriteArgs a) {
    grid_launch_dependents();
    grid_wait_prerequisites();
    const uint32_t pieces = (uint32_t)a.c.dim / 8;        // of a row; a multiple of 4
    const uint32_t per_token = pieces * (uint32_t)a.c.heads;
    const uint32_t idx = blockIdx.x * kCopyThreads + threadIdx.x;
    const uint32_t token = idx / per_token;
    const bool live = token < (uint32_t)a.tokens;         // the same for the four lanes of a block
    const uint32_t in = idx - token * per_token;
    const uint32_t head = in / pieces, piece = in - head * pieces;
    int64_t row = kNoRow;
    if (live) {
        const int64_t slot = a.slots[token];
        if (slot >= 0) {
            row = cache_row(a.c, slot >> a.c.page_shift, (int)head, (int)(slot & ((1 << a.c.page_shift) - 1)));
            if (row == kNoRow && in == 0 && a.status) atomicOr(a.status, kErrCacheIndex);
        }
    }
    uint4 kv = make_uint4(0u, 0u, 0u, 0u), vv = kv;
    if (row != kNoRow) {
        const int64_t at = 8 * (int64_t)piece;
        kv = load8(a.k + (int64_t)token * a.k_token + (int64_t)head * a.k_head + at, a.k_vec);
        vv = load8(a.v + (int64_t)token * a.v_token + (int64_t)head * a.v_head + at, a.v_vec);
    }
    uint2 kq, vq;
    const uint32_t kb = quantize_quarter<DT>(kv, kq), vb = quantize_quarter<DT>(vv, vq);
    if (row == kNoRow) return;
    gstore_plain(reinterpret_cast<uint2*>(a.k_out + row * a.c.dim + 8 * piece), kq, a.kw, a.status);
    gstore_plain(reinterpret_cast<uint2*>(a.v_out + row * a.c.dim + 8 * piece), vq, a.vw, a.status);
    if ((piece & 3) == 0) {
        const int64_t s = row * (a.c.dim / 32) + (piece >> 2);
        gstore_plain(a.k_scales + s, (uint8_t)kb, a.ksw, a.status);
        gstore_plain(a.v_scales + s, (uint8_t)vb, a.vsw, a.status);
    }
}

__device__ __forceinline__ float2 e4m3_pair(uint32_t two_bytes) {
    uint32_t h2;
    asm("{\n\t.reg .b16 t;\n\tcvt.u16.u32 t, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, t;\n\t}" : "=r"(h2) : "r"(two_bytes));
    return __half22float2(*reinterpret_cast<const __half2*>(&h2));
}

// Eight payload bytes times their block's scale to out (16-byte aligned).
template <int OUT>
__device__ __forceinline__ void widen8(const uint2& q, uint32_t byte, uint8_t* out, const StoreWindow& w,
                                       unsigned int* status) {
    const float scale = ue8m0_value(byte);
    float f[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 t = e4m3_pair(((i & 2 ? q.y : q.x) >> (16 * (i & 1))) & 0xFFFFu);
        f[2 * i] = __fmul_rn(t.x, scale);
        f[2 * i + 1] = __fmul_rn(t.y, scale);
    }
    if constexpr (OUT == MXFP8_F32) {
        gstore(reinterpret_cast<float4*>(out), make_float4(f[0], f[1], f[2], f[3]), w, status);
        gstore(reinterpret_cast<float4*>(out) + 1, make_float4(f[4], f[5], f[6], f[7]), w, status);
    } else {
        uint32_t h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (OUT == MXFP8_BF16) {
                const __nv_bfloat162 t = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
                h[i] = *reinterpret_cast<const uint32_t*>(&t);
            } else {
                const __half2 t = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
                h[i] = *reinterpret_cast<const uint32_t*>(&t);
            }
        }
        gstore(reinterpret_cast<uint4*>(out), make_uint4(h[0], h[1], h[2], h[3]), w, status);
    }
}

constexpr int kReadRows = 8;          // output rows of a CTA
constexpr int64_t kLeave = -2;        // a row that no sequence covers

// A CTA widens kReadRows consecutive output rows.  Their cache rows (of head
// 0) are looked up once, by one thread each: which sequence covers the row,
// then its page.
template <int OUT>
__global__ void __launch_bounds__(kCopyThreads) cache_read_kernel(const CacheReadArgs a) {
    __shared__ int64_t source[kReadRows];
    grid_launch_dependents();
    grid_wait_prerequisites();
    const int64_t row0 = (int64_t)blockIdx.x * kReadRows;
    if (threadIdx.x < kReadRows) {
        const int64_t row = row0 + threadIdx.x;
        int64_t from = kLeave;
        if (row < a.total) {
            const int64_t b = sequence_of(a.starts, a.batch, row);
            if (b >= 0 && b < a.batch) {
                const int64_t at = row - a.starts[b];
                const int64_t page = table_page(a.table, a.table_stride, a.max_pages, b, at, a.c.page_shift);
                from = cache_row(a.c, page, 0, (int)(at & ((1 << a.c.page_shift) - 1)));
                if (from == kNoRow && a.status) atomicOr(a.status, kErrCacheIndex);
            }
        }
        source[threadIdx.x] = from;
    }
    __syncthreads();
    constexpr int kEs = OUT == MXFP8_F32 ? 4 : 2;
    const uint32_t pieces = (uint32_t)a.c.dim / 8;
    const uint32_t per_row = pieces * (uint32_t)a.c.heads;
#pragma unroll 2
    for (uint32_t i = threadIdx.x; i < kReadRows * per_row; i += kCopyThreads) {
        const uint32_t r = i / per_row, in = i - r * per_row;
        const int64_t from = source[r];
        if (from == kLeave) continue;
        const uint32_t head = in / pieces, piece = in - head * pieces;
        uint2 kq = make_uint2(0u, 0u), vq = kq;
        uint32_t kb = 0, vb = 0;
        if (from != kNoRow) {
            const int64_t row = from + ((int64_t)head << a.c.page_shift);
            kq = __ldcs(reinterpret_cast<const uint2*>(a.k + row * a.c.dim + 8 * piece));
            vq = __ldcs(reinterpret_cast<const uint2*>(a.v + row * a.c.dim + 8 * piece));
            const int64_t s = row * (a.c.dim / 32) + (piece >> 2);
            kb = __ldg(a.k_scales + s);
            vb = __ldg(a.v_scales + s);
        }
        const int64_t at = ((row0 + r) * per_row + in) * (8 * kEs);
        widen8<OUT>(kq, kb, a.k_out + at, a.kw, a.status);
        widen8<OUT>(vq, vb, a.v_out + at, a.vw, a.status);
    }
}

template <typename Args>
int launch_copy(void (*kernel)(const Args), int64_t blocks, cudaStream_t stream, const char* what, const Args& a) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(kCopyThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
    if (e == cudaSuccess) e = cudaGetLastError();
    if (e != cudaSuccess) {
        set_last_error(what, (int)e);
        return MXFP8_ERR_CUDA;
    }
    return MXFP8_OK;
}

}  // namespace

int launch_cache_write(const CacheWriteArgs& a, int dtype, cudaStream_t stream) {
    const int64_t threads = a.tokens * a.c.heads * (a.c.dim / 8);
    const int64_t blocks = (threads + kCopyThreads - 1) / kCopyThreads;
    return launch_copy(dtype == MXFP8_BF16 ? cache_write_kernel<kBF16> : cache_write_kernel<kFP16>, blocks, stream,
                       "cache_write_kernel launch", a);
}

int launch_cache_read(const CacheReadArgs& a, int out_dtype, cudaStream_t stream) {
    const int64_t blocks = (a.total + kReadRows - 1) / kReadRows;
    auto kernel = out_dtype == MXFP8_F32    ? cache_read_kernel<MXFP8_F32>
                  : out_dtype == MXFP8_BF16 ? cache_read_kernel<MXFP8_BF16>
                                            : cache_read_kernel<MXFP8_FP16>;
    return launch_copy(kernel, blocks, stream, "cache_read_kernel launch", a);
}

}  // namespace mxfp8
