// cache_copy.cu -- rows into and out of the paged MXFP8 cache.
//
// Both are byte streams bound by HBM (3 + 1/32 bytes an element to write, 1 +
// 1/32 + the output's to read back), and by latency for a decode step's few
// rows, so K and V go in one launch and every thread has both in flight, 16
// elements of each: 32-byte loads of what is written, 32-byte stores of what is read.
// Measured: 8191 tokens of 8 x 128 written at scattered slots 9.3 us = 5.5 TB/s
// (10.3 with 8 elements a thread); 67.7 k rows of them read back 68.7 us = 6.1 TB/s
// (80.8 with 8 elements and a binary search a row); 64 tokens 1.8 us.
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

// Sixteen 16-bit values at p, half a block; 32-byte load where `vec` says it is aligned.
__device__ __forceinline__ void load_half_block(const uint16_t* p, bool vec, uint32_t (&w)[8]) {
    if (vec) {
        asm volatile("ld.global.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                     : "l"(p));
    } else {
        const uint4 a = load8(p, (reinterpret_cast<uintptr_t>(p) & 15) == 0);
        const uint4 b = load8(p + 8, (reinterpret_cast<uintptr_t>(p) & 15) == 0);
        w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
        w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
    }
}

// The recipe of mxfp8_quantize on a block of 32 held by two lanes: this lane's
// payload bytes and the block's scale byte.
template <int DT>
__device__ __forceinline__ uint32_t quantize_half(const uint32_t (&w)[8], uint4& q) {
    uint32_t a = w[0] & 0x7FFF7FFFu;
#pragma unroll
    for (int i = 1; i < 8; ++i) a = __vmaxu2(a, w[i] & 0x7FFF7FFFu);
    a = max(a & 0xFFFFu, a >> 16);
    a = max(a, __shfl_xor_sync(0xFFFFFFFFu, a, 1));
    uint32_t byte;
    float inv;
    scale_from_amax<DT>(a, byte, inv);
    q.x = quantize_pair<DT>(w[0], inv) | (quantize_pair<DT>(w[1], inv) << 16);
    q.y = quantize_pair<DT>(w[2], inv) | (quantize_pair<DT>(w[3], inv) << 16);
    q.z = quantize_pair<DT>(w[4], inv) | (quantize_pair<DT>(w[5], inv) << 16);
    q.w = quantize_pair<DT>(w[6], inv) | (quantize_pair<DT>(w[7], inv) << 16);
    return byte;
}

// One thread per half block (16 elements) of a token's (heads, dim) rows, of K
// and of V.
template <int DT>
__global__ void __launch_bounds__(kCopyThreads) cache_write_kernel(const CacheWriteArgs a) {
    grid_launch_dependents();
    grid_wait_prerequisites();
    const uint32_t pieces = (uint32_t)a.c.dim / 16;       // of a row; an even number
    const uint32_t per_token = pieces * (uint32_t)a.c.heads;
    const uint32_t idx = blockIdx.x * kCopyThreads + threadIdx.x;
    const uint32_t token = idx / per_token;
    const bool live = token < (uint32_t)a.tokens;         // the same for the two lanes of a block
    const uint32_t in = idx - token * per_token;
    const uint32_t head = in / pieces, piece = in - head * pieces;
    uint32_t kv[8] = {0u}, vv[8] = {0u};
    int64_t row = kNoRow;
    if (live) {
        // the rows are read whether the slot takes them or not: not to wait for it first
        const int64_t slot = a.slots[token];
        const int64_t at = 16 * (int64_t)piece;
        load_half_block(a.k + (int64_t)token * a.k_token + (int64_t)head * a.k_head + at, a.k_vec, kv);
        load_half_block(a.v + (int64_t)token * a.v_token + (int64_t)head * a.v_head + at, a.v_vec, vv);
        if (slot >= 0) {
            row = cache_row(a.c, slot >> a.c.page_shift, (int)head, (int)(slot & ((1 << a.c.page_shift) - 1)));
            if (row == kNoRow && in == 0 && a.status) atomicOr(a.status, kErrCacheIndex);
        }
    }
    uint4 kq, vq;
    const uint32_t kb = quantize_half<DT>(kv, kq), vb = quantize_half<DT>(vv, vq);
    if (row == kNoRow) return;
    gstore_plain(reinterpret_cast<uint4*>(a.k_out + row * a.c.dim + 16 * piece), kq, a.kw, a.status);
    gstore_plain(reinterpret_cast<uint4*>(a.v_out + row * a.c.dim + 16 * piece), vq, a.vw, a.status);
    if ((piece & 1) == 0) {
        const int64_t s = row * (a.c.dim / 32) + (piece >> 1);
        gstore_plain(a.k_scales + s, (uint8_t)kb, a.ksw, a.status);
        gstore_plain(a.v_scales + s, (uint8_t)vb, a.vsw, a.status);
    }
}

__device__ __forceinline__ float2 e4m3_pair(uint32_t two_bytes) {
    uint32_t h2;
    asm("{\n\t.reg .b16 t;\n\tcvt.u16.u32 t, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, t;\n\t}" : "=r"(h2) : "r"(two_bytes));
    return __half22float2(*reinterpret_cast<const __half2*>(&h2));
}

// Sixteen payload bytes times their block's scale to out (16-byte aligned;
// `vec`: 32).
template <int OUT>
__device__ __forceinline__ void widen16(const uint4& q, uint32_t byte, uint8_t* out, bool vec, const StoreWindow& w,
                                        unsigned int* status) {
    const float scale = ue8m0_value(byte);
    const uint32_t in[4] = {q.x, q.y, q.z, q.w};
    constexpr int kWords = OUT == MXFP8_F32 ? 16 : 8;
    uint32_t h[kWords];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float2 t = e4m3_pair((in[i / 2] >> (16 * (i & 1))) & 0xFFFFu);
        const float x = __fmul_rn(t.x, scale), y = __fmul_rn(t.y, scale);
        if constexpr (OUT == MXFP8_F32) {
            h[2 * i] = __float_as_uint(x);
            h[2 * i + 1] = __float_as_uint(y);
        } else if constexpr (OUT == MXFP8_BF16) {
            const __nv_bfloat162 p = __floats2bfloat162_rn(x, y);
            h[i] = *reinterpret_cast<const uint32_t*>(&p);
        } else {
            const __half2 p = __floats2half2_rn(x, y);
            h[i] = *reinterpret_cast<const uint32_t*>(&p);
        }
    }
#pragma unroll
    for (int i = 0; i < kWords; i += 8) {
        if (vec) {
            gstore32(out + 4 * i, h + i, w, status);
        } else {
            gstore(reinterpret_cast<uint4*>(out + 4 * i), make_uint4(h[i], h[i + 1], h[i + 2], h[i + 3]), w, status);
            gstore(reinterpret_cast<uint4*>(out + 4 * i) + 1, make_uint4(h[i + 4], h[i + 5], h[i + 6], h[i + 7]), w,
                   status);
        }
    }
}

constexpr int kMinReadRows = 8, kMaxReadRows = 128;  // output rows of a CTA: two half blocks a thread where it can be
constexpr int64_t kLeave = -2;        // a row that no sequence covers

// A CTA widens a.cta_rows consecutive output rows.  Their cache rows (of head 0)
// are looked up once: all threads count the starts at or before the first row,
// one round of loads for a batch below 256, then one thread a row goes on from
// there and takes the page.
template <int OUT>
__global__ void __launch_bounds__(kCopyThreads) cache_read_kernel(const CacheReadArgs a) {
    __shared__ int64_t source[kMaxReadRows];
    grid_launch_dependents();
    grid_wait_prerequisites();
    const int64_t row0 = (int64_t)blockIdx.x * a.cta_rows;
    int64_t from = -1;
    for (int64_t b0 = 0; b0 <= a.batch; b0 += kCopyThreads)
        from += __syncthreads_count(b0 + threadIdx.x <= a.batch && a.starts[b0 + threadIdx.x] <= row0);
    if (threadIdx.x < a.cta_rows) {
        const int64_t row = row0 + threadIdx.x;
        int64_t at_row = kLeave;
        if (row < a.total) {
            const int64_t b = sequence_from(a.starts, a.batch, from, row);
            if (b >= 0 && b < a.batch) {
                const int64_t at = row - a.starts[b];
                const int64_t page = table_page(a.table, a.table_stride, a.max_pages, b, at, a.c.page_shift);
                at_row = cache_row(a.c, page, 0, (int)(at & ((1 << a.c.page_shift) - 1)));
                if (at_row == kNoRow && a.status) atomicOr(a.status, kErrCacheIndex);
            }
        }
        source[threadIdx.x] = at_row;
    }
    __syncthreads();
    constexpr int kEs = OUT == MXFP8_F32 ? 4 : 2;
    const bool vec = ((reinterpret_cast<uintptr_t>(a.k_out) | reinterpret_cast<uintptr_t>(a.v_out)) & 31) == 0;
    const uint32_t pieces = (uint32_t)a.c.dim / 16;
    const uint32_t per_row = pieces * (uint32_t)a.c.heads;
#pragma unroll 2
    for (uint32_t i = threadIdx.x; i < a.cta_rows * per_row; i += kCopyThreads) {
        const uint32_t r = i / per_row, in = i - r * per_row;
        const int64_t src = source[r];
        if (src == kLeave) continue;
        const uint32_t head = in / pieces, piece = in - head * pieces;
        uint4 kq = make_uint4(0u, 0u, 0u, 0u), vq = kq;
        uint32_t kb = 0, vb = 0;
        if (src != kNoRow) {
            const int64_t row = src + ((int64_t)head << a.c.page_shift);
            kq = __ldcs(reinterpret_cast<const uint4*>(a.k + row * a.c.dim + 16 * piece));
            vq = __ldcs(reinterpret_cast<const uint4*>(a.v + row * a.c.dim + 16 * piece));
            const int64_t s = row * (a.c.dim / 32) + (piece >> 1);
            kb = a.k_scales[s];
            vb = a.v_scales[s];
        }
        const int64_t at = ((row0 + r) * per_row + in) * (16 * kEs);
        widen16<OUT>(kq, kb, a.k_out + at, vec, a.kw, a.status);
        widen16<OUT>(vq, vb, a.v_out + at, vec, a.vw, a.status);
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
    const int64_t threads = a.tokens * a.c.heads * (a.c.dim / 16);
    const int64_t blocks = (threads + kCopyThreads - 1) / kCopyThreads;
    return launch_copy(dtype == MXFP8_BF16 ? cache_write_kernel<kBF16> : cache_write_kernel<kFP16>, blocks, stream,
                       "cache_write_kernel launch", a);
}

int launch_cache_read(const CacheReadArgs& args, int out_dtype, cudaStream_t stream) {
    CacheReadArgs a = args;
    // narrow rows: more of them a CTA (131 k rows of 1 x 128: 11.1 us, 18.0 with 8 rows a CTA), as long as there are
    // CTAs for the SMs (1 k rows of 4 x 64: 2.4 us, 3.2 with 32)
    int64_t rows = 2 * kCopyThreads / ((int64_t)a.c.heads * (a.c.dim / 16));
    if (rows > a.total / 256) rows = a.total / 256;
    a.cta_rows = (uint32_t)(rows < kMinReadRows ? kMinReadRows : rows > kMaxReadRows ? kMaxReadRows : rows);
    const int64_t blocks = (a.total + a.cta_rows - 1) / a.cta_rows;
    auto kernel = out_dtype == MXFP8_F32    ? cache_read_kernel<MXFP8_F32>
                  : out_dtype == MXFP8_BF16 ? cache_read_kernel<MXFP8_BF16>
                                            : cache_read_kernel<MXFP8_FP16>;
    return launch_copy(kernel, blocks, stream, "cache_read_kernel launch", a);
}

}  // namespace mxfp8
