// cache.cuh -- launch arguments of the paged MXFP8 cache's kernels, after
// validation.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "cache_index.h"
#include "guard.cuh"

namespace mxfp8 {

constexpr unsigned kErrCacheIndex = 64u;  // device status bit: an index was not followed

// Eight 16-bit values at p; 16-byte load where `vec` says it is aligned.
__device__ __forceinline__ uint4 load8(const uint16_t* p, bool vec) {
    if (vec) return __ldcs(reinterpret_cast<const uint4*>(p));
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (uint32_t)p[2 * i] | ((uint32_t)p[2 * i + 1] << 16);
    return make_uint4(w[0], w[1], w[2], w[3]);
}

struct CacheWriteArgs {
    CacheShape c;
    const uint16_t* k;
    const uint16_t* v;
    int64_t k_token, k_head, v_token, v_head;  // strides in elements
    bool k_vec, v_vec;                         // every row starts on a 32-byte boundary
    int64_t tokens;
    const int64_t* slots;
    uint8_t *k_out, *v_out, *k_scales, *v_scales;
    StoreWindow kw, vw, ksw, vsw;
    unsigned int* status;
};

struct CacheReadArgs {
    CacheShape c;
    const uint8_t *k, *v, *k_scales, *v_scales;
    const int32_t* table;
    int64_t table_stride, max_pages, batch;
    const int32_t* starts;
    int64_t total;
    uint32_t cta_rows;  // set by the launch
    uint8_t *k_out, *v_out;
    StoreWindow kw, vw;
    unsigned int* status;
};

struct CacheAttentionArgs {
    CacheShape c;
    const uint8_t *k, *v, *k_scales, *v_scales;
    const uint16_t* q;
    int64_t q_batch, q_head;  // strides in elements
    bool q_bf16;
    int64_t batch;
    int q_heads;
    const int32_t* table;
    int64_t table_stride, max_pages;
    const int32_t* lengths;
    float scale;
    uint16_t* out;
    float* lse;
    void* workspace;
    StoreWindow ow, lw, ww;  // out, lse, workspace
    unsigned int* status;
};

int launch_cache_write(const CacheWriteArgs& a, int dtype, cudaStream_t stream);
int launch_cache_read(const CacheReadArgs& a, int out_dtype, cudaStream_t stream);
int launch_cache_attention(const CacheAttentionArgs& a, int sm_count, cudaStream_t stream);
// Bytes of workspace that launch_cache_attention needs.
int64_t cache_attention_workspace(const CacheShape& c, int64_t batch, int q_heads, int sm_count);

}  // namespace mxfp8
