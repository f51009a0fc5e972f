// capi_cache.cu -- the extern "C" boundary declared in include/mxfp8_cache.h:
// argument validation, then the launches of cache_copy.cu and
// cache_attention.cu.
#include <cuda_runtime.h>

#include "../../include/mxfp8_cache.h"
#include "cache.cuh"
#include "launch.h"

using namespace mxfp8;

namespace {

constexpr int64_t kInt32Max = 2147483647;
constexpr int64_t kMaxStride = int64_t(1) << 38;
constexpr int kMaxHeads = 65536;  // a token's rows are counted in 32 bits

inline bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// Geometry of a cache with pages; *c is filled in.
int check_cache(const mxfp8_cache* cache, CacheShape* c) {
    if (!cache) return MXFP8_ERR_NULL_POINTER;
    const int s = cache->page_size;
    if (cache->num_pages < 0 || cache->heads < 1 || cache->heads > kMaxHeads || s < 1 || s > 4096 ||
        (s & (s - 1)) != 0 || cache->dim < 32 || cache->dim > 1024 || cache->dim % 32 != 0 ||
        cache->num_pages > ((int64_t(1) << 32) - 1) / cache->heads / s)
        return MXFP8_ERR_SHAPE;
    if (cache->num_pages > 0) {
        if (!cache->k || !cache->v || !cache->k_scales || !cache->v_scales) return MXFP8_ERR_NULL_POINTER;
        if (!aligned(cache->k, 16) || !aligned(cache->v, 16) || !aligned(cache->k_scales, 4) ||
            !aligned(cache->v_scales, 4))
            return MXFP8_ERR_ALIGNMENT;
    }
    c->num_pages = cache->num_pages;
    c->heads = cache->heads;
    c->page_shift = 0;
    while ((1 << c->page_shift) < s) ++c->page_shift;
    c->dim = cache->dim;
    return MXFP8_OK;
}

int check_table(const int32_t* table, int64_t stride, int64_t max_pages) {
    if (max_pages < 0 || max_pages > kInt32Max || stride < 0 || stride > kMaxStride) return MXFP8_ERR_SHAPE;
    if (max_pages > 0 && !table) return MXFP8_ERR_NULL_POINTER;
    return aligned(table, 4) ? MXFP8_OK : MXFP8_ERR_ALIGNMENT;
}

inline int64_t positions(const CacheShape& c) { return (c.num_pages * c.heads) << c.page_shift; }

// Whether rows of these strides from p all start on 32 bytes.
inline bool rows_aligned(const void* p, int64_t a, int64_t b) { return aligned(p, 32) && a % 16 == 0 && b % 16 == 0; }

int attention_shape(const CacheShape& c, int64_t batch, int64_t q_heads) {
    if (batch < 0 || q_heads < 1 || q_heads > kMaxHeads || q_heads % c.heads != 0 || batch > kInt32Max / q_heads ||
        c.page_shift < 1 || (c.dim != 64 && c.dim != 128 && c.dim != 192 && c.dim != 256))
        return MXFP8_ERR_SHAPE;
    return MXFP8_OK;
}

}  // namespace

extern "C" MXFP8_API int mxfp8_cache_write(const mxfp8_cache* cache, const void* k, int64_t k_token_stride,
                                           int64_t k_head_stride, const void* v, int64_t v_token_stride,
                                           int64_t v_head_stride, int dtype, int64_t tokens, const int64_t* slots,
                                           mxfp8_stream_t stream) {
    if (dtype != MXFP8_BF16 && dtype != MXFP8_FP16) return MXFP8_ERR_DTYPE;
    CacheWriteArgs a;
    if (int rc = check_cache(cache, &a.c)) return rc;
    for (int64_t s : {k_token_stride, k_head_stride, v_token_stride, v_head_stride})
        if (s < 0 || s > kMaxStride) return MXFP8_ERR_SHAPE;
    if (tokens < 0 || tokens > kInt32Max / (a.c.heads * (a.c.dim / 8))) return MXFP8_ERR_SHAPE;
    if (tokens == 0) return MXFP8_OK;
    if (!k || !v || !slots) return MXFP8_ERR_NULL_POINTER;
    if (!aligned(k, 2) || !aligned(v, 2) || !aligned(slots, 8)) return MXFP8_ERR_ALIGNMENT;
    int sms = 0;
    if (int rc = ready_device(&sms, &a.status)) return rc;
    a.k = static_cast<const uint16_t*>(k);
    a.v = static_cast<const uint16_t*>(v);
    a.k_token = k_token_stride;
    a.k_head = k_head_stride;
    a.v_token = v_token_stride;
    a.v_head = v_head_stride;
    a.k_vec = rows_aligned(k, k_token_stride, k_head_stride);
    a.v_vec = rows_aligned(v, v_token_stride, v_head_stride);
    a.tokens = tokens;
    a.slots = slots;
    a.k_out = static_cast<uint8_t*>(cache->k);
    a.v_out = static_cast<uint8_t*>(cache->v);
    a.k_scales = static_cast<uint8_t*>(cache->k_scales);
    a.v_scales = static_cast<uint8_t*>(cache->v_scales);
    const int64_t rows = positions(a.c);
    a.kw = make_window(cache->k, rows * a.c.dim);
    a.vw = make_window(cache->v, rows * a.c.dim);
    a.ksw = make_window(cache->k_scales, rows * (a.c.dim / 32));
    a.vsw = make_window(cache->v_scales, rows * (a.c.dim / 32));
    return launch_cache_write(a, dtype, static_cast<cudaStream_t>(stream));
}

extern "C" MXFP8_API int mxfp8_cache_read(const mxfp8_cache* cache, const int32_t* table, int64_t table_stride,
                                          int64_t max_pages, int64_t batch, const int32_t* starts, int64_t total,
                                          void* k_out, void* v_out, int out_dtype, mxfp8_stream_t stream) {
    if (out_dtype != MXFP8_BF16 && out_dtype != MXFP8_FP16 && out_dtype != MXFP8_F32) return MXFP8_ERR_DTYPE;
    CacheReadArgs a;
    if (int rc = check_cache(cache, &a.c)) return rc;
    if (batch < 0 || batch > kInt32Max || total < 0 || total > kInt32Max) return MXFP8_ERR_SHAPE;
    if (int rc = check_table(table, table_stride, max_pages)) return rc;
    if (total == 0 || batch == 0) return MXFP8_OK;
    if (!starts || !k_out || !v_out) return MXFP8_ERR_NULL_POINTER;
    if (!aligned(starts, 4) || !aligned(k_out, 16) || !aligned(v_out, 16)) return MXFP8_ERR_ALIGNMENT;
    int sms = 0;
    if (int rc = ready_device(&sms, &a.status)) return rc;
    a.k = static_cast<const uint8_t*>(cache->k);
    a.v = static_cast<const uint8_t*>(cache->v);
    a.k_scales = static_cast<const uint8_t*>(cache->k_scales);
    a.v_scales = static_cast<const uint8_t*>(cache->v_scales);
    a.table = table;
    a.table_stride = table_stride;
    a.max_pages = max_pages;
    a.batch = batch;
    a.starts = starts;
    a.total = total;
    a.k_out = static_cast<uint8_t*>(k_out);
    a.v_out = static_cast<uint8_t*>(v_out);
    const int64_t bytes = total * a.c.heads * a.c.dim * (out_dtype == MXFP8_F32 ? 4 : 2);
    a.kw = make_window(k_out, bytes);
    a.vw = make_window(v_out, bytes);
    return launch_cache_read(a, out_dtype, static_cast<cudaStream_t>(stream));
}

extern "C" MXFP8_API int64_t mxfp8_cache_attention_workspace(const mxfp8_cache* cache, int64_t batch, int64_t q_heads) {
    CacheShape c;
    if (int rc = check_cache(cache, &c)) return rc;
    if (int rc = attention_shape(c, batch, q_heads)) return rc;
    int sms = 0;
    unsigned int* status = nullptr;
    if (int rc = ready_device(&sms, &status)) return rc;
    return cache_attention_workspace(c, batch, (int)q_heads, sms);
}

extern "C" MXFP8_API int mxfp8_cache_attention(const mxfp8_cache* cache, const void* q, int64_t q_batch_stride,
                                               int64_t q_head_stride, int dtype, int64_t batch, int64_t q_heads,
                                               const int32_t* table, int64_t table_stride, int64_t max_pages,
                                               const int32_t* lengths, float scale, void* out, float* lse,
                                               void* workspace, int64_t workspace_bytes, mxfp8_stream_t stream) {
    if (dtype != MXFP8_BF16 && dtype != MXFP8_FP16) return MXFP8_ERR_DTYPE;
    CacheAttentionArgs a;
    if (int rc = check_cache(cache, &a.c)) return rc;
    if (int rc = attention_shape(a.c, batch, q_heads)) return rc;
    if (int rc = check_table(table, table_stride, max_pages)) return rc;
    if ((max_pages << a.c.page_shift) > kInt32Max - 1024 || q_batch_stride < 0 || q_batch_stride > kMaxStride ||
        q_head_stride < 0 || q_head_stride > kMaxStride ||
        batch > (int64_t(1) << 34) / ((max_pages << a.c.page_shift) + 1024))
        return MXFP8_ERR_SHAPE;
    if (batch == 0) return MXFP8_OK;
    if (!q || !lengths || !out || !workspace) return MXFP8_ERR_NULL_POINTER;
    if (!aligned(q, 2) || !aligned(lengths, 4) || !aligned(out, 16) || !aligned(lse, 4) || !aligned(workspace, 16))
        return MXFP8_ERR_ALIGNMENT;
    int sms = 0;
    if (int rc = ready_device(&sms, &a.status)) return rc;
    const int64_t need = cache_attention_workspace(a.c, batch, (int)q_heads, sms);
    if (workspace_bytes < need) return MXFP8_ERR_WORKSPACE;
    a.k = static_cast<const uint8_t*>(cache->k);
    a.v = static_cast<const uint8_t*>(cache->v);
    a.k_scales = static_cast<const uint8_t*>(cache->k_scales);
    a.v_scales = static_cast<const uint8_t*>(cache->v_scales);
    a.q = static_cast<const uint16_t*>(q);
    a.q_batch = q_batch_stride;
    a.q_head = q_head_stride;
    a.q_bf16 = dtype == MXFP8_BF16;
    a.batch = batch;
    a.q_heads = (int)q_heads;
    a.table = table;
    a.table_stride = table_stride;
    a.max_pages = max_pages;
    a.lengths = lengths;
    a.scale = scale;
    a.out = static_cast<uint16_t*>(out);
    a.lse = lse;
    a.workspace = workspace;
    a.ow = make_window(out, batch * q_heads * a.c.dim * 2);
    a.lw = make_window(lse, lse ? batch * q_heads * 4 : 0);
    a.ww = StoreWindow{static_cast<uint8_t*>(workspace), static_cast<uint8_t*>(workspace) + need};
    return launch_cache_attention(a, sms, static_cast<cudaStream_t>(stream));
}
