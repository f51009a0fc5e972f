/*
 * mxfp8_cache.h -- C ABI of the MXFP8 key/value cache in libmxfp8.so: rows
 * quantized into pages as they are written, read back widened, and attended
 * to by single query tokens (sm_100a).
 *
 * A cache is four buffers over num_pages pages of page_size positions (a
 * power of two, at most 4096):
 *   k, v               (num_pages, heads, page_size, dim) E4M3 bytes
 *   k_scales, v_scales (num_pages, heads, page_size, dim / 32) UE8M0 bytes
 * all contiguous, dim % 32 == 0 and dim <= 1024, heads <= 65536, k and v
 * 16-byte aligned, the scales 4-byte aligned, num_pages * heads * page_size <
 * 2^32.  A position
 * (slot) is page * page_size + offset.  Rows are quantized by the recipe of
 * mxfp8_quantize along dim, so a row's bytes equal those of quantizing it
 * alone.
 *
 * Indexes live on the device and are checked there: a page or slot outside
 * the cache, or a sequence that runs past its row of the page table, is never
 * followed; the call does what its entry says instead and sets bit 64 of the
 * device status word (mxfp8_device_status).
 *
 * Conventions, status codes and streams are those of mxfp8.h.  No
 * counterpart in the reference (it has no cache).
 */
#ifndef MXFP8_CACHE_H_
#define MXFP8_CACHE_H_

#include "mxfp8.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct mxfp8_cache {
    void* k;
    void* v;
    void* k_scales;
    void* v_scales;
    int64_t num_pages;
    int32_t heads;
    int32_t page_size;
    int32_t dim;
} mxfp8_cache;

/* Quantize k and v (tokens, heads, dim) of dtype MXFP8_BF16 or MXFP8_FP16 into
 * the positions slots[0 .. tokens - 1].  Strides in elements; the last
 * dimension is contiguous; any strides and any 2-byte aligned base.  A negative slot
 * skips its token; a slot past the cache is skipped and reported.  Slots that
 * are written must differ: where two tokens name the same position, its bytes
 * are an unspecified mix of both.  Other positions keep their bytes. */
MXFP8_API int mxfp8_cache_write(const mxfp8_cache* cache, const void* k, int64_t k_token_stride, int64_t k_head_stride,
                                const void* v, int64_t v_token_stride, int64_t v_head_stride, int dtype,
                                int64_t tokens, const int64_t* slots, mxfp8_stream_t stream);

/* Widen a batch's rows into k_out and v_out (total, heads, dim), contiguous,
 * of out_dtype (MXFP8_BF16, MXFP8_FP16 or MXFP8_F32), 16-byte aligned.
 * Position j of sequence b, j < starts[b + 1] - starts[b], comes from page
 * table[b * table_stride + j / page_size] and goes to row starts[b] + j.
 * starts (batch + 1 values) does not fall.  Rows at or past total, and rows of
 * the outputs that no sequence covers, are left as they were; a row whose page
 * is outside the cache or the table is written as zeros and reported. */
MXFP8_API int mxfp8_cache_read(const mxfp8_cache* cache, const int32_t* table, int64_t table_stride,
                               int64_t max_pages, int64_t batch, const int32_t* starts, int64_t total, void* k_out,
                               void* v_out, int out_dtype, mxfp8_stream_t stream);

/* Workspace of mxfp8_cache_attention in bytes for these sizes on the current
 * device, or a negative mxfp8_status. */
MXFP8_API int64_t mxfp8_cache_attention_workspace(const mxfp8_cache* cache, int64_t batch, int64_t q_heads);

/* out[b, h] = softmax_j(scale * q[b, h] . k_j) v_j over j < lengths[b], the
 * cached rows of KV head h / (q_heads / heads): one query token a sequence.
 * q (batch, q_heads, dim) of dtype MXFP8_BF16 or MXFP8_FP16, strides in
 * elements, last dimension contiguous; out contiguous of the same type and
 * lse (batch, q_heads) f32 or NULL: log of the sum of exp(scale * q . k_j).
 * dim is 64, 128, 192 or 256, page_size at least 2, q_heads a multiple of
 * heads, max_pages * page_size < 2^31 - 1024, and batch times that at most
 * 2^34.  A length of 0 (or below) gives zeros and lse -inf; a position whose
 * page is outside the cache takes no part, as if it were not there, and is
 * reported; a length past the table is cut to it and reported.  Scores and sums
 * are held in f32; a weight is held to 2^-22 of itself or 2^-28 of the largest
 * one, whichever is more, whatever the scales of V's blocks are (V more than
 * 2^70 below its head's sums so far counts as zero); outputs are rounded once.  A score
 * overflows where a K block's scale is 2^96 or more (the query is held with its
 * largest element near 2^14; elements 2^28 below it lose bits).  workspace is 16-byte aligned scratch of
 * one call at a time; its contents do not matter before or after. */
MXFP8_API int mxfp8_cache_attention(const mxfp8_cache* cache, const void* q, int64_t q_batch_stride,
                                    int64_t q_head_stride, int dtype, int64_t batch, int64_t q_heads,
                                    const int32_t* table, int64_t table_stride, int64_t max_pages,
                                    const int32_t* lengths, float scale, void* out, float* lse, void* workspace,
                                    int64_t workspace_bytes, mxfp8_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* MXFP8_CACHE_H_ */
