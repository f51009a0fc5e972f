/*
 * mxfp4.h -- C ABI of the 4-bit half of libmxfp8.so: MXFP4 quantization,
 * its inverse, and the product of two MXFP4 matrices (sm_100a).
 *
 * An MXFP4 matrix (rows, cols), cols % 32 == 0, is a payload of two E2M1
 * codes a byte (the even column in the low four bits), row-major with a row
 * stride of ld bytes, plus one UE8M0 scale byte per 1x32 block along the
 * columns in the same 128x4 chunk layout as the MXFP8 scales (mxfp8.h);
 * mxfp8_scale_storage_bytes(rows, cols) gives the scale storage.  Payloads
 * and scales are 16-byte aligned and ld % 16 == 0, so that the product can
 * read every matrix that the quantizer writes.
 *
 * Conventions, status codes and streams are those of mxfp8.h.  No
 * counterpart in the reference (its quantizer writes E4M3 only).
 */
#ifndef MXFP4_H_
#define MXFP4_H_

#include "mxfp8.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Quantize x (m, k) of dtype MXFP8_BF16 or MXFP8_FP16, row stride ld_x
 * elements (any, >= k; x 2-byte aligned), into q (m, q_cols / 2 bytes) and s,
 * q_cols = ceil(k / 32) * 32; columns k .. q_cols - 1 count as zeros.
 * For a block with largest magnitude a: a finite and not zero: scale 2^e with
 * the smallest e >= -127 such that a <= 6 * 2^e (nothing saturates), byte
 * e + 127, codes x * 2^-e rounded to nearest, ties to the even code; a zero:
 * byte 127, codes 0 (the sign of a zero is kept); an inf or a NaN in the
 * block: byte 255, which decodes to NaN, and codes 0.  Scale bytes of the
 * padding (rows m .. ceil(m / 128) * 128, columns up to the next multiple of
 * 4 blocks) are written as 0.  s_bytes >= mxfp8_scale_storage_bytes(m, q_cols). */
MXFP8_API int mxfp4_quantize(const void* x, int dtype, int64_t m, int64_t k, int64_t ld_x, void* q, int64_t ld_q,
                             void* s, int64_t s_bytes, mxfp8_stream_t stream);

/* out (rows, cols) of out_dtype (MXFP8_BF16, MXFP8_FP16 or MXFP8_F32), row
 * stride ld_out elements = E2M1 value * 2^(scale byte - 127), rounded once;
 * scale byte 255 gives NaN.  out is aligned to its element. */
MXFP8_API int mxfp4_dequantize(const void* q, int64_t rows, int64_t cols, int64_t ld_q, const void* s,
                               int64_t s_bytes, void* out, int out_dtype, int64_t ld_out, mxfp8_stream_t stream);

/* out (m, n) of out_dtype (MXFP8_BF16, MXFP8_FP16 or MXFP8_F32), row stride
 * ld_out elements = A B^T for the MXFP4 matrices A (m, k) and B (n, k),
 * k % 32 == 0: products of E2M1 values scaled by both blocks' powers of two,
 * summed in f32 on the tensor cores, rounded once.  A block whose scale byte is
 * 255 makes its row of A (its row of B) give NaN in every output that it meets.
 * Padding scale bytes must not be 255 (mxfp4_quantize writes 0).  out is
 * aligned to its element; it must not overlap the operands.  k == 0 gives
 * zeros.  Any m from single tokens to long prefills; the sum's order depends on
 * the sizes and the device alone, so equal calls give equal bits.  A pipeline
 * wait that runs out (about 1 s) sets bit 32 of the device status word
 * (mxfp8_device_status). */
MXFP8_API int mxfp4_gemm(const void* a_q, int64_t m, int64_t ld_a, const void* a_s, int64_t a_s_bytes,
                         const void* b_q, int64_t n, int64_t ld_b, const void* b_s, int64_t b_s_bytes, int64_t k,
                         void* out, int out_dtype, int64_t ld_out, mxfp8_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* MXFP4_H_ */
