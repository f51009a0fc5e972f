// capi_mxfp4.cu -- the extern "C" boundary declared in include/mxfp4.h:
// argument validation, then the launches of mxfp4_convert.cu and
// mxfp4_gemm.cu.
#include <cuda_runtime.h>

#include "../../include/mxfp4.h"
#include "launch.h"

using namespace mxfp8;

namespace {

constexpr int64_t kInt32Max = 2147483647;
constexpr int64_t kMaxStride = int64_t(1) << 38;

inline bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int out_bytes(int dtype) { return dtype == MXFP8_F32 ? 4 : 2; }
inline bool is_out_dtype(int dtype) { return dtype == MXFP8_BF16 || dtype == MXFP8_FP16 || dtype == MXFP8_F32; }

// One MXFP4 operand: payload, scales and their strides.
int check_fp4(const void* q, int64_t rows, int64_t cols, int64_t ld_q, const void* s, int64_t s_bytes) {
    if (!q || !s) return MXFP8_ERR_NULL_POINTER;
    if (!aligned(q, 16) || !aligned(s, 16) || ld_q % 16 != 0) return MXFP8_ERR_ALIGNMENT;
    if (s_bytes < mxfp8_scale_storage_bytes(rows, cols)) return MXFP8_ERR_SCALE_BUFFER;
    return MXFP8_OK;
}

}  // namespace

extern "C" MXFP8_API int mxfp4_quantize(const void* x, int dtype, int64_t m, int64_t k, int64_t ld_x, void* q,
                                        int64_t ld_q, void* s, int64_t s_bytes, mxfp8_stream_t stream) {
    if (dtype != MXFP8_BF16 && dtype != MXFP8_FP16) return MXFP8_ERR_DTYPE;
    if (m < 0 || k < 0 || m > kInt32Max || k > kInt32Max - 31 || ld_x < k || ld_x > kMaxStride)
        return MXFP8_ERR_SHAPE;
    const int64_t q_cols = ceil_div(k, 32) * 32;
    if (ld_q < q_cols / 2 || ld_q > kMaxStride) return MXFP8_ERR_SHAPE;
    if (m == 0 || k == 0) return MXFP8_OK;
    if (!x) return MXFP8_ERR_NULL_POINTER;
    if (!aligned(x, 2)) return MXFP8_ERR_ALIGNMENT;
    if (int rc = check_fp4(q, m, q_cols, ld_q, s, s_bytes)) return rc;
    Fp4QuantizeArgs a;
    int sms = 0;
    if (int rc = ready_device(&sms, &a.status)) return rc;
    a.x = x;
    a.dtype = dtype;
    a.m = m;
    a.k = k;
    a.ld_x = ld_x;
    a.q = static_cast<uint8_t*>(q);
    a.q_cols = q_cols;
    a.ld_q = ld_q;
    a.s = static_cast<uint8_t*>(s);
    a.qw = make_window(q, (m - 1) * ld_q + q_cols / 2);
    a.sw = make_window(s, mxfp8_scale_storage_bytes(m, q_cols));
    return launch_mxfp4_quantize(a, static_cast<cudaStream_t>(stream));
}

extern "C" MXFP8_API int mxfp4_dequantize(const void* q, int64_t rows, int64_t cols, int64_t ld_q, const void* s,
                                          int64_t s_bytes, void* out, int out_dtype, int64_t ld_out,
                                          mxfp8_stream_t stream) {
    if (!is_out_dtype(out_dtype)) return MXFP8_ERR_DTYPE;
    if (rows < 0 || cols < 0 || cols % 32 != 0 || rows > kInt32Max || cols > kInt32Max || ld_q < cols / 2 ||
        ld_q > kMaxStride || ld_out < cols || ld_out > kMaxStride)
        return MXFP8_ERR_SHAPE;
    if (rows == 0 || cols == 0) return MXFP8_OK;
    if (!out) return MXFP8_ERR_NULL_POINTER;
    if (int rc = check_fp4(q, rows, cols, ld_q, s, s_bytes)) return rc;
    if (!aligned(out, out_bytes(out_dtype))) return MXFP8_ERR_ALIGNMENT;
    int sms = 0;
    unsigned int* status = nullptr;
    if (int rc = ready_device(&sms, &status)) return rc;
    const StoreWindow ow = make_window(out, ((rows - 1) * ld_out + cols) * out_bytes(out_dtype));
    return launch_mxfp4_dequantize(static_cast<const uint8_t*>(q), rows, cols, ld_q, static_cast<const uint8_t*>(s),
                                   out, out_dtype, ld_out, ow, status, static_cast<cudaStream_t>(stream));
}

extern "C" MXFP8_API int mxfp4_gemm(const void* a_q, int64_t m, int64_t ld_a, const void* a_s, int64_t a_s_bytes,
                                    const void* b_q, int64_t n, int64_t ld_b, const void* b_s, int64_t b_s_bytes,
                                    int64_t k, void* out, int out_dtype, int64_t ld_out, mxfp8_stream_t stream) {
    if (!is_out_dtype(out_dtype)) return MXFP8_ERR_DTYPE;
    if (m < 0 || n < 0 || k < 0 || k % 32 != 0 || m > kInt32Max || n > kInt32Max || k > kInt32Max - 255 ||
        ld_a < k / 2 || ld_b < k / 2 || ld_a > kMaxStride || ld_b > kMaxStride || ld_out < n || ld_out > kMaxStride)
        return MXFP8_ERR_SHAPE;
    if (m == 0 || n == 0) return MXFP8_OK;
    if (!out) return MXFP8_ERR_NULL_POINTER;
    const int es = out_bytes(out_dtype);
    if (!aligned(out, es)) return MXFP8_ERR_ALIGNMENT;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (k == 0) {
        const cudaError_t e = cudaMemset2DAsync(out, (size_t)(ld_out * es), 0, (size_t)(n * es), (size_t)m, st);
        if (e == cudaSuccess) return MXFP8_OK;
        set_last_error("cudaMemset2DAsync", (int)e);
        return MXFP8_ERR_CUDA;
    }
    if (int rc = check_fp4(a_q, m, k, ld_a, a_s, a_s_bytes)) return rc;
    if (int rc = check_fp4(b_q, n, k, ld_b, b_s, b_s_bytes)) return rc;
    Fp4GemmArgs g;
    int sms = 0;
    if (int rc = ready_device(&sms, &g.status)) return rc;
    g.a = Fp4Operand{static_cast<const uint8_t*>(a_q), static_cast<const uint8_t*>(a_s), m, ld_a};
    g.b = Fp4Operand{static_cast<const uint8_t*>(b_q), static_cast<const uint8_t*>(b_s), n, ld_b};
    g.k = k;
    g.out = out;
    g.out_dtype = out_dtype;
    g.ld_out = ld_out;
    g.ow = make_window(out, ((m - 1) * ld_out + n) * es);
    return launch_mxfp4_gemm(g, sms, st);
}
