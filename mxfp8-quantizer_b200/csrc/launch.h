// launch.h -- internal host-side launch interface between the C ABI
// (capi.cu) and the kernel translation units.
#pragma once
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "guard.cuh"

namespace mxfp8 {

// Problem description after argument validation.
struct QuantizeArgs {
    const void* x;
    int dtype;
    int64_t m, k, ld_x;
    uint8_t* q;
    int64_t q_rows, q_cols, ld_q;
    uint8_t* s;
    int64_t scale_rows;   // q_rows rounded up to 128
    int64_t scale_cols;   // q_cols / 32
    int64_t col_chunks;   // ceil(scale_cols / 4)
    unsigned int* status; // device error word (may be null)
    StoreWindow qw, sw;   // bytes the kernels may write: Q rows, S storage
};

// Returned by launchers: 0, or a negative mxfp8_status.
int launch_quantize_tma(const QuantizeArgs& a, int sm_count, cudaStream_t stream);
int launch_quantize_generic(const QuantizeArgs& a, int sm_count, cudaStream_t stream);
// Same kernel as launch_quantize_tma, scratch in a fixed device array (never allocates).
int launch_quantize_tma_noalloc(const QuantizeArgs& a, int dev, int sm_count, cudaStream_t stream);
int launch_dequantize(const uint8_t* q, int64_t rows, int64_t cols, int64_t ld_q, const uint8_t* s,
                      void* out, int out_dtype, int64_t ld_out, StoreWindow ow, unsigned int* status,
                      cudaStream_t stream);

int launch_bounded_wait_selftest(unsigned int* status, uint32_t limit_us, cudaStream_t stream);

// Problem description of an MXFP4 quantization after argument validation.
struct Fp4QuantizeArgs {
    const void* x;
    int dtype;
    int64_t m, k, ld_x;
    uint8_t* q;
    int64_t q_cols, ld_q;  // columns rounded up to 32, row stride in bytes
    uint8_t* s;
    unsigned int* status;
    StoreWindow qw, sw;
};

int launch_mxfp4_quantize(const Fp4QuantizeArgs& a, cudaStream_t stream);
int launch_mxfp4_dequantize(const uint8_t* q, int64_t rows, int64_t cols, int64_t ld_q, const uint8_t* s, void* out,
                            int out_dtype, int64_t ld_out, StoreWindow ow, unsigned int* status, cudaStream_t stream);

// One operand of the MXFP4 product: payload (rows, k / 2 bytes, row stride ld
// bytes) and packed scales.
struct Fp4Operand {
    const uint8_t* q;
    const uint8_t* s;
    int64_t rows, ld;
};

struct Fp4GemmArgs {
    Fp4Operand a, b;
    int64_t k;
    void* out;
    int out_dtype;
    int64_t ld_out;  // elements
    StoreWindow ow;
    unsigned int* status;
};

int launch_mxfp4_gemm(const Fp4GemmArgs& g, int sm_count, cudaStream_t stream);

// The driver's cuTensorMapEncodeTiled, looked up once; null if it is missing.
PFN_cuTensorMapEncodeTiled_v12000 get_encode_fn();

// SM count and device error word of the current device (made ready by the
// first call on it); 0 or a negative mxfp8_status.
int ready_device(int* sm_count, unsigned int** status);

// The bytes [base, base + bytes) a kernel may write.  The checked build
// narrows it by mxfp8_checked_window_slack bytes, to show that its store
// guards fire; the product build ignores the window.
StoreWindow make_window(void* base, int64_t bytes);

// Records the CUDA error text for mxfp8_last_error() on this host thread, and clears the runtime's own note of it.
void set_last_error(const char* what, int code);

// Key of the CUDA context current on this host thread, unique for the
// process's lifetime; 0 if none is current (context_key) or after binding the
// runtime's context to the thread first (bound_context_key, never 0 on
// success).  Per-device caches compare it to notice a new context.
int context_key(uint64_t* key);
int bound_context_key(uint64_t* key);

// A kernel's opt-in to `smem` bytes of dynamic shared memory, and with `most_shared` to the largest share of the SM's
// memory.  It belongs to a context: made by the kernel's first launch in one, so that later launches, captured ones
// among them, make no such call.  `done` is the kernel's own, static; 0 or a negative mxfp8_status.
constexpr int kMaxDevices = 64;
struct OptIn {
    std::atomic<uint64_t> ctx[kMaxDevices];  // context_key() of the context it was made in last
};
int opt_in(const void* kernel, int smem, bool most_shared, OptIn& done);

// Device address of the allocation-free entries' status word (a fixed device
// array of quantize_tma.cu) on device `dev`, the current device.
int noalloc_status_word(int dev, unsigned int** out);

}  // namespace mxfp8
