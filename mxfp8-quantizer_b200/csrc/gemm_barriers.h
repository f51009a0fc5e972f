// gemm_barriers.h -- the mbarriers of the MXFP4 product's pipeline, eight
// bytes each, in the order they lie in shared memory.  Plain C++, so that the
// CPU tests compile it too.
#pragma once

#ifdef __CUDACC__
#define MXFP8_HD_INLINE __host__ __device__ __forceinline__
#else
#define MXFP8_HD_INLINE inline
#endif

namespace mxfp8 {

// `stages` tiles of operands in shared memory, `acc` accumulators in tensor
// memory.  Those two kinds are used in turn, each use one phase; `drained` has
// one phase in a CTA's life: the tensor-core work of all its tiles is done, and
// tensor memory may go.  It shares no barrier with a tile: after an even number
// of uses the phase to wait for would be one that ended long ago, and a commit
// on a tile's barrier would announce a tile that is not there.
template <int STAGES, int ACC>
struct GemmBarriers {
    static constexpr int count = 2 * STAGES + 2 * ACC + 1;
    static constexpr int bytes = 8 * count;
    static MXFP8_HD_INLINE constexpr int full(int s) { return 8 * s; }
    static MXFP8_HD_INLINE constexpr int empty(int s) { return 8 * (STAGES + s); }
    static MXFP8_HD_INLINE constexpr int acc_full(int a) { return 8 * (2 * STAGES + a); }
    static MXFP8_HD_INLINE constexpr int acc_empty(int a) { return 8 * (2 * STAGES + ACC + a); }
    static MXFP8_HD_INLINE constexpr int drained() { return 8 * (2 * STAGES + 2 * ACC); }
};

}  // namespace mxfp8
