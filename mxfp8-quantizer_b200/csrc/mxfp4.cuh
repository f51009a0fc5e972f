// mxfp4.cuh -- the MXFP4 block recipe, shared by the quantizer and its
// inverse.  For a block whose largest magnitude is a > 0, the scale is 2^e
// with the smallest e >= -127 such that a <= 6 * 2^e, 6 being the largest
// E2M1 value: with a = 1.f * 2^E, that is e = E - 2 where 1.f <= 1.5 and
// E - 1 where it is above, an exact rule on the bits.  x * 2^-e is exact in
// f32 (or below a quarter of the smallest code, where it rounds to 0), so
// the conversion's rounding is the only one.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "recipe.cuh"

namespace mxfp8 {

// Bit patterns of |x| from here on are inf or NaN.
template <int DT>
constexpr uint32_t kNonFinite16 = DT == kBF16 ? 0x7F80u : 0x7C00u;

// Scale byte and inverse scale from the block's amax bit pattern.  A block
// with an inf or a NaN has byte 255, the only NaN the format has; its caller
// writes codes 0.
template <int DT>
__device__ __forceinline__ void fp4_scale_from_amax(uint32_t amax_bits, uint32_t& byte, float& inv) {
    const uint32_t b = __float_as_uint(widen<DT>(amax_bits));
    const int e = (int)(b >> 23) - 2 + ((b & 0x7FFFFFu) > 0x400000u ? 1 : 0);
    uint32_t r = (uint32_t)max(e, 0);
    r = amax_bits == 0u ? 127u : r;
    inv = __uint_as_float((254u - r) << 23);
    byte = amax_bits >= kNonFinite16<DT> ? 255u : r;
}

// Eight f32 -> eight E2M1 codes, v[0] in the lowest four bits.
__device__ __forceinline__ uint32_t cvt_e2m1x8(const float (&v)[8]) {
    uint32_t r;
    asm("{\n\t.reg .b8 t0, t1, t2, t3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 t0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 t1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 t2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 t3, %8, %7;\n\t"
        "mov.b32 %0, {t0, t1, t2, t3};\n\t}"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}

// Eight E2M1 codes -> four f16 pairs, in element order.
__device__ __forceinline__ void e2m1x8_to_half2(uint32_t codes, uint32_t (&h)[4]) {
    asm("{\n\t.reg .b8 t0, t1, t2, t3;\n\t"
        "mov.b32 {t0, t1, t2, t3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, t0;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, t1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, t2;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, t3;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(codes));
}

}  // namespace mxfp8
