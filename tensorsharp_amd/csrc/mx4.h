// Values in four bits as a cache holds them: blocks of 32, a code of sign, two bits of exponent and one of mantissa each, and a power of two for
// the block (a byte e: 2^(e - 127), 255: NaN).
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

namespace tship {

// e of a block by the bits of its largest magnitude (of integers: a NaN is the largest of all): the least power of at least 2^-126 with top <= 7 * 2^(e - 127),
// 255 from 2^127 on.  (7 rounds to 6 as 5 to 4 does: one power less would cut values off, one more lose half a step of all others.)
__device__ __forceinline__ uint32_t mx4_scale(uint32_t top)
{
    if (top >= 0x7f000000u) return 255;
    const int e = (int)(top >> 23) - 2 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
    return e < 1 ? 1u : (uint32_t)e;
}
// as a number; 2^-127 and NaN included
__device__ __forceinline__ float mx4_power(uint32_t e) { return __uint_as_float(e == 0 ? 0x00400000u : e == 255 ? 0x7fc00000u : e << 23); }

// Eight values as codes, the first in the lowest bits: the instruction divides by the scale's power, rounds to nearest even and saturates.
__device__ __forceinline__ uint32_t mx4_codes(const float (&x)[8], uint32_t e)
{
    const float scale = __uint_as_float(e == 255 ? 127u << 23 : e << 23);
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[0], x[1], scale, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[2], x[3], scale, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[4], x[5], scale, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[6], x[7], scale, 3);
    return c;
}
// and back
__device__ __forceinline__ void mx4_values(uint32_t c, uint32_t e, float (&x)[8])
{
    typedef float two_t __attribute__((ext_vector_type(2)));
    const float by = mx4_power(e);
    const two_t a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 1);
    const two_t d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 2), f = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 3);
    x[0] = a.x * by, x[1] = a.y * by, x[2] = b.x * by, x[3] = b.y * by;
    x[4] = d.x * by, x[5] = d.y * by, x[6] = f.x * by, x[7] = f.y * by;
}
// the largest magnitude's bits over eight values of each of four lanes that hold a block
__device__ __forceinline__ uint32_t mx4_top(const float (&x)[8])
{
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
    top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xb1, 0xf, 0xf, true));        // lane ^ 1
    return max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4e, 0xf, 0xf, true));       // lane ^ 2
}

}  // namespace tship
