// The integer rint(127 x / top) as the low byte of a float, and four such bytes as one word.
#pragma once

#include "nq_common.h"

namespace nq {

// t = 127 x is exact for an x of up to 16 significant bits (a bf16 value, or a product of two), q = t / top follows from
// t * (1 / top) by one correction, which gives the correctly rounded quotient (checked for all pairs of such x and top);
// a true quotient that is no tie is further from every tie than that rounding moves it: of x = a 2^i and top = b 2^j it
// differs from (2n + 1) / 2 by at least 1 / (254 a) > 2^-24 of itself for a <= 255 * 255.  Adding 1.5 * 2^23 rounds it to
// an integer, ties to even.  A fifth of the instructions of a division and a conversion.
__device__ __forceinline__ uint32_t code_bits(float x, float top, float inv) {
    const float t = x * 127.0f;
    const float q = t * inv;
    return __float_as_uint(fmaf(fmaf(-q, top, t), inv, q) + 12582912.0f);
}
__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0c0c0400u), __builtin_amdgcn_perm(b, a, 0x0c0c0400u),
                                 0x05040100u);
}

}  // namespace nq
