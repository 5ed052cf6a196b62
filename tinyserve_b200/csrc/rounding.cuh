// Quotients rounded to 32 bits, as a division gives them, two at a time and without one.
#pragma once

#include "pairs.cuh"

// y / scale from inverse = 1 / scale, itself rounded correctly, and scale > 1e-30: the product is off by less than two units of its last place;
// what a quotient lacks, y - quotient * scale, is exact in one fused operation, and adding its product with the inverse leaves half a unit
// and 2^-23 of one, the second time the correctly rounded quotient (P. Markstein, 1990).  A quotient next to a half, of which bfloat16
// numbers over their largest have many, is then on the side where a division puts it.
__device__ __forceinline__ F2 f2_quotient(F2 y, F2 minus_scale, F2 inverse) {
  F2 q = f2_mul(y, inverse);
  q = f2_fma(f2_fma(q, minus_scale, y), inverse, q);
  return f2_fma(f2_fma(q, minus_scale, y), inverse, q);
}
