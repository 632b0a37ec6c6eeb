// scores.hpp -- what the attention kernels do to a score between its product and the
// softmax: a cap by tanh, and a bias by distance.
#pragma once

#include <hip/hip_runtime.h>

namespace aq {

constexpr float kLog2e = 1.44269504088896340736f;

// cap * tanh(s / cap) to base 2: in is 1 / cap (of a product), cap2 the cap to base 2.  With
// u = exp(-2|z|), tanh is (1 - u) / (1 + u).  1 - u keeps 2^-24 of 1, so below 0.6 of z the error
// would grow against the value: EXACT takes z times a polynomial of z^2 there (fitted at
// Chebyshev points, 2^-26 of the value), 2^-21 of the value above (the reciprocal is within one
// step, as the exponential is).  Without EXACT the error is 2^-22 of the cap everywhere, whatever
// the score: for half-precision rows and caps up to kRoughCap alone, where it is 2^-16 of a unit,
// as much as their weights are rounded by.
constexpr float kRoughCap = 64.0f;

template <bool EXACT>
__device__ __forceinline__ float capped(float s, float in, float cap2) {
  const float z = s * in;
  const float u = __builtin_amdgcn_exp2f(fabsf(z) * (-2.0f * kLog2e));
  float y = copysignf((1.0f - u) * __builtin_amdgcn_rcpf(1.0f + u), z);
  if constexpr (EXACT) {
    const float z2 = z * z;
    float c = -0.0062691197f;
    c = fmaf(c, z2, 0.02111096f);
    c = fmaf(c, z2, -0.05387395f);
    c = fmaf(c, z2, 0.13332915f);
    c = fmaf(c, z2, -0.3333333f);
    y = fabsf(z) < 0.6f ? fmaf(z * z2, c, z) : y;
  }
  return y * cap2;
}

}  // namespace aq
