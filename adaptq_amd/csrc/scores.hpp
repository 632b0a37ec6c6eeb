// scores.hpp -- what the attention kernels do to a score between its product and the
// softmax: a cap by tanh, and a bias by distance.
#pragma once

#include <hip/hip_runtime.h>

namespace aq {

constexpr float kLog2e = 1.44269504088896340736f;

// tanh: with u = exp(-2|z|), (1 - u) / (1 + u).  1 - u keeps 2^-24 of 1, so below 0.6 of z
// the error would grow against the value: EXACT takes z times a polynomial of z^2 there
// (fitted at Chebyshev points, 2^-26 of the value), 2^-22 of the value above.  Without EXACT
// the error is 2^-23 of the cap everywhere, a thousandth of what scores of half-precision
// rows and weights are rounded by.
template <bool EXACT>
__device__ __forceinline__ float tanh_of(float z) {
  const float u = __builtin_amdgcn_exp2f(fabsf(z) * (-2.0f * kLog2e));
  float y;
  if constexpr (EXACT) {
    y = copysignf((1.0f - u) / (1.0f + u), z);
    const float z2 = z * z;
    float c = -0.0062691197f;
    c = fmaf(c, z2, 0.02111096f);
    c = fmaf(c, z2, -0.05387395f);
    c = fmaf(c, z2, 0.13332915f);
    c = fmaf(c, z2, -0.3333333f);
    y = fabsf(z) < 0.6f ? fmaf(z * z2, c, z) : y;
  } else {
    y = copysignf((1.0f - u) * __builtin_amdgcn_rcpf(1.0f + u), z);
  }
  return y;
}

}  // namespace aq
