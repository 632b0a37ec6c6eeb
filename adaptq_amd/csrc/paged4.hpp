// paged4.hpp -- pages of 4-bit values: the codes, and where a token's lie.
//
// 32 consecutive channels of a row share a power of two, 2^e the smallest that takes their
// largest magnitude to 6 or below (-125 <= e <= 125; beyond, values saturate at 6 * 2^125),
// held as the byte e + 127, or 255 where one of them is infinite or NaN: the 32 read as NaN.
// A value is the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 times 2^e with its sign, of two equally
// near the one with the even code: the format that the card's conversions take (one
// instruction a pair of values and its scale), and exact, as powers of two round nothing.
//
// A (page, head) holds blocks of 16 tokens, each 8 * dim bytes of codes and then 16 * dim / 32
// of scales, so that what a wave reads together lies together:
//   keys    [16 tokens][dim / 2] codes, [16 tokens][dim / 32] scales
//   values  [4 groups of 4 tokens][dim / C][4 tokens][C / 2] codes, C channels of a lane,
//           [4 groups][dim / 32][4 tokens] scales
// A byte holds two neighbouring channels, the first in its low half.
#pragma once

#include "io.hpp"
#include "paged.hpp"
#include "rotary.hpp"

namespace aq {

constexpr int kBlock4 = 32;  // channels that share a scale

__host__ __device__ __forceinline__ int block4_bytes(int dim) { return 17 * dim / 2; }
// Channels of a lane: C above.
__host__ __device__ __forceinline__ int value_channels4(int dim) { return dim <= 64 ? 4 : 8; }

// Byte 16 tokens' blocks of a page's head begin at.
__device__ __forceinline__ int64_t block4_at(const PagedShape &p, int page, int head, int slot) {
  return ((int64_t)page * p.n_heads + head) * (p.page_size / 16) * block4_bytes(p.dim) +
         (int64_t)(slot / 16) * block4_bytes(p.dim);
}

// A byte as the scale of the card's conversions: they take its exponent field alone (so what
// lies above and below may be anything), 255 as NaN.
__device__ __forceinline__ float scale4(uint32_t byte) { return __uint_as_float(byte << 23); }

// The scale's byte for the largest magnitude's bits.
__device__ __forceinline__ int scale4_of(uint32_t top) {
  if (top >= 0x7F800000u) return 255;
  const int e = (int)(top >> 23) - ((top & 0x7FFFFFu) > 0x400000u ? 1 : 2);  // + 127
  return min(max(e, 2), 252);
}

// 8 channels of a row, from channel 8 * chunk on, by a lane of four that hold its 32: their codes,
// and the byte of the scale.  All four lanes take part.
__device__ __forceinline__ uint32_t encode4(const float (&x)[8], int *byte) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
  top = max(top, (uint32_t)__shfl_xor((int)top, 1, 64));
  top = max(top, (uint32_t)__shfl_xor((int)top, 2, 64));
  *byte = scale4_of(top);
  const float scale = scale4(*byte);
  uint32_t codes = 0;
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[0], x[1], scale, 0);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[2], x[3], scale, 1);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[4], x[5], scale, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[6], x[7], scale, 3);
}

// Writes them at a token's place: `at` its block of 16, `in` its number there.
__device__ __forceinline__ void store4(char *at, int in, int chunk, uint32_t codes, int byte,
                                       bool value, int dim) {
  const int blocks = dim / kBlock4;
  char *scales = at + 8 * dim;
  if (!value) {
    *reinterpret_cast<uint32_t *>(at + in * (dim / 2) + 4 * chunk) = codes;
    if (chunk % 4 == 0) scales[in * blocks + chunk / 4] = (char)byte;
    return;
  }
  const int group = in / 4, token = in % 4;
  if (value_channels4(dim) == 8) {
    *reinterpret_cast<uint32_t *>(at + (group * (dim / 8) + chunk) * 16 + 4 * token) = codes;
  } else {
    char *to = at + (group * (dim / 4) + 2 * chunk) * 8 + 2 * token;
    *reinterpret_cast<uint16_t *>(to) = (uint16_t)codes;
    *reinterpret_cast<uint16_t *>(to + 8) = (uint16_t)(codes >> 16);
  }
  if (chunk % 4 == 0) scales[(group * blocks + chunk / 4) * 4 + token] = (char)byte;
}

// 4 channels of a token, from channel d on, and their scale's byte.
__device__ __forceinline__ uint32_t load4(const char *at, int in, int d, bool value, int dim,
                                          int *byte) {
  const int blocks = dim / kBlock4;
  const char *scales = at + 8 * dim;
  if (!value) {
    *byte = (uint8_t)scales[in * blocks + d / kBlock4];
    return *reinterpret_cast<const uint16_t *>(at + in * (dim / 2) + d / 2);
  }
  const int group = in / 4, token = in % 4;
  *byte = (uint8_t)scales[(group * blocks + d / kBlock4) * 4 + token];
  const int c = value_channels4(dim);
  return *reinterpret_cast<const uint16_t *>(at + (group * (dim / c) + d / c) * 2 * c +
                                             token * (c / 2) + d % c / 2);
}

// 8 channels of an input row, from channel 8 * chunk on: a key's rotated to its position and
// rounded to the rows' type, as Rotary's outputs are.
__device__ __forceinline__ float round_to(float x, IoType io) {
  if (io == IoType::F32) return x;
  if (io == IoType::F16) return (float)(_Float16)x;
  Bf16 b;
  row_put(b, x);
  return row_get(b);
}

// cs(pair): cosine and sine of a pair at the row's position.
template <typename CosSin>
__device__ __forceinline__ void rotate8(float (&x)[8], const void *row, int chunk, IoType io,
                                        const RotaryTable &rt, CosSin cs) {
  const int d0 = 8 * chunk;
  if (d0 >= 2 * rt.pairs) return;
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d = d0 + i;
    y[i] = x[i];
    if (d >= 2 * rt.pairs) continue;
    const bool one = rt.interleaved ? !(d & 1) : d < rt.pairs;
    const int pair = rt.interleaved ? d >> 1 : one ? d : d - rt.pairs;
    const int other = rt.interleaved ? d ^ 1 : one ? d + rt.pairs : d - rt.pairs;
    const float v = io_load(row, other, io);
    const float2 a = cs(pair);
    y[i] = round_to(one ? fmaf(x[i], a.x, -(v * a.y)) : fmaf(x[i], a.x, v * a.y), io);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = y[i];
}

}  // namespace aq
