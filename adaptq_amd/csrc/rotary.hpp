// rotary.hpp -- rotary positions: the angle of a position and the rotation of
// vectors of row values, shared by the rotary kernel and the paged cache's.
//
// Pair i of a row at position p turns by p * f_i radians.  A pair's step is held
// as a 64-bit fraction of a turn, round(f_i / 2 pi * 2^64), so p * step mod 2^64 is
// the angle with whole turns dropped, with an error of p * 2^-65 turns (2^-34 at
// the largest position) where p * f_i in fp32 would be off by 2^-24 of the whole
// angle.  The top two bits (after adding an eighth of a turn) are the quadrant and
// the rest is within an eighth of a turn of 0: the only rounding before the sine
// is of that rest to fp32.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "launch.hpp"

namespace aq {

__device__ __forceinline__ float2 rotary_cos_sin(uint64_t step, int position, float amplitude) {
  const uint64_t phase = step * (uint64_t)(int64_t)position;
  const uint32_t quadrant = (uint32_t)((phase + (1ull << 61)) >> 62);
  const int64_t rest = (int64_t)(phase - ((uint64_t)quadrant << 62));  // of 2^64 a turn
  float s, c;
  sincospif((float)rest * 0x1p-63f, &s, &c);  // half turns
  if (quadrant & 1) {
    const float t = c;
    c = -s;
    s = t;
  }
  if (quadrant & 2) {
    c = -c;
    s = -s;
  }
  return make_float2(c * amplitude, s * amplitude);
}

// N consecutive values of a row as one load or store.
template <typename T, int N>
struct alignas(sizeof(T) * N) RowVec {
  T x[N];
};

// The same as one access; NT: marked as not used again soon.
template <int BYTES>
struct Words {
  typedef uint32_t type __attribute__((ext_vector_type(BYTES / 4)));
};
template <>
struct Words<4> {
  typedef uint32_t type;
};
template <>
struct Words<2> {
  typedef uint16_t type;
};

template <bool NT, typename T, int N>
__device__ __forceinline__ RowVec<T, N> load_rows(const T *p) {
  typedef typename Words<sizeof(T) * N>::type W;
  const W *from = reinterpret_cast<const W *>(p);
  return __builtin_bit_cast(RowVec<T, N>, NT ? __builtin_nontemporal_load(from) : *from);
}
template <bool NT, typename T, int N>
__device__ __forceinline__ void store_rows(T *p, const RowVec<T, N> &x) {
  typedef typename Words<sizeof(T) * N>::type W;
  W *to = reinterpret_cast<W *>(p);
  const W w = __builtin_bit_cast(W, x);
  if (NT) __builtin_nontemporal_store(w, to);
  else *to = w;
}

// fp16 and fp32 as their C++ types, bf16 as its bits.
struct Bf16 {
  uint16_t bits;
};

__device__ __forceinline__ float row_get(float v) { return v; }
__device__ __forceinline__ float row_get(_Float16 v) { return (float)v; }
__device__ __forceinline__ float row_get(Bf16 v) { return __uint_as_float((uint32_t)v.bits << 16); }
__device__ __forceinline__ void row_put(float &d, float v) { d = v; }
__device__ __forceinline__ void row_put(_Float16 &d, float v) { d = (_Float16)v; }
__device__ __forceinline__ void row_put(Bf16 &d, float v) {
  d.bits = __builtin_bit_cast(uint16_t, (__bf16)v);  // to nearest even, NaN stays NaN
}

// Where the pairs of a head lie in its first `dim` channels: pair i is (i, i + dim/2),
// or (2i, 2i + 1) when interleaved.
struct RotaryShape {
  const uint64_t *steps;  // [pairs]
  int pairs;
  bool interleaved;
  float amplitude;
};

// N pairs of one row from the two vectors that hold them.  half layout: a holds the
// first members and b the second; interleaved: a and then b hold the pairs in order.
// cs[i]: cosine and sine of pair i.  backward: the transposed rotation.
template <typename T, int N>
__device__ __forceinline__ void rotate_pairs(RowVec<T, N> &a, RowVec<T, N> &b, const float2 *cs,
                                             bool interleaved, bool backward) {
  float y[2 * N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float u, v;
    if (interleaved && N > 1) {
      u = row_get(2 * i < N ? a.x[2 * i % N] : b.x[2 * i % N]);
      v = row_get(2 * i + 1 < N ? a.x[(2 * i + 1) % N] : b.x[(2 * i + 1) % N]);
    } else {
      u = row_get(a.x[i]);
      v = row_get(b.x[i]);
    }
    const float c = cs[i].x, s = backward ? -cs[i].y : cs[i].y;
    y[i] = fmaf(u, c, -(v * s));
    y[N + i] = fmaf(v, c, u * s);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (interleaved && N > 1) {
      // a: u0 v0 u1 v1 ..., b: the later pairs
      row_put(a.x[i], y[(i & 1 ? N : 0) + i / 2]);
      row_put(b.x[i], y[(i & 1 ? N : 0) + (N + i) / 2]);
    } else {
      row_put(a.x[i], y[i]);
      row_put(b.x[i], y[N + i]);
    }
  }
}

// Offsets (in values) of the two vectors of pair chunk j of N pairs.
template <int N>
__device__ __forceinline__ int2 chunk_at(int j, int pairs, bool interleaved) {
  return interleaved ? make_int2(2 * N * j, 2 * N * j + N) : make_int2(N * j, pairs + N * j);
}

}  // namespace aq
