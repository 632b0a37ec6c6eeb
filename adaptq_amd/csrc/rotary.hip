// rotary.hip -- rotary positions on queries and keys, forward and transposed.
//
// y1 = a (x1 cos - x2 sin), y2 = a (x2 cos + x1 sin) for each pair (x1, x2) of a
// row, by the angle of its token's position; the channels behind the pairs pass
// through.  The gradient is the same with -sin.
//
// Bound: the rows' bytes, read and written once.  A block takes a few tokens of all
// heads of both tensors; a thread takes an item of a row, two vectors of up to 16
// bytes (the two members of N pairs, or 2 N channels that pass through), and has
// kRows of them in flight.  The loads go out first; while they are under way the
// tokens' cosines and sines are computed into LDS, once for every head.  8,192 tokens
// of 32 + 8 heads of 128 in bf16: 35.2 us, 4.8 TB/s read and written (a copy of 2 GiB
// moves 5.0), 29.6 where the last cache still holds some of the 168 MB; compared there: 33
// with two rows in flight, 31 to 33 with streaming loads or stores, 41 with the loads
// behind the cosines.
#include <algorithm>

#include "paged.hpp"
#include "rotary.hpp"

namespace aq {

namespace {

constexpr int kThreads = 256;
constexpr int kCosSin = 1024;  // pairs x tokens of a block
constexpr int kRows = 4;

struct RowsArg {
  const char *in;
  char *out;
  int64_t in_nb1, in_nb2, in_nb3, out_nb1, out_nb2, out_nb3;
  int heads;
};

struct Shape {
  RotaryShape r;
  RowsArg a, b;
  const int *positions;
  int64_t pos_stride;
  int n_batch, n_tokens, total, first_token, tokens_per_block;
  int items, pass_vecs;  // items of a row; vectors of it that pass through
  uint64_t head_mul;     // row / heads = row * head_mul >> 32, for row * heads < 2^32
  bool backward;
};

// Cosines and sines of a token's pairs in LDS: two pairs (16 bytes) of each chunk of N side
// by side for all its chunks, then the next two, so that threads of neighbouring chunks read
// neighbouring words: 29.6 us instead of 30.5 with a chunk's pairs in a row (rows in the last
// cache).  (The append keeps them in a row: it gains nothing, and prompts over 4 heads lose
// 5 %.)
template <int N>
__device__ __forceinline__ int cos_sin_at(int pair, int chunks) {
  if (N == 1) return pair;
  const int j = pair % N;
  return (j / 2 * chunks + pair / N) * 2 + j % 2;
}
template <int N>
__device__ __forceinline__ void get_cos_sin(const float2 *of_token, int chunk, int chunks,
                                            float2 (&cs)[N]) {
  if constexpr (N == 1) {
    cs[0] = of_token[chunk];
  } else {
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      const float4 x =
          *reinterpret_cast<const float4 *>(of_token + (j / 2 * chunks + chunk) * 2);
      cs[j] = make_float2(x.x, x.y);
      cs[j + 1] = make_float2(x.z, x.w);
    }
  }
}

template <typename T, int N>
__global__ __launch_bounds__(kThreads) void rotary_kernel(const Shape s) {
  typedef RowVec<T, N> Vec;
  __shared__ __align__(16) float2 s_cs[kCosSin];
  const int tid = threadIdx.x;
  const int t0 = s.first_token + blockIdx.x * s.tokens_per_block;
  const int nt = min(s.tokens_per_block, s.total - t0);
  const int chunks = s.r.pairs / N, heads = s.a.heads + s.b.heads, n_rows = nt * heads;
  const int wide = min(s.items, kThreads), rows_per = kThreads / wide;  // threads of a row
  const bool active = tid < wide * rows_per;
  int item = active ? tid % wide : s.items;
  int row0 = tid / wide;
  int2 at = make_int2(0, 0);  // the item's vectors; .y -1: it has one
  Vec u[kRows], v[kRows];

  const auto place = [&](int row, bool out) {
    const int j = (int)((uint64_t)row * s.head_mul >> 32), head = row - j * heads;
    const int t = t0 + j, batch = s.n_batch > 1 ? t / s.n_tokens : 0;
    const bool first = head < s.a.heads;
    const int64_t h = first ? head : head - s.a.heads, tok = t - batch * s.n_tokens;
    const RowsArg &x = first ? s.a : s.b;
    return out ? x.out + h * x.out_nb1 + tok * x.out_nb2 + batch * x.out_nb3
               : const_cast<char *>(x.in) + h * x.in_nb1 + tok * x.in_nb2 + batch * x.in_nb3;
  };
  const auto load = [&]() {
    if (item >= s.items) return;
    if (item < chunks) {
      at = chunk_at<N>(item, s.r.pairs, s.r.interleaved);
    } else {
      const int i = 2 * (item - chunks);
      at.x = 2 * s.r.pairs + i * N;
      at.y = i + 1 < s.pass_vecs ? at.x + N : -1;
    }
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
      const int row = row0 + j * rows_per;
      if (row >= n_rows) break;
      const T *in = reinterpret_cast<const T *>(place(row, false));
      u[j] = load_rows<false, T, N>(in + at.x);
      if (at.y >= 0) v[j] = load_rows<false, T, N>(in + at.y);
    }
  };
  load();

  for (int i = tid; i < nt * s.r.pairs; i += kThreads) {
    const int j = i / s.r.pairs, t = t0 + j, batch = s.n_batch > 1 ? t / s.n_tokens : 0;
    const int pair = i - j * s.r.pairs;
    s_cs[j * s.r.pairs + cos_sin_at<N>(pair, chunks)] =
        rotary_cos_sin(s.r.steps[pair],
                       s.positions[batch * s.pos_stride + (t - batch * s.n_tokens)],
                       s.r.amplitude);
  }
  __syncthreads();

  while (item < s.items) {
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
      const int row = row0 + j * rows_per;
      if (row >= n_rows) break;
      if (item < chunks) {
        const int tok = (int)((uint64_t)row * s.head_mul >> 32);
        float2 cs[N];
        get_cos_sin<N>(s_cs + tok * s.r.pairs, item, chunks, cs);
        rotate_pairs<T, N>(u[j], v[j], cs, s.r.interleaved, s.backward);
      }
      T *out = reinterpret_cast<T *>(place(row, true));
      store_rows<false>(out + at.x, u[j]);
      if (at.y >= 0) store_rows<false>(out + at.y, v[j]);
    }
    row0 += kRows * rows_per;
    if (row0 >= n_rows) {
      row0 = tid / wide;
      item += wide;
    }
    load();
  }
}

RowsArg rows_arg(const RotaryRows &r) {
  return {static_cast<const char *>(r.in), static_cast<char *>(r.out), (int64_t)r.in_nb[0],
          (int64_t)r.in_nb[1], (int64_t)r.in_nb[2], (int64_t)r.out_nb[0], (int64_t)r.out_nb[1],
          (int64_t)r.out_nb[2], r.n_heads};
}

template <typename T, int N>
hipError_t launch(Shape g, int dim, bool in_place, hipStream_t s) {
  g.pass_vecs = in_place ? 0 : (dim - 2 * g.r.pairs) / N;
  g.items = g.r.pairs / N + (g.pass_vecs + 1) / 2;
  const int heads = g.a.heads + g.b.heads;
  g.head_mul = (((uint64_t)1 << 32) + heads - 1) / heads;
  // tokens of a block: enough rows to fill its threads, LDS for their cosines, and
  // no fewer than 1,024 blocks for it
  int tb = kRows * kThreads / (g.items * heads);
  tb = std::min({tb, kCosSin / std::max(g.r.pairs, 1), g.total / 1024});
  g.tokens_per_block = std::max(tb, 1);
  return launch_over_tokens(g.total, g.tokens_per_block, [&](int first, int blocks) {
    g.first_token = first;
    rotary_kernel<T, N><<<blocks, kThreads, 0, s>>>(g);
  });
}

template <typename T>
hipError_t launch_type(const RotaryTable &t, const RotaryCall &c, hipStream_t s) {
  Shape g{};
  g.r = {t.steps, t.pairs, t.interleaved, t.amplitude};
  g.a = rows_arg(c.rows[0]);
  if (c.n_rows > 1) g.b = rows_arg(c.rows[1]);
  g.positions = c.positions;
  g.pos_stride = (int64_t)c.pos_stride;
  g.n_batch = c.n_batch;
  g.n_tokens = c.n_tokens;
  g.total = c.n_batch * c.n_tokens;
  g.backward = c.backward;
  // the widest vectors that the layout of the pairs and every row's address allow
  int n = 16 / (int)sizeof(T);
  size_t bits = (size_t)t.pairs | (size_t)(c.dim - 2 * t.pairs);
  bool in_place = true;
  for (int i = 0; i < c.n_rows; ++i) {
    const RotaryRows &r = c.rows[i];
    size_t x = reinterpret_cast<uintptr_t>(r.in) | reinterpret_cast<uintptr_t>(r.out);
    for (int k = 0; k < 3; ++k) x |= r.in_nb[k] | r.out_nb[k];
    bits |= x / sizeof(T);
    in_place = in_place && r.in == r.out;
  }
  while (bits % n) n /= 2;
  if (n >= 8) {
    if constexpr (sizeof(T) == 2) return launch<T, 8>(g, c.dim, in_place, s);
  }
  if (n >= 4) return launch<T, 4>(g, c.dim, in_place, s);
  if (n == 2) return launch<T, 2>(g, c.dim, in_place, s);
  return launch<T, 1>(g, c.dim, in_place, s);
}

}  // namespace

hipError_t launch_rotary(const RotaryTable &t, const RotaryCall &c, hipStream_t s) {
  switch (c.io) {
    case IoType::F32: return launch_type<float>(t, c, s);
    case IoType::F16: return launch_type<_Float16>(t, c, s);
    default: return launch_type<Bf16>(t, c, s);
  }
}

}  // namespace aq
