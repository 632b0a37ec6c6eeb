// rotary.hip -- rotary positions on queries and keys, forward and transposed.
//
// y1 = a (x1 cos - x2 sin), y2 = a (x2 cos + x1 sin) for each pair (x1, x2) of a
// row, by the angle of its token's position; the channels behind the pairs pass
// through.  The gradient is the same with -sin.
//
// A block takes a few tokens: cosines and sines of their pairs go to LDS once and
// serve every head of every tensor.  A thread takes a chunk of N pairs (two vector
// loads, two stores), kRows rows in flight.
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

template <typename T, int N>
__global__ __launch_bounds__(kThreads) void rotary_kernel(
    RotaryShape sh, RowsArg a, RowsArg b, const int *__restrict__ positions, int64_t pos_stride,
    int n_tokens, int total, int tokens_per_block, int items, bool backward) {
  __shared__ float2 s_cs[kCosSin];
  const int tid = threadIdx.x;
  const int t0 = blockIdx.x * tokens_per_block;
  const int nt = min(tokens_per_block, total - t0);
  for (int i = tid; i < nt * sh.pairs; i += kThreads) {
    const int t = t0 + i / sh.pairs;
    const int batch = t / n_tokens;
    s_cs[i] = rotary_cos_sin(sh.steps[i % sh.pairs],
                             positions[batch * pos_stride + (t - batch * n_tokens)], sh.amplitude);
  }
  __syncthreads();

  const int chunks = sh.pairs / N;
  const int heads = a.heads + b.heads;
  const int wide = min(items, kThreads);  // threads that share a row
  const int rows_per = kThreads / wide;
  if (tid >= wide * rows_per) return;
  const int n_rows = nt * heads;
  for (int item = tid % wide; item < items; item += wide) {
    const bool pass = item >= chunks;
    const int2 at = pass ? make_int2(2 * sh.pairs + (item - chunks) * N, 0)
                         : chunk_at<N>(item, sh.pairs, sh.interleaved);
    for (int r0 = tid / wide; r0 < n_rows; r0 += kRows * rows_per) {
      RowVec<T, N> u[kRows], v[kRows];
      T *out[kRows];
#pragma unroll
      for (int j = 0; j < kRows; ++j) {
        const int row = r0 + j * rows_per;
        if (row >= n_rows) break;
        const int t = t0 + row / heads, batch = t / n_tokens;
        const int head = row % heads;
        const RowsArg &x = head < a.heads ? a : b;
        const int64_t h = head < a.heads ? head : head - a.heads;
        const T *in = reinterpret_cast<const T *>(x.in + h * x.in_nb1 +
                                                  (t - batch * n_tokens) * x.in_nb2 +
                                                  batch * x.in_nb3);
        out[j] = reinterpret_cast<T *>(x.out + h * x.out_nb1 + (t - batch * n_tokens) * x.out_nb2 +
                                       batch * x.out_nb3);
        u[j] = *reinterpret_cast<const RowVec<T, N> *>(in + at.x);
        if (!pass) v[j] = *reinterpret_cast<const RowVec<T, N> *>(in + at.y);
      }
#pragma unroll
      for (int j = 0; j < kRows; ++j) {
        const int row = r0 + j * rows_per;
        if (row >= n_rows) break;
        if (!pass) {
          rotate_pairs<T, N>(u[j], v[j], s_cs + (row / heads) * sh.pairs + item * N,
                             sh.interleaved, backward);
          *reinterpret_cast<RowVec<T, N> *>(out[j] + at.y) = v[j];
        }
        *reinterpret_cast<RowVec<T, N> *>(out[j] + at.x) = u[j];
      }
    }
  }
}

RowsArg rows_arg(const RotaryRows &r) {
  return {static_cast<const char *>(r.in), static_cast<char *>(r.out), (int64_t)r.in_nb[0],
          (int64_t)r.in_nb[1], (int64_t)r.in_nb[2], (int64_t)r.out_nb[0], (int64_t)r.out_nb[1],
          (int64_t)r.out_nb[2], r.n_heads};
}

template <typename T, int N>
hipError_t launch(const RotaryShape &sh, const RotaryCall &c, int items, hipStream_t s) {
  RowsArg a = rows_arg(c.rows[0]), b{};
  if (c.n_rows > 1) b = rows_arg(c.rows[1]);
  const int total = c.n_batch * c.n_tokens;
  // tokens of a block: enough rows to fill its threads, LDS for their cosines, and
  // no fewer than 1,024 blocks for it
  int tb = kRows * kThreads / (items * (a.heads + b.heads));
  tb = std::min({tb, kCosSin / std::max(sh.pairs, 1), total / 1024});
  tb = std::max(tb, 1);
  rotary_kernel<T, N><<<(total + tb - 1) / tb, kThreads, 0, s>>>(
      sh, a, b, c.positions, (int64_t)c.pos_stride, c.n_tokens, total, tb, items, c.backward);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_type(const RotaryShape &sh, const RotaryCall &c, hipStream_t s) {
  // the widest vectors that the layout of the pairs and every row's address allow
  int n = 16 / (int)sizeof(T);
  size_t bits = (size_t)sh.pairs | (size_t)(c.dim - 2 * sh.pairs);
  bool in_place = true;
  for (int i = 0; i < c.n_rows; ++i) {
    const RotaryRows &r = c.rows[i];
    size_t x = reinterpret_cast<uintptr_t>(r.in) | reinterpret_cast<uintptr_t>(r.out);
    for (int k = 0; k < 3; ++k) x |= r.in_nb[k] | r.out_nb[k];
    bits |= x / sizeof(T);
    in_place = in_place && r.in == r.out;
  }
  while (bits % n) n /= 2;
  const int items = sh.pairs / n + (in_place ? 0 : (c.dim - 2 * sh.pairs) / n);
  if (n >= 8) {
    if constexpr (sizeof(T) == 2) return launch<T, 8>(sh, c, items, s);
  }
  if (n >= 4) return launch<T, 4>(sh, c, items, s);
  if (n == 2) return launch<T, 2>(sh, c, items, s);
  return launch<T, 1>(sh, c, items, s);
}

}  // namespace

hipError_t launch_rotary(const RotaryTable &t, const RotaryCall &c, hipStream_t s) {
  const RotaryShape sh{t.steps, t.pairs, t.interleaved, t.amplitude};
  switch (c.io) {
    case IoType::F32: return launch_type<float>(sh, c, s);
    case IoType::F16: return launch_type<_Float16>(sh, c, s);
    default: return launch_type<Bf16>(sh, c, s);
  }
}

}  // namespace aq
