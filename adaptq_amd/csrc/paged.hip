// paged.hip -- rows written into the pages of their sequences, keys rotated on the
// way.
#include <algorithm>

#include "paged.hpp"
#include "paged_split.hpp"
#include "rotary.hpp"

namespace aq {

namespace {

constexpr int kThreads = 256;

// Page of token `at` of sequence `seq`, or -1 where the table has none for it.
__device__ __forceinline__ int page_of(const PagedSeqs &q, const PagedShape &p, int seq, int at) {
  const int col = at / p.page_size;
  if (at < 0 || col >= q.width) return -1;
  const int page = q.table[(int64_t)seq * q.stride + col];
  return page >= 0 && page < p.n_pages ? page : -1;
}

// A block takes a few tokens of all heads, a thread an item of a (token, head): two
// vectors of the key (the members of N pairs, or 2 N channels that pass through) or of
// the value, kRows of them in flight.  The rows' loads go out first; while they are
// under way the tokens' sequences, positions and pages are looked up, and the cosines
// and sines of their pairs computed, into LDS once for every head.  Bound: the rows'
// bytes, read and written once; 40,000 tokens of 8 heads of 128 in bf16 71 us, 4.6 TB/s
// (a copy of 2 GiB moves 5.0); 16 ragged prompts of fp32 rows of 80 25 us, 4.6 TB/s, 29
// without the mark on the loads that they are not used again, 44 with it on the stores.
// Half or twice the tokens a block, or blocks of 512 threads, were slower.

constexpr int kCosSin = 1024;   // pairs x tokens of a block
constexpr int kBlockTokens = 16;
constexpr int kRows = 4;

struct Shape {
  PagedShape p;
  PagedSeqs q;
  PagedAppend a;
  int first_token, tokens_per_block;
  int chunks, pass, items;  // items of a row: pairs, the rest of the key; with the value
  uint64_t head_mul;        // row / n_heads = row * head_mul >> 32, for row * n_heads < 2^32
};

template <typename T, int N>
__global__ __launch_bounds__(kThreads) void append_kernel(const Shape s) {
  typedef RowVec<T, N> Vec;
  __shared__ __align__(16) float2 s_cs[kCosSin];
  __shared__ int64_t s_row[kBlockTokens];  // row of head 0 in the pages, or -1
  __shared__ int s_pos[kBlockTokens];
  const PagedShape &p = s.p;
  const PagedSeqs &q = s.q;
  const PagedAppend &a = s.a;
  const int tid = threadIdx.x;
  const int t0 = s.first_token + blockIdx.x * s.tokens_per_block;
  const int nt = min(s.tokens_per_block, a.n_tokens - t0), n_rows = nt * p.n_heads;
  const int pairs = p.rotary.pairs;
  const int wide = min(s.items, kThreads), rows_per = kThreads / wide;  // threads of a row
  int item = tid < wide * rows_per ? tid % wide : s.items;
  int row0 = tid / wide;
  int2 at = make_int2(0, 0);  // the item's vectors; .y -1: it has one
  bool value = false;
  Vec u[kRows], v[kRows];

  const auto load = [&]() {
    if (item >= s.items) return;
    value = item >= s.chunks + s.pass;
    if (item < s.chunks) {
      at = chunk_at<N>(item, pairs, p.rotary.interleaved);
    } else {
      at.x = (value ? 0 : 2 * pairs) + 2 * N * (item - s.chunks - (value ? s.pass : 0));
      at.y = at.x + N < p.dim ? at.x + N : -1;
    }
    const char *in = static_cast<const char *>(value ? a.v : a.k);
    const int64_t nb1 = value ? a.v_nb[0] : a.k_nb[0], nb2 = value ? a.v_nb[1] : a.k_nb[1];
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
      const int row = row0 + j * rows_per;
      if (row >= n_rows) break;
      const int t = (int)((uint64_t)row * s.head_mul >> 32), head = row - t * p.n_heads;
      const T *x = reinterpret_cast<const T *>(in + (t0 + t) * nb2 + head * nb1);
      u[j] = load_rows<true, T, N>(x + at.x);
      if (at.y >= 0) v[j] = load_rows<true, T, N>(x + at.y);
    }
  };
  load();

  if (tid < nt) {
    const int t = t0 + tid;
    int seq = t, j = 0;
    if (a.offsets) {
      // the last sequence that begins at or before t
      int lo = 0, hi = q.n_seqs;
      while (hi - lo > 1) {
        const int mid = lo + (hi - lo) / 2;
        if (a.offsets[mid] <= t) lo = mid;
        else hi = mid;
      }
      seq = lo;
      j = a.offsets[lo] <= t && t < a.offsets[lo + 1] ? t - a.offsets[lo] : -1;
    }
    int64_t pos = -1;
    if (j >= 0 && q.lengths[seq] >= 0) pos = (int64_t)q.lengths[seq] + j;
    const int page = pos >= 0 && pos < kMaxTokens ? page_of(q, p, seq, (int)pos) : -1;
    s_pos[tid] = (int)pos;
    s_row[tid] = page < 0 ? -1 : (int64_t)page * p.n_heads * p.page_size + pos % p.page_size;
  }
  __syncthreads();
  if (pairs) {
    for (int i = tid; i < nt * pairs; i += kThreads) {
      const int t = i / pairs;
      s_cs[i] = rotary_cos_sin(p.rotary.steps[i - t * pairs], s_pos[t], p.rotary.amplitude);
    }
    __syncthreads();
  }

  while (item < s.items) {
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
      const int row = row0 + j * rows_per;
      if (row >= n_rows) break;
      const int t = (int)((uint64_t)row * s.head_mul >> 32), head = row - t * p.n_heads;
      const int64_t to = s_row[t];
      if (to < 0) continue;
      if (item < s.chunks)
        rotate_pairs<T, N>(u[j], v[j], s_cs + t * pairs + item * N, p.rotary.interleaved, false);
      T *out = static_cast<T *>(value ? p.v_pages : p.k_pages) +
               (to + (int64_t)head * p.page_size) * p.dim;
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

template <typename T, int N>
hipError_t append_n(const PagedShape &p, const PagedSeqs &q, const PagedAppend &a, hipStream_t s) {
  Shape g{p, q, a};
  const int pairs = p.rotary.pairs, rest = p.dim - 2 * pairs;
  g.chunks = pairs / N;
  g.pass = (rest / N + 1) / 2;
  g.items = g.chunks + g.pass + (p.dim / N + 1) / 2;
  g.head_mul = (((uint64_t)1 << 32) + p.n_heads - 1) / p.n_heads;
  // tokens of a block: enough rows to fill its threads, LDS for their cosines, and
  // no fewer than 1,024 blocks for it
  int tb = kRows * kThreads / (g.items * p.n_heads);
  tb = std::min({tb, kCosSin / std::max(pairs, 1), kBlockTokens, a.n_tokens / 1024});
  g.tokens_per_block = std::max(tb, 1);
  return launch_over_tokens(a.n_tokens, g.tokens_per_block, [&](int first, int blocks) {
    g.first_token = first;
    append_kernel<T, N><<<blocks, kThreads, 0, s>>>(g);
  });
}

template <typename T>
hipError_t append_type(const PagedShape &p, const PagedSeqs &q, const PagedAppend &a,
                       hipStream_t s) {
  // the widest vectors that the layout of the pairs and every row's address allow
  int n = 16 / (int)sizeof(T);
  size_t x = reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v);
  for (int k = 0; k < 2; ++k) x |= a.k_nb[k] | a.v_nb[k];
  const size_t bits = x / sizeof(T) | (size_t)p.rotary.pairs | (size_t)p.dim;
  while (bits % n) n /= 2;
  if (n >= 8) {
    if constexpr (sizeof(T) == 2) return append_n<T, 8>(p, q, a, s);
  }
  if (n >= 4) return append_n<T, 4>(p, q, a, s);
  if (n == 2) return append_n<T, 2>(p, q, a, s);
  return append_n<T, 1>(p, q, a, s);
}

}  // namespace

hipError_t launch_paged_append(const PagedShape &p, const PagedSeqs &q, const PagedAppend &a,
                               hipStream_t s) {
  switch (p.io) {
    case IoType::F32: return append_type<float>(p, q, a, s);
    case IoType::F16: return append_type<_Float16>(p, q, a, s);
    default: return append_type<Bf16>(p, q, a, s);
  }
}

}  // namespace aq
