// paged.hip -- rows written into the pages of their sequences, keys rotated on the
// way.
#include <limits.h>

#include "paged.hpp"
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

// A block takes a few tokens; their sequence, position and page, and the cosines
// and sines of their pairs, go to LDS once for every head.  A thread takes one item
// of a (token, head): a chunk of N pairs of the key, N channels of it that pass
// through, or N channels of the value.

constexpr int kCosSin = 1024;
constexpr int kMaxTokens = 16;  // of a block

template <typename T, int N>
__global__ __launch_bounds__(kThreads) void append_kernel(PagedShape p, PagedSeqs q, PagedAppend a,
                                                          int tokens_per_block) {
  __shared__ float2 s_cs[kCosSin];
  __shared__ int64_t s_row[kMaxTokens];  // row of head 0 in the pages, or -1
  __shared__ int s_pos[kMaxTokens];
  const int tid = threadIdx.x;
  const int t0 = blockIdx.x * tokens_per_block;
  const int nt = min(tokens_per_block, a.n_tokens - t0);
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
    int64_t at = -1;
    if (j >= 0 && seq < q.n_seqs && q.lengths[seq] >= 0) at = (int64_t)q.lengths[seq] + j;
    const int page = at >= 0 && at < INT_MAX ? page_of(q, p, seq, (int)at) : -1;
    s_pos[tid] = (int)at;
    s_row[tid] = page < 0 ? -1 : (int64_t)page * p.n_heads * p.page_size + at % p.page_size;
  }
  __syncthreads();
  const int pairs = p.rotary.pairs;
  for (int i = tid; i < nt * pairs; i += kThreads)
    s_cs[i] = rotary_cos_sin(p.rotary.steps[i % pairs], s_pos[i / pairs], p.rotary.amplitude);
  __syncthreads();

  const int chunks = pairs / N, pass = (p.dim - 2 * pairs) / N;
  const int items = chunks + pass + p.dim / N;
  for (int i = tid; i < nt * p.n_heads * items; i += kThreads) {
    const int row = i / items, item = i % items;
    const int t = row / p.n_heads, head = row % p.n_heads;
    if (s_row[t] < 0) continue;
    const bool value = item >= chunks + pass;
    const T *in = reinterpret_cast<const T *>(
        static_cast<const char *>(value ? a.v : a.k) +
        (size_t)(t0 + t) * (value ? a.v_nb[1] : a.k_nb[1]) +
        (size_t)head * (value ? a.v_nb[0] : a.k_nb[0]));
    T *out = static_cast<T *>(value ? p.v_pages : p.k_pages) +
             (s_row[t] + (int64_t)head * p.page_size) * p.dim;
    if (item < chunks) {
      const int2 at = chunk_at<N>(item, pairs, p.rotary.interleaved);
      RowVec<T, N> u = *reinterpret_cast<const RowVec<T, N> *>(in + at.x);
      RowVec<T, N> v = *reinterpret_cast<const RowVec<T, N> *>(in + at.y);
      rotate_pairs<T, N>(u, v, s_cs + t * pairs + item * N, p.rotary.interleaved, false);
      *reinterpret_cast<RowVec<T, N> *>(out + at.x) = u;
      *reinterpret_cast<RowVec<T, N> *>(out + at.y) = v;
    } else {
      const int at = value ? (item - chunks - pass) * N : 2 * pairs + (item - chunks) * N;
      *reinterpret_cast<RowVec<T, N> *>(out + at) = *reinterpret_cast<const RowVec<T, N> *>(in + at);
    }
  }
}

template <typename T, int N>
hipError_t append_n(const PagedShape &p, const PagedSeqs &q, const PagedAppend &a, hipStream_t s) {
  const int items = (2 * p.dim - p.rotary.pairs) / N * p.n_heads;
  int tb = 4 * kThreads / items;
  tb = std::min({tb, kCosSin / std::max(p.rotary.pairs, 1), kMaxTokens, a.n_tokens / 1024});
  tb = std::max(tb, 1);
  append_kernel<T, N><<<(a.n_tokens + tb - 1) / tb, kThreads, 0, s>>>(p, q, a, tb);
  return hipGetLastError();
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
