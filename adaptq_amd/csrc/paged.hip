// paged.hip -- a cache of exact key and value rows in pages: rows written into the
// pages of their sequences, keys rotated on the way, and the attention of one new
// token per sequence.
#include <float.h>
#include <limits.h>

#include "paged.hpp"
#include "rotary.hpp"

namespace aq {

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ RotaryShape rotary_shape(const RotaryTable &t) {
  return {t.steps, t.pairs, t.interleaved, t.amplitude};
}

// Page of token `at` of sequence `seq`, or -1 where the table has none for it.
__device__ __forceinline__ int page_of(const PagedSeqs &q, const PagedShape &p, int seq, int at) {
  const int col = at / p.page_size;
  if (at < 0 || col >= q.width) return -1;
  const int page = q.table[(int64_t)seq * q.stride + col];
  return page >= 0 && page < p.n_pages ? page : -1;
}

// ---- append ----
//
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

// ---- attention ----
//
// o = sum_t p_t v_t / sum_t p_t, p_t = exp(scale <q, k_t> - max), over the tokens
// [lo, n) of a sequence.  A block takes one (sequence, query head); its waves take
// every fourth token with a running maximum and sum each, and join in LDS.

constexpr int kMaxDim = 256;

template <typename T>
__global__ __launch_bounds__(kThreads) void attend_kernel(PagedShape p, PagedSeqs q,
                                                          PagedAttend a) {
  constexpr int E = kMaxDim / 64;
  __shared__ float s_q[kMaxDim];
  __shared__ float s_acc[4][kMaxDim], s_m[4], s_l[4];
  const int seq = blockIdx.x / a.q_heads, qh = blockIdx.x % a.q_heads;
  const int head = qh / (a.q_heads / p.n_heads);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t cap = (int64_t)q.width * p.page_size;
  const int64_t held = q.lengths[seq] < 0 ? 0 : (int64_t)q.lengths[seq] + a.extra;
  const int at_q = (int)(held - 1);  // the query's position
  const int n = (int)min(min(held, cap), (int64_t)INT_MAX);
  const int lo = a.window > 0 && n > a.window ? n - a.window : 0;
  const T *qr = reinterpret_cast<const T *>(static_cast<const char *>(a.q) +
                                            (size_t)seq * a.q_nb[1] + (size_t)qh * a.q_nb[0]);
  const RotaryTable &r = p.rotary;
  for (int i = tid; i < r.pairs; i += kThreads) {
    const float2 cs = rotary_cos_sin(r.steps[i], at_q, r.amplitude);
    const int2 at = chunk_at<1>(i, r.pairs, r.interleaved);
    const float u = row_get(qr[at.x]), v = row_get(qr[at.y]);
    s_q[at.x] = fmaf(u, cs.x, -(v * cs.y));
    s_q[at.y] = fmaf(v, cs.x, u * cs.y);
  }
  for (int i = 2 * r.pairs + tid; i < p.dim; i += kThreads) s_q[i] = row_get(qr[i]);
  __syncthreads();
  float acc[E] = {}, m = -INFINITY, l = 0.0f;
  for (int t = lo + wave; t < n; t += 4) {
    const int page = page_of(q, p, seq, t);
    if (page < 0) continue;
    const int64_t row =
        (((int64_t)page * p.n_heads + head) * p.page_size + t % p.page_size) * p.dim;
    const T *k = static_cast<const T *>(p.k_pages) + row, *v = static_cast<const T *>(p.v_pages) + row;
    float x = 0.0f;
    for (int i = lane; i < p.dim; i += 64) x = fmaf(row_get(k[i]), s_q[i], x);
#pragma unroll
    for (int k2 = 32; k2 >= 1; k2 >>= 1) x += __shfl_xor(x, k2, 64);
    x *= a.scale;
    const float top = fmaxf(fmaxf(m, x), -FLT_MAX);  // finite: a token was there
    const float keep = expf(m - top), w = expf(x - top);
    m = top;
    l = l * keep + w;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int i = lane + 64 * e;
      if (i < p.dim) acc[e] = fmaf(w, row_get(v[i]), acc[e] * keep);
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e) s_acc[wave][lane + 64 * e] = acc[e];
  if (lane == 0) {
    s_m[wave] = m;
    s_l[wave] = l;
  }
  __syncthreads();
  float top = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
  const bool none = top == -INFINITY;
  if (none) top = 0.0f;
  float w[4], sum = 0.0f;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    w[k] = expf(s_m[k] - top);
    sum += w[k] * s_l[k];
  }
  T *out = reinterpret_cast<T *>(static_cast<char *>(a.out) + (size_t)seq * a.out_nb[1] +
                                 (size_t)qh * a.out_nb[0]);
  for (int i = tid; i < p.dim; i += kThreads) {
    float y = 0.0f;
#pragma unroll
    for (int k = 0; k < 4; ++k) y = fmaf(w[k], s_acc[k][i], y);
    row_put(out[i], none ? 0.0f : y / sum);
  }
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

size_t paged_workspace_bytes(const PagedShape &) { return 0; }

hipError_t launch_paged_attend(const PagedShape &p, const PagedSeqs &q, const PagedAttend &a,
                               void *, hipStream_t s) {
  const unsigned grid = (unsigned)q.n_seqs * a.q_heads;
  switch (p.io) {
    case IoType::F32: attend_kernel<float><<<grid, kThreads, 0, s>>>(p, q, a); break;
    case IoType::F16: attend_kernel<_Float16><<<grid, kThreads, 0, s>>>(p, q, a); break;
    default: attend_kernel<Bf16><<<grid, kThreads, 0, s>>>(p, q, a); break;
  }
  return hipGetLastError();
}

}  // namespace aq
