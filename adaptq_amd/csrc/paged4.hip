// paged4.hip -- rows written into pages of 4-bit values, and read back (paged4.hpp).
#include <algorithm>

#include "paged4.hpp"
#include "paged_split.hpp"

namespace aq {

namespace {

constexpr int kThreads = 256;
constexpr int kBlockTokens = 64;
constexpr int kCosSin = 2048;  // pairs x tokens of a block

struct Args {
  PagedShape p;
  PagedSeqs q;
  PagedAppend a;
  float *k_out, *v_out;  // read: [n_tokens][n_heads][dim]
  int first_token, tokens_per_block;
  bool vec;              // rows of 16 bytes' alignment
};

// A token's page, slot and position, or a page of -1: as the exact cache's append has it.
__device__ __forceinline__ void find_token(const Args &g, int t, int *page, int *pos) {
  int seq = t, j = 0;
  if (g.a.offsets) {
    int lo = 0, hi = g.q.n_seqs;  // the last sequence that begins at or before t
    while (hi - lo > 1) {
      const int mid = lo + (hi - lo) / 2;
      if (g.a.offsets[mid] <= t) lo = mid;
      else hi = mid;
    }
    seq = lo;
    j = g.a.offsets[lo] <= t && t < g.a.offsets[lo + 1] ? t - g.a.offsets[lo] : -1;
  }
  *page = -1;
  *pos = 0;
  if (j < 0 || g.q.lengths[seq] < 0) return;
  const int64_t at = (int64_t)g.q.lengths[seq] + j;
  if (at >= kMaxTokens) return;
  *pos = (int)at;
  const int col = *pos / g.p.page_size;
  if (col >= g.q.width) return;
  const int x = g.q.table[(int64_t)seq * g.q.stride + col];
  if (x >= 0 && x < g.p.n_pages) *page = x;
}

// A block takes a few tokens of all heads; a lane 8 channels of a (token, head)'s key and value,
// four neighbours a scale.  Bound: the input rows' bytes.
template <typename T>
__global__ __launch_bounds__(kThreads) void append4_kernel(const Args g) {
  __shared__ float2 s_cs[kCosSin];
  __shared__ int s_page[kBlockTokens], s_pos[kBlockTokens];
  const int tid = threadIdx.x, dim = g.p.dim, heads = g.p.n_heads;
  const int t0 = g.first_token + blockIdx.x * g.tokens_per_block;
  const int nt = min(g.tokens_per_block, g.a.n_tokens - t0);
  for (int t = tid; t < nt; t += kThreads) find_token(g, t0 + t, &s_page[t], &s_pos[t]);
  __syncthreads();
  const RotaryTable &rt = g.p.rotary;
  if (rt.pairs) {
    for (int i = tid; i < nt * rt.pairs; i += kThreads) {
      const int t = i / rt.pairs;
      s_cs[i] = rotary_cos_sin(rt.steps[i - t * rt.pairs], s_pos[t], rt.amplitude);
    }
    __syncthreads();
  }
  const int lanes = dim / 8, items = nt * heads * lanes;
  // (whole groups of four lanes: items is a multiple of 4)
  for (int i = tid; i < items; i += kThreads) {
    const int row = i / lanes, chunk = i - row * lanes;
    const int t = row / heads, head = row - t * heads;
    const void *rows[2] = {
        static_cast<const char *>(g.a.k) + (t0 + t) * (int64_t)g.a.k_nb[1] + head * (int64_t)g.a.k_nb[0],
        static_cast<const char *>(g.a.v) + (t0 + t) * (int64_t)g.a.v_nb[1] + head * (int64_t)g.a.v_nb[0]};
    float x[2][8];
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      const T *from = static_cast<const T *>(rows[v]) + 8 * chunk;
      if (g.vec) {
        constexpr int N = 16 / sizeof(T);
#pragma unroll
        for (int k = 0; k < 8; k += N) {
          const RowVec<T, N> y = load_rows<true, T, N>(from + k);
#pragma unroll
          for (int j = 0; j < N; ++j) x[v][k + j] = row_get(y.x[j]);
        }
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) x[v][k] = row_get(from[k]);
      }
    }
    if (rt.pairs)
      rotate8(x[0], rows[0], chunk, g.p.io, rt, [&](int pair) { return s_cs[t * rt.pairs + pair]; });
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      int byte;
      const uint32_t codes = encode4(x[v], &byte);
      if (s_page[t] < 0) continue;
      const int slot = s_pos[t] % g.p.page_size;
      store4(static_cast<char *>(v ? g.p.v_pages : g.p.k_pages) + block4_at(g.p, s_page[t], head, slot),
             slot & 15, chunk, codes, byte, v, dim);
    }
  }
}

__global__ __launch_bounds__(kThreads) void read4_kernel(const Args g) {
  __shared__ int s_page[kBlockTokens], s_pos[kBlockTokens];
  const int tid = threadIdx.x, dim = g.p.dim, heads = g.p.n_heads;
  const int t0 = g.first_token + blockIdx.x * g.tokens_per_block;
  const int nt = min(g.tokens_per_block, g.a.n_tokens - t0);
  for (int t = tid; t < nt; t += kThreads) find_token(g, t0 + t, &s_page[t], &s_pos[t]);
  __syncthreads();
  const int lanes = dim / 8, items = nt * heads * lanes;
  for (int i = tid; i < items; i += kThreads) {
    const int row = i / lanes, chunk = i - row * lanes;
    const int t = row / heads, head = row - t * heads;
    const int64_t to = ((int64_t)(t0 + t) * heads + head) * dim + 8 * chunk;
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      uint32_t codes = 0;
      int byte = 127;
      if (s_page[t] >= 0) {
        const int slot = s_pos[t] % g.p.page_size;
        codes = load4(static_cast<const char *>(v ? g.p.v_pages : g.p.k_pages) +
                          block4_at(g.p, s_page[t], head, slot),
                      slot & 15, chunk, v, dim, &byte);
      }
      const float scale = scale4(byte);
      float *out = (v ? g.v_out : g.k_out) + to;
#pragma unroll
      for (int k = 0; k < 8; k += 4) {
        RowVec<float, 4> y;
#pragma unroll
        for (int j = 0; j < 4; ++j) y.x[j] = value4(codes >> 4 * (k + j), scale);
        store_rows<true>(out + k, y);
      }
    }
  }
}

// Tokens of a block: a few rounds of its threads, and no fewer than 2,048 blocks for it.
int tokens_per_block(const PagedShape &p, int n_tokens, bool rotates) {
  int tb = std::max(1, 8 * kThreads / (p.n_heads * p.dim / 8));
  if (rotates && p.rotary.pairs) tb = std::min(tb, kCosSin / p.rotary.pairs);
  return std::max(1, std::min({tb, kBlockTokens, n_tokens / 2048}));
}

}  // namespace

hipError_t launch_paged4_append(const PagedShape &p, const PagedSeqs &q, const PagedAppend &a,
                                hipStream_t s) {
  Args g{p, q, a};
  size_t x = reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v);
  for (int k = 0; k < 2; ++k) x |= a.k_nb[k] | a.v_nb[k];
  g.vec = x % 16 == 0;
  g.tokens_per_block = tokens_per_block(p, a.n_tokens, true);
  return launch_over_tokens(a.n_tokens, g.tokens_per_block, [&](int first, int blocks) {
    g.first_token = first;
    switch (p.io) {
      case IoType::F32: append4_kernel<float><<<blocks, kThreads, 0, s>>>(g); break;
      case IoType::F16: append4_kernel<_Float16><<<blocks, kThreads, 0, s>>>(g); break;
      default: append4_kernel<Bf16><<<blocks, kThreads, 0, s>>>(g);
    }
  });
}

hipError_t launch_paged4_read(const PagedShape &p, const PagedSeqs &q, int n_tokens,
                              const int *offsets, float *k, float *v, hipStream_t s) {
  Args g{p, q, PagedAppend{}};
  g.a.n_tokens = n_tokens;
  g.a.offsets = offsets;
  g.k_out = k;
  g.v_out = v;
  g.tokens_per_block = tokens_per_block(p, n_tokens, false);
  return launch_over_tokens(n_tokens, g.tokens_per_block, [&](int first, int blocks) {
    g.first_token = first;
    read4_kernel<<<blocks, kThreads, 0, s>>>(g);
  });
}

}  // namespace aq
