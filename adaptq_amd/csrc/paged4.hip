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
  uint64_t token_mul;    // row / tokens_per_block = row * token_mul >> 32, for a block's rows
  bool vec;              // rows of 16 bytes' alignment
};

// Where a token lies: the byte in the pools that its block of 16 begins at for head 0, or -1, its
// number in it, and its position; as the exact cache's append has it.
__device__ __forceinline__ void find_token(const Args &g, int t, int64_t *at_block, int *in,
                                           int *pos) {
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
  *at_block = -1;
  *in = 0;
  *pos = 0;
  if (j < 0 || g.q.lengths[seq] < 0) return;
  const int64_t at = (int64_t)g.q.lengths[seq] + j;
  if (at >= kMaxTokens) return;
  *pos = (int)at;
  const int col = *pos / g.p.page_size;
  if (col >= g.q.width) return;
  const int x = g.q.table[(int64_t)seq * g.q.stride + col];
  if (x < 0 || x >= g.p.n_pages) return;
  const int slot = *pos - col * g.p.page_size;
  *at_block = block4_at(g.p, x, 0, slot);
  *in = slot & 15;
}

// A block takes a few tokens of all heads; a lane 8 channels of the keys or values of a (token,
// head), four neighbours a scale, kRows rows of them in flight.  Rows go token by token within a
// head, so that neighbouring rows' codes, which lie side by side in a block of 16 tokens, are
// written together.  Bound: the bytes.
constexpr int kRows = 4;

template <typename T>
__global__ __launch_bounds__(kThreads) void append4_kernel(const Args g) {
  __shared__ float2 s_cs[kCosSin];
  __shared__ int64_t s_at[kBlockTokens];
  __shared__ int s_in[kBlockTokens], s_pos[kBlockTokens];
  const int tid = threadIdx.x, dim = g.p.dim, tb = g.tokens_per_block;
  const int t0 = g.first_token + blockIdx.x * tb;
  const int nt = min(tb, g.a.n_tokens - t0);
  const RotaryTable &rt = g.p.rotary;
  const int lanes = dim / 8, rows = g.p.n_heads * tb;
  const int per = kThreads / (2 * lanes);  // rows of a pass: keys, then values
  const int item = tid % (2 * lanes), row0 = tid < per * 2 * lanes ? tid / (2 * lanes) : rows;
  const bool value = item >= lanes;
  const int chunk = value ? item - lanes : item;
  const char *in = static_cast<const char *>(value ? g.a.v : g.a.k) + t0 * (int64_t)(value ? g.a.v_nb[1] : g.a.k_nb[1]);
  const int64_t nb1 = value ? g.a.v_nb[0] : g.a.k_nb[0], nb2 = value ? g.a.v_nb[1] : g.a.k_nb[1];
  float x[kRows][8];
  int tok[kRows], head[kRows];
  const auto load = [&](int r0) {
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
      const int r = r0 + j * per;
      head[j] = (int)((uint64_t)r * g.token_mul >> 32);
      tok[j] = r < rows ? r - head[j] * tb : nt;
      if (tok[j] >= nt) continue;
      const T *from = reinterpret_cast<const T *>(in + tok[j] * nb2 + head[j] * nb1) + 8 * chunk;
      if (g.vec) {
        constexpr int N = 16 / sizeof(T);
#pragma unroll
        for (int k = 0; k < 8; k += N) {
          const RowVec<T, N> y = load_rows<true, T, N>(from + k);
#pragma unroll
          for (int i = 0; i < N; ++i) x[j][k + i] = row_get(y.x[i]);
        }
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) x[j][k] = row_get(from[k]);
      }
    }
  };
  load(row0);
  for (int t = tid; t < nt; t += kThreads) find_token(g, t0 + t, &s_at[t], &s_in[t], &s_pos[t]);
  __syncthreads();
  if (rt.pairs) {
    for (int i = tid; i < nt * rt.pairs; i += kThreads) {
      const int t = i / rt.pairs;
      s_cs[i] = rotary_cos_sin(rt.steps[i - t * rt.pairs], s_pos[t], rt.amplitude);
    }
    __syncthreads();
  }
  char *pool = static_cast<char *>(value ? g.p.v_pages : g.p.k_pages);
  const int head_bytes = g.p.page_size / 16 * block4_bytes(dim);
  // (the four lanes of a scale have the same rows)
  for (int r0 = row0; r0 < rows; r0 += kRows * per) {
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
      const int t = tok[j];
      if (t >= nt) continue;
      if (rt.pairs && !value)
        rotate8(x[j], in + t * nb2 + head[j] * nb1, chunk, g.p.io, rt,
                [&](int pair) { return s_cs[t * rt.pairs + pair]; });
      int byte;
      const uint32_t codes = encode4(x[j], &byte);
      const int64_t at = s_at[t];
      if (at < 0) continue;
      store4(pool + at + (uint64_t)(uint32_t)head[j] * (uint32_t)head_bytes, s_in[t], chunk, codes,
             byte, value, dim);
    }
    load(r0 + kRows * per);
  }
}

// The same way back, a lane 4 channels so that a wave writes whole lines.
__global__ __launch_bounds__(kThreads) void read4_kernel(const Args g) {
  __shared__ int64_t s_at[kBlockTokens];
  __shared__ int s_in[kBlockTokens], s_pos[kBlockTokens];
  const int tid = threadIdx.x, dim = g.p.dim, tb = g.tokens_per_block;
  const int t0 = g.first_token + blockIdx.x * tb;
  const int nt = min(tb, g.a.n_tokens - t0);
  for (int t = tid; t < nt; t += kThreads) find_token(g, t0 + t, &s_at[t], &s_in[t], &s_pos[t]);
  __syncthreads();
  const int lanes = dim / 4, rows = g.p.n_heads * tb;
  const int per = max(kThreads / (2 * lanes), 1);
  const int head_bytes = g.p.page_size / 16 * block4_bytes(dim);
  for (int item = tid; item < per * 2 * lanes; item += kThreads) {
    const int row0 = item / (2 * lanes), c = item - row0 * 2 * lanes;
    const bool value = c >= lanes;
    const int d = 4 * (value ? c - lanes : c);
    const char *pool = static_cast<const char *>(value ? g.p.v_pages : g.p.k_pages);
    float *out = (value ? g.v_out : g.k_out) + (int64_t)t0 * g.p.n_heads * dim + d;
    for (int r0 = row0; r0 < rows; r0 += kRows * per) {
      uint32_t codes[kRows];
      int byte[kRows];
      int64_t to[kRows];
#pragma unroll
      for (int j = 0; j < kRows; ++j) {
        const int r = r0 + j * per;
        const int head = (int)((uint64_t)r * g.token_mul >> 32), t = r - head * tb;
        codes[j] = 0;
        byte[j] = 127;
        to[j] = -1;
        if (r >= rows || t >= nt) continue;
        to[j] = ((int64_t)t * g.p.n_heads + head) * dim;
        const int64_t at = s_at[t];
        if (at < 0) continue;
        codes[j] = load4(pool + at + (uint64_t)(uint32_t)head * (uint32_t)head_bytes, s_in[t], d,
                         value, dim, &byte[j]);
      }
#pragma unroll
      for (int j = 0; j < kRows; ++j) {
        if (to[j] < 0) continue;
        const float scale = scale4(byte[j]);
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[j], scale, 0);
        const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[j], scale, 1);
        store_rows<true>(out + to[j], RowVec<float, 4>{{a[0], a[1], b[0], b[1]}});
      }
    }
  }
}

// Tokens of a block: a few rounds of its threads, of lanes for 8 channels, in fours that share a
// place in the pages, and no fewer than 1,024 blocks for it.
void cut_tokens(Args &g, int lanes, bool rotates) {
  int tb = std::max(1, 4 * kRows * kThreads / (2 * lanes * g.p.n_heads));
  if (rotates && g.p.rotary.pairs) tb = std::min(tb, kCosSin / g.p.rotary.pairs);
  tb = std::max(1, std::min({tb, kBlockTokens, g.a.n_tokens / 1024}));
  if (tb > 4) tb = tb / 4 * 4;
  g.tokens_per_block = tb;
  g.token_mul = (((uint64_t)1 << 32) + tb - 1) / tb;
}

}  // namespace

hipError_t launch_paged4_append(const PagedShape &p, const PagedSeqs &q, const PagedAppend &a,
                                hipStream_t s) {
  Args g{p, q, a};
  size_t x = reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v);
  for (int k = 0; k < 2; ++k) x |= a.k_nb[k] | a.v_nb[k];
  g.vec = x % 16 == 0;
  cut_tokens(g, p.dim / 8, true);
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
  cut_tokens(g, p.dim / 4, false);
  return launch_over_tokens(n_tokens, g.tokens_per_block, [&](int first, int blocks) {
    g.first_token = first;
    read4_kernel<<<blocks, kThreads, 0, s>>>(g);
  });
}

}  // namespace aq
