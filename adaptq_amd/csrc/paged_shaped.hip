// paged_shaped.hip -- the paged attention with scores of its own: capped, biased, masked, and
// with the weight that each token got added up (paged_attend.hpp holds the kernel).
//
// Weights: a token's weight needs the maximum and sum over all tokens, which are there when the
// attention is done.  So it leaves its scores (4 bytes a token and query head, beside rows of
// 4 * dim a token and key head), and a second launch turns them into weights, adds those of a
// key head's query heads in their order, and adds the sum to the token's.  Reading the keys
// again instead would cost half of the attention.
#include "paged_attend.hpp"

namespace aq {

namespace {

// A block takes 1,024 tokens of one sequence and key head, a thread 4 of them.  Bound: the
// scores' bytes, read once, and the weights', read and written.
struct WeightArgs {
  Args g;
  PagedWeights w;
  int chunks;
  int64_t first_block;
};

constexpr int kChunk = 4 * kThreads;

__global__ __launch_bounds__(kThreads) void weights_kernel(const WeightArgs x) {
  const Args &g = x.g;
  const int64_t block = x.first_block + blockIdx.x;
  const int chunk = (int)(block % x.chunks);
  const int64_t rest = block / x.chunks;
  const int head = (int)(rest % g.p.n_heads), seq = (int)(rest / g.p.n_heads);
  const ShapedSpan span = span_of<kShaped>(g, seq, g.q.lengths[seq], 16);
  const int t = chunk * kChunk + 4 * (int)threadIdx.x;
  if (t >= span.n || t + 4 <= span.lo) return;
  const int col = page_column(g.page_of, t >> 4);
  const int page = g.q.table[(int64_t)seq * g.q.stride + col];
  if (page < 0 || page >= g.p.n_pages) return;
  f32x4 sum = {0, 0, 0, 0};
  const int64_t row = seq * (int64_t)g.a.q_heads + head * g.group;
  for (int i = 0; i < g.group; ++i) {
    const float2 ml = g.stats[row + i];
    const f32x4 s = *reinterpret_cast<const f32x4 *>(g.scores + (row + i) * g.score_stride + t);
    const float part = 1.0f / ml.y;
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[j] = fmaf(__builtin_amdgcn_exp2f(s[j] - ml.x), part, sum[j]);
  }
  float *to = x.w.weights + seq * x.w.nb[1] + head * x.w.nb[0] + t;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (span.sees(t + j)) to[j] += sum[j];
}

int64_t score_stride(const PagedShape &p, int width) {
  return std::min((int64_t)width * p.page_size, (int64_t)kMaxTokens);
}

int64_t stats_of(int q_heads, int n_seqs) {  // scores behind them are aligned to 16 bytes
  return ((int64_t)n_seqs * q_heads + 1) / 2 * 2;
}

}  // namespace

size_t paged_weights_workspace(const PagedShape &p, int q_heads, int n_seqs, int width) {
  return (size_t)n_seqs * q_heads * sizeof(float) * score_stride(p, width) +
         sizeof(float2) * stats_of(q_heads, n_seqs);
}

hipError_t launch_paged_shaped(const PagedShape &p, const PagedSeqs &q, const PagedAttend &a,
                               const PagedAppend *step, const PagedScores &sc,
                               const PagedWeights &w, void *workspace, hipStream_t s) {
  WeightArgs x{};
  Args &g = x.g;
  g = attend_args(p, q, a, step, workspace);
  g.sc = sc;
  if (sc.softcap > 0) {
    g.cap_in = a.scale / sc.softcap;
    g.cap2 = sc.softcap * kLog2e;
  }
  if (w.weights) {
    g.score_stride = score_stride(p, q.width);
    g.stats = static_cast<float2 *>(w.workspace);
    g.scores = reinterpret_cast<float *>(g.stats + stats_of(a.q_heads, q.n_seqs));
  }
  hipError_t e;
  switch (p.io) {
    case IoType::F32: e = launch_type<float, true>(g, s); break;
    case IoType::F16: e = launch_type<_Float16, true>(g, s); break;
    default: e = launch_type<Bf16, true>(g, s);
  }
  if (e != hipSuccess || !w.weights || g.cap == 0) return e;
  x.w = w;
  x.chunks = (int)((g.cap + kChunk - 1) / kChunk);
  const int64_t blocks = (int64_t)q.n_seqs * p.n_heads * x.chunks;
  constexpr int64_t kMost = (((int64_t)1 << 32) - 1) / kThreads;
  for (int64_t b = 0; b < blocks; b += kMost) {
    x.first_block = b;
    weights_kernel<<<(int)std::min(kMost, blocks - b), kThreads, 0, s>>>(x);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace aq
