// paged_few.hip -- attention of a few new tokens per sequence (draft tokens, short chunks): the
// single-token kernel (paged_attend.hpp) with a row a (query, query head).
//
// Up to 16 rows cost what one does, straight from the registers that rows were loaded into, and
// the work is cut evenly over the blocks whatever the lengths: bound by the rows' bytes, where a
// prompt's tile of 128 rows would leave three waves of four without any.
#include "paged_attend.hpp"

namespace aq {

namespace {

template <typename T, int DP, bool EXACT>
hipError_t launch_few(const Args &g, hipStream_t s) {
  return launch_attend<DP, Kind<T, DP>::kUnit>(
      g, attend_kernel<Attend<T, DP, EXACT, true, false, true, true>>,
      attend_kernel<Attend<T, DP, EXACT, false, false, true, true>>, s);
}

template <typename T>
hipError_t launch_few_type(const Args &g, hipStream_t s) {
  switch (padded_dim(g.p.dim)) {
    case 64: return g.p.dim == 64 ? launch_few<T, 64, true>(g, s) : launch_few<T, 64, false>(g, s);
    case 128:
      return g.p.dim == 128 ? launch_few<T, 128, true>(g, s) : launch_few<T, 128, false>(g, s);
    default:
      return g.p.dim == 256 ? launch_few<T, 256, true>(g, s) : launch_few<T, 256, false>(g, s);
  }
}

}  // namespace

hipError_t launch_paged_few(const PagedShape &p, const PagedSeqs &q, const PagedPrompt &a,
                            void *workspace, hipStream_t s) {
  PagedAttend t{};
  t.q = a.q;
  t.out = a.out;
  for (int i = 0; i < 2; ++i) {
    t.q_nb[i] = a.q_nb[i];
    t.out_nb[i] = a.out_nb[i];
  }
  t.q_heads = a.q_heads;
  t.scale = a.scale;
  t.window = a.scores.window;
  Args g = attend_args(p, q, t, nullptr, workspace);
  g.sc = a.scores;
  if (g.sc.softcap > 0) {
    g.cap_in = a.scale / g.sc.softcap;
    g.cap2 = g.sc.softcap * kLog2e;
  }
  g.offsets = a.offsets;
  g.n_tokens = a.n_tokens;
  // tiles of a sequence on the average, for the launch's size and the rows' mark
  const int64_t rows = (int64_t)a.n_tokens * g.group;
  g.q_tiles = (int)std::max<int64_t>(1, (rows / q.n_seqs + kTile - 1) / kTile);
  g.segs = p.n_heads * g.q_tiles;
  switch (p.io) {
    case IoType::F32: return launch_few_type<float>(g, s);
    case IoType::F16: return launch_few_type<_Float16>(g, s);
    default: return launch_few_type<Bf16>(g, s);
  }
}

}  // namespace aq
