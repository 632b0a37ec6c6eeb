// paged4_attend.hip -- the attention over pages of 4-bit values (paged4_attend.hpp).
#include "paged4_attend.hpp"

namespace aq {

hipError_t launch_paged4_attend(const PagedShape &p, const PagedSeqs &q, const PagedAttend &a,
                                const PagedAppend *step, const PagedScores &sc, void *workspace,
                                hipStream_t s) {
  Args g = attend_args(p, q, a, step, workspace);
  g.sc = sc;
  if (sc.softcap > 0) {
    g.cap_in = a.scale / sc.softcap;
    g.cap2 = sc.softcap * kLog2e;
  }
  const bool shaped = sc.softcap > 0 || sc.slopes || sc.prefix || sc.first;
  return shaped ? launch4_dim<true>(g, s) : launch4_dim<false>(g, s);
}

}  // namespace aq
