// paged_attend.hip -- attention of one new token per sequence over its pages, scores as they
// are: the kernel's variants (paged_attend.hpp).
#include "paged_attend.hpp"

namespace aq {

size_t paged_workspace_bytes(const PagedShape &p) {
  return 4 * sizeof(int) * kMaxBlocks +
         2 * sizeof(float) * part_floats(padded_dim(p.dim)) * most_blocks(p.cus, padded_dim(p.dim));
}

hipError_t launch_paged_attend(const PagedShape &p, const PagedSeqs &q, const PagedAttend &a,
                               const PagedAppend *step, void *workspace, hipStream_t s) {
  const Args g = attend_args(p, q, a, step, workspace);
  switch (p.io) {
    case IoType::F32: return launch_type<float, false>(g, s);
    case IoType::F16: return launch_type<_Float16, false>(g, s);
    default: return launch_type<Bf16, false>(g, s);
  }
}

}  // namespace aq
