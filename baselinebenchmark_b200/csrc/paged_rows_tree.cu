// Attention over pages for sequences with many new tokens that form trees: each sees its own branch.
#include "paged_rows.cuh"

namespace moba {

size_t paged_rows_tree_workspace(const PagedParams& p) { return rows_workspace(p, true); }

cudaError_t launch_paged_rows_tree(const PagedParams& p, const int32_t* parents, const void* q, const void* kp, const void* vp, const uint8_t* ks,
                                   const uint8_t* vs, void* out, float* lse, void* workspace, cudaStream_t st) {
  return launch_rows<true>(p, parents, q, kp, vp, ks, vs, out, lse, workspace, st);
}

}  // namespace moba
