// Attention over pages for sequences with few drafted tokens that form a tree: each sees its own branch.
#include "paged_few.cuh"

namespace moba {

cudaError_t launch_paged_few_tree(const PagedParams& p, const int32_t* parents, const void* q, const void* kp, const void* vp, const uint8_t* ks,
                                  const uint8_t* vs, void* out, float* lse, void* workspace, cudaStream_t st) {
  return launch_few<true>(p, parents, q, kp, vp, ks, vs, out, lse, workspace, st);
}

}  // namespace moba
