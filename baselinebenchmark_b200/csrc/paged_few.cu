// Attention over pages for sequences with few new tokens: each token sees all positions before it.
#include "paged_few.cuh"

namespace moba {

size_t paged_few_workspace(const PagedParams& p) { return few_workspace(p); }

cudaError_t launch_paged_few(const PagedParams& p, const void* q, const void* kp, const void* vp, const uint8_t* ks,
                             const uint8_t* vs, void* out, float* lse, void* workspace, cudaStream_t st) {
  return launch_few<false>(p, nullptr, q, kp, vp, ks, vs, out, lse, workspace, st);
}

}  // namespace moba
