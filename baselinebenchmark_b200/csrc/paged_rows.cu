// Attention over pages for sequences with many new tokens: each token sees all positions before it.
#include "paged_rows.cuh"

namespace moba {

size_t paged_rows_workspace(const PagedParams& p) { return rows_workspace(p, false); }

cudaError_t launch_paged_rows(const PagedParams& p, const void* q, const void* kp, const void* vp, const uint8_t* ks,
                              const uint8_t* vs, void* out, float* lse, void* workspace, cudaStream_t st) {
  return launch_rows<false>(p, nullptr, q, kp, vp, ks, vs, out, lse, workspace, st);
}

}  // namespace moba
