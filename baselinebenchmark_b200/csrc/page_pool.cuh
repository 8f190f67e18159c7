// Pages taken from and given back to a pool: what the kernels and the C ABI share.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace moba {

// Sequences of a call: two numbers of each lie in shared memory.
constexpr int kPoolMostBatch = 16384;

struct PoolParams {
  int64_t rows, table_stride;
  int batch, per_seq, page_shift, pages;
  const int32_t *cu, *lens;                // cu == null: pages are given back
  const int32_t* parents;
  int32_t *table, *free, *count;
  long long* slots;
  int32_t *positions, *missing;
};
cudaError_t launch_pool(const PoolParams& p, cudaStream_t st);

}  // namespace moba
