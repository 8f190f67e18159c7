// Rotary positions: what the kernel and the C ABI share.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace moba {

struct RotaryParams {
  int64_t rows;
  int heads_q, heads_k, dim, turned, interleaved, inverse, fp16;
  float magnitude;
  int64_t q_t, q_h, k_t, k_h, qo_t, qo_h, ko_t, ko_h;
  const void *q, *k;
  void *q_out, *k_out;
  const int32_t* positions;
  const long long* turns;
  int slots, lanes, units, per_unit;       // set by the launch: see rotary.cu
};
cudaError_t launch_rotary(RotaryParams p, cudaStream_t st);

}  // namespace moba
