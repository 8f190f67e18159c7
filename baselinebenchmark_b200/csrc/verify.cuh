// Verification of drafted tokens: what the kernel and the C ABI share.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace moba {

// Rows of a sequence, and tokens of a vocabulary, that one call takes at most: what the kernel keeps of them lies in shared memory (a row takes 30 bytes,
// a token an eighth of a bit a block).
constexpr int kVerifyMostRows = 1024;
constexpr int64_t kVerifyMostTokens = (int64_t)1 << 22;

struct VerifyParams {
  const void *target, *draft, *tokens;
  int64_t target_stride, draft_stride, rows, vocabulary;
  int64_t part;                            // of the vocabulary, a block's
  int batch, max_new, tokens64;
  const int32_t *cu, *parents;
  const float *accept, *sample;
  int32_t *path, *count;
  void* next;
};
cudaError_t launch_verify(VerifyParams a, int dtype, cudaStream_t st);

}  // namespace moba
