// Keys and values of many sequences in pages: what the kernels that write, read and attend to them share.
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"
#include "moba_b200.h"

namespace moba {

// Launch-time view of a call (struct moba_paged), passed to kernels by value.
struct PagedParams {
  int64_t T;
  int B, Hq, Hkv, G, D;
  int pages, page_shift, per_seq, max_new;
  int fp16, store;
  float sl2;                               // factor of the scores, log2 e included
  int64_t sq_t, sq_h, so_t, so_h, sk_t, sk_h, sv_t, sv_h;
  int64_t kp_p, kp_t, kp_h, vp_p, vp_t, vp_h, table_stride;
  const int32_t* cu;
  const int32_t* lens;
  const int32_t* table;
};

// A sequence of the batch: its packed rows [row0, row0 + n), of which row i is at position pos0 + i.  Numbers that make no
// sense are cut to the rows and the table that there are.
struct PagedSeq {
  int row0, n, pos0;
  int len;                                 // keys that the table has room for
};
__device__ __forceinline__ PagedSeq paged_seq(const PagedParams& p, int b) {
  const int64_t lo = __ldg(p.cu + b), hi = __ldg(p.cu + b + 1);
  const int len = __ldg(p.lens + b);
  PagedSeq s;
  s.row0 = (int)min(max(lo, (int64_t)0), p.T);
  s.n = max((int)min(hi, p.T) - s.row0, 0);
  s.pos0 = (int)max((int64_t)len - s.n, -((int64_t)1 << 31));
  s.len = (int)min((int64_t)max(len, 0), (int64_t)p.per_seq << p.page_shift);
  return s;
}

// Page of a position >= 0 of sequence b, -1 where there is none.
__device__ __forceinline__ int paged_page(const PagedParams& p, int b, int pos) {
  const int i = pos >> p.page_shift;
  if (i >= p.per_seq) return -1;
  const int id = __ldg(p.table + (int64_t)b * p.table_stride + i);
  return (unsigned)id < (unsigned)p.pages ? id : -1;
}

// The least power of two of a row: 2^-96, so that the inverses of a million rows' add up within fp32.
constexpr int kPagedLeastByte = 127 - 96;
__device__ __forceinline__ float paged_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

cudaError_t launch_paged_store(const PagedParams& p, const void* k, const void* v, void* kp, void* vp, uint8_t* ks, uint8_t* vs,
                               cudaStream_t st);
cudaError_t launch_paged_load(const PagedParams& p, const void* kp, const void* vp, const uint8_t* ks, const uint8_t* vs, void* k,
                              void* v, cudaStream_t st);

// Sequences that one launch of an attention kernel takes: their work is added up in shared memory.
constexpr int kPagedBatch = 1024;

// Items of more rows run on tcgen05.  Two new launches (the plan, the join of many rows) cost a small call 8 us there; in a large one the tensor
// memory kernel keeps up with the copies whatever the rows are, where the other's chain grows with them.  8-bit codes are turned once for each
// tile of 16 rows here and once for each of 128 or 256 there, by fewer warps.  (rows: this kernel / tcgen05, us; 16 sequences of 8000 tokens
// over 8 kv heads, the same over one, 2 of 500; 64-token pages)
//   head dim 128          8:  93 / 94, 19 / 33, 12 / 20    16: 120 / 95, 39 / 33, 13 / 21     32: 207 / 96, 43 / 33, 16 / 21
//   head dim 128, e4m3    8:  57 / 157, 17 / 41, 12 / 26   16:  59 / 157, 22 / 41, 13 / 26    32: 100 / 159, 24 / 41, 13 / 26
//                         48 (8 sequences): 79 / 92        64: 100 / 92, 34 / 42
//   head dim 256          8: 179 / 171, 51 / 50, 16 / 27    16: 186 / 171, 49 / 50, 17 / 27    32: 345 / 173, 58 / 51, 23 / 27
inline bool paged_few_rows(const PagedParams& p) {
  const int most = p.store != MOBA_STORE_SAME ? 48 : p.D == 256 ? 16 : 8;
  return (int64_t)p.max_new * p.G <= most;
}

size_t paged_rows_workspace(const PagedParams& p);
cudaError_t launch_paged_rows(const PagedParams& p, const void* q, const void* kp, const void* vp, const uint8_t* ks,
                              const uint8_t* vs, void* out, float* lse, void* workspace, cudaStream_t st);
size_t paged_few_workspace(const PagedParams& p);
cudaError_t launch_paged_few(const PagedParams& p, const void* q, const void* kp, const void* vp, const uint8_t* ks,
                             const uint8_t* vs, void* out, float* lse, void* workspace, cudaStream_t st);

}  // namespace moba
