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
// over 8 kv heads, the same over one, 2 of 500 over 8, one of 40000 over 8; 64-token pages; 16-bit rows are bf16)
//   head dim 64           8: 53 / 71, 14 / 25, 9 / 18, 21 / 39        16: 56 / 72, 17 / 25, 10 / 18, 24 / 39      32: 95 / 73, 20 / 25, 12 / 18, 30 / 40
//   head dim 128          8: 93 / 93, 18 / 33, 11 / 20, 39 / 56       16: 100 / 94, 25 / 31, 14 / 20, 43 / 56     32: 183 / 96, 30 / 31, 16 / 20, 60 / 57
//   head dim 256          8: 182 / 170, 40 / 50, 13 / 25, 65 / 91     16: 187 / 171, 43 / 48, 17 / 26, 70 / 93    32: 331 / 174, 57 / 48, 19 / 26, 119 / 95
//   e4m3, head dim 64    16: 45 / 112, 17 / 30, 12 / 21, 25 / 49      48: 110 / 114, 24 / 30, 14 / 21, 40 / 49    64: 140 / 115, 29 / 31, 15 / 22, 49 / 50
//   e4m3, head dim 96    16: 56 / 147, 19 / 36, 13 / 24, 29 / 61      48: 133 / 149, 29 / 36, 16 / 24, 48 / 62    64: 171 / 150, 34 / 36, 17 / 25, 59 / 62
//   e4m3, head dim 128   16: 65 / 157, 20 / 37, 14 / 26, 29 / 64      48: 161 / 160, 32 / 37, 16 / 26, 55 / 65    64: 206 / 162, 38 / 37, 17 / 25, 69 / 67
//   e4m3, head dim 256   16: 164 / 342, 37 / 57, 21 / 37, 65 / 123    32: 298 / 343, 56 / 59, 22 / 37, 103 / 125  48: 428 / 345, 74 / 60, 23 / 38, 141 / 126
//   int8, fp16, 128      16: 73 / 153, 20 / 36, 14 / 25, 31 / 63      48: 188 / 157, 35 / 37, 16 / 26, 63 / 65    64: 244 / 159, 42 / 37, 17 / 25, 80 / 66
// The limits are those of large calls, where most is at stake.  Calls of one sequence or of short ones would be served better here up to 32 rows
// and more of 16-bit pages; the rule does not look at that.
inline bool paged_few_rows(const PagedParams& p) {
  const int most = p.store != MOBA_STORE_SAME ? (p.D == 256 ? 32 : 48) : p.D == 256 ? 16 : 8;
  return (int64_t)p.max_new * p.G <= most;
}

size_t paged_rows_workspace(const PagedParams& p);
cudaError_t launch_paged_rows(const PagedParams& p, const void* q, const void* kp, const void* vp, const uint8_t* ks,
                              const uint8_t* vs, void* out, float* lse, void* workspace, cudaStream_t st);
size_t paged_few_workspace(const PagedParams& p);
cudaError_t launch_paged_few(const PagedParams& p, const void* q, const void* kp, const void* vp, const uint8_t* ks,
                             const uint8_t* vs, void* out, float* lse, void* workspace, cudaStream_t st);

}  // namespace moba
