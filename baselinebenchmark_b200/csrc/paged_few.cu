// Attention over pages for sequences with few new tokens (decode steps, drafted tokens), with mma.sync.
//
// Rows of an item are the (new token, query head) pairs of one sequence and kv head, token by token, 8 or 16 at a time: the M of one
// m16n8k16, or half of it.  With so few rows the bytes of K and V bound the call (2 * 16 rows of products a key against 4 D bytes of it), so what
// counts is that many bytes are always on their way, and the tensor work only has to keep up: no tcgen05 here, whose 128
// lanes would be mostly empty and whose tiles would have to be handed from warp to warp.
//   - A warp is on its own: TMA brings it blocks of 16 keys (32 of 8-bit pages) of K and V into its own ring of swizzled shared memory, and it
//     runs Q.K^T, the softmax step and P.V on them in registers.  Nothing is waited for but its copies.  (With a copy instruction
//     and its addresses for every 16 bytes a block was 490 instructions; with boxes it is 300.)
//   - The keys of all items are one line of units (a block for each warp of a CTA), cut into equal pieces, one for each CTA: whatever
//     the lengths in the batch are, all SMs read the same number of bytes.  A CTA has at most two items that others share; their
//     results (maximum, sum, unnormalised output, fp32) go through the workspace, and a second kernel joins them in the order of
//     the keys.  No atomics: a call gives the same bits every time.
//   - 8-bit codes become fp16, which holds them exactly, on their way from shared memory to the tensor core.  Scales are applied to
//     scores and probabilities, of which there are fewer than elements of K and V.  The power of two 2^e of a V row is part of its
//     weight: with x = score * log2(e) and M a reference near the running maximum of x + e, a key weighs w = 2^(x + e - M), 2^8 at
//     most; the output is sum(w * code) / sum(w * 2^-e).  Where all weights of a block are 2^-14 and more (or nothing at all) they go to P.V as
//     fp16.  A row of zeros (e = 0) or one with a single large element may put M far above what the other channels are made of: a block with
//     smaller weights takes them as bf16, which has fp32's range, over codes turned to bf16; fp16 rows, which are owed three bits more, as the
//     sum of two bf16 numbers, in two products.
//     bf16 queries become fp16, which holds them exactly where they lie within 2^-23 to 2^10 (or are zeros); a tile with others stays bf16
//     and has the codes turned to bf16 for its Q.K^T.
//   - P is rounded to the 16-bit type that V has (or as said): 2^-8 (bf16), 2^-11 (fp16) relative at most, as in the dense stage of the prefill.
// The reference that weights are taken to is only moved when the maximum exceeds it by more than 8 (a factor of 256); over codes it is set 4
// below the maximum, so that fp16 holds weights down to 2^-18 of the largest at least.
// Measured (replayed from a graph, us; head dim 128, 32/8 heads unless said otherwise; in brackets the bytes at the measured copy bandwidth):
//   one token of 48 requests of 16 to 11001 tokens                        188 -> 172 (boxes) -> 151 (three CTAs an SM) -> 115 (what an item costs besides
//                                                                         its keys counts on the line)                          [103]
//   one token of 16 requests of 16385 to 40001, e4m3                      214 -> 147 (172 where no page is left in L2)          [138]
//     the same where no block's weights fit fp16: bf16 172, fp16 263; where no tile's queries do: 168; fp16 with every block near or beyond 65504: 739
//   one token of 16 requests of 8000, 16/4 heads, head dim 256, e4m3      77; int8, fp16 88                                     [40]
//   five tokens of 12 requests of 338 to 20016, int8, 16/4 heads, fp16    92 -> 52                                              [14]
//   one token behind 20011, 16/4 heads, head dim 64, fp16                 64 -> 19 (pieces joined in parallel) -> 16            [3]
// The last is a chain of latencies, and much of the one before it: the plan of the line, a page's number, its rows, four warps joined, the second kernel.
#include <type_traits>

#include "paged.cuh"
#include "sm100_ptx.cuh"

namespace moba {

bool make_page_map(CUtensorMap* m, int elem, int D, const void* base, int pages, int slots, int H, int64_t sp, int64_t st, int64_t sh,
                   int box_rows);
bool make_page_parts_map(CUtensorMap* m, int elem, int subs, const void* base, int pages, int slots, int H, int64_t sp, int64_t st,
                         int64_t sh, int box_rows);

namespace {

using namespace ptx;

constexpr int kFewWarps = 4, kFewThreads = kFewWarps * 32;
constexpr int kFewMaxCtas = 148 * 3;
constexpr float kLn2 = 0.6931471805599453f;

template <int D, int kStore, int kM> struct FewShape {
  static constexpr bool kCodes = kStore != MOBA_STORE_SAME;
  static constexpr int kKeys = kCodes ? 32 : 16;                     // of a warp's block
  static constexpr int kSpan = kCodes ? 128 : 64;                    // elements of 128 bytes
  static constexpr int kSubs = (D + kSpan - 1) / kSpan;              // sub-blocks [keys][128 bytes] of K, and of V
  static constexpr int kSubBytes = kKeys * 128;
  static constexpr int kSideBytes = kSubs * kSubBytes;               // K; V behind it
  static constexpr int kStageBytes = 2 * kSideBytes;
  static constexpr bool kParts = !kCodes && kSubs > 1 && D % kSpan == 0;   // one box has all sub-blocks (not of head dim 96: a row's would end in the next)
  // Three CTAs, twelve warps, an SM with 16 KB of stages each: what a warp waits for is its own chain of instructions, and there have to be
  // others meanwhile.  One CTA with 48 KB a warp at head dim 256, where output and queries alone are 192 registers (over codes 255 with
  // 100 to 290 bytes spilled); two with 24 KB for 16 rows over codes at head dim 128, which do not fit the registers of three (16 sequences of 8000
  // tokens, 32/8 heads, e4m3 97 us with three, 57 with two; 8 rows of 16 longer ones 169 with three, 175 with two; both before weights were looked at).
  static constexpr int kCtas = kStageBytes == 16384 ? 1 : kCodes && kM == 16 && D == 128 ? 2 : 3;
  static constexpr int kStages = kStageBytes == 16384 || kCtas == 2 ? 3 : kStageBytes == 8192 ? 2 : 4;
  static constexpr int kWarpBytes = kStages * kStageBytes;
  static constexpr int kUnit = kKeys * kFewWarps;                    // keys of a CTA's unit
  static constexpr size_t kSmem = 1024 + (size_t)kFewWarps * kWarpBytes;
  // bf16 queries over codes: turned to fp16 as they come, and read again by a tile that cannot have them so; or kept until that is known, where
  // registers are short (8 rows at head dim 128 and 256; 8 rows of 16 sequences of 8000 tokens, e4m3, 16/4 heads of 256: 86 us at once, 77 kept;
  // 16 rows, 32/8 heads of 128: 65 at once, 68 kept).
  static constexpr bool kAtOnce = kM == 16 || D == 64;
  static_assert(kWarpBytes >= 16 * D * 4, "the output of a warp fits its ring");
};

// `bytes` (a multiple of 16) to shared memory, counted on the barrier
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes),
               "r"(bar)
               : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <bool kHalf>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (kHalf)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Four codes, of which the bytes of `kA` and `kB` (a prmt selector each) are wanted as pairs of fp16.
template <int kStore, uint32_t kLo, uint32_t kHi>
__device__ __forceinline__ void codes_to_half(uint32_t x, uint32_t& lo, uint32_t& hi) {
  if (kStore == MOBA_STORE_E4M3) {
    const uint32_t y = kLo == 0x10 && kHi == 0x32 ? x : __byte_perm(x, 0, kLo | kHi << 8);
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(y));
  } else {
    // u = code + 128 under the exponent of 1024 is 1024 + u: taking 1152 off leaves the code
    const uint32_t u = x ^ 0x80808080u;
    constexpr uint32_t kSelLo = 0x4040 | (kLo & 0xf) | (kLo & 0xf0) << 4, kSelHi = 0x4040 | (kHi & 0xf) | (kHi & 0xf0) << 4;
    const uint32_t a = __byte_perm(u, 0x64u, kSelLo), b = __byte_perm(u, 0x64u, kSelHi);
    const __half2 off = __half2half2(__ushort_as_half(0x6480));                  // 1152
    const __half2 ra = __hsub2(*reinterpret_cast<const __half2*>(&a), off), rb = __hsub2(*reinterpret_cast<const __half2*>(&b), off);
    lo = *reinterpret_cast<const uint32_t*>(&ra);
    hi = *reinterpret_cast<const uint32_t*>(&rb);
  }
}

// Two fp16 codes as bf16, which holds those of both types exactly.
__device__ __forceinline__ uint32_t half_codes_to_bf16(uint32_t x) {
  const float2 f = unpack2<true>(x);
  return pack2_16<false>(f.x, f.y);
}
// bf16 queries over codes are taken 2^6-fold to fp16, where that changes none of a tile's (they are zeros, or 2^-23 to 2^10 in magnitude).
constexpr float kQueryScale = 64.f;
template <bool kHalf>
__device__ __forceinline__ uint32_t scaled_query(uint32_t x, float f) {
  const float2 y = unpack2<false>(x);
  return pack2_16<kHalf>(y.x * f, y.y * f);
}
// Magnitudes of a tile's elements, as pairs of bf16: the least that is not 0 (its bits, less one) and the largest.
struct QueryRange {
  uint32_t least = 0xffffffffu, most = 0;
  __device__ __forceinline__ void add(uint32_t x) {
    const uint32_t y = x & 0x7fff7fffu;
    least = __viaddmin_u16x2(y, 0xffffffffu, least);
    most = __vmaxu2(y, most);
  }
  // the largest is 2^e or more; all that are not 0 are
  __device__ __forceinline__ bool reaches(int e) const { return max(most & 0xffffu, most >> 16) >= (uint32_t)(127 + e) << 7; }
  __device__ __forceinline__ bool all_reach(int e) const { return min(least & 0xffffu, least >> 16) >= ((uint32_t)(127 + e) << 7) - 1; }
};
// fp16 rows: two codes, and what they become where a value is beyond fp16 (pages that were written from bf16 rows).
template <int kStore> constexpr uint32_t kMostHalfByte = kStore == MOBA_STORE_E4M3 ? 134 : 135;   // 448 * 2^7 and -128 * 2^8 are fp16's
__device__ __forceinline__ uint32_t codes_within_half(uint32_t x, float s0, float s1) {
  const float2 c = unpack2<true>(x);
  return pack2_half(fabsf(c.x * s0) >= 65520.f ? copysignf(INFINITY, c.x) : c.x, fabsf(c.y * s1) >= 65520.f ? copysignf(INFINITY, c.y) : c.y);
}
constexpr float kLift = 4.f;               // over codes: how far below the maximum the reference is set
constexpr uint32_t kLeastHalf = 0x38800000;   // 2^-14, fp16's least normal number, as fp32

// ---- the line of units -------------------------------------------------------
// Sequence b has tiles(b) row tiles of kM, each of units(b) units of keys, for every kv head: in the order
// sequence, kv head, row tile, unit.  (Units behind the last key that a tile sees are empty: they differ by the few new tokens.)  In
// front of an item's units lie kItemUnits that stand for what it costs besides (its Q rows, the way of its first copies, its
// output): without them a CTA that got two dozen short sequences came in last, 40 us behind the others of a decode step of 48 requests.
constexpr int kItemUnits = 2;
struct FewPlan {
  int64_t begin[kPagedBatch + 1];          // first unit of a sequence
  int64_t scan[16];
};
struct FewItem {
  int b, h, tile;
  int u0, u1, units;                       // this piece's units of the item's (u1 <= u0: none)
  int64_t end;                             // of the item on the line
};

template <int kM>
__device__ __forceinline__ int few_tiles(const PagedParams& p, const PagedSeq& s) { return (int)(((int64_t)s.n * p.G + kM - 1) / kM); }

// All threads; returns the number of units of the batch.
template <int kM, int kUnit, int kThreads>
__device__ __forceinline__ int64_t few_plan(const PagedParams& p, FewPlan& plan) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t carry = 0;
  for (int base = 0; base < p.B; base += kThreads) {
    const int b = base + threadIdx.x;
    int64_t w = 0;
    if (b < p.B) {
      const PagedSeq s = paged_seq(p, b);
      // (rows without a key need an item too: they are written as zeros)
      const int units = max((s.len + kUnit - 1) / kUnit, 1);
      w = (int64_t)few_tiles<kM>(p, s) * (units + kItemUnits) * p.Hkv;
    }
    int64_t x = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) plan.scan[warp] = x;
    __syncthreads();
    int64_t before = carry;
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) {
      if (i < warp) before += plan.scan[i];
      carry += plan.scan[i];
    }
    if (b < p.B) plan.begin[b] = before + x - w;
    __syncthreads();
  }
  if (threadIdx.x == 0) plan.begin[p.B] = carry;
  __syncthreads();
  return carry;
}

// The item that has unit `u` of the line, from there on up to `end`.
template <int kM, int kUnit>
__device__ __forceinline__ FewItem few_item(const PagedParams& p, const FewPlan& plan, int64_t u, int64_t end, PagedSeq& s) {
  int lo = 0, n = p.B;
  while (n > 1) {                                           // last b with begin[b] <= u: one with units
    const int half = n >> 1;
    const bool up = plan.begin[lo + half] <= u;
    lo = up ? lo + half : lo;
    n = up ? n - half : half;
  }
  s = paged_seq(p, lo);
  FewItem it;
  it.b = lo;
  it.units = max((s.len + kUnit - 1) / kUnit, 1);
  const int line = it.units + kItemUnits;
  const int64_t at = u - plan.begin[lo], item = at / line;
  const int tiles = few_tiles<kM>(p, s);
  it.h = (int)(item / tiles);
  it.tile = (int)(item - (int64_t)it.h * tiles);
  const int on = (int)(at - item * line) - kItemUnits;
  it.u0 = max(on, 0);
  it.u1 = (int)min((int64_t)it.units, on + (end - u));
  it.end = u - on + it.units;
  return it;
}

// CTAs that share the line, and where the units of each begin: as many for all, one more for the first few.  A piece is two units at
// least, so that short lines are joined from fewer pieces.
struct FewCut {
  int ctas, rest;
  int64_t each;
  __device__ __forceinline__ int64_t operator()(int c) const { return each * c + min(c, rest); }
};
__device__ __forceinline__ FewCut few_cut(int64_t units, int grid) {
  FewCut f;
  f.ctas = (int)max(min((units + 1) / 2, (int64_t)grid), (int64_t)1);
  f.each = units / f.ctas;
  f.rest = (int)(units - f.each * f.ctas);
  return f;
}

// For the joining kernel, from each CTA: the item that it began and others end (pieces: theirs and its own; 0: there is none).
struct FewShared {
  int32_t pieces, row0, n, h, tile;
};

struct FewArgs {
  const void* q;
  const void *kp, *vp;
  const uint8_t *ks, *vs;
  void* out;
  float* lse;
  float* part;                             // [2 * CTAs][kM][D]: outputs of shared items, by CTA: 0 one that others began, 1 one that others end
  float2* part_ml;                         // [2 * CTAs][kM]: {maximum, sum}
  FewShared* shared;                       // [CTAs]
};

// Packed row (token, head) of row r of a tile, or -1.
template <int kM>
__device__ __forceinline__ bool few_row(const PagedParams& p, const PagedSeq& s, int h, int tile, int r, int64_t& token, int& head, int& i) {
  const int64_t at = (int64_t)tile * kM + r;
  i = (int)(at / p.G);
  head = h * p.G + (int)(at - (int64_t)i * p.G);
  token = (int64_t)s.row0 + i;
  return i < s.n;
}

// kM: rows of a tile, 8 or 16 (the upper half of the MMA's rows is empty with 8, and its exponentials are left out)
template <bool kHalf, int D, int kStore, int kM>
__global__ void __launch_bounds__(kFewThreads, FewShape<D, kStore, kM>::kCtas)
paged_few_kernel(const PagedParams p, const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, const FewArgs a) {
  using S = FewShape<D, kStore, kM>;
  constexpr bool kCodes = S::kCodes;
  constexpr bool kF16 = kHalf || kCodes;                    // operands of the MMAs
  constexpr int kSteps = D / 16;                            // k-steps of Q.K^T
  constexpr int kBlocksN = S::kKeys / 8;                    // 8-key blocks of scores
  constexpr int kGroups = S::kKeys / 16;                    // groups of 16 keys, each in one page
  constexpr int kE = kM / 8;                                // rows of this thread: g, and g + 8
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  __shared__ FewPlan plan;
  __shared__ float2 warp_ml[kFewWarps][kM];
  __shared__ uint64_t full[kFewWarps][S::kStages];
  __shared__ __align__(16) uint8_t scales[kFewWarps][S::kStages][2][32];
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int g = lane >> 2, t4 = lane & 3;
  if (threadIdx.x == 0) {
    for (int w = 0; w < kFewWarps; ++w)
      for (int i = 0; i < S::kStages; ++i) mbar_init(smem_u32(&full[w][i]), 1);
    fence_barrier_init();
    prefetch_tmap(&tmap_k);
    prefetch_tmap(&tmap_v);
  }
  pdl_wait();
  pdl_trigger();
  const int64_t units = few_plan<kM, S::kUnit, kFewThreads>(p, plan);
  const FewCut cut = few_cut(units, gridDim.x);
  const int64_t first = cut(blockIdx.x), last = cut(blockIdx.x + 1);
  if ((int)blockIdx.x >= cut.ctas || first >= last) {
    if (threadIdx.x == 0) a.shared[blockIdx.x].pieces = 0;
    return;
  }
  const uint32_t ring = smem_u32(smem) + warp * S::kWarpBytes;
  // addresses of ldmatrix within a sub-block: row of this lane, pieces in the order of the swizzle
  const int mrow = lane & 7, mi = lane >> 3;
  const uint32_t k_row = (uint32_t)((mrow + 8 * (kCodes ? mi : mi >> 1)) * 128), v_row = (uint32_t)((mrow + 8 * (kCodes ? mi : mi & 1)) * 128);
  constexpr int kPer = kCodes ? 8 : 4;                      // k-steps, or pairs of pieces, of a sub-block
  uint32_t k_at[kPer], v_at[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    k_at[i] = k_row + (uint32_t)(((kCodes ? i : 2 * i + (mi & 1)) ^ mrow) << 4);
    v_at[i] = v_row + (uint32_t)(((kCodes ? i : 2 * i + (mi >> 1)) ^ mrow) << 4);
  }
  const uint32_t full0 = smem_u32(&full[warp][0]);
  int st_in = 0, st_out = 0;                                // stages that come next: to be filled, to be read
  uint32_t phase = 0;                                       // of st_out
  uint32_t there = 0;                                       // groups in flight that have a page, the oldest block's lowest
  bool ok = true;
  FewShared shared{0, 0, 0, 0, 0};

  for (int64_t u = first; u < last;) {
    PagedSeq s;
    const FewItem it = few_item<kM, S::kUnit>(p, plan, u, last, s);
    u = it.end;
    if (it.u1 <= it.u0) continue;
    // keys that some row of the tile sees: rows of the last new token see the most, the first row sees the least
    const int64_t tile_last = min((int64_t)s.n - 1, ((int64_t)(it.tile + 1) * kM - 1) / p.G);
    const int end = (int)min(max((int64_t)s.pos0 + tile_last + 1, (int64_t)0), (int64_t)s.len);
    const int all_see = (int)min(max((int64_t)s.pos0 + (int64_t)it.tile * kM / p.G + 1, (int64_t)0), (int64_t)s.len);
    const int key_of_warp = warp * S::kKeys;
    // this warp's blocks: unit v of [u0, u1) has keys v * kUnit + key_of_warp ..
    int blocks = 0;
    if (end > key_of_warp) blocks = min(it.u1, (end - key_of_warp + S::kUnit - 1) / S::kUnit) - it.u0;
    blocks = ok ? max(blocks, 0) : 0;

    // ---- copies: the pages of a block are looked up one block ahead of its copies
    int page[kGroups];                                      // as the table has them: they are looked at when the copies are asked for
    const int32_t* row = p.table + (int64_t)it.b * p.table_stride;
    auto lookup = [&](int j) {
#pragma unroll
      for (int gr = 0; gr < kGroups; ++gr) {
        const int key = (it.u0 + j) * S::kUnit + key_of_warp + 16 * gr;
        page[gr] = -1;
        if (j < blocks && key < end) page[gr] = __ldg(row + (key >> p.page_shift));   // (end <= the table's reach)
      }
    };
    int waiting = 0;                                        // blocks asked for and not read yet
    auto copy = [&](int j) {                                // block j into stage st_in; `page` is the block's
      const uint32_t dst = ring + st_in * S::kStageBytes, bar = full0 + 8 * st_in;
      const int key0 = (it.u0 + j) * S::kUnit + key_of_warp;
      // 32 keys in one page come as one box
      const bool one = kGroups == 2 && p.page_shift > 4;
      uint32_t got = 0;
#pragma unroll
      for (int gr = 0; gr < kGroups; ++gr) got |= ((unsigned)page[gr] < (unsigned)p.pages ? 1u : 0u) << gr;
      if (lane == 0) {
        const uint32_t boxes = one ? (got ? 2 : 0) : __popc(got);
        mbar_expect_tx(bar, boxes * (2 * S::kSubs * 16 * 128 + (kCodes ? 2 * 16 : 0)));
#pragma unroll
        for (int gr = 0; gr < kGroups; ++gr) {
          if (!((got >> gr) & 1) || (one && gr > 0)) continue;
          const int slot = (key0 + 16 * gr) & ((1 << p.page_shift) - 1);
          if constexpr (S::kParts) {
            tma_load_5d(dst, &tmap_k, bar, 0, slot, 0, it.h, page[gr]);
            tma_load_5d(dst + S::kSideBytes, &tmap_v, bar, 0, slot, 0, it.h, page[gr]);
          } else {
#pragma unroll
            for (int i = 0; i < S::kSubs; ++i) {
              tma_load_4d(dst + i * S::kSubBytes + gr * 2048, &tmap_k, bar, i * S::kSpan, slot, it.h, page[gr]);
              tma_load_4d(dst + S::kSideBytes + i * S::kSubBytes + gr * 2048, &tmap_v, bar, i * S::kSpan, slot, it.h, page[gr]);
            }
          }
          if (kCodes) {
            const int64_t at = (((int64_t)page[gr] * p.Hkv + it.h) << p.page_shift) + slot;
            bulk_load(smem_u32(&scales[warp][st_in][0][16 * gr]), a.ks + at, one ? 32 : 16, bar);
            bulk_load(smem_u32(&scales[warp][st_in][1][16 * gr]), a.vs + at, one ? 32 : 16, bar);
          }
        }
      }
      // (both groups of one page; the second may lie behind the keys that are seen, and is masked then)
      if (one && got) got = 3;
      there |= got << (kGroups * waiting);
      ++waiting;
      st_in = st_in + 1 == S::kStages ? 0 : st_in + 1;
    };
    there = 0;
    lookup(0);
#pragma unroll
    for (int j = 0; j < S::kStages - 1; ++j) {
      if (j < blocks) copy(j);
      lookup(j + 1);
    }

    // ---- rows of this thread
    int lim[kE];                                            // keys below are visible
    bool wide = false;                                      // over codes: bf16 rows that fp16 does not hold
    QueryRange range;
    uint32_t qa[kSteps][4];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      if (e >= kE) {
#pragma unroll
        for (int k = 0; k < kSteps; ++k) qa[k][e] = qa[k][2 + e] = 0;
        continue;
      }
      int64_t token;
      int head, i;
      const bool on = few_row<kM>(p, s, it.h, it.tile, g + 8 * e, token, head, i);
      lim[e] = on ? (int)min(max((int64_t)s.pos0 + i + 1, (int64_t)0), (int64_t)s.len) : 0;
      const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(a.q) + token * p.sq_t + head * p.sq_h;
      if (!kCodes) {
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
          qa[k][e] = on ? __ldg(reinterpret_cast<const uint32_t*>(q + 16 * k + 2 * t4)) : 0;
          qa[k][2 + e] = on ? __ldg(reinterpret_cast<const uint32_t*>(q + 16 * k + 8 + 2 * t4)) : 0;
        }
      } else {
        // the dims that a lane's four codes of a step are of: 4 t4 .. 4 t4 + 3 of its 16
        uint2 x[kSteps];
#pragma unroll
        for (int k = 0; k < kSteps; ++k) x[k] = on ? __ldg(reinterpret_cast<const uint2*>(q + 16 * k + 4 * t4)) : make_uint2(0, 0);
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
          if (!kHalf) { range.add(x[k].x); range.add(x[k].y); }
          qa[k][e] = S::kAtOnce && !kHalf ? scaled_query<true>(x[k].x, kQueryScale) : x[k].x;
          qa[k][2 + e] = S::kAtOnce && !kHalf ? scaled_query<true>(x[k].y, kQueryScale) : x[k].y;
        }
      }
    }
    float rs = kCodes && !kHalf && S::kAtOnce ? p.sl2 * (1.f / kQueryScale) : p.sl2;   // factor of the scores
    if (kCodes && !kHalf) wide = __any_sync(0xffffffffu, range.reaches(10) || !range.all_reach(-23));
    // (a wide tile's rows are taken as they are, unless sums of their products with codes might leave fp32)
    if constexpr (kCodes && !kHalf && S::kAtOnce) {
      if (wide) {
        const bool large = __any_sync(0xffffffffu, range.reaches(100)), small = !__any_sync(0xffffffffu, range.reaches(-60));
        const float f = large ? 0x1p-64f : small ? 0x1p64f : 1.f;
        rs = p.sl2 * (large ? 0x1p64f : small ? 0x1p-64f : 1.f);
#pragma unroll
        for (int e = 0; e < kE; ++e) {
          int64_t token;
          int head, i;
          if (!few_row<kM>(p, s, it.h, it.tile, g + 8 * e, token, head, i)) continue;
          const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(a.q) + token * p.sq_t + head * p.sq_h;
#pragma unroll
          for (int k = 0; k < kSteps; ++k) {
            const uint2 x = __ldg(reinterpret_cast<const uint2*>(q + 16 * k + 4 * t4));
            qa[k][e] = scaled_query<false>(x.x, f);
            qa[k][2 + e] = scaled_query<false>(x.y, f);
          }
        }
      }
    } else if constexpr (kCodes && !kHalf) {
      auto scale_rows = [&](auto half, float f) {
#pragma unroll
        for (int k = 0; k < kSteps; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if ((i & 1) < kE) qa[k][i] = scaled_query<decltype(half)::value>(qa[k][i], f);
      };
      if (!wide) {
        rs *= 1.f / kQueryScale;
        scale_rows(std::true_type(), kQueryScale);
      } else {
        const bool large = __any_sync(0xffffffffu, range.reaches(100)), small = !__any_sync(0xffffffffu, range.reaches(-60));
        if (large || small) {
          rs *= large ? 0x1p64f : 0x1p-64f;
          scale_rows(std::false_type(), large ? 0x1p-64f : 0x1p64f);
        }
      }
    }
    float o[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
    float m[kE], l[kE];
#pragma unroll
    for (int e = 0; e < kE; ++e) { m[e] = -INFINITY; l[e] = 0.f; }

    for (int j = 0; j < blocks; ++j) {
      if (j + S::kStages - 1 < blocks) copy(j + S::kStages - 1);
      lookup(j + S::kStages);
      ok = __all_sync(0xffffffffu, mbar_wait(full0 + 8 * st_out, phase));
      if (!ok) {                                            // copies that are under way get time to land
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 2000000ull) __nanosleep(1000);
        break;
      }
      const uint32_t sk = ring + st_out * S::kStageBytes, sv = sk + S::kSideBytes;
      const int key0 = (it.u0 + j) * S::kUnit + key_of_warp;
      const uint32_t mine = there & ((1u << kGroups) - 1);
      there >>= kGroups;
      --waiting;
      const bool plain = key0 + S::kKeys <= all_see && mine == (1u << kGroups) - 1;
      if (!plain) {
        // rows of V that nobody may see are zeros: whatever the page, or the stage, holds there, 0 * it stays out of P.V
        for (int n = lane; n < S::kKeys * 8; n += 32) {
          const int r = n >> 3;
          if (key0 + r < end && ((mine >> (r >> 4)) & 1)) continue;
#pragma unroll
          for (int i = 0; i < S::kSubs; ++i)
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(sv + i * S::kSubBytes + n * 16), "r"(0) : "memory");
        }
        fence_proxy_async_smem();
        __syncwarp();
      }
      // ---- S = Q.K^T
      bool beyond = false;                                  // fp16 rows: values of the block may be beyond fp16
      float sc[kBlocksN][4];
#pragma unroll
      for (int n = 0; n < kBlocksN; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[n][e] = 0.f;
      if (kCodes && kHalf) {
        const bool seen = key0 + lane < end && ((mine >> (lane >> 4)) & 1);
        const uint32_t most = max(scales[warp][st_out][0][lane], scales[warp][st_out][1][lane]);
        beyond = __any_sync(0xffffffffu, seen && most > kMostHalfByte<kStore>);
      }
      if (kCodes && kHalf && beyond) {
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
          uint32_t b[4];
          ldsm4(sk + k_at[k % kPer] + (k / kPer) * S::kSubBytes, b);
#pragma unroll
          for (int n = 0; n < kBlocksN; ++n) {
            const float s = paged_scale(scales[warp][st_out][0][8 * n + g]);
            uint32_t b0, b1;
            codes_to_half<kStore, 0x10, 0x32>(b[n], b0, b1);
            mma_16816<true>(sc[n], qa[k], codes_within_half(b0, s, s), codes_within_half(b1, s, s));
          }
        }
      } else if (kCodes && !kHalf && wide) {
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
          uint32_t b[4];
          ldsm4(sk + k_at[k % kPer] + (k / kPer) * S::kSubBytes, b);
#pragma unroll
          for (int n = 0; n < kBlocksN; ++n) {
            uint32_t b0, b1;
            codes_to_half<kStore, 0x10, 0x32>(b[n], b0, b1);
            mma_16816<false>(sc[n], qa[k], half_codes_to_bf16(b0), half_codes_to_bf16(b1));
          }
        }
      } else
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        uint32_t b[4];
        ldsm4(sk + k_at[k % kPer] + (k / kPer) * S::kSubBytes, b);
        if (!kCodes) {                                      // matrices: keys 0-7 pieces 2k, 2k + 1, keys 8-15 the same
          mma_16816<kF16>(sc[0], qa[k], b[0], b[1]);
          mma_16816<kF16>(sc[1], qa[k], b[2], b[3]);
        } else {                                            // matrices: piece k (16 dims) of keys 0-7, 8-15, 16-23, 24-31
#pragma unroll
          for (int n = 0; n < kBlocksN; ++n) {
            uint32_t b0, b1;
            codes_to_half<kStore, 0x10, 0x32>(b[n], b0, b1);
            mma_16816<kF16>(sc[n], qa[k], b0, b1);
          }
        }
      }
      // ---- x = scores in powers of two (+ the exponent of the V row)
      float vinv[kBlocksN][2];
      if (kCodes) {
        const uint8_t(*sb)[32] = scales[warp][st_out];
#pragma unroll
        for (int n = 0; n < kBlocksN; ++n) {
          const uint32_t kb = *reinterpret_cast<const uint16_t*>(sb[0] + 8 * n + 2 * t4), vb = *reinterpret_cast<const uint16_t*>(sb[1] + 8 * n + 2 * t4);
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            // (fp16 rows: from 2^25 all that is not 0 is beyond fp16; how far does not count for the other channels' weights)
            const uint32_t ke = (kb >> (8 * c)) & 255, vs = (vb >> (8 * c)) & 255, ve = kHalf ? min(vs, 127u + 25u) : vs;
            const float kf = paged_scale(ke), vf = (float)((int)ve - 127);
            vinv[n][c] = vs == 255 ? __uint_as_float(0x7fc00000u) : __uint_as_float((254u - ve) << 23);
#pragma unroll
            for (int e = 0; e < kE; ++e) sc[n][2 * e + c] = fmaf(sc[n][2 * e + c], rs * kf, vf);
          }
        }
      } else {
#pragma unroll
        for (int n = 0; n < kBlocksN; ++n)
#pragma unroll
          for (int e = 0; e < 2 * kE; ++e) sc[n][e] *= p.sl2;
      }
      if (!plain) {
#pragma unroll
        for (int n = 0; n < kBlocksN; ++n)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int key = key0 + 8 * n + 2 * t4 + c;
            const bool here = (mine >> (n >> 1)) & 1;
#pragma unroll
            for (int e = 0; e < kE; ++e)
              if (key >= lim[e] || !here) sc[n][2 * e + c] = -INFINITY;
            if (key >= end || !here) vinv[n][c] = 0.f;
          }
      }
      // ---- running maximum
      bool moved = false;
      float alpha[kE];
#pragma unroll
      for (int e = 0; e < kE; ++e) {
        float mx = -INFINITY;
#pragma unroll
        for (int n = 0; n < kBlocksN; ++n) mx = fmaxf(mx, fmaxf(sc[n][2 * e], sc[n][2 * e + 1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        alpha[e] = 1.f;
        if (mx > m[e] + 8.f) {
          const float ref = kCodes ? mx - kLift : mx;
          alpha[e] = exp2f(m[e] - ref);                     // (0 the first time)
          m[e] = ref;
          moved = true;
        }
      }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int e = 0; e < kE; ++e) {
#pragma unroll
          for (int i = 0; i < D / 8; ++i) {
            o[i][2 * e] *= alpha[e];
            o[i][2 * e + 1] *= alpha[e];
          }
          l[e] *= alpha[e];
        }
      }
      uint32_t pa[kGroups][4];
      uint32_t least = 0xffffffffu;                         // the least weight that is not 0 (its bits, less one)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        if (e >= kE) {
#pragma unroll
          for (int gr = 0; gr < kGroups; ++gr) pa[gr][1] = pa[gr][3] = 0;
          continue;
        }
        // a row that has seen nothing yet has no reference: any finite one leaves its weights at 0
        const float ref = m[e] == -INFINITY ? 0.f : m[e];
#pragma unroll
        for (int n = 0; n < kBlocksN; ++n) {
          const float w0 = ex2_approx(sc[n][2 * e] - ref), w1 = ex2_approx(sc[n][2 * e + 1] - ref);
          l[e] += kCodes ? w0 * vinv[n][0] + w1 * vinv[n][1] : w0 + w1;
          pa[n >> 1][(n & 1) * 2 + e] = pack2_16<kF16>(w0, w1);
          if (kCodes) {
            least = min(least, min(__float_as_uint(w0) - 1u, __float_as_uint(w1) - 1u));
            sc[n][2 * e] = w0;
            sc[n][2 * e + 1] = w1;
          }
        }
      }
      // ---- O += P.V
      if (kCodes && (__any_sync(0xffffffffu, least < kLeastHalf - 1u) || beyond)) {
        // weights that fp16 has not: as bf16, and for fp16 rows what that leaves of them, as bf16 again
#pragma unroll 1
        for (int part = 0; part < (kHalf ? 2 : 1); ++part) {
#pragma unroll
          for (int n = 0; n < kBlocksN; ++n)
#pragma unroll
            for (int e = 0; e < kE; ++e) {
              const uint32_t y = pack2_16<false>(sc[n][2 * e], sc[n][2 * e + 1]);
              const float2 f = unpack2<false>(y);
              pa[n >> 1][(n & 1) * 2 + e] = y;
              sc[n][2 * e] -= f.x;
              sc[n][2 * e + 1] -= f.y;
            }
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            uint32_t b[4];
            ldsm4_t(sv + v_at[i % kPer] + (i / kPer) * S::kSubBytes, b);
#pragma unroll
            for (int gr = 0; gr < kGroups; ++gr) {
              uint32_t e0, o0, e1, o1;
              codes_to_half<kStore, 0x20, 0x31>(b[2 * gr], e0, o0);
              codes_to_half<kStore, 0x20, 0x31>(b[2 * gr + 1], e1, o1);
              if (kHalf && beyond) {
                float s[4];                                 // (rows that nobody sees are zeros: their bytes are anything)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                  const int n = 16 * gr + 8 * (c >> 1) + 2 * t4 + (c & 1);
                  s[c] = paged_scale(min((uint32_t)scales[warp][st_out][1][n], 254u));
                }
                e0 = codes_within_half(e0, s[0], s[1]);
                o0 = codes_within_half(o0, s[0], s[1]);
                e1 = codes_within_half(e1, s[2], s[3]);
                o1 = codes_within_half(o1, s[2], s[3]);
              }
              mma_16816<false>(o[2 * i], pa[gr], half_codes_to_bf16(e0), half_codes_to_bf16(e1));
              mma_16816<false>(o[2 * i + 1], pa[gr], half_codes_to_bf16(o0), half_codes_to_bf16(o1));
            }
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          uint32_t b[4];
          ldsm4_t(sv + v_at[i % kPer] + (i / kPer) * S::kSubBytes, b);
          if (!kCodes) {                                    // matrices: keys 0-7, 8-15 of pieces 2i, the same of 2i + 1
            mma_16816<kF16>(o[2 * i], pa[0], b[0], b[1]);
            mma_16816<kF16>(o[2 * i + 1], pa[0], b[2], b[3]);
          } else {
            // matrices: keys 0-7, 8-15, 16-23, 24-31 of piece i; pairs of dims are their 16-bit elements: the even dims of 16, and the odd ones
#pragma unroll
            for (int gr = 0; gr < kGroups; ++gr) {
              uint32_t e0, o0, e1, o1;
              codes_to_half<kStore, 0x20, 0x31>(b[2 * gr], e0, o0);
              codes_to_half<kStore, 0x20, 0x31>(b[2 * gr + 1], e1, o1);
              mma_16816<kF16>(o[2 * i], pa[gr], e0, e1);
              mma_16816<kF16>(o[2 * i + 1], pa[gr], o0, o1);
            }
          }
        }
      }
      if (++st_out == S::kStages) { st_out = 0; phase ^= 1; }
      __syncwarp();
    }

    // ---- the warps' results, joined by all threads
    float* so = reinterpret_cast<float*>(smem + warp * S::kWarpBytes);                            // [kM][D]
#pragma unroll
    for (int e = 0; e < kE; ++e) {
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
      // a row with a score that is not a number has no maximum to speak of: with this one it stays NaN in every join (so does one whose
      // copies did not arrive in time)
      if (l[e] != l[e] || !ok) { m[e] = INFINITY; l[e] = __uint_as_float(0x7fc00000u); }
      if (t4 == 0) warp_ml[warp][g + 8 * e] = make_float2(m[e], l[e]);
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        if (!kCodes) {
          *reinterpret_cast<float2*>(so + (g + 8 * e) * D + 8 * i + 2 * t4) = make_float2(o[i][2 * e], o[i][2 * e + 1]);
        } else {                                            // column c of blocks 2i, 2i + 1: dims 2c, 2c + 1 of 16
          float* at = so + (g + 8 * e) * D + 16 * (i >> 1) + (i & 1);
          at[2 * (2 * t4)] = o[i][2 * e];
          at[2 * (2 * t4 + 1)] = o[i][2 * e + 1];
        }
      }
    }
    __syncthreads();
    const bool whole = it.u0 == 0 && it.u1 == it.units;
    if (it.u0 == 0 && !whole) {
      int lo = blockIdx.x + 1, hi = cut.ctas;               // the last CTA that begins before the item's end
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (cut(mid) < it.end) lo = mid; else hi = mid;
      }
      shared = FewShared{lo - (int)blockIdx.x + 1, s.row0, s.n, it.h, it.tile};
    }
    const int64_t slot = 2 * (int64_t)blockIdx.x + (it.u0 == 0 ? 1 : 0);
    for (int n = threadIdx.x; n < kM * (D / 4); n += kFewThreads) {
      const int r = n / (D / 4), c = n % (D / 4) * 4;
      int64_t token;
      int head, i;
      if (!few_row<kM>(p, s, it.h, it.tile, r, token, head, i)) continue;
      float mx = -INFINITY;
#pragma unroll
      for (int w = 0; w < kFewWarps; ++w) mx = fmaxf(mx, warp_ml[w][r].x);
      const float ref = mx == -INFINITY ? 0.f : mx;
      float sum = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kFewWarps; ++w) {
        const float f = exp2f(warp_ml[w][r].x - ref);
        const float4 v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(smem + w * S::kWarpBytes) + r * D + c);
        if (f == 0.f) continue;
        sum += f * warp_ml[w][r].y;
        x[0] += f * v.x; x[1] += f * v.y; x[2] += f * v.z; x[3] += f * v.w;
      }
      if (whole) {
        const float inv = mx == -INFINITY ? 0.f : 1.f / sum;
        uint2 y;
        y.x = pack2_16<kHalf>(x[0] * inv, x[1] * inv);
        y.y = pack2_16<kHalf>(x[2] * inv, x[3] * inv);
        *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out) + token * p.so_t + head * p.so_h + c) = y;
        if (a.lse != nullptr && c == 0) a.lse[(int64_t)head * p.T + token] = (mx + log2f(sum)) * kLn2;
      } else {
        *reinterpret_cast<float4*>(a.part + (slot * kM + r) * D + c) = make_float4(x[0], x[1], x[2], x[3]);
        if (c == 0) a.part_ml[slot * kM + r] = make_float2(mx, sum);
      }
    }
    fence_proxy_async_smem();                               // the ring is copied to again
    __syncthreads();
  }
  if (threadIdx.x == 0) a.shared[blockIdx.x] = shared;
}

// Joins the pieces of the items that several CTAs share.  Block c: the item that CTA c began and did not end.  A few long sequences
// have a hundred pieces an item: blocks share its output, and threads in groups take every so many of the pieces, their sums are added in the
// order of the groups.
constexpr int kJoinThreads = 512, kJoinShare = 128;
template <bool kHalf, int D, int kM>
__global__ void __launch_bounds__(kJoinThreads) paged_few_join_kernel(const PagedParams p, const FewArgs a) {
  extern __shared__ float join_smem[];
  float(*weight)[kM] = reinterpret_cast<float(*)[kM]>(join_smem);
  float(*part_sum)[kM] = weight + kFewMaxCtas;
  __shared__ float most[kM], total[kM];
  __shared__ float4 sums[kJoinThreads];
  pdl_wait();
  pdl_trigger();
  const int c0 = blockIdx.x;
  FewShared it;
  it.pieces = __ldcg(&a.shared[c0].pieces);
  it.row0 = __ldcg(&a.shared[c0].row0);
  it.n = __ldcg(&a.shared[c0].n);
  it.h = __ldcg(&a.shared[c0].h);
  it.tile = __ldcg(&a.shared[c0].tile);
  const int pieces = it.pieces;
  if (pieces == 0) return;
  PagedSeq s;
  s.row0 = it.row0;
  s.n = it.n;
  auto slot = [&](int k) { return 2 * (int64_t)(c0 + k) + (k == 0 ? 1 : 0); };
  const int rows = (int)min((int64_t)kM, (int64_t)s.n * p.G - (int64_t)it.tile * kM);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // this block's share of the item's output, four elements each: [from, from + outputs)
  const int all = rows * (D / 4), share = (all + gridDim.y - 1) / gridDim.y, from = blockIdx.y * share;
  const int outputs = min(share, all - from);
  if (outputs <= 0) return;
  const int groups = kJoinThreads / outputs;                // (a share has at most kJoinShare)
  const int group = threadIdx.x / outputs, n = from + threadIdx.x % outputs;
  // the first pieces of this thread's first output are on their way while the weights are worked out
  constexpr int kAhead = 8;
  float4 ahead[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    const int k = group + i * groups;
    ahead[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (group < groups && k < pieces)
      ahead[i] = __ldcg(reinterpret_cast<const float4*>(a.part + (slot(k) * kM + n / (D / 4)) * D + n % (D / 4) * 4));
  }
  // ---- weights of the pieces
  for (int i = threadIdx.x; i < pieces * rows; i += kJoinThreads) {
    const int k = i / rows, r = i - k * rows;
    const float2 ml = __ldcg(a.part_ml + slot(k) * kM + r);
    weight[k][r] = ml.x;
    part_sum[k][r] = ml.y;
  }
  __syncthreads();
  for (int r = warp; r < rows; r += kJoinThreads / 32) {
    float mx = -INFINITY;
    for (int k = lane; k < pieces; k += 32) mx = fmaxf(mx, weight[k][r]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    float sum = 0.f;
    for (int k = lane; k < pieces; k += 32) {
      const float x = weight[k][r], f = x == -INFINITY ? 0.f : exp2f(x - mx);
      weight[k][r] = f;
      if (f != 0.f) sum += f * part_sum[k][r];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) { most[r] = mx; total[r] = sum; }
  }
  __syncthreads();
  const int r = n / (D / 4), c = n % (D / 4) * 4;
  float x[4] = {0.f, 0.f, 0.f, 0.f};
  // (a piece that saw nothing has no weight; what it holds is no number that counts)
  auto add = [&](float f, const float4& v) {
    if (f == 0.f) return;
    x[0] += f * v.x; x[1] += f * v.y; x[2] += f * v.z; x[3] += f * v.w;
  };
  if (group < groups) {
    int k = group;
#pragma unroll
    for (int i = 0; i < kAhead; ++i, k += groups) add(k < pieces ? weight[k][r] : 0.f, ahead[i]);
#pragma unroll 4
    for (; k < pieces; k += groups) add(weight[k][r], __ldcg(reinterpret_cast<const float4*>(a.part + (slot(k) * kM + r) * D + c)));
  }
  sums[threadIdx.x] = make_float4(x[0], x[1], x[2], x[3]);
  __syncthreads();
  if (group != 0) return;
  for (int k = 1; k < groups; ++k) {
    const float4 v = sums[k * outputs + threadIdx.x];
    x[0] += v.x; x[1] += v.y; x[2] += v.z; x[3] += v.w;
  }
  int64_t token;
  int head, i;
  few_row<kM>(p, s, it.h, it.tile, r, token, head, i);
  const float inv = most[r] == -INFINITY ? 0.f : 1.f / total[r];
  uint2 y;
  y.x = pack2_16<kHalf>(x[0] * inv, x[1] * inv);
  y.y = pack2_16<kHalf>(x[2] * inv, x[3] * inv);
  *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out) + token * p.so_t + head * p.so_h + c) = y;
  if (a.lse != nullptr && c == 0) a.lse[(int64_t)head * p.T + token] = (most[r] + log2f(total[r])) * kLn2;
}

struct FewKernels {
  void (*attend)(const PagedParams, const CUtensorMap, const CUtensorMap, const FewArgs);
  void (*join)(const PagedParams, const FewArgs);
  size_t smem;
  int per_sm;
  bool parts;                              // of the tensor maps
};
template <bool kHalf, int D, int kStore, int kM>
FewKernels few_kernels() {
  using S = FewShape<D, kStore, kM>;
  return FewKernels{paged_few_kernel<kHalf, D, kStore, kM>, paged_few_join_kernel<kHalf, D, kM>, S::kSmem, S::kCtas, S::kParts};
}
template <bool kHalf, int D, int kM>
FewKernels pick_few(int store) {
  return store == MOBA_STORE_SAME ? few_kernels<kHalf, D, MOBA_STORE_SAME, kM>() : store == MOBA_STORE_E4M3 ? few_kernels<kHalf, D, MOBA_STORE_E4M3, kM>()
                                                                                 : few_kernels<kHalf, D, MOBA_STORE_INT8, kM>();
}
template <bool kHalf, int kM>
FewKernels pick_few_dim(int D, int store) {
  return D == 64 ? pick_few<kHalf, 64, kM>(store) : D == 96 ? pick_few<kHalf, 96, kM>(store) : D == 128 ? pick_few<kHalf, 128, kM>(store)
                                                                                                       : pick_few<kHalf, 256, kM>(store);
}


constexpr size_t kSharedBytes = (kFewMaxCtas * sizeof(FewShared) + 255) / 256 * 256;

}  // namespace

size_t paged_few_workspace(const PagedParams& p) { return kSharedBytes + (size_t)2 * kFewMaxCtas * 16 * (p.D * sizeof(float) + sizeof(float2)); }

cudaError_t launch_paged_few(const PagedParams& all, const void* q, const void* kp, const void* vp, const uint8_t* ks,
                             const uint8_t* vs, void* out, float* lse, void* workspace, cudaStream_t st) {
  const bool eight = (int64_t)all.max_new * all.G <= 8;
  const int tile_rows = eight ? 8 : 16;
  const FewKernels k = all.fp16 ? (eight ? pick_few_dim<true, 8>(all.D, all.store) : pick_few_dim<true, 16>(all.D, all.store))
                                : (eight ? pick_few_dim<false, 8>(all.D, all.store) : pick_few_dim<false, 16>(all.D, all.store));
  FewArgs a{q, kp, vp, ks, vs, out, lse, nullptr, nullptr, nullptr};
  a.shared = static_cast<FewShared*>(workspace);
  a.part_ml = reinterpret_cast<float2*>(static_cast<char*>(workspace) + kSharedBytes);
  a.part = reinterpret_cast<float*>(a.part_ml + 2 * kFewMaxCtas * 16);
  const int slots = 1 << all.page_shift, box = all.store == MOBA_STORE_SAME || slots < 32 ? 16 : 32;
  const int elem = all.store != MOBA_STORE_SAME ? 1 : all.fp16 ? 2 : 3;
  CUtensorMap mk, mv;
  const bool ok = k.parts ? make_page_parts_map(&mk, elem, all.D / 64, kp, all.pages, slots, all.Hkv, all.kp_p, all.kp_t, all.kp_h, box) &&
                                make_page_parts_map(&mv, elem, all.D / 64, vp, all.pages, slots, all.Hkv, all.vp_p, all.vp_t, all.vp_h, box)
                          : make_page_map(&mk, elem, all.D, kp, all.pages, slots, all.Hkv, all.kp_p, all.kp_t, all.kp_h, box) &&
                                make_page_map(&mv, elem, all.D, vp, all.pages, slots, all.Hkv, all.vp_p, all.vp_t, all.vp_h, box);
  if (!ok)
    return cudaErrorNotSupported;
  cudaError_t e = prepare_kernel(k.attend, k.smem, nullptr, true);
  if (e != cudaSuccess) return e;
  if ((e = prepare_kernel(k.join, 2 * kFewMaxCtas * tile_rows * sizeof(float))) != cudaSuccess) return e;
  const int sms = device_info().sms;
  const int grid = k.per_sm * sms < kFewMaxCtas ? k.per_sm * sms : kFewMaxCtas;
  for (int b = 0; b < all.B; b += kPagedBatch) {
    PagedParams p = all;
    p.B = all.B - b < kPagedBatch ? all.B - b : kPagedBatch;
    p.cu += b;
    p.lens += b;
    p.table += b * all.table_stride;
    if ((e = launch_pdl(k.attend, dim3(grid), kFewThreads, k.smem, st, p, mk, mv, a)) != cudaSuccess) return e;
    if ((e = launch_pdl(k.join, dim3(grid, (tile_rows * (all.D / 4) + kJoinShare - 1) / kJoinShare), kJoinThreads, 2 * kFewMaxCtas * tile_rows * sizeof(float), st, p, a)) != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace moba
