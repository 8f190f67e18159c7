// Attention over pages for sequences with many new tokens (blocks of a prompt, whole prompts), on tcgen05 / TMEM / TMA.
//
// Rows of an item are the (new token, query head) pairs of one sequence and kv head, token by token, 256 at a time (two 128-row MMA tiles, "A"
// and "B"): all query heads of a group share one stream of K and V.  An item is such rows against a piece of the sequence's keys, in
// tiles of 128.
//   - 16-bit pages: TMA copies the pages of a tile straight into the swizzled operand tiles, one box for each page (or 128 slots of
//     one).  Warp 0 brings K, warp 3 V.  What lies behind the sequence's end in its last page, or where a page is missing, may be
//     anything: scores there are masked, and those rows of V are overwritten with zeros before the tensor core sees them (0 * NaN).
//   - 8-bit pages: eight warps (3, and 12-18) read the codes, multiply by the row's power of two (exact: see moba_b200.h) and store the operand
//     tiles in the rows' 16-bit type; from there on nothing differs, and no pass over the cache writes it out in 16 bits.  They run through one
//     stream of tiles, without a barrier at an item's end; warp 0 tells them where the codes are.  All 19 warps live with 96 registers,
//     which is what bounds this form: the softmax reads its scores twice, 16 at a time (with 32 at a time its loop kept values in
//     local memory, in an L1 of the few KB that shared memory leaves, and each look at them went to L2; 4 to 8 bytes are spilled now, 48 at
//     head dim 96, and 16 bytes by the form for 16-bit pages).
//   - An item of at most 128 rows (drafted tokens, a small group) has them in both row tiles: A takes every other key tile, B the ones between,
//     each with its own output, and the two are joined at the end.  One softmax at a time left the copies waiting.
//   - Pieces: a first kernel (one CTA) adds up the work of the batch and picks how many pieces an item is cut into, so that
//     the waves of items on the SMs are full; pieces of a sequence and kv head lie next to one another in the order in which CTAs draw
//     them, row tiles fastest, so that those that run together read the same K and V and find them in L2.  Cut items
//     leave {output, maximum, sum} in fp32 for a last kernel, a warp for each row, which joins them in order of the keys: the same bits every
//     time, whichever CTA did what.
// Roles, tensor memory and the order of MMAs are those of the dense stage of the prefill (attend_tc5.cu): warps 4-7 and 8-11 the
// softmax of tiles A and B, a thread a row; warp 1 issues QK_A(j+1) | PV_B(j) | QK_B(j+1) | PV_A(j+1) ...; warp 2 draws and resolves the
// item after this one.  P is rounded to the rows' type before P.V; scores, sums and the output are fp32.
// Measured (replayed from a graph; 32/8 heads, head dim 128 unless said otherwise; in brackets the products at the measured bf16 rate):
//   700 tokens behind 50021                              527 us, 1095 TFLOP/s [351 us]: 3300 cycles a tile and SM against 2048 of its MMAs
//   2048 behind 30720, e4m3                              7.1 ms (mma.sync) -> 3.1 (four warps for codes) -> 2.0 (eight) -> 1.66 (one stream of tiles)
//                                                        -> 1.28 (next to nothing in local memory), 830 TFLOP/s [648 us]: 4600 cycles a tile
//   prompts of 1023, 4096 and 200, 16 heads, head dim 256   3.8 ms (mma.sync) -> 0.22 [89 us]
//   4 tokens of 16 requests of 8000 over 8 kv heads      127 us (one row tile at work) -> 95 (both, key tiles by turns) [80 us of bytes]
#include "attend_rows.cuh"
#include "fast_div.cuh"
#include "paged.cuh"
#include "sm100_ptx.cuh"

namespace moba {

bool make_page_map(CUtensorMap* m, int elem, int D, const void* base, int pages, int slots, int H, int64_t sp, int64_t st, int64_t sh,
                   int box_rows);

namespace {

// Head dim 256 has one row tile an item; its K, V and Q are handled in halves of 128 dims, which take the places of the two stages and of the two
// row tiles: S = Q_lo.K_lo^T + Q_hi.K_hi^T in one of two accumulators, O_lo += P.V_lo and O_hi += P.V_hi.
constexpr int kMostRows = 2 * kTileM;
__host__ __device__ constexpr int item_rows(int D) { return D == 256 ? kTileM : kMostRows; }
constexpr int kCodeWarps = 8;              // that turn codes into operand tiles: warp 3, which has no V to bring, and warps 12-18
template <int kStore> constexpr int kRowsThreads = kStore == MOBA_STORE_SAME ? 384 : 384 + 32 * (kCodeWarps - 1);
// Results of pieces that the workspace has room for at most (158 MB at head dim 128): with half of them 256 items could not be cut into the four
// pieces each that fill the waves.
constexpr int kMostSlots = 8 * 148;
constexpr int kLeastPiece = 4;             // key tiles
// ... and those that a launch can come to: its row tiles, each in as many pieces as the table has room for.  (Sequences that overlap, which no
// call has, might ask for more: the plan does not go beyond it.)
int rows_slots(const PagedParams& p) {
  const int64_t keys = ((int64_t)p.per_seq << p.page_shift), cuts = ((keys + kBN - 1) / kBN + kLeastPiece - 1) / kLeastPiece;
  if (cuts < 2) return 0;
  const int64_t tiles = p.T * p.G / item_rows(p.D) + (p.T < p.B ? p.T : p.B);
  return (int)(tiles * p.Hkv >= kMostSlots ? kMostSlots : tiles * p.Hkv * cuts < kMostSlots ? tiles * p.Hkv * cuts : kMostSlots);
}
constexpr float kLn2 = 0.6931471805599453f;

// ---- the plan ------------------------------------------------------------------
// In the workspace, one for each launch.
struct RowsPlan {
  int32_t counter, status;                 // items drawn; a bounded wait gave up
  int32_t items;
  int32_t pad;
  int32_t begin[kPagedBatch + 1];          // first item of a sequence
  int32_t slot0[kPagedBatch];              // first result slot of a sequence whose items are cut
  int32_t piece[kPagedBatch];              // key tiles of a piece
};

__device__ __forceinline__ int rows_tiles(const PagedParams& p, int n) {
  const int rows = item_rows(p.D);
  return (int)(((int64_t)n * p.G + rows - 1) / rows);
}
// Keys that the rows of tile t see at most, and their tiles.
__device__ __forceinline__ int rows_end(const PagedParams& p, const PagedSeq& s, int t) {
  const int64_t last = min((int64_t)s.n - 1, ((int64_t)(t + 1) * item_rows(p.D) - 1) / p.G);
  return (int)min(max((int64_t)s.pos0 + last + 1, (int64_t)0), (int64_t)s.len);
}
// (an item without a key has one tile, all masked: its rows are written as zeros)
__device__ __forceinline__ int key_tiles(int keys) { return max((keys + kBN - 1) / kBN, 1); }

// What an item costs besides its key tiles (its Q rows, the first and the last tile's latency, its output), in tiles.
constexpr float kItemCost = 3.f;

// Tiles of a piece when `tiles` are cut into as many as pieces of `piece` make, evenly (there may be one piece fewer then).
__device__ __forceinline__ int even_piece(int tiles, int piece) {
  const int cuts = (tiles + piece - 1) / piece;
  return (tiles + cuts - 1) / cuts;
}

// Candidate k cuts the batch into about k / 4 pieces a CTA, candidate 0 not at all.  With equal pieces the time is that of the waves;
// longer ones than the average may come last.
__global__ void __launch_bounds__(1024) paged_plan_kernel(const PagedParams p, RowsPlan* plan, int sms, int most_slots) {
  __shared__ int rows_s[kPagedBatch], most_s[kPagedBatch], least_s[kPagedBatch];
  __shared__ float cost_s[32];
  __shared__ int piece_s[32];
  __shared__ int scan_s[2][32];
  pdl_wait();
  pdl_trigger();
  const int b = threadIdx.x, warp = b >> 5, lane = b & 31;
  int rows = 0, most = 1, least = 1;
  if (b < p.B) {
    const PagedSeq s = paged_seq(p, b);
    const int tiles = rows_tiles(p, s.n);
    rows = tiles * p.Hkv;
    if (tiles > 0) {
      most = key_tiles(rows_end(p, s, tiles - 1));
      least = key_tiles(rows_end(p, s, 0));
    }
  }
  rows_s[b] = rows;
  most_s[b] = most;
  least_s[b] = least;
  __syncthreads();
  // every warp: the work of the batch, then its own candidate
  float work = 0.f;
  int longest = 1;
  for (int i = lane; i < p.B; i += 32) {
    if (rows_s[i] == 0) continue;
    work += 0.5f * (float)rows_s[i] * (float)(most_s[i] + least_s[i]);
    longest = max(longest, most_s[i]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) work += __shfl_xor_sync(0xffffffffu, work, o);
  longest = __reduce_max_sync(0xffffffffu, longest);
  const int piece = warp == 0 ? longest : max((int)ceilf(4.f * work / (float)(sms * warp)), kLeastPiece);
  float items = 0.f;
  int slots = 0, top = 1;
  for (int i = lane; i < p.B; i += 32) {
    if (rows_s[i] == 0) continue;
    const int even = even_piece(most_s[i], piece), cuts = (most_s[i] + even - 1) / even;
    items += 0.5f * (float)rows_s[i] * (float)(cuts + (least_s[i] + even - 1) / even);
    if (cuts > 1) slots += (int)min((int64_t)rows_s[i] * cuts, (int64_t)(1 << 20));
    top = max(top, even);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) items += __shfl_xor_sync(0xffffffffu, items, o);
  slots = __reduce_add_sync(0xffffffffu, min(slots, 1 << 25));
  top = __reduce_max_sync(0xffffffffu, top);
  if (lane == 0) {
    const float average = work / fmaxf(items, 1.f);
    const float cost = ceilf(items / (float)sms) * (average + kItemCost) + 0.5f * fmaxf((float)top - average, 0.f);
    cost_s[warp] = slots > most_slots ? INFINITY : cost;
    piece_s[warp] = piece;
  }
  __syncthreads();
  // every warp for itself: the cheapest, of equal ones the first (costs are not negative: they compare as integers)
  const uint32_t mine = __float_as_uint(cost_s[lane]);
  const int best = piece_s[__ffs(__ballot_sync(0xffffffffu, mine == __reduce_min_sync(0xffffffffu, mine))) - 1];
  // first items and slots of the sequences
  const int even = even_piece(most, best), cuts = (most + even - 1) / even;
  const int n = rows * cuts, m = cuts > 1 ? n : 0;
  int x = n, y = m;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, x, o), v = __shfl_up_sync(0xffffffffu, y, o);
    if (lane >= o) { x += u; y += v; }
  }
  if (lane == 31) { scan_s[0][warp] = x; scan_s[1][warp] = y; }
  __syncthreads();
  const int bx = __reduce_add_sync(0xffffffffu, lane < warp ? scan_s[0][lane] : 0);
  const int by = __reduce_add_sync(0xffffffffu, lane < warp ? scan_s[1][lane] : 0);
  if (b < p.B) {
    plan->begin[b] = bx + x - n;
    plan->slot0[b] = m > 0 ? by + y - m : -1;
    plan->piece[b] = even;
    if (b == p.B - 1) {
      plan->begin[p.B] = bx + x;
      plan->items = bx + x;
      plan->counter = 0;
      plan->status = 0;
    }
  }
}

// ---- items ---------------------------------------------------------------------
struct RowsItem {
  int b, h, tile;                          // sequence, kv head, row tile
  int nrows;
  int j0, ntiles;                          // key tiles [j0, j0 + ntiles) of the sequence
  int row0, pos0, len;                     // the sequence's (PagedSeq)
  int slot;                                // of its results; -1: not cut
};

// Where the codes of a key tile lie: for its eight groups of 16 keys, which have a page each.
struct TileInfo {
  int64_t k[8], v[8], scale[8];            // offsets in the pools; k < 0: no page
  int32_t keys;                            // of the tile in the sequence; 0: there are no more tiles
  uint32_t there;
};
constexpr int kInfoSlots = 4;

struct RowsCtrl {
  uint64_t info_full[kInfoSlots], info_empty[kInfoSlots];
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], v_raw;
  uint64_t s_full[2], p_full[2], o_full[2];
  uint64_t item_ready[2];
  uint32_t tmem_slot;
  volatile int32_t abort;
  int32_t items;
  RowsItem item[2];
  int32_t done[2];
  uint32_t there[4];                       // [key tile mod 4]: which groups of 16 keys have a page
  int64_t qoff[2][kMostRows], ooff[2][kMostRows];   // of a row in q and out; -1: no row
  float2 pair_ml[2][kTileM];               // {maximum, sum} of a row in tiles A and B, where both have it
  float row_inv[kTileM];                   // head dim 256: the row's factor (0: nothing is seen), for the warps that write the second half of O
  TileInfo info[kInfoSlots];
};
constexpr size_t kRowsSmem = 1024 + 6 * kTileBytes + sizeof(RowsCtrl);
static_assert(kRowsSmem <= 232448, "shared memory of one CTA");

struct RowsArgs {
  const __nv_bfloat16* q;
  const uint8_t *kp, *vp, *ks, *vs;        // pools as bytes
  __nv_bfloat16* out;
  float* lse;
  RowsPlan* plan;
  float* part;                             // [slots][rows of an item][D]
  float2* part_ml;                         // the same rows: {maximum, sum}
  FastDiv by_group;
};

// Items that are not cut come longest first, all heads by turns, where the K and V of all heads stay in L2 together; otherwise head by head, so that
// the last head's long items may come late (prompts of 1023, 4096 and 200 tokens, 16 heads of 256: 228 us head by head, 190 by turns).
constexpr int64_t kAllHeadsBytes = (int64_t)80 << 20;

// Both row tiles have the item's rows, and the key tiles by turns.
__device__ __forceinline__ bool rows_twice(int D, const RowsItem& it) { return D != 256 && it.nrows <= kTileM; }

// Warp 2, one item ahead of the others.
__device__ __forceinline__ void rows_prefetch(const PagedParams& p, const RowsArgs& a, RowsCtrl& c, int at) {
  const int lane = threadIdx.x & 31;
  RowsItem it;
  bool done = false;
  for (;;) {
    int idx = 0;
    if (lane == 0) idx = c.abort ? 0x7fffffff : atomicAdd(&a.plan->counter, 1);
    idx = __shfl_sync(0xffffffffu, idx, 0);
    if (idx >= c.items) { done = true; break; }
    it.b = search_warp(p.B, idx, [&](int k) { return __ldcg(a.plan->begin + k); });
    const PagedSeq s = paged_seq(p, it.b);
    const int tiles = rows_tiles(p, s.n), piece = __ldcg(a.plan->piece + it.b);
    const int most = key_tiles(rows_end(p, s, tiles - 1)), cuts = (most + piece - 1) / piece;
    const int i = idx - __ldcg(a.plan->begin + it.b);      // kv head, piece, row tile, the last one first
    int cut = 0;
    if (cuts == 1 && (int64_t)s.len * p.Hkv * p.D * 4 <= kAllHeadsBytes) {
      it.tile = tiles - 1 - i / p.Hkv;
      it.h = i % p.Hkv;
    } else {
      const int hc = i / tiles;
      it.tile = tiles - 1 - (i - hc * tiles);
      it.h = hc / cuts;
      cut = hc - it.h * cuts;
    }
    it.j0 = cut * piece;
    it.ntiles = min(key_tiles(rows_end(p, s, it.tile)) - it.j0, piece);
    if (it.ntiles <= 0) continue;
    const int rows = item_rows(p.D);
    it.nrows = (int)min((int64_t)s.n * p.G - (int64_t)it.tile * rows, (int64_t)rows);
    it.row0 = s.row0;
    it.pos0 = s.pos0;
    it.len = s.len;
    it.slot = cuts > 1 ? __ldcg(a.plan->slot0 + it.b) + i : -1;
    break;
  }
  if (lane == 0) { c.item[at] = it; c.done[at] = done; }
  if (!done) {
#pragma unroll
    for (int u = 0; u < kMostRows / 32; ++u) {
      const int r = lane + 32 * u;
      int64_t qo = -1, oo = -1;
      const int rt = rows_twice(p.D, it) ? r & (kTileM - 1) : r;
      if (rt < it.nrows) {
        const int row = it.tile * item_rows(p.D) + rt, i = row / a.by_group, head = it.h * p.G + row - i * p.G;
        const int64_t token = (int64_t)it.row0 + i;
        qo = token * p.sq_t + (int64_t)head * p.sq_h;
        oo = token * p.so_t + (int64_t)head * p.so_h;
        asm volatile("prefetch.global.L2 [%0];" ::"l"(a.q + qo));
        if (p.D > 64) asm volatile("prefetch.global.L2 [%0];" ::"l"(a.q + qo + 64));
        if (p.D > 128) {
          asm volatile("prefetch.global.L2 [%0];" ::"l"(a.q + qo + 128));
          asm volatile("prefetch.global.L2 [%0];" ::"l"(a.q + qo + 192));
        }
      }
      c.qoff[at][r] = qo;
      c.ooff[at][r] = oo;
    }
  }
  __syncwarp();
  if (lane == 0) mbar_arrive(smem_u32(&c.item_ready[at]));
}

__device__ __forceinline__ void rows_pair_barrier() { asm volatile("bar.sync 2, 256;" ::: "memory"); }   // warps 4-11
// The warps that go item by item: all but those that turn codes into tiles.
template <bool kCodes>
__device__ __forceinline__ void rows_barrier() { asm volatile("bar.sync 1, %0;" ::"n"(kCodes ? 352 : 384) : "memory"); }
// The item of slot `at` begins; the softmax warps copy its Q rows into the swizzled tiles.  False: there is none.
template <bool kGather, int D, bool kCodes>
__device__ __forceinline__ bool rows_next(const RowsArgs& a, const RowsCtrl& c, unsigned char* smem, int at) {
  rows_barrier<kCodes>();
  if (c.done[at]) return false;
  if (kGather) {
    constexpr int kChunks = D / 8;
    constexpr int kPieces = item_rows(D) * kChunks / 256;
    const int t = threadIdx.x - 128;
    uint4 val[kPieces];
#pragma unroll
    for (int u = 0; u < kPieces; ++u) {
      const int i = t + u * 256;
      const int r = i / kChunks, ch = i % kChunks;
      const int64_t off = c.qoff[at][r];
      val[u] = make_uint4(0, 0, 0, 0);
      if (off >= 0) val[u] = __ldg(reinterpret_cast<const uint4*>(a.q + off + ch * 8));
    }
#pragma unroll
    for (int u = 0; u < kPieces; ++u) {
      const int i = t + u * 256;
      const int r = i / kChunks, ch = i % kChunks;
      // row tile, or half of the dims
      const int tile = D == 256 ? ch >> 4 : r >> 7;
      const uint32_t dst = (uint32_t)(tile * kTileBytes + ((ch >> 3) & 1) * kHalfBytes + (r & 127) * 128 + (((ch & 7) ^ (r & 7)) << 4));
      *reinterpret_cast<uint4*>(smem + dst) = val[u];
    }
  }
  fence_proxy_async_smem();
  rows_barrier<kCodes>();
  return true;
}

// ---- codes -> operand tiles ------------------------------------------------------
// Four codes and the row's byte -> four elements.  `byte` may be anything here.
template <bool kHalf, int kStore>
__device__ __noinline__ uint2 decode4_any(uint32_t w, uint32_t byte) {
  const float s = paged_scale(byte);
  float f[4];
  if (kStore == MOBA_STORE_E4M3) {
    uint32_t lo, hi;
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
    const float2 x = unpack2<true>(lo), y = unpack2<true>(hi);
    f[0] = x.x; f[1] = x.y; f[2] = y.x; f[3] = y.y;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = (float)(int8_t)(w >> (8 * i));
  }
  return make_uint2(pack2_16<kHalf>(f[0] * s, f[1] * s), pack2_16<kHalf>(f[2] * s, f[3] * s));
}
__device__ __forceinline__ uint32_t mul2_bf16(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t sub2_bf16(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t mul2_f16(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t sub2_f16(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// The factor that the quick way multiplies by: a float, or both halves of a word; 0 where the type has none.
template <bool kHalf, int kStore>
__device__ __forceinline__ uint32_t quick_factor(uint32_t byte) {
  if (!kHalf && kStore == MOBA_STORE_E4M3) return byte << 23;
  const uint32_t f = !kHalf ? byte << 7 : byte >= 113 && byte <= 142 ? (byte - 112) << 10 : 0;
  return f | f << 16;
}
template <bool kHalf, int kStore>
__device__ __forceinline__ uint2 decode4_quick(uint32_t w, uint32_t factor) {
  uint32_t lo, hi;
  if (kHalf && kStore == MOBA_STORE_E4M3) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
    return make_uint2(mul2_f16(lo, factor), mul2_f16(hi, factor));
  }
  if (kHalf) {                             // 1024 + (code + 128) - 1152
    const uint32_t u = w ^ 0x80808080u;
    lo = sub2_f16(__byte_perm(u, 0x64u, 0x4140), 0x64806480u);
    hi = sub2_f16(__byte_perm(u, 0x64u, 0x4342), 0x64806480u);
    return make_uint2(mul2_f16(lo, factor), mul2_f16(hi, factor));
  }
  if (kStore == MOBA_STORE_E4M3) {
    // through fp16 and fp32: two of five instructions for two elements are the integer unit's, which the softmax needs too (moving sign,
    // exponent and mantissa to their places in bf16 takes four there)
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
    const float2 x = unpack2<true>(lo), y = unpack2<true>(hi);
    const float f = __uint_as_float(factor);
    const uint64_t f2 = pack2(f, f), u = mul2(pack2(x.x, x.y), f2), v = mul2(pack2(y.x, y.y), f2);
    return make_uint2(pack2_16<false>(lo2(u), hi2(u)), pack2_16<false>(lo2(v), hi2(v)));
  }
  // code = (128 + its low seven bits) - (128, or 256 with the sign bit set)
  const uint32_t a = __byte_perm(w, 0x43u, 0x4140), b = __byte_perm(w, 0x43u, 0x4342);
  lo = sub2_bf16(a & 0xff7fff7fu, (a & 0x00800080u) | 0x43004300u);
  hi = sub2_bf16(b & 0xff7fff7fu, (b & 0x00800080u) | 0x43004300u);
  return make_uint2(mul2_bf16(lo, factor), mul2_bf16(hi, factor));
}

// A tile of codes on its way.  A warp has one group of 16 keys; a lane's pieces of 16 codes are of rows r and r + 8 with r = lane % 8, so that
// eight lanes in a row store to different banks.
template <int D> constexpr int kRawPieces = D / 32;
template <int D> struct RawTile {
  uint4 code[kRawPieces<D>];
  uint32_t byte[2];                        // of rows r and r + 8
};
// Row (0: r, 1: r + 8) and piece of the row of a lane's piece i.
template <int D> __device__ __forceinline__ int raw_row(int i, int lane) { return ((lane >> 3) + 4 * i) / (D / 16); }
template <int D> __device__ __forceinline__ int raw_piece(int i, int lane) { return ((lane >> 3) + 4 * i) % (D / 16); }

// (past L1, which is what shared memory leaves of it: values that the compiler keeps there would go with every tile)
__device__ __forceinline__ uint4 load_codes(const uint8_t* at) {
  uint4 x;
  asm volatile("ld.global.nc.L1::no_allocate.L2::128B.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "l"(at));
  return x;
}
template <int D>
__device__ __forceinline__ void raw_load(const uint8_t* pool, const uint8_t* scales, int64_t at, int64_t scale, int64_t st, int keys,
                                         int lane, RawTile<D>& raw) {
  const int r = lane & 7;
#pragma unroll
  for (int i = 0; i < kRawPieces<D>; ++i) raw.code[i] = make_uint4(0, 0, 0, 0);
  raw.byte[0] = raw.byte[1] = 127;
  if (at < 0 || keys <= 0) return;                          // (the warp as one)
  const uint8_t* from = pool + at + r * st;
#pragma unroll
  for (int i = 0; i < kRawPieces<D>; ++i) {
    const int up = raw_row<D>(i, lane);
    if (r + 8 * up < keys) raw.code[i] = load_codes(from + (up ? 8 * st : 0) + 16 * raw_piece<D>(i, lane));
  }
#pragma unroll
  for (int u = 0; u < 2; ++u)
    if (r + 8 * u < keys) raw.byte[u] = __ldg(scales + scale + r + 8 * u);
}
// `dst`: the operand tile's first row of the warp's group.
template <bool kHalf, int D, int kStore>
__device__ __forceinline__ void raw_store(const RawTile<D>& raw, uint32_t dst, int lane) {
  const uint32_t f0 = quick_factor<kHalf, kStore>(raw.byte[0]), f1 = quick_factor<kHalf, kStore>(raw.byte[1]);
  const int r = lane & 7;
  const bool quick = __all_sync(0xffffffffu, f0 != 0 && f1 != 0);
#pragma unroll
  for (int i = 0; i < kRawPieces<D>; ++i) {
    const int up = raw_row<D>(i, lane), c = raw_piece<D>(i, lane);
    const uint32_t w[4] = {raw.code[i].x, raw.code[i].y, raw.code[i].z, raw.code[i].w};
    uint2 y[4];
    if (quick) {
#pragma unroll
      for (int u = 0; u < 4; ++u) y[u] = decode4_quick<kHalf, kStore>(w[u], up ? f1 : f0);
    } else {
#pragma unroll
      for (int u = 0; u < 4; ++u) y[u] = decode4_any<kHalf, kStore>(w[u], raw.byte[up]);
    }
    // pieces 2c and 2c + 1 of the row in 16 bits
    const uint32_t at = dst + (uint32_t)((c >> 2) * kHalfBytes + (r + 8 * up) * 128 + ((((2 * c) & 7) ^ r) << 4));
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(y[0].x), "r"(y[0].y), "r"(y[1].x), "r"(y[1].y) : "memory");
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at ^ 16u), "r"(y[2].x), "r"(y[2].y), "r"(y[3].x), "r"(y[3].y) : "memory");
  }
}

// ---- softmax ---------------------------------------------------------------------
// Reference of a row's weights: a score, and the score in powers of two.  A weight is 2^(score * factor - ref); where scores are so large that
// the rounding of `ref` would be powers of two itself (kLarge), it is 2^((score - raw) * factor).
struct RowRef { float raw, ref, l; };
constexpr float kLarge = 1048576.f;

// One step of one row: S (128 fp32 columns of this thread's lane) -> P over its first 64, running reference and sum.
// As softmax_row of attend_tc5.cu, but for rows that have seen nothing yet (no reference: weights are 0), and with exponentials of masked tiles by the
// special-function unit alone, which makes them exactly 0 where nothing is seen.  kTwice: the scores are read twice, 16 at a time, for
// launches whose threads have fewer registers.  !kMasked returns false, with nothing done, where a score is large: the
// other form then takes the tile.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
                 "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
// `quiet` runs (the warp as one) before O is touched: where the P.V of the tile before may still be executing it waits for that.
template <bool kMasked, bool kHalf, int D, bool kTwice, typename F>
__device__ __forceinline__ bool rows_softmax(uint32_t tS, uint32_t tO, bool first, int rem, uint32_t there, float sl2, RowRef& row, F&& quiet) {
  constexpr int kW = kTwice ? 16 : 128, kP = kTwice ? 8 : 16;   // columns, and words of P, at a time
  uint32_t v[kTwice ? 2 : 1][kW];
  // runs `step(columns, first column)` over the scores; twice as it says: 16 columns travel while the 16 before them are worked on
  auto mask = [&](uint32_t (&x)[kW], int at) {
    if (kMasked) {
#pragma unroll
      for (int i = 0; i < kW; ++i) {
        const int seen = (there >> ((at + i) >> 4)) & 1 ? rem : 0;
        x[i] = at + i < seen ? x[i] : 0xff800000u;          // -inf
      }
    }
  };
  auto over = [&](auto&& step) {
    if constexpr (kTwice) {
      tmem_ld16(tS, v[0]);
#pragma unroll 1
      for (int at = 0; at < 128; at += 32) {                // (a loop: the code of the two roles is fetched all the time)
        tmem_wait_ld();
        tmem_ld16(tS + at + 16, v[1]);
        mask(v[0], at);
        step(v[0], at);
        tmem_wait_ld();
        if (at < 96) tmem_ld16(tS + at + 32, v[0]);
        mask(v[1], at + 16);
        step(v[1], at + 16);
      }
    } else {
      step(v[0], 0);
    }
  };
  if constexpr (!kTwice) {
    tmem_ld128(tS, v[0]);
    tmem_wait_ld();
    mask(v[0], 0);
  }
  float mx0 = -INFINITY, mx1 = -INFINITY, mx2 = -INFINITY, mx3 = -INFINITY;
  over([&](uint32_t (&x)[kW], int) {
#pragma unroll
    for (int i = 0; i < kW; i += 8) {
      mx0 = max3(mx0, __uint_as_float(x[i]), __uint_as_float(x[i + 1]));
      mx1 = max3(mx1, __uint_as_float(x[i + 2]), __uint_as_float(x[i + 3]));
      mx2 = max3(mx2, __uint_as_float(x[i + 4]), __uint_as_float(x[i + 5]));
      mx3 = max3(mx3, __uint_as_float(x[i + 6]), __uint_as_float(x[i + 7]));
    }
  });
  const float raw = fmaxf(row.raw, fmaxf(fmaxf(mx0, mx1), fmaxf(mx2, mx3))), ref = raw * sl2;
  // (a row whose reference is large has it from a tile of the other form, and rises from there)
  if (!kMasked && __any_sync(0xffffffffu, fabsf(ref) > kLarge)) return false;
  const bool up = ref > row.ref + 8.f;
  if (__any_sync(0xffffffffu, up)) {
    float alpha = up ? ex2_approx(row.ref - ref) : 1.f;
    if (kMasked && up && fabsf(ref) > kLarge) alpha = ex2_approx((row.raw - raw) * sl2);
    if (!first) {
      quiet();
      uint32_t o[32];
#pragma unroll 1
      for (int ch = 0; ch < D / 32; ++ch) {
        tmem_ld32(tO + ch * 32, o);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
        tmem_st32(tO + ch * 32, o);
      }
    }
    row.l *= alpha;
    if (up) { row.raw = raw; row.ref = ref; }
  }
  const bool large = kMasked && fabsf(row.ref) > kLarge, none = row.ref == -INFINITY;
  const float neg = none || large ? 0.f : -row.ref, base = none || !large ? 0.f : row.raw;
  const uint64_t scale2 = pack2(sl2, sl2), negm2 = pack2(neg, neg), base2 = pack2(base, base);
  uint64_t sum_a = 0, sum_b = 0;
  over([&](uint32_t (&y)[kW], int at) {
#pragma unroll
    for (int ch = 0; ch < kW / (2 * kP); ++ch) {
      uint32_t pk[kP];
#pragma unroll
      for (int i = 0; i < kP; ++i) {
        const int e = ch * 2 * kP + 2 * i;
        uint64_t x = pack2(__uint_as_float(y[e]), __uint_as_float(y[e + 1]));
        if (kMasked) x = sub2(x, base2);
        x = fma2(x, scale2, negm2);
        const uint64_t pr = !kMasked && (i & 7) < kPolyPairs ? ex2_poly2(x) : pack2(ex2_approx(lo2(x)), ex2_approx(hi2(x)));
        if (i & 1) sum_b = add2(sum_b, pr); else sum_a = add2(sum_a, pr);
        pk[i] = pack2_16<kHalf>(lo2(pr), hi2(pr));
      }
      if constexpr (kTwice) tmem_st8(tS + at / 2 + ch * kP, pk); else tmem_st16(tS + at / 2 + ch * kP, pk);
    }
  });
  const uint64_t sum = add2(sum_a, sum_b);
  row.l += lo2(sum) + hi2(sum);
  tmem_wait_st();
  return true;
}

// D dims (at most 128): S at `d` (+)= the Q tile X . K^T; O at `d` (+)= P . V
template <int X, bool kHalf, int D>
__device__ __forceinline__ void rows_qk(uint32_t d, uint32_t dq, uint32_t dk, bool more = false) {
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) {
    const uint32_t koff = (uint32_t)((ks >> 2) * (kHalfBytes >> 4) + (ks & 3) * 2);
    mma_ss(d, desc64(dq + X * (kTileBytes >> 4) + koff), desc64(dk + koff), kIdescQK<kHalf>, more || ks > 0);
  }
}
template <bool kHalf, int D>
__device__ __forceinline__ void rows_pv(uint32_t d, uint32_t tp, uint32_t dv, bool first) {
#pragma unroll
  for (int ks = 0; ks < 8; ++ks) mma_ts(d, tp + ks * 8, desc64(dv + ks * (2048 >> 4)), kIdescPV<kHalf, D>, (!first) || ks > 0);
}

// Rows of V that nobody may see become zeros: slots behind the sequence's end, and groups without a page.  One warp.
template <int D>
__device__ __forceinline__ void zero_rows(unsigned char* tile, const RowsItem& it, int key0, uint32_t there) {
  const int lane = threadIdx.x & 31;
  for (int r0 = 0; r0 < kBN; r0 += 4) {                     // four rows of eight pieces at a time
    const int r = r0 + (lane >> 3);
    if (key0 + r < it.len && ((there >> (r >> 4)) & 1)) continue;
#pragma unroll
    for (int blk = 0; blk < (D + 63) / 64; ++blk)
      *reinterpret_cast<uint4*>(tile + blk * kHalfBytes + r * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
  }
}

enum { RS_PRODUCER = 1, RS_MMA = 2, RS_SOFTMAX = 3 };

template <bool kHalf, int D, int kStore>
__global__ void __launch_bounds__(kRowsThreads<kStore>, 1)
paged_rows_kernel(const PagedParams p, const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                  const RowsArgs a) {
  constexpr bool kCodes = kStore != MOBA_STORE_SAME;
  constexpr bool kWide = D == 256;
  constexpr int kParts = kWide ? 2 : 1, kPart = D / kParts;   // parts of the dims, each a tile of its own
  constexpr int kBlocks = (kPart + 63) / 64;
  constexpr int kRows = item_rows(D);
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const uint32_t sQ = smem_u32(smem), sK = sQ + 2 * kTileBytes, sV = sK + 2 * kTileBytes;
  RowsCtrl& c = *reinterpret_cast<RowsCtrl*>(smem + 6 * kTileBytes);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&c.k_full[i]), kCodes ? kCodeWarps : 1);
      mbar_init(smem_u32(&c.k_empty[i]), 1);
      mbar_init(smem_u32(&c.v_full[i]), kCodes ? kCodeWarps : 1);
      mbar_init(smem_u32(&c.v_empty[i]), 1);
      mbar_init(smem_u32(&c.s_full[i]), 1);
      mbar_init(smem_u32(&c.p_full[i]), kTileM);
      mbar_init(smem_u32(&c.o_full[i]), 1);
      mbar_init(smem_u32(&c.item_ready[i]), 1);
    }
    mbar_init(smem_u32(&c.v_raw), 1);
    for (int i = 0; i < kInfoSlots; ++i) {
      mbar_init(smem_u32(&c.info_full[i]), 1);
      mbar_init(smem_u32(&c.info_empty[i]), kCodeWarps);
    }
    c.abort = 0;
    fence_barrier_init();
    if (!kCodes) {
      prefetch_tmap(&tmap_k);
      prefetch_tmap(&tmap_v);
    }
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&c.tmem_slot), 512);
    tmem_relinquish();
  }
  pdl_wait();
  pdl_trigger();
  if (threadIdx.x == 0) c.items = __ldcg(&a.plan->items);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = c.tmem_slot;

  if (warp < (kCodes ? 3 : 4)) {
    // ---- warps 0-3: K (TMA, or where its codes are), MMA, items, V (TMA)
    if (!kCodes) setmaxnreg_dec<72>();
    uint32_t kc = 0, vc = 0;               // K / V tiles (of a part of the dims) produced (warps 0, 3) or consumed (warp 1) so far
    uint32_t pph0 = 0, pph1 = 0, raw = 0;
    uint32_t gq = 0, gp = 0;               // head dim 256: tiles whose Q.K^T, whose P.V has been issued
    int pre = 0;                           // tiles of the coming item already requested
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    const uint32_t dq = __shfl_sync(0xffffffffu, desc_lo(sQ, 16), 0);
    const uint32_t dk = __shfl_sync(0xffffffffu, desc_lo(sK, 16), 0);
    const uint32_t dv = __shfl_sync(0xffffffffu, desc_lo(sV, kHalfBytes), 0);
    const uint32_t el = elect_one();
    bool ended = false;
    auto end_tiles = [&] {                                  // warp 0: there are no more tiles of codes
      const uint32_t s = kc % kInfoSlots;
      if (lane == 0 && mbar_wait(smem_u32(&c.info_empty[s]), ((kc / kInfoSlots) & 1) ^ 1)) {
        c.info[s].keys = 0;
        mbar_arrive(smem_u32(&c.info_full[s]));
      }
      __syncwarp();
      ended = true;
    };
    for (int n = 0;; ++n) {
      if (warp == 2) rows_prefetch(p, a, c, n & 1);
      if (!rows_next<false, D, kCodes>(a, c, smem, n & 1)) break;
      const RowsItem& it = c.item[n & 1];
      if (kCodes && warp == 0) {
        // where the tiles' codes are
        auto describe = [&](const RowsItem& w, int j) -> bool {
          const uint32_t s = kc % kInfoSlots;
          const int key0 = (w.j0 + j) * kBN, key = key0 + 16 * lane;
          const int id = lane < 8 && key < w.len ? paged_page(p, w.b, key) : -1;
          const uint32_t there = __ballot_sync(0xffffffffu, id >= 0);
          if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&c.info_empty[s]), ((kc / kInfoSlots) & 1) ^ 1))) return false;
          TileInfo& info = c.info[s];
          if (lane < 8) {
            const int slot = key & ((1 << p.page_shift) - 1);
            info.k[lane] = id >= 0 ? id * p.kp_p + slot * p.kp_t + w.h * p.kp_h : -1;
            info.v[lane] = id >= 0 ? id * p.vp_p + slot * p.vp_t + w.h * p.vp_h : -1;
            info.scale[lane] = (((int64_t)id * p.Hkv + w.h) << p.page_shift) + slot;
          }
          if (lane == 0) {
            info.keys = max(w.len - key0, 1);
            info.there = there;
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&c.info_full[s]));
          ++kc;
          return true;
        };
        bool alive = true;
        for (int j = pre; alive && j < it.ntiles; ++j) alive = describe(it, j);
        pre = 0;
        if (alive) {
          const int s1 = (n + 1) & 1;
          alive = __all_sync(0xffffffffu, mbar_wait(smem_u32(&c.item_ready[s1]), ((n + 1) >> 1) & 1));
          if (alive && !c.done[s1]) {
            const int nt = min(2, c.item[s1].ntiles);
            for (; alive && pre < nt; ++pre) alive = describe(c.item[s1], pre);
          } else if (alive) {
            end_tiles();                                    // (now: the last V tile is turned behind the look for a next one)
          }
        }
        if (!alive && lane == 0) { atomicExch(&a.plan->status, RS_PRODUCER); c.abort = 1; }
      } else if (!kCodes && (warp == 0 || warp == 3)) {
        // a tile's pages: lanes 0 .. boxes - 1 have one each
        const int box_rows = min(1 << p.page_shift, kBN), boxes = kBN / box_rows;
        auto load_tile = [&](const RowsItem& w, int jj) -> bool {
          const int j = jj / kParts, dim0 = jj % kParts * kPart;
          const int key0 = (w.j0 + j) * kBN, key = key0 + lane * box_rows;
          const int id = lane < boxes && key < w.len ? paged_page(p, w.b, key) : -1;
          const uint32_t got = __ballot_sync(0xffffffffu, id >= 0);
          const uint32_t bytes = (uint32_t)(__popc(got) * box_rows * 128 * kBlocks);
          // groups of 16 keys that have a page (boxes of at most 128 rows: 8, 4, 2 or 1 of them)
          const uint32_t there = __ballot_sync(0xffffffffu, lane < 8 && ((got >> (lane * 16 / box_rows)) & 1));
          const uint32_t s = (warp == 0 ? kc : vc) & 1;
          const uint32_t at = (warp == 0 ? sK : sV) + s * kTileBytes + lane * box_rows * 128;
          const int slot = key & ((1 << p.page_shift) - 1);
          if (warp == 0) {
            if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&c.k_empty[s]), ((kc >> 1) & 1) ^ 1))) return false;
            const uint32_t bar = smem_u32(&c.k_full[s]);
            // (tiles of the other parity may still be in use, and one more softmax may read its word: hence four)
            if (lane == 0) {
              c.there[kc / kParts & 3] = there;
              mbar_expect_tx(bar, bytes);
            }
            __syncwarp();
            if (id >= 0) {
#pragma unroll
              for (int blk = 0; blk < kBlocks; ++blk) tma_load_4d(at + blk * kHalfBytes, &tmap_k, bar, dim0 + 64 * blk, slot, w.h, id);
            }
            ++kc;
          } else {
            if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&c.v_empty[s]), ((vc >> 1) & 1) ^ 1))) return false;
            const bool whole = key0 + kBN <= w.len && there == 0xff;
            const uint32_t bar = smem_u32(whole ? &c.v_full[s] : &c.v_raw);
            if (lane == 0) mbar_expect_tx(bar, bytes);
            __syncwarp();
            if (id >= 0) {
#pragma unroll
              for (int blk = 0; blk < kBlocks; ++blk) tma_load_4d(at + blk * kHalfBytes, &tmap_v, bar, dim0 + 64 * blk, slot, w.h, id);
            }
            if (!whole) {
              if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&c.v_raw), raw))) return false;
              raw ^= 1;
              zero_rows<kPart>(smem + 4 * kTileBytes + s * kTileBytes, w, key0, there);
              fence_proxy_async_smem();
              __syncwarp();
              if (lane == 0) mbar_arrive(smem_u32(&c.v_full[s]));
            }
            ++vc;
          }
          return true;
        };
        bool alive = true;
        for (int j = pre; alive && j < it.ntiles * kParts; ++j) alive = load_tile(it, j);
        pre = 0;
        // the first tiles of the next item, as soon as stages free up
        if (alive) {
          const int s1 = (n + 1) & 1;
          alive = __all_sync(0xffffffffu, mbar_wait(smem_u32(&c.item_ready[s1]), ((n + 1) >> 1) & 1));
          if (alive && !c.done[s1]) {
            const int nt = min(2, c.item[s1].ntiles * kParts);
            for (; alive && pre < nt; ++pre) alive = load_tile(c.item[s1], pre);
          }
        }
        if (!alive && lane == 0) { atomicExch(&a.plan->status, RS_PRODUCER); c.abort = 1; }
      } else if (kWide && warp == 1) {
        // QK(0) QK(1) PV(0) QK(2) PV(1) ...: S of tile g of the CTA in accumulator g & 1
        const int ntiles = it.ntiles;
        auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(smem_u32(bar), parity)); };
        tc_fence_after();
        auto qk = [&]() -> bool {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (!wait(&c.k_full[h], (kc >> 1) & 1)) return false;
            tc_fence_after();
            if (el) {
              if (h == 0) rows_qk<0, kHalf, kPart>(tm + (gq & 1) * kBN, dq, dk);
              else rows_qk<1, kHalf, kPart>(tm + (gq & 1) * kBN, dq, dk + (kTileBytes >> 4), true);
              tc_commit(smem_u32(&c.k_empty[h]));
              if (h == 1) tc_commit(smem_u32(&c.s_full[gq & 1]));
            }
            __syncwarp();
            ++kc;
          }
          ++gq;
          return true;
        };
        bool ok = qk();
        if (ok && ntiles > 1) ok = qk();
        for (int j = 0; ok && j < ntiles; ++j) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            ok = ok && wait(&c.v_full[h], (vc >> 1) & 1) && (h == 1 || wait(&c.p_full[0], gp & 1));
            if (!ok) break;
            tc_fence_after();
            if (el) {
              rows_pv<kHalf, kPart>(tm + 256 + 128 * h, tm + (gp & 1) * kBN, dv + h * (kTileBytes >> 4), j == 0);
              tc_commit(smem_u32(&c.v_empty[h]));
              if (h == 1) tc_commit(smem_u32(&c.o_full[0]));
            }
            __syncwarp();
            ++vc;
          }
          ++gp;
          if (ok && j + 2 < ntiles) ok = qk();
        }
        if (!ok && lane == 0) { atomicExch(&a.plan->status, RS_MMA); c.abort = 1; }
      } else if (warp == 1) {
        const int ntiles = it.ntiles;
        auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(smem_u32(bar), parity)); };
        auto kd = [&](uint32_t s) { return dk + s * (kTileBytes >> 4); };
        auto vd = [&](uint32_t s) { return dv + s * (kTileBytes >> 4); };
        tc_fence_after();
        bool ok = true;
        if (rows_twice(D, it)) {
          auto qk = [&](int t) -> bool {
            const uint32_t s = kc & 1;
            if (!wait(&c.k_full[s], (kc >> 1) & 1)) return false;
            tc_fence_after();
            if (el) {
              if (t & 1) rows_qk<1, kHalf, kPart>(tm + kBN, dq, kd(s)); else rows_qk<0, kHalf, kPart>(tm, dq, kd(s));
              tc_commit(smem_u32(&c.s_full[t & 1]));
              tc_commit(smem_u32(&c.k_empty[s]));
            }
            __syncwarp();
            ++kc;
            return true;
          };
          ok = qk(0);
          if (ok && ntiles > 1) ok = qk(1);
          for (int t = 0; ok && t < ntiles; ++t) {
            const int x = t & 1;
            const uint32_t vs = vc & 1;
            ok = wait(&c.v_full[vs], (vc >> 1) & 1) && wait(&c.p_full[x], x ? pph1 : pph0);
            if (!ok) break;
            if (x) pph1 ^= 1; else pph0 ^= 1;
            tc_fence_after();
            if (el) {
              rows_pv<kHalf, kPart>(tm + 256 + 128 * x, tm + x * kBN, vd(vs), t < 2);
              tc_commit(smem_u32(&c.v_empty[vs]));
              if (t + 2 >= ntiles) tc_commit(smem_u32(&c.o_full[x]));
            }
            __syncwarp();
            ++vc;
            if (t + 2 < ntiles) ok = qk(t + 2);
          }
          if (!ok && lane == 0) { atomicExch(&a.plan->status, RS_MMA); c.abort = 1; }
          __syncwarp();
          continue;
        }
        ok = wait(&c.k_full[kc & 1], (kc >> 1) & 1);
        if (ok) {
          tc_fence_after();
          if (el) {
            rows_qk<0, kHalf, kPart>(tm, dq, kd(kc & 1));
            tc_commit(smem_u32(&c.s_full[0]));
            rows_qk<1, kHalf, kPart>(tm + kBN, dq, kd(kc & 1));
            tc_commit(smem_u32(&c.s_full[1]));
            tc_commit(smem_u32(&c.k_empty[kc & 1]));
          }
          __syncwarp();
          ++kc;
        }
        for (int j = 0; ok && j < ntiles; ++j) {
          const bool more = j + 1 < ntiles;
          const uint32_t vs = vc & 1, ks = kc & 1;
          ok = wait(&c.v_full[vs], (vc >> 1) & 1) && wait(&c.p_full[0], pph0);
          if (!ok) break;
          pph0 ^= 1;
          tc_fence_after();
          if (el) {
            rows_pv<kHalf, kPart>(tm + 256, tm, vd(vs), j == 0);
          }
          __syncwarp();
          if (more) {
            ok = wait(&c.k_full[ks], (kc >> 1) & 1);
            if (!ok) break;
            tc_fence_after();
            if (el) {
              rows_qk<0, kHalf, kPart>(tm, dq, kd(ks));
              tc_commit(smem_u32(&c.s_full[0]));
            }
          } else if (el) {
            tc_commit(smem_u32(&c.o_full[0]));
          }
          __syncwarp();
          ok = wait(&c.p_full[1], pph1);
          if (!ok) break;
          pph1 ^= 1;
          tc_fence_after();
          if (el) {
            rows_pv<kHalf, kPart>(tm + 384, tm + kBN, vd(vs), j == 0);
            tc_commit(smem_u32(&c.v_empty[vs]));
            if (more) {
              rows_qk<1, kHalf, kPart>(tm + kBN, dq, kd(ks));
              tc_commit(smem_u32(&c.s_full[1]));
              tc_commit(smem_u32(&c.k_empty[ks]));
            } else {
              tc_commit(smem_u32(&c.o_full[1]));
            }
          }
          __syncwarp();
          ++vc;
          if (more) ++kc;
        }
        if (!ok && lane == 0) { atomicExch(&a.plan->status, RS_MMA); c.abort = 1; }
      }
      __syncwarp();
    }
    if (kCodes && warp == 0 && !ended) end_tiles();
  } else if (warp >= 4 && warp < 12) {
    // ---- warps 4-11: softmax and output, a thread a row
    if (!kCodes) setmaxnreg_inc<216>();
    const int x = (warp - 4) >> 2;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + lane_base + x * kBN, tO = tmem + lane_base + 256 + (kWide ? 0 : x * 128);
    uint32_t sph = 0, oph = 0, kt = 0;     // kt: key tiles of this CTA before the item's
    // head dim 256: the softmax of an item, by warps 4-7; all eight leave when its last P.V has executed
    auto wide_rows = [&](int ntiles, int j0, int lim, int lim_first, int x, uint32_t kt, RowRef& rr, bool& ok) {
      uint32_t g = kt;                                      // the CTA's tiles before this one
      if (x == 0) {
        for (int j = 0; ok && j < ntiles; ++j, ++g) {
          ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&c.s_full[g & 1]), (g >> 1) & 1));
          if (!ok) break;
          tc_fence_after();
          const uint32_t tSg = tmem + lane_base + (g & 1) * kBN;
          const int key0 = (j0 + j) * kBN;
          const uint32_t there = c.there[g & 3];
          // the P.V of tile g - 1 must have executed before O is touched (that of tile g - 2 has)
          auto quiet = [&] {
            if (!mbar_wait(smem_u32(&c.o_full[0]), (g - 1) & 1)) ok = false;
            tc_fence_after();
          };
          if (key0 + kBN > lim_first || there != 0xff || !rows_softmax<false, kHalf, D, kCodes>(tSg, tO, j == 0, 0, 0, p.sl2, rr, quiet))
            rows_softmax<true, kHalf, D, kCodes>(tSg, tO, j == 0, lim - key0, there, p.sl2, rr, quiet);
          // completions of o_full stay at most one behind: the parity of a tile never answers for an older one
          if (j > 0 && !mbar_wait(smem_u32(&c.o_full[0]), (g - 1) & 1)) ok = false;
          ok = __all_sync(0xffffffffu, ok);
          tc_fence_before();
          mbar_arrive(smem_u32(&c.p_full[0]));
        }
      } else {
        g += (uint32_t)ntiles;
      }
      rows_pair_barrier();                                  // the last P has been published
      if (ok) ok = mbar_wait(smem_u32(&c.o_full[0]), (g - 1) & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (x == 0) c.row_inv[row] = rr.ref == -INFINITY && rr.l == 0.f ? 0.f : 1.f / rr.l;
      rows_pair_barrier();                                  // the rows' factors are visible to warps 8-11
    };
    for (int n = 0; rows_next<true, D, kCodes>(a, c, smem, n & 1); ++n) {
      const RowsItem& it = c.item[n & 1];
      const int ntiles = it.ntiles, j0 = it.j0;
      const bool twice = rows_twice(D, it);
      const int base = kWide || twice ? 0 : x * kTileM;    // first row of the item in this row tile
      const int at = it.tile * kRows + base;
      const int i_row = (at + row) / a.by_group, i_first = at / a.by_group;
      const bool on = base + row < it.nrows;
      const int lim = on ? min(max(it.pos0 + i_row + 1, 0), it.len) : 0;
      const int lim_first = min(max(it.pos0 + i_first + 1, 0), it.len);
      RowRef rr{-INFINITY, -INFINITY, 0.f};
      bool ok = true;
      if constexpr (kWide) {
        wide_rows(ntiles, j0, lim, lim_first, x, kt, rr, ok);
      } else {
        const int j1 = twice ? x : 0, by = twice ? 2 : 1;
        for (int j = j1; ok && j < ntiles; j += by) {
          ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&c.s_full[x]), sph));
          if (!ok) break;
          sph ^= 1;
          tc_fence_after();
          const int key0 = (j0 + j) * kBN;
          const uint32_t there = c.there[(kt + j) & 3];
          if (key0 + kBN > lim_first || there != 0xff || !rows_softmax<false, kHalf, D, kCodes>(tS, tO, j == j1, 0, 0, p.sl2, rr, [] {}))
            rows_softmax<true, kHalf, D, kCodes>(tS, tO, j == j1, lim - key0, there, p.sl2, rr, [] {});
          tc_fence_before();
          mbar_arrive(smem_u32(&c.p_full[x]));
        }
        if (j1 < ntiles) {
          if (ok) ok = mbar_wait(smem_u32(&c.o_full[x]), oph);
          ok = __all_sync(0xffffffffu, ok);
          oph ^= 1;
        }
      }
      kt += ntiles;
      if (!kWide && twice) {
        // the row's two results joined; each tile's warps write every other 32 columns
        c.pair_ml[x][row] = make_float2(rr.l != rr.l ? INFINITY : rr.ref, rr.l);
        tc_fence_before();
        rows_pair_barrier();
        tc_fence_after();
        const float2 ml0 = c.pair_ml[0][row], ml1 = c.pair_ml[1][row];
        const float m = fmaxf(ml0.x, ml1.x);
        const float f0 = ml0.x == -INFINITY ? 0.f : exp2f(ml0.x - m), f1 = ml1.x == -INFINITY ? 0.f : exp2f(ml1.x - m);
        const float sum = (f0 == 0.f ? 0.f : f0 * ml0.y) + (f1 == 0.f ? 0.f : f1 * ml1.y);
        const bool empty = m == -INFINITY;
        if (ok) {
          const float inv = it.slot >= 0 ? 1.f : empty ? 0.f : 1.f / sum;
          const int64_t part_row = (int64_t)it.slot * kRows + row, off = c.ooff[n & 1][row];
#pragma unroll 1
          for (int ch = 32 * x; ch < kPart; ch += 64) {
            uint32_t v[32], w[32];
            tmem_ld32(tmem + lane_base + 256 + ch, v);
            tmem_ld32(tmem + lane_base + 384 + ch, w);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const float e0 = f0 == 0.f ? 0.f : f0 * __uint_as_float(v[i]), e1 = f1 == 0.f ? 0.f : f1 * __uint_as_float(w[i]);
              v[i] = __float_as_uint((e0 + e1) * inv);
            }
            if (on && it.slot >= 0) {
#pragma unroll
              for (int u = 0; u < 32; u += 8) store32(a.part + part_row * D + ch + u, v + u);
            } else if (on) {
#pragma unroll
              for (int u = 0; u < 32; u += 8) {
                uint32_t y[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) y[i] = pack2_16<kHalf>(__uint_as_float(v[u + 2 * i]), __uint_as_float(v[u + 2 * i + 1]));
                *reinterpret_cast<uint4*>(a.out + off + ch + u) = make_uint4(y[0], y[1], y[2], y[3]);
              }
            }
            __syncwarp();
          }
          if (on && x == 0) {
            if (it.slot >= 0) a.part_ml[part_row] = make_float2(m, sum);
            else if (a.lse != nullptr) a.lse[(int64_t)(it.h * p.G + (at + row) - i_row * p.G) * p.T + it.row0 + i_row] = (m + log2f(sum)) * kLn2;
          }
          tc_fence_before();
        } else {
          atomicExch(&a.plan->status, RS_SOFTMAX);
          c.abort = 1;
        }
        continue;
      }
      if (ok) {
        tc_fence_after();
        float m_ref = rr.ref;
        const float l = rr.l;
        const float row_inv = kWide ? c.row_inv[row] : 0.f;
        const bool empty = kWide ? row_inv == 0.f : m_ref == -INFINITY && l == 0.f;
        // a sum that is not a number stays one whatever it is joined with
        if (l != l) m_ref = INFINITY;
        const int col0 = kWide ? x * kPart : 0;              // this warp's columns of O
        if (it.slot >= 0) {
          const int64_t part_row = (int64_t)it.slot * kRows + base + row;
          if (on && col0 == 0) a.part_ml[part_row] = make_float2(m_ref, l);
          float* dst = a.part + part_row * D + col0;
#pragma unroll 1
          for (int ch = 0; ch < kPart; ch += 32) {
            uint32_t v[32];
            tmem_ld32(tO + col0 + ch, v);
            tmem_wait_ld();
            if (on) {
#pragma unroll
              for (int u = 0; u < 32; u += 8) store32(dst + ch + u, v + u);
            }
            __syncwarp();
          }
        } else {
          const float inv = kWide ? row_inv : empty ? 0.f : 1.f / l;
          // rows pass through this warp's 8 KB of the idle Q tile: 64 columns at a time, rows 144 bytes apart
          unsigned char* stage = smem + x * kTileBytes + (warp & 3) * 8192;
          const int64_t* ooff = c.ooff[n & 1] + base + (warp & 3) * 32;
#pragma unroll 1
          for (int ch = 0; ch < kPart; ch += 64) {
            const int cols = min(kPart - ch, 64);
#pragma unroll 1
            for (int half = 0; half < cols; half += 32) {
              uint32_t v[32];
              tmem_ld32(tO + col0 + ch + half, v);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                uint32_t w[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                  // (an accumulator of a row that saw nothing holds no number that counts)
                  const float e0 = empty ? 0.f : __uint_as_float(v[8 * i + 2 * u]) * inv, e1 = empty ? 0.f : __uint_as_float(v[8 * i + 2 * u + 1]) * inv;
                  w[u] = pack2_16<kHalf>(e0, e1);
                }
                *reinterpret_cast<uint4*>(stage + lane * 144 + half * 2 + i * 16) = make_uint4(w[0], w[1], w[2], w[3]);
              }
            }
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int rl = i * 4 + (lane >> 3), c16 = lane & 7;
              const int64_t off = ooff[rl];
              if (off >= 0 && c16 * 8 < cols)
                *reinterpret_cast<uint4*>(a.out + off + col0 + ch + c16 * 8) = *reinterpret_cast<const uint4*>(stage + rl * 144 + c16 * 16);
            }
            __syncwarp();
          }
          if (a.lse != nullptr && on && col0 == 0) {
            const int head = it.h * p.G + (at + row) - i_row * p.G;
            a.lse[(int64_t)head * p.T + it.row0 + i_row] = empty ? -INFINITY : (m_ref + log2f(l)) * kLn2;
          }
        }
        tc_fence_before();
      } else {
        atomicExch(&a.plan->status, RS_SOFTMAX);
        c.abort = 1;
      }
    }
  } else {
    // ---- warps 3 and 12-18: codes into operand tiles, one stream of tiles whatever the items are
    const int group = warp == 3 ? 7 : warp - 12;   // of 16 keys
    RawTile<kPart> ra, rb;                 // two parts of operands: one on its way while the other is turned
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      ok = ok && __all_sync(0xffffffffu, mbar_wait(smem_u32(bar), parity));
      return ok;
    };
    // a tile's parts in order: K, V; K_lo, K_hi, V_lo, V_hi.  The first of the next tile is asked for while the last one is turned.
    auto ask_k = [&](uint32_t t, int part, RawTile<kPart>& raw) {
      const TileInfo& info = c.info[t % kInfoSlots];
      raw_load<kPart>(a.kp + part * kPart, a.ks, info.k[group], info.scale[group], p.kp_t, info.keys - 16 * group, lane, raw);
    };
    auto ask_v = [&](uint32_t t, int part, RawTile<kPart>& raw) {
      const TileInfo& info = c.info[t % kInfoSlots];
      raw_load<kPart>(a.vp + part * kPart, a.vs, info.v[group], info.scale[group], p.vp_t, info.keys - 16 * group, lane, raw);
    };
    auto more_tiles = [&](uint32_t t) {                     // false: there are no more
      return wait(&c.info_full[t % kInfoSlots], (t / kInfoSlots) & 1) && c.info[t % kInfoSlots].keys != 0;
    };
    // into stage s, of which this is use number `use`
    auto turn = [&](const RawTile<kPart>& raw, uint64_t* empty, uint64_t* full, uint32_t base, uint32_t s, uint32_t use) {
      if (!wait(&empty[s], (use & 1) ^ 1)) return false;
      raw_store<kHalf, kPart, kStore>(raw, base + s * kTileBytes + group * 2048, lane);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&full[s]));
      return true;
    };
    bool more = more_tiles(0);
    if (more) ask_k(0, 0, ra);
    for (uint32_t t = 0; more; ++t) {
      const uint32_t there = c.info[t % kInfoSlots].there;
      auto asked = [&] {                                    // for all of the tile: its description may go
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&c.info_empty[t % kInfoSlots]));
      };
      // (in front of the arrival on k_full, behind the wait that frees the stage)
      auto tell = [&] { if (group == 0 && lane == 0) c.there[t & 3] = there; };
      if constexpr (kWide) {
        ask_k(t, 1, rb);
        if (!wait(&c.k_empty[0], (t & 1) ^ 1)) break;
        tell();
        if (!turn(ra, c.k_empty, c.k_full, sK, 0, t)) break;
        ask_v(t, 0, ra);
        if (!turn(rb, c.k_empty, c.k_full, sK, 1, t)) break;
        ask_v(t, 1, rb);
        asked();
        if (!turn(ra, c.v_empty, c.v_full, sV, 0, t)) break;
        if ((more = more_tiles(t + 1))) ask_k(t + 1, 0, ra);
        if (!turn(rb, c.v_empty, c.v_full, sV, 1, t)) break;
      } else {
        ask_v(t, 0, rb);
        asked();
        if (!wait(&c.k_empty[t & 1], ((t >> 1) & 1) ^ 1)) break;
        tell();
        if (!turn(ra, c.k_empty, c.k_full, sK, t & 1, t >> 1)) break;
        if ((more = more_tiles(t + 1))) ask_k(t + 1, 0, ra);
        if (!turn(rb, c.v_empty, c.v_full, sV, t & 1, t >> 1)) break;
      }
    }
    if (!ok && lane == 0) { atomicExch(&a.plan->status, RS_PRODUCER); c.abort = 1; }
    __syncwarp();
  }

  // teardown: after an abort copies in flight get time to land
  if (c.abort) {
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 2000000ull) __nanosleep(1000);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

// ---- the pieces' results, joined -------------------------------------------------
// A warp for each packed row (token, head).  Rows whose items were not cut are there already.
constexpr int kJoinThreads = 256;
template <bool kHalf, int D>
__global__ void __launch_bounds__(kJoinThreads) paged_rows_join_kernel(const PagedParams p, const RowsArgs a) {
  pdl_wait();
  pdl_trigger();
  const int64_t g = (int64_t)blockIdx.x * (kJoinThreads / 32) + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const int64_t token = g / p.Hq;
  const int head = (int)(g - token * p.Hq);
  if (token >= p.T || token < __ldg(p.cu) || token >= __ldg(p.cu + p.B)) return;
  const int b = search_warp(p.B, (int)token, [&](int k) { return __ldg(p.cu + k); });
  const PagedSeq s = paged_seq(p, b);
  const int i = (int)(token - s.row0);
  if (i < 0 || i >= s.n) return;
  constexpr int kPer = D / 32;                              // elements of a lane
  __nv_bfloat16* dst = a.out + token * p.so_t + (int64_t)head * p.so_h + lane * kPer;
  float x[kPer];
#pragma unroll
  for (int u = 0; u < kPer; ++u) x[u] = 0.f;
  float mx = -INFINITY, sum = 0.f;
  if (__ldcg(&a.plan->status) != 0) {
    sum = __uint_as_float(0x7fc00000u);                     // a bounded wait gave up: NaN in place of half a result
    mx = 0.f;
  } else {
    const int slot0 = __ldcg(a.plan->slot0 + b);
    if (slot0 < 0) return;
    const int tiles = rows_tiles(p, s.n), piece = __ldcg(a.plan->piece + b);
    const int cuts = (key_tiles(rows_end(p, s, tiles - 1)) + piece - 1) / piece;
    const int h = head / p.G;
    constexpr int kRows = item_rows(D);
    const int row = i * p.G + head - h * p.G, tile = row / kRows, r = row - tile * kRows;
    const int mine = (key_tiles(rows_end(p, s, tile)) + piece - 1) / piece;
    // several pieces under way at a time
    constexpr int kAhead = kPer > 4 ? 4 : 8;
    for (int k0 = 0; k0 < mine; k0 += kAhead) {
      float2 ml[kAhead];
      float v[kAhead][kPer];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        ml[k] = make_float2(-INFINITY, 0.f);
        if (k0 + k >= mine) continue;
        const int64_t at = ((int64_t)slot0 + ((int64_t)h * cuts + k0 + k) * tiles + tiles - 1 - tile) * kRows + r;
        ml[k] = __ldcg(a.part_ml + at);
        const float* src = a.part + at * D + lane * kPer;
        if constexpr (kPer % 4 == 0) {
#pragma unroll
          for (int u = 0; u < kPer; u += 4) {
            const float4 f = __ldcg(reinterpret_cast<const float4*>(src + u));
            v[k][u] = f.x; v[k][u + 1] = f.y; v[k][u + 2] = f.z; v[k][u + 3] = f.w;
          }
        } else {
#pragma unroll
          for (int u = 0; u < kPer; ++u) v[k][u] = __ldcg(src + u);
        }
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        if (ml[k].x == -INFINITY) continue;
        const float up = fmaxf(mx, ml[k].x), f0 = exp2f(mx - up), f1 = exp2f(ml[k].x - up);
        mx = up;
        sum = sum * f0 + ml[k].y * f1;
#pragma unroll
        for (int u = 0; u < kPer; ++u) x[u] = x[u] * f0 + v[k][u] * f1;
      }
    }
  }
  const float inv = mx == -INFINITY ? 0.f : 1.f / sum;
#pragma unroll
  for (int u = 0; u < kPer; ++u) x[u] *= inv;
  if constexpr (kPer % 2 == 0) {
#pragma unroll
    for (int u = 0; u < kPer; u += 2) *reinterpret_cast<uint32_t*>(dst + u) = pack2_16<kHalf>(x[u], x[u + 1]);
  } else {                                                  // head dim 96
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      const uint16_t y = (uint16_t)pack2_16<kHalf>(x[u], 0.f);
      *reinterpret_cast<uint16_t*>(dst + u) = y;
    }
  }
  if (a.lse != nullptr && lane == 0) a.lse[(int64_t)head * p.T + token] = (mx + log2f(sum)) * kLn2;
}

template <bool kHalf, int D>
cudaError_t launch_rows_dim(const PagedParams& p, const CUtensorMap& mk, const CUtensorMap& mv, const RowsArgs& a, int sms, int slots, cudaStream_t st) {
  auto kernel = p.store == MOBA_STORE_SAME ? paged_rows_kernel<kHalf, D, MOBA_STORE_SAME>
              : p.store == MOBA_STORE_E4M3 ? paged_rows_kernel<kHalf, D, MOBA_STORE_E4M3> : paged_rows_kernel<kHalf, D, MOBA_STORE_INT8>;
  const int threads = p.store == MOBA_STORE_SAME ? kRowsThreads<MOBA_STORE_SAME> : kRowsThreads<MOBA_STORE_E4M3>;
  cudaError_t e = prepare_kernel(kernel, kRowsSmem);
  if (e != cudaSuccess) return e;
  if ((e = launch_pdl(paged_plan_kernel, dim3(1), kPagedBatch, 0, st, p, a.plan, sms, slots)) != cudaSuccess) return e;
  if ((e = launch_pdl(kernel, dim3(sms), threads, kRowsSmem, st, p, mk, mv, a)) != cudaSuccess) return e;
  const int64_t warps = p.T * p.Hq, per = kJoinThreads / 32;
  return launch_pdl(paged_rows_join_kernel<kHalf, D>, dim3((unsigned)((warps + per - 1) / per)), kJoinThreads, 0, st, p, a);
}
static_assert(kPagedBatch == 1024, "a thread of the plan kernel for each sequence");

constexpr size_t kPlanBytes = (sizeof(RowsPlan) + 255) / 256 * 256;

}  // namespace

size_t paged_rows_workspace(const PagedParams& p) {
  return kPlanBytes + (size_t)rows_slots(p) * item_rows(p.D) * (sizeof(float2) + p.D * sizeof(float));
}

cudaError_t launch_paged_rows(const PagedParams& all, const void* q, const void* kp, const void* vp, const uint8_t* ks,
                              const uint8_t* vs, void* out, float* lse, void* workspace, cudaStream_t st) {
  RowsArgs a;
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.kp = static_cast<const uint8_t*>(kp);
  a.vp = static_cast<const uint8_t*>(vp);
  a.ks = ks;
  a.vs = vs;
  a.out = static_cast<__nv_bfloat16*>(out);
  a.lse = lse;
  a.plan = static_cast<RowsPlan*>(workspace);
  a.part_ml = reinterpret_cast<float2*>(static_cast<char*>(workspace) + kPlanBytes);
  const int slots_of_results = rows_slots(all);
  a.part = reinterpret_cast<float*>(a.part_ml + (size_t)slots_of_results * item_rows(all.D));
  a.by_group = fast_div(all.G);
  CUtensorMap mk{}, mv{};
  if (all.store == MOBA_STORE_SAME) {
    const int slots = 1 << all.page_shift, box = slots < kBN ? slots : kBN;
    if (!make_page_map(&mk, all.fp16 ? 2 : 3, all.D, kp, all.pages, slots, all.Hkv, all.kp_p, all.kp_t, all.kp_h, box) ||
        !make_page_map(&mv, all.fp16 ? 2 : 3, all.D, vp, all.pages, slots, all.Hkv, all.vp_p, all.vp_t, all.vp_h, box))
      return cudaErrorNotSupported;
  }
  const int sms = device_info().sms;
  for (int b = 0; b < all.B; b += kPagedBatch) {
    PagedParams p = all;
    p.B = all.B - b < kPagedBatch ? all.B - b : kPagedBatch;
    p.cu += b;
    p.lens += b;
    p.table += b * all.table_stride;
    const cudaError_t e = p.D == 64 ? (p.fp16 ? launch_rows_dim<true, 64>(p, mk, mv, a, sms, slots_of_results, st) : launch_rows_dim<false, 64>(p, mk, mv, a, sms, slots_of_results, st))
                        : p.D == 96 ? (p.fp16 ? launch_rows_dim<true, 96>(p, mk, mv, a, sms, slots_of_results, st) : launch_rows_dim<false, 96>(p, mk, mv, a, sms, slots_of_results, st))
                        : p.D == 128 ? (p.fp16 ? launch_rows_dim<true, 128>(p, mk, mv, a, sms, slots_of_results, st) : launch_rows_dim<false, 128>(p, mk, mv, a, sms, slots_of_results, st))
                                     : (p.fp16 ? launch_rows_dim<true, 256>(p, mk, mv, a, sms, slots_of_results, st) : launch_rows_dim<false, 256>(p, mk, mv, a, sms, slots_of_results, st));
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace moba
