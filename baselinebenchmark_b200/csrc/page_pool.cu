// Page tables, slots and positions from the lengths of requests, and pages given back, without the host.
//
// Free pages lie on a stack of numbers.  The entries that a call's new tokens lie in are one line, sequence by sequence.  One that lacks a page is
// number r of those, a prefix sum, and takes the r-th page from the top; pages given back are numbered the same way, and the stack is left as the reserve that took
// them found it.  A warp has a stretch of the line, its count goes to all blocks of the cluster, and every entry then knows its number: no
// atomics, the same pages every time.
// Slots and positions follow row by row; the depth of a row in a tree of drafted tokens by doubling, d(i) += d(up(i)), up(i) <- up(up(i)), which takes
// as many rounds as the depth has bits.
// All of it is a few KB: what bounds it is the chain of dependent loads and barriers, and the launches.  Small calls are one block, one launch.
// Measured (replayed from a graph, us): 64 sequences of one new token 6.3, their pages back 6.2; 40000 new tokens of 1000 sequences 10.3; 200000 in 32 sequences,
// prompts and trees 24.7 (four launches; 118 more with a sequence's rows in one block); 1.9 million entries looked through for pages to give back 33
// (300 entry by entry, in one cluster as now).
#include "page_pool.cuh"

#include "cluster.cuh"
#include "common.cuh"

namespace moba {
namespace {

constexpr int kThreads = 1024, kWarps = kThreads / 32;
constexpr int kBlocks = 8;                 // of the cluster, where there is much to do
constexpr int kSmallRows = 2048;            // that one block does

// Pages of a sequence's tokens, as many as its row of the table has room for.
__device__ __forceinline__ int pages_of(const PoolParams& p, int b) {
  const int64_t room = (int64_t)p.per_seq << p.page_shift, mask = ((int64_t)1 << p.page_shift) - 1;
  return (int)((min(max((int64_t)__ldg(p.lens + b), (int64_t)0), room) + mask) >> p.page_shift);
}
struct Range {                             // entries of a sequence's packed tokens
  int first, count;
};
__device__ __forceinline__ Range entries_of(const PoolParams& p, int b) {
  const int64_t room = (int64_t)p.per_seq << p.page_shift;
  const int up = pages_of(p, b);
  const int64_t n = (int64_t)__ldg(p.cu + b + 1) - __ldg(p.cu + b);
  if (n <= 0) return Range{0, 0};
  const int from = (int)(min(max((int64_t)__ldg(p.lens + b) - n, (int64_t)0), room) >> p.page_shift);
  return Range{from, max(up - from, 0)};
}

// Last b with start[b] <= x.
template <typename F>
__device__ __forceinline__ int search(int n, int64_t x, F&& start) {
  int lo = 0;
  while (n > 1) {
    const int half = n >> 1;
    const bool up = start(lo + half) <= x;
    lo = up ? lo + half : lo;
    n = up ? n - half : half;
  }
  return lo;
}

struct Row {                               // a packed row: its sequence, index in it, first row and position of index 0
  int b, i;
  int64_t row0, pos0;
};
__device__ __forceinline__ bool row_of(const PoolParams& p, int64_t row, Row& r) {
  if (row >= p.rows) return false;
  r.b = search(p.batch, row, [&](int b) { return (int64_t)__ldg(p.cu + b); });
  r.row0 = __ldg(p.cu + r.b);
  const int64_t n = __ldg(p.cu + r.b + 1) - r.row0;
  r.i = (int)(row - r.row0);
  r.pos0 = __ldg(p.lens + r.b) - n;
  return row >= r.row0 && r.i < n;
}
// (the table was written by this launch, or by the one before it: past the read-only path)
__device__ __forceinline__ long long slot_of(const PoolParams& p, const Row& r) {
  const int64_t pos = r.pos0 + r.i;
  if (pos < 0 || (pos >> p.page_shift) >= p.per_seq) return -1;
  const int id = __ldcg(p.table + r.b * p.table_stride + (pos >> p.page_shift));
  if ((unsigned)id >= (unsigned)p.pages) return -1;
  return ((long long)id << p.page_shift) + (pos & (((int64_t)1 << p.page_shift) - 1));
}
__device__ __forceinline__ int clamp_position(int64_t x) { return (int)min(max(x, -((int64_t)1 << 31)), (((int64_t)1 << 31) - 1)); }

// Depths of `rows` rows (a thread has rows tid, tid + kThreads ..; a parent in the block is its place there, depth known so far in `depth`).
template <int kPer>
__device__ __forceinline__ void double_depths(int* up, int* depth) {
  for (;;) {
    int u[kPer], d[kPer];
    bool more = false;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int i = threadIdx.x + k * kThreads;
      u[k] = up[i];
      d[k] = depth[i];
      if (u[k] >= 0) {
        d[k] += depth[u[k]];
        u[k] = up[u[k]];
        more |= u[k] >= 0;
      }
    }
    more = __syncthreads_or(more);
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      up[threadIdx.x + k * kThreads] = u[k];
      depth[threadIdx.x + k * kThreads] = d[k];
    }
    __syncthreads();
    if (!more) return;
  }
}

// Pages taken.  kRows: one block, which also does the rows.
template <bool kRows>
__global__ void __launch_bounds__(kThreads) pool_kernel(const PoolParams p) {
  extern __shared__ int32_t smem[];
  int32_t* begin = smem;                                    // [batch + 1]: first entry of a sequence on the line
  int32_t* first = begin + p.batch + 1;                     // [batch]: its first entry in the table
  __shared__ int32_t scan[kWarps], counts[kWarps], block_total[kBlocks];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = kRows ? 0 : cluster_rank(), blocks = kRows ? 1 : cluster_size();
  if (!kRows) cluster_sync();                               // (all blocks are there)
  pdl_wait();
  pdl_trigger();
  const int have = min(max(__ldcg(p.count), 0), p.pages);
  // ---- the line (every block for itself)
  int carry = 0;
  for (int base = 0; base < p.batch; base += kThreads) {
    const int b = base + tid;
    Range r{0, 0};
    if (b < p.batch) r = entries_of(p, b);
    int x = r.count;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) scan[warp] = x;
    __syncthreads();
    const int s = scan[lane], before = __reduce_add_sync(0xffffffffu, lane < warp ? s : 0), all = __reduce_add_sync(0xffffffffu, s);
    if (b < p.batch) {
      begin[b] = carry + before + x - r.count;
      first[b] = r.first;
    }
    carry += all;
    __syncthreads();
  }
  if (tid == 0) begin[p.batch] = carry;
  __syncthreads();
  // ---- how many of each warp's entries count
  const int warps = (int)blocks * kWarps, me = (int)rank * kWarps + warp;
  const int per = ((carry + warps - 1) / warps + 31) / 32 * 32;
  constexpr int kRound = 4, kStep = 32 * kRound;            // entries under way: of a lane, of a warp
  const int lo = (int)min((int64_t)per * me, (int64_t)carry), hi = (int)min((int64_t)lo + per, (int64_t)carry);
  auto entry = [&](int at, int32_t*& place) {               // not below 0: it lacks a page
    const int b = search(p.batch, at, [&](int k) { return (int64_t)begin[k]; });
    place = p.table + b * p.table_stride + first[b] + (at - begin[b]);
    const int id = *place;
    return (unsigned)id < (unsigned)p.pages ? -1 : 0;
  };
  int mine = 0, ids[kRound];
  int32_t* places[kRound];
  auto load_round = [&](int at) {
#pragma unroll
    for (int k = 0; k < kRound; ++k) {
      ids[k] = -1;
      if (at + 32 * k + lane < hi) ids[k] = entry(at + 32 * k + lane, places[k]);
    }
  };
  // (the last round first: where there is one, as a rule, it is kept for what follows)
  for (int at = lo + (hi - lo - 1) / kStep * kStep; at >= lo && lo < hi; at -= kStep) {
    load_round(at);
#pragma unroll
    for (int k = 0; k < kRound; ++k) mine += __popc(__ballot_sync(0xffffffffu, ids[k] >= 0));
  }
  if (lane == 0) counts[warp] = mine;
  __syncthreads();
  const int c = counts[lane], block_sum = __reduce_add_sync(0xffffffffu, c);
  int before = __reduce_add_sync(0xffffffffu, lane < warp ? c : 0), total = block_sum;
  if (!kRows) {
    if (warp == 0 && lane < (int)blocks) cluster_store(cluster_place(&block_total[rank], lane), (uint32_t)block_sum);
    cluster_sync();
    total = 0;
    for (int i = 0; i < (int)blocks; ++i) {
      if (i < (int)rank) before += block_total[i];
      total += block_total[i];
    }
  }
  // ---- pages taken
  for (int at = lo; at < hi; at += kStep) {
    if (at > lo) load_round(at);
#pragma unroll
    for (int k = 0; k < kRound; ++k) {
      const uint32_t votes = __ballot_sync(0xffffffffu, ids[k] >= 0);
      const int r = before + __popc(votes & ((1u << lane) - 1));
      before += __popc(votes);
      if (ids[k] >= 0 && r < have) *places[k] = p.free[have - 1 - r];
    }
  }
  if (rank == 0 && tid == 0) {
    *p.count = max(have - total, 0);
    *p.missing = max(total - have, 0);
  }
  if constexpr (kRows) {
    // ---- the rows
    __shared__ int32_t up[kSmallRows], depth[kSmallRows];
    constexpr int kPer = kSmallRows / kThreads;
    __threadfence_block();
    __syncthreads();
    Row r[kPer];
    bool on[kPer];
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int64_t row = tid + k * kThreads;
      on[k] = row_of(p, row, r[k]);
      if (p.parents != nullptr) {
        const int parent = on[k] ? __ldg(p.parents + row) : -1;
        const bool has = parent >= 0 && parent < r[k].i;
        up[row] = has ? (int)r[k].row0 + parent : -1;
        depth[row] = has ? 1 : 0;
      }
    }
    if (p.parents != nullptr) {
      __syncthreads();
      double_depths<kPer>(up, depth);
    }
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int64_t row = tid + k * kThreads;
      if (row >= p.rows) continue;
      p.slots[row] = on[k] ? slot_of(p, r[k]) : -1;
      p.positions[row] = on[k] ? clamp_position(r[k].pos0 + (p.parents != nullptr ? depth[row] : r[k].i)) : -1;
  }
  }
}

// Pages given back.  The tables are looked through in units of kSegment entries of a row, an even share of them a warp: counted, then (units that
// have some) numbered and moved.
constexpr int kSegment = 1024, kAbreast = 8;   // entries that a lane has under way
template <bool kOne>
__global__ void __launch_bounds__(kThreads) pool_cut_kernel(const PoolParams p) {
  __shared__ int32_t counts[kWarps], block_total[kBlocks];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = kOne ? 0 : cluster_rank(), blocks = kOne ? 1 : cluster_size();
  if (!kOne) cluster_sync();                                // (all blocks are there)
  pdl_wait();
  pdl_trigger();
  const int have = min(max(__ldcg(p.count), 0), p.pages);
  const int segments = (p.per_seq + kSegment - 1) / kSegment, warps = (int)blocks * kWarps, me = (int)rank * kWarps + warp;
  const int64_t units = (int64_t)p.batch * segments, lo = units * me / warps, hi = units * (me + 1) / warps;
  // runs `step(entries, first column, end)` over a unit, 32 * kAbreast entries at a time
  auto over = [&](int64_t unit, auto&& step) {
    const int b = (int)(unit / segments), from = (int)(unit - (int64_t)b * segments) * kSegment;
    const int end = min(from + kSegment, p.per_seq);
    int32_t* row = p.table + b * p.table_stride;
    for (int at = max(from, pages_of(p, b)); at < end; at += 32 * kAbreast) {
      int ids[kAbreast];
#pragma unroll
      for (int k = 0; k < kAbreast; ++k) {
        const int column = at + 32 * k + lane;
        ids[k] = column < end ? __ldcg(row + column) : -1;
        if ((unsigned)ids[k] >= (unsigned)p.pages) ids[k] = -1;
      }
      step(ids, row + at);
    }
  };
  int mine = 0;
  uint32_t some = 0;                                        // units with pages; those from the 32nd on as one
  for (int64_t unit = lo; unit < hi; ++unit) {
    int n = 0;
    over(unit, [&](const int (&ids)[kAbreast], int32_t*) {
#pragma unroll
      for (int k = 0; k < kAbreast; ++k) n += __popc(__ballot_sync(0xffffffffu, ids[k] >= 0));
    });
    mine += n;
    if (n > 0) some |= 1u << (int)min(unit - lo, (int64_t)31);
  }
  if (lane == 0) counts[warp] = mine;
  __syncthreads();
  const int c = counts[lane], block_sum = __reduce_add_sync(0xffffffffu, c);
  int before = __reduce_add_sync(0xffffffffu, lane < warp ? c : 0), total = block_sum;
  if (!kOne) {
    if (warp == 0 && lane < (int)blocks) cluster_store(cluster_place(&block_total[rank], lane), (uint32_t)block_sum);
    cluster_sync();
    total = 0;
    for (int i = 0; i < (int)blocks; ++i) {
      if (i < (int)rank) before += block_total[i];
      total += block_total[i];
    }
  }
  for (int64_t unit = lo; unit < hi; ++unit) {
    if (!((some >> (int)min(unit - lo, (int64_t)31)) & 1)) continue;
    over(unit, [&](const int (&ids)[kAbreast], int32_t* row) {
#pragma unroll
      for (int k = 0; k < kAbreast; ++k) {
        const uint32_t votes = __ballot_sync(0xffffffffu, ids[k] >= 0);
        const int64_t to = (int64_t)have + total - 1 - before - __popc(votes & ((1u << lane) - 1));
        before += __popc(votes);
        if (ids[k] < 0) continue;
        if (to >= 0 && to < p.pages) p.free[to] = ids[k];
        row[32 * k + lane] = -1;
      }
    });
  }
  if (rank == 0 && threadIdx.x == 0) *p.count = (int)min((int64_t)have + total, (int64_t)p.pages);
}

// A row a thread.  With parents the position is there already.
constexpr int kRowThreads = 256;
__global__ void __launch_bounds__(kRowThreads) pool_rows_kernel(const PoolParams p) {
  pdl_wait();
  pdl_trigger();
  const int64_t row = (int64_t)blockIdx.x * kRowThreads + threadIdx.x;
  if (row >= p.rows) return;
  Row r;
  const bool on = row_of(p, row, r);
  p.slots[row] = on ? slot_of(p, r) : -1;
  if (p.parents == nullptr) p.positions[row] = on ? clamp_position(r.pos0 + r.i) : -1;
}

// Depths of many rows, in two steps.  First blocks of kWayRows rows for themselves: by doubling each row gets the way to the first ancestor in front
// of the block's rows (or its root) and how long it is, kept in the row's slot until that is written.  Then every row goes from block to block; a
// prompt without branches has a step for each kWayRows rows.
constexpr int kWayPer = 4, kWayRows = kWayPer * kThreads;
__device__ __forceinline__ long long pack_way(int exit, int length) { return ((long long)exit << 32) | (unsigned)length; }
__global__ void __launch_bounds__(kThreads) pool_ways_kernel(const PoolParams p) {
  extern __shared__ int32_t smem[];
  int32_t *up = smem, *depth = up + kWayRows, *out = depth + kWayRows;
  pdl_wait();
  pdl_trigger();
  const int64_t base = (int64_t)blockIdx.x * kWayRows;
  int u[kWayPer], d[kWayPer], e[kWayPer];
#pragma unroll
  for (int k = 0; k < kWayPer; ++k) {
    const int64_t row = base + threadIdx.x + k * kThreads;
    Row r;
    const bool on = row_of(p, row, r);
    const int parent = on ? __ldg(p.parents + row) : -1;
    const bool has = parent >= 0 && parent < r.i;
    const int64_t to = has ? r.row0 + parent : -1;
    u[k] = to >= base ? (int)(to - base) : -1;
    d[k] = has ? 1 : 0;
    e[k] = has && u[k] < 0 ? (int)to : -1;
  }
  for (;;) {
    bool more = false;
#pragma unroll
    for (int k = 0; k < kWayPer; ++k) {
      const int i = threadIdx.x + k * kThreads;
      up[i] = u[k];
      depth[i] = d[k];
      out[i] = e[k];
      more |= u[k] >= 0;
    }
    if (!__syncthreads_or(more)) break;
#pragma unroll
    for (int k = 0; k < kWayPer; ++k) {
      const int at = u[k];
      if (at >= 0) { d[k] += depth[at]; e[k] = out[at]; u[k] = up[at]; }
    }
    __syncthreads();
  }
#pragma unroll
  for (int k = 0; k < kWayPer; ++k) {
    const int64_t row = base + threadIdx.x + k * kThreads;
    if (row < p.rows) p.slots[row] = pack_way(e[k], d[k]);
  }
}
__global__ void __launch_bounds__(kRowThreads) pool_depths_kernel(const PoolParams p) {
  pdl_wait();
  pdl_trigger();
  const int64_t row = (int64_t)blockIdx.x * kRowThreads + threadIdx.x;
  if (row >= p.rows) return;
  Row r;
  const bool on = row_of(p, row, r);
  int64_t depth = 0;
  for (int64_t at = row; on && at >= 0;) {                  // (an exit lies in front of its row)
    const long long way = __ldcg(p.slots + at);
    depth += (int)way;
    const int exit = (int)(way >> 32);
    at = exit < at ? exit : -1;
  }
  p.positions[row] = on ? clamp_position(r.pos0 + depth) : -1;
}

}  // namespace

cudaError_t launch_pool(const PoolParams& p, cudaStream_t st) {
  const size_t smem = (2 * (size_t)p.batch + 1) * sizeof(int32_t);
  cudaError_t e;
  if (p.cu == nullptr) {
    // (units: two for each warp of a block)
    const int64_t units = (int64_t)p.batch * ((p.per_seq + kSegment - 1) / kSegment);
    return units <= 2 * kWarps ? launch_pdl(pool_cut_kernel<true>, dim3(1), kThreads, 0, st, p)
                               : launch_clusters(pool_cut_kernel<false>, kBlocks, dim3(kBlocks), kThreads, 0, st, p);
  }
  if (p.rows <= kSmallRows) {
    if ((e = prepare_kernel(pool_kernel<true>, smem)) != cudaSuccess) return e;
    return launch_pdl(pool_kernel<true>, dim3(1), kThreads, smem, st, p);
  }
  if ((e = prepare_kernel(pool_kernel<false>, smem)) != cudaSuccess) return e;
  if ((e = launch_clusters(pool_kernel<false>, kBlocks, dim3(kBlocks), kThreads, smem, st, p)) != cudaSuccess) return e;
  const dim3 grid((unsigned)((p.rows + kRowThreads - 1) / kRowThreads));
  if (p.parents != nullptr) {
    constexpr size_t way_smem = 3 * kWayRows * sizeof(int32_t);
    if ((e = prepare_kernel(pool_ways_kernel, way_smem)) != cudaSuccess) return e;
    if ((e = launch_pdl(pool_ways_kernel, dim3((unsigned)((p.rows + kWayRows - 1) / kWayRows)), kThreads, way_smem, st, p)) != cudaSuccess) return e;
    if ((e = launch_pdl(pool_depths_kernel, grid, kRowThreads, 0, st, p)) != cudaSuccess) return e;
  }
  return launch_pdl(pool_rows_kernel, grid, kRowThreads, 0, st, p);
}

}  // namespace moba
