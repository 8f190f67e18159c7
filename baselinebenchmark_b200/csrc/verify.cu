// Drafted tokens checked against the target's probabilities, with given random numbers.
//
// The packed rows of a sequence are a tree: row 0 is its last accepted token, row i > 0 a drafted token x_i that follows row parent(i).  p_v is the
// target's distribution behind row v, q_v the draft's, of which v's children were drawn.  From row 0 on, the children of a row v are looked at in the
// order of their rows, t being what is left of p_v and S its sum (at first t = p_v and S = 1):
//     child c is accepted      where t(x_c) > 0 and u_c q_v(x_c) S < t(x_c);            the walk goes on from c
//     otherwise                t <- max(t / S - q_v, 0), S <- sum of t
// and where no child is left, or none was accepted, the next token is the first whose sum of t up to and with it exceeds u sum(t).  So the
// accepted tokens and the next one are distributed as the target's.  Without q the children are given tokens and not draws (q is 1 for each
// in its turn): t loses x_c, S its probability.  All in 64 bits, in which the probabilities' differences and sums are next to exact: an answer
// does not depend on the order of the sums but for borders that lie within 1e-13 of a random number.
//
// A cluster of blocks has a sequence.  The first block knows all rows' tokens and probabilities after one round of loads and walks the tree on its own;
// it tells the others what sum is needed next (so that no block takes another way than its neighbours, whatever the tensors hold), all blocks add up
// their part of the vocabulary and tell one another.  A walk needs one pass over one row of p and q, one more for each drafted
// sibling beyond the first that is not accepted; the token is found in the one block, warp and thread whose sums the random number falls to.
// The sums are quick where no child or one was rejected: max(p - q, 0) = max(p, q) - q takes the maximum in 32 bits, exactly, and two
// conversions; a sum that is not finite tells of infinities, and is taken again the careful way.
// Bound by the bytes of that row where there are many sequences, else by the chain of loads and barriers.
// Measured (replayed from a graph, us; in brackets the bytes at the measured copy bandwidth):
//   5 rows of 64 sequences over 128000 tokens, fp32      35.4 -> 28.8 (four blocks an SM in place of one) -> 20.6 (quick sums)   [10.0]
//   6 rows of one sequence over 32000, fp32              10.3                                                                [0.04]
//   40 rows of 16 over 100003, bf16, no draft            18.5 -> 14.4 (the rejected tokens' bits looked at a vector at a time) [0.5]
//   32 rows of 24 over 64000, many siblings              141 (divided by S) -> 56 (by 1 / S, and quick sums)
// The second is: launch 2.5, tokens and their probabilities (three dependent loads), the walk, three barriers of the cluster, one pass, one look for the token.
#include <cuda_fp16.h>
#include <cuda_bf16.h>

#include <type_traits>

#include "cluster.cuh"
#include "common.cuh"
#include "moba_b200.h"
#include "verify.cuh"

namespace moba {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kAbreast = 2;               // vectors of p, and of q, that a lane has under way
constexpr int kMostBlocks = 8;             // of a cluster

struct Node {                              // a row: what its test needs
  int32_t parent, token;
  float have, drawn, u;                    // p and q of its token behind its parent
};
struct Command {
  int32_t row;                             // whose distributions; -1: there is nothing to add up
  int32_t rejected;                        // children that were not accepted
  int32_t last;                            // nothing left to look at: a token is wanted
};

__device__ __forceinline__ float element(const float* p) { return __ldg(p); }
__device__ __forceinline__ float element(const __half* p) { return __half2float(__ldg(p)); }
__device__ __forceinline__ float element(const __nv_bfloat16* p) { return __bfloat162float(__ldg(p)); }
// What is no probability (negative, infinite, not a number) counts as 0.
__device__ __forceinline__ float probability(float x) { return x > 0.f && x < INFINITY ? x : 0.f; }

template <typename T> constexpr int kVector = 16 / sizeof(T);
template <typename T>
__device__ __forceinline__ void widen(const uint4& w, float (&x)[kVector<T>]) {
  if constexpr (std::is_same<T, float>::value) {
    x[0] = __uint_as_float(w.x); x[1] = __uint_as_float(w.y); x[2] = __uint_as_float(w.z); x[3] = __uint_as_float(w.w);
  } else {
    unpack8<std::is_same<T, __half>::value>(w, x);
  }
}

// What is left of an element after the rejections of a row's children.
struct Residual {
  const double* inverse;                   // 1 / S after each rejection, from the first on (0: nothing is left); the last one may not be known yet
  int rejected;
  const uint32_t* taken;                   // without a draft: tokens that were rejected, bits from `taken0` on; null: none
  int64_t taken0;
  // bit of element `at`, and those behind it in its word
  __device__ __forceinline__ uint32_t gone(int64_t at) const { return taken == nullptr ? 0u : taken[(at - taken0) >> 5] >> ((at - taken0) & 31); }
  template <bool kDraft>
  __device__ __forceinline__ double operator()(float p, float q, int64_t at) const {
    double t = (double)probability(p);
    if (kDraft) {
      if (rejected > 0) {
        const double d = (double)probability(q);
        t = fmax(t - d, 0.0);
#pragma unroll 1
        for (int j = 0; j + 1 < rejected; ++j) t = fmax(__dsub_rn(__dmul_rn(t, inverse[j]), d), 0.0);
      }
    } else if (gone(at) & 1) {
      t = 0.0;
    }
    return t;
  }
};

__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// The next step of the walk, by the first warp of the first block: from row `at`, behind its first `rejected` children (of which `before` was the last),
// with the sum of what is left of its row (rejected > 0).
struct Walk {
  int at, before, rejected, length;
  double mass;
};
template <bool kDraft>
__device__ __forceinline__ Command walk_on(const Node* nodes, int n, Walk& w, const double* inverse, int16_t* path) {
  const int lane = threadIdx.x & 31;
  for (;;) {
    // the next child of row `at`, behind row `before`
    int child = -1;
    for (int base = (w.before + 1) & ~31; base < n; base += 32) {
      const int i = base + lane;
      const uint32_t mine = __ballot_sync(0xffffffffu, i > w.before && i < n && nodes[i].parent == w.at);
      if (mine) { child = base + __ffs(mine) - 1; break; }
    }
    if (child < 0) return Command{w.at, w.rejected, 1};
    const Node c = nodes[child];
    double have = (double)probability(c.have), drawn = kDraft ? (double)probability(c.drawn) : 1.0;
    if (kDraft) {
      // (the sum after the last rejection is asked for when a sibling needs it)
      if (w.rejected > 0 && w.mass < 0.0) return Command{w.at, w.rejected, 0};
      if (w.rejected > 0) {
        have = fmax(have - drawn, 0.0);
        for (int j = 0; j + 1 < w.rejected; ++j) have = fmax(__dsub_rn(__dmul_rn(have, inverse[j]), drawn), 0.0);
      }
    } else if (w.rejected > 0) {
      bool twice = false;                                   // a sibling had the token
      for (int i = w.at + 1 + lane; i < child; i += 32) twice |= nodes[i].parent == w.at && nodes[i].token == c.token;
      if (__any_sync(0xffffffffu, twice)) have = 0.0;
    }
    const double mass = w.rejected > 0 ? w.mass : 1.0;
    if (have > 0.0 && (double)c.u * mass * drawn < have) {
      if (lane == 0) path[w.length] = (int16_t)child;
      w = Walk{child, child, 0, w.length + 1, 1.0};
    } else {
      w.before = child;
      ++w.rejected;
      w.mass = kDraft ? -1.0 : mass - have;
    }
  }
}

// (four blocks an SM: a batch of 74 sequences is resident at once)
template <typename T, bool kDraft>
__global__ void __launch_bounds__(kThreads, 4) verify_kernel(const VerifyParams a) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ double totals[kMostBlocks], warp_total[kWarps];
  __shared__ Command told;
  __shared__ int first_at, last_at;
  const int most = a.max_new;
  double* inverse = reinterpret_cast<double*>(smem);        // [max_new]
  Node* nodes = reinterpret_cast<Node*>(inverse + most);    // [max_new]
  int16_t* path = reinterpret_cast<int16_t*>(nodes + most);   // [max_new, even]
  uint32_t* taken = reinterpret_cast<uint32_t*>(path + ((most + 1) & ~1));   // a bit for each token of this block's part
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cluster_rank(), blocks = cluster_size();
  const int b = blockIdx.x / blocks;
  cluster_sync();                                           // (all blocks are there)
  pdl_wait();
  pdl_trigger();
  const int64_t row0 = min(max((int64_t)__ldg(a.cu + b), (int64_t)0), a.rows), end = min((int64_t)__ldg(a.cu + b + 1), a.rows);
  const int n = (int)min(max(end - row0, (int64_t)0), (int64_t)most);
  const T* target = static_cast<const T*>(a.target) + row0 * a.target_stride;
  const T* draft = kDraft ? static_cast<const T*>(a.draft) + row0 * a.draft_stride : nullptr;
  auto token_of = [&](int64_t i) { return a.tokens64 ? (int64_t)__ldg(static_cast<const long long*>(a.tokens) + i) : (int64_t)__ldg(static_cast<const int*>(a.tokens) + i); };
  // this block's part of the vocabulary, and each warp's of it
  const int64_t part = a.part, share = part / kWarps;
  constexpr int kV = kVector<T>;
  Walk walk{0, 0, 0, 1, 1.0};
  if (rank == 0) {
    for (int i = tid; i < n; i += kThreads) {
      Node c{-1, -1, 0.f, 0.f, 0.f};
      if (i > 0) {
        const int parent = a.parents != nullptr ? __ldg(a.parents + row0 + i) : i - 1;
        const int64_t x = token_of(row0 + i);
        if (parent >= 0 && parent < i) {
          c.parent = parent;
          c.u = __ldg(a.accept + row0 + i);
          if (x >= 0 && x < a.vocabulary) {
            c.token = (int)x;
            c.have = element(target + parent * a.target_stride + x);
            if (kDraft) c.drawn = element(draft + parent * a.draft_stride + x);
          }
        }
      }
      nodes[i] = c;
    }
    if (tid == 0) path[0] = 0;
    __syncthreads();
  }
  bool raw = false;                                         // nothing was left of the row: the token is drawn from all of it
  bool infinite = false, again = false;                     // the sum was: there are infinities, which the quick way does not look for
  for (;;) {
    // ---- what is needed next: the first block tells all
    if (rank == 0 && warp == 0) {
      Command c = n == 0 ? Command{-1, 0, 1} : again ? told : raw ? Command{walk.at, 0, 1} : walk_on<kDraft>(nodes, n, walk, inverse, path);
      __syncwarp();
      for (uint32_t i = lane; i < blocks * 3; i += 32) {
        const uint32_t to = i / 3, word = i - to * 3;
        cluster_store(cluster_place(&told, to) + 4 * word, (uint32_t)(word == 0 ? c.row : word == 1 ? c.rejected : c.last));
      }
      // the sums of the rejections (the other blocks need them, the newest one excepted)
      if (kDraft && c.rejected > 1)
        for (uint32_t to = 1 + lane; to < blocks; to += 32)
          cluster_store(cluster_place(&inverse[c.rejected - 2], to), (uint64_t)__double_as_longlong(inverse[c.rejected - 2]));
    }
    // without a draft the rejected tokens do not count any more
    if (!kDraft) for (int i = tid; i < (int)((part + 2 * kV + 31) / 32); i += kThreads) taken[i] = 0;
    cluster_sync();
    const Command c = told;
    if (c.row < 0) break;
    const T* p = target + c.row * a.target_stride;
    const T* q = kDraft ? draft + c.row * a.draft_stride : nullptr;
    const bool with_draft = kDraft && c.rejected > 0;
    // parts begin where p is aligned for vectors, `head` elements behind a multiple of their size; the first part has those too
    const int head = (int)(((16 - ((uintptr_t)p & 15)) & 15) / sizeof(T));
    const bool vectors = !with_draft || (((uintptr_t)p ^ (uintptr_t)q) & 15) == 0;
    const int64_t lo = rank == 0 ? 0 : min((int64_t)rank * part + head, a.vocabulary), hi = min(((int64_t)rank + 1) * part + head, a.vocabulary);
    const int64_t taken0 = (int64_t)rank * part + head - kV;   // a vector's bits lie in one word
    auto first_of = [&](int w) { return w == 0 ? lo : min((int64_t)rank * part + head + w * share, hi); };
    auto end_of = [&](int w) { return min((int64_t)rank * part + head + (w + 1) * share, hi); };
    const int64_t wlo = first_of(warp), whi = end_of(warp);
    if (!kDraft && c.rejected > 0) {
      // (of the children of a row all were rejected)
      for (int i = c.row + 1 + tid; i < n; i += kThreads) {
        const int parent = a.parents != nullptr ? __ldg(a.parents + row0 + i) : i - 1;
        const int64_t x = token_of(row0 + i);
        if (parent == c.row && x >= lo && x < hi) atomicOr(&taken[(x - taken0) >> 5], 1u << ((x - taken0) & 31));
      }
      __syncthreads();
    }
    // ---- the sum of what is left, warp by warp
    const Residual left{inverse, c.rejected, !kDraft && c.rejected > 0 ? taken : nullptr, taken0};
    // quick: t is p, or max(p - q, 0) = max(p, q) - q with p and q no less than 0 (which drops what is not a number)
    const bool quick = !infinite && (!kDraft || c.rejected <= 1);
    double s0 = 0.0, s1 = 0.0;
    auto one = [&](float x, float y, int64_t e, int i, uint32_t gone) {
      double t;
      if (quick) {
        const float d = fmaxf(y, 0.f);
        t = kDraft ? (double)fmaxf(fmaxf(x, 0.f), d) - (double)d : (double)(gone & 1 ? 0.f : fmaxf(x, 0.f));
      } else {
        t = left.template operator()<kDraft>(x, y, e);
      }
      if (i & 1) s1 += t; else s0 += t;
    };
    int64_t at = wlo;
    if (vectors) {
      if (rank == 0 && warp == 0 && lane < head && lane < whi) one(element(p + lane), with_draft ? element(q + lane) : 0.f, lane, 0, left.gone(lane));
      if (rank == 0 && warp == 0) at = min((int64_t)head, whi);
      for (; at + 32 * kV * kAbreast <= whi; at += 32 * kV * kAbreast) {
        uint4 x[kAbreast], y[kAbreast];
#pragma unroll
        for (int k = 0; k < kAbreast; ++k) {
          const int64_t e = at + (k * 32 + lane) * kV;
          x[k] = __ldg(reinterpret_cast<const uint4*>(p + e));
          y[k] = with_draft ? __ldg(reinterpret_cast<const uint4*>(q + e)) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int k = 0; k < kAbreast; ++k) {
          float f[kV], g[kV];
          widen<T>(x[k], f);
          widen<T>(y[k], g);
          const int64_t e = at + (k * 32 + lane) * kV;
          const uint32_t gone = kDraft ? 0u : left.gone(e);
#pragma unroll
          for (int i = 0; i < kV; ++i) one(f[i], g[i], e + i, i, gone >> i);
        }
      }
#pragma unroll 1
      for (; at + 32 * kV <= whi; at += 32 * kV) {
        const int64_t e = at + lane * kV;
        float f[kV], g[kV];
        const uint32_t gone = kDraft ? 0u : left.gone(e);
        widen<T>(__ldg(reinterpret_cast<const uint4*>(p + e)), f);
        widen<T>(with_draft ? __ldg(reinterpret_cast<const uint4*>(q + e)) : make_uint4(0, 0, 0, 0), g);
#pragma unroll
        for (int i = 0; i < kV; ++i) one(f[i], g[i], e + i, i, gone >> i);
      }
    }
    for (; at < whi; at += 32 * kV) {
      float x[kV], y[kV];
#pragma unroll
      for (int i = 0; i < kV; ++i) {
        const int64_t e = at + lane + 32 * i;
        x[i] = e < whi ? element(p + e) : 0.f;
        y[i] = with_draft && e < whi ? element(q + e) : 0.f;
      }
#pragma unroll
      for (int i = 0; i < kV; ++i) {
        const int64_t e = at + lane + 32 * i;
        if (e < whi) one(x[i], y[i], e, i, kDraft ? 0u : left.gone(e));
      }
    }
    const double mine = warp_sum(s0 + s1);
    if (lane == 0) warp_total[warp] = mine;
    if (tid == 0) { first_at = 0x7fffffff; last_at = -1; }
    __syncthreads();
    if (warp == 0 && lane < (int)blocks) {
      double sum = 0.0;
      for (int w = 0; w < kWarps; ++w) sum += warp_total[w];
      cluster_store(cluster_place(&totals[rank], lane), (uint64_t)__double_as_longlong(sum));
    }
    cluster_sync();
    double total = 0.0;
    for (uint32_t i = 0; i < blocks; ++i) total += totals[i];
    again = quick && !(total <= 1e300);
    if (again) { infinite = true; continue; }
    if (!c.last) {
      if (rank == 0 && warp == 0) {
        walk.mass = total;
        if (lane == 0) inverse[c.rejected - 1] = total > 0.0 ? 1.0 / total : 0.0;
        __syncwarp();
      }
      continue;
    }
    if (!(total > 0.0) && c.rejected > 0) { raw = true; continue; }
    // ---- the token: the block, the warp, the element whose sum exceeds the random number's
    int64_t token = -1;
    if (total > 0.0) {
      const double bar = (double)__ldg(a.sample + b) * total;
      auto pick = [&](const double* parts, int count, double& before) {
        int found = -1, last = 0;
        double sum = before;
        for (int i = 0; i < count; ++i) {
          if (parts[i] > 0.0) last = i;
          if (found < 0 && parts[i] > 0.0 && sum + parts[i] > bar) { found = i; before = sum; }
          sum += parts[i];
        }
        if (found >= 0) return found;
        // (rounded, or a number from 1 on: the last that has any)
        before = INFINITY;
        return last;
      };
      double before = 0.0;
      const int in_block = pick(totals, (int)blocks, before);
      if (in_block != (int)rank) break;                     // (no barrier of the cluster comes behind this)
      const int in_warp = before == INFINITY ? -1 : pick(warp_total, kWarps, before);
      int64_t flo, fhi;
      if (before == INFINITY) { flo = lo; fhi = hi; } else { flo = first_of(in_warp); fhi = end_of(in_warp); }
      // each thread has a few elements that lie together
      const int64_t per = (fhi - flo + kThreads - 1) / kThreads, from = min(flo + tid * per, fhi), to = min(from + per, fhi);
      auto value = [&](int64_t e) { return left.template operator()<kDraft>(element(p + e), with_draft ? element(q + e) : 0.f, e); };
      double own = 0.0;
      int64_t has = -1;
      for (int64_t e = from; e < to; ++e) {
        const double t = value(e);
        if (t > 0.0) has = e;
        own += t;
      }
      double x = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      __syncthreads();                                      // (warp_total has been read)
      if (lane == 31) warp_total[warp] = x;
      __syncthreads();
      double sum = before + (x - own);
      for (int w = 0; w < warp; ++w) sum += warp_total[w];
      for (int64_t e = from; e < to; ++e) {
        const double t = value(e);
        sum += t;
        if (t > 0.0 && sum > bar && before != INFINITY) {
          atomicMin(&first_at, (int)e);
          break;
        }
      }
      if (has >= 0) atomicMax(&last_at, (int)has);
      __syncthreads();
      token = first_at != 0x7fffffff ? first_at : last_at;
    } else if (rank != 0) {
      break;
    }
    if (tid == 0) {
      if (a.tokens64) static_cast<long long*>(a.next)[b] = token; else static_cast<int*>(a.next)[b] = (int)token;
    }
    break;
  }
  // ---- the accepted rows
  if (rank == 0) {
    __syncthreads();
    if (tid == 0) {
      last_at = n == 0 ? 0 : walk.length;
      a.count[b] = last_at;
      if (n == 0) {
        if (a.tokens64) static_cast<long long*>(a.next)[b] = -1; else static_cast<int*>(a.next)[b] = -1;
      }
    }
    __syncthreads();
    for (int i = tid; i < most; i += kThreads) a.path[(int64_t)b * most + i] = i < last_at ? path[i] : -1;
  }
}

typedef void (*VerifyKernel)(const VerifyParams);
template <typename T> VerifyKernel pick_kernel(bool draft) { return draft ? verify_kernel<T, true> : verify_kernel<T, false>; }

}  // namespace

cudaError_t launch_verify(VerifyParams a, int dtype, cudaStream_t st) {
  const VerifyKernel kernel = dtype == MOBA_DTYPE_FP32 ? pick_kernel<float>(a.draft != nullptr)
                            : dtype == MOBA_DTYPE_FP16 ? pick_kernel<__half>(a.draft != nullptr) : pick_kernel<__nv_bfloat16>(a.draft != nullptr);
  const int64_t step = (int64_t)kWarps * 32 * (dtype == MOBA_DTYPE_FP32 ? 4 : 8);   // whole vectors of all warps
  // Blocks of a cluster: a round of them (four an SM, as many as fit of fp32 rows with a draft and few new ones; the bits of a wide part and max_new of 1024 leave
  // fewer, which costs time only) takes 8 us and 0.5 us for each 1000 tokens of a part.  (fp32 with a draft, sequences x tokens, us with 8 / 4 / 2 / 1 blocks:
  // 1 x 32000 10 / 12 / 16 / 23, 100 x 32000 19 / 14 / 18 / 25, 300 x 32000 44 / 32 / 29 / 31, 64 x 128000 21 / 29 / 51 / 93, 300 x 128000 86 / 83 / 107 / 124,
  // 600 x 1000 65 / 37 / 23 / 16)
  const int64_t round = 4 * (int64_t)device_info().sms;
  int blocks = 0;
  int64_t least = 0;
  for (int n = kMostBlocks; n >= 1; n /= 2) {
    const int64_t part = (a.vocabulary + n * step - 1) / (n * step) * step;
    if (blocks != 0 && a.draft == nullptr && part / 8 > (128 << 10)) break;   // (the bits of a part lie in shared memory)
    const int64_t cost = (a.batch * (int64_t)n + round - 1) / round * (16000 + a.vocabulary / n);
    if (blocks == 0 || cost < least) { blocks = n; least = cost; a.part = part; }
  }
  const size_t smem = (size_t)a.max_new * (sizeof(double) + sizeof(Node)) + (size_t)((a.max_new + 1) & ~1) * sizeof(int16_t) +
                      (a.draft == nullptr ? (size_t)((a.part + 16 + 31) / 32) * 4 : 0);
  cudaError_t e = prepare_kernel(kernel, smem);
  if (e != cudaSuccess) return e;
  return launch_clusters(kernel, blocks, dim3((unsigned)(a.batch * blocks)), kThreads, smem, st, a);
}

}  // namespace moba
