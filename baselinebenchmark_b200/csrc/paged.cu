// New K and V rows into the pages of their sequences, and back.
//
// Both are bound by bytes (a row in, a row out: 4 bytes an element of 16-bit pages, 3 of 8-bit ones) and, for the few rows of a decode step, by
// the chain of dependent loads from a row to its sequence, its page and its slot.  A warp takes kTokens packed tokens
// and a few heads of them: the rows are asked for first, the chain runs while they travel.  D / 8 lanes have a row, 8 elements each, so
// that a warp's accesses are whole rows; the largest magnitude of a row goes through the lanes as an integer (the bits of
// |x| rise with it, and a NaN is above them all).
#include <cuda_fp8.h>

#include "paged.cuh"

namespace moba {
namespace {

constexpr int kRowThreads = 256;

// lanes of a row: D / 8, in a group of a power of two
template <int D> constexpr int kRowLanes = D == 64 ? 8 : D == 256 ? 32 : 16;

template <bool kHalf> __device__ __forceinline__ uint32_t abs_bits_max(uint4 x) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack2<kHalf>(w[i]);
    m = max(m, max(__float_as_uint(f.x) & 0x7fffffffu, __float_as_uint(f.y) & 0x7fffffffu));
  }
  return m;
}

// The byte of a row whose largest magnitude has these bits (see moba_b200.h).  amax = m * 2^k with m in [1, 2); the largest code is
// 1.75 * 2^8 (e4m3) or 1.984375 * 2^6 (int8).
template <int kStore>
__device__ __forceinline__ uint32_t row_byte(uint32_t amax) {
  if (amax == 0) return 127;
  const int k = (int)(amax >> 23);
  if (k == 255) return 255;
  const uint32_t m = amax & 0x7fffffu;
  const int e = kStore == MOBA_STORE_E4M3 ? k - 8 + (m > 0x600000u) : k - 6 + (m > 0x7e0000u);
  return (uint32_t)max(e, kPagedLeastByte);
}

// 8 elements -> 8 codes.  x * 2^-e is exact (or far below a code's step), so that a code is rounded once.
template <bool kHalf, int kStore>
__device__ __forceinline__ uint2 encode8(uint4 x, uint32_t byte) {
  if (byte == 255) return make_uint2(0, 0);                // 0 * 2^128 reads back as NaN
  // what a code may stand for at most: the next one up would be an infinity of the 16-bit type
  constexpr float kMost = kStore == MOBA_STORE_E4M3 ? (kHalf ? 61440.f : 0x1.ep127f) : (kHalf ? 64512.f : 0x1.f8p127f);
  const float inv = __uint_as_float((254u - byte) << 23);
  float f[8];
  unpack8<kHalf>(x, f);
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = fminf(fmaxf(f[4 * h + i], -kMost), kMost) * inv;
    if (kStore == MOBA_STORE_E4M3) {
      const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(y[0], y[1]), __NV_SATFINITE, __NV_E4M3);
      const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(y[2], y[3]), __NV_SATFINITE, __NV_E4M3);
      w[h] = lo | hi << 16;
    } else {
      w[h] = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[h] |= (uint32_t)(__float2int_rn(y[i]) & 255) << (8 * i);
    }
  }
  return make_uint2(w[0], w[1]);
}

// 8 codes -> 8 elements
template <bool kHalf, int kStore>
__device__ __forceinline__ uint4 decode8(uint2 c, uint32_t byte) {
  const float s = paged_scale(byte);
  const uint32_t w[2] = {c.x, c.y};
  uint32_t o[4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float f[4];
    if (kStore == MOBA_STORE_E4M3) {
      const __half2_raw lo = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[h] & 0xffff), __NV_E4M3);
      const __half2_raw hi = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[h] >> 16), __NV_E4M3);
      const float2 a = __half22float2(__half2(lo)), b = __half22float2(__half2(hi));
      f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = (float)(int8_t)(w[h] >> (8 * i));
    }
    o[2 * h] = pack2_16<kHalf>(f[0] * s, f[1] * s);
    o[2 * h + 1] = pack2_16<kHalf>(f[2] * s, f[3] * s);
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

struct Place { int page, slot; };          // page < 0: nowhere

// Place of packed row `row` (the last sequence b with cu[b] <= row has it).
__device__ __forceinline__ Place place_of(const PagedParams& p, int64_t row) {
  Place at{-1, 0};
  if (row >= p.T) return at;
  int lo = 0, n = p.B;
  while (n > 1) {
    const int half = n >> 1;
    const bool up = __ldg(p.cu + lo + half) <= row;
    lo = up ? lo + half : lo;
    n = up ? n - half : half;
  }
  const PagedSeq s = paged_seq(p, lo);
  const int64_t i = row - s.row0;
  if (i < 0 || i >= s.n) return at;
  const int64_t pos = s.pos0 + i;
  if (pos < 0 || pos > 0x7fffffff) return at;
  at.page = paged_page(p, lo, (int)pos);
  at.slot = (int)pos & ((1 << p.page_shift) - 1);
  return at;
}

struct RowArgs {
  void *kp, *vp, *k, *v;
  uint8_t *ks, *vs;
  int units, heads;                        // warps of a token, heads of each
};

// The warp's tokens, heads and lane; rows of K and V of head h, token t of the warp: [t0 + t][h].
template <int D> struct RowWork {
  int64_t t0;
  int head0, sub, c;
  bool on;                                 // head dim 96: 12 of 16 lanes have elements
};
template <int D, int kTokens>
__device__ __forceinline__ bool row_work(const PagedParams& p, const RowArgs& a, RowWork<D>& w) {
  const int lane = threadIdx.x & 31;
  const int64_t g = (int64_t)blockIdx.x * (kRowThreads / 32) + (threadIdx.x >> 5);
  w.t0 = g / a.units * kTokens;
  w.head0 = (int)(g % a.units) * a.heads;
  w.sub = lane / kRowLanes<D>;
  w.c = (lane % kRowLanes<D>) * 8;
  w.on = w.c < D;
  return w.t0 < p.T;
}

template <bool kHalf, int D, int kStore, int kTokens>
__global__ void __launch_bounds__(kRowThreads) paged_store_kernel(const PagedParams p, const RowArgs a) {
  pdl_wait();
  pdl_trigger();
  RowWork<D> w;
  if (!row_work<D, kTokens>(p, a, w)) return;
  constexpr int kRows = 32 / kRowLanes<D>;                  // rows of a warp access
  const int lane = threadIdx.x & 31;
  const uint4 none = make_uint4(0, 0, 0, 0);
  Place mine{-1, 0};
  for (int h0 = w.head0; h0 < min(w.head0 + a.heads, p.Hkv); h0 += kRows) {
    const int h = h0 + w.sub;
    const bool on = w.on && h < p.Hkv;
    uint4 x[kTokens][2];
#pragma unroll
    for (int t = 0; t < kTokens; ++t) {
      const int64_t row = w.t0 + t;
      const bool got = on && row < p.T;
      x[t][0] = got ? __ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.k) + row * p.sk_t + h * p.sk_h + w.c)) : none;
      x[t][1] = got ? __ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.v) + row * p.sv_t + h * p.sv_h + w.c)) : none;
    }
    if (h0 == w.head0 && lane < kTokens) mine = place_of(p, w.t0 + lane);
#pragma unroll
    for (int t = 0; t < kTokens; ++t) {
      const int page = __shfl_sync(0xffffffffu, mine.page, t), slot = __shfl_sync(0xffffffffu, mine.slot, t);
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const int64_t at = kv == 0 ? page * p.kp_p + slot * p.kp_t + h * p.kp_h + w.c : page * p.vp_p + slot * p.vp_t + h * p.vp_h + w.c;
        void* pool = kv == 0 ? a.kp : a.vp;
        if (kStore == MOBA_STORE_SAME) {
          if (on && page >= 0) *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(pool) + at) = x[t][kv];
        } else {
          uint32_t amax = abs_bits_max<kHalf>(x[t][kv]);
#pragma unroll
          for (int o = kRowLanes<D> / 2; o > 0; o >>= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
          const uint32_t byte = row_byte<kStore>(amax);
          if (on && page >= 0) {
            *reinterpret_cast<uint2*>(static_cast<uint8_t*>(pool) + at) = encode8<kHalf, kStore>(x[t][kv], byte);
            if (w.c == 0) (kv == 0 ? a.ks : a.vs)[(((int64_t)page * p.Hkv + h) << p.page_shift) + slot] = (uint8_t)byte;
          }
        }
      }
    }
  }
}

template <bool kHalf, int D, int kStore, int kTokens>
__global__ void __launch_bounds__(kRowThreads) paged_load_kernel(const PagedParams p, const RowArgs a) {
  pdl_wait();
  pdl_trigger();
  RowWork<D> w;
  if (!row_work<D, kTokens>(p, a, w)) return;
  constexpr int kRows = 32 / kRowLanes<D>;
  const int lane = threadIdx.x & 31;
  Place mine{-1, 0};
  if (lane < kTokens) mine = place_of(p, w.t0 + lane);
  // rows behind the last sequence are left as they are
  const int64_t end = min((int64_t)__ldg(p.cu + p.B), p.T);
  for (int h0 = w.head0; h0 < min(w.head0 + a.heads, p.Hkv); h0 += kRows) {
    const int h = h0 + w.sub;
    const bool on = w.on && h < p.Hkv;
    uint4 x[kTokens][2];
    uint32_t byte[kTokens][2];
#pragma unroll
    for (int t = 0; t < kTokens; ++t) {
      const int page = __shfl_sync(0xffffffffu, mine.page, t), slot = __shfl_sync(0xffffffffu, mine.slot, t);
      const bool got = on && page >= 0;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const int64_t at = kv == 0 ? page * p.kp_p + slot * p.kp_t + h * p.kp_h + w.c : page * p.vp_p + slot * p.vp_t + h * p.vp_h + w.c;
        const void* pool = kv == 0 ? a.kp : a.vp;
        x[t][kv] = make_uint4(0, 0, 0, 0);
        byte[t][kv] = 127;
        if (got) {
          if (kStore == MOBA_STORE_SAME) {
            x[t][kv] = __ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(pool) + at));
          } else {
            const uint2 c = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(pool) + at));
            x[t][kv].x = c.x;
            x[t][kv].y = c.y;
            byte[t][kv] = __ldg((kv == 0 ? a.ks : a.vs) + (((int64_t)page * p.Hkv + h) << p.page_shift) + slot);
          }
        }
      }
    }
#pragma unroll
    for (int t = 0; t < kTokens; ++t) {
      const int64_t row = w.t0 + t;
      if (!on || row >= end) continue;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const uint4 y = kStore == MOBA_STORE_SAME ? x[t][kv]
                                                  : decode8<kHalf, kStore>(make_uint2(x[t][kv].x, x[t][kv].y), byte[t][kv]);
        __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(kv == 0 ? a.k : a.v) + (kv == 0 ? row * p.sk_t + h * p.sk_h : row * p.sv_t + h * p.sv_h) + w.c;
        *reinterpret_cast<uint4*>(dst) = y;
      }
    }
  }
}

typedef void (*RowKernel)(const PagedParams, const RowArgs);
constexpr int kManyLoad = 4, kManyStore = 2;   // tokens of a warp, where there are many

template <bool kHalf, int D, int kTokens>
RowKernel pick_store(bool load, int store) {
  if constexpr (kTokens != kManyStore) {
    if (load)
      return store == MOBA_STORE_SAME ? paged_load_kernel<kHalf, D, MOBA_STORE_SAME, kTokens>
           : store == MOBA_STORE_E4M3 ? paged_load_kernel<kHalf, D, MOBA_STORE_E4M3, kTokens>
                                      : paged_load_kernel<kHalf, D, MOBA_STORE_INT8, kTokens>;
  }
  if constexpr (kTokens == kManyLoad) return nullptr;
  else return store == MOBA_STORE_SAME ? paged_store_kernel<kHalf, D, MOBA_STORE_SAME, kTokens>
       : store == MOBA_STORE_E4M3 ? paged_store_kernel<kHalf, D, MOBA_STORE_E4M3, kTokens>
                                  : paged_store_kernel<kHalf, D, MOBA_STORE_INT8, kTokens>;
}
template <bool kHalf, int kTokens>
RowKernel pick_dim(bool load, int D, int store) {
  return D == 64 ? pick_store<kHalf, 64, kTokens>(load, store) : D == 96 ? pick_store<kHalf, 96, kTokens>(load, store)
       : D == 128 ? pick_store<kHalf, 128, kTokens>(load, store) : pick_store<kHalf, 256, kTokens>(load, store);
}
template <int kTokens>
RowKernel pick_row_kernel(bool load, const PagedParams& p) {
  // (rows that are copied as they are have no type)
  return p.fp16 && p.store != MOBA_STORE_SAME ? pick_dim<true, kTokens>(load, p.D, p.store) : pick_dim<false, kTokens>(load, p.D, p.store);
}

cudaError_t launch_rows(bool load, const PagedParams& p, RowArgs a, cudaStream_t st) {
  const int rows = 32 * 8 / (p.D == 96 ? 128 : p.D);        // heads of one warp access
  // A few tokens a warp where that still gives every SM its warps: more loads under way.  Four rows read back at a time, two written (131072 tokens
  // of e4m3 read back, 8 heads of 128: 1 165, 2 165, 4 144, 8 148 us; 8191 written to int8 and read back, written by 4 30.5, by 2 28.1).
  const int passes = (p.Hkv + rows - 1) / rows, several = load ? kManyLoad : kManyStore;
  const bool many = p.T * passes >= (int64_t)several * 148 * 64;
  a.units = passes;
  a.heads = rows;
  const int64_t warps = (p.T + (many ? several : 1) - 1) / (many ? several : 1) * a.units;
  const int64_t blocks = (warps + kRowThreads / 32 - 1) / (kRowThreads / 32);
  return launch_pdl(!many ? pick_row_kernel<1>(load, p) : load ? pick_row_kernel<kManyLoad>(load, p) : pick_row_kernel<kManyStore>(load, p), dim3((unsigned)blocks), kRowThreads, 0, st, p, a);
}

}  // namespace

cudaError_t launch_paged_store(const PagedParams& p, const void* k, const void* v, void* kp, void* vp, uint8_t* ks, uint8_t* vs,
                               cudaStream_t st) {
  return launch_rows(false, p, RowArgs{kp, vp, const_cast<void*>(k), const_cast<void*>(v), ks, vs, 0, 0}, st);
}
cudaError_t launch_paged_load(const PagedParams& p, const void* kp, const void* vp, const uint8_t* ks, const uint8_t* vs, void* k,
                              void* v, cudaStream_t st) {
  return launch_rows(true, p, RowArgs{const_cast<void*>(kp), const_cast<void*>(vp), k, v, const_cast<uint8_t*>(ks),
                                      const_cast<uint8_t*>(vs), 0, 0}, st);
}

}  // namespace moba
