// Rotary positions of queries and keys: pair j of a head's first `turned` dims, (x, y), becomes
//     m (x cos a - y sin a), m (x sin a + y cos a)      with a = position * frequency[j]
// where a pair is dims j and j + turned / 2, or 2 j and 2 j + 1.  The gradient is the turn by -a.
//
// An angle far from 0 has few digits left in 32 bits (position 10^6: 0.06 radians).  Here a frequency is a part of a whole turn in 64 bits of fixed
// point; position * frequency modulo 2^64 drops whole turns exactly, and its upper 32 bits, an angle of -1/2 to 1/2 turns, go to sincospif.  So the
// error of an angle is that of the frequency, 2^-65 turns a position, and a rounding of the reduced angle to 24 bits.
//
// Bound by bytes: rows in, rows out.  A warp has a token and some of its heads; a lane has a few pairs of a head (16 bytes of each half), works out their
// sines once and goes from head to head with them; lanes that lie a head apart have the same ones.
// Measured (replayed from a graph): 16384 tokens of 32/8 heads of 128, all of each turned 57.5 us, 89 % of the measured copy bandwidth; half of each, there and
// back 111 us, 92 %; 64 tokens 4.2 us, which is the launch and two dependent loads.
#include "rotary.cuh"

#include "common.cuh"

namespace moba {
namespace {

// (16384 tokens of 32/8 heads of 128, us: one head of a lane under way 64, two 57.5, four 58; 256 threads a block 57.5, at head dim 96 47.7 for 47.2)
constexpr int kThreads = 128, kWarps = kThreads / 32;
constexpr int kHeads = 2;                  // of a lane under way

// kPairs: of a lane.  Untouched dims are copied, as many as two halves of a lane's at a time.
template <int kPairs> struct Piece;
template <> struct Piece<8> { using Word = uint4; };
template <> struct Piece<4> { using Word = uint2; };
template <> struct Piece<1> { using Word = uint16_t; };

template <bool kHalf, int kPairs>
__device__ __forceinline__ void widen(const typename Piece<kPairs>::Word& w, float (&f)[kPairs]) {
  if constexpr (kPairs == 8) {
    unpack8<kHalf>(w, f);
  } else if constexpr (kPairs == 4) {
    const float2 a = unpack2<kHalf>(w.x), b = unpack2<kHalf>(w.y);
    f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
  } else {
    f[0] = unpack2<kHalf>((uint32_t)w).x;
  }
}
template <bool kHalf, int kPairs>
__device__ __forceinline__ typename Piece<kPairs>::Word narrow(const float (&f)[kPairs]) {
  if constexpr (kPairs == 8) {
    return make_uint4(pack2_16<kHalf>(f[0], f[1]), pack2_16<kHalf>(f[2], f[3]), pack2_16<kHalf>(f[4], f[5]), pack2_16<kHalf>(f[6], f[7]));
  } else if constexpr (kPairs == 4) {
    return make_uint2(pack2_16<kHalf>(f[0], f[1]), pack2_16<kHalf>(f[2], f[3]));
  } else {
    return (uint16_t)pack2_16<kHalf>(f[0], 0.f);
  }
}

template <bool kHalf, int kPairs, bool kInterleaved>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryParams p) {
  using Word = typename Piece<kPairs>::Word;
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const int64_t g = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  const int64_t row = g / p.units;
  if (row >= p.rows) return;
  const int unit = (int)(g - row * p.units), heads = p.heads_q + p.heads_k;
  const int sub = lane / p.lanes, abreast = 32 / p.lanes;
  const int pos = __ldg(p.positions + row);
  const int last = min((unit + 1) * p.per_unit, heads);
  for (int slot = lane % p.lanes; slot < p.slots; slot += p.lanes) {
    const int j0 = slot * kPairs;                           // first pair, or (behind the turned ones) two pieces of other dims
    const bool turned = 2 * j0 < p.turned;
    const int at0 = turned && !kInterleaved ? j0 : 2 * j0, at1 = turned && !kInterleaved ? j0 + p.turned / 2 : 2 * j0 + kPairs;
    const bool turn = turned && pos >= 0;                   // (a row of no sequence has no position)
    float c[kPairs], s[kPairs];
    if (turn) {
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        const unsigned long long a = (unsigned long long)__ldg(p.turns + j0 + i) * (unsigned long long)(long long)pos;
        const int part = (int)((a + 0x80000000ull) >> 32);
        sincospif((float)part * 0x1p-31f, &s[i], &c[i]);
        c[i] *= p.magnitude;
        s[i] *= p.inverse ? -p.magnitude : p.magnitude;
      }
    }
    // (loads of kHeads heads before their stores: rows may be turned where they are, so that the compiler does not bring loads forward)
    for (int h0 = unit * p.per_unit + sub; h0 < last; h0 += kHeads * abreast) {
      Word w[kHeads][2];
      uint16_t* to[kHeads];
#pragma unroll
      for (int k = 0; k < kHeads; ++k) {
        const int h = h0 + k * abreast, hh = h < p.heads_q ? h : h - p.heads_q;
        to[k] = nullptr;
        if (h >= last) continue;
        const bool of_q = h < p.heads_q;
        const uint16_t* src = static_cast<const uint16_t*>(of_q ? p.q : p.k) + (of_q ? row * p.q_t + hh * p.q_h : row * p.k_t + hh * p.k_h);
        to[k] = static_cast<uint16_t*>(of_q ? p.q_out : p.k_out) + (of_q ? row * p.qo_t + hh * p.qo_h : row * p.ko_t + hh * p.ko_h);
        w[k][0] = *reinterpret_cast<const Word*>(src + at0);
        w[k][1] = *reinterpret_cast<const Word*>(src + at1);
      }
#pragma unroll
      for (int k = 0; k < kHeads; ++k) {
        if (to[k] == nullptr) continue;
        if (turn) {
          float f0[kPairs], f1[kPairs];
          widen<kHalf, kPairs>(w[k][0], f0);
          widen<kHalf, kPairs>(w[k][1], f1);
          float x[2 * kPairs];                              // both pieces
#pragma unroll
          for (int i = 0; i < kPairs; ++i) { x[i] = f0[i]; x[kPairs + i] = f1[i]; }
#pragma unroll
          for (int i = 0; i < kPairs; ++i) {
            const int a = kInterleaved ? 2 * i : i, b = kInterleaved ? 2 * i + 1 : kPairs + i;
            const float u = x[a], v = x[b];
            x[a] = u * c[i] - v * s[i];
            x[b] = u * s[i] + v * c[i];
          }
#pragma unroll
          for (int i = 0; i < kPairs; ++i) { f0[i] = x[i]; f1[i] = x[kPairs + i]; }
          w[k][0] = narrow<kHalf, kPairs>(f0);
          w[k][1] = narrow<kHalf, kPairs>(f1);
        }
        *reinterpret_cast<Word*>(to[k] + at0) = w[k][0];
        *reinterpret_cast<Word*>(to[k] + at1) = w[k][1];
      }
    }
  }
}

typedef void (*RotaryKernel)(const RotaryParams);
template <bool kHalf, int kPairs>
RotaryKernel pick_form(bool interleaved) { return interleaved ? rotary_kernel<kHalf, kPairs, true> : rotary_kernel<kHalf, kPairs, false>; }
template <bool kHalf>
RotaryKernel pick_kernel(int pairs, bool interleaved) {
  return pairs == 8 ? pick_form<kHalf, 8>(interleaved) : pairs == 4 ? pick_form<kHalf, 4>(interleaved) : pick_form<kHalf, 1>(interleaved);
}

}  // namespace

cudaError_t launch_rotary(RotaryParams p, cudaStream_t st) {
  // the widest piece that the turned dims' halves, and what lies behind them, are whole numbers of
  const int pairs = p.turned % 16 == 0 ? 8 : p.turned % 8 == 0 ? 4 : 1;
  p.slots = p.dim / (2 * pairs);
  p.lanes = 1;
  while (p.lanes < p.slots && p.lanes < 32) p.lanes *= 2;
  const int heads = p.heads_q + p.heads_k, abreast = 32 / p.lanes;
  // as many warps a token as its heads give, where there are few tokens; else one, so that its sines are worked out once
  const int most = (heads + abreast - 1) / abreast;
  int64_t units = (148 * 16 + p.rows - 1) / p.rows;
  units = units < most ? units : most;
  p.per_unit = (int)((most + units - 1) / units) * abreast;
  p.units = (heads + p.per_unit - 1) / p.per_unit;
  const int64_t warps = p.rows * p.units;
  const RotaryKernel kernel = p.fp16 ? pick_kernel<true>(pairs, p.interleaved != 0) : pick_kernel<false>(pairs, p.interleaved != 0);
  return launch_pdl(kernel, dim3((unsigned)((warps + kWarps - 1) / kWarps)), kThreads, 0, st, p);
}

}  // namespace moba
