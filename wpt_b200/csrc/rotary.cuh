// Rotary positions: pairs of channels (a, b) of a head turned by an angle
// that grows with the token's position p,
//
//   y_a = m (x_a cos t - x_b sin t),  y_b = m (x_b cos t + x_a sin t),  t = p f_i,
//
// pair i of `dims / 2` either (start + i, start + dims / 2 + i) (halves) or
// (start + 2 i, start + 2 i + 1) (interleaved); channels outside start ..
// start + dims - 1 are copied. The window layers of WPT turn the last 64
// channels of queries and keys (packages/wpt-model/src/wpt_model/
// attention.py:59). The gradient of x is the same turn by -t.
//
// Angles. A position is whole, so p f in turns, modulo a turn, is a product
// of whole numbers that wraps: f / (2 pi) as a fraction of 2^64 (turn_of), times
// p, modulo 2^64 (turn_sincos). The product is exact at any position, where
// p f in fp32 is off by 2^-24 p f radians (0.03 at a million). What is left, in
// radians: 2^-52 p f, since f / (2 pi) is rounded to double twice (the constant
// and the product); 2 pi 2^-65 p, since its fraction of a turn is rounded to
// 2^-64 (2e-13 at a million positions, 2e-7 at 2^40: what grows for slow pairs);
// and 2 pi 2^-32, of which the phase is cut. The nearest quarter turn is taken off
// in whole numbers too, and sine and cosine of the rest, |x| <= pi / 4, are
// their Taylor series: to x^9 and x^10, whose next terms are under 1.8e-9 and
// 1.2e-10 there (the math library's function, made for any argument, took five
// times the instructions).
#pragma once

#include <cstdint>

#include "common.cuh"

namespace wpt {

// A frequency (radians a position) in 2^-64 turns a position. (By its size: 1
// less a small number would keep 2^-54 of it.)
__device__ __forceinline__ uint64_t turn_of(double f) {
  double t = fabs(f) * 0.15915494309189535;  // 1 / (2 pi)
  t -= floor(t);
  const uint64_t turn = __double2ull_rn(t * 18446744073709551616.0);
  return f < 0.0 ? 0 - turn : turn;
}

// sin and cos of position p at `turn` 2^-64 turns a position.
__device__ __forceinline__ void turn_sincos(int64_t p, uint64_t turn, float& s, float& c) {
  const uint32_t a = static_cast<uint32_t>((static_cast<uint64_t>(p) * turn) >> 32);  // 2^-32 turns
  const uint32_t q = (a + 0x20000000u) >> 30;                                          // quarter turns, to the nearest
  const float x = static_cast<float>(static_cast<int32_t>(a - (q << 30))) * 1.4629180792671596e-9f;  // 2 pi 2^-32
  const float z = x * x;
  float u = fmaf(z, 2.7557319e-6f, -1.9841270e-4f);  // 1 / 9!, -1 / 7!, 1 / 5!, -1 / 3!
  u = fmaf(z, u, 8.3333333e-3f);
  u = fmaf(z, u, -1.6666667e-1f);
  u = fmaf(z * x, u, x);
  float w = fmaf(z, -2.7557319e-7f, 2.4801587e-5f);  // -1 / 10!, 1 / 8!, -1 / 6!, 1 / 4!, -1 / 2!
  w = fmaf(z, w, -1.3888889e-3f);
  w = fmaf(z, w, 4.1666667e-2f);
  w = fmaf(z, w, -0.5f);
  w = fmaf(z, w, 1.f);
  const float ss = (q & 1u) ? w : u, cc = (q & 1u) ? u : w;
  s = __uint_as_float(__float_as_uint(ss) ^ ((q & 2u) << 30));
  c = __uint_as_float(__float_as_uint(cc) ^ (((q + 1u) & 2u) << 30));
}

// One pair's turn. The products are rounded before their sum, as elementary
// fp32 operations round them, not fused.
__device__ __forceinline__ void turn_pair(float a, float b, float s, float c, float& ya, float& yb) {
  ya = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
  yb = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
}

// VE consecutive elements of T as one access, widened to and rounded from fp32.
template <class T, int VE>
struct Vec;
template <>
struct Vec<__nv_bfloat16, 8> {
  using Raw = uint4;
  static __device__ __forceinline__ void widen(const uint4& r, float* x) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint4 round(const float* x) {
    return make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
  }
  static __device__ __forceinline__ uint4 from_lane(const uint4& r, int lane) {  // the whole warp
    return make_uint4(__shfl_sync(0xffffffffu, r.x, lane), __shfl_sync(0xffffffffu, r.y, lane),
                      __shfl_sync(0xffffffffu, r.z, lane), __shfl_sync(0xffffffffu, r.w, lane));
  }
};
template <>
struct Vec<float, 4> {
  using Raw = float4;
  static __device__ __forceinline__ void widen(const float4& r, float* x) {
    x[0] = r.x;
    x[1] = r.y;
    x[2] = r.z;
    x[3] = r.w;
  }
  static __device__ __forceinline__ float4 round(const float* x) { return make_float4(x[0], x[1], x[2], x[3]); }
  static __device__ __forceinline__ float4 from_lane(const float4& r, int lane) {
    return make_float4(__shfl_sync(0xffffffffu, r.x, lane), __shfl_sync(0xffffffffu, r.y, lane),
                       __shfl_sync(0xffffffffu, r.z, lane), __shfl_sync(0xffffffffu, r.w, lane));
  }
};
template <>
struct Vec<__nv_bfloat16, 2> {
  using Raw = uint32_t;
  static __device__ __forceinline__ void widen(const Raw& r, float* x) {
    x[0] = __uint_as_float(r << 16);
    x[1] = __uint_as_float(r & 0xffff0000u);
  }
  static __device__ __forceinline__ Raw round(const float* x) { return pack_bf16(x[0], x[1]); }
};
template <>
struct Vec<float, 2> {
  using Raw = float2;
  static __device__ __forceinline__ void widen(const Raw& r, float* x) {
    x[0] = r.x;
    x[1] = r.y;
  }
  static __device__ __forceinline__ Raw round(const float* x) { return make_float2(x[0], x[1]); }
};
template <>
struct Vec<__nv_bfloat16, 1> {
  using Raw = __nv_bfloat16;
  static __device__ __forceinline__ void widen(const Raw& r, float* x) { x[0] = __bfloat162float(r); }
  static __device__ __forceinline__ Raw round(const float* x) { return __float2bfloat16_rn(x[0]); }
};
template <>
struct Vec<float, 1> {
  using Raw = float;
  static __device__ __forceinline__ void widen(const Raw& r, float* x) { x[0] = r; }
  static __device__ __forceinline__ Raw round(const float* x) { return x[0]; }
};

struct RotateParams {
  const void* x;
  void* y;                      // (B, T, H, C) contiguous
  int64_t xsb, xst, xsh;        // strides of x, elements
  const int64_t* positions;     // positions[b * psb + t]
  int64_t psb;
  const void* frequencies;      // (dims / 2,) fp64, or fp32
  int64_t total;                // threads with work: B T lanes items
  int T, H, C, dims, start;
  unsigned items, lanes;        // items of a head; heads go over `lanes` threads
  int f64;
  float sign, magnitude;        // sign -1: the gradient's turn
};

__device__ __forceinline__ uint64_t rotate_turn(const void* frequencies, int f64, int i) {
  return turn_of(f64 ? static_cast<const double*>(frequencies)[i]
                     : static_cast<double>(static_cast<const float*>(frequencies)[i]));
}

// The block's frequencies as turns, in shared memory (dims / 2 of them): a
// thread's own would be up to 8 conversions from fp64 each.
__device__ __forceinline__ void turns_of(const RotateParams& p, uint64_t* s_turns) {
  for (int k = threadIdx.x; k < p.dims / 2; k += blockDim.x) s_turns[k] = rotate_turn(p.frequencies, p.f64, k);
  __syncthreads();
}

// Thread i's item (the fastest), head lane, and token (b, t). Divisions of 32 bits
// where they do, as nearly always: three of 64 took more than all else in a thread.
struct RotateAt {
  int item, lane;
  int64_t token, b, t;
  __device__ __forceinline__ RotateAt(const RotateParams& p, int64_t i) {
    if (p.total <= 0x7fffffff) {
      const unsigned n = static_cast<unsigned>(i), lane_at = n / p.items;
      item = n - lane_at * p.items;
      const unsigned at = lane_at / p.lanes;
      lane = lane_at - at * p.lanes;
      token = at;
      b = at / static_cast<unsigned>(p.T);
    } else {
      const int64_t lane_at = i / p.items;
      item = static_cast<int>(i - lane_at * p.items);
      token = lane_at / p.lanes;
      lane = static_cast<int>(lane_at - token * p.lanes);
      b = token / p.T;
    }
    t = token - b * p.T;
  }
};

// A thread owns one item of a token (a vector of VE channels; with halves, the
// vector and its partner `dims / 2` on), works out its angles once and walks
// the heads h = lane, lane + lanes, ... Neighbouring threads take
// neighbouring items, then heads, so a warp reads and writes whole lines.
// Channels that do not turn: COPIES vectors ride along with each item where they
// come out even (0, 1 or 2: all lanes then do the same work and have 2 to 4
// loads in flight for each of two heads); else (-1) they are items of their own.
// Bound by HBM: 8 x 4,096 tokens of 16 heads of 128, 64 turned (134 MB in, 134
// out) take 44 us, 6.1 TB/s. A vector a thread, its partner from the lane that owns it (51 us there)
// or from L1 (67 us: it was read from L2 twice), was no faster.
template <class T, int VE, bool INTERLEAVED, int COPIES>
__global__ void __launch_bounds__(256) rotate_kernel(const RotateParams p) {
  using V = Vec<T, VE>;
  using Raw = typename V::Raw;
  extern __shared__ uint64_t s_turns[];
  griddep_wait();
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const bool mine = at < p.total;  // the last block's other threads help with the turns
  const RotateAt where(p, mine ? at : p.total - 1);
  const int item = where.item, lane = where.lane, lanes = p.lanes;
  constexpr bool WHOLE = INTERLEAVED && VE > 1;  // a vector holds whole pairs
  constexpr int PAIRS = WHOLE ? VE / 2 : VE;     // pairs of an item
  const int half = p.dims >> 1, turned = half / PAIRS;
  const T* x = static_cast<const T*>(p.x) + where.b * p.xsb + where.t * p.xst;
  T* y = static_cast<T*>(p.y) + where.token * p.H * p.C;
  if constexpr (COPIES < 0) {
    turns_of(p, s_turns);  // all threads, before they part
    if (!mine) return;
  }
  if (COPIES < 0 && item >= turned) {
    int c = (item - turned) * VE;
    if (c >= p.start) c += p.dims;
    constexpr int U = 4;
    for (int h0 = lane; h0 < p.H; h0 += U * lanes) {
      Raw r[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (h0 + u * lanes < p.H) r[u] = *reinterpret_cast<const Raw*>(x + (h0 + u * lanes) * p.xsh + c);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (h0 + u * lanes < p.H) *reinterpret_cast<Raw*>(y + static_cast<int64_t>(h0 + u * lanes) * p.C + c) = r[u];
    }
    return;
  }
  constexpr int K = COPIES > 0 ? COPIES : 0, U = 2;
  const int ca = p.start + (INTERLEAVED ? 2 * PAIRS : PAIRS) * item;
  const int cb = INTERLEAVED ? ca + 1 : ca + half;
  int cc[K > 0 ? K : 1];  // the copied vectors: item, item + turned, ... of those that do not turn
#pragma unroll
  for (int k = 0; k < K; ++k) {
    cc[k] = (item + k * turned) * VE;
    if (cc[k] >= p.start) cc[k] += p.dims;
  }
  Raw ra[U], rb[U], rc[U][K > 0 ? K : 1];
  auto load = [&](int h0) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (h0 + u * lanes < p.H) {
        const T* from = x + (h0 + u * lanes) * p.xsh;
        ra[u] = *reinterpret_cast<const Raw*>(from + ca);
        if constexpr (!WHOLE) rb[u] = *reinterpret_cast<const Raw*>(from + cb);
#pragma unroll
        for (int k = 0; k < K; ++k) rc[u][k] = *reinterpret_cast<const Raw*>(from + cc[k]);
      }
  };
  load(lane);  // in flight while the angles are worked out
  const int64_t pos = p.positions[where.b * p.psb + where.t];
  if constexpr (COPIES >= 0) {
    turns_of(p, s_turns);
    if (!mine) return;
  }
  float sn[PAIRS], cs[PAIRS];
#pragma unroll
  for (int k = 0; k < PAIRS; ++k) {
    turn_sincos(pos, s_turns[item * PAIRS + k], sn[k], cs[k]);
    sn[k] *= p.sign;
  }
  const float m = p.magnitude;
  for (int h0 = lane; h0 < p.H; h0 += U * lanes) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (h0 + u * lanes < p.H) {
        T* to = y + static_cast<int64_t>(h0 + u * lanes) * p.C;
        float a[VE], z[VE];
        V::widen(ra[u], a);
        if constexpr (!WHOLE) V::widen(rb[u], z);
#pragma unroll
        for (int k = 0; k < PAIRS; ++k) {
          float& one = a[WHOLE ? 2 * k : k];
          float& two = WHOLE ? a[WHOLE ? 2 * k + 1 : 0] : z[k];
          float o, q;
          turn_pair(one, two, sn[k], cs[k], o, q);
          one = o * m;
          two = q * m;
        }
        *reinterpret_cast<Raw*>(to + ca) = V::round(a);
        if constexpr (!WHOLE) *reinterpret_cast<Raw*>(to + cb) = V::round(z);
#pragma unroll
        for (int k = 0; k < K; ++k) *reinterpret_cast<Raw*>(to + cc[k]) = rc[u][k];
      }
    load(h0 + U * lanes);
  }
}

}  // namespace wpt
