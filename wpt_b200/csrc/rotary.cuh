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
// p f in fp32 is off by 2^-24 p f radians (0.03 at a million); what is left
// is the rounding of f / (2 pi) to double, 2^-53 p f, and of the fraction of
// half a turn to fp32, 2^-25, before sincospif.
#pragma once

#include <cstdint>

#include "common.cuh"

namespace wpt {

// A frequency (radians a position) in 2^-64 turns a position.
__device__ __forceinline__ uint64_t turn_of(double f) {
  double t = f * 0.15915494309189535;  // 1 / (2 pi)
  t -= floor(t);
  return __double2ull_rz(t * 18446744073709551616.0);
}

// sin and cos of position p at `turn` 2^-64 turns a position.
__device__ __forceinline__ void turn_sincos(int64_t p, uint64_t turn, float& s, float& c) {
  const int32_t a = static_cast<int32_t>((static_cast<uint64_t>(p) * turn) >> 32);  // -1/2 .. 1/2 turn
  sincospif(static_cast<float>(a) * 4.656612873077393e-10f, &s, &c);                // 2^-31 half turns
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
  int items, lanes;             // items of a head; heads go over `lanes` threads
  int f64;
  float sign, magnitude;        // sign -1: the gradient's turn
};

__device__ __forceinline__ uint64_t rotate_turn(const void* frequencies, int f64, int i) {
  return turn_of(f64 ? static_cast<const double*>(frequencies)[i]
                     : static_cast<double>(static_cast<const float*>(frequencies)[i]));
}

// A thread owns one item of a token (a vector of VE channels; with halves, the
// vector and its partner `dims / 2` on), works out its angles once and walks
// the heads h = lane, lane + lanes, ... Neighbouring threads take
// neighbouring items, then heads, so a warp reads and writes whole lines.
template <class T, int VE, bool INTERLEAVED>
__global__ void __launch_bounds__(256) rotate_kernel(const RotateParams p) {
  using V = Vec<T, VE>;
  using Raw = typename V::Raw;
  griddep_wait();
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= p.total) return;
  const int64_t lane_at = i / p.items;
  const int item = static_cast<int>(i - lane_at * p.items);
  const int64_t token = lane_at / p.lanes;
  const int lane = static_cast<int>(lane_at - token * p.lanes);
  const int64_t b = token / p.T, t = token - b * p.T;
  // items: the turned ones, then the copied ones (before `start`, then behind)
  constexpr int PAIRS = INTERLEAVED && VE > 1 ? VE / 2 : VE;  // pairs of an item
  const int half = p.dims >> 1;
  const int turned = half / PAIRS;
  const T* x = static_cast<const T*>(p.x) + b * p.xsb + t * p.xst;
  T* y = static_cast<T*>(p.y) + token * p.H * p.C;
  const int64_t xstep = p.xsh, ystep = p.C;
  if (item >= turned) {
    int c = (item - turned) * VE;
    if (c >= p.start) c += p.dims;
    constexpr int U = 4;
    for (int h0 = lane; h0 < p.H; h0 += U * p.lanes) {
      Raw r[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (h0 + u * p.lanes < p.H) r[u] = *reinterpret_cast<const Raw*>(x + (h0 + u * p.lanes) * xstep + c);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (h0 + u * p.lanes < p.H) *reinterpret_cast<Raw*>(y + (h0 + u * p.lanes) * ystep + c) = r[u];
    }
    return;
  }
  const int64_t pos = p.positions[b * p.psb + t];
  float sn[PAIRS], cs[PAIRS];
#pragma unroll
  for (int k = 0; k < PAIRS; ++k) {
    turn_sincos(pos, rotate_turn(p.frequencies, p.f64, item * PAIRS + k), sn[k], cs[k]);
    sn[k] *= p.sign;
  }
  const float m = p.magnitude;
  constexpr bool ONE = INTERLEAVED && VE > 1;  // an item is one vector of whole pairs
  const int ca = p.start + (INTERLEAVED ? 2 * PAIRS : PAIRS) * item;
  const int cb = INTERLEAVED ? ca + 1 : ca + half;
  constexpr int U = 2;
  for (int h0 = lane; h0 < p.H; h0 += U * p.lanes) {
    Raw ra[U], rb[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (h0 + u * p.lanes < p.H) {
        const T* at = x + (h0 + u * p.lanes) * xstep;
        ra[u] = *reinterpret_cast<const Raw*>(at + ca);
        if constexpr (!ONE) rb[u] = *reinterpret_cast<const Raw*>(at + cb);
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (h0 + u * p.lanes < p.H) {
        T* at = y + (h0 + u * p.lanes) * ystep;
        float a[VE], o[VE];
        V::widen(ra[u], a);
        if constexpr (ONE) {
#pragma unroll
          for (int k = 0; k < PAIRS; ++k) {
            turn_pair(a[2 * k], a[2 * k + 1], sn[k], cs[k], o[2 * k], o[2 * k + 1]);
            o[2 * k] *= m;
            o[2 * k + 1] *= m;
          }
        } else {
          float z[VE], q[VE];
          V::widen(rb[u], z);
#pragma unroll
          for (int k = 0; k < VE; ++k) {
            turn_pair(a[k], z[k], sn[k], cs[k], o[k], q[k]);
            o[k] *= m;
            q[k] *= m;
          }
          *reinterpret_cast<Raw*>(at + cb) = V::round(q);
        }
        *reinterpret_cast<Raw*>(at + ca) = V::round(o);
      }
  }
}

}  // namespace wpt
