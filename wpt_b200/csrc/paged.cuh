// The paged generation cache held in 8 bits, and attention over it.
//
// Layout. pages (P, S, 2 C) e4m3: an entry's key, then its value, as in the
// plain entries table (packages/wpt-model/src/wpt_model/cache.py:110-128), S
// entries a page. scales (P, S / 16, 2) fp32: block k of a page (its entries
// 16 k .. 16 k + 15) stands for scales[k][0] * keys and scales[k][1] * values.
// Entry n of batch row b is entry n % S of page table[b, n / S].
//
// Scales are powers of two: e4m3 keeps its 4 significant bits whatever the
// scale, so a finer scale would gain nothing, multiplying by one is exact, and
// a block whose scale grows loses only what falls under its new smallest step.
#pragma once

#include "rotary.cuh"

namespace wpt {

constexpr int PAGE_BLOCK = 16;  // entries that share a scale

// cvt to a pair of e4m3 (lo in the low byte), to nearest even; finite values past 448 become 448
__device__ __forceinline__ uint32_t pack_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t pack_e4m3x4(float a, float b, float c, float d) {
  return pack_e4m3x2(a, b) | (pack_e4m3x2(c, d) << 16);
}
// both e4m3 of a pair, as fp16 (exact)
__device__ __forceinline__ uint32_t unpack_e4m3x2(uint32_t pair) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(pair)));
  return r;
}
__device__ __forceinline__ float half_lo(uint32_t h) {
  float f;
  asm("{\n\t.reg .f16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.f32.f16 %0, l;\n\t}" : "=f"(f) : "r"(h));
  return f;
}
__device__ __forceinline__ float half_hi(uint32_t h) {
  float f;
  asm("{\n\t.reg .f16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.f32.f16 %0, h;\n\t}" : "=f"(f) : "r"(h));
  return f;
}

// The exponent of the least power of two 2^e with |x| <= 448 * 2^e, at least
// `least`, from the bits of |x| (448 = 1.75 * 2^8).
__device__ __forceinline__ int scale_exponent(uint32_t abs_bits, int least) {
  const int e = static_cast<int>(abs_bits >> 23) - 135 + ((abs_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e > least ? e : least;
}
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }

constexpr int SCALE_LEAST = -60;
constexpr uint32_t SCALE_TOP_BITS = (60u + 8u + 127u) << 23 | 0x600000u;  // 448 * 2^60: larger values count as infinite

struct AppendParams {
  const void* src;                 // new entries: (B, n, 2 C)
  int64_t ssb, ssn;                // strides, elements
  uint8_t* pages;
  int64_t psp, psr;                // strides of a page and of an entry, bytes
  float* scales;
  int64_t scp;                     // stride of a page's scales, elements
  const void* table;               // (B, M) int32 or int64
  int64_t tsb;
  const int64_t* first;            // (B,)
  const int64_t* counts;           // (B,)
  const int64_t* positions;        // (B, n) or null: first + i
  const void* frequencies;         // (dims / 2,) or null
  unsigned* status;
  int t64, f64;
  int B, n, C, M, P, S, dims, start;
  int blocks;                      // grid blocks a row
  float magnitude;
};

__device__ __forceinline__ int64_t page_of(const void* table, int t64, int64_t at, int P) {
  const int64_t id = t64 ? static_cast<const int64_t*>(table)[at] : static_cast<const int32_t*>(table)[at];
  return id >= 0 && id < P ? id : -1;
}

// Appending. One CTA a block of 16 entries (and batch row), so a block's scale
// needs no exchange: the block's new entries are turned, widened to fp32 in
// shared memory, their largest value gives the scale, and a second pass
// rounds them. Bound by HBM for prompts; a step of one entry a row is a chain
// of three loads (first, the page's number, its scale).
template <class T, int VE, bool INTERLEAVED>
__global__ void __launch_bounds__(128) paged_append_kernel(const AppendParams p) {
  using V = Vec<T, VE>;
  using Raw = typename V::Raw;
  extern __shared__ float s_val[];  // (16, 2 C)
  __shared__ uint32_t s_red[4][2];
  griddep_wait();
  const int b = blockIdx.x / p.blocks;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t capacity = static_cast<int64_t>(p.M) * p.S;
  const int64_t first = p.first[b];
  int64_t count = p.counts[b];
  if (count > p.n) count = p.n;
  if (count <= 0) return;
  // entries lo .. hi - 1 of the row are new; those outside the table are dropped
  const bool out = first < 0 || first > capacity - count;
  int64_t lo = first < 0 ? 0 : first, hi = first > capacity - count ? capacity : first + count;
  const int64_t block = lo / PAGE_BLOCK + (blockIdx.x - b * p.blocks);
  if (out && tid == 0 && blockIdx.x == b * p.blocks) atomicOr(p.status, STATUS_BAD_SHAPE);
  const int64_t n0 = block * PAGE_BLOCK;
  if (n0 >= hi) return;
  const int64_t begun = lo;  // entries before it are earlier ones
  if (lo < n0) lo = n0;
  if (hi > n0 + PAGE_BLOCK) hi = n0 + PAGE_BLOCK;
  const int64_t page = page_of(p.table, p.t64, b * p.tsb + n0 / p.S, p.P);
  if (page < 0) {
    if (tid == 0) atomicOr(p.status, STATUS_BAD_SHAPE);
    return;
  }
  const int in_page = static_cast<int>(n0 % p.S);
  uint8_t* rows = p.pages + page * p.psp + in_page * p.psr;
  float* scale_at = p.scales + page * p.scp + in_page / PAGE_BLOCK * 2;
  const bool older = n0 < begun;  // the block holds earlier entries
  float old[2] = {0.f, 0.f};
  if (older) {
    old[0] = scale_at[0];
    old[1] = scale_at[1];
  }

  // first pass: turn, widen, largest value
  constexpr int PAIRS = INTERLEAVED && VE > 1 ? VE / 2 : VE;
  const int half = p.dims >> 1, turned = half / PAIRS;
  const int items = turned + (2 * p.C - p.dims) / VE;
  const int live = static_cast<int>(hi - lo);
  const int slot0 = static_cast<int>(lo - n0);
  const T* src = static_cast<const T*>(p.src) + b * p.ssb + (lo - first) * p.ssn;
  uint32_t amax[2] = {0u, 0u};
  auto size = [](float v) {  // |v|'s bits, 0 for what counts as infinite
    const uint32_t bits = __float_as_uint(v) & 0x7fffffffu;
    return bits <= SCALE_TOP_BITS ? bits : 0u;
  };
  for (int at = tid; at < live * items; at += 128) {
    const int i = at / items, item = at - i * items;
    const T* x = src + i * p.ssn;
    float* out_at = s_val + (slot0 + i) * 2 * p.C;
    if (item >= turned) {
      int c = (item - turned) * VE;
      if (c >= p.start) c += p.dims;
      float v[VE];
      V::widen(*reinterpret_cast<const Raw*>(x + c), v);
#pragma unroll
      for (int k = 0; k < VE; ++k) {
        out_at[c + k] = v[k];
        const uint32_t bits = size(v[k]);
        amax[0] = c < p.C ? max(amax[0], bits) : amax[0];
        amax[1] = c < p.C ? amax[1] : max(amax[1], bits);
      }
    } else {
      const int64_t row = lo - first + i;
      const int64_t pos = p.positions ? p.positions[static_cast<int64_t>(b) * p.n + row] : lo + i;
      constexpr bool ONE = INTERLEAVED && VE > 1;
      const int ca = p.start + (INTERLEAVED ? 2 * PAIRS : PAIRS) * item;
      const int cb = INTERLEAVED ? ca + 1 : ca + half;
      float a[VE], z[VE];
      V::widen(*reinterpret_cast<const Raw*>(x + ca), a);
      if constexpr (!ONE) V::widen(*reinterpret_cast<const Raw*>(x + cb), z);
#pragma unroll
      for (int k = 0; k < PAIRS; ++k) {
        float sn, cs, u, w;
        turn_sincos(pos, rotate_turn(p.frequencies, p.f64, item * PAIRS + k), sn, cs);
        turn_pair(ONE ? a[ONE ? 2 * k : 0] : a[k], ONE ? a[ONE ? 2 * k + 1 : 0] : z[k], sn, cs, u, w);
        u *= p.magnitude;
        w *= p.magnitude;
        out_at[ONE ? ca + 2 * k : ca + k] = u;
        out_at[ONE ? ca + 2 * k + 1 : cb + k] = w;
        amax[0] = max(amax[0], max(size(u), size(w)));
      }
    }
  }
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    amax[w] = __reduce_max_sync(0xffffffffu, amax[w]);
    if (lane == 0) s_red[warp][w] = amax[w];
  }
  __syncthreads();
  float scale[2], inv[2];
  bool grown[2];
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const uint32_t m = max(max(s_red[0][w], s_red[1][w]), max(s_red[2][w], s_red[3][w]));
    scale[w] = power_of_two(scale_exponent(m, SCALE_LEAST));
    grown[w] = old[w] < scale[w];
    if (!grown[w]) scale[w] = old[w];
    inv[w] = 1.f / scale[w];
  }
  // second pass: round, four channels a thread
  const int quads = p.C / 2;
  for (int at = tid; at < live * quads; at += 128) {
    const int i = slot0 + at / quads, c = 4 * (at % quads);
    const float4 v = *reinterpret_cast<const float4*>(s_val + i * 2 * p.C + c);
    const float f = c >= p.C ? inv[1] : inv[0];
    float q[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const bool fits = (__float_as_uint(q[k]) & 0x7fffffffu) <= SCALE_TOP_BITS;
      q[k] = fits ? q[k] * f : __int_as_float(0x7fffffff);  // infinities and what counts as one: NaN
    }
    *reinterpret_cast<uint32_t*>(rows + i * p.psr + c) = pack_e4m3x4(q[0], q[1], q[2], q[3]);
  }
  if (older) {  // a larger scale: the earlier entries are rounded again
    const float shrink[2] = {old[0] * inv[0], old[1] * inv[1]};
    for (int at = tid; at < slot0 * quads; at += 128) {
      const int i = at / quads, c = 4 * (at % quads);
      if (!(c >= p.C ? grown[1] : grown[0])) continue;
      const float f = c >= p.C ? shrink[1] : shrink[0];
      uint32_t* word = reinterpret_cast<uint32_t*>(rows + i * p.psr + c);
      const uint32_t x = *word, u = unpack_e4m3x2(x & 0xffffu), w = unpack_e4m3x2(x >> 16);
      *word = pack_e4m3x4(half_lo(u) * f, half_hi(u) * f, half_lo(w) * f, half_hi(w) * f);
    }
  }
  if (tid == 0) {
    scale_at[0] = scale[0];
    scale_at[1] = scale[1];
  }
}


// ------------------------------------------------------------- attention
//
// Few queries a batch row over the paged cache, out = softmax(scale q.k) v
// with the keys as the MMA's M, as in the key-stream kernel, and straight from
// the 8-bit pages: no entry is widened.
//
//   S^T = K Q^T      M = 128 keys,     K = 128 channels, e4m3 x e4m3
//   O^T += V^T P^T   M = 128 channels, K = 128 keys,     e4m3 x e5m2
//
// What e4m3 and e5m2 cannot hold of q and of the weights goes into more
// columns of the same product, whose M (the streamed side) is read once:
//   q (bf16, 8 significant bits), by a power of two of its row into 224 ..
//   448, is hi + lo / 16, both e4m3: exact down to 2^-10 of the row's
//   largest value and within 2^-22.8 of that below.
//   a weight w = 2^x, as fp16 (11 significant bits) 3 e5m2 numbers, each the
//   upper byte (e5m2 is fp16's) of what the ones before it leave, rounded:
//   within 2^-10 w down to 2^-21 of the largest weight (bf16's 2^-8 would
//   do), and an absolute 2^-30 of it under that, so that a long tail of small
//   weights keeps its sum.
// Scales. A key's scale multiplies its score. A value's scale 2^lv joins the
// exponent, w = 2^(s + lv - m), m the running maximum of s + lv, so O needs no
// scaling; the softmax's sum takes w 2^-lv. Sums, maxima and accumulators are
// fp32.
//
// Warps 0-3 prepare q, then take thread r = key r of a tile of 128 (as the
// key-stream kernel's do); warp 4 issues products; warp 5 brings K and V by
// TMA, a box for each page of a tile; warp 6 brings the scales.
struct PagedParams {
  const __nv_bfloat16* q;        // (B, T, H, 128) contiguous
  const float* scales;
  int64_t scp;                   // stride of a page's scales, elements
  const void* table;
  int64_t tsb;
  const int64_t* positions;      // (B, T)
  const float* sink;             // (H,) or null
  __nv_bfloat16* out;            // (B, T, H, 128)
  float* lse;                    // (B, T, H)
  float* part_o;                 // (groups * splits, NCOL, 128), not normalised
  float2* part_ml;               // (groups * splits, NCOL): exponent of the maximum, sum
  unsigned* status;
  int t64;
  int B, T, H, M, P, S, window, TQ, groups_per_row, splits, chunk_tiles;
  int cluster;                   // > 1: the splits of a group are one cluster
  float scale_log2;
};

// The exponent unit's weights come out 2^13 times as large: with a lazy
// maximum at most 2 under the true one they reach 2^15 (fp16 ends at 2^16).
constexpr float PAGED_UP = 13.f, PAGED_SLACK = 2.f;

template <int NCOL>
struct PagedLayout {
  static constexpr int C = 128, BN = 128;
  static constexpr int NK = NCOL == 64 ? 4 : 2, NV = NCOL == 64 ? 5 : 3;  // ring stages of keys and of values
  static constexpr int CTAS = NCOL == 64 ? 1 : 2;                         // a SM
  static constexpr int TILE = BN * C;
  static constexpr int Q_BYTES = 2 * NCOL * C;
  static constexpr int P_BYTES = BN * (NCOL == 64 ? 256 : 128);
  static constexpr int OFF_K = ((Q_BYTES + 1023) / 1024) * 1024;
  static constexpr int OFF_V = OFF_K + NK * TILE;
  static constexpr int OFF_P = OFF_V + NV * TILE;
  static constexpr int OFF_COL = OFF_P + P_BYTES;            // float4 a column: factor, base, bound, -
  static constexpr int OFF_RED = OFF_COL + NCOL * 16;        // 4 x NCOL floats
  static constexpr int OFF_ALPHA = OFF_RED + 4 * NCOL * 4;   // float2 a column: factor, shift
  static constexpr int OFF_L = OFF_ALPHA + NCOL * 8;
  static constexpr int OFF_SCALE = OFF_L + NCOL * 4;         // NV x 8 blocks x float4
  static constexpr int OFF_NAN = OFF_SCALE + NV * 8 * 16;    // 4 words a column
  static constexpr int OFF_QLO = OFF_NAN + NCOL * 16;
  static constexpr int OFF_QHI = OFF_QLO + 64 * 4;
  static constexpr int OFF_BAR = OFF_QHI + 64 * 4;
  static constexpr int NBAR = 1 + 2 * NK + 3 * NV + 2 + 1 + 1;
  static constexpr int OFF_MISC = OFF_BAR + NBAR * 8;
  static constexpr int BYTES = OFF_MISC + 32 + 1024;
  static constexpr int S_COLS = 2 * NCOL, O_COLS = 3 * NCOL;
  static constexpr int TMEM_COLS = 2 * S_COLS + O_COLS <= 128 ? 128 : 2 * S_COLS + O_COLS <= 256 ? 256 : 512;
};

constexpr int PAGED_THREADS = 224;

// kind::f8f6f4, fp32 accumulators; types 0 e4m3, 1 e5m2
__host__ __device__ constexpr uint32_t idesc_f8(int M, int N, int a_type, int b_type, int a_mn, int b_mn) {
  return (1u << 4) | (static_cast<uint32_t>(a_type) << 7) | (static_cast<uint32_t>(b_type) << 10) |
         (static_cast<uint32_t>(a_mn) << 15) | (static_cast<uint32_t>(b_mn) << 16) |
         (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}
template <uint32_t OFF_A, uint32_t OFF_B>
__device__ __forceinline__ void mma_f8_off_warp(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                                uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b64 da, db;\n\t"
      "add.s64 da, %1, %5;\n\tadd.s64 db, %2, %6;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "n"(OFF_A), "n"(OFF_B)
      : "memory");
}
// S^T = K Q^T, 4 steps of 32 channels; both K-major rows of 128 bytes.
template <int KK>
__device__ __forceinline__ void paged_s_steps(uint32_t d, uint64_t dk, uint64_t dq, uint32_t idesc) {
  if constexpr (KK > 0) paged_s_steps<KK - 1>(d, dk, dq, idesc);
  constexpr uint32_t off = KK * 32 / 16;
  mma_f8_off_warp<off, off>(d, dk, dq, idesc, KK > 0 ? 1u : 0u);
}
// O^T += V^T P^T, 4 steps of 32 keys; both MN-major, 128 bytes a key.
template <int KK>
__device__ __forceinline__ void paged_pv_steps(uint32_t d, uint64_t dv, uint64_t dp, uint32_t idesc, uint32_t acc0) {
  if constexpr (KK > 0) paged_pv_steps<KK - 1>(d, dv, dp, idesc, acc0);
  constexpr uint32_t off = KK * 32 * 128 / 16;
  mma_f8_off_warp<off, off>(d, dv, dp, idesc, KK > 0 ? 1u : acc0);
}

// The rows a query reads: lo .. hi of its batch row (hi < lo: none).
__device__ __forceinline__ void paged_query_rows(const PagedParams& p, int b, int t, int& lo, int& hi) {
  const int64_t pos = p.positions[static_cast<int64_t>(b) * p.T + t];
  const int64_t last = static_cast<int64_t>(p.M) * p.S - 1;
  const int64_t top = pos < last ? pos : last;
  int64_t low = 0;
  if (p.window > 0 && pos >= p.window) low = pos - p.window + 1;
  hi = top < -1 ? -1 : static_cast<int>(top);
  lo = low > INT_MAX ? INT_MAX : static_cast<int>(low);
}

// fp16 pair -> its rounded upper bytes (kept in place) and what they leave
__device__ __forceinline__ uint32_t e5m2_part(uint32_t& h) {
  const uint32_t part = (h + 0x00800080u) & 0xff00ff00u;
  asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(h) : "r"(part));
  return part;
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// One column's parts from several splits (m_i, l_i): the weights w_i = 2^(m_i
// - M) / L and the log-sum. l_i = 0: a split that read nothing.
__device__ __forceinline__ float paged_total(float M, float L, const float* sink, int h, float& inv) {
  float top = M;
  if (sink != nullptr) {
    const float s2 = sink[h] * LOG2E;
    top = fmaxf(M, s2);
    const float keep = M == -INFINITY ? 0.f : fast_exp2(M - top);
    inv = keep;
    L = L * keep + (s2 == -INFINITY ? 0.f : fast_exp2(s2 - top));
  } else {
    inv = 1.f;
  }
  inv = L == 0.f ? 0.f : inv / L;
  return L == 0.f ? -INFINITY : (top + log2f(L)) * LN2;
}

// Cluster mode: a group's splits, one CTA each, merge through distributed
// shared memory; CTA k owns columns k, k + S, ... (as stream_cluster_merge).
template <int NCOL>
__device__ __forceinline__ void paged_cluster_merge(const PagedParams& p, const float4* s_col, const float* s_l,
                                                    const float* s_o, float* s_w, int64_t row0, int ncols) {
  constexpr int C = 128;
  cluster_sync();
  const int S = p.cluster;
  const int rank = static_cast<int>(cluster_rank());
  const int mine = ncols > rank ? (ncols - rank + S - 1) / S : 0;
  const uint32_t am = smem_u32(s_col), al = smem_u32(s_l), ao = smem_u32(s_o);
  if (static_cast<int>(threadIdx.x) < mine) {
    const int cl = threadIdx.x, c = rank + cl * S;
    float mi[8], li[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      mi[i] = -INFINITY;
      li[i] = 0.f;
      if (i < S) {
        mi[i] = dsmem_ld(dsmem_map(am + c * 16 + 4, i));
        li[i] = dsmem_ld(dsmem_map(al + c * 4, i));
      }
    }
    float M = -INFINITY;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (li[i] != 0.f) M = fmaxf(M, mi[i]);
    float w[8], L = 0.f, inv;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      w[i] = li[i] != 0.f ? fast_exp2(mi[i] - M) : 0.f;
      L += li[i] != 0.f ? w[i] * li[i] : 0.f;
    }
    s_w[cl * 9 + 8] = paged_total(M, L, p.sink, c % p.H, inv);
#pragma unroll
    for (int i = 0; i < 8; ++i) s_w[cl * 9 + i] = li[i] != 0.f ? w[i] * inv : 0.f;
  }
  __syncthreads();
  for (int item = threadIdx.x; item < mine * (C / 4); item += blockDim.x) {
    const int cl = item / (C / 4), quad = item % (C / 4), c = rank + cl * S;
    float4 o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < S && s_w[cl * 9 + i] != 0.f) o[i] = dsmem_ld4(dsmem_map(ao + (c * C + quad * 4) * 4, i));
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float w = i < S ? s_w[cl * 9 + i] : 0.f;
      if (w != 0.f) {
        acc.x = fmaf(w, o[i].x, acc.x);
        acc.y = fmaf(w, o[i].y, acc.y);
        acc.z = fmaf(w, o[i].z, acc.z);
        acc.w = fmaf(w, o[i].w, acc.w);
      }
    }
    uint2 packed;
    packed.x = pack_bf16(acc.x, acc.y);
    packed.y = pack_bf16(acc.z, acc.w);
    *reinterpret_cast<uint2*>(p.out + (row0 + c) * C + quad * 4) = packed;
    if (quad == 0) p.lse[row0 + c] = s_w[cl * 9 + 8];
  }
  cluster_sync();
}

template <int NCOL>
__global__ void __launch_bounds__(PAGED_THREADS, PagedLayout<NCOL>::CTAS)
    paged_kernel(const __grid_constant__ CUtensorMap tm, const PagedParams p) {
  using L = PagedLayout<NCOL>;
  constexpr int C = L::C, BN = L::BN, NK = L::NK, NV = L::NV;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sK = smem + L::OFF_K;
  uint8_t* sV = smem + L::OFF_V;
  uint8_t* sP = smem + L::OFF_P;
  float4* s_col = reinterpret_cast<float4*>(smem + L::OFF_COL);
  float* s_red = reinterpret_cast<float*>(smem + L::OFF_RED);
  float2* s_alpha = reinterpret_cast<float2*>(smem + L::OFF_ALPHA);
  float* s_l = reinterpret_cast<float*>(smem + L::OFF_L);
  float4* s_scale = reinterpret_cast<float4*>(smem + L::OFF_SCALE);
  uint32_t* s_nan = reinterpret_cast<uint32_t*>(smem + L::OFF_NAN);
  int* s_qlo = reinterpret_cast<int*>(smem + L::OFF_QLO);
  int* s_qhi = reinterpret_cast<int*>(smem + L::OFF_QHI);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  uint64_t* q_full = bars;
  uint64_t* k_full = bars + 1;
  uint64_t* k_empty = k_full + NK;
  uint64_t* v_full = k_empty + NK;
  uint64_t* v_empty = v_full + NV;
  uint64_t* sc_full = v_empty + NV;
  uint64_t* s_full = sc_full + NV;
  uint64_t* p_ready = s_full + 2;
  uint64_t* o_done = p_ready + 1;
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(smem + L::OFF_MISC);
  int* s_range = reinterpret_cast<int*>(smem + L::OFF_MISC + 4);  // rows read by some query, rows read by all, any NaN

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = blockIdx.x, split = blockIdx.y;
  const int b = group / p.groups_per_row;
  const int t0 = (group - b * p.groups_per_row) * p.TQ;
  const int TQg = min(p.TQ, p.T - t0);
  const int ncols = TQg * p.H;
  const int64_t row0 = (static_cast<int64_t>(b) * p.T + t0) * p.H;

  if (warp == 0) {
    griddep_wait();
    int rlo = INT_MAX, rhi = -1, alo = 0, ahi = INT_MAX;
    for (int tq = lane; tq < TQg; tq += 32) {
      int lo, hi;
      paged_query_rows(p, b, t0 + tq, lo, hi);
      s_qlo[tq] = lo;
      s_qhi[tq] = hi;
      if (hi >= lo) {
        rlo = min(rlo, lo);
        rhi = max(rhi, hi);
      }
      alo = max(alo, lo);
      ahi = min(ahi, hi);
    }
    rlo = __reduce_min_sync(0xffffffffu, rlo);
    rhi = __reduce_max_sync(0xffffffffu, rhi);
    alo = __reduce_max_sync(0xffffffffu, alo);
    ahi = __reduce_min_sync(0xffffffffu, ahi);
    if (lane == 0) {
      s_range[0] = rlo;
      s_range[1] = rhi;
      s_range[2] = alo;
      s_range[3] = ahi;
      s_range[4] = 0;
    }
  } else if (warp == 1) {
    for (int i = lane; i < NCOL; i += 32) {
      s_col[i] = make_float4(0.f, -PAGED_UP, -INFINITY, 0.f);
      s_l[i] = 0.f;
    }
  } else if (warp == 2) {
    for (int i = lane; i < NCOL * 4; i += 32) s_nan[i] = 0u;
  } else if (warp == 3 && lane == 0) {
    mbar_init(q_full, 128);
    for (int s = 0; s < NK; ++s) {
      mbar_init(k_full + s, 1);
      mbar_init(k_empty + s, 1);
    }
    for (int s = 0; s < NV; ++s) {
      mbar_init(v_full + s, 1);
      mbar_init(v_empty + s, 1);
      mbar_init(sc_full + s, 1);
    }
    mbar_init(s_full, 1);
    mbar_init(s_full + 1, 1);
    mbar_init(p_ready, 128);
    mbar_init(o_done, 1);
    fence_mbar_init();
  } else if (warp == 4) {
    tmem_alloc(s_tmem, L::TMEM_COLS);
    tmem_relinquish();
  }
  griddep_wait();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // tiles of 128 entries, from the one that holds the first row read
  const int rlo = s_range[0], rhi = s_range[1];
  const int tile0 = rhi >= rlo ? rlo / BN + split * p.chunk_tiles : 0;
  const int ntiles = rhi >= rlo ? max(0, min(p.chunk_tiles, rhi / BN - tile0 + 1)) : 0;
  const int64_t seg = static_cast<int64_t>(group) * p.splits + split;

  if (ntiles == 0) {
    if (p.cluster > 1) {
      paged_cluster_merge<NCOL>(p, s_col, s_l, reinterpret_cast<const float*>(sK), reinterpret_cast<float*>(sP), row0,
                                ncols);
    } else if (p.splits > 1) {
      if (static_cast<int>(threadIdx.x) < ncols) p.part_ml[seg * NCOL + threadIdx.x] = make_float2(-INFINITY, 0.f);
    } else {
      for (int i = threadIdx.x; i < ncols * (C / 2); i += PAGED_THREADS)
        reinterpret_cast<uint32_t*>(p.out + row0 * C)[i] = 0u;
      if (static_cast<int>(threadIdx.x) < ncols)
        p.lse[row0 + threadIdx.x] = p.sink != nullptr ? p.sink[threadIdx.x % p.H] : -INFINITY;
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 4) {
      tc_fence_after();
      tmem_dealloc(*s_tmem, L::TMEM_COLS);
    }
    return;
  }
  const uint32_t tmem = *s_tmem;
  griddep_launch();

  if (warp == 5) {
    // ------------------------------------------------ keys and values by TMA
    const int rows = min(p.S, BN), per = BN / rows;  // entries of a box, boxes of a tile
    const int batch = 32 / per;                      // tiles whose page numbers the warp holds, a lane a box
    const int part = lane % per;
    auto lookup = [&](int j0) {  // the page of this lane's box in tile j0 + lane / per
      const int64_t n = static_cast<int64_t>(tile0 + j0 + lane / per) * BN + part * rows;
      if (j0 + lane / per >= ntiles || n / p.S >= p.M) return -1;
      return static_cast<int>(page_of(p.table, p.t64, b * p.tsb + n / p.S, p.P));
    };
    int mine = lookup(0), next = lookup(batch);
    bool ok = true;
    for (int j = 0; ok && j < ntiles; ++j) {
      const int in = j % batch;
      if (in == 0 && j > 0) {
        mine = next;
        next = lookup(j + batch);
      }
      const int row = static_cast<int>((static_cast<int64_t>(tile0 + j) * BN) % p.S);  // 0 for pages within a tile
      const int sk = j % NK, sv = j % NV;
      if (j >= NK) ok = __all_sync(0xffffffffu, mbar_wait(k_empty + sk, ((j / NK) & 1) ^ 1, p.status));
      if (!ok) break;
      if (lane == 0) mbar_expect_tx(k_full + sk, L::TILE);
      __syncwarp();
      if (lane / per == in) tma_load_3d(sK + sk * L::TILE + part * rows * C, &tm, k_full + sk, 0, row, mine);
      if (j >= NV) ok = __all_sync(0xffffffffu, mbar_wait(v_empty + sv, ((j / NV) & 1) ^ 1, p.status));
      if (!ok) break;
      if (lane == 0) mbar_expect_tx(v_full + sv, L::TILE);
      __syncwarp();
      if (lane / per == in) tma_load_3d(sV + sv * L::TILE + part * rows * C, &tm, v_full + sv, C, row, mine);
    }
  } else if (warp == 6) {
    // ------------------------------------- scales: a lane a block, four tiles at a time
    auto lookup = [&](int j0) {
      float4 r = make_float4(0.f, 0.f, 0.f, 0.f);  // key scale, log2 of the value scale, its inverse, 1: there
      const int j = j0 + (lane >> 3);
      const int64_t n = static_cast<int64_t>(tile0 + j) * BN + (lane & 7) * PAGE_BLOCK;
      if (j >= ntiles || n / p.S >= p.M) return r;
      const int64_t page = page_of(p.table, p.t64, b * p.tsb + n / p.S, p.P);
      if (page < 0) return r;
      const float* at = p.scales + page * p.scp + (n % p.S) / PAGE_BLOCK * 2;
      r.x = at[0];
      // 2^-60 at least: what is scaled by less (0: an empty block) is nothing; over 2^60: NaN
      const float v = at[1];
      r.y = v < power_of_two(SCALE_LEAST) && v >= 0.f ? static_cast<float>(SCALE_LEAST)
            : v <= power_of_two(60)                   ? log2f(v)
                                                      : __int_as_float(0x7fffffff);
      r.z = fast_exp2(-r.y);
      r.w = 1.f;
      return r;
    };
    float4 mine = lookup(0), next = lookup(4);
    bool ok = true;
    for (int j = 0; ok && j < ntiles; ++j) {
      if ((j & 3) == 0 && j > 0) {
        mine = next;
        next = lookup(j + 4);
      }
      const int st = j % NV;
      if (j >= NV) ok = __all_sync(0xffffffffu, mbar_wait(v_empty + st, ((j / NV) & 1) ^ 1, p.status));
      if (!ok) break;
      if ((lane >> 3) == (j & 3)) s_scale[st * 8 + (lane & 7)] = mine;
      __syncwarp();
      if (lane == 0) mbar_arrive(sc_full + st);
    }
  } else if (warp == 4) {
    // --------------------------------------------------------- MMA issuer
    constexpr uint32_t IDESC_S = idesc_f8(128, 2 * NCOL, 0, 0, 0, 0);
    constexpr uint32_t IDESC_O = idesc_f8(128, 3 * NCOL, 0, 1, 1, 1);
    const uint32_t tS = tmem, tO = tmem + 2 * L::S_COLS;
    const uint32_t k_addr = smem_u32(sK), v_addr = smem_u32(sV);
    const uint64_t dq = sdesc_sw128(smem_u32(sQ), 16, 1024);
    const uint64_t dp = sdesc_sw128(smem_u32(sP), BN * 128, 1024);
    auto wait = [&](uint64_t* bar, int parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, p.status)); };
    bool ok = wait(q_full, 0);
    for (int j = 0; ok && j <= ntiles; ++j) {
      if (j < ntiles) {
        const int st = j % NK;
        if (!(ok = wait(k_full + st, (j / NK) & 1))) break;
        tc_fence_after();
        paged_s_steps<3>(tS + (j & 1) * L::S_COLS, sdesc_sw128(k_addr + st * L::TILE, 16, 1024), dq, IDESC_S);
        mma_commit_warp(s_full + (j & 1));
        mma_commit_warp(k_empty + st);
      }
      if (j > 0) {
        const int jp = j - 1, st = jp % NV;
        if (!(ok = wait(v_full + st, (jp / NV) & 1))) break;
        if (!(ok = wait(p_ready, jp & 1))) break;
        tc_fence_after();
        paged_pv_steps<3>(tO, sdesc_sw128(v_addr + st * L::TILE, BN * 128, 1024), dp, IDESC_O, jp > 0 ? 1u : 0u);
        mma_commit_warp(v_empty + st);
        mma_commit_warp(o_done);
      }
    }
  } else {
    const int r = threadIdx.x;
    // ------------------------------------------- q: hi and lo rows, a warp a column
    for (int col = warp; col < NCOL; col += 4) {
      uint2 raw = make_uint2(0u, 0u);
      if (col < ncols) raw = *reinterpret_cast<const uint2*>(p.q + (row0 + col) * C + lane * 4);
      const float x[4] = {__uint_as_float(raw.x << 16), __uint_as_float(raw.x & 0xffff0000u),
                          __uint_as_float(raw.y << 16), __uint_as_float(raw.y & 0xffff0000u)};
      uint32_t top = 0u;
#pragma unroll
      for (int k = 0; k < 4; ++k) top = max(top, __float_as_uint(x[k]) & 0x7fffffffu);
      top = __reduce_max_sync(0xffffffffu, top);
      const bool finite = top < 0x7f800000u;
      const int e = finite ? scale_exponent(top, -100) : 0;
      const float inv = power_of_two(-e);
      float hi[4], lo[4];
      uint32_t packed_hi = 0u, packed_lo = 0u;
      if (finite) {
#pragma unroll
        for (int k = 0; k < 4; ++k) hi[k] = x[k] * inv;
        packed_hi = pack_e4m3x4(hi[0], hi[1], hi[2], hi[3]);
        const uint32_t u = unpack_e4m3x2(packed_hi & 0xffffu), w = unpack_e4m3x2(packed_hi >> 16);
        lo[0] = (hi[0] - half_lo(u)) * 16.f;
        lo[1] = (hi[1] - half_hi(u)) * 16.f;
        lo[2] = (hi[2] - half_lo(w)) * 16.f;
        lo[3] = (hi[3] - half_hi(w)) * 16.f;
        packed_lo = pack_e4m3x4(lo[0], lo[1], lo[2], lo[3]);
      }
      const uint32_t chunk = lane >> 2, in = (lane & 3) * 4;
      *reinterpret_cast<uint32_t*>(sQ + sw128_offset(col, chunk) + in) = packed_hi;
      *reinterpret_cast<uint32_t*>(sQ + sw128_offset(NCOL + col, chunk) + in) = packed_lo;
      // a query with an infinity or NaN has no result but NaN
      if (lane == 0)
        s_col[col].x = finite ? power_of_two(e) * p.scale_log2 : __int_as_float(0x7fffffff);
    }
    fence_proxy_async();
    mbar_arrive(q_full);
    named_barrier(1, 128);  // s_col

    // --------------------------------------------------- softmax: thread r = key r
    const uint32_t lane_addr = tmem + (static_cast<uint32_t>(warp * 32) << 16);
    const uint32_t tO = lane_addr + 2 * L::S_COLS;
    const uint64_t head_bits = p.H >= 64 ? ~0ull : ((1ull << p.H) - 1);
    const uint64_t all_cols = ncols >= 64 ? ~0ull : ((1ull << ncols) - 1);
    const int alo = s_range[2], ahi = s_range[3];
    float lp[NCOL];
#pragma unroll
    for (int c = 0; c < NCOL; ++c) lp[c] = 0.f;
    bool ok = true;
    for (int j = 0; j < ntiles; ++j) {
      const int st = j % NV;
      ok = __all_sync(0xffffffffu, mbar_wait(sc_full + st, (j / NV) & 1, p.status));
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait(s_full + (j & 1), (j >> 1) & 1, p.status));
      tc_fence_after();
      const float4 sc = s_scale[st * 8 + (r >> 4)];
      const int n0 = (tile0 + j) * BN;
      float s[NCOL];
      {
        const uint32_t sa = lane_addr + (j & 1) * L::S_COLS;
        if constexpr (NCOL == 16) {
          uint32_t x[32];
          tmem_ld32(sa, x);
#pragma unroll
          for (int c = 0; c < 16; ++c) s[c] = fmaf(__uint_as_float(x[16 + c]), 0.0625f, __uint_as_float(x[c]));
        } else {
#pragma unroll
          for (int c0 = 0; c0 < NCOL; c0 += 32) {
            uint32_t x[32], y[32];
            tmem_ld32x2(sa + c0, sa + NCOL + c0, x, y);
#pragma unroll
            for (int c = 0; c < 32; ++c) s[c0 + c] = fmaf(__uint_as_float(y[c]), 0.0625f, __uint_as_float(x[c]));
          }
        }
      }
      // exponents relative to the columns' bases; a row that nothing masks keeps padding columns too
      uint64_t vis = ~0ull;
      const bool inside = n0 >= alo && n0 + BN - 1 <= ahi;
      if (!inside) {
        const int row = n0 + r;
        vis = 0ull;
        for (int tq = 0; tq < TQg; ++tq)
          if (row >= s_qlo[tq] && row <= s_qhi[tq]) vis |= head_bits << (tq * p.H);
        if (vis == all_cols) vis = ~0ull;
      }
      if (sc.w == 0.f) vis = 0ull;
      bool raise = false;
#pragma unroll
      for (int c = 0; c < NCOL; ++c) {
        const float4 col = s_col[c];
        s[c] = fmaf(s[c] * sc.x, col.x, sc.y) - col.y;
        if (vis != ~0ull && !((vis >> c) & 1ull)) s[c] = -INFINITY;
        raise |= s[c] > col.z;
      }
      // values that nothing may read hold nothing; one that some columns may read and that holds NaN is taken
      // out of the product and noted for those columns
      if (vis != ~0ull) {
        if (ok) ok = mbar_wait(v_full + st, (j / NV) & 1, p.status);
        uint8_t* vr = sV + st * L::TILE + r * 128;
        bool clear = vis == 0ull;
        if (!clear && ok) {
          uint32_t bits[4] = {0u, 0u, 0u, 0u};
          for (int ch = 0; ch < 32; ++ch) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(vr + (((ch >> 2) ^ (r & 7)) << 4) + (ch & 3) * 4);
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (((w >> (8 * k)) & 0x7fu) == 0x7fu) bits[ch >> 3] |= 1u << ((ch & 7) * 4 + k);
          }
          if (bits[0] | bits[1] | bits[2] | bits[3]) {
            clear = true;
            s_range[4] = 1;
            for (int c = 0; c < ncols; ++c)
              if ((vis >> c) & 1ull)
                for (int k = 0; k < 4; ++k) atomicOr(s_nan + c * 4 + k, bits[k]);
          }
        }
        if (clear && ok)
          for (int ch = 0; ch < 8; ++ch) *reinterpret_cast<uint4*>(vr + ch * 16) = make_uint4(0u, 0u, 0u, 0u);
      }
      // the lazy maximum, as in the key-stream kernel: most tiles raise no column's
      if (named_barrier_or(1, 128, raise || !ok)) {
#pragma unroll
        for (int c32 = 0; c32 < (NCOL + 31) / 32; ++c32) {
          float tmp[32];
#pragma unroll
          for (int c = 0; c < 32; ++c) tmp[c] = (c32 * 32 + c < NCOL) ? s[(c32 * 32 + c) % NCOL] : -INFINITY;
          const float m = transpose_reduce32(tmp, MaxOp());
          if (c32 * 32 + lane < NCOL) s_red[warp * NCOL + c32 * 32 + lane] = m;
        }
        ok = named_barrier_and(1, 128, ok);
        if (!ok) break;
        if (r < NCOL) {
          const float top = fmaxf(fmaxf(s_red[r], s_red[NCOL + r]), fmaxf(s_red[2 * NCOL + r], s_red[3 * NCOL + r]));
          const float4 col = s_col[r];
          float2 a = make_float2(1.f, 0.f);
          if (top > col.z) {
            a.y = top - PAGED_UP;
            if (col.z != -INFINITY) a.x = fast_exp2(-a.y);  // else nothing was added up yet
            s_col[r] = make_float4(col.x, col.y + a.y, PAGED_UP + PAGED_SLACK, 0.f);
          }
          s_alpha[r] = a;
        }
        named_barrier(1, 128);
        bool any = false;
#pragma unroll
        for (int c = 0; c < NCOL; ++c) {
          const float2 a = s_alpha[c];
          s[c] -= a.y;
          lp[c] *= a.x;
          any |= a.x != 1.f;
        }
        if (any && j > 0) {
          ok = __all_sync(0xffffffffu, mbar_wait(o_done, (j - 1) & 1, p.status));
          if (ok) {
            tc_fence_after();
#pragma unroll
            for (int c0 = 0; c0 < L::O_COLS; c0 += 16) {
              uint32_t x[16];
              tmem_ld16(tO + c0, x);
#pragma unroll
              for (int c = 0; c < 16; ++c)
                x[c] = __float_as_uint(__uint_as_float(x[c]) * s_alpha[(c0 + c) % NCOL].x);
              tmem_st16(tO + c0, x);
            }
            tmem_wait_st();
          }
        }
      }
      // weights, their sums, and their three parts
#pragma unroll
      for (int c = 0; c < NCOL; ++c) {
        s[c] = fast_exp2(s[c]);
        lp[c] = fmaf(s[c], sc.z, lp[c]);
      }
      // a row without a value scale adds nothing (its inverse is 0 too)
      if (j > 0 && ok) ok = __all_sync(0xffffffffu, mbar_wait(o_done, (j - 1) & 1, p.status));  // P's buffer is free
      if (ok) {
#pragma unroll
        for (int c0 = 0; c0 < NCOL; c0 += 16) {
          uint32_t part[3][4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t x = pack_half2(s[c0 + 4 * k], s[c0 + 4 * k + 1]);
            uint32_t y = pack_half2(s[c0 + 4 * k + 2], s[c0 + 4 * k + 3]);
#pragma unroll
            for (int i = 0; i < 3; ++i) part[i][k] = __byte_perm(e5m2_part(x), e5m2_part(y), 0x7531);
          }
#pragma unroll
          for (int i = 0; i < 3; ++i) {
            const int at = i * NCOL + c0;  // the column's byte in the key's row
            *reinterpret_cast<uint4*>(sP + (at >> 7) * (BN * 128) + sw128_offset(r, (at & 127) >> 4)) =
                make_uint4(part[i][0], part[i][1], part[i][2], part[i][3]);
          }
        }
      }
      tc_fence_before();
      fence_proxy_async();
      mbar_arrive(p_ready);
    }
    if (ok) ok = __all_sync(0xffffffffu, mbar_wait(o_done, (ntiles - 1) & 1, p.status));
    tc_fence_after();
    // per-column sums over the 128 keys
#pragma unroll
    for (int c32 = 0; c32 < (NCOL + 31) / 32; ++c32) {
      float tmp[32];
#pragma unroll
      for (int c = 0; c < 32; ++c) tmp[c] = (c32 * 32 + c < NCOL) ? lp[(c32 * 32 + c) % NCOL] : 0.f;
      const float sum = transpose_reduce32(tmp, SumOp());
      if (c32 * 32 + lane < NCOL) s_red[warp * NCOL + c32 * 32 + lane] = sum;
    }
    ok = named_barrier_and(1, 128, ok);
    if (r < ncols) {
      const float l = (s_red[r] + s_red[NCOL + r]) + (s_red[2 * NCOL + r] + s_red[3 * NCOL + r]);
      if (p.cluster > 1) {
        s_l[r] = ok ? l : 0.f;
      } else if (p.splits == 1) {
        float inv;
        const float lse = paged_total(l != 0.f ? s_col[r].y : -INFINITY, l, p.sink, r % p.H, inv);
        s_l[r] = inv;
        if (ok) p.lse[row0 + r] = lse;
      } else {
        p.part_ml[seg * NCOL + r] = ok ? make_float2(s_col[r].y, l) : make_float2(-INFINITY, 0.f);
      }
    }
    named_barrier(1, 128);
    const bool any_nan = s_range[4] != 0;
    if (ok) {
#pragma unroll
      for (int c0 = 0; c0 < NCOL; c0 += 16) {  // thread r: channel r
        uint32_t x[16], y[16], z[16];
        tmem_ld16(tO + c0, x);
        tmem_ld16(tO + NCOL + c0, y);
        tmem_ld16(tO + 2 * NCOL + c0, z);
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          const int col = c0 + c;
          float o = __uint_as_float(x[c]) + (__uint_as_float(y[c]) + __uint_as_float(z[c]));
          if (any_nan && ((s_nan[col * 4 + (r >> 5)] >> lane) & 1u)) o = __int_as_float(0x7fffffff);
          if (p.cluster > 1) {
            reinterpret_cast<float*>(sK)[col * C + r] = o;  // the rings hold no tile any more
          } else if (col < ncols) {
            if (p.splits == 1) {
              p.out[(row0 + col) * C + r] = __float2bfloat16_rn(o * s_l[col]);
            } else {
              p.part_o[(seg * NCOL + col) * C + r] = o;
            }
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 4) {
    tc_fence_after();
    tmem_dealloc(tmem, L::TMEM_COLS);
  }
  if (p.cluster > 1)
    paged_cluster_merge<NCOL>(p, s_col, s_l, reinterpret_cast<const float*>(sK), reinterpret_cast<float*>(sP), row0,
                              ncols);
}

// Splits that wrote partials: one warp a row (query, head), four channels a lane.
__global__ void __launch_bounds__(256) paged_merge_kernel(const PagedParams p, int ncol) {
  griddep_wait();
  constexpr int C = 128;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= static_cast<int64_t>(p.B) * p.T * p.H) return;
  const int64_t query = row / p.H;
  const int h = static_cast<int>(row - query * p.H);
  const int64_t b = query / p.T;
  const int t = static_cast<int>(query - b * p.T);
  const int64_t group = b * p.groups_per_row + t / p.TQ;
  const int col = (t % p.TQ) * p.H + h;
  float M = -INFINITY, L = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = 0; s0 < p.splits; s0 += 8) {
    float2 ml[8];
    float4 o[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      ml[k] = make_float2(-INFINITY, 0.f);
      o[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (s0 + k < p.splits) {
        const int64_t at = (group * p.splits + s0 + k) * ncol + col;
        ml[k] = p.part_ml[at];
        o[k] = *reinterpret_cast<const float4*>(p.part_o + at * C + lane * 4);
      }
    }
    float top = M;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (ml[k].y != 0.f) top = fmaxf(top, ml[k].x);
    if (top != M) {
      const float a = M == -INFINITY ? 0.f : fast_exp2(M - top);
      L *= a;
      acc = make_float4(acc.x * a, acc.y * a, acc.z * a, acc.w * a);
      M = top;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (ml[k].y == 0.f) continue;  // the split read nothing: its output was not written
      const float w = fast_exp2(ml[k].x - M);
      L = fmaf(w, ml[k].y, L);
      acc.x = fmaf(w, o[k].x, acc.x);
      acc.y = fmaf(w, o[k].y, acc.y);
      acc.z = fmaf(w, o[k].z, acc.z);
      acc.w = fmaf(w, o[k].w, acc.w);
    }
  }
  float inv;
  const float lse = paged_total(M, L, p.sink, h, inv);
  uint2 packed;
  packed.x = pack_bf16(acc.x * inv, acc.y * inv);
  packed.y = pack_bf16(acc.z * inv, acc.w * inv);
  *reinterpret_cast<uint2*>(p.out + row * C + lane * 4) = packed;
  if (lane == 0) p.lse[row] = lse;
}

}  // namespace wpt
