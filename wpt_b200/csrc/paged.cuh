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
  unsigned S;                      // entries a page
  int B, n, C, M, P, dims, start;
  int blocks;                      // grid blocks a row
  int turn_rows, turn_pairs;       // APPEND_THREADS / (dims / 2), and the rest
  int vecs, inv_vecs;              // ROWS: vectors of a key, and 65536 / vecs + 1
  float magnitude;
};

__device__ __forceinline__ int64_t page_number(const void* table, int t64, int64_t at) {
  return t64 ? static_cast<const int64_t*>(table)[at] : static_cast<const int32_t*>(table)[at];
}
__device__ __forceinline__ int64_t page_of(const void* table, int t64, int64_t at, int P) {
  const int64_t id = page_number(table, t64, at);
  return id >= 0 && id < P ? id : -1;
}

// Where an entry's vector v sits among its key's turned channels: whether it is
// one of them, its first pair, whether it holds the first channels of its pairs
// (halves), and how many vectors on its pairs' others are.
template <int VE, bool INTERLEAVED>
struct TurnedVector {
  bool turned, front;
  int pair, partner;
  __device__ __forceinline__ TurnedVector(int v, int start, int dims) {
    const int at = v * VE - start, half = dims >> 1;
    turned = at >= 0 && at < dims;
    front = INTERLEAVED || at < half;
    pair = INTERLEAVED ? at / 2 : front ? at : at - half;
    partner = !turned || INTERLEAVED ? 0 : front ? half / VE : -half / VE;
  }
  // u, widened, turned in place; z: its partner vector, widened (halves); sn, cs: of its pairs
  __device__ __forceinline__ void turn(float (&u)[VE], const float (&z)[VE], const float* sn, const float* cs) const {
    if constexpr (INTERLEAVED) {
#pragma unroll
      for (int k = 0; k < VE / 2; ++k) {
        float a, b;
        turn_pair(u[2 * k], u[2 * k + 1], sn[k], cs[k], a, b);
        u[2 * k] = a;
        u[2 * k + 1] = b;
      }
    } else {
      const float sign = front ? -1.f : 1.f;
#pragma unroll
      for (int k = 0; k < VE; ++k) {  // x_a cos - x_b sin, or x_b cos + x_a sin
        u[k] = __fmaf_rn(__fmul_rn(z[k], sn[k]), sign, __fmul_rn(u[k], cs[k]));
      }
    }
  }
};

// max(|x|, |y|, m), NaN ignored
__device__ __forceinline__ float max_abs(float x, float y, float m) {
  float r;
  asm("max.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(m));
  return r;
}

constexpr int APPEND_THREADS = 128;

// Appending. One CTA a block of 16 entries (and batch row), so a block's scale
// needs no exchange: all threads work out the sines and cosines of its entries
// (a table in shared memory: 16 x dims / 2 pairs, where the lanes that turn
// would each compute 8 a token while the others wait), the new entries are
// turned and widened to fp32, their largest value gives the scale, and they are
// rounded. ROWS: a warp takes four entries, their keys and values apart, so that
// all its lanes turn or none; a lane has a vector (with halves, the other
// channels of its pairs come from the lane that loaded them), and the entries
// stay in registers; else they go through shared memory. Prompts (16 rows of
// 4,096, 2 x 128, all key channels turned: 23 us for 50 MB) are bound by issue
// slots, a third of them for angles; a step of one entry a row (2.8 us) is a
// chain of three loads (first, the page's number, its scale).
template <class T, int VE, bool INTERLEAVED, int ROWS>
__global__ void __launch_bounds__(APPEND_THREADS, ROWS == 2 ? 8 : ROWS == 4 ? 4 : 1) paged_append_kernel(const AppendParams p) {
  using V = Vec<T, VE>;
  using Raw = typename V::Raw;
  constexpr int WARPS = APPEND_THREADS / 32;
  extern __shared__ float s_all[];  // sines and cosines (16, dims / 2), then, unless ROWS, values (16, 2 C)
  __shared__ uint32_t s_red[WARPS][2];
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
  const unsigned at_entry = static_cast<unsigned>(n0);  // under the table's capacity
  const int64_t page = page_of(p.table, p.t64, b * p.tsb + at_entry / p.S, p.P);
  const int live = static_cast<int>(hi - lo);
  const int slot0 = static_cast<int>(lo - n0);
  const int64_t row0 = lo - first;  // the first new entry's number
  const T* src = static_cast<const T*>(p.src) + b * p.ssb + row0 * p.ssn;
  const int half = p.dims >> 1;
  // ROWS: a warp has 4 entries, 32 / vecs of them at a time (a group; up to ROWS), first their keys, then their values
  constexpr int MINE = PAGE_BLOCK / WARPS, GROUPS = ROWS > 0 ? ROWS : 1;
  const int sub = lane * p.inv_vecs >> 16, vec = lane - sub * p.vecs, each = (32 * p.inv_vecs) >> 16;
  auto entry_of = [&](int g) {  // this lane's of group g, `live` or more: none
    const int e = g * each + sub;
    return sub < each && e < MINE ? MINE * warp + e : PAGE_BLOCK;
  };
  Raw raw[GROUPS][2];
  if constexpr (ROWS) {
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      const int i = entry_of(g);
      if (i < live) {
        const T* x = src + i * p.ssn + vec * VE;
        raw[g][0] = *reinterpret_cast<const Raw*>(x);
        raw[g][1] = *reinterpret_cast<const Raw*>(x + p.C);
      }
    }
  }
  float2* s_turn = reinterpret_cast<float2*>(s_all);
  float* s_val = s_all + PAGE_BLOCK * p.dims;
  {
    int i = half > 0 ? tid / half : live, k = tid - i * half, last = -1;
    uint64_t turn = 0;
    while (i < live) {
      if (k != last) turn = rotate_turn(p.frequencies, p.f64, k);
      last = k;
      const int64_t pos = p.positions ? p.positions[static_cast<int64_t>(b) * p.n + row0 + i] : lo + i;
      float sn, cs;
      turn_sincos(pos, turn, sn, cs);
      s_turn[i * half + k] = make_float2(sn * p.magnitude, cs * p.magnitude);
      i += p.turn_rows;
      k += p.turn_pairs;
      if (k >= half) {
        k -= half;
        ++i;
      }
    }
  }
  if (page < 0) {
    if (tid == 0) atomicOr(p.status, STATUS_BAD_SHAPE);
    return;
  }
  const int in_page = static_cast<int>(at_entry % p.S);
  uint8_t* rows = p.pages + page * p.psp + in_page * p.psr;
  float* scale_at = p.scales + page * p.scp + in_page / PAGE_BLOCK * 2;
  const bool older = n0 < begun;  // the block holds earlier entries
  float old[2] = {0.f, 0.f};
  if (older) {
    old[0] = scale_at[0];
    old[1] = scale_at[1];
  }
  if (p.dims > 0) __syncthreads();

  // turned and widened values, and the bits of the largest absolute ones of keys and values
  uint32_t amax[2] = {0u, 0u};
  auto note = [](float v, uint32_t& m) { m = max(m, __float_as_uint(v) & 0x7fffffffu); };
  float u[ROWS ? 2 * GROUPS : 1][VE];
  if constexpr (ROWS) {
    const TurnedVector<VE, INTERLEAVED> tv(vec, p.start, p.dims);
    float most[2] = {0.f, 0.f};
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      if (MINE * warp + g * each >= live || g * each >= MINE) break;  // the whole warp
      const int i = entry_of(g);
      Raw z = raw[g][0];
      if constexpr (!INTERLEAVED) {
        if (p.dims > 0) z = V::from_lane(raw[g][0], lane + tv.partner);
      }
      if (i < live) {
        float(&key)[VE] = u[2 * g];
        float(&value)[VE] = u[ROWS ? 2 * g + 1 : 0];
        V::widen(raw[g][0], key);
        V::widen(raw[g][1], value);
        if (tv.turned) {
          float c[VE], sn[VE], cs[VE];
          V::widen(z, c);
          const float4* at = reinterpret_cast<const float4*>(s_turn + i * half + tv.pair);
#pragma unroll
          for (int k = 0; k < (INTERLEAVED ? VE / 2 : VE); k += 2) {
            const float4 t = at[k / 2];
            sn[k] = t.x;
            cs[k] = t.y;
            sn[k + 1] = t.z;
            cs[k + 1] = t.w;
          }
          tv.turn(key, c, sn, cs);
        }
#pragma unroll
        for (int k = 0; k < VE; k += 2) {
          most[0] = max_abs(key[k], key[k + 1], most[0]);
          most[1] = max_abs(value[k], value[k + 1], most[1]);
        }
      }
    }
    amax[0] = __float_as_uint(most[0]);
    amax[1] = __float_as_uint(most[1]);
  } else {
    // items: pairs (with VE > 1, vectors of them), then the channels that do not turn
    constexpr bool ONE = INTERLEAVED && VE > 1;  // an item is one vector of whole pairs
    constexpr int PAIRS = ONE ? VE / 2 : VE;
    const int turned = half / PAIRS, items = turned + (2 * p.C - p.dims) / VE;
    for (int at = tid; at < live * items; at += APPEND_THREADS) {
      const int i = at / items, item = at - i * items;
      const T* x = src + i * p.ssn;
      float* to = s_val + (slot0 + i) * 2 * p.C;
      uint32_t m = 0u;
      int c = (item - turned) * VE;
      if (item >= turned) {
        if (c >= p.start) c += p.dims;
        V::widen(*reinterpret_cast<const Raw*>(x + c), u[0]);
      } else {
        c = p.start + (INTERLEAVED ? 2 * PAIRS : PAIRS) * item;
        const int cb = INTERLEAVED ? c + 1 : c + half;
        float w[VE];
        V::widen(*reinterpret_cast<const Raw*>(x + c), u[0]);
        if constexpr (!ONE) V::widen(*reinterpret_cast<const Raw*>(x + cb), w);
#pragma unroll
        for (int k = 0; k < PAIRS; ++k) {
          const float2 t = s_turn[i * half + item * PAIRS + k];
          float& a = u[0][ONE ? 2 * k : k];
          float& z = ONE ? u[0][ONE ? 2 * k + 1 : 0] : w[k];
          float y0, y1;
          turn_pair(a, z, t.x, t.y, y0, y1);
          a = y0;
          z = y1;
        }
        if constexpr (!ONE) {
#pragma unroll
          for (int k = 0; k < VE; ++k) {
            to[cb + k] = w[k];
            note(w[k], m);
          }
        }
      }
#pragma unroll
      for (int k = 0; k < VE; ++k) {
        to[c + k] = u[0][k];
        note(u[0][k], m);
      }
      amax[0] = max(amax[0], c < p.C ? m : 0u);
      amax[1] = max(amax[1], c < p.C ? 0u : m);
    }
  }
  auto largest = [&]() {  // of the block, in amax
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t m = __reduce_max_sync(0xffffffffu, amax[h]);
      if (lane == 0) s_red[warp][h] = m;
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) amax[h] = __reduce_max_sync(0xffffffffu, s_red[lane % WARPS][h]);
  };
  largest();
  // infinities and values past 448 * 2^60 do not count (seldom: looked at again without them), and become NaN
  if (max(amax[0], amax[1]) > SCALE_TOP_BITS) {
    amax[0] = amax[1] = 0u;
    auto again = [&](float& v, uint32_t& m) {
      if ((__float_as_uint(v) & 0x7fffffffu) <= SCALE_TOP_BITS)
        note(v, m);
      else
        v = __int_as_float(0x7fffffff);
    };
    if constexpr (ROWS) {
#pragma unroll
      for (int g = 0; g < GROUPS; ++g)
        if (entry_of(g) < live) {
#pragma unroll
          for (int k = 0; k < VE; ++k) {
            again(u[2 * g][k], amax[0]);
            again(u[ROWS ? 2 * g + 1 : 0][k], amax[1]);
          }
        }
    } else {
      for (int at = tid; at < live * 2 * p.C; at += APPEND_THREADS)
        again(s_val[slot0 * 2 * p.C + at], amax[at % (2 * p.C) < p.C ? 0 : 1]);
    }
    __syncthreads();  // s_red has been read
    largest();
  }
  float scale[2], inv[2];
  bool grown[2] = {true, true};
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int e = scale_exponent(amax[h], SCALE_LEAST);
    scale[h] = power_of_two(e);
    inv[h] = power_of_two(-e);
    if (older && !(old[h] < scale[h])) {
      grown[h] = false;
      scale[h] = old[h];
      inv[h] = 1.f / old[h];
    }
  }
  if constexpr (ROWS) {
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      const int i = entry_of(g);
      if (i < live) {
        uint8_t* to = rows + (slot0 + i) * p.psr + vec * VE;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float(&x)[VE] = u[ROWS ? 2 * g + h : 0];
          uint32_t out4[VE / 4];
#pragma unroll
          for (int k = 0; k < VE; k += 4)
            out4[k / 4] = pack_e4m3x4(x[k] * inv[h], x[k + 1] * inv[h], x[k + 2] * inv[h], x[k + 3] * inv[h]);
          if constexpr (VE == 8)
            *reinterpret_cast<uint2*>(to + h * p.C) = make_uint2(out4[0], out4[VE / 4 - 1]);
          else
            *reinterpret_cast<uint32_t*>(to + h * p.C) = out4[0];
        }
      }
    }
  } else {
    const int quads = p.C / 2;
    for (int at = tid; at < live * quads; at += APPEND_THREADS) {
      const int i = slot0 + at / quads, c = 4 * (at % quads);
      const float4 v = *reinterpret_cast<const float4*>(s_val + i * 2 * p.C + c);
      const float f = c >= p.C ? inv[1] : inv[0];
      *reinterpret_cast<uint32_t*>(rows + i * p.psr + c) =
          pack_e4m3x4(v.x * f, v.y * f, v.z * f, v.w * f);
    }
  }
  if (older && (grown[0] || grown[1])) {  // a larger scale: the earlier entries are rounded again
    const int quads = p.C / 2;
    const float shrink[2] = {old[0] * inv[0], old[1] * inv[1]};
    for (int at = tid; at < slot0 * quads; at += APPEND_THREADS) {
      const int i = at / quads, c = 4 * (at % quads);
      if (!(c >= p.C ? grown[1] : grown[0])) continue;
      const float f = c >= p.C ? shrink[1] : shrink[0];
      uint32_t* word = reinterpret_cast<uint32_t*>(rows + i * p.psr + c);
      const uint32_t x = *word, y = unpack_e4m3x2(x & 0xffffu), z = unpack_e4m3x2(x >> 16);
      *word = pack_e4m3x4(half_lo(y) * f, half_hi(y) * f, half_lo(z) * f, half_hi(z) * f);
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
//   q (bf16, 8 significant bits), by a power of two that brings the group's
//   largest value into 224 .. 448, is hi + lo / 16, both e4m3: exact down to
//   2^-10 of that value, and within 2^-22.8 of it below. Where a column's own
//   largest value is under 2^-6 of the group's (a head that is off, or a
//   padding query of anything next to it), each column has a power of two of
//   its own, and a tile's scores are multiplied by them where they lie.
//   a weight w = 2^x, as fp16 (11 significant bits) 3 e5m2 numbers, each the
//   upper byte (e5m2 is fp16's) of what the ones before it leave, the second times
//   4 and the last times 32 and rounded to nearest: within 2^-8.6 w (2^-9, and
//   fp16's 2^-11; a bf16 weight's is 2^-8), or 2^-21.8 where w is under 2^-13 (2^-20
//   were the second part not enlarged: under 2^-16 it would hold nothing). 2^15
//   is the largest weight that fits. So what 2^-22 is worth hangs on a column's
//   base, the exponent that stands for a weight of 1, and a key that takes nearly
//   all of the weight (while its value may be next to nothing) must not set it:
//     the first base is the maximum over 32 keys of the first tile, but not more
//     than 8 (base 2) above the least of the maxima over each eight of them;
//     a score 15 above its base raises it, to 12 below that score.
//   A weight under 2^-34 of that of a key that raised the base, or under 2^-14 of
//   the largest of such eight keys, adds nothing to O (all add to the sum). With
//   bases at the maxima themselves, one key of 0.98 of the weight whose value is 0
//   and 32,768 or 262,144 others in one run: off by 20% and 73% of the result;
//   with these 0.18% (the result's own rounding) and 0.21%. Price: 64 rows 59.7
//   us (59.1), scores of four times the deviation 126 (107).
// Scales. A key's scale multiplies its score. A value's scale 2^lv joins the
// exponent, w = 2^(s + lv - m), m the running maximum of s + lv, so O needs no
// scaling; the softmax's sum takes w 2^-lv. Sums, maxima and accumulators are
// fp32.
//
// Work. A group is up to 32 columns (query, head) of a batch row, its tiles
// those that its queries read. (Groups of 64 read each tile once for twice the
// columns, but leave room for one CTA of them on an SM, whose four softmax warps
// are what the time goes to: 45 queries of 24 heads over 1,261 keys 25 us against
// 13, 59 of 32 in 13 rows over 1,073 51 against 41.) Balanced: every CTA works out the groups' tile
// counts and takes an equal run of all tiles in a row, a part of one group or
// of several (segments); a group in several CTAs leaves parts for
// paged_merge_kernel. Otherwise a group's tiles go in equal runs to a cluster of
// up to 8 CTAs that merges through distributed shared memory.
//
// Warps 0-3 prepare q, then take thread r = key r of a tile of 128 (as the
// key-stream kernel's do); warp 4 issues products; warp 5 brings K and V by
// TMA, a box for each page of a tile; warp 6 brings the scales. Two CTAs share
// an SM, so that one's exponents run under the other's loads.
//
// What bounds it: at 64 rows of 1,024 to 32,768 keys and 32 columns HBM and the
// softmax warps' instructions about equally, 61 us for 278 MB (4.5 TB/s), of
// which 5 are the merge; one row of 262,144 keys (27 us) and 7 rows of 5 drafts
// of 12 heads over up to 6,007 (16 us) are chains of latencies: the groups'
// tiles, a page's number, its tile, the products, the parts, the merge. A
// segment's fixed cost is code that is fetched anew for it (the kernel is larger
// than the instruction cache), which is why what runs once a segment is in loops
// that are not unrolled.
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
  float* part_o;                 // (parts, NCOL, 128), not normalised
  float2* part_ml;               // (parts, NCOL): exponent of the maximum, sum
  int2* info;                    // balanced: each group's first part and its parts
  unsigned* status;
  int t64;
  unsigned M, S;                 // pages a row, entries a page
  int B, T, H, P, window;
  int TQ, HG, chunks;            // queries and heads of a group; groups that the heads of a query take (TQ is 1 then)
  int groups_per_row, groups;
  int splits;                    // CTAs of a group, a cluster where > 1; 0: balanced, all groups' tiles over the grid
  float scale_log2;
};

constexpr float PAGED_TOP = 15.f;    // weights up to 2^15 (fp16 ends at 2^16)
constexpr float PAGED_LIFT = 12.f;   // how far a raised base stays below the score that raised it
constexpr float PAGED_APART = 8.f;   // and a first one at most above the least of four maxima
constexpr uint32_t PAGED_EVEN = 6u << 23;  // 2^6 between columns' largest values, up to which they share a power of two
// Minus the base of a column that has read nothing: any score is past it.
constexpr float PAGED_UNSET = 3e38f;

constexpr int PAGED_GROUPS = 256;  // of a balanced call, at most
constexpr int PAGED_SEGMENT = 4;   // what a segment costs beside its tiles, in tiles

template <int NCOL>
struct PagedLayout {
  static constexpr int C = 128, BN = 128;
  static constexpr int NK = 2, NV = 2;  // ring stages of keys and of values
  static constexpr int TILE = BN * C;
  static constexpr int Q_BYTES = 2 * NCOL * C;
  static constexpr int P_BYTES = BN * 128;
  static constexpr int OFF_K = ((Q_BYTES + 1023) / 1024) * 1024;
  static constexpr int OFF_V = OFF_K + NK * TILE;
  static constexpr int OFF_P = OFF_V + NV * TILE;
  static constexpr int OFF_BASE = OFF_P + 2 * P_BYTES;       // minus a column's base, PAGED_UNSET while none is set
  static constexpr int OFF_RED = OFF_BASE + NCOL * 4;        // 4 x NCOL floats
  static constexpr int OFF_ALPHA = OFF_RED + 4 * NCOL * 4;   // the factor of a rescaled column, 1 for others
  static constexpr int OFF_L = OFF_ALPHA + NCOL * 4;
  static constexpr int OFF_TOP = OFF_L + NCOL * 4;           // a column's largest exponent, where it is to be raised
  static constexpr int OFF_POWER = OFF_TOP + NCOL * 4;       // a column's own power of two, where they are uneven
  static constexpr int OFF_SCALE = OFF_POWER + NCOL * 4;       // 2 tiles x 8 blocks x float4
  static constexpr int OFF_NAN = OFF_SCALE + 2 * 8 * 16;     // 4 words a column
  static constexpr int OFF_QLO = OFF_NAN + NCOL * 16;
  static constexpr int OFF_QHI = OFF_QLO + 32 * 4;
  static constexpr int OFF_TILES = OFF_QHI + 32 * 4;         // groups: tiles before each, and the first tile
  static constexpr int OFF_BAR = OFF_TILES + (2 * PAGED_GROUPS + 2) * 4;
  static constexpr int NBAR = 1 + 2 * NK + 2 * NV + 2 + 2 + 1 + 1;
  static constexpr int OFF_MISC = OFF_BAR + NBAR * 8;
  static constexpr int BYTES = OFF_MISC + 64 + 1024;
  static constexpr int S_COLS = 2 * NCOL, O_COLS = 3 * NCOL;
  static constexpr int TMEM_COLS = 2 * S_COLS + O_COLS <= 128 ? 128 : 256;
};

constexpr int PAGED_THREADS = 256;
// Registers: the softmax warps hold a column's score, sum, factor and base
// each, the others little. 128 threads of 200 and 128 of 56 are the 256 of 128
// that a block of two on an SM is launched with.
constexpr int PAGED_REGS = 128, PAGED_REGS_SOFTMAX = 200, PAGED_REGS_OTHERS = 56;

// kind::f8f6f4, fp32 accumulators; types 0 e4m3, 1 e5m2
__host__ __device__ constexpr uint32_t idesc_f8(int M, int N, int a_type, int b_type, int a_mn, int b_mn) {
  return (1u << 4) | (static_cast<uint32_t>(a_type) << 7) | (static_cast<uint32_t>(b_type) << 10) |
         (static_cast<uint32_t>(a_mn) << 15) | (static_cast<uint32_t>(b_mn) << 16) |
         (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}
__device__ __forceinline__ void mma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Four steps of 32 along K, `step` 16-byte units on in both operands: S^T = K
// Q^T (32 channels, rows of 128 bytes: 32 bytes on) or O^T += V^T P^T (32 keys of
// 128 bytes). One thread issues these and their commits.
__device__ __forceinline__ void paged_steps(uint32_t d, uint64_t da, uint64_t db, uint32_t step, uint32_t idesc,
                                            uint32_t accumulate) {
#pragma unroll
  for (int k = 0; k < 4; ++k) mma_f8(d, da + k * step, db + k * step, idesc, k > 0 ? 1u : accumulate);
}

// Group g: the batch row, its queries (query .. query + queries - 1 of the B T), their heads h0 .. h0 + heads - 1;
// rows row0 .. row0 + columns - 1 of the (B T H, 128) queries and results.
struct PagedGroup {
  int b, queries, h0, heads, columns, query, row0;  // (B T H is under 2^31)
  __device__ __forceinline__ PagedGroup(const PagedParams& p, int g) {
    b = g / p.groups_per_row;
    int at = g - b * p.groups_per_row;
    h0 = 0;
    if (p.chunks > 1) {
      h0 = at % p.chunks * p.HG;
      at /= p.chunks;
    }
    const int t0 = at * p.TQ;
    queries = min(p.TQ, p.T - t0);
    heads = min(p.HG, p.H - h0);
    columns = queries * heads;
    query = b * p.T + t0;
    row0 = query * p.H + h0;
  }
};

// The rows that a query at `pos` reads: lo .. hi of its batch row (hi < lo: none).
__device__ __forceinline__ void paged_rows(const PagedParams& p, int64_t pos, int& lo, int& hi) {
  const int64_t last = static_cast<int64_t>(p.M) * p.S - 1;
  const int64_t top = pos < last ? pos : last;
  int64_t low = 0;
  if (p.window > 0 && pos >= p.window) low = pos - p.window + 1;
  hi = top < -1 ? -1 : static_cast<int>(top);
  lo = low > INT_MAX ? INT_MAX : static_cast<int>(low);
}

// fp16 pair (not negative) -> its upper bytes, cut off, and in h what they leave
__device__ __forceinline__ uint32_t e5m2_part(uint32_t& h) {
  const uint32_t part = h & 0xff00ff00u;
  asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(h) : "r"(part));
  return part;
}
// floats in the order of their ints (NaN aside), and back
__device__ __forceinline__ int ordered(float x) {
  const int i = __float_as_int(x);
  return i ^ ((i >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float unordered(int i) { return __int_as_float(i ^ ((i >> 31) & 0x7fffffff)); }
template <uint32_t POWER>  // fp16: both halves times it
__device__ __forceinline__ uint32_t half2_times(uint32_t h) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(h), "r"(POWER * 0x10001u));
  return r;
}
// two fp16 pairs as four e5m2, to nearest even
__device__ __forceinline__ uint32_t pack_e5m2x4(uint32_t ab, uint32_t cd) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e5m2x2.f16x2 %0, %1;" : "=h"(lo) : "r"(ab));
  asm("cvt.rn.satfinite.e5m2x2.f16x2 %0, %1;" : "=h"(hi) : "r"(cd));
  return lo | (static_cast<uint32_t>(hi) << 16);
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
__device__ __forceinline__ void paged_cluster_merge(const PagedParams& p, const float* s_base, const float* s_l,
                                                    const float* s_o, float* s_w, const PagedGroup& group) {
  constexpr int C = 128;
  cluster_sync();
  const int S = p.splits, ncols = group.columns;
  const int64_t row0 = group.row0;
  const int rank = static_cast<int>(cluster_rank());
  const int mine = ncols > rank ? (ncols - rank + S - 1) / S : 0;
  const uint32_t am = smem_u32(s_base), al = smem_u32(s_l), ao = smem_u32(s_o);
  if (static_cast<int>(threadIdx.x) < mine) {
    const int cl = threadIdx.x, c = rank + cl * S;
    float mi[8], li[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      mi[i] = -INFINITY;
      li[i] = 0.f;
      if (i < S) {
        mi[i] = -dsmem_ld(dsmem_map(am + c * 4, i));
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
    s_w[cl * 9 + 8] = paged_total(M, L, p.sink, group.h0 + c % p.HG, inv);
#pragma unroll
    for (int i = 0; i < 8; ++i) s_w[cl * 9 + i] = li[i] != 0.f ? w[i] * inv : 0.f;
  }
  __syncthreads();
#pragma unroll 1
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
__global__ void __launch_bounds__(PAGED_THREADS, 2)
    paged_kernel(const __grid_constant__ CUtensorMap tm, const PagedParams p) {
  using L = PagedLayout<NCOL>;
  constexpr int C = L::C, BN = L::BN, NK = L::NK, NV = L::NV;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sK = smem + L::OFF_K;
  uint8_t* sV = smem + L::OFF_V;
  uint8_t* sP = smem + L::OFF_P;
  float* s_base = reinterpret_cast<float*>(smem + L::OFF_BASE);
  float* s_red = reinterpret_cast<float*>(smem + L::OFF_RED);
  float* s_alpha = reinterpret_cast<float*>(smem + L::OFF_ALPHA);
  float* s_l = reinterpret_cast<float*>(smem + L::OFF_L);
  int* s_top = reinterpret_cast<int*>(smem + L::OFF_TOP);
  float* s_power = reinterpret_cast<float*>(smem + L::OFF_POWER);
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
  uint64_t* s_full = v_empty + NV;  // a tile's scores, and its scales
  uint64_t* p_ready = s_full + 2;
  uint64_t* o_done = p_ready + 2;
  uint64_t* o_final = o_done + 1;   // a segment's last product has completed: a phase a segment
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(smem + L::OFF_MISC);
  int* s_any_nan = reinterpret_cast<int*>(smem + L::OFF_MISC + 4);
  int* s_sum = reinterpret_cast<int*>(smem + L::OFF_MISC + 8);  // 8 warps; later the largest |q| of four
  int* s_before = reinterpret_cast<int*>(smem + L::OFF_TILES);  // [g]: the groups before g, tiles and what is set aside
  int* s_first = s_before + PAGED_GROUPS + 1;                   // [g]: its first tile

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool balanced = p.splits == 0;
  const int gbase = balanced ? 0 : blockIdx.x;  // the group that s_before[0] stands for
  const int gcount = balanced ? p.groups : 1;

  if (warp == 3) {
#pragma unroll 1
    for (int i = lane; i < NCOL * 4; i += 32) s_nan[i] = 0u;
#pragma unroll 1
    for (int i = lane; i < NCOL; i += 32) {
      s_base[i] = PAGED_UNSET;
      s_l[i] = 0.f;
      s_top[i] = INT_MIN;
    }
    if (lane == 0) {
      mbar_init(q_full, 128);
      for (int s = 0; s < NK; ++s) {
        mbar_init(k_full + s, 1);
        mbar_init(k_empty + s, 1);
      }
      for (int s = 0; s < NV; ++s) {
        mbar_init(v_full + s, 1);
        mbar_init(v_empty + s, 1);
      }
      for (int s = 0; s < 2; ++s) {
        mbar_init(s_full + s, 2);
        mbar_init(p_ready + s, 128);
      }
      mbar_init(o_done, 1);
      mbar_init(o_final, 1);
      fence_mbar_init();
      *s_any_nan = 0;
    }
  } else if (warp == 4) {
    tmem_alloc(s_tmem, L::TMEM_COLS);
    tmem_relinquish();
  }
  griddep_wait();
  // the groups' tiles: thread g counts group g's, a scan adds them up
  int count = 0;
  if (static_cast<int>(threadIdx.x) < gcount) {
    const PagedGroup group(p, gbase + threadIdx.x);
    int rlo = INT_MAX, rhi = -1;
#pragma unroll 1
    for (int t = 0; t < group.queries; ++t) {
      int lo, hi;
      paged_rows(p, p.positions[group.query + t], lo, hi);
      if (hi >= lo) {
        rlo = min(rlo, lo);
        rhi = max(rhi, hi);
      }
    }
    int first = 0;
    if (rhi >= 0) {
      first = rlo / BN;
      count = rhi / BN - first + 1;
    }
    s_first[threadIdx.x] = first;
  }
  const int aside = balanced ? PAGED_SEGMENT : 0;
  if (count > 0) count += aside;
  int upto = count;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += x;
  }
  if (lane == 31) s_sum[warp] = upto;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  int all = 0;
#pragma unroll
  for (int w = 0; w < PAGED_THREADS / 32; ++w) {
    if (w < warp) upto += s_sum[w];
    all += s_sum[w];
  }
  s_before[threadIdx.x + 1] = upto;
  if (threadIdx.x == 0) s_before[0] = 0;
  // this CTA's run of tiles
  // no more runs than tiles, so that every CTA from a group's first to its last has a part of it
  const int parts = balanced ? max(1, min(static_cast<int>(gridDim.x), all)) : p.splits;
  const int part_of = balanced ? min(static_cast<int>(blockIdx.x), parts) : blockIdx.y;
  // (all * part_of / parts without 64 bits: parts are under 2^16)
  const unsigned share = static_cast<unsigned>(all) / parts, rest = all - share * parts;
  const int begin = share * part_of + rest * part_of / parts;
  const int end = part_of < parts ? share * (part_of + 1) + rest * (part_of + 1) / parts : begin;
  __syncthreads();
  const uint32_t tmem = *s_tmem;
  griddep_launch();

  // The segments of the run, the same for every warp: next() until false.
  struct Segments {
    const int *before, *first;
    int aside, at, end, g;  // the run's next place; the group (from gbase) of the segment
    int tile0, n;           // its first tile and its tiles
    bool whole;             // all of its group's
    __device__ __forceinline__ bool next() {
#pragma unroll 1
      while (at < end) {
#pragma unroll 1
        while (before[g + 1] <= at) ++g;
        const int from = before[g] + aside, stop = min(end, before[g + 1]);
        tile0 = max(at, from);
        n = stop - tile0;
        tile0 += first[g] - from;
        whole = n == before[g + 1] - from;
        at = stop;
        if (n > 0) return true;  // else the run ends in what is set aside for the group
      }
      return false;
    }
  };
  Segments sg{s_before, s_first, aside, begin, end, 0, 0, 0, false};

  if (balanced && blockIdx.x == 0 && warp == 7) {
    // parts of group g, for the merge: from the CTA whose run holds its first tile to the one that holds its last
    auto holder = [&](int64_t tile) { return static_cast<int>(((tile + 1) * parts + all - 1) / all) - 1; };
#pragma unroll 1
    for (int g = lane; g < gcount; g += 32) {
      const int before = s_before[g], last = s_before[g + 1];
      const int from = last > before ? holder(before + aside) : 0;
      p.info[g] = last > before ? make_int2(from + g, holder(last - 1) - from + 1) : make_int2(0, 0);
    }
  }
  if (begin == end) {  // nothing to read (a cluster's share of that is merged below)
    if (p.splits == 1) {
      const PagedGroup group(p, gbase);
#pragma unroll 1
      for (int i = threadIdx.x; i < group.columns * (C / 2); i += PAGED_THREADS)
        reinterpret_cast<uint32_t*>(p.out + static_cast<int64_t>(group.row0) * C)[i] = 0u;
      if (static_cast<int>(threadIdx.x) < group.columns)
        p.lse[group.row0 + threadIdx.x] = p.sink != nullptr ? p.sink[group.h0 + threadIdx.x % p.HG] : -INFINITY;
    }
  } else if (warp == 5) {
    setmaxnreg_dec<PAGED_REGS_OTHERS>();
    // ------------------------------------------------ keys and values by TMA
    const int rows = min(static_cast<int>(p.S), BN), per = BN / rows;  // entries of a box, boxes of a tile
    const int batch = 32 / per;                      // tiles whose page numbers the warp holds, a lane a box
    const int part = lane % per;
    bool ok = true;
    int j = 0;  // the ring's tile
#pragma unroll 1
    while (ok && sg.next()) {
      const int b = (gbase + sg.g) / p.groups_per_row;
      // the number of this lane's page in tile i0 + lane / per: loaded a batch ahead, checked when it is used
      auto lookup = [&](int i0) {
        const unsigned at = (static_cast<unsigned>(sg.tile0 + i0 + lane / per) * BN + part * rows) / p.S;
        const bool there = i0 + lane / per < sg.n && at < p.M;
        return there ? page_number(p.table, p.t64, b * p.tsb + at) : -1;
      };
      int64_t next = lookup(0);
      int page = -1;
#pragma unroll 1
      for (int i = 0; i < sg.n; ++i, ++j) {
        const int in = i % batch;
        if (in == 0) {
          page = next >= 0 && next < p.P ? static_cast<int>(next) : -1;
          next = lookup(i + batch);
        }
        const int row = static_cast<int>(static_cast<unsigned>(sg.tile0 + i) * BN % p.S);  // 0 for pages within a tile
        const int sk = j % NK, sv = j % NV;
        if (j >= NK) ok = __all_sync(0xffffffffu, mbar_wait(k_empty + sk, ((j / NK) & 1) ^ 1, p.status));
        if (!ok) break;
        if (lane == 0) mbar_expect_tx(k_full + sk, L::TILE);
        __syncwarp();
        if (lane / per == in) tma_load_3d(sK + sk * L::TILE + part * rows * C, &tm, k_full + sk, 0, row, page);
        if (j >= NV) ok = __all_sync(0xffffffffu, mbar_wait(v_empty + sv, ((j / NV) & 1) ^ 1, p.status));
        if (!ok) break;
        if (lane == 0) mbar_expect_tx(v_full + sv, L::TILE);
        __syncwarp();
        if (lane / per == in) tma_load_3d(sV + sv * L::TILE + part * rows * C, &tm, v_full + sv, C, row, page);
      }
    }
  } else if (warp == 6) {
    setmaxnreg_dec<PAGED_REGS_OTHERS>();
    // ------------------------------------- scales: a lane a block, four tiles at a time
    bool ok = true;
    int j = 0;
#pragma unroll 1
    while (ok && sg.next()) {
      const int b = (gbase + sg.g) / p.groups_per_row;
      // page numbers are loaded two batches ahead, scales one
      auto number = [&](int i0) {
        const unsigned at = (static_cast<unsigned>(sg.tile0 + i0 + (lane >> 3)) * BN + (lane & 7) * PAGE_BLOCK) / p.S;
        const bool there = i0 + (lane >> 3) < sg.n && at < p.M;
        return there ? page_number(p.table, p.t64, b * p.tsb + at) : -1;
      };
      auto pair = [&](int i0, int64_t page) {
        if (page < 0 || page >= p.P) return make_float2(0.f, -1.f);  // no page
        const unsigned n = static_cast<unsigned>(sg.tile0 + i0 + (lane >> 3)) * BN + (lane & 7) * PAGE_BLOCK;
        const float* at = p.scales + page * p.scp + n % p.S / PAGE_BLOCK * 2;
        return make_float2(at[0], at[1]);
      };
      int64_t page = number(0);
      float2 raw = pair(0, page);
      bool there = page >= 0 && page < p.P;
      page = number(4);
      float4 mine;
#pragma unroll 1
      for (int i = 0; i < sg.n; ++i, ++j) {
        if ((i & 3) == 0) {
          // key scale; log2 of the value scale, 2^-60 at least (what is scaled by less, as the 0 of an empty
          // block, is nothing), NaN over 2^60; its inverse; 1: there
          const float v = raw.y;
          mine.x = raw.x;
          mine.y = v < power_of_two(SCALE_LEAST) && v >= 0.f ? static_cast<float>(SCALE_LEAST)
                   : v <= power_of_two(60)                   ? log2f(v)
                                                             : __int_as_float(0x7fffffff);
          mine.z = mine.y == mine.y ? fast_exp2(-mine.y) : 1.f;  // (a NaN is in the exponents that are read)
          mine.w = 1.f;
          if (!there) mine = make_float4(0.f, 0.f, 0.f, 0.f);
          raw = pair(i + 4, page);
          there = page >= 0 && page < p.P;
          page = number(i + 8);
        }
        // the slot of tile j - 2 is free once its P V is done (its scores' phase, which this arrival must not
        // fall into, ended before)
        if (j >= 2)
          ok = __all_sync(0xffffffffu, mbar_wait(v_empty + (j - 2) % NV, ((j - 2) / NV) & 1, p.status));
        if (!ok) break;
        if ((lane >> 3) == (i & 3)) s_scale[(j & 1) * 8 + (lane & 7)] = mine;
        __syncwarp();
        if (lane == 0) mbar_arrive(s_full + (j & 1));
      }
    }
  } else if (warp == 4) {
    setmaxnreg_dec<PAGED_REGS_OTHERS>();
    // --------------------------------------------------------- MMA issuer
    constexpr uint32_t IDESC_S = idesc_f8(128, 2 * NCOL, 0, 0, 0, 0);
    constexpr uint32_t IDESC_O = idesc_f8(128, 3 * NCOL, 0, 1, 1, 1);
    const uint32_t tS = tmem, tO = tmem + 2 * L::S_COLS;
    const uint32_t k_addr = smem_u32(sK), v_addr = smem_u32(sV);
    const uint64_t dq = sdesc_sw128(smem_u32(sQ), 16, 1024);
    const uint32_t p_addr = smem_u32(sP);
    auto wait = [&](uint64_t* bar, int parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, p.status)); };
    bool ok = true;
    int j = 0, nseg = 0;
#pragma unroll 1
    while (ok && sg.next()) {
      ok = wait(q_full, nseg++ & 1);
#pragma unroll 1
      for (int i = 0; ok && i <= sg.n; ++i) {
        if (i < sg.n) {
          const int st = j % NK;
          if (!(ok = wait(k_full + st, (j / NK) & 1))) break;
          tc_fence_after();
          if (lane == 0) {
            paged_steps(tS + (j & 1) * L::S_COLS, sdesc_sw128(k_addr + st * L::TILE, 16, 1024), dq, 32 / 16, IDESC_S, 0u);
            mma_commit(s_full + (j & 1));
            mma_commit(k_empty + st);
          }
          __syncwarp();
          ++j;
        }
        if (i > 0) {
          const int jp = i < sg.n ? j - 2 : j - 1, st = jp % NV;
          if (!(ok = wait(v_full + st, (jp / NV) & 1))) break;
          if (!(ok = wait(p_ready + (jp & 1), (jp >> 1) & 1))) break;
          tc_fence_after();
          if (lane == 0) {
            paged_steps(tO, sdesc_sw128(v_addr + st * L::TILE, BN * 128, 1024),
                        sdesc_sw128(p_addr + (jp & 1) * L::P_BYTES, BN * 128, 1024), 32 * 128 / 16, IDESC_O,
                        i > 1 ? 1u : 0u);
            mma_commit(v_empty + st);
            mma_commit(o_done);
            if (i == sg.n) mma_commit(o_final);
          }
          __syncwarp();
        }
      }
    }
  } else if (warp == 7) {
    setmaxnreg_dec<PAGED_REGS_OTHERS>();
  } else {
    setmaxnreg_inc<PAGED_REGS_SOFTMAX>();
    const int r = threadIdx.x;
    const uint32_t lane_addr = tmem + (static_cast<uint32_t>(warp * 32) << 16);
    const uint32_t tO = lane_addr + 2 * L::S_COLS;
    // A segment's queries: each warp's columns (warp, warp + 4, ...), four channels a lane, and a lane's
    // positions, loaded while the segment before ends.
    uint2 ahead_q[NCOL / 4];
    int64_t ahead_pos;
    Segments nx = sg;
    bool more = nx.next();
    auto load_ahead = [&]() {
      const PagedGroup group(p, gbase + nx.g);
      const __nv_bfloat16* q = p.q + static_cast<int64_t>(group.row0) * C + lane * 4;
#pragma unroll
      for (int i = 0; i < NCOL / 4; ++i)
        if (warp + 4 * i < group.columns) ahead_q[i] = *reinterpret_cast<const uint2*>(q + (warp + 4 * i) * C);
      if (lane < group.queries) ahead_pos = p.positions[group.query + lane];
    };
    if (more) load_ahead();
    bool ok = true;
    int j = 0, nseg = 0;
#pragma unroll 1
    while (ok && more) {
      sg = nx;
      const PagedGroup group(p, gbase + sg.g);
      const int ncols = group.columns;
      const uint32_t head_bits = 0xffffffffu >> (32 - group.heads), all_cols = 0xffffffffu >> (32 - ncols);
      // each query's rows, and those that all of them read
      int alo = 0, ahi = INT_MAX;
      if (lane < group.queries) {
        paged_rows(p, ahead_pos, alo, ahi);
        if (warp == 0) {
          s_qlo[lane] = alo;
          s_qhi[lane] = ahi;
        }
      }
      alo = __reduce_max_sync(0xffffffffu, alo);
      ahi = __reduce_min_sync(0xffffffffu, ahi);
      // q: the group's largest value, then hi and lo rows. A query with an infinity or NaN has no result but NaN.
      uint32_t col_q[NCOL / 4], top_q = 0u;
#pragma unroll
      for (int i = 0; i < NCOL / 4; ++i) {
        if (warp + 4 * i >= ncols) ahead_q[i] = make_uint2(0u, 0u);
        const uint2 raw = ahead_q[i];
        col_q[i] = 0u;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t bits = (((k & 2) ? raw.y : raw.x) << ((k & 1) ? 0 : 16)) & 0x7fff0000u;
          col_q[i] = max(col_q[i], bits < 0x7f800000u ? bits : 0u);
        }
        top_q = max(top_q, col_q[i]);
      }
      top_q = __reduce_max_sync(0xffffffffu, top_q);
      if (lane == 0) s_sum[warp] = static_cast<int>(top_q);
      named_barrier(1, 128);
      top_q = max(max(s_sum[0], s_sum[1]), max(s_sum[2], s_sum[3]));
      auto put_q = [&](int col, const uint2& raw, float inv) {  // a column's hi and lo rows, this lane's four channels
        float x[4] = {__uint_as_float(raw.x << 16), __uint_as_float(raw.x & 0xffff0000u),
                      __uint_as_float(raw.y << 16), __uint_as_float(raw.y & 0xffff0000u)};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const bool finite = (__float_as_uint(x[k]) & 0x7fffffffu) < 0x7f800000u;
          x[k] = finite ? x[k] * inv : __int_as_float(0x7fffffff);
        }
        const uint32_t hi = pack_e4m3x4(x[0], x[1], x[2], x[3]);
        const uint32_t u = unpack_e4m3x2(hi & 0xffffu), w = unpack_e4m3x2(hi >> 16);
        const uint32_t lo = pack_e4m3x4((x[0] - half_lo(u)) * 16.f, (x[1] - half_hi(u)) * 16.f,
                                        (x[2] - half_lo(w)) * 16.f, (x[3] - half_hi(w)) * 16.f);
        const uint32_t chunk = lane >> 2, in = (lane & 3) * 4;
        *reinterpret_cast<uint32_t*>(sQ + sw128_offset(col, chunk) + in) = hi;
        *reinterpret_cast<uint32_t*>(sQ + sw128_offset(NCOL + col, chunk) + in) = lo;
      };
      const int e_q = scale_exponent(top_q, -100);
      const float inv_q = power_of_two(-e_q);
      float factor = power_of_two(e_q) * p.scale_log2;
      const uint32_t small = top_q > PAGED_EVEN ? top_q - PAGED_EVEN : 0u;
      bool uneven = false;
#pragma unroll
      for (int i = 0; i < NCOL / 4; ++i) {
        put_q(warp + 4 * i, ahead_q[i], inv_q);
        uneven |= !__any_sync(0xffffffffu, col_q[i] >= small) && __any_sync(0xffffffffu, col_q[i] != 0u);
      }
      uneven = named_barrier_or(1, 128, uneven);  // s_qlo, s_qhi too; s_sum is read
      if (uneven) {
        // (what is over 2^90 stays in the factor, where it meets the key's scale: 2^24 times a column's power of two may
        // be past fp32 although the score is not)
        const int high = max(0, e_q - 90);
        factor = power_of_two(high) * p.scale_log2;
#pragma unroll 1
        for (int col = warp; col < ncols; col += 4) {
          const uint2 raw = *reinterpret_cast<const uint2*>(p.q + (static_cast<int64_t>(group.row0) + col) * C + lane * 4);
          uint32_t top = 0u;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t bits = (((k & 2) ? raw.y : raw.x) << ((k & 1) ? 0 : 16)) & 0x7fff0000u;
            top = max(top, bits < 0x7f800000u ? bits : 0u);
          }
          const int e_col = scale_exponent(__reduce_max_sync(0xffffffffu, top), -100);
          put_q(col, raw, power_of_two(-e_col));
          if (lane == 0) s_power[col] = power_of_two(max(e_col - high, -126));
        }
        if (r >= ncols && r < NCOL) s_power[r] = 0.f;
        named_barrier(1, 128);
      }
      fence_proxy_async();
      mbar_arrive(q_full);

      // softmax: thread r = key r. Pairs of columns: minus bases, sums, exponents
      uint64_t nb[NCOL / 2], lp[NCOL / 2], e[NCOL / 2];
      auto two = [](const float* at, int i) { return reinterpret_cast<const uint64_t*>(at)[i]; };
#pragma unroll
      for (int i = 0; i < NCOL / 2; ++i) lp[i] = 0ull;
#pragma unroll 1
      for (int i = 0; i < sg.n; ++i, ++j) {
        ok = __all_sync(0xffffffffu, mbar_wait(s_full + (j & 1), (j >> 1) & 1, p.status));
        tc_fence_after();
        const float4 sc = s_scale[(j & 1) * 8 + (r >> 4)];
        const float fk = sc.x * factor;
        const uint64_t ks = f2_pack(fk, fk), lv = f2_pack(sc.y, sc.y);
        // which columns read this key; ~0 (padding columns too) where all do
        const int n0 = (sg.tile0 + i) * BN;
        uint32_t vis = ~0u;
        if (n0 < alo || n0 + BN - 1 > ahi) {
          const int row = n0 + r;
          vis = 0u;
#pragma unroll 1
          for (int tq = 0; tq < group.queries; ++tq)
            if (row >= s_qlo[tq] && row <= s_qhi[tq]) vis |= head_bits << (tq * group.heads);
          if (vis == all_cols) vis = ~0u;
        }
        if (sc.w == 0.f) vis = 0u;
        // The maximum is lazy, as in the key-stream kernel: a column's base changes only when a score is PAGED_TOP past
        // it. A segment's first tile sets the bases: the warps with keys that all columns read share the columns, and
        // set each by their own 32 keys (no such key: by the tile's). A tile with a score past its column's bound is
        // taken twice, that column's base being PAGED_LIFT below its maximum then. What is run once in a segment is
        // kept short: such code is fetched anew each time. (A wait that failed is carried to the barriers, where all
        // warps agree to stop.)
        const uint32_t sa = lane_addr + (j & 1) * L::S_COLS;
        if (uneven) {
#pragma unroll 1
          for (int c = 0; c < NCOL; c += 16) {
            uint32_t x[16], y[16];
            tmem_ld16x2(sa + c, sa + NCOL + c, x, y);
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              x[k] = __float_as_uint(fmaf(__uint_as_float(y[k]), 0.0625f, __uint_as_float(x[k])) * s_power[c + k]);
              y[k] = 0u;
            }
            tmem_st16(sa + c, x);
            tmem_st16(sa + NCOL + c, y);
          }
          tmem_wait_st();
        }
        auto score = [&](uint32_t hi, uint32_t lo) {
          return fmaf(fmaf(__uint_as_float(lo), 0.0625f, __uint_as_float(hi)), fk, sc.y);
        };
        if (i == 0) {
          const int from = max(alo, n0), upto = min(ahi, n0 + BN - 1);
          const bool shared = from <= upto;
          const int w0 = (from - n0) >> 5, per = shared ? (NCOL / 8 + ((upto - n0) >> 5) - w0) / (((upto - n0) >> 5) - w0 + 1) * 8 : 0;
          float* to = shared ? s_base : s_red + warp * NCOL;
          const int c_end = !shared ? NCOL : n0 + 32 * warp > upto ? 0 : min(NCOL, (warp - w0 + 1) * per);
#pragma unroll 1
          for (int c = shared ? max(0, warp - w0) * per : 0; c < c_end; c += 8) {
            uint32_t x[8], y[8];
            tmem_ld8x2(sa + c, sa + NCOL + c, x, y);
            float m[8];
            const uint32_t sees = vis >> c;
#pragma unroll
            for (int k = 0; k < 8; ++k) m[k] = (sees >> k) & 1u ? score(x[k], y[k]) : -INFINITY;
            // the maximum over each eight lanes, column c + lane % 8's in m[0]; the largest and the least of the four
            // (of those that read a key)
#pragma unroll
            for (int step = 4; step > 0; step >>= 1)
#pragma unroll
              for (int k = 0; k < step; ++k) {
                const bool up = (lane & step) != 0;
                const float other = __shfl_xor_sync(0xffffffffu, up ? m[k] : m[k + step], step);
                m[k] = fmaxf(up ? m[k + step] : m[k], other);
              }
            float most = m[0], least = m[0] == -INFINITY ? INFINITY : m[0];
#pragma unroll
            for (int step = 8; step < 32; step <<= 1) {
              most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, step));
              least = fminf(least, __shfl_xor_sync(0xffffffffu, least, step));
            }
            if (lane < 8) to[c + lane] = most == -INFINITY ? PAGED_UNSET : -fminf(most, least + PAGED_APART);
          }
          if (!shared) {
            named_barrier(1, 128);
            if (r < NCOL)
              s_base[r] = fminf(fminf(s_red[r], s_red[NCOL + r]), fminf(s_red[2 * NCOL + r], s_red[3 * NCOL + r]));
          }
          if (r == 0) bulk_wait_read();  // the segment before has left P's buffers
          named_barrier(1, 128);
        }
        bool stop = false;
#pragma unroll 1
        for (int pass = 0;; ++pass) {
          // the exponents s + lv - base, the scores rounded as where they set bases: else half a unit in the last place of
          // a score of 2^28 is 2^4 and more of exponent
          if (pass != 0 || i == 0) {
#pragma unroll
            for (int k = 0; k < NCOL / 2; ++k) nb[k] = two(s_base, k);
          }
          const uint64_t low = f2_pack(0.0625f, 0.0625f);
#pragma unroll
          for (int c0 = 0; c0 < NCOL; c0 += 16) {
            uint32_t x[16], y[16];
            tmem_ld16x2(sa + c0, sa + NCOL + c0, x, y);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const int at = c0 / 2 + k;
              const uint64_t t = f2_fma(f2_pack(__uint_as_float(y[2 * k]), __uint_as_float(y[2 * k + 1])), low,
                                        f2_pack(__uint_as_float(x[2 * k]), __uint_as_float(x[2 * k + 1])));
              e[at] = f2_add(f2_fma(t, ks, lv), nb[at]);
            }
          }
          if (vis != ~0u) {
#pragma unroll
            for (int k = 0; k < NCOL / 2; ++k) {
              float x, y;
              f2_unpack(e[k], x, y);
              e[k] = f2_pack((vis >> (2 * k)) & 1u ? x : -INFINITY, (vis >> (2 * k + 1)) & 1u ? y : -INFINITY);
            }
          }
          if (pass == 1) break;
          float top = -INFINITY;
#pragma unroll
          for (int k = 0; k < NCOL / 2; ++k) {
            float x, y;
            f2_unpack(e[k], x, y);
            top = fmaxf(fmaxf(x, y), top);
          }
          if (!named_barrier_or(1, 128, top > PAGED_TOP || !ok)) break;
#pragma unroll 1
          for (int c = 0; c < NCOL; c += 4) {
            uint32_t x[4], y[4];
            tmem_ld4x2(sa + c, sa + NCOL + c, x, y);
            const float4 base = *reinterpret_cast<const float4*>(s_base + c);
            const float past[4] = {base.x, base.y, base.z, base.w};
            const uint32_t sees = vis >> c;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float v = score(x[k], y[k]);
              if (((sees >> k) & 1u) && v + past[k] > PAGED_TOP) atomicMax(s_top + c + k, ordered(v));
            }
          }
          stop = !named_barrier_and(1, 128, ok);
          if (stop) break;
          if (r < NCOL) {
            float a = 1.f;
            if (s_top[r] != INT_MIN) {
              const float base = PAGED_LIFT - unordered(s_top[r]);
              if (s_base[r] != PAGED_UNSET) a = fast_exp2(base - s_base[r]);  // else nothing was added up
              s_base[r] = base;
              s_top[r] = INT_MIN;
            }
            s_alpha[r] = a;
          }
          named_barrier(1, 128);
#pragma unroll
          for (int k = 0; k < NCOL / 2; ++k) lp[k] = f2_mul(lp[k], two(s_alpha, k));
          if (i > 0) {
            // (its parity tells the product before this tile's from the one before that, which is complete: this tile's
            // scores were issued after it)
            ok = __all_sync(0xffffffffu, mbar_wait(o_done, (j - 1) & 1, p.status));
            if (ok) {
              tc_fence_after();
#pragma unroll 1
              for (int c0 = 0; c0 < L::O_COLS; c0 += 16) {
                const float* alpha = s_alpha + c0 % NCOL;
                bool some = false;
#pragma unroll
                for (int c = 0; c < 16; ++c) some |= alpha[c] != 1.f;
                if (!some) continue;
                uint32_t x[16];
                tmem_ld16(tO + c0, x);
#pragma unroll
                for (int c = 0; c < 16; ++c) x[c] = __float_as_uint(__uint_as_float(x[c]) * alpha[c]);
                tmem_st16(tO + c0, x);
              }
              tmem_wait_st();
            }
          }
        }
        if (stop) {
          ok = false;
          break;
        }
        // A value that no column may read is 0 in the product; where only some may (drafts that come before it do
        // not), a NaN in it is taken out of the product and noted for those columns.
        if (vis != ~0u) {
          if (ok) ok = mbar_wait(v_full + j % NV, (j / NV) & 1, p.status);
          uint4* vr = reinterpret_cast<uint4*>(sV + j % NV * L::TILE + r * 128);
          if (vis == 0u && ok) {
#pragma unroll
            for (int i8 = 0; i8 < 8; ++i8) vr[i8 ^ (r & 7)] = make_uint4(0u, 0u, 0u, 0u);
          }
#pragma unroll 1
          for (int i8 = 0; ok && vis != 0u && i8 < 8; ++i8) {  // 16 channels each, others in each lane
            const int at = i8 ^ (r & 7);
            uint4 v = vr[at];
            uint32_t* w = reinterpret_cast<uint32_t*>(&v);
            uint32_t any = 0u, bits = 0u;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint32_t nan = __vcmpeq4(w[k] & 0x7f7f7f7fu, 0x7f7f7f7fu);
              w[k] &= ~nan;
              any |= nan;
              bits |= ((nan & 1u) | (nan >> 7 & 2u) | (nan >> 14 & 4u) | (nan >> 21 & 8u)) << 4 * k;
            }
            if (any != 0u) {
              vr[at] = v;
              *s_any_nan = 1;
              const int ch = (at ^ (r & 7)) * 16;  // the first channel
#pragma unroll 1
              for (int c = 0; c < ncols; ++c)
                if ((vis >> c) & 1u) atomicOr(s_nan + c * 4 + (ch >> 5), bits << (ch & 31));
            }
          }
        }
        __syncwarp();
        // weights, their sums (a key on no page adds 0 times 0), and as fp16 pairs
        uint32_t h[NCOL / 2];
        const uint64_t iv = f2_pack(sc.z, sc.z);
#pragma unroll
        for (int k = 0; k < NCOL / 2; ++k) {
          float x, y;
          f2_unpack(e[k], x, y);
          x = fast_exp2(x);
          y = fast_exp2(y);
          lp[k] = f2_fma(f2_pack(x, y), iv, lp[k]);
          h[k] = pack_half2(x, y);
        }
        // P's buffer is free: the scores came after tile j - 2's P V
        {
          uint8_t* pj = sP + (j & 1) * L::P_BYTES;
#pragma unroll
          for (int c0 = 0; c0 < NCOL; c0 += 16) {
            uint32_t part[3][4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              uint32_t x = h[c0 / 2 + 2 * k], y = h[c0 / 2 + 2 * k + 1];
              part[0][k] = __byte_perm(e5m2_part(x), e5m2_part(y), 0x7531);
              x = half2_times<0x4400>(x);  // 4
              y = half2_times<0x4400>(y);
              part[1][k] = __byte_perm(e5m2_part(x), e5m2_part(y), 0x7531);
              part[2][k] = pack_e5m2x4(half2_times<0x4800>(x), half2_times<0x4800>(y));  // 8
            }
#pragma unroll
            for (int n = 0; n < 3; ++n) {
              const int at = n * NCOL + c0;  // the column's byte in the key's row
              *reinterpret_cast<uint4*>(pj + sw128_offset(r, at >> 4)) =
                  make_uint4(part[n][0], part[n][1], part[n][2], part[n][3]);
            }
          }
        }
        tc_fence_before();
        fence_proxy_async();
        mbar_arrive(p_ready + (j & 1));
      }
      more = nx.next();
      if (more) load_ahead();
      // o_done's parity cannot name the last product here: the last tile's scores vouch for the products up to two tiles
      // before it, whose phase has the same parity, and the two after may still wait for their values. o_final completes
      // once a segment, and every one of its phases is waited for.
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait(o_final, nseg & 1, p.status));
      ++nseg;
      tc_fence_after();
      // per-column sums over the 128 keys
      {
        float tmp[32];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          tmp[2 * i] = tmp[2 * i + 1] = 0.f;
          if (i < NCOL / 2) f2_unpack(lp[i % (NCOL / 2)], tmp[2 * i], tmp[2 * i + 1]);
        }
        const float sum = transpose_reduce32(tmp, SumOp());
        if (lane < NCOL) s_red[warp * NCOL + lane] = sum;
      }
      ok = named_barrier_and(1, 128, ok);
      // a whole group's result is final; else a part
      const bool final = balanced ? sg.whole : p.splits == 1;
      const int64_t seg = static_cast<int64_t>(blockIdx.x) + gbase + sg.g;
      if (r < NCOL) {
        const float l = (s_red[r] + s_red[NCOL + r]) + (s_red[2 * NCOL + r] + s_red[3 * NCOL + r]);
        if (p.splits > 1) {
          s_l[r] = ok ? l : 0.f;
        } else if (r < ncols && final) {
          float inv;
          const float lse = paged_total(l != 0.f ? -s_base[r] : -INFINITY, l, p.sink, group.h0 + r % p.HG, inv);
          s_l[r] = inv;
          if (ok) p.lse[group.row0 + r] = lse;
        } else {
          s_l[r] = 1.f;
          if (r < ncols) p.part_ml[seg * NCOL + r] = ok ? make_float2(-s_base[r], l) : make_float2(-INFINITY, 0.f);
        }
      }
      named_barrier(1, 128);
      // thread r: channel r. The result goes through shared memory, in the P buffers that no product reads any more
      // (a cluster's to be merged from there), and leaves as one bulk copy.
      const bool any_nan = *s_any_nan != 0, wide = !final || p.splits > 1;
#pragma unroll 1
      for (int c = 0; ok && c < NCOL; c += 8) {
        uint32_t x[8], y[8], z[8];
        tmem_ld8x3(tO + c, tO + NCOL + c, tO + 2 * NCOL + c, x, y, z);
        float o[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
          o[k] = fmaf(fmaf(__uint_as_float(z[k]), 0.125f, __uint_as_float(y[k])), 0.25f, __uint_as_float(x[k]));
        if (any_nan) {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if ((s_nan[(c + k) * 4 + (r >> 5)] >> lane) & 1u) o[k] = __int_as_float(0x7fffffff);
        }
        if (wide) {
#pragma unroll
          for (int k = 0; k < 8; ++k) reinterpret_cast<float*>(sP)[(c + k) * C + r] = o[k];
        } else {
          const float4 f0 = *reinterpret_cast<const float4*>(s_l + c), f1 = *reinterpret_cast<const float4*>(s_l + c + 4);
          const float f[8] = {f0.x, f0.y, f0.z, f0.w, f1.x, f1.y, f1.z, f1.w};
#pragma unroll
          for (int k = 0; k < 8; ++k)
            reinterpret_cast<__nv_bfloat16*>(sP)[(c + k) * C + r] = __float2bfloat16_rn(o[k] * f[k]);
        }
      }
      if (p.splits <= 1) {
        fence_proxy_async();
        named_barrier(1, 128);
        if (r == 0 && ok) {
          if (wide)
            bulk_store(p.part_o + seg * NCOL * C, sP, ncols * C * 4);
          else
            bulk_store(p.out + static_cast<int64_t>(group.row0) * C, sP, ncols * C * 2);
          bulk_commit();
        }
      }
      tc_fence_before();
      if (any_nan && more) {  // for the next segment
        if (r < NCOL) {
#pragma unroll
          for (int k = 0; k < 4; ++k) s_nan[r * 4 + k] = 0u;
        }
        if (r == 0) *s_any_nan = 0;
      }
    }
    if (r == 0) bulk_wait_all();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 4) {
    tc_fence_after();
    tmem_dealloc(tmem, L::TMEM_COLS);
  }
  if (p.splits > 1) {
    paged_cluster_merge<NCOL>(p, s_base, s_l, reinterpret_cast<const float*>(sP), reinterpret_cast<float*>(sK),
                              PagedGroup(p, gbase));
  }
}

// Balanced: groups in several CTAs, or in none. A warp a row (query, head),
// four channels a lane; with SPREAD (8 or 32) a row's parts go over that many
// warps of a CTA and are added up in shared memory. One long row has a part in
// every CTA: 8 warps take its 296 parts in 10 rounds of loads, 32 in 3; for
// hundreds of rows of 22 parts CTAs of 32 warps cost more than they save (24 us a
// call against 17).
template <int SPREAD>
__global__ void __launch_bounds__(SPREAD ? SPREAD * 32 : 256) paged_merge_kernel(const PagedParams p, int ncol) {
  griddep_wait();
  constexpr int C = 128, WARPS = SPREAD ? SPREAD : 8, STEP = SPREAD ? WARPS : 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = SPREAD ? blockIdx.x : static_cast<int64_t>(blockIdx.x) * WARPS + warp;
  if (row >= static_cast<int64_t>(p.B) * p.T * p.H) return;
  const int64_t query = row / p.H;
  const int h = static_cast<int>(row - query * p.H);
  const int64_t b = query / p.T;
  const int t = static_cast<int>(query - b * p.T);
  const int64_t group = b * p.groups_per_row + t / p.TQ * p.chunks + h / p.HG;
  const int col = (t % p.TQ) * p.HG + h % p.HG;
  const int2 info = p.info[group];
  if (info.y == 1) return;  // one CTA had all of it
  float M = -INFINITY, L = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  // adds parts (exponents and sums ml, outputs o; a sum of 0: nothing was read, nothing was written)
  constexpr int MOST = 4;
  auto add = [&](const float2 (&ml)[MOST], const float4 (&o)[MOST]) {
    float top = M;
#pragma unroll
    for (int k = 0; k < MOST; ++k)
      if (ml[k].y != 0.f) top = fmaxf(top, ml[k].x);
    if (top != M) {
      const float a = M == -INFINITY ? 0.f : fast_exp2(M - top);
      L *= a;
      acc = make_float4(acc.x * a, acc.y * a, acc.z * a, acc.w * a);
      M = top;
    }
#pragma unroll
    for (int k = 0; k < MOST; ++k) {
      if (ml[k].y == 0.f) continue;
      const float w = fast_exp2(ml[k].x - M);
      L = fmaf(w, ml[k].y, L);
      acc.x = fmaf(w, o[k].x, acc.x);
      acc.y = fmaf(w, o[k].y, acc.y);
      acc.z = fmaf(w, o[k].z, acc.z);
      acc.w = fmaf(w, o[k].w, acc.w);
    }
  };
  for (int s0 = SPREAD ? warp : 0; s0 < info.y; s0 += MOST * STEP) {
    float2 ml[MOST];
    float4 o[MOST];
#pragma unroll
    for (int k = 0; k < MOST; ++k) {
      ml[k] = make_float2(-INFINITY, 0.f);
      o[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (s0 + k * STEP < info.y) {
        const int64_t at = static_cast<int64_t>(info.x + s0 + k * STEP) * ncol + col;
        ml[k] = p.part_ml[at];
        o[k] = *reinterpret_cast<const float4*>(p.part_o + at * C + lane * 4);
      }
    }
    add(ml, o);
  }
  if constexpr (SPREAD) {
    __shared__ float4 s_acc[WARPS][32];
    __shared__ float2 s_ml[WARPS];
    s_acc[warp][lane] = acc;
    if (lane == 0) s_ml[warp] = make_float2(M, L);
    __syncthreads();
    if (warp > 0) return;
    M = -INFINITY;
    L = 0.f;
    acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int w0 = 0; w0 < WARPS && w0 < info.y; w0 += MOST) {
      float2 ml[MOST];
      float4 o[MOST];
#pragma unroll
      for (int k = 0; k < MOST; ++k) {
        ml[k] = s_ml[w0 + k];
        o[k] = s_acc[w0 + k][lane];
      }
      add(ml, o);
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
