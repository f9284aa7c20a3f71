// Beam search between two steps: the selection over beams and vocabulary,
// and the reordering of the beams' cached rows.
//
// Selection. Text r's candidate (beam w, token v) has the value
//     totals[r, w] + ((x - m) - log s),  x = scores[r, w, v], m = max_v x,
//     s = sum_v exp(x - m);
// the `beams` largest win (ties: the lowest w * V + v). Within a beam the
// value grows with x, so a beam's best candidates are its largest scores and
// one pass over the scores finds both them and (m, s). beam_scan_kernel: each
// CTA takes a run of one beam's scores, keeps a running (m, s) a thread and
// the run's best candidates in shared memory; a tile of scores is looked at
// again only when one of them beats the worst of the best so far.
// beam_merge_kernel: one CTA a text joins the runs' (m, s), turns the
// candidates into values and ranks them. Bound: HBM, the scores read once.
//
// Reordering, in place. Every thread owns one unit of bytes of a table place
// across all of a text's beams: it loads that unit of each beam that another
// one takes, and only then stores, so no copy of the table is needed.
#pragma once

#include <cstdint>

#include "common.cuh"
#include "select.cuh"  // order_key

namespace wpt {

constexpr int BEAM_MAX = 64;  // beams in and out
constexpr int BEAM_THREADS = 256;
constexpr int BEAM_PER = 16;  // scores a thread holds at once
constexpr int BEAM_TILE = BEAM_THREADS * BEAM_PER;
constexpr int BEAM_ROOM = 1024;  // candidates of a run above its bound, before they are ranked
constexpr int BEAM_GROUPS = 64;  // groups of threads whose maxima give the gather's bound

struct BeamParams {
  const void* scores;  // (R, W, V)
  int64_t stride_r, stride_w;  // elements
  const float* totals;         // (R, W)
  const uint8_t* done;         // (R, W) or NULL
  float2* stats;               // (R, W, splits): maximum, sum of exp(x - maximum)
  uint64_t* cand;              // (R, W, splits, K): (score, token) keys, best first, 0 for none
  float* out_totals;           // (R, K)
  int64_t* parents;            // (R, K)
  int64_t* tokens;             // (R, K)
  int R, W, V, K, splits;
  int tiles;  // tiles of BEAM_TILE scores a run
  int end;
};

// Orders by value, then by the lower index: unique for unique indices.
__device__ __forceinline__ uint64_t beam_key(float x, uint32_t index) {
  return (static_cast<uint64_t>(order_key(x + 0.f)) << 32) | (0xFFFFFFFFu - index);
}
__device__ __forceinline__ float beam_key_value(uint64_t key) {
  const uint32_t k = static_cast<uint32_t>(key >> 32);
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}

__device__ __forceinline__ float beam_load(const float* p) { return *p; }
__device__ __forceinline__ float beam_load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void beam_load16(const float* p, float (&x)[4]) {
  const float4 f = *reinterpret_cast<const float4*>(p);
  x[0] = f.x;
  x[1] = f.y;
  x[2] = f.z;
  x[3] = f.w;
}
__device__ __forceinline__ void beam_load16(const __nv_bfloat16* p, float (&x)[8]) {
  const uint4 f = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}

// The K best keys of BEAM_THREADS * PER offered ones and of the list of the
// best so far, by all BEAM_THREADS threads. key(j): this thread's j-th key (0
// for none). s_buf holds the list in its first *count entries and has room
// for BEAM_MAX + BEAM_THREADS * PER. Keys are unique, so ranks are.
struct BeamShared {
  uint64_t list[BEAM_MAX];                 // the best so far, best first
  uint64_t buf[BEAM_MAX + BEAM_TILE];      // gathered keys
  uint32_t group[BEAM_GROUPS];
  uint32_t bound;
  int count, listed;
};

// A bound that the K best of the threads' keys reach: the K-th largest of the
// maxima of BEAM_GROUPS groups of threads (top: a thread's largest key's
// upper half, 0 for none). Ends after a barrier.
__device__ __forceinline__ uint32_t beam_bound(BeamShared& s, int K, uint32_t top) {
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
  if ((threadIdx.x & 3) == 0) s.group[threadIdx.x >> 2] = top;
  __syncthreads();
  if (threadIdx.x < 32) {
    const uint32_t a = s.group[threadIdx.x], b = s.group[threadIdx.x + 32];
    uint32_t bound = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t mid = bound | (1u << bit);
      const int at_least = __popc(__ballot_sync(0xffffffffu, a >= mid)) + __popc(__ballot_sync(0xffffffffu, b >= mid));
      if (at_least >= K) bound = mid;
    }
    if (threadIdx.x == 0) s.bound = bound;
  }
  __syncthreads();
  return s.bound;
}

// s.list = the K best of the n unique keys in s.buf, best first.
__device__ __forceinline__ void beam_rank(BeamShared& s, int K, int n) {
  for (int i = threadIdx.x; i < n; i += BEAM_THREADS) {
    const uint64_t mine = s.buf[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += s.buf[j] > mine;
    if (rank < K) s.list[rank] = mine;
  }
  if (threadIdx.x == 0) s.listed = min(n, K);
  __syncthreads();
}

template <int PER, class Key>
__device__ __forceinline__ void beam_keep_best(BeamShared& s, int K, Key key) {
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) top = max(top, static_cast<uint32_t>(key(j) >> 32));
  if (threadIdx.x < s.listed) s.buf[threadIdx.x] = s.list[threadIdx.x];
  if (threadIdx.x == 0) s.count = s.listed;
  const uint32_t bound = beam_bound(s, K, top);
  const uint64_t worst = s.listed == K ? s.list[K - 1] : 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const uint64_t k = key(j);
    if (k > worst && static_cast<uint32_t>(k >> 32) >= bound) s.buf[atomicAdd(&s.count, 1)] = k;
  }
  __syncthreads();
  beam_rank(s, K, s.count);
}

// A thread's BEAM_PER scores of the tile at e0 (positions are counted from the
// 16-byte boundary at or before the row; off: the row's first): -inf outside it.
template <typename T>
__device__ __forceinline__ void beam_load_tile(const T* from, int64_t e0, int off, int64_t end, float (&x)[BEAM_PER]) {
  constexpr int VEC = 16 / sizeof(T);
#pragma unroll
  for (int l = 0; l < BEAM_PER / VEC; ++l) {
    const int64_t e = e0 + (l * BEAM_THREADS + threadIdx.x) * VEC;
    float f[VEC];
    if (e >= off && e + VEC <= end) {
      beam_load16(from + e, f);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) f[i] = e + i >= off && e + i < end ? beam_load(from + e + i) : -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) x[l * VEC + i] = f[i];
  }
}

template <typename T>
__global__ void __launch_bounds__(BEAM_THREADS, 4) beam_scan_kernel(const BeamParams p) {
  constexpr int VEC = 16 / sizeof(T);
  __shared__ BeamShared s;
  __shared__ float s_m[BEAM_THREADS / 32], s_s[BEAM_THREADS / 32];
  const int split = blockIdx.x % p.splits;
  const int64_t rw = blockIdx.x / p.splits;
  const int64_t r = rw / p.W, w = rw - r * p.W;
  griddep_wait();
  if (p.done != nullptr && p.done[rw]) return;  // an ended beam's scores are not read
  const T* row = static_cast<const T*>(p.scores) + r * p.stride_r + w * p.stride_w;
  const int off = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
  const int64_t end = static_cast<int64_t>(off) + p.V;
  const T* from = row - off;
  const int64_t run0 = static_cast<int64_t>(split) * p.tiles * BEAM_TILE;
  const int64_t run1 = min(end, run0 + static_cast<int64_t>(p.tiles) * BEAM_TILE);
  auto key_of = [&](float x, int64_t e0, int j) -> uint64_t {
    const int64_t e = e0 + ((j / VEC) * BEAM_THREADS + threadIdx.x) * VEC + j % VEC;
    return x > -INFINITY ? beam_key(x, static_cast<uint32_t>(e - off)) : 0;
  };
  if (threadIdx.x == 0) s.count = s.listed = 0;
  float m = -INFINITY, sum = 0.f, least = -INFINITY;
  float x[BEAM_PER];
  beam_load_tile(from, run0, off, end, x);
  for (int64_t e0 = run0; e0 < run1; e0 += BEAM_TILE) {
    float next[BEAM_PER];
    if (e0 + BEAM_TILE < run1) beam_load_tile(from, e0 + BEAM_TILE, off, end, next);
    float top = x[0];
#pragma unroll
    for (int j = 1; j < BEAM_PER; ++j) top = fmaxf(top, x[j]);
    if (e0 == run0) {
      // the bound that every candidate has to reach, from the run's first tile
      const uint32_t bound = beam_bound(s, p.K, top > -INFINITY ? order_key(top + 0.f) : 0u);
      least = bound == 0 ? -INFINITY : beam_key_value(static_cast<uint64_t>(bound) << 32);
    }
    if (top >= least && top > -INFINITY) {
#pragma unroll
      for (int j = 0; j < BEAM_PER; ++j)
        if (x[j] >= least && x[j] > -INFINITY) {
          const int i = atomicAdd(&s.count, 1);
          if (i < BEAM_ROOM) s.buf[i] = key_of(x[j], e0, j);
        }
    }
    if (top > m) {
      sum *= fast_exp2((m - top) * LOG2E);
      m = top;
    }
    // a NaN score makes the sum NaN, and so does +inf (inf - inf)
    const float shift = m == -INFINITY ? 0.f : m;
    float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < BEAM_PER; ++j) part[j & 3] += fast_exp2((x[j] - shift) * LOG2E);
    sum += (part[0] + part[1]) + (part[2] + part[3]);
#pragma unroll
    for (int j = 0; j < BEAM_PER; ++j) x[j] = next[j];
  }
  griddep_launch();
  // (m, sum) over the block
  float mm = m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) s_m[warp] = mm;
  __syncthreads();
  mm = s_m[0];
#pragma unroll
  for (int i = 1; i < BEAM_THREADS / 32; ++i) mm = fmaxf(mm, s_m[i]);
  // a thread that met nothing above -inf holds 0, or NaN
  if (m > -INFINITY) sum *= fast_exp2((m - mm) * LOG2E);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) s_s[warp] = sum;
  __syncthreads();
  const int64_t run = rw * p.splits + split;
  if (threadIdx.x == 0) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < BEAM_THREADS / 32; ++i) t += s_s[i];
    p.stats[run] = make_float2(mm, t);
  }
  if (s.count <= BEAM_ROOM) {
    beam_rank(s, p.K, s.count);
  } else {
    // more scores reached the first tile's bound than there is room for
    // (scores that rise along the vocabulary, or many equal ones): once more
    // over the run, keeping the best after every tile
    for (int64_t e0 = run0; e0 < run1; e0 += BEAM_TILE) {
      beam_load_tile(from, e0, off, end, x);
      float top = x[0];
#pragma unroll
      for (int j = 1; j < BEAM_PER; ++j) top = fmaxf(top, x[j]);
      const float worst = s.listed == p.K ? beam_key_value(s.list[p.K - 1]) : -INFINITY;
      if (__syncthreads_or(top > worst)) beam_keep_best<BEAM_PER>(s, p.K, [&](int j) { return key_of(x[j], e0, j); });
    }
  }
  if (threadIdx.x < p.K) p.cand[run * p.K + threadIdx.x] = threadIdx.x < s.listed ? s.list[threadIdx.x] : 0;
}

__global__ void __launch_bounds__(BEAM_THREADS) beam_merge_kernel(const BeamParams p) {
  constexpr int PER = 4;
  __shared__ BeamShared s;
  __shared__ float s_m[BEAM_MAX], s_log[BEAM_MAX];
  const int64_t r = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  griddep_wait();
  for (int w = warp; w < p.W; w += BEAM_THREADS / 32) {
    if (p.done != nullptr && p.done[r * p.W + w]) continue;
    const float2* st = p.stats + (r * p.W + w) * p.splits;
    float m = -INFINITY;
    for (int i = lane; i < p.splits; i += 32) m = fmaxf(m, st[i].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    float sum = 0.f;
    for (int i = lane; i < p.splits; i += 32) {
      const float2 v = st[i];
      // a run of -inf scores only adds nothing; a NaN sum stays NaN
      sum += v.x > -INFINITY || isnan(v.y) ? v.y * expf(v.x - m) : 0.f;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) {
      s_m[w] = m;
      s_log[w] = logf(sum);
    }
  }
  if (threadIdx.x == 0) s.listed = 0;
  __syncthreads();
  const int per_beam = p.splits * p.K;
  const int total = p.W * per_beam;
  for (int c0 = 0; c0 < total; c0 += BEAM_THREADS * PER) {
    uint64_t keys[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int c = c0 + j * BEAM_THREADS + threadIdx.x;
      uint64_t key = 0;
      if (c < total) {
        const int w = c / per_beam;
        const float t = p.totals[r * p.W + w];
        float value = -INFINITY;
        uint32_t token = 0;
        if (p.done != nullptr && p.done[r * p.W + w]) {
          if (c == w * per_beam) value = t, token = p.end;
        } else {
          const uint64_t k = p.cand[(r * p.W + w) * per_beam + (c - w * per_beam)];
          if (k) {
            value = t + ((beam_key_value(k) - s_m[w]) - s_log[w]);
            token = 0xFFFFFFFFu - static_cast<uint32_t>(k);
          }
        }
        if (value > -INFINITY) key = beam_key(value, static_cast<uint32_t>(w) * p.V + token);
      }
      keys[j] = key;
    }
    beam_keep_best<PER>(s, p.K, [&](int j) { return keys[j]; });
  }
  if (threadIdx.x < p.K) {
    const int64_t o = r * p.K + threadIdx.x;
    const bool some = threadIdx.x < s.listed;
    const uint64_t k = some ? s.list[threadIdx.x] : 0;
    const uint32_t flat = 0xFFFFFFFFu - static_cast<uint32_t>(k);
    p.out_totals[o] = some ? beam_key_value(k) : -INFINITY;
    p.parents[o] = some ? static_cast<int64_t>(flat / static_cast<uint32_t>(p.V)) : -1;
    p.tokens[o] = some ? static_cast<int64_t>(flat % static_cast<uint32_t>(p.V)) : -1;
  }
}

// --------------------------------------------------------------- reordering

constexpr int REORDER_TABLES = 32;  // tables a launch
constexpr int REORDER_THREADS = 256;

struct ReorderTable {
  uint8_t* base;
  int64_t stride_b, stride_n;  // bytes
  int units;                   // units of a row
  int capacity;                // rows
};

struct ReorderParams {
  ReorderTable table[REORDER_TABLES];
  const int64_t* parents;  // (R, W)
  const int64_t* lengths;  // (R * W,)
  const int64_t* first;    // (R,) or NULL
  unsigned* status;
  int R, W, chunks;  // chunks: CTAs a (table, text)
};

// MAXW: the most beams an instance takes (its units in registers).
template <typename Unit, int MAXW>
__global__ void __launch_bounds__(REORDER_THREADS) reorder_kernel(const __grid_constant__ ReorderParams p) {
  __shared__ int s_src[MAXW], s_len[MAXW], s_n, s_top;
  __shared__ unsigned long long s_dst[MAXW];  // the beams that take source i
  __shared__ unsigned long long s_takers[MAXW];
  const int chunk = blockIdx.x % p.chunks;
  const int tr = blockIdx.x / p.chunks;
  const int r = tr % p.R;
  const ReorderTable& t = p.table[tr / p.R];
  const int w = threadIdx.x;
  if (w < MAXW) s_takers[w] = 0;
  if (w == 0) s_n = s_top = 0;
  griddep_wait();
  __syncthreads();
  int64_t len = 0;
  if (w < p.W) {
    const int64_t parent = p.parents[static_cast<int64_t>(r) * p.W + w];
    len = p.lengths[static_cast<int64_t>(r) * p.W + w];
    if (parent >= p.W)
      atomicOr(p.status, STATUS_BAD_SHAPE);
    else if (parent >= 0 && parent != w)
      atomicOr(&s_takers[parent], 1ull << w);
  }
  __syncthreads();
  if (w < p.W && s_takers[w] != 0) {  // a source: its slot may be any
    const int i = atomicAdd(&s_n, 1);
    s_src[i] = w;
    s_dst[i] = s_takers[w];
    s_len[i] = len < 0 ? 0 : len > t.capacity ? t.capacity : static_cast<int>(len);
    atomicMax(&s_top, s_len[i]);
  }
  __syncthreads();
  const int n_src = s_n;
  const int64_t asked = p.first == nullptr ? 0 : p.first[r];
  const int64_t first = asked < 0 ? 0 : asked > t.capacity ? t.capacity : asked;
  const int64_t u1 = static_cast<int64_t>(s_top) * t.units;
  uint8_t* base = t.base + static_cast<int64_t>(r) * p.W * t.stride_b;
  for (int64_t u = first * t.units + chunk * REORDER_THREADS + threadIdx.x; u < u1;
       u += static_cast<int64_t>(p.chunks) * REORDER_THREADS) {
    const int row = static_cast<int>(u / t.units), c = static_cast<int>(u - static_cast<int64_t>(row) * t.units);
    uint8_t* at = base + row * t.stride_n + c * static_cast<int64_t>(sizeof(Unit));
    Unit v[MAXW];
#pragma unroll
    for (int i = 0; i < MAXW; ++i)
      if (i < n_src && row < s_len[i]) v[i] = *reinterpret_cast<const Unit*>(at + s_src[i] * t.stride_b);
#pragma unroll
    for (int i = 0; i < MAXW; ++i)
      if (i < n_src && row < s_len[i])
        for (unsigned long long d = s_dst[i]; d; d &= d - 1)
          *reinterpret_cast<Unit*>(at + (__ffsll(static_cast<long long>(d)) - 1) * t.stride_b) = v[i];
  }
}

}  // namespace wpt
