// Beam search between two steps: the selection over beams and vocabulary,
// and the reordering of the beams' cached rows.
//
// Selection. Text r's candidate (beam w, token v) has the value
//     totals[r, w] + ((x - m) - log s),  x = scores[r, w, v], m = max_v x,
//     s = sum_v exp(x - m);
// the `beams` largest win (ties: the lowest w * V + v). Within a beam the
// value grows with x, so a beam's best candidates are its largest scores and
// one pass over the scores finds both them and (m, s). beam_scan_kernel: each
// CTA takes a run of one beam's scores. Its first tile gives a bound that the
// K best of the run reach; scores that do go to shared memory, and after 1, 2,
// 4, ... tiles those are ranked and the bound becomes the K-th best so far, so
// that a run of n tiles looks at about K (2 + log2 n) scores twice. Scores equal to
// the bound count only in tokens up to its own.
// beam_merge_kernel: one CTA a text joins the runs' sums, turns the candidates
// into values and ranks them. Bound: HBM, the scores read once.
//
// Different scores can round to one value, of which the lowest index wins, while
// a run keeps its largest scores. So a run ranks one candidate more and hands over
// its score, which no token that it left out passes. Where that score's value is
// the last chosen one's (scores a rounding of the total apart), the merge reads the
// run again for tokens of this value.
//
// The sums are kept in base 2 with a whole number in place of the maximum:
// sum 2^(x L - M), L = log2(e) in fp32, M = round(m L). Moving to a larger M
// is then exact, and the product's one rounding is that of the difference.
//
// Reordering, in place. Every thread owns one unit of bytes of a table place
// across all of a text's beams: it loads that unit of each beam that another
// one takes, and only then stores, so no copy of the table is needed.
#pragma once

#include <cfloat>
#include <cstdint>

#include "common.cuh"
#include "select.cuh"  // order_key

namespace wpt {

constexpr int BEAM_MAX = 64;  // beams in and out
constexpr int BEAM_THREADS = 256;
constexpr int BEAM_PER = 16;    // scores a thread holds at once
constexpr int BEAM_STAGES = 3;  // tiles of 64 bytes a thread on their way to a block
constexpr int BEAM_ROOM = 512;  // candidates of a run above its bound, before they are ranked

struct BeamParams {
  const void* scores;  // (R, W, V)
  int64_t stride_r, stride_w;  // elements
  const float* totals;         // (R, W)
  const uint8_t* done;         // (R, W) or NULL
  float2* stats;               // (R, W, splits): maximum, sum of exp(x - maximum)
  uint64_t* cand;              // (R, W, splits, K + 1): (score, token) keys, best first, 0 for none; the last without token
  float* out_totals;           // (R, K)
  int64_t* parents;            // (R, K)
  int64_t* tokens;             // (R, K)
  int R, W, V, K, splits;
  int tiles;  // tiles of 64 bytes a thread a run
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

// The next number above a key's.
__device__ __forceinline__ float beam_above(uint64_t key) { return beam_key_value(key + (1ull << 32)); }

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

// The upper half of an ended beam's key: that of a NaN, which no candidate has.
constexpr uint64_t BEAM_ENDED = 0xFFFFFFFFull << 32;

// A block's list of the best keys so far, and what it is made from (buf: room for
// the list and the keys offered at once). Keys are unique, so ranks are.
struct BeamShared {
  uint64_t list[BEAM_MAX + 1];  // best first
  uint64_t* buf;            // gathered keys
  alignas(16) uint64_t group[BEAM_THREADS];
  uint64_t bound;
  int count, listed;
};

// A bound that the K best of the threads' keys reach: the K-th largest of the
// maxima of GROUPS >= K groups of threads (top: a thread's largest, 0 for none), 0
// where fewer have one. Of whole keys, or of their upper halves, which is quicker,
// but equal scores then all reach it. Ends after a barrier.
template <int GROUPS, typename Key>
__device__ __forceinline__ void beam_bound_of(BeamShared& s, int K, Key top) {
  constexpr int VEC = 16 / sizeof(Key);
  Key* group = reinterpret_cast<Key*>(s.group);
#pragma unroll
  for (int o = 1; o < BEAM_THREADS / GROUPS; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (threadIdx.x % (BEAM_THREADS / GROUPS) == 0) group[threadIdx.x / (BEAM_THREADS / GROUPS)] = top;
  __syncthreads();
  if (threadIdx.x < GROUPS) {
    const int me = threadIdx.x;
    const Key mine = group[me];
    int rank = 0;
#pragma unroll 8
    for (int i = 0; i < GROUPS; i += VEC) {
      const uint4 raw = *reinterpret_cast<const uint4*>(group + i);
      Key v[VEC];
      if constexpr (VEC == 4) {
        v[0] = raw.x, v[1] = raw.y, v[2] = raw.z, v[3] = raw.w;
      } else {
        v[0] = static_cast<uint64_t>(raw.y) << 32 | raw.x, v[1] = static_cast<uint64_t>(raw.w) << 32 | raw.z;
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) rank += v[j] > mine || (v[j] == mine && i + j < me);
    }
    if (rank == K - 1) s.bound = mine;
  }
  __syncthreads();
}
// The more groups, the fewer keys reach the bound (K = 16 of 64: about 18 a
// tile; K = 64 of 256: 74), and the longer it takes to rank them.
template <typename Key>
__device__ __forceinline__ Key beam_bound(BeamShared& s, int K, Key top) {
  if (K <= 17)
    beam_bound_of<64>(s, K, top);
  else
    beam_bound_of<BEAM_THREADS>(s, K, top);
  return static_cast<Key>(s.bound);
}

// s.list = the K best of the n keys in s.buf, best first.
__device__ __forceinline__ void beam_rank(BeamShared& s, int K, int n) {
  for (int i = threadIdx.x; i < n; i += BEAM_THREADS) {
    const uint64_t mine = s.buf[i];
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) rank += s.buf[j] > mine;
    if (rank < K) s.list[rank] = mine;
  }
  if (threadIdx.x == 0) s.listed = min(n, K);
  __syncthreads();
}

// The list's K best after BEAM_THREADS * PER more keys (key(j): this thread's
// j-th, 0 for none). Bound: whole keys (uint64_t) or upper halves.
template <int PER, typename Bound, class Key>
__device__ __forceinline__ void beam_keep_best(BeamShared& s, int K, Key key) {
  constexpr int SHIFT = 64 - 8 * static_cast<int>(sizeof(Bound));
  Bound top = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) top = max(top, static_cast<Bound>(key(j) >> SHIFT));
  if (threadIdx.x < s.listed) s.buf[threadIdx.x] = s.list[threadIdx.x];
  if (threadIdx.x == 0) s.count = s.listed;
  const Bound bound = beam_bound(s, K, top);
  const uint64_t worst = s.listed == K ? s.list[K - 1] : 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const uint64_t k = key(j);
    if (k > worst && static_cast<Bound>(k >> SHIFT) >= bound) s.buf[atomicAdd(&s.count, 1)] = k;
  }
  __syncthreads();
  beam_rank(s, K, s.count);
}

// Scores past this, 2^29, are at least 32 apart, so that a sum holds only those
// equal to the maximum (e^-32 for the next); where the maximum is past it, they
// are counted in a pass of their own and the running sums stay 0 (masks of a large
// finite value alone in a row, or in all that a thread reads). Up to it M, a rounded
// product, is within 32 of m L, so that no term is out of fp32's range.
constexpr float BEAM_FAR = 536870912.f;

// M for a maximum m: -M has to take every score to 0 or, by its rounding, little more.
__device__ __forceinline__ float beam_shift(float m) {
  return m < -BEAM_FAR ? 0.f : m > BEAM_FAR ? INFINITY : rintf(m * LOG2E);
}
// 2^(from - to) for whole numbers from <= to (0 under 2^-126; to may be infinite).
__device__ __forceinline__ float beam_rescale(float from, float to) {
  return __int_as_float((127 + static_cast<int>(fmaxf(from - to, -127.f))) << 23);
}

// A scan block's shared memory: its tiles, which the second pass of a run with
// too many candidates uses for their keys.
constexpr int BEAM_TILES_BYTES = BEAM_STAGES * BEAM_THREADS * 64;
static_assert(BEAM_TILES_BYTES >= (BEAM_MAX + 1 + BEAM_THREADS * BEAM_PER) * 8, "room for a tile's keys");
template <typename T>
constexpr int BEAM_TILE = BEAM_THREADS * 64 / static_cast<int>(sizeof(T));

// Sends for the 64 bytes of scores that this thread takes of the tile at e0
// (positions are counted from the 16-byte boundary at or before the row; off:
// the row's first, end: past its last), 16 at a time, into its own part of the
// stage; -inf outside the row. Only the thread itself reads them.
template <typename T>
__device__ __forceinline__ void beam_send(uint8_t* stage, const T* from, int64_t e0, int off, int64_t end) {
  constexpr int VEC = 16 / sizeof(T);
  if (e0 >= off && e0 + BEAM_TILE<T> <= end) {
#pragma unroll
    for (int l = 0; l < 4; ++l)
      cp_async_16(smem_u32(stage) + (l * BEAM_THREADS + threadIdx.x) * 16,
                  from + e0 + (l * BEAM_THREADS + threadIdx.x) * VEC, true);
  } else if (e0 < end) {
    for (int l = 0; l < 4; ++l) {
      const int64_t e = e0 + (l * BEAM_THREADS + threadIdx.x) * VEC;
      T* to = reinterpret_cast<T*>(stage) + (l * BEAM_THREADS + threadIdx.x) * VEC;
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        to[i] = e + i >= off && e + i < end ? from[e + i] : static_cast<T>(-INFINITY);
    }
  }
  cp_async_commit();
}

// After a first tile with more scores equal to the bound than there is room for (a
// finite mask over most tokens, equal scores): its candidates again, of equal
// scores those of the lowest tokens. Returns the bound from here on. stage: the
// tile, from token `token0` on. (64 texts of 8 beams with all but
// 65 tokens a beam at -1e9: 36 us, 2,300 without.)
template <typename T>
__device__ __noinline__ float beam_gather_keys(BeamShared& s, uint64_t* room, int K, const uint8_t* stage, int64_t token0) {
  constexpr int PER = 64 / sizeof(T), VEC = 16 / sizeof(T);
  auto key = [&](int j) -> uint64_t {
    const int at = (j / VEC * BEAM_THREADS + threadIdx.x) * VEC + j % VEC;
    const float x = beam_load(reinterpret_cast<const T*>(stage) + at);
    return x > -INFINITY ? beam_key(x, static_cast<uint32_t>(token0 + at)) : 0;
  };
  uint64_t top = 0;
  for (int j = 0; j < PER; ++j) top = max(top, key(j));
  const uint64_t bound = beam_bound(s, K, top);
  if (threadIdx.x == 0) s.count = 0;
  __syncthreads();
  if (top >= bound)
    for (int j = 0; j < PER; ++j) {
      const uint64_t k = key(j);
      if (k == 0 || k < bound) continue;
      const int i = atomicAdd(&s.count, 1);
      if (i < BEAM_ROOM) room[i] = k;
    }
  __syncthreads();
  return bound != 0 ? beam_above(bound) : -FLT_MAX;
}

struct BeamScanShared {
  BeamShared s;
  uint64_t room[BEAM_ROOM];
  float m[BEAM_THREADS / 32], sum[BEAM_THREADS / 32];
};

// One run: `tiles` tiles of beam rw's scores from tile split * tiles on. Returns
// its maximum and sum (in every thread; a NaN or +inf score makes the sum NaN),
// its K best candidates' (score, token) keys in sh.s.list[0 .. sh.s.listed).
template <typename T>
__device__ __forceinline__ float2 beam_scan_run(const BeamParams& p, int K, BeamScanShared& sh, uint8_t* s_tiles,
                                                int64_t rw, int split) {
  constexpr int VEC = 16 / sizeof(T), HALVES = 4 / sizeof(T), TILE = BEAM_TILE<T>;
  BeamShared& s = sh.s;
  const int64_t r = rw / p.W, w = rw - r * p.W;
  const T* row = static_cast<const T*>(p.scores) + r * p.stride_r + w * p.stride_w;
  const int off = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
  const int64_t end = static_cast<int64_t>(off) + p.V;
  const T* from = row - off;
  const int64_t run0 = static_cast<int64_t>(split) * p.tiles * TILE;
  const int64_t run1 = min(end, run0 + static_cast<int64_t>(p.tiles) * TILE);
  // thread t's j-th score of the h-th 16 of its 64 bytes
  auto place = [&](int h, int j) { return ((h * (BEAM_PER / VEC) + j / VEC) * BEAM_THREADS + threadIdx.x) * VEC + j % VEC; };
  if (threadIdx.x == 0) {
    s.count = s.listed = 0;
    s.buf = sh.room;
  }
  int at_stage = 0;
#pragma unroll
  for (int i = 0; i < BEAM_STAGES - 1; ++i)
    beam_send(s_tiles + i * BEAM_THREADS * 64, from, run0 + i * TILE, off, run1);
  float m = -INFINITY, least = -FLT_MAX, shift = 0.f;  // -inf is no candidate
  uint64_t sums[2] = {0, 0};
  int tile = 0;
  for (int64_t e0 = run0; e0 < run1; e0 += TILE, ++tile) {
    cp_async_wait<BEAM_STAGES - 2>();
    const uint8_t* stage = s_tiles + at_stage * BEAM_THREADS * 64;
    float x[BEAM_PER];
#pragma unroll 1
    for (int h = 0; h < HALVES; ++h) {
#pragma unroll
      for (int l = 0; l < BEAM_PER / VEC; ++l)
        beam_load16(reinterpret_cast<const T*>(stage) + ((h * (BEAM_PER / VEC) + l) * BEAM_THREADS + threadIdx.x) * VEC,
                    *reinterpret_cast<float(*)[VEC]>(x + l * VEC));
      if (h == HALVES - 1) {
        // the next tile, into the stage read one tile ago, by this thread
        const int to = at_stage == 0 ? BEAM_STAGES - 1 : at_stage - 1;
        beam_send(s_tiles + to * BEAM_THREADS * 64, from, e0 + (BEAM_STAGES - 1) * TILE, off, run1);
      }
      float top = x[0];
#pragma unroll
      for (int j = 1; j < BEAM_PER; ++j) top = fmaxf(top, x[j]);
      if (e0 == run0 && h == 0) {
        // the bound that every candidate has to reach, from the run's first scores
        const uint32_t bound = beam_bound(s, K, top > -INFINITY ? order_key(top + 0.f) : 0u);
        if (bound != 0) least = beam_key_value(static_cast<uint64_t>(bound) << 32);
      }
      if (top >= least) {
        unsigned found = 0;
#pragma unroll
        for (int j = 0; j < BEAM_PER; ++j) found |= (x[j] >= least ? 1u : 0u) << j;
        int i = atomicAdd(&s.count, __popc(found));
        for (; found && i < BEAM_ROOM; found &= found - 1, ++i) {
          const int at = __ffs(found) - 1;
          float value = x[0];
#pragma unroll
          for (int j = 1; j < BEAM_PER; ++j) value = at == j ? x[j] : value;
          sh.room[i] = beam_key(value, static_cast<uint32_t>(e0 + place(h, at) - off));
        }
      }
      if (top > m) {
        m = top;
        const float was = shift;
        shift = beam_shift(m);
        const float f = sums[0] == 0 && sums[1] == 0 ? 1.f : beam_rescale(was, shift);
        sums[0] = f2_mul(sums[0], f2_pack(f, f));
        sums[1] = f2_mul(sums[1], f2_pack(f, f));
      }
      // a NaN score makes the sum NaN, and so does +inf (inf - inf)
      const uint64_t l2 = f2_pack(LOG2E, LOG2E), s2 = f2_pack(-shift, -shift);
#pragma unroll
      for (int j = 0; j < BEAM_PER; j += 2) {
        float a, b;
        f2_unpack(f2_fma(f2_pack(x[j], x[j + 1]), l2, s2), a, b);
        sums[(j / 2) & 1] = f2_add(sums[(j / 2) & 1], f2_pack(fast_exp2(a), fast_exp2(b)));
      }
    }
    at_stage = at_stage == BEAM_STAGES - 1 ? 0 : at_stage + 1;
    if ((tile & (tile + 1)) == 0 && e0 + TILE < run1) {
      // after 1, 2, 4, ... tiles: the K best so far give a better bound
      __syncthreads();
      const int n = s.count;
      __syncthreads();
      if (n <= BEAM_ROOM) {
        beam_rank(s, K, n);
        if (threadIdx.x < s.listed) sh.room[threadIdx.x] = s.list[threadIdx.x];
        if (threadIdx.x == 0) s.count = s.listed;
        // the tokens from here on are higher: scores equal to the last one do not count
        if (s.listed == K) least = fmaxf(least, beam_above(s.list[K - 1]));
        __syncthreads();
      } else if (tile == 0) {
        least = beam_gather_keys<T>(s, sh.room, K, stage, e0 - off);
      }
    }
  }
  // (m, sum) over the block
  float sum, other;
  f2_unpack(f2_add(sums[0], sums[1]), sum, other);
  sum += other;
  float mm = m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) sh.m[warp] = mm;
  __syncthreads();
  mm = sh.m[0];
#pragma unroll
  for (int i = 1; i < BEAM_THREADS / 32; ++i) mm = fmaxf(mm, sh.m[i]);
  if (sum != 0.f) sum *= beam_rescale(shift, beam_shift(mm));
  if (fabsf(mm) > BEAM_FAR && fabsf(mm) < INFINITY)
    for (int64_t e = max(run0, static_cast<int64_t>(off)) + threadIdx.x; e < run1; e += BEAM_THREADS)
      sum += beam_load(from + e) == mm ? 1.f : 0.f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) sh.sum[warp] = sum;
  __syncthreads();
  sum = 0.f;
#pragma unroll
  for (int i = 0; i < BEAM_THREADS / 32; ++i) sum += sh.sum[i];
  if (s.count <= BEAM_ROOM) {
    beam_rank(s, K, s.count);
  } else {
    // more scores reached the bound than there is room for (scores that rise
    // along the vocabulary, or many equal ones): once more over the run,
    // keeping the best after every 16 scores a thread
    cp_async_wait<0>();
    __syncthreads();
    if (threadIdx.x == 0) {
      s.buf = reinterpret_cast<uint64_t*>(s_tiles);
      s.listed = 0;
    }
    __syncthreads();
    for (int64_t e0 = run0; e0 < run1; e0 += TILE) {
      for (int h = 0; h < HALVES; ++h) {
        float x[BEAM_PER], top = -INFINITY;
#pragma unroll
        for (int j = 0; j < BEAM_PER; ++j) {
          const int64_t e = e0 + place(h, j);
          x[j] = e >= off && e < run1 ? beam_load(from + e) : -INFINITY;
          top = fmaxf(top, x[j]);
        }
        const float worst = s.listed == K ? beam_key_value(s.list[K - 1]) : -INFINITY;
        if (__syncthreads_or(top > worst))
          beam_keep_best<BEAM_PER, uint64_t>(s, K, [&](int j) -> uint64_t {
            return x[j] > -INFINITY ? beam_key(x[j], static_cast<uint32_t>(e0 + place(h, j) - off)) : 0;
          });
      }
    }
  }
  return make_float2(mm, sum);
}

struct BeamMergeShared {
  BeamShared s;
  uint64_t keys[BEAM_MAX + BEAM_THREADS * 4];
  float m[BEAM_MAX], log[BEAM_MAX];
  uint8_t again[BEAM_THREADS];
};

// The value of a candidate with the score x: it does not fall where x grows.
__device__ __forceinline__ float beam_value(float total, float x, float m, float log) { return total + ((x - m) - log); }

// Offers the tokens that their run left out and whose value is the last chosen one's.
template <typename T, class Cand>
__device__ __noinline__ void beam_read_again(const BeamParams& p, BeamMergeShared& sh, int64_t r, Cand cand) {
  constexpr int TILE = BEAM_TILE<T>, GROUPS = 4, PER = 4;
  constexpr uint64_t STEP = (sizeof(T) == 2 ? 0x10000ull : 1ull) << 32;  // between the keys of T's neighbouring numbers
  BeamShared& s = sh.s;
  const float tie = beam_key_value(s.list[p.K - 1]);
  const int runs = p.W * p.splits;
  for (int c0 = 0; c0 < runs; c0 += BEAM_THREADS) {
    bool again = false;
    if (c0 + static_cast<int>(threadIdx.x) < runs) {
      const int w = (c0 + threadIdx.x) / p.splits, i = (c0 + threadIdx.x) - w * p.splits;
      if (p.done == nullptr || !p.done[r * p.W + w]) {
        const uint64_t key = cand(w, i, p.K);
        const float total = p.totals[r * p.W + w];
        auto value = [&](uint64_t k) { return beam_value(total, beam_key_value(k), sh.m[w], sh.log[w]); };
        // where no other score has this value, what was left out has higher tokens than what was kept
        again = key != 0 && value(key) == tie && !(value(key + STEP) > tie && value(key - STEP) < tie);
      }
    }
    sh.again[threadIdx.x] = again;
    __syncthreads();
    for (int t = 0; t < BEAM_THREADS && c0 + t < runs; ++t) {
      if (!sh.again[t]) continue;
      const int w = (c0 + t) / p.splits, i = (c0 + t) - w * p.splits;
      const T* row = static_cast<const T*>(p.scores) + r * p.stride_r + w * p.stride_w;
      const float total = p.totals[r * p.W + w], m = sh.m[w], log = sh.log[w];
      // the run's scores, as beam_scan_run counts them, without the part before the row
      const int off = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
      const int64_t v0 = max(static_cast<int64_t>(0), static_cast<int64_t>(i) * p.tiles * TILE - off);
      const int64_t v1 = min(static_cast<int64_t>(p.V), static_cast<int64_t>(i + 1) * p.tiles * TILE - off);
      for (int64_t v = v0 + threadIdx.x; v - threadIdx.x < v1; v += BEAM_THREADS * GROUPS * PER) {
        uint64_t key[GROUPS * PER];
        bool any = false;
#pragma unroll
        for (int j = 0; j < GROUPS * PER; ++j) {
          const int64_t at = v + j * BEAM_THREADS;
          const float value = at < v1 ? beam_value(total, beam_load(row + at), m, log) : -INFINITY;
          key[j] = value == tie ? beam_key(value, static_cast<uint32_t>(w) * p.V + static_cast<uint32_t>(at)) : 0;
          if (key[j] <= s.list[p.K - 1]) key[j] = 0;
          for (int k = 0; key[j] != 0 && k < p.K; ++k)
            if (s.list[k] == key[j]) key[j] = 0;  // it is chosen already
          any |= key[j] != 0;
        }
        if (!__syncthreads_or(any)) continue;
#pragma unroll
        for (int g = 0; g < GROUPS; ++g)
          beam_keep_best<PER, uint32_t>(s, p.K, [&](int j) { return key[g * PER + j]; });
      }
    }
    __syncthreads();
  }
}

// Text r's choice from its runs: stat(w, i) the maximum and sum of beam w's i-th
// of `splits` runs, cand(w, i, k) its k-th candidate, 0 for none, and for k = K
// the score that no other of its tokens passes, without a token (neither is
// asked of an ended beam).
template <typename T, class Stat, class Cand>
__device__ __forceinline__ void beam_merge(const BeamParams& p, BeamMergeShared& sh, int64_t r, Stat stat, Cand cand) {
  constexpr int PER = 4;
  BeamShared& s = sh.s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slots = p.K + 1, per_beam = p.splits * slots;
  const int total = p.W * per_beam;
  // a thread's candidates of the tile at c0: (score, token) keys (an ended
  // beam's first place: its end token), and their beams' totals
  uint64_t found[PER];
  float before[PER];
  auto load = [&](int c0) {
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int c = c0 + j * BEAM_THREADS + threadIdx.x;
      found[j] = 0;
      if (c >= total) continue;
      const int w = c / per_beam, i = c - w * per_beam;
      before[j] = p.totals[r * p.W + w];
      if (p.done == nullptr || !p.done[r * p.W + w])
        found[j] = cand(w, i / slots, i % slots);
      else if (i == 0)
        found[j] = BEAM_ENDED | (0xFFFFFFFFu - static_cast<uint32_t>(p.end));
    }
  };
  load(0);
  for (int w = warp; w < p.W; w += BEAM_THREADS / 32) {
    if (p.done != nullptr && p.done[r * p.W + w]) continue;
    float m = -INFINITY;
    for (int i = lane; i < p.splits; i += 32) m = fmaxf(m, stat(w, i).x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float shift = beam_shift(m);
    float sum = 0.f;
    for (int i = lane; i < p.splits; i += 32) {
      const float2 v = stat(w, i);
      // a NaN stays one whatever its weight
      const float weight = fabsf(m) > BEAM_FAR ? (v.x == m ? 1.f : 0.f)
                           : v.x < -BEAM_FAR   ? 0.f
                                               : beam_rescale(beam_shift(v.x), shift);
      sum += v.y * weight;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) {
      // log sum exp(x - m) from sum 2^(x L - M), where 2^L = e^(L ln 2)
      sh.m[w] = m;
      const double moved =
          fabsf(m) > BEAM_FAR ? 0. : (static_cast<double>(shift) - static_cast<double>(m) * LOG2E) * 0.69314718055994531;
      sh.log[w] = static_cast<float>(moved + log(static_cast<double>(sum)));
    }
  }
  if (threadIdx.x == 0) {
    s.listed = 0;
    s.buf = sh.keys;
  }
  __syncthreads();
  float others = -INFINITY;  // no other token of this thread's runs passes this value
  for (int c0 = 0; c0 < total; c0 += BEAM_THREADS * PER) {
    if (c0 > 0) load(c0);
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if (found[j] == 0) continue;
      const int w = (c0 + j * BEAM_THREADS + static_cast<int>(threadIdx.x)) / per_beam;
      const uint32_t token = 0xFFFFFFFFu - static_cast<uint32_t>(found[j]);
      const float value = (found[j] >> 32) == (BEAM_ENDED >> 32)
                              ? before[j]
                              : beam_value(before[j], beam_key_value(found[j]), sh.m[w], sh.log[w]);
      if (token == 0xFFFFFFFFu) others = fmaxf(others, value);
      found[j] = value > -INFINITY && token != 0xFFFFFFFFu ? beam_key(value, static_cast<uint32_t>(w) * p.V + token) : 0;
    }
    beam_keep_best<PER, uint32_t>(s, p.K, [&](int j) { return found[j]; });
  }
  if (__syncthreads_or(others > -INFINITY && s.listed == p.K && others >= beam_key_value(s.list[p.K - 1])))
    beam_read_again<T>(p, sh, r, cand);
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

template <typename T>
__global__ void __launch_bounds__(BEAM_THREADS, 4) beam_scan_kernel(const __grid_constant__ BeamParams p) {
  extern __shared__ __align__(16) uint8_t s_tiles[];
  __shared__ BeamScanShared sh;
  const int split = blockIdx.x % p.splits;
  const int64_t rw = blockIdx.x / p.splits;
  griddep_wait();
  if (p.done != nullptr && p.done[rw]) return;  // an ended beam's scores are not read
  const float2 stat = beam_scan_run<T>(p, p.K + 1, sh, s_tiles, rw, split);
  const int64_t run = rw * p.splits + split;
  griddep_launch();
  if (threadIdx.x == 0) p.stats[run] = stat;
  if (threadIdx.x <= p.K) {
    const uint64_t key = threadIdx.x < sh.s.listed ? sh.s.list[threadIdx.x] : 0;
    p.cand[run * (p.K + 1) + threadIdx.x] = threadIdx.x < p.K ? key : key >> 32 << 32;
  }
}

template <typename T>
__global__ void __launch_bounds__(BEAM_THREADS) beam_merge_kernel(const __grid_constant__ BeamParams p) {
  __shared__ BeamMergeShared sh;
  const int64_t r = blockIdx.x;
  griddep_wait();
  beam_merge<T>(
      p, sh, r, [&](int w, int i) { return p.stats[(r * p.W + w) * p.splits + i]; },
      [&](int w, int i, int k) { return p.cand[((r * p.W + w) * p.splits + i) * (p.K + 1) + k]; });
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
