// Eviction from the generation cache by accumulated attention weight: each
// cache row b keeps, of its lengths[b] live table rows, the first `first`
// and the last `recent` ones and those of the others with the largest
// weights (ties: the lowest row), `keep` in all, in their order, at the
// front of new tables.
//
// evict_rows_kernel finds them: a cluster of `slices` CTAs a row, each with a
// contiguous slice of the row's keys in shared memory. The threshold key is
// found by histograms over equal ranges, first of all keys (lowest to highest:
// a float's bits grow like its logarithm, so skewed weights spread over the
// bins), then of the one bin that holds it, until a bin's keys are all kept or
// all equal; the slices' histograms are summed over distributed shared memory.
// A count of the kept rows before each warp's run of keys gives their places.
// evict_gather_kernel copies the kept entries: the selection wants few CTAs a
// row, the copy every SM. A few of them the selection's own CTAs copy. 64 rows of
// 8,192 keys to 2,048 entries of 512 bytes: 31 us, of them 22 for the copy's 134
// MB (6.1 TB/s).
#pragma once

#include <cstdint>

#include "common.cuh"
#include "select.cuh"  // order_key

namespace wpt {

constexpr int EVICT_THREADS = 1024;  // a whole block a row, or slice: the selection is a chain of block steps
constexpr int EVICT_BINS = 2048;
constexpr int EVICT_SLICES = 8;  // most CTAs a row (a portable cluster)
constexpr int EVICT_QUADS = 4 * EVICT_THREADS;  // a slice is a multiple of this: whole quads a thread
constexpr int EVICT_COPY_THREADS = 256, EVICT_COPY_CTAS = 5;  // CTAs an SM

struct GatherParams {
  const uint8_t* src;
  int64_t src_sb, src_sn;  // bytes
  uint8_t* dst;            // (B, capacity, row_bytes), contiguous
  const int64_t* rows;     // (B, keep)
  int keep, capacity, units;  // units of a row (row_bytes / sizeof(Unit))
  int chunks;                 // CTAs a cache row
};

// Copies row rows[b, i] to place i of the new table, for the places of chunk
// `chunk`, and writes zeros where there is none (rows[b, i] = -1, and the places
// from keep to capacity: a product over a whole tile of the new table
// multiplies its unread rows by zero weights, which must not meet a NaN).
template <typename Unit, int THREADS>
__device__ __forceinline__ void evict_copy(const GatherParams& p, int b, int chunk) {
  constexpr int ROWS = 4;  // places a thread has in flight
  const uint8_t* src = p.src + b * p.src_sb;
  Unit* dst = reinterpret_cast<Unit*>(p.dst) + static_cast<int64_t>(b) * p.capacity * p.units;
  const int64_t* rows = p.rows + static_cast<int64_t>(b) * p.keep;
  // a group of threads a place, a unit each (long rows: several)
  const int group = min(p.units, THREADS), groups = THREADS / group;
  const int mine = threadIdx.x / group, unit = threadIdx.x - mine * group;
  if (mine >= groups) return;
  const int step = p.chunks * groups;
  auto row_of = [&](int64_t i) { return i < p.keep ? static_cast<int>(__ldcg(rows + i)) : -1; };
  int next[ROWS];  // the rows of the places after these, read while these are copied
  const int64_t begin = static_cast<int64_t>(chunk) * groups + mine;
#pragma unroll
  for (int k = 0; k < ROWS; ++k) next[k] = row_of(begin + static_cast<int64_t>(k) * step);
  for (int64_t i0 = begin; i0 < p.capacity; i0 += static_cast<int64_t>(ROWS) * step) {
    const Unit* from[ROWS];
#pragma unroll
    for (int k = 0; k < ROWS; ++k)
      from[k] = next[k] >= 0 ? reinterpret_cast<const Unit*>(src + next[k] * p.src_sn) : nullptr;
#pragma unroll
    for (int k = 0; k < ROWS; ++k) next[k] = row_of(i0 + static_cast<int64_t>(ROWS + k) * step);
    for (int c = unit; c < p.units; c += group) {
      Unit v[ROWS];
#pragma unroll
      for (int k = 0; k < ROWS; ++k) v[k] = from[k] != nullptr ? from[k][c] : Unit{};
#pragma unroll
      for (int k = 0; k < ROWS; ++k) {
        const int64_t i = i0 + static_cast<int64_t>(k) * step;
        if (i < p.capacity) dst[i * p.units + c] = v[k];
      }
    }
  }
}

template <typename Unit>
__global__ void __launch_bounds__(EVICT_COPY_THREADS, EVICT_COPY_CTAS) evict_gather_kernel(const GatherParams p) {
  griddep_wait();
  const int b = blockIdx.x / p.chunks;
  evict_copy<Unit, EVICT_COPY_THREADS>(p, b, blockIdx.x - b * p.chunks);
}

struct EvictParams {
  const float* weights;  // (B, N), row stride weights_ld
  int64_t weights_ld;
  const int64_t* lengths;  // (B,)
  int64_t* rows;           // (B, keep)
  float* weights_out;      // (B, capacity)
  int64_t* counts;         // (B,)
  int N, keep, recent, first, capacity;
  int slices;     // CTAs (one cluster) a row
  int cache_cap;  // keys of a slice that shared memory holds
  int copy;       // 16 or 4: this kernel copies the entries too, in units of so many bytes; 0: another does
  GatherParams gather;
};

// The key that orders weights: larger weights, larger keys; -0 as +0; NaN as
// -inf (a poisoned weight does not hold its row).
__device__ __forceinline__ uint32_t evict_key(float x) {
  return order_key(isnan(x) ? -INFINITY : x + 0.f);
}

__device__ __forceinline__ uint32_t dsmem_ld_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ uint2 dsmem_ld_u32x2(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared::cluster.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
  return v;
}

// The copy by the row's own CTAs, once all of them have written their rows.
__device__ __forceinline__ void evict_copy_here(const EvictParams& p, int b, int rank) {
  if (p.copy == 0) return;
  if (p.slices > 1)
    cluster_sync();
  else
    __syncthreads();
  if (p.copy == 16)
    evict_copy<uint4, EVICT_THREADS>(p.gather, b, rank);
  else
    evict_copy<uint32_t, EVICT_THREADS>(p.gather, b, rank);
}

__global__ void __launch_bounds__(EVICT_THREADS) evict_rows_kernel(const EvictParams p) {
  extern __shared__ __align__(16) uint32_t s_keys[];  // cache_cap keys
  __shared__ __align__(16) uint32_t s_hist[2][EVICT_BINS];
  __shared__ int s_warp[EVICT_THREADS / 32];
  __shared__ uint32_t s_red[EVICT_THREADS / 16];
  __shared__ int s_gt[EVICT_THREADS / 32], s_eq[EVICT_THREADS / 32];
  __shared__ int s_tot[2];
  __shared__ uint32_t s_mm[2];
  __shared__ int s_bin, s_above, s_in;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.x / p.slices;
  const uint32_t rank = p.slices > 1 ? cluster_rank() : 0u;
  reinterpret_cast<uint4*>(s_hist)[threadIdx.x] = make_uint4(0, 0, 0, 0);
  static_assert(sizeof(s_hist) == EVICT_THREADS * 16, "a quad a thread");
  griddep_wait();
  const int64_t raw = p.lengths[b];
  const int len = raw < 0 ? 0 : raw > p.N ? p.N : static_cast<int>(raw);
  const int count = len < p.keep ? len : p.keep;
  const float* src = p.weights + static_cast<int64_t>(b) * p.weights_ld;
  int64_t* rows = p.rows + static_cast<int64_t>(b) * p.keep;
  float* kept = p.weights_out + static_cast<int64_t>(b) * p.capacity;
  if (rank == 0) {
    for (int i = count + threadIdx.x; i < p.keep; i += EVICT_THREADS) rows[i] = -1;
    for (int i = count + threadIdx.x; i < p.capacity; i += EVICT_THREADS) kept[i] = 0.f;
    if (threadIdx.x == 0) p.counts[b] = count;
  }
  if (len <= p.keep) {  // everything is kept (the same decision on all CTAs of the cluster)
    for (int i = rank * EVICT_THREADS + threadIdx.x; i < len; i += p.slices * EVICT_THREADS) {
      rows[i] = i;
      kept[i] = src[i];
    }
    evict_copy_here(p, b, rank);
    return;
  }

  // this CTA's slice [base, base + n), in quads; `quads` of them a thread
  const int quads = ((len + p.slices - 1) / p.slices + EVICT_QUADS - 1) / EVICT_QUADS, slice = quads * EVICT_QUADS;
  const int64_t base64 = static_cast<int64_t>(rank) * slice;
  const int base = base64 < len ? static_cast<int>(base64) : len;
  const int n = min(slice, len - base);
  const bool cached = slice <= p.cache_cap;
  const int kept_from = len - p.recent - base;  // slice indices from here on, and under kept_to, are always kept
  const int kept_to = p.first - base;
  constexpr uint32_t ALWAYS = 0xFFFFFFFFu;  // their key; the others' are from 0x007FFFFF (-inf) to 0xFF800000; none: 0
  const bool aligned = (reinterpret_cast<uintptr_t>(src + base) & 15) == 0;
  // the weights' keys of quad c, whether always kept or not
  auto load4 = [&](int c) {
    const int i = 4 * c;
    if (aligned && i + 4 <= n) {
      const float4 f = *reinterpret_cast<const float4*>(src + base + i);
      return make_uint4(evict_key(f.x), evict_key(f.y), evict_key(f.z), evict_key(f.w));
    }
    uint4 k = make_uint4(0, 0, 0, 0);
    if (i < n) k.x = evict_key(src[base + i]);
    if (i + 1 < n) k.y = evict_key(src[base + i + 1]);
    if (i + 2 < n) k.z = evict_key(src[base + i + 2]);
    if (i + 3 < n) k.w = evict_key(src[base + i + 3]);
    return k;
  };
  auto keys4 = [&](int c) {
    if (cached) return reinterpret_cast<const uint4*>(s_keys)[c];
    uint4 k = load4(c);
    const int i = 4 * c;
    if (i < kept_to || i + 3 >= kept_from) {
      if (i < n && (i < kept_to || i >= kept_from)) k.x = ALWAYS;
      if (i + 1 < n && (i + 1 < kept_to || i + 1 >= kept_from)) k.y = ALWAYS;
      if (i + 2 < n && (i + 2 < kept_to || i + 2 >= kept_from)) k.z = ALWAYS;
      if (i + 3 < n && (i + 3 < kept_to || i + 3 >= kept_from)) k.w = ALWAYS;
    }
    return k;
  };
  auto meet = [&] {
    if (p.slices > 1)
      cluster_sync();
    else
      __syncthreads();
  };

  // bounds of the keys, and the keys into shared memory
  uint32_t lo = ALWAYS, hi = 0;
  for (int c0 = 0; c0 < quads * EVICT_THREADS; c0 += 4 * EVICT_THREADS) {
    uint4 k[4];
    const int in = min(4, quads - c0 / EVICT_THREADS);  // quads a thread takes now
#pragma unroll
    for (int h = 0; h < 4; ++h)
      if (h < in) k[h] = load4(c0 + h * EVICT_THREADS + threadIdx.x);
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      if (h >= in) break;
      if (cached) reinterpret_cast<uint4*>(s_keys)[c0 + h * EVICT_THREADS + threadIdx.x] = k[h];
      hi = max(max(hi, max(k[h].x, k[h].y)), max(k[h].z, k[h].w));
      // 0, past the slice's end, wraps to the largest
      lo = min(min(lo, min(k[h].x - 1, k[h].y - 1)), min(k[h].z - 1, k[h].w - 1));
    }
  }
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  if (lane == 0) {
    s_red[warp] = lo;
    s_red[32 + warp] = hi;
  }
  __syncthreads();
  if (cached) {  // the always kept rows' keys
    for (int i = threadIdx.x; i < min(kept_to, n); i += EVICT_THREADS) s_keys[i] = ALWAYS;
    for (int i = max(kept_from, 0) + threadIdx.x; i < n; i += EVICT_THREADS) s_keys[i] = ALWAYS;
  }
  lo = __reduce_min_sync(0xffffffffu, s_red[lane]);
  hi = __reduce_max_sync(0xffffffffu, s_red[32 + lane]);
  if (p.slices > 1) {
    if (threadIdx.x == 0) {
      s_mm[0] = lo;
      s_mm[1] = hi;
    }
    cluster_sync();
    for (int r = 0; r < p.slices; ++r) {
      lo = min(lo, dsmem_ld_u32(dsmem_map(smem_u32(s_mm), r)));
      hi = max(hi, dsmem_ld_u32(dsmem_map(smem_u32(s_mm + 1), r)));
    }
  } else {
    __syncthreads();
  }
  lo += 1;

  // the threshold: keys above it are kept, and the first `ties` of those equal to it
  uint32_t threshold = ALWAYS - 1;
  int ties = 0, need = p.keep - p.first - p.recent;
  for (int pass = 0; need > 0; ++pass) {
    // keys in [lo, hi], in bins of 2^shift
    const uint32_t range = hi - lo;
    const int shift = range < EVICT_BINS ? 0 : 32 - __clz(range) - 11;
    uint32_t* hist = s_hist[pass & 1];
    auto tally = [&](uint32_t key) {  // 0 and ALWAYS are out of the range
      const uint32_t d = key - lo;
      if (d <= range) atomicAdd(&hist[d >> shift], 1u);
    };
    for (int c = threadIdx.x; c < quads * EVICT_THREADS; c += EVICT_THREADS) {
      const uint4 k = keys4(c);
      tally(k.x);
      tally(k.y);
      tally(k.z);
      tally(k.w);
    }
    meet();
    // The bins from the top, two a thread: each warp's sum, the warps above
    // it, and the bin where the count reaches `need`.
    const int top_bin = EVICT_BINS - 1 - 2 * threadIdx.x;
    int c0 = 0, c1 = 0;
    if (p.slices > 1) {
      uint2 c[EVICT_SLICES];  // all slices' loads in flight at once
#pragma unroll
      for (int r = 0; r < EVICT_SLICES; ++r)
        c[r] = r < p.slices ? dsmem_ld_u32x2(dsmem_map(smem_u32(hist + top_bin - 1), r)) : make_uint2(0, 0);
#pragma unroll
      for (int r = 0; r < EVICT_SLICES; ++r) {
        c0 += c[r].y;
        c1 += c[r].x;
      }
    } else {
      c0 = hist[top_bin];
      c1 = hist[top_bin - 1];
    }
    const int sum = __reduce_add_sync(0xffffffffu, c0 + c1);
    if (lane == 0) s_warp[warp] = sum;
    __syncthreads();
    int before = __reduce_add_sync(0xffffffffu, lane < warp ? s_warp[lane] : 0);
    if (before < need && need <= before + sum) {
      int incl = c0 + c1;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
      }
      before += incl - c0 - c1;
      if (before < need && need <= before + c0) {
        s_bin = top_bin;
        s_above = before;
        s_in = c0;
      } else if (before + c0 < need && need <= before + c0 + c1) {
        s_bin = top_bin - 1;
        s_above = before + c0;
        s_in = c1;
      }
    }
    __syncthreads();
    const uint32_t bin_lo = lo + (static_cast<uint32_t>(s_bin) << shift);
    need -= s_above;
    if (s_in == need) {  // the whole bin is kept
      threshold = bin_lo - 1;
      break;
    }
    if (shift == 0) {  // one key's bin
      threshold = bin_lo;
      ties = need;
      break;
    }
    lo = bin_lo;
    hi = min(hi, bin_lo + ((1u << shift) - 1u));
    // The two histograms take turns. The next one was last read in the pass
    // before this one, by CTAs that have all come to this pass's meeting.
    if (pass > 0) {
      uint32_t* next = s_hist[(pass + 1) & 1];
      for (int i = threadIdx.x; i < EVICT_BINS; i += EVICT_THREADS) next[i] = 0;
      __syncthreads();
    }
  }

  // kept rows of each warp's run of quads, and of the warps and slices before it
  int gt = 0, eq = 0;
  const int run0 = warp * 32 * quads + lane;
  for (int q = 0; q < quads; ++q) {
    const uint4 k = keys4(run0 + 32 * q);
    gt += (k.x > threshold) + (k.y > threshold) + (k.z > threshold) + (k.w > threshold);
    eq += (k.x == threshold) + (k.y == threshold) + (k.z == threshold) + (k.w == threshold);
  }
  gt = __reduce_add_sync(0xffffffffu, gt);
  eq = __reduce_add_sync(0xffffffffu, eq);
  if (lane == 0) {
    s_gt[warp] = gt;
    s_eq[warp] = eq;
  }
  __syncthreads();
  if (p.slices > 1) {
    if (warp == 0) {
      gt = __reduce_add_sync(0xffffffffu, s_gt[lane]);
      eq = __reduce_add_sync(0xffffffffu, s_eq[lane]);
      if (lane == 0) {
        s_tot[0] = gt;
        s_tot[1] = eq;
      }
    }
    cluster_sync();
  }
  gt = __reduce_add_sync(0xffffffffu, lane < warp ? s_gt[lane] : 0);
  eq = __reduce_add_sync(0xffffffffu, lane < warp ? s_eq[lane] : 0);
  for (uint32_t r = 0; r < rank; ++r) {
    gt += dsmem_ld_u32(dsmem_map(smem_u32(s_tot), r));
    eq += dsmem_ld_u32(dsmem_map(smem_u32(s_tot + 1), r));
  }
  // their places: lanes hold consecutive quads, so that a warp's stores are next to each other
  for (int q = 0; q < quads; ++q) {
    const int c = run0 + 32 * q;
    const uint4 k = keys4(c);
    const uint32_t key[4] = {k.x, k.y, k.z, k.w};
    int mine = 0;  // above the threshold, and 2^16 times equal to it
#pragma unroll
    for (int h = 0; h < 4; ++h) mine += key[h] > threshold ? 1 : key[h] == threshold ? 1 << 16 : 0;
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    const int all = __shfl_sync(0xffffffffu, incl, 31);
    int g = gt + ((incl - mine) & 0xFFFF), e = eq + ((incl - mine) >> 16);
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      const bool above = key[h] > threshold, equal = key[h] == threshold;
      if (above || (equal && e < ties)) {
        const int place = g + min(e, ties);
        rows[place] = base + 4 * c + h;
        // the key gives the weight back, but for -0, -inf and NaN and always kept rows
        const uint32_t x = key[h];
        kept[place] = x > 0x80000000u && x < ALWAYS       ? __uint_as_float(x & 0x7FFFFFFFu)
                      : x > 0x007FFFFFu && x < 0x80000000u ? __uint_as_float(~x)
                                                           : src[base + 4 * c + h];
      }
      g += above;
      e += equal;
    }
    gt += all & 0xFFFF;
    eq += all >> 16;
  }
  // a CTA's totals stay readable until every CTA has read them
  if (p.copy != 0)
    evict_copy_here(p, b, rank);
  else if (p.slices > 1)
    cluster_sync();
}

}  // namespace wpt
