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
// evict_gather_kernel copies the kept entries. Two kernels rather than one:
// the selection wants few CTAs a row, the copy wants every SM.
#pragma once

#include <cstdint>

#include "common.cuh"
#include "select.cuh"  // order_key, block_exclusive_scan

namespace wpt {

constexpr int EVICT_THREADS = TOPK_THREADS;  // block_exclusive_scan's block
constexpr int EVICT_BINS = 2048;
constexpr int EVICT_COPY_THREADS = 256;

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

__global__ void __launch_bounds__(EVICT_THREADS) evict_rows_kernel(const EvictParams p) {
  extern __shared__ uint32_t s_keys[];  // cache_cap keys
  __shared__ uint32_t s_hist[2][EVICT_BINS];
  __shared__ int s_warp[EVICT_THREADS / 32];
  __shared__ uint32_t s_red[EVICT_THREADS / 16];
  __shared__ int s_gt[EVICT_THREADS / 32], s_eq[EVICT_THREADS / 32];
  __shared__ int s_tot[2];
  __shared__ uint32_t s_mm[2];
  __shared__ int s_bin, s_above, s_in;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.x / p.slices;
  const uint32_t rank = p.slices > 1 ? cluster_rank() : 0u;
  for (int i = threadIdx.x; i < 2 * EVICT_BINS; i += EVICT_THREADS) (&s_hist[0][0])[i] = 0;
  griddep_wait();
  const int64_t raw = p.lengths[b];
  const int len = raw < 0 ? 0 : raw > p.N ? p.N : static_cast<int>(raw);
  const int count = len < p.keep ? len : p.keep;
  const bool cut = len > p.keep;
  const float* src = p.weights + static_cast<int64_t>(b) * p.weights_ld;

  // this CTA's slice [base, base + n), cut into one run of `run` keys a warp
  const int slice = ((len + p.slices - 1) / p.slices + EVICT_THREADS - 1) / EVICT_THREADS * EVICT_THREADS;
  const int64_t base64 = static_cast<int64_t>(rank) * slice;
  const int base = base64 < len ? static_cast<int>(base64) : len;
  const int n = min(slice, len - base);
  const int run = slice / (EVICT_THREADS / 32);
  const bool cached = n <= p.cache_cap;
  const int kept_from = len - p.recent;  // rows from here on, and those before `first`, are always kept
  constexpr uint32_t ALWAYS = 0xFFFFFFFFu;  // their key; the others' are at most +inf's, 0xFF800000
  auto make_key = [&](int i) -> uint32_t {  // i: index in the slice
    const int row = base + i;
    return row < p.first || row >= kept_from ? ALWAYS : evict_key(src[row]);
  };
  // (nothing competes, and nothing is cached, when the always kept rows fill the budget)
  auto key_at = [&](int i) { return cached && p.keep > p.first + p.recent ? s_keys[i] : make_key(i); };
  auto meet = [&] {
    if (p.slices > 1)
      cluster_sync();
    else
      __syncthreads();
  };

  // the threshold: keys above it are kept, and the first `ties` of those equal to it
  uint32_t threshold = ALWAYS - 1;
  int ties = 0, need = p.keep - p.first - p.recent;
  if (cut && need > 0) {
    uint32_t lo = ALWAYS, hi = 0;  // of the keys that compete
    if (cached) {
#pragma unroll 4
      for (int i = threadIdx.x; i < n; i += EVICT_THREADS) {
        const uint32_t key = make_key(i);
        s_keys[i] = key;
        if (key != ALWAYS) {
          lo = min(lo, key);
          hi = max(hi, key);
        }
      }
    } else {
      for (int i = threadIdx.x; i < n; i += EVICT_THREADS) {
        const uint32_t key = make_key(i);
        if (key != ALWAYS) {
          lo = min(lo, key);
          hi = max(hi, key);
        }
      }
    }
    block_minmax(lo, hi, s_red);
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
    }
    for (int pass = 0;; ++pass) {
      // keys in [lo, hi], in bins of 2^shift
      const uint32_t range = hi - lo;
      const int shift = range < EVICT_BINS ? 0 : 32 - __clz(range) - 11;
      uint32_t* hist = s_hist[pass & 1];
#pragma unroll 4
      for (int i = threadIdx.x; i < n; i += EVICT_THREADS) {
        const uint32_t d = key_at(i) - lo;  // ALWAYS is above hi
        if (d <= range) atomicAdd(&hist[d >> shift], 1u);
      }
      meet();
      // The bins from the top, two a thread.
      const int top_bin = EVICT_BINS - 1 - 2 * threadIdx.x;
      uint32_t c0 = 0, c1 = 0;
      if (p.slices > 1) {
        for (int r = 0; r < p.slices; ++r) {
          c0 += dsmem_ld_u32(dsmem_map(smem_u32(hist + top_bin), r));
          c1 += dsmem_ld_u32(dsmem_map(smem_u32(hist + top_bin - 1), r));
        }
      } else {
        c0 = hist[top_bin];
        c1 = hist[top_bin - 1];
      }
      int total;
      const int above = block_exclusive_scan(static_cast<int>(c0 + c1), s_warp, &total);
      if (above < need && need <= above + static_cast<int>(c0)) {
        s_bin = top_bin;
        s_above = above;
        s_in = c0;
      } else if (above + static_cast<int>(c0) < need && need <= above + static_cast<int>(c0 + c1)) {
        s_bin = top_bin - 1;
        s_above = above + c0;
        s_in = c1;
      }
      __syncthreads();
      const uint32_t bin_lo = lo + (static_cast<uint32_t>(s_bin) << shift);
      need -= s_above;
      if (s_in == need) {  // the whole bin is kept
        threshold = bin_lo - 1;  // keys are at least -inf's, 0x007FFFFF: no wrap
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
  }

  // kept rows of each warp's run of keys, then of the warps and slices before it
  const int run0 = min(n, warp * run), run1 = min(n, run0 + run);
  int gt = 0, eq = 0;
  if (cut) {
    for (int i0 = run0; i0 < run1; i0 += 32) {
      const int i = i0 + lane;
      const uint32_t key = i < run1 ? key_at(i) : 0u;
      gt += __popc(__ballot_sync(0xffffffffu, i < run1 && key > threshold));
      eq += __popc(__ballot_sync(0xffffffffu, i < run1 && ties > 0 && key == threshold));
    }
  } else {
    gt = run1 - run0;
  }
  if (lane == 0) {
    s_gt[warp] = gt;
    s_eq[warp] = eq;
  }
  __syncthreads();
  if (warp == 0) {
    int g = s_gt[lane], e = s_eq[lane];
    const int g1 = g, e1 = e;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int gy = __shfl_up_sync(0xffffffffu, g, o), ey = __shfl_up_sync(0xffffffffu, e, o);
      if (lane >= o) {
        g += gy;
        e += ey;
      }
    }
    s_gt[lane] = g - g1;
    s_eq[lane] = e - e1;
    if (lane == 31) {
      s_tot[0] = g;
      s_tot[1] = e;
    }
  }
  meet();
  gt = s_gt[warp];
  eq = s_eq[warp];
  for (uint32_t r = 0; r < rank; ++r) {
    gt += dsmem_ld_u32(dsmem_map(smem_u32(s_tot), r));
    eq += dsmem_ld_u32(dsmem_map(smem_u32(s_tot + 1), r));
  }
  int64_t* rows = p.rows + static_cast<int64_t>(b) * p.keep;
  float* kept = p.weights_out + static_cast<int64_t>(b) * p.capacity;
  for (int i0 = run0; i0 < run1; i0 += 32) {
    const int i = i0 + lane;
    bool above = i < run1, equal = false;
    if (cut) {
      const uint32_t key = i < run1 ? key_at(i) : 0u;
      above = above && key > threshold;
      equal = i < run1 && ties > 0 && key == threshold;
    }
    const unsigned ga = __ballot_sync(0xffffffffu, above), ea = __ballot_sync(0xffffffffu, equal);
    const unsigned before = (1u << lane) - 1u;
    const int g = gt + __popc(ga & before), e = eq + __popc(ea & before);
    if (above || (equal && e < ties)) {
      const int place = g + min(e, ties);
      rows[place] = base + i;
      kept[place] = src[base + i];
    }
    gt += __popc(ga);
    eq += __popc(ea);
  }
  if (rank == 0) {
    for (int i = count + threadIdx.x; i < p.keep; i += EVICT_THREADS) rows[i] = -1;
    for (int i = count + threadIdx.x; i < p.capacity; i += EVICT_THREADS) kept[i] = 0.f;
    if (threadIdx.x == 0) p.counts[b] = count;
  }
  if (p.slices > 1) cluster_sync();  // a CTA's totals stay readable until every CTA has read them
}

struct GatherParams {
  const uint8_t* src;
  int64_t src_sb, src_sn;  // bytes
  uint8_t* dst;            // (B, capacity, row_bytes), contiguous
  const int64_t* rows;     // (B, keep)
  int keep, capacity, units;  // units of a row (row_bytes / sizeof(Unit))
  int chunks;                 // CTAs a cache row
};

// Copies row rows[b, i] to place i of the new table, and writes zeros where
// there is none (rows[b, i] = -1, and the places from keep to capacity: a
// product over a whole tile of the new table multiplies its unread rows by
// zero weights, which must not meet a NaN).
template <typename Unit>
__global__ void __launch_bounds__(EVICT_COPY_THREADS) evict_gather_kernel(const GatherParams p) {
  constexpr int ROWS = 4;  // places a thread has in flight
  const int b = blockIdx.x / p.chunks, chunk = blockIdx.x - b * p.chunks;
  const uint8_t* src = p.src + b * p.src_sb;
  Unit* dst = reinterpret_cast<Unit*>(p.dst) + static_cast<int64_t>(b) * p.capacity * p.units;
  const int64_t* rows = p.rows + static_cast<int64_t>(b) * p.keep;
  // a group of threads a place, a unit each (long rows: several)
  const int group = min(p.units, EVICT_COPY_THREADS), groups = EVICT_COPY_THREADS / group;
  const int mine = threadIdx.x / group, unit = threadIdx.x - mine * group;
  griddep_wait();
  if (mine >= groups) return;
  const int step = p.chunks * groups;
  for (int64_t i0 = chunk * groups + mine; i0 < p.capacity; i0 += static_cast<int64_t>(ROWS) * step) {
    const Unit* from[ROWS];
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      const int64_t i = i0 + static_cast<int64_t>(k) * step;
      const int64_t row = i < p.keep ? rows[i] : -1;
      from[k] = row >= 0 ? reinterpret_cast<const Unit*>(src + row * p.src_sn) : nullptr;
    }
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

}  // namespace wpt
