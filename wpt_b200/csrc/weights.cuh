// The attention weight that each cached row collects: for a pass of queries
// q (B, T, H, C) over keys k (B, N, C) with the forward pass's log-sum-exp,
//
//   weights[b, n] += sum over t, h of exp(scale q_bth . k_bn - lse_bth)
//
// over the queries that read row n (max(0, p - window + 1, floor) <= n <=
// min(p, N - 1), p the query's position). With lse known there is no running
// maximum: a key's weight is a plain sum over the (query, head) columns, so
// the keys are the product's M (S^T = K Q^T), thread r owns key r and no sum
// crosses threads. Every key's columns are summed in a fixed order, so
// repeated calls agree bit for bit.
//
// weights_stream_kernel (T * H up to 256 columns, one decode step): the
// queries stay in shared memory and the keys stream through it. The rows'
// live key tiles are laid end to end and cut into one equal range a CTA, so
// rows of any lengths keep the SMs equally busy. Bound: HBM (2 C bytes a key).
//
// 64 rows of 1,024 to 32,768 keys, 32 heads: 54 us for 308 MB (5.7 TB/s).
//
// weights_tile_kernel (more columns, a prompt): up to four tiles of 128 keys
// stay in shared memory and the queries stream past them, 128 columns at a
// time. A warpgroup a key tile adds up the exponentials of its scores from its
// quarter of TMEM while the others' products run. Items of (key tiles, a run
// of column tiles) are handed out by an atomic ticket; where a key's columns
// are cut into several runs, their sums go to scratch and weights_reduce_kernel
// adds them in order. weights_prep_kernel lays out each column's constant and
// rows, and each column tile's extremes, by which tiles that no query reads are
// skipped and tiles read whole need no mask. Bound: the exponentials (16 a clock
// an SM: 1,024 clocks for 128 keys x 128 columns, whose products take 512), so
// an eighth of them take the FMA pipe. 8 x 4,096 places of 16 heads, causal, width
// 128: 364 us, 755 TFLOP/s (0.47 of the measured bf16 peak, at 1.53 GHz under the
// power limit). A run of 32 columns keeps a scheduler's exponential unit busy for
// 896 clocks (28 exponentials a thread, four warps). Over the whole kernel the unit
// is busy 71% of the time and the issue slots 46%; loads from TMEM and waits make up
// the rest.
#pragma once

#include <climits>

#include "common.cuh"

namespace wpt {

// The rows [lo, hi] that the query at `pos` reads; hi < lo for none.
__device__ __forceinline__ int2 weights_range(int64_t pos, const int64_t* floor, int64_t at, int window, int N) {
  int64_t hi = pos < N - 1 ? pos : N - 1;
  int64_t lo = window > 0 ? pos - window + 1 : 0;
  if (floor != nullptr && floor[at] > lo) lo = floor[at];
  if (lo < 0) lo = 0;
  if (hi < lo) return make_int2(INT_MAX, -1);
  return make_int2(static_cast<int>(lo), static_cast<int>(hi));
}

// The exponent's constant of a column: exp(x - lse) = 2^(x log2e + this). A
// query without rows has lse -inf; it adds nothing.
__device__ __forceinline__ float weights_offset(float lse) { return lse == -INFINITY ? -INFINITY : -lse * LOG2E; }

__device__ __forceinline__ float weights_clamp(float x, float lo, float hi) {  // a NaN stays one
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(x) : "f"(lo));
  asm("min.NaN.f32 %0, %0, %1;" : "+f"(x) : "f"(hi));
  return x;
}

// 2^x for a pair of floats on the FMA pipe, for the terms whose turn it is not
// on the exponential unit. 2^x = 2^r 2^f with r = round(x) and f = x - r in
// [-1/2, 1/2]: 2^f is a polynomial of degree 5 fitted for this library by
// iterated weighted least squares (relative error 1.5e-7, a rounding of the sum it
// goes into). Adding 1.5 * 2^23 + 127 rounds x and leaves r + 127 in the low bits,
// which shifted are 2^r: 0 at r = -127 and +inf at 128, where x is clamped. A
// product with it, and not an addition to the exponent, keeps a NaN.
__device__ __forceinline__ uint64_t weights_exp2_poly(uint64_t x) {
  constexpr float MAGIC = 12582912.0f + 127.0f;
  float x0, x1;
  f2_unpack(x, x0, x1);
  x = f2_pack(weights_clamp(x0, -127.f, 128.f), weights_clamp(x1, -127.f, 128.f));
  const uint64_t t = f2_add(x, f2_pack(MAGIC, MAGIC));
  const uint64_t r = f2_add(t, f2_pack(-MAGIC, -MAGIC));
  const uint64_t f = f2_fma(r, f2_pack(-1.f, -1.f), x);
  uint64_t q = f2_fma(f2_pack(0.0013264717999845743f, 0.0013264717999845743f), f, f2_pack(0.009671512991189957f, 0.009671512991189957f));
  q = f2_fma(q, f, f2_pack(0.05550733953714371f, 0.05550733953714371f));
  q = f2_fma(q, f, f2_pack(0.24022242426872253f, 0.24022242426872253f));
  q = f2_fma(q, f, f2_pack(0.6931470036506653f, 0.6931470036506653f));
  q = f2_fma(q, f, f2_pack(1.f, 1.f));
  float t0, t1;
  f2_unpack(t, t0, t1);
  return f2_mul(q, f2_pack(__int_as_float(__float_as_int(t0) << 23), __int_as_float(__float_as_int(t1) << 23)));
}

// Adds exp2(x scale + cols[0][c]) over 2 * PAIRS columns c to the four partial
// sums, POLY of every 8 pairs on the FMA pipe; MASK: of those with cols[1][c] <= n <=
// cols[2][c] (whole numbers). cols: rows of STRIDE columns in shared memory,
// 16-byte aligned.
template <int PAIRS, int POLY, bool MASK, int STRIDE>
__device__ __forceinline__ void weights_terms(uint64_t (&sum)[2], const uint32_t* x, float scale, const float* cols,
                                              int n) {
  const uint64_t scale2 = f2_pack(scale, scale);
#pragma unroll
  for (int i = 0; i < PAIRS; i += 2) {
    const float4 o = *reinterpret_cast<const float4*>(cols + 2 * i);
    uint64_t a[2];
    a[0] = f2_fma(f2_pack(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])), scale2, f2_pack(o.x, o.y));
    a[1] = f2_fma(f2_pack(__uint_as_float(x[2 * i + 2]), __uint_as_float(x[2 * i + 3])), scale2, f2_pack(o.z, o.w));
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if constexpr (!MASK) {
        if (((i + h) * POLY) % 8 < POLY) {
          sum[h] = f2_add(sum[h], weights_exp2_poly(a[h]));
          continue;
        }
      }
      float a0, a1;
      f2_unpack(a[h], a0, a1);
      a0 = fast_exp2(a0);
      a1 = fast_exp2(a1);
      if constexpr (MASK) {
        const int2 lo = *reinterpret_cast<const int2*>(cols + STRIDE + 2 * (i + h));
        const int2 hi = *reinterpret_cast<const int2*>(cols + 2 * STRIDE + 2 * (i + h));
        a0 = n >= lo.x && n <= hi.x ? a0 : 0.f;
        a1 = n >= lo.y && n <= hi.y ? a1 : 0.f;
      }
      sum[h] = f2_add(sum[h], f2_pack(a0, a1));
    }
  }
}

// D = A B^T over KK + 1 steps of 16 columns, A 128 rows and B `cols` rows in
// 64-column chunks of 128-byte-swizzled rows; issued by one lane of the warp.
template <int KK, int COLS>
__device__ __forceinline__ void weights_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc) {
  if constexpr (KK > 0) weights_mma<KK - 1, COLS>(d, a, b, idesc);
  constexpr uint32_t OFF_A = ((KK / 4) * 128 * 128 + (KK % 4) * 32) / 16, OFF_B = ((KK / 4) * COLS * 128 + (KK % 4) * 32) / 16;
  mma_ss_off_warp<OFF_A, OFF_B>(d, a, b, idesc, KK > 0 ? 1u : 0u);
}

// ------------------------------------------------------------- key stream

constexpr int WEIGHTS_BAL_ROWS = 1024;  // most batch rows whose tiles are laid end to end
constexpr int WEIGHTS_STREAM_THREADS = 192;  // warps 0-3 epilogue, 4 MMA, 5 loader

struct WeightsParams {
  const int64_t* positions;  // (B, T)
  const int64_t* floor;      // (B, T) or NULL
  const float* lse;          // (B, T, H)
  float* weights;            // (B, N), row stride weights_ld
  int64_t weights_ld;
  unsigned* status;
  int B, T, H, N, window;
  float scale_log2;  // scale * log2(e)
};

template <int C, int NCOL, int STAGES>
struct WeightsStreamLayout {
  static constexpr int Q_BYTES = NCOL * C * 2, K_BYTES = 128 * C * 2;
  static constexpr int OFF_Q = 0;  // two buffers
  static constexpr int OFF_K = 2 * Q_BYTES;
  static constexpr int OFF_COL = OFF_K + STAGES * K_BYTES;  // each column's constant (float), then its lowest and highest row
  static constexpr int OFF_PRE = OFF_COL + NCOL * 12;
  static constexpr int OFF_FIRST = OFF_PRE + (WEIGHTS_BAL_ROWS + 2) * 4;
  static constexpr int OFF_BAR = OFF_FIRST + WEIGHTS_BAL_ROWS * 4;
  // TMEM buffers: enough tiles for the epilogue's change of rows
  static constexpr int BUFS = NCOL <= 64 ? 8 : 512 / NCOL;
  // q_full[2], q_empty[2], drained, s_full[BUFS], s_free[BUFS], k_full[STAGES], k_empty[STAGES]
  static constexpr int NBAR = 5 + 2 * BUFS + 2 * STAGES;
  static constexpr int OFF_MISC = OFF_BAR + NBAR * 8;
  static constexpr int BYTES = OFF_MISC + 64 + 1024;
  static constexpr int TMEM_COLS = BUFS * NCOL;
};

// The lowest and highest row that batch row b's queries from `first` on, `step`
// apart, read; (INT_MAX, -1) for none.
__device__ __forceinline__ int2 weights_row_range(const WeightsParams& p, int b, int first, int step) {
  int lo = INT_MAX, hi = -1;
  for (int t = first; t < p.T; t += step) {
    const int64_t at = static_cast<int64_t>(b) * p.T + t;
    const int2 r = weights_range(p.positions[at], p.floor, at, p.window, p.N);
    lo = min(lo, r.x);
    hi = max(hi, r.y);
  }
  return make_int2(lo, hi);
}

// A role's walk over its CTA's work: segments of (batch row, key tiles).
struct WeightsWalk {
  int b, tile0, ntiles;
  const int *pre, *first;  // balanced: live tiles of the rows before each row, and each row's first
  int64_t lo, hi;          // balanced: the CTA's range of the tiles laid end to end
  bool balanced;
  int next;

  __device__ __forceinline__ void start(const WeightsParams& p, const int* s_pre, const int* s_first) {
    pre = s_pre;
    first = s_first;
    balanced = p.B <= WEIGHTS_BAL_ROWS;
    if (balanced) {
      const int64_t total = pre[p.B];
      lo = total * blockIdx.x / gridDim.x;
      hi = total * (blockIdx.x + 1) / gridDim.x;
      // the first row that ends after lo
      int a = 0, z = p.B;
      while (a < z) {
        const int m = (a + z) >> 1;
        if (pre[m + 1] > lo)
          z = m;
        else
          a = m + 1;
      }
      next = a;
    } else {
      next = blockIdx.x;
    }
  }
  __device__ __forceinline__ bool step(const WeightsParams& p) {
    if (balanced) {
      while (next < p.B && pre[next + 1] == pre[next]) ++next;
      if (next >= p.B || pre[next] >= hi || lo >= hi) return false;
      b = next++;
      const int64_t a = max(lo, static_cast<int64_t>(pre[b])), z = min(hi, static_cast<int64_t>(pre[b + 1]));
      tile0 = first[b] + static_cast<int>(a - pre[b]);
      ntiles = static_cast<int>(z - a);
      return true;
    }
    for (; next < p.B; next += gridDim.x) {
      const int2 rows = weights_row_range(p, next, 0, 1);
      if (rows.y >= rows.x) {
        b = next;
        tile0 = rows.x / 128;
        ntiles = rows.y / 128 - tile0 + 1;
        next += gridDim.x;
        return true;
      }
    }
    return false;
  }
};

template <int C, int NCOL, int STAGES>
__global__ void __launch_bounds__(WEIGHTS_STREAM_THREADS, 1)
    weights_stream_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                          const WeightsParams p) {
  using L = WeightsStreamLayout<C, NCOL, STAGES>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* s_off = reinterpret_cast<float*>(smem + L::OFF_COL);
  int* s_lo = reinterpret_cast<int*>(smem + L::OFF_COL + NCOL * 4);
  int* s_hi = reinterpret_cast<int*>(smem + L::OFF_COL + NCOL * 8);
  int* s_pre = reinterpret_cast<int*>(smem + L::OFF_PRE);
  int* s_first = reinterpret_cast<int*>(smem + L::OFF_FIRST);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  uint64_t* q_full = bars;
  uint64_t* q_empty = bars + 2;
  uint64_t* drained = bars + 4;
  uint64_t* s_full = bars + 5;
  uint64_t* s_free = s_full + L::BUFS;
  uint64_t* k_full = s_free + L::BUFS;
  uint64_t* k_empty = k_full + STAGES;
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(smem + L::OFF_MISC);
  int* s_scan = reinterpret_cast<int*>(smem + L::OFF_MISC + 16);  // 6 warp totals
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    mbar_init(drained, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(q_full + i, 1);
      mbar_init(q_empty + i, 1);
    }
    for (int i = 0; i < L::BUFS; ++i) {
      mbar_init(s_full + i, 1);
      mbar_init(s_free + i, 4);
    }
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(k_full + s, 1);
      mbar_init(k_empty + s, 1);
    }
    fence_mbar_init();
  }
  if (warp == 4) {
    tmem_alloc(s_tmem, L::TMEM_COLS);
    tmem_relinquish();
  }
  if (warp == 5 && lane == 0) {
    tma_prefetch(&tm_q);
    tma_prefetch(&tm_k);
  }
  griddep_wait();
  if (p.B <= WEIGHTS_BAL_ROWS) {
    // each row's first live tile and their number: a thread a row, or with
    // many queries a row, a warp
    auto put = [&](int b, int2 rows) {
      s_first[b] = rows.y < rows.x ? 0 : rows.x / 128;
      s_pre[b + 1] = rows.y < rows.x ? 0 : rows.y / 128 - rows.x / 128 + 1;
    };
    if (p.T <= 8) {
      for (int b = threadIdx.x; b < p.B; b += WEIGHTS_STREAM_THREADS) put(b, weights_row_range(p, b, 0, 1));
    } else {
      for (int b = warp; b < p.B; b += WEIGHTS_STREAM_THREADS / 32) {
        int2 rows = weights_row_range(p, b, lane, 32);
        rows.x = __reduce_min_sync(0xffffffffu, rows.x);
        rows.y = __reduce_max_sync(0xffffffffu, rows.y);
        if (lane == 0) put(b, rows);
      }
    }
    __syncthreads();
    // live tiles of the rows before each row
    const int per = (p.B + WEIGHTS_STREAM_THREADS - 1) / WEIGHTS_STREAM_THREADS;
    const int b0 = min(p.B, static_cast<int>(threadIdx.x) * per), b1 = min(p.B, b0 + per);
    int sum = 0;
    for (int b = b0; b < b1; ++b) sum += s_pre[b + 1];
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    if (lane == 31) s_scan[warp] = incl;
    __syncthreads();
    int at = incl - sum;
    for (int w = 0; w < warp; ++w) at += s_scan[w];
    for (int b = b0; b < b1; ++b) {
      at += s_pre[b + 1];
      s_pre[b + 1] = at;
    }
    if (threadIdx.x == 0) s_pre[0] = 0;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  WeightsWalk walk;
  walk.start(p, s_pre, s_first);

  if (warp == 5) {
    if (lane == 0) {
      bool ok = true;
      int j = 0;
      for (int seg = 0; ok && walk.step(p); ++seg) {
        uint8_t* sQ = smem + L::OFF_Q + (seg & 1) * L::Q_BYTES;
        if (seg >= 2 && !(ok = mbar_wait(q_empty + (seg & 1), ((seg >> 1) & 1) ^ 1, p.status))) break;
        mbar_expect_tx(q_full + (seg & 1), L::Q_BYTES);
#pragma unroll
        for (int c = 0; c < C / 64; ++c)
          tma_load_3d(sQ + c * NCOL * 128, &tm_q, q_full + (seg & 1), c * 64, 0, walk.b);
        for (int jj = 0; jj < walk.ntiles; ++jj, ++j) {
          const int st = j % STAGES;
          if (j >= STAGES && !(ok = mbar_wait(k_empty + st, ((j / STAGES) & 1) ^ 1, p.status))) break;
          uint8_t* sK = smem + L::OFF_K + st * L::K_BYTES;
          mbar_expect_tx(k_full + st, L::K_BYTES);
#pragma unroll
          for (int c = 0; c < C / 64; ++c)
            tma_load_3d(sK + c * 128 * 128, &tm_k, k_full + st, c * 64, (walk.tile0 + jj) * 128, walk.b);
        }
      }
      // after a wait that ran out: the copies in flight land before the block leaves
      for (int st = 0; !ok && st < STAGES && st < j; ++st)
        mbar_wait(k_full + st, ((j - 1 - st) / STAGES) & 1, p.status);
    }
    __syncwarp();
  } else if (warp == 4) {
    constexpr uint32_t IDESC = idesc_bf16(128, NCOL, 0, 0);
    auto wait = [&](uint64_t* bar, int parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, p.status)); };
    bool ok = true;
    int j = 0;
    for (int seg = 0; ok && walk.step(p); ++seg) {
      const uint64_t q_desc = sdesc_sw128(smem_u32(smem + L::OFF_Q + (seg & 1) * L::Q_BYTES), 16, 1024);
      if (!(ok = wait(q_full + (seg & 1), (seg >> 1) & 1))) break;
      for (int jj = 0; jj < walk.ntiles; ++jj, ++j) {
        const int st = j % STAGES, buf = j % L::BUFS;
        if (!(ok = wait(k_full + st, (j / STAGES) & 1))) break;
        if (j >= L::BUFS && !(ok = wait(s_free + buf, ((j / L::BUFS) & 1) ^ 1))) break;
        tc_fence_after();
        weights_mma<C / 16 - 1, NCOL>(tmem + buf * NCOL, sdesc_sw128(smem_u32(smem + L::OFF_K + st * L::K_BYTES), 16, 1024),
                                      q_desc, IDESC);
        mma_commit_warp(k_empty + st);
        mma_commit_warp(s_full + buf);
      }
      if (ok) mma_commit_warp(q_empty + (seg & 1));
    }
    mma_commit_warp(drained);  // TMEM is freed with no product in flight
    wait(drained, 0);
  } else {
    const int r = threadIdx.x;
    const uint32_t lane_addr = tmem + (static_cast<uint32_t>(warp * 32) << 16);
    const int cols = p.T * p.H;
    const bool padded = cols < NCOL;
    bool ok = true;
    int j = 0;
    while (walk.step(p)) {
      const int b = walk.b;
      // the previous segment's columns were read; a wait that ran out stops all four warps
      if (!named_barrier_and(1, 128, ok)) break;
      for (int c = r; c < NCOL; c += 128) {
        const int t = c / p.H;
        float off = -INFINITY;  // a padding column reads nothing
        int2 range = make_int2(INT_MAX, -1);
        if (t < p.T) {
          const int64_t at = static_cast<int64_t>(b) * p.T + t;
          range = weights_range(p.positions[at], p.floor, at, p.window, p.N);
          off = weights_offset(p.lse[at * p.H + (c - t * p.H)]);
        }
        s_off[c] = off;
        s_lo[c] = range.x;
        s_hi[c] = range.y;
      }
      named_barrier(1, 128);
      // rows that every column reads, and that any does
      int all_lo = 0, all_hi = INT_MAX, any_lo = INT_MAX, any_hi = -1;
      for (int c = 0; c < cols; c += p.H) {
        all_lo = max(all_lo, s_lo[c]);
        all_hi = min(all_hi, s_hi[c]);
        any_lo = min(any_lo, s_lo[c]);
        any_hi = max(any_hi, s_hi[c]);
      }
      for (int jj = 0; jj < walk.ntiles; ++jj, ++j) {
        const int n0 = (walk.tile0 + jj) * 128, n = n0 + r, buf = j % L::BUFS;
        const bool mine = n >= any_lo && n <= any_hi;
        if (!(ok = __all_sync(0xffffffffu, mbar_wait(s_full + buf, (j / L::BUFS) & 1, p.status)))) break;
        tc_fence_after();
        const bool whole = n0 >= all_lo && n0 + 127 <= all_hi;
        uint64_t sums[2] = {0, 0};
        constexpr int W = NCOL < 32 ? NCOL : 32;
        uint32_t x[W];
        auto load = [&](int c0) {
          if constexpr (W == 32)
            tmem_ld32(lane_addr + buf * NCOL + c0, x);
          else
            tmem_ld16(lane_addr + buf * NCOL + c0, x);
        };
        auto release = [&] {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(s_free + buf);
        };
#pragma unroll 2
        for (int c0 = 0; c0 < NCOL; c0 += W) {
          load(c0);
          if (c0 + W == NCOL && !padded) release();  // the scores are in registers
          if (whole)
            weights_terms<W / 2, 0, false, NCOL>(sums, x, p.scale_log2, s_off + c0, n);
          else
            weights_terms<W / 2, 0, true, NCOL>(sums, x, p.scale_log2, s_off + c0, n);
        }
        float s0, s1;
        f2_unpack(f2_add(sums[0], sums[1]), s0, s1);
        if (padded) {
          // A padding column's score is 0 times the key, which is NaN where the key is not
          // finite: then once more with the mask. (The mask for every tile: 44.7 us for 64
          // rows of 8,192 keys and 100 heads, this 42.2.)
          if (whole && __any_sync(0xffffffffu, isnan(s0 + s1))) {
            sums[0] = sums[1] = 0;
#pragma unroll 1
            for (int c0 = 0; c0 < NCOL; c0 += W) {
              load(c0);
              weights_terms<W / 2, 0, true, NCOL>(sums, x, p.scale_log2, s_off + c0, n);
            }
            f2_unpack(f2_add(sums[0], sums[1]), s0, s1);
          }
          release();
        }
        // A reduction in L2 instead of a load, which each tile would wait for: 64
        // rows of 1,024 to 32,768 keys take 54 us with it, 58 without. A key has one
        // such addition a call, so their order cannot matter.
        if (mine) atomicAdd(p.weights + static_cast<int64_t>(b) * p.weights_ld + n, s0 + s1);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 4) {
    tc_fence_after();
    tmem_dealloc(tmem, L::TMEM_COLS);
  }
}

// ------------------------------------------------------------ query stream

constexpr int WEIGHTS_TILE_THREADS = 576;  // warps 0-15 epilogue, 16 MMA, 17 loader
constexpr int WEIGHTS_TILE_GROUPS = 4;     // key tiles of 128 an item, one for each epilogue warpgroup
constexpr int WEIGHTS_TILE_COLS = 128;
constexpr int WEIGHTS_Q_STAGES = 2, WEIGHTS_C_STAGES = 4;
// Pairs in every 8 whose exponentials take the FMA pipe. 8 x 4,096 places of 16
// heads, causal: 0 take 389 us, 1 364, 2 368, 3 387.
constexpr int WEIGHTS_POLY8 = 1;

struct WeightsTileParams {
  float* weights;      // (B, N), row stride weights_ld
  int64_t weights_ld;
  const int4* meta;    // (B, tiles): lowest and highest row any column reads, then that all of them read
  const float* cols;   // (B, tiles, 3, 128): each column's exponent constant, then its lowest and highest row (int)
  float* partial;      // (chunks, B, N) when chunks > 1
  unsigned* ticket;
  unsigned* status;
  int B, N, tiles, key_blocks, chunks, chunk_tiles, items;
  int groups;  // key tiles an item has, up to WEIGHTS_TILE_GROUPS
  float scale_log2;
};

// One CTA a column tile: its columns' constants and rows, and the tile's.
__global__ void __launch_bounds__(WEIGHTS_TILE_COLS)
    weights_prep_kernel(const WeightsParams p, int tiles, int4* meta, float* cols, unsigned* ticket) {
  __shared__ int s_red[4][4];
  const int b = blockIdx.x / tiles, tile = blockIdx.x - b * tiles;
  // A small grid lets the next kernel set itself up meanwhile; a large one
  // would share its SMs with it.
  if (gridDim.x <= 256) griddep_launch();
  griddep_wait();
  if (blockIdx.x == 0 && threadIdx.x == 0) *ticket = 0;
  const int64_t c = static_cast<int64_t>(tile) * WEIGHTS_TILE_COLS + threadIdx.x;
  const int t = static_cast<int>(c / p.H);
  float off = -INFINITY;
  int2 r = make_int2(INT_MAX, -1);
  // A column past the last reads nothing. Its score is 0 times the key, which is NaN
  // where the key is not finite, so its tile always takes the mask.
  int4 m = make_int4(INT_MAX, -1, INT_MAX, -1);
  if (t < p.T) {
    const int64_t at = static_cast<int64_t>(b) * p.T + t;
    r = weights_range(p.positions[at], p.floor, at, p.window, p.N);
    off = weights_offset(p.lse[at * p.H + (c - static_cast<int64_t>(t) * p.H)]);
    m = make_int4(r.x, r.y, r.x, r.y);
  }
  float* to = cols + (static_cast<int64_t>(b) * tiles + tile) * (3 * WEIGHTS_TILE_COLS) + threadIdx.x;
  to[0] = off;
  to[WEIGHTS_TILE_COLS] = __int_as_float(r.x);
  to[2 * WEIGHTS_TILE_COLS] = __int_as_float(r.y);
  m.x = __reduce_min_sync(0xffffffffu, m.x);
  m.y = __reduce_max_sync(0xffffffffu, m.y);
  m.z = __reduce_max_sync(0xffffffffu, m.z);
  m.w = __reduce_min_sync(0xffffffffu, m.w);
  const int warp = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0) {
    s_red[0][warp] = m.x;
    s_red[1][warp] = m.y;
    s_red[2][warp] = m.z;
    s_red[3][warp] = m.w;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 4; ++w) {
      m.x = min(m.x, s_red[0][w]);
      m.y = max(m.y, s_red[1][w]);
      m.z = max(m.z, s_red[2][w]);
      m.w = min(m.w, s_red[3][w]);
    }
    meta[static_cast<int64_t>(b) * tiles + tile] = m;
  }
}

template <int C>
struct WeightsTileLayout {
  static constexpr int K_BYTES = 128 * C * 2;  // a key tile
  static constexpr int Q_BYTES = WEIGHTS_TILE_COLS * C * 2, COL_BYTES = WEIGHTS_TILE_COLS * 12;
  static constexpr int OFF_K = 0;
  static constexpr int OFF_Q = WEIGHTS_TILE_GROUPS * K_BYTES;
  static constexpr int OFF_COL = OFF_Q + WEIGHTS_Q_STAGES * Q_BYTES;
  static constexpr int OFF_BAR = OFF_COL + WEIGHTS_C_STAGES * COL_BYTES;
  // k_full, k_empty, drained, item_full[2], item_empty[2], s_full[4], s_free[4], then q and c full, empty
  static constexpr int NBAR = 15 + 2 * WEIGHTS_Q_STAGES + 2 * WEIGHTS_C_STAGES;
  static constexpr int OFF_MISC = OFF_BAR + NBAR * 8;
  static constexpr int BYTES = OFF_MISC + 32 + 1024;
};

// A walk over the column tiles of an item that read any of its keys, found 32
// at a time by the warp: step() gives the next one, or -1.
struct WeightsTiles {
  const int4* meta;
  int at, end, lo, hi;
  unsigned mask;
  int4 mine;  // of the tile at + lane
  __device__ __forceinline__ void start(const int4* m, int first, int last, int n0, int n1) {
    meta = m;
    at = first - 32;
    end = last;
    lo = n0;
    hi = n1;
    mask = 0;
  }
  __device__ __forceinline__ int step() {
    while (mask == 0) {
      at += 32;
      if (at >= end) return -1;
      const int i = at + (threadIdx.x & 31);
      mine = i < end ? meta[i] : make_int4(INT_MAX, -1, INT_MAX, -1);
      mask = __ballot_sync(0xffffffffu, mine.x <= hi && mine.y >= lo);
    }
    const int i = __ffs(mask) - 1;
    mask &= mask - 1;
    return at + i;
  }
  // Of the tiles at .. at + 31: which have a column that reads one of rows n .. n + 127, and whose columns all read them all.
  __device__ __forceinline__ unsigned any(int n) const {
    return __ballot_sync(0xffffffffu, mine.x <= n + 127 && mine.y >= n);
  }
  __device__ __forceinline__ unsigned all(int n) const {
    return __ballot_sync(0xffffffffu, mine.z <= n && mine.w >= n + 127);
  }
};

template <int C>
__global__ void __launch_bounds__(WEIGHTS_TILE_THREADS, 1)
    weights_tile_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                        const WeightsTileParams p) {
  using L = WeightsTileLayout<C>;
  constexpr int COLS = WEIGHTS_TILE_COLS, GROUPS = WEIGHTS_TILE_GROUPS;
  constexpr int QS = WEIGHTS_Q_STAGES, CS = WEIGHTS_C_STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  uint64_t* k_full = bars;
  uint64_t* k_empty = bars + 1;
  uint64_t* drained = bars + 2;
  uint64_t* item_full = bars + 3;
  uint64_t* item_empty = bars + 5;
  uint64_t* s_full = bars + 7;   // a key tile's scores are in TMEM
  uint64_t* s_free = bars + 11;  // and have been read
  uint64_t* q_full = bars + 15;
  uint64_t* q_empty = q_full + QS;
  uint64_t* c_full = q_empty + QS;
  uint64_t* c_empty = c_full + CS;
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(smem + L::OFF_MISC);
  volatile int* s_item = reinterpret_cast<volatile int*>(smem + L::OFF_MISC + 8);  // two slots
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    mbar_init(k_full, 1);
    mbar_init(k_empty, 1);
    mbar_init(drained, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(item_full + i, 1);
      mbar_init(item_empty + i, 17);  // the MMA warp and the 16 epilogue warps
    }
    for (int i = 0; i < GROUPS; ++i) {
      mbar_init(s_full + i, 1);
      mbar_init(s_free + i, 4);
    }
    for (int s = 0; s < QS; ++s) {
      mbar_init(q_full + s, 1);
      mbar_init(q_empty + s, 1);
    }
    for (int s = 0; s < CS; ++s) {
      mbar_init(c_full + s, 1);
      mbar_init(c_empty + s, 16);
    }
    fence_mbar_init();
  }
  if (warp == 16) {
    tmem_alloc(s_tmem, 512);
    tmem_relinquish();
  }
  if (warp == 17 && lane == 0) {
    tma_prefetch(&tm_q);
    tma_prefetch(&tm_k);
  }
  griddep_wait();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;

  // an item: keys [n0, n0 + 128 groups) of row b against a run of column tiles
  struct Item {
    int b, n0, chunk;
    WeightsTiles tiles;
  };
  auto open = [&](int item, Item& it) {
    const int per = p.B * p.key_blocks;
    it.chunk = p.chunks - 1 - item / per;  // a causal pass's last columns read the most keys: first
    const int rest = item % per;
    it.b = rest % p.B;
    it.n0 = rest / p.B * (128 * p.groups);
    const int c0 = it.chunk * p.chunk_tiles;
    it.tiles.start(p.meta + static_cast<int64_t>(it.b) * p.tiles, c0, min(p.tiles, c0 + p.chunk_tiles), it.n0,
                   it.n0 + 128 * p.groups - 1);
  };
  auto wait = [&](uint64_t* bar, int parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, p.status)); };

  if (warp == 17) {
    // ------------------------------------------------------------ loader
    bool ok = true;
    int u = 0, k_uses = 0;
    for (int i = 0; ok; ++i) {
      int item = 0;
      if (lane == 0) item = static_cast<int>(atomicAdd(p.ticket, 1u));
      item = __shfl_sync(0xffffffffu, item, 0);
      if (item >= p.items) item = -1;
      if (i >= 2 && !(ok = wait(item_empty + (i & 1), ((i >> 1) & 1) ^ 1))) break;
      if (lane == 0) {
        s_item[i & 1] = item;
        mbar_arrive(item_full + (i & 1));
      }
      if (item < 0) break;
      Item it;
      open(item, it);
      bool first = true;
      for (int ct = it.tiles.step(); ok && ct >= 0; ct = it.tiles.step(), ++u) {
        if (first) {
          first = false;
          if (k_uses > 0 && !(ok = wait(k_empty, (k_uses - 1) & 1))) break;
          ++k_uses;
          if (lane == 0) {
            mbar_expect_tx(k_full, p.groups * L::K_BYTES);
            for (int g = 0; g < p.groups; ++g)
#pragma unroll
              for (int c = 0; c < C / 64; ++c)
                tma_load_3d(smem + L::OFF_K + g * L::K_BYTES + c * 128 * 128, &tm_k, k_full, c * 64, it.n0 + g * 128,
                            it.b);
          }
        }
        const int qs = u % QS, cs = u % CS;
        if (u >= QS && !(ok = wait(q_empty + qs, ((u / QS) & 1) ^ 1))) break;
        if (lane == 0) {
          mbar_expect_tx(q_full + qs, L::Q_BYTES);
#pragma unroll
          for (int c = 0; c < C / 64; ++c)
            tma_load_3d(smem + L::OFF_Q + qs * L::Q_BYTES + c * COLS * 128, &tm_q, q_full + qs, c * 64, ct * COLS, it.b);
        }
        if (u >= CS && !(ok = wait(c_empty + cs, ((u / CS) & 1) ^ 1))) {
          ++u;  // its queries are on their way
          break;
        }
        if (lane == 0) {
          mbar_expect_tx(c_full + cs, L::COL_BYTES);
          bulk_load(smem + L::OFF_COL + cs * L::COL_BYTES,
                    p.cols + (static_cast<int64_t>(it.b) * p.tiles + ct) * (3 * COLS), L::COL_BYTES, c_full + cs);
        }
        __syncwarp();
      }
    }
    // after a wait that ran out: the copies in flight land before the block leaves
    if (!ok) {
      if (k_uses > 0) mbar_wait(k_full, (k_uses - 1) & 1, p.status);
      for (int st = 0; st < QS && st < u; ++st) mbar_wait(q_full + st, ((u - 1 - st) / QS) & 1, p.status);
      for (int st = 0; st < CS && st < u; ++st) mbar_wait(c_full + st, ((u - 1 - st) / CS) & 1, p.status);
    }
  } else if (warp == 16) {
    // ------------------------------------------------------- MMA issuer
    constexpr uint32_t IDESC = idesc_bf16(128, COLS, 0, 0);
    const uint32_t k_addr = smem_u32(smem + L::OFF_K);
    bool ok = true;
    int u = 0, k_uses = 0;
    unsigned uses = 0;  // parity of each key tile's uses (bits 0-3), and whether it had one (bits 4-7)
    for (int i = 0; ok; ++i) {
      if (!(ok = wait(item_full + (i & 1), (i >> 1) & 1))) break;
      const int item = s_item[i & 1];
      __syncwarp();
      if (lane == 0) mbar_arrive(item_empty + (i & 1));
      if (item < 0) break;
      Item it;
      open(item, it);
      bool first = true;
      unsigned any[GROUPS];
      int from = -1;
      for (int ct = it.tiles.step(); ok && ct >= 0; ct = it.tiles.step(), ++u) {
        if (it.tiles.at != from) {
          from = it.tiles.at;
#pragma unroll
          for (int g = 0; g < GROUPS; ++g) any[g] = g < p.groups ? it.tiles.any(it.n0 + g * 128) : 0u;
        }
        if (first) {
          first = false;
          if (!(ok = wait(k_full, k_uses & 1))) break;
          ++k_uses;
        }
        const int qs = u % QS;
        if (!(ok = wait(q_full + qs, (u / QS) & 1))) break;
        const uint64_t q_desc = sdesc_sw128(smem_u32(smem + L::OFF_Q + qs * L::Q_BYTES), 16, 1024);
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
          if (!ok || !((any[g] >> (ct - from)) & 1u)) continue;
          if ((uses >> (4 + g)) & 1u) ok = wait(s_free + g, ((uses >> g) & 1u) ^ 1u);
          if (!ok) continue;
          uses = (uses ^ (1u << g)) | (16u << g);
          tc_fence_after();
          weights_mma<C / 16 - 1, COLS>(tmem + g * COLS, sdesc_sw128(k_addr + g * L::K_BYTES, 16, 1024), q_desc, IDESC);
          mma_commit_warp(s_full + g);
        }
        if (ok) mma_commit_warp(q_empty + qs);
      }
      if (ok && !first) mma_commit_warp(k_empty);
    }
    mma_commit_warp(drained);  // TMEM is freed with no product in flight
    wait(drained, 0);
  } else {
    // ----------------------------------------------------------- epilogue
    // A warpgroup takes one of the item's key tiles, a thread one key, in runs
    // of 32 columns. It waits for each run's scores from TMEM and then adds them up;
    // while a warpgroup waits, the others compute (the next run's load under way
    // meanwhile took as long or longer).
    const int g = warp >> 2;
    const uint32_t from = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + g * COLS;
    bool ok = true;
    int u = 0, used = 0;
    for (int i = 0; ok; ++i) {
      if (!(ok = wait(item_full + (i & 1), (i >> 1) & 1))) break;
      const int item = s_item[i & 1];
      __syncwarp();
      if (lane == 0) mbar_arrive(item_empty + (i & 1));
      if (item < 0) break;
      Item it;
      open(item, it);
      const int n0 = it.n0 + g * 128, n = n0 + (threadIdx.x & 127);
      uint64_t sum[2] = {0, 0};
      unsigned any = 0, all = 0;
      int first = -1;
      for (int ct = it.tiles.step(); ok && ct >= 0; ct = it.tiles.step(), ++u) {
        if (it.tiles.at != first) {
          first = it.tiles.at;
          any = g < p.groups ? it.tiles.any(n0) : 0u;
          all = it.tiles.all(n0);
        }
        const int cs = u % CS;
        if (!(ok = wait(c_full + cs, (u / CS) & 1))) break;
        if ((any >> (ct - first)) & 1u) {
          const float* off = reinterpret_cast<const float*>(smem + L::OFF_COL + cs * L::COL_BYTES);
          if (!(ok = wait(s_full + g, used & 1))) break;
          ++used;
          tc_fence_after();
          const bool whole = (all >> (ct - first)) & 1u;
#pragma unroll
          for (int run = 0; run < COLS / 32; ++run) {
            uint32_t x[32];
            tmem_ld32(from + run * 32, x);
            if (run == COLS / 32 - 1) {  // the scores are in registers
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(s_free + g);
            }
            if (whole)
              weights_terms<16, WEIGHTS_POLY8, false, COLS>(sum, x, p.scale_log2, off + run * 32, n);
            else
              weights_terms<16, 0, true, COLS>(sum, x, p.scale_log2, off + run * 32, n);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(c_empty + cs);
      }
      if (!ok || g >= p.groups || n >= p.N) continue;
      float s0, s1;
      f2_unpack(f2_add(sum[0], sum[1]), s0, s1);
      if (p.chunks > 1)
        p.partial[(static_cast<int64_t>(it.chunk) * p.B + it.b) * p.N + n] = s0 + s1;
      else
        p.weights[static_cast<int64_t>(it.b) * p.weights_ld + n] += s0 + s1;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 16) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// weights += the chunks' sums, in their order.
__global__ void __launch_bounds__(256)
    weights_reduce_kernel(const float* partial, float* weights, int64_t weights_ld, int chunks, int B, int N) {
  griddep_wait();
  const int64_t rows = static_cast<int64_t>(B) * N;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= rows) return;
  float sum = 0.f;
  for (int c = 0; c < chunks; ++c) sum += partial[c * rows + i];
  weights[i / N * weights_ld + i % N] += sum;
}

}  // namespace wpt
