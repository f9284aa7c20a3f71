// The one translation unit of libwpt_b200.so: the kernels (headers beside
// this file) and the extern "C" launchers declared in include/wpt_attn.h.
#include <algorithm>
#include <atomic>
#include <climits>
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <map>
#include <mutex>
#include <utility>
#include <string>

#include "../../include/wpt_attn.h"
#include "accept.cuh"
#include "backward.cuh"
#include "beam.cuh"
#include "cache.cuh"
#include "common.cuh"
#include "evict.cuh"
#include "exchange.cuh"
#include "head.cuh"
#include "merge.cuh"
#include "paged.cuh"
#include "prefill.cuh"
#include "rotary.cuh"
#include "select.cuh"
#include "stream.cuh"
#include "tree.cuh"
#include "weights.cuh"

namespace {

thread_local std::string g_error;

int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  g_error = buf;
  return code;
}

int cuda_fail(cudaError_t e, const char* what) {
  return fail(WPT_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

__device__ unsigned g_status_word;

// One lock for every per-device cache of a device symbol's address (the
// status word here, the no-alloc scratch below). The caches are filled once
// per device and never refreshed: the library must not be used across a
// cudaDeviceReset (or any teardown of the device's primary context), after
// which the cached addresses would be stale.
std::mutex g_symbol_lock;

// The device address of the status word on the current device.
int status_word(unsigned** out) {
  static unsigned* cached[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  if (dev < 0 || dev >= 64) return fail(WPT_ERR_INVALID, "device %d out of range", dev);
  std::lock_guard<std::mutex> guard(g_symbol_lock);
  if (cached[dev] == nullptr) {
    void* p = nullptr;
    e = cudaGetSymbolAddress(&p, g_status_word);
    if (e != cudaSuccess) return cuda_fail(e, "cudaGetSymbolAddress(status)");
    cached[dev] = static_cast<unsigned*>(p);
  }
  *out = cached[dev];
  return WPT_OK;
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

int encoder(EncodeTiled* out) {
  static EncodeTiled fn = nullptr;
  if (fn == nullptr) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q);
    if (e != cudaSuccess || q != cudaDriverEntryPointSuccess || p == nullptr)
      return fail(WPT_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    fn = reinterpret_cast<EncodeTiled>(p);
  }
  *out = fn;
  return WPT_OK;
}

// A tensor map with 128-byte swizzle, of bf16 where nothing else is said.
// Makes the current device's primary context current on this host thread.
// Runtime calls bind it lazily, but the driver's tensor-map encoder needs it
// bound already, and a thread that has made no runtime call on the device
// yet (autograd's backward worker, for one) has none: cudaSetDevice binds it.
// Once per thread and device.
int bind_context() {
  static thread_local int bound = -1;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  if (bound != dev) {
    e = cudaSetDevice(dev);
    if (e != cudaSuccess) return cuda_fail(e, "cudaSetDevice");
    bound = dev;
  }
  return WPT_OK;
}

// A tensor map depends only on its base address, shape, strides and box, so
// each host thread keeps its last few encodings and a repeated call (a
// decode loop over the same tables) skips the driver's encoder.
struct MapKey {
  const void* base;
  int rank, dev;
  CUtensorMapDataType type;
  cuuint64_t dims[3], strides[2];
  cuuint32_t box[3];
};

int tensor_map_encode(CUtensorMap* map, const void* base, int rank, const cuuint64_t* dims,
                      const cuuint64_t* strides_bytes, const cuuint32_t* box, CUtensorMapDataType type);
int current_device(int* sms = nullptr);

int tensor_map(CUtensorMap* map, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides_bytes,
               const cuuint32_t* box, CUtensorMapDataType type = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16) {
  constexpr int SLOTS = 16;
  static thread_local MapKey keys[SLOTS];
  static thread_local CUtensorMap maps[SLOTS];
  static thread_local int used = 0, next = 0;
  MapKey key;
  memset(&key, 0, sizeof(key));
  key.base = base;
  key.rank = rank;
  key.dev = current_device();
  key.type = type;
  for (int i = 0; i < rank; ++i) {
    key.dims[i] = dims[i];
    key.box[i] = box[i];
    if (i + 1 < rank) key.strides[i] = strides_bytes[i];
  }
  for (int i = 0; i < used; ++i)
    if (memcmp(&keys[i], &key, sizeof(key)) == 0) {
      *map = maps[i];
      return WPT_OK;
    }
  if (int rc = tensor_map_encode(map, base, rank, dims, strides_bytes, box, type)) return rc;
  keys[next] = key;
  maps[next] = *map;
  next = (next + 1) % SLOTS;
  if (used < SLOTS) ++used;
  return WPT_OK;
}

int tensor_map_encode(CUtensorMap* map, const void* base, int rank, const cuuint64_t* dims,
                      const cuuint64_t* strides_bytes, const cuuint32_t* box, CUtensorMapDataType type) {
  EncodeTiled encode;
  if (int rc = encoder(&encode)) return rc;
  if (int rc = bind_context()) return rc;
  cuuint32_t elem[3] = {1, 1, 1};
  CUresult r = encode(map, type, rank, const_cast<void*>(base), dims, strides_bytes,
                      box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(WPT_ERR_INVALID, "cuTensorMapEncodeTiled failed (%d)", static_cast<int>(r));
  return WPT_OK;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// A (B, N, C) table as a 3-D map {C, N, B} with boxes of {64, 128, 1}.
int table_map(CUtensorMap* map, const void* base, int64_t stride_b, int64_t stride_n, int B, int N, int C) {
  if (!aligned16(base)) return fail(WPT_ERR_INVALID, "a key/value table is not 16-byte aligned");
  if (stride_n % 8 != 0 || (B > 1 && stride_b % 8 != 0) || stride_n < C)
    return fail(WPT_ERR_INVALID, "key/value strides must be multiples of 8 elements (got %lld, %lld)",
                static_cast<long long>(stride_b), static_cast<long long>(stride_n));
  if (B == 1) stride_b = static_cast<int64_t>(N) * stride_n;
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(C), static_cast<cuuint64_t>(N), static_cast<cuuint64_t>(B)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(stride_n) * 2, static_cast<cuuint64_t>(stride_b) * 2};
  cuuint32_t box[3] = {64, 128, 1};
  return tensor_map(map, base, 3, dims, strides, box);
}

// The current device (and its SM count), asked of the runtime once per
// thread and device change rather than on every launch.
int current_device(int* sms) {
  static thread_local int cached_sms[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = 0;
  if (sms) {
    if (cached_sms[dev] == 0) {
      int v = 148;
      if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) v = 148;
      cached_sms[dev] = v;
    }
    *sms = cached_sms[dev];
  }
  return dev;
}

// Raises a kernel's dynamic shared memory limit to `bytes` on the current
// device, once per (kernel, device, size): the attribute call costs
// microseconds that a decode step should not pay on every launch.
template <typename Kernel>
int allow_smem(Kernel kernel, int bytes) {
  static std::mutex mu;
  static std::map<std::pair<const void*, int>, int> done;
  const int dev = current_device();
  const auto key = std::make_pair(reinterpret_cast<const void*>(kernel), dev);
  // one lock over the check and the call: the limit never falls under what another thread's launch needs
  std::lock_guard<std::mutex> lock(mu);
  auto it = done.find(key);
  if (it != done.end() && it->second >= bytes) return WPT_OK;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(max dynamic shared memory)");
  done[key] = bytes;
  return WPT_OK;
}

// Q-pair buffers and K/V ring stages of the prefill kernel: the ring gets
// what 227 KB leaves after the Q buffers (the next item's Q is prefetched
// into L2 instead of a second buffer when C = 128).
template <int C>
struct PrefillShape {
  static constexpr int QB = C == 128 ? 1 : 2, NS = C == 128 ? 5 : 8;
};

// Pairs of weights in every 8 computed on the FMA pipe (WPT_B200_POLY8 = 0..4 overrides).
int prefill_poly8() {
  static int v = -1;
  if (v < 0) {
    const char* env = getenv("WPT_B200_POLY8");
    const int e = env ? atoi(env) : 1;
    v = (e >= 0 && e <= 4) ? e : 1;
  }
  return v;
}

template <int C, int POLY8, bool CLUSTER>
int launch_prefill_p(const wpt::PrefillParams& p, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                     const CUtensorMap& to, cudaStream_t stream) {
  constexpr int QB = PrefillShape<C>::QB, NS = PrefillShape<C>::NS;
  using L = wpt::PrefillLayout<C, QB, NS>;
  static_assert(L::BYTES <= 232448, "prefill kernel shared memory exceeds 227 KB");
  auto kernel = wpt::prefill_kernel<C, QB, NS, POLY8, CLUSTER>;
  if (int rc = allow_smem(kernel, L::BYTES)) return rc;
  // setmaxnreg redistributes the registers the block was launched with: a
  // kernel built with fewer than REGS_LAUNCH would leave the softmax
  // warpgroups' increase waiting forever, so it is refused here instead
  static int regs = -1;
  if (regs < 0) {
    cudaFuncAttributes fa;
    cudaError_t e = cudaFuncGetAttributes(&fa, kernel);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncGetAttributes(prefill_kernel)");
    regs = fa.numRegs;
  }
  if (regs != L::REGS_LAUNCH)
    return fail(WPT_ERR_CUDA, "prefill_kernel built with %d registers a thread, its register split needs %d", regs,
                L::REGS_LAUNCH);
  int sms = 148;
  current_device(&sms);
  const int grid = p.items < sms ? p.items : sms;  // persistent: one CTA per SM walks the items
  if (p.cluster && (grid != p.items || p.items % 2 != 0))
    return fail(WPT_ERR_INVALID, "prefill cluster mode needs one item per CTA (%d items, %d SMs)", p.items, sms);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;  // cluster mode: a pair's two splits per cluster
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.cluster ? 1 : 0;
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(L::THREADS);
  cfg.dynamicSmemBytes = L::BYTES;
  cfg.stream = stream;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, tq, tk, tv, to, p);
  if (e != cudaSuccess) return cuda_fail(e, "prefill_kernel launch");
  return WPT_OK;
}

template <int C>
int launch_prefill(const wpt::PrefillParams& p, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                   const CUtensorMap& to,
                   cudaStream_t stream) {
  // the cluster-combine instance (the POLY8 overrides are for sweeps of the plain one)
  if (p.cluster) return launch_prefill_p<C, 1, true>(p, tq, tk, tv, to, stream);
  switch (prefill_poly8()) {
    case 0: return launch_prefill_p<C, 0, false>(p, tq, tk, tv, to, stream);
    case 3: return launch_prefill_p<C, 3, false>(p, tq, tk, tv, to, stream);
    case 4: return launch_prefill_p<C, 4, false>(p, tq, tk, tv, to, stream);
    case 2: return launch_prefill_p<C, 2, false>(p, tq, tk, tv, to, stream);
    default: return launch_prefill_p<C, 1, false>(p, tq, tk, tv, to, stream);
  }
}

// 1: the key-stream kernel launches as a programmatic dependent of the
// kernel before it on the stream (WPT_B200_PDL = 0 or 1 overrides).
int stream_pdl() {
  static int v = -1;
  if (v < 0) {
    const char* env = getenv("WPT_B200_PDL");
    v = env ? (atoi(env) != 0) : 1;
  }
  return v;
}

template <int NCOL, int STAGES, bool GATHER>
int launch_stream_n(const CUtensorMap& tk, const CUtensorMap& tv, const wpt::StreamParams& p, int groups,
                    cudaStream_t stream) {
  using L = wpt::StreamLayout<NCOL, STAGES>;
  static_assert(L::BYTES <= 232448, "key-stream kernel shared memory exceeds 227 KB");
  auto kernel = wpt::stream_kernel<NCOL, STAGES, GATHER>;
  if (int rc = allow_smem(kernel, L::BYTES)) return rc;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  int na = 0;
  if (stream_pdl()) {  // its set-up overlaps the tail of the kernel before it (it waits on the device)
    attr[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[na++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (p.cluster > 1) {  // cluster mode: one group's splits per cluster
    attr[na].id = cudaLaunchAttributeClusterDimension;
    attr[na].val.clusterDim.x = 1;
    attr[na].val.clusterDim.y = p.cluster;
    attr[na++].val.clusterDim.z = 1;
  }
  cfg.attrs = attr;
  cfg.numAttrs = na;
  cfg.gridDim = dim3(groups, p.splits);
  cfg.blockDim = dim3(wpt::STREAM_THREADS);
  cfg.dynamicSmemBytes = L::BYTES;
  cfg.stream = stream;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, tk, tv, p);
  if (e != cudaSuccess) return cuda_fail(e, "stream_kernel launch");
  return WPT_OK;
}

template <bool GATHER>
int launch_stream_g(const CUtensorMap& tk, const CUtensorMap& tv, const wpt::StreamParams& p, int ncol, int groups,
                    cudaStream_t stream) {
  switch (ncol) {
    case 16: return launch_stream_n<16, 3, GATHER>(tk, tv, p, groups, stream);
    case 32: return launch_stream_n<32, 3, GATHER>(tk, tv, p, groups, stream);
    default: return launch_stream_n<64, 2, GATHER>(tk, tv, p, groups, stream);
  }
}

template <int NCOL>
int launch_score(const CUtensorMap& tq, const CUtensorMap& tk, const wpt::ScoreParams& p, int groups, int splits,
                 cudaStream_t stream) {
  constexpr int STAGES = 4;
  using L = wpt::ScoreLayout<NCOL, STAGES>;
  static_assert(L::BYTES <= 232448, "score kernel shared memory exceeds 227 KB");
  auto kernel = wpt::score_kernel<NCOL, STAGES>;
  if (int rc = allow_smem(kernel, L::BYTES)) return rc;
  int sms = 148;
  current_device(&sms);
  const dim3 grid = p.balanced ? dim3(sms) : dim3(groups, splits);  // balanced: one CTA per SM
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // waits for lse on the device
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.gridDim = grid;
  cfg.blockDim = dim3(192);
  cfg.dynamicSmemBytes = L::BYTES;
  cfg.stream = stream;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, tq, tk, p);
  if (e != cudaSuccess) return cuda_fail(e, "score_kernel launch");
  return WPT_OK;
}

template <int C>
// pdl: the merge directly follows the attention kernel that wrote the
// partials, and launches while that kernel finishes (programmatic dependent
// launch; the merge waits for it on the device before reading).
int launch_merge(const float* part_o, const float* part_lse, int splits, int64_t rows, wpt::SplitLayout lay, int H,
                 const float* sink, void* out, float* lse, cudaStream_t stream, bool pdl = false,
                 float* out_f32 = nullptr) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 1 : 0;
  cfg.stream = stream;
  cfg.dynamicSmemBytes = 0;
  __nv_bfloat16* o = static_cast<__nv_bfloat16*>(out);
  cudaError_t e;
  if (splits >= 16 && splits <= wpt::MERGE_MAX_SPLITS && rows <= 4096) {  // few rows, many splits: a CTA per row
    cfg.gridDim = dim3(static_cast<unsigned>(rows));
    cfg.blockDim = dim3(wpt::MERGE_THREADS);
    e = cudaLaunchKernelEx(&cfg, wpt::merge_wide_kernel<C>, part_o, part_lse, splits, lay, H, sink, o, lse, out_f32);
  } else {
    const int warps = 8;
    const int64_t blocks = (rows + warps - 1) / warps;
    cfg.gridDim = dim3(static_cast<unsigned>(blocks));
    cfg.blockDim = dim3(warps * 32);
    e = cudaLaunchKernelEx(&cfg, wpt::merge_kernel<C>, part_o, part_lse, splits, rows, lay, H, sink, o, lse,
                           out_f32);
  }
  if (e != cudaSuccess) return cuda_fail(e, "merge_kernel launch");
  return WPT_OK;
}

// The plain (splits, rows) layout at split stride `split_stride` rows.
template <int C>
int launch_merge(const float* part_o, const float* part_lse, int splits, int64_t rows, int64_t split_stride, int H,
                 const float* sink, void* out, float* lse, cudaStream_t stream, bool pdl = false) {
  wpt::SplitLayout lay;
  lay.per = splits;
  lay.stride = split_stride;
  lay.group_o = 0;
  lay.group_l = 0;
  return launch_merge<C>(part_o, part_lse, splits, rows, lay, H, sink, out, lse, stream, pdl);
}

}  // namespace

extern "C" const char* wpt_last_error(void) { return g_error.c_str(); }

extern "C" int wpt_status(unsigned* status, int reset) {
  unsigned* word = nullptr;
  if (int rc = status_word(&word)) return rc;
  cudaError_t e = cudaDeviceSynchronize();
  if (e != cudaSuccess) return cuda_fail(e, "cudaDeviceSynchronize");
  unsigned value = 0;
  e = cudaMemcpy(&value, word, sizeof(value), cudaMemcpyDeviceToHost);
  if (e != cudaSuccess) return cuda_fail(e, "read status");
  if (reset) {
    e = cudaMemset(word, 0, sizeof(unsigned));
    if (e != cudaSuccess) return cuda_fail(e, "reset status");
    e = cudaDeviceSynchronize();
    if (e != cudaSuccess) return cuda_fail(e, "cudaDeviceSynchronize");
  }
  if (status) *status = value;
  return WPT_OK;
}

extern "C" int wpt_attn_prefill(const void* q, const void* k, const void* v, int64_t k_stride_b, int64_t k_stride_n,
                                int64_t v_stride_b, int64_t v_stride_n, const int64_t* positions,
                                const int64_t* floor_rows, const uint64_t* tree_bits, const int64_t* tree_base,
                                const float* sink, void* out, float* lse, float* part_o, float* part_lse, int splits,
                                int B, int T, int H, int C, int N, int window, float scale, void* stream) {
  if (C != 64 && C != 128) return fail(WPT_ERR_UNSUPPORTED, "head width %d: the kernels take 64 or 128", C);
  if (H < 1 || H > 128) return fail(WPT_ERR_UNSUPPORTED, "%d heads: the kernels take 1 to 128", H);
  if (B < 1 || T < 1 || N < 1) return fail(WPT_ERR_INVALID, "empty shape B=%d T=%d N=%d", B, T, N);
  if (static_cast<int64_t>(B) * T * H + 256 >= (int64_t(1) << 31)) return fail(WPT_ERR_UNSUPPORTED, "B*T*H too large");
  if (splits < 1) return fail(WPT_ERR_INVALID, "splits must be >= 1");
  // part_o and part_lse both NULL with 2 splits: cluster mode (a pair's two
  // splits combine in shared memory; no scratch, no merge launch)
  const bool cluster = splits == 2 && part_o == nullptr && part_lse == nullptr;
  if (splits > 1 && !cluster && (part_o == nullptr || part_lse == nullptr))
    return fail(WPT_ERR_INVALID, "splits > 1 needs part_o and part_lse scratch (or neither, for 2)");
  if (tree_bits != nullptr && tree_base == nullptr) return fail(WPT_ERR_INVALID, "tree_bits needs tree_base");
  if (!q || !k || !v || !positions || !out || !lse) return fail(WPT_ERR_INVALID, "a required pointer is NULL");
  if (!aligned16(q) || !aligned16(out)) return fail(WPT_ERR_INVALID, "q and out must be 16-byte aligned");
  if (!(scale > 0.f)) return fail(WPT_ERR_INVALID, "scale must be positive");

  CUtensorMap tq, tk, tv, to;  // to: the output, same shape as q (full query tiles leave by TMA store)
  {
    cuuint64_t dims[2] = {static_cast<cuuint64_t>(C), static_cast<cuuint64_t>(B) * T * H};
    cuuint64_t strides[1] = {static_cast<cuuint64_t>(C) * 2};
    cuuint32_t box[2] = {64, 128};
    if (int rc = tensor_map(&tq, q, 2, dims, strides, box)) return rc;
    if (int rc = tensor_map(&to, out, 2, dims, strides, box)) return rc;
  }
  if (int rc = table_map(&tk, k, k_stride_b, k_stride_n, B, N, C)) return rc;
  if (int rc = table_map(&tv, v, v_stride_b, v_stride_n, B, N, C)) return rc;

  wpt::PrefillParams p;
  p.positions = positions;
  p.floor_rows = floor_rows;
  p.tree_bits = tree_bits;
  p.tree_base = tree_base;
  p.sink = splits > 1 && !cluster ? nullptr : sink;  // cluster mode: its combine adds the sink
  p.cluster = cluster ? 1 : 0;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.lse = lse;
  p.part_o = part_o;
  p.part_lse = part_lse;
  p.tma_out = splits > 1 ? 0 : 1;
  if (int rc = status_word(&p.status)) return rc;
  p.B = B;
  p.T = T;
  p.H = H;
  p.N = N;
  p.window = window > 0 ? window : 0;
  p.TQ = 128 / H;
  p.splits = splits;
  {
    const int64_t items = static_cast<int64_t>((T + 2 * p.TQ - 1) / (2 * p.TQ)) * B * splits;  // query-tile pairs
    if (items >= (int64_t(1) << 31)) return fail(WPT_ERR_UNSUPPORTED, "too many prefill work items");
    p.items = static_cast<int>(items);
  }
  p.scale_log2 = scale * wpt::LOG2E;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int rc = C == 128 ? launch_prefill<128>(p, tq, tk, tv, to, s) : launch_prefill<64>(p, tq, tk, tv, to, s);
  if (rc) return rc;
  if (splits > 1 && !cluster) {
    const int64_t rows = static_cast<int64_t>(B) * T * H;
    rc = C == 128 ? launch_merge<128>(part_o, part_lse, splits, rows, rows, H, sink, out, lse, s, true)
                  : launch_merge<64>(part_o, part_lse, splits, rows, rows, H, sink, out, lse, s, true);
  }
  return rc;
}

// ---------------------------------------------------------------- backward
namespace {

struct BwdScratch {
  int64_t ld, ranges, bounds, sink_part, kv_part, total;  // byte offsets, each 256-aligned
  int kv_parts;
};

// Parts per key tile of the key-tile kernel: enough CTAs for about two per
// SM, since under a causal mask key tile 0 is read by every query tile and
// the last one by a few, and the most-read tile sets the kernel's length.
int bwd_kv_parts(int B, int N) {
  int sms = 148;
  current_device(&sms);
  const int64_t units = static_cast<int64_t>(B) * ((N + 127) / 128);
  const int64_t want = (2 * static_cast<int64_t>(sms) + units - 1) / units;
  return static_cast<int>(want < 1 ? 1 : want > 8 ? 8 : want);
}

BwdScratch bwd_scratch(int B, int T, int H, int N) {
  const int TQ = 128 / H;
  const int64_t qtiles = (T + TQ - 1) / TQ;
  auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
  BwdScratch s;
  s.kv_parts = bwd_kv_parts(B, N);
  s.ld = 0;
  s.ranges = s.ld + up(static_cast<int64_t>(B) * qtiles * 256 * 4);
  s.bounds = s.ranges + up(static_cast<int64_t>(B) * qtiles * 8);
  s.sink_part = s.bounds + up(static_cast<int64_t>(B) * T * 8);
  s.kv_part = s.sink_part + up(static_cast<int64_t>(B) * qtiles * H * 4);
  s.total = s.kv_part + (s.kv_parts > 1 ? up(static_cast<int64_t>(s.kv_parts) * B * N * 256 * 4) : 0);
  return s;
}

}  // namespace

// The failure-detection test hook of wpt_debug_backward_fault.
std::atomic<int> g_bwd_skip_key_tile{-1};
std::atomic<unsigned long long> g_bwd_wait_ns{0};

extern "C" int wpt_debug_backward_fault(int skip_key_tile, unsigned long long wait_ns) {
  if (skip_key_tile < -1) return fail(WPT_ERR_INVALID, "skip_key_tile must be -1 (off) or a key tile index");
  g_bwd_skip_key_tile.store(skip_key_tile);
  g_bwd_wait_ns.store(wait_ns);
  return WPT_OK;
}

extern "C" size_t wpt_attn_backward_scratch_bytes(int B, int T, int H, int C, int N) {
  if (B < 1 || T < 1 || H < 1 || H > 128 || C != 128 || N < 1) return 0;
  return static_cast<size_t>(bwd_scratch(B, T, H, N).total);
}

template <int NCOL>
int launch_gather_bwd(const wpt::GatherBwdParams& g, cudaStream_t st) {
  using L = wpt::GatherBwdLayout<NCOL>;
  static_assert(L::BYTES <= 232448, "gathered-rows backward shared memory exceeds 227 KB");
  if (int rc = allow_smem(wpt::bwd_gather_kernel<NCOL>, L::BYTES)) return rc;
  wpt::bwd_gather_kernel<NCOL><<<static_cast<unsigned>(static_cast<int64_t>(g.B) * g.T), wpt::GBWD_THREADS, L::BYTES,
                                 st>>>(g);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "bwd_gather_kernel launch");
  return WPT_OK;
}

extern "C" int wpt_attn_backward(const void* q, const void* k, const void* v, int64_t k_stride_b, int64_t k_stride_n,
                                 int64_t v_stride_b, int64_t v_stride_n, const int64_t* positions,
                                 const int64_t* floor_rows, const int64_t* idx, int K, const float* sink,
                                 const void* out, const float* lse, const void* d_out, void* dq, void* dk, void* dv,
                                 float* d_sink, void* scratch, int f32_grads, int B, int T, int H, int C, int N,
                                 int window, float scale, void* stream) {
  if (K < 0 || (K > 0 && idx == nullptr)) return fail(WPT_ERR_INVALID, "K=%d chosen rows need idx", K);
  if (K > 0 && !f32_grads)
    return fail(WPT_ERR_INVALID, "gradients over chosen rows accumulate in fp32: pass f32_grads = 1");
  if (K > 0 && H > 64) return fail(WPT_ERR_UNSUPPORTED, "%d heads: the gathered-rows backward takes up to 64", H);
  if (C != 128) return fail(WPT_ERR_UNSUPPORTED, "head width %d: the backward kernels take 128", C);
  if (H < 1 || H > 128) return fail(WPT_ERR_UNSUPPORTED, "%d heads: the kernels take 1 to 128", H);
  if (B < 1 || T < 1 || N < 1) return fail(WPT_ERR_INVALID, "empty shape B=%d T=%d N=%d", B, T, N);
  if (static_cast<int64_t>(B) * T * H + 256 >= (int64_t(1) << 31)) return fail(WPT_ERR_UNSUPPORTED, "B*T*H too large");
  if (static_cast<int64_t>(B) * N * C >= (int64_t(1) << 40)) return fail(WPT_ERR_UNSUPPORTED, "B*N too large");
  if (!q || !k || !v || !positions || !out || !lse || !d_out || !dq || !dk || !dv || !scratch)
    return fail(WPT_ERR_INVALID, "a required pointer is NULL");
  if (!aligned16(q) || !aligned16(out) || !aligned16(d_out) || !aligned16(dq) || !aligned16(dk) || !aligned16(dv) ||
      !aligned16(scratch))
    return fail(WPT_ERR_INVALID, "q, out, d_out, dq, dk, dv and scratch must be 16-byte aligned");
  if (sink == nullptr && d_sink != nullptr) return fail(WPT_ERR_INVALID, "d_sink needs sink");
  if (!(scale > 0.f)) return fail(WPT_ERR_INVALID, "scale must be positive");
  CUtensorMap tq, tdo, tk, tv;
  {
    cuuint64_t dims[2] = {static_cast<cuuint64_t>(C), static_cast<cuuint64_t>(B) * T * H};
    cuuint64_t strides[1] = {static_cast<cuuint64_t>(C) * 2};
    cuuint32_t box[2] = {64, 128};
    if (int rc = tensor_map(&tq, q, 2, dims, strides, box)) return rc;
    if (int rc = tensor_map(&tdo, d_out, 2, dims, strides, box)) return rc;
  }
  if (int rc = table_map(&tk, k, k_stride_b, k_stride_n, B, N, C)) return rc;
  if (int rc = table_map(&tv, v, v_stride_b, v_stride_n, B, N, C)) return rc;
  const BwdScratch lay = bwd_scratch(B, T, H, N);
  uint8_t* base = static_cast<uint8_t*>(scratch);
  wpt::BwdParams p;
  p.positions = positions;
  p.floor_rows = floor_rows;
  p.out = static_cast<const __nv_bfloat16*>(out);
  p.d_out = static_cast<const __nv_bfloat16*>(d_out);
  p.lse = lse;
  p.sink = sink;
  p.ld = reinterpret_cast<float*>(base + lay.ld);
  p.ranges = reinterpret_cast<int2*>(base + lay.ranges);
  p.bounds = reinterpret_cast<int2*>(base + lay.bounds);
  p.sink_part = reinterpret_cast<float*>(base + lay.sink_part);
  p.dq = dq;
  p.dk = dk;
  p.dv = dv;
  p.d_sink = d_sink;
  if (int rc = status_word(&p.status)) return rc;
  p.B = B;
  p.T = T;
  p.H = H;
  p.N = N;
  p.window = window > 0 ? window : 0;
  p.TQ = 128 / H;
  p.qtiles = (T + p.TQ - 1) / p.TQ;
  p.ktiles = (N + 127) / 128;
  p.f32_grads = f32_grads ? 1 : 0;
  p.scale = scale;
  p.scale_log2 = scale * wpt::LOG2E;
  p.kv_parts = lay.kv_parts;
  p.kv_part = reinterpret_cast<float*>(base + lay.kv_part);
  p.skip_key_tile = g_bwd_skip_key_tile.load();
  p.wait_ns = g_bwd_wait_ns.load();
  if (p.wait_ns == 0) p.wait_ns = wpt::WAIT_LIMIT_NS;
  if (static_cast<int64_t>(p.qtiles) * B >= (int64_t(1) << 31) ||
      static_cast<int64_t>(p.ktiles) * B * p.kv_parts >= (int64_t(1) << 31) || B > 65535)
    return fail(WPT_ERR_UNSUPPORTED, "backward grid too large");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  wpt::bwd_prep_kernel<<<dim3(p.qtiles, B), 128, 0, st>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "bwd_prep_kernel launch");
  if (d_sink != nullptr) {
    wpt::bwd_sink_kernel<<<H, 256, 0, st>>>(p.sink_part, static_cast<int64_t>(B) * p.qtiles, H, d_sink);
    e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_fail(e, "bwd_sink_kernel launch");
  }
  static_assert(wpt::BwdKvLayout::BYTES <= 232448, "backward key kernel shared memory exceeds 227 KB");
  static_assert(wpt::BwdQLayout::BYTES <= 232448, "backward query kernel shared memory exceeds 227 KB");
  if (int rc = allow_smem(wpt::bwd_kv_kernel, wpt::BwdKvLayout::BYTES)) return rc;
  if (int rc = allow_smem(wpt::bwd_q_kernel, wpt::BwdQLayout::BYTES)) return rc;
  wpt::bwd_kv_kernel<<<static_cast<unsigned>(static_cast<int64_t>(p.ktiles) * B * p.kv_parts), wpt::BWD_THREADS,
                       wpt::BwdKvLayout::BYTES, st>>>(tq, tdo, tk, tv, p);
  e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "bwd_kv_kernel launch");
  if (p.kv_parts > 1) {
    int sms = 148;
    current_device(&sms);
    const int64_t n4 = static_cast<int64_t>(B) * N * 64;
    const int blocks = static_cast<int>(std::min<int64_t>((n4 + 255) / 256, static_cast<int64_t>(sms) * 8));
    wpt::bwd_kv_reduce_kernel<<<blocks, 256, 0, st>>>(p.kv_part, p.kv_parts, static_cast<int64_t>(B) * N, dk, dv,
                                                      p.f32_grads);
    e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_fail(e, "bwd_kv_reduce_kernel launch");
  }
  wpt::bwd_q_kernel<<<static_cast<unsigned>(p.qtiles * B), wpt::BWD_THREADS, wpt::BwdQLayout::BYTES, st>>>(
      tq, tdo, tk, tv, p);
  e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "bwd_q_kernel launch");
  if (K > 0) {  // the chosen rows' share, added to the fp32 gradients above
    wpt::GatherBwdParams g;
    g.q = static_cast<const __nv_bfloat16*>(q);
    g.d_out = static_cast<const __nv_bfloat16*>(d_out);
    g.k = static_cast<const __nv_bfloat16*>(k);
    g.v = static_cast<const __nv_bfloat16*>(v);
    g.ksb = k_stride_b;
    g.ksn = k_stride_n;
    g.vsb = v_stride_b;
    g.vsn = v_stride_n;
    g.idx = idx;
    g.ld = p.ld;
    g.dq = static_cast<float*>(dq);
    g.dk = static_cast<float*>(dk);
    g.dv = static_cast<float*>(dv);
    g.status = p.status;
    g.B = B;
    g.T = T;
    g.H = H;
    g.N = N;
    g.K = K;
    g.TQ = p.TQ;
    g.qtiles = p.qtiles;
    g.scale = scale;
    g.scale_log2 = p.scale_log2;
    const int rc = H <= 16 ? launch_gather_bwd<16>(g, st) : H <= 32 ? launch_gather_bwd<32>(g, st)
                                                                     : launch_gather_bwd<64>(g, st);
    if (rc) return rc;
  }
  return WPT_OK;
}

extern "C" int wpt_f32_to_bf16(const float* x, int64_t n, void* y, void* stream) {
  if (n < 0 || (n > 0 && (!x || !y))) return fail(WPT_ERR_INVALID, "bad f32_to_bf16 arguments");
  if (n % 4 || !aligned16(x) || reinterpret_cast<uintptr_t>(y) % 8)
    return fail(WPT_ERR_INVALID, "f32_to_bf16 takes a multiple of 4 values, x 16-byte and y 8-byte aligned");
  if (n == 0) return WPT_OK;
  int sms = 148;
  current_device(&sms);
  const int64_t want = (n / 4 + 255) / 256;
  const int blocks = static_cast<int>(std::min<int64_t>(want, static_cast<int64_t>(sms) * 8));
  wpt::f32_to_bf16_kernel<<<blocks, 256, 0, static_cast<cudaStream_t>(stream)>>>(
      reinterpret_cast<const float4*>(x), n / 4, static_cast<uint2*>(y));
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "f32_to_bf16_kernel launch");
  return WPT_OK;
}

extern "C" int wpt_attn_merge(const float* part_o, const float* part_lse, int splits, int64_t rows,
                              int64_t split_stride, int H, int C, const float* sink, void* out, float* lse,
                              void* stream) {
  if (C != 64 && C != 128) return fail(WPT_ERR_UNSUPPORTED, "head width %d: the kernels take 64 or 128", C);
  if (splits < 1 || rows < 0 || split_stride < rows || H < 1)
    return fail(WPT_ERR_INVALID, "bad merge shape splits=%d rows=%lld", splits, static_cast<long long>(rows));
  if (rows == 0) return WPT_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return C == 128 ? launch_merge<128>(part_o, part_lse, splits, rows, split_stride, H, sink, out, lse, s)
                  : launch_merge<64>(part_o, part_lse, splits, rows, split_stride, H, sink, out, lse, s);
}

extern "C" int wpt_attn_merge_partial(const float* part_o, const float* part_lse, int splits, int64_t rows,
                                      int64_t split_stride, int C, float* out_o, float* out_lse, void* stream) {
  if (C != 64 && C != 128) return fail(WPT_ERR_UNSUPPORTED, "head width %d: the kernels take 64 or 128", C);
  if (splits < 1 || rows < 0 || split_stride < rows)
    return fail(WPT_ERR_INVALID, "bad merge shape splits=%d rows=%lld", splits, static_cast<long long>(rows));
  if (!part_o || !part_lse || !out_o || !out_lse) return fail(WPT_ERR_INVALID, "a required pointer is NULL");
  if (rows == 0) return WPT_OK;
  wpt::SplitLayout lay;
  lay.per = splits;
  lay.stride = split_stride;
  lay.group_o = 0;
  lay.group_l = 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return C == 128 ? launch_merge<128>(part_o, part_lse, splits, rows, lay, 1, nullptr, nullptr, out_lse, s, false, out_o)
                  : launch_merge<64>(part_o, part_lse, splits, rows, lay, 1, nullptr, nullptr, out_lse, s, false, out_o);
}

extern "C" int wpt_attn_merge_groups(const float* parts, int groups, int per, int64_t rows, int64_t group_floats,
                                     int H, int C, const float* sink, void* out, float* lse, void* stream) {
  if (C != 64 && C != 128) return fail(WPT_ERR_UNSUPPORTED, "head width %d: the kernels take 64 or 128", C);
  if (groups < 1 || per < 1 || rows < 0 || H < 1)
    return fail(WPT_ERR_INVALID, "bad merge shape groups=%d per=%d rows=%lld", groups, per,
                static_cast<long long>(rows));
  if (static_cast<int64_t>(groups) * per > wpt::MERGE_MAX_SPLITS * 32)
    return fail(WPT_ERR_UNSUPPORTED, "%d x %d splits: too many", groups, per);
  if (group_floats < static_cast<int64_t>(per) * rows * (C + 1))
    return fail(WPT_ERR_INVALID, "group_floats %lld < per * rows * (C + 1)", static_cast<long long>(group_floats));
  if (!parts || !out || !lse) return fail(WPT_ERR_INVALID, "a required pointer is NULL");
  if (rows == 0) return WPT_OK;
  wpt::SplitLayout lay;
  lay.per = per;
  lay.stride = rows;
  lay.group_o = group_floats;
  lay.group_l = group_floats;
  const float* part_lse = parts + static_cast<int64_t>(per) * rows * C;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int splits = groups * per;
  return C == 128 ? launch_merge<128>(parts, part_lse, splits, rows, lay, H, sink, out, lse, s)
                  : launch_merge<64>(parts, part_lse, splits, rows, lay, H, sink, out, lse, s);
}

extern "C" size_t wpt_peer_bytes(int world, int64_t rows, int C) {
  if (C != 128 || world < 1 || world > wpt::EXCH_MAX_WORLD || rows < 1 || rows > wpt::EXCH_MAX_CTAS) return 0;
  const int64_t chunk = (rows * (C + 1) + 3) / 4 * 4;
  return static_cast<size_t>(wpt::EXCH_CTRL_BYTES + 2 * world * chunk * 4);
}

extern "C" int wpt_peer_alloc(size_t bytes, void** buffer, void* handle) {
  if (bytes == 0 || !buffer || !handle) return fail(WPT_ERR_INVALID, "peer buffer: bad arguments");
  void* p = nullptr;
  cudaError_t e = cudaMalloc(&p, bytes);
  if (e != cudaSuccess) return cuda_fail(e, "cudaMalloc(peer buffer)");
  e = cudaMemset(p, 0, bytes);
  if (e == cudaSuccess) e = cudaDeviceSynchronize();  // zeroed before any peer can write into it
  cudaIpcMemHandle_t h;
  if (e == cudaSuccess) e = cudaIpcGetMemHandle(&h, p);
  if (e != cudaSuccess) {
    cudaFree(p);
    return cuda_fail(e, "peer buffer set-up");
  }
  std::memcpy(handle, &h, sizeof(h));
  *buffer = p;
  return WPT_OK;
}

extern "C" int wpt_peer_open(const void* handle, void** buffer) {
  if (!handle || !buffer) return fail(WPT_ERR_INVALID, "peer open: bad arguments");
  cudaIpcMemHandle_t h;
  std::memcpy(&h, handle, sizeof(h));
  cudaError_t e = cudaIpcOpenMemHandle(buffer, h, cudaIpcMemLazyEnablePeerAccess);
  if (e != cudaSuccess) return cuda_fail(e, "cudaIpcOpenMemHandle");
  return WPT_OK;
}

extern "C" int wpt_peer_close(void* buffer, int opened) {
  cudaError_t e = opened ? cudaIpcCloseMemHandle(buffer) : cudaFree(buffer);
  if (e != cudaSuccess) return cuda_fail(e, opened ? "cudaIpcCloseMemHandle" : "cudaFree(peer buffer)");
  return WPT_OK;
}

extern "C" int wpt_attn_exchange(const float* part_o, const float* part_lse, int splits, int64_t rows, int H, int C,
                                 const float* sink, void* const* peers, int world, int rank, void* out, float* lse,
                                 void* stream) {
  if (C != 128) return fail(WPT_ERR_UNSUPPORTED, "head width %d: the exchange takes 128", C);
  if (world < 1 || world > wpt::EXCH_MAX_WORLD || rank < 0 || rank >= world)
    return fail(WPT_ERR_UNSUPPORTED, "world %d rank %d: 1 to %d ranks", world, rank, wpt::EXCH_MAX_WORLD);
  if (rows < 1 || rows > wpt::EXCH_MAX_CTAS)
    return fail(WPT_ERR_UNSUPPORTED, "%lld rows: the exchange takes 1 to %d", static_cast<long long>(rows),
                wpt::EXCH_MAX_CTAS);
  if (splits < 1 || H < 1) return fail(WPT_ERR_INVALID, "bad exchange shape splits=%d H=%d", splits, H);
  if (!part_o || !part_lse || !peers || !out || !lse) return fail(WPT_ERR_INVALID, "a required pointer is NULL");
  wpt::ExchangeParams p = {};
  p.part_o = part_o;
  p.part_lse = part_lse;
  p.sink = sink;
  for (int g = 0; g < world; ++g) {
    if (!peers[g] || reinterpret_cast<uintptr_t>(peers[g]) % 256 != 0)
      return fail(WPT_ERR_INVALID, "peer buffer %d is NULL or not 256-byte aligned", g);
    p.peers[g] = static_cast<uint8_t*>(peers[g]);
  }
  p.local = p.peers[rank];
  p.out = static_cast<__nv_bfloat16*>(out);
  p.lse = lse;
  if (int rc = status_word(&p.status)) return rc;
  p.chunk = (rows * (C + 1) + 3) / 4 * 4;
  p.splits = splits;
  p.rows = static_cast<int>(rows);
  p.H = H;
  p.world = world;
  p.rank = rank;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // waits for the partials on the device
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(rows));  // one row per CTA
  cfg.blockDim = dim3(wpt::EXCH_THREADS);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaLaunchKernelEx(&cfg, wpt::exchange_kernel<128>, p);
  if (e != cudaSuccess) return cuda_fail(e, "exchange_kernel launch");
  return WPT_OK;
}

extern "C" int wpt_attn_decode(const void* q, const void* k, const void* v, int64_t k_stride_b, int64_t k_stride_n,
                               int64_t v_stride_b, int64_t v_stride_n, const int64_t* positions,
                               const int64_t* floor_rows, const int64_t* idx, int K, const float* sink, void* out,
                               float* lse, float* part_o, float* part_lse, int splits, int chunk_tiles, int B, int T,
                               int H, int C, int N, int window, float scale, void* stream) {
  if (C != 128) return fail(WPT_ERR_UNSUPPORTED, "head width %d: the key-stream kernel takes 128", C);
  if (H < 1 || H > 64) return fail(WPT_ERR_UNSUPPORTED, "%d heads: the key-stream kernel takes 1 to 64", H);
  if (B < 1 || T < 1 || N < 1) return fail(WPT_ERR_INVALID, "empty shape B=%d T=%d N=%d", B, T, N);
  if (static_cast<int64_t>(B) * T * H >= (int64_t(1) << 31)) return fail(WPT_ERR_UNSUPPORTED, "B*T*H too large");
  if (splits < 1 || chunk_tiles < 1) return fail(WPT_ERR_INVALID, "splits and chunk_tiles must be >= 1");
  if (splits > 65535) return fail(WPT_ERR_UNSUPPORTED, "%d splits: at most 65535", splits);
  // part_o and part_lse both NULL with 2..8 splits: cluster mode (the splits
  // of a group merge in shared memory; no scratch, no merge launch)
  const bool cluster = splits > 1 && part_o == nullptr && part_lse == nullptr;
  if (cluster && splits > 8) return fail(WPT_ERR_INVALID, "%d splits without scratch: at most 8", splits);
  if (splits > 1 && !cluster && (part_o == nullptr || part_lse == nullptr))
    return fail(WPT_ERR_INVALID, "splits > 1 needs both part_o and part_lse scratch (or neither, for 2 to 8)");
  if (idx != nullptr && K < 0) return fail(WPT_ERR_INVALID, "K must be >= 0");
  // out and lse both NULL with splits > 1: partials only, merged by the caller
  const bool partials_only = splits > 1 && !cluster && out == nullptr && lse == nullptr;
  if (!q || !k || !v || !positions || ((!out || !lse) && !partials_only))
    return fail(WPT_ERR_INVALID, "a required pointer is NULL");
  if (!aligned16(q) || !aligned16(k) || !aligned16(v)) return fail(WPT_ERR_INVALID, "q, k, v must be 16-byte aligned");
  if (k_stride_n % 8 || v_stride_n % 8 || (B > 1 && (k_stride_b % 8 || v_stride_b % 8)))
    return fail(WPT_ERR_INVALID, "key/value strides must be multiples of 8 elements");
  if (!(scale > 0.f)) return fail(WPT_ERR_INVALID, "scale must be positive");
  const bool gather = idx != nullptr;
  const int cols = gather ? H : (T * H < 64 ? T * H : 64);
  const int ncol = cols <= 16 ? 16 : cols <= 32 ? 32 : 64;
  wpt::StreamParams p;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.k = static_cast<const __nv_bfloat16*>(k);
  p.v = static_cast<const __nv_bfloat16*>(v);
  p.ksb = k_stride_b;
  p.ksn = k_stride_n;
  p.vsb = v_stride_b;
  p.vsn = v_stride_n;
  p.positions = positions;
  p.floor_rows = gather ? nullptr : floor_rows;
  p.idx = idx;
  p.K = gather ? K : 0;
  p.sink = splits > 1 && !cluster ? nullptr : sink;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.lse = lse;
  p.part_o = part_o;
  p.part_lse = part_lse;
  if (int rc = status_word(&p.status)) return rc;
  p.B = B;
  p.T = T;
  p.H = H;
  p.N = N;
  p.window = window > 0 ? window : 0;
  p.TQ = gather ? 1 : ncol / H;
  p.groups_per_row = (T + p.TQ - 1) / p.TQ;
  p.splits = splits;
  p.chunk_tiles = chunk_tiles;
  p.cluster = cluster ? splits : 0;
  p.scale_log2 = scale * wpt::LOG2E;
  const int64_t groups = static_cast<int64_t>(B) * p.groups_per_row;
  if (groups >= (int64_t(1) << 31)) return fail(WPT_ERR_UNSUPPORTED, "too many query groups");
  // range mode loads whole tiles by TMA; gather mode loads its window's
  // tiles by TMA when the tables allow tensor maps, else copies every row
  CUtensorMap tk, tv;
  memset(&tk, 0, sizeof(tk));
  memset(&tv, 0, sizeof(tv));
  const auto mappable = [&](const void* t, int64_t sb, int64_t sn) {
    return aligned16(t) && sn % 8 == 0 && (B == 1 || sb % 8 == 0) && sn >= C;
  };
  p.window_tma = 0;
  if (!gather || (mappable(k, k_stride_b, k_stride_n) && mappable(v, v_stride_b, v_stride_n) && window > 0)) {
    if (int rc = table_map(&tk, k, k_stride_b, k_stride_n, B, N, C)) return rc;
    if (int rc = table_map(&tv, v, v_stride_b, v_stride_n, B, N, C)) return rc;
    p.window_tma = gather ? 1 : 0;
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int rc = gather ? launch_stream_g<true>(tk, tv, p, ncol, static_cast<int>(groups), s)
                        : launch_stream_g<false>(tk, tv, p, ncol, static_cast<int>(groups), s);
  if (rc) return rc;
  if (splits > 1 && !partials_only && !cluster) {
    const int64_t rows = static_cast<int64_t>(B) * T * H;
    return launch_merge<128>(part_o, part_lse, splits, rows, rows, H, sink, out, lse, s, true);
  }
  return WPT_OK;
}

extern "C" int wpt_attn_topk(const void* q, const void* k, int64_t k_stride_b, int64_t k_stride_n,
                             const int64_t* positions, const float* lse, float* scores, int64_t ld_scores,
                             int64_t* chosen, int K, int B, int T, int H, int C, int N, int window, float scale,
                             void* stream) {
  if (C != 128) return fail(WPT_ERR_UNSUPPORTED, "head width %d: the selection kernel takes 128", C);
  if (H < 1 || H > 128) return fail(WPT_ERR_UNSUPPORTED, "%d heads: the selection kernel takes 1 to 128", H);
  if (B < 1 || T < 1 || N < 1 || K < 0) return fail(WPT_ERR_INVALID, "bad shape B=%d T=%d N=%d K=%d", B, T, N, K);
  if (K == 0) return WPT_OK;
  if (ld_scores < N) return fail(WPT_ERR_INVALID, "ld_scores %lld < N %d", static_cast<long long>(ld_scores), N);
  if (!q || !k || !positions || !lse || !scores || !chosen) return fail(WPT_ERR_INVALID, "a required pointer is NULL");
  if (!aligned16(q)) return fail(WPT_ERR_INVALID, "q must be 16-byte aligned");
  if (static_cast<int64_t>(B) * T * H >= (int64_t(1) << 31)) return fail(WPT_ERR_UNSUPPORTED, "B*T*H too large");
  const int cols = T * H < 256 ? T * H : 256;
  const int ncol = cols <= 16 ? 16 : cols <= 32 ? 32 : cols <= 64 ? 64 : cols <= 128 ? 128 : 256;
  wpt::ScoreParams p;
  p.positions = positions;
  p.lse = lse;
  p.scores = scores;
  p.ld = ld_scores;
  if (int rc = status_word(&p.status)) return rc;
  p.B = B;
  p.T = T;
  p.H = H;
  p.N = N;
  p.window = window;
  p.TQ = ncol / H;
  if (p.TQ < 1) return fail(WPT_ERR_UNSUPPORTED, "%d heads exceed the selection kernel's columns", H);
  p.groups_per_row = (T + p.TQ - 1) / p.TQ;
  p.scale = scale;
  const int64_t groups = static_cast<int64_t>(B) * p.groups_per_row;
  // one query per group (decode) and few groups: the groups' live key tiles
  // split evenly over one CTA per SM, whatever the rows' lengths
  p.balanced = T == 1 && p.TQ == 1 && groups <= wpt::SCORE_BAL_GROUPS ? 1 : 0;
  const int tiles = (N + 127) / 128;
  int64_t chunk = (static_cast<int64_t>(tiles) * groups + 4 * 148 - 1) / (4 * 148);
  if (chunk < 4) chunk = 4;
  if (chunk > tiles) chunk = tiles;
  p.chunk_tiles = static_cast<int>(chunk);
  const int splits = (tiles + p.chunk_tiles - 1) / p.chunk_tiles;
  if (groups >= (int64_t(1) << 31) || splits > 65535) return fail(WPT_ERR_UNSUPPORTED, "selection grid too large");
  CUtensorMap tq, tk;
  {
    cuuint64_t dims[2] = {static_cast<cuuint64_t>(C), static_cast<cuuint64_t>(B) * T * H};
    cuuint64_t strides[1] = {static_cast<cuuint64_t>(C) * 2};
    cuuint32_t box[2] = {64, static_cast<cuuint32_t>(ncol)};
    if (int rc = tensor_map(&tq, q, 2, dims, strides, box)) return rc;
  }
  if (int rc = table_map(&tk, k, k_stride_b, k_stride_n, B, N, C)) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int rc;
  switch (ncol) {
    case 16: rc = launch_score<16>(tq, tk, p, static_cast<int>(groups), splits, s); break;
    case 32: rc = launch_score<32>(tq, tk, p, static_cast<int>(groups), splits, s); break;
    case 64: rc = launch_score<64>(tq, tk, p, static_cast<int>(groups), splits, s); break;
    case 128: rc = launch_score<128>(tq, tk, p, static_cast<int>(groups), splits, s); break;
    default: rc = launch_score<256>(tq, tk, p, static_cast<int>(groups), splits, s); break;
  }
  if (rc) return rc;
  const int cap = N < 47104 ? N : 47104;  // keys cached in shared memory (the rest of it: bins, candidates)
  const int smem = (cap + 1 + wpt::SELECT_BINS + 2 * wpt::SELECT_CAND + 64) * 4;
  int sms = 148;
  current_device(&sms);
  const int64_t queries = static_cast<int64_t>(B) * T;
  // fewer queries than SMs: each query's candidates in two slices, a 2-CTA
  // cluster per query (WPT_B200_TOPK_PAIR=0 keeps one CTA)
  static const int pair_env = [] {
    const char* env = getenv("WPT_B200_TOPK_PAIR");
    return env ? atoi(env) : 1;
  }();
  const bool pair = pair_env != 0 && queries < sms;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // waits for the scores on the device
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pair ? 2 : 1;
  cfg.gridDim = dim3(static_cast<unsigned>(pair ? 2 * queries : queries));
  cfg.blockDim = dim3(wpt::TOPK_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaError_t e;
  if (pair) {
    if (int rc2 = allow_smem(wpt::topk_kernel<2>, smem)) return rc2;
    e = cudaLaunchKernelEx(&cfg, wpt::topk_kernel<2>, scores, ld_scores, positions, chosen, T, N, K, window, cap);
  } else {
    if (int rc2 = allow_smem(wpt::topk_kernel<1>, smem)) return rc2;
    e = cudaLaunchKernelEx(&cfg, wpt::topk_kernel<1>, scores, ld_scores, positions, chosen, T, N, K, window, cap);
  }
  if (e != cudaSuccess) return cuda_fail(e, "topk_kernel launch");
  return WPT_OK;
}

extern "C" int wpt_tree_bits(const int64_t* parents, int64_t parents_stride_b, int B, int n, uint64_t* bits,
                             const int64_t* base, int64_t* positions, void* stream) {
  if (B < 1 || n < 1) return fail(WPT_ERR_INVALID, "empty tree batch B=%d n=%d", B, n);
  if (n > 64) return fail(WPT_ERR_UNSUPPORTED, "a tree of %d nodes: the kernels take up to 64", n);
  if (!parents || !bits || (positions && !base)) return fail(WPT_ERR_INVALID, "a required pointer is NULL");
  if (parents_stride_b != 0 && parents_stride_b < n)
    return fail(WPT_ERR_INVALID, "parents_stride_b must be 0 (one tree for every row) or at least n");
  const int64_t total = static_cast<int64_t>(B) * n;
  const int64_t blocks = (total + 255) / 256;
  if (blocks >= (int64_t(1) << 31)) return fail(WPT_ERR_UNSUPPORTED, "too many tree rows");
  wpt::tree_bits_kernel<<<static_cast<unsigned>(blocks), 256, 0, static_cast<cudaStream_t>(stream)>>>(
      parents, parents_stride_b, B, n, bits, base, positions);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "tree_bits_kernel launch");
  return WPT_OK;
}

extern "C" int wpt_cache_append(const void* src, int64_t src_stride_b, int64_t src_stride_n, void* dst,
                                int64_t dst_stride_b, int64_t dst_stride_n, const int64_t* first,
                                const int64_t* counts, int B, int n, int row_bytes, int64_t capacity, void* stream) {
  if (B < 0 || n < 0 || row_bytes < 0 || capacity < 0) return fail(WPT_ERR_INVALID, "bad cache_append shape");
  if (B == 0 || n == 0 || row_bytes == 0) return WPT_OK;
  if (!src || !dst || !first || !counts) return fail(WPT_ERR_INVALID, "a required pointer is NULL");
  if (row_bytes % 16 || src_stride_b % 16 || src_stride_n % 16 || dst_stride_b % 16 || dst_stride_n % 16 ||
      !aligned16(src) || !aligned16(dst))
    return fail(WPT_ERR_INVALID, "cache_append copies 16-byte units: rows, strides and bases must be 16-byte multiples");
  unsigned* status = nullptr;
  if (int rc = status_word(&status)) return rc;
  const int64_t warps = static_cast<int64_t>(B) * n;
  const int64_t blocks = (warps + 7) / 8;
  if (blocks >= (int64_t(1) << 31)) return fail(WPT_ERR_UNSUPPORTED, "too many rows to append");
  wpt::cache_append_kernel<<<static_cast<unsigned>(blocks), 256, 0, static_cast<cudaStream_t>(stream)>>>(
      static_cast<const uint8_t*>(src), src_stride_b, src_stride_n, static_cast<uint8_t*>(dst), dst_stride_b,
      dst_stride_n, first, counts, B, n, row_bytes, capacity, status);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "cache_append_kernel launch");
  return WPT_OK;
}

extern "C" int wpt_temperature_scale(const float* x, int64_t n, float temperature, float* out, void* stream) {
  if (n < 0 || (n > 0 && (!x || !out))) return fail(WPT_ERR_INVALID, "bad temperature_scale arguments");
  if (!(temperature > 0.f)) return fail(WPT_ERR_INVALID, "temperature must be positive");
  if (n == 0) return WPT_OK;
  int sms = 148;
  current_device(&sms);
  const int64_t want = (n + 255) / 256;
  const int blocks = static_cast<int>(std::min<int64_t>(want, static_cast<int64_t>(sms) * 8));
  wpt::temperature_scale_kernel<<<blocks, 256, 0, static_cast<cudaStream_t>(stream)>>>(x, n, temperature, out);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "temperature_scale_kernel launch");
  return WPT_OK;
}

extern "C" size_t wpt_accept_scratch_bytes(int R, int n, int V) {
  if (R < 0 || n < 0 || V < 1) return 0;
  return wpt::accept_scratch(R, n, V).bytes;
}

namespace {
template <int N>
int launch_head(const CUtensorMap& tw, const CUtensorMap& th, const wpt::HeadParams& p, cudaStream_t stream) {
  using L = wpt::HeadLayout<N>;
  static_assert(L::BYTES <= 232448, "head kernel shared memory exceeds 227 KB");
  auto kernel = wpt::head_kernel<N>;
  if (int rc = allow_smem(kernel, L::BYTES)) return rc;
  int sms = 148;
  current_device(&sms);
  const int grid = p.tiles < sms ? p.tiles : sms;  // persistent: one CTA per SM walks the vocabulary tiles
  kernel<<<grid, wpt::HEAD_THREADS, L::BYTES, stream>>>(tw, th, p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "head_kernel launch");
  return WPT_OK;
}
}  // namespace

extern "C" int wpt_head_scores(const void* h, int64_t h_stride, const void* w, int64_t w_stride, int R, int D,
                               int V, int round_bf16, float* scores, void* stream) {
  if (R < 1 || D < 1 || V < 1) return fail(WPT_ERR_INVALID, "empty shape R=%d D=%d V=%d", R, D, V);
  if (D % 64 != 0) return fail(WPT_ERR_UNSUPPORTED, "model width %d: the head kernel takes multiples of 64", D);
  if (!h || !w || !scores) return fail(WPT_ERR_INVALID, "a required pointer is NULL");
  if (!aligned16(h) || !aligned16(w)) return fail(WPT_ERR_INVALID, "h and the head weight must be 16-byte aligned");
  if (h_stride < D || w_stride < D || h_stride % 8 || w_stride % 8)
    return fail(WPT_ERR_INVALID, "row strides must be at least D and multiples of 8 elements");
  if (static_cast<int64_t>(R) * V >= (int64_t(1) << 40)) return fail(WPT_ERR_UNSUPPORTED, "R*V too large");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int tiles = (V + 127) / 128;
  CUtensorMap tw;
  {
    cuuint64_t dims[2] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(V)};
    cuuint64_t strides[1] = {static_cast<cuuint64_t>(w_stride) * 2};
    cuuint32_t box[2] = {64, 128};
    if (int rc = tensor_map(&tw, w, 2, dims, strides, box)) return rc;
  }
  for (int r0 = 0; r0 < R; r0 += 128) {  // up to 128 rows of h per launch (the MMA's N)
    const int rows = R - r0 < 128 ? R - r0 : 128;
    const int n = rows <= 32 ? 32 : rows <= 64 ? 64 : 128;
    const void* hb = static_cast<const __nv_bfloat16*>(h) + static_cast<int64_t>(r0) * h_stride;
    CUtensorMap th;
    cuuint64_t dims[2] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(rows)};
    cuuint64_t strides[1] = {static_cast<cuuint64_t>(h_stride) * 2};
    cuuint32_t box[2] = {64, static_cast<cuuint32_t>(n)};
    if (int rc = tensor_map(&th, hb, 2, dims, strides, box)) return rc;
    wpt::HeadParams p;
    p.scores = scores + static_cast<int64_t>(r0) * V;
    if (int rc = status_word(&p.status)) return rc;
    p.R = rows;
    p.V = V;
    p.D = D;
    p.tiles = tiles;
    p.round_bf16 = round_bf16 ? 1 : 0;
    const int rc = n == 32 ? launch_head<32>(tw, th, p, s) : n == 64 ? launch_head<64>(tw, th, p, s)
                                                                     : launch_head<128>(tw, th, p, s);
    if (rc) return rc;
  }
  return WPT_OK;
}

extern "C" int wpt_accept(const float* scores, const int64_t* drafted, const float* q, const float* uniforms,
                          const float* resample, const int64_t* lengths, void* scratch, int64_t* tokens,
                          int64_t* accepted, int R, int n, int V, float temperature, int top_k, void* stream) {
  if (R < 0 || n < 0 || V < 1) return fail(WPT_ERR_INVALID, "bad accept shape R=%d n=%d V=%d", R, n, V);
  if (R == 0) return WPT_OK;
  if (R > 65535 || n + 1 > 65535) return fail(WPT_ERR_UNSUPPORTED, "accept grid too large (R=%d, n=%d)", R, n);
  if (!(temperature > 0.f)) return fail(WPT_ERR_INVALID, "temperature must be positive");
  if (!scores || !scratch || !tokens || !accepted || !resample || (n > 0 && (!drafted || !q || !uniforms)))
    return fail(WPT_ERR_INVALID, "a required pointer is NULL");
  if (reinterpret_cast<uintptr_t>(scratch) % 16 != 0) return fail(WPT_ERR_INVALID, "accept scratch not 16-byte aligned");
  const wpt::AcceptScratch layout = wpt::accept_scratch(R, n, V);
  char* base = static_cast<char*>(scratch);
  wpt::AcceptParams p;
  p.scores = scores;
  p.drafted = drafted;
  p.q = q;
  p.uniforms = uniforms;
  p.resample = resample;
  p.lengths = lengths;
  p.part = reinterpret_cast<float2*>(base + layout.part);
  p.pos_stat = reinterpret_cast<float2*>(base + layout.pos_stat);
  p.thr = reinterpret_cast<float*>(base + layout.thr);
  p.keep = reinterpret_cast<int*>(base + layout.keep);
  p.chunk_sum = reinterpret_cast<double*>(base + layout.chunk_sum);
  p.pos_count = reinterpret_cast<unsigned*>(base + layout.pos_count);
  p.count = reinterpret_cast<unsigned*>(base + layout.count);
  p.ticket = reinterpret_cast<unsigned long long*>(base + layout.ticket);
  p.tokens = tokens;
  p.accepted = accepted;
  p.R = R;
  p.n = n;
  p.V = V;
  p.top_k = top_k;
  p.S = (V + wpt::STAT_SEG - 1) / wpt::STAT_SEG;
  p.chunks = (V + wpt::DRAW_CHUNK - 1) / wpt::DRAW_CHUNK;
  p.temperature = temperature;
  const int slices = (p.chunks + wpt::DRAW_CPS - 1) / wpt::DRAW_CPS;
  if (slices > 65535) return fail(WPT_ERR_UNSUPPORTED, "vocabulary of %d entries is too large", V);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // the arrival counters (positions', rows') and the unit ticket start at zero
  cudaError_t e = cudaMemsetAsync(base + layout.pos_count, 0, layout.bytes - layout.pos_count, s);
  if (e != cudaSuccess) return cuda_fail(e, "cudaMemsetAsync(accept counters)");
  if (top_k > 1 && top_k < V) {
    wpt::accept_topk_stats_kernel<<<dim3(n + 1, R), wpt::ACCEPT_THREADS, 0, s>>>(p);
    e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_fail(e, "accept_topk_stats_kernel launch");
  } else {
    // a grid the SMs hold at once: its warps take the units in turn
    const bool greedy = top_k == 1 && V > 1;
    const int variant = (greedy ? 2 : 0) + (temperature == 1.f ? 1 : 0);
    void (*const kernels[4])(const wpt::AcceptParams) = {
        wpt::accept_stats_kernel<false, false>, wpt::accept_stats_kernel<false, true>,
        wpt::accept_stats_kernel<true, false>, wpt::accept_stats_kernel<true, true>};
    auto kernel = kernels[variant];
    static int resident[4][64] = {};
    int sms = 148;
    const int dev = current_device(&sms);
    if (resident[variant][dev] == 0) {
      int per_sm = 0;
      e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, wpt::STAT_THREADS, 0);
      if (e != cudaSuccess) return cuda_fail(e, "cudaOccupancyMaxActiveBlocksPerMultiprocessor");
      resident[variant][dev] = per_sm > 0 ? per_sm : 1;
    }
    const int64_t units = static_cast<int64_t>(R) * (n + 1) * p.S;
    const int64_t want = (units + wpt::STAT_THREADS / 32 - 1) / (wpt::STAT_THREADS / 32);
    const int blocks = static_cast<int>(
        std::max<int64_t>(1, std::min<int64_t>(want, static_cast<int64_t>(sms) * resident[variant][dev])));
    kernel<<<blocks, wpt::STAT_THREADS, 0, s>>>(p);
    e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_fail(e, "accept_stats_kernel launch");
  }
  // the draw launches while the statistics finish (programmatic dependent
  // launch) and waits for them on the device
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(R, slices);
  cfg.blockDim = dim3(wpt::DRAW_THREADS);
  cfg.dynamicSmemBytes = 0;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, wpt::accept_draw_kernel, p);
  if (e != cudaSuccess) return cuda_fail(e, "accept_draw_kernel launch");
  return WPT_OK;
}

// ---------------------------------------------------------------- no-alloc
// Scratch of wpt_attn_decode_noalloc: the per-split partial outputs and
// log-sum-exps live in this file-scope device array instead of buffers the
// caller allocates. Every GPU that loads the library holds these 8 MiB
// until the process exits. In host code the array's name is only a
// host-side stand-in: its device address comes from cudaGetSymbolAddress,
// once per device, with that device current.
constexpr size_t WPT_NOALLOC_SCRATCH_FLOATS = size_t(1) << 21;  // 8 MiB of fp32
static __device__ __align__(256) float g_noalloc_scratch[WPT_NOALLOC_SCRATCH_FLOATS];

namespace {

int noalloc_scratch(float** out) {
  static float* cached[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  if (dev < 0 || dev >= 64) return fail(WPT_ERR_INVALID, "device %d out of range", dev);
  std::lock_guard<std::mutex> guard(g_symbol_lock);
  if (cached[dev] == nullptr) {
    void* p = nullptr;
    e = cudaGetSymbolAddress(&p, g_noalloc_scratch);
    if (e != cudaSuccess) return cuda_fail(e, "cudaGetSymbolAddress(no-alloc scratch)");
    cached[dev] = static_cast<float*>(p);
  }
  *out = cached[dev];
  return WPT_OK;
}

}  // namespace

extern "C" int wpt_attn_decode_noalloc(const void* q, const void* k, const void* v, int64_t k_stride_b,
                                       int64_t k_stride_n, int64_t v_stride_b, int64_t v_stride_n,
                                       const int64_t* positions, const int64_t* floor_rows, const int64_t* idx,
                                       int K, const float* sink, void* out, float* lse, int splits, int chunk_tiles,
                                       int B, int T, int H, int C, int N, int window, float scale, void* stream) {
  // The partials live in the library's private array, where the caller
  // cannot read them: the partials-only mode of wpt_attn_decode
  // (out == lse == NULL) would compute nothing the caller can see.
  if (out == nullptr || lse == nullptr)
    return fail(WPT_ERR_INVALID, "no-alloc decode: out and lse are required (its partials are not readable)");
  if (C != 128) return fail(WPT_ERR_UNSUPPORTED, "head width %d: the key-stream kernel takes 128", C);
  if (H < 1 || H > 64) return fail(WPT_ERR_UNSUPPORTED, "%d heads: the key-stream kernel takes 1 to 64", H);
  if (B < 1 || T < 1) return fail(WPT_ERR_INVALID, "empty shape B=%d T=%d", B, T);
  if (splits < 1) return fail(WPT_ERR_INVALID, "splits must be >= 1");
  if (splits > 65535) return fail(WPT_ERR_UNSUPPORTED, "%d splits: at most 65535", splits);
  const int64_t rows = static_cast<int64_t>(B) * T * H;
  if (rows >= (int64_t(1) << 31)) return fail(WPT_ERR_UNSUPPORTED, "B*T*H = %lld rows is too many",
                                              static_cast<long long>(rows));
  float* part_o = nullptr;
  float* part_lse = nullptr;
  if (splits > 1) {
    // splits < 2^16 and rows < 2^31, so the product fits in 64 bits
    const int64_t need = static_cast<int64_t>(splits) * rows * (C + 1);
    if (need > static_cast<int64_t>(WPT_NOALLOC_SCRATCH_FLOATS))
      return fail(WPT_ERR_UNSUPPORTED,
                  "no-alloc decode: %d splits x %lld rows x (%d + 1) floats = %lld floats exceed the %lld-float "
                  "(8 MiB) static scratch; use fewer splits or rows, or wpt_attn_decode with caller buffers",
                  splits, static_cast<long long>(rows), C, static_cast<long long>(need),
                  static_cast<long long>(WPT_NOALLOC_SCRATCH_FLOATS));
    float* scratch = nullptr;
    if (int rc = noalloc_scratch(&scratch)) return rc;
    part_o = scratch;                                   // (splits, rows, C), 256-byte aligned
    part_lse = scratch + static_cast<int64_t>(splits) * rows * C;  // (splits, rows)
  }
  return wpt_attn_decode(q, k, v, k_stride_b, k_stride_n, v_stride_b, v_stride_n, positions, floor_rows, idx, K, sink,
                         out, lse, part_o, part_lse, splits, chunk_tiles, B, T, H, C, N, window, scale, stream);
}

// ----------------------------------------- the cache between two decode steps

namespace {

// A launch as a programmatic dependent of the kernel before it on the stream
// (every kernel launched so waits for it on the device before its first
// global access), with a cluster of `cluster` CTAs when that is above 1.
template <typename Kernel, typename... Args>
int launch_dependent(const char* what, Kernel kernel, int64_t grid, int threads, int smem, int cluster,
                     cudaStream_t stream, const Args&... args) {
  if (grid >= (int64_t(1) << 31)) return fail(WPT_ERR_UNSUPPORTED, "%s: too large a grid", what);
  if (smem > 0)
    if (int rc = allow_smem(kernel, smem)) return rc;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e != cudaSuccess) return cuda_fail(e, what);
  return WPT_OK;
}

// The query-stream form's cut, and its scratch in bytes from its start.
struct WeightsPlan {
  int tiles, groups, key_blocks, chunks, chunk_tiles;
  int64_t meta, cols, partial, ticket, bytes;
};

WeightsPlan weights_plan(int64_t B, int64_t T, int64_t H, int64_t N) {
  WeightsPlan w = {};
  const int64_t cols = T * H, sms = 148;
  if (cols <= 256) return w;  // the key-stream form needs none
  w.tiles = static_cast<int>((cols + wpt::WEIGHTS_TILE_COLS - 1) / wpt::WEIGHTS_TILE_COLS);
  // Items of 1 or 2 key tiles where one wave of them (of 4 column tiles each)
  // covers the call: 5 rows of 6,007 keys of width 64 and 444 columns take 13.3
  // us with 2, 19.1 with 1 (two waves), 16.0 with 4 (60 SMs). Else 4, so that
  // four warpgroups share the exponential unit: 2,000 keys of 32 rows and 1,024
  // columns take 34.6 us with 4, 38.7 with 2, 53.5 with 1.
  auto blocks = [&](int64_t groups) { return (N + 128 * groups - 1) / (128 * groups); };
  w.groups = 1;
  while (w.groups < wpt::WEIGHTS_TILE_GROUPS && B * blocks(w.groups) * ((w.tiles + 3) / 4) > sms) w.groups *= 2;
  w.key_blocks = static_cast<int>(blocks(w.groups));
  // runs of 16 column tiles, shorter ones (not under 4) to four items an SM
  int64_t per = 16;
  while (per > 4 && B * w.key_blocks * ((w.tiles + per - 1) / per) < 4 * sms) per /= 2;
  // Longer ones where there are more than 64 a key and eight items an SM are left:
  // each run leaves a sum a key, B N T H / 512 bytes with runs of 16 (1 GB for a row
  // of 131,072 places of 32 heads), so at most 256 bytes a key or 5 MB in all. A row
  // of 32,768 places takes 4.9 to 5.1 ms either way.
  while ((w.tiles + per - 1) / per > 64 && B * w.key_blocks * ((w.tiles + 2 * per - 1) / (2 * per)) >= 8 * sms) per *= 2;
  w.chunk_tiles = static_cast<int>(per < w.tiles ? per : w.tiles);
  w.chunks = (w.tiles + w.chunk_tiles - 1) / w.chunk_tiles;
  int64_t at = 0;
  const int64_t n = B * w.tiles;
  w.meta = at, at += n * 16;
  w.cols = at, at += n * wpt::WEIGHTS_TILE_COLS * 12;
  w.partial = at, at += w.chunks > 1 ? (w.chunks * B * N * 4 + 15) / 16 * 16 : 0;
  w.ticket = at, at += 16;
  w.bytes = at;
  return w;
}

template <int C, int NCOL, int STAGES>
int launch_weights_stream(const CUtensorMap& tq, const CUtensorMap& tk, const wpt::WeightsParams& p,
                          cudaStream_t stream) {
  using L = wpt::WeightsStreamLayout<C, NCOL, STAGES>;
  static_assert(L::BYTES <= 232448, "attention-weight kernel shared memory exceeds 227 KB");
  int sms = 148;
  current_device(&sms);
  return launch_dependent("weights_stream_kernel launch", wpt::weights_stream_kernel<C, NCOL, STAGES>, sms,
                          wpt::WEIGHTS_STREAM_THREADS, L::BYTES, 1, stream, tq, tk, p);
}

template <int C>
int weights_call(const void* q, const CUtensorMap& tk, const wpt::WeightsParams& p, uint8_t* scratch,
                 cudaStream_t stream) {
  const int64_t cols = static_cast<int64_t>(p.T) * p.H;
  const bool few = cols <= 256;
  const int ncol = !few ? 128 : cols <= 16 ? 16 : cols <= 32 ? 32 : cols <= 64 ? 64 : cols <= 128 ? 128 : 256;
  CUtensorMap tq;
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(C), static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(p.B)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(C) * 2, static_cast<cuuint64_t>(cols) * C * 2};
  cuuint32_t box[3] = {64, static_cast<cuuint32_t>(ncol), 1};
  if (int rc = tensor_map(&tq, q, 3, dims, strides, box)) return rc;
  if (few) {
    switch (ncol) {
      case 16: return launch_weights_stream<C, 16, 6>(tq, tk, p, stream);
      case 32: return launch_weights_stream<C, 32, 6>(tq, tk, p, stream);
      case 64: return launch_weights_stream<C, 64, 5>(tq, tk, p, stream);
      case 128: return launch_weights_stream<C, 128, 4>(tq, tk, p, stream);
      default: return launch_weights_stream<C, 256, 2>(tq, tk, p, stream);
    }
  }
  const WeightsPlan w = weights_plan(p.B, p.T, p.H, p.N);
  using L = wpt::WeightsTileLayout<C>;
  static_assert(L::BYTES <= 232448, "attention-weight kernel shared memory exceeds 227 KB");
  wpt::WeightsTileParams t;
  t.weights = p.weights;
  t.weights_ld = p.weights_ld;
  int4* meta = reinterpret_cast<int4*>(scratch + w.meta);
  float* columns = reinterpret_cast<float*>(scratch + w.cols);
  t.meta = meta;
  t.cols = columns;
  t.partial = reinterpret_cast<float*>(scratch + w.partial);
  t.ticket = reinterpret_cast<unsigned*>(scratch + w.ticket);
  t.status = p.status;
  t.B = p.B;
  t.N = p.N;
  t.tiles = w.tiles;
  t.groups = w.groups;
  t.key_blocks = w.key_blocks;
  t.chunks = w.chunks;
  t.chunk_tiles = w.chunk_tiles;
  t.scale_log2 = p.scale_log2;
  const int64_t items = static_cast<int64_t>(p.B) * w.key_blocks * w.chunks;
  if (items >= (int64_t(1) << 30)) return fail(WPT_ERR_UNSUPPORTED, "attention weights: too many keys and queries");
  t.items = static_cast<int>(items);
  if (int rc = launch_dependent("weights_prep_kernel launch", wpt::weights_prep_kernel,
                                static_cast<int64_t>(p.B) * w.tiles, wpt::WEIGHTS_TILE_COLS, 0, 1, stream, p, w.tiles,
                                meta, columns, t.ticket))
    return rc;
  int sms = 148;
  current_device(&sms);
  if (int rc = launch_dependent("weights_tile_kernel launch", wpt::weights_tile_kernel<C>, std::min<int64_t>(items, sms),
                                wpt::WEIGHTS_TILE_THREADS, L::BYTES, 1, stream, tq, tk, t))
    return rc;
  if (w.chunks == 1) return WPT_OK;
  return launch_dependent("weights_reduce_kernel launch", wpt::weights_reduce_kernel,
                          (static_cast<int64_t>(p.B) * p.N + 255) / 256, 256, 0, 1, stream,
                          static_cast<const float*>(t.partial), p.weights, p.weights_ld, w.chunks, p.B, p.N);
}

}  // namespace

extern "C" size_t wpt_attn_weights_scratch_bytes(int B, int T, int H, int N) {
  if (B < 1 || T < 1 || H < 1 || N < 1 || static_cast<int64_t>(T) * H >= (int64_t(1) << 31)) return 0;
  return static_cast<size_t>(weights_plan(B, T, H, N).bytes);
}

extern "C" int wpt_attn_weights(const void* q, const void* k, int64_t k_stride_b, int64_t k_stride_n,
                                const int64_t* positions, const int64_t* floor, const float* lse, float* weights,
                                int64_t weights_ld, void* scratch, int B, int T, int H, int C, int N, int window,
                                float scale, void* stream) {
  if (C != 64 && C != 128)
    return fail(WPT_ERR_UNSUPPORTED, "head width %d: the attention-weight kernels take 64 and 128", C);
  if (B < 0 || T < 0 || H < 1 || N < 0 || window < 0)
    return fail(WPT_ERR_INVALID, "bad shape B=%d T=%d H=%d N=%d window=%d", B, T, H, N, window);
  if (B == 0 || T == 0 || N == 0) return WPT_OK;
  if (static_cast<int64_t>(T) * H >= (int64_t(1) << 31) || B >= (1 << 24) || N > INT_MAX - 512)
    return fail(WPT_ERR_UNSUPPORTED, "attention weights: shape too large");
  if (static_cast<int64_t>(B) * ((static_cast<int64_t>(T) * H + 127) / 128) >= (int64_t(1) << 31))
    return fail(WPT_ERR_UNSUPPORTED, "attention weights: B*T*H too large");
  if (!q || !k || !positions || !lse || !weights) return fail(WPT_ERR_INVALID, "a required pointer is NULL");
  if (weights_ld < N && B > 1) return fail(WPT_ERR_INVALID, "the weights' row stride is under N");
  if (!aligned16(q)) return fail(WPT_ERR_INVALID, "q must be 16-byte aligned");
  if (static_cast<int64_t>(T) * H > 256 && (!scratch || !aligned16(scratch)))
    return fail(WPT_ERR_INVALID, "attention weights: scratch is missing or not 16-byte aligned");
  CUtensorMap tk;
  if (int rc = table_map(&tk, k, k_stride_b, k_stride_n, B, N, C)) return rc;
  wpt::WeightsParams p;
  p.positions = positions;
  p.floor = floor;
  p.lse = lse;
  p.weights = weights;
  p.weights_ld = weights_ld;
  if (int rc = status_word(&p.status)) return rc;
  p.B = B;
  p.T = T;
  p.H = H;
  p.N = N;
  p.window = window;
  p.scale_log2 = scale * wpt::LOG2E;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  uint8_t* at = static_cast<uint8_t*>(scratch);
  return C == 64 ? weights_call<64>(q, tk, p, at, s) : weights_call<128>(q, tk, p, at, s);
}

extern "C" int wpt_cache_evict(const void* held, int64_t held_stride_b, int64_t held_stride_n, const float* weights,
                               int64_t weights_ld, const int64_t* lengths, void* kept, float* kept_weights,
                               int64_t* rows, int64_t* counts, int B, int N, int row_bytes, int keep, int recent,
                               int first, int capacity, void* stream) {
  if (B < 0 || N < 0 || row_bytes < 0 || keep < 0 || capacity < keep || recent < 0 || first < 0)
    return fail(WPT_ERR_INVALID, "bad eviction shape B=%d N=%d keep=%d recent=%d first=%d capacity=%d", B, N, keep,
                recent, first, capacity);
  if (static_cast<int64_t>(recent) + first > keep)
    return fail(WPT_ERR_INVALID, "%d first and %d recent rows do not fit in the %d kept", first, recent, keep);
  if (row_bytes % 4)
    return fail(WPT_ERR_UNSUPPORTED, "cache rows of %d bytes: the eviction kernel copies multiples of 4", row_bytes);
  if (N > INT_MAX - (1 << 20) || capacity > INT_MAX - (1 << 20))
    return fail(WPT_ERR_UNSUPPORTED, "eviction: table too long");
  if (B == 0) return WPT_OK;
  const bool copies = capacity > 0 && row_bytes > 0;
  if (!lengths || !counts || (N > 0 && !weights) || (keep > 0 && !rows) || (capacity > 0 && !kept_weights) ||
      (copies && (!kept || (N > 0 && !held))))
    return fail(WPT_ERR_INVALID, "a required pointer is NULL");
  if (weights_ld < N && B > 1) return fail(WPT_ERR_INVALID, "the weights' row stride is under N");
  const auto at = reinterpret_cast<uintptr_t>(held) | reinterpret_cast<uintptr_t>(kept) |
                  static_cast<uintptr_t>(held_stride_b) | static_cast<uintptr_t>(held_stride_n) |
                  static_cast<uintptr_t>(row_bytes);
  if (at % 4) return fail(WPT_ERR_INVALID, "cache tables and strides must be multiples of 4 bytes");
  int sms = 148;
  current_device(&sms);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  wpt::EvictParams p;
  p.weights = weights;
  p.weights_ld = weights_ld;
  p.lengths = lengths;
  p.rows = rows;
  p.weights_out = kept_weights;
  p.counts = counts;
  p.N = N;
  p.keep = keep;
  p.recent = recent;
  p.first = first;
  p.capacity = capacity;
  // One CTA a row up to 12,288 keys (7 rows of 10,007: 13.4 us with one, 14.5 with
  // two), then a cluster (1 row of 32,768: 24 us with one, 17.4 with two, 14.6 with
  // four), while the SMs are not all taken.
  p.slices = 1;
  while (p.slices < wpt::EVICT_SLICES && N > 12288 * p.slices && static_cast<int64_t>(B) * p.slices * 2 <= sms)
    p.slices *= 2;
  const int slice = (N / p.slices + wpt::EVICT_QUADS) / wpt::EVICT_QUADS * wpt::EVICT_QUADS;
  p.cache_cap = slice < 49152 ? slice : 49152;
  const bool wide = at % 16 == 0;
  wpt::GatherParams& g = p.gather;
  g.src = static_cast<const uint8_t*>(held);
  g.src_sb = held_stride_b;
  g.src_sn = held_stride_n;
  g.dst = static_cast<uint8_t*>(kept);
  g.rows = rows;
  g.keep = keep;
  g.capacity = capacity;
  g.units = row_bytes / (wide ? 16 : 4);
  g.chunks = p.slices;
  // A CTA that keeps up to 128 KB copies it itself, which saves a launch (a call
  // takes 15 us of the host instead of 17); on the device 64 KB take 8.2 us so, 7.0
  // with a kernel of their own for one row, 9.0 and 9.4 for 64 rows, 256 KB 13.6
  // and 8.0 for one row.
  const bool here = static_cast<int64_t>(capacity) * row_bytes <= 128 * 1024 * static_cast<int64_t>(p.slices);
  p.copy = !copies || !here ? 0 : wide ? 16 : 4;
  if (int rc = launch_dependent("evict_rows_kernel launch", wpt::evict_rows_kernel, static_cast<int64_t>(B) * p.slices,
                                wpt::EVICT_THREADS, p.cache_cap * 4, p.slices, s, p))
    return rc;
  if (!copies || here) return WPT_OK;
  // one wave of CTAs, no more than have a place for every group of threads
  const int groups = wpt::EVICT_COPY_THREADS / std::min(std::max(g.units, 1), wpt::EVICT_COPY_THREADS);
  const int64_t blocks = (static_cast<int64_t>(capacity) + groups - 1) / groups;
  g.chunks = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(blocks, int64_t(wpt::EVICT_COPY_CTAS) * sms / B)));
  if (wide)
    return launch_dependent("evict_gather_kernel launch", wpt::evict_gather_kernel<uint4>,
                            static_cast<int64_t>(B) * g.chunks, wpt::EVICT_COPY_THREADS, 0, 1, s, g);
  return launch_dependent("evict_gather_kernel launch", wpt::evict_gather_kernel<uint32_t>,
                          static_cast<int64_t>(B) * g.chunks, wpt::EVICT_COPY_THREADS, 0, 1, s, g);
}

namespace {
// Runs a beam's scores are cut into, and tiles a run: enough runs for two an SM
// (64 texts of 8 beams: whole beams 29.8 us, halves 30.6, quarters 32.0).
void beam_plan(int64_t R, int64_t W, int64_t V, bool bf16, int* splits, int* tiles) {
  constexpr int64_t sms = 148;  // whichever device the scratch is asked for on
  const int es = bf16 ? 2 : 4;
  const int64_t tile = wpt::BEAM_THREADS * 64 / es;
  const int64_t all = (V + 16 / es - 1 + tile - 1) / tile;  // a row may start off a 16-byte boundary
  int64_t want = (2 * sms + R * W - 1) / (R * W);
  if (want > all) want = all;
  if (want < 1) want = 1;
  *tiles = static_cast<int>((all + want - 1) / want);
  *splits = static_cast<int>((all + *tiles - 1) / *tiles);
}

template <typename T>
int launch_beam_scan(const wpt::BeamParams& p, cudaStream_t stream) {
  return launch_dependent("beam_scan_kernel launch", wpt::beam_scan_kernel<T>, static_cast<int64_t>(p.R) * p.W * p.splits,
                          wpt::BEAM_THREADS, wpt::BEAM_TILES_BYTES, 1, stream, p);
}
}  // namespace

extern "C" size_t wpt_beam_scratch_bytes(int R, int W, int V, int K, int bf16) {
  if (R < 1 || W < 1 || V < 1 || K < 1) return 0;
  int splits, tiles;
  beam_plan(R, W, V, bf16 != 0, &splits, &tiles);
  return static_cast<size_t>(R) * W * splits * (8 + 8 * (static_cast<size_t>(K) + 1));
}

extern "C" int wpt_beam_select(const void* scores, int bf16, int64_t stride_r, int64_t stride_w, const float* totals,
                               const uint8_t* done, int end, void* scratch, float* out_totals, int64_t* parents,
                               int64_t* tokens, int R, int W, int V, int K, void* stream) {
  if (R < 0 || W < 1 || V < 1 || K < 1) return fail(WPT_ERR_INVALID, "bad shape R=%d W=%d V=%d beams=%d", R, W, V, K);
  if (W > wpt::BEAM_MAX || K > wpt::BEAM_MAX)
    return fail(WPT_ERR_UNSUPPORTED, "%d beams in, %d out: the selection kernels take up to %d", W, K, wpt::BEAM_MAX);
  if (V > INT_MAX - (1 << 20) || static_cast<int64_t>(W) * V > UINT_MAX)
    return fail(WPT_ERR_UNSUPPORTED, "%d beams of %d scores are too many", W, V);
  if (R == 0) return WPT_OK;
  if (!scores || !totals || !scratch || !out_totals || !parents || !tokens)
    return fail(WPT_ERR_INVALID, "a required pointer is NULL");
  if (reinterpret_cast<uintptr_t>(scratch) & 7) return fail(WPT_ERR_INVALID, "scratch must be 8-byte aligned");
  if (done && (end < 0 || end >= V)) return fail(WPT_ERR_INVALID, "end token %d of a vocabulary of %d", end, V);
  if (reinterpret_cast<uintptr_t>(scores) & (bf16 ? 1 : 3)) return fail(WPT_ERR_INVALID, "scores are misaligned");
  wpt::BeamParams p;
  beam_plan(R, W, V, bf16 != 0, &p.splits, &p.tiles);
  p.scores = scores;
  p.stride_r = stride_r;
  p.stride_w = stride_w;
  p.totals = totals;
  p.done = done;
  p.stats = static_cast<float2*>(scratch);
  p.cand = reinterpret_cast<uint64_t*>(p.stats + static_cast<int64_t>(R) * W * p.splits);
  p.out_totals = out_totals;
  p.parents = parents;
  p.tokens = tokens;
  p.R = R;
  p.W = W;
  p.V = V;
  p.K = K;
  p.end = end;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (int rc = bf16 ? launch_beam_scan<__nv_bfloat16>(p, s) : launch_beam_scan<float>(p, s)) return rc;
  if (bf16)
    return launch_dependent("beam_merge_kernel launch", wpt::beam_merge_kernel<__nv_bfloat16>, R, wpt::BEAM_THREADS, 0, 1,
                            s, p);
  return launch_dependent("beam_merge_kernel launch", wpt::beam_merge_kernel<float>, R, wpt::BEAM_THREADS, 0, 1, s, p);
}

namespace {
template <typename Unit, int MAXW>
int launch_reorder(const wpt::ReorderParams& p, int tables, cudaStream_t stream) {
  return launch_dependent("reorder_kernel launch", wpt::reorder_kernel<Unit, MAXW>,
                          static_cast<int64_t>(tables) * p.R * p.chunks, wpt::REORDER_THREADS, 0, 1, stream, p);
}
}  // namespace

extern "C" int wpt_cache_reorder(const wpt_cache_table* tables, int count, const int64_t* parents,
                                 const int64_t* lengths, const int64_t* first, int R, int W, void* stream) {
  if (count < 0 || R < 0 || W < 1) return fail(WPT_ERR_INVALID, "bad reorder shape");
  if (W > wpt::BEAM_MAX)
    return fail(WPT_ERR_UNSUPPORTED, "%d beams: the reordering kernel takes up to %d", W, wpt::BEAM_MAX);
  if (count > wpt::REORDER_TABLES)
    return fail(WPT_ERR_UNSUPPORTED, "%d tables: a call takes up to %d", count, wpt::REORDER_TABLES);
  if (count == 0 || R == 0) return WPT_OK;
  if (!tables || !parents || !lengths) return fail(WPT_ERR_INVALID, "a required pointer is NULL");
  wpt::ReorderParams p;
  int64_t all = 0;
  for (int i = 0; i < count; ++i) {
    const wpt_cache_table& t = tables[i];
    if (t.row_bytes < 0 || t.row_bytes > INT_MAX || t.capacity < 0 || t.capacity > INT_MAX)
      return fail(WPT_ERR_INVALID, "bad table %d", i);
    if (t.row_bytes > 0 && t.capacity > 0 && !t.address) return fail(WPT_ERR_INVALID, "table %d is NULL", i);
    all |= t.address | t.stride_b | t.stride_n | t.row_bytes;
  }
  if (all % 4)
    return fail(WPT_ERR_UNSUPPORTED, "the reordering kernel moves units of 4 bytes: tables, strides and rows must be "
                                     "multiples of 4 bytes");
  if (int rc = status_word(&p.status)) return rc;
  // 16-byte units, one register quad a beam; above 32 beams, or for rows that
  // are not 16-byte multiples, 4-byte units
  const bool wide = all % 16 == 0 && W <= 32;
  int64_t most = 0;
  for (int i = 0; i < count; ++i) {
    const wpt_cache_table& t = tables[i];
    p.table[i].base = reinterpret_cast<uint8_t*>(t.address);
    p.table[i].stride_b = t.stride_b;
    p.table[i].stride_n = t.stride_n;
    p.table[i].units = static_cast<int>(t.row_bytes / (wide ? 16 : 4));
    p.table[i].capacity = static_cast<int>(t.capacity);
    most = std::max(most, t.capacity * p.table[i].units);
  }
  p.parents = parents;
  p.lengths = lengths;
  p.first = first;
  p.R = R;
  p.W = W;
  int sms = 148;
  current_device(&sms);
  const int64_t blocks = (most + wpt::REORDER_THREADS - 1) / wpt::REORDER_THREADS;
  const int64_t groups = static_cast<int64_t>(count) * R;
  p.chunks = static_cast<int>(std::max<int64_t>(1, std::min(blocks, (int64_t(8) * sms + groups - 1) / groups)));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (wide) {
    if (W <= 8) return launch_reorder<uint4, 8>(p, count, s);
    if (W <= 16) return launch_reorder<uint4, 16>(p, count, s);
    return launch_reorder<uint4, 32>(p, count, s);
  }
  if (W <= 16) return launch_reorder<uint32_t, 16>(p, count, s);
  return launch_reorder<uint32_t, 64>(p, count, s);
}

// --------------------------------------- rotary positions, the 8-bit paged cache

namespace {

// A launch as a programmatic dependent of the kernel before it on the stream
// (each of these kernels waits on the device before it touches memory).
template <class... Args>
cudaError_t launch_dependent(void (*kernel)(Args...), dim3 grid, int threads, int smem, int cluster_y,
                             cudaStream_t stream, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 1;
  attr[1].val.clusterDim.y = cluster_y;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster_y > 1 ? 2 : 1;
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Elements of a vector: `wide` (16 bytes), 2 or 1, the most of which turned and copied channels are whole vectors and
// x, its strides and y are multiples. (Vectors of 2 where whole ones do not fit: 88,000 heads of 232 bf16 channels, 52
// turned, 36 us against 60 one by one; 81 entries of 2 x 224, 46 turned, appended in 11 against 17.)
int rotary_elements(int wide, int C, int dims, int start, int interleaved, const void* x, int64_t strides,
                    const void* y) {
  const int64_t units = C | start | (interleaved ? dims : dims / 2) | strides;
  const uintptr_t at = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y);
  for (int ve : {wide, 2})
    if (units % ve == 0 && at % (16 / wide * ve) == 0) return ve;
  return 1;
}

int check_rotary(int C, int dims, int start, const void* frequencies) {
  if (dims < 0 || dims % 2 || start < 0 || static_cast<int64_t>(start) + dims > C)
    return fail(WPT_ERR_INVALID, "%d turned channels from %d on of %d", dims, start, C);
  if (dims > 0 && !frequencies) return fail(WPT_ERR_INVALID, "a required pointer is NULL");
  return WPT_OK;
}

template <class T, int VE, bool INTERLEAVED>
auto rotate_kernel_for(int copies) {
  void (*kernel)(wpt::RotateParams) = wpt::rotate_kernel<T, VE, INTERLEAVED, -1>;
  if constexpr (VE > 2) {
    if (copies == 0) kernel = wpt::rotate_kernel<T, VE, INTERLEAVED, 0>;
    if (copies == 1) kernel = wpt::rotate_kernel<T, VE, INTERLEAVED, 1>;
    if (copies == 2) kernel = wpt::rotate_kernel<T, VE, INTERLEAVED, 2>;
  }
  return kernel;
}
template <class T, int VE>
cudaError_t launch_rotate(const wpt::RotateParams& p, int interleaved, int copies, int64_t blocks, cudaStream_t s) {
  const auto kernel = interleaved ? rotate_kernel_for<T, VE, true>(copies) : rotate_kernel_for<T, VE, false>(copies);
  const int smem = p.dims / 2 * 8;
  if (smem > 48 * 1024 && allow_smem(kernel, smem) != WPT_OK) return cudaErrorInvalidValue;
  return launch_dependent(kernel, dim3(static_cast<unsigned>(blocks)), 256, smem, 1, s, p);
}

template <class T, int VE>
int launch_append(const wpt::AppendParams& p, int interleaved, unsigned blocks, cudaStream_t s) {
  // A warp's lanes cover a key's vectors: the entries stay in registers, half a warp's at a time or one by one, else in
  // shared memory (16 rows of 4,096 fp32 entries of 2 x 128, 64 turned, 22 us against 38; bf16 of 2 x 256 35 against 76).
  const int rows = VE <= 2 || p.vecs > 32 ? 0 : p.vecs <= 16 ? 2 : 4;
  void (*kernel)(wpt::AppendParams) = interleaved ? wpt::paged_append_kernel<T, VE, true, 0>
                                                  : wpt::paged_append_kernel<T, VE, false, 0>;
  if constexpr (VE > 2) {
    if (rows == 2) kernel = interleaved ? wpt::paged_append_kernel<T, VE, true, 2> : wpt::paged_append_kernel<T, VE, false, 2>;
    if (rows == 4) kernel = interleaved ? wpt::paged_append_kernel<T, VE, true, 4> : wpt::paged_append_kernel<T, VE, false, 4>;
  }
  const int smem = wpt::PAGE_BLOCK * (rows ? 0 : 2 * p.C * 4) + wpt::PAGE_BLOCK * p.dims / 2 * 8;
  if (int rc = allow_smem(kernel, smem)) return rc;
  cudaError_t e = launch_dependent(kernel, dim3(blocks), wpt::APPEND_THREADS, smem, 1, s, p);
  if (e != cudaSuccess) return cuda_fail(e, "paged_append_kernel launch");
  return WPT_OK;
}

template <int NCOL>
int launch_paged(const CUtensorMap& tm, const wpt::PagedParams& p, int ctas, cudaStream_t s) {
  using L = wpt::PagedLayout<NCOL>;
  static_assert(L::BYTES <= 115712, "paged attention kernel: too much shared memory");
  auto kernel = wpt::paged_kernel<NCOL>;
  if (int rc = allow_smem(kernel, L::BYTES)) return rc;
  // its register split draws on what the block was launched with: fewer would leave the increase waiting
  static std::atomic<int> regs{0};
  if (regs.load(std::memory_order_relaxed) == 0) {
    cudaFuncAttributes fa;
    cudaError_t e = cudaFuncGetAttributes(&fa, kernel);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncGetAttributes(paged_kernel)");
    regs.store(fa.numRegs, std::memory_order_relaxed);
  }
  if (regs.load(std::memory_order_relaxed) != wpt::PAGED_REGS)
    return fail(WPT_ERR_CUDA, "paged_kernel built with %d registers a thread, its register split needs %d",
                regs.load(std::memory_order_relaxed), wpt::PAGED_REGS);
  const dim3 grid = p.splits == 0 ? dim3(ctas) : dim3(p.groups, p.splits);
  cudaError_t e = launch_dependent(kernel, grid, wpt::PAGED_THREADS, L::BYTES, p.splits, s, tm, p);
  if (e != cudaSuccess) return cuda_fail(e, "paged_kernel launch");
  return WPT_OK;
}

// Columns of a group, its queries and its heads: more than 32 heads are shared out evenly over several groups a query.
struct PagedPlan {
  int ncol, TQ, HG, chunks;
  int64_t per_row;  // groups of a batch row
  PagedPlan(int T, int H) {
    ncol = static_cast<int64_t>(T) * H <= 16 ? 16 : 32;
    chunks = (H + 31) / 32;
    HG = (H + chunks - 1) / chunks;
    TQ = chunks > 1 ? 1 : ncol / H;
    per_row = (static_cast<int64_t>(T) + TQ - 1) / TQ * chunks;
  }
};

bool page_size_ok(int S) { return S == 16 || S == 32 || S == 64 || (S >= 128 && S % 128 == 0); }

}  // namespace

extern "C" int wpt_rotate(const void* x, int64_t x_stride_b, int64_t x_stride_t, int64_t x_stride_h,
                          const int64_t* positions, int64_t positions_stride_b, const void* frequencies,
                          int frequencies_f64, void* y, int f32, int B, int T, int H, int C, int dims, int start,
                          int interleaved, float magnitude, int inverse, void* stream) {
  if (B < 0 || T < 0 || H < 0 || C < 1) return fail(WPT_ERR_INVALID, "bad shape B=%d T=%d H=%d C=%d", B, T, H, C);
  if (int rc = check_rotary(C, dims, start, frequencies)) return rc;
  if (dims > 32768) return fail(WPT_ERR_UNSUPPORTED, "%d turned channels: up to 32768", dims);
  if (B == 0 || T == 0 || H == 0) return WPT_OK;
  if (!x || !y || !positions) return fail(WPT_ERR_INVALID, "a required pointer is NULL");
  wpt::RotateParams p;
  p.x = x;
  p.y = y;
  p.xsb = x_stride_b;
  p.xst = x_stride_t;
  p.xsh = x_stride_h;
  p.positions = positions;
  p.psb = positions_stride_b;
  p.frequencies = frequencies;
  p.f64 = frequencies_f64;
  p.T = T;
  p.H = H;
  p.C = C;
  p.dims = dims;
  p.start = start;
  p.sign = inverse ? -1.f : 1.f;
  p.magnitude = magnitude;
  const int wide = f32 ? 4 : 8;
  const int64_t strides = x_stride_b | x_stride_t | x_stride_h;
  const int ve = rotary_elements(wide, C, dims, start, interleaved, x, strides, y);
  const int turned = dims / 2 / (interleaved && ve > 1 ? ve / 2 : ve), rest = (C - dims) / ve;
  const int copies = ve == wide && turned > 0 && rest % turned == 0 && rest / turned <= 2 ? rest / turned : -1;
  p.items = copies < 0 ? turned + rest : turned;
  // a thread's angles serve up to 8 heads, fewer where that would leave SMs without threads
  int sms = 148;
  current_device(&sms);
  const int64_t tokens = static_cast<int64_t>(B) * T;
  int heads = 8;
  while (heads > 1 && tokens * p.items * ((H + heads - 1) / heads) < static_cast<int64_t>(sms) * 1024) heads /= 2;
  p.lanes = (H + heads - 1) / heads;
  p.total = tokens * p.items * p.lanes;
  const int64_t blocks = (p.total + 255) / 256;
  if (blocks >= (int64_t(1) << 31)) return fail(WPT_ERR_UNSUPPORTED, "too much to rotate in one call");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (f32)
    e = ve == 4   ? launch_rotate<float, 4>(p, interleaved, copies, blocks, s)
        : ve == 2 ? launch_rotate<float, 2>(p, interleaved, copies, blocks, s)
                  : launch_rotate<float, 1>(p, interleaved, copies, blocks, s);
  else
    e = ve == 8   ? launch_rotate<__nv_bfloat16, 8>(p, interleaved, copies, blocks, s)
        : ve == 2 ? launch_rotate<__nv_bfloat16, 2>(p, interleaved, copies, blocks, s)
                  : launch_rotate<__nv_bfloat16, 1>(p, interleaved, copies, blocks, s);
  if (e != cudaSuccess) return cuda_fail(e, "rotate_kernel launch");
  return WPT_OK;
}

extern "C" int wpt_paged_append(const void* src, int f32, int64_t src_stride_b, int64_t src_stride_n, void* pages,
                                int64_t page_stride, int64_t entry_stride, float* scales, int64_t scales_stride,
                                const void* table, int table_i64, int64_t table_stride_b, const int64_t* first,
                                const int64_t* counts, const int64_t* positions, const void* frequencies,
                                int frequencies_f64, int B, int n, int C, int M, int P, int S, int dims, int start,
                                int interleaved, float magnitude, void* stream) {
  if (B < 0 || n < 0 || M < 0 || P < 0 || C < 1) return fail(WPT_ERR_INVALID, "bad paged_append shape");
  if (C % 16 || C > 512) return fail(WPT_ERR_UNSUPPORTED, "entries of 2 x %d: the paged cache takes multiples of 16 up to 512", C);
  if (!page_size_ok(S)) return fail(WPT_ERR_UNSUPPORTED, "pages of %d entries: 16, 32, 64 or a multiple of 128", S);
  if (int rc = check_rotary(C, dims, start, frequencies)) return rc;
  if (B == 0 || n == 0 || M == 0 || P == 0) return WPT_OK;
  if (!src || !pages || !scales || !table || !first || !counts) return fail(WPT_ERR_INVALID, "a required pointer is NULL");
  if (static_cast<int64_t>(M) * S > INT_MAX - 1024) return fail(WPT_ERR_UNSUPPORTED, "a table of %d pages of %d entries", M, S);
  if (!aligned16(pages) || page_stride % 16 || entry_stride % 16 || entry_stride < 2 * C)
    return fail(WPT_ERR_INVALID, "pages and their strides must be multiples of 16 bytes");
  const int wide = f32 ? 4 : 8;
  const int ve = rotary_elements(wide, C, dims, start, interleaved, src, src_stride_b | src_stride_n, nullptr);
  wpt::AppendParams p;
  p.src = src;
  p.ssb = src_stride_b;
  p.ssn = src_stride_n;
  p.pages = static_cast<uint8_t*>(pages);
  p.psp = page_stride;
  p.psr = entry_stride;
  p.scales = scales;
  p.scp = scales_stride;
  p.table = table;
  p.tsb = table_stride_b;
  p.first = first;
  p.counts = counts;
  p.positions = positions;
  p.frequencies = frequencies;
  if (int rc = status_word(&p.status)) return rc;
  p.t64 = table_i64;
  p.f64 = frequencies_f64;
  p.B = B;
  p.n = n;
  p.C = C;
  p.M = M;
  p.P = P;
  p.S = S;
  p.dims = dims;
  p.start = start;
  p.magnitude = magnitude;
  p.vecs = C / ve;
  p.inv_vecs = 65536 / p.vecs + 1;
  p.turn_rows = dims > 0 ? wpt::APPEND_THREADS / (dims / 2) : 0;
  p.turn_pairs = dims > 0 ? wpt::APPEND_THREADS % (dims / 2) : 0;
  p.blocks = (n - 1) / wpt::PAGE_BLOCK + 2;  // n entries reach into that many blocks at most
  const int64_t blocks = static_cast<int64_t>(B) * p.blocks;
  if (blocks >= (int64_t(1) << 31)) return fail(WPT_ERR_UNSUPPORTED, "too many entries to append");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const unsigned grid = static_cast<unsigned>(blocks);
  if (f32)
    return ve == 4   ? launch_append<float, 4>(p, interleaved, grid, s)
           : ve == 2 ? launch_append<float, 2>(p, interleaved, grid, s)
                     : launch_append<float, 1>(p, interleaved, grid, s);
  return ve == 8   ? launch_append<__nv_bfloat16, 8>(p, interleaved, grid, s)
         : ve == 2 ? launch_append<__nv_bfloat16, 2>(p, interleaved, grid, s)
                   : launch_append<__nv_bfloat16, 1>(p, interleaved, grid, s);
}

extern "C" size_t wpt_paged_scratch_bytes(int B, int T, int H, int splits, int ctas) {
  if (B < 1 || T < 1 || H < 1 || H > 64 || splits != 0 || ctas < 1) return 0;
  const PagedPlan plan(T, H);
  const size_t groups = static_cast<size_t>(B) * plan.per_row;
  return (groups + ctas) * plan.ncol * (128 * 4 + 8) + groups * 8;
}

extern "C" int wpt_paged_attention(const void* q, const void* pages, int64_t page_stride, int64_t entry_stride,
                                   const float* scales, int64_t scales_stride, const void* table, int table_i64,
                                   int64_t table_stride_b, const int64_t* positions, const float* sink, void* out,
                                   float* lse, void* scratch, int splits, int ctas, int B, int T, int H, int C, int M, int P, int S, int window, float scale, void* stream) {
  if (C != 128) return fail(WPT_ERR_UNSUPPORTED, "head width %d: the paged attention kernel takes 128", C);
  if (H < 1 || H > 64) return fail(WPT_ERR_UNSUPPORTED, "%d heads: the paged attention kernel takes 1 to 64", H);
  if (!page_size_ok(S)) return fail(WPT_ERR_UNSUPPORTED, "pages of %d entries: 16, 32, 64 or a multiple of 128", S);
  if (B < 0 || T < 0 || M < 0 || P < 0 || window < 0) return fail(WPT_ERR_INVALID, "bad shape B=%d T=%d M=%d P=%d", B, T, M, P);
  if (B == 0 || T == 0) return WPT_OK;
  if (static_cast<int64_t>(M) * S > INT_MAX - 1024) return fail(WPT_ERR_UNSUPPORTED, "a table of %d pages of %d entries", M, S);
  if (static_cast<int64_t>(B) * T >= (int64_t(1) << 31) / H) return fail(WPT_ERR_UNSUPPORTED, "B*T*H too large");
  if (splits < 0 || splits > 8) return fail(WPT_ERR_INVALID, "%d splits: 1 to 8, or 0 for a balanced call", splits);
  if (!q || !positions || !out || !lse || (M > 0 && P > 0 && (!pages || !scales || !table)))
    return fail(WPT_ERR_INVALID, "a required pointer is NULL");
  if (!aligned16(q) || !aligned16(out) || (scratch && !aligned16(scratch)))
    return fail(WPT_ERR_INVALID, "q, out and scratch must be 16-byte aligned");
  const PagedPlan plan(T, H);
  const int ncol = plan.ncol;
  const int64_t groups = static_cast<int64_t>(B) * plan.per_row;
  if (splits == 0) {
    if (!scratch || ctas < 1) return fail(WPT_ERR_INVALID, "a balanced call needs scratch and CTAs");
    if (groups > wpt::PAGED_GROUPS || groups * ((static_cast<int64_t>(M) * S + 127) / 128 + wpt::PAGED_SEGMENT) >= (int64_t(1) << 31) ||
        ctas >= (1 << 16))
      return fail(WPT_ERR_UNSUPPORTED, "a balanced call takes up to %d query groups (got %lld) and 2^31 tiles",
                  wpt::PAGED_GROUPS, static_cast<long long>(groups));
  }
  CUtensorMap tm;
  memset(&tm, 0, sizeof(tm));
  if (M > 0 && P > 0) {
    if (!aligned16(pages) || page_stride % 16 || entry_stride % 16 || entry_stride < 2 * C)
      return fail(WPT_ERR_INVALID, "pages and their strides must be multiples of 16 bytes");
    const cuuint64_t dims[3] = {2 * 128, static_cast<cuuint64_t>(S), static_cast<cuuint64_t>(P)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(entry_stride),
                                   static_cast<cuuint64_t>(P > 1 ? page_stride : entry_stride * S)};
    const cuuint32_t box[3] = {128, static_cast<cuuint32_t>(S < 128 ? S : 128), 1};
    if (int rc = tensor_map(&tm, pages, 3, dims, strides, box, CU_TENSOR_MAP_DATA_TYPE_UINT8)) return rc;
  }
  wpt::PagedParams p;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.scales = scales;
  p.scp = scales_stride;
  p.table = table;
  p.tsb = table_stride_b;
  p.positions = positions;
  p.sink = sink;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.lse = lse;
  p.t64 = table_i64;
  if (int rc = status_word(&p.status)) return rc;
  p.B = B;
  p.T = T;
  p.H = H;
  p.M = P > 0 ? M : 0;  // no page: no row
  p.P = P;
  p.S = S;
  p.window = window;
  p.TQ = plan.TQ;
  p.HG = plan.HG;
  p.chunks = plan.chunks;
  p.groups_per_row = static_cast<int>(plan.per_row);
  p.groups = static_cast<int>(groups);
  p.splits = splits;
  p.scale_log2 = scale * wpt::LOG2E;
  const int64_t parts = splits == 0 ? groups + ctas : 0;
  p.part_o = static_cast<float*>(scratch);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + parts * ncol * 128);
  p.info = reinterpret_cast<int2*>(p.part_ml + parts * ncol);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int rc = ncol == 16 ? launch_paged<16>(tm, p, ctas, s) : launch_paged<32>(tm, p, ctas, s);
  if (rc || splits != 0) return rc;
  const int64_t rows = static_cast<int64_t>(B) * T * H;
  // parts of a group: about ctas / groups + 1
  const int spread = ctas <= 7 * groups ? 0 : ctas > 31 * groups && rows <= 256 ? 32 : 8;
  cudaError_t e = launch_dependent(spread == 0   ? wpt::paged_merge_kernel<0>
                                   : spread == 8 ? wpt::paged_merge_kernel<8>
                                                 : wpt::paged_merge_kernel<32>,
                                   dim3(static_cast<unsigned>(spread ? rows : (rows + 7) / 8)), spread ? spread * 32 : 256,
                                   0, 1, s, p, ncol);
  if (e != cudaSuccess) return cuda_fail(e, "paged_merge_kernel launch");
  return WPT_OK;
}
