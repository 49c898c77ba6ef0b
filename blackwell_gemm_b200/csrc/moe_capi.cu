// C-ABI launchers of the mixture-of-experts operators (include/b200_moe.h).
//
// Per call: check the arguments, encode the tensor maps, choose a kernel and
// launch it on the caller's stream.  Per device, once: shared-memory limits
// and the number of 2-CTA clusters that can be resident.
#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <mutex>

#include "b200_moe.h"
#include "device_state.h"
#include "grouped_gemm.cuh"
#include "moe_route.cuh"
#include "moe_stream.cuh"
#include "moe_w4.cuh"

using namespace b200;

namespace {

constexpr int kMaxDevices = 64;
// The kernels index an extent in 32 bits and may look a tile, a block's step or
// a block's chunk of tokens past its end.
constexpr int kMaxExtent = 0x7FFFFFFF - (1 << 25) + 1;

struct MoeDevice {
  bool ready = false;
  int init_status = B200_OK;
  int pairs[3] = {};  // resident clusters per GroupedMode
};

std::mutex g_mu;
MoeDevice g_moe[kMaxDevices];
std::atomic<int> g_kernel{0};

long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <class F>
bool set_smem(F* fn, int bytes) {
  return cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) ==
         cudaSuccess;
}

// dB: experts whose table fits beside six stages.
constexpr int kFewExperts = 128;

template <int kMode, bool kMany, class T>
bool init_pair(int sms, int* pairs) {
  using C = GroupedCfg<kMode, kMany>;
  constexpr int experts = kMode == kGroupedDB && !kMany ? kFewExperts : kMaxExperts;
  // (512 B: more than the kernel's static shared memory)
  static_assert(C::smem_bytes(experts) <= 227 * 1024 - 512, "shared memory of one CTA");
  auto* fn = grouped_pair_kernel<kMode, kMany, T>;
  if (!set_smem(fn, C::smem_bytes(experts))) return false;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * sms);
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = C::smem_bytes(experts);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, fn, &cfg) != cudaSuccess || n < 1) return false;
  if (*pairs == 0 || n < *pairs) *pairs = n;
  return true;
}

template <bool kDA, class T>
bool init_stream() {
  return set_smem(grouped_stream_kernel<kDA, 16, T>, StreamCfg<16>::smem_bytes(kMaxExperts)) &&
         set_smem(grouped_stream_kernel<kDA, 64, T>, StreamCfg<64>::smem_bytes(kMaxExperts));
}

template <int kGroup, class T>
constexpr bool kSplits = kFormat<T> == 1 && kGroup < 128;  // many rows: w4_split_kernel

template <int kGroup, bool kZeros, class T>
bool init_w4_one() {
  if constexpr (kSplits<kGroup, T>) {
    if (!set_smem(w4_split_kernel<64, kGroup, kZeros>,
                  W4SplitCfg<64, kGroup>::smem_bytes(kMaxExperts)) ||
        !set_smem(w4_split_kernel<128, kGroup, kZeros>,
                  W4SplitCfg<128, kGroup>::smem_bytes(kMaxExperts)))
      return false;
  } else {
    if (!set_smem(w4_stream_kernel<kGroup, kZeros, T>, W4Cfg<kGroup>::smem_bytes(kMaxExperts)) ||
        !set_smem(w4_wide_kernel<kGroup, kZeros, T>, W4WideCfg<kGroup>::smem_bytes(kMaxExperts)))
      return false;
  }
  if constexpr (kGroup < 128) {
    if (!set_smem(w4_rows_kernel<32, kGroup, kZeros, T>,
                  W4RowsCfg<32, kGroup>::smem_bytes(kMaxExperts)))
      return false;
  }
  return set_smem(w4_rows_kernel<8, kGroup, kZeros, T>,
                  W4RowsCfg<8, kGroup>::smem_bytes(kMaxExperts)) &&
         set_smem(w4_rows_kernel<16, kGroup, kZeros, T>,
                  W4RowsCfg<16, kGroup>::smem_bytes(kMaxExperts));
}

template <int kGroup, class T>
bool init_w4() {
  return init_w4_one<kGroup, false, T>() && init_w4_one<kGroup, true, T>();
}

template <class T>
bool init_type(MoeDevice& m, int sms) {
  return init_pair<kGroupedFwd, false, T>(sms, &m.pairs[0]) &&
         init_pair<kGroupedDA, false, T>(sms, &m.pairs[1]) &&
         init_pair<kGroupedDB, false, T>(sms, &m.pairs[2]) &&
         init_pair<kGroupedDB, true, T>(sms, &m.pairs[2]) && init_stream<false, T>() &&
         init_stream<true, T>() && init_w4<32, T>() && init_w4<64, T>() && init_w4<128, T>();
}

template <int kPer>
bool init_choose() {
  return set_smem(route_choose_kernel<kPer>, (1 + kRouteWarps) * kMaxExperts * (int)sizeof(int));
}

bool init_route() {
  return init_choose<1>() && init_choose<2>() && init_choose<4>() && init_choose<8>() &&
         init_choose<32>() &&
         set_smem(route_rank_kernel, (1 + kRouteWarps) * kMaxExperts * (int)sizeof(int));
}

int moe_device(DeviceView* v, MoeDevice** out) {
  const int st = device_view(v);
  if (st != B200_OK) return st;
  std::lock_guard<std::mutex> lock(g_mu);
  MoeDevice& m = g_moe[v->device];
  if (!m.ready) {
    m.ready = true;
    m.init_status =
        init_type<__nv_bfloat16>(m, v->sms) && init_type<__half>(m, v->sms) && init_route()
            ? B200_OK
            : B200_ERR_LAUNCH;
    if (m.init_status != B200_OK) cudaGetLastError();
  }
  if (m.init_status != B200_OK) return m.init_status;
  *out = &m;
  return B200_OK;
}

// Arrival counts of the streaming kernels: one array per (device, stream),
// made on the stream's first call; every launch leaves it at zero.  Null when
// none can be made, as for streams after the first 256 (the caller then clears
// counts of its own).
constexpr size_t kCountBytes = 4096 * sizeof(unsigned int);
struct StreamCounts {
  int device;
  unsigned long long stream;  // stream_id
  unsigned int* counts;
};
constexpr int kMaxStreamCounts = 256;
StreamCounts g_counts[kMaxStreamCounts];
int g_num_counts = 0;

unsigned int* stream_counts(const DeviceView& v, cudaStream_t stream) {
  unsigned long long id = 0;
  if (!stream_id(stream, &id)) return nullptr;
  std::lock_guard<std::mutex> lock(g_mu);
  for (int i = 0; i < g_num_counts; ++i)
    if (g_counts[i].device == v.device && g_counts[i].stream == id) return g_counts[i].counts;
  if (g_num_counts == kMaxStreamCounts) return nullptr;
  unsigned int* p = nullptr;
  if (!pool_take(&p, kCountBytes, v.pool, stream)) return nullptr;
  if (cudaMemsetAsync(p, 0, kCountBytes, stream) != cudaSuccess) {
    cudaGetLastError();
    pool_give(p, stream);
    return nullptr;
  }
  g_counts[g_num_counts++] = {v.device, id, p};
  return p;
}

// Slots and counts of one streaming launch.  Counts are the stream's own
// array, except under capture (a graph may be replayed on another stream),
// where they come with the slots and are cleared in the graph.
struct Workspace {
  char* base = nullptr;
  cudaStream_t stream = nullptr;
  int take(const DeviceView& v, size_t slot_bytes, cudaStream_t s, StreamArgs* args) {
    stream = s;
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(s, &cap) != cudaSuccess) {
      cudaGetLastError();
      cap = cudaStreamCaptureStatusActive;
    }
    args->counts = cap == cudaStreamCaptureStatusNone ? stream_counts(v, s) : nullptr;
    if (!pool_take(&base, kCountBytes + slot_bytes, v.pool, s)) return B200_ERR_LAUNCH;
    args->slots = reinterpret_cast<float*>(base + kCountBytes);
    if (args->counts == nullptr) {
      args->counts = reinterpret_cast<unsigned int*>(base);
      if (cudaMemsetAsync(base, 0, kCountBytes, s) != cudaSuccess) {
        cudaGetLastError();
        return B200_ERR_LAUNCH;
      }
    }
    return B200_OK;
  }
  ~Workspace() {
    if (base) pool_give(base, stream);
  }
};

// A buffer of the device's pool for one call, freed in stream order.
struct PoolBuffer {
  char* p = nullptr;
  cudaStream_t stream = nullptr;
  int take(const DeviceView& v, size_t bytes, cudaStream_t s) {
    stream = s;
    return pool_take(&p, bytes, v.pool, s) ? B200_OK : B200_ERR_LAUNCH;
  }
  ~PoolBuffer() {
    if (p) pool_give(p, stream);
  }
};

CUtensorMapDataType map_type(int dtype) {
  return dtype == B200_FP16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
}

int map_rows(CUtensorMap* m, int dtype, const void* p, int cols, int rows, int ld, int box_rows) {
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
  const cuuint32_t box[2] = {kSlabK, (cuuint32_t)box_rows};
  return encode_tensor(m, map_type(dtype), 2, p, dims, strides, box);
}

int map_bank(CUtensorMap* m, int dtype, const void* p, int K, int N, int experts, int ld,
             long long expert_stride, int box_rows) {
  const cuuint64_t dims[3] = {(cuuint64_t)K, (cuuint64_t)N, (cuuint64_t)experts};
  // (the stride of a bank of one is never used; any valid one will do)
  const cuuint64_t far = experts > 1 ? (cuuint64_t)expert_stride * 2 : (cuuint64_t)N * ld * 2;
  const cuuint64_t strides[2] = {(cuuint64_t)ld * 2, far};
  const cuuint32_t box[3] = {kSlabK, (cuuint32_t)box_rows, 1};
  return encode_tensor(m, map_type(dtype), 3, p, dims, strides, box);
}

// One call's operands: t the token operand read (A or dC), u the token
// operand written (C or dA) or, for dB, the other one read (A).
struct Call {
  const void* t;
  void* u;
  void* bank;
  const int* offsets;
  int rows, experts, N, K;
  int ldt, ldu, ldb;
  long long expert_stride;
  int dtype;
};

bool tma_rows(const void* p, long long ld) { return aligned16(p) && (ld & 7) == 0; }
bool tma_bank(const Call& c) {
  return tma_rows(c.bank, c.ldb) && (c.experts <= 1 || (c.expert_stride & 7) == 0);
}

int check_call(const Call& c, int mode) {
  if (c.rows < 0 || c.experts < 0 || c.N < 0 || c.K < 0) return B200_ERR_INVALID_ARGUMENT;
  if (c.dtype != B200_BF16 && c.dtype != B200_FP16) return B200_ERR_INVALID_ARGUMENT;
  if (c.experts > kMaxExperts) return B200_ERR_TOO_LARGE;
  const int wt = mode == kGroupedFwd ? c.K : c.N;  // width of t
  const int wu = mode == kGroupedFwd ? c.N : c.K;  // width of u
  const bool has_t = c.rows > 0 && wt > 0, has_u = c.rows > 0 && wu > 0;
  const bool has_bank = c.experts > 0 && c.N > 0 && c.K > 0;
  if ((has_t && !c.t) || (has_u && !c.u) || (has_bank && !c.bank) || (c.experts > 0 && !c.offsets))
    return B200_ERR_INVALID_ARGUMENT;
  if ((has_t && c.ldt < wt) || (has_u && c.ldu < wu) || (has_bank && c.ldb < c.K) ||
      (has_bank && c.experts > 1 && c.expert_stride < (long long)c.N * c.ldb))
    return B200_ERR_INVALID_ARGUMENT;
  // What is read must suit TMA; what is written, its elements.
  const bool bank_in = mode != kGroupedDB;
  if ((has_t && !tma_rows(c.t, c.ldt)) ||
      (has_u && (mode == kGroupedDB ? !tma_rows(c.u, c.ldu)
                                    : (reinterpret_cast<uintptr_t>(c.u) & 1u) != 0)) ||
      (has_bank && (bank_in ? !tma_bank(c) : (reinterpret_cast<uintptr_t>(c.bank) & 1u) != 0)) ||
      (reinterpret_cast<uintptr_t>(c.offsets) & 3u))
    return B200_ERR_ALIGNMENT;
  if (c.rows > kMaxExtent || c.N > kMaxExtent || c.K > kMaxExtent) return B200_ERR_TOO_LARGE;
  // unit numbers are 32-bit
  const int feat = mode == kGroupedDA ? c.K : c.N;
  const long long units = mode == kGroupedDB
                              ? ceil_div(c.N, 256) * ceil_div(c.K, 256) * c.experts
                              : (ceil_div(c.rows, 16) + c.experts) * ceil_div(feat, 128);
  return units < (1ll << 30) ? B200_OK : B200_ERR_TOO_LARGE;
}

int zero_rows(void* p, int ld, int width, int rows, cudaStream_t stream) {
  if (rows == 0 || width == 0) return B200_OK;
  return cudaMemset2DAsync(p, (size_t)ld * 2, 0, (size_t)width * 2, rows, stream) == cudaSuccess
             ? B200_OK
             : B200_ERR_LAUNCH;
}

// Launch with programmatic stream serialization: the kernel's set-up overlaps
// the end of the one before it (every kernel of this file waits, grid_wait,
// before it touches global memory).
template <class... P, class... A>
int launch(void (*fn)(P...), int blocks, int threads, size_t smem, cudaStream_t stream,
           A&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, fn, static_cast<P>(args)...) == cudaSuccess) return B200_OK;
  cudaGetLastError();
  return B200_ERR_LAUNCH;
}

template <int kMode, bool kMany, class T>
int launch_pair(const Call& c, const DeviceView& v, const MoeDevice& m, cudaStream_t stream) {
  using C = GroupedCfg<kMode, kMany>;
  CUtensorMap tw, tt, ts;
  int st;
  if (kMode == kGroupedDB) {
    st = map_rows(&tw, c.dtype, c.t, c.N, c.rows, c.ldt, 64);
    if (st == B200_OK) st = map_rows(&tt, c.dtype, c.u, c.K, c.rows, c.ldu, 64);
    if (st == B200_OK && tma_bank(c))
      st = map_bank(&ts, c.dtype, c.bank, c.K, c.N, c.experts, c.ldb, c.expert_stride, 32);
    else
      ts = tt;  // (not used: the kernel stores to `out`)
  } else {
    const int red = kMode == kGroupedFwd ? c.K : c.N;
    st = map_bank(&tw, c.dtype, c.bank, c.K, c.N, c.experts, c.ldb, c.expert_stride,
                  kMode == kGroupedFwd ? 128 : 64);
    if (st == B200_OK) st = map_rows(&tt, c.dtype, c.t, red, c.rows, c.ldt, 128);
    if (st == B200_OK) st = map_rows(&ts, c.dtype, c.t, red, c.rows, c.ldt, 16);
  }
  if (st != B200_OK) return st;
  PoolBuffer maps;
  if (kMode == kGroupedDB) {
    st = maps.take(v, (size_t)c.experts * 2 * sizeof(CUtensorMap), stream);
    if (st == B200_OK)
      st = launch(grouped_maps_kernel, c.experts, 32, 0, stream, tw, tt, c.offsets, c.rows,
                  reinterpret_cast<CUtensorMap*>(maps.p));
    if (st != B200_OK) return st;
  }
  GroupedArgs a = {};
  a.offsets = c.offsets;
  a.experts = c.experts;
  a.rows = c.rows;
  a.feat = kMode == kGroupedDA ? c.K : c.N;
  a.red = kMode == kGroupedFwd ? c.K : c.N;
  a.cols = c.K;
  a.out = kMode != kGroupedDB ? c.u : tma_bank(c) ? nullptr : c.bank;
  a.ldo = kMode == kGroupedDB ? c.ldb : c.ldu;
  a.expert_stride = c.expert_stride;
  a.group = 8;
  a.maps = reinterpret_cast<const CUtensorMap*>(maps.p);
  a.status = v.status;
  a.timeout_ns = v.timeout_ns;
  const long long tf = ceil_div(a.feat, 256);
  const long long most = kMode == kGroupedDB
                             ? tf * ceil_div(c.K, 256) * c.experts
                             : tf * (ceil_div(c.rows, 256) + (c.experts < c.rows ? c.experts : c.rows));
  const int pairs = (int)(most < m.pairs[kMode] ? most : m.pairs[kMode]);
  return launch(grouped_pair_kernel<kMode, kMany, T>, 2 * pairs, C::kThreads,
                C::smem_bytes(c.experts), stream, tw, tt, ts, a);
}

template <bool kDA, int kTok, class T>
int launch_stream(const Call& c, const DeviceView& v, cudaStream_t stream) {
  using C = StreamCfg<kTok>;
  CUtensorMap tw, tt;
  int st = map_bank(&tw, c.dtype, c.bank, c.K, c.N, c.experts, c.ldb, c.expert_stride,
                    kDA ? 64 : 128);
  const int red = kDA ? c.N : c.K;
  if (st == B200_OK) st = map_rows(&tt, c.dtype, c.t, red, c.rows, c.ldt, 16);
  if (st != B200_OK) return st;
  StreamArgs a = {};
  a.offsets = c.offsets;
  a.experts = c.experts;
  a.rows = c.rows;
  a.feat = kDA ? c.K : c.N;
  a.feat_blocks = (int)ceil_div(a.feat, 128);
  a.red = red;
  a.red_blocks = (int)ceil_div(red, kSlabK);
  a.min_items = 16;
  a.out = c.u;
  a.ldo = c.ldu;
  a.status = v.status;
  a.timeout_ns = v.timeout_ns;
  Workspace ws;
  st = ws.take(v, (size_t)v.sms * 2 * kTok * 128 * sizeof(float), stream, &a);
  if (st != B200_OK) return st;
  return launch(grouped_stream_kernel<kDA, kTok, T>, v.sms, C::kThreads,
                C::smem_bytes(c.experts), stream, tw, tt, a);
}

// The streaming kernel splits every contraction evenly over the SMs and takes
// 64 rows of an expert at a time; the pair kernel 256, but deals whole tiles.
// Streaming is faster while most experts fit one of its tiles (48 rows on
// average) and either the contraction is long or there are too few tiles to
// go round.  Measured, us, streaming / pair, for experts x N x K at rows per
// expert: 8 x 14336 x 4096 at 2: 112 / 122, at 48: 153 / 172, at 64: 205 /
// 175; 16 x 512 x 8192 at 16: 32 / 40; 32 x 2056 x 1032 at 16: 33 / 32, its
// gradient in A 45 / 37; 64 x 1024 x 2048 at 16: 54 / 55, 54 / 51.  With more
// rows it still is where three of four pairs would have no tile: 4 x 744 x
// 6200 at 100: 24 / 35, at 256: 39 / 48, at 400: 50 / 45.
bool use_stream(const Call& c, int feat, int red, int pairs) {
  const int k = g_kernel.load();
  if (k != 0) return k == 1;
  const long long groups = c.experts < c.rows ? c.experts : c.rows;
  const long long tiles = groups * ceil_div(feat, 256);  // of the pair kernel, at the least
  if (c.rows <= 48ll * c.experts) return red >= 4096 || tiles < 2ll * pairs;
  return c.rows <= 256ll * c.experts && red >= 4096 && 4 * tiles <= pairs;
}

template <int kMode, class T>
int run_typed(const Call& c, const DeviceView& v, const MoeDevice& m, cudaStream_t stream) {
  if constexpr (kMode != kGroupedDB) {
    constexpr bool kDA = kMode == kGroupedDA;
    if (use_stream(c, kDA ? c.K : c.N, kDA ? c.N : c.K, m.pairs[kMode]))
      return c.rows <= 16 ? launch_stream<kDA, 16, T>(c, v, stream)
                          : launch_stream<kDA, 64, T>(c, v, stream);
  }
  if constexpr (kMode == kGroupedDB) {
    if (c.experts > kFewExperts) return launch_pair<kMode, true, T>(c, v, m, stream);
  }
  return launch_pair<kMode, false, T>(c, v, m, stream);
}

template <int kMode>
int run_grouped(const Call& c, cudaStream_t stream) {
  int st = check_call(c, kMode);
  if (st != B200_OK) return st;
  const bool no_bank = c.experts == 0 || c.N == 0 || c.K == 0;
  if (kMode == kGroupedDB ? no_bank : c.rows == 0 || (kMode == kGroupedDA ? c.K : c.N) == 0)
    return B200_OK;  // nothing to write
  DeviceView v;
  MoeDevice* m = nullptr;
  st = moe_device(&v, &m);
  if (st != B200_OK) return st;
  if (kMode != kGroupedDB && no_bank)  // an empty contraction, or no expert at all
    return zero_rows(c.u, c.ldu, kMode == kGroupedDA ? c.K : c.N, c.rows, stream);
  if (kMode == kGroupedDB && c.rows == 0) {
    for (int e = 0; e < c.experts; ++e) {
      st = zero_rows(static_cast<char*>(c.bank) + 2 * e * c.expert_stride, c.ldb, c.K, c.N, stream);
      if (st != B200_OK) return st;
    }
    return B200_OK;
  }
  return c.dtype == B200_FP16 ? run_typed<kMode, __half>(c, v, *m, stream)
                              : run_typed<kMode, __nv_bfloat16>(c, v, *m, stream);
}

// ------------------------------------------------------------- 4-bit weights
struct W4Call {
  const void* a;
  const void* packed;
  void* c;
  const int* offsets;
  int rows, experts, N, K, group, zeros, lda, ldc, dtype;
};

int check_w4_shape(int experts, int N, int K, int group) {
  if (experts < 0 || N < 0 || K < 0) return B200_ERR_INVALID_ARGUMENT;
  if ((group != 32 && group != 64 && group != 128) || K % group != 0)
    return B200_ERR_INVALID_ARGUMENT;
  if (experts > kMaxExperts || N > kMaxExtent || K > kMaxExtent) return B200_ERR_TOO_LARGE;
  // record numbers are launch indexes
  return (long long)experts * ceil_div(N, kW4Rows) * ceil_div(K, kW4K) < (1ll << 31)
             ? B200_OK
             : B200_ERR_TOO_LARGE;
}

enum W4Kind { kW4Few, kW4Some, kW4Wide, kW4Split };  // rows, stream, wide, split kernel

template <W4Kind kKind, int kTok, int kGroup, bool kZeros, class T>
int launch_w4(const W4Call& c, const DeviceView& v, cudaStream_t stream) {
  constexpr int box_rows = W4Ring<kTok, kGroup>::kSlabRows;
  CUtensorMap tt;
  int st;
  if (kKind == kW4Split) {
    st = map_rows(&tt, c.dtype, c.a, c.K, c.rows, c.lda, kTok);
  } else if (kKind == kW4Wide) {
    st = map_rows(&tt, c.dtype, c.a, c.K, c.rows, c.lda, W4WideCfg<kGroup>::kBox);
  } else if (c.K % kSlabK == 0) {  // (k in a slab, row, slab)
    const cuuint64_t dims[3] = {kSlabK, (cuuint64_t)c.rows, (cuuint64_t)(c.K / kSlabK)};
    const cuuint64_t strides[2] = {(cuuint64_t)c.lda * 2, kSlabK * 2};
    const cuuint32_t box[3] = {kSlabK, box_rows, 4};
    st = encode_tensor(&tt, map_type(c.dtype), 3, c.a, dims, strides, box);
  } else {
    st = map_rows(&tt, c.dtype, c.a, c.K, c.rows, c.lda, box_rows);
  }
  if (st != B200_OK) return st;
  StreamArgs a = {};
  a.offsets = c.offsets;
  a.experts = c.experts;
  a.rows = c.rows;
  a.feat = c.N;
  a.feat_blocks = (int)ceil_div(c.N, kW4Rows);
  a.red = c.K;
  a.red_blocks = (int)ceil_div(c.K, kW4K);
  a.min_items = kKind == kW4Few ? 8 : 4;
  a.out = c.c;
  a.ldo = c.ldc;
  a.status = v.status;
  a.timeout_ns = v.timeout_ns;
  a.packed = static_cast<const uint8_t*>(c.packed);
  a.record_bytes = w4_record_bytes(kGroup, kZeros);
  a.expert_bytes = (long long)a.feat_blocks * a.red_blocks * a.record_bytes;
  Workspace ws;
  st = ws.take(v, (size_t)v.sms * (kKind == kW4Wide ? 3 : 2) * kTok * 128 * sizeof(float), stream, &a);
  if (st != B200_OK) return st;
  if constexpr (kKind == kW4Few) {
    using C = W4RowsCfg<kTok, kGroup>;
    return launch(w4_rows_kernel<kTok, kGroup, kZeros, T>, v.sms, C::kThreads,
                  C::smem_bytes(c.experts), stream, tt, a);
  } else if constexpr (kKind == kW4Split) {
    using C = W4SplitCfg<kTok, kGroup>;
    return launch(w4_split_kernel<kTok, kGroup, kZeros>, v.sms, C::kThreads,
                  C::smem_bytes(c.experts), stream, tt, a);
  } else if constexpr (kKind == kW4Wide) {
    using C = W4WideCfg<kGroup>;
    return launch(w4_wide_kernel<kGroup, kZeros, T>, v.sms, C::kThreads, C::smem_bytes(c.experts),
                  stream, tt, a);
  } else {
    using C = W4Cfg<kGroup>;
    return launch(w4_stream_kernel<kGroup, kZeros, T>, v.sms, C::kThreads,
                  C::smem_bytes(c.experts), stream, tt, a);
  }
}

template <int kGroup, bool kZeros, class T>
int run_w4_group(const W4Call& c, const DeviceView& v, cudaStream_t stream) {
  // A tile as wide as most experts' rows: an expert with more takes another
  // tile, that is, reads its weights again.
  if (c.rows <= 8 || c.rows <= 4ll * c.experts)
    return launch_w4<kW4Few, 8, kGroup, kZeros, T>(c, v, stream);
  if (c.rows <= 16 || c.rows <= 8ll * c.experts)
    return launch_w4<kW4Few, 16, kGroup, kZeros, T>(c, v, stream);
  // Small groups: warp MMAs take a tile of 32 as well, because the way through
  // TMEM reads a product back for every group (24 rows x 14336 x 4096: groups
  // of 32 40.2 and 30.0 us, of 64 36.1 and 31.9, of 128 26.5 and 27.2; 128
  // rows over 8 experts, groups of 32: 200 and 122).
  if constexpr (kGroup < 128) {
    if (c.rows <= 32 || c.rows <= 16ll * c.experts)
      return launch_w4<kW4Few, 32, kGroup, kZeros, T>(c, v, stream);
  }
  // bf16, small groups: weights as the sum of two bf16, so that no group's sums
  // are read back (one matrix of 14336 x 4096, groups of 32: 64 rows 43 and 34
  // us, 2048 rows 602 and 333; of 64: 37 and 34, 354 and 333; 1024 rows over 8
  // experts 520 and 251, 345 and 237).  Groups of 128 are better off without
  // (2048 rows 272 and 333).
  if constexpr (kSplits<kGroup, T>) {
    if (c.rows <= 64ll * c.experts)
      return launch_w4<kW4Split, 64, kGroup, kZeros, T>(c, v, stream);
    return launch_w4<kW4Split, 128, kGroup, kZeros, T>(c, v, stream);
  } else {
    // Tiles of 64 rows or of 256.  One matrix: as soon as 64 do not hold them
    // (96 rows x 14336 x 4096: 42.2 us in two tiles, 40.2 in a wide one; groups
    // of 32 66.8 and 62.8).  A bank: a wide tile costs the same from 129 rows
    // on, so experts must fill it by half, in groups of 32 altogether (8
    // experts of 14336 x 4096, groups of 128: 512 rows 153 and 184 us, 1024
    // rows 262 and 236; groups of 32: 1024 rows 483 and 601, 2048 rows 900 and
    // 890).
    const long long some = c.experts == 1 ? 64 : kGroup == 32 ? 256ll * c.experts : 96ll * c.experts;
    if (c.rows <= some)
      return launch_w4<kW4Some, 64, kGroup, kZeros, T>(c, v, stream);
    return launch_w4<kW4Wide, 256, kGroup, kZeros, T>(c, v, stream);
  }
}

template <class T>
int run_w4_typed(const W4Call& c, const DeviceView& v, cudaStream_t stream) {
  if (c.zeros)
    return c.group == 32   ? run_w4_group<32, true, T>(c, v, stream)
           : c.group == 64 ? run_w4_group<64, true, T>(c, v, stream)
                           : run_w4_group<128, true, T>(c, v, stream);
  return c.group == 32   ? run_w4_group<32, false, T>(c, v, stream)
         : c.group == 64 ? run_w4_group<64, false, T>(c, v, stream)
                         : run_w4_group<128, false, T>(c, v, stream);
}

int run_w4(const W4Call& c, cudaStream_t stream) {
  int st = check_w4_shape(c.experts, c.N, c.K, c.group);
  if (st != B200_OK) return st;
  if (c.rows < 0 || (c.dtype != B200_BF16 && c.dtype != B200_FP16) ||
      (c.offsets == nullptr && c.experts > 1))
    return B200_ERR_INVALID_ARGUMENT;
  if (c.rows == 0 || c.N == 0) return B200_OK;
  const bool empty = c.K == 0 || c.experts == 0;
  if (!c.c || c.ldc < c.N || (!empty && (!c.a || !c.packed || c.lda < c.K)))
    return B200_ERR_INVALID_ARGUMENT;
  if ((reinterpret_cast<uintptr_t>(c.c) & 1u) ||
      (!empty && (!tma_rows(c.a, c.lda) || !aligned16(c.packed))) ||
      (reinterpret_cast<uintptr_t>(c.offsets) & 3u))
    return B200_ERR_ALIGNMENT;
  if (c.rows > kMaxExtent ||
      (ceil_div(c.rows, 16) + c.experts) * ceil_div(c.N, kW4Rows) >= (1ll << 30))
    return B200_ERR_TOO_LARGE;
  DeviceView v;
  MoeDevice* m = nullptr;
  st = moe_device(&v, &m);
  if (st != B200_OK) return st;
  if (empty) return zero_rows(c.c, c.ldc, c.N, c.rows, stream);
  return c.dtype == B200_FP16 ? run_w4_typed<__half>(c, v, stream)
                              : run_w4_typed<__nv_bfloat16>(c, v, stream);
}

int run_w4_pack(const void* q, const void* scales, const void* zeros, void* packed, int experts,
                int N, int K, int group, cudaStream_t stream) {
  int st = check_w4_shape(experts, N, K, group);
  if (st != B200_OK) return st;
  const int blocks = (int)ceil_div(N, kW4Rows), red = (int)ceil_div(K, kW4K);
  const long long records = (long long)experts * blocks * red;
  if (records == 0) return B200_OK;
  if (!q || !scales || !packed) return B200_ERR_INVALID_ARGUMENT;
  if (!aligned16(packed) || (reinterpret_cast<uintptr_t>(scales) & 1u)) return B200_ERR_ALIGNMENT;
  DeviceView v;
  MoeDevice* m = nullptr;
  st = moe_device(&v, &m);
  if (st != B200_OK) return st;
  return launch(w4_pack_kernel, (int)records, 256, 0, stream, static_cast<const uint8_t*>(q),
                static_cast<const uint16_t*>(scales), static_cast<const uint8_t*>(zeros),
                static_cast<uint8_t*>(packed), N, K, group, blocks, red,
                w4_record_bytes(group, zeros != nullptr), v.status);
}

// -------------------------------------------------------------------- routing
template <int kPer>
int launch_choose(const RouteArgs& a, int blocks, size_t smem, cudaStream_t stream) {
  return launch(route_choose_kernel<kPer>, blocks, kRouteThreads, smem, stream, a);
}

int run_route(RouteArgs a, const DeviceView& v, cudaStream_t stream) {
  // Up to 256 tokens one block does everything in one launch; beyond that
  // one chunk per SM (two choose faster but rank slower: 10.2 + 18.7 us against
  // 11 + 13 at 16383 tokens, 64 experts).
  a.chunk = a.tokens <= 256 ? a.tokens : (int)ceil_div(a.tokens, v.sms);
  const int blocks = (int)ceil_div(a.tokens, a.chunk);
  const size_t smem = (size_t)(1 + kRouteWarps) * a.experts * sizeof(int);
  int* counts = nullptr;
  if (blocks > 1) {
    if (!pool_take(&counts, (size_t)blocks * a.experts * sizeof(int), v.pool, stream))
      return B200_ERR_LAUNCH;
    a.counts = counts;
  }
  int st = a.experts <= 32    ? launch_choose<1>(a, blocks, smem, stream)
           : a.experts <= 64  ? launch_choose<2>(a, blocks, smem, stream)
           : a.experts <= 128 ? launch_choose<4>(a, blocks, smem, stream)
           : a.experts <= 256 ? launch_choose<8>(a, blocks, smem, stream)
                              : launch_choose<32>(a, blocks, smem, stream);
  if (st == B200_OK && blocks > 1) {
    st = launch(route_rank_kernel, blocks, kRouteThreads, smem, stream, a);
  }
  if (counts) pool_give(counts, stream);
  return st;
}

enum Move { kDispatch, kCombine, kCombineGrad };

template <class T, int kVec>
int launch_move(Move what, const MoveArgs& a, cudaStream_t stream) {
  const long long lanes = ceil_div(a.width, kVec);
  const int threads = lanes >= 256 ? 256 : (int)(lanes < 32 ? 32 : (lanes + 31) / 32 * 32);
  switch (what) {
    case kDispatch: return launch(dispatch_kernel<T, kVec>, a.tokens, threads, 0, stream, a);
    case kCombine: return launch(combine_kernel<T, kVec>, a.tokens, threads, 0, stream, a);
    default: return launch(combine_grad_kernel<T, kVec>, a.tokens, threads, 0, stream, a);
  }
}

int run_move(Move what, MoveArgs a, const int* total, int dtype, cudaStream_t stream) {
  if (a.tokens < 0 || a.top_k < 0 || a.width < 0 || a.top_k > kMaxTopK ||
      (dtype != B200_BF16 && dtype != B200_FP16))
    return B200_ERR_INVALID_ARGUMENT;
  if ((long long)a.tokens * a.top_k >= (1ll << 31) || a.tokens > kMaxExtent ||
      a.width > kMaxExtent)
    return B200_ERR_TOO_LARGE;
  // no slots: dispatch and the gradient write nothing, combine writes zeros
  if (a.tokens == 0 || (a.top_k == 0 && what != kCombine)) return B200_OK;
  if (a.width == 0 && what != kCombineGrad) return B200_OK;
  const bool any = a.top_k > 0, wide = a.width > 0;
  if ((any && !a.rows) || (wide && (!a.out || (any && !a.in))) ||
      (what != kCombine && !total) ||
      (what == kCombineGrad && ((wide && !a.in2) || !a.weights)))
    return B200_ERR_INVALID_ARGUMENT;
  if (wide && (a.ld_in < a.width || a.ld_out < a.width ||
               (what == kCombineGrad && a.ld_in2 < a.width)))
    return B200_ERR_INVALID_ARGUMENT;
  if (((reinterpret_cast<uintptr_t>(a.in) | reinterpret_cast<uintptr_t>(a.in2) |
        reinterpret_cast<uintptr_t>(a.out)) & 1u) ||
      ((reinterpret_cast<uintptr_t>(a.rows) | reinterpret_cast<uintptr_t>(total) |
        reinterpret_cast<uintptr_t>(a.weights) | reinterpret_cast<uintptr_t>(a.dweights)) & 3u))
    return B200_ERR_ALIGNMENT;
  DeviceView v;
  MoeDevice* m = nullptr;
  const int st = moe_device(&v, &m);
  if (st != B200_OK) return st;
  const bool vec = aligned16(a.in) && aligned16(a.out) && aligned16(a.in2) &&
                   ((a.width | a.ld_in | a.ld_out | a.ld_in2) & 7) == 0;
  const int pairs = a.tokens * a.top_k;
  PoolBuffer named;
  if (what != kCombine && pairs > kScanPairs) {
    int got = named.take(v, (size_t)pairs * sizeof(int), stream);
    const int blocks = (int)ceil_div(pairs, 256);
    if (got == B200_OK)
      got = launch(mark_rows_kernel, blocks < 8 * v.sms ? blocks : 8 * v.sms, 256, 0, stream, a.rows,
                   reinterpret_cast<int*>(named.p), pairs);
    if (got != B200_OK) return got;
    a.named = reinterpret_cast<const int*>(named.p);
  }
  if (dtype == B200_FP16)
    return vec ? launch_move<__half, 8>(what, a, stream) : launch_move<__half, 1>(what, a, stream);
  return vec ? launch_move<__nv_bfloat16, 8>(what, a, stream)
             : launch_move<__nv_bfloat16, 1>(what, a, stream);
}

}  // namespace

extern "C" {

int b200_grouped_gemm(const void* A, const void* B, void* C, const int* offsets, int rows,
                      int experts, int N, int K, int lda, int ldb, long long expert_stride,
                      int ldc, int dtype, void* stream) {
  const Call c = {A, C, const_cast<void*>(B), offsets, rows, experts, N, K,
                  lda, ldc, ldb, expert_stride, dtype};
  return run_grouped<kGroupedFwd>(c, static_cast<cudaStream_t>(stream));
}

int b200_grouped_gemm_da(const void* dC, const void* B, void* dA, const int* offsets, int rows,
                         int experts, int N, int K, int ldc, int ldb, long long expert_stride,
                         int lda, int dtype, void* stream) {
  const Call c = {dC, dA, const_cast<void*>(B), offsets, rows, experts, N, K,
                  ldc, lda, ldb, expert_stride, dtype};
  return run_grouped<kGroupedDA>(c, static_cast<cudaStream_t>(stream));
}

int b200_grouped_gemm_db(const void* dC, const void* A, void* dB, const int* offsets, int rows,
                         int experts, int N, int K, int ldc, int lda, int ldb,
                         long long expert_stride, int dtype, void* stream) {
  const Call c = {dC, const_cast<void*>(A), dB, offsets, rows, experts, N, K,
                  ldc, lda, ldb, expert_stride, dtype};
  return run_grouped<kGroupedDB>(c, static_cast<cudaStream_t>(stream));
}

int b200_align_rows(const void* src, long long matrix_stride, long long row_stride, void* dst,
                    int matrices, int rows, int cols, int ld, void* stream) {
  if (matrices < 0 || rows < 0 || cols < 0 || ld < cols) return B200_ERR_INVALID_ARGUMENT;
  if (matrices == 0 || rows == 0 || cols == 0) return B200_OK;
  if (!src || !dst || row_stride < 0 || matrix_stride < 0) return B200_ERR_INVALID_ARGUMENT;
  if (!tma_rows(dst, ld) || (reinterpret_cast<uintptr_t>(src) & 1u)) return B200_ERR_ALIGNMENT;
  if (ld > kMaxExtent) return B200_ERR_TOO_LARGE;
  DeviceView v;
  MoeDevice* m = nullptr;
  const int st = moe_device(&v, &m);
  if (st != B200_OK) return st;
  const long long blocks = ceil_div((long long)matrices * rows * (ld / 8), 256);
  const long long most = 16ll * v.sms;
  return launch(align_rows_kernel, (int)(blocks < most ? blocks : most), 256, 0,
                static_cast<cudaStream_t>(stream), static_cast<const uint16_t*>(src),
                matrix_stride, row_stride, static_cast<uint16_t*>(dst), matrices, rows, cols, ld);
}

int b200_narrow_offsets(const void* offsets, long long stride, int count, int* out, void* stream) {
  if (count < 0 || stride < 0) return B200_ERR_INVALID_ARGUMENT;
  if (count == 0) return B200_OK;
  if (count > kMaxExperts + 1) return B200_ERR_TOO_LARGE;
  if (!offsets || !out) return B200_ERR_INVALID_ARGUMENT;
  if ((reinterpret_cast<uintptr_t>(offsets) & 7u) || (reinterpret_cast<uintptr_t>(out) & 3u))
    return B200_ERR_ALIGNMENT;
  DeviceView v;
  MoeDevice* m = nullptr;
  const int st = moe_device(&v, &m);
  if (st != B200_OK) return st;
  return launch(narrow_offsets_kernel, 1, 256, 0, static_cast<cudaStream_t>(stream),
                static_cast<const long long*>(offsets), stride, count, out);
}

int b200_grouped_set_kernel(int kernel) {
  if (kernel < 0 || kernel > 2) return B200_ERR_INVALID_ARGUMENT;
  g_kernel.store(kernel);
  return B200_OK;
}

int b200_w4_packed_bytes(int experts, int N, int K, int group, int zeros, size_t* bytes) {
  if (!bytes) return B200_ERR_INVALID_ARGUMENT;
  const int st = check_w4_shape(experts, N, K, group);
  if (st != B200_OK) return st;
  *bytes = (size_t)experts * ceil_div(N, kW4Rows) * ceil_div(K, kW4K) *
           w4_record_bytes(group, zeros != 0);
  return B200_OK;
}

int b200_w4_pack(const void* q, const void* scales, const void* zeros, void* packed, int experts,
                 int N, int K, int group, void* stream) {
  return run_w4_pack(q, scales, zeros, packed, experts, N, K, group,
                     static_cast<cudaStream_t>(stream));
}

int b200_w4_gemm(const void* A, const void* packed, void* C, const int* offsets, int rows,
                 int experts, int N, int K, int group, int zeros, int lda, int ldc, int dtype,
                 void* stream) {
  const W4Call c = {A, packed, C, offsets, rows, experts, N, K, group, zeros, lda, ldc, dtype};
  return run_w4(c, static_cast<cudaStream_t>(stream));
}

int b200_route(const void* logits, int tokens, int experts, long long ld, int type, int top_k,
               int normalize, float* weights, int* chosen, int* rows, int* sources, int* offsets,
               void* stream) {
  if (tokens < 0 || experts < 0 || top_k < 0 || top_k > experts || top_k > kMaxTopK ||
      type < B200_BF16 || type > B200_FP32)
    return B200_ERR_INVALID_ARGUMENT;
  if (experts > kMaxExperts || tokens > kMaxExtent || (long long)tokens * top_k >= (1ll << 31))
    return B200_ERR_TOO_LARGE;
  if (!offsets) return B200_ERR_INVALID_ARGUMENT;
  const bool any = tokens > 0 && top_k > 0;
  if (any && (!logits || ld < experts || !weights || !chosen || !rows || !sources))
    return B200_ERR_INVALID_ARGUMENT;
  if ((reinterpret_cast<uintptr_t>(logits) & (type == B200_FP32 ? 3u : 1u)) ||
      ((reinterpret_cast<uintptr_t>(weights) | reinterpret_cast<uintptr_t>(chosen) |
        reinterpret_cast<uintptr_t>(rows) | reinterpret_cast<uintptr_t>(sources) |
        reinterpret_cast<uintptr_t>(offsets)) & 3u))
    return B200_ERR_ALIGNMENT;
  DeviceView v;
  MoeDevice* m = nullptr;
  const int st = moe_device(&v, &m);
  if (st != B200_OK) return st;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (!any)
    return cudaMemsetAsync(offsets, 0, (size_t)(experts + 1) * sizeof(int), s) == cudaSuccess
               ? B200_OK
               : B200_ERR_LAUNCH;
  RouteArgs a = {};
  a.logits = logits;
  a.ld = ld;
  a.type = type;
  a.tokens = tokens;
  a.experts = experts;
  a.top_k = top_k;
  a.normalize = normalize != 0;
  a.weights = weights;
  a.chosen = chosen;
  a.rows = rows;
  a.sources = sources;
  a.offsets = offsets;
  return run_route(a, v, s);
}

int b200_route_grad(const void* logits, int tokens, int experts, long long ld, int type, int top_k,
                    int normalize, const int* chosen, const float* weights, const float* dweights,
                    void* dlogits, void* stream) {
  if (tokens < 0 || experts < 0 || top_k < 0 || top_k > experts || top_k > kMaxTopK ||
      type < B200_BF16 || type > B200_FP32)
    return B200_ERR_INVALID_ARGUMENT;
  if (experts > kMaxExperts || tokens > kMaxExtent) return B200_ERR_TOO_LARGE;
  if (tokens == 0 || experts == 0) return B200_OK;
  if (!logits || ld < experts || !dlogits || (top_k > 0 && (!chosen || !weights || !dweights)))
    return B200_ERR_INVALID_ARGUMENT;
  if (((reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(dlogits)) &
       (type == B200_FP32 ? 3u : 1u)) ||
      ((reinterpret_cast<uintptr_t>(chosen) | reinterpret_cast<uintptr_t>(weights) |
        reinterpret_cast<uintptr_t>(dweights)) & 3u))
    return B200_ERR_ALIGNMENT;
  DeviceView v;
  MoeDevice* m = nullptr;
  const int st = moe_device(&v, &m);
  if (st != B200_OK) return st;
  RouteArgs a = {};
  a.logits = logits;
  a.ld = ld;
  a.type = type;
  a.tokens = tokens;
  a.experts = experts;
  a.top_k = top_k;
  a.normalize = normalize != 0;
  a.weights = const_cast<float*>(weights);
  a.chosen = const_cast<int*>(chosen);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int blocks = (int)ceil_div(tokens, 8);
  return experts <= 32    ? launch(route_grad_kernel<1>, blocks, 256, 0, s, a, dweights, dlogits)
         : experts <= 64  ? launch(route_grad_kernel<2>, blocks, 256, 0, s, a, dweights, dlogits)
         : experts <= 128 ? launch(route_grad_kernel<4>, blocks, 256, 0, s, a, dweights, dlogits)
         : experts <= 256 ? launch(route_grad_kernel<8>, blocks, 256, 0, s, a, dweights, dlogits)
                          : launch(route_grad_kernel<32>, blocks, 256, 0, s, a, dweights, dlogits);
}

int b200_dispatch(const void* x, const int* rows, const int* total, void* xs, int tokens, int top_k,
                  int width, long long ldx, long long ldxs, int dtype, void* stream) {
  MoveArgs a = {};
  a.in = x;
  a.ld_in = ldx;
  a.out = xs;
  a.ld_out = ldxs;
  a.rows = rows;
  a.tokens = tokens;
  a.top_k = top_k;
  a.width = width;
  return run_move(kDispatch, a, total, dtype, static_cast<cudaStream_t>(stream));
}

int b200_combine(const void* y, const float* weights, const int* rows, void* out, int tokens,
                 int top_k, int width, long long ldy, long long ldo, int dtype, void* stream) {
  MoveArgs a = {};
  a.in = y;
  a.ld_in = ldy;
  a.out = out;
  a.ld_out = ldo;
  a.weights = weights;
  a.rows = rows;
  a.tokens = tokens;
  a.top_k = top_k;
  a.width = width;
  return run_move(kCombine, a, nullptr, dtype, static_cast<cudaStream_t>(stream));
}

int b200_combine_grad(const void* dout, const void* y, const float* weights, const int* rows,
                      const int* total, void* dy, float* dweights, int tokens, int top_k, int width,
                      long long ldo, long long ldy, long long lddy, int dtype, void* stream) {
  MoveArgs a = {};
  a.in = dout;
  a.ld_in = ldo;
  a.in2 = y;
  a.ld_in2 = ldy;
  a.out = dy;
  a.ld_out = lddy;
  a.weights = weights;
  a.dweights = dweights;
  a.rows = rows;
  a.tokens = tokens;
  a.top_k = top_k;
  a.width = width;
  return run_move(kCombineGrad, a, total, dtype, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
