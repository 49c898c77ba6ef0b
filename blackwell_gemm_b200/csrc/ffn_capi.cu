// C-ABI launchers of the feed-forward operators (include/b200_ffn.h).
//
// Per call: check the arguments, encode the tensor maps, choose a kernel and
// launch it on the caller's stream.  Per device, once: shared-memory limits
// and the number of 2-CTA clusters that can be resident.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <mutex>

#include "b200_ffn.h"
#include "device_state.h"
#include "ffn_cluster.cuh"
#include "ffn_gemm.cuh"
#include "ffn_grad.cuh"
#include "ffn_stream.cuh"
#include "grad_norm.cuh"
#include "launch.h"

using namespace b200;

namespace {

struct FfnDevice {
  bool ready = false;
  int init_status = B200_OK;
  int pairs[4] = {};  // resident clusters per FfnMode
  int clusters[2][4] = {};  // resident clusters of parts of 1 or 2 CTAs, 1, 2, 4 or 8 parts
};

std::mutex g_mu;
FfnDevice g_ffn[kMaxDevices];
std::atomic<int> g_kernel{0};

// Experts whose table fits beside six stages.
constexpr int kFewExperts = 128;

template <int kMode, bool kMany, class T>
bool init_pair(int sms, int* pairs) {
  using C = FfnCfg<kMode, kMany>;
  constexpr int experts = kMany ? kMaxExperts : kFewExperts;
  // (512 B: more than the kernel's static shared memory)
  static_assert(C::smem_bytes(experts) <= 227 * 1024 - 512, "shared memory of one CTA");
  auto* fn = ffn_pair_kernel<kMode, kMany, T>;
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

template <bool kGated, int kTok, class T>
bool init_stream() {
  using C = FfnStreamCfg<kTok>;
  static_assert(C::smem_bytes(kMaxExperts) <= 227 * 1024 - 512, "shared memory of one CTA");
  return set_smem(ffn_stream_kernel<kGated, kTok, T>, C::smem_bytes(kMaxExperts));
}

template <int kMode, bool kPair, class T>
bool init_cluster(int sms, int* clusters) {
  using C = FfnClusterCfg<kPair>;
  static_assert(C::kSmem <= 227 * 1024 - 512, "shared memory of one CTA");
  auto* fn = ffn_cluster_kernel<kMode, kPair, T>;
  if (!set_smem(fn, C::kSmem)) return false;
  for (int i = 0; i < (kPair ? 3 : 4); ++i) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    const int ctas = (kPair ? 2 : 1) << i;
    cfg.gridDim = dim3((unsigned)(sms / ctas * ctas));
    cfg.blockDim = dim3(C::kThreads);
    cfg.dynamicSmemBytes = C::kSmem;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, fn, &cfg) != cudaSuccess || n < 1) return false;
    if (clusters[i] == 0 || n < clusters[i]) clusters[i] = n;
  }
  return true;
}

template <int kMode, class T>
bool init_clusters(FfnDevice& d, int sms) {
  return init_cluster<kMode, false, T>(sms, d.clusters[0]) &&
         init_cluster<kMode, true, T>(sms, d.clusters[1]);
}

template <class T>
bool init_type(FfnDevice& d, int sms) {
  return init_clusters<kFfnGated, T>(d, sms) && init_clusters<kFfnAct, T>(d, sms) &&
         init_clusters<kFfnDA, T>(d, sms) &&
         init_pair<kFfnGated, false, T>(sms, &d.pairs[0]) &&
         init_pair<kFfnGated, true, T>(sms, &d.pairs[0]) &&
         init_pair<kFfnAct, false, T>(sms, &d.pairs[1]) &&
         init_pair<kFfnDA, false, T>(sms, &d.pairs[2]) &&
         init_pair<kFfnDA, true, T>(sms, &d.pairs[2]) &&
         init_pair<kFfnDW, false, T>(sms, &d.pairs[3]) &&
         init_pair<kFfnDW, true, T>(sms, &d.pairs[3]) && init_stream<true, 16, T>() &&
         init_stream<true, 64, T>() && init_stream<true, 128, T>() &&
         init_stream<true, 256, T>() && init_stream<false, 16, T>() &&
         init_stream<false, 64, T>();
}

int ffn_device(DeviceView* v, FfnDevice** out) {
  const int st = device_view(v);
  if (st != B200_OK) return st;
  std::lock_guard<std::mutex> lock(g_mu);
  FfnDevice& d = g_ffn[v->device];
  if (!d.ready) {
    d.ready = true;
    d.init_status = init_type<__nv_bfloat16>(d, v->sms) && init_type<__half>(d, v->sms)
                        ? B200_OK
                        : B200_ERR_LAUNCH;
    if (d.init_status != B200_OK) cudaGetLastError();
  }
  if (d.init_status != B200_OK) return d.init_status;
  *out = &d;
  return B200_OK;
}

// A bank of matrices, or one: read by TMA.
struct Bank {
  const void* p;
  int ld;
  long long stride;
};

// One product.  t: the token operand read; out: what is written.
struct FfnCall {
  const void* t;
  Bank w[2];
  int weights;  // 1 or 2
  const int* offsets;
  int rows, experts, N, K;
  int ldt;
  FfnOut o;
  int dtype;
};

bool on(const void* p, unsigned bytes) {
  return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0;
}

// What all the operators' sizes have to be; experts counts matrices.
int check_sizes(int rows, int experts, int N, int K, const int* offsets, int dtype) {
  if (rows < 0 || experts < 0 || N < 0 || K < 0) return B200_ERR_INVALID_ARGUMENT;
  if (dtype != B200_BF16 && dtype != B200_FP16) return B200_ERR_INVALID_ARGUMENT;
  if (offsets == nullptr && experts != 1) return B200_ERR_INVALID_ARGUMENT;
  if (experts > kMaxExperts) return B200_ERR_TOO_LARGE;
  if (!on(offsets, 4)) return B200_ERR_ALIGNMENT;
  if (rows > kMaxExtent || N > kMaxExtent || K > kMaxExtent) return B200_ERR_TOO_LARGE;
  return B200_OK;
}

// A matrix (or bank) that TMA reads; null is allowed where it is empty.
int check_bank(const Bank& w, int experts, int N, int K) {
  if (experts == 0 || N == 0 || K == 0) return B200_OK;
  if (!w.p || w.ld < K || (experts > 1 && w.stride < (long long)N * w.ld))
    return B200_ERR_INVALID_ARGUMENT;
  return tma_rows(w.p, w.ld) && (experts <= 1 || (w.stride & 7) == 0) ? B200_OK
                                                                       : B200_ERR_ALIGNMENT;
}

int check_rows(const void* p, int ld, int rows, int cols) {
  if (rows == 0 || cols == 0) return B200_OK;
  if (!p || ld < cols) return B200_ERR_INVALID_ARGUMENT;
  return tma_rows(p, ld) ? B200_OK : B200_ERR_ALIGNMENT;
}

// A row operand that kernels read or write element by element.
int check_plain(const void* p, int ld, int rows, int cols, bool may_be_null) {
  if (rows == 0 || cols == 0 || (p == nullptr && may_be_null)) return B200_OK;
  if (!p || ld < cols) return B200_ERR_INVALID_ARGUMENT;
  return on(p, 2) ? B200_OK : B200_ERR_ALIGNMENT;
}

int check_z(const float* z, int ldz, int rows, int cols) {
  if (z == nullptr || rows == 0 || cols == 0) return B200_OK;
  if (ldz < cols) return B200_ERR_INVALID_ARGUMENT;
  return on(z, 16) && (ldz & 3) == 0 ? B200_OK : B200_ERR_ALIGNMENT;
}

// unit numbers are 32-bit
int check_units(long long row_tiles, long long experts, long long feat, long long times) {
  return (row_tiles + experts) * ceil_div(feat, 64) * times < (1ll << 30) ? B200_OK
                                                                         : B200_ERR_TOO_LARGE;
}

#define CHECK(x)                     \
  do {                               \
    const int st_ = (x);             \
    if (st_ != B200_OK) return st_;  \
  } while (0)

// (columns, rows, halves), the halves rows * ld apart.
int map_halves(CUtensorMap* m, int dtype, const void* p, int cols, int rows, int halves, int ld,
               int box_rows) {
  return map_bank(m, dtype, p, cols, rows, halves, ld, (long long)rows * ld, box_rows);
}

template <int kMode, bool kMany, class T>
int launch_pair(FfnArgs& a, const CUtensorMap& w0, const CUtensorMap& w1, const CUtensorMap& t,
                const CUtensorMap& h, const CUtensorMap& s, const DeviceView& v,
                const FfnDevice& d, cudaStream_t stream) {
  using C = FfnCfg<kMode, kMany>;
  // Bands of token tiles: wide ones read the weights less often, narrow ones the tokens.
  // (8, 16 and 32 wide, us: gated 8192 x 28672 x 4096 1190, 1180, 1308; its dA 1254, 1288,
  // 1366 and dW 1247, 1290, 1355; dA of 4095 rows, all in one band of 16, 697 and 679.)
  const bool few = ceil_div(a.rows, 256) <= 16;
  a.group = kMode == kFfnDW || (kMode == kFfnDA && !few) ? 8 : 16;
  a.status = v.status;
  a.timeout_ns = v.timeout_ns;
  const long long tf = ceil_div(a.feat, C::kFeat);
  const long long most =
      kMode == kFfnDW ? tf * ceil_div(a.cols, 256) * a.halves * a.experts
      : a.offsets == nullptr
          ? tf * ceil_div(a.rows, 256)
          : tf * (ceil_div(a.rows, 256) + (a.experts < a.rows ? a.experts : a.rows));
  // Tiles of equal contractions may be divided, where some are left over: the kernel
  // sees whether that pays.
  const int blocks = (int)ceil_div(kMode == kFfnDW ? a.rows : a.red, kSlabK) *
                     (kMode == kFfnDA ? a.halves : 1);
  const bool divide = (kMode != kFfnDW || a.offsets == nullptr) &&
                      blocks > FfnWalk<kMode>::kJoinBlocks && most > d.pairs[kMode] &&
                      (a.offsets != nullptr || most % d.pairs[kMode] != 0);
  a.tile_n = kMode == kFfnDW || a.offsets != nullptr
                 ? 256
                 : (int)ceil_div(ceil_div(a.rows, ceil_div(a.rows, 256)), 32) * 32;
  const int pairs = (int)(most < d.pairs[kMode] ? most : d.pairs[kMode]);
  Workspace ws;
  if (divide) CHECK(ws.take(v, (size_t)2 * pairs * 2 * 256 * 128 * sizeof(float), stream, &a));
  return launch(ffn_pair_kernel<kMode, kMany, T>, 2 * pairs, C::kThreads,
                C::smem_bytes(a.experts), stream, w0, w1, t, h, s, a);
}

// The forward products and dA: a bank of matrices times rows.
template <int kMode, class T>
int run_pair(const FfnCall& c, const DeviceView& v, const FfnDevice& d, cudaStream_t stream) {
  constexpr bool kDA = kMode == kFfnDA;
  const int red = kDA ? c.N : c.K;
  CUtensorMap w[2], t, h, s;
  for (int i = 0; i < c.weights; ++i)
    CHECK(map_bank(&w[i], c.dtype, c.w[i].p, c.K, c.N, c.experts, c.w[i].ld, c.w[i].stride,
                   kMode == kFfnAct ? 128 : 64));
  if (c.weights == 1) w[1] = w[0];
  const int halves = kDA ? c.weights : 1;
  CHECK(map_halves(&t, c.dtype, c.t, red, c.rows, halves, c.ldt, 128));
  CHECK(map_halves(&h, c.dtype, c.t, red, c.rows, halves, c.ldt, 64));
  CHECK(map_halves(&s, c.dtype, c.t, red, c.rows, halves, c.ldt, 16));
  FfnArgs a = {};
  a.offsets = c.offsets;
  a.experts = c.experts;
  a.rows = c.rows;
  a.feat = c.o.feat;
  a.red = red;
  a.halves = halves;
  a.o = c.o;
  if constexpr (kMode != kFfnAct) {  // (which has one matrix)
    if (c.experts > kFewExperts)
      return launch_pair<kMode, true, T>(a, w[0], w[1], t, h, s, v, d, stream);
  }
  return launch_pair<kMode, false, T>(a, w[0], w[1], t, h, s, v, d, stream);
}

// How the cluster kernel would take a product, and about how long, in us.
struct ClusterPlan {
  bool pair = false;
  int splits = 0, tokens = 0;  // splits 0: it cannot
  double us = 1e30;
};

// Every way that fits one wave, by what was measured: 6.5 us for the launch, the ring's
// first loads and the last barrier; a stage's 16 KiB of weights and box of tokens at 95
// GB/s to a CTA, 70 in a pair, or the weights at HBM's 6.3 TB/s; 16 tokens of the
// epilogue 0.55 us to a group of warps, of the exchange 0.25.  (2048 x 8192 at 256
// rows: 22.9 us in 64 CTAs, 22.1 in 32 pairs, where the persistent pairs took 48; 4096
// x 14336 at 128 rows 27.0, 44 through slots in L2.)
ClusterPlan plan_cluster(int rows, int feat, int blocks, int feat_cta, const FfnDevice& d) {
  ClusterPlan best;
  for (int pair = 0; pair < 2; ++pair) {
    const int step = pair ? 32 : 16;
    int last = 0;
    for (int most = 256; most >= step; most /= 2) {
      const long long tt = ceil_div(rows, most);
      const int tokens = (int)(ceil_div(ceil_div(rows, tt), step) * step);
      if (tokens == last) continue;
      last = tokens;
      const long long tiles = ceil_div(feat, feat_cta << pair) * ceil_div(rows, tokens);
      for (int i = 0; i < (pair ? 3 : 4); ++i) {
        const int splits = 1 << i;
        if (tiles > d.clusters[pair][i] || splits > blocks) continue;
        const double share = (double)ceil_div(blocks, splits);
        const double load = (16384.0 + (pair ? tokens / 2 : tokens) * 128) / (pair ? 70e3 : 95e3);
        const double hbm = 16384.0 * (double)(tiles / ceil_div(rows, tokens) * splits) *
                           (pair ? 2 : 1) / 6.3e6;
        const double chunks = tokens / 32.0;  // to a group of warps
        const double us = 6.5 + share * std::max(load, hbm) + 0.55 * chunks / splits +
                          (splits > 1 ? 0.7 + 0.25 * chunks * (1.0 - 1.0 / splits) : 0.0);
        if (us < best.us) best = {pair != 0, splits, tokens, us};
      }
    }
  }
  return best;
}

// One tile to a cluster, its contraction over `splits` parts of one CTA or two.
template <int kMode, bool kPair, class T>
int run_cluster(const FfnCall& c, const ClusterPlan& plan, const DeviceView& v,
                cudaStream_t stream) {
  using C = FfnClusterCfg<kPair>;
  constexpr bool kDA = kMode == kFfnDA;
  const int red = kDA ? c.N : c.K, halves = kDA ? c.weights : 1;
  FfnClusterArgs a = {};
  a.rows = c.rows;
  a.feat = c.o.feat;
  a.red = red;
  a.halves = halves;
  a.splits = plan.splits;
  a.tokens = plan.tokens;
  a.tiles_t = (int)ceil_div(c.rows, a.tokens);
  a.box = kPair ? a.tokens / 2 : a.tokens;
  a.stage_bytes = C::kWeight + a.box * 128;
  a.stages = std::min(C::kMaxStages, C::kRing / a.stage_bytes);
  a.o = c.o;
  a.status = v.status;
  a.timeout_ns = v.timeout_ns;
  CUtensorMap w[2], t;
  for (int i = 0; i < c.weights; ++i)
    CHECK(map_bank(&w[i], c.dtype, c.w[i].p, c.K, c.N, 1, c.w[i].ld, 0,
                   kMode == kFfnAct ? 128 : 64));
  if (c.weights == 1) w[1] = w[0];
  CHECK(map_halves(&t, c.dtype, c.t, red, c.rows, halves, c.ldt, a.box));
  const int feat = (kPair ? 2 : 1) * (kMode == kFfnGated ? 64 : 128);
  const int ctas = a.splits * (kPair ? 2 : 1);
  return launch_clusters(ffn_cluster_kernel<kMode, kPair, T>,
                         (int)ceil_div(c.o.feat, feat) * a.tiles_t * ctas, ctas, C::kThreads,
                         C::kSmem, stream, w[0], w[1], t, a);
}

// The cluster kernel's plan for a call, if it has one.
template <int kMode>
ClusterPlan cluster_plan(const FfnCall& c, const FfnDevice& d) {
  constexpr bool kDA = kMode == kFfnDA;
  const int k = g_kernel.load();
  if (c.offsets != nullptr || (k != 0 && k != 3)) return {};
  const int blocks = (int)ceil_div(kDA ? c.N : c.K, kSlabK) * (kDA ? c.weights : 1);
  return plan_cluster(c.rows, c.o.feat, blocks, kMode == kFfnGated ? 64 : 128, d);
}

template <int kMode, class T>
int run_plan(const FfnCall& c, const ClusterPlan& plan, const DeviceView& v,
             cudaStream_t stream) {
  return plan.pair ? run_cluster<kMode, true, T>(c, plan, v, stream)
                   : run_cluster<kMode, false, T>(c, plan, v, stream);
}

template <bool kGated, int kTok, class T>
int run_stream(const FfnCall& c, const DeviceView& v, cudaStream_t stream) {
  using C = FfnStreamCfg<kTok>;
  CUtensorMap w[2], t, h;
  for (int i = 0; i < c.weights; ++i)
    CHECK(map_bank(&w[i], c.dtype, c.w[i].p, c.K, c.N, c.experts, c.w[i].ld, c.w[i].stride,
                   kGated ? 64 : 128));
  if (c.weights == 1) w[1] = w[0];
  CHECK(map_rows(&t, c.dtype, c.t, c.K, c.rows, c.ldt, 16));
  h = t;
  if (kTok > 16) CHECK(map_rows(&h, c.dtype, c.t, c.K, c.rows, c.ldt, 64));
  StreamArgs a = {};
  a.offsets = c.offsets;
  a.experts = c.experts;
  a.rows = c.rows;
  a.feat = c.N;
  a.feat_blocks = (int)ceil_div(c.N, kGated ? 64 : 128);
  a.red = c.K;
  a.red_blocks = (int)ceil_div(c.K, kSlabK);
  a.min_items = 16;
  a.status = v.status;
  a.timeout_ns = v.timeout_ns;
  Workspace ws;
  CHECK(ws.take(v, (size_t)v.sms * 2 * kTok * 128 * sizeof(float), stream, &a));
  return launch(ffn_stream_kernel<kGated, kTok, T>, v.sms, C::kThreads, C::smem_bytes(c.experts),
                stream, w[0], w[1], t, h, a, c.o);
}

// f with the activation as a constant.
template <class F>
void by_act(int act, F&& f) {
  switch (act) {
    case B200_ACT_RELU: f(ActCode<B200_ACT_RELU>()); break;
    case B200_ACT_SILU: f(ActCode<B200_ACT_SILU>()); break;
    case B200_ACT_GELU: f(ActCode<B200_ACT_GELU>()); break;
    case B200_ACT_GELU_TANH: f(ActCode<B200_ACT_GELU_TANH>()); break;
    case B200_ACT_SIGMOID: f(ActCode<B200_ACT_SIGMOID>()); break;
    default: f(ActCode<B200_ACT_NONE>()); break;
  }
}

// The streaming kernel spreads any number of tiles over the SMs, but takes 64 rows of an
// expert at a time and joins divided tiles through L2.  One matrix: where no cluster
// fits or is estimated slower (14336 x 4096 gated, 1 row: 41.0 us, pairs 45.3; 64 rows
// 45.6 and 47.2, 96 rows 53.4 and 48.5).  A bank: up to 64 rows an expert on average, 48
// in short contractions, and up to 256 where half of the pairs would have no tile (8 x
// 14336 x 4096 gated, 512 rows: 297 us, pairs 330; 1024 rows 361 and 332; 32 x 1032 x
// 1032, 1024 rows 30.5 and 31.9, 2048 rows 34.8 and 33.4; 4 x 744 x 6200, 400 rows 29
// and 36).  Where the steps lie, streaming's time over the pairs', banks of 8 x 8192, 16 x
// 4096, 32 x 1032 and 64 x 1024 features, skewed counts: K = 1032 at 32 rows an expert 0.90
// to 1.02, at 48 0.99 to 1.09; K = 2048 to 3584 at 48 0.90 to 1.01, at 64 (the pairs', by
// this rule) 0.92 to 1.03; K = 4096 and 6144 at 64 0.92 to 1.02, at 80 1.04 to 1.20.
template <bool kGated>
bool use_stream(const FfnCall& c, const ClusterPlan& plan, const DeviceView& v,
                const FfnDevice& d) {
  const int k = g_kernel.load();
  if (k != 0) return k == 1;
  if (c.offsets != nullptr) {
    if (c.rows <= (c.K >= 4096 ? 64ll : 48ll) * c.experts) return true;
    return c.rows <= 256ll * c.experts &&
           2 * c.experts * ceil_div(c.N, kGated ? 128 : 256) <=
               d.pairs[kGated ? kFfnGated : kFfnAct];
  }
  if (c.rows > 64) return false;
  const long long units = ceil_div(c.N, kGated ? 64 : 128), items = units * ceil_div(c.K, kSlabK);
  const double box = (double)ceil_div(c.rows, 16) * 16 * 128;
  const double us = 7.7 + 0.15 * c.rows +
                    (double)items * std::max((16384 + box) / 95e3 / v.sms, 16384 / 6.3e6);
  return us < plan.us;
}

template <bool kGated, class T>
int run_forward(const FfnCall& c, const DeviceView& v, const FfnDevice& d, cudaStream_t stream) {
  constexpr int kMode = kGated ? kFfnGated : kFfnAct;
  const ClusterPlan plan = cluster_plan<kMode>(c, d);
  if (use_stream<kGated>(c, plan, v, d)) {
    if (c.rows <= 16) return run_stream<kGated, 16, T>(c, v, stream);
    // A tile that holds most experts' rows: an expert with more reads its weights again.
    if constexpr (kGated) {
      if (c.rows > 64ll * c.experts) return run_stream<kGated, 256, T>(c, v, stream);
      if (c.rows > 24ll * c.experts && c.experts > 1)
        return run_stream<kGated, 128, T>(c, v, stream);
    }
    return run_stream<kGated, 64, T>(c, v, stream);
  }
  if (plan.splits > 0) return run_plan<kMode, T>(c, plan, v, stream);
  return run_pair<kMode, T>(c, v, d, stream);
}

template <bool kGated>
int run_product(FfnCall& c, cudaStream_t stream) {
  if (c.rows == 0 || c.N == 0) return B200_OK;
  DeviceView v;
  FfnDevice* d = nullptr;
  CHECK(ffn_device(&v, &d));
  if (c.experts == 0 || c.K == 0) {
    if (kGated) {  // act(0) * 0
      if (c.o.z != nullptr &&
          cudaMemset2DAsync(c.o.z, c.o.ldz * sizeof(float), 0, c.N * sizeof(float), 2ll * c.rows,
                            stream) != cudaSuccess)
        return B200_ERR_LAUNCH;
      return zero_rows(c.o.out, (int)c.o.ldo, c.N, c.rows, stream);
    }
    const int blocks = (int)std::min(ceil_div((long long)c.rows * c.N, 256), 8ll * v.sms);
    int st = B200_OK;
    by_act(c.o.act, [&](auto code) {
      constexpr int kAct = decltype(code)::value;
      st = c.dtype == B200_FP16
               ? launch(ffn_empty_kernel<kAct, __half>, blocks, 256, 0, stream, c.o, c.rows)
               : launch(ffn_empty_kernel<kAct, __nv_bfloat16>, blocks, 256, 0, stream, c.o, c.rows);
    });
    return st;
  }
  c.o.vec_out = on(c.o.out, 8) && (c.o.ldo & 3) == 0;
  c.o.vec_res = on(c.o.residual, 8) && (c.o.ldr & 3) == 0;
  return c.dtype == B200_FP16 ? run_forward<kGated, __half>(c, v, *d, stream)
                              : run_forward<kGated, __nv_bfloat16>(c, v, *d, stream);
}

int check_act(int act) {
  return act >= B200_ACT_NONE && act <= B200_ACT_SIGMOID ? B200_OK : B200_ERR_INVALID_ARGUMENT;
}

template <class T>
int launch_grad(const FfnGradArgs& a, bool gated, int act, int blocks, cudaStream_t stream) {
  int st = B200_OK;
  by_act(act, [&](auto code) {
    constexpr int kAct = decltype(code)::value;
    st = gated ? launch(ffn_grad_kernel<true, kAct, T>, blocks, 256, 0, stream, a)
               : launch(ffn_grad_kernel<false, kAct, T>, blocks, 256, 0, stream, a);
  });
  return st;
}

int run_grad(FfnGradArgs a, bool gated, int act, void* dbias, int dtype, cudaStream_t stream) {
  DeviceView v;
  FfnDevice* d = nullptr;
  CHECK(ffn_device(&v, &d));
  a.strips = (int)ceil_div(a.feat, 256);
  // About eight blocks to an SM, of 32 rows at least.  Up to 64 rows one block to a strip,
  // which then has the whole sum (x 4096, silu: 64 rows 5.8 us in one kernel, 65 rows 5.1 in
  // two, whose second launch and buffer cost the caller 3.4 us).
  const long long want = std::max(1ll, 8ll * v.sms / a.strips);
  a.block_rows = (int)std::max(dbias != nullptr && a.rows <= 64 ? 64ll : 32ll,
                               ceil_div(ceil_div(a.rows, want), 8) * 8);
  const int row_blocks = (int)ceil_div(a.rows, a.block_rows);
  PoolBuffer partial;
  if (row_blocks > 1 && dbias != nullptr) {
    CHECK(partial.take(v, (size_t)row_blocks * a.feat * sizeof(float), stream));
    a.partial = reinterpret_cast<float*>(partial.p);
  } else {
    a.dbias = dbias;
  }
  const int blocks = a.strips * row_blocks;
  const bool half = dtype == B200_FP16;
  CHECK(half ? launch_grad<__half>(a, gated, act, blocks, stream)
             : launch_grad<__nv_bfloat16>(a, gated, act, blocks, stream));
  if (a.partial == nullptr) return B200_OK;
  const int columns = (int)ceil_div(a.feat, 32);
  return half ? launch(ffn_bias_kernel<__half>, columns, 256, 0, stream, a.partial, row_blocks,
                       a.feat, static_cast<__half*>(dbias))
              : launch(ffn_bias_kernel<__nv_bfloat16>, columns, 256, 0, stream, a.partial,
                       row_blocks, a.feat, static_cast<__nv_bfloat16*>(dbias));
}

// ------------------------------------------------------------ norm, clipping
constexpr int kNormBlocks = 4;  // per SM

// The tables of one call: tensors in launches of up to kNormTensors.
int norm_tables(const b200_tensor* tensors, int n, int* at, NormTable* table) {
  table->tensors = table->chunks = 0;
  long long chunks = 0;
  while (*at < n && table->tensors < kNormTensors) {
    const b200_tensor& t = tensors[*at];
    const long long more = ceil_div(t.count, kNormChunk);
    if (chunks + more > 0x7FFFFFFFll - (1 << 20)) {
      if (table->tensors == 0) return B200_ERR_TOO_LARGE;
      break;
    }
    ++*at;
    if (t.count == 0) continue;
    table->t[table->tensors++] = {t.data, t.count, (int)chunks, t.type};
    chunks += more;
  }
  table->chunks = (int)chunks;
  return B200_OK;
}

int run_norm(const b200_tensor* tensors, int n, bool clip, float max_norm, float* norm,
             cudaStream_t stream) {
  if (n < 0 || (n > 0 && !tensors) || !norm) return B200_ERR_INVALID_ARGUMENT;
  if (clip && !(max_norm >= 0.0f)) return B200_ERR_INVALID_ARGUMENT;
  if (!on(norm, 4)) return B200_ERR_ALIGNMENT;
  for (int i = 0; i < n; ++i) {
    const b200_tensor& t = tensors[i];
    if (t.type != B200_BF16 && t.type != B200_FP16 && t.type != B200_FP32)
      return B200_ERR_INVALID_ARGUMENT;
    if (t.count < 0 || (t.count > 0 && !t.data)) return B200_ERR_INVALID_ARGUMENT;
    if (!on(t.data, t.type == B200_FP32 ? 4 : 2)) return B200_ERR_ALIGNMENT;
  }
  DeviceView v;
  FfnDevice* d = nullptr;
  CHECK(ffn_device(&v, &d));
  const int most = kNormBlocks * v.sms;
  // (a table holds kNormTensors tensors, or all the chunks that 31 bits count)
  NormTable table;
  int launches = 0, partials = 0;
  for (int at = 0; at < n; ++launches) CHECK(norm_tables(tensors, n, &at, &table));
  PoolBuffer sums;
  CHECK(sums.take(v, (size_t)std::max(launches, 1) * most * sizeof(double), stream));
  double* partial = reinterpret_cast<double*>(sums.p);
  for (int at = 0; at < n;) {
    CHECK(norm_tables(tensors, n, &at, &table));
    const int blocks = std::min(table.chunks, most);
    if (blocks == 0) continue;
    CHECK(launch(norm_kernel<>, blocks, kNormThreads, 0, stream, table, partial + partials));
    partials += blocks;
  }
  if (!clip || partials == 0)
    return launch(norm_finish_kernel<>, 1, kNormThreads, 0, stream, partial, partials, norm);
  for (int at = 0; at < n;) {
    CHECK(norm_tables(tensors, n, &at, &table));
    const int blocks = table.chunks;
    if (blocks == 0) continue;
    CHECK(launch(clip_kernel<>, blocks, kNormThreads, 0, stream, table, partial, partials,
                 max_norm, norm));
    norm = nullptr;  // (the first of them writes it)
  }
  return B200_OK;
}

}  // namespace

extern "C" {

int b200_ffn_act(const void* A, const void* W, const void* bias, const void* residual, void* C,
                 float* z, int rows, int N, int K, int lda, int ldw, int ldr, int ldc, int ldz,
                 int act, int dtype, void* stream) {
  CHECK(check_sizes(rows, 1, N, K, nullptr, dtype));
  CHECK(check_act(act));
  FfnCall c = {A, {{W, ldw, 0}, {}}, 1, nullptr, rows, 1, N, K, lda, {}, dtype};
  if (N > 0) CHECK(check_bank(c.w[0], rows > 0, N, K));
  CHECK(check_rows(A, lda, N > 0 ? rows : 0, K));
  CHECK(check_plain(C, ldc, rows, N, false));
  CHECK(check_plain(residual, ldr, rows, N, true));
  CHECK(check_plain(bias, N, 1, N, true));
  CHECK(check_z(z, ldz, rows, N));
  CHECK(check_units(ceil_div(rows, 16), 1, N, 1));
  c.o.out = C;
  c.o.ldo = ldc;
  c.o.z = z;
  c.o.ldz = ldz;
  c.o.bias = bias;
  c.o.residual = residual;
  c.o.ldr = ldr;
  c.o.feat = N;
  c.o.act = act;
  return run_product<false>(c, static_cast<cudaStream_t>(stream));
}

int b200_ffn_gated(const void* A, const void* Wg, const void* Wu, const int* offsets, void* H,
                   float* z, int rows, int experts, int N, int K, int lda, int ldg,
                   long long stride_g, int ldu, long long stride_u, int ldh, int ldz, int act,
                   int dtype, void* stream) {
  CHECK(check_sizes(rows, experts, N, K, offsets, dtype));
  CHECK(check_act(act));
  FfnCall c = {A, {{Wg, ldg, stride_g}, {Wu, ldu, stride_u}}, 2, offsets, rows, experts, N, K,
               lda, {}, dtype};
  if (rows > 0) {
    CHECK(check_bank(c.w[0], experts, N, K));
    CHECK(check_bank(c.w[1], experts, N, K));
  }
  CHECK(check_rows(A, lda, N > 0 && experts > 0 ? rows : 0, K));
  CHECK(check_plain(H, ldh, rows, N, false));
  CHECK(check_z(z, ldz, rows, N));
  CHECK(check_units(ceil_div(rows, 16), experts, N, 1));
  c.o.out = H;
  c.o.ldo = ldh;
  c.o.z = z;
  c.o.ldz = ldz;
  c.o.z_half = (long long)rows * ldz;
  c.o.feat = N;
  c.o.act = act;
  return run_product<true>(c, static_cast<cudaStream_t>(stream));
}

int b200_ffn_act_grad(const void* dC, const float* z, void* dz, void* dbias, int rows, int N,
                      int ldc, int ldz, int lddz, int act, int dtype, void* stream) {
  CHECK(check_sizes(rows, 1, N, 0, nullptr, dtype));
  CHECK(check_act(act));
  CHECK(check_rows(dC, ldc, rows, N));
  if (act != B200_ACT_NONE && !z && rows > 0 && N > 0) return B200_ERR_INVALID_ARGUMENT;
  CHECK(check_z(act != B200_ACT_NONE ? z : nullptr, ldz, rows, N));
  if (dz) CHECK(check_rows(dz, lddz, rows, N));
  CHECK(check_plain(dbias, N, 1, N, true));
  CHECK(check_units(ceil_div(rows, 32), 1, N, 1));
  if (N == 0 || (!dz && !dbias) || (rows == 0 && !dbias)) return B200_OK;
  if (rows == 0) return zero_rows(dbias, N, N, 1, static_cast<cudaStream_t>(stream));
  FfnGradArgs a = {};
  a.dout = dC;
  a.ldd = ldc;
  a.z = z;
  a.ldz = ldz;
  a.dz = dz;
  a.lddz = lddz;
  a.experts = 1;
  a.rows = rows;
  a.feat = N;
  return run_grad(a, false, act, dbias, dtype, static_cast<cudaStream_t>(stream));
}

int b200_ffn_gated_grad(const void* dH, const float* z, const int* offsets, void* dz, int rows,
                        int experts, int N, int ldh, int ldz, int lddz, int act, int dtype,
                        void* stream) {
  CHECK(check_sizes(rows, experts, N, 0, offsets, dtype));
  CHECK(check_act(act));
  CHECK(check_rows(dH, ldh, rows, N));
  CHECK(check_rows(dz, lddz, rows, N));
  if (!z && rows > 0 && N > 0) return B200_ERR_INVALID_ARGUMENT;
  CHECK(check_z(z, ldz, rows, N));
  CHECK(check_units(ceil_div(rows, 32), experts, N, 1));
  if (rows == 0 || N == 0 || experts == 0) return B200_OK;
  FfnGradArgs a = {};
  a.dout = dH;
  a.ldd = ldh;
  a.z = z;
  a.ldz = ldz;
  a.z_half = (long long)rows * ldz;
  a.dz = dz;
  a.lddz = lddz;
  a.dz_half = (long long)rows * lddz;
  a.offsets = offsets;
  a.experts = experts;
  a.rows = rows;
  a.feat = N;
  return run_grad(a, true, act, nullptr, dtype, static_cast<cudaStream_t>(stream));
}

int b200_ffn_da(const void* dz, const void* W0, const void* W1, const int* offsets, void* dA,
                int halves, int rows, int experts, int N, int K, int lddz, int ld0,
                long long stride0, int ld1, long long stride1, int lda, int dtype, void* stream) {
  CHECK(check_sizes(rows, experts, N, K, offsets, dtype));
  if (halves != 1 && halves != 2) return B200_ERR_INVALID_ARGUMENT;
  FfnCall c = {dz, {{W0, ld0, stride0}, {W1, ld1, stride1}}, halves, offsets, rows, experts, N, K,
               lddz, {}, dtype};
  for (int i = 0; i < halves && rows > 0; ++i) CHECK(check_bank(c.w[i], experts, N, K));
  CHECK(check_rows(dz, lddz, K > 0 && experts > 0 ? rows : 0, N));
  CHECK(check_plain(dA, lda, rows, K, false));
  CHECK(check_units(ceil_div(rows, 16), experts, K, 1));
  if (rows == 0 || K == 0) return B200_OK;
  DeviceView v;
  FfnDevice* d = nullptr;
  CHECK(ffn_device(&v, &d));
  if (experts == 0 || N == 0) return zero_rows(dA, lda, K, rows, static_cast<cudaStream_t>(stream));
  c.o.out = dA;
  c.o.ldo = lda;
  c.o.feat = K;
  c.o.act = B200_ACT_NONE;
  c.o.vec_out = on(dA, 8) && (lda & 3) == 0;
  const ClusterPlan plan = cluster_plan<kFfnDA>(c, *d);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (plan.splits > 0)
    return dtype == B200_FP16 ? run_plan<kFfnDA, __half>(c, plan, v, s)
                              : run_plan<kFfnDA, __nv_bfloat16>(c, plan, v, s);
  return dtype == B200_FP16 ? run_pair<kFfnDA, __half>(c, v, *d, s)
                            : run_pair<kFfnDA, __nv_bfloat16>(c, v, *d, s);
}

}  // extern "C"

namespace {

template <class T>
int run_dw(const void* dz, const void* A, const int* offsets, void* dW, int halves, int rows,
           int experts, int N, int K, int lddz, int lda, int dtype, cudaStream_t stream) {
  DeviceView v;
  FfnDevice* d = nullptr;
  CHECK(ffn_device(&v, &d));
  CUtensorMap tz, ta, ts;
  CHECK(map_halves(&tz, dtype, dz, N, rows, halves, lddz, 64));
  CHECK(map_rows(&ta, dtype, A, K, rows, lda, 64));
  const bool tma = tma_rows(dW, K);
  if (tma)
    CHECK(map_bank(&ts, dtype, dW, K, N, halves * experts, K, (long long)N * K, 32));
  else
    ts = ta;  // (not used: the kernel stores to `out`)
  FfnArgs a = {};
  PoolBuffer maps;
  if (offsets != nullptr) {
    CHECK(maps.take(v, (size_t)experts * 2 * sizeof(CUtensorMap), stream));
    CHECK(launch(ffn_maps_kernel<>, experts, 32, 0, stream, tz, ta, offsets, rows,
                 reinterpret_cast<CUtensorMap*>(maps.p)));
    a.maps = reinterpret_cast<const CUtensorMap*>(maps.p);
  }
  a.offsets = offsets;
  a.experts = experts;
  a.rows = rows;
  a.feat = N;
  a.cols = K;
  a.halves = halves;
  a.o.out = tma ? nullptr : dW;
  if (experts > kFewExperts)
    return launch_pair<kFfnDW, true, T>(a, tz, ta, tz, tz, ts, v, *d, stream);
  return launch_pair<kFfnDW, false, T>(a, tz, ta, tz, tz, ts, v, *d, stream);
}

}  // namespace

extern "C" {

int b200_ffn_dw(const void* dz, const void* A, const int* offsets, void* dW, int halves, int rows,
                int experts, int N, int K, int lddz, int lda, int dtype, void* stream) {
  CHECK(check_sizes(rows, experts, N, K, offsets, dtype));
  if (halves != 1 && halves != 2) return B200_ERR_INVALID_ARGUMENT;
  const bool any = experts > 0 && N > 0 && K > 0;
  if (!any) return B200_OK;
  CHECK(check_rows(dz, lddz, rows, N));
  CHECK(check_rows(A, lda, rows, K));
  if (!dW) return B200_ERR_INVALID_ARGUMENT;
  if (!on(dW, 2)) return B200_ERR_ALIGNMENT;
  CHECK(check_units(ceil_div(N, 256), 0, K, (long long)halves * experts));
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (rows == 0)
    return cudaMemsetAsync(dW, 0, (size_t)2 * halves * experts * N * K, s) == cudaSuccess
               ? B200_OK
               : B200_ERR_LAUNCH;
  return dtype == B200_FP16 ? run_dw<__half>(dz, A, offsets, dW, halves, rows, experts, N, K, lddz,
                                             lda, dtype, s)
                            : run_dw<__nv_bfloat16>(dz, A, offsets, dW, halves, rows, experts, N,
                                                    K, lddz, lda, dtype, s);
}

int b200_ffn_set_kernel(int kernel) {
  if (kernel < 0 || kernel > 3) return B200_ERR_INVALID_ARGUMENT;
  g_kernel.store(kernel);
  return B200_OK;
}

int b200_grad_norm(const b200_tensor* tensors, int n, float* norm, void* stream) {
  return run_norm(tensors, n, false, 0.0f, norm, static_cast<cudaStream_t>(stream));
}

int b200_clip_grads(const b200_tensor* tensors, int n, float max_norm, float* norm, void* stream) {
  return run_norm(tensors, n, true, max_norm, norm, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
