// Routing: each token's top-k experts, their softmax weights, and the order
// that sorts (token, slot) pairs by expert; rows moved there and back.
//
//   chosen     the k largest logits of a token, the lower index first on a
//              tie; NaN counts as largest, -inf is a closed expert: never
//              chosen, its slot stays empty (expert, row -1, weight 0)
//   weights    softmax over the chosen, or over all, experts; fp32
//   row        offsets[e] + the number of earlier pairs, by token then slot,
//              that chose e too: the order does not depend on timing
//   dispatch   xs[row(t, j)] = x[t]          combine  out[t] = sum_j w y[row]
//
// A warp holds a token's logits in registers (with more than 256 experts not all
// of them: 1 KB a thread is spilled there).  The tokens are cut into one
// chunk per block: counts per (chunk, expert) first, then every block adds
// up the chunks before its own and ranks its pairs (two launches; one when a
// single block does it all).  Moving rows is bound by memory: one block per
// token, every row read once and written once, sums in fp32.
// 8192 tokens, 64 experts, two each, width 4096: choose 6.6 us and rank 11.7
// (a chain of counts, barriers and ranks over 1024 threads; 3 MB), dispatch
// 36 (202 MB, 5.6 TB/s, 2 us of it the search for rows without a slot), combine
// 37 (202 MB, 5.4 TB/s), its gradient 59 (336 MB, 5.7 TB/s, the same), the
// logits' gradient 6.4.
#pragma once
#include "moe_groups.cuh"

namespace b200 {

constexpr int kRouteThreads = 1024;
constexpr int kRouteWarps = kRouteThreads / 32;
constexpr int kMaxTopK = 32;

// Logit types: 0 bf16, 1 f16, 2 f32.
struct RouteArgs {
  const void* logits;
  long long ld;
  int type;
  int tokens, experts, top_k;
  int chunk;        // tokens per block
  bool normalize;
  float* weights;   // tokens x top_k
  int* chosen;      // tokens x top_k
  int* rows;        // tokens x top_k
  int* sources;     // tokens * top_k
  int* offsets;     // experts + 1
  int* counts;      // blocks x experts (several blocks)
};

__device__ __forceinline__ float load_logit(const void* p, int type, long long i) {
  if (type == 2) return static_cast<const float*>(p)[i];
  if (type == 1) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

// An unsigned key in the order of the values: NaN above all, -0 = +0.
__device__ __forceinline__ uint32_t order_key(float v) {
  if (v != v) return 0xFFFFFFFFu;
  const uint32_t b = __float_as_uint(v + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
constexpr uint32_t kClosedKey = 0x007FFFFFu;  // order_key(-inf)

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

// A token's logits in a warp: expert i of the row is value i / 32 of lane i % 32.
template <int kPer>
__device__ __forceinline__ void load_token(const RouteArgs& a, int t, float (&v)[kPer]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int e = i * 32 + lane;
    v[i] = e < a.experts ? load_logit(a.logits, a.type, t * a.ld + e) : -INFINITY;
  }
}

template <int kPer>
__device__ __forceinline__ void choose_token(const RouteArgs& a, int t, const float (&v)[kPer],
                                             int* hist) {
  const int lane = threadIdx.x & 31;
  uint32_t key[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) key[i] = order_key(v[i]);
  float base = 0.0f, mine = 0.0f, sum = 0.0f;
  int slot_expert = -1;  // lane j keeps slot j
  for (int j = 0; j < a.top_k; ++j) {
    uint32_t best = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) best = max(best, key[i]);
    best = __reduce_max_sync(0xffffffffu, best);
    if (best <= kClosedKey) break;
    int at = 0x7FFFFFFF;
#pragma unroll
    for (int i = kPer - 1; i >= 0; --i)
      if (key[i] == best) at = i * 32 + lane;
    at = __reduce_min_sync(0xffffffffu, at);
    float val = 0.0f;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (at == i * 32 + lane) {
        val = v[i];
        key[i] = 0;
      }
    val = __shfl_sync(0xffffffffu, val, at & 31);
    if (j == 0) base = val;
    const float p = expf(val - base);
    if (a.normalize) sum += p;
    if (lane == j) {
      slot_expert = at;
      mine = p;
    }
  }
  if (!a.normalize) {
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (i * 32 + lane < a.experts) sum += expf(v[i] - base);
    sum = warp_sum(sum);
  }
  if (lane < a.top_k) {
    const long long at = (long long)t * a.top_k + lane;
    a.weights[at] = slot_expert >= 0 ? mine / sum : 0.0f;
    a.chosen[at] = slot_expert;
    if (slot_expert >= 0) atomicAdd(hist + slot_expert, 1);
  }
}

template <int kPer>
__device__ __forceinline__ void choose_chunk(const RouteArgs& a, int first, int last, int* hist) {
  for (int i = threadIdx.x; i < a.experts; i += kRouteThreads) hist[i] = 0;
  __syncthreads();
  // (a warp's next token is on its way while it chooses for this one)
  int t = first + (threadIdx.x >> 5);
  float v[kPer], next[kPer];
  if (t < last) load_token<kPer>(a, t, v);
  for (; t < last; t += kRouteWarps) {
    if (t + kRouteWarps < last) load_token<kPer>(a, t + kRouteWarps, next);
    choose_token<kPer>(a, t, v, hist);
#pragma unroll
    for (int i = 0; i < kPer; ++i) v[i] = next[i];
  }
  __syncthreads();
}

// Exclusive prefix sum of totals[0 .. n) by one warp; returns the sum.
__device__ __forceinline__ int scan_experts(int* totals, int n) {
  const int lane = threadIdx.x & 31;
  int run = 0;
  for (int base = 0; base < n; base += 32) {
    const int i = base + lane;
    const int own = i < n ? totals[i] : 0;
    int v = own;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, v, d);
      if (lane >= d) v += o;
    }
    if (i < n) totals[i] = run + v - own;
    run += __shfl_sync(0xffffffffu, v, 31);
  }
  return run;
}

// A warp's part of a chunk's pairs, [lo, hi) from `base`, in steps of 32.
struct RoutePart {
  long long base;
  int lo, hi;
  int first;  // the expert of pair lo + lane, -1 past the end
};
__device__ __forceinline__ RoutePart route_part(const RouteArgs& a, int first, int last) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int pairs = (last - first) * a.top_k;
  const int part = ((pairs + kRouteWarps - 1) / kRouteWarps + 31) & ~31;
  RoutePart p;
  p.base = (long long)first * a.top_k;
  p.lo = min(warp * part, pairs);
  p.hi = min(p.lo + part, pairs);
  p.first = p.lo + lane < p.hi ? a.chosen[p.base + p.lo + lane] : -1;
  return p;
}

// Rows of the chunk's pairs.  start[e]: offsets[e] + pairs of earlier chunks;
// cursor[warp][e]: next row of this warp's part of the chunk.
__device__ __forceinline__ void rank_chunk(const RouteArgs& a, const RoutePart& p,
                                           const int* start, int* cursor) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < kRouteWarps * a.experts; i += kRouteThreads) cursor[i] = 0;
  __syncthreads();
  int* mine = cursor + warp * a.experts;
  for (int i = p.lo + lane; i < p.hi; i += 32) {
    const int e = i == p.lo + lane ? p.first : a.chosen[p.base + i];
    if (e >= 0) atomicAdd(mine + e, 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < a.experts; e += kRouteThreads) {
    int at = start[e];
#pragma unroll 8
    for (int w = 0; w < kRouteWarps; ++w) {
      const int n = cursor[w * a.experts + e];
      cursor[w * a.experts + e] = at;
      at += n;
    }
  }
  __syncthreads();
  for (int i = p.lo; i < p.hi; i += 32) {
    const bool in = i + lane < p.hi;
    const int e = i == p.lo ? p.first : in ? a.chosen[p.base + i + lane] : -1;
    const unsigned int same = __match_any_sync(0xffffffffu, e);
    const int before = __popc(same & ((1u << lane) - 1u));
    int row = -1;
    if (e >= 0) {
      row = mine[e] + before;
      a.sources[row] = (int)((p.base + i + lane) / a.top_k);
    }
    __syncwarp();
    if (e >= 0 && before == 0) mine[e] += __popc(same);
    __syncwarp();
    if (in) a.rows[p.base + i + lane] = row;
  }
}

// Pairs that went nowhere leave rows without an expert at the end.
__device__ __forceinline__ void mark_unowned(const RouteArgs& a, int total) {
  const long long pairs = (long long)a.tokens * a.top_k;
  for (long long r = total + (long long)blockIdx.x * kRouteThreads + threadIdx.x; r < pairs;
       r += (long long)gridDim.x * kRouteThreads)
    a.sources[r] = -1;
}

// Dynamic shared memory: hist/start [experts], cursor [warps][experts].
template <int kPer>
__global__ void __launch_bounds__(kRouteThreads) route_choose_kernel(const RouteArgs a) {
  grid_wait();
  grid_launch_next();
  extern __shared__ int s_route[];
  int* hist = s_route;
  const int first = blockIdx.x * a.chunk;
  const int last = min(a.tokens, first + a.chunk);
  choose_chunk<kPer>(a, first, last, hist);
  if (gridDim.x > 1) {
    for (int e = threadIdx.x; e < a.experts; e += kRouteThreads)
      a.counts[(long long)blockIdx.x * a.experts + e] = hist[e];
    return;
  }
  __shared__ int total;
  if (threadIdx.x < 32) {
    const int n = scan_experts(hist, a.experts);
    if (threadIdx.x == 0) total = n;
  }
  __syncthreads();
  for (int e = threadIdx.x; e <= a.experts; e += kRouteThreads)
    a.offsets[e] = e < a.experts ? hist[e] : total;
  rank_chunk(a, route_part(a, first, last), hist, s_route + a.experts);
  mark_unowned(a, total);
}

__global__ void __launch_bounds__(kRouteThreads) route_rank_kernel(const RouteArgs a) {
  grid_wait();
  grid_launch_next();
  extern __shared__ int s_route[];
  int* start = s_route;                 // totals, then offsets, then + earlier chunks
  int* earlier = s_route + a.experts;   // (the cursors take this over)
  __shared__ int total;
  const int first = blockIdx.x * a.chunk;
  const RoutePart part = route_part(a, first, min(a.tokens, first + a.chunk));
  // Counts of all chunks and of the earlier ones: a thread adds up a share of
  // the chunks for one expert (16 loads in flight), shared memory the shares.
  for (int e = threadIdx.x; e < a.experts; e += kRouteThreads) start[e] = earlier[e] = 0;
  __syncthreads();
  const int shares = a.experts < kRouteThreads ? kRouteThreads / a.experts : 1;
  for (int i = threadIdx.x; i < shares * a.experts; i += kRouteThreads) {
    const int e = i % a.experts;
    int all = 0, before = 0;
#pragma unroll 16
    for (int b = i / a.experts; b < (int)gridDim.x; b += shares) {
      const int n = __ldg(a.counts + (long long)b * a.experts + e);
      all += n;
      before += b < (int)blockIdx.x ? n : 0;
    }
    atomicAdd(start + e, all);
    atomicAdd(earlier + e, before);
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    const int n = scan_experts(start, a.experts);
    if (threadIdx.x == 0) total = n;
  }
  __syncthreads();
  if (blockIdx.x == 0)
    for (int e = threadIdx.x; e <= a.experts; e += kRouteThreads)
      a.offsets[e] = e < a.experts ? start[e] : total;
  __syncthreads();
  for (int e = threadIdx.x; e < a.experts; e += kRouteThreads) start[e] += earlier[e];
  __syncthreads();
  rank_chunk(a, part, start, s_route + a.experts);
  mark_unowned(a, total);
}

// Gradient in the logits, one warp per token:
//   over the chosen:  w_j (dw_j - sum_i w_i dw_i) at chosen experts, else 0
//   over all:         p_e ([e chosen] dw_e - sum_j w_j dw_j)
template <int kPer>
__global__ void __launch_bounds__(256)
route_grad_kernel(const RouteArgs a, const float* __restrict__ dweights, void* dlogits) {
  grid_wait();
  grid_launch_next();
  const int lane = threadIdx.x & 31;
  const int t = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (t >= a.tokens) return;
  float v[kPer];
  if (!a.normalize) load_token<kPer>(a, t, v);
  const long long at = (long long)t * a.top_k + lane;
  const int e = lane < a.top_k ? a.chosen[at] : -1;
  const float w = e >= 0 ? a.weights[at] : 0.0f;
  const float dw = e >= 0 ? dweights[at] : 0.0f;
  const float inner = warp_sum(e >= 0 ? w * dw : 0.0f);
  // what the chosen experts get: their weights and the weights' gradients
  float share[kPer], hit[kPer];
  uint32_t took = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) share[i] = hit[i] = 0.0f;
  for (int j = 0; j < a.top_k; ++j) {
    const int ej = __shfl_sync(0xffffffffu, e, j);
    const float wj = __shfl_sync(0xffffffffu, w, j), dj = __shfl_sync(0xffffffffu, dw, j);
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (ej == i * 32 + lane) {
        share[i] = wj;
        hit[i] = dj;
        took |= 1u << i;
      }
  }
  float base = 0.0f, sum = 1.0f;
  const int top = __shfl_sync(0xffffffffu, e, 0);
  if (!a.normalize && top >= 0) {
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (i == top >> 5) base = v[i];
    base = __shfl_sync(0xffffffffu, base, top & 31);
    float part = 0.0f;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (i * 32 + lane < a.experts) part += expf(v[i] - base);
    sum = warp_sum(part);
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int ei = i * 32 + lane;
    if (ei >= a.experts) continue;
    const bool mine = took >> i & 1u;
    float g = 0.0f;
    if (a.normalize) {
      if (mine) g = share[i] * (hit[i] - inner);
    } else if (top >= 0 && v[i] != -INFINITY) {
      // (a closed expert has no share; NaN and inf take part as they are)
      g = (mine ? share[i] : expf(v[i] - base) / sum) * (hit[i] - inner);
    }
    const long long o = (long long)t * a.experts + ei;
    if (a.type == 2) static_cast<float*>(dlogits)[o] = g;
    else if (a.type == 1) static_cast<__half*>(dlogits)[o] = __float2half_rn(g);
    else static_cast<__nv_bfloat16*>(dlogits)[o] = __float2bfloat16_rn(g);
  }
}

// ------------------------------------------------------------------ moving rows
struct MoveArgs {
  const void* in;         // x, y or dout
  long long ld_in;
  const void* in2;        // combine's gradient: y
  long long ld_in2;
  void* out;              // xs, out or dy
  long long ld_out;
  const float* weights;   // tokens x top_k, or null: 1
  float* dweights;        // combine's gradient
  const int* rows;        // tokens x top_k
  const int* named;       // per sorted row a slot that may name it, or null
  int tokens, top_k, width;
};

// kVec elements of a row at once: 8 (16 bytes, aligned rows) or 1.
template <class T, int kVec>
struct Pack {
  T v[kVec];
};
template <class T, int kVec>
__device__ __forceinline__ Pack<T, kVec> load_pack(const void* base, long long i) {
  Pack<T, kVec> p;
  if constexpr (kVec == 8)
    *reinterpret_cast<uint4*>(&p) =
        __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(base) + i));
  else
    p.v[0] = static_cast<const T*>(base)[i];
  return p;
}
template <class T, int kVec>
__device__ __forceinline__ void store_pack(void* base, long long i, const Pack<T, kVec>& p) {
  if constexpr (kVec == 8)
    *reinterpret_cast<uint4*>(static_cast<T*>(base) + i) = *reinterpret_cast<const uint4*>(&p);
  else
    static_cast<T*>(base)[i] = p.v[0];
}
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }

// A token's rows and weights into shared memory; a row that is no row of the
// operand is treated as none.
__device__ __forceinline__ void load_slots(const MoveArgs& a, long long t, int* s_row, float* s_w) {
  if ((int)threadIdx.x < a.top_k) {
    const long long at = t * a.top_k + threadIdx.x;
    const int r = a.rows[at];
    s_row[threadIdx.x] = r >= 0 && r < (long long)a.tokens * a.top_k ? r : -1;
    s_w[threadIdx.x] = a.weights != nullptr ? a.weights[at] : 1.0f;
  }
  __syncthreads();
}

// Sorted rows that no slot names -- past the owned ones or, where slots were
// taken out of a routing, among them -- are zero.  named[r] is a slot that
// names row r, if there is any: memory that nobody cleared, so an entry counts
// only where that slot's row is r.
__global__ void __launch_bounds__(256)
mark_rows_kernel(const int* __restrict__ rows, int* __restrict__ named, int pairs) {
  grid_wait();
  grid_launch_next();
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < pairs; i += gridDim.x * 256ll) {
    const int r = rows[i];
    if (r >= 0 && r < pairs) named[r] = (int)i;
  }
}

// Token t's block zeroes those of rows t * top_k .. that no slot names.  Up to
// kScanPairs slots it looks through all of them itself; beyond, mark_rows_kernel
// has been there (a launch more, but no work that grows with the square).
// Dispatch, us, looking through / marked: 32 slots 2.5 / 5.1, 2048 4.8 / 5.2,
// 4096 7.8 / 6.5, 65532 691 / 57; with rows left as they are 2.3, 3.2, 4.6, 54.
constexpr int kScanPairs = 2048;
template <class T, int kVec>
__device__ __forceinline__ void zero_unnamed(const MoveArgs& a, long long t) {
  __shared__ uint32_t s_named[8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int pairs = a.tokens * a.top_k, first = (int)t * a.top_k;
  uint32_t bits = 0;
  if (a.named == nullptr) {
    for (int i = threadIdx.x; i < pairs; i += blockDim.x) {
      const uint32_t r = (uint32_t)(a.rows[i] - first);
      if (r < (uint32_t)a.top_k) bits |= 1u << r;
    }
    bits = __reduce_or_sync(0xffffffffu, bits);
  } else if (warp == 0) {
    const int at = lane < a.top_k ? a.named[first + lane] : -1;
    bits = __ballot_sync(0xffffffffu, (uint32_t)at < (uint32_t)pairs && a.rows[at] == first + lane);
  }
  if (lane == 0) s_named[warp] = bits;
  __syncthreads();
  bits = 0;
  for (int w = 0; w < (int)(blockDim.x >> 5); ++w) bits |= s_named[w];
  for (int j = 0; j < a.top_k; ++j) {
    if (bits >> j & 1u) continue;
    Pack<T, kVec> z;
#pragma unroll
    for (int i = 0; i < kVec; ++i) z.v[i] = round_one<T>(0.0f);
    for (int c = threadIdx.x * kVec; c < a.width; c += blockDim.x * kVec)
      store_pack<T, kVec>(a.out, (long long)(first + j) * a.ld_out + c, z);
  }
}

template <class T, int kVec>
__global__ void __launch_bounds__(256) dispatch_kernel(const MoveArgs a) {
  grid_wait();
  grid_launch_next();
  __shared__ int s_row[kMaxTopK];
  __shared__ float s_w[kMaxTopK];
  const long long t = blockIdx.x;
  load_slots(a, t, s_row, s_w);
  for (int c = threadIdx.x * kVec; c < a.width; c += blockDim.x * kVec) {
    const Pack<T, kVec> p = load_pack<T, kVec>(a.in, t * a.ld_in + c);
    for (int j = 0; j < a.top_k; ++j)
      if (s_row[j] >= 0) store_pack<T, kVec>(a.out, (long long)s_row[j] * a.ld_out + c, p);
  }
  zero_unnamed<T, kVec>(a, t);
}

template <class T, int kVec>
__global__ void __launch_bounds__(256) combine_kernel(const MoveArgs a) {
  grid_wait();
  grid_launch_next();
  __shared__ int s_row[kMaxTopK];
  __shared__ float s_w[kMaxTopK];
  const long long t = blockIdx.x;
  load_slots(a, t, s_row, s_w);
  for (int c = threadIdx.x * kVec; c < a.width; c += blockDim.x * kVec) {
    float sum[kVec];
#pragma unroll
    for (int i = 0; i < kVec; ++i) sum[i] = 0.0f;
#pragma unroll 4
    for (int j = 0; j < a.top_k; ++j) {
      if (s_row[j] < 0) continue;
      const Pack<T, kVec> p = load_pack<T, kVec>(a.in, (long long)s_row[j] * a.ld_in + c);
#pragma unroll
      for (int i = 0; i < kVec; ++i) sum[i] = fmaf(s_w[j], widen(p.v[i]), sum[i]);
    }
    Pack<T, kVec> o;
#pragma unroll
    for (int i = 0; i < kVec; ++i) o.v[i] = round_one<T>(sum[i]);
    store_pack<T, kVec>(a.out, t * a.ld_out + c, o);
  }
}

// dy[row] = w dout[t], dw[t, j] = <dout[t], y[row]>.  Slot by slot, without a
// barrier between them, so warps spread over the slots; dout comes from cache
// after the first.  (All of a token's loads ahead of its stores takes twice
// the registers and half the occupancy: 131 us against 108 for 16383 x 4 rows
// of 2048.)
template <class T, int kVec>
__global__ void __launch_bounds__(256) combine_grad_kernel(const MoveArgs a) {
  grid_wait();
  grid_launch_next();
  __shared__ int s_row[kMaxTopK];
  __shared__ float s_w[kMaxTopK];
  __shared__ float s_part[8][kMaxTopK];
  const long long t = blockIdx.x;
  load_slots(a, t, s_row, s_w);
#pragma unroll 1
  for (int j = 0; j < a.top_k; ++j) {
    const long long r = s_row[j];
    const float w = s_w[j];
    float dot = 0.0f;
    if (r >= 0) {
      for (int c = threadIdx.x * kVec; c < a.width; c += blockDim.x * kVec) {
        const Pack<T, kVec> y = load_pack<T, kVec>(a.in2, r * a.ld_in2 + c);
        const Pack<T, kVec> d = load_pack<T, kVec>(a.in, t * a.ld_in + c);
        Pack<T, kVec> o;
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          const float v = widen(d.v[i]);
          dot = fmaf(v, widen(y.v[i]), dot);
          o.v[i] = round_one<T>(w * v);
        }
        store_pack<T, kVec>(a.out, r * a.ld_out + c, o);
      }
    }
    dot = warp_sum(dot);
    if ((threadIdx.x & 31) == 0) s_part[threadIdx.x >> 5][j] = dot;
  }
  zero_unnamed<T, kVec>(a, t);
  // (zero_unnamed's barrier lies between the parts and their sum)
  if (a.dweights != nullptr && (int)threadIdx.x < a.top_k) {
    float all = 0.0f;
    for (int w = 0; w < (int)(blockDim.x >> 5); ++w) all += s_part[w][threadIdx.x];
    a.dweights[t * a.top_k + threadIdx.x] = all;
  }
}

}  // namespace b200
