// The 2-norm of many tensors together, and their scaling by it.
//
//   norm = sqrt(sum x^2),  x *= min(1, max_norm / (norm + 1e-6))
//
// A launch takes a table of tensors in its parameters -- nothing is copied to the
// device, so a captured graph holds all it needs -- and cuts them into chunks of
// 16384 elements, dealt to the blocks in turn.  Eight elements' squares are added in
// fp32 and those sums in fp64; where such a sum leaves the range in which fp32 keeps
// its precision (a square overflows or is subnormal) the eight are squared in fp64
// instead.  Every block leaves its sum; whoever needs the norm adds them all in one
// order, so no atomics and the same bits every time.
//
// Bound by HBM: read once for the norm, read and written for the scale.  Four blocks to an
// SM walk the chunks for the norm (950 MB 142 us, 6.7 TB/s; eight 167); for the scale each
// chunk has a block of its own, which keeps reads and writes further apart (299 us, 6.4
// TB/s; four blocks to an SM 404, eight 337).  Chunks are scaled from the last to the
// first, so that what the first pass read last still lies in L2, and past it (120 MB: 49 us
// where plain accesses take 53).
#pragma once
#include "ffn_grad.cuh"

namespace b200 {

struct NormTensor {
  void* data;
  long long count;
  int first;  // chunk
  int type;
};

constexpr int kNormTensors = 320;  // of one launch (7.5 KiB of parameters)
constexpr int kNormChunk = 16384;
constexpr int kNormThreads = 256;

struct NormTable {
  int tensors, chunks;
  NormTensor t[kNormTensors];
};

// The tensor that chunk c belongs to.
__device__ __forceinline__ int norm_find(const NormTable& table, int c) {
  int lo = 0, hi = table.tensors - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (table.t[mid].first <= c) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ float norm_widen(const float* p) { return *p; }
template <class T>
__device__ __forceinline__ float norm_widen(const T* p) {
  return widen<T>(*reinterpret_cast<const uint16_t*>(p));
}
__device__ __forceinline__ void norm_round(float* p, float v) { *p = v; }
template <class T>
__device__ __forceinline__ void norm_round(T* p, float v) { *p = round_one<T>(v); }

template <class T>
struct NormVector {  // 16 bytes
  static constexpr int kN = 16 / sizeof(T);
  uint4 w;
  __device__ __forceinline__ void widen_all(float (&v)[kN]) const {
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        v[i] = __uint_as_float(x[i]);
      } else {
        v[2 * i] = widen<T>((uint16_t)x[i]);
        v[2 * i + 1] = widen<T>((uint16_t)(x[i] >> 16));
      }
    }
  }
  __device__ __forceinline__ void round_all(const float (&v)[kN]) {
    uint32_t x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) x[i] = __float_as_uint(v[i]);
      else x[i] = pack_pair<T>(v[2 * i], v[2 * i + 1]);
    }
    w = make_uint4(x[0], x[1], x[2], x[3]);
  }
};

// Elements [0, n) from p: `head` to the first 16-byte boundary, whole vectors, rest.
template <class T>
__device__ __forceinline__ void norm_span(const T* p, int n, int* head, int* vectors) {
  const int off = (int)(reinterpret_cast<uintptr_t>(p) & 15u);
  int h = off == 0 ? 0 : (16 - off) / (int)sizeof(T);
  if (h > n) h = n;
  *head = h;
  *vectors = (n - h) / (16 / (int)sizeof(T));
}

template <int kN>
__device__ __forceinline__ double norm_add(const float (&v)[kN]) {
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < kN; ++i) s = fmaf(v[i], v[i], s);
  if (s > 0x1p-90f && s < 0x1p126f) return (double)s;
  // Squares that fp32 does not hold, or nothing but zeros.
  double d = 0.0;
#pragma unroll
  for (int i = 0; i < kN; ++i) d = fma((double)v[i], (double)v[i], d);
  return d;
}

template <class T>
__device__ __forceinline__ double norm_chunk(const T* p, int n) {
  constexpr int kN = NormVector<T>::kN;
  constexpr int kDepth = 4;  // loads in flight
  int head, vectors;
  norm_span(p, n, &head, &vectors);
  double sum = 0.0;
  const int edge = n - vectors * kN;  // elements before and after the vectors
  if ((int)threadIdx.x < edge) {
    const int i = (int)threadIdx.x < head ? (int)threadIdx.x : (int)threadIdx.x + vectors * kN;
    const double x = norm_widen(p + i);
    sum = x * x;
  }
  const uint4* q = reinterpret_cast<const uint4*>(p + head);
  int i = threadIdx.x;
  for (; i + (kDepth - 1) * kNormThreads < vectors; i += kDepth * kNormThreads) {
    NormVector<T> x[kDepth];
#pragma unroll
    for (int j = 0; j < kDepth; ++j) x[j].w = __ldcg(q + i + j * kNormThreads);
#pragma unroll
    for (int j = 0; j < kDepth; ++j) {
      float v[kN];
      x[j].widen_all(v);
      sum += norm_add(v);
    }
  }
  for (; i < vectors; i += kNormThreads) {
    NormVector<T> x;
    x.w = __ldcg(q + i);
    float v[kN];
    x.widen_all(v);
    sum += norm_add(v);
  }
  return sum;
}

template <class T>
__device__ __forceinline__ void scale_chunk(T* p, int n, float scale) {
  constexpr int kN = NormVector<T>::kN;
  constexpr int kDepth = 4;
  int head, vectors;
  norm_span(p, n, &head, &vectors);
  const int edge = n - vectors * kN;
  if ((int)threadIdx.x < edge) {
    const int i = (int)threadIdx.x < head ? (int)threadIdx.x : (int)threadIdx.x + vectors * kN;
    norm_round(p + i, norm_widen(p + i) * scale);
  }
  uint4* q = reinterpret_cast<uint4*>(p + head);
  int i = threadIdx.x;
  for (; i + (kDepth - 1) * kNormThreads < vectors; i += kDepth * kNormThreads) {
    NormVector<T> x[kDepth];
#pragma unroll
    for (int j = 0; j < kDepth; ++j) x[j].w = __ldcs(q + i + j * kNormThreads);
#pragma unroll
    for (int j = 0; j < kDepth; ++j) {
      float v[kN];
      x[j].widen_all(v);
#pragma unroll
      for (int e = 0; e < kN; ++e) v[e] *= scale;
      x[j].round_all(v);
      __stcs(q + i + j * kNormThreads, x[j].w);
    }
  }
  for (; i < vectors; i += kNormThreads) {
    NormVector<T> x;
    x.w = q[i];
    float v[kN];
    x.widen_all(v);
#pragma unroll
    for (int e = 0; e < kN; ++e) v[e] *= scale;
    x.round_all(v);
    q[i] = x.w;
  }
}

// The sum over the block, on every thread.
__device__ __forceinline__ double norm_block_sum(double v) {
  __shared__ double warps[kNormThreads / 32];
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int i = 0; i < kNormThreads / 32; ++i) s += warps[i];
  return s;
}

// partial[block] = the sum of the squares of its chunks.
template <int kUnused = 0>
__global__ void __launch_bounds__(kNormThreads)
norm_kernel(const __grid_constant__ NormTable table, double* partial) {
  grid_wait();
  grid_launch_next();
  double sum = 0.0;
  for (int c = blockIdx.x; c < table.chunks; c += gridDim.x) {
    const NormTensor& t = table.t[norm_find(table, c)];
    const long long at = (long long)(c - t.first) * kNormChunk;
    const int n = (int)min((long long)kNormChunk, t.count - at);
    sum += t.type == B200_FP32   ? norm_chunk(static_cast<const float*>(t.data) + at, n)
           : t.type == B200_FP16 ? norm_chunk(static_cast<const __half*>(t.data) + at, n)
                                 : norm_chunk(static_cast<const __nv_bfloat16*>(t.data) + at, n);
  }
  sum = norm_block_sum(sum);
  if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

__device__ __forceinline__ double norm_total(const double* partial, int partials) {
  double sum = 0.0;
  for (int i = threadIdx.x; i < partials; i += kNormThreads) sum += __ldcg(partial + i);
  return sqrt(norm_block_sum(sum));
}

// One block: *norm from all partial sums.
template <int kUnused = 0>
__global__ void __launch_bounds__(kNormThreads)
norm_finish_kernel(const double* partial, int partials, float* norm) {
  grid_wait();
  grid_launch_next();
  const double n = norm_total(partial, partials);
  if (threadIdx.x == 0) *norm = (float)n;
}

// A block to a chunk; each adds the partial sums up for itself.
template <int kUnused = 0>
__global__ void __launch_bounds__(kNormThreads)
clip_kernel(const __grid_constant__ NormTable table, const double* partial, int partials,
            float max_norm, float* norm) {
  grid_wait();
  grid_launch_next();
  const double n = norm_total(partial, partials);
  if (norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n;
  const double ratio = (double)max_norm / (n + 1e-6);
  if (ratio >= 1.0) return;
  const float scale = (float)ratio;  // (of a norm that is not a number, not one either)
  const int c = table.chunks - 1 - (int)blockIdx.x;
  const NormTensor& t = table.t[norm_find(table, c)];
  const long long at = (long long)(c - t.first) * kNormChunk;
  const int count = (int)min((long long)kNormChunk, t.count - at);
  if (t.type == B200_FP32) scale_chunk(static_cast<float*>(t.data) + at, count, scale);
  else if (t.type == B200_FP16) scale_chunk(static_cast<__half*>(t.data) + at, count, scale);
  else scale_chunk(static_cast<__nv_bfloat16*>(t.data) + at, count, scale);
}

}  // namespace b200
