// The elementwise step of the feed-forward gradients, between their products:
//
//   gated  dz[0] = dh * u * act'(g),  dz[1] = dh * act(g)
//   act    dz = dc * act'(z),  dbias = the sum of its rows before rounding
//
// z (g and u) is fp32 as the forward product left it.  dz is rounded to the
// operands' type, because the products that follow take 16-bit operands: an error
// of half a step in each element, which over a sum of N or of rows is as large as
// the gradient's own last rounding.
//
// Bound by HBM: gated reads 10 and writes 4 bytes an element (4095 x 14336: 128 us, 6.4
// TB/s), act 6 and 2 (8191 x 8192 with the bias' sums: 105 us, 5.1 TB/s; four rows'
// loads in flight, with two 113).  A block takes 256 columns, a thread eight of them and
// every eighth of its rows.
#pragma once
#include "ffn_epilogue.cuh"

namespace b200 {

struct FfnGradArgs {
  const void* dout;
  long long ldd;
  const float* z;
  long long ldz, z_half;
  void* dz;  // null: only the bias
  long long lddz, dz_half;
  float* partial;      // (row blocks, N) sums, or null
  void* dbias;         // the sums themselves, rounded, where one block takes all rows
  const int* offsets;  // null: all rows
  int experts, rows, feat;
  int strips;      // blocks along a row; the rest of the grid goes over the rows
  int block_rows;
};

__device__ __forceinline__ void load_eight(const float* p, int n, float (&v)[8]) {
  if (n >= 8) {
    const float4 a = __ldcg(reinterpret_cast<const float4*>(p));
    const float4 b = __ldcg(reinterpret_cast<const float4*>(p) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? __ldcg(p + i) : 0.0f;
  }
}

template <class T>
__device__ __forceinline__ void load_eight(const T* p, int n, float (&v)[8]) {
  const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
  if (n >= 8) {
    const uint4 w = __ldcg(reinterpret_cast<const uint4*>(h));
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = widen<T>((uint16_t)x[i]);
      v[2 * i + 1] = widen<T>((uint16_t)(x[i] >> 16));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? widen<T>(__ldcg(h + i)) : 0.0f;
  }
}

template <class T>
__device__ __forceinline__ void store_eight(T* p, int n, const float (&v)[8]) {
  if (n >= 8) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_pair<T>(v[0], v[1]), pack_pair<T>(v[2], v[3]),
                                              pack_pair<T>(v[4], v[5]), pack_pair<T>(v[6], v[7]));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = round_one<T>(v[i]);
  }
}

// dout, z and dz have rows on 16 bytes.
template <bool kGated, int kAct, class T>
__global__ void __launch_bounds__(256)
ffn_grad_kernel(const FfnGradArgs a) {
  __shared__ float sums[kGated ? 1 : 8][256];
  grid_wait();
  grid_launch_next();
  const int lane = threadIdx.x & 31, part = threadIdx.x >> 5;
  const int block = blockIdx.x / a.strips, strip = blockIdx.x - block * a.strips;
  const int f = strip * 256 + lane * 8, n = a.feat - f;
  int lo = block * a.block_rows, hi = min(lo + a.block_rows, a.rows);
  if (a.offsets != nullptr) {
    // The owned rows, as build_groups has them: from the first offset to the
    // largest of the clamped ones.
    int end = 0;
    for (int i = lane; i <= a.experts; i += 32) end = max(end, min(a.offsets[i], a.rows));
    end = __reduce_max_sync(0xffffffffu, end);
    lo = max(lo, min(max(a.offsets[0], 0), a.rows));
    hi = min(hi, end);
  }
  float total[8] = {};
  if (n > 0) {
#pragma unroll(kGated ? 2 : 4)
    for (int r = lo + part; r < hi; r += 8) {
      float d[8], z[8];
      load_eight<T>(static_cast<const T*>(a.dout) + r * a.ldd + f, n, d);
      if constexpr (kGated) {
        float u[8], g[8], slope[8];
        load_eight(a.z + r * a.ldz + f, n, z);
        load_eight(a.z + a.z_half + r * a.ldz + f, n, u);
        activate_slope<kAct>(z, g, slope);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          slope[i] = times_slope<kAct>(d[i] * u[i], slope[i]);
          g[i] = d[i] * g[i];
        }
        T* to = static_cast<T*>(a.dz) + r * a.lddz + f;
        store_eight(to, n, slope);
        store_eight(to + a.dz_half, n, g);
      } else {
        if constexpr (kAct != B200_ACT_NONE) {
          float y[8], slope[8];
          load_eight(a.z + r * a.ldz + f, n, z);
          activate_slope<kAct>(z, y, slope);
#pragma unroll
          for (int i = 0; i < 8; ++i) d[i] = times_slope<kAct>(d[i], slope[i]);
        }
        if (a.dz != nullptr) store_eight(static_cast<T*>(a.dz) + r * a.lddz + f, n, d);
#pragma unroll
        for (int i = 0; i < 8; ++i) total[i] += d[i];
      }
    }
  }
  if constexpr (!kGated) {
    if (a.partial == nullptr && a.dbias == nullptr) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) sums[part][lane * 8 + i] = total[i];
    __syncthreads();
    const int col = strip * 256 + threadIdx.x;
    if (col < a.feat) {
      float s = 0.0f;
#pragma unroll
      for (int p = 0; p < 8; ++p) s += sums[p][threadIdx.x];
      if (a.partial != nullptr) a.partial[(long long)block * a.feat + col] = s;
      else static_cast<T*>(a.dbias)[col] = round_one<T>(s);
    }
  }
}

// dbias[n] = the row blocks' sums: 32 columns to a block, each warp every eighth of the
// sums in order, and the eight of them in order.
template <class T>
__global__ void __launch_bounds__(256)
ffn_bias_kernel(const float* partial, int blocks, int feat, T* __restrict__ dbias) {
  __shared__ float sums[8][32];
  grid_wait();
  grid_launch_next();
  const int lane = threadIdx.x & 31, part = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + lane;
  float s = 0.0f;
  if (col < feat) {
#pragma unroll 4
    for (int b = part; b < blocks; b += 8) s += __ldcg(partial + (long long)b * feat + col);
  }
  sums[part][lane] = s;
  __syncthreads();
  if (part != 0 || col >= feat) return;
#pragma unroll
  for (int p = 1; p < 8; ++p) s += sums[p][lane];
  dbias[col] = round_one<T>(s);
}

// C = act(bias) + residual, and z = bias: a product with an empty contraction.
template <int kAct, class T>
__global__ void __launch_bounds__(256)
ffn_empty_kernel(const FfnOut o, int rows) {
  grid_wait();
  grid_launch_next();
  const long long total = (long long)rows * o.feat;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    const long long r = i / o.feat;
    const int f = (int)(i - r * o.feat);
    float v[1] = {o.bias != nullptr
                      ? widen<T>(static_cast<const uint16_t*>(o.bias)[f]) : 0.0f};
    if (o.z != nullptr) o.z[r * o.ldz + f] = v[0];
    activate<kAct>(v);
    if (o.residual != nullptr)
      v[0] += widen<T>(static_cast<const uint16_t*>(o.residual)[r * o.ldr + f]);
    static_cast<T*>(o.out)[r * o.ldo + f] = round_one<T>(v[0]);
  }
}

}  // namespace b200
