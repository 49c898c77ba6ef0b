// The end of a feed-forward product, shared by its kernels: 16 tokens x 128
// accumulator rows, staged in shared memory so that a thread finds what belongs
// together (a feature's gate and up product lie in different TMEM lanes) and
// rows are written in long pieces.
//
//   gated: rows 0..63 are gate products, 64..127 the up products of the same 64
//          features; h = act(g) * u
//   else:  128 features; y = act(acc + bias) + residual
//
// All of it in fp32, rounded once.  With z the pre-activations are kept in fp32:
// rounding them to 16 bits would put errors as large as the result's own
// rounding into the gradient two more times.
#pragma once
#include "ffn_act.cuh"
#include "moe_groups.cuh"

namespace b200 {

struct FfnOut {
  void* out;
  long long ldo;
  float* z;               // null: not kept
  long long ldz, z_half;  // z_half: from the gate's to the up products'
  const void* bias;
  const void* residual;
  long long ldr;
  int feat;  // output columns
  int act;
  int vec_out, vec_res;  // rows on 8 bytes
};

constexpr int kStageTokens = 16;
constexpr int kFfnStageBytes = kStageTokens * 128 * 4;

template <class T>
__device__ __forceinline__ float widen(uint16_t bits);
template <>
__device__ __forceinline__ float widen<__nv_bfloat16>(uint16_t bits) {
  return __uint_as_float((uint32_t)bits << 16);
}
template <>
__device__ __forceinline__ float widen<__half>(uint16_t bits) {
  return __half2float(__ushort_as_half(bits));
}

template <class T>
__device__ __forceinline__ void store_four(T* p, const float (&v)[4]) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_pair<T>(v[0], v[1]), pack_pair<T>(v[2], v[3]));
}

// One warp's part of the staging: lane's accumulator row `quarter * 32 + lane`
// of 16 tokens.
__device__ __forceinline__ void stage_put(uint32_t stage, int quarter, const float (&v)[16]) {
  const uint32_t at = stage + (uint32_t)(quarter * 32 + (threadIdx.x & 31)) * 4u;
#pragma unroll
  for (int t = 0; t < kStageTokens; ++t) st_shared_u32(at + t * 512u, __float_as_uint(v[t]));
}

// What a thread keeps over a tile: its features' bias, and whether all of the tile's
// features are there, in rows that it reads and writes four at a time.
template <bool kGated>
struct FfnTile {
  float bias[kGated ? 1 : 8];
  bool whole;
};

// feat0: the first feature of the 64 or 128; tid: 0..127 of the group of warps.
template <bool kGated, class T>
__device__ __forceinline__ void ffn_tile(const FfnOut& o, int feat0, int tid, FfnTile<kGated>& s) {
  s.whole = feat0 + (kGated ? 64 : 128) <= o.feat && o.vec_out &&
            (kGated || o.residual == nullptr || o.vec_res);
  if constexpr (!kGated) {
    const int f = feat0 + (tid & 15) * 4;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        s.bias[h * 4 + i] =
            s.whole && o.bias != nullptr
                ? widen<T>(static_cast<const uint16_t*>(o.bias)[f + h * 64 + i]) : 0.0f;
    }
  }
}

// A thread's part of 16 staged tokens: token tid / 16 and eight further, features
// 4 (tid % 16) on and, not gated, 64 further.  All of it is there (FfnTile::whole, 16
// tokens), so the loads and the arithmetic of all values run side by side.  The residual
// is asked for before the barrier that the staged values wait at.
template <bool kGated, int kAct, class T>
__device__ __forceinline__ void ffn_rows_whole(const FfnOut& o, uint32_t stage, uint32_t bar,
                                               int quarter, const float (&acc)[16],
                                               long long row0, int feat0, int tid,
                                               const FfnTile<kGated>& s) {
  const int f = feat0 + (tid & 15) * 4;
  const long long row = row0 + (tid >> 4);
  uint2 res[2][2];
  const bool add = !kGated && o.residual != nullptr;
  if constexpr (!kGated) {
    const T* r = static_cast<const T*>(o.residual) + row * o.ldr + f;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        res[j][h] = add ? *reinterpret_cast<const uint2*>(r + j * 8 * o.ldr + h * 64)
                        : make_uint2(0, 0);
  }
  stage_put(stage, quarter, acc);
  named_bar_sync(bar, 128);
  const uint32_t at = stage + (uint32_t)(tid >> 4) * 512u + (uint32_t)(tid & 15) * 16u;
  float v[2][2][4];
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int h = 0; h < 2; ++h)
      ld_shared_v4_f32(at + j * 8u * 512u + h * 256u, v[j][h][0], v[j][h][1], v[j][h][2],
                       v[j][h][3]);
  T* out = static_cast<T*>(o.out) + row * o.ldo + f;
  if constexpr (!kGated) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[j][h][i] += s.bias[h * 4 + i];
  }
  if (o.z != nullptr) {
    float* z = o.z + row * o.ldz + f;
    const long long second = kGated ? o.z_half : 64;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float(&w)[4] = v[j][h];
        *reinterpret_cast<float4*>(z + j * 8 * o.ldz + h * second) =
            make_float4(w[0], w[1], w[2], w[3]);
      }
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    activate<kAct>(v[j][0]);
    if constexpr (!kGated) activate<kAct>(v[j][1]);
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    T* to = out + j * 8 * o.ldo;
    if constexpr (kGated) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[j][0][i] *= v[j][1][i];
      store_four(to, v[j][0]);
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float(&w)[4] = v[j][h];
        w[0] += widen<T>((uint16_t)res[j][h].x);
        w[1] += widen<T>((uint16_t)(res[j][h].x >> 16));
        w[2] += widen<T>((uint16_t)res[j][h].y);
        w[3] += widen<T>((uint16_t)(res[j][h].y >> 16));
        store_four(to + h * 64, w);
      }
    }
  }
  named_bar_sync(bar, 128);
}

// The same where features or tokens (of which `tokens` are there) end, or rows lie on
// odd addresses: a warp takes every fourth token and a thread every 32nd feature, so that
// 32 neighbours are written by one instruction wherever the row begins.  (Four features to
// a thread, as above, took a store each: 2036 rows over 32 experts of 1031 x 1032 47 us.)
template <bool kGated, int kAct, class T>
__device__ __forceinline__ void ffn_rows_ragged(const FfnOut& o, uint32_t stage, long long row0,
                                                int tokens, int feat0, int tid) {
  constexpr int kN = kGated ? 2 : 4;
  const int f = feat0 + (tid & 31), n = o.feat - f;
  float bias[kN];
  if constexpr (!kGated) {
#pragma unroll
    for (int i = 0; i < kN; ++i)
      bias[i] = o.bias != nullptr && 32 * i < n
                    ? widen<T>(static_cast<const uint16_t*>(o.bias)[f + 32 * i]) : 0.0f;
  }
#pragma unroll 2
  for (int t = tid >> 5; t < kStageTokens; t += 4) {
    if (t >= tokens) break;
    const long long row = row0 + t;
    const uint32_t at = stage + (uint32_t)t * 512u + (uint32_t)(tid & 31) * 4u;
    float v[kN], u[kN];
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      v[i] = ld_shared_f32(at + i * 128u);
      if constexpr (kGated) u[i] = ld_shared_f32(at + 256u + i * 128u);
      else v[i] += bias[i];
    }
    if (o.z != nullptr) {
      float* z = o.z + row * o.ldz + f;
#pragma unroll
      for (int i = 0; i < kN; ++i)
        if (32 * i < n) {
          z[32 * i] = v[i];
          if constexpr (kGated) z[o.z_half + 32 * i] = u[i];
        }
    }
    activate<kAct>(v);
    T* out = static_cast<T*>(o.out) + row * o.ldo + f;
    const uint16_t* r = static_cast<const uint16_t*>(o.residual) + row * o.ldr + f;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      if (32 * i >= n) continue;
      if constexpr (kGated) v[i] *= u[i];
      else if (o.residual != nullptr) v[i] += widen<T>(r[32 * i]);
      out[32 * i] = round_one<T>(v[i]);
    }
  }
}

// A group of four warps: `v` staged, finished and the staging free again.
template <bool kGated, int kAct, class T>
__device__ __forceinline__ void ffn_finish(const FfnOut& o, uint32_t stage, uint32_t bar,
                                           int quarter, const float (&v)[16], long long row0,
                                           int tokens, int feat0, int tid,
                                           const FfnTile<kGated>& s) {
  if (s.whole && tokens >= kStageTokens) {
    ffn_rows_whole<kGated, kAct, T>(o, stage, bar, quarter, v, row0, feat0, tid, s);
  } else {
    stage_put(stage, quarter, v);
    named_bar_sync(bar, 128);
    ffn_rows_ragged<kGated, kAct, T>(o, stage, row0, tokens, feat0, tid);
    named_bar_sync(bar, 128);
  }
}

}  // namespace b200
