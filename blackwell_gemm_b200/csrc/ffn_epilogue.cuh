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
constexpr int kFfnStageBytes = kStageTokens * 128 * 4;  // (a power of two)

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
template <int kFrom = 0>
__device__ __forceinline__ void stage_put(uint32_t at, const float (&v)[16]) {
  if constexpr (kFrom < kStageTokens) {
    st_shared_f32_at<kFrom * 512>(at, v[kFrom]);
    stage_put<kFrom + 1>(at, v);
  }
}

// What a thread keeps over a tile: where its part of the first token begins, its features'
// bias, and whether all of the tile's features are there, in rows that it reads and writes
// four at a time.
template <bool kGated, class T>
struct FfnTile {
  T* out;
  const T* residual;
  float* z;
  F32x2 bias[kGated ? 1 : 4];
  bool whole;
};

// feat0: the first feature of the 64 or 128; row0: the tile's first row; tid: 0..127 of the
// group of warps.  A thread has token tid / 16 and eight further of 16, features 4 (tid %
// 16) on and, not gated, 64 further.
template <bool kGated, class T>
__device__ __forceinline__ void ffn_tile(const FfnOut& o, int feat0, long long row0, int tid,
                                         FfnTile<kGated, T>& s) {
  const int f = feat0 + (tid & 15) * 4;
  const long long row = row0 + (tid >> 4);
  s.whole = feat0 + (kGated ? 64 : 128) <= o.feat && o.vec_out &&
            (kGated || o.residual == nullptr || o.vec_res);
  s.out = static_cast<T*>(o.out) + row * o.ldo + f;
  s.residual = static_cast<const T*>(o.residual) + row * o.ldr + f;
  s.z = o.z + row * o.ldz + f;
  if constexpr (!kGated) {
    if (o.bias != nullptr && s.whole) {
      const uint16_t* b = static_cast<const uint16_t*>(o.bias) + f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint16_t* p = b + (i >> 1) * 64 + (i & 1) * 2;
        s.bias[i] = pair_of(widen<T>(p[0]), widen<T>(p[1]));
      }
    }
  }
}

// A thread's residual of 16 tokens, `c` from the tile's first.  The pair and cluster kernels
// ask for it a round ahead: from HBM it takes longer than all the rest that is done with
// them (4096 rows x 8192 x 512 with gelu 59 us; with a residual 82, and 65 so).
template <bool kGated, class T>
struct FfnResidual {
  uint2 v[2][2];
  __device__ __forceinline__ void fetch(const FfnOut& o, int c, int tokens,
                                        const FfnTile<kGated, T>& s) {
    if constexpr (!kGated) {
      if (o.residual == nullptr || !s.whole || tokens < kStageTokens) return;
      const T* r = s.residual + c * o.ldr;
      const T* r8 = r + 8 * o.ldr;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        v[0][h] = *reinterpret_cast<const uint2*>(r + h * 64);
        v[1][h] = *reinterpret_cast<const uint2*>(r8 + h * 64);
      }
    }
  }
};

template <class T>
__device__ __forceinline__ F32x2 widen_pair(uint32_t w) {
  return pair_of(widen<T>((uint16_t)w), widen<T>((uint16_t)(w >> 16)));
}

// A thread's part of 16 staged tokens, `c` from the tile's first.  All of it is there
// (FfnTile::whole, 16 tokens), so the arithmetic of all values runs side by side.
template <bool kGated, int kAct, class T>
__device__ __forceinline__ void ffn_rows_whole(const FfnOut& o, uint32_t stage, int c, int tid,
                                               const FfnTile<kGated, T>& s,
                                               const FfnResidual<kGated, T>& res) {
  const uint32_t at = stage + (uint32_t)(tid >> 4) * 512u + (uint32_t)(tid & 15) * 16u;
  float v[2][2][4];
  ld_shared_v4_f32_at<0>(at, v[0][0]);
  ld_shared_v4_f32_at<256>(at, v[0][1]);
  ld_shared_v4_f32_at<8 * 512>(at, v[1][0]);
  ld_shared_v4_f32_at<8 * 512 + 256>(at, v[1][1]);
  if constexpr (!kGated) {
    if (o.bias != nullptr) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float(&w)[4] = v[j][i >> 1];
          const int k = (i & 1) * 2;
          halves_of(add2(pair_of(w[k], w[k + 1]), s.bias[i]), w[k], w[k + 1]);
        }
    }
  }
  if (o.z != nullptr) {
    float* z = s.z + c * o.ldz;
    float* z8 = z + 8 * o.ldz;
    const long long second = kGated ? o.z_half : 64;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float(&a)[4] = v[0][h];
      const float(&b)[4] = v[1][h];
      *reinterpret_cast<float4*>(z + h * second) = make_float4(a[0], a[1], a[2], a[3]);
      *reinterpret_cast<float4*>(z8 + h * second) = make_float4(b[0], b[1], b[2], b[3]);
    }
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    activate<kAct>(v[j][0]);
    if constexpr (!kGated) activate<kAct>(v[j][1]);
  }
  T* to = s.out + c * o.ldo;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    if constexpr (kGated) {
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        float(&w)[4] = v[j][0];
        halves_of(mul2(pair_of(w[i], w[i + 1]), pair_of(v[j][1][i], v[j][1][i + 1])), w[i],
                  w[i + 1]);
      }
      store_four(to, v[j][0]);
    } else {
      if (o.residual != nullptr) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float(&w)[4] = v[j][h];
          halves_of(add2(pair_of(w[0], w[1]), widen_pair<T>(res.v[j][h].x)), w[0], w[1]);
          halves_of(add2(pair_of(w[2], w[3]), widen_pair<T>(res.v[j][h].y)), w[2], w[3]);
        }
      }
      store_four(to, v[j][0]);
      store_four(to + 64, v[j][1]);
    }
    to += 8 * o.ldo;
  }
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

// A group of four warps: `v`, 16 tokens from the tile's token c on, staged and finished.
// kTwo: there are two stagings, taken in turn (`turn`), so that one barrier is enough --
// who writes the same one again has passed the barrier of the other, where all that read
// this one had come by -- and the warps overlap; else the staging is free again at the end.
template <bool kGated, int kAct, class T, bool kTwo>
__device__ __forceinline__ void ffn_finish(const FfnOut& o, uint32_t stage, uint32_t* turn,
                                           uint32_t bar, int quarter, const float (&v)[16],
                                           long long row0, int c, int tokens, int feat0, int tid,
                                           const FfnTile<kGated, T>& s,
                                           const FfnResidual<kGated, T>& res) {
  if constexpr (kTwo) {
    stage += *turn;
    *turn ^= (uint32_t)kFfnStageBytes;
  }
  stage_put(stage + (uint32_t)(quarter * 32 + (threadIdx.x & 31)) * 4u, v);
  named_bar_sync(bar, 128);
  if (s.whole && tokens >= kStageTokens)
    ffn_rows_whole<kGated, kAct, T>(o, stage, c, tid, s, res);
  else
    ffn_rows_ragged<kGated, kAct, T>(o, stage, row0 + c, tokens, feat0, tid);
  if constexpr (!kTwo) named_bar_sync(bar, 128);
}

}  // namespace b200
