// Ragged groups of rows: expert e of a bank owns rows offsets[e] ..
// offsets[e+1] - 1 of the token operand.  The offsets are read on the device
// (no host synchronisation), so every kernel first builds the same table in
// its shared memory and walks its work from it.
#pragma once
#include <stdint.h>

#include "gemm_kernel.cuh"

namespace b200 {

// wait_bounded for a barrier that has usually completed already.
__device__ __forceinline__ bool wait_ready(uint32_t bar, uint32_t parity, const WaitCtx& w,
                                           int code) {
  if (mbar_test_wait(bar, parity)) return true;
  return wait_slow(bar, parity, w, code, true);
}

// The same with nothing called (a kernel that moves registers between its
// warps may not call functions).  draining: the abort word does not end it.
__device__ __forceinline__ bool wait_inline(uint32_t bar, uint32_t parity, const WaitCtx& w,
                                            int code, bool draining = false) {
  if (mbar_test_wait(bar, parity)) return true;
  const unsigned long long t0 = globaltimer_ns();
  for (;;) {
#pragma unroll 1
    for (int i = 0; i < 32; ++i)
      if (mbar_try_wait(bar, parity)) return true;
    if (!draining && ld_volatile_shared(w.abort_local) != 0) return false;
    if (globaltimer_ns() - t0 > w.timeout_ns) {
      atomicCAS(w.status, 0, code);
      asm volatile("st.volatile.shared.u32 [%0], %1;" :: "r"(w.abort_local), "r"(1u) : "memory");
      return false;
    }
  }
}

// End of a producing thread: its last copies have landed before the CTA may
// leave, also where a wait elsewhere ran out.  `stage` and `phase` are what
// comes next, `full` the ring's barriers.
template <int kStages>
__device__ __forceinline__ void drain_copies(uint32_t full, uint32_t stage, uint32_t phase,
                                             long long issued, const WaitCtx& w) {
#pragma unroll 1
  for (int i = 0; i < kStages && i < issued; ++i) {
    if (stage == 0) { stage = kStages; phase ^= 1u; }
    --stage;
    if (!wait_inline(full + stage * 8u, phase, w, kErrWaitDrain, true)) break;
  }
}

constexpr int kMaxExperts = 1024;
// Device error word: offsets that fall or leave [0, rows] (they are clamped).
constexpr int kErrOffsets = 0x100A;
// The same: 4-bit zero points above 15 (their low four bits were packed).
constexpr int kErrZeroPoint = 0x100B;

__host__ __device__ constexpr int group_table_bytes(int experts) {
  return ((2 * (experts + 1) * 4 + 15) / 16) * 16;
}

// One warp: s_off[0..E] = the offsets clamped to [0, rows] and made
// non-decreasing (so no later index can leave the operands whatever the
// offsets hold); s_tiles[e] = token tiles of `tile` rows before expert e.
// Returns true when the offsets had to be changed.
__device__ __forceinline__ bool build_groups(const int* offsets, int experts, int rows, int tile,
                                             int* s_off, int* s_tiles) {
  const int lane = threadIdx.x & 31;
  int top = 0;
  bool bad = false;
  for (int base = 0; base <= experts; base += 32) {
    const int i = base + lane;
    const int raw = i <= experts ? offsets[i] : rows;
    int v = min(max(raw, 0), rows);
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, v, d);
      if (lane >= d) v = max(v, o);
    }
    v = max(v, top);
    if (i <= experts) {
      s_off[i] = v;
      bad |= v != raw;
    }
    top = __shfl_sync(0xffffffffu, v, 31);
  }
  __syncwarp();
  int sum = 0;
  if (lane == 0) s_tiles[0] = 0;
  for (int base = 0; base < experts; base += 32) {
    const int i = base + lane;
    int v = i < experts ? (s_off[i + 1] - s_off[i] + tile - 1) / tile : 0;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, v, d);
      if (lane >= d) v += o;
    }
    v += sum;
    if (i < experts) s_tiles[i + 1] = v;
    sum = __shfl_sync(0xffffffffu, v, 31);
  }
  return __any_sync(0xffffffffu, bad);
}

// 64-bit offsets as the kernels read them: what 32 bits do not hold becomes
// something outside the rows, which build_groups clamps and reports.
__global__ void __launch_bounds__(256)
narrow_offsets_kernel(const long long* __restrict__ offsets, long long stride, int count,
                      int* __restrict__ out) {
  grid_wait();
  grid_launch_next();
  for (int i = threadIdx.x; i < count; i += 256)
    out[i] = (int)min(max(offsets[i * stride], -1ll), 0x7FFFFFFFll);
}

// The 16-bit output formats: round to nearest even, two at a time or one.
template <class T>
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack_pair<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack_pair<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <class T>
__device__ __forceinline__ T round_one(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 round_one<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half round_one<__half>(float v) {
  return __float2half_rn(v);
}
template <class T>
constexpr int kFormat = 0;  // tcgen05 16-bit format codes: 0 = f16, 1 = bf16
template <>
constexpr int kFormat<__nv_bfloat16> = 1;

// Rows no expert owns, [0, first) and [last, rows), are zero in an output of
// `cols` columns; thread `t` of `threads` writes its share.
template <class T>
__device__ __forceinline__ void zero_unowned_rows(T* out, long long ld, int cols, int first,
                                                  int last, int rows, long long t,
                                                  long long threads) {
  const bool wide = (ld & 7) == 0 && (reinterpret_cast<uintptr_t>(out) & 15u) == 0;
  const int groups = (cols + 7) / 8;
  const long long total = (long long)(first + rows - last) * groups;
  for (long long i = t; i < total; i += threads) {
    const long long r = i / groups;
    const int c = (int)(i - r * groups) * 8;
    T* p = out + (r < first ? r : r - first + last) * ld + c;
    if (wide && c + 8 <= cols) {
      *reinterpret_cast<uint4*>(p) = make_uint4(0, 0, 0, 0);
    } else {
      for (int j = 0; j < 8 && c + j < cols; ++j) p[j] = round_one<T>(0.0f);
    }
  }
}

// Copies an operand whose rows TMA cannot take (a row stride or base that is
// no multiple of 16 bytes) into rows that it can: `matrices` matrices of rows
// x cols 16-bit elements with unit column stride into rows of ld (a multiple
// of 8).  A thread makes 16 bytes of a row from the five words that hold them
// -- a row may start on any 2 bytes -- so loads and stores stay wide.  Bound
// by memory: each element read and written once.
__global__ void __launch_bounds__(256)
align_rows_kernel(const uint16_t* __restrict__ src, long long matrix_stride, long long row_stride,
                  uint16_t* __restrict__ dst, int matrices, int rows, int cols, int ld) {
  grid_wait();
  grid_launch_next();
  const int groups = ld / 8;
  const long long total = (long long)matrices * rows * groups;
  const uintptr_t begin = reinterpret_cast<uintptr_t>(src);
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    const long long r = i / groups;
    const int c = (int)(i - r * groups) * 8;
    const int m = (int)(r / rows);
    const uint16_t* from = src + m * matrix_stride + (r - (long long)m * rows) * row_stride + c;
    const uintptr_t at = reinterpret_cast<uintptr_t>(from);
    uint32_t w[4];
    // Words that reach past the row are read only inside the operand.
    if (c + 9 <= cols && (at & ~3ull) >= begin) {
      const uint32_t* words = reinterpret_cast<const uint32_t*>(at & ~3ull);
      uint32_t v[5];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = __ldg(words + j);
      if (at & 2) {
        v[4] = __ldg(words + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = __funnelshift_r(v[j], v[j + 1], 16);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = v[j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t lo = c + 2 * j < cols ? from[2 * j] : 0;
        const uint32_t hi = c + 2 * j + 1 < cols ? from[2 * j + 1] : 0;
        w[j] = lo | hi << 16;
      }
    }
    *reinterpret_cast<uint4*>(dst + r * ld + c) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

}  // namespace b200
