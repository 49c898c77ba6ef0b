// Operands made readable for the products: offsets of 64 bits, rows that TMA
// cannot take.
#pragma once
#include <stdint.h>

#include "sm100_ptx.cuh"

namespace b200 {

// 64-bit offsets as the kernels read them: what 32 bits do not hold becomes
// something outside the rows, which build_groups clamps and reports.
__global__ void __launch_bounds__(256)
narrow_offsets_kernel(const long long* offsets, long long stride, int count, int* out) {
  grid_wait();
  grid_launch_next();
  for (int i = threadIdx.x; i < count; i += 256)
    out[i] = (int)min(max(offsets[i * stride], -1ll), 0x7FFFFFFFll);
}

// Copies an operand whose rows TMA cannot take (a row stride or base that is
// no multiple of 16 bytes) into rows that it can: `matrices` matrices of rows
// x cols 16-bit elements with unit column stride into rows of ld (a multiple
// of 8).  A thread makes 16 bytes of a row from the five words that hold them
// -- a row may start on any 2 bytes -- so loads and stores stay wide.  Bound
// by memory: each element read and written once.  With offsets, a bank: the
// matrices of experts without rows are left out.
__global__ void __launch_bounds__(256)
align_rows_kernel(const uint16_t* src, long long matrix_stride, long long row_stride, uint16_t* dst,
                  int matrices, int rows, int cols, int ld, const int* offsets) {
  grid_wait();
  grid_launch_next();
  const int groups = ld / 8;
  const long long total = (long long)matrices * rows * groups;
  const uintptr_t begin = reinterpret_cast<uintptr_t>(src);
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    const long long r = i / groups;
    const int c = (int)(i - r * groups) * 8;
    const int m = (int)(r / rows);
    if (offsets != nullptr && offsets[m + 1] <= offsets[m]) continue;
    const uint16_t* from = src + m * matrix_stride + (r - (long long)m * rows) * row_stride + c;
    const uintptr_t at = reinterpret_cast<uintptr_t>(from);
    uint32_t w[4];
    // Words that reach past the row are read only inside the operand.
    if (c + 9 <= cols && (at & ~3ull) >= begin) {
      const uint32_t* words = reinterpret_cast<const uint32_t*>(at & ~3ull);
      uint32_t v[5];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = __ldcg(words + j);
      if (at & 2) {
        v[4] = __ldcg(words + 4);
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
