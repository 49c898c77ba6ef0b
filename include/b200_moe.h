/* C ABI of the sm_100a mixture-of-experts operators (libb200gemm.so).
 *
 * The products of b200_gemm.h where the weight is a bank of experts and every
 * row of the other operand names one.  Conventions are those of b200_gemm.h:
 * device pointers, strides in elements, asynchronous on `stream`, a status
 * code back (B200_OK ...), pipeline waits bounded and reported through
 * b200_gemm_device_status.
 *
 * Rows are sorted by expert: expert e owns rows offsets[e] .. offsets[e+1]-1
 * of the row operands; offsets is experts + 1 int32 values in device memory,
 * read by the kernels (nothing waits for the host).  An expert may own no
 * row.  Rows before offsets[0] or from offsets[experts] on belong to no
 * expert.  Offsets that decrease or leave [0, rows] are clamped, and device
 * error word 0x100A is set (b200_gemm_device_status).
 * Element types: dtype = B200_BF16 or B200_FP16, for every 16-bit operand of
 * a call; sums are fp32, rounded to the output once. */
#ifndef B200_MOE_H_
#define B200_MOE_H_

#include <stddef.h>
#include <stdint.h>

#include "b200_gemm.h"

#ifdef __cplusplus
extern "C" {
#endif

#define B200_BF16 0
#define B200_FP16 1
#define B200_MAX_EXPERTS 1024

/* C[r, :] = A[r, :] B[e]^T for the rows r of every expert e.
 * A: rows x K, stride lda.  B: experts x N x K, row stride ldb, matrix stride
 * expert_stride (elements).  C: rows x N, stride ldc; rows of no expert are
 * set to zero.  Pointers 16-byte aligned; lda, ldb, ldc and expert_stride
 * multiples of 8; lda, ldb >= K, ldc >= N, expert_stride >= N * ldb (or
 * experts <= 1); sizes >= 0.  K == 0 gives zeros. */
int b200_grouped_gemm(const void* A, const void* B, void* C, const int* offsets, int rows,
                      int experts, int N, int K, int lda, int ldb, long long expert_stride,
                      int ldc, int dtype, void* stream);

/* Gradient of the above in A: dA[r, :] = dC[r, :] B[e].  dC: rows x N, stride
 * ldc; dA: rows x K, stride lda; rows of no expert are set to zero. */
int b200_grouped_gemm_da(const void* dC, const void* B, void* dA, const int* offsets, int rows,
                         int experts, int N, int K, int ldc, int ldb, long long expert_stride,
                         int lda, int dtype, void* stream);

/* Gradient in B: dB[e] = sum over expert e's rows r of dC[r, :]^T A[r, :];
 * every element of every N x K matrix is written, zeros for an expert
 * without rows.  Rows of no expert are never read into a sum. */
int b200_grouped_gemm_db(const void* dC, const void* A, void* dB, const int* offsets, int rows,
                         int experts, int N, int K, int ldc, int lda, int ldb,
                         long long expert_stride, int dtype, void* stream);

/* Kernel for b200_grouped_gemm and _da: 0 = chosen by rows per expert
 * (default), 1 = the streaming kernel (few rows), 2 = the pair kernel. */
int b200_grouped_set_kernel(int kernel);

/* ---- 4-bit weights with group scales ---------------------------------------
 * A weight is (q - z) * s: q in 0..15, one scale s (16-bit, the type of A) and
 * one zero point z in 0..15 (8 where none are given) per `group` consecutive
 * k of a row; group = 32, 64 or 128 and K a multiple of it.
 *
 * b200_w4_pack lays a matrix, or a bank of them, out once in the order the
 * kernel reads it.  q: experts x N x K/2 bytes, the low nibble the even k;
 * scales: experts x N x K/group; zeros: the same shape, one byte each, or
 * NULL; all contiguous.  packed: b200_w4_packed_bytes bytes, 16-byte aligned
 * (zeros != 0 when zero points are given). */
int b200_w4_packed_bytes(int experts, int N, int K, int group, int zeros, size_t* bytes);
int b200_w4_pack(const void* q, const void* scales, const void* zeros, void* packed, int experts,
                 int N, int K, int group, void* stream);

/* C[r, :] = A[r, :] W[e]^T with packed weights.  offsets as for
 * b200_grouped_gemm, or NULL for experts = 1: every row takes the one matrix.
 * A: rows x K, stride lda; C: rows x N, stride ldc; alignment as above.  The
 * weights enter as exact integers, the scales multiply fp32 sums.  Any number
 * of rows; made for few (the weights are read once per 64 rows of an expert,
 * 32 when group is 32). */
int b200_w4_gemm(const void* A, const void* packed, void* C, const int* offsets, int rows,
                 int experts, int N, int K, int group, int zeros, int lda, int ldc, int dtype,
                 void* stream);

#ifdef __cplusplus
}
#endif

#endif /* B200_MOE_H_ */
