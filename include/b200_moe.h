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
 * Rows, columns, tokens and widths are at most 2^31 - 2^25 (B200_ERR_TOO_LARGE).
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
#define B200_FP32 2 /* logits only */
#define B200_MAX_EXPERTS 1024
#define B200_MAX_TOP_K 32

/* C[r, :] = A[r, :] B[e]^T for the rows r of every expert e.
 * A: rows x K, stride lda.  B: experts x N x K, row stride ldb, matrix stride
 * expert_stride (elements).  C: rows x N, stride ldc; rows of no expert are
 * set to zero.  What is read (here A and B) has 16-byte aligned pointers and
 * strides that are multiples of 8 (b200_align_rows makes such rows); what is
 * written (here C) may lie anywhere its elements can.  lda, ldb >= K, ldc >=
 * N, expert_stride >= N * ldb (or experts <= 1); sizes >= 0.  K == 0 gives
 * zeros. */
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

/* Copies `matrices` matrices of rows x cols 16-bit elements (strides in
 * elements, unit column stride, any alignment) into rows of ld elements, ld a
 * multiple of 8 and dst 16-byte aligned: what the products above can read.
 * The columns past cols are zero. */
int b200_align_rows(const void* src, long long matrix_stride, long long row_stride, void* dst,
                    int matrices, int rows, int cols, int ld, void* stream);

/* The same for a bank whose offsets say which experts own rows (or NULL): the
 * matrices of the others are not copied, and what dst holds of them is left. */
int b200_align_bank(const void* src, long long matrix_stride, long long row_stride, void* dst,
                    const int* offsets, int matrices, int rows, int cols, int ld, void* stream);

/* int64 offsets as the calls here take them: `count` values, `stride` elements
 * apart, to int32.  One that 32 bits do not hold becomes -1 or 2^31 - 1: outside
 * the rows, as it was, and so clamped and reported. */
int b200_narrow_offsets(const void* offsets, long long stride, int count, int* out, void* stream);

/* Kernel for b200_grouped_gemm and _da: 0 = chosen by rows per expert
 * (default), 1 = the streaming kernel (few rows), 2 = the pair kernel. */
int b200_grouped_set_kernel(int kernel);

/* ---- Routing -----------------------------------------------------------------
 * Each token's top_k experts (largest logits; the lower index first on a tie;
 * NaN counts as largest), their softmax weights and the order that sorts the
 * tokens * top_k (token, slot) pairs by expert, pairs of one expert by token
 * and slot.  An expert whose logit is -inf is closed: never chosen.  A slot
 * left empty for want of open experts has expert -1, row -1 and weight 0.
 * logits: tokens x experts, stride ld, type B200_BF16, _FP16 or _FP32.
 * normalize != 0: softmax over the chosen experts, else over all of them.
 * weights, chosen, rows: tokens x top_k; sources: tokens * top_k, the token of
 * each sorted row, -1 past the last owned row; offsets: experts + 1, what
 * b200_grouped_gemm takes.  top_k <= experts, top_k <= 32. */
int b200_route(const void* logits, int tokens, int experts, long long ld, int type, int top_k,
               int normalize, float* weights, int* chosen, int* rows, int* sources, int* offsets,
               void* stream);

/* Gradient of the weights in the logits; dlogits: tokens x experts,
 * contiguous, of the logits' type; zero at closed experts. */
int b200_route_grad(const void* logits, int tokens, int experts, long long ld, int type, int top_k,
                    int normalize, const int* chosen, const float* weights, const float* dweights,
                    void* dlogits, void* stream);

/* xs[rows[t][j], :] = x[t, :]; rows of xs that no slot names are zero (of a
 * routing as b200_route makes it those from the last entry of offsets on; of one
 * that slots were taken out of, theirs too).  A row outside 0 .. tokens * top_k
 * - 1 is an empty slot; no two slots name the same row.  total: the last entry
 * of offsets, not null (its value is not needed).  xs: tokens * top_k rows.
 * 16-bit elements; strides in elements; 16-byte aligned rows of a multiple of 8
 * elements move fastest, any others work. */
int b200_dispatch(const void* x, const int* rows, const int* total, void* xs, int tokens, int top_k,
                  int width, long long ldx, long long ldxs, int dtype, void* stream);

/* out[t, :] = sum over t's non-empty slots j of weights[t][j] y[rows[t][j], :],
 * summed in fp32 in slot order, rounded once; weights NULL: all 1 (which is
 * the gradient of b200_dispatch). */
int b200_combine(const void* y, const float* weights, const int* rows, void* out, int tokens,
                 int top_k, int width, long long ldy, long long ldo, int dtype, void* stream);

/* Gradients of b200_combine: dy[rows[t][j], :] = weights[t][j] dout[t, :] (rows
 * that no slot names zero; total as above), dweights[t][j] = <dout[t, :], y[rows[t][j], :]> (0 at
 * empty slots; dweights may be NULL). */
int b200_combine_grad(const void* dout, const void* y, const float* weights, const int* rows,
                      const int* total, void* dy, float* dweights, int tokens, int top_k, int width,
                      long long ldo, long long ldy, long long lddy, int dtype, void* stream);

/* ---- 4-bit weights with group scales ---------------------------------------
 * A weight is (q - z) * s: q in 0..15, one scale s (16-bit, the type of A) and
 * one zero point z in 0..15 (8 where none are given) per `group` consecutive
 * k of a row; group = 32, 64 or 128 and K a multiple of it.
 *
 * b200_w4_pack lays a matrix, or a bank of them, out once in the order the
 * kernel reads it.  q: experts x N x K/2 bytes, the low nibble the even k;
 * scales: experts x N x K/group; zeros: the same shape, one byte each, or
 * NULL; all contiguous.  packed: b200_w4_packed_bytes bytes, 16-byte aligned
 * (zeros != 0 when zero points are given).  Of a zero point above 15 the low four
 * bits are taken and device error word 0x100B is set. */
int b200_w4_packed_bytes(int experts, int N, int K, int group, int zeros, size_t* bytes);
int b200_w4_pack(const void* q, const void* scales, const void* zeros, void* packed, int experts,
                 int N, int K, int group, void* stream);

/* C[r, :] = A[r, :] W[e]^T with packed weights.  offsets as for
 * b200_grouped_gemm, or NULL for experts = 1: every row takes the one matrix.
 * A: rows x K, stride lda; C: rows x N, stride ldc; alignment as there.  The
 * weights enter unrounded: as exact integers whose fp32 sums the scales
 * multiply, or (bf16 in groups of 32 and 64, from 33 rows on, a bank from 17 rows
 * an expert on average) as the sum of two bf16, exact for scales of 2^-120 and
 * more.  The result is then rounded once.  With an infinite scale the first way
 * gives the sum's sign times infinity, the second the sum of infinite weights,
 * NaN where their signs differ or q = z.  Any number of rows (the weights are read
 * once per 8 to 256 rows of an expert). */
int b200_w4_gemm(const void* A, const void* packed, void* C, const int* offsets, int rows,
                 int experts, int N, int K, int group, int zeros, int lda, int ldc, int dtype,
                 void* stream);

#ifdef __cplusplus
}
#endif

#endif /* B200_MOE_H_ */
