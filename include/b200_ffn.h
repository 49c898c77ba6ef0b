/* C ABI of the sm_100a feed-forward operators (libb200gemm.so): products with
 * the activation, gate, bias and residual of a transformer's feed-forward layer
 * in their epilogue, their gradients, and the norm and clipping of many gradients.
 *
 * Conventions are those of b200_gemm.h and b200_moe.h: device pointers, strides
 * in elements, asynchronous on `stream`, a status code back, pipeline waits
 * bounded and reported through b200_gemm_device_status; dtype = B200_BF16 or
 * B200_FP16 for every 16-bit operand of a call; sums are fp32, rounded to the
 * output once; extents at most 2^31 - 2^25 (B200_ERR_TOO_LARGE).  What is read
 * by rows has 16-byte aligned pointers and strides that are multiples of 8
 * (b200_align_rows makes such rows); what is written, and a residual and a bias,
 * may lie anywhere its elements can.
 *
 * offsets: as in b200_moe.h, experts + 1 int32 values in device memory; or NULL
 * for experts = 1: every row takes the one matrix. */
#ifndef B200_FFN_H_
#define B200_FFN_H_

#include <stddef.h>
#include <stdint.h>

#include "b200_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Activations.  s: the logistic function, Phi: the normal distribution's. */
#define B200_ACT_NONE 0
#define B200_ACT_RELU 1      /* max(z, 0); up to z = 0 nothing comes back, inf and NaN neither */
#define B200_ACT_SILU 2      /* z s(z) */
#define B200_ACT_GELU 3      /* z Phi(z) */
#define B200_ACT_GELU_TANH 4 /* z (1 + tanh(c (z + 0.044715 z^3))) / 2, c = sqrt(2 / pi) */
#define B200_ACT_SIGMOID 5   /* s(z) */

/* C = act(A W^T + bias) + residual.  A: rows x K; W: N x K; bias: N or NULL;
 * residual: rows x N or NULL; C: rows x N (not overlapping what is read, but it
 * may be the residual itself).  z: NULL, or rows x N fp32 that receive the
 * activation's argument (16-byte aligned, ldz >= N a multiple of 4). */
int b200_ffn_act(const void* A, const void* W, const void* bias, const void* residual, void* C,
                 float* z, int rows, int N, int K, int lda, int ldw, int ldr, int ldc, int ldz,
                 int act, int dtype, void* stream);

/* H[r, :] = act(A[r, :] Wg[e]^T) * (A[r, :] Wu[e]^T) for the rows r of every
 * expert e; rows of no expert are zero.  Wg, Wu: experts x N x K, row strides
 * ldg, ldu, matrix strides stride_g, stride_u.  z: NULL, or 2 x rows x N fp32 that
 * receive the products themselves, gate then up (16-byte aligned, ldz >= N a
 * multiple of 4, the second half at rows * ldz; rows of no expert are left). */
int b200_ffn_gated(const void* A, const void* Wg, const void* Wu, const int* offsets, void* H,
                   float* z, int rows, int experts, int N, int K, int lda, int ldg,
                   long long stride_g, int ldu, long long stride_u, int ldh, int ldz, int act,
                   int dtype, void* stream);

/* From the gradient of b200_ffn_act's C that of its product: dz = dC * act'(z),
 * rounded (fp16: infinite beyond 65504; dz: rows x lddz, 16-byte aligned, lddz >= N a
 * multiple of 8; or NULL), and dbias = the unrounded sum of its rows, rounded once
 * (N elements, or NULL).  z: as b200_ffn_act left it; with B200_ACT_NONE it is not read. */
int b200_ffn_act_grad(const void* dC, const float* z, void* dz, void* dbias, int rows, int N,
                      int ldc, int ldz, int lddz, int act, int dtype, void* stream);

/* From the gradient of b200_ffn_gated's H those of its two products, rounded:
 * dz[0] = dH * u * act'(g), dz[1] = dH * act(g) (dz: 2 x rows x lddz, as above).
 * Rows of no expert are left as they are. */
int b200_ffn_gated_grad(const void* dH, const float* z, const int* offsets, void* dz, int rows,
                        int experts, int N, int ldh, int ldz, int lddz, int act, int dtype,
                        void* stream);

/* Gradient in A: dA[r, :] = dz[0][r, :] W0[e] + dz[1][r, :] W1[e].  dz: halves x
 * rows x N, row stride lddz, halves rows * lddz apart; halves = 1 (W1 NULL) or 2.
 * Rows of no expert are zero. */
int b200_ffn_da(const void* dz, const void* W0, const void* W1, const int* offsets, void* dA,
                int halves, int rows, int experts, int N, int K, int lddz, int ld0,
                long long stride0, int ld1, long long stride1, int lda, int dtype, void* stream);

/* Gradients in the weights: dW[h][e] = sum over expert e's rows r of dz[h][r, :]^T
 * A[r, :].  dW: halves x experts x N x K, contiguous.  Rows of no expert are never
 * read into a sum; an expert without rows gets zeros. */
int b200_ffn_dw(const void* dz, const void* A, const int* offsets, void* dW, int halves, int rows,
                int experts, int N, int K, int lddz, int lda, int dtype, void* stream);

/* Kernel for b200_ffn_act, b200_ffn_gated and b200_ffn_da: 0 = chosen by sizes
 * (default), 1 = the streaming kernel (few rows; b200_ffn_da has none), 2 = the pair
 * kernel, 3 = the cluster kernel (one matrix, where its tiles fit the device; else pairs). */
int b200_ffn_set_kernel(int kernel);

/* ---- Norm of many gradients, clipping -----------------------------------------
 * A tensor is `count` consecutive elements of type B200_BF16, B200_FP16 or
 * B200_FP32, on its element's boundary; the list is read before the call returns. */
typedef struct {
  void* data;
  long long count;
  int type;
} b200_tensor;

/* *norm (device memory, fp32) = the 2-norm of all elements together.  Squares are
 * added 16 bytes of a tensor at a time in fp32 (in fp64 where fp32 does not hold them)
 * and those sums in fp64, in one order; within 2^-21 of the norm. */
int b200_grad_norm(const b200_tensor* tensors, int n, float* norm, void* stream);

/* The same, and every element multiplied by min(1, max_norm / (norm + 1e-6)) in
 * fp32 and rounded; nothing is written where that is 1.  Tensors must not overlap.
 * A norm that is not a number makes every element one; an infinite one makes them
 * zero, and infinite elements not a number (all of them, if max_norm is infinite
 * too).  max_norm >= 0. */
int b200_clip_grads(const b200_tensor* tensors, int n, float max_norm, float* norm, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* B200_FFN_H_ */
