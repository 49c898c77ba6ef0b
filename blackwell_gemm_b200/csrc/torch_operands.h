// Operands of the torch bindings (moe_torch.cpp, ffn_torch.cpp): checks, copies
// into rows that the kernels read, results past the dispatcher.
#pragma once
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include "b200_moe.h"

namespace b200_torch {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

inline void check_status(int st, const char* what) {
  TORCH_CHECK(st == B200_OK, what, " failed: ", b200_gemm_status_string(st), " (status ", st, ")");
}

inline int64_t round_up8(int64_t x) { return (x + 7) / 8 * 8; }

inline bool aligned16(const at::Tensor& t) {
  return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0;
}

inline void* current_stream() { return at::cuda::getCurrentCUDAStream().stream(); }

// A new contiguous tensor on `like`'s device, past the dispatcher (0.9 us a
// tensor against 1.8: a decode step makes a dozen of them).
inline at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& like) {
  return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}

inline int dtype_code(const at::Tensor& t) {
  return t.scalar_type() == at::kHalf ? B200_FP16 : B200_BF16;
}

inline void check_16bit(const at::Tensor& t, const char* who, const char* name) {
  TORCH_CHECK(t.is_cuda(), who, ": ", name, " must be a CUDA tensor");
  TORCH_CHECK(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf, who, ": ", name,
              " must be bfloat16 or float16");
}

inline void check_same(const at::Tensor& t, const at::Tensor& like, const char* who,
                       const char* name) {
  TORCH_CHECK(t.device() == like.device(), who, ": ", name, " is on another device");
  TORCH_CHECK(t.scalar_type() == like.scalar_type(), who, ": ", name, " has another dtype");
}

// Whether any tensor can have a tangent: forward mode has one level, and without it
// none has (a look at 60 views of one buffer took 4 us).
inline bool tangents_possible() {
  return torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr;
}

// There are no forward-mode derivatives: a tangent would be lost.
inline void check_no_tangent(std::initializer_list<at::Tensor> operands, const char* who) {
  if (!tangents_possible()) return;
  for (const at::Tensor& t : operands)
    TORCH_CHECK(!t._fw_grad(0).defined(), who,
                ": forward-mode derivatives are not defined; use the backward pass");
}

// Nor second ones: where a backward pass is itself recorded and its results
// depend on something differentiable, walking through them is an error.
inline variable_list differentiable_once(variable_list grads, bool depends, const char* who) {
  if (!depends || !at::GradMode::is_enabled()) return grads;
  for (at::Tensor& g : grads)
    if (g.defined()) g = g.detach().requires_grad_(true);
  torch::autograd::DelayedError error(
      std::string(who) + ": second derivatives are not defined (trying to differentiate twice)",
      (int64_t)grads.size());
  return error.apply(std::move(grads));
}

// A copy that no graph records (a backward pass may itself be recorded).
inline void copy_plain(const at::Tensor& to, const at::Tensor& from) {
  const at::NoGradGuard plain;
  to.copy_(from);
}

// A rows x cols operand as the kernels read it (unit column stride, rows and
// base on 16 bytes): `t` itself where it is one, else a copy.
struct Rows {
  at::Tensor t;
  int ld;
};

inline Rows as_rows(const at::Tensor& t) {
  const int64_t rows = t.size(0), cols = t.size(1), pad = std::max<int64_t>(round_up8(cols), 8);
  if (rows == 0 || cols == 0) return {t, (int)pad};
  const int64_t ld = rows > 1 ? t.stride(0) : pad;
  if ((cols == 1 || t.stride(1) == 1) && ld >= cols && ld % 8 == 0 && ld < (1ll << 31) &&
      aligned16(t))
    return {t, (int)ld};
  auto buf = fresh({rows, pad}, t.scalar_type(), t);
  const at::Tensor to = buf.narrow(1, 0, cols);
  if (cols == 1 || t.stride(1) == 1)
    check_status(b200_align_rows(t.data_ptr(), 0, rows > 1 ? t.stride(0) : cols, buf.data_ptr(), 1,
                                 (int)rows, (int)cols, (int)pad, current_stream()),
                 "aligning rows");
  else
    copy_plain(to, t);  // (transposed: what lies past cols is never read)
  return {to, (int)pad};
}

// The same for a bank of matrices, given as (experts, N, K).
struct Bank {
  at::Tensor t;
  int ld;
  int64_t stride;
};

// With offsets only the matrices of experts with rows are copied.
inline Bank as_bank(const at::Tensor& t, const at::Tensor& offsets = {}) {
  const int64_t e = t.size(0), n = t.size(1), k = t.size(2);
  const int64_t pad = std::max<int64_t>(round_up8(k), 8);
  if (t.numel() == 0) return {t, (int)pad, n * pad};
  const int64_t ld = n > 1 ? t.stride(1) : pad;
  const int64_t stride = e > 1 ? t.stride(0) : n * ld;
  if ((k == 1 || t.stride(2) == 1) && ld >= k && ld % 8 == 0 && ld < (1ll << 31) &&
      stride % 8 == 0 && stride >= n * ld && aligned16(t))
    return {t, (int)ld, stride};
  auto buf = fresh({e, n, pad}, t.scalar_type(), t);
  const at::Tensor to = buf.narrow(2, 0, k);
  if (k == 1 || t.stride(2) == 1)
    check_status(b200_align_bank(t.data_ptr(), t.stride(0), t.stride(1), buf.data_ptr(),
                                 offsets.defined() ? offsets.data_ptr<int>() : nullptr, (int)e,
                                 (int)n, (int)k, (int)pad, current_stream()),
                 "aligning a bank");
  else
    copy_plain(to, t);
  return {to, (int)pad, n * pad};
}

inline at::Tensor check_offsets(const at::Tensor& offsets, int64_t experts,
                                const at::Tensor& like, const char* who) {
  TORCH_CHECK(offsets.dim() == 1 && offsets.size(0) == experts + 1, who, ": offsets must have ",
              experts + 1, " entries (one more than there are experts)");
  TORCH_CHECK(offsets.device() == like.device(), who, ": offsets must be on the operands' device");
  TORCH_CHECK(offsets.scalar_type() == at::kInt || offsets.scalar_type() == at::kLong, who,
              ": offsets must be int32 or int64");
  if (offsets.scalar_type() == at::kInt) return offsets.contiguous();
  const c10::cuda::CUDAGuard guard(offsets.device());
  auto narrow = fresh({offsets.size(0)}, at::kInt, offsets);
  check_status(b200_narrow_offsets(offsets.data_ptr(), offsets.stride(0), (int)offsets.size(0),
                                   narrow.data_ptr<int>(), current_stream()),
               who);
  return narrow;
}

inline void check_sizes(std::initializer_list<int64_t> sizes, const char* who) {
  for (int64_t s : sizes)
    TORCH_CHECK(s < (1ll << 31) - 8, who, ": dimension exceeds 2^31-1");
}

}  // namespace b200_torch
