// Torch bindings of the mixture-of-experts operators (include/b200_moe.h).
//
// As for matmul_b200: dtype, device, rank and shape are checked and raise
// RuntimeError; an operand whose rows are not 16-byte aligned is first copied
// into a layout the kernels read; launches go on the current torch stream.
// Operators with gradients are autograd functions here in C++, so a training
// step pays no Python call per node.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include "b200_moe.h"
#include "moe_torch.h"

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void check_status(int st, const char* what) {
  TORCH_CHECK(st == B200_OK, what, " failed: ", b200_gemm_status_string(st), " (status ", st, ")");
}

int64_t round_up8(int64_t x) { return (x + 7) / 8 * 8; }

bool aligned16(const at::Tensor& t) {
  return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0;
}

void* current_stream() { return at::cuda::getCurrentCUDAStream().stream(); }

// A new contiguous tensor on `like`'s device, past the dispatcher (0.9 us a
// tensor against 1.8: a decode step makes a dozen of them).
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& like) {
  return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}

int dtype_code(const at::Tensor& t) {
  return t.scalar_type() == at::kHalf ? B200_FP16 : B200_BF16;
}

void check_16bit(const at::Tensor& t, const char* who, const char* name) {
  TORCH_CHECK(t.is_cuda(), who, ": ", name, " must be a CUDA tensor");
  TORCH_CHECK(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf, who, ": ", name,
              " must be bfloat16 or float16");
}

void check_same(const at::Tensor& t, const at::Tensor& like, const char* who, const char* name) {
  TORCH_CHECK(t.device() == like.device(), who, ": ", name, " is on another device");
  TORCH_CHECK(t.scalar_type() == like.scalar_type(), who, ": ", name, " has another dtype");
}

// There are no forward-mode derivatives: a tangent would be lost.
void check_no_tangent(std::initializer_list<at::Tensor> operands, const char* who) {
  for (const at::Tensor& t : operands)
    TORCH_CHECK(!t._fw_grad(0).defined(), who,
                ": forward-mode derivatives are not defined; use the backward pass");
}

// Nor second ones: where a backward pass is itself recorded and its results
// depend on something differentiable, walking through them is an error.
variable_list differentiable_once(variable_list grads, bool depends, const char* who) {
  if (!depends || !at::GradMode::is_enabled()) return grads;
  for (at::Tensor& g : grads)
    if (g.defined()) g = g.detach().requires_grad_(true);
  torch::autograd::DelayedError error(
      std::string(who) + ": second derivatives are not defined (trying to differentiate twice)",
      (int64_t)grads.size());
  return error.apply(std::move(grads));
}

// A copy that no graph records (a backward pass may itself be recorded).
void copy_plain(const at::Tensor& to, const at::Tensor& from) {
  const at::NoGradGuard plain;
  to.copy_(from);
}

// A rows x cols operand as the kernels read it (unit column stride, rows and
// base on 16 bytes): `t` itself where it is one, else a copy.
struct Rows {
  at::Tensor t;
  int ld;
};

Rows as_rows(const at::Tensor& t) {
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

Bank as_bank(const at::Tensor& t) {
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
    check_status(b200_align_rows(t.data_ptr(), t.stride(0), t.stride(1), buf.data_ptr(), (int)e,
                                 (int)n, (int)k, (int)pad, current_stream()),
                 "aligning a bank");
  else
    copy_plain(to, t);
  return {to, (int)pad, n * pad};
}

at::Tensor check_offsets(const at::Tensor& offsets, int64_t experts, const at::Tensor& like,
                         const char* who) {
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

void check_sizes(std::initializer_list<int64_t> sizes, const char* who) {
  for (int64_t s : sizes)
    TORCH_CHECK(s < (1ll << 31) - 8, who, ": dimension exceeds 2^31-1");
}

// ------------------------------------------------------------ grouped product
constexpr const char* kGrouped = "matmul_b200_grouped";

at::Tensor grouped_forward(const Rows& a, const Bank& bank, const at::Tensor& offsets) {
  const int64_t rows = a.t.size(0), e = bank.t.size(0), n = bank.t.size(1), k = bank.t.size(2);
  auto c = fresh({rows, n}, a.t.scalar_type(), a.t);
  check_status(b200_grouped_gemm(a.t.data_ptr(), bank.t.data_ptr(), c.data_ptr(),
                                 offsets.data_ptr<int>(), (int)rows, (int)e, (int)n, (int)k, a.ld,
                                 bank.ld, bank.stride, (int)n, dtype_code(a.t), current_stream()),
               kGrouped);
  return c;
}

at::Tensor grouped_da(const Rows& dc, const Bank& bank, const at::Tensor& offsets) {
  const int64_t rows = dc.t.size(0), e = bank.t.size(0), n = bank.t.size(1), k = bank.t.size(2);
  auto da = fresh({rows, k}, dc.t.scalar_type(), dc.t);
  check_status(b200_grouped_gemm_da(dc.t.data_ptr(), bank.t.data_ptr(), da.data_ptr(),
                                    offsets.data_ptr<int>(), (int)rows, (int)e, (int)n, (int)k,
                                    dc.ld, bank.ld, bank.stride, (int)k, dtype_code(dc.t),
                                    current_stream()),
               "matmul_b200_grouped backward (A)");
  return da;
}

at::Tensor grouped_db(const Rows& dc, const Rows& a, const at::Tensor& offsets) {
  const int64_t e = offsets.size(0) - 1, rows = a.t.size(0), n = dc.t.size(1), k = a.t.size(1);
  auto db = fresh({e, n, k}, dc.t.scalar_type(), dc.t);
  check_status(b200_grouped_gemm_db(dc.t.data_ptr(), a.t.data_ptr(), db.data_ptr(),
                                    offsets.data_ptr<int>(), (int)rows, (int)e, (int)n, (int)k,
                                    dc.ld, a.ld, (int)k, n * k, dtype_code(dc.t),
                                    current_stream()),
               "matmul_b200_grouped backward (B)");
  return db;
}

// An operand that had to be copied into aligned rows is kept as that copy, so
// that a training step copies it once.
struct GroupedMatmul : torch::autograd::Function<GroupedMatmul> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& a, const at::Tensor& b,
                            const at::Tensor& offsets) {
    const c10::cuda::CUDAGuard guard(a.device());
    const Rows ra = as_rows(a);
    const Bank rb = as_bank(b.transpose(1, 2));
    ctx->save_for_backward({ra.t, rb.t, offsets});
    ctx->saved_data["both"] = a.requires_grad() && b.requires_grad();
    return grouped_forward(ra, rb, offsets);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &a = saved[0], &bank = saved[1], &offsets = saved[2];
    at::Tensor da, db;
    if (grads[0].defined()) {
      const c10::cuda::CUDAGuard guard(a.device());
      const Rows dc = as_rows(grads[0].scalar_type() == a.scalar_type()
                                  ? grads[0]
                                  : grads[0].to(a.scalar_type()));
      if (ctx->needs_input_grad(0)) da = grouped_da(dc, as_bank(bank), offsets);
      if (ctx->needs_input_grad(1)) db = grouped_db(dc, as_rows(a), offsets).transpose(1, 2);
    }
    // (linear in each operand: a gradient is constant unless both are variables)
    return differentiable_once({da, db, at::Tensor()},
                               ctx->saved_data["both"].toBool() || grads[0].requires_grad(),
                               kGrouped);
  }
};

at::Tensor matmul_b200_grouped(const at::Tensor& A, const at::Tensor& B,
                               const at::Tensor& offsets) {
  TORCH_CHECK(A.dim() == 2 && B.dim() == 3, kGrouped,
              ": A must be (rows, K) and B (experts, K, N)");
  check_no_tangent({A, B}, kGrouped);
  check_16bit(A, kGrouped, "A");
  check_16bit(B, kGrouped, "B");
  check_same(B, A, kGrouped, "B");
  TORCH_CHECK(B.size(1) == A.size(1), kGrouped, ": inner dimensions differ (A has K = ", A.size(1),
              ", B has K = ", B.size(1), ")");
  TORCH_CHECK(B.size(0) <= B200_MAX_EXPERTS, kGrouped, ": more than ", B200_MAX_EXPERTS,
              " experts");
  check_sizes({A.size(0), A.size(1), B.size(2)}, kGrouped);
  const at::Tensor off = check_offsets(offsets, B.size(0), A, kGrouped);
  if (at::GradMode::is_enabled() && (A.requires_grad() || B.requires_grad()))
    return GroupedMatmul::apply(A, B, off);
  const c10::cuda::CUDAGuard guard(A.device());
  return grouped_forward(as_rows(A), as_bank(B.transpose(1, 2)), off);
}

// -------------------------------------------------------------------- routing
constexpr const char* kRoute = "route_b200";
constexpr const char* kDispatch = "dispatch_b200";
constexpr const char* kCombine = "combine_b200";

int logit_code(const at::Tensor& t) {
  return t.scalar_type() == at::kFloat ? B200_FP32 : dtype_code(t);
}

// Rows with unit column stride; any row stride of at least the width.
at::Tensor unit_rows(const at::Tensor& t) {
  return (t.size(1) <= 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1))
             ? t
             : t.contiguous();
}
int64_t row_stride(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

// weights, experts, rows, tokens, offsets
std::vector<at::Tensor> route_forward(const at::Tensor& logits, int64_t top_k, bool normalize) {
  const c10::cuda::CUDAGuard guard(logits.device());
  const int64_t t = logits.size(0), e = logits.size(1);
  const at::Tensor l = unit_rows(logits);
  auto weights = fresh({t, top_k}, at::kFloat, logits);
  auto chosen = fresh({t, top_k}, at::kInt, logits), rows = fresh({t, top_k}, at::kInt, logits);
  auto sources = fresh({t * top_k}, at::kInt, logits), offsets = fresh({e + 1}, at::kInt, logits);
  check_status(b200_route(l.data_ptr(), (int)t, (int)e, row_stride(l), logit_code(l), (int)top_k,
                          normalize, weights.data_ptr<float>(), chosen.data_ptr<int>(),
                          rows.data_ptr<int>(), sources.data_ptr<int>(), offsets.data_ptr<int>(),
                          current_stream()),
               kRoute);
  return {weights, chosen, rows, sources, offsets};
}

struct Route : torch::autograd::Function<Route> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& logits, int64_t top_k,
                               bool normalize) {
    auto r = route_forward(logits, top_k, normalize);
    ctx->save_for_backward({logits, r[1], r[0]});
    ctx->saved_data["normalize"] = normalize;
    ctx->mark_non_differentiable({r[1], r[2], r[3], r[4]});
    return r;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &logits = saved[0], &chosen = saved[1], &weights = saved[2];
    at::Tensor dlogits;
    if (grads[0].defined()) {
      const c10::cuda::CUDAGuard guard(logits.device());
      const at::Tensor l = unit_rows(logits);
      const at::Tensor dw = grads[0].to(at::kFloat).contiguous();
      dlogits = fresh({l.size(0), l.size(1)}, l.scalar_type(), l);
      check_status(b200_route_grad(l.data_ptr(), (int)l.size(0), (int)l.size(1), row_stride(l),
                                   logit_code(l), (int)chosen.size(1),
                                   ctx->saved_data["normalize"].toBool(), chosen.data_ptr<int>(),
                                   weights.data_ptr<float>(), dw.data_ptr<float>(),
                                   dlogits.data_ptr(), current_stream()),
                   "route_b200 backward");
    }
    return differentiable_once({dlogits, at::Tensor(), at::Tensor()}, true, kRoute);
  }
};

std::vector<at::Tensor> route_b200(const at::Tensor& logits, int64_t top_k, bool normalize) {
  TORCH_CHECK(logits.dim() == 2, kRoute, ": logits must be (tokens, experts)");
  check_no_tangent({logits}, kRoute);
  TORCH_CHECK(logits.is_cuda(), kRoute, ": logits must be a CUDA tensor");
  TORCH_CHECK(logits.scalar_type() == at::kFloat || logits.scalar_type() == at::kBFloat16 ||
                  logits.scalar_type() == at::kHalf,
              kRoute, ": logits must be float32, bfloat16 or float16");
  const int64_t t = logits.size(0), e = logits.size(1);
  TORCH_CHECK(e <= B200_MAX_EXPERTS, kRoute, ": more than ", B200_MAX_EXPERTS, " experts");
  TORCH_CHECK(top_k >= 1 && top_k <= e && top_k <= B200_MAX_TOP_K, kRoute, ": top_k = ", top_k,
              " must be 1 .. min(experts, ", B200_MAX_TOP_K, ")");
  check_sizes({t * top_k}, kRoute);
  if (at::GradMode::is_enabled() && logits.requires_grad())
    return Route::apply(logits, top_k, normalize);
  return route_forward(logits, top_k, normalize);
}

// A sorted operand's rows and a token operand's, checked against the routing.
void check_routing(const at::Tensor& t, const at::Tensor& rows, const at::Tensor& offsets,
                   bool sorted, const char* who, const char* name) {
  TORCH_CHECK(t.dim() == 2, who, ": ", name, " must be 2-D");
  check_no_tangent({t}, who);
  check_16bit(t, who, name);
  TORCH_CHECK(rows.dim() == 2 && rows.is_contiguous() && rows.scalar_type() == at::kInt &&
                  offsets.dim() == 1 && offsets.size(0) >= 1 && offsets.is_contiguous() &&
                  offsets.scalar_type() == at::kInt,
              who, ": routing must come from route_b200");
  TORCH_CHECK(rows.device() == t.device() && offsets.device() == t.device(), who, ": ", name,
              " and the routing are on different devices");
  TORCH_CHECK(rows.size(1) <= B200_MAX_TOP_K, who, ": more than ", B200_MAX_TOP_K, " slots");
  const int64_t want = sorted ? rows.numel() : rows.size(0);
  TORCH_CHECK(t.size(0) == want, who, ": ", name, " has ", t.size(0), " rows, the routing ", want);
  check_sizes({rows.numel(), t.size(1)}, who);
}

const int* total_of(const at::Tensor& offsets) {
  return offsets.data_ptr<int>() + (offsets.size(0) - 1);
}

at::Tensor dispatch_forward(const at::Tensor& x, const at::Tensor& rows,
                            const at::Tensor& offsets) {
  const c10::cuda::CUDAGuard guard(x.device());
  const at::Tensor in = unit_rows(x);
  auto xs = fresh({rows.numel(), x.size(1)}, x.scalar_type(), x);
  check_status(b200_dispatch(in.data_ptr(), rows.data_ptr<int>(), total_of(offsets), xs.data_ptr(),
                             (int)rows.size(0), (int)rows.size(1), (int)x.size(1), row_stride(in),
                             x.size(1), dtype_code(x), current_stream()),
               kDispatch);
  return xs;
}

at::Tensor combine_forward(const at::Tensor& y, const float* weights, const at::Tensor& rows,
                           const char* who) {
  const c10::cuda::CUDAGuard guard(y.device());
  const at::Tensor in = unit_rows(y);
  auto out = fresh({rows.size(0), y.size(1)}, y.scalar_type(), y);
  check_status(b200_combine(in.data_ptr(), weights, rows.data_ptr<int>(), out.data_ptr(),
                            (int)rows.size(0), (int)rows.size(1), (int)y.size(1), row_stride(in),
                            y.size(1), dtype_code(y), current_stream()),
               who);
  return out;
}

struct Dispatch : torch::autograd::Function<Dispatch> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& rows,
                            const at::Tensor& offsets) {
    ctx->save_for_backward({rows});
    ctx->saved_data["dtype"] = x.scalar_type();
    return dispatch_forward(x, rows, offsets);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    at::Tensor dx;
    if (grads[0].defined())
      dx = combine_forward(grads[0].to(ctx->saved_data["dtype"].toScalarType()), nullptr,
                           ctx->get_saved_variables()[0], "dispatch_b200 backward");
    return differentiable_once({dx, at::Tensor(), at::Tensor()}, grads[0].requires_grad(),
                               kDispatch);
  }
};

at::Tensor dispatch_b200(const at::Tensor& x, const at::Tensor& rows, const at::Tensor& offsets) {
  check_routing(x, rows, offsets, false, kDispatch, "x");
  if (at::GradMode::is_enabled() && x.requires_grad()) return Dispatch::apply(x, rows, offsets);
  return dispatch_forward(x, rows, offsets);
}

struct Combine : torch::autograd::Function<Combine> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& y, const at::Tensor& weights,
                            const at::Tensor& rows, const at::Tensor& offsets) {
    ctx->save_for_backward({y, weights, rows, offsets});
    ctx->saved_data["both"] = y.requires_grad() && weights.requires_grad();
    return combine_forward(y, weights.data_ptr<float>(), rows, kCombine);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &y = saved[0], &weights = saved[1], &rows = saved[2], &offsets = saved[3];
    at::Tensor dy, dweights;
    if (grads[0].defined()) {
      const c10::cuda::CUDAGuard guard(y.device());
      const at::Tensor dout = unit_rows(grads[0].to(y.scalar_type())), in = unit_rows(y);
      dy = fresh({y.size(0), y.size(1)}, y.scalar_type(), y);
      if (ctx->needs_input_grad(1))
        dweights = fresh({rows.size(0), rows.size(1)}, at::kFloat, weights);
      check_status(
          b200_combine_grad(dout.data_ptr(), in.data_ptr(), weights.data_ptr<float>(),
                            rows.data_ptr<int>(), total_of(offsets), dy.data_ptr(),
                            dweights.defined() ? dweights.data_ptr<float>() : nullptr,
                            (int)rows.size(0), (int)rows.size(1), (int)y.size(1), row_stride(dout),
                            row_stride(in), y.size(1), dtype_code(y), current_stream()),
          "combine_b200 backward");
    }
    return differentiable_once({dy, dweights, at::Tensor(), at::Tensor()},
                               ctx->saved_data["both"].toBool() || grads[0].requires_grad(),
                               kCombine);
  }
};

at::Tensor combine_b200(const at::Tensor& y, const at::Tensor& weights, const at::Tensor& rows,
                        const at::Tensor& offsets) {
  check_no_tangent({weights}, kCombine);
  check_routing(y, rows, offsets, true, kCombine, "y");
  TORCH_CHECK(weights.sizes() == rows.sizes() && weights.scalar_type() == at::kFloat &&
                  weights.device() == y.device(),
              kCombine, ": weights must be float32 (tokens, top_k) on y's device");
  const at::Tensor w = weights.is_contiguous() ? weights : weights.contiguous();
  if (at::GradMode::is_enabled() && (y.requires_grad() || w.requires_grad()))
    return Combine::apply(y, w, rows, offsets);
  return combine_forward(y, w.data_ptr<float>(), rows, kCombine);
}

// -------------------------------------------------------------- 4-bit weights
constexpr const char* kPack = "pack_w4";
constexpr const char* kW4 = "matmul_b200_w4";

// q (experts, N, K / 2), scales and zeros (experts, N, K / group): the packed bytes.
at::Tensor w4_pack(const at::Tensor& q, const at::Tensor& scales,
                   const std::optional<at::Tensor>& zeros) {
  TORCH_CHECK(q.dim() == 3 && scales.dim() == 3, kPack,
              ": q must be (N, K/2) or (experts, N, K/2) and scales (.., N, K/group)");
  TORCH_CHECK(q.is_cuda() && q.scalar_type() == at::kByte, kPack,
              ": q must be a uint8 CUDA tensor");
  check_16bit(scales, kPack, "scales");
  TORCH_CHECK(scales.device() == q.device(), kPack, ": scales is on another device");
  const int64_t e = q.size(0), n = q.size(1), k = 2 * q.size(2), groups = scales.size(2);
  TORCH_CHECK(scales.size(0) == e && scales.size(1) == n, kPack,
              ": scales must have q's experts and rows");
  check_sizes({n, k}, kPack);
  TORCH_CHECK(groups > 0 ? k % groups == 0 : k == 0, kPack, ": K = ", k,
              " is not a whole number of groups (", groups, " scales to a row)");
  const int64_t group = groups > 0 ? k / groups : 128;
  TORCH_CHECK(group == 32 || group == 64 || group == 128, kPack,
              ": groups must hold 32, 64 or 128 weights, not ", group);
  TORCH_CHECK(e <= B200_MAX_EXPERTS, kPack, ": more than ", B200_MAX_EXPERTS, " experts");
  at::Tensor z;
  if (zeros.has_value()) {
    TORCH_CHECK(zeros->sizes() == scales.sizes() && zeros->scalar_type() == at::kByte &&
                    zeros->device() == q.device(),
                kPack, ": zeros must be uint8, of scales' shape, on q's device");
    z = zeros->contiguous();
  }
  const c10::cuda::CUDAGuard guard(q.device());
  // (the one wait for the device here, once per weight; in a capture the
  // packing kernel alone reports it)
  if (z.defined() && z.numel() > 0 &&
      c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None)
    TORCH_CHECK(z.max().item<int64_t>() <= 15, kPack, ": zeros must be 0 .. 15");
  size_t bytes = 0;
  check_status(b200_w4_packed_bytes((int)e, (int)n, (int)k, (int)group, z.defined(), &bytes),
               kPack);
  auto packed = fresh({(int64_t)bytes}, at::kByte, q);
  const at::Tensor qc = q.contiguous(), sc = scales.contiguous();
  check_status(b200_w4_pack(qc.data_ptr(), sc.data_ptr(), z.defined() ? z.data_ptr() : nullptr,
                            packed.data_ptr(), (int)e, (int)n, (int)k, (int)group,
                            current_stream()),
               kPack);
  return packed;
}

at::Tensor w4_matmul(const at::Tensor& A, const at::Tensor& packed, int64_t experts, int64_t N,
                     int64_t K, int64_t group, bool zeros, bool half,
                     const std::optional<at::Tensor>& offsets) {
  TORCH_CHECK(A.dim() == 2, kW4, ": A must be (rows, K)");
  check_no_tangent({A}, kW4);
  check_16bit(A, kW4, "A");
  TORCH_CHECK(A.scalar_type() == (half ? at::kHalf : at::kBFloat16), kW4,
              ": A and the scales must have the same dtype");
  TORCH_CHECK(A.device() == packed.device(), kW4, ": A and the weight are on different devices");
  TORCH_CHECK(A.size(1) == K, kW4, ": inner dimensions differ (A has K = ", A.size(1),
              ", the weight has K = ", K, ")");
  TORCH_CHECK(experts >= 0 && N >= 0 && K >= 0 && group >= 0, kW4,
              ": the weight's sizes must not be negative");
  TORCH_CHECK(experts <= B200_MAX_EXPERTS, kW4, ": more than ", B200_MAX_EXPERTS, " experts");
  check_sizes({N, K, group}, kW4);
  size_t bytes = 0;
  check_status(b200_w4_packed_bytes((int)experts, (int)N, (int)K, (int)group, zeros, &bytes), kW4);
  TORCH_CHECK(packed.scalar_type() == at::kByte && packed.is_contiguous() &&
                  packed.numel() == (int64_t)bytes,
              kW4, ": the weight's data must be pack_w4's, ", bytes,
              " contiguous bytes (uint8) for its sizes");
  TORCH_CHECK(!(at::GradMode::is_enabled() && A.requires_grad()), kW4,
              ": no gradient is defined (4-bit weights serve); use torch.no_grad()");
  check_sizes({A.size(0)}, kW4);
  at::Tensor off;
  if (offsets.has_value())
    off = check_offsets(*offsets, experts, A, kW4);
  else
    TORCH_CHECK(experts == 1, kW4, ": a bank of experts needs offsets");
  const c10::cuda::CUDAGuard guard(A.device());
  const Rows ra = as_rows(A);
  auto c = fresh({A.size(0), N}, A.scalar_type(), A);
  check_status(b200_w4_gemm(ra.t.data_ptr(), packed.data_ptr(), c.data_ptr(),
                            off.defined() ? off.data_ptr<int>() : nullptr, (int)A.size(0),
                            (int)experts, (int)N, (int)K, (int)group, zeros, ra.ld, (int)N,
                            dtype_code(A), current_stream()),
               kW4);
  return c;
}

}  // namespace

void register_moe(pybind11::module_& m) {
  m.def("matmul_b200_grouped", &matmul_b200_grouped,
        "C[r] = A[r] @ B[e] for rows r of expert e (offsets on the device)");
  m.def("route_b200", &route_b200, "top-k experts, weights and the order sorted by expert");
  m.def("dispatch_b200", &dispatch_b200, "rows of x in the order sorted by expert");
  m.def("combine_b200", &combine_b200, "weighted sum of each token's rows");
  m.def("w4_pack", &w4_pack, "4-bit weights in the order the kernel reads them",
        pybind11::arg("q"), pybind11::arg("scales"), pybind11::arg("zeros") = std::nullopt);
  m.def("w4_matmul", &w4_matmul, "C = A @ W^T with packed 4-bit weights");
}
