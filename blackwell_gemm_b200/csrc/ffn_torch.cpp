// Torch bindings of the feed-forward operators (include/b200_ffn.h).
//
// As for the grouped products: dtype, device, rank and shape are checked and
// raise RuntimeError; an operand whose rows are not 16-byte aligned is first
// copied into a layout the kernels read, once per training step; launches go on
// the current torch stream; the autograd functions are C++.
#include "ffn_torch.h"

#include "b200_ffn.h"
#include "torch_operands.h"

using namespace b200_torch;

namespace {

constexpr const char* kAct = "matmul_b200_act";
constexpr const char* kGated = "matmul_b200_gated";
constexpr const char* kNorm = "grad_norm_b200";
constexpr const char* kClip = "clip_grads_b200";

using OptTensor = std::optional<at::Tensor>;

int act_code(const std::string& name, const char* who) {
  static const char* const names[] = {"none", "relu", "silu", "gelu", "gelu_tanh", "sigmoid"};
  for (int i = 0; i < 6; ++i)
    if (name == names[i]) return i;
  TORCH_CHECK(false, who, ": unknown activation '", name,
              "' (none, relu, silu, gelu, gelu_tanh, sigmoid)");
}

// Columns of an fp32 or 16-bit buffer made here: whole 16 bytes to a row.
int64_t padded(int64_t n) { return std::max<int64_t>(round_up8(n), 8); }

at::Tensor defined_or_empty(const OptTensor& t) { return t.has_value() ? *t : at::Tensor(); }

void* data_or_null(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// A gradient in the operands' type.
at::Tensor like_operand(const at::Tensor& g, at::ScalarType type) {
  return g.scalar_type() == type ? g : g.to(type);
}

// ---------------------------------------- product with bias, activation, residual
// A residual with unit column stride, whatever its row stride.
at::Tensor unit_columns(const at::Tensor& t) {
  return (t.size(1) <= 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1)) &&
                 (t.size(0) <= 1 || t.stride(0) < (1ll << 31))
             ? t
             : t.contiguous();
}

at::Tensor act_forward(const Rows& a, const Rows& w, const at::Tensor& bias,
                       const at::Tensor& residual, int act, at::Tensor* z) {
  const int64_t m = a.t.size(0), n = w.t.size(0), k = a.t.size(1);
  auto c = fresh({m, n}, a.t.scalar_type(), a.t);
  if (z != nullptr) *z = fresh({m, padded(n)}, at::kFloat, a.t);
  const at::Tensor r = residual.defined() ? unit_columns(residual) : residual;
  const int64_t ldr = !r.defined() || m <= 1 ? n : r.stride(0);
  const at::Tensor b = bias.defined() ? bias.contiguous() : bias;
  check_status(b200_ffn_act(a.t.data_ptr(), w.t.data_ptr(), data_or_null(b), data_or_null(r),
                            c.data_ptr(), z != nullptr ? z->data_ptr<float>() : nullptr, (int)m,
                            (int)n, (int)k, a.ld, w.ld, (int)ldr, (int)n, (int)padded(n), act,
                            dtype_code(a.t), current_stream()),
               kAct);
  return c;
}

struct ActMatmul : torch::autograd::Function<ActMatmul> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& a, const at::Tensor& b,
                            const OptTensor& bias_, const OptTensor& residual_, int64_t act) {
    const at::Tensor bias = defined_or_empty(bias_), residual = defined_or_empty(residual_);
    const c10::cuda::CUDAGuard guard(a.device());
    const Rows ra = as_rows(a), rw = as_rows(b.t());
    const bool through = a.requires_grad() || b.requires_grad() ||
                         (bias.defined() && bias.requires_grad());
    at::Tensor z;
    at::Tensor c = act_forward(ra, rw, bias, residual, (int)act,
                               through && act != B200_ACT_NONE ? &z : nullptr);
    // What a gradient that nobody asks for would need is not kept.
    const bool keep_a = b.requires_grad(), keep_w = a.requires_grad();
    // (detached: a view made here would answer for a weight changed meanwhile in its words)
    ctx->save_for_backward(
        {keep_a ? ra.t : at::Tensor(), keep_w ? rw.t.detach() : at::Tensor(), z});
    ctx->saved_data["act"] = act;
    ctx->saved_data["bias"] = bias.defined();
    ctx->saved_data["residual"] = residual.defined();
    ctx->saved_data["m"] = a.size(0);
    ctx->saved_data["n"] = b.size(1);
    ctx->saved_data["k"] = a.size(1);
    ctx->saved_data["dtype"] = a.scalar_type();
    // (linear in each operand without an activation)
    ctx->saved_data["bends"] =
        through && (act != B200_ACT_NONE || (a.requires_grad() && b.requires_grad()));
    return c;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &a = saved[0], &w = saved[1], &z = saved[2];
    const int act = (int)ctx->saved_data["act"].toInt();
    const int64_t m = ctx->saved_data["m"].toInt(), n = ctx->saved_data["n"].toInt(),
                  k = ctx->saved_data["k"].toInt();
    const bool has_bias = ctx->saved_data["bias"].toBool(),
               has_residual = ctx->saved_data["residual"].toBool();
    at::Tensor da, db, dbias, dresidual;
    if (grads[0].defined()) {
      const at::ScalarType type = ctx->saved_data["dtype"].toScalarType();
      const at::Tensor dc = like_operand(grads[0], type);
      const c10::cuda::CUDAGuard guard(dc.device());
      const bool want_a = ctx->needs_input_grad(0), want_b = ctx->needs_input_grad(1),
                 want_bias = has_bias && ctx->needs_input_grad(2);
      // (edges are numbered past an operand that is not there)
      if (has_residual && ctx->needs_input_grad(2 + has_bias)) dresidual = dc;
      if (want_a || want_b || want_bias) {
        Rows dz = as_rows(dc);
        const Rows rows = dz;
        const bool bent = act != B200_ACT_NONE && (want_a || want_b);
        if (bent) dz = {fresh({m, padded(n)}, type, dc), (int)padded(n)};
        if (want_bias) dbias = fresh({n}, type, dc);
        if (bent || want_bias)
          check_status(
              b200_ffn_act_grad(rows.t.data_ptr(), z.defined() ? z.data_ptr<float>() : nullptr,
                                bent ? dz.t.data_ptr() : nullptr, data_or_null(dbias), (int)m,
                                (int)n, rows.ld, (int)padded(n), (int)padded(n), act,
                                dtype_code(dc), current_stream()),
              "matmul_b200_act backward");
        if (want_a) {
          const Rows rw = as_rows(w);
          da = fresh({m, k}, type, dc);
          check_status(b200_ffn_da(dz.t.data_ptr(), rw.t.data_ptr(), nullptr, nullptr,
                                   da.data_ptr(), 1, (int)m, 1, (int)n, (int)k, dz.ld, rw.ld, 0, 0,
                                   0, (int)k, dtype_code(dc), current_stream()),
                       "matmul_b200_act backward (A)");
        }
        if (want_b) {
          const Rows ra = as_rows(a);
          db = fresh({n, k}, type, dc);
          check_status(b200_ffn_dw(dz.t.data_ptr(), ra.t.data_ptr(), nullptr, db.data_ptr(), 1,
                                   (int)m, 1, (int)n, (int)k, dz.ld, ra.ld, dtype_code(dc),
                                   current_stream()),
                       "matmul_b200_act backward (B)");
          db = db.t();
        }
      }
    }
    return differentiable_once({da, db, dbias, dresidual, at::Tensor()},
                               ctx->saved_data["bends"].toBool() || grads[0].requires_grad(),
                               kAct);
  }
};

at::Tensor matmul_b200_act(const at::Tensor& A, const at::Tensor& B, const OptTensor& bias_,
                           const OptTensor& residual_, const std::string& activation) {
  const at::Tensor bias = defined_or_empty(bias_), residual = defined_or_empty(residual_);
  TORCH_CHECK(A.dim() == 2 && B.dim() == 2, kAct, ": A must be (M, K) and B (K, N)");
  const int act = act_code(activation, kAct);
  check_no_tangent({A, B}, kAct);
  if (bias.defined()) check_no_tangent({bias}, kAct);
  if (residual.defined()) check_no_tangent({residual}, kAct);
  check_16bit(A, kAct, "A");
  check_16bit(B, kAct, "B");
  check_same(B, A, kAct, "B");
  TORCH_CHECK(B.size(0) == A.size(1), kAct, ": inner dimensions differ (A has K = ", A.size(1),
              ", B has K = ", B.size(0), ")");
  const int64_t m = A.size(0), n = B.size(1);
  check_sizes({m, n, A.size(1)}, kAct);
  bool any = A.requires_grad() || B.requires_grad();
  if (bias.defined()) {
    check_same(bias, A, kAct, "bias");
    TORCH_CHECK(bias.dim() == 1 && bias.size(0) == n, kAct, ": bias must have shape (", n, ",)");
    any = any || bias.requires_grad();
  }
  if (residual.defined()) {
    check_same(residual, A, kAct, "residual");
    TORCH_CHECK(residual.dim() == 2 && residual.size(0) == m && residual.size(1) == n, kAct,
                ": residual must have shape (", m, ", ", n, ")");
    any = any || residual.requires_grad();
  }
  if (at::GradMode::is_enabled() && any) return ActMatmul::apply(A, B, bias_, residual_, act);
  const c10::cuda::CUDAGuard guard(A.device());
  return act_forward(as_rows(A), as_rows(B.t()), bias, residual, act, nullptr);
}

// ------------------------------------------------------------------ gated product
// Weights as banks (experts, N, K); without offsets a bank of one.
at::Tensor gated_forward(const Rows& a, const Bank& g, const Bank& u, const at::Tensor& offsets,
                         int act, at::Tensor* z) {
  const int64_t m = a.t.size(0), e = g.t.size(0), n = g.t.size(1), k = a.t.size(1);
  auto h = fresh({m, n}, a.t.scalar_type(), a.t);
  if (z != nullptr) *z = fresh({2, m, padded(n)}, at::kFloat, a.t);
  check_status(b200_ffn_gated(a.t.data_ptr(), g.t.data_ptr(), u.t.data_ptr(),
                              offsets.defined() ? offsets.data_ptr<int>() : nullptr, h.data_ptr(),
                              z != nullptr ? z->data_ptr<float>() : nullptr, (int)m, (int)e,
                              (int)n, (int)k, a.ld, g.ld, g.stride, u.ld, u.stride, (int)n,
                              (int)padded(n), act, dtype_code(a.t), current_stream()),
               kGated);
  return h;
}

// (.., K, N) to (experts, N, K)
at::Tensor bank_of(const at::Tensor& b) {
  return b.dim() == 3 ? b.transpose(1, 2) : b.t().unsqueeze(0);
}

struct GatedMatmul : torch::autograd::Function<GatedMatmul> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& a, const at::Tensor& gate,
                            const at::Tensor& up, const OptTensor& offsets_, int64_t act) {
    const at::Tensor offsets = defined_or_empty(offsets_);
    const c10::cuda::CUDAGuard guard(a.device());
    const Rows ra = as_rows(a);
    const Bank g = as_bank(bank_of(gate), offsets), u = as_bank(bank_of(up), offsets);
    at::Tensor z;
    at::Tensor h = gated_forward(ra, g, u, offsets, (int)act, &z);
    const bool keep_a = gate.requires_grad() || up.requires_grad(), keep_w = a.requires_grad();
    ctx->save_for_backward({keep_a ? ra.t : at::Tensor(), keep_w ? g.t.detach() : at::Tensor(),
                            keep_w ? u.t.detach() : at::Tensor(), offsets, z});
    ctx->saved_data["act"] = act;
    ctx->saved_data["experts"] = g.t.size(0);
    ctx->saved_data["n"] = g.t.size(1);
    ctx->saved_data["k"] = a.size(1);
    ctx->saved_data["bank"] = gate.dim() == 3;
    ctx->saved_data["dtype"] = a.scalar_type();
    return h;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &a = saved[0], &offsets = saved[3], &z = saved[4];
    const int act = (int)ctx->saved_data["act"].toInt();
    const int64_t e = ctx->saved_data["experts"].toInt(), n = ctx->saved_data["n"].toInt(),
                  k = ctx->saved_data["k"].toInt(), m = z.size(1);
    const bool bank = ctx->saved_data["bank"].toBool();
    const int* off = offsets.defined() ? offsets.data_ptr<int>() : nullptr;
    at::Tensor da, dgate, dup;
    if (grads[0].defined()) {
      const c10::cuda::CUDAGuard guard(z.device());
      const at::ScalarType type = ctx->saved_data["dtype"].toScalarType();
      const Rows dh = as_rows(like_operand(grads[0], type));
      const auto dz = fresh({2, m, padded(n)}, type, z);
      check_status(b200_ffn_gated_grad(dh.t.data_ptr(), z.data_ptr<float>(), off, dz.data_ptr(),
                                       (int)m, (int)e, (int)n, dh.ld, (int)padded(n),
                                       (int)padded(n), act, dtype_code(dz), current_stream()),
                   "matmul_b200_gated backward");
      if (ctx->needs_input_grad(0)) {
        const Bank g = as_bank(saved[1], offsets), u = as_bank(saved[2], offsets);
        da = fresh({m, k}, type, z);
        check_status(b200_ffn_da(dz.data_ptr(), g.t.data_ptr(), u.t.data_ptr(), off, da.data_ptr(),
                                 2, (int)m, (int)e, (int)n, (int)k, (int)padded(n), g.ld, g.stride,
                                 u.ld, u.stride, (int)k, dtype_code(dz), current_stream()),
                     "matmul_b200_gated backward (A)");
      }
      const bool want_gate = ctx->needs_input_grad(1), want_up = ctx->needs_input_grad(2);
      if (want_gate || want_up) {
        // Both halves in one launch, or the one that is asked for.
        const int64_t halves = want_gate && want_up ? 2 : 1;
        const Rows ra = as_rows(a);
        const auto dw = fresh({halves, e, n, k}, type, z);
        const at::Tensor from = halves == 1 && want_up ? dz.select(0, 1) : dz;
        check_status(b200_ffn_dw(from.data_ptr(), ra.t.data_ptr(), off, dw.data_ptr(), (int)halves,
                                 (int)m, (int)e, (int)n, (int)k, (int)padded(n), ra.ld,
                                 dtype_code(dz), current_stream()),
                     "matmul_b200_gated backward (B)");
        auto half = [&](int64_t i) {
          const at::Tensor t = dw.select(0, i);
          return bank ? t.transpose(1, 2) : t.select(0, 0).t();
        };
        if (want_gate) dgate = half(0);
        if (want_up) dup = half(halves - 1);
      }
    }
    return differentiable_once({da, dgate, dup, at::Tensor(), at::Tensor()}, true, kGated);
  }
};

at::Tensor matmul_b200_gated(const at::Tensor& A, const at::Tensor& gate, const at::Tensor& up,
                             const OptTensor& offsets_, const std::string& activation) {
  TORCH_CHECK(A.dim() == 2 && (gate.dim() == 2 || gate.dim() == 3), kGated,
              ": A must be (rows, K), B_gate and B_up (K, N) or (experts, K, N)");
  const int act = act_code(activation, kGated);
  check_no_tangent({A, gate, up}, kGated);
  check_16bit(A, kGated, "A");
  check_16bit(gate, kGated, "B_gate");
  check_same(gate, A, kGated, "B_gate");
  check_16bit(up, kGated, "B_up");
  check_same(up, A, kGated, "B_up");
  TORCH_CHECK(gate.sizes() == up.sizes(), kGated, ": B_gate and B_up must have the same shape");
  const int64_t k = gate.size(-2), experts = gate.dim() == 3 ? gate.size(0) : 1;
  TORCH_CHECK(k == A.size(1), kGated, ": inner dimensions differ (A has K = ", A.size(1),
              ", the weights have K = ", k, ")");
  TORCH_CHECK(experts <= B200_MAX_EXPERTS, kGated, ": more than ", B200_MAX_EXPERTS, " experts");
  check_sizes({A.size(0), k, gate.size(-1)}, kGated);
  at::Tensor offsets;
  if (offsets_.has_value()) {
    TORCH_CHECK(gate.dim() == 3, kGated, ": offsets go with a bank of experts (experts, K, N)");
    offsets = check_offsets(*offsets_, experts, A, kGated);
  } else {
    TORCH_CHECK(experts == 1, kGated, ": a bank of experts needs offsets");
  }
  if (at::GradMode::is_enabled() &&
      (A.requires_grad() || gate.requires_grad() || up.requires_grad()))
    return GatedMatmul::apply(A, gate, up, offsets.defined() ? OptTensor(offsets) : OptTensor(),
                              act);
  const c10::cuda::CUDAGuard guard(A.device());
  return gated_forward(as_rows(A), as_bank(bank_of(gate), offsets),
                       as_bank(bank_of(up), offsets), offsets, act, nullptr);
}

// -------------------------------------------------------- gradient norm, clipping
// The tensors as flat runs of elements.  One that has gaps is taken through a copy
// (`back`: what is copied back into it).
struct Flat {
  std::vector<b200_tensor> list;
  std::vector<std::pair<at::Tensor, at::Tensor>> back;
};

Flat flatten(const std::vector<at::Tensor>& grads, bool written, const char* who) {
  TORCH_CHECK(!grads.empty(), who, ": needs at least one gradient");
  const bool tangents = tangents_possible();
  for (const at::Tensor& g : grads) {
    TORCH_CHECK(g.defined(), who, ": gradients must be dense CUDA tensors");
    if (tangents) check_no_tangent({g}, who);
  }
  const c10::Device device = grads[0].device();
  const bool recording = at::GradMode::is_enabled();
  Flat f;
  f.list.reserve(grads.size());
  for (const at::Tensor& g : grads) {
    TORCH_CHECK(g.layout() == at::kStrided && g.is_cuda(), who,
                ": gradients must be dense CUDA tensors");
    TORCH_CHECK(g.device() == device, who, ": gradients are on different devices");
    const at::ScalarType type = g.scalar_type();
    TORCH_CHECK(type == at::kFloat || type == at::kBFloat16 || type == at::kHalf, who,
                ": gradients must be float32, bfloat16 or float16");
    TORCH_CHECK(!(recording && g.requires_grad()), who,
                ": no gradient is defined for it; use torch.no_grad()");
    const int64_t n = g.numel();
    if (n == 0) continue;
    const int code = type == at::kFloat ? B200_FP32 : dtype_code(g);
    if (g.is_non_overlapping_and_dense() && !g.is_neg()) {
      f.list.push_back({g.data_ptr(), n, code});
      continue;
    }
    if (written)
      for (int64_t i = 0; i < g.dim(); ++i)
        TORCH_CHECK(g.size(i) <= 1 || g.stride(i) != 0, who,
                    ": an expanded tensor cannot be scaled in place");
    const at::NoGradGuard plain;
    f.back.emplace_back(g, g.clone(at::MemoryFormat::Contiguous));
    f.list.push_back({f.back.back().second.data_ptr(), n, code});
  }
  return f;
}

// Where a tensor's bytes lie: begin + the sum of stride k, 0 <= k < count, over the terms.
struct Bytes {
  const char *begin, *end;
  bool dense;  // every byte from begin to end
  const at::Tensor* t;
};

Bytes bytes_of(const at::Tensor& t) {
  const char* p = static_cast<const char*>(t.data_ptr());
  const bool dense = t.is_non_overlapping_and_dense();
  int64_t last = dense ? t.numel() - 1 : 0;
  for (int64_t i = 0; i < t.dim() && !dense; ++i) last += (t.size(i) - 1) * t.stride(i);
  return {p, p + (last + 1) * (int64_t)t.element_size(), dense, &t};
}

// Whether two tensors have a byte in common: whether the terms of the one less those of
// the other can make the distance of their beginnings.  Or two elements of one tensor:
// whether differences of its indexes that are not all zero make none.  A search from the
// largest stride down, in which each term has only the few values that leave a distance the
// rest can make; one that takes too long (strides without order among many dimensions)
// counts as one that was found.
struct Meeting {
  struct Term {
    int64_t stride, lo, hi;
    int64_t least, most;  // what the smaller strides' terms make together
  };
  std::vector<Term> terms;
  int budget = 100000;

  void add(int64_t stride, int64_t lo, int64_t hi) {
    for (Term& t : terms)
      if (t.stride == stride) {
        t.lo += lo;
        t.hi += hi;
        return;
      }
    terms.push_back({stride, lo, hi, 0, 0});
  }
  void add(const Bytes& b, int sign) {
    auto term = [&](int64_t stride, int64_t count) {
      if (count > 1 && stride > 0)
        add(stride, sign < 0 ? -(count - 1) : 0, sign < 0 ? 0 : count - 1);
    };
    const int64_t size = b.t->element_size();
    term(1, b.dense ? b.end - b.begin : size);
    for (int64_t i = 0; i < b.t->dim() && !b.dense; ++i)
      term(b.t->stride(i) * size, b.t->size(i));
  }
  bool reach(size_t i, int64_t distance) {
    if (i == terms.size()) return distance == 0;
    if (--budget < 0) return true;
    const Term& t = terms[i];
    auto floor_div = [](int64_t a, int64_t b) { return a / b - (a % b < 0); };
    const int64_t lo = std::max(t.lo, -floor_div(t.most - distance, t.stride)),
                  hi = std::min(t.hi, floor_div(distance - t.least, t.stride));
    for (int64_t k = lo; k <= hi; ++k)
      if (reach(i + 1, distance - k * t.stride)) return true;
    return false;
  }
  void order() {
    std::sort(terms.begin(), terms.end(),
              [](const Term& x, const Term& y) { return x.stride > y.stride; });
    int64_t least = 0, most = 0;
    for (size_t i = terms.size(); i-- > 0;) {
      Term& t = terms[i];
      t.least = least;
      t.most = most;
      least += t.lo * t.stride;
      most += t.hi * t.stride;
    }
  }
  static bool between(const Bytes& a, const Bytes& b) {
    if (a.dense && b.dense) return true;  // (whose extents cross)
    Meeting m;
    m.add(a, 1);
    m.add(b, -1);
    m.order();
    return m.reach(0, b.begin - a.begin);
  }
  static bool within(const at::Tensor& t) {
    Meeting m;
    for (int64_t i = 0; i < t.dim(); ++i)
      if (t.size(i) > 1) m.terms.push_back({t.stride(i), 1 - t.size(i), t.size(i) - 1, 0, 0});
    m.order();
    // (the first difference that is not zero may be taken as positive)
    for (size_t i = 0; i < m.terms.size(); ++i)
      for (int64_t k = 1; k <= m.terms[i].hi && k * m.terms[i].stride <= m.terms[i].most; ++k)
        if (m.reach(i + 1, -k * m.terms[i].stride)) return true;
    return false;
  }
};

// No element may be scaled twice, nor counted twice in the norm.  (Tensors with gaps may
// interleave, as columns do.)
void check_apart(const std::vector<at::Tensor>& grads, const char* who) {
  std::vector<Bytes> spans;
  spans.reserve(grads.size());
  for (const at::Tensor& g : grads) {
    if (g.numel() == 0) continue;
    spans.push_back(bytes_of(g));
    TORCH_CHECK(spans.back().dense || !Meeting::within(g), who,
                ": gradients must not share memory");
  }
  auto before = [](const Bytes& a, const Bytes& b) { return a.begin < b.begin; };
  if (!std::is_sorted(spans.begin(), spans.end(), before))
    std::sort(spans.begin(), spans.end(), before);
  for (size_t i = 0; i < spans.size(); ++i)
    for (size_t j = i + 1; j < spans.size() && spans[j].begin < spans[i].end; ++j)
      TORCH_CHECK(!Meeting::between(spans[i], spans[j]), who, ": gradients must not share memory");
}

// Where the work goes; nowhere yet if the checks are going to refuse it.
std::optional<c10::Device> device_of(const std::vector<at::Tensor>& grads) {
  return !grads.empty() && grads[0].defined() && grads[0].is_cuda()
             ? std::optional<c10::Device>(grads[0].device())
             : std::nullopt;
}

at::Tensor grad_norm_b200(const std::vector<at::Tensor>& grads) {
  const c10::cuda::OptionalCUDAGuard guard(device_of(grads));
  const Flat f = flatten(grads, false, kNorm);
  auto norm = fresh({}, at::kFloat, grads[0]);
  check_status(b200_grad_norm(f.list.data(), (int)f.list.size(), norm.data_ptr<float>(),
                              current_stream()),
               kNorm);
  return norm;
}

at::Tensor clip_grads_b200(const std::vector<at::Tensor>& grads, double max_norm) {
  TORCH_CHECK(max_norm >= 0, kClip, ": max_norm must not be negative");
  const c10::cuda::OptionalCUDAGuard guard(device_of(grads));
  const Flat f = flatten(grads, true, kClip);
  check_apart(grads, kClip);
  auto norm = fresh({}, at::kFloat, grads[0]);
  check_status(b200_clip_grads(f.list.data(), (int)f.list.size(), (float)max_norm,
                               norm.data_ptr<float>(), current_stream()),
               kClip);
  const at::NoGradGuard plain;
  for (const auto& [to, from] : f.back) to.copy_(from);
  // (written past autograd: what it saved of them is no longer that)
  for (const at::Tensor& g : grads)
    if (!g.is_inference()) g.unsafeGetTensorImpl()->bump_version();
  return norm;
}

}  // namespace

void register_ffn(pybind11::module_& m) {
  namespace py = pybind11;
  m.def("matmul_b200_act", &matmul_b200_act, "C = act(A @ B + bias) + residual", py::arg("A"),
        py::arg("B"), py::arg("bias") = std::nullopt, py::arg("residual") = std::nullopt,
        py::arg("activation") = "none");
  m.def("matmul_b200_gated", &matmul_b200_gated, "H = act(A @ B_gate) * (A @ B_up)", py::arg("A"),
        py::arg("B_gate"), py::arg("B_up"), py::arg("offsets") = std::nullopt,
        py::arg("activation") = "silu");
  m.def("grad_norm_b200", &grad_norm_b200, "2-norm of many tensors together");
  m.def("clip_grads_b200", &clip_grads_b200, "many tensors scaled in place by their norm");
}
