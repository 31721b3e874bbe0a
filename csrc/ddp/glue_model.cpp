// Bindings of the model and update operators: RMS norm, rotary positions, orthogonalised updates. The checks of arguments are here, for
// tensors of either device; CPU tensors take the formulas in ATen operations, CUDA tensors the kernels, on the current stream of their device.
#include <ATen/cuda/CUDAContext.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <tuple>
#include <vector>

#include "nangila_kernels.h"
#include "nangila_model_kernels.h"

namespace py = pybind11;

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

bool known(at::ScalarType t) { return t == at::kFloat || t == at::kHalf || t == at::kBFloat16; }
int dtype_code(const Tensor& t) { return t.scalar_type() == at::kFloat ? NANGILA_F32 : t.scalar_type() == at::kHalf ? NANGILA_F16 : NANGILA_BF16; }
void check_launch(int err, const char* what) { TORCH_CHECK(err == 0, "nangila: ", what, " failed: ", cudaGetErrorString(static_cast<cudaError_t>(err))); }
void check_plain(const Tensor& t, const char* name) {
  TORCH_CHECK_TYPE(!t.unsafeGetTensorImpl()->is_python_dispatch(), "nangila: ", name, " must be a plain tensor, not one that wraps another (a sharded one has to be gathered first)");
  TORCH_CHECK_TYPE(t.layout() == at::kStrided, "nangila: ", name, " must be dense");
  TORCH_CHECK_TYPE(t.is_cuda() || t.is_cpu(), "nangila: ", name, " must be on a CUDA device or the CPU");
}
void check_tensor(const Tensor& t, const char* name) {
  check_plain(t, name);
  TORCH_CHECK_TYPE(known(t.scalar_type()), "nangila: ", name, " must be float32, float16 or bfloat16, not ", t.scalar_type());
}
// The kernels write into fresh memory behind the dispatcher's back. What follows the operations of PyTorch from there (forward-mode derivatives, tracers,
// tensors that stand for others) would not see them, and go on as if the results were constants: such calls are refused.
void check_followed(const Tensor& t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(0).defined(),
                              "nangila: the kernels have no forward-mode derivative; give them tensors without a tangent (forward_ad.unpack_dual(..).primal), or CPU tensors");
}
void check_no_tracer() {
  using c10::impl::TorchDispatchModeKey;
  using c10::impl::TorchDispatchModeTLS;
  TORCH_CHECK_NOT_IMPLEMENTED(!torch::jit::tracer::isTracing(), "nangila: the kernels cannot be traced (torch.jit.trace)");
  if (!TorchDispatchModeTLS::any_modes_set()) return;
  for (const TorchDispatchModeKey key : {TorchDispatchModeKey::FAKE, TorchDispatchModeKey::PROXY, TorchDispatchModeKey::FUNCTIONAL})
    TORCH_CHECK_NOT_IMPLEMENTED(!TorchDispatchModeTLS::get_mode(key).has_value(), "nangila: the kernels cannot be traced (make_fx, export or fake tensors)");
}
void check_unseen(std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts) check_followed(*t);
  check_no_tracer();
}
bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}
void once_only() {
  TORCH_CHECK(!at::GradMode::is_enabled(), "nangila: this gradient cannot be differentiated again (create_graph=True)");
}

// The tensor with its values in memory: a view that is negated only when it is read has others there, zeros that nobody has read yet have none.
Tensor in_memory(const Tensor& t) {
  if (t._is_zerotensor()) return at::zeros(t.sizes(), t.options());
  return t.is_neg() ? t.resolve_neg() : t;
}

// ---- RMS norm --------------------------------------------------------------------------------------------------
// `t` as rows of d adjacent values, `stride` apart: the tensor itself where its strides allow that, else a packed copy.
Tensor as_rows(const Tensor& given, int64_t d, int64_t* stride) {
  const Tensor t = in_memory(given);
  *stride = d;
  if (t.is_contiguous()) return t;
  if (t.dim() >= 2 && t.stride(-1) == 1) {
    int64_t step = -1, expected = -1;  // between rows; what the next outer dimension's stride has to be
    bool uniform = true;
    for (int64_t i = t.dim() - 2; i >= 0; --i) {
      if (t.size(i) == 1) continue;
      if (step < 0) step = t.stride(i);
      else if (t.stride(i) != expected) uniform = false;
      expected = t.stride(i) * t.size(i);
    }
    if (uniform && step >= 0) {
      *stride = step;
      return t;
    }
  }
  return t.contiguous();
}
struct NormArgs {
  int64_t d, rows;
};
NormArgs check_norm(const Tensor& x, const Tensor& residual, const Tensor& weight, double eps) {
  check_tensor(x, "x");
  check_tensor(weight, "weight");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= NANGILA_NORM_MAX_D, "nangila: the last dimension of x must have 1 to ", NANGILA_NORM_MAX_D,
                    " values, got shape ", x.sizes());
  TORCH_CHECK_VALUE(weight.dim() == 1 && weight.size(0) == x.size(-1), "nangila: weight must have shape [", x.size(-1), "], not ", weight.sizes());
  TORCH_CHECK_VALUE(weight.device() == x.device(), "nangila: weight is on ", weight.device(), ", x on ", x.device());
  if (residual.defined()) {
    TORCH_CHECK_VALUE(residual.sizes() == x.sizes(), "nangila: residual has shape ", residual.sizes(), ", x ", x.sizes());
    TORCH_CHECK_TYPE(residual.scalar_type() == x.scalar_type(), "nangila: residual is ", residual.scalar_type(), ", x ", x.scalar_type());
    TORCH_CHECK_VALUE(residual.device() == x.device(), "nangila: residual is on ", residual.device(), ", x on ", x.device());
  }
  TORCH_CHECK_VALUE(std::isfinite(eps) && eps >= 0, "nangila: eps must be finite and not negative, got ", eps);
  return {x.size(-1), x.numel() / x.size(-1)};
}
// y, h and rstd (or q, h and scales) of CUDA rows
struct NormOut {
  Tensor y, h, rstd, q, scale;
};
NormOut norm_forward(const Tensor& x_in, const Tensor& residual_in, const Tensor& weight_in, double eps, bool keep_rstd, bool fp8, int64_t group) {
  c10::cuda::CUDAGuard guard(x_in.device());
  const int64_t d = x_in.size(-1), rows = x_in.numel() / d;
  NormOut o;
  if (residual_in.defined()) o.h = at::empty(x_in.sizes(), x_in.options());
  if (fp8) {
    o.q = at::empty(x_in.sizes(), x_in.options().dtype(at::kFloat8_e4m3fn));
    std::vector<int64_t> shape = x_in.sizes().vec();
    shape.back() = group ? d / group : 1;
    o.scale = at::empty(shape, x_in.options().dtype(at::kFloat));
  } else {
    o.y = at::empty(x_in.sizes(), x_in.options());
  }
  if (keep_rstd) o.rstd = at::empty({rows}, x_in.options().dtype(at::kFloat));
  if (rows == 0) return o;
  NangilaNormParams p;
  std::memset(&p, 0, sizeof p);
  Tensor x = as_rows(x_in, d, &p.x_stride), residual = residual_in, weight = in_memory(weight_in).contiguous();
  if (residual.defined()) residual = as_rows(residual, d, &p.residual_stride);
  if (group) {  // a group's columns are read sixteen bytes at a time
    auto packed = [&](Tensor& t, int64_t* stride) {
      if ((reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0 && (stride == nullptr || *stride % 8 == 0)) return;
      t = t.clone(at::MemoryFormat::Contiguous);
      if (stride != nullptr) *stride = d;
    };
    packed(x, &p.x_stride);
    if (residual.defined()) packed(residual, &p.residual_stride);
    packed(weight, nullptr);
  }
  p.x = x.data_ptr();
  p.residual = residual.defined() ? residual.data_ptr() : nullptr;
  p.weight = weight.data_ptr();
  p.h = o.h.defined() ? o.h.data_ptr() : nullptr;
  p.y = o.y.defined() ? o.y.data_ptr() : nullptr;
  p.rstd = o.rstd.defined() ? o.rstd.data_ptr<float>() : nullptr;
  p.q = o.q.defined() ? static_cast<uint8_t*>(o.q.data_ptr()) : nullptr;
  p.scale = o.scale.defined() ? o.scale.data_ptr<float>() : nullptr;
  p.rows = rows;
  p.d = int32_t(d);
  p.group = int32_t(group);
  p.dtype = dtype_code(x);
  p.weight_dtype = dtype_code(weight);
  p.eps = float(eps);
  check_launch(nangila_rms_norm_forward(&p, at::cuda::getCurrentCUDAStream()), "rms_norm");
  return o;
}

class RmsNorm : public torch::autograd::Function<RmsNorm> {
 public:
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const c10::optional<Tensor>& residual_in, const Tensor& weight, double eps) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor residual = residual_in.value_or(Tensor());
    NormOut o = norm_forward(x, residual, weight, eps, true, false, 0);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({residual.defined() ? o.h : x, weight, o.rstd});
    ctx->saved_data["residual"] = residual.defined();
    if (residual.defined()) return {o.y, o.h};
    return {o.y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once_only();
    const variable_list saved = ctx->get_saved_variables();
    Tensor h = saved[0], weight = in_memory(saved[1]).contiguous();
    const Tensor& rstd = saved[2];
    Tensor dy = grads[0], dh = grads.size() > 1 ? grads[1] : Tensor();
    variable_list out(4);
    if (!dy.defined() && !dh.defined()) return out;
    check_unseen({&dy, &dh});
    // (asked for by the place among the tensors that were given)
    const bool two = ctx->saved_data["residual"].toBool(), for_x = ctx->needs_input_grad(0), for_residual = two && ctx->needs_input_grad(1);
    const bool want_x = for_x || for_residual, want_w = ctx->needs_input_grad(two ? 2 : 1) && dy.defined();
    if (!want_x && !want_w) return out;
    c10::cuda::CUDAGuard guard(h.device());
    const int64_t d = h.size(-1), rows = h.numel() / d;
    Tensor dx, dw, partial;
    if (want_x) dx = at::empty(h.sizes(), h.options());
    if (rows == 0) {
      if (want_w) dw = at::zeros_like(weight);
    } else {
      NangilaNormGradParams p;
      std::memset(&p, 0, sizeof p);
      auto rows_of = [&](Tensor& t, int64_t* stride) {
        if (t.scalar_type() != h.scalar_type()) t = t.to(h.scalar_type());
        t = as_rows(t, d, stride);
        return t.data_ptr();
      };
      p.h = rows_of(h, &p.h_stride);
      if (dy.defined()) p.dy = rows_of(dy, &p.dy_stride);
      if (dh.defined()) p.dh = rows_of(dh, &p.dh_stride);
      p.weight = weight.data_ptr();
      p.rstd = rstd.data_ptr<float>();
      p.dx = want_x ? dx.data_ptr() : nullptr;
      p.rows = rows;
      p.d = int32_t(d);
      p.dtype = dtype_code(h);
      p.weight_dtype = dtype_code(weight);
      if (want_w) {
        int32_t parts = 0;
        check_launch(nangila_rms_norm_partials(rows, p.d, p.dtype, &parts), "rms_norm gradient");
        dw = at::empty({d}, weight.options());
        partial = at::empty({int64_t(parts) * d}, h.options().dtype(at::kFloat));
        p.dw = dw.data_ptr();
        p.partial = partial.data_ptr<float>();
      }
      check_launch(nangila_rms_norm_backward(&p, at::cuda::getCurrentCUDAStream()), "rms_norm gradient");
    }
    if (for_x) out[0] = dx;
    if (for_residual) out[1] = dx;
    out[2] = dw;
    return out;
  }
};

Tensor cpu_unit(const Tensor& h, const Tensor& weight, double eps) {
  const Tensor f = h.to(at::kFloat);
  return f * at::rsqrt(f.square().mean(-1, true) + eps) * weight.to(at::kFloat);
}
Tensor rms_norm(const Tensor& x, const Tensor& weight, double eps) {
  check_norm(x, Tensor(), weight, eps);
  if (x.is_cpu()) return cpu_unit(x, weight, eps).to(x.scalar_type());
  check_unseen({&x, &weight});
  if (!wants_grad({&x, &weight})) return norm_forward(x, Tensor(), weight, eps, false, false, 0).y;
  return RmsNorm::apply(x, c10::optional<Tensor>(), weight, eps)[0];
}
std::tuple<Tensor, Tensor> add_rms_norm(const Tensor& x, const Tensor& residual, const Tensor& weight, double eps) {
  check_norm(x, residual, weight, eps);
  if (x.is_cpu()) {
    const Tensor h = x + residual;
    return {cpu_unit(h, weight, eps).to(x.scalar_type()), h};
  }
  check_unseen({&x, &residual, &weight});
  if (!wants_grad({&x, &residual, &weight})) {
    NormOut o = norm_forward(x, residual, weight, eps, false, false, 0);
    return {o.y, o.h};
  }
  variable_list o = RmsNorm::apply(x, c10::optional<Tensor>(residual), weight, eps);
  return {o[0], o[1]};
}
std::tuple<Tensor, Tensor, c10::optional<Tensor>> rms_norm_fp8(const Tensor& x, const Tensor& weight, double eps, const c10::optional<Tensor>& residual_in, int64_t group) {
  const Tensor residual = residual_in.value_or(Tensor());
  const NormArgs a = check_norm(x, residual, weight, eps);
  TORCH_CHECK_VALUE(group == 0 || group == 128, "nangila: group must be None (one scale for each row) or 128, got ", group);
  TORCH_CHECK_VALUE(group == 0 || a.d % 128 == 0, "nangila: groups of 128 need a last dimension that is a multiple of 128, got ", a.d);
  TORCH_CHECK(!wants_grad({&x, &residual, &weight}), "nangila: the 8-bit output has no gradient; call it under torch.no_grad() or on detached tensors");
  if (x.is_cpu()) {
    const Tensor h = residual.defined() ? x + residual : x;
    Tensor f = cpu_unit(h, weight, eps);
    const std::vector<int64_t> shape = f.sizes().vec();
    f = f.unflatten(-1, {group ? a.d / group : 1, group ? group : a.d});
    Tensor amax = f.abs().amax(-1);
    Tensor scale = at::where(at::isfinite(amax), amax.clamp_min(1e-12) / 448.0, at::full_like(amax, NAN));
    Tensor q = (f / scale.unsqueeze(-1)).clamp(-448.0, 448.0).to(at::kFloat8_e4m3fn).reshape(shape);
    return {q, scale, residual.defined() ? c10::optional<Tensor>(h) : c10::nullopt};
  }
  check_unseen({&x, &residual, &weight});
  NormOut o = norm_forward(x, residual, weight, eps, false, true, group);
  return {o.q, o.scale, residual.defined() ? c10::optional<Tensor>(o.h) : c10::nullopt};
}

// ---- rotary positions --------------------------------------------------------------------------------------------
void check_rotary(const Tensor& q, const Tensor& k, const Tensor& table, const Tensor& positions) {
  check_tensor(q, "q");
  TORCH_CHECK_VALUE(q.dim() == 4 && q.size(3) >= 2 && q.size(3) <= 65536, "nangila: q must have shape [batch, seq, heads, head_dim], got ", q.sizes());
  if (k.defined()) {
    check_tensor(k, "k");
    TORCH_CHECK_VALUE(k.dim() == 4 && k.size(0) == q.size(0) && k.size(1) == q.size(1) && k.size(3) == q.size(3), "nangila: k must have q's batch, seq and head_dim, got ",
                      k.sizes(), " for q ", q.sizes());
    TORCH_CHECK_TYPE(k.scalar_type() == q.scalar_type(), "nangila: k is ", k.scalar_type(), ", q ", q.scalar_type());
    TORCH_CHECK_VALUE(k.device() == q.device(), "nangila: k is on ", k.device(), ", q on ", q.device());
  }
  check_plain(table, "the table");
  TORCH_CHECK_VALUE(table.dim() == 3 && table.size(2) == 2 && table.scalar_type() == at::kFloat && table.size(0) >= 1 && table.size(1) >= 1,
                    "nangila: the table must be float32 of shape [positions, rot / 2, 2], got ", table.scalar_type(), " ", table.sizes());
  TORCH_CHECK_VALUE(2 * table.size(1) <= q.size(3), "nangila: the table turns ", 2 * table.size(1), " columns, a head has ", q.size(3));
  TORCH_CHECK_VALUE(table.device() == q.device(), "nangila: the table is on ", table.device(), ", q on ", q.device());
  TORCH_CHECK_VALUE(!table.requires_grad(), "nangila: the table has no gradient");
  if (positions.defined()) {
    check_plain(positions, "positions");
    TORCH_CHECK_TYPE(positions.scalar_type() == at::kLong || positions.scalar_type() == at::kInt, "nangila: positions must be int64 or int32, not ", positions.scalar_type());
    TORCH_CHECK_VALUE(positions.device() == q.device(), "nangila: positions are on ", positions.device(), ", q on ", q.device());
    TORCH_CHECK_VALUE((positions.dim() == 1 && positions.size(0) == q.size(1)) ||
                          (positions.dim() == 2 && (positions.size(0) == q.size(0) || positions.size(0) == 1) && positions.size(1) == q.size(1)),
                      "nangila: positions must have shape [seq] or [batch, seq], got ", positions.sizes(), " for q ", q.sizes());
  } else {
    TORCH_CHECK_VALUE(q.size(1) <= table.size(0), "nangila: the table has ", table.size(0), " positions, the sequence ", q.size(1));
  }
}
// one or two tensors turned; an undefined one is left out
std::tuple<Tensor, Tensor> rotary_launch(const Tensor& q, const Tensor& k, const Tensor& table_in, const Tensor& positions_in, bool half, bool inverse) {
  const Tensor& some = q.defined() ? q : k;
  c10::cuda::CUDAGuard guard(some.device());
  const Tensor table = in_memory(table_in).contiguous(), positions = positions_in.defined() ? in_memory(positions_in) : positions_in;
  NangilaRotaryParams p;
  std::memset(&p, 0, sizeof p);
  Tensor out[2], in[2];
  int n = 0;
  for (const Tensor* t : {&q, &k}) {
    Tensor& o = out[t == &q ? 0 : 1];
    if (!t->defined()) continue;
    o = at::empty(t->sizes(), t->options());
    if (t->numel() == 0) continue;
    in[n] = in_memory(*t);
    if (in[n].stride(3) != 1) in[n] = in[n].contiguous();
    p.in[n] = in[n].data_ptr();
    p.out[n] = o.data_ptr();
    p.stride_b[n] = in[n].stride(0);
    p.stride_t[n] = in[n].stride(1);
    p.stride_h[n] = in[n].stride(2);
    p.heads[n] = int32_t(t->size(2));
    ++n;
  }
  if (n == 0) return {out[0], out[1]};
  p.batch = some.size(0);
  p.seq = some.size(1);
  p.d = int32_t(some.size(3));
  p.rot = int32_t(2 * table.size(1));
  p.half = half ? 1 : 0;
  p.inverse = inverse ? 1 : 0;
  p.table = table.data_ptr<float>();
  p.table_rows = table.size(0);
  if (positions.defined()) {
    p.positions = positions.data_ptr();
    p.positions_64 = positions.scalar_type() == at::kLong ? 1 : 0;
    p.pos_stride_b = positions.dim() == 2 && positions.size(0) > 1 ? positions.stride(0) : 0;
    p.pos_stride_t = positions.stride(-1);
  }
  p.dtype = dtype_code(some);
  check_launch(nangila_rotary(&p, at::cuda::getCurrentCUDAStream()), "rotary");
  return {out[0], out[1]};
}
class Rotary : public torch::autograd::Function<Rotary> {
 public:
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const c10::optional<Tensor>& k_in, const Tensor& table, const c10::optional<Tensor>& positions_in,
                               bool half) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor k = k_in.value_or(Tensor()), positions = positions_in.value_or(Tensor());
    auto [oq, ok] = rotary_launch(q, k, table, positions, half, false);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({table, positions});
    ctx->saved_data["half"] = half;
    if (k.defined()) return {oq, ok};
    return {oq};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once_only();
    const variable_list saved = ctx->get_saved_variables();
    variable_list out(5);
    Tensor gq = ctx->needs_input_grad(0) ? grads[0] : Tensor(), gk = grads.size() > 1 && ctx->needs_input_grad(1) ? grads[1] : Tensor();
    if (!gq.defined() && !gk.defined()) return out;
    check_unseen({&gq, &gk});
    std::tie(out[0], out[1]) = rotary_launch(gq, gk, saved[0], saved[1], ctx->saved_data["half"].toBool(), true);
    return out;
  }
};
Tensor cpu_turn(const Tensor& x, const Tensor& angles, bool half) {  // angles: [.., seq, 1, rot / 2, 2]
  const int64_t n = angles.size(-2);
  const Tensor c = angles.select(-1, 0), s = angles.select(-1, 1), f = x.to(at::kFloat);
  Tensor turned;
  if (half) {
    const Tensor a = f.narrow(-1, 0, n), b = f.narrow(-1, n, n);
    turned = at::cat({a * c - b * s, a * s + b * c}, -1);
  } else {
    const Tensor pairs = f.narrow(-1, 0, 2 * n).unflatten(-1, {n, 2}), a = pairs.select(-1, 0), b = pairs.select(-1, 1);
    turned = at::stack({a * c - b * s, a * s + b * c}, -1).flatten(-2);
  }
  return at::cat({turned, f.narrow(-1, 2 * n, x.size(-1) - 2 * n)}, -1).to(x.scalar_type());
}
std::tuple<Tensor, c10::optional<Tensor>> rotary(const Tensor& q, const c10::optional<Tensor>& k_in, const Tensor& table, const c10::optional<Tensor>& positions_in, bool half) {
  const Tensor k = k_in.value_or(Tensor()), positions = positions_in.value_or(Tensor());
  check_rotary(q, k, table, positions);
  Tensor oq, ok;
  if (q.is_cpu()) {
    Tensor angles;
    if (positions.defined()) {
      const Tensor out = (positions < 0).logical_or(positions >= table.size(0));
      angles = table.index({positions.to(at::kLong).clamp(0, table.size(0) - 1)});
      angles = at::where(out.unsqueeze(-1).unsqueeze(-1), at::full({}, NAN, table.options()), angles);
    } else {
      angles = table.narrow(0, 0, q.size(1));
    }
    angles = angles.unsqueeze(-3);
    oq = cpu_turn(q, angles, half);
    if (k.defined()) ok = cpu_turn(k, angles, half);
    return {oq, k.defined() ? c10::optional<Tensor>(ok) : c10::nullopt};
  }
  check_unseen({&q, &k, &table});
  for (const Tensor* t : {&q, &k})
    TORCH_CHECK_VALUE(!t->defined() || t->size(2) <= (int64_t(1) << 30), "nangila: the kernels take up to 2^30 heads, got ", t->sizes());
  if (wants_grad({&q, &k})) {
    variable_list o = Rotary::apply(q, k_in, table, positions_in, half);
    oq = o[0];
    if (k.defined()) ok = o[1];
  } else {
    std::tie(oq, ok) = rotary_launch(q, k, table, positions, half, false);
  }
  return {oq, k.defined() ? c10::optional<Tensor>(ok) : c10::nullopt};
}

// ---- orthogonalised updates ----------------------------------------------------------------------------------------
struct OrthArgs {
  std::vector<double> coefficients;  // three for each step
  double eps, mu, decay, rate;
  bool nesterov;
};
void check_schedule(const std::vector<double>& coefficients) {
  TORCH_CHECK_VALUE(!coefficients.empty() && coefficients.size() % 3 == 0 && coefficients.size() / 3 <= NANGILA_ORTH_MAX_STEPS, "nangila: three coefficients for each of 1 to ",
                    NANGILA_ORTH_MAX_STEPS, " steps");
}
// Packed CUDA matrices of one shape, type and device, which the callers below have checked. With params: param = param * decay - rate * result
// and nothing is returned; else the results, bf16, one behind the other.
Tensor orth_group(const std::vector<Tensor>& grads, const std::vector<Tensor>& momenta, const std::vector<Tensor>& params, const OrthArgs& args) {
  const int64_t total = int64_t(grads.size());
  const Tensor& first = grads[0];
  const int64_t rows = first.size(0), cols = first.size(1);
  const std::vector<double>& coefficients = args.coefficients;
  c10::cuda::CUDAGuard guard(first.device());
  Tensor out;
  if (params.empty()) out = at::empty({total, rows, cols}, first.options().dtype(at::kBFloat16));
  // as many matrices at a time as fit into a workspace of a gigabyte, one at least
  const int64_t each = nangila_orth_workspace(1, int32_t(rows), int32_t(cols));
  const int64_t most = std::max<int64_t>(1, std::min<int64_t>(NANGILA_ORTH_MAX_COUNT, (int64_t(1) << 30) / each));
  const int64_t groups = (total + most - 1) / most, size = (total + groups - 1) / groups;
  const Tensor workspace = at::empty({nangila_orth_workspace(int32_t(std::min(size, total)), int32_t(rows), int32_t(cols))}, first.options().dtype(at::kByte));
  for (int64_t at = 0; at < total; at += size) {
    NangilaOrthParams p;
    std::memset(&p, 0, sizeof p);
    p.count = int32_t(std::min(size, total - at));
    for (int32_t i = 0; i < p.count; ++i) {
      p.grad[i] = grads[at + i].data_ptr();
      if (!momenta.empty()) p.momentum[i] = momenta[at + i].data_ptr<float>();
      if (!params.empty()) p.param[i] = params[at + i].data_ptr();
    }
    if (params.empty()) p.out = static_cast<uint16_t*>(out.data_ptr()) + at * rows * cols;
    p.rows = int32_t(rows);
    p.cols = int32_t(cols);
    p.grad_dtype = dtype_code(first);
    p.param_dtype = params.empty() ? 0 : dtype_code(params[0]);
    p.steps = int32_t(coefficients.size() / 3);
    for (size_t i = 0; i < coefficients.size(); ++i) p.coefficients[i / 3][i % 3] = float(coefficients[i]);
    p.nesterov = args.nesterov ? 1 : 0;
    p.eps = float(args.eps);
    p.mu = float(args.mu);
    p.decay = float(args.decay);
    p.rate = float(args.rate);
    p.workspace = workspace.data_ptr();
    check_launch(nangila_orth(&p, at::cuda::getCurrentCUDAStream()), "orthogonalize");
  }
  return out;
}
// Whether what is written (params and momenta) shares memory with anything else in the lists: the updates would depend on an order.
bool overlapping(const std::vector<Tensor>& written, const std::vector<Tensor>& read) {
  struct Span {
    uintptr_t from, to;
    bool written;
  };
  std::vector<Span> spans;
  auto add = [&](const std::vector<Tensor>& ts, bool w) {
    for (const Tensor& t : ts) {
      if (t.numel() == 0) continue;
      int64_t last = 0;
      for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
      const auto from = reinterpret_cast<uintptr_t>(t.data_ptr());
      spans.push_back({from, from + uintptr_t((last + 1) * t.element_size()), w});
    }
  };
  add(written, true);
  add(read, false);
  std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) { return a.from < b.from; });
  uintptr_t end_any = 0, end_written = 0;
  for (const Span& s : spans) {
    if (s.from < (s.written ? end_any : end_written)) return true;
    end_any = std::max(end_any, s.to);
    if (s.written) end_written = std::max(end_written, s.to);
  }
  return false;
}

void check_matrix(const Tensor& t, const char* name) {
  check_tensor(t, name);
  TORCH_CHECK_VALUE(t.dim() == 2 && t.size(0) >= 1 && t.size(1) >= 1 && t.size(0) <= 65536 && t.size(1) <= 65536, "nangila: ", name,
                    " must be matrices of 1 x 1 to 65536 x 65536, got shape ", t.sizes());
}
template <typename Same>
std::vector<std::vector<int64_t>> grouped(size_t n, const Same& same) {
  std::vector<std::vector<int64_t>> groups;
  for (size_t i = 0; i < n; ++i) {
    auto it = std::find_if(groups.begin(), groups.end(), [&](const std::vector<int64_t>& g) { return same(size_t(g[0]), i); });
    if (it == groups.end()) groups.push_back({int64_t(i)});
    else it->push_back(int64_t(i));
  }
  return groups;
}
std::vector<Tensor> chosen(const std::vector<Tensor>& ts, const std::vector<int64_t>& which, bool packed = false) {
  std::vector<Tensor> out;
  out.reserve(which.size());
  for (const int64_t i : which) out.push_back(packed ? in_memory(ts[i]).contiguous() : ts[i]);
  return out;
}
// Results for the CUDA matrices among the updates; nothing (None) in the place of the others.
std::vector<c10::optional<Tensor>> orthogonalize(const std::vector<Tensor>& updates, const std::vector<double>& coefficients, double eps) {
  at::NoGradGuard no_grad;
  check_schedule(coefficients);
  bool cuda = false;
  for (const Tensor& t : updates) {
    check_matrix(t, "updates");
    if (!t.is_cuda()) continue;
    check_followed(t);
    cuda = true;
  }
  if (cuda) check_no_tracer();
  std::vector<c10::optional<Tensor>> out(updates.size());
  for (const auto& g : grouped(updates.size(), [&](size_t i, size_t j) {
         return updates[i].sizes() == updates[j].sizes() && updates[i].scalar_type() == updates[j].scalar_type() && updates[i].device() == updates[j].device();
       })) {
    if (!updates[g[0]].is_cuda()) continue;
    const Tensor stack = orth_group(chosen(updates, g, true), {}, {}, OrthArgs{coefficients, eps, 0.0, 1.0, 0.0, false});
    for (size_t k = 0; k < g.size(); ++k) out[g[k]] = stack.select(0, int64_t(k));
  }
  return out;
}
// The step of the CUDA parameters among them; returns the indices of the others. scale: 0 sqrt(max(1, rows / cols)), 1 0.2 sqrt(max(rows, cols)), 2 one.
// Everything is checked before anything changes.
std::vector<int64_t> muon_step(const std::vector<Tensor>& params, const std::vector<Tensor>& grads, const std::vector<Tensor>& momenta, const std::vector<double>& coefficients, double eps,
                               double mu, bool nesterov, double lr, double weight_decay, int64_t scale) {
  at::NoGradGuard no_grad;
  check_schedule(coefficients);
  TORCH_CHECK_VALUE(params.size() == grads.size() && params.size() == momenta.size(), "nangila: ", params.size(), " parameters, ", grads.size(), " gradients and ",
                    momenta.size(), " momenta");
  bool cuda = false;
  for (size_t i = 0; i < params.size(); ++i) {
    const Tensor &p = params[i], &g = grads[i], &m = momenta[i];
    check_matrix(p, "parameters");
    check_matrix(g, "gradients");
    check_matrix(m, "momenta");
    TORCH_CHECK_VALUE(p.sizes() == g.sizes() && p.sizes() == m.sizes() && p.device() == g.device() && p.device() == m.device(), "nangila: parameter ", i, " is ", p.sizes(), " on ",
                      p.device(), ", its gradient ", g.sizes(), " on ", g.device(), ", its momentum ", m.sizes(), " on ", m.device());
    TORCH_CHECK_TYPE(m.scalar_type() == at::kFloat, "nangila: momenta must be float32, got ", m.scalar_type());
    TORCH_CHECK_VALUE(p.is_contiguous() && m.is_contiguous(), "nangila: parameter ", i, " and its momentum must be packed (contiguous)");
    if (!p.is_cuda()) continue;
    TORCH_CHECK_VALUE(!p.is_neg() && !m.is_neg() && !p._is_zerotensor() && !m._is_zerotensor(), "nangila: parameter ", i, " or its momentum is a view whose values are not in memory");
    for (const Tensor* t : {&p, &g, &m}) check_followed(*t);
    cuda = true;
  }
  if (cuda) check_no_tracer();
  std::vector<Tensor> written = params;
  written.insert(written.end(), momenta.begin(), momenta.end());
  TORCH_CHECK_VALUE(!overlapping(written, grads), "nangila: parameters and momenta must not share memory with one another or with the gradients");
  std::vector<int64_t> others;
  for (const auto& g : grouped(params.size(), [&](size_t i, size_t j) {
         return params[i].sizes() == params[j].sizes() && params[i].scalar_type() == params[j].scalar_type() && grads[i].scalar_type() == grads[j].scalar_type() &&
                params[i].device() == params[j].device();
       })) {
    const Tensor& first = params[g[0]];
    if (!first.is_cuda()) {
      others.insert(others.end(), g.begin(), g.end());
      continue;
    }
    const double rows = double(first.size(0)), cols = double(first.size(1));
    const double size = scale == 0 ? std::sqrt(std::max(1.0, rows / cols)) : scale == 1 ? 0.2 * std::sqrt(std::max(rows, cols)) : 1.0;
    orth_group(chosen(grads, g, true), chosen(momenta, g), chosen(params, g), OrthArgs{coefficients, eps, mu, 1.0 - lr * weight_decay, lr * size, nesterov});
    // the kernels write where autograd does not look: what was saved for a backward pass is not what it was
    for (const int64_t i : g)
      for (const Tensor* t : {&params[i], &momenta[i]})
        if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
  }
  return others;
}

}  // namespace

void register_model(py::module_& m) {
  m.def("rms_norm", &rms_norm, py::arg("x"), py::arg("weight"), py::arg("eps"));
  m.def("add_rms_norm", &add_rms_norm, py::arg("x"), py::arg("residual"), py::arg("weight"), py::arg("eps"));
  m.def("rms_norm_fp8", &rms_norm_fp8, py::arg("x"), py::arg("weight"), py::arg("eps"), py::arg("residual") = py::none(), py::arg("group") = 0);
  m.def("rotary", &rotary, py::arg("q"), py::arg("k"), py::arg("table"), py::arg("positions"), py::arg("half"));
  m.def("orthogonalize", &orthogonalize, py::arg("updates"), py::arg("coefficients"), py::arg("eps"));
  m.def("muon_step", &muon_step, py::arg("params"), py::arg("grads"), py::arg("momenta"), py::arg("coefficients"), py::arg("eps"), py::arg("mu"), py::arg("nesterov"), py::arg("lr"),
        py::arg("weight_decay"), py::arg("scale"));
}
