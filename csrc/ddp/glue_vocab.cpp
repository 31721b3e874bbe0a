// Bindings of the operators at a language model's two ends: token embeddings, dropout, the loss of a head whose logits are not kept. The checks of arguments are
// here, for tensors of either device; CPU tensors take the formulas in ATen operations, CUDA tensors the kernels, on the current stream of their device.
#include <ATen/CPUGeneratorImpl.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/CUDAGraphsUtils.cuh>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/engine.h>
#include <torch/extension.h>

#include <cmath>
#include <cstring>
#include <mutex>
#include <tuple>
#include <vector>

#include "glue_checks.hpp"
#include "nangila_kernels.h"
#include "nangila_vocab_kernels.h"

namespace py = pybind11;

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

using namespace nangila::glue;

bool capturing() { return at::cuda::currentStreamCaptureStatusMayInitCtx() != at::cuda::CaptureStatus::None; }

// ---- dropout -----------------------------------------------------------------------------------------------------
struct Mask {
  int64_t least, draw, seed;  // the seed's 64 bits
  Tensor seed_tensor;         // in its place
  double scale() const { return least == int64_t(1) << 32 ? 0.0 : 1.0 / (1.0 - double(least) / 4294967296.0); }
};
Tensor dropout_launch(const Tensor& x_in, const Tensor& residual_in, const Mask& mask) {
  c10::cuda::CUDAGuard guard(x_in.device());
  const Tensor x = in_memory(x_in).contiguous(), residual = residual_in.defined() ? in_memory(residual_in).contiguous() : residual_in;
  const Tensor out = at::empty(x.sizes(), x.options());
  NangilaDropoutParams p;
  std::memset(&p, 0, sizeof p);
  p.n = x.numel();
  if (p.n == 0) return out;
  p.x = x.data_ptr();
  p.residual = residual.defined() ? residual.data_ptr() : nullptr;
  p.out = out.data_ptr();
  p.seed = uint64_t(mask.seed);
  p.seed_ptr = mask.seed_tensor.defined() ? mask.seed_tensor.data_ptr<int64_t>() : nullptr;
  p.least = uint64_t(mask.least);
  p.draw = uint32_t(mask.draw);
  p.dtype = dtype_code(x);
  p.scale = float(mask.scale());
  check_launch(nangila_dropout(&p, at::cuda::getCurrentCUDAStream()), "dropout");
  return out;
}
void philox(uint32_t (&c)[4], uint64_t seed) {
  uint32_t k0 = uint32_t(seed), k1 = uint32_t(seed >> 32);
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = uint64_t(0xD2511F53u) * c[0], b = uint64_t(0xCD9E8D57u) * c[2];
    const uint32_t n[4] = {uint32_t(b >> 32) ^ c[1] ^ k0, uint32_t(b), uint32_t(a >> 32) ^ c[3] ^ k1, uint32_t(a)};
    std::memcpy(c, n, sizeof n);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
}
// Which elements are kept, as the kernel has it.
Tensor cpu_kept(at::IntArrayRef sizes, const Mask& mask) {
  Tensor kept = at::empty(sizes, at::TensorOptions().dtype(at::kBool));
  const uint64_t seed = mask.seed_tensor.defined() ? uint64_t(mask.seed_tensor.item<int64_t>()) : uint64_t(mask.seed);
  bool* to = kept.data_ptr<bool>();
  const int64_t n = kept.numel();
  for (int64_t block = 0; block * 8 < n; ++block) {
    uint32_t upper[4] = {uint32_t(block), uint32_t(uint64_t(block) >> 32), uint32_t(mask.draw), 0}, lower[4] = {upper[0], upper[1], upper[2], 1};
    philox(upper, seed);
    philox(lower, seed);
    for (int64_t i = 0; i < 8 && block * 8 + i < n; ++i) {
      const int s = (i & 1) ? 16 : 0;
      const uint32_t number = (upper[i / 2] >> s & 0xffffu) << 16 | (lower[i / 2] >> s & 0xffffu);
      to[block * 8 + i] = int64_t(number) >= mask.least;
    }
  }
  return kept;
}
class Dropout : public torch::autograd::Function<Dropout> {
 public:
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const c10::optional<Tensor>& residual, const c10::optional<Tensor>& seed_tensor, int64_t least, int64_t draw, int64_t seed) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Mask mask{least, draw, seed, seed_tensor.value_or(Tensor())};
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({mask.seed_tensor});
    ctx->saved_data["residual"] = residual.has_value();
    ctx->saved_data["least"] = least;
    ctx->saved_data["draw"] = draw;
    ctx->saved_data["seed"] = seed;
    return dropout_launch(x, residual.value_or(Tensor()), mask);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once_only();
    variable_list out(6);
    const Tensor& dy = grads[0];
    if (!dy.defined()) return out;
    check_unseen({&dy});
    const bool residual = ctx->saved_data["residual"].toBool();
    const Mask mask{ctx->saved_data["least"].toInt(), ctx->saved_data["draw"].toInt(), ctx->saved_data["seed"].toInt(), ctx->get_saved_variables()[0]};
    check_saved(!mask.seed_tensor.defined() || saved_as(mask.seed_tensor, at::kLong, 1, dy.device()));
    if (ctx->needs_input_grad(0)) out[0] = dropout_launch(dy, Tensor(), mask);
    if (residual && ctx->needs_input_grad(1)) out[1] = dy;
    return out;
  }
};
Tensor dropout(const Tensor& x, const c10::optional<Tensor>& residual_in, int64_t least, int64_t draw, const c10::optional<int64_t>& seed_in, const c10::optional<Tensor>& seed_tensor) {
  const Tensor residual = residual_in.value_or(Tensor());
  check_tensor(x, "x");
  if (residual.defined()) {
    check_plain(residual, "residual");
    TORCH_CHECK_VALUE(residual.sizes() == x.sizes(), "nangila: residual has shape ", residual.sizes(), ", x ", x.sizes());
    TORCH_CHECK_TYPE(residual.scalar_type() == x.scalar_type(), "nangila: residual is ", residual.scalar_type(), ", x ", x.scalar_type());
    TORCH_CHECK_VALUE(residual.device() == x.device(), "nangila: residual is on ", residual.device(), ", x on ", x.device());
  }
  check_no_tracer();  // (a mask would become a constant)
  if (x.is_cuda()) check_unseen({&x, &residual});
  TORCH_CHECK_VALUE(least >= 0 && least <= int64_t(1) << 32 && draw >= 0 && draw < int64_t(1) << 32, "nangila: p or draw out of range");
  Mask mask{least, draw, seed_in.value_or(0), seed_tensor.value_or(Tensor())};
  if (mask.seed_tensor.defined()) {
    const Tensor& t = mask.seed_tensor;
    check_plain(t, "the seed");
    TORCH_CHECK_TYPE(t.scalar_type() == at::kLong, "nangila: the seed must be int64, not ", t.scalar_type());
    TORCH_CHECK_VALUE(t.numel() == 1, "nangila: the seed must be one number, got shape ", t.sizes());
    TORCH_CHECK_VALUE(t.device() == x.device(), "nangila: the seed is on ", t.device(), ", x on ", x.device());
    mask.seed_tensor = in_memory(t);
  } else if (!seed_in.has_value()) {
    c10::cuda::OptionalCUDAGuard guard;
    if (x.is_cuda()) guard.set_device(x.device());
    TORCH_CHECK(!x.is_cuda() || !capturing(), "nangila: a captured graph would repeat one mask for ever; give it a seed (a tensor, which can be changed between replays)");
    auto* gen = at::get_generator_or_default<at::CPUGeneratorImpl>(c10::nullopt, at::detail::getDefaultCPUGenerator());
    std::lock_guard<std::mutex> lock(gen->mutex_);
    mask.seed = int64_t(gen->random64());
  }
  if (x.is_cpu()) {
    // (formed in float32 and rounded once, like the kernel)
    const Tensor kept = cpu_kept(x.sizes(), mask);
    Tensor y = at::where(kept, x.to(at::kFloat) * mask.scale(), at::zeros({}, x.options().dtype(at::kFloat)));
    if (residual.defined()) y = y + residual.to(at::kFloat);
    return y.to(x.scalar_type());
  }
  if (!wants_grad({&x, &residual})) return dropout_launch(x, residual, mask);
  return Dropout::apply(x, residual_in, mask.seed_tensor.defined() ? c10::optional<Tensor>(mask.seed_tensor) : c10::nullopt, mask.least, mask.draw, mask.seed);
}

// ---- token embeddings -----------------------------------------------------------------------------------------------
void check_ids(const Tensor& ids, const char* name) {
  check_plain(ids, name);
  TORCH_CHECK_TYPE(ids.scalar_type() == at::kLong || ids.scalar_type() == at::kInt, "nangila: ", name, " must be int64 or int32, not ", ids.scalar_type());
}
std::vector<int64_t> with_width(at::IntArrayRef sizes, int64_t d) {
  std::vector<int64_t> shape = sizes.vec();
  shape.push_back(d);
  return shape;
}
Tensor embedding_launch(const Tensor& ids_in, const Tensor& weight_in, double scale) {
  c10::cuda::CUDAGuard guard(weight_in.device());
  const int64_t d = weight_in.size(1);
  const Tensor ids = in_memory(ids_in).contiguous();
  const Tensor out = at::empty(with_width(ids.sizes(), d), weight_in.options());
  NangilaEmbeddingParams p;
  std::memset(&p, 0, sizeof p);
  p.n = ids.numel();
  if (p.n == 0) return out;
  const Tensor weight = as_rows(weight_in, d, &p.weight_stride);
  p.ids = ids.data_ptr();
  p.weight = weight.data_ptr();
  p.out = out.data_ptr();
  p.rows = weight.size(0);
  p.d = int32_t(d);
  p.dtype = dtype_code(weight);
  p.ids_64 = ids.scalar_type() == at::kLong ? 1 : 0;
  p.scale = float(scale);
  check_launch(nangila_embedding(&p, at::cuda::getCurrentCUDAStream()), "embedding");
  return out;
}
class Embedding : public torch::autograd::Function<Embedding> {
 public:
  static Tensor forward(AutogradContext* ctx, const Tensor& weight, const Tensor& ids, double scale, int64_t padding) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({ids});
    ctx->saved_data["rows"] = weight.size(0);
    ctx->saved_data["d"] = weight.size(1);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding"] = padding;
    return embedding_launch(ids, weight, scale);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once_only();
    variable_list out(4);
    const Tensor& dy_in = grads[0];
    if (!dy_in.defined() || !ctx->needs_input_grad(0)) return out;
    check_unseen({&dy_in});
    c10::cuda::CUDAGuard guard(dy_in.device());
    const Tensor saved = ctx->get_saved_variables()[0];
    NangilaEmbeddingGradParams p;
    std::memset(&p, 0, sizeof p);
    p.rows = ctx->saved_data["rows"].toInt();
    p.d = int32_t(ctx->saved_data["d"].toInt());
    p.n = dy_in.numel() / p.d;
    check_saved(saved_as(saved, at::kLong, p.n, dy_in.device()) || saved_as(saved, at::kInt, p.n, dy_in.device()));
    const Tensor ids = in_memory(saved).contiguous();
    if (p.n == 0) {
      out[0] = at::zeros({p.rows, p.d}, dy_in.options());
      return out;
    }
    const Tensor dy = as_rows(dy_in, p.d, &p.dy_stride);
    out[0] = at::empty({p.rows, p.d}, dy.options());
    const Tensor workspace = at::empty({nangila_embedding_workspace(p.n, p.rows, p.d)}, dy.options().dtype(at::kByte));
    p.ids = ids.data_ptr();
    p.dy = dy.data_ptr();
    p.dw = out[0].data_ptr();
    p.workspace = workspace.data_ptr();
    p.padding = ctx->saved_data["padding"].toInt();
    p.dtype = dtype_code(dy);
    p.ids_64 = ids.scalar_type() == at::kLong ? 1 : 0;
    p.scale = float(ctx->saved_data["scale"].toDouble());
    check_launch(nangila_embedding_backward(&p, at::cuda::getCurrentCUDAStream()), "embedding gradient");
    return out;
  }
};
Tensor embedding(const Tensor& ids, const Tensor& weight, double scale, const c10::optional<int64_t>& padding_in) {
  check_ids(ids, "ids");
  check_tensor(weight, "weight");
  TORCH_CHECK_VALUE(weight.dim() == 2 && weight.size(0) >= 1 && weight.size(1) >= 1 && weight.size(0) <= NANGILA_EMBEDDING_MAX_ROWS && weight.size(1) <= NANGILA_EMBEDDING_MAX_WIDTH,
                    "nangila: weight must have shape [rows, width], up to ", NANGILA_EMBEDDING_MAX_ROWS, " and ", NANGILA_EMBEDDING_MAX_WIDTH, ", got ", weight.sizes());
  TORCH_CHECK_VALUE(ids.device() == weight.device(), "nangila: ids are on ", ids.device(), ", weight on ", weight.device());
  TORCH_CHECK_VALUE(std::isfinite(scale), "nangila: scale must be finite, got ", scale);
  TORCH_CHECK_VALUE(ids.numel() <= NANGILA_EMBEDDING_MAX_TOKENS, "nangila: up to ", NANGILA_EMBEDDING_MAX_TOKENS, " ids, got ", ids.numel());
  int64_t padding = -1;
  if (padding_in.has_value()) {
    padding = *padding_in;
    TORCH_CHECK_VALUE(padding >= -weight.size(0) && padding < weight.size(0), "nangila: padding_idx must be a row of weight (", weight.size(0), " rows), got ", padding);
    if (padding < 0) padding += weight.size(0);
  }
  if (weight.is_cpu()) {
    const Tensor outside = (ids < 0).logical_or(ids >= weight.size(0));
    const Tensor y = at::embedding(weight.to(at::kFloat), ids.to(at::kLong).clamp(0, weight.size(0) - 1), padding) * scale;
    return at::where(outside.unsqueeze(-1), at::full({}, NAN, y.options()), y).to(weight.scalar_type()).contiguous();
  }
  check_unseen({&weight});
  if (!wants_grad({&weight})) return embedding_launch(ids, weight, scale);
  return Embedding::apply(weight, ids, scale, padding);
}

// ---- the head's loss -----------------------------------------------------------------------------------------------
enum Reduction { kNone, kMean, kSum };
struct Head {
  Tensor x, weight, bias, targets;  // x and weight as the kernels take them
  int64_t n, d, width;              // columns; of x and weight as they are given
  NangilaLinearCeParams p;
};
// Rows that the kernels' copies of tiles can start from: packed to a multiple of eight columns where they are not.
Tensor tile_rows(const Tensor& t, int64_t width, int64_t d, int64_t* stride) {
  Tensor rows = as_rows(t, width, stride);
  if (width == d && *stride % 8 == 0 && *stride >= d && (reinterpret_cast<uintptr_t>(rows.data_ptr()) & 15u) == 0) return rows;
  *stride = d;
  rows = rows.reshape({-1, width});
  return width == d ? rows.clone(at::MemoryFormat::Contiguous) : at::constant_pad_nd(rows, {0, d - width});
}
Head head_of(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& targets, int64_t classes, int64_t ignore, bool mean) {
  Head h;
  std::memset(&h.p, 0, sizeof h.p);
  h.width = x.size(-1);
  h.d = (h.width + 7) / 8 * 8;
  h.n = targets.numel();
  h.x = tile_rows(x, h.width, h.d, &h.p.x_stride);
  h.weight = tile_rows(weight, h.width, h.d, &h.p.w_stride);
  h.targets = in_memory(targets).to(at::kLong).contiguous();
  if (bias.defined()) h.bias = in_memory(bias).contiguous();
  h.p.x = h.x.data_ptr();
  h.p.w = h.weight.data_ptr();
  h.p.bias = h.bias.defined() ? h.bias.data_ptr() : nullptr;
  h.p.targets = h.targets.data_ptr<int64_t>();
  h.p.n = h.n;
  h.p.ignore = ignore;
  h.p.d = int32_t(h.d);
  h.p.rows = int32_t(weight.size(0));
  h.p.classes = int32_t(classes);
  h.p.dtype = dtype_code(x);
  h.p.bias_dtype = h.bias.defined() ? dtype_code(h.bias) : 0;
  h.p.mean = mean ? 1 : 0;
  return h;
}
void head_launch(Head& h, int what) {
  const int64_t bytes = nangila_linear_ce_workspace(&h.p, what);
  TORCH_CHECK(bytes >= 0, "nangila: linear_cross_entropy failed: invalid argument");
  const Tensor workspace = at::empty({bytes}, h.x.options().dtype(at::kByte));
  h.p.workspace = workspace.data_ptr();
  check_launch(nangila_linear_ce(&h.p, what, at::cuda::getCurrentCUDAStream()), "linear_cross_entropy");
}
struct HeadGrads {
  Tensor dx, dw, db;  // dx and dw with padded columns
};
HeadGrads head_gradients(Head& h, bool want_x, bool want_w, bool want_b, at::ScalarType db_type) {
  HeadGrads g;
  if (want_x) g.dx = at::empty({h.n, h.d}, h.x.options());
  if (want_w) g.dw = at::empty({h.p.rows, h.d}, h.weight.options());
  if (want_b) g.db = at::empty({h.p.rows}, h.bias.options().dtype(db_type));
  h.p.dx = want_x ? g.dx.data_ptr() : nullptr;
  h.p.dw = want_w ? g.dw.data_ptr() : nullptr;
  h.p.dbias = want_b ? g.db.data_ptr() : nullptr;
  return g;
}
// the loss or losses, and what a backward pass needs: losses and lse, and with `both` the gradients for an upstream gradient of one
struct HeadOut {
  Tensor result, losses, lse;  // (losses of their own, where the result may change under a caller's hands)
  HeadGrads grads;
};
HeadOut head_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& targets, int64_t classes, int64_t ignore, int64_t reduction, bool both, bool keep) {
  c10::cuda::CUDAGuard guard(x.device());
  const at::TensorOptions f32 = x.options().dtype(at::kFloat);
  HeadOut o;
  o.losses = at::empty(targets.sizes(), f32);
  o.lse = at::empty(targets.sizes(), f32);
  if (reduction != kNone) o.result = targets.numel() == 0 ? at::full({}, reduction == kMean ? NAN : 0.0, f32) : at::empty({}, f32);
  else o.result = keep ? at::empty(targets.sizes(), f32) : o.losses;
  if (targets.numel() == 0) return o;
  Head h = head_of(x, weight, bias, targets, classes, ignore, reduction == kMean);
  h.p.losses = o.losses.data_ptr<float>();
  h.p.lse = o.lse.data_ptr<float>();
  h.p.loss = reduction != kNone ? o.result.data_ptr<float>() : nullptr;
  h.p.losses_too = reduction == kNone && keep ? o.result.data_ptr<float>() : nullptr;
  if (both) o.grads = head_gradients(h, x.requires_grad(), weight.requires_grad(), bias.defined() && bias.requires_grad(), at::kFloat);
  head_launch(h, both ? NANGILA_CE_BOTH : NANGILA_CE_LOSSES);
  return o;
}
class LinearCrossEntropy : public torch::autograd::Function<LinearCrossEntropy> {
 public:
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const c10::optional<Tensor>& bias_in, const Tensor& targets, int64_t classes, int64_t ignore, int64_t reduction) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor bias = bias_in.value_or(Tensor());
    // One upstream gradient for all rows: bf16 has the range to form the gradients along with the losses. (Half precision waits for the scale of its loss.)
    const bool both = reduction != kNone && x.scalar_type() == at::kBFloat16 && targets.numel() > 0;
    HeadOut o = head_forward(x, weight, bias, targets, classes, ignore, reduction, both, true);
    ctx->set_materialize_grads(false);
    // (what has been formed among them: hooks on saved tensors, and checkpoints, have it in their hands)
    ctx->save_for_backward({x, weight, bias, targets, o.losses, o.lse, o.grads.dx, o.grads.dw, o.grads.db});
    ctx->saved_data["rows"] = weight.size(0);
    ctx->saved_data["classes"] = classes;
    ctx->saved_data["ignore"] = ignore;
    ctx->saved_data["reduction"] = reduction;
    ctx->saved_data["both"] = both;
    return o.result;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once_only();
    variable_list out(7);
    const Tensor& upstream_in = grads[0];
    if (!upstream_in.defined()) return out;
    check_unseen({&upstream_in});
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1], &bias = saved[2], &targets = saved[3];
    const bool want_x = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1), want_b = bias.defined() && ctx->needs_input_grad(2);
    const int64_t reduction = ctx->saved_data["reduction"].toInt(), width = x.size(-1);
    const int64_t n = targets.numel(), rows = weight.size(0), padded = (width + 7) / 8 * 8;
    const at::ScalarType type = x.scalar_type();
    const at::Device device = upstream_in.device();
    check_saved((type == at::kHalf || type == at::kBFloat16) && saved_as(x, type, n * width, device) && saved_as(weight, type, rows * width, device) && weight.dim() == 2 &&
                rows == ctx->saved_data["rows"].toInt() && (saved_as(targets, at::kLong, n, device) || saved_as(targets, at::kInt, n, device)) && saved_as(saved[4], at::kFloat, n, device) &&
                saved_as(saved[5], at::kFloat, n, device) && upstream_in.numel() == (reduction == kNone ? n : 1) &&
                (!bias.defined() || (known(bias.scalar_type()) && saved_as(bias, bias.scalar_type(), rows, device))));
    if (n == 0) {
      if (want_x) out[0] = at::zeros_like(x);
      if (want_w) out[1] = at::zeros_like(weight);
      if (want_b) out[2] = at::zeros_like(bias);
      return out;
    }
    c10::cuda::CUDAGuard guard(x.device());
    const Tensor upstream = in_memory(upstream_in).to(at::kFloat).contiguous();
    HeadGrads g;
    if (ctx->saved_data["both"].toBool()) {
      // What the forward pass has formed is multiplied in place and given away, unless it is wanted again: by another pass over the same graph, or when a captured pass is replayed.
      const bool keep = capturing() || torch::autograd::get_current_graph_task_keep_graph();
      NangilaRescaleParams r;
      std::memset(&r, 0, sizeof r);
      int i = 0;
      Tensor formed_db;
      auto scaled = [&](const Tensor& formed, bool want) {
        if (!want) return Tensor();
        const Tensor t = keep ? formed.clone(at::MemoryFormat::Contiguous) : formed.contiguous();
        r.array[i] = t.data_ptr();
        r.count[i] = t.numel();
        r.dtype[i] = dtype_code(t);
        ++i;
        return t;
      };
      check_saved((!want_x || saved_as(saved[6], type, n * padded, device)) && (!want_w || saved_as(saved[7], type, rows * padded, device)) &&
                  (!want_b || saved_as(saved[8], at::kFloat, rows, device)));
      g.dx = scaled(saved[6], want_x);
      g.dw = scaled(saved[7], want_w);
      if (want_b) {  // (held in float32 until now: the rounding is that of the bias's type, which may have no place for what comes before the upstream gradient)
        formed_db = saved[8].contiguous();
        g.db = at::empty({rows}, bias.options());
        r.wide = formed_db.data_ptr<float>();
        r.narrow = g.db.data_ptr();
        r.narrow_count = g.db.numel();
        r.narrow_dtype = dtype_code(g.db);
      }
      r.factor = upstream.data_ptr<float>();
      check_launch(nangila_rescale(&r, at::cuda::getCurrentCUDAStream()), "linear_cross_entropy gradient");
    } else {
      Head h = head_of(x, weight, bias, targets, ctx->saved_data["classes"].toInt(), ctx->saved_data["ignore"].toInt(), reduction == kMean);
      const Tensor losses = saved[4].contiguous(), lse = saved[5].contiguous();
      h.p.losses = losses.data_ptr<float>();
      h.p.lse = lse.data_ptr<float>();
      h.p.upstream = upstream.data_ptr<float>();
      h.p.upstream_rows = reduction == kNone ? 1 : 0;
      g = head_gradients(h, want_x, want_w, want_b, want_b ? bias.scalar_type() : at::kFloat);
      head_launch(h, NANGILA_CE_GRADIENTS);
    }
    auto unpadded = [&](const Tensor& t) { return t.size(1) == width ? t : t.narrow(1, 0, width).contiguous(); };
    if (want_x) out[0] = unpadded(g.dx).view(x.sizes());
    if (want_w) out[1] = unpadded(g.dw);
    if (want_b) out[2] = g.db;
    return out;
  }
};
Tensor linear_cross_entropy(const Tensor& x, const Tensor& weight, const Tensor& targets, const c10::optional<Tensor>& bias_in, const c10::optional<int64_t>& classes_in, int64_t ignore,
                            int64_t reduction) {
  const Tensor bias = bias_in.value_or(Tensor());
  check_tensor(x, "x");
  check_tensor(weight, "weight");
  check_ids(targets, "targets");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= NANGILA_CE_MAX_WIDTH, "nangila: the last dimension of x must have 1 to ", NANGILA_CE_MAX_WIDTH, " values, got shape ", x.sizes());
  TORCH_CHECK_VALUE(weight.dim() == 2 && weight.size(1) == x.size(-1) && weight.size(0) >= 1 && weight.size(0) <= NANGILA_CE_MAX_CLASSES, "nangila: weight must have shape [classes, ", x.size(-1),
                    "], 1 to ", NANGILA_CE_MAX_CLASSES, " classes, not ", weight.sizes());
  TORCH_CHECK_TYPE(weight.scalar_type() == x.scalar_type(), "nangila: weight is ", weight.scalar_type(), ", x ", x.scalar_type());
  TORCH_CHECK_VALUE(weight.device() == x.device(), "nangila: weight is on ", weight.device(), ", x on ", x.device());
  TORCH_CHECK_VALUE(targets.sizes() == x.sizes().slice(0, x.dim() - 1), "nangila: targets have shape ", targets.sizes(), ", x ", x.sizes());
  TORCH_CHECK_VALUE(targets.device() == x.device(), "nangila: targets are on ", targets.device(), ", x on ", x.device());
  if (bias.defined()) {
    check_tensor(bias, "bias");
    TORCH_CHECK_VALUE(bias.dim() == 1 && bias.size(0) == weight.size(0), "nangila: bias must have shape [", weight.size(0), "], not ", bias.sizes());
    TORCH_CHECK_VALUE(bias.device() == x.device(), "nangila: bias is on ", bias.device(), ", x on ", x.device());
  }
  const int64_t classes = classes_in.value_or(weight.size(0));
  TORCH_CHECK_VALUE(classes >= 1 && classes <= weight.size(0), "nangila: num_classes must be 1 to ", weight.size(0), " (the rows of weight), got ", classes);
  TORCH_CHECK_VALUE(reduction >= kNone && reduction <= kSum, "nangila: unknown reduction");
  if (x.is_cpu()) {
    c10::impl::ExcludeDispatchKeyGuard in_float(c10::autocast_dispatch_keyset);  // (autocast would form the logits in 16 bits)
    // (rows that add nothing and the padding stay out of the products: what they hold would come back as 0 times that)
    const Tensor t = targets.to(at::kLong), ignored = t == ignore, outside = (t < 0).logical_or(t >= classes).logical_and(ignored.logical_not());
    const Tensor rows = x.to(at::kFloat).masked_fill(ignored.logical_or(outside).unsqueeze(-1), 0.0);
    const Tensor z = at::linear(rows, weight.narrow(0, 0, classes).to(at::kFloat), bias.defined() ? bias.narrow(0, 0, classes).to(at::kFloat) : bias);
    const Tensor zt = z.gather(-1, t.clamp(0, classes - 1).unsqueeze(-1)).squeeze(-1);
    Tensor losses = at::where(ignored, at::zeros({}, z.options()), z.logsumexp(-1) - zt);
    losses = at::where(outside, at::full({}, NAN, z.options()), losses);
    if (reduction == kNone) return losses;
    return reduction == kSum ? losses.sum() : losses.sum() / ignored.logical_not().sum();
  }
  TORCH_CHECK_TYPE(x.scalar_type() != at::kFloat, "nangila: the kernels take float16 and bfloat16 on a CUDA device, not float32 (under torch.autocast it is cast)");
  check_unseen({&x, &weight, &bias});
  if (!wants_grad({&x, &weight, &bias})) return head_forward(x, weight, bias, targets, classes, ignore, reduction, false, false).result;
  return LinearCrossEntropy::apply(x, weight, bias_in, targets, classes, ignore, reduction);
}

}  // namespace

void register_vocab(py::module_& m) {
  m.def("dropout", &dropout, py::arg("x"), py::arg("residual"), py::arg("least"), py::arg("draw"), py::arg("seed"), py::arg("seed_tensor"));
  m.def("embedding", &embedding, py::arg("ids"), py::arg("weight"), py::arg("scale"), py::arg("padding_idx"));
  m.def("linear_cross_entropy", &linear_cross_entropy, py::arg("x"), py::arg("weight"), py::arg("targets"), py::arg("bias"), py::arg("num_classes"), py::arg("ignore_index"), py::arg("reduction"));
}
