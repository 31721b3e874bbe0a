// Checks of arguments that the bindings of the model's operators share.
#pragma once
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <cuda_runtime.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <initializer_list>

#include "nangila_kernels.h"

namespace nangila {
namespace glue {

using at::Tensor;

inline bool known(at::ScalarType t) { return t == at::kFloat || t == at::kHalf || t == at::kBFloat16; }
inline int dtype_code(const Tensor& t) { return t.scalar_type() == at::kFloat ? NANGILA_F32 : t.scalar_type() == at::kHalf ? NANGILA_F16 : NANGILA_BF16; }
inline void check_launch(int err, const char* what) { TORCH_CHECK(err == 0, "nangila: ", what, " failed: ", cudaGetErrorString(static_cast<cudaError_t>(err))); }
inline void check_plain(const Tensor& t, const char* name) {
  TORCH_CHECK_TYPE(!t.unsafeGetTensorImpl()->is_python_dispatch(), "nangila: ", name, " must be a plain tensor, not one that wraps another (a sharded one has to be gathered first)");
  TORCH_CHECK_TYPE(t.layout() == at::kStrided, "nangila: ", name, " must be dense");
  TORCH_CHECK_TYPE(t.is_cuda() || t.is_cpu(), "nangila: ", name, " must be on a CUDA device or the CPU");
}
inline void check_tensor(const Tensor& t, const char* name) {
  check_plain(t, name);
  TORCH_CHECK_TYPE(known(t.scalar_type()), "nangila: ", name, " must be float32, float16 or bfloat16, not ", t.scalar_type());
}
// The kernels write into fresh memory behind the dispatcher's back. What follows the operations of PyTorch from there (forward-mode derivatives, tracers,
// tensors that stand for others) would not see them, and go on as if the results were constants: such calls are refused.
inline void check_followed(const Tensor& t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(0).defined(),
                              "nangila: the kernels have no forward-mode derivative; give them tensors without a tangent (forward_ad.unpack_dual(..).primal), or CPU tensors");
}
inline void check_no_tracer() {
  using c10::impl::TorchDispatchModeKey;
  using c10::impl::TorchDispatchModeTLS;
  TORCH_CHECK_NOT_IMPLEMENTED(!torch::jit::tracer::isTracing(), "nangila: the kernels cannot be traced (torch.jit.trace)");
  if (!TorchDispatchModeTLS::any_modes_set()) return;
  for (const TorchDispatchModeKey key : {TorchDispatchModeKey::FAKE, TorchDispatchModeKey::PROXY, TorchDispatchModeKey::FUNCTIONAL})
    TORCH_CHECK_NOT_IMPLEMENTED(!TorchDispatchModeTLS::get_mode(key).has_value(), "nangila: the kernels cannot be traced (make_fx, export or fake tensors)");
}
inline void check_unseen(std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts) check_followed(*t);
  check_no_tracer();
}
inline bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}
inline void once_only() {
  TORCH_CHECK(!at::GradMode::is_enabled(), "nangila: this gradient cannot be differentiated again (create_graph=True)");
}

// What comes back of a saved tensor goes through a user's hooks, if there are some, and the kernels take its memory as it is.
inline void check_saved(bool as_it_was) { TORCH_CHECK_VALUE(as_it_was, "nangila: a hook on saved tensors gave back a tensor of another shape, type or device than it was given"); }
inline bool saved_as(const Tensor& t, at::ScalarType type, int64_t numel, const at::Device& device) {
  return t.defined() && t.layout() == at::kStrided && t.scalar_type() == type && t.numel() == numel && t.device() == device;
}

// The tensor with its values in memory: a view that is negated only when it is read has others there, zeros that nobody has read yet have none.
inline Tensor in_memory(const Tensor& t) {
  if (t._is_zerotensor()) return at::zeros(t.sizes(), t.options());
  return t.is_neg() ? t.resolve_neg() : t;
}

// `t` as rows of d adjacent values, `stride` apart: the tensor itself where its strides allow that, else a packed copy.
inline Tensor as_rows(const Tensor& given, int64_t d, int64_t* stride) {
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

}  // namespace glue
}  // namespace nangila
