// What the Python module's operators share (dense_autograd.cpp, moe_autograd.cpp): argument checks, the C
// ABI's errors as exceptions, the modes that a launch cannot take part in.
#pragma once
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include "../../include/lazylora_mxfp4.h"

namespace lazylora {


using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

inline int dtype_code(const Tensor& t)
{
  switch (t.scalar_type()) {
    case at::kFloat: return MXFP4_F32;
    case at::kBFloat16: return MXFP4_BF16;
    case at::kHalf: return MXFP4_F16;
    default: return -1;
  }
}

inline void check(int rc)
{
  if (rc == MXFP4_OK) return;
  TORCH_CHECK_VALUE(rc != MXFP4_EINVAL, mxfp4_last_error());
  TORCH_CHECK(false, "MXFP4 kernel failed (", rc, "): ", mxfp4_last_error());
}

inline hipStream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

// t with its values as they lie in memory: contiguous, and no view that stands for its negative (the imaginary part
// of a conjugate; one of a single element is contiguous).
inline Tensor laid_out(const Tensor& t) { return t.resolve_neg().contiguous(); }
// The same and 16-byte aligned (a copy where it is not).
inline Tensor tidy(const Tensor& t)
{
  Tensor c = laid_out(t);
  return reinterpret_cast<uintptr_t>(c.data_ptr()) & 15 ? c.clone() : c;
}
inline Tensor arg(const Tensor& t, const char* name, at::IntArrayRef shape, const Tensor& like, at::ScalarType dtype)
{
  TORCH_CHECK_VALUE(t.sizes() == shape && t.scalar_type() == dtype && t.device() == like.device(), name, " must be ",
                    dtype, " ", shape, " on ", like.device(), ", got ", t.scalar_type(), " ", t.sizes(), " on ",
                    t.device());
  return tidy(t);
}
inline void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
inline float* fptr(const Tensor& t) { return static_cast<float*>(ptr(t)); }
inline Tensor given(const OptTensor& t) { return t ? *t : Tensor(); }
inline bool records(at::ArrayRef<Tensor> ts)
{
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor& t : ts)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}
// A launch computes values and records nothing: it would drop a tensor's forward-mode tangent, which says that
// the derivative along it is zero, and a tracer would see the outputs allocated but not filled. The tensors of a
// function transform (vmap, batched gradients, torch.func.grad, functionalize) have no memory to launch over. Every
// call and every backward pass looks for these first.
inline void check_modes(at::ArrayRef<Tensor> ts)
{
  using c10::impl::TorchDispatchModeTLS;
  const bool traced = torch::jit::tracer::isTracing() ||
                      c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch) ||
                      (TorchDispatchModeTLS::any_modes_set() &&
                       TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value());
  TORCH_CHECK_NOT_IMPLEMENTED(!traced, "the operators of this package cannot be traced (torch.jit.trace, make_fx, "
                                       "torch.export): a trace would not hold their launches");
  using c10::DispatchKey;
  constexpr c10::DispatchKeySet transformed({DispatchKey::Batched, DispatchKey::FuncTorchBatched,
                                             DispatchKey::FuncTorchGradWrapper, DispatchKey::Functionalize});
  for (const Tensor& t : ts)
    TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t.key_set().has_any(transformed),
                                "the operators of this package cannot be transformed (torch.func.vmap, grad, functionalize, "
                                "batched gradients)");
  for (const Tensor& t : ts)
    TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(/*level=*/0).defined(),
                                "the operators of this package have no forward-mode derivative (an input or upstream gradient "
                                "carries a tangent)");
}
// Gradients that autograd may use but not differentiate: where a graph of them is asked for, a second
// derivative raises instead of coming out as zero.
inline variable_list once(variable_list grads)
{
  if (!at::GradMode::is_enabled()) return grads;
  variable_list some;
  for (const Tensor& g : grads)
    if (g.defined()) some.push_back(g.detach().requires_grad_(true));
  auto node = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function that was marked with once_differentiable", (int64_t)some.size());
  const variable_list marked = (*node)(std::move(some));
  size_t i = 0;
  for (Tensor& g : grads)
    if (g.defined()) g = marked[i++];
  return grads;
}

// The operators of moe_autograd.cpp.
void bind_moe(py::module_& m);

}  // namespace lazylora
