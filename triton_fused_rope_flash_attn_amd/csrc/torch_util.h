// Helpers shared by the torch ops' native kernels (torch_ops.cpp, torch_seq_ops.cpp).
#pragma once

#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/function.h>
#include <torch/library.h>

#include <sstream>

#include "farope.h"

namespace farope_torch {

using at::Tensor;
using torch::autograd::variable_list;

inline int dtype_code(at::ScalarType t) {
  return t == at::kFloat ? FAROPE_F32 : t == at::kHalf ? FAROPE_F16 : t == at::kBFloat16 ? FAROPE_BF16 : -1;
}
inline std::string shape_str(const Tensor& t) {
  std::ostringstream s;
  s << '(';
  for (int64_t i = 0; i < t.dim(); ++i) s << (i ? ", " : "") << t.size(i);
  s << (t.dim() == 1 ? ",)" : ")");
  return s.str();
}
inline std::string dtype_str(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return "torch.float32";
    case at::kHalf: return "torch.float16";
    case at::kBFloat16: return "torch.bfloat16";
    case at::kDouble: return "torch.float64";
    default: return std::string("torch.") + c10::toString(t.scalar_type());
  }
}

inline void check_rc(int rc, const char* what) {
  TORCH_CHECK(rc == FAROPE_OK, what, ": ", farope_strerror(rc), " (status ", rc, ")");
}

inline const int64_t* strides(const Tensor& t) { return t.strides().data(); }
inline float* floats(const Tensor& t) { return t.defined() && t.numel() ? t.data_ptr<float>() : nullptr; }
inline void* data(const Tensor& t) { return t.numel() ? t.data_ptr() : nullptr; }
inline void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream(); }
inline Tensor workspace(const Tensor& like, size_t elems) {
  return elems ? at::empty({(int64_t)elems}, like.options().dtype(at::kFloat)) : Tensor();
}

inline bool any_requires_grad(std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// None of the ops has a forward-mode derivative: a tangent is refused, whether gradients are enabled or not.
inline void refuse_tangents(const char* op, std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    TORCH_CHECK(!t->defined() || !t->_fw_grad(0).defined(), "farope: ", op,
                " has no forward-mode derivative; detach the tangents of its inputs (torch.autograd.forward_ad)");
}

}  // namespace farope_torch
