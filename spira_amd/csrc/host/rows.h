// What the row operators' sources share: checks of their tensors, and what their
// gradients need of autograd.
#pragma once

#include "host_common.h"

#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

namespace spira_host {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Tensor = torch::Tensor;
using OptTensor = std::optional<torch::Tensor>;

inline int row_dtype(const Tensor &t) {
  switch (t.scalar_type()) {
    case torch::kHalf: return SPIRA_F16;
    case torch::kBFloat16: return SPIRA_BF16;
    case torch::kFloat: return SPIRA_F32;
    default: fail("Cannot find implementation for feature dtype ", t.scalar_type());
  }
}

inline const void *ptr(const OptTensor &t) { return t ? t->data_ptr() : nullptr; }

// t is a contiguous tensor of this type, on x's device, of these sizes (-1: any)
inline void require(const Tensor &t, const char *name, const Tensor &x, torch::ScalarType type,
                    std::initializer_list<int64_t> sizes) {
  require_device(t, name);
  SPIRA_CHECK_ARG(t.device() == x.device(), name, " must be on ", x.device());
  SPIRA_CHECK_ARG(t.scalar_type() == type, name, " must be ", type, ", got ", t.scalar_type());
  bool fits = t.dim() == static_cast<int64_t>(sizes.size());
  int64_t d = 0;
  for (int64_t s : sizes) {
    if (fits && s >= 0 && t.size(d) != s) fits = false;
    ++d;
  }
  if (!fits) {
    std::ostringstream os;
    for (int64_t s : sizes) os << (os.tellp() > 0 ? ", " : "") << (s < 0 ? std::string("any") : std::to_string(s));
    fail(name, " must have the shape [", os.str(), "], got ", t.sizes());
  }
}
inline void require(const OptTensor &t, const char *name, const Tensor &x, torch::ScalarType type,
                    std::initializer_list<int64_t> sizes) {
  if (t) require(*t, name, x, type, sizes);
}

inline Tensor like(const Tensor &x, torch::IntArrayRef sizes) { return torch::empty(sizes, x.options()); }
inline Tensor floats(const Tensor &x, torch::IntArrayRef sizes) {
  return torch::empty(sizes, x.options().dtype(torch::kFloat));
}

inline Tensor dense(const Tensor &t) { return t.contiguous(); }
inline OptTensor dense(const OptTensor &t) { return t ? OptTensor(t->contiguous()) : t; }

// Whether the call needs a node in the graph.  A tangent of forward mode would be
// lost without a word, here and within a node, and read as zero: it is refused.
inline bool tracked(const char *name, std::initializer_list<const OptTensor *> ts) {
  if (c10::AutogradState::get_tls_state().get_fw_grad_mode())
    for (const OptTensor *t : ts)
      SPIRA_CHECK_ARG(!*t || !(*t)->_fw_grad(0).defined(), name, ": there are no derivatives of forward mode");
  if (!torch::GradMode::is_enabled()) return false;
  for (const OptTensor *t : ts)
    if (*t && (*t)->requires_grad()) return true;
  return false;
}
inline bool wants(const OptTensor &t) { return t && t->requires_grad(); }

inline Tensor given(const OptTensor &t) { return t ? *t : Tensor(); }
inline OptTensor maybe(const Tensor &t) { return t.defined() ? OptTensor(t) : std::nullopt; }

// Gradients are of first order: with a graph of them asked for, they carry a
// node that fails when it is differentiated.
inline variable_list once(variable_list grads, const char *name) {
  if (!torch::GradMode::is_enabled()) return grads;
  variable_list some;
  for (const Tensor &g : grads)
    if (g.defined()) some.push_back(g.detach().requires_grad_(true));
  auto error = std::make_shared<torch::autograd::DelayedError>(
      std::string("[Spira] ") + name + ": gradients are of first order", static_cast<int64_t>(some.size()));
  some = (*error)(std::move(some));
  size_t i = 0;
  for (Tensor &g : grads)
    if (g.defined()) g = some[i++];
  return grads;
}

}  // namespace spira_host
