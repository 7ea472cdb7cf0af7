// Refusal of derivatives by operators that have none: forward-mode ones (the kernels would
// return values without the tangents) and those of gradients.
#pragma once

#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/types.h>
#include <c10/core/AutogradState.h>

#include "../common/check.hpp"

namespace mgfa {

// `name` is the operator; undefined tensors count as absent.
inline void refuse_tangents(const char* name, std::initializer_list<torch::Tensor> inputs) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const torch::Tensor& t : inputs)
    MGFA_CHECK(!t.defined() || !t._fw_grad(/*level=*/0).defined(), name,
               " has no forward-mode derivative");
}

// Gradients that cannot be differentiated again: an error where that is tried.
inline torch::autograd::variable_list once(torch::autograd::variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  for (auto& g : grads)
    if (g.defined()) g = g.detach().requires_grad_(true);
  auto node = std::make_shared<torch::autograd::DelayedError>(
      "this operator's gradient has no gradient of its own", int(grads.size()));
  return (*node)(std::move(grads));
}

}  // namespace mgfa
