// Refusal of forward-mode derivatives by operators that have none: the kernels would
// return values without the tangents.
#pragma once

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

}  // namespace mgfa
