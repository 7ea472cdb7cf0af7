// Arguments that the operators with rotary positions share: checks, and the kernels' view.
#pragma once

#include <torch/types.h>
#include "../common/check.hpp"

#include "../kernels/norm_rotary.cuh"

namespace mgfa {

inline RotaryTensor rotary_tensor(const torch::Tensor& t) {
  RotaryTensor r;
  r.in = t.data_ptr();
  r.stride_b = t.dim() == 4 ? t.stride(0) : 0;
  r.stride_t = t.stride(-3);
  r.stride_h = t.stride(-2);
  r.heads = int(t.size(-2));
  return r;
}

// Whether every head of t starts on a 16-byte boundary. (The strides of dimensions of size 1
// mean nothing.)
inline bool rotary_vec(const RotaryTensor& r, const torch::Tensor& t) {
  const int64_t v = 16 / t.element_size();
  auto fits = [&](int64_t dim, int64_t stride) { return t.size(dim) <= 1 || stride % v == 0; };
  return reinterpret_cast<uintptr_t>(r.in) % 16 == 0 && (t.dim() < 4 || fits(0, r.stride_b)) &&
         fits(-3, r.stride_t) && fits(-2, r.stride_h);
}

// All of p but the outputs; q and k are made contiguous where their last dimension is not.
inline RotaryType rotary_args(RotaryParams& p, torch::Tensor& q, torch::Tensor& k,
                              const torch::Tensor& positions, const torch::Tensor& inv_freq,
                              bool interleaved, double magnitude) {
  MGFA_CHECK(q.is_cuda(), "q must be a CUDA tensor");
  MGFA_CHECK(q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf ||
                 q.scalar_type() == at::kFloat,
             "q must be bfloat16, float16 or float32");
  MGFA_CHECK(q.dim() == 3 || q.dim() == 4,
             "q must be [tokens, heads, head_dim] or [batch, tokens, heads, head_dim]");
  const int64_t D = q.size(-1), L = q.size(-3), B = q.dim() == 4 ? q.size(0) : 1;
  MGFA_CHECK(D >= 2 && D <= 256, "head_dim must be 2 to 256, got ", D);
  MGFA_CHECK(inv_freq.is_cuda() && inv_freq.scalar_type() == at::kDouble && inv_freq.dim() == 1 &&
                 inv_freq.is_contiguous() && inv_freq.device() == q.device(),
             "inv_freq must be a contiguous float64 CUDA tensor [rotary_dim / 2] on q's device");
  MGFA_CHECK(inv_freq.numel() >= 1 && 2 * inv_freq.numel() <= D,
             "inv_freq has ", inv_freq.numel(), " entries for head_dim ", D);
  MGFA_CHECK(positions.is_cuda() && positions.device() == q.device() &&
                 (positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong),
             "positions must be an int32 or int64 CUDA tensor on q's device");
  MGFA_CHECK((positions.dim() == 1 && positions.size(0) == L) ||
                 (q.dim() == 4 && positions.dim() == 2 && positions.size(0) == B &&
                  positions.size(1) == L),
             "positions must be [tokens], or [batch, tokens] for a batch");
  if (q.stride(-1) != 1) q = q.contiguous();
  if (k.defined()) {
    MGFA_CHECK(k.is_cuda() && k.device() == q.device() && k.scalar_type() == q.scalar_type() &&
                   k.dim() == q.dim() && k.size(-1) == D && k.size(-3) == L &&
                   (k.dim() == 3 || k.size(0) == B),
               "k must match q in all but the number of heads");
    if (k.stride(-1) != 1) k = k.contiguous();
  }
  MGFA_CHECK(q.size(-2) + (k.defined() ? k.size(-2) : 0) <= 4096, "at most 4096 heads");
  MGFA_CHECK(B * L < (int64_t(1) << 31), "too many tokens");
  p.x[0] = rotary_tensor(q);
  if (k.defined()) p.x[1] = rotary_tensor(k);
  p.positions = positions.data_ptr();
  p.positions64 = positions.scalar_type() == at::kLong;
  p.pos_stride_b = positions.dim() == 2 ? positions.stride(0) : 0;
  p.pos_stride_t = positions.stride(-1);
  p.inv_freq = inv_freq.data_ptr<double>();
  p.batch = B;
  p.tokens = L;
  p.head_dim = int(D);
  p.rotary_dim = int(2 * inv_freq.numel());
  p.interleaved = interleaved;
  p.magnitude = float(magnitude);
  p.vec = D % (16 / q.element_size()) == 0 && rotary_vec(p.x[0], q) &&
          (!k.defined() || rotary_vec(p.x[1], k));
  return q.scalar_type() == at::kBFloat16 ? RotaryType::kBf16
         : q.scalar_type() == at::kHalf   ? RotaryType::kF16
                                          : RotaryType::kF32;
}

// The norms' weights and eps; `w` keeps the weights that the kernels read.
inline void norm_weight_args(NormRotaryParams& p, const torch::Tensor& q, const torch::Tensor& k,
                             const torch::Tensor& q_weight,
                             const c10::optional<torch::Tensor>& k_weight, double eps,
                             torch::Tensor (&w)[2]) {
  MGFA_CHECK(eps >= 0.0, "eps must not be negative");
  MGFA_CHECK(k.defined() == k_weight.has_value(), "k and k_weight come together");
  for (int i = 0; i < (k.defined() ? 2 : 1); ++i) {
    w[i] = i ? *k_weight : q_weight;
    const char* name = i ? "k_weight" : "q_weight";
    MGFA_CHECK(w[i].is_cuda() && w[i].dim() == 1 && w[i].size(0) == q.size(-1) && w[i].device() == q.device(),
               name, " must be a CUDA tensor [head_dim] on q's device");
    MGFA_CHECK(w[i].scalar_type() == q.scalar_type() || w[i].scalar_type() == at::kFloat, name,
               " must have q's dtype or be float32");
    MGFA_CHECK(w[i].scalar_type() == w[0].scalar_type(), "q_weight and k_weight must have one dtype");
    w[i] = w[i].contiguous();
    p.weight[i] = w[i].data_ptr();
  }
  p.weight_f32 = w[0].scalar_type() == at::kFloat;
  p.eps = float(eps);
}

}  // namespace mgfa
