// Torch-facing entry point of the token log probabilities (token_logprobs.cu).
#include <torch/csrc/autograd/custom_function.h>
#include <torch/types.h>
#include "../common/check.hpp"
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <tuple>
#include <vector>

#include "forward_ad.hpp"
#include "../kernels/token_logprobs.cuh"

namespace mgfa {

int device_sm_count(int device);
uint32_t* status_ptr(const torch::Tensor& t, const torch::Tensor& like);

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = c10::optional<torch::Tensor>;

LogitType logit_type(const torch::Tensor& t) {
  return t.scalar_type() == at::kBFloat16 ? LogitType::kBf16
         : t.scalar_type() == at::kHalf   ? LogitType::kF16
                                          : LogitType::kF32;
}

// [..., vocab] as rows of one stride with a contiguous last dimension (copied where the
// strides do not allow it).
torch::Tensor logit_rows(const torch::Tensor& x) {
  torch::Tensor r = x.dim() == 2 ? x : x.reshape({x.numel() / x.size(-1), x.size(-1)});
  return r.stride(1) != 1 ? r.contiguous() : r;
}

void check_logits(const torch::Tensor& x, const torch::Tensor& targets, int64_t top) {
  MGFA_CHECK(x.is_cuda(), "logits must be a CUDA tensor");
  MGFA_CHECK(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf || x.scalar_type() == at::kFloat,
             "logits must be bfloat16, float16 or float32");
  MGFA_CHECK(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) < (int64_t(1) << 30),
             "logits must be [..., vocab] with 1 to 2^30 - 1 entries");
  MGFA_CHECK(targets.is_cuda() && targets.device() == x.device() &&
                 (targets.scalar_type() == at::kInt || targets.scalar_type() == at::kLong),
             "targets must be an int32 or int64 CUDA tensor on the logits' device");
  MGFA_CHECK(targets.sizes() == x.sizes().slice(0, x.dim() - 1), "targets must have the logits' shape without the vocab");
  MGFA_CHECK(top >= 0 && top <= kLogprobMaxTop && top <= x.size(-1), "top must be 0 to ", kLogprobMaxTop,
             " and not above the vocab, got ", top);
}

struct Logprobs {
  torch::Tensor logprobs, entropy, top_logprobs, top_indices, stats;
};

Logprobs logprobs_fwd(const torch::Tensor& x, const torch::Tensor& targets_in, int64_t top, int64_t ignore,
                      const torch::Tensor& status, bool need_stats) {
  check_logits(x, targets_in, top);
  c10::cuda::CUDAGuard guard(x.device());
  const torch::Tensor rows = logit_rows(x), targets = targets_in.contiguous();
  const auto f32 = x.options().dtype(at::kFloat);
  std::vector<int64_t> sizes = targets.sizes().vec();
  Logprobs o;
  o.logprobs = torch::empty(sizes, f32);
  o.entropy = torch::empty(sizes, f32);
  if (need_stats) o.stats = torch::empty({rows.size(0), 4}, f32);
  LogprobParams p;
  if (top) {
    sizes.push_back(top);
    o.top_logprobs = torch::empty(sizes, f32);
    o.top_indices = torch::empty(sizes, x.options().dtype(at::kLong));
    p.top_logprobs = o.top_logprobs.data_ptr<float>();
    p.top_indices = o.top_indices.data_ptr<int64_t>();
  }
  p.x = rows.data_ptr();
  p.stride = rows.stride(0);
  p.rows = rows.size(0);
  p.vocab = int(rows.size(1));
  p.targets = targets.data_ptr();
  p.targets64 = targets.scalar_type() == at::kLong;
  p.ignore = ignore;
  p.logprobs = o.logprobs.data_ptr<float>();
  p.entropy = o.entropy.data_ptr<float>();
  p.stats = need_stats ? o.stats.data_ptr<float>() : nullptr;
  p.top = int(top);
  p.status = status_ptr(status, x);
  if (p.rows > 0)
    token_logprobs_launch(logit_type(x), p, device_sm_count(x.get_device()), at::cuda::getCurrentCUDAStream());
  return o;
}

// A gradient [rows] with the stride of its only dimension.
const float* grad_rows(torch::Tensor& g, int64_t& stride) {
  if (!g.defined()) return nullptr;
  g = g.reshape({-1});
  stride = g.stride(0);
  return g.data_ptr<float>();
}

struct TokenLogprobsFn : torch::autograd::Function<TokenLogprobsFn> {
  static variable_list forward(AutogradContext* ctx, const torch::Tensor& x, const torch::Tensor& targets,
                               int64_t top, int64_t ignore, const torch::Tensor& status) {
    Logprobs o = logprobs_fwd(x, targets, top, ignore, status, true);
    ctx->save_for_backward({x, targets, o.stats});
    ctx->saved_data["ignore"] = ignore;
    ctx->set_materialize_grads(false);
    if (!top) return {o.logprobs, o.entropy};
    ctx->mark_non_differentiable({o.top_logprobs, o.top_indices});
    return {o.logprobs, o.entropy, o.top_logprobs, o.top_indices};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    torch::Tensor dl = grads[0], dh = grads[1];
    if (!dl.defined() && !dh.defined()) return variable_list(5);
    refuse_tangents("token_logprobs' gradient", {dl, dh});
    const variable_list saved = ctx->get_saved_variables();
    const torch::Tensor &x = saved[0], targets = saved[1].contiguous(), &stats = saved[2];
    c10::cuda::CUDAGuard guard(x.device());
    const torch::Tensor rows = logit_rows(x);
    torch::Tensor dx = torch::empty(x.sizes(), x.options());
    LogprobBwdParams p;
    p.x = rows.data_ptr();
    p.stride = rows.stride(0);
    p.rows = rows.size(0);
    p.vocab = int(rows.size(1));
    p.targets = targets.data_ptr();
    p.targets64 = targets.scalar_type() == at::kLong;
    p.ignore = ctx->saved_data["ignore"].toInt();
    p.stats = stats.data_ptr<float>();
    p.dl = grad_rows(dl, p.dl_stride);
    p.dh = grad_rows(dh, p.dh_stride);
    p.dx = dx.data_ptr();
    if (p.rows > 0) 
      token_logprobs_bwd_launch(logit_type(x), p, device_sm_count(x.get_device()), at::cuda::getCurrentCUDAStream());
    return once({dx, {}, {}, {}, {}});
  }
};

}  // namespace

// logprobs and entropy (float32, the targets' shape) and, with `top`, the likeliest
// alternatives' log probabilities and indices [..., top].
std::tuple<torch::Tensor, torch::Tensor, OptTensor, OptTensor> token_logprobs(
    torch::Tensor logits, torch::Tensor targets, int64_t top, int64_t ignore, torch::Tensor status) {
  refuse_tangents("token_logprobs", {logits});
  if (at::GradMode::is_enabled() && logits.requires_grad()) {
    variable_list o = TokenLogprobsFn::apply(logits, targets, top, ignore, status);
    if (!top) return {o[0], o[1], {}, {}};
    return {o[0], o[1], o[2], o[3]};
  }
  Logprobs o = logprobs_fwd(logits, targets, top, ignore, status, false);
  if (!top) return {o.logprobs, o.entropy, {}, {}};
  return {o.logprobs, o.entropy, o.top_logprobs, o.top_indices};
}

}  // namespace mgfa
