// Torch-facing entry points of the per-token operators of a decoder layer:
// root-mean-square norm (rms_norm.cu) and rotary positions (rotary.cu).
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/types.h>
#include "../common/check.hpp"
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <algorithm>
#include <tuple>
#include <vector>

#include "forward_ad.hpp"
#include "../kernels/rms_norm.cuh"
#include "../kernels/rotary.cuh"

namespace mgfa {

int device_sm_count(int device);

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = c10::optional<torch::Tensor>;

NormType norm_type(const torch::Tensor& t, const char* name) {
  MGFA_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  switch (t.scalar_type()) {
    case at::kBFloat16: return NormType::kBf16;
    case at::kHalf: return NormType::kF16;
    case at::kFloat: return NormType::kF32;
    default: MGFA_CHECK(false, name, " must be bfloat16, float16 or float32");
  }
  return NormType::kF32;
}

// [..., dim] as rows of one stride with a contiguous last dimension (copied where the
// strides do not allow it).
torch::Tensor as_rows(const torch::Tensor& t) {
  const int64_t dim = t.size(-1);
  torch::Tensor r = t.dim() == 2 ? t : t.reshape({t.numel() / dim, dim});
  if (r.stride(1) != 1 || r.stride(0) < 0) r = r.contiguous();
  return r;
}

// Whether row i of r starts i * dim elements behind a 16-byte boundary, up to whole
// vectors of v elements. A width that is no multiple of a vector has its rows' edges read
// with their neighbours', so the rows must not overlap.
bool rows_vec(const torch::Tensor& r, int64_t dim, int v) {
  return reinterpret_cast<uintptr_t>(r.data_ptr()) % 16 == 0 &&
         (r.size(0) <= 1 ||
          ((r.stride(0) - dim) % v == 0 && (dim % v == 0 || r.stride(0) >= dim)));
}

// NormFwdParams::layout of rows (of undefined tensors: none); the outputs are packed. A
// weight of x's type is read in vectors where the rows are aligned.
int norm_layout(int64_t dim, std::initializer_list<const torch::Tensor*> rows,
                const torch::Tensor& weight) {
  const torch::Tensor& x = **rows.begin();
  const int v = 16 / int(x.element_size());
  for (const torch::Tensor* r : rows)
    if (r->defined() && !rows_vec(*r, dim, v)) return 2;
  // A shifted row's vectors reach up to v - 1 columns into its neighbours: it has to fit a
  // block with them, and the row behind it has to hold them.
  if (dim % v) return dim >= v - 1 && dim + v - 1 <= kNormMaxDim ? 1 : 2;
  return weight.scalar_type() != x.scalar_type() ||
                 reinterpret_cast<uintptr_t>(weight.data_ptr()) % 16 == 0
             ? 0 : 1;
}

void check_norm_inputs(const torch::Tensor& x, const torch::Tensor& weight,
                       const OptTensor& residual) {
  norm_type(x, "x");
  MGFA_CHECK(x.dim() >= 1, "x must be [..., dim]");
  const int64_t dim = x.size(-1);
  MGFA_CHECK(dim >= 1 && dim <= kNormMaxDim, "x: the last dimension must be 1 to ", kNormMaxDim,
             ", got ", dim);
  MGFA_CHECK(weight.is_cuda() && weight.dim() == 1 && weight.size(0) == dim,
             "weight must be a CUDA tensor [dim]");
  MGFA_CHECK(weight.scalar_type() == x.scalar_type() || weight.scalar_type() == at::kFloat,
             "weight must have x's dtype or be float32");
  MGFA_CHECK(weight.device() == x.device(), "weight must be on x's device");
  if (residual.has_value()) {
    MGFA_CHECK(residual->scalar_type() == x.scalar_type() && residual->sizes() == x.sizes(),
               "residual must have x's dtype and shape");
    MGFA_CHECK(residual->device() == x.device(), "residual must be on x's device");
  }
}

struct NormFwd {
  torch::Tensor y, h, rstd, scale;
};

NormFwd norm_fwd(const torch::Tensor& x, const torch::Tensor& weight_in, const OptTensor& residual,
                 double eps, bool need_rstd, bool eight, int64_t group) {
  check_norm_inputs(x, weight_in, residual);
  const int dim = int(x.size(-1));
  MGFA_CHECK(eps >= 0.0, "eps must not be negative");
  if (eight)
    MGFA_CHECK(group == 0 || ((group == 16 || group == 32 || group == 64 || group == 128) &&
                              dim % group == 0),
               "group must be 0 (a scale for each row) or 16, 32, 64 or 128 columns that divide dim");
  c10::cuda::CUDAGuard guard(x.device());
  const NormType t = norm_type(x, "x");
  const int v = t == NormType::kF32 ? 4 : 8;
  torch::Tensor xr = as_rows(x), rr, weight = weight_in.contiguous();
  if (residual.has_value()) rr = as_rows(*residual);
  int layout = norm_layout(dim, {&xr, &rr}, weight);
  if (group && layout != 0) {  // the scales of column groups need aligned vectors
    if (!rows_vec(xr, dim, v)) xr = xr.clone(at::MemoryFormat::Contiguous);
    if (rr.defined() && !rows_vec(rr, dim, v)) rr = rr.clone(at::MemoryFormat::Contiguous);
    weight = weight.clone();
    layout = 0;
  }
  NormFwd out;
  out.y = torch::empty(x.sizes(), x.options().dtype(eight ? at::kFloat8_e4m3fn : x.scalar_type()));
  if (rr.defined()) out.h = torch::empty(x.sizes(), x.options());
  const auto f32 = x.options().dtype(at::kFloat);
  if (need_rstd) out.rstd = torch::empty({xr.size(0)}, f32);
  if (eight) {
    std::vector<int64_t> sizes = x.sizes().vec();
    sizes.back() = group ? dim / group : 1;
    out.scale = torch::empty(sizes, f32);
  }
  NormFwdParams p;
  p.x = xr.data_ptr();
  p.weight = weight.data_ptr();
  p.weight_f32 = weight.scalar_type() != x.scalar_type();
  p.y = out.y.data_ptr();
  p.rows = xr.size(0);
  p.x_stride = xr.stride(0);
  if (rr.defined()) {
    p.residual = rr.data_ptr();
    p.r_stride = rr.stride(0);
    p.h = out.h.data_ptr();
  }
  p.rstd = need_rstd ? out.rstd.data_ptr<float>() : nullptr;
  p.scale = eight ? out.scale.data_ptr<float>() : nullptr;
  p.dim = dim;
  p.group = int(group);
  p.layout = layout;
  p.eps = float(eps);
  MGFA_CHECK(p.rows < (int64_t(1) << 31), "too many rows");
  if (p.rows > 0) {
    rms_norm_fwd_launch(t, p, device_sm_count(x.get_device()), at::cuda::getCurrentCUDAStream());
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
  return out;
}

OptTensor opt(const torch::Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }

}  // namespace

// y (e4m3), scale [..., dim / group] (group 0: [..., 1]) and h (with a residual).
std::tuple<torch::Tensor, torch::Tensor, OptTensor> rms_norm_fp8(torch::Tensor x,
                                                                 torch::Tensor weight,
                                                                 OptTensor residual, double eps,
                                                                 int64_t group) {
  refuse_tangents("rms_norm_fp8", {x, weight, residual.value_or(torch::Tensor())});
  NormFwd o = norm_fwd(x, weight, residual, eps, false, true, group);
  return {o.y, o.scale, opt(o.h)};
}

namespace {

// dx (which is the residual's gradient too) and the weight's gradient (when asked for)
// from the gradients of y and h, either of which may be undefined.
std::tuple<torch::Tensor, torch::Tensor> norm_bwd(const torch::Tensor& dy, const torch::Tensor& dh,
                                                  const torch::Tensor& h,
                                                  const torch::Tensor& weight_in,
                                                  const torch::Tensor& rstd, bool need_dw) {
  check_norm_inputs(h, weight_in, opt(dh));
  if (dy.defined())
    MGFA_CHECK(dy.scalar_type() == h.scalar_type() && dy.sizes() == h.sizes() &&
                   dy.device() == h.device(),
               "dy must match the stream's dtype, shape and device");
  const int dim = int(h.size(-1));
  c10::cuda::CUDAGuard guard(h.device());
  const NormType t = norm_type(h, "h");
  torch::Tensor hr = as_rows(h), dyr, dhr, weight = weight_in.contiguous();
  if (dy.defined()) dyr = as_rows(dy);
  if (dh.defined()) dhr = as_rows(dh);
  torch::Tensor dx = torch::empty(h.sizes(), h.options()), dw, part;
  NormBwdParams p;
  p.h = hr.data_ptr();
  p.h_stride = hr.stride(0);
  if (dyr.defined()) {
    p.dy = dyr.data_ptr();
    p.dy_stride = dyr.stride(0);
  }
  if (dhr.defined()) {
    p.dh = dhr.data_ptr();
    p.dh_stride = dhr.stride(0);
  }
  p.weight = weight.data_ptr();
  p.weight_f32 = weight.scalar_type() != h.scalar_type();
  p.rstd = rstd.data_ptr<float>();
  p.dx = dx.data_ptr();
  p.rows = hr.size(0);
  p.dim = dim;
  p.layout = norm_layout(dim, {&hr, &dyr, &dhr}, weight);
  if (p.rows == 0) {
    if (need_dw) dw = torch::zeros({dim}, weight.options());
    return {dx, dw};
  }
  const int parts = rms_norm_bwd_parts(t, p, device_sm_count(h.get_device()));
  if (need_dw) {
    dw = torch::empty({dim}, weight.options());
    part = torch::empty({parts, dim}, h.options().dtype(at::kFloat));
    p.dw = dw.data_ptr();
    p.dw_part = part.data_ptr<float>();
  }
  rms_norm_bwd_launch(t, p, parts, at::cuda::getCurrentCUDAStream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {dx, dw};
}

// Gradients that cannot be differentiated again: an error where that is tried.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  for (auto& g : grads)
    if (g.defined()) g = g.detach().requires_grad_(true);
  auto node = std::make_shared<torch::autograd::DelayedError>(
      "this operator's gradient has no gradient of its own", int(grads.size()));
  return (*node)(std::move(grads));
}

struct RmsNormFn : torch::autograd::Function<RmsNormFn> {
  static variable_list forward(AutogradContext* ctx, const torch::Tensor& x,
                               const torch::Tensor& weight, const OptTensor& residual, double eps) {
    NormFwd o = norm_fwd(x, weight, residual, eps, true, false, 0);
    ctx->save_for_backward({o.h.defined() ? o.h : x, weight, o.rstd});
    ctx->set_materialize_grads(false);
    if (!o.h.defined()) return {o.y};
    return {o.y, o.h};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const bool res = grads.size() > 1;
    const torch::Tensor dy = grads[0], dh = res ? grads[1] : torch::Tensor();
    if (!dy.defined() && !dh.defined()) return {{}, {}, {}, {}};
    refuse_tangents("rms_norm's gradient", {dy, dh});
    const variable_list saved = ctx->get_saved_variables();
    auto [dx, dw] = norm_bwd(dy, dh, saved[0], saved[1], saved[2], ctx->needs_input_grad(1));
    return once({ctx->needs_input_grad(0) ? dx : torch::Tensor(), dw,
                 res && ctx->needs_input_grad(2) ? dx : torch::Tensor(), {}});
  }
};

bool wants_grad(const torch::Tensor& a, const OptTensor& b) {
  return at::GradMode::is_enabled() && (a.requires_grad() || (b.has_value() && b->requires_grad()));
}

}  // namespace

// y and h (with a residual); differentiable.
std::tuple<torch::Tensor, OptTensor> rms_norm(torch::Tensor x, torch::Tensor weight,
                                              OptTensor residual, double eps) {
  refuse_tangents("rms_norm", {x, weight, residual.value_or(torch::Tensor())});
  if (wants_grad(x, residual) || wants_grad(weight, {})) {
    variable_list o = RmsNormFn::apply(x, weight, residual, eps);
    return {o[0], o.size() > 1 ? OptTensor(o[1]) : OptTensor()};
  }
  NormFwd o = norm_fwd(x, weight, residual, eps, false, false, 0);
  return {o.y, opt(o.h)};
}

// How the kernels read the rows of x, weight and residual (NormFwdParams::layout), on any
// device: for tests of the rule.
int64_t norm_layout_of(torch::Tensor x, torch::Tensor weight, OptTensor residual) {
  const torch::Tensor xr = as_rows(x), rr = residual.has_value() ? as_rows(*residual) : torch::Tensor();
  return norm_layout(x.size(-1), {&xr, &rr}, weight);
}

// ------------------------------------------------------------------ rotary positions
namespace {

RotaryTensor rotary_tensor(const torch::Tensor& t, torch::Tensor& out, const char* name) {
  MGFA_CHECK(t.dim() == 3 || t.dim() == 4, name,
             " must be [tokens, heads, head_dim] or [batch, tokens, heads, head_dim]");
  RotaryTensor r;
  out = torch::empty(t.sizes(), t.options());
  r.in = t.data_ptr();
  r.out = out.data_ptr();
  r.stride_b = t.dim() == 4 ? t.stride(0) : 0;
  r.stride_t = t.stride(-3);
  r.stride_h = t.stride(-2);
  r.heads = int(t.size(-2));
  return r;
}

}  // namespace

namespace {

// q (and k) with rotary positions; sign -1 rotates back (the gradient).
std::tuple<torch::Tensor, torch::Tensor> rotary(torch::Tensor q, const OptTensor& k_in,
                                                const torch::Tensor& positions,
                                                const torch::Tensor& inv_freq, bool interleaved,
                                                double magnitude, double sign) {
  const NormType t = norm_type(q, "q");
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
  torch::Tensor k, qo, ko;
  if (q.stride(-1) != 1) q = q.contiguous();
  if (k_in.has_value()) {
    k = *k_in;
    MGFA_CHECK(k.is_cuda() && k.device() == q.device() && k.scalar_type() == q.scalar_type() &&
                   k.dim() == q.dim() && k.size(-1) == D && k.size(-3) == L &&
                   (k.dim() == 3 || k.size(0) == B),
               "k must match q in all but the number of heads");
    if (k.stride(-1) != 1) k = k.contiguous();
  }
  c10::cuda::CUDAGuard guard(q.device());
  RotaryParams p;
  p.x[0] = rotary_tensor(q, qo, "q");
  if (k.defined()) p.x[1] = rotary_tensor(k, ko, "k");
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
  p.sign = float(sign);
  const int v = t == NormType::kF32 ? 4 : 8;
  auto vec_tensor = [&](const RotaryTensor& r) {
    return reinterpret_cast<uintptr_t>(r.in) % 16 == 0 && r.stride_b % v == 0 &&
           r.stride_t % v == 0 && r.stride_h % v == 0;
  };
  p.vec = D % v == 0 && vec_tensor(p.x[0]) && (!k.defined() || vec_tensor(p.x[1]));
  MGFA_CHECK(p.x[0].heads + int64_t(p.x[1].heads) <= 4096, "at most 4096 heads");
  MGFA_CHECK(B * L < (int64_t(1) << 31), "too many tokens");
  if (B * L > 0 && p.x[0].heads + p.x[1].heads > 0) {
    rotary_launch(RotaryType(int(t)), p, device_sm_count(q.get_device()),
                  at::cuda::getCurrentCUDAStream());
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
  return {qo, ko};
}

struct RotaryFn : torch::autograd::Function<RotaryFn> {
  static variable_list forward(AutogradContext* ctx, const torch::Tensor& q, const OptTensor& k,
                               const torch::Tensor& positions, const torch::Tensor& inv_freq,
                               bool interleaved, double magnitude) {
    auto [qo, ko] = rotary(q, k, positions, inv_freq, interleaved, magnitude, 1.0);
    ctx->save_for_backward({positions, inv_freq});
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["magnitude"] = magnitude;
    ctx->set_materialize_grads(false);
    if (!ko.defined()) return {qo};
    return {qo, ko};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const torch::Tensor dq = grads[0], dk = grads.size() > 1 ? grads[1] : torch::Tensor();
    if (!dq.defined() && !dk.defined()) return {{}, {}, {}, {}, {}, {}};
    refuse_tangents("apply_rotary's gradient", {dq, dk});
    const variable_list saved = ctx->get_saved_variables();
    const bool il = ctx->saved_data["interleaved"].toBool();
    const double mag = ctx->saved_data["magnitude"].toDouble();
    if (!dq.defined())
      return once({{}, std::get<0>(rotary(dk, {}, saved[0], saved[1], il, mag, -1.0)), {}, {}, {}, {}});
    auto [gq, gk] = rotary(dq, opt(dk), saved[0], saved[1], il, mag, -1.0);
    return once({gq, gk, {}, {}, {}, {}});
  }
};

}  // namespace

std::tuple<torch::Tensor, OptTensor> apply_rotary(torch::Tensor q, OptTensor k,
                                                  torch::Tensor positions, torch::Tensor inv_freq,
                                                  bool interleaved, double magnitude) {
  refuse_tangents("apply_rotary", {q, k.value_or(torch::Tensor()), inv_freq});
  if (wants_grad(q, k)) {
    variable_list o = RotaryFn::apply(q, k, positions, inv_freq, interleaved, magnitude);
    return {o[0], o.size() > 1 ? OptTensor(o[1]) : OptTensor()};
  }
  auto [qo, ko] = rotary(q, k, positions, inv_freq, interleaved, magnitude, 1.0);
  return {qo, opt(ko)};
}

}  // namespace mgfa
