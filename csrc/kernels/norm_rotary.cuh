// Launch interface of the kernels that norm and rotate query and key heads (norm_rotary.cu).
#pragma once

#include "paged_cache.cuh"
#include "rotary.cuh"

namespace mgfa {

struct NormRotaryParams : RotaryParams {
  const void* weight[2] = {nullptr, nullptr};  // [head_dim], x's type or (weight_f32) fp32
  int weight_f32 = 0;
  float eps = 0.f;
  // backward: x[i].in are the forward's inputs and x[i].out their gradients
  RotaryTensor dy[2];        // the outputs' gradients (in and strides)
  float* dw_part = nullptr;  // [parts, 2, head_dim]; null: no weight gradient
  void* dw[2] = {nullptr, nullptr};
};

// The same on the way into a cache: x[0].out packed, keys and values to their pages.
struct CacheAppendParams : NormRotaryParams {
  int norm = 0;    // 0: positions alone
  RotaryTensor v;  // values (in and strides)
  CacheState c;
  void* k_pool = nullptr;  // the layer's
  void* v_pool = nullptr;
  int64_t k_stride[3] = {0, 0, 0}, v_stride[3] = {0, 0, 0};  // page, token, head
  const int* slots = nullptr;
  const int* cu = nullptr;
  int seqs = 0;
};

void norm_rotary_launch(RotaryType t, const NormRotaryParams& p, int sm_count, cudaStream_t stream);
// Rows of dw_part: one per CTA of the backward kernel.
int norm_rotary_bwd_parts(RotaryType t, const NormRotaryParams& p, int sm_count);
void norm_rotary_bwd_launch(RotaryType t, const NormRotaryParams& p, int parts, int sm_count,
                            cudaStream_t stream);
// 16-bit types, p.vec.
void cache_append_launch(RotaryType t, const CacheAppendParams& p, int sm_count, cudaStream_t stream);

}  // namespace mgfa
