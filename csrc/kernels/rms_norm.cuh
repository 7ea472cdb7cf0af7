// Launch interface of the root-mean-square norm kernels (rms_norm.cu).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace mgfa {

enum class NormType : int { kBf16 = 0, kF16 = 1, kF32 = 2 };

// Rows [rows, dim]; a row stride per tensor in elements, the last dimension contiguous.
struct NormFwdParams {
  const void* x = nullptr;
  const void* residual = nullptr;  // null: h = x
  const void* weight = nullptr;    // [dim], x's type or (weight_f32, where that is another) fp32
  void* y = nullptr;               // [rows, dim] packed, x's type; or 8-bit when scale is set
  void* h = nullptr;               // [rows, dim] packed, written when residual is set
  float* rstd = nullptr;           // [rows], written when set
  float* scale = nullptr;          // 8-bit output: [rows, dim / group] (group 0: [rows])
  int64_t rows = 0;
  int64_t x_stride = 0, r_stride = 0;
  int dim = 0;
  int group = 0;
  int weight_f32 = 0;
  int layout = 2;  // 0: rows on 16-byte boundaries, dim a multiple of 16 bytes; 1: row r is
                   // r * dim elements behind such a boundary; 2: any
  float eps = 0.f;
};

struct NormBwdParams {
  const void* dy = nullptr;      // null: no gradient reaches y
  const void* dh = nullptr;      // null: no gradient reaches h
  const void* h = nullptr;       // the stream that the norm read
  const void* weight = nullptr;
  const float* rstd = nullptr;   // [rows]
  void* dx = nullptr;            // [rows, dim] packed
  float* dw_part = nullptr;      // [norm_bwd_parts(...), dim]; null: no weight gradient
  void* dw = nullptr;            // [dim], the weight's type
  int64_t rows = 0;
  int64_t dy_stride = 0, dh_stride = 0, h_stride = 0;
  int dim = 0;
  int weight_f32 = 0;
  int layout = 2;
};

constexpr int kNormMaxDim = 16384;

void rms_norm_fwd_launch(NormType t, const NormFwdParams& p, int sm_count, cudaStream_t stream);
// Rows of dw_part: one per CTA of the backward kernel.
int rms_norm_bwd_parts(NormType t, const NormBwdParams& p, int sm_count);
void rms_norm_bwd_launch(NormType t, const NormBwdParams& p, int parts, cudaStream_t stream);

}  // namespace mgfa
