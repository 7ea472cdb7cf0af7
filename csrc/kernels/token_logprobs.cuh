// Launch interface of the token log probabilities (token_logprobs.cu).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace mgfa {

enum class LogitType : int { kBf16 = 0, kF16 = 1, kF32 = 2 };

constexpr int kLogprobMaxTop = 32;

// Rows [rows, vocab] with a contiguous vocab.
struct LogprobParams {
  const void* x = nullptr;
  int64_t stride = 0;  // of rows, in elements
  int64_t rows = 0;
  int vocab = 0;
  const void* targets = nullptr;  // [rows]
  int targets64 = 0;              // int64 (else int32)
  int64_t ignore = 0;
  float* logprobs = nullptr;  // [rows]
  float* entropy = nullptr;   // [rows]
  float* stats = nullptr;     // [rows, 4]: the largest logit m, S = sum e^(x - m), ln S, entropy; or null
  int top = 0;                // 0 to kLogprobMaxTop
  float* top_logprobs = nullptr;    // [rows, top]
  int64_t* top_indices = nullptr;
  uint32_t* status = nullptr;
};

struct LogprobBwdParams : LogprobParams {
  const float* dl = nullptr;  // gradients of logprobs and entropy: [rows] with strides, or null
  const float* dh = nullptr;
  int64_t dl_stride = 0, dh_stride = 0;
  void* dx = nullptr;  // [rows, vocab] packed, x's type
};

void token_logprobs_launch(LogitType t, const LogprobParams& p, int sm_count, cudaStream_t stream);
void token_logprobs_bwd_launch(LogitType t, const LogprobBwdParams& p, int sm_count, cudaStream_t stream);

}  // namespace mgfa
