// Launch interface of the rotary position kernel (rotary.cu), and a pair's angle, which
// norm_rotary.cu uses too.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace mgfa {

enum class RotaryType : int { kBf16 = 0, kF16 = 1, kF32 = 2 };

// One of the tensors that are rotated together: [batch, tokens, heads, head_dim] with
// strides in elements and a contiguous head_dim; the output is packed.
struct RotaryTensor {
  const void* in = nullptr;
  void* out = nullptr;
  int64_t stride_b = 0, stride_t = 0, stride_h = 0;
  int heads = 0;
};

struct RotaryParams {
  RotaryTensor x[2];               // queries and keys (heads 0: absent)
  const void* positions = nullptr;  // [tokens], or [batch, tokens] when pos_stride_b != 0
  const double* inv_freq = nullptr; // [rotary_dim / 2], radians a position
  int64_t pos_stride_b = 0, pos_stride_t = 0;
  int64_t batch = 0, tokens = 0;
  int head_dim = 0, rotary_dim = 0;
  int positions64 = 0;   // int64 positions (else int32)
  int interleaved = 0;   // pairs (2i, 2i + 1); else (i, i + rotary_dim / 2)
  int vec = 0;           // 1: every head starts and ends on a 16-byte boundary
  float magnitude = 1.f; // factor on the rotated values
  float sign = 1.f;      // -1: the transpose, for gradients
};

#ifdef __CUDACC__
namespace dev {

__device__ __forceinline__ double rotary_position(const RotaryParams& p, int64_t token) {
  const int64_t b = p.batch == 1 ? 0 : token / p.tokens, l = token - b * p.tokens;
  const int64_t at = b * p.pos_stride_b + l * p.pos_stride_t;
  return p.positions64 ? double(static_cast<const int64_t*>(p.positions)[at])
                       : double(static_cast<const int32_t*>(p.positions)[at]);
}

// (cos, sin) * magnitude of pair f at a token.
__device__ __forceinline__ float2 rotary_angle(const RotaryParams& p, int64_t token, int f) {
  double turns = rotary_position(p, token) * p.inv_freq[f] * 0.15915494309189535;  // 1 / (2 pi)
  turns -= rint(turns);
  float s, c;
  sincospif(float(2.0 * turns), &s, &c);
  return make_float2(c * p.magnitude, s * p.magnitude * p.sign);
}

}  // namespace dev
#endif

void rotary_launch(RotaryType t, const RotaryParams& p, int sm_count, cudaStream_t stream);

}  // namespace mgfa
