// Rotary positions: each pair (a, b) of a head's first rotary_dim elements becomes
//   (a cos t - b sin t, a sin t + b cos t) * magnitude,   t = position * inv_freq[i],
// and the elements behind them are copied. The gradient is the rotation by -t.
//
// Bound by memory: every element is read and written once. The angle belongs to a
// (token, pair), not to a head, so a CTA computes its tokens' sines and cosines once
// in shared memory and all heads of q and k use them. t is formed in 64 bits as a
// fraction of a turn and reduced there: at position 10^6 a 32-bit angle would be off
// by 2^-24 * 10^6 = 0.06 radians. Sine and cosine of the reduced angle are 32-bit.
#include "rotary.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

namespace mgfa {
namespace {

constexpr int kThreads = 256;

template <class E>
__device__ __forceinline__ float to_f(E v) { return float(v); }
template <>
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <class E>
__device__ __forceinline__ E from_f(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ float from_f(float v) { return v; }

template <class E, int V>
struct alignas(sizeof(E) * V) Pack {
  E e[V];
};

// A head is `units` units of work: V pairs each (V elements of either half, or
// 2V neighbours), then copies of V elements behind rotary_dim.
template <class E, int V, bool kInterleaved>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryParams p, int tile) {
  extern __shared__ float2 cs[];  // [tile][rotary_dim / 2]: (cos, sin) * magnitude
  const int pairs = p.rotary_dim >> 1;
  const int64_t all = p.batch * p.tokens;
  const int64_t first = int64_t(blockIdx.x) * tile;
  const int here = int(all - first < tile ? all - first : tile);
  for (int i = threadIdx.x; i < here * pairs; i += kThreads) {
    const int t = i / pairs, f = i - t * pairs;
    const int64_t b = (first + t) / p.tokens, l = (first + t) - b * p.tokens;
    const int64_t at = b * p.pos_stride_b + l * p.pos_stride_t;
    const double pos = p.positions64 ? double(static_cast<const int64_t*>(p.positions)[at])
                                     : double(static_cast<const int32_t*>(p.positions)[at]);
    double turns = pos * p.inv_freq[f] * 0.15915494309189535;  // 1 / (2 pi)
    turns -= rint(turns);
    float s, c;
    sincospif(float(2.0 * turns), &s, &c);
    cs[i] = make_float2(c * p.magnitude, s * p.magnitude * p.sign);
  }
  __syncthreads();
  const int rot_units = pairs / V, units = rot_units + (p.head_dim - p.rotary_dim) / V;
  const int heads = p.x[0].heads + p.x[1].heads;
  const int per_token = heads * units;
  const int total = here * per_token;
#pragma unroll 4
  for (int i = threadIdx.x; i < total; i += kThreads) {
    const int t = i / per_token, rest = i - t * per_token;
    int h = rest / units;
    const int u = rest - h * units;
    const int which = h >= p.x[0].heads;
    if (which) h -= p.x[0].heads;
    const RotaryTensor& x = p.x[which];
    const int64_t b = p.batch == 1 ? 0 : (first + t) / p.tokens, l = (first + t) - b * p.tokens;
    const E* in = static_cast<const E*>(x.in) + b * x.stride_b + l * x.stride_t + h * x.stride_h;
    E* out = static_cast<E*>(x.out) + ((first + t) * x.heads + h) * p.head_dim;
    if (u >= rot_units) {
      const int c = p.rotary_dim + (u - rot_units) * V;
      *reinterpret_cast<Pack<E, V>*>(out + c) = *reinterpret_cast<const Pack<E, V>*>(in + c);
      continue;
    }
    const int c0 = kInterleaved ? 2 * u * V : u * V, c1 = kInterleaved ? c0 + V : c0 + pairs;
    Pack<E, V> x0 = *reinterpret_cast<const Pack<E, V>*>(in + c0);
    Pack<E, V> x1 = *reinterpret_cast<const Pack<E, V>*>(in + c1);
    const float2* w = cs + t * pairs + u * V;
    float a[V], d[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      // pair j's elements: neighbours of the 2V, or element j of both halves
      a[j] = to_f(kInterleaved ? (2 * j < V ? x0.e[(2 * j) % V] : x1.e[(2 * j) % V]) : x0.e[j]);
      d[j] = to_f(kInterleaved ? (2 * j + 1 < V ? x0.e[(2 * j + 1) % V] : x1.e[(2 * j + 1) % V]) : x1.e[j]);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float2 k = w[j];
      const E ra = from_f<E>(a[j] * k.x - d[j] * k.y), rd = from_f<E>(a[j] * k.y + d[j] * k.x);
      if (kInterleaved) {
        (2 * j < V ? x0.e[(2 * j) % V] : x1.e[(2 * j) % V]) = ra;
        (2 * j + 1 < V ? x0.e[(2 * j + 1) % V] : x1.e[(2 * j + 1) % V]) = rd;
      } else {
        x0.e[j] = ra;
        x1.e[j] = rd;
      }
    }
    *reinterpret_cast<Pack<E, V>*>(out + c0) = x0;
    *reinterpret_cast<Pack<E, V>*>(out + c1) = x1;
  }
}

template <class E, int V>
void launch_v(const RotaryParams& p, int sm_count, cudaStream_t s) {
  const int pairs = p.rotary_dim / 2;
  const int64_t all = p.batch * p.tokens;
  const int per_token = (p.x[0].heads + p.x[1].heads) * (pairs / V + (p.head_dim - p.rotary_dim) / V);
  // Tokens a CTA: 4 units of work a thread and at most 32 KB of angles, but no fewer
  // CTAs than two for each SM.
  int64_t tile = std::max(1, 4 * kThreads / std::max(1, per_token));
  tile = std::min<int64_t>(tile, 32768 / (8 * std::max(1, pairs)));
  tile = std::max<int64_t>(1, std::min<int64_t>(tile, all / (2 * sm_count)));
  const unsigned grid = unsigned((all + tile - 1) / tile);
  const size_t smem = size_t(tile) * pairs * sizeof(float2);
  if (p.interleaved) rotary_kernel<E, V, true><<<grid, kThreads, smem, s>>>(p, int(tile));
  else rotary_kernel<E, V, false><<<grid, kThreads, smem, s>>>(p, int(tile));
}

template <class E>
void launch_e(const RotaryParams& p, int sm_count, cudaStream_t s) {
  if (p.vec) launch_v<E, 16 / sizeof(E)>(p, sm_count, s);
  else launch_v<E, 1>(p, sm_count, s);
}

}  // namespace

void rotary_launch(RotaryType t, const RotaryParams& p, int sm_count, cudaStream_t stream) {
  switch (t) {
    case RotaryType::kBf16: return launch_e<__nv_bfloat16>(p, sm_count, stream);
    case RotaryType::kF16: return launch_e<__half>(p, sm_count, stream);
    default: return launch_e<float>(p, sm_count, stream);
  }
}

}  // namespace mgfa
