// Rotary positions: each pair (a, b) of a head's first rotary_dim elements becomes
//   (a cos t - b sin t, a sin t + b cos t) * magnitude,   t = position * inv_freq[i],
// and the elements behind them are copied. The gradient is the rotation by -t.
//
// Bound by memory: every element is read and written once; 32768 tokens of 40 heads of
// 128 in bf16 take 117 us, 5.7 TB/s. The angle belongs to a
// (token, pair), not to a head, so a CTA computes its tokens' sines and cosines once
// in shared memory and all heads of q and k use them. t is formed in 64 bits as a
// fraction of a turn and reduced there: at position 10^6 a 32-bit angle would be off
// by 2^-24 * 10^6 = 0.06 radians. Sine and cosine of the reduced angle are 32-bit.
#include "rotary.cuh"

#include <algorithm>

#include "pairs.cuh"

namespace mgfa {
namespace {

using namespace mgfa::dev;

constexpr int kThreads = 256;

// How a head is cut into units of work, each a load and a store of 16 bytes, V elements:
enum : int {
  kHalves = 0,      // V elements of either half (two loads), V dividing rotary_dim / 2; then copies
  kNeighbours = 1,  // V elements with the pairs (2i, 2i + 1) inside
  kAny = 2,         // V elements; each one's partner is fetched by itself (from L1)
};

// Heads whose loads a thread has under way. At 32768 tokens of 32 + 8 heads of 128 in
// bf16 (671 MB moved) 2, 3 and 4 take 121, 120 and 117 us (halves) and 174, 149 and
// 121 us (neighbours). At 4 CTAs an SM a thread has 64 registers: 4 heads spill 176 bytes in
// the 16-bit halves and none in the neighbours, 8 more than they gain.
constexpr int kBatch = 4;

__host__ __device__ inline int units_of(int mode, int v, int head_dim, int rotary_dim) {
  return mode == kHalves ? rotary_dim / 2 / v + (head_dim - rotary_dim) / v : head_dim / v;
}

// CTA: `tile` tokens; of each, `slots` groups of `units` threads, each of which takes
// every slots-th head, at the same columns c0 (and c1) throughout. So a thread reads its
// columns' sines and cosines once from shared memory, and its first loads are under way
// while they are computed.
template <class E, int kMode>
__global__ void __launch_bounds__(kThreads, 4) rotary_kernel(const RotaryParams p, int tile, int slots) {
  constexpr int V = 16 / sizeof(E), kPairs = V / 2;
  using P = PairOf<E>;
  union Vec {
    uint4 v;
    typename P::Raw w[kPairs];
  };
  extern __shared__ float2 cs[];  // [tile][rotary_dim / 2]: (cos, sin) * magnitude
  const int half = p.rotary_dim >> 1;
  const int units = units_of(kMode, V, p.head_dim, p.rotary_dim);
  const int64_t first = int64_t(blockIdx.x) * tile, all = p.batch * p.tokens;
  const int here = int(all - first < tile ? all - first : tile);
  const int t = threadIdx.x / (units * slots);
  const int slot = threadIdx.x / units - t * slots, u = threadIdx.x - (t * slots + slot) * units;
  const bool rotates = kMode != kHalves || u < half / V;
  const int c0 = rotates ? u * V : p.rotary_dim + (u - half / V) * V;
  const int c1 = kMode == kHalves && rotates ? c0 + half : c0;
  const int heads = t < here ? p.x[0].heads + p.x[1].heads : 0;
  const int64_t token = first + t, b = p.batch == 1 ? 0 : token / p.tokens, l = token - b * p.tokens;
  const E* const in0 = static_cast<const E*>(p.x[0].in) + b * p.x[0].stride_b + l * p.x[0].stride_t;
  const E* const in1 = static_cast<const E*>(p.x[1].in) + b * p.x[1].stride_b + l * p.x[1].stride_t;
  E* const out0 = static_cast<E*>(p.x[0].out) + token * p.x[0].heads * p.head_dim;
  E* const out1 = static_cast<E*>(p.x[1].out) + token * p.x[1].heads * p.head_dim;

  Vec x0[kBatch], x1[kMode == kHalves ? kBatch : 1];
  uint64_t other[kMode == kAny ? kBatch : 1][kPairs];
  auto load = [&](int h0) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int h = h0 + i * slots, hk = h - p.x[0].heads;
      const E* in = hk < 0 ? in0 + h * p.x[0].stride_h : in1 + hk * p.x[1].stride_h;
      if (h < heads) {
        x0[i].v = __ldg(reinterpret_cast<const uint4*>(in + c0));
        if constexpr (kMode == kHalves) x1[i].v = __ldg(reinterpret_cast<const uint4*>(in + c1));
        if constexpr (kMode == kAny) {
#pragma unroll
          for (int k = 0; k < kPairs; ++k) {
            const int c = c0 + 2 * k;
            // rotary_dim is even, but half may be odd: the two elements' partners lie apart
            const int a = c >= p.rotary_dim ? c : c < half ? c + half : c - half;
            const int d = c >= p.rotary_dim ? c : c + 1 < half ? c + 1 + half : c + 1 - half;
            other[i][k] = f2_pack(to_f(in[a]), to_f(in[d]));
          }
        }
      }
    }
  };
  load(slot);

  for (int i = threadIdx.x; i < here * half; i += blockDim.x) {
    const int tt = i / half;
    cs[i] = rotary_angle(p, first + tt, i - tt * half);
  }
  __syncthreads();
  if (slot >= heads) return;
  // out = own * co + partner * si for this thread's columns
  uint64_t co[kPairs], si[kPairs];
#pragma unroll
  for (int k = 0; k < kPairs; ++k) {
    const int c = c0 + 2 * k;
    co[k] = si[k] = 0;
    if (c < p.rotary_dim) {
      const float2* w = cs + t * half;
      if (kMode == kNeighbours) {
        const float2 f = w[c >> 1];
        co[k] = f2_pack(f.x, f.x);
        si[k] = f2_pack(-f.y, f.y);
      } else {
        const float2 f = w[c < half ? c : c - half], g = w[c + 1 < half ? c + 1 : c + 1 - half];
        co[k] = f2_pack(f.x, g.x);
        si[k] = f2_pack(c < half ? -f.y : f.y, c + 1 < half ? -g.y : g.y);
      }
    }
  }
  for (int h0 = slot; h0 < heads; h0 += slots * kBatch) {
    if (h0 != slot) load(h0);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int h = h0 + i * slots, hk = h - p.x[0].heads;
      if (h >= heads) continue;
      E* out = hk < 0 ? out0 + h * p.head_dim : out1 + hk * p.head_dim;
#pragma unroll
      for (int k = 0; k < kPairs; ++k) {
        const uint64_t a = P::wide(x0[i].w[k]);
        if constexpr (kMode == kHalves) {
          const uint64_t d = P::wide(x1[i].w[k]);
          if (rotates) x0[i].w[k] = P::narrow(f2_fma(a, co[k], f2_mul(d, si[k])));
          x1[i].w[k] = P::narrow(f2_sub(f2_mul(d, co[k]), f2_mul(a, si[k])));
        } else {
          uint64_t d = other[kMode == kAny ? i : 0][k];
          if constexpr (kMode == kNeighbours) {
            float e0, e1;
            f2_unpack(a, e0, e1);
            d = f2_pack(e1, e0);
          }
          if (c0 + 2 * k < p.rotary_dim) x0[i].w[k] = P::narrow(f2_fma(a, co[k], f2_mul(d, si[k])));
        }
      }
      *reinterpret_cast<uint4*>(out + c0) = x0[i].v;
      if constexpr (kMode == kHalves)
        if (rotates) *reinterpret_cast<uint4*>(out + c1) = x1[i].v;
    }
  }
}

// Heads that start or end off a 16-byte boundary: one element a thread, its partner from L1.
template <class E>
__global__ void __launch_bounds__(kThreads) rotary_element_kernel(const RotaryParams p) {
  extern __shared__ float2 cs[];  // [rotary_dim / 2]
  const int half = p.rotary_dim >> 1;
  const int64_t token = blockIdx.x, b = token / p.tokens, l = token - b * p.tokens;
  for (int i = threadIdx.x; i < half; i += kThreads) cs[i] = rotary_angle(p, token, i);
  __syncthreads();
  for (int k = 0; k < 2; ++k) {
    const RotaryTensor& x = p.x[k];
    const E* in = static_cast<const E*>(x.in) + b * x.stride_b + l * x.stride_t;
    E* out = static_cast<E*>(x.out) + token * x.heads * p.head_dim;
    for (int i = threadIdx.x; i < x.heads * p.head_dim; i += kThreads) {
      const int h = i / p.head_dim, c = i - h * p.head_dim;
      const E* row = in + h * x.stride_h;
      E v = row[c];
      if (c < p.rotary_dim) {
        const bool second = p.interleaved ? c & 1 : c >= half;
        const float2 f = cs[p.interleaved ? c >> 1 : second ? c - half : c];
        const float d = to_f(row[p.interleaved ? c ^ 1 : second ? c - half : c + half]);
        v = from_f<E>(to_f(v) * f.x + d * (second ? f.y : -f.y));
      }
      out[i] = v;
    }
  }
}

template <class E, int kMode>
void launch_mode(const RotaryParams& p, int sm_count, cudaStream_t s) {
  constexpr int V = 16 / sizeof(E);
  const int heads = p.x[0].heads + p.x[1].heads;
  const int units = units_of(kMode, V, p.head_dim, p.rotary_dim);
  const int64_t all = p.batch * p.tokens;
  // A batch of heads a thread; then as many tokens as a CTA has threads for, but no fewer
  // CTAs than two for each SM.
  const int slots = std::max(1, std::min(kThreads / units, (heads + kBatch - 1) / kBatch));
  int64_t tile = kThreads / (units * slots);
  tile = std::max<int64_t>(1, std::min<int64_t>(tile, all / (2 * sm_count)));
  const unsigned grid = unsigned((all + tile - 1) / tile);
  const int threads = int(tile) * units * slots;
  rotary_kernel<E, kMode><<<grid, (threads + 31) / 32 * 32,
                            size_t(tile) * (p.rotary_dim / 2) * sizeof(float2), s>>>(p, int(tile), slots);
}

// The widest accesses that the pairs' layout and (p.vec) the strides allow.
template <class E>
void launch_e(const RotaryParams& p, int sm_count, cudaStream_t s) {
  constexpr int kV = 16 / sizeof(E);
  const int pairs = p.rotary_dim / 2;
  if (!p.vec) {
    rotary_element_kernel<E><<<unsigned(p.batch * p.tokens), kThreads, pairs * sizeof(float2), s>>>(p);
    return;
  }
  if (p.interleaved) return launch_mode<E, kNeighbours>(p, sm_count, s);
  if (pairs % kV == 0 && (p.head_dim - p.rotary_dim) % kV == 0)
    return launch_mode<E, kHalves>(p, sm_count, s);
  launch_mode<E, kAny>(p, sm_count, s);
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
