// Root-mean-square norm with the residual's addition, its 8-bit output, and its
// gradients.
//
//   h = round(x + r)               the new residual stream (an output: x's type)
//   y = h * rstd * w               rstd = 1 / sqrt(mean(h^2) + eps)
//   y8 = e4m3(y / scale)           scale = max|y| / 448 over a row or `group` columns
//   dx = dr = dh + rstd (w dy - n mean(w dy n)),  n = h rstd;  dw = sum over rows of dy n
//
// h is rounded before the norm reads it, so that y, and the backward pass that has
// only the stored h, belong to the same stream. All sums are in fp32.
//
// Bound by memory: every tensor is read or written once. A row stays in the
// registers of the T threads that own it (N vectors of 16 bytes each, or single
// elements where a row is not 16-byte aligned), so the statistics and the output
// need one pass; T grows with the row so that a thread holds at most 8 vectors.
#include "rms_norm.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>

namespace mgfa {
namespace {

constexpr int kMaxThreads = 512;

template <class E>
__device__ __forceinline__ float to_f(E v);
template <>
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f(float v) { return v; }
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

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

struct Sum {
  static __device__ __forceinline__ float of(float a, float b) { return a + b; }
};
struct MaxNan {
  static __device__ __forceinline__ float of(float a, float b) { return max_nan(a, b); }
};

// Over the blockDim.x threads of one row (a multiple of 32); `buf` holds
// blockDim.y * 32 floats. Every thread gets the same value, added in the same order.
template <class Op>
__device__ __forceinline__ float row_reduce(float v, float* buf) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = Op::of(v, __shfl_xor_sync(0xffffffffu, v, o));
  if (blockDim.x == 32) return v;
  const int warps = blockDim.x >> 5;
  float* row = buf + threadIdx.y * 32;
  __syncthreads();  // the previous reduction's readers are done
  if ((threadIdx.x & 31) == 0) row[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = row[0];
  for (int i = 1; i < warps; ++i) t = Op::of(t, row[i]);
  return t;
}

template <class E, int V, int N>
__device__ __forceinline__ void load_w(const void* w, int weight_f32, int dim, float (&f)[N][V]) {
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = (j * blockDim.x + threadIdx.x) * V;
    if (c < dim) {
      if (weight_f32) {
#pragma unroll
        for (int i = 0; i < V; ++i) f[j][i] = __ldg(static_cast<const float*>(w) + c + i);
      } else {
        const Pack<E, V> p = *reinterpret_cast<const Pack<E, V>*>(static_cast<const E*>(w) + c);
#pragma unroll
        for (int i = 0; i < V; ++i) f[j][i] = to_f(p.e[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) f[j][i] = 0.f;
    }
  }
}

// V elements per vector, N vectors per thread; block (T, R): R rows of T threads.
template <class E, int V, int N, bool kRes, bool k8>
__global__ void __launch_bounds__(kMaxThreads) rms_norm_fwd_kernel(const NormFwdParams p) {
  __shared__ float buf[8 * 32];
  const int64_t row = int64_t(blockIdx.x) * blockDim.y + threadIdx.y;
  const bool live = row < p.rows;  // rows past the end take part in the barriers only
  const E* x = static_cast<const E*>(p.x) + (live ? row : 0) * p.x_stride;
  const E* r = kRes ? static_cast<const E*>(p.residual) + (live ? row : 0) * p.r_stride : nullptr;
  Pack<E, V> h[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = (j * blockDim.x + threadIdx.x) * V;
    if (c < p.dim) h[j] = *reinterpret_cast<const Pack<E, V>*>(x + c);
  }
  if constexpr (kRes) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = (j * blockDim.x + threadIdx.x) * V;
      if (c < p.dim) {
        const Pack<E, V> q = *reinterpret_cast<const Pack<E, V>*>(r + c);
#pragma unroll
        for (int i = 0; i < V; ++i) h[j].e[i] = from_f<E>(to_f(h[j].e[i]) + to_f(q.e[i]));
      }
    }
  }
  float w[N][V];
  load_w<E, V, N>(p.weight, p.weight_f32, p.dim, w);
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = (j * blockDim.x + threadIdx.x) * V;
    if (c < p.dim) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float f = to_f(h[j].e[i]);
        sum = fmaf(f, f, sum);
      }
      if (kRes && live)
        *reinterpret_cast<Pack<E, V>*>(static_cast<E*>(p.h) + row * p.dim + c) = h[j];
    }
  }
  sum = row_reduce<Sum>(sum, buf);
  const float rstd = 1.f / sqrtf(sum / float(p.dim) + p.eps);
  if (p.rstd && live && threadIdx.x == 0) p.rstd[row] = rstd;
  if constexpr (!k8) {
    if (!live) return;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = (j * blockDim.x + threadIdx.x) * V;
      if (c < p.dim) {
        Pack<E, V> o;
#pragma unroll
        for (int i = 0; i < V; ++i) o.e[i] = from_f<E>(to_f(h[j].e[i]) * rstd * w[j][i]);
        *reinterpret_cast<Pack<E, V>*>(static_cast<E*>(p.y) + row * p.dim + c) = o;
      }
    }
  } else {
    float top[N], row_top = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = (j * blockDim.x + threadIdx.x) * V;
      top[j] = 0.f;
      if (c < p.dim) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          w[j][i] *= to_f(h[j].e[i]) * rstd;  // from here on the output
          top[j] = max_nan(top[j], fabsf(w[j][i]));
        }
      }
      row_top = max_nan(row_top, top[j]);
    }
    // A group is a power of two of columns, V * (at most 32) aligned lanes of a warp.
    if (p.group == 0) {
      row_top = row_reduce<MaxNan>(row_top, buf);
#pragma unroll
      for (int j = 0; j < N; ++j) top[j] = row_top;
    } else {
      const int lanes = p.group / V;
#pragma unroll
      for (int j = 0; j < N; ++j)
        for (int o = lanes >> 1; o > 0; o >>= 1)
          top[j] = max_nan(top[j], __shfl_xor_sync(0xffffffffu, top[j], o));
    }
    if (!live) return;
    const int groups = p.group ? p.dim / p.group : 1;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = (j * blockDim.x + threadIdx.x) * V;
      if (c >= p.dim) continue;
      float scale = top[j] / 448.f;      // 448: the largest e4m3 value
      if (!(scale > 0.f)) scale = 1.f;   // nothing but zeros, or a NaN
      if (p.group ? c % p.group == 0 : c == 0)
        p.scale[row * groups + (p.group ? c / p.group : 0)] = scale;
      Pack<uint8_t, V> o;
#pragma unroll
      for (int i = 0; i < V; ++i)
        o.e[i] = __nv_cvt_float_to_fp8(w[j][i] / scale, __NV_SATFINITE, __NV_E4M3);
      *reinterpret_cast<Pack<uint8_t, V>*>(static_cast<uint8_t*>(p.y) + row * p.dim + c) = o;
    }
  }
}

// Each CTA takes every gridDim.x-th set of R rows and keeps its columns' part of dw
// in registers. While a row is reduced, the next one's loads are under way (N <= 2;
// wider rows have the loads of 4 vectors and more a tensor in flight as it is, and
// no registers to hold two rows). The parts are added by norm_dw_kernel, in the CTAs'
// order, so dw does not depend on timing.
template <class E, int V, int N>
__global__ void __launch_bounds__(kMaxThreads) rms_norm_bwd_kernel(const NormBwdParams p) {
  constexpr bool kAhead = N * V * sizeof(E) <= 32;
  extern __shared__ float sh[];  // row_reduce: blockDim.y * 32; then dw: blockDim.y * dim
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int64_t step = int64_t(gridDim.x) * blockDim.y;
  float w[N][V], dw[N][V];
  if constexpr (kAhead) load_w<E, V, N>(p.weight, p.weight_f32, p.dim, w);
#pragma unroll
  for (int j = 0; j < N; ++j)
#pragma unroll
    for (int i = 0; i < V; ++i) dw[j][i] = 0.f;
  Pack<E, V> h[N], dy[N], dh[N];
  float rstd = 0.f;
  auto load = [&](int64_t row) {
    const bool live = row < p.rows;
    const int64_t at = live ? row : 0;
    rstd = live ? __ldg(p.rstd + at) : 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = (j * blockDim.x + threadIdx.x) * V;
#pragma unroll
      for (int i = 0; i < V; ++i) h[j].e[i] = dy[j].e[i] = dh[j].e[i] = from_f<E>(0.f);
      if (live && c < p.dim) {
        if (p.dy) {
          h[j] = *reinterpret_cast<const Pack<E, V>*>(static_cast<const E*>(p.h) + at * p.h_stride + c);
          dy[j] = *reinterpret_cast<const Pack<E, V>*>(static_cast<const E*>(p.dy) + at * p.dy_stride + c);
        }
        if (p.dh)
          dh[j] = *reinterpret_cast<const Pack<E, V>*>(static_cast<const E*>(p.dh) + at * p.dh_stride + c);
      }
    }
  };
  // A CTA's first row exists, so every thread of the CTA makes the same number of steps.
  const int64_t first = int64_t(blockIdx.x) * blockDim.y;
  if (kAhead && first < p.rows) load(first + threadIdx.y);
  for (int64_t base = first; base < p.rows; base += step) {
    const int64_t row = base + threadIdx.y;
    if constexpr (!kAhead) {
      load(row);
      load_w<E, V, N>(p.weight, p.weight_f32, p.dim, w);
    }
    Pack<E, V> h1[N], dy1[N], dh1[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      h1[j] = h[j];
      dy1[j] = dy[j];
      dh1[j] = dh[j];
    }
    const float rs = rstd;
    if (kAhead && base + step < p.rows) load(row + step);
    float dot = 0.f;  // sum of w dy n
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float dn = to_f(dy1[j].e[i]) * (to_f(h1[j].e[i]) * rs);
        dw[j][i] += dn;
        dot = fmaf(dn, w[j][i], dot);
      }
    dot = row_reduce<Sum>(dot, sh) / float(p.dim);
    if (row < p.rows) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int c = (j * blockDim.x + threadIdx.x) * V;
        if (c < p.dim) {
          Pack<E, V> o;
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float g = to_f(dy1[j].e[i]) * w[j][i] - to_f(h1[j].e[i]) * rs * dot;
            o.e[i] = from_f<E>(fmaf(rs, g, to_f(dh1[j].e[i])));
          }
          *reinterpret_cast<Pack<E, V>*>(static_cast<E*>(p.dx) + row * p.dim + c) = o;
        }
      }
    }
  }
  if (!p.dw_part) return;
  float* part = p.dw_part + int64_t(blockIdx.x) * p.dim;
  if (blockDim.y == 1) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = (j * blockDim.x + threadIdx.x) * V;
      if (c < p.dim)
#pragma unroll
        for (int i = 0; i < V; ++i) part[c + i] = dw[j][i];
    }
    return;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = (j * blockDim.x + threadIdx.x) * V;
    if (c < p.dim)
#pragma unroll
      for (int i = 0; i < V; ++i) sh[threadIdx.y * p.dim + c + i] = dw[j][i];
  }
  __syncthreads();
  for (int c = threadIdx.y * blockDim.x + threadIdx.x; c < p.dim; c += blockDim.x * blockDim.y) {
    float t = 0.f;
    for (int y = 0; y < blockDim.y; ++y) t += sh[y * p.dim + c];
    part[c] = t;
  }
}

// dw[c] = sum of the parts, 32 columns a CTA: warp w adds parts w, w + 32, ..., then
// the 32 warps' sums are added in order.
template <class E>
__global__ void __launch_bounds__(1024) norm_dw_kernel(const float* part, int parts, int dim, E* dw) {
  __shared__ float sh[32][33];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float t = 0.f;
  if (c < dim)
    for (int i = warp; i < parts; i += 32) t += part[int64_t(i) * dim + c];
  sh[warp][lane] = t;
  __syncthreads();
  if (warp == 0 && c < dim) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) s += sh[i][lane];
    dw[c] = from_f<E>(s);
  }
}

struct Shape {
  int n;      // vectors per thread
  dim3 block;
};

// T threads (a multiple of 32) per row with n vectors each, and rows packed until a
// block has 256 threads. dim <= 16384, so n <= 4 (16-bit vectors), 8 (fp32 vectors) or
// 32 (single elements).
Shape shape_of(int dim, int v) {
  const int vecs = (dim + v - 1) / v;
  int n = vecs > 256 ? 2 : 1;
  while (vecs > n * kMaxThreads) n *= 2;
  const int t = ((vecs + n - 1) / n + 31) / 32 * 32;
  return {n, dim3(t, std::max(1, std::min(8, 256 / t)))};
}

template <class E, int V, int N>
void fwd_n(const NormFwdParams& p, dim3 block, cudaStream_t s) {
  const dim3 grid(unsigned((p.rows + block.y - 1) / block.y));
  if (p.scale) {
    if (p.residual) rms_norm_fwd_kernel<E, V, N, true, true><<<grid, block, 0, s>>>(p);
    else rms_norm_fwd_kernel<E, V, N, false, true><<<grid, block, 0, s>>>(p);
  } else {
    if (p.residual) rms_norm_fwd_kernel<E, V, N, true, false><<<grid, block, 0, s>>>(p);
    else rms_norm_fwd_kernel<E, V, N, false, false><<<grid, block, 0, s>>>(p);
  }
}

template <class E>
void fwd_e(const NormFwdParams& p, cudaStream_t s) {
  constexpr int kV = 16 / sizeof(E);
  const Shape sh = shape_of(p.dim, p.vec ? kV : 1);
  if (p.vec) {
    switch (sh.n) {
      case 1: return fwd_n<E, kV, 1>(p, sh.block, s);
      case 2: return fwd_n<E, kV, 2>(p, sh.block, s);
      case 4: return fwd_n<E, kV, 4>(p, sh.block, s);
      default:
        if constexpr (sizeof(E) == 4) fwd_n<E, kV, 8>(p, sh.block, s);
        return;
    }
  }
  switch (sh.n) {
    case 1: case 2: return fwd_n<E, 1, 2>(p, sh.block, s);
    case 4: case 8: return fwd_n<E, 1, 8>(p, sh.block, s);
    default: return fwd_n<E, 1, 32>(p, sh.block, s);
  }
}

template <class E, int V, int N>
void bwd_n(const NormBwdParams& p, dim3 block, int parts, cudaStream_t s) {
  size_t smem = block.y * 32 * sizeof(float);
  if (block.y > 1) smem = std::max(smem, size_t(block.y) * p.dim * sizeof(float));
  rms_norm_bwd_kernel<E, V, N><<<parts, block, smem, s>>>(p);
}

template <class E>
void bwd_e(const NormBwdParams& p, int parts, cudaStream_t s) {
  constexpr int kV = 16 / sizeof(E);
  const Shape sh = shape_of(p.dim, p.vec ? kV : 1);
  if (p.vec) {
    switch (sh.n) {
      case 1: bwd_n<E, kV, 1>(p, sh.block, parts, s); break;
      case 2: bwd_n<E, kV, 2>(p, sh.block, parts, s); break;
      case 4: bwd_n<E, kV, 4>(p, sh.block, parts, s); break;
      default:
        if constexpr (sizeof(E) == 4) bwd_n<E, kV, 8>(p, sh.block, parts, s);
    }
  } else {
    switch (sh.n) {
      case 1: case 2: bwd_n<E, 1, 2>(p, sh.block, parts, s); break;
      case 4: case 8: bwd_n<E, 1, 8>(p, sh.block, parts, s); break;
      default: bwd_n<E, 1, 32>(p, sh.block, parts, s);
    }
  }
  if (!p.dw_part) return;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((p.dim + 31) / 32);
  cfg.blockDim = dim3(1024);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const float* part = p.dw_part;
  if (p.weight_f32) cudaLaunchKernelEx(&cfg, norm_dw_kernel<float>, part, parts, p.dim, static_cast<float*>(p.dw));
  else cudaLaunchKernelEx(&cfg, norm_dw_kernel<E>, part, parts, p.dim, static_cast<E*>(p.dw));
}

int vec_of(NormType t, int vec) { return vec ? (t == NormType::kF32 ? 4 : 8) : 1; }

}  // namespace

void rms_norm_fwd_launch(NormType t, const NormFwdParams& p, cudaStream_t stream) {
  switch (t) {
    case NormType::kBf16: return fwd_e<__nv_bfloat16>(p, stream);
    case NormType::kF16: return fwd_e<__half>(p, stream);
    default: return fwd_e<float>(p, stream);
  }
}

int rms_norm_bwd_parts(NormType t, int64_t rows, int dim, int vec, int sm_count) {
  const Shape sh = shape_of(dim, vec_of(t, vec));
  const int threads = int(sh.block.x * sh.block.y);
  const int64_t sets = (rows + sh.block.y - 1) / sh.block.y;
  return int(std::min<int64_t>(sets, int64_t(sm_count) * std::max(1, 768 / threads)));
}

void rms_norm_bwd_launch(NormType t, const NormBwdParams& p, int parts, cudaStream_t stream) {
  switch (t) {
    case NormType::kBf16: return bwd_e<__nv_bfloat16>(p, parts, stream);
    case NormType::kF16: return bwd_e<__half>(p, parts, stream);
    default: return bwd_e<float>(p, parts, stream);
  }
}

}  // namespace mgfa
