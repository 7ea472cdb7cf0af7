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
// Bound by memory: every tensor is read or written once. At 16384 x 4096 bf16 with a
// residual the forward takes 84 us (6.4 TB/s) and the backward 111 us (4.8 TB/s, with
// 9 us for dw's parts); without the packed pairs and with the weights in registers they
// took 120 and 210 us. A row stays with the T threads that own it (N vectors each), so the
// statistics and the output need one pass. A vector is 16 bytes, also where the width is no
// multiple of that (kShifted: 16384 x 4095 takes 150 + 241 us, half the aligned rate; by
// single elements 255 + 374), and one element for other strides. T grows with the row, which
// leaves a thread 8 to 16 elements up to a width of 4096, and 32 beyond: there the backward's
// three tensors do not fit 128 registers (392 bytes of spills in 16 bits, 608 in fp32), and
// 8192 x 8192 takes 90 us forward and 123 us back in bf16, 160 and 222 us in fp32, against
// 82 and 164 us of each at the copy's rate. The 8-bit output of 16384 x 4096 takes 111 us
// with a scale a row and 129 us with one for each 128 columns (72 us for its bytes): the
// division of every value by its scale comes on top.
#include "rms_norm.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <type_traits>

#include "pairs.cuh"

namespace mgfa {
namespace {

using namespace mgfa::dev;

// Threads of a block whose threads hold `elements` (shape_of).
constexpr int max_threads(int elements) { return elements <= 16 ? 256 : 512; }

// How a thread's share of a row lies in memory.
enum : int {
  kAligned = 0,  // rows start on 16-byte boundaries and dim is a multiple of a vector
  kShifted = 1,  // row r starts r * dim elements behind one: the vectors are the aligned ones
                 // that cover the row, and its first and last are taken by elements; for
                 // widths from a vector less one element on, so that the vectors end inside
                 // the next row
  kSingle = 2,   // single elements, for any strides
};

// A thread's share of a row: N vectors of V elements, vector j at column
// (j * blockDim.x + threadIdx.x) * V - shift. N * V is even; columns outside the row are
// zero.
template <class E, int V, int N, int kLay>
struct Share {
  using P = PairOf<E>;
  using Raw = typename P::Raw;
  using Vec = typename Bytes<V * sizeof(E)>::T;
  static constexpr int kPairs = N * V / 2;
  union {
    Raw raw[kPairs];
    Vec vec[N];
  };
  static __device__ __forceinline__ int shift(int64_t row, int dim) {
    return kLay == kShifted ? int(uint32_t(row) * uint32_t(dim) % V) : 0;
  }
  static __device__ __forceinline__ int col(int j, int shift) {
    return (j * int(blockDim.x) + int(threadIdx.x)) * V - shift;
  }
  static __device__ __forceinline__ bool whole(int c, int dim) {
    return kLay == kShifted ? c >= 0 && c + V <= dim : c < dim;
  }
  // `last`: no row follows. Elsewhere a shifted row's first and last vector reach into its
  // neighbours, whose elements are cut.
  __device__ __forceinline__ void load(const void* row_at, int dim, int shift, bool live, bool last) {
    const E* row = static_cast<const E*>(row_at);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = col(j, shift);
      Vec v = {};
      if (live && c < dim && (kLay != kShifted || !last || c + V <= dim))
        v = __ldg(reinterpret_cast<const Vec*>(row + c));
      vec[j] = v;
    }
    if constexpr (kLay == kShifted) {
      constexpr int kBits = 8 * sizeof(E);
      constexpr Raw kOne = (Raw(1) << kBits) - 1;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int c = col(j, shift);
        if (!live || c >= dim || whole(c, dim)) continue;
        if (last && c + V > dim) {
          float e[V];
#pragma unroll
          for (int i = 0; i < V; ++i) e[i] = c + i >= 0 && c + i < dim ? to_f(row[c + i]) : 0.f;
#pragma unroll
          for (int i = 0; i < V / 2; ++i) raw[j * V / 2 + i] = P::narrow(f2_pack(e[2 * i], e[2 * i + 1]));
        } else {
#pragma unroll
          for (int i = 0; i < V / 2; ++i) {
            const uint32_t a = uint32_t(c + 2 * i);
            raw[j * V / 2 + i] &= (a < uint32_t(dim) ? kOne : Raw(0)) |
                                  (a + 1 < uint32_t(dim) ? kOne << kBits : Raw(0));
          }
        }
      }
    }
  }
  __device__ __forceinline__ void store(void* row_at, int dim, int shift) const {
    E* row = static_cast<E*>(row_at);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = col(j, shift);
      if (whole(c, dim)) *reinterpret_cast<Vec*>(row + c) = vec[j];
      if constexpr (kLay == kShifted) {
        if (c < dim && !whole(c, dim)) {
#pragma unroll
          for (int i = 0; i < V / 2; ++i) {
            float e[2];
            f2_unpack(at(j * V / 2 + i), e[0], e[1]);  // exact: they are E's already
#pragma unroll
            for (int k = 0; k < 2; ++k)
              if (c + 2 * i + k >= 0 && c + 2 * i + k < dim) row[c + 2 * i + k] = from_f<E>(e[k]);
          }
        }
      }
    }
  }
  __device__ __forceinline__ uint64_t at(int k) const { return P::wide(raw[k]); }
  __device__ __forceinline__ void put(int k, uint64_t v) { raw[k] = P::narrow(v); }
  // Says that the pairs may have changed, so that the compiler widens them again instead
  // of keeping both forms in registers.
  __device__ __forceinline__ void renew() {
#pragma unroll
    for (int k = 0; k < kPairs; ++k) {
      if constexpr (sizeof(Raw) == 4) asm volatile("" : "+r"(raw[k]));
      else asm volatile("" : "+l"(raw[k]));
    }
  }
};

// The weights of a thread's columns as fp32 pairs, from E or fp32.
template <class E, int V, int N, int kLay>
__device__ __forceinline__ void load_w(const void* w, int weight_f32, int dim, int shift,
                                       uint64_t (&f)[N * V / 2]) {
  using S = Share<E, V, N, kLay>;
  if (kLay != kShifted && !weight_f32) {
    S s;
    s.load(w, dim, 0, true, true);
#pragma unroll
    for (int k = 0; k < N * V / 2; ++k) f[k] = s.at(k);
  } else {
    float e[N * V];
#pragma unroll
    for (int i = 0; i < N * V; ++i) {
      const int c = S::col(i / V, shift) + i % V;
      e[i] = c < 0 || c >= dim ? 0.f
             : weight_f32     ? __ldg(static_cast<const float*>(w) + c)
                              : to_f(static_cast<const E*>(w)[c]);
    }
#pragma unroll
    for (int k = 0; k < N * V / 2; ++k) f[k] = f2_pack(e[2 * k], e[2 * k + 1]);
  }
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float f2_sum(uint64_t v) {
  float a, b;
  f2_unpack(v, a, b);
  return a + b;
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
  // at most 16 warps, in an order that is every thread's
  const int lane = threadIdx.x & 31;
  v = lane < warps ? row[lane] : 0.f;
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = Op::of(v, __shfl_xor_sync(0xffffffffu, v, o));
  return __shfl_sync(0xffffffffu, v, 0);
}

// The rows that a CTA of block (T, R) takes, R at a time (T threads a row): every
// gridDim.x-th set. kShifted: those whose columns are the same threads', rows V * k apart;
// gridDim.x is a multiple of V.
template <int V, int kLay>
struct Rows {
  static constexpr int kApart = kLay == kShifted ? V : 1;
  int64_t lead, step;  // the first row, and from set to set
  __device__ __forceinline__ Rows()
      : lead(int64_t(blockIdx.x / kApart) * blockDim.y * kApart + blockIdx.x % kApart),
        step(int64_t(gridDim.x) * blockDim.y) {}
  static __device__ __forceinline__ int64_t mine(int64_t base) { return base + threadIdx.y * kApart; }
};

// The thread's weights in E, held in registers where no vector load reaches them.
template <class E, int V, int N, int kLay>
struct Weights {
  Share<E, V, N, kLay> held;
  const void* w;
  int weight_f32, dim, shift;
  __device__ __forceinline__ Weights(const void* weight, int f32, int d, int s)
      : w(weight), weight_f32(f32), dim(d), shift(s) {
    if constexpr (kLay == kShifted) {
      if (sizeof(E) == 4 || !f32) {
        uint64_t f[N * V / 2];
        load_w<E, V, N, kLay>(w, f32, dim, shift, f);
#pragma unroll
        for (int k = 0; k < N * V / 2; ++k) held.put(k, f[k]);
      }
    }
  }
  __device__ __forceinline__ void get(uint64_t (&f)[N * V / 2]) {
    if (kLay == kShifted && (sizeof(E) == 4 || !weight_f32)) {
      held.renew();
#pragma unroll
      for (int k = 0; k < N * V / 2; ++k) f[k] = held.at(k);
    } else {
      asm volatile("" : "+l"(w));  // read them again
      load_w<E, V, N, kLay>(w, weight_f32, dim, shift, f);
    }
  }
};

template <class E, int V, int N, int kLay, bool kRes, bool k8>
__global__ void __launch_bounds__(max_threads(N * V)) rms_norm_fwd_kernel(const NormFwdParams p) {
  using S = Share<E, V, N, kLay>;
  __shared__ float buf[8 * 32];
  constexpr int kPairs = N * V / 2;
  const Rows<V, kLay> rows;
  const int shift = S::shift(rows.mine(rows.lead), p.dim);
  Weights<E, V, N, kLay> weights(p.weight, p.weight_f32, p.dim, shift);
  for (int64_t base = rows.lead; base < p.rows; base += rows.step) {
    const int64_t row = rows.mine(base);
    const bool live = row < p.rows;  // rows past the end take part in the barriers only
    S h;
    h.load(static_cast<const E*>(p.x) + row * p.x_stride, p.dim, shift, live, row + 1 >= p.rows);
    if constexpr (kRes) {
      S r;
      r.load(static_cast<const E*>(p.residual) + row * p.r_stride, p.dim, shift, live, row + 1 >= p.rows);
#pragma unroll
      for (int k = 0; k < kPairs; ++k) h.put(k, f2_add(h.at(k), r.at(k)));
      if (live) h.store(static_cast<E*>(p.h) + row * p.dim, p.dim, shift);
    }
    uint64_t w[kPairs];
    weights.get(w);
    uint64_t acc[2] = {f2_pack(0.f, 0.f), f2_pack(0.f, 0.f)};
#pragma unroll
    for (int k = 0; k < kPairs; ++k) acc[k & 1] = f2_fma(h.at(k), h.at(k), acc[k & 1]);
    const float sum = row_reduce<Sum>(f2_sum(f2_add(acc[0], acc[1])), buf);
    const float rstd = 1.f / sqrtf(sum / float(p.dim) + p.eps);
    const uint64_t rstd2 = f2_pack(rstd, rstd);
    if (p.rstd && live && threadIdx.x == 0) p.rstd[row] = rstd;
#pragma unroll
    for (int k = 0; k < kPairs; ++k) w[k] = f2_mul(f2_mul(h.at(k), rstd2), w[k]);  // the output
    if constexpr (!k8) {
#pragma unroll
      for (int k = 0; k < kPairs; ++k) h.put(k, w[k]);
      if (live) h.store(static_cast<E*>(p.y) + row * p.dim, p.dim, shift);
    } else {
      float y[N * V];
#pragma unroll
      for (int k = 0; k < kPairs; ++k) f2_unpack(w[k], y[2 * k], y[2 * k + 1]);
      float top[N], row_top = 0.f;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        top[j] = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i)  // a NaN statistic makes 0 * NaN of columns outside the row
          if (S::col(j, shift) + i >= 0 && S::col(j, shift) + i < p.dim)
            top[j] = max_nan(top[j], fabsf(y[j * V + i]));
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
      const int groups = p.group ? p.dim / p.group : 1;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int c = S::col(j, shift);
        if (!live || c >= p.dim) continue;
        float scale = top[j] / 448.f;      // 448: the largest e4m3 value
        if (!(scale > 0.f)) scale = 1.f;   // nothing but zeros, or a NaN
        if (p.group ? c % p.group == 0 : c <= 0)
          p.scale[row * groups + (p.group ? c / p.group : 0)] = scale;
        uint8_t* dst = static_cast<uint8_t*>(p.y) + row * p.dim + c;
        if (V == 1 || !S::whole(c, p.dim)) {
#pragma unroll
          for (int i = 0; i < V; ++i)
            if (c + i >= 0 && c + i < p.dim)
              dst[i] = __nv_cvt_float_to_fp8(y[j * V + i] / scale, __NV_SATFINITE, __NV_E4M3);
        } else if constexpr (V > 1) {
          uint16_t o[V / 2];
#pragma unroll
          for (int i = 0; i < V / 2; ++i)
            o[i] = __nv_cvt_float2_to_fp8x2(make_float2(y[j * V + 2 * i] / scale, y[j * V + 2 * i + 1] / scale),
                                            __NV_SATFINITE, __NV_E4M3);
          *reinterpret_cast<typename Bytes<V>::T*>(dst) = *reinterpret_cast<typename Bytes<V>::T*>(o);
        }
      }
    }
  }
}

// A CTA keeps its columns' part of dw in registers over all its rows; several CTAs of an
// SM cover one another's reductions. Aligned weights are read again for every row (they
// stay in L1) to leave the registers to the rows. The parts are added by norm_dw_kernel,
// in the CTAs' order, so dw does not depend on timing.
template <class E, int V, int N, int kLay>
__global__ void __launch_bounds__(max_threads(N * V), N * V > 16 ? 1 : sizeof(E) == 4 ? 2 : 3)
    rms_norm_bwd_kernel(const NormBwdParams p) {
  using S = Share<E, V, N, kLay>;
  constexpr int kPairs = N * V / 2;
  extern __shared__ float sh[];  // row_reduce: blockDim.y * 32; then dw: blockDim.y * dim
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  uint64_t dw[kPairs];
#pragma unroll
  for (int k = 0; k < kPairs; ++k) dw[k] = f2_pack(0.f, 0.f);
  const float inv_dim = 1.f / float(p.dim);
  const Rows<V, kLay> rows;
  const int shift = S::shift(rows.mine(rows.lead), p.dim);
  Weights<E, V, N, kLay> weights(p.weight, p.weight_f32, p.dim, shift);
  for (int64_t base = rows.lead; base < p.rows; base += rows.step) {
    const int64_t row = rows.mine(base);
    const bool live = row < p.rows;
    const bool last = row + 1 >= p.rows;
    S h, dy, dh;
    h.load(static_cast<const E*>(p.h) + row * p.h_stride, p.dim, shift, live && p.dy, last);
    dy.load(static_cast<const E*>(p.dy) + row * p.dy_stride, p.dim, shift, live && p.dy, last);
    dh.load(static_cast<const E*>(p.dh) + row * p.dh_stride, p.dim, shift, live && p.dh, last);
    const float rstd = live ? __ldg(p.rstd + row) : 0.f;
    const uint64_t rstd2 = f2_pack(rstd, rstd);
    uint64_t acc = f2_pack(0.f, 0.f);  // sum of w dy n
    {
      uint64_t w[kPairs];
      weights.get(w);
#pragma unroll
      for (int k = 0; k < kPairs; ++k) {
        const uint64_t t = f2_mul(dy.at(k), f2_mul(h.at(k), rstd2));
        dw[k] = f2_add(dw[k], t);
        acc = f2_fma(t, w[k], acc);
      }
    }
    const float dot = row_reduce<Sum>(f2_sum(acc), sh) * inv_dim;  // mean of w dy n
    const float c = -dot * rstd;                                    // dx = rstd (w dy + c h) + dh
    const uint64_t c2 = f2_pack(c, c);
    h.renew();
    dy.renew();
    {
      uint64_t w[kPairs];
      weights.get(w);
#pragma unroll
      for (int k = 0; k < kPairs; ++k)
        dh.put(k, f2_fma(rstd2, f2_fma(dy.at(k), w[k], f2_mul(c2, h.at(k))), dh.at(k)));
    }
    if (live) dh.store(static_cast<E*>(p.dx) + row * p.dim, p.dim, shift);
  }
  if (!p.dw_part) return;
  float* part = p.dw_part + int64_t(blockIdx.x) * p.dim;
  float* to = blockDim.y == 1 ? part : sh + threadIdx.y * p.dim;
  if (blockDim.y > 1) __syncthreads();
#pragma unroll
  for (int k = 0; k < kPairs; ++k) {
    float e[2];
    f2_unpack(dw[k], e[0], e[1]);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int at = 2 * k + i, col = S::col(at / V, shift) + at % V;
      if (col >= 0 && col < p.dim) to[col] = e[i];
    }
  }
  if (blockDim.y == 1) return;
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
  int n;      // vectors of a thread
  dim3 block;
};

// Elements of a thread, then T threads (a multiple of 32) for a row, and rows packed
// until a block has 256 threads. At 16384 x 4096 and 32768 x 2048 bf16, 16 elements take
// 84 and 84 us forward and 107 and 108 us back; 32 take 83 us and 131 us at 4096, and 8
// take 91 us and 126 us at 2048.
Shape shape_of(int dim, int v, int lay) {
  const int covered = lay == kShifted ? dim + v - 1 : dim;
  int e = covered <= 512 ? 8 : covered <= 4096 ? 16 : 32;
  if (e < v) e = v;
  const int t = ((covered + e - 1) / e + 31) / 32 * 32;
  return {e / v, dim3(t, std::max(1, std::min(8, 256 / t)))};
}

template <class E>
int vec_elements(int lay) { return lay == kSingle ? 1 : 16 / int(sizeof(E)); }

// f(vector's elements, number, layout) as compile-time constants, for what shape_of gives.
template <class E, class F>
void with_shape(int lay, int n, F f) {
  auto pick = [&](auto vc, auto lc) {
    constexpr int V = decltype(vc)::value;
    switch (n * V) {
      case 8: return f(vc, std::integral_constant<int, 8 / V>(), lc);
      case 16: return f(vc, std::integral_constant<int, 16 / V>(), lc);
      default: return f(vc, std::integral_constant<int, 32 / V>(), lc);
    }
  };
  using Full = std::integral_constant<int, 16 / sizeof(E)>;
  if (lay == kAligned) pick(Full(), std::integral_constant<int, kAligned>());
  else if (lay == kShifted) pick(Full(), std::integral_constant<int, kShifted>());
  else pick(std::integral_constant<int, 1>(), std::integral_constant<int, kSingle>());
}

// CTAs for all rows, `most` a SM at a time; kShifted: a multiple of the vectors' elements.
int64_t ctas_of(const Shape& sh, int layout, int v, int64_t rows, int64_t most) {
  const int64_t sets = (rows + sh.block.y - 1) / sh.block.y, apart = layout == kShifted ? v : 1;
  // no more than run at once: a CTA left over would take as long again
  return std::min((sets + apart - 1) / apart, std::max<int64_t>(1, most / apart)) * apart;
}

template <class E>
void fwd_e(const NormFwdParams& p, int sm_count, cudaStream_t s) {
  const int v = vec_elements<E>(p.layout);
  const Shape sh = shape_of(p.dim, v, p.layout);
  with_shape<E>(p.layout, sh.n, [&](auto vc, auto n, auto lay) {
    constexpr int V = decltype(vc)::value, N = decltype(n)::value, L = decltype(lay)::value;
    auto fn = p.scale ? (p.residual ? rms_norm_fwd_kernel<E, V, N, L, true, true>
                                    : rms_norm_fwd_kernel<E, V, N, L, false, true>)
                      : (p.residual ? rms_norm_fwd_kernel<E, V, N, L, true, false>
                                    : rms_norm_fwd_kernel<E, V, N, L, false, false>);
    // A CTA a set of rows; kShifted, whose weights are slow to load, as many as run at once.
    int64_t most = p.rows;
    if (L == kShifted) {
      int n_sm = 1;
      cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n_sm, fn, int(sh.block.x * sh.block.y), 0);
      most = int64_t(sm_count) * std::max(1, n_sm);
    }
    fn<<<unsigned(ctas_of(sh, L, v, p.rows, most)), sh.block, 0, s>>>(p);
  });
}

size_t bwd_smem(int dim, const Shape& sh) {
  const size_t sums = sh.block.y * 32 * sizeof(float);
  return sh.block.y > 1 ? std::max(sums, size_t(sh.block.y) * dim * sizeof(float)) : sums;
}

template <class E>
int bwd_resident(const NormBwdParams& p, const Shape& sh) {
  int n = 1;
  with_shape<E>(p.layout, sh.n, [&](auto v, auto k, auto lay) {
    cudaOccupancyMaxActiveBlocksPerMultiprocessor(
        &n, rms_norm_bwd_kernel<E, decltype(v)::value, decltype(k)::value, decltype(lay)::value>,
        int(sh.block.x * sh.block.y), bwd_smem(p.dim, sh));
  });
  return std::max(1, n);
}

template <class E>
void bwd_e(const NormBwdParams& p, int parts, cudaStream_t s) {
  const Shape sh = shape_of(p.dim, vec_elements<E>(p.layout), p.layout);
  with_shape<E>(p.layout, sh.n, [&](auto v, auto n, auto lay) {
    rms_norm_bwd_kernel<E, decltype(v)::value, decltype(n)::value, decltype(lay)::value>
        <<<parts, sh.block, bwd_smem(p.dim, sh), s>>>(p);
  });
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

}  // namespace

void rms_norm_fwd_launch(NormType t, const NormFwdParams& p, int sm_count, cudaStream_t stream) {
  switch (t) {
    case NormType::kBf16: return fwd_e<__nv_bfloat16>(p, sm_count, stream);
    case NormType::kF16: return fwd_e<__half>(p, sm_count, stream);
    default: return fwd_e<float>(p, sm_count, stream);
  }
}

template <class E>
static int bwd_parts(const NormBwdParams& p, int sm_count) {
  const int v = vec_elements<E>(p.layout);
  const Shape sh = shape_of(p.dim, v, p.layout);
  return int(ctas_of(sh, p.layout, v, p.rows, int64_t(sm_count) * bwd_resident<E>(p, sh)));
}

int rms_norm_bwd_parts(NormType t, const NormBwdParams& p, int sm_count) {
  switch (t) {
    case NormType::kBf16: return bwd_parts<__nv_bfloat16>(p, sm_count);
    case NormType::kF16: return bwd_parts<__half>(p, sm_count);
    default: return bwd_parts<float>(p, sm_count);
  }
}

void rms_norm_bwd_launch(NormType t, const NormBwdParams& p, int parts, cudaStream_t stream) {
  switch (t) {
    case NormType::kBf16: return bwd_e<__nv_bfloat16>(p, parts, stream);
    case NormType::kF16: return bwd_e<__half>(p, parts, stream);
    default: return bwd_e<float>(p, parts, stream);
  }
}

}  // namespace mgfa
