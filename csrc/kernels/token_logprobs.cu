// Log probabilities of given tokens, the entropy of their distributions and the likeliest
// alternatives, in one pass over the logits; and the gradient.
//
//   m = max x,  S = sum e^(x - m),  logprob = x_t - m - ln S
//   H = -sum p ln p = ln S - (1/S) sum (x - m) e^(x - m)
//   dx_j = dl (1[j = t] - p_j) - dh p_j (ln p_j + H)
//
// Bound by memory: forward reads the logits, back reads them and writes dx. A row is cut
// into segments that its threads hold in registers while they need them three times (the
// maximum, the sums, the alternatives), so the logits are read once. Each thread keeps
// (m, S, sum) of its own, rescaled when its maximum grows; a row's are joined at the end:
// by shuffles, through shared memory and, where few rows share the SMs, across the CTAs of
// a cluster. Exponents are of base 2: sums hold W = sum (x - m) log2(e) e^(x - m).
//
// The alternatives are kept by each warp, one a lane, as 64-bit keys that order by value
// and then by lower index, so that any order of work gives the same ones. A NaN counts as
// the largest value; it makes its row's sums NaN.
#include "token_logprobs.cuh"

#include <cooperative_groups.h>

#include <algorithm>
#include <stdexcept>
#include <string>

#include "pairs.cuh"

namespace mgfa {
namespace {

using namespace mgfa::dev;
namespace cg = cooperative_groups;

constexpr int kThreads = 256;
constexpr int kWarpsCta = kThreads / 32;
constexpr int kVecs = 8;  // 16-byte vectors of a segment that a thread holds
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kLog2eRest = float(1.4426950408889634 - double(kLog2e));
// Exponents below this are taken as it: 2^it is 0 in float32, and so is the product of both
// (where the difference is infinite it would be NaN).
constexpr float kLeast = -200.f;

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// The sums of some of a row's elements, relative to their maximum.
struct Sums {
  float m, s, w;
};

__device__ __forceinline__ Sums join(const Sums& a, const Sums& b) {
  const float m = max_nan(a.m, b.m), base = m == -INFINITY ? 0.f : m;
  const float da = max_nan((a.m - base) * kLog2e, kLeast), db = max_nan((b.m - base) * kLog2e, kLeast);
  const float fa = ex2_approx(da), fb = ex2_approx(db);
  return {m, a.s * fa + b.s * fb, fa * (a.w + da * a.s) + fb * (b.w + db * b.s)};
}

__device__ __forceinline__ Sums warp_join(Sums v) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1)
    v = join(v, {__shfl_xor_sync(0xffffffffu, v.m, o), __shfl_xor_sync(0xffffffffu, v.s, o),
                 __shfl_xor_sync(0xffffffffu, v.w, o)});
  return v;
}

// Larger for larger values; equal for equal ones (both zeros); NaN above all. Never 0.
__device__ __forceinline__ uint32_t order_of(float v) {
  uint32_t b = __float_as_uint(v + 0.f);
  if (v != v) b = 0x7fffffffu;
  return b ^ (b & 0x80000000u ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t o) {
  return __uint_as_float(o ^ (o & 0x80000000u ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ uint64_t key_of(uint32_t order, int index) {
  return uint64_t(order) << 32 | uint32_t(~index);
}

// The largest of the warp's keys.
__device__ __forceinline__ uint64_t warp_top(uint64_t key) {
  const uint32_t hi = __reduce_max_sync(0xffffffffu, uint32_t(key >> 32));
  const uint32_t lo = __reduce_max_sync(0xffffffffu, uint32_t(key >> 32) == hi ? uint32_t(key) : 0u);
  return uint64_t(hi) << 32 | lo;
}

template <class E>
struct Logits {
  static constexpr int V = 16 / sizeof(E), kPairs = V / 2;
  using P = PairOf<E>;
  union Vec {
    uint4 v;
    typename P::Raw w[kPairs];
    E e[V];
  };
  // Row r as aligned vectors: element j of vector v is column v * V + j - head.
  const uint4* base;
  int head, vecs, vocab;
  __device__ __forceinline__ Logits(const void* x, int64_t offset, int n) : vocab(n) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(static_cast<const E*>(x) + offset);
    head = int(at % 16) / int(sizeof(E));
    base = reinterpret_cast<const uint4*>(at - at % 16);
    vecs = int((int64_t(head) + n + V - 1) / V);
  }
  __device__ __forceinline__ bool inside(int64_t v) const { return v * V >= head && (v + 1) * V <= int64_t(head) + vocab; }
  // -inf outside the row, whose first and last elements are read by themselves
  __device__ __forceinline__ void load(int64_t v, Vec& to) const {
    if (inside(v)) {
      to.v = __ldg(base + v);
    } else if (v >= vecs) {
#pragma unroll
      for (int k = 0; k < kPairs; ++k) to.w[k] = P::narrow(f2_pack(-INFINITY, -INFINITY));
    } else {
      const E* at = reinterpret_cast<const E*>(base) + v * V;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int64_t c = v * V + j - head;
        to.e[j] = c >= 0 && c < vocab ? at[j] : from_f<E>(-INFINITY);
      }
    }
  }
};

__device__ __forceinline__ int64_t target_of(const LogprobParams& p, int64_t row) {
  return p.targets64 ? static_cast<const int64_t*>(p.targets)[row]
                     : int64_t(static_cast<const int32_t*>(p.targets)[row]);
}

// A row's given token: its logit, and whether it has one.
struct Given {
  float x;
  bool ignored, known;
};
template <class E>
__device__ __forceinline__ Given given_of(const LogprobParams& p, int64_t row) {
  const int64_t t = target_of(p, row);
  Given g{0.f, t == p.ignore, t >= 0 && t < p.vocab};
  if (g.known) g.x = to_f(static_cast<const E*>(p.x)[row * p.stride + t]);
  return g;
}

// A row's results, by one thread.
__device__ __forceinline__ void finish(const LogprobParams& p, int64_t row, const Sums& v, const Given& g) {
  const bool none = v.m == -INFINITY;  // nothing but -inf: probabilities of 0
  const float ln_s = none ? 0.f : logf(v.s);
  const float h = none ? 0.f : ln_s - kLn2 * (v.w / v.s);
  if (!g.ignored && !g.known) record_error(p.status, kErrBadArgument, 68, 0);
  p.logprobs[row] = g.ignored ? 0.f : !g.known ? NAN : none ? -INFINITY : g.x - v.m - ln_s;
  p.entropy[row] = h;
  if (p.stats) reinterpret_cast<float4*>(p.stats)[row] = make_float4(v.m, v.s, ln_s, h);
}

__device__ __forceinline__ void put_top(const LogprobParams& p, int64_t row, int rank, uint64_t key,
                                        float m, float ln_s) {
  const float x = value_of(uint32_t(key >> 32));
  p.top_logprobs[row * p.top + rank] = m == -INFINITY ? -INFINITY : x - m - ln_s;
  p.top_indices[row * p.top + rank] = int64_t(uint32_t(~uint32_t(key)));
}

// kWarps 8: a row for a cluster of CTAs, which take its segments in turn; 1: a row a warp.
template <class E, int kWarps, bool kTop>
__global__ void __launch_bounds__(kThreads, kTop ? 2 : 3) token_logprobs_kernel(const LogprobParams p, int ctas) {
  using L = Logits<E>;
  using P = typename L::P;
  constexpr int V = L::V, kPairs = L::kPairs, kT = kWarps * 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int tid = kWarps == 1 ? lane : int(threadIdx.x);
  const int rank = kWarps == 1 ? 0 : int(blockIdx.x % unsigned(ctas));
  const int64_t row = kWarps == 1 ? int64_t(blockIdx.x) * kWarpsCta + warp : int64_t(blockIdx.x / unsigned(ctas));
  if (kWarps == 1 && row >= p.rows) return;  // the whole warp, which no other waits for
  const L x(p.x, row * p.stride, p.vocab);
  const Given given = given_of<E>(p, row);
  Sums mine{-INFINITY, 0.f, 0.f};
  uint64_t best = 0;  // the lane's of the warp's alternatives, the largest in lane 0
  for (int64_t first = int64_t(rank) * kVecs * kT; first < x.vecs; first += int64_t(ctas) * kVecs * kT) {
    typename L::Vec at[kVecs];
#pragma unroll
    for (int i = 0; i < kVecs; ++i) x.load(first + i * kT + tid, at[i]);
    // vectors of a thread that the row reaches
    const int n = x.vecs - first < kVecs * kT ? int((x.vecs - first + kT - 1) / kT) : kVecs;
    // the maximum
    float m = mine.m;
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      if (i >= n) break;
#pragma unroll
      for (int k = 0; k < kPairs; ++k) {
        float a, b;
        f2_unpack(P::wide(at[i].w[k]), a, b);
        m = max_nan(m, max_nan(a, b));
      }
    }
    const float base = m == -INFINITY ? 0.f : m;
    uint64_t s = f2_pack(0.f, 0.f), w = s;
    if (m != mine.m && mine.m != -INFINITY) {
      const Sums moved = join(mine, {m, 0.f, 0.f});
      mine.s = moved.s;
      mine.w = moved.w;
    }
    mine.m = m;
    const uint64_t minus = f2_pack(-base, -base), log2e = f2_pack(kLog2e, kLog2e);
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      if (i >= n) break;
#pragma unroll
      for (int k = 0; k < kPairs; ++k) {
        // the difference first: it is exact or nearly so where the exponential counts
        float a, b;
        f2_unpack(f2_mul(f2_add(P::wide(at[i].w[k]), minus), log2e), a, b);
        a = max_nan(a, kLeast);
        b = max_nan(b, kLeast);
        const uint64_t e = f2_pack(ex2_approx(a), ex2_approx(b));
        s = f2_add(s, e);
        w = f2_fma(e, f2_pack(a, b), w);
      }
    }
    float a, b;
    f2_unpack(s, a, b);
    mine.s += a + b;
    f2_unpack(w, a, b);
    mine.w += a + b;
    if constexpr (kTop) {
      // Each lane offers its largest element that has not been taken; the warp's largest is
      // put in its place in the list, while it is above the last one there.
      uint64_t tops[kVecs];
      auto top_of = [&](int i, uint64_t below) {
        uint64_t t = 0;
        const int64_t v = first + i * kT + tid;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const int64_t c = v * V + j - x.head;
          const uint64_t key = key_of(order_of(to_f(at[i].e[j])), int(c));
          if (c >= 0 && c < x.vocab && key < below && key > t) t = key;
        }
        return t;
      };
      uint64_t offer = 0;
#pragma unroll
      for (int i = 0; i < kVecs; ++i) {
        tops[i] = i < n ? top_of(i, ~uint64_t(0)) : 0;
        offer = tops[i] > offer ? tops[i] : offer;
      }
      for (;;) {
        const uint64_t key = warp_top(offer);
        if (key <= __shfl_sync(0xffffffffu, best, p.top - 1)) break;
        const int place = __popc(__ballot_sync(0xffffffffu, best > key));
        const uint64_t up = __shfl_up_sync(0xffffffffu, best, 1);
        best = lane < place ? best : lane == place ? key : up;
        if (offer == key) {
          offer = 0;
#pragma unroll
          for (int i = 0; i < kVecs; ++i) {
            if (tops[i] == key) tops[i] = top_of(i, key);
            offer = tops[i] > offer ? tops[i] : offer;
          }
        }
      }
    }
  }
  mine = warp_join(mine);
  if constexpr (kWarps == 1) {
    if (lane == 0) finish(p, row, mine, given);
    if (kTop && lane < p.top) put_top(p, row, lane, best, mine.m, logf(mine.s));
  } else {
    __shared__ Sums sums[kWarps];
    __shared__ uint64_t tops[kTop ? kThreads : 1];  // of the CTA's warps, then of the cluster's CTAs
    __shared__ uint64_t list[kTop ? 32 : 1];        // the CTA's, in order
    if (lane == 0) sums[warp] = mine;
    if constexpr (kTop) {
      tops[threadIdx.x] = lane < p.top ? best : 0;
      if (threadIdx.x < 32) list[threadIdx.x] = 0;
    }
    __syncthreads();
    Sums all = lane < kWarps ? sums[lane] : Sums{-INFINITY, 0.f, 0.f};
    all = warp_join(all);
    // the place of a thread's key among `tops`, or 32
    auto place = [&](uint64_t key) {
      int n = key ? 0 : 32;
      for (int i = 0; i < kThreads; ++i) n += tops[i] > key;
      return n < 32 ? n : 32;
    };
    if constexpr (kTop) {
      const uint64_t key = tops[threadIdx.x];
      const int n = place(key);
      if (n < p.top) list[n] = key;
      __syncthreads();
    }
    if (ctas > 1) {
      cg::cluster_group cluster = cg::this_cluster();
      __shared__ Sums cta_sums;
      if (threadIdx.x == 0) cta_sums = all;
      cluster.sync();
      if (rank == 0) {
        all = lane < ctas ? *cluster.map_shared_rank(&cta_sums, lane) : Sums{-INFINITY, 0.f, 0.f};
        all = warp_join(all);
        if constexpr (kTop) tops[threadIdx.x] = warp < ctas ? cluster.map_shared_rank(list, warp)[lane] : 0;
      }
      cluster.sync();  // nobody leaves before the first CTA has read its results
      if (rank) return;
      if constexpr (kTop) {
        const uint64_t key = tops[threadIdx.x];
        const int n = place(key);
        if (n < p.top) put_top(p, row, n, key, all.m, logf(all.s));
      }
    } else if constexpr (kTop) {
      if (int(threadIdx.x) < p.top) put_top(p, row, threadIdx.x, list[threadIdx.x], all.m, logf(all.s));
    }
    if (threadIdx.x == 0) finish(p, row, all, given);
  }
}

// dx of a row's segments. Where x's and dx's rows lie differently to 16-byte boundaries, dx
// is written by elements.
constexpr int kBackVecs = 4;
// kT threads a segment: a CTA, or a warp for rows of few vectors.
template <class E, int kT>
__global__ void __launch_bounds__(kThreads) token_logprobs_bwd_kernel(const LogprobBwdParams p, int segments) {
  using L = Logits<E>;
  using P = typename L::P;
  constexpr int V = L::V, kPairs = L::kPairs;
  const int64_t unit = kT == kThreads ? int64_t(blockIdx.x) : int64_t(blockIdx.x) * (kThreads / kT) + threadIdx.x / kT;
  const int64_t row = unit / segments;
  if (row >= p.rows) return;
  const int tid = threadIdx.x % kT;
  const int64_t first = (unit - row * segments) * kBackVecs * kT;
  const L x(p.x, row * p.stride, p.vocab);
  E* const dx = static_cast<E*>(p.dx) + row * p.vocab;
  typename L::Vec at[kBackVecs];
#pragma unroll
  for (int i = 0; i < kBackVecs; ++i) x.load(first + i * kT + tid, at[i]);
  const int64_t t = target_of(p, row);
  const bool known = t != p.ignore && t >= 0 && t < p.vocab;
  const float4 stats = reinterpret_cast<const float4*>(p.stats)[row];
  const float m = stats.x, ln_s = stats.z, h = stats.w;
  const bool none = m == -INFINITY;
  const float dl = known && p.dl && !none ? p.dl[row * p.dl_stride] : 0.f;
  const float dh = p.dh && !none ? p.dh[row * p.dh_stride] : 0.f;
  const float base = none ? 0.f : m, inv = none ? 0.f : 1.f / stats.y;
  const bool alike = (reinterpret_cast<uintptr_t>(dx) - reinterpret_cast<uintptr_t>(static_cast<const E*>(p.x) + row * p.stride)) % 16 == 0;
  const int place = known ? int(t) : -1;
#pragma unroll
  for (int i = 0; i < kBackVecs; ++i) {
    const int64_t v = first + i * kT + tid, c0 = v * V - x.head;
    if (v >= x.vecs) break;
#pragma unroll
    for (int k = 0; k < kPairs; ++k) {
      float z[2], d[2];
      f2_unpack(f2_add(P::wide(at[i].w[k]), f2_pack(-base, -base)), z[0], z[1]);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        // 2^(z log2 e) with the product in two parts: rounding it would cost up to |z| steps
        const float y = max_nan(z[j] * kLog2e, kLeast), lo = y > kLeast ? fmaf(z[j], kLog2eRest, fmaf(z[j], kLog2e, -y)) : 0.f;
        const float e = ex2_approx(y), prob = fmaf(e, lo * kLn2, e) * inv;
        // where z is -inf, ln p times p is 0
        const float lnp = max_nan(z[j], kLeast) - ln_s;
        d[j] = -prob * fmaf(dh, lnp + h, dl);
        if (c0 + 2 * k + j == place) d[j] += dl;
      }
      at[i].w[k] = P::narrow(f2_pack(d[0], d[1]));
    }
    if (alike && x.inside(v)) {
      *reinterpret_cast<uint4*>(dx + c0) = at[i].v;
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (c0 + j >= 0 && c0 + j < p.vocab) dx[c0 + j] = at[i].e[j];
    }
  }
}

void cuda_ok(cudaError_t e) {
  if (e != cudaSuccess) throw std::runtime_error(std::string("token_logprobs: ") + cudaGetErrorString(e));
}

unsigned grid_of(int64_t n) {
  if (n >= int64_t(1) << 31) throw std::runtime_error("token_logprobs: too many logits");
  return unsigned(n);
}

template <class E, bool kTop>
void launch_e(const LogprobParams& p, int sm_count, cudaStream_t s) {
  constexpr int V = 16 / sizeof(E);
  const int64_t vecs = (int64_t(p.vocab) + V - 1) / V + 1;
  if (vecs <= 32 * kVecs) {  // a segment of a warp
    token_logprobs_kernel<E, 1, kTop><<<grid_of((p.rows + kWarpsCta - 1) / kWarpsCta), kThreads, 0, s>>>(p, 1);
    return cuda_ok(cudaGetLastError());
  }
  // CTAs of a row: as many as it has segments, up to 8, while the rows alone do not fill the
  // SMs four times over.
  const int64_t segments = (vecs + kThreads * kVecs - 1) / (kThreads * kVecs);
  int ctas = 1;
  while (ctas < 8 && ctas < segments && p.rows * ctas < 16 * sm_count) ctas *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid_of(p.rows * ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cuda_ok(cudaLaunchKernelEx(&cfg, token_logprobs_kernel<E, 8, kTop>, p, ctas));
}

template <class E, int kT>
void bwd_t(const LogprobBwdParams& p, int64_t vecs, cudaStream_t s) {
  const int64_t segments = (vecs + kT * kBackVecs - 1) / (kT * kBackVecs);
  token_logprobs_bwd_kernel<E, kT>
      <<<grid_of((p.rows * segments + kThreads / kT - 1) / (kThreads / kT)), kThreads, 0, s>>>(p, int(segments));
  cuda_ok(cudaGetLastError());
}

template <class E>
void bwd_e(const LogprobBwdParams& p, cudaStream_t s) {
  constexpr int V = 16 / sizeof(E);
  const int64_t vecs = (int64_t(p.vocab) + V - 1) / V + 1;
  if (vecs < kThreads * kBackVecs) bwd_t<E, 32>(p, vecs, s);
  else bwd_t<E, kThreads>(p, vecs, s);
}

}  // namespace

void token_logprobs_launch(LogitType t, const LogprobParams& p, int sm_count, cudaStream_t s) {
  switch (t) {
    case LogitType::kBf16: return p.top ? launch_e<__nv_bfloat16, true>(p, sm_count, s) : launch_e<__nv_bfloat16, false>(p, sm_count, s);
    case LogitType::kF16: return p.top ? launch_e<__half, true>(p, sm_count, s) : launch_e<__half, false>(p, sm_count, s);
    default: return p.top ? launch_e<float, true>(p, sm_count, s) : launch_e<float, false>(p, sm_count, s);
  }
}

void token_logprobs_bwd_launch(LogitType t, const LogprobBwdParams& p, cudaStream_t s) {
  switch (t) {
    case LogitType::kBf16: return bwd_e<__nv_bfloat16>(p, s);
    case LogitType::kF16: return bwd_e<__half>(p, s);
    default: return bwd_e<float>(p, s);
  }
}

}  // namespace mgfa
