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
// The alternatives are 64-bit keys that order by value and then by lower index, so that any
// order of work gives the same ones. Of a segment's threads, `top` have a largest key that is
// not below the top-th largest of these; so none of the segment's alternatives is below it,
// and few other elements are above: these are gathered in shared memory and ranked by
// counting, together with those of the segments before. A NaN counts as the largest value;
// it makes its row's sums NaN.
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

constexpr int kGather = 256;  // keys of a segment that are gathered at once

// What the threads that share a row (a CTA, or a warp) need for its alternatives.
struct Gather {
  uint64_t keys[kGather + 32];  // lanes' largest, then candidates
  uint64_t list[32];            // the alternatives so far, the largest first; 0: none
  uint64_t floor;
  int count;
};

template <int kT>
__device__ __forceinline__ void group_sync() {
  if constexpr (kT == 32) __syncwarp();
  else __syncthreads();
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
  // The largest element, NaN where one is: 16-bit ones in pairs as they lie.
  static __device__ __forceinline__ float largest(const Vec& a) {
    if constexpr (sizeof(E) == 4) {
      return max_nan(max_nan(a.e[0], a.e[1]), max_nan(a.e[2], a.e[3]));
    } else {
      using E2 = std::conditional_t<std::is_same_v<E, __half>, __half2, __nv_bfloat162>;
      auto pair = [&](int k) { return *reinterpret_cast<const E2*>(&a.w[k]); };
      const E2 m = __hmax2_nan(__hmax2_nan(pair(0), pair(1)), __hmax2_nan(pair(2), pair(3)));
      return max_nan(to_f(m.x), to_f(m.y));
    }
  }
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

// Adds a segment's elements to the alternatives of the threads that share the row: `at` are a
// thread's vectors, n of them in use, `top` its largest element.
template <class E, int kWarps>
__device__ __forceinline__ void add_segment(const Logits<E>& x, const typename Logits<E>::Vec (&at)[kVecs], int64_t first,
                                            int n, float top, int want, Gather& g) {
  constexpr int V = Logits<E>::V, kT = kWarps * 32;
  const int lane = threadIdx.x & 31, warp = kWarps == 1 ? 0 : int(threadIdx.x) >> 5, tid = warp * 32 + lane;
  using L = Logits<E>;
  using Vec = typename L::Vec;
  // calls take(key) for the elements of a vector of the thread
  auto each = [&](const Vec& v, int i, auto take) {
    const int64_t c0 = (first + i * kT + tid) * V - x.head;
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (c0 + j >= 0 && c0 + j < x.vocab) take(key_of(order_of(to_f(v.e[j])), int(c0) + j));
  };
  const bool any = first + tid < x.vecs;  // (a vector may hold nothing of the row but at its ends)
  uint32_t order = any ? order_of(top) : 0;
  // A bound that is quick to have: in each warp, a want / kWarps-th of the threads is not below.
  uint32_t bound = 0;
  if constexpr (kWarps > 1) {
    __shared__ uint32_t bounds[kWarps];
    uint32_t left = order;
    for (int j = (want + kWarps - 1) / kWarps; j > 0; --j) {
      bound = __reduce_max_sync(0xffffffffu, left);
      if (lane == __ffs(__ballot_sync(0xffffffffu, left == bound)) - 1) left = 0;
    }
    if (lane == 0) bounds[warp] = bound;
    if (tid == 0) g.count = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kWarps; ++j) bound = bounds[j] < bound ? bounds[j] : bound;
  } else {
    if (lane == 0) g.count = 0;
    __syncwarp();
  }
  // The want-th largest of the threads' largest keys.
  uint64_t mine = 0;
  const bool offers = any && order >= bound;
  if (offers) {
    // it is in the first vector whose largest element it is
    Vec in = at[0];
    int which = 0;
#pragma unroll
    for (int i = kVecs - 1; i > 0; --i)
      if (i < n && order_of(L::largest(at[i])) == order) {
        in = at[i];
        which = i;
      }
    if (order_of(L::largest(at[0])) == order) {
      in = at[0];
      which = 0;
    }
    each(in, which, [&](uint64_t key) { mine = key > mine ? key : mine; });
    if (mine) g.keys[atomicAdd(&g.count, 1)] = mine;
  }
  if (tid == 0) g.floor = 0;
  group_sync<kT>();
  const int offered = g.count;
  if (tid < offered) {
    const uint64_t key = g.keys[tid];
    int above = 0;
    for (int i = 0; i < offered; ++i) above += g.keys[i] > key;
    if (above == want - 1) g.floor = key;
  }
  group_sync<kT>();
  const uint64_t floor = g.floor > g.list[want - 1] ? g.floor : g.list[want - 1];
  if (tid == 0) g.count = 0;
  group_sync<kT>();
  // Only a thread whose largest key is not below the floor has others that are not.
  if (mine >= floor && mine) {
#pragma unroll
    for (int i = 0; i < kVecs; ++i)
      if (i < n && order_of(L::largest(at[i])) >= uint32_t(floor >> 32))
        each(at[i], i, [&](uint64_t key) {
          if (key >= floor) {
            const int to = atomicAdd(&g.count, 1);
            if (to < kGather) g.keys[to] = key;
          }
        });
  }
  group_sync<kT>();
  int gathered = g.count;
  if (gathered > kGather) {
    // Too many (a few threads with all that is large): the largest, the next one, and so on.
    __shared__ uint64_t tops[kWarpsCta];
    uint64_t below = ~uint64_t(0);
    for (int r = 0; r < want; ++r) {
      uint64_t key = 0;
#pragma unroll
      for (int i = 0; i < kVecs; ++i)
        if (i < n) each(at[i], i, [&](uint64_t k) { key = k < below && k > key ? k : key; });
      key = warp_top(key);
      if constexpr (kWarps > 1) {
        if (lane == 0) tops[warp] = key;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kWarps; ++j) key = tops[j] > key ? tops[j] : key;
        __syncthreads();
      }
      if (tid == 0) g.keys[r] = key;
      below = key;
    }
    gathered = want;
  }
  // The list so far joins them (its keys are others: of columns before).
  const uint64_t kept = tid < 32 ? g.list[tid] : 0;
  if (tid < 32) g.keys[gathered + tid] = kept;
  group_sync<kT>();
  const int all = gathered + 32;
  for (int c = tid; c < all; c += kT) {
    const uint64_t key = g.keys[c];
    int above = key ? 0 : 32;
    for (int i = 0; i < all; ++i) above += g.keys[i] > key;
    if (above < 32) g.list[above] = key;
  }
  group_sync<kT>();
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
  __shared__ Gather gathers[kTop ? kWarpsCta / kWarps : 1];
  Gather* const gather = kTop ? &gathers[kWarps == 1 ? warp : 0] : nullptr;
  if constexpr (kTop) {
    if (tid < 32) gather->list[tid] = 0;
  }
  for (int64_t first = int64_t(rank) * kVecs * kT; first < x.vecs; first += int64_t(ctas) * kVecs * kT) {
    typename L::Vec at[kVecs];
#pragma unroll
    for (int i = 0; i < kVecs; ++i) x.load(first + i * kT + tid, at[i]);
    // vectors of a thread that the row reaches
    const int n = x.vecs - first < kVecs * kT ? int((x.vecs - first + kT - 1) / kT) : kVecs;
    // the maximum
    float m = mine.m, top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      if (i >= n) break;
      top = max_nan(top, L::largest(at[i]));
    }
    m = max_nan(m, top);
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
      add_segment<E, kWarps>(x, at, first, n, top, p.top, *gather);
    }
  }
  mine = warp_join(mine);
  if constexpr (kWarps == 1) {
    if (lane == 0) finish(p, row, mine, given);
    if constexpr (kTop) {
      if (lane < p.top) put_top(p, row, lane, gather->list[lane], mine.m, logf(mine.s));
    }
  } else {
    __shared__ Sums sums[kWarps];
    if (lane == 0) sums[warp] = mine;
    __syncthreads();
    Sums all = lane < kWarps ? sums[lane] : Sums{-INFINITY, 0.f, 0.f};
    all = warp_join(all);
    if (ctas > 1) {
      cg::cluster_group cluster = cg::this_cluster();
      __shared__ Sums cta_sums;
      if (threadIdx.x == 0) cta_sums = all;
      cluster.sync();
      if (rank == 0) {
        all = lane < ctas ? *cluster.map_shared_rank(&cta_sums, lane) : Sums{-INFINITY, 0.f, 0.f};
        all = warp_join(all);
        if constexpr (kTop) gather->keys[threadIdx.x] = warp < ctas ? cluster.map_shared_rank(gather, warp)->list[lane] : 0;
      }
      cluster.sync();  // nobody leaves before the first CTA has read its results
      if (rank) return;
      if constexpr (kTop) {
        // the CTAs' lists: a key's place is how many are above it in each of them
        const uint64_t key = gather->keys[threadIdx.x];
        int place = key ? 0 : 32;
#pragma unroll
        for (int l = 0; l < kWarps; ++l) {
          const uint64_t* list = gather->keys + l * 32;
          int above = 0;
#pragma unroll
          for (int step = 16; step > 0; step >>= 1) above += list[above + step - 1] > key ? step : 0;
          place += above + (list[above] > key);
        }
        if (place < p.top) put_top(p, row, place, key, all.m, logf(all.s));
      }
    } else if constexpr (kTop) {
      if (int(threadIdx.x) < p.top) put_top(p, row, threadIdx.x, gather->list[threadIdx.x], all.m, logf(all.s));
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
  while (ctas < 8 && ctas < segments && p.rows * ctas < (kTop ? 1 : 16) * sm_count) ctas *= 2;
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
