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
// order of work gives the same ones. What is not below a bound that the threads' largest
// elements give is gathered in shared memory and ranked by counting, together with the
// alternatives of the segments before. A NaN counts as the largest value; it makes its row's
// sums NaN.
//
// Bound by memory: 4096 rows of 131072 in bf16 take 195 us (1.07 GB, 5.5 TB/s) and 311 us back
// (2.15 GB, 6.9 TB/s; 517 us before a segment was loaded while the one before is worked on).
// 1021 rows of 50001 in fp32 take 46 and 62 us (4.4 and 6.6 TB/s). 64 rows of 131072 with 20
// alternatives, 17 MB, take 17 us, bound by the steps of a segment one behind another. The whole
// call took 79 us when a warp inserted its alternatives one by one, and 23 us with a second
// pass over the segment for those above the bound.
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
  uint64_t keys[kGather + 32];
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
  static __device__ __forceinline__ float element(const Vec& a, int j) {
    if constexpr (sizeof(E) == 4) {
      return j & 2 ? (j & 1 ? a.e[3] : a.e[2]) : (j & 1 ? a.e[1] : a.e[0]);
    } else {
      const uint32_t w = j & 4 ? (j & 2 ? a.w[3] : a.w[2]) : (j & 2 ? a.w[1] : a.w[0]);
      const uint16_t h = uint16_t(j & 1 ? w >> 16 : w);
      return to_f(*reinterpret_cast<const E*>(&h));
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
  float x = 0.f;
  bool ignored = true, known = false;
};
template <class E>
__device__ __forceinline__ Given given_of(const LogprobParams& p, int64_t row) {
  const int64_t t = target_of(p, row);
  Given g;
  g.ignored = t == p.ignore;
  g.known = t >= 0 && t < p.vocab;
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

// The elements of vector v, each as take(key).
template <class E, class Take>
__device__ __forceinline__ void each_key(const Logits<E>& x, const typename Logits<E>::Vec& a, int64_t v, Take take) {
  constexpr int V = Logits<E>::V;
  const int64_t c0 = v * V - x.head;
#pragma unroll
  for (int j = 0; j < V; ++j)
    if (c0 + j >= 0 && c0 + j < x.vocab) take(key_of(order_of(to_f(a.e[j])), int(c0) + j));
}

// A segment's elements join the alternatives of the threads that share the row, in two steps.
// First all that is not below a bound is gathered, which is quick to have: in each warp a
// want / kWarps-th of the threads have a largest element (`top`, of the n vectors `at` in use)
// that is not below it, so that the segment's `want` largest are among them. (A NaN bound, of
// a segment with fewer threads, takes all.)
template <class E, int kWarps>
__device__ __forceinline__ void gather_segment(const Logits<E>& x, const typename Logits<E>::Vec (&at)[kVecs],
                                               int64_t first, int n, float top, int want, Gather& g) {
  using L = Logits<E>;
  constexpr int V = L::V, kT = kWarps * 32;
  const int lane = threadIdx.x & 31, warp = kWarps == 1 ? 0 : int(threadIdx.x) >> 5, tid = warp * 32 + lane;
  const uint32_t order = first + tid < x.vecs ? order_of(top) : 0;
  uint32_t bound = 0;
  if (tid == 0) g.count = 0;
  if constexpr (kWarps > 1) {
    __shared__ uint32_t bounds[kWarps];
    uint32_t left = order;
    for (int j = (want + kWarps - 1) / kWarps; j > 0; --j) {
      bound = __reduce_max_sync(0xffffffffu, left);
      if (lane == __ffs(__ballot_sync(0xffffffffu, left == bound)) - 1) left = 0;
    }
    if (lane == 0) bounds[warp] = bound;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kWarps; ++j) bound = bounds[j] < bound ? bounds[j] : bound;
  } else {
    __syncwarp();
    int above = 0;  // lanes before this one in the order of their largest elements
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      const uint32_t other = __shfl_sync(0xffffffffu, order, j);
      above += other > order || (other == order && j < lane);
    }
    bound = __shfl_sync(0xffffffffu, order, __ffs(__ballot_sync(0xffffffffu, above == want - 1)) - 1);
  }
  const float least = value_of(bound);
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    if (i >= n) break;
    if (L::largest(at[i]) < least) continue;
    uint32_t mask = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) mask |= uint32_t(!(to_f(at[i].e[j]) < least)) << j;
    const int64_t c0 = (first + i * kT + tid) * V - x.head;
    for (; mask; mask &= mask - 1) {
      const int j = __ffs(mask) - 1;
      if (c0 + j < 0 || c0 + j >= x.vocab) continue;
      const int to = atomicAdd(&g.count, 1);
      if (to < kGather) g.keys[to] = key_of(order_of(L::element(at[i], j)), int(c0) + j);
    }
  }
  group_sync<kT>();
}

// Then they are ranked together with the list so far. Where too many were gathered (equal
// logits, a few threads with all that is large), the segment is read again.
template <class E, int kWarps>
__device__ __forceinline__ void rank_segment(const Logits<E>& x, int64_t first, int n, int want, Gather& g) {
  using L = Logits<E>;
  constexpr int kT = kWarps * 32;
  const int lane = threadIdx.x & 31, warp = kWarps == 1 ? 0 : int(threadIdx.x) >> 5, tid = warp * 32 + lane;
  int gathered = g.count;
  if (gathered > kGather) {
    group_sync<kT>();
    auto each = [&](auto take) {
#pragma unroll 1
      for (int i = 0; i < n; ++i) {
        typename L::Vec a;
        x.load(first + i * kT + tid, a);
        each_key<E>(x, a, first + i * kT + tid, take);
      }
    };
    // The want-th largest of the threads' largest keys is a better bound.
    uint64_t mine = 0;
    each([&](uint64_t key) { mine = key > mine ? key : mine; });
    g.keys[tid] = mine;
    if (tid == 0) {
      g.count = 0;
      g.floor = 0;
    }
    group_sync<kT>();
    int above = 0;
    for (int i = 0; i < kT; ++i) above += g.keys[i] > mine;
    if (mine && above == want - 1) g.floor = mine;
    group_sync<kT>();
    const uint64_t floor = g.floor;
    if (mine >= floor)
      each([&](uint64_t key) {
        if (key >= floor) {
          const int to = atomicAdd(&g.count, 1);
          if (to < kGather) g.keys[to] = key;
        }
      });
    group_sync<kT>();
    gathered = g.count;
    if (gathered > kGather) {
      // Still too many: the largest, the next one, and so on.
      __shared__ uint64_t tops[kWarpsCta];
      uint64_t below = ~uint64_t(0);
      for (int r = 0; r < want; ++r) {
        uint64_t key = 0;
        each([&](uint64_t k) { key = k < below && k > key ? k : key; });
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
  }
  // (the list's keys are others: of columns before)
  if (tid < 32) g.keys[gathered + tid] = g.list[tid];
  group_sync<kT>();
  const int all = gathered + 32;
  for (int c = tid; c < all; c += kT) {
    const uint64_t key = g.keys[c];
    int above = key ? 0 : 32;
#pragma unroll 4
    for (int i = 0; i < all; ++i) above += g.keys[i] > key;
    if (above < 32) g.list[above] = key;
  }
  group_sync<kT>();
}

// kWarps 8: a row for a cluster of CTAs, which take its segments in turn; 1: a row a warp.
template <class E, int kWarps, bool kTop>
__global__ void __launch_bounds__(kThreads, kTop ? 2 : 4) token_logprobs_kernel(const LogprobParams p, int ctas) {
  using L = Logits<E>;
  using P = typename L::P;
  constexpr int V = L::V, kPairs = L::kPairs, kT = kWarps * 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int tid = kWarps == 1 ? lane : int(threadIdx.x);
  const int rank = kWarps == 1 ? 0 : int(blockIdx.x % unsigned(ctas));
  const int64_t row = kWarps == 1 ? int64_t(blockIdx.x) * kWarpsCta + warp : int64_t(blockIdx.x / unsigned(ctas));
  if (kWarps == 1 && row >= p.rows) return;  // the whole warp, which no other waits for
  const L x(p.x, row * p.stride, p.vocab);
  Given given;
  Sums mine{-INFINITY, 0.f, 0.f};
  __shared__ Gather gathers[kTop ? kWarpsCta / kWarps : 1];
  Gather* const gather = kTop ? &gathers[kWarps == 1 ? warp : 0] : nullptr;
  if constexpr (kTop) {
    if (tid < 32) gather->list[tid] = 0;
  }
  const int64_t step = int64_t(ctas) * kVecs * kT;
  typename L::Vec at[kVecs];
  auto load = [&](int64_t first) {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) x.load(first + i * kT + tid, at[i]);
  };
  if (kTop) load(int64_t(rank) * kVecs * kT);
  for (int64_t first = int64_t(rank) * kVecs * kT; first < x.vecs; first += step) {
    if (!kTop) load(first);
    if (first == int64_t(rank) * kVecs * kT) given = given_of<E>(p, row);  // behind the first loads
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
      gather_segment<E, kWarps>(x, at, first, n, top, p.top, *gather);
      if (first + step < x.vecs) load(first + step);
      rank_segment<E, kWarps>(x, first, n, p.top, *gather);
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

// dx. A row's segments go to `parts` units of kT threads (a CTA, or a warp where rows have few
// vectors), each of which loads its next segment before it works on one. Where x's and dx's
// rows lie differently to 16-byte boundaries, dx is written by elements.
constexpr int kBackVecs = 4;
template <class E, int kT>
__global__ void __launch_bounds__(kThreads) token_logprobs_bwd_kernel(const LogprobBwdParams p, int parts) {
  using L = Logits<E>;
  using P = typename L::P;
  constexpr int V = L::V, kPairs = L::kPairs;
  const int64_t unit = kT == kThreads ? int64_t(blockIdx.x) : int64_t(blockIdx.x) * (kThreads / kT) + threadIdx.x / kT;
  const int64_t row = unit / parts;
  if (row >= p.rows) return;
  const int tid = threadIdx.x % kT;
  const int64_t step = int64_t(parts) * kBackVecs * kT;
  int64_t first = (unit - row * parts) * kBackVecs * kT;
  const L x(p.x, row * p.stride, p.vocab);
  E* const dx = static_cast<E*>(p.dx) + row * p.vocab;
  typename L::Vec at[kBackVecs], ahead[kBackVecs];
  auto load = [&](int64_t from, typename L::Vec (&to)[kBackVecs]) {
#pragma unroll
    for (int i = 0; i < kBackVecs; ++i) x.load(from + i * kT + tid, to[i]);
  };
  load(first, at);
  const int64_t t = target_of(p, row);
  const bool known = t != p.ignore && t >= 0 && t < p.vocab;
  const float4 stats = reinterpret_cast<const float4*>(p.stats)[row];
  const float m = stats.x, ln_s = stats.z, h = stats.w;
  const bool none = m == -INFINITY;
  const float dl = known && p.dl && !none ? p.dl[row * p.dl_stride] : 0.f;
  const float dh = p.dh && !none ? p.dh[row * p.dh_stride] : 0.f;
  const float base = none ? 0.f : m, inv = none ? 0.f : 1.f / stats.y;
  const bool alike = (reinterpret_cast<uintptr_t>(dx) - reinterpret_cast<uintptr_t>(static_cast<const E*>(p.x) + row * p.stride)) % 16 == 0;
  const int64_t place = known ? t : -1;
  // dl + dh (ln p + H) = rest + dh z
  const float rest = fmaf(dh, h - ln_s, dl);
  const uint64_t minus = f2_pack(-base, -base), log2e = f2_pack(kLog2e, kLog2e), inv2 = f2_pack(-inv, -inv),
                 dh2 = f2_pack(dh, dh), rest2 = f2_pack(rest, rest);
  for (; first < x.vecs; first += step) {
    if (first + step < x.vecs) load(first + step, ahead);
#pragma unroll
    for (int i = 0; i < kBackVecs; ++i) {
      const int64_t v = first + i * kT + tid, c0 = v * V - x.head;
      if (v >= x.vecs) break;
      float d[V];
#pragma unroll
      for (int k = 0; k < kPairs; ++k) {
        float z[2], y[2], e[2];
        f2_unpack(f2_add(P::wide(at[i].w[k]), minus), z[0], z[1]);
        // (-inf would be NaN in the products below; e^kLeast is 0 already)
        z[0] = max_nan(z[0], kLeast);
        z[1] = max_nan(z[1], kLeast);
        const uint64_t zz = f2_pack(z[0], z[1]), yy = f2_mul(zz, log2e);
        f2_unpack(yy, y[0], y[1]);
        e[0] = ex2_approx(y[0]);
        e[1] = ex2_approx(y[1]);
        uint64_t ee = f2_pack(e[0], e[1]);
        if constexpr (sizeof(E) == 4) {
          // z log2 e in two parts: rounding it costs up to |z| steps of float32 (of which 16-bit
          // results see nothing)
          const uint64_t minus1 = f2_pack(-1.f, -1.f), more = f2_pack(kLog2eRest, kLog2eRest), ln2 = f2_pack(kLn2, kLn2);
          const uint64_t lo = f2_fma(zz, more, f2_fma(zz, log2e, f2_mul(yy, minus1)));
          ee = f2_fma(ee, f2_mul(lo, ln2), ee);
        }
        f2_unpack(f2_mul(f2_mul(ee, inv2), f2_fma(dh2, zz, rest2)), d[2 * k], d[2 * k + 1]);
      }
      if (place >= c0 && place < c0 + V) {
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (c0 + j == place) d[j] += dl;
      }
#pragma unroll
      for (int k = 0; k < kPairs; ++k) at[i].w[k] = P::narrow(f2_pack(d[2 * k], d[2 * k + 1]));
      if (alike && x.inside(v)) {
        *reinterpret_cast<uint4*>(dx + c0) = at[i].v;
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (c0 + j >= 0 && c0 + j < p.vocab) dx[c0 + j] = at[i].e[j];
      }
    }
#pragma unroll
    for (int i = 0; i < kBackVecs; ++i) at[i].v = ahead[i].v;
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
  // CTAs of a row: as many as it has segments, up to 8, while the rows alone do not fill the SMs
  // (1021 rows of 50001 in fp32: with one 46 us, with four 69 us; 64 rows of 131072 with
  // alternatives: with four or eight 17 us, 4096 rows: 195 us with one).
  const int64_t segments = (vecs + kThreads * kVecs - 1) / (kThreads * kVecs);
  int ctas = 1;
  while (ctas < 8 && ctas < segments && p.rows * ctas < (kTop ? 1 : 4) * sm_count) ctas *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid_of(p.rows * ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = ctas > 1 ? 1 : 0;
  cuda_ok(cudaLaunchKernelEx(&cfg, token_logprobs_kernel<E, 8, kTop>, p, ctas));
}

template <class E, int kT>
void bwd_t(const LogprobBwdParams& p, int64_t vecs, int sm_count, cudaStream_t s) {
  const int64_t segments = (vecs + kT * kBackVecs - 1) / (kT * kBackVecs);
  // as few units as keep the SMs evenly loaded
  int64_t parts = 1;
  while (parts * 2 <= segments && p.rows * parts * kT < 16 * int64_t(kThreads) * sm_count * 4) parts *= 2;
  token_logprobs_bwd_kernel<E, kT>
      <<<grid_of((p.rows * parts + kThreads / kT - 1) / (kThreads / kT)), kThreads, 0, s>>>(p, int(parts));
  cuda_ok(cudaGetLastError());
}

template <class E>
void bwd_e(const LogprobBwdParams& p, int sm_count, cudaStream_t s) {
  constexpr int V = 16 / sizeof(E);
  const int64_t vecs = (int64_t(p.vocab) + V - 1) / V + 1;
  if (vecs < kThreads * kBackVecs) bwd_t<E, 32>(p, vecs, sm_count, s);
  else bwd_t<E, kThreads>(p, vecs, sm_count, s);
}

}  // namespace

void token_logprobs_launch(LogitType t, const LogprobParams& p, int sm_count, cudaStream_t s) {
  switch (t) {
    case LogitType::kBf16: return p.top ? launch_e<__nv_bfloat16, true>(p, sm_count, s) : launch_e<__nv_bfloat16, false>(p, sm_count, s);
    case LogitType::kF16: return p.top ? launch_e<__half, true>(p, sm_count, s) : launch_e<__half, false>(p, sm_count, s);
    default: return p.top ? launch_e<float, true>(p, sm_count, s) : launch_e<float, false>(p, sm_count, s);
  }
}

void token_logprobs_bwd_launch(LogitType t, const LogprobBwdParams& p, int sm_count, cudaStream_t s) {
  switch (t) {
    case LogitType::kBf16: return bwd_e<__nv_bfloat16>(p, sm_count, s);
    case LogitType::kF16: return bwd_e<__half>(p, sm_count, s);
    default: return bwd_e<float>(p, sm_count, s);
  }
}

}  // namespace mgfa
