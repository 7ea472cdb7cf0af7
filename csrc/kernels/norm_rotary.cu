// Root-mean-square norm of each query and key head with the rotary positions in the same
// pass, its gradients, and the same on the way into a paged cache:
//
//   n = x * rstd * w,  rstd = 1 / sqrt(mean(x^2) + eps) over the head,  y = R(t) n
//
// R(t) rotates the pairs of the first rotary_dim columns (rotary.cu). Back, with
// g = R(-t) dy (the transpose):
//
//   dw = sum over tokens and heads of g * x * rstd
//   dx = rstd * (g w - x * rstd^2 * mean(g w x))
//
// Bound by memory: forward reads x and writes y, back reads x and dy and writes dx. A
// head's sums stay within the 1 to 32 lanes that hold it, so neither pass waits for more
// than shuffles; rstd is computed again from x in the backward pass, which reads x anyway.
// The sines, cosines and weights of a thread's columns take the registers that loads under
// way would need: so each thread has a ring in shared memory, into which it copies (cp.async)
// what it will work on 4 or 8 heads later, and no other thread waits for it. 16384 tokens of
// 32 + 8 heads of 128 in bf16 take 60 us forward (336 MB, 5.6 TB/s) and 97 us back (503 MB,
// 5.2 TB/s), the sum of the weights' parts 7 us more; the first version, which loaded into
// registers, took 88 and 188 us. At four heads a thread the angles were 8 of 67 us forward and
// 9 of 106 back; eight heads that share them (make_cut) gained that much. 8.4K tokens into a
// cache, 214 MB, take 42 us; 64 single tokens 6.6 us, which is latency. In fp32 8192 tokens of
// the same heads take 63 us forward (336 MB, 5.3 TB/s) and 95 us back, with the weights' sum
// (503 MB, 5.3 TB/s).
#include "norm_rotary.cuh"

#include <algorithm>
#include <atomic>
#include <cmath>
#include <stdexcept>
#include <string>

#include "pairs.cuh"
#include "paged_attn.cuh"

namespace mgfa {
namespace {

using namespace mgfa::dev;

constexpr int kThreads = 256;
// Heads of a unit, two units being a thread's ring (kHalves: 256 bytes either way).
constexpr int kFwdUnit = 4, kBwdUnit = 2;

// How a head's columns are cut (V elements are 16 bytes):
enum : int {
  kHalves = 0,      // a lane has V columns of either half of the pairs, then V others
  kNeighbours = 1,  // V columns with the pairs (2i, 2i + 1) inside
  kAny = 2,         // V columns; each one's partner is fetched by itself (from L1)
};

inline int lanes_of(int mode, int v, int head_dim, int rotary_dim) {
  return mode == kHalves ? rotary_dim / 2 / v + (head_dim - rotary_dim) / v : head_dim / v;
}

// A CTA's threads: `tile` tokens, of each slots[0] + slots[1] + slots[2] groups of
// 2^lanes_log threads, for query, key and (append) value heads. Group i of n takes heads
// i, i + n, ... of its kind, `rounds` of them at most. The CTA takes every gridDim.x-th tile.
struct Cut {
  int tile, threads, lanes, lanes_log, rounds;
  int slots[3];
};

Cut make_cut(int lanes, const int (&heads)[3], int64_t tokens, int sm_count) {
  Cut c;
  c.lanes = lanes;
  c.lanes_log = 0;
  while (1 << c.lanes_log < lanes) ++c.lanes_log;
  const int most = kThreads >> c.lanes_log;
  // Heads a thread, which share its columns' angles: not so many that threads run out; of
  // these the number whose groups are the least idle, a head and a half for the angles counted.
  // (16384 tokens of 32 + 8 heads of 128: with 4, 8, 10 and 16 heads 67, 60, 61 and 66 us
  // forward; 900 tokens of 3 times 8 heads of 64 into the cache: with 8 10.8 us, with 1 6.7 us.)
  const int64_t all = tokens * (heads[0] + heads[1] + heads[2]) << c.lanes_log;
  const int limit = int(std::max<int64_t>(1, std::min<int64_t>(16, all / (2 * int64_t(kThreads) * sm_count))));
  int batch = 1, total = 0;
  float least = INFINITY;
  for (int i = limit; i > 0; --i) {
    int slots = 0;
    for (int h : heads) slots += (h + i - 1) / i;
    int rounds = 0;
    for (int h : heads)
      if (h) rounds = std::max(rounds, (h + (h + i - 1) / i - 1) / ((h + i - 1) / i));
    if (slots * (rounds + 1.5f) < least) {
      least = slots * (rounds + 1.5f);
      batch = i;
    }
  }
  int want[3], sum = 0;
  for (int i = 0; i < 3; ++i) sum += want[i] = (heads[i] + batch - 1) / batch;
  for (int i = 0; i < 3; ++i) {
    c.slots[i] = sum <= most ? want[i] : want[i] ? std::max<int>(1, int64_t(most) * want[i] / sum) : 0;
    total += c.slots[i];
  }
  for (; total > most; --total) --*std::max_element(c.slots, c.slots + 3);
  c.rounds = 0;
  for (int i = 0; i < 3; ++i)
    if (c.slots[i]) c.rounds = std::max(c.rounds, (heads[i] + c.slots[i] - 1) / c.slots[i]);
  c.tile = int(std::max<int64_t>(1, std::min<int64_t>(most / std::max(1, total), tokens / (2 * sm_count))));
  c.threads = ((c.tile * total << c.lanes_log) + 31) / 32 * 32;
  return c;
}

// A thread's place: token `t` of the tile, lane u of the group for head `slot` and every
// `step`-th behind it, of `kind`. live: it has columns of a head; its first is c0 and, in
// kHalves, its second vector's c1 (rotates: c0 and c1 are pairs, otherwise c1 alone).
template <int kMode, int V>
struct Place {
  int t, u, kind, slot, step, c0, c1;
  bool live, rotates;
  __device__ __forceinline__ Place(const RotaryParams& p, const Cut& cut) {
    const int group = threadIdx.x >> cut.lanes_log, all = cut.slots[0] + cut.slots[1] + cut.slots[2];
    u = threadIdx.x & ((1 << cut.lanes_log) - 1);
    t = group / all;
    slot = group - t * all;
    kind = 0;
    if (slot >= cut.slots[0]) {
      slot -= cut.slots[0];
      kind = 1;
      if (slot >= cut.slots[1]) {
        slot -= cut.slots[1];
        kind = 2;
      }
    }
    step = cut.slots[kind];
    live = t < cut.tile && u < cut.lanes;
    const int half = p.rotary_dim >> 1;
    rotates = kMode != kHalves || u < half / V;
    c0 = live ? u * V : 0;
    c1 = kMode != kHalves ? c0 : rotates ? c0 + half : p.rotary_dim + (u - half / V) * V;
  }
};

// The sum over the 2^log lanes of a group.
__device__ __forceinline__ float group_sum(float v, int log) {
#pragma unroll
  for (int o = 0; o < 5; ++o)
    if (o < log) v += __shfl_xor_sync(0xffffffffu, v, 1 << o);
  return v;
}

__device__ __forceinline__ float pair_sum(uint64_t v) {
  float a, b;
  f2_unpack(v, a, b);
  return a + b;
}

__device__ __forceinline__ uint64_t swapped(uint64_t v) {
  float a, b;
  f2_unpack(v, a, b);
  return f2_pack(b, a);
}

// The partners of columns c and c + 1 (pairs (i, i + half)).
__device__ __forceinline__ int partner(int c, int half) {
  return c >= 2 * half ? c : c < half ? c + half : c - half;
}

__device__ __forceinline__ float weight_at(const NormRotaryParams& p, int kind, int c, bool half_type) {
  if (p.weight_f32) return static_cast<const float*>(p.weight[kind])[c];
  return half_type ? __half2float(static_cast<const __half*>(p.weight[kind])[c])
                   : __bfloat162float(static_cast<const __nv_bfloat16*>(p.weight[kind])[c]);
}

// A tile's angles in shared memory, by token: cosines, then sines with the sign that the first
// of a pair takes them with, each `angle_row` floats.
__host__ __device__ inline int angle_row(int rotary_dim) { return (rotary_dim / 2 + 3) / 4 * 4; }

// Those of a tile of tokens [first, first + here), formed as rotary_angle() does. inv_freq: the
// frequencies in shared memory, or p's own before these are there. kFast: sine and cosine of the
// reduced angle to 2^-21, of which 16-bit results see nothing; otherwise to two steps of float32.
template <bool kFast>
__device__ __forceinline__ void tile_angles(const RotaryParams& p, const double* inv_freq, int64_t first, int here, float* to) {
  const int half = p.rotary_dim >> 1, row = angle_row(p.rotary_dim);
  for (int i = threadIdx.x; i < here * half; i += blockDim.x) {
    const int tt = i / half, f = i - tt * half;
    double t = rotary_position(p, first + tt) * inv_freq[f] * 0.15915494309189535;  // 1 / (2 pi)
    t -= rint(t);
    float s, c;
    if constexpr (kFast) {
      const float radians = float(t) * 6.283185307179586f;
      s = __sinf(radians);
      c = __cosf(radians);
    } else {
      sincospif(float(2.0 * t), &s, &c);
    }
    to[2 * tt * row + f] = c * p.magnitude;
    to[(2 * tt + 1) * row + f] = -s * p.magnitude * p.sign;
  }
}

// out = own * co + partner * si for columns c0.. of a token whose angles are `cs`. (kHalves: of
// the first half's columns, or of none.)
template <int kMode, int kPairs>
__device__ __forceinline__ void column_angles(const RotaryParams& p, const float* cs, int c0,
                                              uint64_t (&co)[kPairs], uint64_t (&si)[kPairs]) {
  const int half = p.rotary_dim >> 1;
  const float* const sn = cs + angle_row(p.rotary_dim);
  if constexpr (kMode == kHalves) {
#pragma unroll
    for (int k = 0; k < kPairs; ++k) {
      co[k] = f2_pack(1.f, 1.f);
      si[k] = 0;
    }
    if (c0 < p.rotary_dim) {
#pragma unroll
      for (int k = 0; k < kPairs; k += 2) {
        const ulonglong2 u = *reinterpret_cast<const ulonglong2*>(cs + c0 + 2 * k);
        const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(sn + c0 + 2 * k);
        co[k] = u.x;
        co[k + 1] = u.y;
        si[k] = v.x;
        si[k + 1] = v.y;
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < kPairs; ++k) {
      const int c = c0 + 2 * k;
      co[k] = f2_pack(1.f, 1.f);
      si[k] = 0;
      if (c >= p.rotary_dim) continue;
      if (kMode == kNeighbours) {
        const float u = cs[c >> 1], v = sn[c >> 1];
        co[k] = f2_pack(u, u);
        si[k] = f2_pack(v, -v);
      } else {
        const bool second = c >= half, next = c + 1 >= half;
        const int i = second ? c - half : c, j = next ? c + 1 - half : c + 1;
        co[k] = f2_pack(cs[i], cs[j]);
        si[k] = f2_pack(second ? -sn[i] : sn[i], next ? -sn[j] : sn[j]);
      }
    }
  }
}

// Where a new token's keys and values go, in elements; < 0: nowhere. Called by a whole warp.
struct AppendPlace {
  int64_t k, v;
};
__device__ __forceinline__ AppendPlace append_place(const CacheAppendParams& p, int t, int lane) {
  AppendPlace none{-1, -1};
  if (t < __ldg(p.cu) || t >= __ldg(p.cu + p.seqs)) return none;
  int slot, q0, n, len;
  if (!row_grew(p.c, p.slots, p.cu, p.seqs, t, lane, slot, q0, n, len)) return none;
  const int pos = len - n + t - q0;
  if (pos < 0 || pos >= int64_t(p.c.width) * p.c.page) return none;
  const int page = p.c.table[int64_t(slot) * p.c.width + pos / p.c.page];
  if (page < 0 || page >= p.c.pages) {
    if (lane == 0) record_error(p.c.status, kErrBadArgument, 67, 0);
    return none;
  }
  const int row = pos % p.c.page;
  return {page * p.k_stride[0] + row * p.k_stride[1], page * p.v_stride[0] + row * p.v_stride[1]};
}

__device__ __forceinline__ void copy16(uint4* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// All but the last n copies' groups have arrived (the thread's own).
template <int n>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(n) : "memory"); }

// What a thread works on in turn: units of kUnit heads of one token, of which it has two in its
// ring: while it works on one, it copies the next but one, head for head, into the place of
// what it has read. Unit (tile j, pass i) of the CTA is heads slot + (i * kUnit + r) * step of
// token t of its tile j. Of each head kIn times (kHalves: 2) 16 bytes; a head's lanes lie side
// by side in shared memory.
template <class E, int kMode, int kIn, int kUnit>
struct Units {
  static constexpr int kPer = kMode == kHalves ? 2 : 1, kVecs = kIn * kPer, kRing = 2 * kUnit;
  const RotaryParams& p;
  const Cut& cut;
  const Place<kMode, 16 / sizeof(E)>& at;
  const int64_t all;  // tokens
  int64_t tiles;      // of this CTA
  int passes;
  uint4* mine;
  // the unit to copy into next, and its first head's rows
  int64_t j = 0;
  int pass = 0, heads_left = 0;
  const E* row[kIn];
  int64_t row_step[kIn];

  __device__ __forceinline__ Units(const RotaryParams& params, const Cut& c, const Place<kMode, 16 / sizeof(E)>& place,
                                   const RotaryTensor (&in)[kIn], uint4* ring)
      : p(params), cut(c), at(place), all(params.batch * params.tokens), mine(ring + threadIdx.x) {
    const int64_t n = (all + cut.tile - 1) / cut.tile;
    tiles = n > blockIdx.x ? (n - blockIdx.x + gridDim.x - 1) / gridDim.x : 0;
    passes = (cut.rounds + kUnit - 1) / kUnit;
#pragma unroll
    for (int i = 0; i < kIn; ++i) row_step[i] = at.step * in[i].stride_h;
    for (int k = 0; k < 2; ++k) {
      begin(in);
#pragma unroll
      for (int r = 0; r < kUnit; ++r) copy(k, r);
    }
  }
  __device__ __forceinline__ int64_t first(int64_t tile) const { return (blockIdx.x + tile * gridDim.x) * cut.tile; }
  // Before a unit's copies.
  __device__ __forceinline__ void begin(const RotaryTensor (&in)[kIn]) {
    if (pass == 0) {
      const int64_t token = first(j) + at.t;
      heads_left = at.live && j < tiles && token < all ? in[0].heads - at.slot : 0;
      if (heads_left > 0) {
        const int64_t b = p.batch == 1 ? 0 : token / p.tokens, l = token - b * p.tokens;
#pragma unroll
        for (int i = 0; i < kIn; ++i)
          row[i] = static_cast<const E*>(in[i].in) + b * in[i].stride_b + l * in[i].stride_t + at.slot * in[i].stride_h;
      }
    }
    if (++pass == passes) {
      pass = 0;
      ++j;
    }
  }
  // Head r of the unit, into half k of the ring.
  __device__ __forceinline__ void copy(int k, int r) {
    if (heads_left > 0) {
      uint4* to = mine + (k * kUnit + r) * kVecs * kThreads;
#pragma unroll
      for (int i = 0; i < kIn; ++i) {
        if (at.rotates) copy16(to + i * kPer * kThreads, row[i] + at.c0);
        if constexpr (kMode == kHalves) copy16(to + (i * kPer + 1) * kThreads, row[i] + at.c1);
        row[i] += row_step[i];
      }
    }
    heads_left -= at.step;
    copies_commit();
  }
  // The oldest head has arrived. (kAny reads its neighbours' columns.)
  __device__ __forceinline__ void arrived() const {
    copies_wait<kRing - 1>();
    if constexpr (kMode == kAny) __syncwarp();
  }
  __device__ __forceinline__ uint4 get(int k, int r, int v) const { return mine[((k * kUnit + r) * kVecs + v) * kThreads]; }
  // Column c of the head, of input i (kAny).
  __device__ __forceinline__ float element(int k, int r, int i, int c) const {
    return to_f(reinterpret_cast<const E*>(mine + ((k * kUnit + r) * kVecs + i * kPer) * kThreads - at.u)[c]);
  }
};

// kNorm: with the norm. P: NormRotaryParams, or CacheAppendParams to write into a cache.
template <class E, int kMode, bool kNorm, class P>
__global__ void __launch_bounds__(kThreads, 2) norm_rotary_kernel(const P p, const Cut cut) {
  constexpr bool kAppend = std::is_same_v<P, CacheAppendParams>;
  constexpr int V = 16 / sizeof(E), kPairs = V / 2, kTwo = kMode == kHalves ? kPairs : 1;
  using Pair = PairOf<E>;
  using U = Units<E, kMode, 1, kFwdUnit>;
  union Vec {
    uint4 v;
    typename Pair::Raw w[kPairs];
  };
  // inv_freq; twice a tile's (append) places and angles; the ring
  extern __shared__ uint4 shared[];
  const int half = p.rotary_dim >> 1, angles = 2 * cut.tile * angle_row(p.rotary_dim);
  double* const freqs = reinterpret_cast<double*>(shared);
  AppendPlace* const places = reinterpret_cast<AppendPlace*>(freqs + (half + 1) / 2 * 2);
  float* const cs = reinterpret_cast<float*>(places + (kAppend ? 2 * cut.tile : 0));
  const Place<kMode, V> at(p, cut);
  RotaryTensor x[1] = {p.x[at.kind & 1]};
  if constexpr (kAppend)
    if (at.kind == 2) x[0] = p.v;
  U units(p, cut, at, x, reinterpret_cast<uint4*>(cs + 2 * angles));

  // angles and places of the CTA's tile j
  auto prepare = [&](int64_t j) {
    const int64_t first = units.first(j);
    const int here = int(units.all - first < cut.tile ? units.all - first : cut.tile);
    if constexpr (kAppend) {
      for (int i = threadIdx.x >> 5; i < here; i += blockDim.x >> 5) {
        const AppendPlace to = append_place(p, int(first) + i, threadIdx.x & 31);
        if ((threadIdx.x & 31) == 0) places[(j & 1) * cut.tile + i] = to;
      }
    }
    // (the positions alone as apply_rotary does them, to the bit)
    tile_angles<kNorm && sizeof(E) == 2>(p, j ? freqs : p.inv_freq, first, here, cs + (j & 1) * angles);
  };
  if (units.tiles > 0) prepare(0);
  if (units.tiles > 1)
    for (int i = threadIdx.x; i < half; i += blockDim.x) freqs[i] = p.inv_freq[i];
  uint64_t w0[kPairs], w1[kTwo], wo[kMode == kAny ? kPairs : 1];
  if constexpr (kNorm) {
    constexpr bool kHalfType = std::is_same_v<E, __half>;
    auto weights = [&](int c, int d) {
      return at.live && at.kind < 2 ? f2_pack(weight_at(p, at.kind, c, kHalfType), weight_at(p, at.kind, d, kHalfType))
                                    : uint64_t(0);
    };
#pragma unroll
    for (int k = 0; k < kPairs; ++k) {
      const int c = at.c0 + 2 * k;
      w0[k] = weights(c, c + 1);
      if constexpr (kMode == kHalves) w1[k] = weights(at.c1 + 2 * k, at.c1 + 2 * k + 1);
      if constexpr (kMode == kAny) wo[k] = weights(partner(c, half), partner(c + 1, half));
    }
  }
  const bool rotated = !kAppend || at.kind < 2;
  const float inv = 1.f / float(p.head_dim);
  int k = 0;  // half of the ring
  for (int64_t j = 0; j < units.tiles; ++j) {
    __syncthreads();  // the tile's angles are there, and those of the tile before have been read
    if (j + 1 < units.tiles) prepare(j + 1);
    const int64_t token = units.first(j) + at.t;
    int left = at.live && token < units.all ? x[0].heads - at.slot : 0;  // heads from this one on
    E* out = nullptr;
    int64_t out_h = p.head_dim;
    uint64_t co[kPairs], si[kPairs];
    if (left > 0) {
      if (!kAppend || at.kind == 0) out = static_cast<E*>(x[0].out) + token * x[0].heads * p.head_dim;
      if constexpr (kAppend) {
        const AppendPlace to = places[(j & 1) * cut.tile + at.t];
        if (at.kind == 1 && to.k >= 0) out = static_cast<E*>(p.k_pool) + to.k;
        if (at.kind == 2 && to.v >= 0) out = static_cast<E*>(p.v_pool) + to.v;
        if (at.kind) out_h = at.kind == 1 ? p.k_stride[2] : p.v_stride[2];
      }
      column_angles<kMode>(p, cs + (j & 1) * angles + 2 * at.t * angle_row(p.rotary_dim),
                           kMode == kHalves && !at.rotates ? p.rotary_dim : at.c0, co, si);
    }
    E* row = out + at.slot * out_h;
    for (int i = 0; i < units.passes; ++i, k ^= 1) {
      units.begin(x);
#pragma unroll
      for (int r = 0; r < kFwdUnit; ++r) {
        units.arrived();
        if (i * kFwdUnit + r < cut.rounds) {
          Vec x0, x1;
          x0.v = x1.v = make_uint4(0, 0, 0, 0);
          if (left > 0) {
            if (at.rotates) x0.v = units.get(k, r, 0);
            if constexpr (kMode == kHalves) x1.v = units.get(k, r, 1);
          }
          uint64_t a[kPairs], d[kPairs];
#pragma unroll
          for (int n = 0; n < kPairs; ++n) {
            a[n] = Pair::wide(x0.w[n]);
            if constexpr (kMode == kHalves) d[n] = Pair::wide(x1.w[n]);
            if constexpr (kMode == kNeighbours) d[n] = swapped(a[n]);
            if constexpr (kMode == kAny) {
              const int c = at.c0 + 2 * n;
              d[n] = left > 0 ? f2_pack(units.element(k, r, 0, partner(c, half)), units.element(k, r, 0, partner(c + 1, half))) : 0;
            }
          }
          uint64_t scale = 0;
          if constexpr (kNorm) {
            uint64_t sq = 0;
#pragma unroll
            for (int n = 0; n < kPairs; ++n) {
              sq = f2_fma(a[n], a[n], sq);
              if constexpr (kMode == kHalves) sq = f2_fma(d[n], d[n], sq);
            }
            const float rstd = rsqrtf(group_sum(pair_sum(sq), cut.lanes_log) * inv + p.eps);
            scale = f2_pack(rstd, rstd);
          }
          if (left > 0 && out) {
            if (rotated) {
#pragma unroll
              for (int n = 0; n < kPairs; ++n) {
                if constexpr (kNorm) {
                  a[n] = f2_mul(f2_mul(a[n], scale), w0[n]);
                  d[n] = f2_mul(f2_mul(d[n], scale), kMode == kHalves ? w1[kMode == kHalves ? n : 0]
                                                     : kMode == kAny  ? wo[kMode == kAny ? n : 0]
                                                                      : swapped(w0[n]));
                }
                // without the norm the columns behind rotary_dim are copies, bit for bit
                if (kNorm || (kMode == kHalves ? at.rotates : at.c0 + 2 * n < p.rotary_dim))
                  x0.w[n] = Pair::narrow(f2_fma(a[n], co[n], f2_mul(d[n], si[n])));
                if constexpr (kMode == kHalves)
                  if (kNorm || at.rotates)
                    x1.w[n] = Pair::narrow(at.rotates ? f2_sub(f2_mul(d[n], co[n]), f2_mul(a[n], si[n])) : d[n]);
              }
            }
            if (at.rotates) *reinterpret_cast<uint4*>(row + at.c0) = x0.v;
            if constexpr (kMode == kHalves) *reinterpret_cast<uint4*>(row + at.c1) = x1.v;
          }
          left -= at.step;
          row += at.step * out_h;
        }
        if constexpr (kMode == kAny) __syncwarp();
        units.copy(k, r);
      }
    }
  }
  copies_wait<0>();
}

// Gradients. Each thread keeps its columns' share of the weights' gradients in registers; the
// shares are added in the groups' order.
template <class E, int kMode>
__global__ void __launch_bounds__(kThreads, 2) norm_rotary_bwd_kernel(const NormRotaryParams p, const Cut cut) {
  constexpr int V = 16 / sizeof(E), kPairs = V / 2, kTwo = kMode == kHalves ? kPairs : 1;
  using Pair = PairOf<E>;
  using U = Units<E, kMode, 2, kBwdUnit>;
  union Vec {
    uint4 v;
    typename Pair::Raw w[kPairs];
  };
  // inv_freq, twice a tile's angles, the ring; at the end the weights' gradients
  extern __shared__ uint4 shared[];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int half = p.rotary_dim >> 1, angles = 2 * cut.tile * angle_row(p.rotary_dim);
  double* const freqs = reinterpret_cast<double*>(shared);
  float* const cs = reinterpret_cast<float*>(freqs + (half + 1) / 2 * 2);
  const Place<kMode, V> at(p, cut);
  const RotaryTensor in[2] = {p.x[at.kind], p.dy[at.kind]};
  U units(p, cut, at, in, reinterpret_cast<uint4*>(cs + 2 * angles));
  auto prepare = [&](int64_t j) {
    const int64_t first = units.first(j);
    const int here = int(units.all - first < cut.tile ? units.all - first : cut.tile);
    tile_angles<sizeof(E) == 2>(p, j ? freqs : p.inv_freq, first, here, cs + (j & 1) * angles);
  };
  if (units.tiles > 0) prepare(0);
  if (units.tiles > 1)
    for (int i = threadIdx.x; i < half; i += blockDim.x) freqs[i] = p.inv_freq[i];
  constexpr bool kHalfType = std::is_same_v<E, __half>;
  uint64_t w0[kPairs], w1[kTwo], acc0[kPairs], acc1[kTwo];
#pragma unroll
  for (int n = 0; n < kPairs; ++n) {
    acc0[n] = w0[n] = 0;
    if (at.live)
      w0[n] = f2_pack(weight_at(p, at.kind, at.c0 + 2 * n, kHalfType), weight_at(p, at.kind, at.c0 + 2 * n + 1, kHalfType));
    if constexpr (kMode == kHalves) {
      acc1[n] = w1[n] = 0;
      if (at.live)
        w1[n] = f2_pack(weight_at(p, at.kind, at.c1 + 2 * n, kHalfType), weight_at(p, at.kind, at.c1 + 2 * n + 1, kHalfType));
    }
  }
  const float inv = 1.f / float(p.head_dim);
  int k = 0;  // half of the ring
  for (int64_t j = 0; j < units.tiles; ++j) {
    __syncthreads();  // the tile's angles are there, and those of the tile before have been read
    if (j + 1 < units.tiles) prepare(j + 1);
    const int64_t token = units.first(j) + at.t;
    int left = at.live && token < units.all ? in[0].heads - at.slot : 0;  // heads from this one on
    E* row = static_cast<E*>(in[0].out) + (token * in[0].heads + at.slot) * p.head_dim;
    uint64_t co[kPairs], si[kPairs];
    // (lanes without columns have to add nothing to their group's sums, whatever lies there)
    column_angles<kMode>(p, cs + (j & 1) * angles + 2 * (left > 0 ? at.t : 0) * angle_row(p.rotary_dim),
                         left > 0 && (kMode != kHalves || at.rotates) ? at.c0 : p.rotary_dim, co, si);
    for (int i = 0; i < units.passes; ++i, k ^= 1) {
      units.begin(in);
#pragma unroll
      for (int r = 0; r < kBwdUnit; ++r) {
        units.arrived();
        if (i * kBwdUnit + r >= cut.rounds) {
          units.copy(k, r);
          continue;
        }
        Vec x0, x1, y0, y1;
        x0.v = x1.v = y0.v = y1.v = make_uint4(0, 0, 0, 0);
        if (left > 0) {
          if (at.rotates) {
            x0.v = units.get(k, r, 0);
            y0.v = units.get(k, r, U::kPer);
          }
          if constexpr (kMode == kHalves) {
            x1.v = units.get(k, r, 1);
            y1.v = units.get(k, r, 3);
          }
        }
        uint64_t g0[kPairs], g1[kTwo], sq = 0, dot = 0;
#pragma unroll
        for (int n = 0; n < kPairs; ++n) {
          const uint64_t e = Pair::wide(y0.w[n]), a = Pair::wide(x0.w[n]);
          uint64_t f = 0;
          if constexpr (kMode == kHalves) f = Pair::wide(y1.w[n]);
          if constexpr (kMode == kNeighbours) f = swapped(e);
          if constexpr (kMode == kAny) {
            const int c = at.c0 + 2 * n;
            if (left > 0) f = f2_pack(units.element(k, r, 1, partner(c, half)), units.element(k, r, 1, partner(c + 1, half)));
          }
          g0[n] = f2_fma(e, co[n], f2_mul(f, si[n]));
          sq = f2_fma(a, a, sq);
          dot = f2_fma(f2_mul(g0[n], w0[n]), a, dot);
          if constexpr (kMode == kHalves) {
            const uint64_t d = Pair::wide(x1.w[n]);
            g1[n] = f2_sub(f2_mul(f, co[n]), f2_mul(e, si[n]));
            sq = f2_fma(d, d, sq);
            dot = f2_fma(f2_mul(g1[n], w1[n]), d, dot);
          }
        }
        if constexpr (kMode == kAny) __syncwarp();
        units.copy(k, r);
        // (groups without a head have the sums of nothing)
        float both[2] = {pair_sum(sq), pair_sum(dot)};
#pragma unroll
        for (int o = 0; o < 5; ++o)
          if (o < cut.lanes_log) {
            both[0] += __shfl_xor_sync(0xffffffffu, both[0], 1 << o);
            both[1] += __shfl_xor_sync(0xffffffffu, both[1], 1 << o);
          }
        const float rstd = rsqrtf(both[0] * inv + p.eps), along = both[1] * inv * rstd * rstd;
        if (left > 0) {
          const uint64_t scale = f2_pack(rstd, rstd), minus = f2_pack(-along, -along);
#pragma unroll
          for (int n = 0; n < kPairs; ++n) {
            const uint64_t a = Pair::wide(x0.w[n]);
            acc0[n] = f2_fma(g0[n], f2_mul(a, scale), acc0[n]);
            x0.w[n] = Pair::narrow(f2_mul(scale, f2_fma(g0[n], w0[n], f2_mul(a, minus))));
            if constexpr (kMode == kHalves) {
              const uint64_t d = Pair::wide(x1.w[n]);
              acc1[n] = f2_fma(g1[n], f2_mul(d, scale), acc1[n]);
              x1.w[n] = Pair::narrow(f2_mul(scale, f2_fma(g1[n], w1[n], f2_mul(d, minus))));
            }
          }
          if (at.rotates) *reinterpret_cast<uint4*>(row + at.c0) = x0.v;
          if constexpr (kMode == kHalves) *reinterpret_cast<uint4*>(row + at.c1) = x1.v;
        }
        left -= at.step;
        row += at.step * p.head_dim;
      }
    }
  }
  copies_wait<0>();
  if (!p.dw_part) return;
  // [group][head_dim]
  float* const sums = reinterpret_cast<float*>(shared);
  __syncthreads();
  if (at.live) {
    float* mine = sums + (threadIdx.x >> cut.lanes_log) * p.head_dim;
#pragma unroll
    for (int k = 0; k < kPairs; ++k) {
      if (at.rotates) f2_unpack(acc0[k], mine[at.c0 + 2 * k], mine[at.c0 + 2 * k + 1]);
      if constexpr (kMode == kHalves) f2_unpack(acc1[k], mine[at.c1 + 2 * k], mine[at.c1 + 2 * k + 1]);
    }
  }
  __syncthreads();
  const int step = cut.slots[0] + cut.slots[1];
  for (int i = threadIdx.x; i < 2 * p.head_dim; i += blockDim.x) {
    const int kind = i / p.head_dim, c = i - kind * p.head_dim;
    float sum = 0.f;
    for (int t = 0; t < cut.tile; ++t)
      for (int j = 0; j < cut.slots[kind]; ++j)
        sum += sums[(t * step + (kind ? cut.slots[0] : 0) + j) * p.head_dim + c];
    p.dw_part[int64_t(blockIdx.x) * 2 * p.head_dim + i] = sum;
  }
}

// Heads that start or end off a 16-byte boundary, or need more than 32 lanes: a warp a head,
// its columns lane by lane, a CTA a token (back: every gridDim.x-th). head_dim is at most 256.
// Bound by its single loads and angles: 8192 tokens of 32 + 8 heads of 100 in bf16 take 272 us
// forward and 361 us back (0.5 TB/s), of 162 in fp32 453 and 480 us.
constexpr int kPerLane = 8;

template <class E, bool kBack>
__global__ void __launch_bounds__(kThreads) norm_rotary_element_kernel(const NormRotaryParams p) {
  extern __shared__ float2 cs[];  // [rotary_dim / 2]; at the end the weights' gradients
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  constexpr int kWarps = kThreads / 32;
  constexpr bool kHalfType = std::is_same_v<E, __half>;
  const int half = p.rotary_dim >> 1, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float inv = 1.f / float(p.head_dim);
  float acc[kBack ? 2 : 1][kPerLane] = {};
  for (int64_t token = blockIdx.x; token < p.batch * p.tokens; token += gridDim.x) {
    const int64_t b = token / p.tokens, l = token - b * p.tokens;
    __syncthreads();
    for (int i = threadIdx.x; i < half; i += kThreads) cs[i] = rotary_angle(p, token, i);
    __syncthreads();
#pragma unroll
    for (int kind = 0; kind < 2; ++kind) {
      const RotaryTensor& x = p.x[kind];
      const RotaryTensor& y = p.dy[kind];
      for (int h = warp; h < x.heads; h += kWarps) {
        const E* row = static_cast<const E*>(x.in) + b * x.stride_b + l * x.stride_t + h * x.stride_h;
        const E* back = kBack ? static_cast<const E*>(y.in) + b * y.stride_b + l * y.stride_t + h * y.stride_h : row;
        E* out = static_cast<E*>(x.out) + (token * x.heads + h) * p.head_dim;
        float sq = 0.f, dot = 0.f, v[kPerLane], g[kPerLane], w[kPerLane];
#pragma unroll
        for (int k = 0; k < kPerLane; ++k) {
          const int c = lane + 32 * k;
          v[k] = g[k] = w[k] = 0.f;
          if (c >= p.head_dim) continue;
          v[k] = to_f(row[c]);
          w[k] = weight_at(p, kind, c, kHalfType);
          sq += v[k] * v[k];
          // the rotation's own and partner's terms: of the weighted inputs, or of dy
          const bool turns = c < p.rotary_dim, second = p.interleaved ? c & 1 : c >= half;
          const int pair = p.interleaved ? c >> 1 : second ? c - half : c;
          const int o = p.interleaved ? c ^ 1 : second ? c - half : c + half;
          g[k] = kBack ? to_f(back[c]) : v[k] * w[k];
          if (turns) {
            const float2 f = cs[pair];
            const float other = to_f(back[o]) * (kBack ? 1.f : weight_at(p, kind, o, kHalfType));
            g[k] = g[k] * f.x + other * (second ? f.y : -f.y);
          }
          if (kBack) dot += g[k] * w[k] * v[k];
        }
        const float rstd = rsqrtf(group_sum(sq, 5) * inv + p.eps);
        const float along = kBack ? group_sum(dot, 5) * inv * rstd * rstd : 0.f;
#pragma unroll
        for (int k = 0; k < kPerLane; ++k) {
          const int c = lane + 32 * k;
          if (c >= p.head_dim) continue;
          if (kBack) acc[kBack ? kind : 0][k] += g[k] * (v[k] * rstd);
          out[c] = from_f<E>(kBack ? rstd * (g[k] * w[k] - v[k] * along) : rstd * g[k]);
        }
      }
    }
  }
  if constexpr (kBack) {
    if (!p.dw_part) return;
    float* const sums = reinterpret_cast<float*>(cs);  // [warp][2][head_dim]
    __syncthreads();
#pragma unroll
    for (int kind = 0; kind < 2; ++kind)
#pragma unroll
      for (int k = 0; k < kPerLane; ++k)
        if (lane + 32 * k < p.head_dim) sums[(warp * 2 + kind) * p.head_dim + lane + 32 * k] = acc[kind][k];
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * p.head_dim; i += kThreads) {
      float sum = 0.f;
      for (int j = 0; j < kWarps; ++j) sum += sums[j * 2 * p.head_dim + i];
      p.dw_part[int64_t(blockIdx.x) * 2 * p.head_dim + i] = sum;
    }
  }
}

// dw from the CTAs' parts, in an order that `parts` alone decides: warp j of a CTA adds
// parts j, j + kDwWarps, ... of 32 columns, then the warps' sums are added.
constexpr int kDwWarps = 16;
template <class E>
__global__ void __launch_bounds__(kDwWarps * 32) norm_rotary_dw_kernel(const NormRotaryParams p, int parts) {
  __shared__ float sums[kDwWarps][32];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, i = blockIdx.x * 32 + lane;
  const int columns = 2 * p.head_dim;
  float sum = 0.f;
  if (i < columns) {
#pragma unroll 8
    for (int j = warp; j < parts; j += kDwWarps) sum += p.dw_part[int64_t(j) * columns + i];
  }
  sums[warp][lane] = sum;
  __syncthreads();
  if (warp || i >= columns) return;
  sum = 0.f;
#pragma unroll
  for (int j = 0; j < kDwWarps; ++j) sum += sums[j][lane];
  const int kind = i / p.head_dim, c = i - kind * p.head_dim;
  if (!p.dw[kind]) return;
  if (p.weight_f32) static_cast<float*>(p.dw[kind])[c] = sum;
  else static_cast<E*>(p.dw[kind])[c] = from_f<E>(sum);
}

// The widest accesses that the pairs' layout and (p.vec) the strides allow; < 0: by elements.
template <class E>
int mode_of(const RotaryParams& p) {
  constexpr int V = 16 / sizeof(E);
  if (!p.vec) return -1;
  const int pairs = p.rotary_dim / 2;
  const int mode = p.interleaved ? kNeighbours
                   : pairs % V == 0 && (p.head_dim - p.rotary_dim) % V == 0 ? kHalves : kAny;
  return lanes_of(mode, V, p.head_dim, p.rotary_dim) <= 32 ? mode : -1;
}

void cuda_ok(cudaError_t e) {
  if (e != cudaSuccess) throw std::runtime_error(std::string("norm and rotary positions: ") + cudaGetErrorString(e));
}

// Bytes of the frequencies and of two tiles' angles in shared memory.
size_t freqs_and_angles(const RotaryParams& p, const Cut& cut) {
  return size_t(p.rotary_dim / 2 + 1) / 2 * 2 * sizeof(double) + 4 * size_t(cut.tile) * angle_row(p.rotary_dim) * sizeof(float);
}

// The CTAs of a launch: as many as run at once.
template <auto fn, class P>
void launch_tiles(const P& p, const Cut& cut, int64_t tokens, int ctas, size_t smem, cudaStream_t s) {
  static std::atomic<uint64_t> allowed{0};  // (of this kernel)
  cuda_ok(paged_allow_smem(fn, allowed));
  fn<<<unsigned(std::min<int64_t>((tokens + cut.tile - 1) / cut.tile, ctas)), cut.threads, smem, s>>>(p, cut);
  cuda_ok(cudaGetLastError());
}

template <class E, int kMode, bool kNorm, class P>
void fwd_mode(const P& p, int sm_count, cudaStream_t s) {
  constexpr int V = 16 / sizeof(E);
  constexpr bool kAppend = std::is_same_v<P, CacheAppendParams>;
  int heads[3] = {p.x[0].heads, p.x[1].heads, 0};
  if constexpr (kAppend) heads[2] = p.v.heads;
  const int64_t all = p.batch * p.tokens;
  const Cut cut = make_cut(lanes_of(kMode, V, p.head_dim, p.rotary_dim), heads, all, sm_count);
  using U = Units<E, kMode, 1, kFwdUnit>;
  const size_t smem = freqs_and_angles(p, cut) + sizeof(uint4) * U::kRing * U::kVecs * kThreads +
                      (kAppend ? 2 * cut.tile * sizeof(AppendPlace) : 0);
  launch_tiles<norm_rotary_kernel<E, kMode, kNorm, P>>(p, cut, all, 2 * sm_count, smem, s);
}

template <class E, bool kNorm, class P>
void fwd_e(const P& p, int sm_count, cudaStream_t s) {
  switch (mode_of<E>(p)) {
    case kHalves: return fwd_mode<E, kHalves, kNorm>(p, sm_count, s);
    case kNeighbours: return fwd_mode<E, kNeighbours, kNorm>(p, sm_count, s);
    case kAny: return fwd_mode<E, kAny, kNorm>(p, sm_count, s);
    default: break;
  }
  if constexpr (!std::is_same_v<P, CacheAppendParams>)
    norm_rotary_element_kernel<E, false>
        <<<unsigned(p.batch * p.tokens), kThreads, (p.rotary_dim / 2) * sizeof(float2), s>>>(p);
}

template <class E>
Cut bwd_cut(const NormRotaryParams& p, int mode, int sm_count) {
  return make_cut(lanes_of(mode, 16 / sizeof(E), p.head_dim, p.rotary_dim),
                  {p.x[0].heads, p.x[1].heads, 0}, p.batch * p.tokens, sm_count);
}

// Two CTAs an SM, each with every parts-th tile.
template <class E>
int bwd_parts(const NormRotaryParams& p, int sm_count) {
  const int mode = mode_of<E>(p);
  const int64_t tiles = mode < 0 ? p.batch * p.tokens
                                 : (p.batch * p.tokens + bwd_cut<E>(p, mode, sm_count).tile - 1) / bwd_cut<E>(p, mode, sm_count).tile;
  return int(std::min<int64_t>(tiles, 2 * sm_count));
}

template <class E, int kMode>
void bwd_mode(const NormRotaryParams& p, int parts, int sm_count, cudaStream_t s) {
  const Cut cut = bwd_cut<E>(p, kMode, sm_count);
  using U = Units<E, kMode, 2, kBwdUnit>;
  const size_t ring = freqs_and_angles(p, cut) + sizeof(uint4) * U::kRing * U::kVecs * kThreads;
  const size_t sums = p.dw_part ? size_t(cut.threads >> cut.lanes_log) * p.head_dim * sizeof(float) : 0;
  launch_tiles<norm_rotary_bwd_kernel<E, kMode>>(p, cut, p.batch * p.tokens, parts, std::max(ring, sums), s);
}

template <class E>
void bwd_e(const NormRotaryParams& p, int parts, int sm_count, cudaStream_t s) {
  switch (mode_of<E>(p)) {
    case kHalves: bwd_mode<E, kHalves>(p, parts, sm_count, s); break;
    case kNeighbours: bwd_mode<E, kNeighbours>(p, parts, sm_count, s); break;
    case kAny: bwd_mode<E, kAny>(p, parts, sm_count, s); break;
    default:
      norm_rotary_element_kernel<E, true>
          <<<parts, kThreads, std::max(p.rotary_dim / 2 * sizeof(float2), 2 * kThreads / 32 * p.head_dim * sizeof(float)), s>>>(p);
  }
  if (!p.dw_part) return;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((2 * p.head_dim + 31) / 32);
  cfg.blockDim = dim3(kDwWarps * 32);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cuda_ok(cudaLaunchKernelEx(&cfg, norm_rotary_dw_kernel<E>, p, parts));
}

}  // namespace

void norm_rotary_launch(RotaryType t, const NormRotaryParams& p, int sm_count, cudaStream_t s) {
  switch (t) {
    case RotaryType::kBf16: return fwd_e<__nv_bfloat16, true>(p, sm_count, s);
    case RotaryType::kF16: return fwd_e<__half, true>(p, sm_count, s);
    default: return fwd_e<float, true>(p, sm_count, s);
  }
}

int norm_rotary_bwd_parts(RotaryType t, const NormRotaryParams& p, int sm_count) {
  return t == RotaryType::kF32 ? bwd_parts<float>(p, sm_count) : bwd_parts<__half>(p, sm_count);
}

void norm_rotary_bwd_launch(RotaryType t, const NormRotaryParams& p, int parts, int sm_count, cudaStream_t s) {
  switch (t) {
    case RotaryType::kBf16: return bwd_e<__nv_bfloat16>(p, parts, sm_count, s);
    case RotaryType::kF16: return bwd_e<__half>(p, parts, sm_count, s);
    default: return bwd_e<float>(p, parts, sm_count, s);
  }
}

void cache_append_launch(RotaryType t, const CacheAppendParams& p, int sm_count, cudaStream_t s) {
  if (t == RotaryType::kBf16)
    p.norm ? fwd_e<__nv_bfloat16, true>(p, sm_count, s) : fwd_e<__nv_bfloat16, false>(p, sm_count, s);
  else
    p.norm ? fwd_e<__half, true>(p, sm_count, s) : fwd_e<__half, false>(p, sm_count, s);
}

}  // namespace mgfa
