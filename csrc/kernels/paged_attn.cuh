// Attention of new tokens over a paged cache: parameters, the division of the work
// that the kernels share, and their launch functions.
//
// Sequence b has n_b new tokens (rows [cu_q[b], cu_q[b + 1]) of q), which are the last
// of its kv_b tokens; token i sees keys [0, kv_b - n_b + i] (causal) or all of them.
// The `group` query heads of a key head share its keys, so a unit of work packs them:
// row r of (b, key head) is token r / group, head r % group.
//
// Division of the work. A unit (b, key head, block of tokens) reads a run of key
// tiles; all units' runs, laid end to end, are cut into equal shares, one per CTA,
// whatever the sequences' lengths. A share covers whole units, which the CTA finishes,
// and at most two parts (its first and last), which it leaves, unnormalised in fp32, in
// a workspace for paged_merge_kernel. A cut that would leave `snap` tiles or fewer of a
// unit on one side moves to the unit's border: a part's way through the workspace costs
// more than that (`snap` is at most half a share). The shares follow from the lengths alone, which the kernel reads on
// the device: the host knows none of them, nothing waits for it, and the result does not
// depend on timing. Where the host can see that every unit is short, they are dealt out
// whole instead, which needs neither the lengths' sum nor a join.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <type_traits>

#ifdef __CUDACC__
#include "sm100_ptx.cuh"
#endif

namespace mgfa {

constexpr int kPagedMaxSeqs = 4096;
constexpr int kPagedMaxGroup = 128;
constexpr size_t kPagedMaxSmem = 232448;  // shared memory of a CTA (227 KB)

// Forms of the decode kernel that a launch may ask for; otherwise the rows of a unit decide.
enum : int {
  kPagedByRows = 0,
  kPagedHeadsApart = 1,  // units of four key heads, up to 16 rows each
  kPagedRowsApart = 2,   // units of up to 32 rows, which eight warps share
};

// Shared memory of a kernel that needs `used` bytes from a 1024-byte boundary on, and behind
// them prefix[] of `seqs` sequences (with the number of CTAs, PagedShare).
constexpr size_t paged_smem(size_t used, int seqs) { return 1024 + used + 4 * (size_t(seqs) + 2); }

struct PagedParams {
  // problem
  const void* q = nullptr;      // [tokens, heads, head_dim], strides in elements
  int64_t q_stride_t = 0, q_stride_h = 0;
  void* out = nullptr;          // q's type
  int64_t o_stride_t = 0, o_stride_h = 0;
  float* lse = nullptr;         // [heads, tokens] natural log, or null
  const int* page_table = nullptr;  // [rows, width]
  int64_t table_stride = 0;
  const int* kv_lens = nullptr;     // [rows]
  const int* slots = nullptr;       // [seqs]: row of the table and of kv_lens (null: b)
  const int* cu_q = nullptr;        // [seqs + 1]
  int seqs = 0, rows = 0, width = 0, page = 0, pages = 0;
  int tokens = 0, heads = 0, kv_heads = 0, group = 0, head_dim = 0;
  int max_new = 0;
  int causal = 1, fp16 = 0;
  float scale_log2 = 0.f;
  // division of the work
  int block_tokens = 0;  // new tokens of a unit
  int tile = 0;          // keys of a tile
  int min_share = 1;     // tiles
  int snap = 0;          // tiles
  int max_units = 0;     // of a sequence and key head
  int units = 0;         // seqs * kv_heads * max_units
  int whole = 0;         // 1: the units are dealt out whole: no shares, no parts
  int grid = 0;          // CTAs
  int unit_rows = 0;     // rows of a part in the workspace
  // workspace: parts [2 * grid][unit_rows][head_dim] and their (max, sum), log2 units; the
  // parts of share c are 2 c (a unit that an earlier share began) and 2 c + 1
  float* part_o = nullptr;
  float2* part_ml = nullptr;
  int4* join = nullptr;  // [grid] of the unit that share c began and others go on with:
                         // its first row of q, first head, rows (0: none), last share
  uint32_t* status = nullptr;
  uint64_t wait_limit_ns = 0;
};

// A launch for sequences that share a prefix (paged_shared.cu): sequences [0, own) come without
// the first[b] tokens that their group shares, and behind them the groups, each the new tokens
// of its sequences over the shared[g] tokens before; `seqs` counts both. The kernels are
// compiled for either type of parameters, so that calls without a plan pay nothing for what
// only these need (in one kernel 64 sequences of six new tokens over up to 1024 keys took 139
// us instead of 133, chunks of 16 tokens 98 instead of 94).
struct PagedGroupParams : PagedParams {
  int form = kPagedByRows;  // (kPagedHeadsApart: unit_rows are those of each of its heads)
  const int* first = nullptr;   // [own] tokens that sequence b shares; behind it member, [own]: a
                                // sequence's group, -1: none; -2 - b where a group's first one
                                // shares nothing, b being the first that does
  const int* groups = nullptr;  // [seqs - own + 1] sequences
  const int* shared = nullptr;  // [seqs - own] tokens
  int own = 0;
  int no_own = 0;                        // this launch leaves the sequences' own keys to another
  int64_t least_rows = 0, most_rows = 0;  // of a group a key head: those that it takes
  float* acc_o = nullptr;    // [2 (own, shared)][tokens][heads][head_dim]: rows of whole units,
  float2* acc_ml = nullptr;  // as parts
  int2* desc = nullptr;      // of the units (paged_desc): the shares that have parts of it, first
                             // and last, or -1 where it is whole
  // Launches that run side by side take SMs in proportion to their work, which the device
  // knows: tiles[b] are the tiles a key head of those before sequence or group b, and the same
  // of the others; a tile takes `cost`.
  uint32_t* tiles = nullptr;  // [seqs + 1], or null: the launch is alone, and finds out itself
  const uint32_t* other_tiles[2] = {nullptr, nullptr};
  float cost = 0.f, other_cost[2] = {0.f, 0.f};  // kv_heads times a tile's time on an SM
  int sms = 0, sm_ctas = 0;  // of the device; of this launch on an SM
};

// The launches for sequences that share prefixes: one of the sequences' own keys, others of
// groups, by their rows.
struct PagedSharedParams {
  PagedGroupParams launch[3];
  int launches = 0;
  int own = 0;  // which one
  const int* member = nullptr;  // [sequences], behind PagedGroupParams::first
};

// Entries of PagedGroupParams::desc a key head, of `seqs` sequences or groups. Their units are
// numbered by their rows (two sequences' never meet, as every sequence before adds one); the
// groups' come behind the sequences'.
#ifdef __CUDACC__
__host__ __device__
#endif
inline int64_t paged_desc_rows(const PagedParams& p, int seqs) {
  return int64_t(p.tokens) / p.block_tokens + seqs + 1;
}

#ifdef __CUDACC__
namespace dev {

// A row's probabilities are 2^(score - base) with base = its running maximum - kLift. Their
// rounding to 16 bits for the product with V (half a step of the type) is relative, as the
// output's own, down to the type's smallest normal number: 2^-126 in bf16, but 2^-14 in fp16,
// where weights of 2^-25 would vanish beside the largest, while the fp32 sum counts them. So
// fp16's are lifted to just below its largest number, 65504: up to 2^(kLift + kStale) = 2^15,
// kStale the powers of two by which the kernel lets its maximum lag. The common factor goes
// out with the sum, and the rest of the kernels sees base as the maximum. Both roundings are
// upwards, so that no probability passes 2^15 (and, at scores whose last place is worth
// more than a power of two, infinity).
template <bool kF16, int kStale>
struct PagedBase {
  static constexpr float kLift = kF16 ? 15.f - kStale : 0.f;
  static __device__ __forceinline__ float of(float top, float scale_log2) {
    if constexpr (kF16) return __fadd_ru(__fmul_ru(top, scale_log2), -kLift);
    return top * scale_log2;
  }
};

template <class P>
constexpr bool kShares = std::is_same_v<P, PagedGroupParams>;

// Sequence b as the kernels use it, whatever the arrays say: n new tokens from row q0,
// all inside [0, tokens) and at most max_new; kv within the table's row, behind `skip` pages;
// new token i sees keys [0, base + i], those below kv. `bad` says that something had to be
// cut.
struct PagedSeq {
  int q0, n, kv, base, row, skip;
  bool bad;
};

// Group g (PagedGroupParams::groups) as a sequence.
__device__ __forceinline__ PagedSeq paged_group(const PagedGroupParams& p, int g) {
  PagedSeq s;
  s.n = s.kv = s.base = s.q0 = s.row = s.skip = 0;
  const int a = __ldg(p.groups + g), e = __ldg(p.groups + g + 1), kv = __ldg(p.shared + g);
  s.bad = a < 0 || e < a || e > p.own || kv < 0 || kv > int64_t(p.width) * p.page || kv % p.page;
  if (s.bad || kv == 0 || a == e) return s;
  // (a sequence whose rows leave the batch is served by none, the others of its group are)
  const int q0 = max(__ldg(p.cu_q + a), 0), end = min(__ldg(p.cu_q + e), p.tokens);
  const int other = -2 - __ldg(p.first + p.own + a);
  int row = p.slots ? __ldg(p.slots + a) : a;
  if (other > a && other < e) row = p.slots ? __ldg(p.slots + other) : other;
  s.bad = end < q0 || row < 0 || row >= p.rows;
  const int64_t rows = int64_t(end - q0) * p.group;
  if (s.bad || rows < p.least_rows || rows > p.most_rows) return s;
  s.n = end - q0;
  s.q0 = q0;
  s.kv = s.base = kv;
  s.row = row;
  return s;
}

template <class P>
__device__ __forceinline__ PagedSeq paged_seq(const P& p, int b) {
  PagedSeq s;
  if constexpr (kShares<P>) {
    if (b >= p.own) return paged_group(p, b - p.own);
    if (p.no_own) {
      s.q0 = s.n = s.kv = s.base = s.row = s.skip = 0;
      s.bad = false;
      return s;
    }
  }
  s.skip = 0;
  s.q0 = __ldg(p.cu_q + b);
  int end = __ldg(p.cu_q + b + 1);
  s.row = p.slots ? __ldg(p.slots + b) : b;
  s.bad = s.q0 < 0 || end < s.q0 || end > p.tokens || end - s.q0 > p.max_new || s.row < 0 ||
          s.row >= p.rows;
  if (s.bad) {
    s.n = s.kv = s.base = s.q0 = s.row = 0;
    return s;
  }
  s.n = end - s.q0;
  s.kv = __ldg(p.kv_lens + s.row);
  const int64_t most = int64_t(p.width) * p.page;
  if (s.kv < 0 || s.kv > most) {
    s.bad = true;
    s.kv = s.kv < 0 ? 0 : int(most);
  }
  if constexpr (kShares<P>) {
    const int first = __ldg(p.first + b);
    if (first < 0 || first > s.kv || first % p.page) {
      s.bad = true;
      s.n = 0;
    } else {
      s.skip = first / p.page;
      s.kv -= first;
    }
  }
  s.base = p.causal ? s.kv - s.n : s.kv;
  return s;
}

// Keys that the last of tokens [t, t + block) sees; tiles of that run, at least one (a
// unit without a visible key still writes its rows).
__device__ __forceinline__ int paged_unit_tiles(const PagedParams& p, const PagedSeq& s, int unit) {
  int last = (unit + 1) * p.block_tokens;
  last = last < s.n ? last : s.n;
  int seen = s.base + last;
  seen = seen < s.kv ? seen : s.kv;
  return seen > 0 ? (seen + p.tile - 1) / p.tile : 1;
}

__device__ __forceinline__ int paged_units(const PagedParams& p, const PagedSeq& s) {
  return (s.n + p.block_tokens - 1) / p.block_tokens;
}

__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) {
  const uint32_t v = a + b;
  return v < a ? 0xffffffffu : v;
}

// prefix[b] = tiles of one key head's units of the sequences before b; prefix[seqs] the
// total, which is 0, and an error, where it does not fit 32 bits: nothing is done then.
// Called by all kThreads threads of the CTA; `sums` holds kThreads / 32 values. report: this
// CTA, one for each launch, tells the status word what is wrong with the sequences.
template <int kThreads, class P>
__device__ __forceinline__ void paged_prefix(const P& p, uint32_t* prefix,
                                             uint32_t* sums, bool report) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t before = 0;
  bool bad = false;
  for (int base = 0; base < p.seqs; base += kThreads) {
    const int b = base + int(threadIdx.x);
    uint32_t mine = 0;
    if (b < p.seqs) {
      const PagedSeq s = paged_seq(p, b);
      bad |= s.bad;
      const int units = paged_units(p, s);
      for (int u = 0; u < units; ++u) mine = add_sat(mine, uint32_t(paged_unit_tiles(p, s, u)));
    }
    uint32_t scan = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, scan, o);
      if (lane >= o) scan = add_sat(scan, v);
    }
    if (lane == 31) sums[warp] = scan;
    __syncthreads();
    uint32_t here = before, all = before;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      const uint32_t v = sums[w];
      if (w < warp) here = add_sat(here, v);
      all = add_sat(all, v);
    }
    if (b < p.seqs) prefix[b] = add_sat(here, scan - mine);
    before = all;
    __syncthreads();
  }
  if (before == 0xffffffffu) {
    bad = true;
    before = 0;
  }
  if (threadIdx.x == 0) prefix[p.seqs] = before;
  if (bad && report) record_error(p.status, kErrBadArgument, 60, 0);
  __syncthreads();
}

// The unit that contains tile w of the whole run, and the tiles [first, first + tiles)
// that are the unit's.
struct PagedUnit {
  PagedSeq s;
  int b, hk, unit, tiles;
  uint64_t first;
};

template <class P>
__device__ __forceinline__ PagedUnit paged_find(const P& p, const uint32_t* prefix,
                                                uint64_t w) {
  PagedUnit u;
  int lo = 0, hi = p.seqs;  // the last b with prefix[b] * kv_heads <= w
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (uint64_t(prefix[mid]) * uint32_t(p.kv_heads) <= w) lo = mid;
    else hi = mid;
  }
  u.b = lo;
  u.s = paged_seq(p, lo);
  const uint32_t per_head = prefix[lo + 1] - prefix[lo];
  const uint64_t base = uint64_t(prefix[lo]) * uint32_t(p.kv_heads);
  u.hk = int((w - base) / per_head);
  u.first = base + uint64_t(u.hk) * per_head;
  u.unit = 0;
  u.tiles = paged_unit_tiles(p, u.s, 0);
  while (u.first + uint32_t(u.tiles) <= w) {
    u.first += uint32_t(u.tiles);
    u.tiles = paged_unit_tiles(p, u.s, ++u.unit);
  }
  return u;
}

// The unit behind `u`, which is not the last.
template <class P>
__device__ __forceinline__ void paged_next(const P& p, const uint32_t* prefix,
                                           PagedUnit& u) {
  u.first += uint32_t(u.tiles);
  if (++u.unit >= paged_units(p, u.s)) {
    u.unit = 0;
    if (++u.hk >= p.kv_heads) {
      u.hk = 0;
      do ++u.b;
      while (u.b + 1 < p.seqs && prefix[u.b + 1] == prefix[u.b]);
      u.s = paged_seq(p, u.b);
    }
  }
  u.tiles = paged_unit_tiles(p, u.s, u.unit);
}

// The place of a unit in PagedGroupParams::desc.
__device__ __forceinline__ int64_t paged_desc(const PagedGroupParams& p, const PagedSeq& s, int b, int unit, int hk) {
  const int64_t at = b < p.own ? b : paged_desc_rows(p, p.own) + b - p.own;
  return (at + s.q0 / p.block_tokens + unit) * p.kv_heads + hk;
}

// At the end of a launch that may have begun early: it ends behind the one before it, so that
// what waits for this one sees the results of both. One CTA is enough, the last, which the others
// have all begun before: more would keep the SMs from the launch that comes next.
template <class P>
__device__ __forceinline__ void paged_behind() {
  if (kShares<P> && blockIdx.x == gridDim.x - 1) asm volatile("griddepcontrol.wait;" ::: "memory");
}

template <class P>
struct PagedShare {
  const P& p;
  const uint32_t* prefix;
  uint64_t total, per;
  uint32_t snap;
  __device__ __forceinline__ PagedShare(const P& params, const uint32_t* pre)
      : p(params), prefix(pre) {
    total = uint64_t(prefix[p.seqs]) * uint32_t(p.kv_heads);
    uint32_t grid = uint32_t(p.grid);
    if constexpr (kShares<P>)
      if (p.tiles) grid = prefix[p.seqs + 1];
    per = (total + grid - 1) / grid;
    if (per < uint32_t(p.min_share)) per = uint32_t(p.min_share);
    snap = per / 2 < uint32_t(p.snap) ? uint32_t(per / 2) : uint32_t(p.snap);
  }
  // The first tile of share c; `u`, the unit that it lies in, where there is one.
  __device__ __forceinline__ uint64_t begin(int c, PagedUnit& u) const {
    uint64_t w = per * uint32_t(c);
    if (w >= total) return total;
    u = paged_find(p, prefix, w);
    const uint64_t end = u.first + uint32_t(u.tiles);
    if (w - u.first <= snap) return u.first;
    if (end - w <= snap) {
      w = end;
      if (w < total) paged_next(p, prefix, u);
    }
    return w;
  }
  // The first tile behind share c.
  __device__ __forceinline__ uint64_t end(int c) const {
    PagedUnit u;
    const uint64_t w = per * uint32_t(c + 1);
    return snap ? begin(c + 1, u) : w < total ? w : total;
  }
  // The share of a unit's last tile.
  __device__ __forceinline__ int last(const PagedUnit& u) const {
    const uint64_t end = u.first + uint32_t(u.tiles);
    int c = int((end - 1) / per);
    if (!snap) return c;
    PagedUnit v;
    while (begin(c, v) >= end) --c;  // a cut that has moved to this unit's end
    return c;
  }
};

// Unit number `id` where p.whole: they count key heads, then units from the last (in a
// causal chunk the longest) to the first, then sequences. False where there is none.
__device__ __forceinline__ bool paged_whole(const PagedParams& p, int id, PagedUnit& u) {
  const int rest = id / p.kv_heads, k = rest % p.max_units;
  u.b = rest / p.max_units;
  u.hk = id - rest * p.kv_heads;
  u.unit = p.max_units - 1 - k;
  u.s = paged_seq(p, u.b);
  if (u.s.bad && k == 0 && u.hk == 0) record_error(p.status, kErrBadArgument, 60, 0);
  if (u.unit >= paged_units(p, u.s)) return false;
  u.first = 0;
  u.tiles = paged_unit_tiles(p, u.s, u.unit);
  return true;
}

// What share c, of tiles [begin, end), leaves for others to go on with. `u` is its last
// unit.
__device__ __forceinline__ void paged_join(const PagedShare<PagedParams>& share, const PagedUnit& u, bool any,
                                           uint64_t begin, uint64_t end) {
  const PagedParams& p = share.p;
  if (!p.join) return;  // one share: nothing is left
  int4 j = make_int4(0, 0, 0, 0);
  if (any && u.first >= begin && u.first + uint32_t(u.tiles) > end) {
    int n = u.s.n - u.unit * p.block_tokens;
    n = n < p.block_tokens ? n : p.block_tokens;
    j = make_int4(u.s.q0 + u.unit * p.block_tokens, u.hk * p.group, n * p.group, share.last(u));
  }
  p.join[blockIdx.x] = j;
}

// prefix[] from p.tiles, and behind it the CTAs among which the launch's work is divided: its
// share of the SMs, at least one, the largest launch taking what the others' leave. False for a
// CTA that is none of them: it should end at once.
template <int kThreads>
__device__ __forceinline__ bool paged_divide(const PagedGroupParams& p, uint32_t* prefix) {
  const uint32_t mine = p.tiles[p.seqs];
  float work = float(mine) * p.cost, all = work;
  float others[2];
  bool largest = true;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    others[i] = p.other_tiles[i] ? float(p.other_tiles[i][p.seqs]) * p.other_cost[i] : 0.f;
    all += others[i];
    largest = largest && (others[i] < work || (others[i] == work && p.other_tiles[i] < p.tiles));
  }
  if (mine == 0) return false;
  auto part = [&](float w) { return w > 0.f ? max(1, int(float(p.sms) * (w / all))) : 0; };
  int sms = part(work);
  if (largest) sms = max(1, p.sms - part(others[0]) - part(others[1]));
  const int ctas = min(sms * p.sm_ctas, p.grid);
  if (int(blockIdx.x) >= ctas) return false;
  for (int i = threadIdx.x; i < p.seqs; i += kThreads) prefix[i] = p.tiles[i];
  if (threadIdx.x == 0) {
    prefix[p.seqs] = mine;
    prefix[p.seqs + 1] = uint32_t(ctas);
  }
  __syncthreads();
  return true;
}

// Where a row of a unit that is not written out goes, unnormalised: a whole unit's to its place in
// acc_o and acc_ml (PagedGroupParams; of a group's unit if `group`), a part's to row `part` of
// the workspace. It is row `at` of o and of ml.
struct PagedRow {
  float* o;
  float2* ml;
  int64_t at;
};
template <class P>
__device__ __forceinline__ PagedRow paged_row(const P& p, bool whole, bool group, int64_t token, int64_t head, int64_t part) {
  if constexpr (kShares<P>)
    if (whole) return {p.acc_o, p.acc_ml, ((group ? int64_t(p.tokens) : 0) + token) * p.heads + head};
  return {p.part_o, p.part_ml, part};
}

// A CTA's way through its work, run by run: tiles [t0, t1) of unit u. Its threads walk
// alike, each warp's or each its own copy.
template <class P>
struct PagedWalk {
  PagedUnit u;
  int t0, t1;
  uint64_t begin, end;  // shares: of tiles
  int id;               // p.whole: the unit's number

  // The first run; false where there is none. Called by all kThreads threads, whose
  // earlier writes to shared memory all see after it.
  template <int kThreads>
  __device__ __forceinline__ bool start(const P& p, uint32_t* prefix, uint32_t* sums) {
    bool divided = false;
    if constexpr (kShares<P>) {
      divided = p.tiles;
      if (divided && !paged_divide<kThreads>(p, prefix)) return false;
    } else if (p.whole) {
      id = int(blockIdx.x) - int(gridDim.x);
      const bool any = next(p, prefix);
      __syncthreads();
      return any;
    }
    if (!divided) paged_prefix<kThreads>(p, prefix, sums, blockIdx.x == 0);
    const PagedShare<P> share(p, prefix);
    begin = share.begin(blockIdx.x, u);
    end = share.end(blockIdx.x);
    if (begin >= end) {
      if constexpr (!kShares<P>)
        if (threadIdx.x == 0) paged_join(share, u, false, begin, end);
      return false;
    }
    run(begin);
    return true;
  }
  __device__ __forceinline__ void run(uint64_t w) {
    t0 = int(w - u.first);
    t1 = end - u.first < uint64_t(u.tiles) ? int(end - u.first) : u.tiles;
  }
  __device__ __forceinline__ bool next(const P& p, const uint32_t* prefix) {
    if constexpr (!kShares<P>) {
      if (p.whole) {
        do {
          id += int(gridDim.x);
          if (id >= p.units) return false;
        } while (!paged_whole(p, id, u));
        t0 = 0;
        t1 = u.tiles;
        return true;
      }
    }
    const uint64_t w = u.first + uint32_t(t1);
    if (w >= end) return false;
    paged_next(p, prefix, u);
    run(w);
    return true;
  }
  __device__ __forceinline__ bool complete() const { return t0 == 0 && t1 == u.tiles; }
  // The workspace's part that takes an incomplete run.
  __device__ __forceinline__ int64_t part() const { return 2 * int64_t(blockIdx.x) + (t0 > 0 ? 0 : 1); }
  // Of each run, by one thread (PagedGroupParams::desc).
  __device__ __forceinline__ void note(const P& p, const uint32_t* prefix) const {
    if constexpr (kShares<P>)
      if (t0 == 0)
        p.desc[paged_desc(p, u.s, u.b, u.unit, u.hk)] =
            complete() ? make_int2(-1, -1) : make_int2(int(blockIdx.x), PagedShare<P>(p, prefix).last(u));
  }
  // After the last run, by one thread.
  __device__ __forceinline__ void leave(const P& p, const uint32_t* prefix) const {
    if constexpr (!kShares<P>)
      if (!p.whole) paged_join(PagedShare<P>(p, prefix), u, true, begin, end);
  }
};

}  // namespace dev
#endif

// Lets `fn` use all of an SM's shared memory; once for each device that it runs on.
template <class Fn>
cudaError_t paged_allow_smem(Fn fn, std::atomic<uint64_t>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || (dev < 64 && done.load() >> dev & 1)) return e;
  e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kPagedMaxSmem));
  if (e == cudaSuccess && dev < 64) done.fetch_or(uint64_t(1) << dev);
  return e;
}

// Few rows a key head (max_new * group <= 32).
// early: may begin while the launch before, which it does not need, still runs.
void paged_decode_launch(const CUtensorMap& mk, const CUtensorMap& mv, const PagedParams& p, cudaStream_t stream);
void paged_decode_launch(const CUtensorMap& mk, const CUtensorMap& mv, const PagedGroupParams& p,
                         cudaStream_t stream, bool early);
// More rows: tcgen05 tiles.
void paged_chunk_launch(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv,
                        const PagedParams& p, cudaStream_t stream);
void paged_chunk_launch(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv,
                        const PagedGroupParams& p, cudaStream_t stream, bool early);
// The most local memory a thread of its forms was compiled with, which has to be none.
int64_t paged_chunk_local_bytes();
// Joins the parts; launched behind either.
void paged_merge_launch(const PagedParams& p, cudaStream_t stream);
// Sequences that share a prefix: `shared`, `first` and `member` (PagedGroupParams::first) from
// the page table, for the groups of p. (Nothing but the arrays of the problem is read.)
void paged_plan_launch(const PagedGroupParams& p, int* shared, int* first, int* member, cudaStream_t stream);
// Fills the launches' PagedGroupParams::tiles, where they have it.
void paged_split_launch(const PagedSharedParams& p, cudaStream_t stream);
// Joins own and shared parts, behind the launches that left them.
void paged_shared_launch(const PagedSharedParams& p, cudaStream_t stream);

}  // namespace mgfa
