// The pages of a cache, kept on the device: room for new tokens is reserved, the
// tokens' keys and values are written, sequences are forked and freed and the pool is
// compacted without the host knowing a length, so a serving step needs no
// synchronisation and can be captured into a graph.
//
// Which pages are taken depends on the state alone: always the lowest free ones, in the
// order of the call's sequences. Deciding that is a scan over the pool's reference
// counts by one CTA (4 bytes a page, 4096 pages a step); what moves data is a grid.
// Bound by memory: a byte written or moved is read once and written once. Moving 534 MB
// of pages takes 83 us (6.4 TB/s), the plan over 2048 pages before it 5 us. A step that
// reserves and writes 2100 tokens of 16 sequences (18 MB) is bound by two launches and
// their chains of look-ups: 19 us.
//
// A sequence is served whole or not at all: where its pages do not suffice, its slot is
// named twice or out of range, or its row is too short, it stays as it was (its `grown`
// is 0, so that write() leaves it alone) and the status word says so.
#include "paged_attn.cuh"
#include "paged_cache.cuh"
#include "sm100_ptx.cuh"

#include <algorithm>
#include <stdexcept>
#include <string>

namespace mgfa {
namespace {

using namespace mgfa::dev;

constexpr int kPlanThreads = 1024;
constexpr int kPlanWarps = kPlanThreads / 32;
constexpr int kMaxSeqs = 4096;

static_assert(kMaxSeqs <= kCacheMaxSlots, "owner[] takes an entry a sequence too");

struct PlanSmem {
  int first[kMaxSeqs + 1];     // pages needed by the sequences before b
  int owner[kCacheMaxSlots];   // the first b that names the slot; then (reserve) the place
                               // of sequence b's first new token
  int sums[kPlanWarps];
};

// Exclusive scan over the CTA's threads of `mine`; `total` gets the sum.
__device__ __forceinline__ int cta_scan(int mine, int* sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int scan = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, scan, o);
    if (lane >= o) scan += v;
  }
  __syncthreads();  // the last scan's readers are done
  if (lane == 31) sums[warp] = scan;
  __syncthreads();
  int w = sums[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += v;
  }
  total = __shfl_sync(0xffffffffu, w, 31);
  const int before = __shfl_sync(0xffffffffu, w, warp ? warp - 1 : 0);
  return (warp ? before : 0) + scan - mine;
}

__device__ __forceinline__ int pages_of(int tokens, int page) { return (tokens + page - 1) / page; }

// owner[slot] = the first b of list[0, n) that names it; INT_MAX where none does.
__device__ __forceinline__ void plan_owners(PlanSmem& s, const int* list, int n, int slots) {
  for (int i = threadIdx.x; i < slots; i += kPlanThreads) s.owner[i] = 0x7fffffff;
  __syncthreads();
  for (int b = threadIdx.x; b < n; b += kPlanThreads) {
    const int slot = list[b];
    if (slot >= 0 && slot < slots) atomicMin(&s.owner[slot], b);
  }
  __syncthreads();
}

// first[] from need(b), whose calls see every b once.
template <class Need>
__device__ __forceinline__ void plan_needs(PlanSmem& s, int n, Need need) {
  int before = 0;
  for (int base = 0; base < n; base += kPlanThreads) {
    const int b = base + int(threadIdx.x);
    const int mine = b < n ? need(b) : 0;
    int total;
    const int at = cta_scan(mine, s.sums, total);
    if (b < n) s.first[b] = before + at;
    before += total;
  }
  if (threadIdx.x == 0) s.first[n] = before;
  __syncthreads();
}

// The sequence that page number `rank` of the needed ones is for.
__device__ __forceinline__ int plan_find(const PlanSmem& s, int n, int rank) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (s.first[mid] <= rank) lo = mid;
    else hi = mid;
  }
  return lo;  // the last b with first[b] <= rank: those before it with the same need none
}

// Calls take(rank, page) for the lowest first[n] free pages, as far as there are so
// many, in order, and returns how many there were.
template <class Take>
__device__ __forceinline__ int plan_pages(PlanSmem& s, const CacheState& c, int wanted, Take take) {
  int found = 0;
  for (int base = 0; base < c.pages && found < wanted; base += 4 * kPlanThreads) {
    const int p0 = base + 4 * int(threadIdx.x);
    int ref[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) ref[i] = p0 + i < c.pages ? c.refs[p0 + i] : 1;
    int mine = 0, total;
#pragma unroll
    for (int i = 0; i < 4; ++i) mine += ref[i] == 0;
    int rank = found + cta_scan(mine, s.sums, total);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (ref[i] == 0) {
        if (rank < wanted) take(rank, p0 + i);
        ++rank;
      }
    found += total;
  }
  __syncthreads();
  return found < wanted ? found : wanted;
}

// Position of row t of the batch: behind what its sequence held before it grew.
__device__ __forceinline__ int token_position(const CacheState& c, const int* slots, const int* cu,
                                              int seqs, int t) {
  if (t < __ldg(cu) || t >= __ldg(cu + seqs)) return 0;
  const int b = token_seq(cu, seqs, t), slot = __ldg(slots + b);
  const int n = __ldg(cu + b + 1) - __ldg(cu + b);
  if (slot < 0 || slot >= c.slots) return t - __ldg(cu + b);
  // a sequence that could not grow: where its tokens would have gone (as in the plan)
  const int old = c.grown[slot] == n ? c.lens[slot] - n : c.lens[slot];
  return old + t - __ldg(cu + b);
}

constexpr int kPositionsInPlan = 4096;

__global__ void __launch_bounds__(kPlanThreads)
    cache_reserve_kernel(const CacheState c, const int* slots, const int* cu, int seqs,
                         int* positions, int tokens) {
  extern __shared__ __align__(16) uint8_t raw[];
  PlanSmem& s = *reinterpret_cast<PlanSmem*>(raw);
  plan_owners(s, slots, seqs, c.slots);
  auto grows = [&](int b, int& slot, int& old) {  // tokens that b adds; 0: none, < 0: an error
    slot = slots[b];
    const int n = cu[b + 1] - cu[b];
    if (slot < 0 || slot >= c.slots || s.owner[slot] != b || n < 0 || cu[b] < 0 ||
        cu[b + 1] > tokens)
      return -1;
    old = c.lens[slot];
    if (old < 0 || int64_t(old) + n > int64_t(c.width) * c.page) return -1;
    return n;
  };
  plan_needs(s, seqs, [&](int b) {
    int slot, old = 0;
    const int n = grows(b, slot, old);
    if (n < 0) record_error(c.status, kErrBadArgument, 64, 0);
    return n <= 0 ? 0 : pages_of(old + n, c.page) - pages_of(old, c.page);
  });
  const int wanted = s.first[seqs];
  const int found = plan_pages(s, c, wanted, [&](int rank, int page) {
    const int b = plan_find(s, seqs, rank), slot = slots[b];
    c.table[int64_t(slot) * c.width + pages_of(c.lens[slot], c.page) + rank - s.first[b]] = page;
    c.refs[page] = 1;
  });
  if (found < wanted) {
    if (threadIdx.x == 0) record_error(c.status, kErrNoPages, 64, 0);
    // the sequence that got some but not all of its pages gives them back
    const int b = plan_find(s, seqs, found), slot = slots[b];
    const int have = pages_of(c.lens[slot], c.page);
    for (int i = threadIdx.x; i < found - s.first[b]; i += kPlanThreads) {
      int& entry = c.table[int64_t(slot) * c.width + have + i];
      c.refs[entry] = 0;
      entry = -1;
    }
  }
  __syncthreads();
  for (int b = threadIdx.x; b < seqs; b += kPlanThreads) {
    int slot, old = 0;
    int n = grows(b, slot, old);
    if (n < 0) {
      // a slot named again belongs to its first sequence
      if (slot >= 0 && slot < c.slots && s.owner[slot] == b) c.grown[slot] = 0;
      continue;
    }
    if (s.first[b + 1] > found && s.first[b + 1] > s.first[b]) n = 0;
    c.grown[slot] = n;
    c.lens[slot] = old + n;
  }
  if (tokens > kPositionsInPlan) return;  // cache_positions_kernel
  // From here on first[] is cu and owner[b] what has to be added to a row's number.
  __syncthreads();
  for (int b = threadIdx.x; b <= seqs; b += kPlanThreads) s.first[b] = cu[b];
  __syncthreads();
  for (int b = threadIdx.x; b < seqs; b += kPlanThreads) {
    const int slot = slots[b], n = s.first[b + 1] - s.first[b];
    const bool known = slot >= 0 && slot < c.slots;
    const int old = known ? c.lens[slot] - (c.grown[slot] == n ? n : 0) : 0;
    s.owner[b] = old - s.first[b];
  }
  __syncthreads();
  for (int t = threadIdx.x; t < tokens; t += kPlanThreads) {
    const int b = plan_find(s, seqs, t);
    const bool in = t >= s.first[0] && t < s.first[seqs];
    positions[t] = in ? s.owner[b] + t : 0;
  }
}

__global__ void cache_positions_kernel(const CacheState c, const int* slots, const int* cu,
                                       int seqs, int* positions, int tokens) {
  const int t = blockIdx.x * blockDim.x + threadIdx.x;
  if (t < tokens) positions[t] = token_position(c, slots, cu, seqs, t);
}

struct WriteParams {
  CacheState c;
  CachePool pool;  // one layer: strides [1, 4)
  const void* k;
  const void* v;
  int64_t k_stride[2], v_stride[2];  // token, head
  const int* slots;
  const int* cu;
  int seqs, tokens;
};

// One warp per (row of the batch, key or value): the row's place is looked up once, then
// its heads * head_dim values are copied in 16-byte pieces.
__global__ void __launch_bounds__(256) cache_write_kernel(const WriteParams p) {
  const int64_t id = (int64_t(blockIdx.x) * 256 + threadIdx.x) >> 5;
  const int t = int(id >> 1), lane = threadIdx.x & 31;
  const bool value = id & 1;
  if (t >= p.tokens || t < __ldg(p.cu) || t >= __ldg(p.cu + p.seqs)) return;
  int slot, q0, n, len;
  if (!row_grew(p.c, p.slots, p.cu, p.seqs, t, lane, slot, q0, n, len)) return;
  const int pos = len - n + t - q0;
  if (pos < 0 || pos >= int64_t(p.c.width) * p.c.page) return;
  const int page = p.c.table[int64_t(slot) * p.c.width + pos / p.c.page];
  if (page < 0 || page >= p.c.pages) {
    if (lane == 0) record_error(p.c.status, kErrBadArgument, 65, 0);
    return;
  }
  const int64_t* stride = value ? p.pool.v_stride : p.pool.k_stride;
  const int64_t* from = value ? p.v_stride : p.k_stride;
  uint16_t* dst = static_cast<uint16_t*>(value ? p.pool.v : p.pool.k) + page * stride[1] +
                  (pos % p.c.page) * stride[2];
  const uint16_t* src = static_cast<const uint16_t*>(value ? p.v : p.k) + t * from[0];
  const int per = p.pool.head_dim / 8, pieces = p.pool.heads * per;
#pragma unroll 4
  for (int i = lane; i < pieces; i += 32) {
    const int h = i / per, c = (i % per) * 8;
    *reinterpret_cast<uint4*>(dst + h * stride[3] + c) =
        *reinterpret_cast<const uint4*>(src + h * from[1] + c);
  }
}

// One warp per row: whether it belongs to a sequence that reserve() left as it was.
__global__ void __launch_bounds__(256)
    cache_refused_kernel(const CacheState c, const int* slots, const int* cu, int seqs,
                         bool* refused, int tokens) {
  const int t = int((int64_t(blockIdx.x) * 256 + threadIdx.x) >> 5), lane = threadIdx.x & 31;
  if (t >= tokens) return;
  int slot, q0, n, len;
  const bool in = t >= __ldg(cu) && t < __ldg(cu + seqs);
  const bool no = in && !row_grew(c, slots, cu, seqs, t, lane, slot, q0, n, len);
  if (lane == 0) refused[t] = no;
}

// One CTA per entry; a slot named again is freed once.
__global__ void __launch_bounds__(128) cache_free_kernel(const CacheState c, const int* slots) {
  const int slot = slots[blockIdx.x];
  bool again = false;
  for (int i = threadIdx.x; i < blockIdx.x; i += 128) again |= slots[i] == slot;
  if (__syncthreads_or(again)) return;
  if (slot < 0 || slot >= c.slots) {
    if (threadIdx.x == 0) record_error(c.status, kErrBadArgument, 66, 0);
    return;
  }
  int* row = c.table + int64_t(slot) * c.width;
  for (int i = threadIdx.x; i < c.width; i += 128) {
    const int page = row[i];
    if (page >= 0 && page < c.pages) atomicSub(c.refs + page, 1);
    row[i] = -1;
  }
  if (threadIdx.x == 0) c.lens[slot] = c.grown[slot] = 0;
}

__global__ void __launch_bounds__(kPlanThreads)
    cache_fork_kernel(const CacheState c, const int* src, const int* dst, int n, int share,
                      int* count, PageMove* moves) {
  extern __shared__ __align__(16) uint8_t raw[];
  PlanSmem& s = *reinterpret_cast<PlanSmem*>(raw);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  plan_owners(s, dst, n, c.slots);
  // The source's length, or < 0: a slot out of range or named as a target before, a
  // target that holds something, a source that is a target of this call.
  auto length = [&](int b) {
    const int from = src[b], to = dst[b];
    if (from < 0 || from >= c.slots || to < 0 || to >= c.slots || s.owner[to] != b ||
        s.owner[from] != 0x7fffffff || c.table[int64_t(to) * c.width] >= 0)
      return -1;
    const int l = c.lens[from];
    return l < 0 || l > int64_t(c.width) * c.page ? -1 : l;
  };
  plan_needs(s, n, [&](int b) {
    const int l = length(b);
    if (l < 0) record_error(c.status, kErrBadArgument, 67, 0);
    return l < 0 ? 0 : share ? (l % c.page != 0) : pages_of(l, c.page);
  });
  const int wanted = s.first[n];
  // A page of its own for the rest of a last page that is not full, or for every page.
  const int found = plan_pages(s, c, wanted, [&](int rank, int page) {
    const int b = plan_find(s, n, rank);
    const int l = c.lens[src[b]], col = share ? l / c.page : rank - s.first[b];
    const int left = l - col * c.page;
    moves[rank] = {c.table[int64_t(src[b]) * c.width + col], page, left < c.page ? left : c.page};
    c.refs[page] = 1;
  });
  if (found < wanted) {
    if (threadIdx.x == 0) record_error(c.status, kErrNoPages, 67, 0);
    const int b = plan_find(s, n, found);  // got some but not all: gives them back
    for (int i = s.first[b] + threadIdx.x; i < found; i += kPlanThreads) {
      c.refs[moves[i].to] = 0;
      moves[i].from = -1;
    }
  }
  __syncthreads();
  // The new rows, one warp each. (No source is a target, so the rows read do not change.)
  const int lane = threadIdx.x & 31;
  for (int b = threadIdx.x >> 5; b < n; b += kPlanWarps) {
    const int l = length(b);
    if (l < 0 || (s.first[b + 1] > found && s.first[b + 1] > s.first[b])) continue;
    __syncwarp();  // every lane has read the target's row before lane 0 changes it
    const int* from = c.table + int64_t(src[b]) * c.width;
    int* to = c.table + int64_t(dst[b]) * c.width;
    const int whole = l / c.page, all = pages_of(l, c.page);
    for (int i = lane; i < all; i += 32) {
      if (share && i < whole) {
        to[i] = from[i];
        if (from[i] >= 0 && from[i] < c.pages) atomicAdd(c.refs + from[i], 1);
      } else {
        to[i] = moves[s.first[b] + (share ? 0 : i)].to;
      }
    }
    if (lane == 0) {
      c.lens[dst[b]] = l;
      c.grown[dst[b]] = 0;
    }
  }
  if (threadIdx.x == 0) *count = found;
}

// Pairs the live pages behind the first `live` places with the holes before them, both
// in order: moves[i], place[page] = its new place, count = {pairs, live}.
__global__ void __launch_bounds__(kPlanThreads)
    cache_compact_kernel(const CacheState c, int* count, PageMove* moves, int* place) {
  __shared__ int sums[kPlanWarps];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  int mine = 0, live;
  for (int i = threadIdx.x; i < c.pages; i += kPlanThreads) mine += c.refs[i] != 0;
  cta_scan(mine, sums, live);
  int holes = 0, movers = 0;
  for (int base = 0; base < c.pages; base += 4 * kPlanThreads) {
    const int p0 = base + 4 * int(threadIdx.x);
    int hole[4], mover[4], a = 0, b = 0, total;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int page = p0 + i, ref = page < c.pages ? c.refs[page] : 0;
      hole[i] = page < live && ref == 0;
      mover[i] = page >= live && page < c.pages && ref != 0;
      a += hole[i];
      b += mover[i];
    }
    // both counts in one scan: each is at most 4096 here
    const int both = cta_scan(a | (b << 16), sums, total);
    int h = holes + (both & 0xffff), m = movers + (both >> 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (hole[i]) moves[h++].to = p0 + i;
      if (mover[i]) {
        moves[m].from = p0 + i;
        moves[m++].tokens = c.page;
      }
    }
    holes += total & 0xffff;
    movers += total >> 16;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < holes; i += kPlanThreads) {  // as many movers as holes
    const PageMove mv = moves[i];
    place[mv.from] = mv.to;
    c.refs[mv.to] = c.refs[mv.from];
    c.refs[mv.from] = 0;
  }
  if (threadIdx.x == 0) {
    count[0] = holes;
    count[1] = live;
  }
}

// Carries out the moves over all layers, keys and values, in pieces of kPiece 16-byte
// vectors; with `place`, the table's entries behind the live pages first.
constexpr int kMoveThreads = 256;
constexpr int kPiece = 4 * kMoveThreads;

__global__ void __launch_bounds__(kMoveThreads)
    cache_move_kernel(const CacheState c, const CachePool pool, const int* count,
                      const PageMove* moves, const int* place) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int n = count[0];
  if (place) {
    const int live = count[1];
    const int64_t all = int64_t(c.slots) * c.width;
    for (int64_t i = int64_t(blockIdx.x) * kMoveThreads + threadIdx.x; i < all;
         i += int64_t(gridDim.x) * kMoveThreads) {
      const int page = c.table[i];
      if (page >= live && page < c.pages) c.table[i] = place[page];
    }
  }
  const int per_row = pool.head_dim / 8, per_token = pool.heads * per_row;
  const int pieces = (c.page * per_token + kPiece - 1) / kPiece;
  const int64_t work = int64_t(n) * pool.layers * 2 * pieces;
  for (int64_t w = blockIdx.x; w < work; w += gridDim.x) {
    const int piece = int(w % pieces);
    const int64_t rest = w / pieces;
    const bool value = rest & 1;
    const int layer = int((rest >> 1) % pool.layers);
    const PageMove mv = moves[(rest >> 1) / pool.layers];
    if (mv.from < 0 || mv.from >= c.pages) continue;
    const int64_t* stride = value ? pool.v_stride : pool.k_stride;
    uint16_t* base = static_cast<uint16_t*>(value ? pool.v : pool.k) + layer * stride[0];
    const uint16_t* src = base + mv.from * stride[1];
    uint16_t* dst = base + mv.to * stride[1];
    const int end = mv.tokens * per_token;
    uint4 val[kPiece / kMoveThreads];
    int64_t at[kPiece / kMoveThreads];
#pragma unroll
    for (int i = 0; i < kPiece / kMoveThreads; ++i) {
      const int x = piece * kPiece + i * kMoveThreads + threadIdx.x;
      const int tok = x / per_token, h = (x % per_token) / per_row, col = (x % per_row) * 8;
      at[i] = x < end ? tok * stride[2] + h * stride[3] + col : -1;
      if (at[i] >= 0) val[i] = *reinterpret_cast<const uint4*>(src + at[i]);
    }
#pragma unroll
    for (int i = 0; i < kPiece / kMoveThreads; ++i)
      if (at[i] >= 0) *reinterpret_cast<uint4*>(dst + at[i]) = val[i];
  }
}

void cuda_ok(cudaError_t e) {
  if (e != cudaSuccess) throw std::runtime_error(std::string("cache pages: ") + cudaGetErrorString(e));
}

void move_launch(const CacheState& c, const CachePool& pool, const int* count, const PageMove* moves,
                 const int* place, int64_t most, int sm_count, cudaStream_t s) {
  const int64_t pieces = (int64_t(c.page) * pool.heads * pool.head_dim / 8 + kPiece - 1) / kPiece;
  cudaLaunchConfig_t cfg = {};
  // the number of moves is known on the device only: a few waves, or fewer where even
  // `most` moves are less
  cfg.gridDim = dim3(unsigned(std::max<int64_t>(1, std::min<int64_t>(most * pool.layers * 2 * pieces, 16 * sm_count))));
  cfg.blockDim = dim3(kMoveThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cuda_ok(cudaLaunchKernelEx(&cfg, cache_move_kernel, c, pool, count, moves, place));
}

}  // namespace

void cache_reserve_launch(const CacheState& c, const int* slots, const int* cu, int seqs,
                          int* positions, int tokens, cudaStream_t s) {
  static std::atomic<uint64_t> allowed{0};
  cuda_ok(paged_allow_smem(cache_reserve_kernel, allowed));
  cache_reserve_kernel<<<1, kPlanThreads, sizeof(PlanSmem), s>>>(c, slots, cu, seqs, positions, tokens);
  if (tokens > kPositionsInPlan)
    cache_positions_kernel<<<(tokens + 255) / 256, 256, 0, s>>>(c, slots, cu, seqs, positions, tokens);
  cuda_ok(cudaGetLastError());
}

void cache_refused_launch(const CacheState& c, const int* slots, const int* cu, int seqs,
                          bool* refused, int tokens, cudaStream_t s) {
  cache_refused_kernel<<<unsigned((int64_t(tokens) + 7) / 8), 256, 0, s>>>(c, slots, cu, seqs, refused, tokens);
  cuda_ok(cudaGetLastError());
}

void cache_write_launch(const CacheState& c, const CachePool& pool, const void* k, const void* v,
                        const int64_t* k_stride, const int64_t* v_stride, const int* slots,
                        const int* cu, int seqs, int tokens, cudaStream_t s) {
  WriteParams p{c, pool, k, v, {k_stride[0], k_stride[1]}, {v_stride[0], v_stride[1]}, slots, cu, seqs, tokens};
  cache_write_kernel<<<unsigned((int64_t(tokens) * 2 + 7) / 8), 256, 0, s>>>(p);
  cuda_ok(cudaGetLastError());
}

void cache_free_launch(const CacheState& c, const int* slots, int n, cudaStream_t s) {
  cache_free_kernel<<<n, 128, 0, s>>>(c, slots);
  cuda_ok(cudaGetLastError());
}

void cache_fork_launch(const CacheState& c, const CachePool& pool, const int* src, const int* dst,
                       int n, bool share, int* count, PageMove* moves, int sm_count, cudaStream_t s) {
  static std::atomic<uint64_t> allowed{0};
  cuda_ok(paged_allow_smem(cache_fork_kernel, allowed));
  cache_fork_kernel<<<1, kPlanThreads, sizeof(PlanSmem), s>>>(c, src, dst, n, share ? 1 : 0, count, moves);
  cuda_ok(cudaGetLastError());
  move_launch(c, pool, count, moves, nullptr, share ? n : int64_t(n) * c.width, sm_count, s);
}

void cache_compact_launch(const CacheState& c, const CachePool& pool, int* count, PageMove* moves,
                          int* place, int sm_count, cudaStream_t s) {
  cache_compact_kernel<<<1, kPlanThreads, 0, s>>>(c, count, moves, place);
  cuda_ok(cudaGetLastError());
  move_launch(c, pool, count, moves, place, c.pages, sm_count, s);
}

}  // namespace mgfa
