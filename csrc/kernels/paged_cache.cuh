// The pages of a cache: which sequence holds which, and what moves them (paged_cache.cu).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace mgfa {

constexpr int kCacheMaxSlots = 8192;

// The state that the kernels change. A page is free where refs is 0; a sequence (slot)
// holds the pages of its table row up to ceil(lens / page), the rest of the row is -1.
// Only a full page is ever held by several sequences.
struct CacheState {
  int* table = nullptr;  // [slots, width]
  int* lens = nullptr;   // [slots] tokens
  int* refs = nullptr;   // [pages] sequences that hold the page
  int* grown = nullptr;  // [slots] tokens that the last reserve() added
  int slots = 0, width = 0, pages = 0, page = 0;
  uint32_t* status = nullptr;
};

// [layers, pages, page, heads, head_dim] of 16-bit values, strides in elements.
struct CachePool {
  void* k = nullptr;
  void* v = nullptr;
  int64_t k_stride[4] = {0, 0, 0, 0};  // layer, page, token, head
  int64_t v_stride[4] = {0, 0, 0, 0};
  int layers = 0, heads = 0, head_dim = 0;
};

// A copy of the first `tokens` tokens of a page; from < 0: none.
struct PageMove {
  int from, to, tokens;
};

#ifdef __CUDACC__
namespace dev {

__device__ __forceinline__ int token_seq(const int* cu, int seqs, int t) {
  int lo = 0, hi = seqs;  // the last b with cu[b] <= t
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(cu + mid) <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

// token_seq() by a whole warp: 32 entries a step.
__device__ __forceinline__ int token_seq_warp(const int* cu, int seqs, int t, int lane) {
  int lo = 0, n = seqs;  // the last b with cu[b] <= t is in [lo, lo + n)
  while (n > 1) {
    const int step = (n + 31) / 32, at = lo + lane * step;
    const bool below = lane * step < n && (lane == 0 || __ldg(cu + at) <= t);
    const int last = 31 - __clz(__ballot_sync(0xffffffffu, below));
    lo += last * step;
    n = n - last * step < step ? n - last * step : step;
  }
  return lo;
}

// Whether reserve() has made room for row t of the batch, which is row t - q0 of the n that
// sequence `slot`, now of `len` tokens, has grown by. Called by a whole warp, for
// cu[0] <= t < cu[seqs]. (Loads that do not need one another are issued together.)
__device__ __forceinline__ bool row_grew(const CacheState& c, const int* slots, const int* cu,
                                         int seqs, int t, int lane, int& slot, int& q0, int& n, int& len) {
  const int b = token_seq_warp(cu, seqs, t, lane);
  slot = __ldg(slots + b);
  q0 = __ldg(cu + b);
  n = __ldg(cu + b + 1) - q0;
  if (slot < 0 || slot >= c.slots) return false;
  const int grown = c.grown[slot];
  len = c.lens[slot];
  // a slot named again, with as many tokens, would pass the test below too: its first
  // sequence alone has grown
  bool again = false;
  for (int i = lane; i < b; i += 32) again |= __ldg(slots + i) == slot;
  if (__any_sync(0xffffffffu, again)) return false;
  return grown == n && t - q0 < n;
}

}  // namespace dev
#endif

void cache_reserve_launch(const CacheState& c, const int* slots, const int* cu, int seqs,
                          int* positions, int tokens, cudaStream_t stream);
// refused[t]: whether row t belongs to a sequence that the reserve before left as it was.
void cache_refused_launch(const CacheState& c, const int* slots, const int* cu, int seqs,
                          bool* refused, int tokens, cudaStream_t stream);
void cache_write_launch(const CacheState& c, const CachePool& pool, const void* k, const void* v,
                        const int64_t* k_stride, const int64_t* v_stride, const int* slots,
                        const int* cu, int seqs, int tokens, cudaStream_t stream);
void cache_free_launch(const CacheState& c, const int* slots, int n, cudaStream_t stream);
// `count` one int, `moves` n (share) or n * width entries of scratch.
void cache_fork_launch(const CacheState& c, const CachePool& pool, const int* src, const int* dst,
                       int n, bool share, int* count, PageMove* moves, int sm_count,
                       cudaStream_t stream);
// `count` two ints, `moves` and `place` one entry a page of scratch.
void cache_compact_launch(const CacheState& c, const CachePool& pool, int* count, PageMove* moves,
                          int* place, int sm_count, cudaStream_t stream);

}  // namespace mgfa
