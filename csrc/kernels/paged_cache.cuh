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
