// Torch-facing entry points of attention over a paged cache (paged_decode.cu,
// paged_chunk.cu) and of the cache's pages (paged_cache.cu).
#include <torch/types.h>
#include "../common/check.hpp"
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstring>
#include <tuple>

#include "forward_ad.hpp"
#include "rotary_args.hpp"
#include "../kernels/paged_attn.cuh"
#include "../kernels/paged_cache.cuh"
#include "../kernels/tma_host.hpp"

namespace mgfa {

int device_sm_count(int device);

namespace {

using OptTensor = c10::optional<torch::Tensor>;

void check_ints(const torch::Tensor& t, const torch::Tensor& like, int64_t dims, const char* name) {
  MGFA_CHECK(t.is_cuda() && t.scalar_type() == at::kInt && t.dim() == dims && t.is_contiguous() &&
                 t.device() == like.device(),
             name, " must be a contiguous int32 CUDA tensor of ", dims, " dimension(s) on the cache's device");
}

// The words of host_status_word(), which are never freed.
constexpr int kHostWords = 1024;
int* host_words() {
  static int* words = [] {
    void* p = nullptr;
    // also while a stream of this thread is being captured: the allocation is no part of it
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    C10_CUDA_CHECK(cudaThreadExchangeStreamCaptureMode(&mode));
    const cudaError_t e = cudaHostAlloc(&p, kHostWords * sizeof(int), cudaHostAllocPortable | cudaHostAllocMapped);
    C10_CUDA_CHECK(cudaThreadExchangeStreamCaptureMode(&mode));
    C10_CUDA_CHECK(e);
    return static_cast<int*>(std::memset(p, 0, kHostWords * sizeof(int)));
  }();
  return words;
}
std::atomic<int> host_words_used{0};

}  // namespace

// The kernels' status word in `t`, which is on `like`'s device or in pinned host memory.
uint32_t* status_ptr(const torch::Tensor& t, const torch::Tensor& like) {
  MGFA_CHECK(t.scalar_type() == at::kInt && t.numel() >= 1, "status must be an int32 tensor");
  int* p = t.data_ptr<int>();
  // asking the driver about a pointer costs as much as a launch
  if (!t.is_cuda() && !(host_words_used.load() && p >= host_words() && p < host_words() + kHostWords))
    MGFA_CHECK(t.is_pinned(), "status must be in CUDA or pinned host memory");
  MGFA_CHECK(!t.is_cuda() || t.device() == like.device(), "status must be on q's device or in pinned host memory");
  return reinterpret_cast<uint32_t*>(p);
}

namespace {

// 16-bit values, head_dim 64 or 128 (the last dimension, contiguous), every row on a
// 16-byte boundary.
void check_rows16(const torch::Tensor& t, int64_t dims, const char* name) {
  MGFA_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  MGFA_CHECK(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf, name,
             " must be bfloat16 or float16");
  MGFA_CHECK(t.dim() == dims, name, " must have ", dims, " dimensions");
  MGFA_CHECK(t.size(-1) == 64 || t.size(-1) == 128, name, ": unsupported head_dim ", t.size(-1));
  MGFA_CHECK(t.stride(-1) == 1, name, " must have a contiguous head_dim");
  bool ok = reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int64_t d = 0; d + 1 < dims; ++d)
    ok = ok && (t.size(d) <= 1 || (t.stride(d) > 0 && t.stride(d) % 8 == 0));
  MGFA_CHECK(ok, name, " must have rows on 16-byte boundaries and no repeated ones");
}

bool power_of_two(int64_t n) { return n > 0 && (n & (n - 1)) == 0; }

// A tensor map over `rank` dimensions (innermost first, the first contiguous) with the
// strides of dimensions of size 1, which mean nothing, made legal.
CUtensorMap map16(const torch::Tensor& t, std::initializer_list<int64_t> order,
                  std::initializer_list<uint32_t> box) {
  uint64_t dims[4], strides[3];
  uint32_t b[4];
  int i = 0;
  for (int64_t d : order) {
    dims[i] = d < 0 ? 1 : uint64_t(t.size(d));
    if (i > 0) strides[i - 1] = dims[i] <= 1 ? 16 : uint64_t(t.stride(d)) * 2;
    ++i;
  }
  i = 0;
  for (uint32_t x : box) b[i++] = x;
  return host::make_bf16_map(t.data_ptr(), 4, dims, strides, b, CU_TENSOR_MAP_SWIZZLE_128B,
                             t.scalar_type() == at::kHalf ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                          : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16);
}

}  // namespace

// A status word in pinned host memory, for the life of the process.
torch::Tensor host_status_word() {
  const int i = host_words_used.fetch_add(1);
  MGFA_CHECK(i < kHostWords, "too many status words");
  return torch::from_blob(host_words() + i, {1}, torch::TensorOptions().dtype(at::kInt));
}

namespace {

// How many groups cu_groups counts of a batch of `seqs` sequences.
int64_t check_groups(const torch::Tensor& groups, const torch::Tensor& like, int64_t seqs) {
  check_ints(groups, like, 1, "cu_groups");
  MGFA_CHECK(groups.size(0) >= 1, "cu_groups must be [groups + 1]");
  const int64_t n = groups.size(0) - 1;
  MGFA_CHECK(seqs + n <= kPagedMaxSeqs, "at most ", kPagedMaxSeqs, " sequences and groups a call");
  return n;
}

// A group's rows a key head up to which its prefix goes to the decode kernel, in units of 32
// rows; above, to 128-row tiles. Units more than one read the prefix again (from L2), but start
// and end much sooner: in a small call up to four of them.
int64_t group_few_rows(const PagedParams& p) {
  const int64_t rows = int64_t(p.tokens) * p.group;
  return rows <= 128 && int64_t(p.width) * p.page <= 8192 ? 128 : 32;
}

// The launches for sequences that share prefixes (paged_shared.cu).
void attend_shared(const PagedParams& problem, bool few, const torch::Tensor& q, const torch::Tensor& k,
                   const torch::Tensor& v, const torch::Tensor& groups, const torch::Tensor& plan, int sms) {
  const int64_t T = problem.tokens, D = problem.head_dim, n_groups = groups.size(0) - 1;
  const auto f32 = q.options().dtype(at::kFloat);
  PagedSharedParams j;
  PagedGroupParams p;
  static_cast<PagedParams&>(p) = problem;
  p.own = p.seqs;
  p.seqs += int(n_groups);
  p.groups = groups.data_ptr<int>();
  p.shared = plan.data_ptr<int>();
  p.first = p.shared + n_groups;
  p.most_rows = -1;  // no groups
  p.sms = sms;
  j.member = p.first + p.own;
  // rows of whole units, of what is a sequence's own and of what its group shares
  torch::Tensor acc = torch::empty({2 * T * p.heads * (D + 2)}, f32), work[3];
  p.acc_o = acc.data_ptr<float>();
  p.acc_ml = reinterpret_cast<float2*>(p.acc_o + 2 * T * p.heads * D);

  // A launch of 128-row tiles, or (block_tokens set) of the decode kernel, for the groups
  // of least_rows to most_rows rows, and the sequences' own keys unless no_own.
  auto add = [&](PagedGroupParams l) {
    if (l.block_tokens) {
      l.tile = l.form == kPagedHeadsApart ? 16 : 64;
      l.sm_ctas = l.form == kPagedRowsApart ? 1 : 2;
      // (a tile takes 0.9 us of an SM with 32 rows, 0.57 with 16 and two CTAs at work)
      l.cost = l.form == kPagedRowsApart ? 0.9f : 0.57f;
      if (l.form == kPagedHeadsApart) l.kv_heads /= 4;
    } else {
      l.block_tokens = 2 * std::max(1, 128 / l.group);
      l.tile = 128;
      l.snap = 4;
      l.sm_ctas = 1;
      l.cost = 3.f;
    }
    l.cost *= float(l.kv_heads);
    l.unit_rows = l.block_tokens * l.group;
    l.min_share = 2;
    const int64_t units = ((l.no_own ? 0 : T / l.block_tokens + l.own) +
                           (l.most_rows < 0 ? 0 : T / l.block_tokens + n_groups)) * l.kv_heads;
    const int64_t tiles = std::max<int64_t>(1, (int64_t(l.width) * l.page + l.tile - 1) / l.tile);
    l.grid = int(std::min<int64_t>(l.sm_ctas * sms, (units * tiles + l.min_share - 1) / l.min_share));
    j.launch[j.launches++] = l;
  };
  PagedGroupParams over = p;  // groups alone
  over.no_own = 1;
  const int64_t group_rows = group_few_rows(p);
  const bool small = p.group <= 32 && T * p.group <= group_rows;
  if (small) {
    // Few rows in all: one launch of units of up to 32 rows takes everything (24 to 29 us a
    // call, several launches 30 to 36).
    p.most_rows = INT64_MAX;
    p.form = kPagedRowsApart;
    p.block_tokens = 32 / p.group;
    add(p);
  } else if (few) {
    // The groups, by their rows, of which the host knows the bounds and the mean. Launches of
    // whole SMs that have work come before the sequences' own keys, whose CTAs would otherwise
    // take half of many (eight groups of up to 32 rows: 84 us, in the other order 126); the one
    // that probably has none comes last.
    p.block_tokens = p.max_new;
    if (p.max_new * p.group <= 16 && p.kv_heads % 4 == 0) p.form = kPagedHeadsApart;
    const bool large_first = T * p.group > group_rows * n_groups;
    for (int i = 0; i < 3; ++i) {
      if (i == 1) {
        j.own = j.launches;
        add(p);
      } else if (large_first == (i == 0)) {  // on 128-row tiles
        PagedGroupParams large = over;
        large.least_rows = group_rows + 1;
        large.most_rows = INT64_MAX;
        add(large);
      } else {
        PagedGroupParams small = over;
        small.least_rows = 0;
        small.most_rows = group_rows;
        small.form = kPagedRowsApart;
        small.block_tokens = 32 / p.group;
        add(small);
      }
    }
  } else {  // one launch of 128-row tiles
    p.most_rows = INT64_MAX;
    add(p);
  }

  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  const int64_t counts = p.seqs + 1;
  torch::Tensor tiles;
  if (j.launches > 1) tiles = torch::empty({j.launches * counts}, plan.options());
  for (int i = 0; i < j.launches; ++i) {
    PagedGroupParams& l = j.launch[i];
    const int64_t rows = 2 * int64_t(l.grid) * l.unit_rows * (l.form == kPagedHeadsApart ? 4 : 1);
    const int64_t descs = (paged_desc_rows(l, l.own) + paged_desc_rows(l, int(n_groups))) * l.kv_heads;
    work[i] = torch::empty({rows * (D + 2) + 2 * descs}, f32);
    l.part_o = work[i].data_ptr<float>();
    l.part_ml = reinterpret_cast<float2*>(l.part_o + rows * D);
    l.desc = reinterpret_cast<int2*>(l.part_ml + rows);
    if (!tiles.defined()) continue;
    uint32_t* at = reinterpret_cast<uint32_t*>(tiles.data_ptr<int>());
    l.tiles = at + i * counts;
    for (int k = 0, n = 0; k < j.launches; ++k)
      if (k != i) {
        l.other_tiles[n] = at + k * counts;
        l.other_cost[n++] = j.launch[k].cost;
      }
  }
  if (j.launches > 1) paged_split_launch(j, stream);
  for (int i = 0; i < j.launches; ++i) {
    const PagedGroupParams& l = j.launch[i];
    const uint32_t chunk = uint32_t(std::min<int64_t>(l.page, l.tile)), heads = l.form == kPagedHeadsApart ? 4 : 1;
    const CUtensorMap mk = map16(k, {3, 1, 2, 0}, {64, chunk, heads, 1});
    const CUtensorMap mv = map16(v, {3, 1, 2, 0}, {64, chunk, heads, 1});
    if (l.tile == 128) {
      const CUtensorMap mq = map16(q, {2, 1, 0, -1}, {64, uint32_t(l.group), uint32_t(l.block_tokens / 2), 1});
      paged_chunk_launch(mq, mk, mv, l, stream, i > 0);
    } else {
      paged_decode_launch(mk, mv, l, stream, i > 0);
    }
  }
  paged_shared_launch(j, stream);
}

}  // namespace

// int32 [groups + 2 * sequences]: the tokens that each group shares, then those that each
// sequence shares with its group, then each one's group, or below 0 (PagedGroupParams::first).
torch::Tensor shared_prefix(torch::Tensor page_table, torch::Tensor kv_lens, torch::Tensor cu_q,
                            torch::Tensor groups, int64_t page, OptTensor slots, torch::Tensor status) {
  MGFA_CHECK(page_table.is_cuda(), "page_table must be a CUDA tensor");
  check_ints(page_table, page_table, 2, "page_table");
  check_ints(kv_lens, page_table, 1, "kv_lens");
  check_ints(cu_q, page_table, 1, "cu_seqlens_q");
  MGFA_CHECK(power_of_two(page) && page >= 16 && page <= 1024,
             "the page size must be a power of two from 16 to 1024, got ", page);
  MGFA_CHECK(page_table.size(1) * page < (int64_t(1) << 30), "page_table is too wide");
  MGFA_CHECK(kv_lens.size(0) == page_table.size(0), "kv_lens must have an entry for each row of page_table");
  MGFA_CHECK(cu_q.size(0) >= 1, "cu_seqlens_q must be [sequences + 1]");
  const int64_t seqs = cu_q.size(0) - 1;
  if (slots.has_value()) {
    check_ints(*slots, page_table, 1, "slots");
    MGFA_CHECK(slots->size(0) == seqs, "slots must have an entry for each sequence");
  } else {
    MGFA_CHECK(page_table.size(0) >= seqs, "page_table must have a row for each sequence");
  }
  const int64_t n = check_groups(groups, page_table, seqs);
  c10::cuda::CUDAGuard guard(page_table.device());
  torch::Tensor plan = torch::empty({n + 2 * seqs}, page_table.options());
  PagedGroupParams p;
  p.status = status_ptr(status, page_table);
  if (n == 0) return plan;
  p.page_table = page_table.data_ptr<int>();
  p.table_stride = page_table.stride(0);
  p.kv_lens = kv_lens.data_ptr<int>();
  p.slots = slots.has_value() ? slots->data_ptr<int>() : nullptr;
  p.cu_q = cu_q.data_ptr<int>();
  p.groups = groups.data_ptr<int>();
  p.own = int(seqs);
  p.seqs = int(seqs + n);
  p.rows = int(page_table.size(0));
  p.width = int(page_table.size(1));
  p.page = int(page);
  int* shared = plan.data_ptr<int>();
  paged_plan_launch(p, shared, shared + n, shared + n + seqs, at::cuda::getCurrentCUDAStream());
  return plan;
}

std::tuple<torch::Tensor, OptTensor> paged_attention(
    torch::Tensor q, torch::Tensor k, torch::Tensor v, torch::Tensor page_table,
    torch::Tensor kv_lens, torch::Tensor cu_q, int64_t max_new, OptTensor slots, bool causal,
    double scale, OptTensor out_in, bool want_lse, torch::Tensor status, int64_t wait_limit_ns,
    OptTensor groups, OptTensor plan) {
  refuse_tangents("paged_attention", {q, k, v});
  check_rows16(q, 3, "q");
  check_rows16(k, 4, "k_pages");
  check_rows16(v, 4, "v_pages");
  MGFA_CHECK(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
             "q, k_pages and v_pages must have one dtype");
  MGFA_CHECK(k.device() == q.device() && v.device() == q.device(), "q and the pages must be on one device");
  MGFA_CHECK(k.sizes() == v.sizes(), "k_pages and v_pages must have one shape");
  MGFA_CHECK(k.size(3) == q.size(2), "q and the pages must have one head_dim");
  const int64_t T = q.size(0), Hq = q.size(1), D = q.size(2);
  const int64_t pages = k.size(0), page = k.size(1), Hk = k.size(2);
  MGFA_CHECK(power_of_two(page) && page >= 16 && page <= 1024,
             "the page size must be a power of two from 16 to 1024, got ", page);
  MGFA_CHECK(Hk >= 1 && Hq >= 1 && Hq % Hk == 0, "query heads must be a multiple of kv heads");
  const int64_t group = Hq / Hk;
  MGFA_CHECK(group <= kPagedMaxGroup, "at most ", kPagedMaxGroup, " query heads a kv head");
  MGFA_CHECK(pages >= 1 && pages < (int64_t(1) << 30) && T < (int64_t(1) << 30), "too many pages or tokens, or no page");
  check_ints(page_table, k, 2, "page_table");
  check_ints(kv_lens, k, 1, "kv_lens");
  check_ints(cu_q, k, 1, "cu_seqlens_q");
  MGFA_CHECK(kv_lens.size(0) == page_table.size(0), "kv_lens must have an entry for each row of page_table");
  MGFA_CHECK(cu_q.size(0) >= 1, "cu_seqlens_q must be [sequences + 1]");
  const int64_t seqs = cu_q.size(0) - 1;
  MGFA_CHECK(seqs <= kPagedMaxSeqs, "at most ", kPagedMaxSeqs, " sequences a call");
  if (slots.has_value()) {
    check_ints(*slots, k, 1, "slots");
    MGFA_CHECK(slots->size(0) == seqs, "slots must have an entry for each sequence");
  } else {
    MGFA_CHECK(page_table.size(0) >= seqs, "page_table must have a row for each sequence");
  }
  MGFA_CHECK(page_table.size(1) * page < (int64_t(1) << 30), "page_table is too wide");
  MGFA_CHECK(max_new >= 0, "max_seqlen_q must not be negative");
  MGFA_CHECK(groups.has_value() == plan.has_value(), "cu_groups and the plan of the shared prefixes come together");
  const int64_t n_groups = groups.has_value() ? check_groups(*groups, k, seqs) : 0;
  if (n_groups) {
    check_ints(*plan, k, 1, "the plan");
    MGFA_CHECK(plan->size(0) == n_groups + 2 * seqs, "the plan of the shared prefixes is of another batch");
  }
  const float scale_log2 = float(scale * 1.4426950408889634);  // the kernels' own
  MGFA_CHECK(scale_log2 > 0.f && std::isfinite(scale_log2), "softmax_scale must be positive (in float32)");
  c10::cuda::CUDAGuard guard(q.device());
  torch::Tensor out, lse;
  if (out_in.has_value()) {
    out = *out_in;
    check_rows16(out, 3, "out");
    MGFA_CHECK(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type() && out.device() == q.device(),
               "out must have q's shape, dtype and device");
  } else {
    out = torch::empty({T, Hq, D}, q.options());
  }
  if (want_lse) lse = torch::empty({Hq, T}, q.options().dtype(at::kFloat));
  PagedParams p;
  p.status = status_ptr(status, q);
  p.max_new = int(std::min(max_new, T));
  if (seqs == 0 || p.max_new == 0) return {out, want_lse ? OptTensor(lse) : OptTensor()};
  p.q = q.data_ptr();
  p.q_stride_t = q.stride(0);
  p.q_stride_h = q.stride(1);
  p.out = out.data_ptr();
  p.o_stride_t = out.stride(0);
  p.o_stride_h = out.stride(1);
  p.lse = want_lse ? lse.data_ptr<float>() : nullptr;
  p.page_table = page_table.data_ptr<int>();
  p.table_stride = page_table.stride(0);
  p.kv_lens = kv_lens.data_ptr<int>();
  p.slots = slots.has_value() ? slots->data_ptr<int>() : nullptr;
  p.cu_q = cu_q.data_ptr<int>();
  p.seqs = int(seqs);
  p.rows = int(page_table.size(0));
  p.width = int(page_table.size(1));
  p.page = int(page);
  p.pages = int(pages);
  p.tokens = int(T);
  p.heads = int(Hq);
  p.kv_heads = int(Hk);
  p.group = int(group);
  p.head_dim = int(D);
  p.causal = causal ? 1 : 0;
  p.fp16 = q.scalar_type() == at::kHalf;
  p.scale_log2 = scale_log2;
  p.wait_limit_ns = uint64_t(wait_limit_ns);
  const int sms = device_sm_count(q.get_device());
  // Up to 32 rows a key head pad to 16 or 32 on mma.sync; more fill 128-row tiles.
  const bool few = int64_t(p.max_new) * p.group <= 32;
  if (n_groups) {
    attend_shared(p, few, q, k, v, *groups, *plan, sms);
    return {out, want_lse ? OptTensor(lse) : OptTensor()};
  }
  int64_t units;  // at most
  if (few) {
    p.block_tokens = p.max_new;
    p.unit_rows = p.max_new * p.group;
    p.tile = 64;
    p.min_share = 2;
    units = seqs * Hk;
    p.grid = 2 * sms;
  } else {
    const int tile_tokens = std::max(1, 128 / p.group);
    p.block_tokens = 2 * tile_tokens;
    p.unit_rows = p.block_tokens * p.group;
    p.tile = 128;
    p.min_share = 2;
    p.snap = 4;
    units = (T / p.block_tokens + seqs) * Hk;
    p.grid = sms;
  }
  const int64_t tiles = std::max<int64_t>(1, (int64_t(p.width) * page + p.tile - 1) / p.tile);
  p.max_units = (p.max_new + p.block_tokens - 1) / p.block_tokens;
  const int64_t allowed = seqs * Hk * p.max_units;  // units, by max_new
  // Tables of at most 8 tiles a sequence: the units are dealt out whole, which takes neither
  // the lengths' sum nor a join. One token each over 100 to 320 keys: 9.6 us, in shares
  // 15.4 us; 64 chunks of 128 tokens over 128 keys: 61 us, in shares 76 us. A CTA looks at
  // every unit that max_new allows, though (0.3 us each), so not where these are many times
  // those that there can be: one chunk of 1000 tokens and 255 of one, 15 times as many, 206 us, in
  // shares 220 us; 512 chunks of 100 announced as up to 3200, 19 times, 671 us and 325 us,
  // announced as up to the batch's 51200, 7199 us and 325 us.
  p.whole = tiles <= 8 && allowed <= 16 * units && allowed < (int64_t(1) << 30);
  p.units = p.whole ? int(allowed) : 0;
  p.grid = int(std::min<int64_t>(p.grid, p.whole ? p.units : (units * tiles + p.min_share - 1) / p.min_share));
  torch::Tensor work;
  const bool parts = p.grid > 1 && !p.whole;
  if (parts) {
    const int64_t rows = 2 * int64_t(p.grid) * p.unit_rows;
    work = torch::empty({rows * (D + 2) + 4 * int64_t(p.grid)}, q.options().dtype(at::kFloat));
    p.part_o = work.data_ptr<float>();
    p.join = reinterpret_cast<int4*>(p.part_o + rows * D);
    p.part_ml = reinterpret_cast<float2*>(p.join + p.grid);
  }
  const uint32_t chunk = uint32_t(std::min<int64_t>(page, p.tile));
  const CUtensorMap mk = map16(k, {3, 1, 2, 0}, {64, chunk, 1, 1});
  const CUtensorMap mv = map16(v, {3, 1, 2, 0}, {64, chunk, 1, 1});
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  if (few) {
    paged_decode_launch(mk, mv, p, stream);
  } else {
    const CUtensorMap mq = map16(q, {2, 1, 0, -1}, {64, uint32_t(group), uint32_t(p.block_tokens / 2), 1});
    paged_chunk_launch(mq, mk, mv, p, stream);
  }
  if (parts) paged_merge_launch(p, stream);
  return {out, want_lse ? OptTensor(lse) : OptTensor()};
}

// ------------------------------------------------------------------ the cache's pages
namespace {

CacheState cache_state(const torch::Tensor& k, const torch::Tensor& table, const torch::Tensor& lens,
                       const torch::Tensor& refs, const torch::Tensor& grown,
                       const torch::Tensor& status) {
  CacheState c;
  c.table = table.data_ptr<int>();
  c.lens = lens.data_ptr<int>();
  c.refs = refs.data_ptr<int>();
  c.grown = grown.data_ptr<int>();
  c.slots = int(table.size(0));
  c.width = int(table.size(1));
  c.pages = int(k.size(1));
  c.page = int(k.size(2));
  c.status = status_ptr(status, k);
  return c;
}

CachePool cache_pool(const torch::Tensor& k, const torch::Tensor& v) {
  CachePool p;
  p.k = k.data_ptr();
  p.v = v.data_ptr();
  for (int i = 0; i < 4; ++i) {
    p.k_stride[i] = k.stride(i);
    p.v_stride[i] = v.stride(i);
  }
  p.layers = int(k.size(0));
  p.heads = int(k.size(3));
  p.head_dim = int(k.size(4));
  return p;
}

int check_slots(const torch::Tensor& slots, const torch::Tensor& k, const char* name) {
  check_ints(slots, k, 1, name);
  MGFA_CHECK(slots.size(0) <= kPagedMaxSeqs, name, ": at most ", kPagedMaxSeqs, " sequences a call");
  return int(slots.size(0));
}

}  // namespace

// Checks the tensors of a cache once, when it is made.
void cache_check(torch::Tensor k, torch::Tensor v, torch::Tensor table, torch::Tensor lens,
                 torch::Tensor refs, torch::Tensor grown) {
  check_rows16(k, 5, "k");
  check_rows16(v, 5, "v");
  MGFA_CHECK(k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type() && k.device() == v.device(),
             "k and v must have one shape, dtype and device");
  MGFA_CHECK(power_of_two(k.size(2)) && k.size(2) >= 16 && k.size(2) <= 1024,
             "the page size must be a power of two from 16 to 1024, got ", k.size(2));
  MGFA_CHECK(k.size(0) >= 1 && k.size(1) >= 1 && k.size(3) >= 1, "a cache needs layers, pages and heads");
  MGFA_CHECK(k.size(1) < (int64_t(1) << 30), "too many pages");
  check_ints(table, k, 2, "page_table");
  check_ints(lens, k, 1, "lens");
  check_ints(refs, k, 1, "refs");
  check_ints(grown, k, 1, "grown");
  const int64_t slots = table.size(0);
  MGFA_CHECK(slots >= 1 && slots <= kCacheMaxSlots, "page_table must have 1 to ", kCacheMaxSlots, " rows");
  MGFA_CHECK(table.size(1) >= 1 && table.size(1) * k.size(2) < (int64_t(1) << 30), "page_table is empty or too wide");
  // a call's pages are counted in 32 bits
  MGFA_CHECK(table.numel() < (int64_t(1) << 31), "page_table has too many entries");
  MGFA_CHECK(lens.size(0) == slots && grown.size(0) == slots, "lens and grown must have an entry for each row of page_table");
  MGFA_CHECK(refs.size(0) == k.size(1), "refs must have an entry for each page");
}

torch::Tensor cache_reserve(torch::Tensor k, torch::Tensor table, torch::Tensor lens,
                            torch::Tensor refs, torch::Tensor grown, torch::Tensor status,
                            torch::Tensor slots, torch::Tensor cu, int64_t tokens) {
  const int n = check_slots(slots, k, "slots");
  check_ints(cu, k, 1, "cu_seqlens");
  MGFA_CHECK(cu.size(0) == n + 1, "cu_seqlens must be [sequences + 1]");
  MGFA_CHECK(tokens >= 0 && tokens < (int64_t(1) << 30), "n_tokens is out of range");
  c10::cuda::CUDAGuard guard(k.device());
  torch::Tensor pos = torch::empty({tokens}, lens.options());
  const CacheState c = cache_state(k, table, lens, refs, grown, status);
  if (n > 0)
    cache_reserve_launch(c, slots.data_ptr<int>(), cu.data_ptr<int>(), n, pos.data_ptr<int>(),
                         int(tokens), at::cuda::getCurrentCUDAStream());
  else
    pos.zero_();
  return pos;
}

// bool [tokens]: the rows of sequences that cache_reserve, called with the same slots and
// cu, left as they were.
torch::Tensor cache_refused(torch::Tensor k, torch::Tensor table, torch::Tensor lens,
                            torch::Tensor refs, torch::Tensor grown, torch::Tensor status,
                            torch::Tensor slots, torch::Tensor cu, int64_t tokens) {
  const int n = check_slots(slots, k, "slots");
  check_ints(cu, k, 1, "cu_seqlens");
  MGFA_CHECK(cu.size(0) == n + 1, "cu_seqlens must be [sequences + 1]");
  MGFA_CHECK(tokens >= 0 && tokens < (int64_t(1) << 30), "n_tokens is out of range");
  c10::cuda::CUDAGuard guard(k.device());
  torch::Tensor refused = torch::empty({tokens}, lens.options().dtype(at::kBool));
  if (n > 0 && tokens > 0)
    cache_refused_launch(cache_state(k, table, lens, refs, grown, status), slots.data_ptr<int>(),
                         cu.data_ptr<int>(), n, refused.data_ptr<bool>(), int(tokens),
                         at::cuda::getCurrentCUDAStream());
  else
    refused.zero_();
  return refused;
}

void cache_write(torch::Tensor k, torch::Tensor v, torch::Tensor table, torch::Tensor lens,
                 torch::Tensor refs, torch::Tensor grown, torch::Tensor status, int64_t layer,
                 torch::Tensor new_k, torch::Tensor new_v, torch::Tensor slots, torch::Tensor cu) {
  refuse_tangents("PagedKVCache.write", {new_k, new_v});
  MGFA_CHECK(layer >= 0 && layer < k.size(0), "layer ", layer, " is not one of the cache's ", k.size(0));
  const int n = check_slots(slots, k, "slots");
  check_ints(cu, k, 1, "cu_seqlens");
  MGFA_CHECK(cu.size(0) == n + 1, "cu_seqlens must be [sequences + 1]");
  check_rows16(new_k, 3, "new_k");
  check_rows16(new_v, 3, "new_v");
  MGFA_CHECK(new_k.sizes() == new_v.sizes() && new_k.size(1) == k.size(3) && new_k.size(2) == k.size(4),
             "new_k and new_v must be [tokens, kv_heads, head_dim] as in the cache");
  MGFA_CHECK(new_k.scalar_type() == k.scalar_type() && new_v.scalar_type() == k.scalar_type() &&
                 new_k.device() == k.device() && new_v.device() == k.device(),
             "new_k and new_v must have the cache's dtype and device");
  MGFA_CHECK(new_k.size(0) < (int64_t(1) << 30), "too many tokens");
  if (n == 0 || new_k.size(0) == 0) return;
  c10::cuda::CUDAGuard guard(k.device());
  const CacheState c = cache_state(k, table, lens, refs, grown, status);
  CachePool pool = cache_pool(k, v);
  pool.k = static_cast<uint16_t*>(pool.k) + layer * pool.k_stride[0];
  pool.v = static_cast<uint16_t*>(pool.v) + layer * pool.v_stride[0];
  const int64_t ks[2] = {new_k.stride(0), new_k.stride(1)}, vs[2] = {new_v.stride(0), new_v.stride(1)};
  cache_write_launch(c, pool, new_k.data_ptr(), new_v.data_ptr(), ks, vs, slots.data_ptr<int>(),
                     cu.data_ptr<int>(), n, int(new_k.size(0)), at::cuda::getCurrentCUDAStream());
}

// q with its heads normed (with weights) and rotated; k's, treated alike, and v go to the
// pages of the batch that cache_reserve made room for.
torch::Tensor cache_append(torch::Tensor k, torch::Tensor v, torch::Tensor table, torch::Tensor lens,
                           torch::Tensor refs, torch::Tensor grown, torch::Tensor status,
                           int64_t layer, torch::Tensor q, torch::Tensor new_k, torch::Tensor new_v,
                           torch::Tensor positions, torch::Tensor inv_freq, torch::Tensor slots,
                           torch::Tensor cu, OptTensor q_weight, OptTensor k_weight, double eps,
                           bool interleaved, double magnitude) {
  const torch::Tensor none;
  refuse_tangents("PagedKVCache.append", {q, new_k, new_v, inv_freq, q_weight.value_or(none), k_weight.value_or(none)});
  MGFA_CHECK(layer >= 0 && layer < k.size(0), "layer ", layer, " is not one of the cache's ", k.size(0));
  const int n = check_slots(slots, k, "slots");
  check_ints(cu, k, 1, "cu_seqlens");
  MGFA_CHECK(cu.size(0) == n + 1, "cu_seqlens must be [sequences + 1]");
  check_rows16(q, 3, "q");
  check_rows16(new_k, 3, "new_k");
  check_rows16(new_v, 3, "new_v");
  MGFA_CHECK(new_k.sizes() == new_v.sizes() && new_k.size(1) == k.size(3) && new_k.size(2) == k.size(4),
             "new_k and new_v must be [tokens, kv_heads, head_dim] as in the cache");
  MGFA_CHECK(q.size(0) == new_k.size(0) && q.size(2) == k.size(4), "q must be [tokens, heads, head_dim] with new_k's tokens and head_dim");
  for (const torch::Tensor* t : {&q, &new_k, &new_v})
    MGFA_CHECK(t->scalar_type() == k.scalar_type() && t->device() == k.device(),
               "q, new_k and new_v must have the cache's dtype and device");
  MGFA_CHECK(q.size(0) < (int64_t(1) << 30), "too many tokens");
  MGFA_CHECK(q_weight.has_value() == k_weight.has_value(), "q_weight and k_weight come together");
  c10::cuda::CUDAGuard guard(k.device());
  CacheAppendParams p;
  const RotaryType t = rotary_args(p, q, new_k, positions, inv_freq, interleaved, magnitude);
  torch::Tensor w[2], out = torch::empty(q.sizes(), q.options());
  if (q_weight.has_value()) {
    norm_weight_args(p, q, new_k, *q_weight, k_weight, eps, w);
    p.norm = 1;
  }
  if (q.size(0) == 0) return out;
  MGFA_CHECK(p.vec, "q and new_k must have rows on 16-byte boundaries");  // (checked above)
  p.x[0].out = out.data_ptr();
  p.v = rotary_tensor(new_v);
  p.c = cache_state(k, table, lens, refs, grown, status);
  p.k_pool = static_cast<uint16_t*>(k.data_ptr()) + layer * k.stride(0);
  p.v_pool = static_cast<uint16_t*>(v.data_ptr()) + layer * v.stride(0);
  for (int i = 0; i < 3; ++i) {
    p.k_stride[i] = k.stride(i + 1);
    p.v_stride[i] = v.stride(i + 1);
  }
  p.slots = slots.data_ptr<int>();
  p.cu = cu.data_ptr<int>();
  p.seqs = n;
  cache_append_launch(t, p, device_sm_count(k.get_device()), at::cuda::getCurrentCUDAStream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return out;
}

void cache_free(torch::Tensor k, torch::Tensor table, torch::Tensor lens, torch::Tensor refs,
                torch::Tensor grown, torch::Tensor status, torch::Tensor slots) {
  const int n = check_slots(slots, k, "slots");
  if (n == 0) return;
  c10::cuda::CUDAGuard guard(k.device());
  cache_free_launch(cache_state(k, table, lens, refs, grown, status), slots.data_ptr<int>(), n,
                    at::cuda::getCurrentCUDAStream());
}

void cache_fork(torch::Tensor k, torch::Tensor v, torch::Tensor table, torch::Tensor lens,
                torch::Tensor refs, torch::Tensor grown, torch::Tensor status, torch::Tensor src,
                torch::Tensor dst, bool share) {
  const int n = check_slots(src, k, "src");
  MGFA_CHECK(check_slots(dst, k, "dst") == n, "src and dst must have one length");
  if (n == 0) return;
  c10::cuda::CUDAGuard guard(k.device());
  const CacheState c = cache_state(k, table, lens, refs, grown, status);
  const int64_t most = share ? n : int64_t(n) * c.width;
  torch::Tensor scratch = torch::empty({1 + 3 * most}, lens.options());
  int* at = scratch.data_ptr<int>();
  cache_fork_launch(c, cache_pool(k, v), src.data_ptr<int>(), dst.data_ptr<int>(), n, share, at,
                    reinterpret_cast<PageMove*>(at + 1), device_sm_count(k.get_device()),
                    at::cuda::getCurrentCUDAStream());
}

void cache_compact(torch::Tensor k, torch::Tensor v, torch::Tensor table, torch::Tensor lens,
                   torch::Tensor refs, torch::Tensor grown, torch::Tensor status) {
  c10::cuda::CUDAGuard guard(k.device());
  const CacheState c = cache_state(k, table, lens, refs, grown, status);
  torch::Tensor scratch = torch::empty({2 + 4 * int64_t(c.pages)}, lens.options());
  int* at = scratch.data_ptr<int>();
  cache_compact_launch(c, cache_pool(k, v), at, reinterpret_cast<PageMove*>(at + 2),
                       at + 2 + 3 * int64_t(c.pages), device_sm_count(k.get_device()),
                       at::cuda::getCurrentCUDAStream());
}

}  // namespace mgfa
