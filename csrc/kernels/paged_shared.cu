// Attention of sequences that share a prefix: what they share, and the join of their parts.
//
// Sequences that were forked from one prompt hold the same pages for its full ones. A group
// is a run of the batch's sequences; its first shared[g] tokens are read once for the new
// tokens of all of them, as one more sequence whose every row sees every key, and each
// sequence's own keys are read for itself. Both come as (O, m, l): O = sum 2^(s - m) v,
// l = sum 2^(s - m), unnormalised in fp32, from paged_decode.cu and paged_chunk.cu, whose
// shares may cut them further. A row's result is
//
//   out = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i,   M = max m_i
//
// over its own parts and its group's, in that order: one softmax over all keys, whose two
// halves are never rounded to 16 bits.
//
// The prefix of many rows is work for the tensor cores (paged_chunk.cu), own keys and the prefix
// of few rows are bound by reading them (paged_decode.cu). The launches run side by side, on SMs
// in proportion to their work: one token each of 128 sequences over 32768 shared and up to 512
// own keys (32/8 heads of 128) takes 113 to 118 us that way, 139 us one behind another. The plan
// takes 11 us of that call (once a step, not once a layer), the tiles before each sequence 4 us,
// the join 9 us. Eight groups of up to eight sequences over up to 8192 keys: 59 of 79 us.
#include "paged_attn.cuh"
#include "sm100_ptx.cuh"

#include <cooperative_groups.h>

#include <algorithm>
#include <stdexcept>
#include <string>

namespace mgfa {
namespace {

using namespace mgfa::dev;
namespace cg = cooperative_groups;

// ---------------------------------------------------------------------- what is shared
constexpr int kPlanThreads = 512;
constexpr int kPlanCtas = 8;   // of a group, a cluster
constexpr int kPlanLoads = 8;  // of each table that a lane has under way

// shared[g]: the leading pages that all of the group's sequences with new tokens name alike, as
// far as these are full and hold none of the new tokens; 0 for one alone, which reads them once
// anyway. A sequence without new tokens (an answer that has ended, whose pages may be gone) or
// without a row of the table has no say, and shares nothing; where none has new tokens, shared[g]
// is of all. Groups whose cu_seqlens fall share nothing; invalid ones neither, nor do all others
// of the call then.
__global__ void __launch_bounds__(kPlanThreads)
    paged_plan_kernel(const PagedGroupParams p, int* shared, int* first, int* member) {
  const int g = blockIdx.x / kPlanCtas, cta = blockIdx.x % kPlanCtas, n_groups = p.seqs - p.own;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  __shared__ int least;
  if (threadIdx.x == 0) least = p.width;
  bool bad = false;
  for (int i = threadIdx.x; i < n_groups; i += kPlanThreads) {
    const int a = __ldg(p.groups + i), e = __ldg(p.groups + i + 1);
    bad |= a < 0 || e < a || e > p.own;
  }
  bad = __syncthreads_or(bad);
  const int from = bad ? 0 : __ldg(p.groups + g), to = bad ? 0 : __ldg(p.groups + g + 1);
  auto row_of = [&](int b) { return p.slots ? __ldg(p.slots + b) : b; };
  auto new_of = [&](int b) { return __ldg(p.cu_q + b + 1) - __ldg(p.cu_q + b); };
  auto counts = [&](int row, int n, int any) { return row >= 0 && row < p.rows && n >= any; };
  const int mine_first = from + cta * (kPlanThreads / 32) + warp;  // of this warp's sequences
  int row = 0, n = 0;
  if (mine_first < to) {
    row = row_of(mine_first);
    n = new_of(mine_first);
  }
  // Each warp finds the first that counts, and whether there is a second, for itself: mostly
  // among the first 32, and nothing has to wait for other warps. [1]: with new tokens.
  int lead_of[2] = {to, to}, lead_row[2] = {0, 0}, live[2] = {0, 0};
  for (int b0 = from; b0 < to && live[1] < 2; b0 += 32) {
    const int b = b0 + lane, r = b < to ? row_of(b) : -1, m = b < to ? new_of(b) : 0;
#pragma unroll
    for (int any = 0; any < 2; ++any) {
      const uint32_t mask = __ballot_sync(0xffffffffu, counts(r, m, any));
      if (mask && live[any] == 0) {
        lead_of[any] = b0 + __ffs(mask) - 1;
        lead_row[any] = __shfl_sync(0xffffffffu, r, __ffs(mask) - 1);
      }
      live[any] += __popc(mask);
    }
  }
  const int any = live[1] > 0, lead = any ? lead_of[1] : lead_of[0];
  const bool several = (any ? live[1] : live[0]) > 1;
  if (several) {
    const int* theirs = p.page_table + int64_t(any ? lead_row[1] : lead_row[0]) * p.table_stride;
    for (int b = mine_first; b < to; b += kPlanCtas * (kPlanThreads / 32)) {
      if (b > mine_first) {
        row = row_of(b);
        n = new_of(b);
      }
      if (n < 0 && lane == 0) atomicMin(&least, 0);
      if (!counts(row, n, any)) continue;
      const int64_t kv = std::min<int64_t>(__ldg(p.kv_lens + row), int64_t(p.width) * p.page);
      int pages = int(std::max<int64_t>(kv - n, 0) / p.page);
      const int* mine = p.page_table + int64_t(row) * p.table_stride;
      for (int j0 = 0; j0 < pages; j0 += 32 * kPlanLoads) {
        bool differ[kPlanLoads];
#pragma unroll
        for (int k = 0; k < kPlanLoads; ++k) {
          const int j = j0 + k * 32 + lane;
          differ[k] = false;
          if (j < pages) {
            const int page = __ldg(mine + j);
            differ[k] = page != __ldg(theirs + j) || page < 0;
          }
        }
#pragma unroll
        for (int k = 0; k < kPlanLoads; ++k) {
          const uint32_t at = __ballot_sync(0xffffffffu, differ[k]);
          if (at) pages = std::min(pages, j0 + k * 32 + __ffs(at) - 1);
        }
      }
      if (lane == 0) atomicMin(&least, pages);
    }
  }
  const int id = cta * kPlanThreads + int(threadIdx.x), step = kPlanCtas * kPlanThreads;
  auto shares_of = [&](int b) { return counts(row_of(b), new_of(b), 1); };
  bool shares = from + id < to && shares_of(from + id);
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  int all = several ? least : 0;
  for (int i = 0; i < kPlanCtas; ++i) all = std::min(all, *cluster.map_shared_rank(&least, i));
  cluster.sync();
  for (int b = from + id; b < to; b += step) {
    if (b > from + id) shares = shares_of(b);
    first[b] = shares ? all * p.page : 0;
    member[b] = shares ? g : b == from && all > 0 ? -2 - lead : -1;
  }
  if (id == 0) shared[g] = all * p.page;
  if (g == 0) {  // sequences of no group
    const int begin = bad ? p.own : __ldg(p.groups), end = bad ? p.own : __ldg(p.groups + n_groups);
    for (int b = id; b < p.own; b += step)
      if (b < begin || b >= end) {
        first[b] = 0;
        member[b] = -1;
      }
    if (bad && id == 0) record_error(p.status, kErrBadArgument, 69, 0);
  }
}

// ---------------------------------------------------------------------- who does what
constexpr int kSplitThreads = 1024;

// CTA l: the tiles before each sequence and group of launch l (PagedGroupParams::tiles), which its
// CTAs then need not find out for themselves. Each reports what its own launch's sequences and
// groups have wrong: a launch of the groups alone looks at no sequence's own arguments.
__global__ void __launch_bounds__(kSplitThreads) paged_split_kernel(const __grid_constant__ PagedSharedParams p) {
  extern __shared__ uint32_t prefix[];
  __shared__ uint32_t sums[kSplitThreads / 32];
  const PagedGroupParams& l = p.launch[blockIdx.x];
  paged_prefix<kSplitThreads>(l, prefix, sums, true);
  for (int i = threadIdx.x; i <= l.seqs; i += kSplitThreads) l.tiles[i] = prefix[i];
}

// ---------------------------------------------------------------------- the join
constexpr int kJoinWarps = 16;

// A row's parts of one kind: whole, or those of shares [c, c + n).
struct RowParts {
  const float* o;
  const float2* ml;
  int64_t row, first, step;  // part i: at `row` (n == 1), or first + i * step
  int n;
  __device__ __forceinline__ int64_t at(int i) const { return i ? first + i * step : row; }
};

// Of row (i, head) of sequence or group b, whose keys launch p took; heads: key heads of a unit.
__device__ __forceinline__ RowParts row_parts(const PagedGroupParams& p, const PagedSeq& s, int b, int i, int head) {
  const int heads = p.form == kPagedHeadsApart ? 4 : 1, hk = head / p.group;
  const int unit = i / p.block_tokens, tok = i - unit * p.block_tokens;
  const int2 d = p.desc[paged_desc(p, s, b, unit, hk / heads)];
  RowParts r;
  r.first = r.step = 0;
  if (d.x < 0) {
    r.o = p.acc_o;
    r.ml = p.acc_ml;
    r.row = ((b < p.own ? 0 : int64_t(p.tokens)) + s.q0 + i) * p.heads + head;
    r.n = 1;
  } else {
    // share c's parts are 2 c and 2 c + 1, which is the one of the unit that it begins
    const int64_t at = int64_t(hk % heads) * p.unit_rows + tok * p.group + head - hk * p.group;
    r.o = p.part_o;
    r.ml = p.part_ml;
    r.step = 2 * int64_t(heads) * p.unit_rows;
    r.first = d.x * r.step + at;
    r.row = r.first + r.step / 2;
    // (of a unit that a wait which ran out has left alone: none)
    r.n = d.y >= d.x && d.y < p.grid ? d.y - d.x + 1 : 0;
  }
  return r;
}

// CTA (b, y): every gridDim.y-th block of rows of sequence b, a row for each new token and head.
// kSplit warps share a row, as in paged_merge_kernel.
template <int kD, bool kF16, int kSplit>
__global__ void __launch_bounds__(kJoinWarps * 32) paged_shared_kernel(const __grid_constant__ PagedSharedParams p) {
  constexpr int kE = kD / 32, kRows = kJoinWarps / kSplit;
  __shared__ float sh[kSplit > 1 ? kJoinWarps : 1][kD];
  const PagedGroupParams& a = p.launch[p.own];
  const int b = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = warp % kSplit;
  const PagedSeq own = paged_seq(a, b);
  const int64_t rows = int64_t(own.n) * a.heads;
  // the group, and which launch took it (none a group without new tokens)
  PagedSeq over;
  over.n = 0;
  int taken = 0, g = -1;
  if (rows > 0 && own.skip > 0) {
    g = p.member[b];
    if (g >= 0 && g < a.seqs - a.own) {
      for (; taken < p.launches; ++taken) {
        over = paged_group(p.launch[taken], g);
        if (over.n > 0) break;
      }
      const bool inside = own.q0 >= over.q0 && own.q0 + own.n <= over.q0 + over.n;
      if (!inside || over.kv != own.skip * a.page) over.n = 0;
    }
    if (over.n == 0 && blockIdx.y == 0 && threadIdx.x == 0)
      record_error(a.status, kErrBadArgument, 69, 0);  // first[] and the groups do not fit
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int64_t r0 = int64_t(blockIdx.y) * kRows; r0 < rows; r0 += int64_t(gridDim.y) * kRows) {
    const int64_t r = r0 + warp / kSplit;
    const bool live = r < rows;
    const int i = live ? int(r / a.heads) : 0, head = live ? int(r - int64_t(i) * a.heads) : 0;
    float top = -INFINITY, total = 0.f, acc[kE];
#pragma unroll
    for (int e = 0; e < kE; ++e) acc[e] = 0.f;
    if (live) {
      RowParts side[2];
      side[0] = row_parts(a, own, b, i, head);
      side[1].n = 0;
      if (over.n > 0) side[1] = row_parts(p.launch[taken], over, a.own + g, own.q0 + i - over.q0, head);
#pragma unroll
      for (int k = 0; k < 2; ++k)
        for (int j = lane; j < side[k].n; j += 32) top = fmaxf(top, side[k].ml[side[k].at(j)].x);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int k = 0; k < 2; ++k)
        for (int j0 = 0; j0 < side[k].n; j0 += 32) {
          float2 ml = make_float2(-INFINITY, 0.f);
          if (j0 + lane < side[k].n) ml = side[k].ml[side[k].at(j0 + lane)];
          const float wt = ex2_approx(ml.x - base);
          total += ml.y * wt;
          const int n = side[k].n - j0 < 32 ? side[k].n - j0 : 32;
#pragma unroll 8
          for (int j = part; j < n; j += kSplit) {
            const float f = __shfl_sync(0xffffffffu, wt, j);
            const float* src = side[k].o + side[k].at(j0 + j) * kD + lane * kE;
            if constexpr (kE == 4) {
              const float4 v = *reinterpret_cast<const float4*>(src);
              acc[0] = fmaf(f, v.x, acc[0]);
              acc[1] = fmaf(f, v.y, acc[1]);
              acc[2] = fmaf(f, v.z, acc[2]);
              acc[3] = fmaf(f, v.w, acc[3]);
            } else {
              const float2 v = *reinterpret_cast<const float2*>(src);
              acc[0] = fmaf(f, v.x, acc[0]);
              acc[1] = fmaf(f, v.y, acc[1]);
            }
          }
        }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    }
    if constexpr (kSplit > 1) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < kE; ++e) sh[warp][lane * kE + e] = acc[e];
      __syncthreads();
      if (part == 0) {
#pragma unroll
        for (int k = 1; k < kSplit; ++k)
#pragma unroll
          for (int e = 0; e < kE; ++e) acc[e] += sh[warp + k][lane * kE + e];
      }
    }
    if (!live || part) continue;
    const float base = top == -INFINITY ? 0.f : top;
    const float inv = total == 0.f ? 0.f : 1.f / total;  // 0: no visible key
    const int tok = own.q0 + i;
    uint16_t* out = static_cast<uint16_t*>(a.out) + int64_t(tok) * a.o_stride_t +
                    int64_t(head) * a.o_stride_h + lane * kE;
    if constexpr (kE == 4)
      *reinterpret_cast<uint2*>(out) =
          make_uint2(pack16<kF16>(acc[0] * inv, acc[1] * inv), pack16<kF16>(acc[2] * inv, acc[3] * inv));
    else
      *reinterpret_cast<uint32_t*>(out) = pack16<kF16>(acc[0] * inv, acc[1] * inv);
    if (a.lse && lane == 0)
      a.lse[int64_t(head) * a.tokens + tok] =
          total == 0.f ? -INFINITY : (base + log2f(total)) * 0.6931471805599453f;
  }
}

void cuda_ok(cudaError_t e) {
  if (e != cudaSuccess) throw std::runtime_error(std::string("paged attention: ") + cudaGetErrorString(e));
}

template <int kD, bool kF16>
void join_launch(const PagedSharedParams& p, cudaStream_t s) {
  // Few rows may have many parts each, many rows have few.
  const PagedGroupParams& a = p.launch[p.own];
  const int64_t rows = int64_t(a.max_new) * a.heads;
  const bool few = int64_t(a.own) * rows <= 1024;
  const int per = few ? kJoinWarps / 4 : kJoinWarps;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.own, unsigned(std::min<int64_t>((rows + per - 1) / per, 256)));
  cfg.blockDim = dim3(kJoinWarps * 32);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cuda_ok(cudaLaunchKernelEx(&cfg, few ? paged_shared_kernel<kD, kF16, 4> : paged_shared_kernel<kD, kF16, 1>, p));
}

}  // namespace

void paged_plan_launch(const PagedGroupParams& p, int* shared, int* first, int* member, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((p.seqs - p.own) * kPlanCtas);
  cfg.blockDim = dim3(kPlanThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kPlanCtas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cuda_ok(cudaLaunchKernelEx(&cfg, paged_plan_kernel, p, shared, first, member));
}

void paged_split_launch(const PagedSharedParams& p, cudaStream_t s) {
  paged_split_kernel<<<p.launches, kSplitThreads, 4 * (p.launch[0].seqs + 1), s>>>(p);
  cuda_ok(cudaGetLastError());
}

void paged_shared_launch(const PagedSharedParams& p, cudaStream_t s) {
  const PagedGroupParams& a = p.launch[0];
  if (a.head_dim == 64) a.fp16 ? join_launch<64, true>(p, s) : join_launch<64, false>(p, s);
  else a.fp16 ? join_launch<128, true>(p, s) : join_launch<128, false>(p, s);
}

}  // namespace mgfa
