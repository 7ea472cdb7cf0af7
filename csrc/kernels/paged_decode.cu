// Attention over a paged cache for few new tokens (max_new * group <= 32 rows a key
// head: decoding, and a few speculative tokens), and the kernel that joins the parts.
//
//   out = sum_j p_j v_j / sum_j p_j,  p_j = 2^(scale_log2 q.k_j - m),  lse = ln sum e^(s)
//
// Bound by memory: K and V are read once, at 2 * rows * 2 operations for each 2-byte
// element, 4 to 64 a byte. So the matrix work goes to mma.sync with rows padded to 16
// or 32 (a 128-row tcgen05 tile would be empty but for those rows), and the layout
// serves the loads: a producer warp keeps up to three tiles of 64 keys (K and V, 32 KB
// at head_dim 128) on their way by TMA, page by page, and two CTAs share an SM. Each of
// the four consumer warps takes 16 keys of a tile for itself, scores and values, with a
// running maximum, sum and output of its own in registers, so the loop has no barrier
// but the tile's; the four are added when a unit ends. 32 sequences of 8192 keys (8 key
// heads of 128, pages of 16) take 171 us for 1.07 GB, 6.3 TB/s; one of 131072 keys 86 us,
// and 9 us for joining 296 parts; with 4 new tokens each (16 rows) the 32 sequences take
// 1.03 times as long, with 8 (32 rows, whose second block of 16 spills 468 bytes at head_dim
// 128) 1.3 times. For short sequences the time is latency: one token each
// over 100 to 320 keys takes 9.6 us.
#include "paged_attn.cuh"
#include "sm100_ptx.cuh"

#include <stdexcept>

namespace mgfa {
namespace {

using namespace mgfa::dev;

constexpr int kConsumers = 4;
constexpr int kThreads = (kConsumers + 1) * 32;
constexpr int kKeys = 64;

template <int kD, int kMT>
struct __align__(1024) DecodeSmem {
  static constexpr int kHalves = kD / 64;
  static constexpr int kStages = kD == 64 ? 6 : (kMT == 1 ? 3 : 2);
  uint16_t kv[kStages][2][kHalves][kKeys * 64];  // [stage][K, V][64 columns][key][column]
  union {  // the queries are last read before a unit's results are added
    uint16_t q[16 * kMT][kD + 8];
    float acc[16 * kMT][kD + 4];
  };
  float2 ml[kConsumers][16 * kMT];
  uint64_t full[kStages], empty[kStages];
  uint32_t abort_flag, stop;
  uint32_t sums[kThreads / 32];
};

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

// c += a b, 16 x 8 x 16
template <bool kF16>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (kF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

// kD head_dim, kF16 type, kMT blocks of 16 rows.
template <int kD, bool kF16, int kMT>
__global__ void __launch_bounds__(kThreads, 2)
    paged_decode_kernel(const __grid_constant__ CUtensorMap map_k,
                        const __grid_constant__ CUtensorMap map_v, const PagedParams p) {
  using Smem = DecodeSmem<kD, kMT>;
  constexpr int kStages = Smem::kStages, kHalves = kD / 64, kR = 16 * kMT;
  extern __shared__ uint8_t raw[];
  Smem& s = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  uint32_t* prefix = reinterpret_cast<uint32_t*>(&s + 1);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t warp = warp_id(), lane = lane_id();
  AbortState ab{&s.abort_flag, p.status, p.wait_limit_ns};
  if (threadIdx.x == 0) {
    s.abort_flag = 0;
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&s.full[i], 1);
      mbar_init(&s.empty[i], kConsumers);
    }
    fence_mbar_init();
  }
  PagedWalk at;
  if (!at.start<kThreads>(p, prefix, s.sums)) return;  // the whole CTA
  uint32_t it = 0;

  if (warp == kConsumers) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      tma_prefetch_desc(&map_k);
      tma_prefetch_desc(&map_v);
    }
    const int chunk = p.page < kKeys ? p.page : kKeys;  // keys of one box
    bool ok = true;
    do {
      const PagedUnit& u = at.u;
      const int* row = p.page_table + int64_t(u.s.row) * p.table_stride;
      for (int t = at.t0; t < at.t1; ++t, ++it) {
        const int st = it % kStages;
        if (!__all_sync(0xffffffffu, mbar_wait(&s.empty[st], ((it / kStages) & 1) ^ 1, ab, 61))) {
          ok = false;
          break;
        }
        // boxes that hold a key below kv; the others' keys are masked
        const int left = u.s.kv - t * kKeys;
        const int boxes = left <= 0 ? 0 : ((left < kKeys ? left : kKeys) + chunk - 1) / chunk;
        if (lane == 0)
          mbar_arrive_expect_tx(&s.full[st], uint32_t(boxes * chunk * kD * 2 * 2));
        __syncwarp();
        for (int c = lane; c < boxes; c += 32) {
          const int key = t * kKeys + c * chunk;
          int page = __ldg(row + key / p.page);
          if (page < 0 || page >= p.pages) {
            record_error(p.status, kErrBadArgument, 62, 0);
            page = p.pages;  // outside the map: the box reads zeros
          }
#pragma unroll
          for (int hf = 0; hf < kHalves; ++hf) {
            tma_load_4d(&s.kv[st][0][hf][c * chunk * 64], &map_k, &s.full[st], hf * 64,
                        key % p.page, u.hk, page);
            tma_load_4d(&s.kv[st][1][hf][c * chunk * 64], &map_v, &s.full[st], hf * 64,
                        key % p.page, u.hk, page);
          }
        }
        __syncwarp();
      }
    } while (ok && at.next(p, prefix));
    if (lane == 0) at.leave(p, prefix);
    // Never leave with a copy outstanding: the last kStages tiles' barriers.
    volatile uint32_t never = 0;
    AbortState drain{&never, nullptr, p.wait_limit_ns};
    for (uint32_t i = it > kStages ? it - kStages : 0; i < it; ++i)
      mbar_wait(&s.full[i % kStages], (i / kStages) & 1, drain, 0);
    return;
  }

  // -------------------------------------------------------------- consumers
  const int mi = lane >> 3, lr = lane & 7;  // matrix and row of this lane's ldmatrix address
  // K: matrices (keys 0-7, 8 columns), (keys 0-7, next 8), (keys 8-15, ..) twice
  const uint32_t k_row = warp * 16 + (mi >> 1) * 8 + lr, k_col = (mi & 1) * 8;
  // V, transposed: (keys 0-7), (keys 8-15), then the next 8 columns
  const uint32_t v_row = warp * 16 + (mi & 1) * 8 + lr, v_col = (mi >> 1) * 8;
  const uint32_t kv_base = smem_u32(&s.kv[0][0][0][0]);
  constexpr uint32_t kHalfBytes = kKeys * 128;
  // A wait that ran out must not leave the other warps in a barrier: such a warp goes on
  // to the unit's end without its tiles, and there all four stop.
  bool ok = true;
  do {
    const PagedUnit& u = at.u;
    const int rows = u.s.n * p.group;
    // queries: row r = token r / group, head r % group
    for (int i = threadIdx.x; i < kR * (kD / 8); i += kConsumers * 32) {
      const int r = i / (kD / 8), c = (i % (kD / 8)) * 8;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (r < rows)
        v = *reinterpret_cast<const uint4*>(
            static_cast<const uint16_t*>(p.q) + int64_t(u.s.q0 + r / p.group) * p.q_stride_t +
            int64_t(u.hk * p.group + r % p.group) * p.q_stride_h + c);
      *reinterpret_cast<uint4*>(&s.q[r][c]) = v;
    }
    consumers_sync();
    const uint32_t q_addr = smem_u32(&s.q[(mi & 1) * 8 + lr][(mi >> 1) * 8]);
    uint32_t qf[kMT == 1 ? kD / 16 : 1][4];
    if constexpr (kMT == 1) {
#pragma unroll
      for (int ks = 0; ks < kD / 16; ++ks) ldsm4(q_addr + ks * 32, qf[ks]);
    }
    // keys seen by this thread's rows (lane / 4 and that + 8 of each block)
    int lim[kMT][2];
#pragma unroll
    for (int m = 0; m < kMT; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = m * 16 + h * 8 + (lane >> 2);
        int l = p.causal ? u.s.kv - u.s.n + r / p.group + 1 : u.s.kv;
        l = l < u.s.kv ? l : u.s.kv;
        lim[m][h] = r < rows ? l : 0;
      }
    const int full_keys = (p.causal ? u.s.kv - u.s.n + 1 : u.s.kv);  // seen by every row
    float o[kMT][kD / 8][4], mx[kMT][2], sum[kMT][2];
#pragma unroll
    for (int m = 0; m < kMT; ++m) {
      mx[m][0] = mx[m][1] = -INFINITY;
      sum[m][0] = sum[m][1] = 0.f;
#pragma unroll
      for (int n = 0; n < kD / 8; ++n) o[m][n][0] = o[m][n][1] = o[m][n][2] = o[m][n][3] = 0.f;
    }
    for (int t = at.t0; t < at.t1; ++t, ++it) {
      const int st = it % kStages;
      ok = __all_sync(0xffffffffu, mbar_wait(&s.full[st], (it / kStages) & 1, ab, 63));
      if (!ok) break;
      const uint32_t kb = kv_base + st * (2 * kHalves * kHalfBytes), vb = kb + kHalves * kHalfBytes;
      float sc[kMT][2][4];
#pragma unroll
      for (int m = 0; m < kMT; ++m)
#pragma unroll
        for (int n = 0; n < 2; ++n) sc[m][n][0] = sc[m][n][1] = sc[m][n][2] = sc[m][n][3] = 0.f;
#pragma unroll
      for (int ks = 0; ks < kD / 16; ++ks) {
        uint32_t b[4];
        const uint32_t byte = ((ks & 3) * 16 + k_col) * 2;
        ldsm4(kb + (ks >> 2) * kHalfBytes + k_row * 128 + (byte ^ ((k_row & 7) << 4)), b);
#pragma unroll
        for (int m = 0; m < kMT; ++m) {
          if constexpr (kMT == 1) {
            mma<kF16>(sc[m][0], qf[ks], b[0], b[1]);
            mma<kF16>(sc[m][1], qf[ks], b[2], b[3]);
          } else {
            uint32_t a[4];
            ldsm4(q_addr + m * 16 * (kD + 8) * 2 + ks * 32, a);
            mma<kF16>(sc[m][0], a, b[0], b[1]);
            mma<kF16>(sc[m][1], a, b[2], b[3]);
          }
        }
      }
      const int key0 = t * kKeys + warp * 16;
      const bool whole = key0 + 16 <= full_keys;
      uint32_t pf[kMT][4];
#pragma unroll
      for (int m = 0; m < kMT; ++m) {
        if (!whole) {
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (key0 + n * 8 + int(lane & 3) * 2 + (e & 1) >= lim[m][e >> 1]) sc[m][n][e] = -INFINITY;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float top = fmaxf(fmaxf(sc[m][0][2 * h], sc[m][0][2 * h + 1]),
                            fmaxf(sc[m][1][2 * h], sc[m][1][2 * h + 1]));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          const float now = fmaxf(mx[m][h], PagedBase<kF16, 0>::of(top, p.scale_log2));
          const float base = now == -INFINITY ? 0.f : now;
          const float keep = ex2_approx(mx[m][h] - base);  // -inf: 0, nothing was kept
          mx[m][h] = now;
          float part = 0.f;
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float& x = sc[m][n][2 * h + e];
              x = ex2_approx(fmaf(x, p.scale_log2, -base));
              part += x;
            }
          sum[m][h] = sum[m][h] * keep + part;
          if (__any_sync(0xffffffffu, keep != 1.f)) {
#pragma unroll
            for (int n = 0; n < kD / 8; ++n) {
              o[m][n][2 * h] *= keep;
              o[m][n][2 * h + 1] *= keep;
            }
          }
        }
        // rounded to 16 bits (PagedBase); the sum above keeps them in fp32
        pf[m][0] = pack16<kF16>(sc[m][0][0], sc[m][0][1]);
        pf[m][1] = pack16<kF16>(sc[m][0][2], sc[m][0][3]);
        pf[m][2] = pack16<kF16>(sc[m][1][0], sc[m][1][1]);
        pf[m][3] = pack16<kF16>(sc[m][1][2], sc[m][1][3]);
      }
      // Values behind the sequence's end may be anything, and 0 * NaN is NaN: they are
      // cut to zero where a tile has any.
      const bool cut = key0 + 16 > u.s.kv;
      uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;
      if (cut) {
        const int a = u.s.kv - key0 - int(lane & 3) * 2;  // keys from this thread's first on
        keep0 = a <= 0 ? 0u : a == 1 ? 0xffffu : 0xffffffffu;
        keep1 = a <= 8 ? 0u : a == 9 ? 0xffffu : 0xffffffffu;
      }
#pragma unroll
      for (int n = 0; n < kD / 16; ++n) {
        uint32_t b[4];
        const uint32_t byte = ((n & 3) * 16 + v_col) * 2;
        ldsm4t(vb + (n >> 2) * kHalfBytes + v_row * 128 + (byte ^ ((v_row & 7) << 4)), b);
        if (cut) {
          b[0] &= keep0;
          b[1] &= keep1;
          b[2] &= keep0;
          b[3] &= keep1;
        }
#pragma unroll
        for (int m = 0; m < kMT; ++m) {
          mma<kF16>(o[m][2 * n], pf[m], b[0], b[1]);
          mma<kF16>(o[m][2 * n + 1], pf[m], b[2], b[3]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.empty[st]);
    }
    // ---- the four warps' results, in the warps' order
#pragma unroll
    for (int m = 0; m < kMT; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        sum[m][h] += __shfl_xor_sync(0xffffffffu, sum[m][h], 1);
        sum[m][h] += __shfl_xor_sync(0xffffffffu, sum[m][h], 2);
        if ((lane & 3) == 0)
          s.ml[warp][m * 16 + h * 8 + (lane >> 2)] = make_float2(mx[m][h], sum[m][h]);
      }
    consumers_sync();
    float weight[kMT][2];
#pragma unroll
    for (int m = 0; m < kMT; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = m * 16 + h * 8 + (lane >> 2);
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < kConsumers; ++i) top = fmaxf(top, s.ml[i][r].x);
        weight[m][h] = ex2_approx(mx[m][h] - (top == -INFINITY ? 0.f : top));
      }
    for (int i = 0; i < kConsumers; ++i) {
      if (int(warp) == i) {
#pragma unroll
        for (int m = 0; m < kMT; ++m)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int r = m * 16 + h * 8 + (lane >> 2);
#pragma unroll
            for (int n = 0; n < kD / 8; ++n) {
              float2* at = reinterpret_cast<float2*>(&s.acc[r][n * 8 + (lane & 3) * 2]);
              float2 v = make_float2(o[m][n][2 * h] * weight[m][h], o[m][n][2 * h + 1] * weight[m][h]);
              if (i > 0) {
                v.x += at->x;
                v.y += at->y;
              }
              *at = v;
            }
          }
      }
      consumers_sync();
    }
    const bool done = at.complete();
    const int64_t slot = at.part();
    for (int i = threadIdx.x; i < kR * (kD / 8); i += kConsumers * 32) {
      const int r = i / (kD / 8), c = (i % (kD / 8)) * 8;
      if (r >= rows || *ab.flag) continue;
      float top = -INFINITY, total = 0.f;
#pragma unroll
      for (int k = 0; k < kConsumers; ++k) top = fmaxf(top, s.ml[k][r].x);
      const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int k = 0; k < kConsumers; ++k) total += s.ml[k][r].y * ex2_approx(s.ml[k][r].x - base);
      const float* a = &s.acc[r][c];
      if (done) {
        const float inv = total == 0.f ? 0.f : 1.f / total;  // 0: no visible key
        const int tok = u.s.q0 + r / p.group, head = u.hk * p.group + r % p.group;
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + int64_t(tok) * p.o_stride_t +
                                  int64_t(head) * p.o_stride_h + c) =
            make_uint4(pack16<kF16>(a[0] * inv, a[1] * inv), pack16<kF16>(a[2] * inv, a[3] * inv),
                       pack16<kF16>(a[4] * inv, a[5] * inv), pack16<kF16>(a[6] * inv, a[7] * inv));
        if (p.lse && c == 0)
          p.lse[int64_t(head) * p.tokens + tok] =
              total == 0.f ? -INFINITY : (base + log2f(total)) * 0.6931471805599453f;
      } else {
        float* dst = p.part_o + (slot * p.unit_rows + r) * kD + c;
        *reinterpret_cast<float4*>(dst) = make_float4(a[0], a[1], a[2], a[3]);
        *reinterpret_cast<float4*>(dst + 4) = make_float4(a[4], a[5], a[6], a[7]);
        if (c == 0) p.part_ml[slot * p.unit_rows + r] = make_float2(top, total);
      }
    }
    if (threadIdx.x == 0) s.stop = *ab.flag;
    consumers_sync();  // q, acc and ml are free again
  } while (!s.stop && at.next(p, prefix));
}

// ---------------------------------------------------------------------- joining the parts
// CTA (c, y): rows [y * kRows, y * kRows + kRows) of the unit that share c began and
// others went on with (join[c]), if there is one. kSplit warps share a row: each first
// finds the row's maximum over all parts (lane i holds part i), then adds every kSplit-th
// part's row, weighted by 2^(m_i - max); the warps' sums are added in order.
constexpr int kMergeWarps = 16;

template <int kD, bool kF16, int kSplit, int kRows>
__global__ void __launch_bounds__(kMergeWarps * 32) paged_merge_kernel(const PagedParams p) {
  constexpr int kE = kD / 32, kAtOnce = kMergeWarps / kSplit;
  __shared__ float sh[kSplit > 1 ? kMergeWarps : 1][kD];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int c = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int4 j = p.join[c];
  const int part = warp % kSplit;
  for (int r0 = blockIdx.y * kRows; r0 < j.z && r0 < int(blockIdx.y + 1) * kRows; r0 += kAtOnce) {
    const int r = r0 + warp / kSplit;
    const bool live = r < j.z;
    auto slot = [&](int i) { return (2 * int64_t(i) + (i == c ? 1 : 0)) * p.unit_rows + r; };
    float top = -INFINITY, total = 0.f, acc[kE];
#pragma unroll
    for (int e = 0; e < kE; ++e) acc[e] = 0.f;
    if (live) {
      for (int i = c + lane; i <= j.w; i += 32) top = fmaxf(top, p.part_ml[slot(i)].x);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float base = top == -INFINITY ? 0.f : top;
      for (int i0 = c; i0 <= j.w; i0 += 32) {
        float2 ml = make_float2(-INFINITY, 0.f);
        if (i0 + lane <= j.w) ml = p.part_ml[slot(i0 + lane)];
        const float wt = ex2_approx(ml.x - base);
        total += ml.y * wt;
        const int n = j.w - i0 + 1 < 32 ? j.w - i0 + 1 : 32;
#pragma unroll 8
        for (int i = part; i < n; i += kSplit) {
          const float f = __shfl_sync(0xffffffffu, wt, i);
          const float* src = p.part_o + slot(i0 + i) * kD + lane * kE;
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
    const float inv = total == 0.f ? 0.f : 1.f / total;
    const int tok = j.x + r / p.group, head = j.y + r % p.group;
    uint16_t* out = static_cast<uint16_t*>(p.out) + int64_t(tok) * p.o_stride_t +
                    int64_t(head) * p.o_stride_h + lane * kE;
    if constexpr (kE == 4)
      *reinterpret_cast<uint2*>(out) =
          make_uint2(pack16<kF16>(acc[0] * inv, acc[1] * inv), pack16<kF16>(acc[2] * inv, acc[3] * inv));
    else
      *reinterpret_cast<uint32_t*>(out) = pack16<kF16>(acc[0] * inv, acc[1] * inv);
    if (p.lse && lane == 0)
      p.lse[int64_t(head) * p.tokens + tok] =
          total == 0.f ? -INFINITY : (base + log2f(total)) * 0.6931471805599453f;
  }
}

void cuda_ok(cudaError_t e) {
  if (e != cudaSuccess) throw std::runtime_error(std::string("paged attention: ") + cudaGetErrorString(e));
}

template <int kD, bool kF16, int kMT>
void decode_launch(const CUtensorMap& mk, const CUtensorMap& mv, const PagedParams& p, cudaStream_t s) {
  const int smem = int(sizeof(DecodeSmem<kD, kMT>)) + 1024 + 4 * (p.seqs + 1);
  auto fn = paged_decode_kernel<kD, kF16, kMT>;
  static std::atomic<uint64_t> allowed{0};
  cuda_ok(paged_allow_smem(fn, allowed));
  fn<<<p.grid, kThreads, smem, s>>>(mk, mv, p);
  cuda_ok(cudaGetLastError());
}

template <int kD, bool kF16>
void decode_rows(const CUtensorMap& mk, const CUtensorMap& mv, const PagedParams& p, cudaStream_t s) {
  if (p.unit_rows <= 16) decode_launch<kD, kF16, 1>(mk, mv, p, s);
  else decode_launch<kD, kF16, 2>(mk, mv, p, s);
}

}  // namespace

void paged_decode_launch(const CUtensorMap& mk, const CUtensorMap& mv, const PagedParams& p,
                         cudaStream_t s) {
  if (p.head_dim == 64) p.fp16 ? decode_rows<64, true>(mk, mv, p, s) : decode_rows<64, false>(mk, mv, p, s);
  else p.fp16 ? decode_rows<128, true>(mk, mv, p, s) : decode_rows<128, false>(mk, mv, p, s);
}

template <int kD, bool kF16>
void merge_launch(const PagedParams& p, cudaStream_t s) {
  // A few rows and up to a part of every share, or many rows and mostly two or three
  // parts.
  const bool few = p.unit_rows <= 32;
  const int rows = few ? 4 : 32;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.grid - 1, (p.unit_rows + rows - 1) / rows);
  cfg.blockDim = dim3(kMergeWarps * 32);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cuda_ok(cudaLaunchKernelEx(&cfg, few ? paged_merge_kernel<kD, kF16, 4, 4> : paged_merge_kernel<kD, kF16, 1, 32>, p));
}

void paged_merge_launch(const PagedParams& p, cudaStream_t s) {
  if (p.head_dim == 64) p.fp16 ? merge_launch<64, true>(p, s) : merge_launch<64, false>(p, s);
  else p.fp16 ? merge_launch<128, true>(p, s) : merge_launch<128, false>(p, s);
}

}  // namespace mgfa
