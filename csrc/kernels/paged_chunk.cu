// Attention of a chunk of new tokens over a paged cache on the tensor cores
// (tcgen05 + TMEM + TMA).
//
// A unit packs up to 256 rows (token, query head) of one key head in two 128-row
// tiles, so that grouped heads and short chunks fill the tiles: row r of a tile is
// token r / group, head r % group, one TMA box of [tokens, group heads, 64 columns].
// K and V tiles are 128 keys, one box per page (or per 128 keys of a larger page).
//   warps 0-3, 4-7  softmax of tile 0, 1 (thread t owns row t / TMEM lane t)
//   warp 8          TMA producer: Q of a unit, K and V through two stages each
//   warp 9          MMA: S_t = Q_t K^T (both operands in shared memory), O_t += P_t V
//                   (P read from TMEM, where it overwrote S)
// TMEM (512 columns): S0/P0 [0, 128), S1/P1 [128, 256), O0 and O1 from 256.
// While one tile's softmax runs, the tensor cores work for the other; a CTA runs its
// whole share of the work (paged_attn.cuh) through the same barriers, so the next
// unit's Q, K and first scores are under way during a unit's epilogue.
// Bound by the tensor cores and the exponentials for long chunks, and by memory when a
// unit has few rows.
// O is rescaled only when the running maximum grows by more than 2^8: with the stale
// one P stays below 2^8, whose 16-bit rounding is relative, and sums are fp32.
#include "paged_attn.cuh"
#include "sm100_ptx.cuh"
#include "softmax_exp.cuh"

#include <stdexcept>
#include <string>

namespace mgfa {
namespace {

using namespace mgfa::dev;

constexpr int kTile = 128;
constexpr int kHalfBytes = kTile * 64 * 2;  // one 128 x 64 16-bit swizzled box
constexpr int kWarps = 10;
constexpr int kThreads = kWarps * 32;
constexpr float kRescaleThreshold = 8.0f;   // log2 units

template <int kD>
struct __align__(1024) ChunkSmem {
  static constexpr int kHalves = kD / 64;
  uint16_t q[2][kHalves][kTile * 64];  // [tile][64 columns]
  uint16_t k[2][kHalves][kTile * 64];  // [stage][64 columns]
  uint16_t v[2][kHalves][kTile * 64];
  uint64_t q_full, q_empty;
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2];
  uint64_t s_full[2], p_full[2], o_full[2];
  uint64_t drain;
  uint32_t tmem_base;
  uint32_t abort_flag;
  uint32_t sums[kWarps];
  PagedUnit unit[8];  // of the softmax warps, whose registers hold scores
};

template <int kD, bool kF16>
__global__ void __launch_bounds__(kThreads, 1)
    paged_chunk_kernel(const __grid_constant__ CUtensorMap map_q,
                       const __grid_constant__ CUtensorMap map_k,
                       const __grid_constant__ CUtensorMap map_v, const PagedParams p) {
  constexpr int kHalves = kD / 64;
  constexpr int kKSteps = kD / 16;  // MMA steps of S = Q K^T
  constexpr int kOChunks = kD / 32;
  constexpr uint32_t kOCol = 256;
  extern __shared__ uint8_t smem_raw[];
  ChunkSmem<kD>& s = *reinterpret_cast<ChunkSmem<kD>*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint32_t* prefix = reinterpret_cast<uint32_t*>(&s + 1);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t warp = warp_id(), lane = lane_id();
  AbortState ab{&s.abort_flag, p.status, p.wait_limit_ns};
  if (threadIdx.x == 0) {
    s.abort_flag = 0;
    mbar_init(&s.q_full, 1);
    mbar_init(&s.q_empty, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.k_full[i], 1);
      mbar_init(&s.k_empty[i], 1);
      mbar_init(&s.v_full[i], 1);
      mbar_init(&s.v_empty[i], 1);
      mbar_init(&s.s_full[i], 1);
      mbar_init(&s.p_full[i], 4);  // one arrival per softmax warp
      mbar_init(&s.o_full[i], 1);
    }
    mbar_init(&s.drain, 1);
    fence_mbar_init();
  }
  paged_prefix<kThreads>(p, prefix, s.sums);
  const PagedShare share(p, prefix);
  PagedUnit u, behind;
  const uint64_t begin = share.begin(blockIdx.x, u), end = share.begin(blockIdx.x + 1, behind);
  if (begin >= end) {  // the whole CTA
    if (threadIdx.x == 0) paged_join(share, u, false, begin, end);
    return;
  }
  if (warp == 0) tmem_alloc<512>(&s.tmem_base);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s.tmem_base;
  const int tile_tokens = p.block_tokens / 2;

  if (warp == 8) {
    // ------------------------------------------------------------ TMA producer
    if (lane == 0) {
      tma_prefetch_desc(&map_q);
      tma_prefetch_desc(&map_k);
      tma_prefetch_desc(&map_v);
    }
    const int chunk = p.page < kTile ? p.page : kTile;  // keys of one box
    const uint32_t q_bytes = uint32_t(tile_tokens * p.group * kD * 2);
    uint32_t it = 0, seg = 0;
    bool ok = true;
    for (uint64_t w = begin; ok && w < end; ++seg) {
      const int t0 = int(w - u.first);
      const int t1 = end - u.first < uint64_t(u.tiles) ? int(end - u.first) : u.tiles;
      const int tok0 = u.unit * p.block_tokens;
      const int tiles = u.s.n - tok0 > tile_tokens ? 2 : 1;
      ok = __all_sync(0xffffffffu, mbar_wait(&s.q_empty, (seg & 1) ^ 1, ab, 70));
      if (!ok) break;
      if (lane == 0) {
        mbar_arrive_expect_tx(&s.q_full, tiles * q_bytes);
        for (int t = 0; t < tiles; ++t)
          for (int hf = 0; hf < kHalves; ++hf)
            tma_load_4d(s.q[t][hf], &map_q, &s.q_full, hf * 64, u.hk * p.group,
                        u.s.q0 + tok0 + t * tile_tokens, 0);
      }
      const int* row = p.page_table + int64_t(u.s.row) * p.table_stride;
      for (int j = t0; j < t1; ++j, ++it) {
        const int st = it & 1;
        const uint32_t ph = ((it >> 1) & 1) ^ 1;
        // boxes that hold a key below kv; the others' keys are masked, their values cut
        const int left = u.s.kv - j * kTile;
        const int boxes = left <= 0 ? 0 : ((left < kTile ? left : kTile) + chunk - 1) / chunk;
        const uint32_t bytes = uint32_t(boxes * chunk * kD * 2);
        const int key = j * kTile + int(lane) * chunk;
        int page = 0;
        if (int(lane) < boxes) {
          page = __ldg(row + key / p.page);
          if (page < 0 || page >= p.pages) {
            record_error(p.status, kErrBadArgument, 62, 0);
            page = p.pages;  // outside the map: the box reads zeros
          }
        }
        if (!(ok = __all_sync(0xffffffffu, mbar_wait(&s.k_empty[st], ph, ab, 71)))) break;
        if (lane == 0) mbar_arrive_expect_tx(&s.k_full[st], bytes);
        __syncwarp();
        if (int(lane) < boxes)
          for (int hf = 0; hf < kHalves; ++hf)
            tma_load_4d(&s.k[st][hf][lane * chunk * 64], &map_k, &s.k_full[st], hf * 64,
                        key % p.page, u.hk, page);
        __syncwarp();
        if (!(ok = __all_sync(0xffffffffu, mbar_wait(&s.v_empty[st], ph, ab, 72)))) {
          // K of this tile is on its way all the same
          volatile uint32_t never = 0;
          AbortState drain{&never, nullptr, p.wait_limit_ns};
          mbar_wait(&s.k_full[st], (it >> 1) & 1, drain, 0);
          break;
        }
        if (lane == 0) mbar_arrive_expect_tx(&s.v_full[st], bytes);
        __syncwarp();
        if (int(lane) < boxes)
          for (int hf = 0; hf < kHalves; ++hf)
            tma_load_4d(&s.v[st][hf][lane * chunk * 64], &map_v, &s.v_full[st], hf * 64,
                        key % p.page, u.hk, page);
        __syncwarp();
      }
      if (!ok) {
        ++seg;  // this unit's Q is on its way
        break;
      }
      w = u.first + uint32_t(t1);
      if (w < end) paged_next(p, prefix, u);
    }
    if (lane == 0) paged_join(share, u, true, begin, end);
    // Never leave with a copy outstanding.
    volatile uint32_t never = 0;
    AbortState drain{&never, nullptr, p.wait_limit_ns};
    if (seg > 0) mbar_wait(&s.q_full, (seg - 1) & 1, drain, 0);
    for (uint32_t i = it > 2 ? it - 2 : 0; i < it; ++i) {
      mbar_wait(&s.k_full[i & 1], (i >> 1) & 1, drain, 0);
      mbar_wait(&s.v_full[i & 1], (i >> 1) & 1, drain, 0);
    }
  } else if (warp == 9) {
    // ------------------------------------------------------------ MMA issuer
    const uint32_t idesc_s = make_idesc_16(128, 128, 0, 0, kF16);
    const uint32_t idesc_o = make_idesc_16(128, kD, 0, 1, kF16);
    auto issue_s = [&](int t, int st) {
      const uint32_t qb = smem_u32(s.q[t][0]), kb = smem_u32(s.k[st][0]);
#pragma unroll
      for (int kk = 0; kk < kKSteps; ++kk) {
        const uint32_t off = (kk >> 2) * kHalfBytes + (kk & 3) * 32;
        mma_ss(tmem + t * 128, make_sdesc_sw128(qb + off, 16, 1024),
               make_sdesc_sw128(kb + off, 16, 1024), idesc_s, kk > 0);
      }
    };
    auto issue_o = [&](int t, int st, uint32_t acc) {
      const uint32_t vb = smem_u32(s.v[st][0]);
#pragma unroll
      for (int kk = 0; kk < 8; ++kk)  // 128 keys, 16 a step
        mma_ts(tmem + kOCol + t * kD, tmem + t * 128 + kk * 8,
               make_sdesc_sw128(vb + kk * 2048, kHalfBytes, 1024), idesc_o,
               (acc || kk > 0) ? 1u : 0u);
    };
    auto wait = [&](uint64_t* bar, uint32_t parity, uint32_t site) {
      return bool(__all_sync(0xffffffffu, mbar_wait(bar, parity, ab, site)));
    };
    uint32_t it = 0, seg = 0, pc[2] = {0, 0};  // phases used so far
    bool ok = true;
    for (uint64_t w = begin; ok && w < end; ++seg) {
      const int t0 = int(w - u.first);
      const int t1 = end - u.first < uint64_t(u.tiles) ? int(end - u.first) : u.tiles;
      const bool two = u.s.n - u.unit * p.block_tokens > tile_tokens;
      if (!(ok = wait(&s.q_full, seg & 1, 80))) break;
      if (!(ok = wait(&s.k_full[it & 1], (it >> 1) & 1, 81))) break;
      tc_fence_after();
      if (lane == 0) {
        issue_s(0, it & 1);
        mma_commit(&s.s_full[0]);
        if (two) {
          issue_s(1, it & 1);
          mma_commit(&s.s_full[1]);
        }
        mma_commit(&s.k_empty[it & 1]);
        if (t0 + 1 == t1) mma_commit(&s.q_empty);
      }
      for (int j = t0; j < t1; ++j, ++it) {
        const int st = it & 1, st1 = st ^ 1;
        const uint32_t ph = (it >> 1) & 1, ph1 = ((it + 1) >> 1) & 1;
        const bool more = j + 1 < t1;
        if (!(ok = wait(&s.v_full[st], ph, 82))) break;
        const int left = u.s.kv - j * kTile;
        if (left < kTile) {
          // Values behind the sequence's end may be anything, and 0 * NaN is NaN. Swizzling
          // stays within a 128-byte row, so rows [left, 128) are one run of each half.
          const int from = (left < 0 ? 0 : left) * 8;  // 16-byte pieces
          for (int hf = 0; hf < kHalves; ++hf)
            for (int i = from + int(lane); i < kTile * 8; i += 32)
              reinterpret_cast<uint4*>(s.v[st][hf])[i] = make_uint4(0, 0, 0, 0);
          fence_proxy_async_smem();
          __syncwarp();
        }
        // A unit's first P_t also says that all four warps have read the last unit's O_t.
        if (!(ok = wait(&s.p_full[0], pc[0] & 1, 85))) break;
        ++pc[0];
        tc_fence_after();
        if (lane == 0) issue_o(0, st, j > t0);
        if (more) {
          if (!(ok = wait(&s.k_full[st1], ph1, 86))) break;
          tc_fence_after();
          if (lane == 0) {
            issue_s(0, st1);
            mma_commit(&s.s_full[0]);
          }
        } else if (lane == 0) {
          mma_commit(&s.o_full[0]);
        }
        if (two) {
          if (!(ok = wait(&s.p_full[1], pc[1] & 1, 87))) break;
          ++pc[1];
          tc_fence_after();
          if (lane == 0) issue_o(1, st, j > t0);
        }
        if (lane == 0) {
          mma_commit(&s.v_empty[st]);
          if (more) {
            if (two) {
              issue_s(1, st1);
              mma_commit(&s.s_full[1]);
            }
            mma_commit(&s.k_empty[st1]);
            if (j + 2 == t1) mma_commit(&s.q_empty);
          } else if (two) {
            mma_commit(&s.o_full[1]);
          }
        }
        __syncwarp();
      }
      if (!ok) break;
      w = u.first + uint32_t(t1);
      if (w < end) paged_next(p, prefix, u);
    }
    // Every issued MMA has finished before TMEM is released.
    if (lane == 0) {
      mma_commit(&s.drain);
      volatile uint32_t never = 0;
      AbortState drain{&never, nullptr, p.wait_limit_ns};
      mbar_wait(&s.drain, 0, drain, 0);
    }
  } else {
    // ------------------------------------------------------------ softmax, epilogue
    const int t = warp >> 2;
    const int r = threadIdx.x & 127;  // row of the tile, TMEM lane
    const uint32_t lane_off = uint32_t((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem + lane_off + t * 128;
    const uint32_t o_addr = tmem + lane_off + kOCol + t * kD;
    PagedUnit& su = s.unit[warp];
    if (lane == 0) su = u;
    __syncwarp();
    uint32_t sc = 0, oc = 0;  // phases used so far
    bool ok = true;
    for (uint64_t w = begin; ok && w < end;) {
      const int t0 = int(w - su.first);
      const int t1 = end - su.first < uint64_t(su.tiles) ? int(end - su.first) : su.tiles;
      const int tok0 = su.unit * p.block_tokens + t * tile_tokens;  // this tile's first token
      if (su.s.n > tok0) {
        // keys that this row sees, and those that the tile's first row, hence each, does
        const int n = su.s.n, kv = su.s.kv;
        const int tok = tok0 + r / p.group;
        int lim = p.causal ? kv - n + tok + 1 : kv;
        lim = r >= tile_tokens * p.group || tok >= n ? 0 : lim < kv ? lim : kv;
        int full = p.causal ? kv - n + tok0 + 1 : kv;
        full = full < kv ? full : kv;
        float m = -INFINITY, l = 0.f;
        for (int j = t0; j < t1; ++j) {
          ok = __all_sync(0xffffffffu, mbar_wait(&s.s_full[t], sc & 1, ab, 90 + t));
          if (!ok) break;
          ++sc;
          tc_fence_after();
          uint32_t sr[128];
          tmem_ld64_sync(s_addr, &sr[0]);
          tmem_ld64_sync(s_addr + 64, &sr[64]);
          if ((j + 1) * kTile > full) {
            const int n_vis = lim - j * kTile;
#pragma unroll
            for (int c = 0; c < 128; ++c)
              if (c >= n_vis) sr[c] = 0xff800000u;  // -inf
          }
          const float m_new = fmaxf(m, row_max<128>(sr) * p.scale_log2);
          float alpha = 1.f;
          bool rescale = false;
          if (j == t0) {
            m = m_new;
          } else if (m_new > m + kRescaleThreshold) {
            alpha = ex2_approx(m - m_new);
            m = m_new;
            rescale = true;
          }
          const float neg_m = m == -INFINITY ? 0.f : -m;
          l *= alpha;
          uint32_t pk[2][32];
          float lacc[4] = {0.f, 0.f, 0.f, 0.f};
          exp_half<kF16, 0, true>(sr, 0, p.scale_log2, neg_m, pk[0], lacc);
          tmem_st32(s_addr, pk[0]);
          exp_half<kF16, 0, true>(sr, 1, p.scale_log2, neg_m, pk[1], lacc);
          tmem_st32(s_addr + 32, pk[1]);
          l += (lacc[0] + lacc[1]) + (lacc[2] + lacc[3]);
          // S(j) was issued behind PV(j - 1), and its barrier has completed: O is at rest
          if (__any_sync(0xffffffffu, rescale)) {
#pragma unroll
            for (int ch = 0; ch < kOChunks; ++ch) {
              uint32_t orow[32];
              tmem_ld32_sync(o_addr + ch * 32, orow);
#pragma unroll
              for (int c = 0; c < 32; ++c)
                orow[c] = __float_as_uint(__uint_as_float(orow[c]) * alpha);
              tmem_st32_sync(o_addr + ch * 32, orow);
            }
          }
          tmem_wait_st();
          regs_live32(pk[0]);
          regs_live32(pk[1]);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s.p_full[t]);
        }
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&s.o_full[t], oc & 1, ab, 92 + t));
        if (!ok) break;
        ++oc;
        tc_fence_after();
        const bool done = t0 == 0 && t1 == su.tiles;
        const bool valid = r < tile_tokens * p.group && tok < su.s.n;
        const float scale = !done ? 1.f : l == 0.f ? 0.f : 1.f / l;
        const int r_head = r % p.group;
        const int64_t row_tok = su.s.q0 + tok, head = int64_t(su.hk) * p.group + r_head;
        const int64_t slot = 2 * int64_t(blockIdx.x) + (t0 > 0 ? 0 : 1);
        const int64_t part = slot * p.unit_rows + (tok - su.unit * p.block_tokens) * p.group + r_head;
#pragma unroll
        for (int ch = 0; ch < kOChunks; ++ch) {
          uint32_t orow[32];
          tmem_ld32_sync(o_addr + ch * 32, orow);
          if (!valid) continue;
          if (done) {
            uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) +
                                                  row_tok * p.o_stride_t + head * p.o_stride_h + ch * 32);
            float v[32];
#pragma unroll
            for (int c = 0; c < 32; ++c) v[c] = __uint_as_float(orow[c]) * scale;
#pragma unroll
            for (int c = 0; c < 4; ++c)
              dst[c] = make_uint4(pack16<kF16>(v[8 * c], v[8 * c + 1]), pack16<kF16>(v[8 * c + 2], v[8 * c + 3]),
                                  pack16<kF16>(v[8 * c + 4], v[8 * c + 5]), pack16<kF16>(v[8 * c + 6], v[8 * c + 7]));
          } else {
            uint4* dst = reinterpret_cast<uint4*>(p.part_o + part * kD + ch * 32);
#pragma unroll
            for (int c = 0; c < 8; ++c)
              dst[c] = make_uint4(orow[4 * c], orow[4 * c + 1], orow[4 * c + 2], orow[4 * c + 3]);
          }
        }
        if (valid) {
          if (!done) p.part_ml[part] = make_float2(m, l);
          else if (p.lse)
            p.lse[head * p.tokens + row_tok] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
        }
      }
      w = su.first + uint32_t(t1);
      __syncwarp();
      if (w < end && lane == 0) paged_next(p, prefix, su);
      __syncwarp();
    }
  }
  // ---- teardown
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 0) tmem_dealloc<512>(tmem);
}

template <int kD, bool kF16>
void chunk_launch(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv,
                  const PagedParams& p, cudaStream_t s) {
  const int smem = int(sizeof(ChunkSmem<kD>)) + 1024 + 4 * (p.seqs + 1);
  auto fn = paged_chunk_kernel<kD, kF16>;
  cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess) {
    fn<<<p.grid, kThreads, smem, s>>>(mq, mk, mv, p);
    e = cudaGetLastError();
  }
  if (e != cudaSuccess) throw std::runtime_error(std::string("paged attention: ") + cudaGetErrorString(e));
}

}  // namespace

void paged_chunk_launch(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv,
                        const PagedParams& p, cudaStream_t s) {
  if (p.head_dim == 64) p.fp16 ? chunk_launch<64, true>(mq, mk, mv, p, s) : chunk_launch<64, false>(mq, mk, mv, p, s);
  else p.fp16 ? chunk_launch<128, true>(mq, mk, mv, p, s) : chunk_launch<128, false>(mq, mk, mv, p, s);
}

}  // namespace mgfa
