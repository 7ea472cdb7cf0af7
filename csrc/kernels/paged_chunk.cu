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
// While one tile's softmax runs, the tensor cores work for the other. A unit of one tile
// (up to 128 rows) gives both halves work all the same: they take its even and odd key
// tiles, each with a maximum, sum and O of its own, which the first joins from TMEM. A
// CTA runs its whole share of the work (paged_attn.cuh) through the same barriers, so
// the next unit's Q, K and first scores are under way during a unit's epilogue.
// Bound by a tile's way from scores to probabilities to the next scores: the softmax of
// 128 keys takes 1.25 us, the two products and their hand-overs 1.1 us, so a key tile of
// both halves takes 2.4 us where the tensor cores alone would need 1.5 us. 2048 tokens of
// 32 heads over 32768 keys (8 key heads of 128, causal) take 1.06 ms, 1.01 PFLOP/s, and
// 1.25 ms (0.85) under the power cap of a long run. Units of few rows are bound by the same
// chain, with two tiles of K and V on their way, and not by memory: 16 tokens of 8 sequences
// over 8192 keys take 87 us for 268 MB, 3.1 TB/s, where the decode kernel reaches 6.3. So do
// single tokens that share a call with a chunk: 512 tokens and 60 sequences of one over 4096
// keys take 329 us together, 77 and 179 us (on the decode kernel) apart.
// O is rescaled only when the running maximum grows by more than 2^8 (fp16: 2^4, which
// leaves 2^11 for PagedBase's lift): with the stale one P stays below 2^8 (2^15). Sums are
// fp32.
#include "paged_attn.cuh"
#include "sm100_ptx.cuh"
#include "softmax_exp.cuh"

#include <algorithm>
#include <stdexcept>
#include <string>

namespace mgfa {
namespace {

using namespace mgfa::dev;

constexpr int kTile = 128;
constexpr int kHalfBytes = kTile * 64 * 2;  // one 128 x 64 16-bit swizzled box
constexpr int kWarps = 10;
constexpr int kThreads = kWarps * 32;
// How far the running maximum may lag, in powers of two.
constexpr int stale(bool f16) { return f16 ? 4 : 8; }

template <int kD>
struct __align__(1024) ChunkSmem {
  static constexpr int kHalves = kD / 64;
  uint16_t q[2][kHalves][kTile * 64];  // [tile][64 columns]
  uint16_t k[2][kHalves][kTile * 64];  // [stage][64 columns]
  uint16_t v[2][kHalves][kTile * 64];
  // Of each softmax warp: 64 bytes of its 32 rows. When the halves join, a warp of the
  // second writes no rows, and leaves their (maximum, sum) here.
  uint4 out[8][32][4];
  uint64_t q_full, q_empty;
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2];
  uint64_t s_full[2], p_full[2], o_full[2], x_full, x_empty;
  uint64_t drain;
  uint32_t tmem_base;
  uint32_t abort_flag;
  uint32_t never;  // 0: the flag of the last waits, which nothing ends early
  uint32_t sums[kWarps];
  // The runs, which the producer finds a few ahead: run number i in slot i & 3.
  struct Run {
    PagedSeq s;
    int hk, unit, t0, t1, complete, part;  // t1 < 0: there is none
  } runs[4];
  uint64_t run_full[4], run_empty[4];
};

// A warp's 32 rows of 64 bytes, one per lane, to the rows' places: through shared memory,
// so that four lanes write 64 bytes in a row at once (a lane writing its own row touches
// 32 lines with each store, which took longer than the softmax of two key tiles).
__device__ __forceinline__ void store_rows(uint4 (&stage)[32][4], const uint4 (&v)[4], uint32_t lane,
                                           uint8_t* row_at, bool valid) {
#pragma unroll
  for (int i = 0; i < 4; ++i) stage[lane][i ^ ((lane >> 1) & 3)] = v[i];
  __syncwarp();
  const uint64_t at = valid ? reinterpret_cast<uint64_t>(row_at) : 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t row = i * 8 + (lane >> 2), piece = lane & 3;
    const uint64_t to = __shfl_sync(0xffffffffu, at, row);
    if (to) *reinterpret_cast<uint4*>(to + piece * 16) = stage[row][piece ^ ((row >> 1) & 3)];
  }
  __syncwarp();
}

// Scores [n, 64) to -inf; n is 64 or more in most tiles.
__device__ __forceinline__ void hide(uint32_t (&sr)[64], int n) {
  if (__any_sync(0xffffffffu, n < 64)) {
#pragma unroll
    for (int c = 0; c < 64; ++c)
      if (c >= n) sr[c] = 0xff800000u;
  }
}

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
    s.abort_flag = s.never = 0;
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
    for (int i = 0; i < 4; ++i) {
      mbar_init(&s.run_full[i], 1);
      mbar_init(&s.run_empty[i], 9);  // the MMA's and the softmax's warps
    }
    mbar_init(&s.x_full, 4);
    mbar_init(&s.x_empty, 4);
    mbar_init(&s.drain, 1);
    fence_mbar_init();
  }
  PagedWalk at;
  if (!at.start<kThreads>(p, prefix, s.sums)) return;  // the whole CTA
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
    uint32_t it = 0, seg = 0, run = 0;
    auto publish = [&](int t1) {
      const bool free = __all_sync(0xffffffffu, mbar_wait(&s.run_empty[run & 3], ((run >> 2) & 1) ^ 1, ab, 73));
      if (free && lane == 0) {
        auto& r = s.runs[run & 3];
        r.s = at.u.s;
        r.hk = at.u.hk;
        r.unit = at.u.unit;
        r.t0 = at.t0;
        r.t1 = t1;
        r.complete = at.complete();
        r.part = int(at.part());
        mbar_arrive(&s.run_full[run & 3]);
      }
      ++run;
      return free;
    };
    bool ok = true;
    do {
      const PagedUnit& u = at.u;
      const int tok0 = u.unit * p.block_tokens;
      const int tiles = u.s.n - tok0 > tile_tokens ? 2 : 1;
      if (!(ok = publish(at.t1))) break;
      ok = __all_sync(0xffffffffu, mbar_wait(&s.q_empty, (seg & 1) ^ 1, ab, 70));
      if (!ok) break;
      ++seg;
      if (lane == 0) {
        mbar_arrive_expect_tx(&s.q_full, tiles * q_bytes);
        for (int t = 0; t < tiles; ++t)
          for (int hf = 0; hf < kHalves; ++hf)
            tma_load_4d(s.q[t][hf], &map_q, &s.q_full, hf * 64, u.hk * p.group,
                        u.s.q0 + tok0 + t * tile_tokens, 0);
      }
      const int* row = p.page_table + int64_t(u.s.row) * p.table_stride;
      for (int j = at.t0; j < at.t1; ++j, ++it) {
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
          AbortState drain{&s.never, nullptr, p.wait_limit_ns};
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
    } while (ok && at.next(p, prefix));
    if (ok) publish(-1);
    if (lane == 0) at.leave(p, prefix);
    // Never leave with a copy outstanding.
    AbortState drain{&s.never, nullptr, p.wait_limit_ns};
    if (seg > 0) mbar_wait(&s.q_full, (seg - 1) & 1, drain, 0);
    for (uint32_t i = it > 2 ? it - 2 : 0; i < it; ++i) {
      mbar_wait(&s.k_full[i & 1], (i >> 1) & 1, drain, 0);
      mbar_wait(&s.v_full[i & 1], (i >> 1) & 1, drain, 0);
    }
  } else if (warp == 9) {
    uint32_t run = 0;
    // ------------------------------------------------------------ MMA issuer
    const uint32_t idesc_s = make_idesc_16(128, 128, 0, 0, kF16);
    const uint32_t idesc_o = make_idesc_16(128, kD, 0, 1, kF16);
    // S_t = Q_qt K(stage)^T, then its barriers
    auto issue_s = [&](int t, int qt, int st, bool k_done, bool q_done) {
      if (lane == 0) {
        const uint32_t qb = smem_u32(s.q[qt][0]), kb = smem_u32(s.k[st][0]);
#pragma unroll
        for (int kk = 0; kk < kKSteps; ++kk) {
          const uint32_t off = (kk >> 2) * kHalfBytes + (kk & 3) * 32;
          mma_ss(tmem + t * 128, make_sdesc_sw128(qb + off, 16, 1024),
                 make_sdesc_sw128(kb + off, 16, 1024), idesc_s, kk > 0);
        }
        mma_commit(&s.s_full[t]);
        if (k_done) mma_commit(&s.k_empty[st]);
        if (q_done) mma_commit(&s.q_empty);
      }
    };
    auto issue_o = [&](int t, int st, bool acc, bool v_done, bool o_done) {
      if (lane == 0) {
        const uint32_t vb = smem_u32(s.v[st][0]);
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)  // 128 keys, 16 a step
          mma_ts(tmem + kOCol + t * kD, tmem + t * 128 + kk * 8,
                 make_sdesc_sw128(vb + kk * 2048, kHalfBytes, 1024), idesc_o,
                 (acc || kk > 0) ? 1u : 0u);
        if (v_done) mma_commit(&s.v_empty[st]);
        if (o_done) mma_commit(&s.o_full[t]);
      }
    };
    auto wait = [&](uint64_t* bar, uint32_t parity, uint32_t site) {
      const bool ok = __all_sync(0xffffffffu, mbar_wait(bar, parity, ab, site));
      tc_fence_after();
      return ok;
    };
    uint32_t it = 0, seg = 0, pc0 = 0, pc1 = 0;  // phases used so far
    bool ok = true;
    // K tile number i has arrived; V tile number i has, and is cut behind the sequence's end
    auto wait_k = [&](uint32_t i) { return wait(&s.k_full[i & 1], (i >> 1) & 1, 81); };
    auto wait_v = [&](uint32_t i, int left) {
      if (!wait(&s.v_full[i & 1], (i >> 1) & 1, 82)) return false;
      if (left < kTile) {
        // Values behind the end may be anything, and 0 * NaN is NaN. Swizzling stays
        // within a 128-byte row, so rows [left, 128) are one run of each half.
        const int from = (left < 0 ? 0 : left) * 8;  // 16-byte pieces
        for (int hf = 0; hf < kHalves; ++hf)
          for (int x = from + int(lane); x < kTile * 8; x += 32)
            reinterpret_cast<uint4*>(s.v[i & 1][hf])[x] = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
        __syncwarp();
      }
      return true;
    };
    // A unit's first P_t also says that the warps have read the last unit's O_t.
    auto wait_p = [&](int t) {
      const uint32_t used = t ? pc1++ : pc0++;
      return wait(&s.p_full[t], used & 1, 85 + t);
    };
    for (;; ++run) {
      if (!(ok = wait(&s.run_full[run & 3], (run >> 2) & 1, 88))) break;
      const auto& u = s.runs[run & 3];
      const int t0 = u.t0, t1 = u.t1, kv = u.s.kv;
      const bool two = u.s.n - u.unit * p.block_tokens > tile_tokens;
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.run_empty[run & 3]);
      if (t1 < 0) break;
      if (!(ok = wait(&s.q_full, seg++ & 1, 80) && wait_k(it))) break;
      if (two) {
        issue_s(0, 0, it & 1, false, false);
        issue_s(1, 1, it & 1, true, t0 + 1 == t1);
        for (int j = t0; j < t1; ++j, ++it) {
          const int st = it & 1;
          const bool more = j + 1 < t1;
          if (!(ok = wait_v(it, kv - j * kTile) && wait_p(0))) break;
          issue_o(0, st, j > t0, false, !more);
          if (more) {
            if (!(ok = wait_k(it + 1))) break;
            issue_s(0, 0, st ^ 1, false, false);
          }
          if (!(ok = wait_p(1))) break;
          issue_o(1, st, j > t0, true, !more);
          if (more) issue_s(1, 1, st ^ 1, true, j + 2 == t1);
        }
      } else {
        // Tile j goes to half (j - t0) & 1.
        issue_s(0, 0, it & 1, true, t0 + 1 == t1);
        if (t0 + 1 < t1) {
          if (!(ok = wait_k(it + 1))) break;
          issue_s(1, 0, (it + 1) & 1, true, t0 + 2 == t1);
        }
        for (int j = t0; j < t1; ++j, ++it) {
          const int t = (j - t0) & 1, st = it & 1;
          const bool more = j + 2 < t1;
          if (!(ok = wait_v(it, kv - j * kTile) && wait_p(t))) break;
          issue_o(t, st, j - t0 >= 2, true, !more);
          if (more) {
            if (!(ok = wait_k(it + 2))) break;
            issue_s(t, 0, st, true, j + 3 == t1);
          }
        }
      }
      if (!ok) break;
    }
    // Every issued MMA has finished before TMEM is released.
    if (lane == 0) {
      mma_commit(&s.drain);
      AbortState drain{&s.never, nullptr, p.wait_limit_ns};
      mbar_wait(&s.drain, 0, drain, 0);
    }
  } else {
    // ------------------------------------------------------------ softmax, epilogue
    const int t = warp >> 2;
    const int r = threadIdx.x & 127;  // row of the tile, TMEM lane
    const uint32_t lane_off = uint32_t((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem + lane_off + t * 128;
    const uint32_t o_addr = tmem + lane_off + kOCol + t * kD;
    float2* const other = reinterpret_cast<float2*>(s.out[4 + (warp & 3)]);  // by lane
    uint32_t sc = 0, oc = 0, xc = 0, run = 0;  // phases used so far
    auto wait = [&](uint64_t* bar, uint32_t parity, uint32_t site) {
      const bool ok = __all_sync(0xffffffffu, mbar_wait(bar, parity, ab, site));
      tc_fence_after();
      return ok;
    };
    bool ok = true;
    for (;; ++run) {
      if (!(ok = wait(&s.run_full[run & 3], (run >> 2) & 1, 96))) break;
      const auto& u = s.runs[run & 3];
      const int n = u.s.n, kv = u.s.kv, t0 = u.t0, t1 = u.t1;
      if (t1 < 0) break;
      const bool two = n - u.unit * p.block_tokens > tile_tokens;
      const int tok0 = u.unit * p.block_tokens + (two ? t * tile_tokens : 0);
      const int j0 = two ? t0 : t0 + t, step = two ? 1 : 2;  // this half's key tiles
      float m = -INFINITY, l = 0.f;
      {
        // keys that this row sees, and those that the tile's first row, hence each, does
        const int tok = tok0 + r / p.group;
        int lim = p.causal ? kv - n + tok + 1 : kv;
        lim = r >= tile_tokens * p.group || tok >= n ? 0 : lim < kv ? lim : kv;
        int full = p.causal ? kv - n + tok0 + 1 : kv;
        full = full < kv ? full : kv;
        for (int j = j0; j < t1; j += step) {
          if (!(ok = wait(&s.s_full[t], sc & 1, 90 + t))) break;
          ++sc;
          // Keys [64, 128) are read twice, for the maximum and for the exponentials, and 64
          // scores are held at a time, which leaves registers to spare. (flash_fwd_sm100.cu
          // holds a row's 128, reads them once, and spills nothing in 168 registers.) Nothing
          // here may spill: a register that tcgen05.ld is still writing was seen to
          // be spilled before its wait, which left other kernels' values in it. (The launch
          // refuses a kernel that has any local memory.)
          // (The probabilities of keys [64, 128) go where scores of [32, 64) lie, so they are
          // stored last.)
          const int n_vis = (j + 1) * kTile > full ? lim - j * kTile : kTile;
          uint32_t sr[64], pk[2][32];
          tmem_ld64_sync(s_addr + 64, sr);
          hide(sr, n_vis - 64);
          float m_new = row_max<64>(sr);
          tmem_ld64_sync(s_addr, sr);
          hide(sr, n_vis);
          m_new = fmaxf(m, PagedBase<kF16, stale(kF16)>::of(fmaxf(m_new, row_max<64>(sr)), p.scale_log2));
          float alpha = 1.f;
          bool rescale = false;
          if (j == j0) {
            m = m_new;
          } else if (kF16 ? m_new - m > stale(kF16) : m_new > m + stale(kF16)) {
            alpha = ex2_approx(m - m_new);
            m = m_new;
            rescale = true;
          }
          // S_t was issued behind the last PV_t, and its barrier has completed: O_t is at rest
          if (__any_sync(0xffffffffu, rescale)) {
#pragma unroll 1
            for (int ch = 0; ch < kOChunks; ++ch) {
              uint32_t orow[32];
              tmem_ld32_sync(o_addr + ch * 32, orow);
#pragma unroll
              for (int c = 0; c < 32; ++c)
                orow[c] = __float_as_uint(__uint_as_float(orow[c]) * alpha);
              tmem_st32_sync(o_addr + ch * 32, orow);
            }
          }
          const float neg_m = m == -INFINITY ? 0.f : -m;
          float lacc[4] = {0.f, 0.f, 0.f, 0.f}, unused[4];
          exp_pairs<kF16, 0, true, 32>(sr, 0, p.scale_log2, neg_m, pk[0], lacc, unused);
          tmem_ld64_sync(s_addr + 64, sr);
          hide(sr, n_vis - 64);
          exp_pairs<kF16, 0, true, 32>(sr, 0, p.scale_log2, neg_m, pk[1], lacc, unused);
          tmem_st32x2_sync(s_addr, pk[0], pk[1]);
          l = l * alpha + ((lacc[0] + lacc[1]) + (lacc[2] + lacc[3]));
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s.p_full[t]);
        }
      }
      if (!ok) break;
      if (j0 < t1) {
        if (!(ok = wait(&s.o_full[t], oc & 1, 92 + t))) break;
        ++oc;
        const bool joined = !two && t0 + 1 < t1;  // both halves have a part of these rows
        if (joined && t == 1) {
          other[lane] = make_float2(m, l);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s.x_full);
          if (!(ok = wait(&s.x_empty, xc & 1, 95))) break;
          ++xc;
        } else {
          float w0 = 1.f, w1 = 0.f;
          if (joined) {
            if (!(ok = wait(&s.x_full, xc & 1, 94))) break;
            ++xc;
            const float2 o = other[lane];
            const float top = fmaxf(m, o.x), base = top == -INFINITY ? 0.f : top;
            w0 = ex2_approx(m - base);
            w1 = ex2_approx(o.x - base);
            l = l * w0 + o.y * w1;
            m = top;
          }
          const bool done = u.complete;
          const int tok = tok0 + r / p.group, r_head = r % p.group;
          const bool valid = r < tile_tokens * p.group && tok < u.s.n;
          const int64_t row_tok = u.s.q0 + tok, head = int64_t(u.hk) * p.group + r_head;
          const int64_t part = int64_t(u.part) * p.unit_rows +
                               (tok - u.unit * p.block_tokens) * p.group + r_head;
          if (done) {
            const float scale = l == 0.f ? 0.f : 1.f / l;
            w0 *= scale;
            w1 *= scale;
          }
          uint8_t* to = done ? reinterpret_cast<uint8_t*>(static_cast<uint16_t*>(p.out) +
                                                          row_tok * p.o_stride_t + head * p.o_stride_h)
                             : reinterpret_cast<uint8_t*>(p.part_o + part * kD);
          // one copy of the code for all columns: fetching it takes longer than running it
#pragma unroll 1
          for (int ch = 0; ch < kOChunks; ++ch) {
            uint32_t orow[32];
            tmem_ld32_sync(o_addr + ch * 32, orow);
#pragma unroll
            for (int c = 0; c < 32; ++c) orow[c] = __float_as_uint(__uint_as_float(orow[c]) * w0);
            if (joined) {
              uint32_t more_o[32];
              tmem_ld32_sync(o_addr + kD + ch * 32, more_o);
#pragma unroll
              for (int c = 0; c < 32; ++c)
                orow[c] = __float_as_uint(fmaf(__uint_as_float(more_o[c]), w1, __uint_as_float(orow[c])));
              if (ch == kOChunks - 1) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&s.x_empty);
              }
            }
            auto f = [&](int c) { return __uint_as_float(orow[c]); };
            if (done) {
              uint4 v[4];
#pragma unroll
              for (int c = 0; c < 4; ++c)
                v[c] = make_uint4(pack16<kF16>(f(8 * c), f(8 * c + 1)), pack16<kF16>(f(8 * c + 2), f(8 * c + 3)),
                                  pack16<kF16>(f(8 * c + 4), f(8 * c + 5)), pack16<kF16>(f(8 * c + 6), f(8 * c + 7)));
              store_rows(s.out[warp], v, lane, to + ch * 64, valid);
            } else {
#pragma unroll
              for (int hf = 0; hf < 2; ++hf) {
                uint4 v[4];
#pragma unroll
                for (int c = 0; c < 4; ++c)
                  v[c] = make_uint4(orow[16 * hf + 4 * c], orow[16 * hf + 4 * c + 1],
                                    orow[16 * hf + 4 * c + 2], orow[16 * hf + 4 * c + 3]);
                store_rows(s.out[warp], v, lane, to + ch * 128 + hf * 64, valid);
              }
            }
          }
          if (valid) {
            if (!done) p.part_ml[part] = make_float2(m, l);
            else if (p.lse)
              p.lse[head * p.tokens + row_tok] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.run_empty[run & 3]);
    }
  }
  // ---- teardown
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 0) tmem_dealloc<512>(tmem);
}

template <int kD, bool kF16>
int64_t chunk_local_bytes() {
  cudaFuncAttributes a;
  const cudaError_t e = cudaFuncGetAttributes(&a, paged_chunk_kernel<kD, kF16>);
  if (e != cudaSuccess) throw std::runtime_error(std::string("paged attention: ") + cudaGetErrorString(e));
  return int64_t(a.localSizeBytes);
}

template <int kD, bool kF16>
void chunk_launch(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv,
                  const PagedParams& p, cudaStream_t s) {
  const int smem = int(sizeof(ChunkSmem<kD>)) + 1024 + 4 * (p.seqs + 1);
  auto fn = paged_chunk_kernel<kD, kF16>;
  static const int64_t local = chunk_local_bytes<kD, kF16>();
  if (local != 0)
    throw std::runtime_error("paged attention: the chunk kernel was compiled with " + std::to_string(local) +
                             " bytes of local memory; its scores must not be spilled");
  static std::atomic<uint64_t> allowed{0};
  cudaError_t e = paged_allow_smem(fn, allowed);
  if (e == cudaSuccess) {
    fn<<<p.grid, kThreads, smem, s>>>(mq, mk, mv, p);
    e = cudaGetLastError();
  }
  if (e != cudaSuccess) throw std::runtime_error(std::string("paged attention: ") + cudaGetErrorString(e));
}

}  // namespace

int64_t paged_chunk_local_bytes() {
  return std::max(std::max(chunk_local_bytes<64, false>(), chunk_local_bytes<64, true>()),
                  std::max(chunk_local_bytes<128, false>(), chunk_local_bytes<128, true>()));
}

void paged_chunk_launch(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv,
                        const PagedParams& p, cudaStream_t s) {
  if (p.head_dim == 64) p.fp16 ? chunk_launch<64, true>(mq, mk, mv, p, s) : chunk_launch<64, false>(mq, mk, mv, p, s);
  else p.fp16 ? chunk_launch<128, true>(mq, mk, mv, p, s) : chunk_launch<128, false>(mq, mk, mv, p, s);
}

}  // namespace mgfa
