// head_fwd.cuh -- the head losses' forward pass: x . w^T on the tensor cores,
// reduced to a (maximum, sum of exp2) pair per row in the epilogue; no logit
// leaves the SM but the targets'.
//
// Rows of x lie along TMEM lanes, ids along its columns, so a thread owns a row
// and reduces without exchanging anything.  Tiles are 128 * CG rows (CTA pairs
// from 129 rows on) by `bn` ids:
//   many rows: bound by the tensor cores, 256 ids;
//   up to 128 rows (one generated token, a decode batch): bound by reading w, so
//     bn is chosen to give every SM the same number of ids, x comes in boxes of
//     as many rows as there are (the lanes behind them compute on what lies in
//     shared memory, and nothing reads them), and a CTA keeps its pairs in
//     registers over all its tiles.
// Producers as in head_bwd.cuh: one warp loads A, another B.
//
// The tensor cores truncate as they accumulate: each addition of 16 products
// loses up to 2^-23 of the partial sum (on average 0.8e-9 to 1.6e-9 of the logit
// per column; nothing where the sum is exact).  So a sum stays in tensor memory for
// at most 384 columns and is added, rounded to nearest, in registers (LONG): 128 of
// them a thread, a tile's half row.  Off by, of the logit at dim 2048: random signs
// 3.6e-7, one sign 5.3e-7, exact sums 0, large products first 1.4e-6 (in one sum
// 1.9e-6, 5.6e-6, 0, 1.1e-5).  4096 rows of 32000 ids at dim 768: 142 us
// (one sum of 768: 140), 50000 ids at dim 1024: 273 (271), at dim 512: 175 (148, two
// runs are shorter than a tile's epilogue); one token of 32000 ids: 14.2 (14.2).
#pragma once
#include "head_bwd.cuh"

namespace ne {

constexpr int HF_MAX_STAGES = 12;
constexpr int HF_HINT_KB = 16;
constexpr int HF_RUN_KB = 6;   // k-blocks of 64 a sum stays in tensor memory for, at most

struct HeadLse {
  HeadTargets t;
  const int* d_rows;     // packed rows (NULL: `rows`)
  int* status;
  float2* stats;         // (max, sum) pairs, [part][row] by the two strides
  long long part_stride, row_stride;
  float* zt;             // [entry][row] the targets' logits, log2 units
  float c2;              // scale / (T ln 2)
  int rows, vocab, dim_kb;
  int bn, n_tiles, group_m;
  int run_kb;            // k-blocks of 64 that a sum stays in tensor memory for (LONG)
  int a_rows, stages;    // rows of a box of x; ring depth
  int one_row_tile;      // all units have the same rows: one pair per CTA
};

__device__ __forceinline__ void tma_hint_2d(const void* tmap, int32_t c0, int32_t c1) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(
                   reinterpret_cast<uint64_t>(tmap)),
               "r"(c0), "r"(c1)
               : "memory");
}

// A row's running statistics: sum of 2^(c2 v - mx) over the columns seen.
struct LseRow {
  float mx, sum;
};
// 32 columns n0 .. of the row, those below n_end; picks out the targets' logits.
__device__ __forceinline__ void lse_chunk(const HeadLse& p, LseRow& r, TargetCursor& cur, float (&v)[32],
                                          int n0, int n_end) {
  if (n0 + 32 > n_end) {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (n0 + j >= n_end) v[j] = -INFINITY;
  }
  float t4[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
  for (int j = 4; j < 32; ++j) t4[j & 3] = fmaxf(t4[j & 3], v[j]);
  const float top = fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3]));
  const float nm = fmaxf(r.mx, top * p.c2);
  float s4[4] = {r.sum * ex2_fast(r.mx - nm), 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < 32; ++j) s4[j & 3] += ex2_fast(fmaf(v[j], p.c2, -nm));
  r.mx = nm;
  r.sum = (s4[0] + s4[1]) + (s4[2] + s4[3]);
  const int stop = min(n0 + 32, n_end);
  while (cur.next < stop) {
    if (cur.next >= n0) {
      const int j = cur.next - n0;
      float z = 0.f;
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (i == j) z = v[i];
      p.zt[cur.at * p.t.ld + cur.row] = z * p.c2;
    }
    cursor_step<false>(p.t, cur);
  }
}

// The same of a warp's half of a tile, four chunks of 32 columns 64 apart that are
// all in registers: one maximum for all (4096 rows of 50000 ids at dim 512: 175 us,
// chunk by chunk 184).
__device__ __forceinline__ void lse_half(const HeadLse& p, LseRow& r, TargetCursor& cur, float (&v)[4][32],
                                         int n0, int n_end) {
  if (n0 + 224 > n_end) {
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (n0 + 64 * g + j >= n_end) v[g][j] = -INFINITY;
  }
  float t4[4] = {v[0][0], v[0][1], v[0][2], v[0][3]};
#pragma unroll
  for (int j = 4; j < 128; ++j) t4[j & 3] = fmaxf(t4[j & 3], v[j >> 5][j & 31]);
  const float top = fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3]));
  const float nm = fmaxf(r.mx, top * p.c2);
  float s4[4] = {r.sum * ex2_fast(r.mx - nm), 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < 128; ++j) s4[j & 3] += ex2_fast(fmaf(v[j >> 5][j & 31], p.c2, -nm));
  r.mx = nm;
  r.sum = (s4[0] + s4[1]) + (s4[2] + s4[3]);
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int first = n0 + 64 * g, stop = min(first + 32, n_end);
    while (cur.next < stop) {
      if (cur.next >= first) {
        const int j = cur.next - first;
        float z = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (i == j) z = v[g][i];
        p.zt[cur.at * p.t.ld + cur.row] = z * p.c2;
      }
      cursor_step<false>(p.t, cur);
    }
  }
}

template <int CG, bool LONG>
__global__ void __launch_bounds__(HB_THREADS, 1)
head_lse_kernel(const __grid_constant__ CUtensorMap x_k, const __grid_constant__ CUtensorMap w_k,
                const HeadLse p) {
  constexpr bool PAIR = CG == 2;
  constexpr int TILE_M = GEMM_BM * CG;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* const gbase = smem_raw + (base - raw);
  const int stages = p.stages;
  const uint32_t a_bytes = p.a_rows * 128, b_bytes = p.bn / CG * 128;
  // barriers first; the boxes of x last, so that the rows an MMA reads behind
  // the last one still lie in the allocation
  const uint32_t full_bar = base;
  const uint32_t empty_bar = full_bar + 8 * HF_MAX_STAGES;
  const uint32_t tfull_bar = empty_bar + 8 * HF_MAX_STAGES;   // [2]
  const uint32_t tempty_bar = tfull_bar + 16;                 // [2]
  const uint32_t drain_bar = tempty_bar + 16;
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(gbase + 16 * HF_MAX_STAGES + 40);
  volatile int* const abort_flag = reinterpret_cast<volatile int*>(gbase + 16 * HF_MAX_STAGES + 44);
  const uint32_t b_at = base + 1024, a_at = b_at + stages * b_bytes;

  const int warp = uniform_warp();
  const int lane = threadIdx.x & 31;
  const uint32_t crank = PAIR ? cluster_ctarank() : 0u;
  const int cluster = PAIR ? (int)(blockIdx.x >> 1) : (int)blockIdx.x;
  const int clusters = PAIR ? (int)(gridDim.x >> 1) : (int)gridDim.x;

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(full_bar + 8 * s, 1);
      mbar_init(empty_bar + 8 * s, 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tfull_bar + 8 * a, 1);
      mbar_init(tempty_bar + 8 * a, CG * GEMM_EPI_WARPS);
    }
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&x_k);
    tma_prefetch_desc(&w_k);
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      tmem_alloc_pair(smem_u32(tmem_slot), 512);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(smem_u32(tmem_slot), 512);
      tmem_relinquish();
    }
  }
  pdl_trigger();
  if (p.one_row_tile && warp == 2 + GEMM_EPI_WARPS && cluster < p.n_tiles) {
    // while the kernel before this one ends: the first tile of w toward L2 (a
    // hint; the loads that count come after the wait): about 1 us of the 15 that
    // one token of 32000 ids, dim 768, takes.
    const int kbs = min(p.dim_kb, HF_HINT_KB), row = cluster * p.bn + (int)crank * (p.bn / CG);
    for (int k = lane; k < kbs; k += 32) tma_hint_2d(&w_k, k * GEMM_BK, row);
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();
  const int M = p.d_rows ? *p.d_rows : p.rows;
  GemmShape sh;
  sh.m_tiles = (M + TILE_M - 1) / TILE_M;
  sh.n_tiles = p.n_tiles;
  sh.group_m = p.group_m;
  const int units = sh.m_tiles * sh.n_tiles;

  if (warp == 0 || warp == 2 + GEMM_EPI_WARPS) {
    // ------------------------------------------------ TMA producers
    const bool is_a = warp == 0;
    const bool arms = is_a && (!PAIR || crank == 0);
    // x is read again for every tile of ids, w once for all tiles of rows
    const uint64_t pol = is_a ? policy_evict_last() : policy_evict_normal();
    const uint32_t full_to = PAIR ? mapa_shared(full_bar, 0) : full_bar;
    const CUtensorMap* tm = is_a ? &x_k : &w_k;
    const uint32_t ring = is_a ? a_at : b_at, bytes = is_a ? a_bytes : b_bytes;
    const uint32_t expect = CG * (a_bytes + b_bytes);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int u = cluster; u < units && ok; u += clusters) {
      int mt, nt, sp_unused;
      unit_coords(sh, u, mt, nt, sp_unused);
      const int first = is_a ? mt * TILE_M + (int)crank * GEMM_BM
                             : nt * p.bn + (int)crank * (p.bn / CG);
      for (int k = 0; k < p.dim_kb; ++k) {
        if (!warp_wait(empty_bar + 8 * stage, phase ^ 1u, p.status, abort_flag)) {
          ok = false;
          break;
        }
        if (elect_one()) {
          if (arms) mbar_arrive_expect_tx(full_bar + 8 * stage, expect);
          if constexpr (PAIR)
            tma_load_2d_pair(ring + stage * bytes, tm, full_to + 8 * stage, k * GEMM_BK, first, pol);
          else
            tma_load_2d(ring + stage * bytes, tm, full_to + 8 * stage, k * GEMM_BK, first, pol);
        }
        if (++stage == stages) { stage = 0; phase ^= 1u; }
      }
    }
    // no load may be in flight when the CTA exits (gemm_tc.cuh)
    if (arms) {
      for (int s = 0; s < stages; ++s) {
        const uint32_t par = (s < stage) ? phase : (phase ^ 1u);
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try_wait(full_bar + 8 * s, par)) {
          if (globaltimer_ns() - t0 > 100000000ull) break;
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------ MMA issuer
    if (!PAIR || crank == 0) {
      const uint32_t idesc = umma_idesc_f16(TILE_M, p.bn, 1);
      int stage = 0;
      uint32_t phase = 0;
      int acc = 0;
      uint32_t acc_phase = 0;
      bool ok = true;
      for (int u = cluster; u < units && ok; u += clusters) {
        for (int k0 = 0; k0 < p.dim_kb && ok; k0 += LONG ? p.run_kb : p.dim_kb) {
          if (!warp_wait(tempty_bar + 8 * acc, acc_phase ^ 1u, p.status, abort_flag)) { ok = false; break; }
          tc_fence_after();
          const uint32_t d_tmem = tmem_base + acc * HB_BN;
          const int kn = LONG ? min(p.run_kb, p.dim_kb - k0) : p.dim_kb;
          for (int k = 0; k < kn; ++k) {
            if (!warp_wait(full_bar + 8 * stage, phase, p.status, abort_flag)) { ok = false; break; }
            tc_fence_after();
            if (elect_one()) {
              const uint64_t ad = smem_desc_k_sw128(a_at + stage * a_bytes);
              const uint64_t bd = smem_desc_k_sw128(b_at + stage * b_bytes);
#pragma unroll
              for (int j = 0; j < GEMM_BK / 16; ++j)
                if constexpr (PAIR) umma_f16_pair(d_tmem, ad + 2 * j, bd + 2 * j, idesc, (k | j) != 0);
                else umma_f16(d_tmem, ad + 2 * j, bd + 2 * j, idesc, (k | j) != 0);
              if constexpr (PAIR) umma_commit_pair(empty_bar + 8 * stage, 0x3);
              else umma_commit(empty_bar + 8 * stage);
            }
            if (++stage == stages) { stage = 0; phase ^= 1u; }
          }
          if (!ok) break;
          if (elect_one()) {
            if constexpr (PAIR) umma_commit_pair(tfull_bar + 8 * acc, 0x3);
            else umma_commit(tfull_bar + 8 * acc);
          }
          if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
        }
      }
      if (elect_one()) {
        if constexpr (PAIR) umma_commit_pair(drain_bar, 0x1);
        else umma_commit(drain_bar);
      }
      const uint64_t t0 = globaltimer_ns();
      while (!mbar_try_wait(drain_bar, 0)) {
        if (globaltimer_ns() - t0 > 100000000ull) break;
      }
    }
  } else {
    // ------------------------------------------------ epilogue (warps 2..9)
    // m, s: the running maximum and sum of exp2(c2 acc - m), fp32
    const int quarter = warp & 3;
    const int half = (warp - 2) >> 2;   // of the two warps of a row: even or odd chunks
    const int lane_row = (int)crank * GEMM_BM + quarter * 32 + lane;
    const LseRow none{-3.402823466e38f, 0.f};
    LseRow r = none;
    int acc = 0;
    uint32_t acc_phase = 0;
    // waits for the accumulator and gives it back
    auto acquire = [&]() -> bool {
      const bool ready = mbar_wait(tfull_bar + 8 * acc, acc_phase, p.status, abort_flag);
      if (!__all_sync(0xffffffffu, ready)) return false;
      tc_fence_after();
      return true;
    };
    auto release = [&] {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (PAIR) mbar_arrive_peer(mapa_shared(tempty_bar + 8 * acc, 0));
        else mbar_arrive(tempty_bar + 8 * acc);
      }
      if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
    };
    const uint32_t t_lane = tmem_base + ((uint32_t)(quarter * 32) << 16);
    for (int u = cluster; u < units; u += clusters) {
      int mt, nt, sp_unused;
      unit_coords(sh, u, mt, nt, sp_unused);
      const int m = mt * TILE_M + lane_row;
      const int n_tile = nt * p.bn, n_end = min(n_tile + p.bn, p.vocab);
      const bool has_rows = m - lane < M;   // the warp's
      TargetCursor cur;
      if (!p.one_row_tile) r = none;
      if constexpr (LONG) {
        float sum[4][32];
        bool ok = true;
#pragma unroll 1
        for (int k = 0; k < p.dim_kb; k += p.run_kb) {
          // a chain of loads: behind the tile's first loads of w where those are the
          // bound, else behind the MMAs of its last run
          if (p.one_row_tile ? k == 0 : k + p.run_kb >= p.dim_kb) cursor_seek<false>(p.t, cur, m, M, n_tile);
          if (!acquire()) { ok = false; break; }
          if (has_rows) {
            const uint32_t t = t_lane + acc * HB_BN + 32 * half;
            if (k == 0) {
#pragma unroll
              for (int g = 0; g < 4; ++g) tmem_ld32_issue(t + 64 * g, sum[g]);
#pragma unroll
              for (int g = 0; g < 4; ++g) tmem_ld32_wait(sum[g]);
            } else {
#pragma unroll
              for (int g = 0; g < 4; ++g) {
                float v[32];
                tmem_ld32(t + 64 * g, v);
#pragma unroll
                for (int j = 0; j < 32; ++j) sum[g][j] += v[j];
              }
            }
          }
          release();
        }
        if (!ok) break;
        if (has_rows) {
          if constexpr (PAIR) {
            lse_half(p, r, cur, sum, n_tile + 32 * half, n_end);
          } else {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const int n0 = n_tile + 32 * half + 64 * g;
              if (n0 < n_end) lse_chunk(p, r, cur, sum[g], n0, n_end);
            }
          }
        }
      } else {
        cursor_seek<false>(p.t, cur, m, M, n_tile);
        if (!acquire()) break;
        if (has_rows) {
#pragma unroll 1
          for (int c = 32 * half; c < p.bn; c += 64) {
            if (n_tile + c >= n_end) break;
            float v[32];
            tmem_ld32(t_lane + acc * HB_BN + c, v);
            lse_chunk(p, r, cur, v, n_tile + c, n_end);
          }
        }
        release();
      }
      if (!p.one_row_tile && cur.row >= 0)
        p.stats[(2 * nt + half) * p.part_stride + m * p.row_stride] = make_float2(r.mx, r.sum);
    }
    if (p.one_row_tile && lane_row < M)
      p.stats[(2 * cluster + half) * p.part_stride + lane_row * p.row_stride] = make_float2(r.mx, r.sum);
  }

  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync_all();
  tc_fence_after();
  if (warp == 1) {
    if constexpr (PAIR) tmem_dealloc_pair(tmem_base, 512);
    else tmem_dealloc(tmem_base, 512);
  }
}

}  // namespace ne
