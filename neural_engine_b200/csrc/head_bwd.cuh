// head_bwd.cuh -- the head losses' backward pass: one persistent launch that
// walks the vocabulary in pieces.
//
//   dz[p] = f(x . w[p]^T)            rows x piece, K = dim
//   dx   += dz[p] . w[p]             rows x dim,   K = piece (in splits)
//   dw[p] = dz[p]^T . x              piece x dim,  K = rows
//
// Bound by the tensor cores: 6 rows vocab dim operations, of which the first
// product is the price of not keeping the logits.  Work units are one 128 * CG x
// 256 tile (dx: of one split of the piece), in the order
//   dz[0],  dz[1] dx[0] dw[0],  dz[2] dx[1] dw[1],  ...,  dx[P-1] dw[P-1]
// so that what a unit reads was made a piece earlier, and pieces are small
// enough to be read back from L2.  The leading CTA's A producer draws units from
// a counter in device memory, waits until the units it depends on have
// signalled, and hands it to the other roles of both CTAs through a ring of
// slots.  A unit depends only on units drawn before it, so the wait ends
// whatever the number of CTAs that run; it is bounded all the same.  Which pair
// computes a unit changes no value: every unit is computed whole, and dx adds
// the pieces in their order.
// The tensor cores truncate as they add (head_fwd.cuh), so a unit of more than 1024
// products a sum is taken out of tensor memory in runs, which are added in registers:
// fp32 dw of 400000 rows of one sign was 1e-3 too small in one sum, and at dim 4096
// logits summed otherwise than the forward pass's put gradients of few rows 9e-4 off
// (1e-4 in runs).  It costs 1 to 2% (4096 rows of 151936 ids, forward and backward:
// 4.06 -> 4.13 ms, 256 rows of 32000 ids 74.2 -> 75.3 us).
// dz goes into the products in bf16.  What rounding takes from it at a row's target,
// where most of its size is, is put back in fp32: into dx by the kernel that adds the
// slabs, into dw by the epilogue (put_back).  Gradients of 294 rows in bf16 are then
// 1.66e-3 off float64 instead of 2.4e-3, as much as rounding them alone makes; it costs
// 4 us of 75 at 256 rows, 7 of 281 at 1638 of 4096, 0.3% at 4096 rows of 151936 ids.
// As launches of their own the products left 14% of the pairs idle in their last
// waves (4096 rows, dim 1024: 64 tiles of dx, 128 of dw, for 74 pairs).
//
// Shared-memory ring, TMEM accumulators and CTA pairs are those of gemm_tc.cuh,
// and so are the warp roles but for the producer: issuing a tensor load takes a
// thread 110 to 150 cycles and the MMA of a k-block 512, so one warp loads A
// (and draws the units), another B.
#pragma once
#include "gemm_tc.cuh"

namespace ne {

constexpr int HB_BN = 256;
constexpr int HB_SLOTS = 8;
constexpr int HB_DRAW = 12, HB_TAKE = 6;        // k-blocks before a unit's end
constexpr int HB_RUN_KB = 16;                   // k-blocks that a sum stays in tensor memory for, at most
constexpr int HB_THREADS = GEMM_THREADS + 32;   // warps: A, MMA, 8 x epilogue, B
constexpr int HB_BOX = 4096;                    // 32 rows of 128 bytes
constexpr int HB_TWIN = 64;                     // up to here rows stand twice
constexpr int HB_TAB = 256;                     // ids per entry of a row's index
constexpr int HB_PUT_BACK = 32;                 // rows that 32 ids' dw takes rests of, at most

template <int CG>
struct HeadCfg {
  static constexpr int A_BYTES = GEMM_BM * GEMM_BK * 2;
  static constexpr int STAGE_BYTES = A_BYTES + HB_BN / CG * GEMM_BK * 2;
  // a load takes up to 3,000 cycles to arrive and a k-block 512 to be used: as
  // many stages as fit
  static constexpr int STAGES = CG == 2 ? 6 : 4;
  // ring, barriers, a box per epilogue warp, alignment
  static constexpr int SMEM = STAGES * STAGE_BYTES + 2048 + GEMM_EPI_WARPS * HB_BOX;
  static_assert(SMEM <= 232448, "shared memory per CTA");
};

constexpr int HB_BUFS = 3;   // pieces of dz alive: made, waited for, read

struct HeadWalk {
  const int* d_rows;        // packed rows
  int* counters;            // units drawn, then head_flag's, all zero at launch
  int* status;
  int rows64;               // rows of a dz buffer and of a slab of dx
  int vocab, dim, dim_kb, dim_tiles;   // dim also in k-blocks of 64 and tiles of 256
  int piece, pieces;        // ids a piece (a multiple of 256)
  int split_n, splits;      // ids a split of dx's product (a multiple of 256), splits a piece
  int own_slabs;            // dx of each piece goes to slabs of its own, else they add up
  int want_dx, want_dw, dw_f32;
};
// Counters of piece p: dz read (per unit), dx added (per epilogue warp), and for
// each split of its ids dz written (per epilogue warp).
__device__ __forceinline__ int* head_flag(const HeadWalk& s, int p, int what) {
  return s.counters + 1 + (2 + s.splits) * p + what;
}
enum HeadFlag : int { HF_READ = 0, HF_ADDED = 1, HF_MADE = 2 };   // HF_MADE + split

// The sparse targets of the rows: sorted ids, [entry][row], INT_MAX behind the
// last.
struct HeadTargets {
  const int* ids;
  const float* prob;           // the probability of each id (NULL: 1)
  const int* row_of;           // packed row -> row of the arrays (NULL: the same)
  const unsigned short* tab;   // [row][tab_ld]: how many ids are below 256 t (NULL: one entry a row)
  long long ld;                // between entries
  int tab_ld;
  int n;                       // entries a row
};

// A walk over a row's entries.  The entry behind the next one is read ahead: a
// chunk of columns passes faster than a load arrives.
struct TargetCursor {
  int row;               // of the arrays (-1: none)
  int at;                // the next entry
  int next, after;       // its id, and the one behind it
  float q, q_after;      // their probabilities
};

template <bool PROB>
__device__ __forceinline__ void cursor_load(const HeadTargets& t, const TargetCursor& c, int at, int& id,
                                            float& q) {
  id = 0x7fffffff;
  q = 1.0f;
  if (at < t.n) {
    id = t.ids[at * t.ld + c.row];
    if (PROB && t.prob) q = t.prob[at * t.ld + c.row];
  }
}
template <bool PROB>
__device__ __forceinline__ void cursor_step(const HeadTargets& t, TargetCursor& c) {
  ++c.at;
  c.next = c.after;
  c.q = c.q_after;
  cursor_load<PROB>(t, c, c.at + 1, c.after, c.q_after);
}
// The first entry of row m with an id of at least col0.  Few entries lie
// between a multiple of 256 and col0, so they are stepped over; a search of the
// whole row would be a chain of log2 n loads, 600 cycles each.
template <bool PROB>
__device__ __forceinline__ void cursor_seek(const HeadTargets& t, TargetCursor& c, int m, int rows,
                                            int col0) {
  c.row = m < rows ? (t.row_of ? t.row_of[m] : m) : -1;
  c.at = 0;
  c.next = c.after = 0x7fffffff;
  if (c.row < 0) return;
  if (t.tab) c.at = t.tab[(long long)c.row * t.tab_ld + col0 / HB_TAB];
  cursor_load<PROB>(t, c, c.at, c.next, c.q);
  cursor_load<PROB>(t, c, c.at + 1, c.after, c.q_after);
  while (c.next < col0) cursor_step<PROB>(t, c);
}

// What turns logits into dz = a (2^(c2 acc - lse log2 e) - p), a = g T scale.
struct HeadDz {
  HeadTargets t;
  const float2* coef;   // packed rows: a, log2|a| - lse log2 e
  float c2;             // scale / (T ln 2)
  // What rounding takes from dz at a row's largest target is put back.
  const int* best;      // packed rows: that target's id (NULL: it is not put back)
  float* rest;          // packed rows: what the rounding of dz there left, 0 before
  int* rests;           // for each 32 ids: rows whose target is among them, 0 before
  int4* list;           // for each 32 ids HB_PUT_BACK of them: row, id, rest
  const __nv_bfloat16* x;   // packed rows
  long long ldp;
};

struct HeadMaps {
  CUtensorMap x_k, w_k;        // dz: operands (K = dim contiguous)
  CUtensorMap twin_k, twin_mn; // x_k, x_mn of the rows that stand twice
  CUtensorMap dz_out;          // dz: [buffers * rows64][piece]
  CUtensorMap dz_k, w_mn;      // dx: dz (K = ids), w as [ids][dim]
  CUtensorMap dx_out;          // dx: [splits * rows64][dim] fp32
  CUtensorMap dz_mn, x_mn;     // dw: both as [rows][...]
  CUtensorMap dw_out;          // dw: [vocab][dim]
};

enum HeadKind : int { HK_DX = 0, HK_DW = 1, HK_DZ = 2, HK_END = 3 };

struct HeadUnit {
  int kind, piece, mt, nt, split, kb0, kb;
  int n;   // columns: 256, or what is left of them in whole 32s
};

// Units of each kind in a piece of `ids` ids.
struct HeadCounts {
  int dz, dx, dw;
};
__device__ __forceinline__ HeadCounts head_counts(const HeadWalk& s, int m_tiles, int tile_m, int ids) {
  HeadCounts c;
  c.dz = m_tiles * ((ids + HB_BN - 1) / HB_BN);
  c.dx = s.want_dx ? m_tiles * s.dim_tiles * ((ids + s.split_n - 1) / s.split_n) : 0;
  c.dw = s.want_dw ? s.dim_tiles * ((ids + tile_m - 1) / tile_m) : 0;
  return c;
}

__device__ __forceinline__ int unit_cols(int cols, int nt) {
  return min(HB_BN, (cols - nt * HB_BN + 31) & ~31);
}

// Division by a number that does not change (d >= 1, u >= 0): the quotient by the
// rounded-down reciprocal is short by one at most.
struct FastDiv {
  unsigned d, r;
  __device__ explicit FastDiv(int by) : d(by), r(0xffffffffu / (unsigned)by) {}
  __device__ __forceinline__ int div(int u) const {
    unsigned q = __umulhi((unsigned)u, r);
    if ((unsigned)u - q * d >= d) ++q;
    return (int)q;
  }
};

// A unit is summed in equal runs: the k-blocks of one.
__device__ __forceinline__ int unit_run(const HeadUnit& w) {
  const int runs = (w.kb + HB_RUN_KB - 1) / HB_RUN_KB;
  return runs < 2 ? w.kb : (w.kb + runs - 1) / runs;
}

// What the walk is made of, derived once from the number of rows.
struct HeadOrder {
  int blocks, m_tiles;
  int last_ids;              // of the last piece
  HeadCounts full, last;     // units of a whole piece and of the last one
  FastDiv by_phase, by_m, by_d;
};

// unit u of the walk (HK_END behind the last one)
__device__ __forceinline__ void head_unit(const HeadWalk& s, const HeadOrder& o, int u, HeadUnit& w) {
  const int P = s.pieces;
  const int made0 = P > 1 ? o.full.dz : o.last.dz;
  int kind_at = -1;   // position among dz, dx, dw units of one phase
  int made = -1, used = -1;
  if (u < made0) {
    made = 0;
    kind_at = u;
  } else {
    u -= made0;
    // phase q makes piece q + 1 and uses piece q; the last one makes none
    const int phase = (int)o.by_phase.d;
    const int whole = max(P - 2, 0);
    int q = min(o.by_phase.div(u), whole);
    u -= q * phase;
    if (q == whole && P > 1) {
      const int n = o.last.dz + o.full.dx + o.full.dw;
      if (u >= n) {
        u -= n;
        ++q;
      }
    }
    used = q;
    const int dz_n = q + 1 >= P ? 0 : q + 1 == P - 1 ? o.last.dz : o.full.dz;
    if (u < dz_n) {
      made = q + 1;
      kind_at = u;
    } else {
      u -= dz_n;
    }
  }
  w.split = 0;
  w.mt = w.nt = 0;
  w.kb0 = w.kb = 0;
  if (made >= 0) {
    w.kind = HK_DZ;
    w.piece = made;
    w.nt = o.by_m.div(kind_at);
    w.mt = kind_at - w.nt * o.m_tiles;
    w.kb = s.dim_kb;
    w.n = unit_cols(made == P - 1 ? o.last_ids : s.piece, w.nt);
    return;
  }
  const HeadCounts& c = used == P - 1 ? o.last : o.full;
  const int ids = used == P - 1 ? o.last_ids : s.piece;
  w.piece = used;
  if (u < c.dx) {
    w.kind = HK_DX;
    const int r = o.by_d.div(u);
    w.nt = u - r * s.dim_tiles;
    w.split = o.by_m.div(r);
    w.mt = r - w.split * o.m_tiles;
    w.kb0 = w.split * (s.split_n / GEMM_BK);
    w.kb = (min(ids - w.split * s.split_n, s.split_n) + GEMM_BK - 1) / GEMM_BK;
  } else if (u - c.dx < c.dw) {
    u -= c.dx;
    w.kind = HK_DW;
    w.mt = o.by_d.div(u);
    w.nt = u - w.mt * s.dim_tiles;
    w.kb = o.blocks;
  } else {
    w.kind = HK_END;
  }
  w.n = unit_cols(s.dim, w.nt);
}

__device__ __forceinline__ void flag_add(int* f) {
  asm volatile("red.release.gpu.global.add.s32 [%0], 1;" ::"l"(f) : "memory");
}
__device__ __forceinline__ bool flag_reached(const int* f, int want) {
  int v;
  asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(f) : "memory");
  return v >= want;
}
// Bounded wait until *f >= want.
__device__ __forceinline__ bool flag_wait(const int* f, int want, int* status, volatile int* abort) {
  const uint64_t t0 = globaltimer_ns();
  while (true) {
    if (flag_reached(f, want)) return true;
    if (*abort) return false;
    if (globaltimer_ns() - t0 > kWaitBudgetNs) {
      atomicExch(status, DEV_ERR_TIMEOUT);
      *abort = 1;
      return false;
    }
  }
}
// What was written through TMA before a flag is read through TMA after it.
__device__ __forceinline__ void fence_async_global() {
  asm volatile("fence.proxy.async.global;" ::: "memory");
}

// Arrivals and writes across the pair.  All that crosses is a work unit, written
// together with its completion (st.async): the hand-over is no release at cluster
// scope, which would cost an epilogue warp about 1,400 cycles, and the matching
// acquire another 1,000.  What other SMs wrote is therefore not passed on by it;
// the peer's A producer acquires the same flags itself (`ready`).
__device__ __forceinline__ void mbar_arrive_peer(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ void post_unit(uint32_t cluster_addr, uint32_t cluster_bar,
                                          const HeadUnit& w) {
  asm volatile("mbarrier.arrive.expect_tx.relaxed.cluster.shared::cluster.b64 _, [%0], 32;" ::"r"(
                   cluster_bar)
               : "memory");
  asm volatile(
      "st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, "
      "[%5];" ::"r"(cluster_addr),
      "r"(w.kind), "r"(w.piece), "r"(w.mt), "r"(w.nt), "r"(cluster_bar)
      : "memory");
  asm volatile(
      "st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, "
      "[%5];" ::"r"(cluster_addr + 16),
      "r"(w.split), "r"(w.kb0), "r"(w.kb), "r"(w.n), "r"(cluster_bar)
      : "memory");
}
__device__ __forceinline__ void read_unit(uint32_t addr, HeadUnit& w) {
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(w.kind), "=r"(w.piece), "=r"(w.mt), "=r"(w.nt)
               : "r"(addr)
               : "memory");
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(w.split), "=r"(w.kb0), "=r"(w.kb), "=r"(w.n)
               : "r"(addr + 16)
               : "memory");
}

// The producer and MMA warps run whole, on values that are the same in every
// lane, and elect a lane for what is issued once: such values live in the
// uniform registers that these instructions take.  Issued from a lane of its
// own branch a k-block costs the MMA warp about 590 cycles, this way 360 (the
// MMAs take 512).
__device__ __forceinline__ bool elect_one() {
  uint32_t x;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(x));
  return x != 0;
}
__device__ __forceinline__ int uniform_warp() {
  return __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0);
}
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, int* status, volatile int* abort) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, status, abort));
}

// 32 values to bf16, the low 16 bits of each word first.
__device__ __forceinline__ void pack_bf16(const float (&v)[32], uint32_t* o) {
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
    o[j] = *reinterpret_cast<const uint32_t*>(&h);
  }
}

// This lane's row of a box of 32 rows of 128 bytes, in the 128-byte swizzle.
__device__ __forceinline__ void stage_words(uint32_t box, int lane, const uint32_t (&o)[32]) {
#pragma unroll
  for (int q = 0; q < 8; ++q)
    st_shared_v4(box + lane * 128 + ((q ^ (lane & 7)) << 4), o[4 * q], o[4 * q + 1], o[4 * q + 2],
                 o[4 * q + 3]);
}

// 32 columns of this lane's row; the registers hold them after tmem_ld32_wait.
__device__ __forceinline__ void tmem_ld32_issue(uint32_t taddr, float (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]),
        "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]),
        "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]),
        "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
        "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]),
        "=f"(v[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld32_wait(float (&v)[32]) {
  asm volatile(
      "tcgen05.wait::ld.sync.aligned;"
      : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]),
        "+f"(v[7]), "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]),
        "+f"(v[13]), "+f"(v[14]), "+f"(v[15]), "+f"(v[16]), "+f"(v[17]), "+f"(v[18]),
        "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]), "+f"(v[23]), "+f"(v[24]),
        "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]), "+f"(v[30]),
        "+f"(v[31])
      :
      : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&v)[32]) {
  tmem_ld32_issue(taddr, v);
  tmem_ld32_wait(v);
}

// Back to tensor memory: 32 columns of this lane's row, there after tmem_st_wait.
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const float (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};"
      :
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]),
        "f"(v[7]), "f"(v[8]), "f"(v[9]), "f"(v[10]), "f"(v[11]), "f"(v[12]), "f"(v[13]),
        "f"(v[14]), "f"(v[15]), "f"(v[16]), "f"(v[17]), "f"(v[18]), "f"(v[19]), "f"(v[20]),
        "f"(v[21]), "f"(v[22]), "f"(v[23]), "f"(v[24]), "f"(v[25]), "f"(v[26]), "f"(v[27]),
        "f"(v[28]), "f"(v[29]), "f"(v[30]), "f"(v[31]),
        "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// dw of 32 ids from `first`, one a lane, takes what rounding left of dz at their `n`
// rows' targets (e: the list's place of this lane), on the accumulator: `cols` columns
// of it, x's from n0.  An id's rows one after the other, in their order, whichever
// entered the list first.  Called by a whole warp; a function of its own so that its
// registers are not the epilogue's.
__device__ __noinline__ void put_back(const HeadDz& p, int4 e, int first, int n, uint32_t taddr, int n0,
                                      int cols) {
  const int lane = threadIdx.x & 31;
  int turn = 0;   // of this place among its id's
#pragma unroll 1
  for (int i = 0; i < n; ++i) {
    const int row = __shfl_sync(0xffffffffu, e.x, i), id = __shfl_sync(0xffffffffu, e.y, i);
    turn += id == e.y && row < e.x;
  }
  const int turns = __reduce_max_sync(0xffffffffu, lane < n ? turn : 0) + 1;
#pragma unroll 1
  for (int t = 0; t < turns; ++t) {
    int row = -1;
    float left = 0.f;
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
      const int r = __shfl_sync(0xffffffffu, e.x, i), id = __shfl_sync(0xffffffffu, e.y, i);
      const int z = __shfl_sync(0xffffffffu, e.z, i), k = __shfl_sync(0xffffffffu, turn, i);
      if (id == first + lane && k == t) {
        row = r;
        left = __int_as_float(z);
      }
    }
    uint4 x[16];
    const uint4* src = reinterpret_cast<const uint4*>(p.x + (row < 0 ? 0 : row) * p.ldp + n0);
#pragma unroll
    for (int q = 0; q < 16; ++q)
      x[q] = row >= 0 && 8 * q < cols ? src[q] : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      if (32 * c >= cols) break;
      float v[32];
      tmem_ld32(taddr + 32 * c, v);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint32_t u[4] = {x[4 * c + q].x, x[4 * c + q].y, x[4 * c + q].z, x[4 * c + q].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float& a = v[8 * q + 2 * i];
          float& b = v[8 * q + 2 * i + 1];
          a = fmaf(left, __uint_as_float(u[i] << 16), a);
          b = fmaf(left, __uint_as_float(u[i] & 0xffff0000u), b);
        }
      }
      tmem_st32(taddr + 32 * c, v);
    }
    tmem_st_wait();
  }
}

template <int CG>
__global__ void __launch_bounds__(HB_THREADS, 1)
head_walk_kernel(const __grid_constant__ HeadMaps maps, const HeadWalk sp,
                 const __grid_constant__ HeadDz dzp) {
  using C = HeadCfg<CG>;
  constexpr bool PAIR = CG == 2;
  constexpr int TILE_M = GEMM_BM * CG;
  constexpr int STAGES = C::STAGES;
  constexpr uint32_t TMEM_COLS = 2 * HB_BN;
  constexpr uint32_t MN_BOX = 64 * GEMM_BK * 2;
  // readers of a slot: the MMA thread, B's producer and 8 epilogue warps, and the
  // other CTA's producers and epilogue warps
  constexpr int SLOT_READERS = CG * (2 + GEMM_EPI_WARPS);

  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* const gbase = smem_raw + (base - raw);
  const uint32_t tiles = base;
  const uint32_t bars = base + STAGES * C::STAGE_BYTES;
  const uint32_t full_bar = bars;                         // [STAGES]
  const uint32_t empty_bar = full_bar + 8 * STAGES;       // [STAGES]
  const uint32_t tfull_bar = empty_bar + 8 * STAGES;      // [2]
  const uint32_t tempty_bar = tfull_bar + 16;             // [2]
  const uint32_t drain_bar = tempty_bar + 16;             // [1]
  const uint32_t sfull_bar = drain_bar + 8;               // [HB_SLOTS]
  const uint32_t sempty_bar = sfull_bar + 8 * HB_SLOTS;   // [HB_SLOTS], the leader's
  const uint32_t misc = sempty_bar + 8 * HB_SLOTS;
  const uint32_t slots = bars + 512;                      // [HB_SLOTS] units of 32 bytes
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(gbase + (misc - base));
  volatile int* const abort_flag = reinterpret_cast<volatile int*>(gbase + (misc - base) + 4);

  const int warp = uniform_warp();
  const int lane = threadIdx.x & 31;
  const uint32_t crank = PAIR ? cluster_ctarank() : 0u;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar + 8 * s, 1);
      mbar_init(empty_bar + 8 * s, 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tfull_bar + 8 * a, 1);
      mbar_init(tempty_bar + 8 * a, CG * GEMM_EPI_WARPS);
    }
    mbar_init(drain_bar, 1);
    for (int s = 0; s < HB_SLOTS; ++s) {
      mbar_init(sfull_bar + 8 * s, 1);
      mbar_init(sempty_bar + 8 * s, SLOT_READERS);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      tmem_alloc_pair(smem_u32(tmem_slot), TMEM_COLS);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(smem_u32(tmem_slot), TMEM_COLS);
      tmem_relinquish();
    }
  }
  pdl_trigger();
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();
  // the leader's A producer draws its first unit while the row count arrives
  int drawn = threadIdx.x == 0 && crank == 0 ? atomicAdd(sp.counters, 1) : 0;
  // whole blocks of 64 rows; rows behind the last are zeros
  const int count = *sp.d_rows;
  // up to 64 rows stand twice in a tile that has room for them anyway, for dz in
  // two bf16 parts
  const bool twin = count <= HB_TWIN;
  const int blocks = twin ? 2 : (count + GEMM_BK - 1) / GEMM_BK;
  const int M = blocks * GEMM_BK, m_tiles = (M + TILE_M - 1) / TILE_M;
  const int last_ids = sp.vocab - (sp.pieces - 1) * sp.piece;
  const HeadCounts full = head_counts(sp, m_tiles, TILE_M, sp.piece);
  const HeadOrder ord{blocks, m_tiles, last_ids, full, head_counts(sp, m_tiles, TILE_M, last_ids),
                      FastDiv(full.dz + full.dx + full.dw), FastDiv(m_tiles), FastDiv(sp.dim_tiles)};

  // a role other than the leader's producer takes the unit of slot `it`
  auto take = [&](int it, HeadUnit& w) -> bool {
    const int s = it % HB_SLOTS;
    if (!warp_wait(sfull_bar + 8 * s, (it / HB_SLOTS) & 1, sp.status, abort_flag)) return false;
    read_unit(slots + 32 * s, w);
    return true;
  };
  auto taken = [&](int it) {
    __syncwarp();
    if (!elect_one()) return;
    const uint32_t b = sempty_bar + 8 * (it % HB_SLOTS);
    if constexpr (PAIR) mbar_arrive_peer(mapa_shared(b, 0));
    else mbar_arrive(b);
  };

  if (warp == 0 || warp == 2 + GEMM_EPI_WARPS) {
    // ------------------------------------------------ TMA producers
    {
      const bool is_a = warp == 0;
      const bool leads = is_a && (!PAIR || crank == 0);   // draws the units, arms the barriers
      const uint64_t pol = policy_evict_normal();
      // pair mode: all loads of both CTAs complete on the even CTA's barriers
      const uint32_t full_to = PAIR ? mapa_shared(full_bar, 0) : full_bar;
      auto ld = [&](uint32_t dst, const CUtensorMap* tm, uint32_t bar, int c0, int c1) {
        if constexpr (PAIR) tma_load_2d_pair(dst, tm, bar, c0, c1, pol);
        else tma_load_2d(dst, tm, bar, c0, c1, pol);
      };
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      HeadUnit nw{};   // the leader's next unit
      // What is known to be done: pieces read and added up to here, and the split
      // written last asked for (units come in the order of pieces and kinds).
      int read_to = -1, added_to = -1, made_piece = -1, made_split = -1;
      auto reached = [&](int* f, int want, bool now) -> bool {
        if (__all_sync(0xffffffffu, flag_reached(f, want))) return true;
        if (now && !__all_sync(0xffffffffu, flag_wait(f, want, sp.status, abort_flag))) ok = false;
        return now && ok;
      };
      // What unit w depends on is done: dz, its buffer was read for the last time;
      // dx and dw, dz was written, and dx was added to by the piece before.  Each
      // CTA's A producer acquires that itself before it loads or lets the CTA's
      // epilogue store.  now: wait for it.
      auto ready = [&](const HeadUnit& w, bool now) -> bool {
        if (w.kind == HK_DZ) {
          const int p = w.piece - HB_BUFS;
          if (p > read_to) {
            if (!reached(head_flag(sp, p, HF_READ), ord.full.dx + ord.full.dw, now)) return false;
            read_to = p;
          }
        } else if (w.kind != HK_END) {
          const int split = w.kind == HK_DX ? w.split : w.mt * TILE_M / sp.split_n;
          if (w.piece != made_piece || split != made_split) {
            const int ids = w.piece == sp.pieces - 1 ? ord.last_ids : sp.piece;
            const int n = (min(ids - split * sp.split_n, sp.split_n) + HB_BN - 1) / HB_BN;
            if (!reached(head_flag(sp, w.piece, HF_MADE + split),
                         n * ord.m_tiles * CG * GEMM_EPI_WARPS, now))
              return false;
            made_piece = w.piece;
            made_split = split;
          }
          if (w.kind == HK_DX && !sp.own_slabs && w.piece - 1 > added_to) {
            if (!reached(head_flag(sp, w.piece - 1, HF_ADDED), ord.full.dx * CG * GEMM_EPI_WARPS, now))
              return false;
            added_to = w.piece - 1;
          }
        }
        return true;
      };
      // hands over the leader's next unit once it is ready
      auto hand_over = [&](int it, bool now) -> bool {
        if (!ready(nw, now)) return false;
        const int s = it % HB_SLOTS;
        const uint32_t at = slots + 32 * s;
        if (!warp_wait(sempty_bar + 8 * s, ((it / HB_SLOTS) & 1) ^ 1, sp.status, abort_flag)) {
          ok = false;
          return false;
        }
        if (elect_one()) {
          st_shared_v4(at, nw.kind, nw.piece, nw.mt, nw.nt);
          st_shared_v4(at + 16, nw.split, nw.kb0, nw.kb, nw.n);
          mbar_arrive(sfull_bar + 8 * s);
          if constexpr (PAIR) post_unit(mapa_shared(at, 1), mapa_shared(sfull_bar + 8 * s, 1), nw);
        }
        return true;
      };
      // Decodes the unit drawn before and draws the one after it; the latency of
      // the counter passes behind a unit's loads.  Behind a long unit that waits
      // until HB_DRAW k-blocks are left: what is drawn early stands behind it while
      // other pairs run out of work (forward and backward of 4096 rows of 32000 ids,
      // six in ten left out: 274 us, 292 with the draw at a unit's start).
      bool draw = false;   // the unit after nw is still to be drawn
      auto draw_unit = [&] {
        if (lane == 0) drawn = atomicAdd(sp.counters, 1);
        draw = false;
      };
      auto next_unit = [&] {
        if (draw) draw_unit();
        head_unit(sp, ord, __shfl_sync(0xffffffffu, drawn, 0), nw);
        draw = nw.kind != HK_END;
        if (draw && nw.kb <= HB_DRAW) draw_unit();
      };
      if (leads) {
        next_unit();
        hand_over(0, true);
      }
      for (int it = 0; ok; ++it) {
        HeadUnit w;
        bool handed = false;
        if (leads) {
          w = nw;
        } else {
          if (!take(it, w)) break;
          taken(it);
        }
        if (w.kind == HK_END) break;
        if (is_a && !leads && !ready(w, true)) break;
        fence_async_global();
        const int buf_row = (w.piece % HB_BUFS) * sp.rows64, id0 = w.piece * sp.piece;
        // this role's operand: K-major is one box, MN-major one per 64 columns
        const bool mn = is_a ? w.kind == HK_DW : w.kind != HK_DZ;
        const CUtensorMap* tm =
            is_a ? (w.kind == HK_DZ ? (twin ? &maps.twin_k : &maps.x_k)
                    : w.kind == HK_DX ? &maps.dz_k : &maps.dz_mn)
                 : (w.kind == HK_DZ ? &maps.w_k
                    : w.kind == HK_DX ? &maps.w_mn : twin ? &maps.twin_mn : &maps.x_mn);
        // first row (K-major) or column (MN-major) of the tile, and where K starts
        const int first = is_a ? w.mt * TILE_M + (int)crank * GEMM_BM + (w.kind == HK_DX ? buf_row : 0)
                               : w.nt * HB_BN + (int)crank * (w.n / CG) + (w.kind == HK_DZ ? id0 : 0);
        int k0 = w.kb0 * GEMM_BK;
        if (is_a && w.kind == HK_DW) k0 += buf_row;
        if (!is_a && w.kind == HK_DX) k0 += id0;
        for (int k = 0; k < w.kb; ++k, k0 += GEMM_BK) {
          const uint32_t bar = full_to + 8 * stage;
          const uint32_t dst = tiles + stage * C::STAGE_BYTES + (is_a ? 0 : C::A_BYTES);
          if (!warp_wait(empty_bar + 8 * stage, phase ^ 1u, sp.status, abort_flag)) {
            ok = false;
            break;
          }
          if (elect_one()) {
            if (leads) mbar_arrive_expect_tx(full_bar + 8 * stage, CG * C::STAGE_BYTES);
            if (!mn) {
              ld(dst, tm, bar, k0, first);
            } else {
              ld(dst, tm, bar, first, k0);
              ld(dst + MN_BOX, tm, bar, first + 64, k0);
              if (!PAIR && !is_a) {   // 256 rows of B in one CTA
                ld(dst + 2 * MN_BOX, tm, bar, first + 128, k0);
                ld(dst + 3 * MN_BOX, tm, bar, first + 192, k0);
              }
            }
          }
          if (++stage == STAGES) { stage = 0; phase ^= 1u; }
          if (leads && draw && k == w.kb - HB_DRAW) draw_unit();
          // the loads are ahead of the MMAs now: time for the next unit
          if (leads && k == max(1, w.kb - HB_TAKE)) {
            next_unit();
            handed = hand_over(it + 1, false);
            if (!ok) break;
          }
        }
        if (leads && ok && !handed) {
          if (w.kb < 2) next_unit();
          hand_over(it + 1, true);
        }
      }
      // no load may be in flight when the CTA exits (gemm_tc.cuh)
      if (leads) {
        for (int s = 0; s < STAGES; ++s) {
          const uint32_t par = (s < stage) ? phase : (phase ^ 1u);
          const uint64_t t0 = globaltimer_ns();
          while (!mbar_try_wait(full_bar + 8 * s, par)) {
            if (globaltimer_ns() - t0 > 100000000ull) break;
          }
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------ MMA issuer
    if (!PAIR || crank == 0) {
      int stage = 0;
      uint32_t phase = 0;
      int acc = 0;
      uint32_t acc_phase = 0;
      for (int it = 0;; ++it) {
        HeadUnit w;
        if (!take(it, w)) break;
        taken(it);
        if (w.kind == HK_END) break;
        const int a_mn = w.kind == HK_DW, b_mn = w.kind != HK_DZ;
        const uint32_t idesc = umma_idesc_f16(TILE_M, w.n, 1) | ((uint32_t)a_mn << 15) |
                               ((uint32_t)b_mn << 16);
        const uint64_t a_step = a_mn ? 128 : 2, b_step = b_mn ? 128 : 2;
        const int run = unit_run(w);
        bool ok = true;
        for (int k0 = 0; k0 < w.kb && ok; k0 += run) {
          if (!warp_wait(tempty_bar + 8 * acc, acc_phase ^ 1u, sp.status, abort_flag)) { ok = false; break; }
          tc_fence_after();
          const uint32_t d_tmem = tmem_base + acc * HB_BN;
          const int kn = min(run, w.kb - k0);
          for (int k = 0; k < kn; ++k) {
            if (!warp_wait(full_bar + 8 * stage, phase, sp.status, abort_flag)) { ok = false; break; }
            tc_fence_after();
            if (elect_one()) {
              const uint32_t sa = tiles + stage * C::STAGE_BYTES;
              const uint64_t ad = a_mn ? smem_desc_mn_sw128(sa, MN_BOX) : smem_desc_k_sw128(sa);
              const uint64_t bd = b_mn ? smem_desc_mn_sw128(sa + C::A_BYTES, MN_BOX)
                                       : smem_desc_k_sw128(sa + C::A_BYTES);
#pragma unroll
              for (int j = 0; j < GEMM_BK / 16; ++j)
                if constexpr (PAIR)
                  umma_f16_pair(d_tmem, ad + a_step * j, bd + b_step * j, idesc, (k | j) != 0);
                else
                  umma_f16(d_tmem, ad + a_step * j, bd + b_step * j, idesc, (k | j) != 0);
              if constexpr (PAIR) umma_commit_pair(empty_bar + 8 * stage, 0x3);
              else umma_commit(empty_bar + 8 * stage);
            }
            if (++stage == STAGES) { stage = 0; phase ^= 1u; }
          }
          if (!ok) break;
          if (elect_one()) {
            if constexpr (PAIR) umma_commit_pair(tfull_bar + 8 * acc, 0x3);
            else umma_commit(tfull_bar + 8 * acc);
          }
          if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
        }
        if (!ok) break;
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
    const int quarter = warp & 3;
    const int half = (warp - 2) >> 2;
    const uint32_t sbuf = base + STAGES * C::STAGE_BYTES + 1024 + (warp - 2) * HB_BOX;
    int acc = 0;
    uint32_t acc_phase = 0;
    // The unit whose stores others wait for: signalled when they are complete,
    // which costs nothing once the next unit's boxes or accumulator are due.
    // Never kept over a wait.
    int* owed = nullptr;
    auto settle = [&] {   // lane 0
      bulk_wait_all();
      if (owed) {
        fence_async_global();
        flag_add(owed);
        owed = nullptr;
      }
    };
    // waits for the accumulator and gives it back
    auto acquire = [&]() -> bool {
      if (lane == 0 && owed && !mbar_try_wait(tfull_bar + 8 * acc, acc_phase)) settle();
      if (!warp_wait(tfull_bar + 8 * acc, acc_phase, sp.status, abort_flag)) return false;
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
    for (int it = 0;; ++it) {
      if (lane == 0 && owed && !mbar_try_wait(sfull_bar + 8 * (it % HB_SLOTS), (it / HB_SLOTS) & 1))
        settle();
      HeadUnit w;
      if (!take(it, w)) break;
      taken(it);
      if (w.kind == HK_END) break;
      const int id0 = w.piece * sp.piece;
      const int ids = w.piece == sp.pieces - 1 ? ord.last_ids : sp.piece;
      const int y0 = w.mt * TILE_M + (int)crank * GEMM_BM + quarter * 32;   // the warp's first row
      const int n_tile = w.nt * HB_BN;
      // |dz| = 2^(c2 acc - lse2 + log2|a|) - |a| p: the coefficient goes into the
      // exponent, its sign and the rows that do not count into two masks
      TargetCursor cur;
      float mag = 0.f, shift = 0.f;
      uint32_t keep = 0u, sign = 0u;
      int best = -1;   // where rows stand twice nothing is left
      if (w.kind == HK_DZ) {
        const int m = (twin ? y0 & (HB_TWIN - 1) : y0) + lane;
        if (m < count) {
          if (!twin && dzp.best) best = dzp.best[m];
          const float2 co = dzp.coef[m];
          mag = fabsf(co.x);
          shift = co.y;
          keep = 0xffffffffu;
          sign = co.x < 0.f ? 0x80008000u : 0u;
        }
        cursor_seek<true>(dzp.t, cur, m, count, id0 + n_tile + 128 * half);
      }
      const uint32_t t_half = tmem_base + ((uint32_t)(quarter * 32) << 16) + 128 * half;
      const bool b16 = w.kind == HK_DZ || (w.kind == HK_DW && !sp.dw_f32);
      const bool rows_in = y0 < (w.kind == HK_DW ? ids : M);
      // dz in whole k-blocks of 64 ids: dx's product reads them
      const int cols_end = w.kind == HK_DZ ? (ids + 63) & ~63 : sp.dim;
      const CUtensorMap* out = w.kind == HK_DZ ? &maps.dz_out
                               : w.kind == HK_DW ? &maps.dw_out : &maps.dx_out;
      const bool add = w.kind == HK_DX ? w.piece > 0 && !sp.own_slabs : w.kind == HK_DW && sp.dw_f32;
      const int y = y0 + (w.kind == HK_DX ? (w.split + (sp.own_slabs ? w.piece * sp.splits : 0)) * sp.rows64
                          : w.kind == HK_DW ? id0 : (w.piece % HB_BUFS) * sp.rows64);
      const int n_half = n_tile + 128 * half;
      // 32 logits of columns n0 .. to dz.
      // dz is rounded once to bf16 by pack_bf16: it is the operand of two tensor-core
      // products.  Where rows stand twice, the second 64 take what the rounding of
      // the first leaves; else what it leaves at the row's (largest) target, most of
      // dz's size in one entry, is written down for dx and dw to take
      auto to_dz = [&](float (&v)[32], int n0) {
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = ex2_fast(fmaf(v[j], dzp.c2, shift));
        if (n0 + 32 > ids) {   // behind the last id of the vocabulary
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (n0 + j >= ids) v[j] = 0.f;
        }
        const int col = id0 + n0;
        while (cur.next < col + 32) {
          if (cur.next >= col) {
            const int j = cur.next - col;
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (i == j) v[i] -= mag * cur.q;
          }
          cursor_step<true>(dzp.t, cur);
        }
        if (twin && y0 >= HB_TWIN) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] -= __bfloat162float(__float2bfloat16_rn(v[j]));
        }
        const int j = best - col;
        if ((unsigned)j < 32u) {
          float d = 0.f;
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (i == j) d = v[i];
          d -= __bfloat162float(__float2bfloat16_rn(d));
          if (sign) d = -d;
          dzp.rest[y0 + lane] = d;
          const int at = atomicAdd(dzp.rests + best / 32, 1);
          if (at < HB_PUT_BACK)
            dzp.list[(best / 32) * HB_PUT_BACK + at] = make_int4(y0 + lane, best, __float_as_int(d), 0);
        }
      };
      // sends a box of 128-byte rows: 64 columns of bf16 or 32 of fp32 from column n0
      auto send = [&](const uint32_t (&o)[32], int n0) {
        if (lane == 0) {   // the previous box has left the slot
          if (owed) settle();
          else bulk_wait_read_all();
        }
        __syncwarp();
        stage_words(sbuf, lane, o);
        fence_async_smem();
        __syncwarp();
        if (lane == 0) {
          if (rows_in) {
            if (add) tma_reduce_add_2d(out, sbuf, n0, y);
            else tma_store_2d(out, sbuf, n0, y);
          }
          bulk_commit_group();
        }
      };
      const int run = unit_run(w);
      if (run < w.kb) {
        // runs before the last are added, rounded to nearest, in registers (128 of
        // them, this lane's half row), and then to the last one's accumulator
        float sum[4][32];
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
          for (int j = 0; j < 32; ++j) sum[g][j] = 0.f;
        bool ok = true;
#pragma unroll 1
        for (int k = 0; k < w.kb; k += run) {
          if (!acquire()) { ok = false; break; }
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            float v[32];
            tmem_ld32(t_half + acc * HB_BN + 32 * g, v);
#pragma unroll
            for (int j = 0; j < 32; ++j) sum[g][j] += v[j];
          }
          if (k + run < w.kb) release();
        }
        if (!ok) break;
#pragma unroll
        for (int g = 0; g < 4; ++g) tmem_st32(t_half + acc * HB_BN + 32 * g, sum[g]);
        tmem_st_wait();
      } else if (!acquire()) {
        break;
      }
      // dz has been read, as far as this unit is concerned: its loads arrived
      // before its products.  The release waits 1,500 to 3,000 cycles for this
      // thread's boxes; a piece has then units long enough to hide it.  With no
      // more pieces than buffers nobody asks.
      if (w.kind != HK_DZ && sp.pieces > HB_BUFS && warp == 2 && lane == 0 && crank == 0)
        flag_add(head_flag(sp, w.piece, HF_READ));
      if (w.kind == HK_DW && !twin && dzp.best && rows_in) {
        const int first = id0 + y0;   // the warp's ids
        const int n = __ldcg(dzp.rests + first / 32);
        const int4 e = __ldcg(dzp.list + first + lane);   // 32 places for 32 ids
        if (n > 0 && n <= HB_PUT_BACK)
          put_back(dzp, e, first, n, t_half + acc * HB_BN, n_half, min(128, sp.dim - n_half));
      }
#pragma unroll 1
      for (int c = 0; c < 128; c += b16 ? 64 : 32) {
        if (n_half + c >= cols_end) break;
        uint32_t o[32];
        if (b16) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float v[32];
            tmem_ld32(t_half + acc * HB_BN + c + 32 * h, v);
            if (w.kind == HK_DZ) to_dz(v, n_half + c + 32 * h);
            pack_bf16(v, o + 16 * h);
          }
          if (w.kind == HK_DZ) {
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] = (o[j] ^ sign) & keep;
          }
        } else {
          float v[32];
          tmem_ld32(t_half + acc * HB_BN + c, v);
#pragma unroll
          for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(v[j]);
        }
        send(o, n_half + c);
      }
      release();
      // others wait for what this unit wrote
      if (lane == 0 && w.kind != HK_DW) {
        if (owed) settle();   // a unit without a box of its own
        owed = head_flag(sp, w.piece,
                         w.kind == HK_DZ ? HF_MADE + w.nt * HB_BN / sp.split_n : HF_ADDED);
      }
    }
    if (lane == 0) settle();
  }

  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync_all();
  tc_fence_after();
  if (warp == 1) {
    if constexpr (PAIR) tmem_dealloc_pair(tmem_base, TMEM_COLS);
    else tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

}  // namespace ne
