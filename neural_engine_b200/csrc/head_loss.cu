// head_loss.cu -- losses of the language-model head straight from the hidden
// states, over a vocabulary that is walked in pieces: no logits are kept.
//
//   z_iv = scale * x_i . w_v                       x [rows, dim], w [vocab, dim], bf16
//   cross entropy:   lse_i = log sum_v exp z_iv,   loss_i = lse_i - z_{i,t_i}
//                    dz_iv = g_i (exp(z_iv - lse_i) - [v = t_i])
//   distillation:    u = z / T,  p_i = softmax of the teacher's K logits / T
//                    loss_i = T^2 sum_k p_ik (log p_ik - u_{i,c_ik} + lse_i)
//                    dz_iv = g_i T (exp(u_iv - lse_i) - sum_{k: c_ik = v} p_ik)
//   dx_i = scale sum_v dz_iv w_v,   dw_v = scale sum_i dz_iv x_i
//
// Cross entropy is the one-entry case of the same product: a dense softmax
// minus a sparse target.  So both run on
//   pack      rows that count, moved together (masked rows cost no product and
//             what stands in them, NaN included, reaches nothing)
//   teacher   p and the ids of each row, sorted (distillation)
//   forward   x . w^T on the tensor cores; the epilogue keeps per row a running
//             maximum and sum of exp2 and picks out the target's logits
//   join      the tiles' (maximum, sum) pairs of a row -> lse, loss
//   backward  per piece of the vocabulary: the logits again, turned into bf16 dz
//             by the epilogue, then dx += dz . w and dw = dz^T . x
// Nothing is added up in an order that could change: the same bits every time.
// Times in these files that stand side by side were measured side by side, on one
// card; cards differ by 5 to 10%, and a later step may have moved both.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>

#include "../../include/ne.h"
#include "gemm_tc.cuh"
#include "gemm_tmap.h"
#include "head_bwd.cuh"
#include "head_fwd.cuh"
#include "ne_ctx.h"
#include "ne_internal.h"
#include "ne_launch.cuh"

namespace ne {

// Workspaces of the head losses (ne_head_alloc), sized for the largest call.
struct HeadState {
  long long max_rows = 0, max_vocab = 0;
  int max_dim = 0, max_topk = 0;
  void* pool = nullptr;
  int* count = nullptr;           // rows that count
  int* row_of = nullptr;          // packed row -> row
  int* pos_of = nullptr;          // row -> packed row, -1 where left out
  int* keep = nullptr;            // distillation: the row has an entry
  int* target = nullptr;          // packed rows: the target, of a teacher's entries the largest
  int* best = nullptr;            // distillation: id of a row's largest entry
  float* rest = nullptr;          // packed rows: what rounding left of dz at the target
  float2* coef = nullptr;         // packed rows: a, log2|a| - lse log2 e
  int* ids = nullptr;             // [topk][rows] sorted, INT_MAX behind the last
  unsigned short* tab = nullptr;  // [rows][ids / 256 + 1] entries below each multiple of 256
  float* prob = nullptr;          // [topk][rows]
  float* neg_entropy = nullptr;   // [rows] sum p log p
  float* zt = nullptr;            // [topk][rows] target logits, log2 units
  float* lse = nullptr;           // [rows] between the passes of head_train
  float2* stats = nullptr;        // (max, sum exp2) of each row and half tile
  __nv_bfloat16* xp = nullptr;    // [rows up to 256][dim up to 64] packed x
  __nv_bfloat16* twin = nullptr;  // [128][dim up to 64] the first 64 packed rows, twice
  __nv_bfloat16* dz = nullptr;    // [3][rows up to 64][piece]
  float* dx = nullptr;            // [splits][rows up to 64][dim] sums over the pieces
  int* counters = nullptr;        // of the backward pass: units drawn, flags of the pieces, rows
                                  // with a target in each 32 ids
  int4* list = nullptr;           // HB_PUT_BACK of them
};

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLowest = -3.402823466e38f;
constexpr int kTopkMax = 256;
// dz of one piece (three are alive), and the slabs dx is summed in where its
// product is split.  Backward pass of 4096 rows with pieces of 32, 64, 128 and 256
// MB: 3.14, 3.15, 3.15, 3.10 ms (151936 ids, dim 1024; all of dz would be 1.2 GB),
// 0.262, 0.261, 0.245, 0.240 (32000 ids, dim 768, six rows in ten left out).
constexpr size_t kPieceBytes = 128u << 20;
constexpr size_t kSlabBytes = 64u << 20;

// Entries a row up to which what rounding left of dz at the largest is put back: that
// is most of the error where a row has one target (gradients of 294 rows of 71946 ids
// off float64 by 2.4e-3 of their norm in bf16, 1.66e-3 with it, which is the output's
// own rounding; of 4 entries 2.4e-3 and 2.2e-3, of 64 2.3e-3 and 2.2e-3 at 6% of the time).
constexpr int kPutBackTopk = 4;

inline size_t up(size_t n, size_t to) { return (n + to - 1) / to * to; }

// ------------------------------------------------------------------ rows
__device__ __forceinline__ bool row_counts(const int32_t* target, const int* keep, int i, int vocab) {
  if (keep) return keep[i] != 0;
  const int t = target[i];
  return t >= 0 && t < vocab;
}

// Moves the rows that count together, in order.  A block takes up to 32 rows at a
// time; how many count before its first one it counts itself (the targets stay
// in L2: 4 bytes a row, once per block), so there is no scan to wait for.  With
// more than 8192 rows a block takes several such groups, which bounds the blocks
// and so the counting.  The last PACK_FILL blocks take no rows: they count all of
// them and share the zeros behind the last (16 rows of 768 columns, forward and backward
// pass: 59.2 us, with one block for the zeros 62.8).
constexpr int PACK_ROWS = 32, PACK_FILL = 8;
int pack_rows(int rows) { return rows <= 2048 ? 8 : rows <= 8192 ? 16 : PACK_ROWS; }
int pack_groups(int rows) { return (rows + 8191) / 8192; }
struct HeadPack {
  const __nv_bfloat16* x;
  long long ldx;
  int rows, dim, vocab;
  int per, groups;          // rows a group, groups a block
  const int32_t* target;    // cross entropy
  const int* keep;          // distillation
  int* row_of;
  int* pos_of;
  int* count;
  int* target_p;
  const int* best;          // distillation: by row
  float* rest;
  __nv_bfloat16* xp;        // rows of whole 128-byte lines: what a box of 64 columns reads
  long long ldp;
  // backward
  const float* lse;
  const float* grad;        // NULL: ones
  float factor;             // T * scale (* the loss's weight)
  float2* coef;             // NULL: forward
  __nv_bfloat16* twin;      // [128][ldp] the first 64 packed rows, twice
  int* counters;
  int n_counters;
  int* status;
};
__global__ void __launch_bounds__(256) head_pack_kernel(const HeadPack p) {
  pdl_trigger();
  pdl_wait();
  for (int i = blockIdx.x * 256 + threadIdx.x; i < p.n_counters; i += gridDim.x * 256) p.counters[i] = 0;
  const int32_t* target = p.target;
  const int* keep = p.keep;
  const int rows = p.rows, vocab = p.vocab, per = p.per;
  __shared__ int before, base_s;
  __shared__ unsigned mask_s;
  const int takers = gridDim.x - PACK_FILL;
  const int block_first = (int)blockIdx.x < takers ? (int)blockIdx.x * per * p.groups : rows;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) before = 0;
  __syncthreads();
  int n = 0;
  for (int i = threadIdx.x; i < block_first; i += 256) n += row_counts(target, keep, i, vocab);
  n = __reduce_add_sync(0xffffffffu, n);
  if (lane == 0 && n) atomicAdd(&before, n);
  __syncthreads();
  for (int g = 0; g < p.groups; ++g) {
    const int first = block_first + g * per;
    if (first >= rows) break;
    if (warp == 0) {
      const int i = first + lane, base = before;
      const bool mine = lane < per && i < rows;
      const bool on = mine && row_counts(target, keep, i, vocab);
      if (!keep && mine && target[i] >= vocab) atomicExch(p.status, DEV_ERR_BOUNDS);
      const unsigned mask = __ballot_sync(0xffffffffu, on);
      const int pos = base + __popc(mask & ((1u << lane) - 1));
      if (mine) p.pos_of[i] = on ? pos : -1;
      if (on) {
        p.row_of[pos] = i;
        p.target_p[pos] = target ? target[i] : p.best[i];
        if (p.coef) {
          p.rest[pos] = 0.f;
          const float a = (p.grad ? p.grad[i] : 1.0f) * p.factor;
          p.coef[pos] = make_float2(a, log2f(fabsf(a)) - p.lse[i] * kLog2e);
        }
      }
      __syncwarp();
      if (lane == 0) {
        mask_s = mask;
        base_s = base;
        before = base + __popc(mask);
      }
    }
    __syncthreads();
    const unsigned mask = mask_s;
    const int base = base_s, vecs = p.dim / 8;
    for (int r = warp; r < per; r += 8) {
      if (!((mask >> r) & 1u)) continue;
      const uint4* src = reinterpret_cast<const uint4*>(p.x + (long long)(first + r) * p.ldx);
      const int pos = base + __popc(mask & ((1u << r) - 1));
      uint4* dst = reinterpret_cast<uint4*>(p.xp + (long long)pos * p.ldp);
      uint4* two = p.coef && pos < HB_TWIN ? reinterpret_cast<uint4*>(p.twin + (long long)pos * p.ldp)
                                           : nullptr;
#pragma unroll 4
      for (int k = lane; k < vecs; k += 32) {
        const uint4 v = src[k];
        dst[k] = v;
        if (two) two[k] = two[k + HB_TWIN * (p.ldp / 8)] = v;
      }
    }
    __syncthreads();   // mask_s and base_s are free again
  }
  if ((int)blockIdx.x >= takers) {
    const int total = before, fill = blockIdx.x - takers;
    const int stop = total > 64 ? (total + 63) / 64 * 64 : 64;
    if (fill == 0 && threadIdx.x == 0) *p.count = total;
    // zero rows up to a whole block of 64, which dw's product reduces over
    const int line = (int)(p.ldp / 8), step = 256 * PACK_FILL, at = fill * 256 + threadIdx.x;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    uint4* z = reinterpret_cast<uint4*>(p.xp + (long long)total * p.ldp);
    for (long long k = at; k < (long long)(stop - total) * line; k += step) z[k] = zero;
    if (p.coef && total < HB_TWIN) {
      z = reinterpret_cast<uint4*>(p.twin + (long long)total * p.ldp);
      for (int k = at; k < (HB_TWIN - total) * line; k += step) z[k] = z[k + HB_TWIN * line] = zero;
    }
  }
}

// One block per row, one thread per entry: the softmax over the row's entries,
// the ids sorted (each entry counts those that go before it, out of shared
// memory; equal ids keep their order and stand beside each other, each with its
// probability), and an index: how many ids are below each multiple of 256.
template <bool MAX>
__device__ __forceinline__ float block_reduce(float v, float* part, int warps) {
  v = MAX ? warp_max(v) : warp_sum(v);
  __syncthreads();   // the last use of `part`
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = part[0];
  for (int w = 1; w < warps; ++w) v = MAX ? fmaxf(v, part[w]) : v + part[w];
  return v;
}
__global__ void __launch_bounds__(kTopkMax) head_teacher_kernel(
    const int32_t* __restrict__ ids_in, const float* __restrict__ logit, int rows, int K, int vocab,
    float temperature, int* ids, float* prob, unsigned short* tab, int tab_ld, float* neg_entropy,
    int* keep, int* best, int* status) {
  pdl_trigger();
  pdl_wait();
  __shared__ int least;
  __shared__ __align__(16) unsigned sid[kTopkMax];
  __shared__ unsigned sorted[kTopkMax];
  __shared__ float part[kTopkMax / 32];
  const int r = blockIdx.x, k = threadIdx.x, warps = blockDim.x >> 5;
  int c = -1;
  float v = -INFINITY;
  if (k < K) {
    c = ids_in[(long long)r * K + k];
    v = logit[(long long)r * K + k];
    if (v == -INFINITY) c = -1;   // absent, whatever its id
    if (c >= vocab) atomicExch(status, DEV_ERR_BOUNDS);
  }
  const bool there = c >= 0 && c < vocab;
  if (!there) c = INT_MAX;
  sid[k] = (unsigned)c;
  if (k == 0) least = INT_MAX;
  const int any = __syncthreads_or(there);
  const float top = block_reduce<true>(there ? v : -INFINITY, part, warps);
  if (there && v == top) atomicMin(&least, c);   // of equal logits the lowest id
  // the differences are divided by T, not the logits: a logit / T may pass the range
  v = (v - top) / temperature;
  const float e = there ? expf(v) : 0.f;
  const float sum = block_reduce<false>(e, part, warps);
  const float p = there ? e / sum : 0.f;
  const float ent = block_reduce<false>(there && p != 0.f ? p * (v - logf(sum)) : 0.f, part, warps);
  int rank = 0;
#pragma unroll 4
  for (int j = 0; j < (int)blockDim.x; j += 4) {
    const uint4 q = *reinterpret_cast<const uint4*>(&sid[j]);
    rank += (q.x < (unsigned)c + (j < k)) + (q.y < (unsigned)c + (j + 1 < k)) +
            (q.z < (unsigned)c + (j + 2 < k)) + (q.w < (unsigned)c + (j + 3 < k));
  }
  sorted[rank] = (unsigned)c;
  if (rank < K) {
    ids[(long long)rank * rows + r] = c;
    prob[(long long)rank * rows + r] = p;
  }
  __syncthreads();
  for (int t = k; t < tab_ld; t += blockDim.x) {
    int lo = 0, hi = K;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (sorted[mid] < (unsigned)t * HB_TAB) lo = mid + 1;
      else hi = mid;
    }
    tab[(long long)r * tab_ld + t] = (unsigned short)lo;
  }
  if (k == 0) {
    keep[r] = any;
    best[r] = least;
    neg_entropy[r] = ent;
  }
}

// Joins the (maximum, sum) pairs of a row in a fixed order.  RPB rows a block
// of 256 threads: 32 where there are many rows (the pairs of 32 rows lie side
// by side), 1 where there are few (the pairs of one row do).
struct HeadJoin {
  const float2* stats;
  long long part_stride, row_stride;
  int parts, rows, vocab, n;      // n: entries a row
  const int* pos_of;              // NULL: rows are not packed
  const int32_t* target;          // cross entropy
  const int* keep;                // distillation
  const float* prob;
  const float* neg_entropy;
  const float* zt;
  float t2;                       // T^2
  float weight;
  int add;                        // to loss
  float* loss;
  float* lse;
  int* status;
};
template <int RPB>
__global__ void __launch_bounds__(256) head_join_kernel(const HeadJoin p) {
  constexpr int SL = 256 / RPB;
  pdl_trigger();
  pdl_wait();
  __shared__ float smx[SL][RPB], ssum[SL][RPB];
  const int rl = threadIdx.x % RPB, sl = threadIdx.x / RPB;
  const int i = blockIdx.x * RPB + rl;
  const bool in = i < p.rows;
  bool on = in && row_counts(p.target, p.keep, i, p.vocab);
  if (in && !p.keep && !p.pos_of && sl == 0 && p.target[i] >= p.vocab)
    atomicExch(p.status, DEV_ERR_BOUNDS);
  const int m = in && p.pos_of ? p.pos_of[i] : i;
  // this thread's first entry, on its way while the pairs are joined (with one row
  // a block it has no other)
  const bool mine = in && p.keep && sl < p.n;
  const float q0 = mine ? p.prob[(long long)sl * p.rows + i] : 0.f;
  const float z0 = mine ? p.zt[(long long)sl * p.rows + i] : 0.f;
  float mx = kLowest, sum = 0.f;
  if (on) {
    const float2* s = p.stats + m * p.row_stride;
    // four loads in flight; pairs of a slice are joined in the order of the tiles
    int k = sl;
    for (; k + 3 * SL < p.parts; k += 4 * SL) {
      float2 q[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) q[u] = s[(k + u * SL) * p.part_stride];
      const float top = fmaxf(fmaxf(fmaxf(q[0].x, q[1].x), fmaxf(q[2].x, q[3].x)), mx);
      sum *= exp2f(mx - top);
#pragma unroll
      for (int u = 0; u < 4; ++u) sum += q[u].y * exp2f(q[u].x - top);
      mx = top;
    }
    for (; k < p.parts; k += SL) {
      const float2 q = s[k * p.part_stride];
      const float top = fmaxf(mx, q.x);
      sum = sum * exp2f(mx - top) + q.y * exp2f(q.x - top);
      mx = top;
    }
  }
  smx[sl][rl] = mx;
  ssum[sl][rl] = sum;
  __syncthreads();
  for (int h = SL / 2; h >= 1; h >>= 1) {
    if (sl < h) {
      const float a = smx[sl][rl], b = smx[sl + h][rl];
      const float top = fmaxf(a, b);
      ssum[sl][rl] = ssum[sl][rl] * exp2f(a - top) + ssum[sl + h][rl] * exp2f(b - top);
      smx[sl][rl] = top;
    }
    __syncthreads();
  }
  const float lse2 = smx[0][rl] + log2f(ssum[0][rl]);
  __syncthreads();
  float part = 0.f;
  if (on && p.keep) {
    if (q0 != 0.f) part = q0 * (lse2 - z0);
    for (int k = sl + SL; k < p.n; k += SL) {
      const float q = p.prob[(long long)k * p.rows + i];
      if (q != 0.f) part += q * (lse2 - p.zt[(long long)k * p.rows + i]);
    }
  }
  ssum[sl][rl] = part;
  __syncthreads();
  if (sl == 0 && in) {
    float loss = 0.f;
    if (on && p.keep) {
      float d = 0.f;
      for (int u = 0; u < SL; ++u) d += ssum[u][rl];
      loss = p.t2 * (p.neg_entropy[i] + kLn2 * d);
    } else if (on) {
      loss = kLn2 * (lse2 - p.zt[m]);
    }
    loss *= p.weight;
    p.loss[i] = p.add ? p.loss[i] + loss : loss;
    p.lse[i] = on ? kLn2 * lse2 : 0.f;
  }
}

// dx of the rows as the caller laid them out, the slabs added in a fixed order;
// zeros where a row was left out.  A thread takes four columns of up to eight
// slabs (with more than eight slabs `groups` threads share the columns, and their
// sums are added in the groups' order): what few rows cost is the chain of loads.
// Forward and backward pass of 64 rows of 768 columns, 14 slabs that stand twice:
// 62.5 us, 67.2 without groups.
// Where rows do not stand twice, what rounding left of dz at a row's largest target
// is put back here: times that row of w.
struct HeadRest {
  const int* best;              // packed rows
  const float* rest;            // NULL: nothing is
  const __nv_bfloat16* w;
  long long ldw;
};
// (4 blocks a SM: the compiler gives the loads of eight slabs registers of their own.)
template <class T>
__global__ void __launch_bounds__(256, 4) head_dx_kernel(const float* __restrict__ acc, int slabs,
                                                      long long slab, int rows, int dim, int groups,
                                                      const int* __restrict__ pos_of, T* dx,
                                                      long long ld, int add, const int* count,
                                                      const HeadRest p) {
  pdl_trigger();
  pdl_wait();
  __shared__ float4 part[256];
  const int quads = dim / 4, cols = 256 / groups;
  const int c = threadIdx.x % cols, g = threadIdx.x / cols;
  const long long at = (long long)blockIdx.x * cols + c;
  const bool in = at < (long long)rows * quads;
  const int i = (int)(at / quads), k = (int)(at - (long long)i * quads);
  const int pos = in ? pos_of[i] : -1;
  const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
  float4 v = zero;
  if (pos >= 0) {
    // where rows stand twice, the products of dz's second part lie 64 rows further
    const bool twin = *count <= HB_TWIN;
    const int all = twin ? 2 * slabs : slabs, each = (all + groups - 1) / groups;
    float left = 0.f;
    int id = 0;
    if (p.rest && !twin && g == 0) {   // on their way while the slabs are added
      left = p.rest[pos];
      id = p.best[pos];
    }
    const float4* src = reinterpret_cast<const float4*>(acc + (long long)pos * dim) + k;
    const int end = min(all, (g + 1) * each);
    for (int u0 = g * each; u0 < end; u0 += 8) {
      float4 q[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int n = u0 + u, second = n >= slabs;
        q[u] = n < end ? src[(n - second * slabs) * (slab / 4) + second * HB_TWIN * quads] : zero;
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        v.x += q[u].x; v.y += q[u].y; v.z += q[u].z; v.w += q[u].w;
      }
    }
    if (left != 0.f) {
      const uint2 wb = *reinterpret_cast<const uint2*>(p.w + id * p.ldw + 4 * k);
      v.x = fmaf(left, __uint_as_float(wb.x << 16), v.x);
      v.y = fmaf(left, __uint_as_float(wb.x & 0xffff0000u), v.y);
      v.z = fmaf(left, __uint_as_float(wb.y << 16), v.z);
      v.w = fmaf(left, __uint_as_float(wb.y & 0xffff0000u), v.w);
    }
  }
  if (groups > 1) {
    part[threadIdx.x] = v;
    __syncthreads();
    if (g > 0) return;
    for (int u = 1; u < groups; ++u) {
      const float4 q = part[u * cols + c];
      v.x += q.x; v.y += q.y; v.z += q.z; v.w += q.w;
    }
  }
  if (!in) return;
  T* dst = dx + (long long)i * ld + 4 * k;
  if constexpr (sizeof(T) == 4) {
    if (add) {
      const float4 q = *reinterpret_cast<const float4*>(dst);
      v.x += q.x; v.y += q.y; v.z += q.z; v.w += q.w;
    }
    *reinterpret_cast<float4*>(dst) = v;
  } else {
    uint2 o;
    *reinterpret_cast<__nv_bfloat162*>(&o.x) = __floats2bfloat162_rn(v.x, v.y);
    *reinterpret_cast<__nv_bfloat162*>(&o.y) = __floats2bfloat162_rn(v.z, v.w);
    *reinterpret_cast<uint2*>(dst) = o;
  }
}

// ------------------------------------------------------------------ host
// How the forward pass tiles rows and ids.
struct LsePlan {
  int cg, clusters;           // CTAs a tile, tiles at once
  bool packed, one_row_tile;
  int bn, a_rows, stages;
  size_t smem;
};

LsePlan lse_plan(int rows, int dim, int vocab, int num_sms) {
  LsePlan p;
  p.cg = rows > GEMM_BM ? 2 : 1;
  p.one_row_tile = rows <= GEMM_BM * p.cg;
  p.packed = !p.one_row_tile;   // within one tile of rows packing saves nothing
  p.clusters = num_sms / p.cg;
  const int tile_m = GEMM_BM * p.cg, m_tiles = (rows + tile_m - 1) / tile_m;
  const double dim_kb = (dim + GEMM_BK - 1) / GEMM_BK;
  // ids a tile: what the busiest SM has to do, in ids -- whole waves of tiles,
  // about 700 cycles of hand-over a tile (a k-block takes 2 an id), and the last
  // tile's epilogue, which nothing hides
  double best = 0;
  p.bn = 256;
  for (int bn = 256; bn >= (p.cg == 2 ? 192 : 96); bn -= 16 * p.cg) {
    const long long units = (long long)m_tiles * ((vocab + bn - 1) / bn);
    const double waves = (double)((units + p.clusters - 1) / p.clusters);
    const double cost = waves * (bn + 350 / dim_kb) + 6 * bn / dim_kb;
    if (bn < 256 && p.packed && waves > 8) break;   // the rows that count are not known: 256
    if (bn == 256 || cost < best) {
      best = cost;
      p.bn = bn;
    }
  }
  p.a_rows = p.cg == 2 ? GEMM_BM : (int)up(rows, 8);
  const int a = p.a_rows * 128, b = p.bn / p.cg * 128;
  // 1 KB each for alignment and barriers; an MMA reads 128 rows of x
  const int fixed = 2048 + GEMM_BM * 128 - a;
  p.stages = std::min(HF_MAX_STAGES, (227 * 1024 - fixed) / (a + b));
  p.smem = (size_t)fixed + (size_t)p.stages * (a + b);
  return p;
}

// m-tiles whose panels of x stay in L2 while a wave of tiles reuses them (as gemm_run)
int raster_group(int rows, int dim, int tile_m) {
  const long long panel = (long long)tile_m * dim * 2, budget = 48ll << 20;
  const long long m_tiles = (rows + tile_m - 1) / tile_m;
  return panel * m_tiles > budget ? (int)std::max<long long>(1, budget / panel) : 0;
}

// What turns a logit into log2 units of the softmax.
float logit_factor(float scale, float t) { return (float)((double)scale / t * 1.4426950408889634); }

// What a call works on, after its arguments were checked.
struct HeadCall {
  const ne_head_desc* d;
  const int32_t* target = nullptr;      // cross entropy
  const ne_teacher_desc* teacher = nullptr;
  float t = 1.0f;
  int n = 1;
  float weight = 1.0f;                  // of the loss and its gradient
  bool add = false;                     // to loss and dx
};

// Arrays of no rows may be NULL, as an empty array's address often is.
ne_status head_check(ne_ctx* ctx, const ne_head_desc* d, const char* what) {
  if ((!d->x && d->rows != 0) || !d->w)
    return fail(ctx, NE_ERR_INVALID, std::string(what) + ": x or w is NULL");
  if (d->rows < 0 || d->dim <= 0 || d->vocab <= 0)
    return fail(ctx, NE_ERR_INVALID, std::string(what) + ": rows, dim or vocab out of range");
  if (d->dim % 8) return fail(ctx, NE_ERR_UNSUPPORTED, std::string(what) + ": dim must be a multiple of 8");
  if (d->ldx < d->dim || d->ldw < d->dim || d->ldx % 8 || d->ldw % 8)
    return fail(ctx, NE_ERR_INVALID,
                std::string(what) + ": ldx and ldw must be multiples of 8, at least dim");
  if ((reinterpret_cast<uintptr_t>(d->x) | reinterpret_cast<uintptr_t>(d->w)) & 15u)
    return fail(ctx, NE_ERR_INVALID, std::string(what) + ": x and w must be 16-byte aligned");
  if (!(d->scale > 0.f) || !std::isfinite(d->scale * kLog2e))
    return fail(ctx, NE_ERR_INVALID, std::string(what) + ": scale must be positive and finite");
  const HeadState* h = ctx->head;
  if (!h || d->rows > h->max_rows || d->dim > h->max_dim || d->vocab > h->max_vocab)
    return fail(ctx, NE_ERR_STATE, std::string(what) + ": ne_head_alloc has no room for this call");
  return NE_OK;
}

ne_status teacher_check(ne_ctx* ctx, const ne_head_desc* d, const ne_teacher_desc* t, const char* what) {
  if ((d->rows != 0 && (!t->ids || !t->logits)) || t->topk <= 0)
    return fail(ctx, NE_ERR_INVALID, std::string(what) + ": teacher ids, logits or topk missing");
  if (t->topk > kTopkMax)
    return fail(ctx, NE_ERR_UNSUPPORTED, std::string(what) + ": topk is at most 256");
  if (!(t->temperature > 0.f) || !std::isfinite(t->temperature))
    return fail(ctx, NE_ERR_INVALID, std::string(what) + ": temperature must be positive and finite");
  // what the kernels multiply by: an id behind the vocabulary's end counts as -inf
  // times scale / T, which may not be 0, and the loss is T^2 times sums that grow
  // with 1 / T, so T^2 may not lose bits to its exponent
  const float u = d->scale / t->temperature * kLog2e, t2 = t->temperature * t->temperature;
  if (!std::isnormal(t2) || !std::isfinite(d->scale * t->temperature) || !std::isfinite(u) || !(u > 0.f))
    return fail(ctx, NE_ERR_INVALID, std::string(what) + ": temperature out of range");
  if (t->topk > ctx->head->max_topk)
    return fail(ctx, NE_ERR_STATE, std::string(what) + ": ne_head_alloc has no room for this topk");
  return NE_OK;
}

int tab_entries(int vocab) { return (vocab + HB_TAB - 1) / HB_TAB; }

ne_status enqueue_teacher(ne_ctx* ctx, const HeadCall& c) {
  if (!c.teacher) return NE_OK;
  HeadState* h = ctx->head;
  const int rows = c.d->rows;
  NE_LAUNCH(launch_k(head_teacher_kernel, dim3(rows), dim3((unsigned)up(c.n, 32)), 0, ctx->st,
                     c.teacher->ids, c.teacher->logits, rows, c.n, c.d->vocab, c.t, h->ids, h->prob,
                     h->tab, tab_entries(c.d->vocab), h->neg_entropy, h->keep, h->best,
                     ctx->d_status));
  return NE_OK;
}

// lse: the backward pass's (NULL: forward)
ne_status enqueue_pack(ne_ctx* ctx, const HeadCall& c, const float* lse, const float* grad, int counters) {
  HeadState* h = ctx->head;
  HeadPack p{};
  p.x = (const __nv_bfloat16*)c.d->x;
  p.ldx = c.d->ldx;
  p.rows = c.d->rows;
  p.dim = c.d->dim;
  p.vocab = c.d->vocab;
  p.per = pack_rows(p.rows);
  p.groups = pack_groups(p.rows);
  const int block_rows = p.per * p.groups;
  p.target = c.target;
  p.keep = c.teacher ? h->keep : nullptr;
  p.row_of = h->row_of;
  p.pos_of = h->pos_of;
  p.count = h->count;
  p.target_p = h->target;
  p.best = h->best;
  p.rest = h->rest;
  p.xp = h->xp;
  p.ldp = (long long)up(p.dim, GEMM_BK);
  p.lse = lse;
  p.grad = grad;
  p.factor = c.t * c.d->scale * c.weight;
  p.coef = lse ? h->coef : nullptr;
  p.counters = h->counters;
  p.n_counters = counters;
  p.twin = h->twin;
  p.status = ctx->d_status;
  NE_LAUNCH(launch_k(head_pack_kernel, dim3((p.rows + block_rows - 1) / block_rows + PACK_FILL),
                     dim3(256), 0, ctx->st, p));
  return NE_OK;
}

// Cross entropy's packed targets lie by packed row, a teacher's entries by row.
HeadTargets targets_of(const HeadState* h, const HeadCall& c, bool packed) {
  HeadTargets t{};
  t.ids = c.teacher ? h->ids : packed ? h->target : c.target;
  t.prob = c.teacher ? h->prob : nullptr;
  t.row_of = packed && c.teacher ? h->row_of : nullptr;
  t.tab = c.teacher ? h->tab : nullptr;
  t.tab_ld = tab_entries(c.d->vocab);
  t.ld = c.d->rows;
  t.n = c.n;
  return t;
}

template <int CG, bool LONG>
cudaError_t launch_lse(const CUtensorMap& x, const CUtensorMap& w, const HeadLse& p,
                       const LsePlan& plan, long long units, cudaStream_t st) {
  auto kern = head_lse_kernel<CG, LONG>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)plan.smem);
  if (e != cudaSuccess) return e;
  const int grid = CG * (int)std::min<long long>(units, plan.clusters);
  if constexpr (CG == 2)
    return launch_k_cluster(kern, dim3(grid), dim3(HB_THREADS), plan.smem, st, 2u, x, w, p);
  else
    return launch_k(kern, dim3(grid), dim3(HB_THREADS), plan.smem, st, x, w, p);
}

ne_status head_forward(ne_ctx* ctx, const HeadCall& c, float* loss, float* lse) {
  HeadState* h = ctx->head;
  const ne_head_desc& d = *c.d;
  const int rows = d.rows, V = d.vocab, D = d.dim;
  ne_status s;
  if ((s = enqueue_teacher(ctx, c)) != NE_OK) return s;
  const LsePlan plan = lse_plan(rows, D, V, ctx->num_sms);
  if (plan.packed && (s = enqueue_pack(ctx, c, nullptr, nullptr, 0)) != NE_OK) return s;
  const int tile_m = GEMM_BM * plan.cg;
  const int n_tiles = (V + plan.bn - 1) / plan.bn;
  const long long units = (long long)((rows + tile_m - 1) / tile_m) * n_tiles;
  const int parts = 2 * (plan.one_row_tile ? (int)std::min<long long>(units, plan.clusters) : n_tiles);
  HeadLse p{};
  p.dim_kb = (D + GEMM_BK - 1) / GEMM_BK;
  const int runs = (p.dim_kb + HF_RUN_KB - 1) / HF_RUN_KB;
  p.run_kb = (p.dim_kb + runs - 1) / runs;
  const bool lng = runs > 1;
  p.t = targets_of(h, c, plan.packed);
  p.d_rows = plan.packed ? h->count : nullptr;
  p.status = ctx->d_status;
  p.stats = h->stats;
  p.part_stride = plan.one_row_tile ? 1 : rows;
  p.row_stride = plan.one_row_tile ? parts : 1;
  p.zt = h->zt;
  p.c2 = logit_factor(d.scale, c.t);
  p.rows = rows;
  p.vocab = V;
  p.bn = plan.bn;
  p.n_tiles = n_tiles;
  p.group_m = raster_group(rows, D, tile_m);
  p.a_rows = plan.a_rows;
  p.stages = plan.stages;
  p.one_row_tile = plan.one_row_tile;
  CUtensorMap x, w;
  const long long ldx = plan.packed ? (long long)up(D, GEMM_BK) : d.ldx;
  if (!make_tmap(&x, plan.packed ? h->xp : d.x, rows, D, ldx, plan.a_rows, 0) ||
      !make_tmap(&w, d.w, V, D, d.ldw, plan.bn / plan.cg, 0))
    return fail(ctx, NE_ERR_CUDA, "head loss: tensor map");
  if (plan.cg == 2 && lng) NE_LAUNCH((launch_lse<2, true>(x, w, p, plan, units, ctx->st)));
  else if (plan.cg == 2) NE_LAUNCH((launch_lse<2, false>(x, w, p, plan, units, ctx->st)));
  else if (lng) NE_LAUNCH((launch_lse<1, true>(x, w, p, plan, units, ctx->st)));
  else NE_LAUNCH((launch_lse<1, false>(x, w, p, plan, units, ctx->st)));
  HeadJoin j{};
  j.stats = h->stats;
  j.part_stride = p.part_stride;
  j.row_stride = p.row_stride;
  j.parts = parts;
  j.rows = rows;
  j.vocab = V;
  j.n = c.n;
  j.pos_of = plan.packed ? h->pos_of : nullptr;
  j.target = c.target;
  j.keep = c.teacher ? h->keep : nullptr;
  j.prob = h->prob;
  j.neg_entropy = h->neg_entropy;
  j.zt = h->zt;
  j.t2 = c.t * c.t;
  j.weight = c.weight;
  j.add = c.add;
  j.loss = loss;
  j.lse = lse;
  j.status = ctx->d_status;
  if (plan.packed)
    NE_LAUNCH(launch_k(head_join_kernel<32>, dim3((rows + 31) / 32), dim3(256), 0, ctx->st, j));
  else
    NE_LAUNCH(launch_k(head_join_kernel<1>, dim3(rows), dim3(256), 0, ctx->st, j));
  return NE_OK;
}

// How the backward pass walks the vocabulary.
struct HeadPlan {
  int cg, tile_m, clusters;   // CTAs a tile, rows a tile, clusters at once
  int piece, pieces;          // ids a piece (whole tiles), pieces
  int split_n, splits;        // ids a split of dx's product
  bool own_slabs;             // pieces do not add up into the same slabs
};

HeadPlan head_plan(int rows, int dim, int vocab, int num_sms) {
  HeadPlan p;
  // one CTA's 128 rows where they are enough, else pairs of CTAs
  p.cg = rows > GEMM_BM ? 2 : 1;
  p.tile_m = GEMM_BM * p.cg;
  p.clusters = num_sms / p.cg;
  const long long rows64 = up(rows, 64);
  const long long room = std::max<long long>(HB_BN, (long long)(kPieceBytes / 2) / rows64 / HB_BN * HB_BN);
  p.pieces = (int)((vocab + room - 1) / room);
  p.piece = (int)up((vocab + p.pieces - 1) / p.pieces, HB_BN);
  p.pieces = (vocab + p.piece - 1) / p.piece;
  // dx's units are the longest: where there are few of them the piece is split
  // until a unit is half of what a pair has to do for dx and dw (64 rows of 32000
  // ids, forward and backward: 62.5 us with two thirds, 59.8, 60.4 with a third; 256
  // rows: 70.7, 71.1, 74.3; each split is a slab more to write and read), but not
  // below 8 k-blocks, about what a unit's own hand-over and epilogue cost (19 rows
  // of 2668 ids: 43.0 us with 8 or 6, 43.8 with 12, 45.4 with 16, 49.0 with 32; calls
  // with more to do than one unit a pair do not come to it).  dw's units cost 9
  // k-blocks at least, their epilogue.
  const double m_tiles = (double)((rows + p.tile_m - 1) / p.tile_m);
  const double d_tiles = (dim + HB_BN - 1) / HB_BN;
  const double piece_kb = p.piece / GEMM_BK;
  const double load = m_tiles * d_tiles * piece_kb +
                      (p.piece / p.tile_m) * d_tiles * std::max(9.0, (double)(rows64 / GEMM_BK));
  const double most = std::max(8.0, load / p.clusters / 2);
  const long long slabs = std::max<long long>(1, (long long)kSlabBytes / (rows64 * dim * 4));
  const long long want =
      std::max<long long>(1, std::min<long long>((long long)std::ceil(piece_kb / most), slabs));
  p.split_n = (int)up((p.piece + want - 1) / want, HB_BN);
  p.splits = (p.piece + p.split_n - 1) / p.split_n;
  // with room for it, no piece's dx waits for the piece before
  p.own_slabs = (long long)p.splits * p.pieces <= slabs;
  return p;
}

template <int CG>
cudaError_t launch_walk(const HeadMaps& maps, const HeadWalk& walk, const HeadDz& dz, int clusters,
                        cudaStream_t st) {
  auto kern = head_walk_kernel<CG>;
  const size_t smem = HeadCfg<CG>::SMEM;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  if constexpr (CG == 2)
    return launch_k_cluster(kern, dim3(2 * clusters), dim3(HB_THREADS), smem, st, 2u, maps, walk, dz);
  else
    return launch_k(kern, dim3(clusters), dim3(HB_THREADS), smem, st, maps, walk, dz);
}

ne_status head_backward(ne_ctx* ctx, const HeadCall& c, const float* lse, const float* grad,
                        const ne_head_grads* g) {
  HeadState* h = ctx->head;
  const ne_head_desc& d = *c.d;
  const int rows = d.rows, V = d.vocab, D = d.dim;
  const int rows64 = std::max((int)up(rows, 64), 2 * HB_TWIN);   // few rows stand twice
  const HeadPlan plan = head_plan(rows64, D, V, ctx->num_sms);
  const int flags = 1 + plan.pieces * (2 + plan.splits);
  const bool put_back = c.n <= kPutBackTopk;
  ne_status s;
  if ((s = enqueue_teacher(ctx, c)) != NE_OK ||
      (s = enqueue_pack(ctx, c, lse, grad, flags + (V + 31) / 32)) != NE_OK)
    return s;
  HeadDz dz{};
  dz.t = targets_of(h, c, true);
  dz.coef = h->coef;
  dz.c2 = logit_factor(d.scale, c.t);
  dz.best = put_back ? h->target : nullptr;
  dz.rest = h->rest;
  dz.rests = h->counters + flags;
  dz.list = h->list;
  dz.x = h->xp;
  dz.ldp = (long long)up(D, GEMM_BK);
  const CUtensorMapDataType bf = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, f32 = CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
  const long long ldp = (long long)up(D, GEMM_BK);
  const int esz = g->dw_f32 ? 4 : 2, dz_rows = HB_BUFS * rows64;
  HeadMaps maps;
  bool ok = make_tmap(&maps.x_k, h->xp, rows64, D, ldp, GEMM_BM, 0) &&
            make_tmap(&maps.w_k, d.w, V, D, d.ldw, HB_BN / plan.cg, 0) &&
            make_tmap_out(&maps.dz_out, h->dz, dz_rows, plan.piece, plan.piece, bf, 2, 64) &&
            make_tmap(&maps.dz_k, h->dz, dz_rows, plan.piece, plan.piece, GEMM_BM, 0) &&
            make_tmap_mn(&maps.w_mn, d.w, D, V, d.ldw) &&
            make_tmap_out(&maps.dx_out, h->dx, plan.splits * (plan.own_slabs ? plan.pieces : 1) * rows64,
                          D, D, f32, 4, 32) &&
            make_tmap_mn(&maps.dz_mn, h->dz, plan.piece, dz_rows, plan.piece) &&
            make_tmap_mn(&maps.x_mn, h->xp, D, rows64, ldp) &&
            make_tmap(&maps.twin_k, h->twin, 2 * HB_TWIN, D, ldp, GEMM_BM, 0) &&
            make_tmap_mn(&maps.twin_mn, h->twin, D, 2 * HB_TWIN, ldp);
  maps.dw_out = maps.dx_out;   // not used without dw
  if (ok && g->dw)
    ok = make_tmap_out(&maps.dw_out, g->dw, V, D, g->lddw, g->dw_f32 ? f32 : bf, esz, 128 / esz);
  if (!ok) return fail(ctx, NE_ERR_CUDA, "head loss: tensor map");
  HeadWalk walk{};
  walk.d_rows = h->count;
  walk.counters = h->counters;
  walk.status = ctx->d_status;
  walk.rows64 = rows64;
  walk.vocab = V;
  walk.dim = D;
  walk.dim_kb = (D + GEMM_BK - 1) / GEMM_BK;
  walk.dim_tiles = (D + HB_BN - 1) / HB_BN;
  walk.piece = plan.piece;
  walk.pieces = plan.pieces;
  walk.split_n = plan.split_n;
  walk.splits = plan.splits;
  walk.own_slabs = plan.own_slabs;
  walk.want_dx = g->dx != nullptr;
  walk.want_dw = g->dw != nullptr;
  walk.dw_f32 = g->dw_f32 != 0;
  if (plan.cg == 2) NE_LAUNCH(launch_walk<2>(maps, walk, dz, plan.clusters, ctx->st));
  else NE_LAUNCH(launch_walk<1>(maps, walk, dz, plan.clusters, ctx->st));
  if (g->dx) {
    const long long slab = (long long)rows64 * D;
    // the last piece may have fewer splits than the others
    const int last = V - (plan.pieces - 1) * plan.piece;
    const int slabs = !plan.own_slabs && plan.pieces > 1
                          ? plan.splits
                          : (plan.pieces - 1) * plan.splits + (last + plan.split_n - 1) / plan.split_n;
    const int loads = rows <= HB_TWIN ? 2 * slabs : slabs;
    int groups = 1;
    while (groups < 8 && loads > 8 * groups) groups *= 2;
    const int cols = 256 / groups;
    const dim3 grid((unsigned)(((long long)rows * (D / 4) + cols - 1) / cols));
    const HeadRest rest{h->target, put_back ? h->rest : nullptr, (const __nv_bfloat16*)d.w, d.ldw};
    if (g->dx_f32)
      NE_LAUNCH(launch_k(head_dx_kernel<float>, grid, dim3(256), 0, ctx->st, (const float*)h->dx,
                         slabs, slab, rows, D, groups, (const int*)h->pos_of, (float*)g->dx, g->lddx,
                         (int)c.add, (const int*)h->count, rest));
    else
      NE_LAUNCH(launch_k(head_dx_kernel<__nv_bfloat16>, grid, dim3(256), 0, ctx->st,
                         (const float*)h->dx, slabs, slab, rows, D, groups, (const int*)h->pos_of,
                         (__nv_bfloat16*)g->dx, g->lddx, 0, (const int*)h->count, rest));
  }
  return NE_OK;
}

ne_status grads_check(ne_ctx* ctx, const ne_head_desc* d, const ne_head_grads* g, const char* what) {
  if (!g->dx && !g->dw && d->rows != 0)
    return fail(ctx, NE_ERR_INVALID, std::string(what) + ": no gradient asked for");
  if ((g->dx && (g->lddx < d->dim || g->lddx % 8)) || (g->dw && (g->lddw < d->dim || g->lddw % 8)))
    return fail(ctx, NE_ERR_INVALID,
                std::string(what) + ": lddx and lddw must be multiples of 8, at least dim");
  if ((reinterpret_cast<uintptr_t>(g->dx) | reinterpret_cast<uintptr_t>(g->dw)) & 15u)
    return fail(ctx, NE_ERR_INVALID, std::string(what) + ": dx and dw must be 16-byte aligned");
  return NE_OK;
}

// No rows: dw of no rows is zero where it is written, and stays where it is added to.
ne_status no_rows(ne_ctx* ctx, const ne_head_desc* d, const ne_head_grads* g) {
  if (g->dw && !g->dw_f32)
    NE_CUDA(cudaMemset2DAsync(g->dw, (size_t)g->lddw * 2, 0, (size_t)d->dim * 2, (size_t)d->vocab,
                              ctx->st));
  return NE_OK;
}

}  // namespace

ne_status head_train(ne_ctx* ctx, const ne_head_desc* d, const int32_t* target,
                     const ne_teacher_desc* teacher, float hard, float weight, float* loss, float* dx,
                     float* dw) {
  const char* what = "ne_lmhead_distill_fwd_bwd";
  ne_status s = head_check(ctx, d, what);
  if (s != NE_OK || (teacher && (s = teacher_check(ctx, d, teacher, what)) != NE_OK)) return s;
  const ne_head_grads g{dx, d->dim, 1, dw, d->dim, 1};
  HeadCall c;
  c.d = d;
  for (int part = 0; part < 2; ++part) {
    const float share = part == 0 ? 1.0f - hard : hard;
    if (share == 0.f) continue;
    c.teacher = part == 0 ? teacher : nullptr;
    c.target = part == 0 ? nullptr : target;
    c.t = c.teacher ? teacher->temperature : 1.0f;
    c.n = c.teacher ? teacher->topk : 1;
    c.weight = share;
    if ((s = head_forward(ctx, c, loss, ctx->head->lse)) != NE_OK) return s;
    c.weight = share * weight;
    if ((s = head_backward(ctx, c, ctx->head->lse, nullptr, &g)) != NE_OK) return s;
    c.add = true;
  }
  return NE_OK;
}

void free_head(ne_ctx* ctx) {
  if (!ctx->head) return;
  if (ctx->head->pool) cudaFree(ctx->head->pool);
  delete ctx->head;
  ctx->head = nullptr;
}

}  // namespace ne

using namespace ne;

extern "C" {

NE_API ne_status ne_head_alloc(ne_ctx* ctx, int max_rows, int max_dim, int max_vocab, int max_topk) {
  if (!ctx) return NE_ERR_INVALID;
  if (max_rows <= 0 || max_dim <= 0 || max_vocab <= 0 || max_topk < 0)
    return fail(ctx, NE_ERR_INVALID, "ne_head_alloc: sizes out of range");
  if (max_dim % 8) return fail(ctx, NE_ERR_UNSUPPORTED, "ne_head_alloc: dim must be a multiple of 8");
  if (max_topk > kTopkMax) return fail(ctx, NE_ERR_UNSUPPORTED, "ne_head_alloc: topk is at most 256");
  if (max_rows > (1 << 22))
    return fail(ctx, NE_ERR_UNSUPPORTED, "ne_head_alloc: at most 4194304 rows a call");
  if (max_dim > (1 << 28) || max_vocab > (1 << 28))   // the kernels count in 32 bits
    return fail(ctx, NE_ERR_UNSUPPORTED, "ne_head_alloc: dim and vocab are at most 268435456");
  HeadState n;
  n.max_rows = max_rows;
  n.max_dim = max_dim;
  n.max_vocab = max_vocab;
  n.max_topk = max_topk;
  if (const HeadState* o = ctx->head) {
    if (max_rows <= o->max_rows && max_dim <= o->max_dim && max_vocab <= o->max_vocab &&
        max_topk <= o->max_topk)
      return NE_OK;
    n.max_rows = std::max(n.max_rows, o->max_rows);
    n.max_dim = std::max(n.max_dim, o->max_dim);
    n.max_vocab = std::max(n.max_vocab, o->max_vocab);
    n.max_topk = std::max(n.max_topk, o->max_topk);
  }
  NE_CUDA(cudaSetDevice(ctx->device));
  cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
  NE_CUDA(cudaStreamIsCapturing(ctx->st, &cs));
  if (cs != cudaStreamCaptureStatusNone)
    return fail(ctx, NE_ERR_STATE, "ne_head_alloc inside a capture");
  NE_CUDA(cudaStreamSynchronize(ctx->st));
  free_head(ctx);
  const size_t R = n.max_rows, R256 = up(R, 256), D = n.max_dim, V = n.max_vocab;
  const size_t R64 = std::max<size_t>(up(R, 64), 2 * HB_TWIN);   // few rows stand twice
  const size_t K = std::max(n.max_topk, 1);
  // a piece is at least 256 ids wide, whatever the rows
  const size_t dz = std::min<size_t>(std::max<size_t>(kPieceBytes, R64 * HB_BN * 2),
                                     R64 * up(V, HB_BN) * 2);
  // pairs of a row: two a tile of at least 192 ids, or two a CTA where there is
  // one tile of rows
  const size_t pairs = std::max(2 * ((V + 191) / 192) * R, (size_t)2 * ctx->num_sms * 2 * GEMM_BM);
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t at = off;
    off += up(bytes, 1024);
    return at;
  };
  const size_t o_count = take(4), o_row = take(up(R, 64) * 4), o_pos = take(R * 4);
  const size_t o_keep = take(R * 4), o_ids = take(K * R * 4), o_prob = take(K * R * 4);
  const size_t o_ent = take(R * 4), o_zt = take(K * R * 4), o_stats = take(pairs * 8);
  const size_t o_lse = take(R * 4), o_xp = take(R256 * up(D, GEMM_BK) * 2);
  const size_t o_twin = take(2 * HB_TWIN * up(D, GEMM_BK) * 2), o_target = take(R * 4);
  const size_t o_coef = take(R * 8), o_dz = take(HB_BUFS * dz);
  const size_t o_tab = take(n.max_topk ? R * (size_t)tab_entries((int)V) * 2 : 2);
  const size_t o_dx = take(std::max(R64 * D * 4, kSlabBytes));
  const size_t o_counters = take((4 * (up(V, HB_BN) / HB_BN + 1) + 1 + (V + 31) / 32) * 4);
  const size_t o_list = take((V + 31) / 32 * HB_PUT_BACK * 16);
  const size_t o_best = take(R * 4), o_rest = take(R * 4);
  uint8_t* b = nullptr;
  ne_status s = dalloc(ctx, &b, off);
  if (s != NE_OK) {
    cudaGetLastError();   // reported here, and not by a later launch
    return s;
  }
  n.pool = b;
  n.count = (int*)(b + o_count);
  n.row_of = (int*)(b + o_row);
  n.pos_of = (int*)(b + o_pos);
  n.keep = (int*)(b + o_keep);
  n.ids = (int*)(b + o_ids);
  n.prob = (float*)(b + o_prob);
  n.target = (int*)(b + o_target);
  n.best = (int*)(b + o_best);
  n.rest = (float*)(b + o_rest);
  n.list = (int4*)(b + o_list);
  n.coef = (float2*)(b + o_coef);
  n.tab = (unsigned short*)(b + o_tab);
  n.neg_entropy = (float*)(b + o_ent);
  n.zt = (float*)(b + o_zt);
  n.stats = (float2*)(b + o_stats);
  n.lse = (float*)(b + o_lse);
  n.xp = (__nv_bfloat16*)(b + o_xp);
  n.twin = (__nv_bfloat16*)(b + o_twin);
  n.dz = (__nv_bfloat16*)(b + o_dz);
  n.dx = (float*)(b + o_dx);
  n.counters = (int*)(b + o_counters);
  ctx->head = new HeadState(n);
  return NE_OK;
}

NE_API ne_status ne_head_ce_fwd(ne_ctx* ctx, const ne_head_desc* d, const int32_t* d_target,
                                float* d_loss, float* d_lse) {
  if (!ctx || !d) return NE_ERR_INVALID;
  if (d->rows != 0 && (!d_target || !d_loss || !d_lse))
    return fail(ctx, NE_ERR_INVALID, "ne_head_ce_fwd: target, loss or lse is NULL");
  ne_status s = head_check(ctx, d, "ne_head_ce_fwd");
  if (s != NE_OK || d->rows == 0) return s;
  NE_CUDA(cudaSetDevice(ctx->device));
  HeadCall c;
  c.d = d;
  c.target = d_target;
  return head_forward(ctx, c, d_loss, d_lse);
}

NE_API ne_status ne_head_ce_bwd(ne_ctx* ctx, const ne_head_desc* d, const int32_t* d_target,
                                const float* d_lse, const float* d_grad, const ne_head_grads* g) {
  if (!ctx || !d || !g) return NE_ERR_INVALID;
  if (d->rows != 0 && (!d_target || !d_lse))
    return fail(ctx, NE_ERR_INVALID, "ne_head_ce_bwd: target or lse is NULL");
  ne_status s = head_check(ctx, d, "ne_head_ce_bwd");
  if (s != NE_OK || (s = grads_check(ctx, d, g, "ne_head_ce_bwd")) != NE_OK) return s;
  NE_CUDA(cudaSetDevice(ctx->device));
  if (d->rows == 0) return no_rows(ctx, d, g);
  HeadCall c;
  c.d = d;
  c.target = d_target;
  return head_backward(ctx, c, d_lse, d_grad, g);
}

NE_API ne_status ne_head_distill_fwd(ne_ctx* ctx, const ne_head_desc* d, const ne_teacher_desc* t,
                                     float* d_loss, float* d_lse) {
  if (!ctx || !d || !t) return NE_ERR_INVALID;
  if (d->rows != 0 && (!d_loss || !d_lse))
    return fail(ctx, NE_ERR_INVALID, "ne_head_distill_fwd: loss or lse is NULL");
  ne_status s = head_check(ctx, d, "ne_head_distill_fwd");
  if (s != NE_OK || (s = teacher_check(ctx, d, t, "ne_head_distill_fwd")) != NE_OK || d->rows == 0)
    return s;
  NE_CUDA(cudaSetDevice(ctx->device));
  HeadCall c;
  c.d = d;
  c.teacher = t;
  c.t = t->temperature;
  c.n = t->topk;
  return head_forward(ctx, c, d_loss, d_lse);
}

NE_API ne_status ne_head_distill_bwd(ne_ctx* ctx, const ne_head_desc* d, const ne_teacher_desc* t,
                                     const float* d_lse, const float* d_grad,
                                     const ne_head_grads* g) {
  if (!ctx || !d || !t || !g) return NE_ERR_INVALID;
  if (d->rows != 0 && !d_lse) return fail(ctx, NE_ERR_INVALID, "ne_head_distill_bwd: lse is NULL");
  ne_status s = head_check(ctx, d, "ne_head_distill_bwd");
  if (s != NE_OK || (s = teacher_check(ctx, d, t, "ne_head_distill_bwd")) != NE_OK ||
      (s = grads_check(ctx, d, g, "ne_head_distill_bwd")) != NE_OK)
    return s;
  NE_CUDA(cudaSetDevice(ctx->device));
  if (d->rows == 0) return no_rows(ctx, d, g);
  HeadCall c;
  c.d = d;
  c.teacher = t;
  c.t = t->temperature;
  c.n = t->topk;
  return head_backward(ctx, c, d_lse, d_grad, g);
}

}  // extern "C"
