// Eviction from a paged cache by a score per row: which rows of each KV head stay, and the move of
// those rows to pages of their own.
//
// A sequence of n > keep rows keeps, per KV head, its first `sinks` rows, its last `recent` rows and
// the keep - sinks - recent rows with the highest scores of those between (equal scores: the lower
// row; NaN counts as lowest); a sequence of at most keep rows keeps them all.  The kept rows stay in
// order, so "the last rows" means the same after the next eviction.
#pragma once

#include <cooperative_groups.h>

#include "paged_cache.cuh"

namespace rib {
namespace paged {

constexpr int kSelBins = 2048;

struct SelectParams {
  const float *scores;         // [B][nkv] rows, strides s_seq, s_head
  const int32_t *lens;         // [B]
  int32_t *rows;               // [B][nkv][keep]: kept rows in order, then -1
  int32_t *new_lens;           // [B]
  float *new_scores;           // [B][nkv][new_width] kept scores, then 0 (strides n_seq, n_head), or null
  long long s_seq, s_head, n_seq, n_head;
  int nkv, keep, sinks, recent, max_len, new_width;
};

// A score as an unsigned number of the same order; NaN lowest, -0 equal to +0.
__device__ __forceinline__ uint32_t order_key(float x) {
  const int u = __float_as_int(x + 0.0f);
  return x == x ? static_cast<uint32_t>(u ^ ((u >> 31) | 0x80000000)) : 0u;
}

constexpr int kSelStepRows = 32;  // rows of a thread that a CTA keeps in shared memory: a lane for each step

// The score that a key stands for (a NaN for NaN, +0 for -0).
__device__ __forceinline__ float score_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

// One cluster per (KV head, sequence); CTA r of it takes the r-th part of the rows, a warp a
// consecutive run of the part, 32 at a time, so the kept rows come out in order.
//
// The threshold, the key of the last row that stays, is found digit by digit, most significant first:
// a histogram of the candidates that match the digits found so far, summed over the cluster through
// distributed shared memory (each CTA sums a slice of the bins and hands it to all), then the bin that
// holds the wanted rank.  The walk ends early when all of that bin stays, mostly after two of the three
// digits.  The first digit is the sign, the exponent and two more bits: accumulated weights have few
// exponents, and with 8 bits a digit their additions queue at a handful of bins.
// kCached: the scores are read once and kept as keys in shared memory; longer parts are read again for
// every digit.  Reading the scores takes a few us at most; the chain of passes over the keys and the
// barriers between them bound it: 35 us for 8 x 8 heads of 65536 rows, 19 us for 32 x 8 of 300-8192.
template <int kThreads, bool kCached>
__global__ void __launch_bounds__(kThreads, 2048 / kThreads) select_rows_kernel(const __grid_constant__ SelectParams p) {
  constexpr int kWarps = kThreads / 32;
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  extern __shared__ __align__(16) uint32_t cached[];
  __shared__ uint32_t hist[2][kSelBins];  // own counts, the cluster's
  __shared__ uint32_t warp_sum[kWarps];
  __shared__ int n_gt[kWarps], n_eq[kWarps];
  __shared__ int cta_gt, cta_eq;
  __shared__ uint32_t pick_bin, pick_rank, pick_count;
  pdl_launch_dependents();
  pdl_wait();
  const int ctas = cluster.num_blocks(), rank_in = cluster.block_rank();
  const int h = blockIdx.x / ctas, b = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int given = p.lens[b];
  const int n = min(max(given, 0), p.max_len);
  if (tid == 0 && blockIdx.x == 0) {
    p.new_lens[b] = min(n, p.keep);
    if (given < 0 || given > p.max_len) atomicExch(&g_device_status, RIB_ECAPACITY);
  }
  const float *sc = p.scores + b * p.s_seq + h * p.s_head;
  int32_t *rows = p.rows + (static_cast<size_t>(b) * p.nkv + h) * p.keep;
  float *ns = p.new_scores ? p.new_scores + b * p.n_seq + h * p.n_head : nullptr;
  if (n <= p.keep) {  // the same for the whole cluster
    for (int i = rank_in * kThreads + tid; i < p.keep; i += ctas * kThreads) rows[i] = i < n ? i : -1;
    if (ns)
      for (int i = rank_in * kThreads + tid; i < p.new_width; i += ctas * kThreads) ns[i] = i < n ? sc[i] : 0.f;
    return;
  }
  // this CTA's part of the rows, and of it each warp's run of `per` times 32 rows
  const int per = (n + ctas * kThreads - 1) / (ctas * kThreads), part = per * kThreads;
  const int base = min(rank_in * part, n), mine = min(part, n - base);
  const float *from = sc + base;
  if (kCached) {
    const int four = (reinterpret_cast<uintptr_t>(from) & 15u) ? 0 : mine / 4;  // rows by 16 bytes where aligned
    for (int i = tid; i < four; i += kThreads)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(cached + 4 * i)), "l"(from + 4 * i)
                   : "memory");
    for (int i = 4 * four + tid; i < mine; i += kThreads)
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(cached + i)), "l"(from + i) : "memory");
    asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
    // a thread turns the scores that it copied itself into keys
    for (int i = tid; i < four; i += kThreads) {
      uint4 x = reinterpret_cast<uint4 *>(cached)[i];
      x = make_uint4(order_key(__uint_as_float(x.x)), order_key(__uint_as_float(x.y)),
                     order_key(__uint_as_float(x.z)), order_key(__uint_as_float(x.w)));
      reinterpret_cast<uint4 *>(cached)[i] = x;
    }
    for (int i = 4 * four + tid; i < mine; i += kThreads) cached[i] = order_key(__uint_as_float(cached[i]));
  }
  auto key_at = [&](int i) { return kCached ? cached[i] : order_key(from[i]); };
  for (int i = tid; i < kSelBins; i += kThreads) hist[0][i] = 0;
  __syncthreads();
  const int lo = p.sinks - base, hi = n - p.recent - base;      // candidates [lo, hi) of the part
  const uint32_t stay = p.keep - p.sinks - p.recent;            // of all candidates, this many stay
  uint32_t rank = stay, prefix = 0, known = 0;                  // `known`: the bits of the key found so far
  if (stay > 0) {
#pragma unroll 1
    for (int digit = 0; digit < 3; ++digit) {
      const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0;
      const uint32_t bits = digit == 2 ? 1023u : 2047u;
#pragma unroll 4
      for (int i = max(lo, 0) + tid; i < min(hi, mine); i += kThreads) {
        const uint32_t key = key_at(i);
        if ((key & known) == prefix) atomicAdd(&hist[0][(key >> shift) & bits], 1u);
      }
      const uint32_t *total = hist[0];
      if (ctas > 1) {
        cluster.sync();
        const int slice = kSelBins / ctas;  // 2, 4 or 8 CTAs
        for (int i = tid; i < slice; i += kThreads) {
          const int bin = rank_in * slice + i;
          uint32_t sum = 0;
          for (int r = 0; r < ctas; ++r) sum += cluster.map_shared_rank(hist[0], r)[bin];
          for (int r = 0; r < ctas; ++r) cluster.map_shared_rank(hist[1], r)[bin] = sum;
        }
        cluster.sync();
        total = hist[1];
      } else {
        __syncthreads();
      }
      // a few bins a thread, from the highest down: their counts, then those above
      constexpr int kBins = kSelBins / kThreads;
      uint32_t count[kBins], sum = 0;
#pragma unroll
      for (int j = 0; j < kBins; ++j) {
        count[j] = total[kSelBins - 1 - kBins * tid - j];
        sum += count[j];
      }
      uint32_t inc = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += up;
      }
      if (lane == 31) warp_sum[warp] = inc;
      __syncthreads();
      uint32_t above = inc - sum + __reduce_add_sync(0xffffffffu, lane < warp ? warp_sum[lane] : 0u);
      if (above < rank && rank <= above + sum) {
#pragma unroll
        for (int j = 0; j < kBins; ++j) {
          if (above < rank && rank <= above + count[j]) {
            pick_bin = kSelBins - 1 - kBins * tid - j;
            pick_rank = rank - above;
            pick_count = count[j];
          }
          above += count[j];
        }
      }
      for (int i = tid; i < kSelBins; i += kThreads) hist[0][i] = 0;
      __syncthreads();
      prefix |= pick_bin << shift;
      known |= bits << shift;
      rank = pick_rank;  // within the bin: at the end, how many of the rows that match the prefix stay
      if (rank == pick_count) break;
    }
  }
  const int ties = static_cast<int>(rank);
  // ---- ordered write: class 2 stays for certain, class 1 matches the threshold
  const int w_lo = warp * per * 32;
  const int in_lo = max(lo, 0), in_hi = stay ? min(hi, mine) : 0;  // rows that go by their keys
  // the classes of rows i0 .. i0 + 31 as masks
  auto classes = [&](int i0, uint32_t &mg, uint32_t &me) {
    if (i0 >= in_lo && i0 + 32 <= in_hi) {  // the same for the whole warp
      const uint32_t key = key_at(i0 + lane) & known;
      mg = __ballot_sync(0xffffffffu, key > prefix);
      me = __ballot_sync(0xffffffffu, key == prefix);
    } else {
      const int i = i0 + lane;
      const bool by_key = i >= in_lo && i < in_hi;
      const uint32_t key = by_key ? key_at(i) & known : 0;
      mg = __ballot_sync(0xffffffffu, by_key ? key > prefix : i < mine && (i < lo || i >= hi));
      me = __ballot_sync(0xffffffffu, by_key && key == prefix);
    }
  };
  // Cached: lane v keeps the classes of the run's v-th 32 rows (there are 32 of those at most), and how
  // many rows of each class come before them in the run.
  uint32_t kept_gt = 0, kept_eq = 0;
  int gt = 0, eq = 0, before_gt = 0, before_eq = 0;
#pragma unroll 4
  for (int v = 0; v < per; ++v) {
    uint32_t mg, me;
    classes(w_lo + v * 32, mg, me);
    if (kCached) {
      if (lane == v) {
        kept_gt = mg;
        kept_eq = me;
      }
    } else {
      gt += __popc(mg);
      eq += __popc(me);
    }
  }
  if (kCached) {
    gt = __popc(kept_gt);
    eq = __popc(kept_eq);
    before_gt = gt;
    before_eq = eq;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int ug = __shfl_up_sync(0xffffffffu, before_gt, o), ue = __shfl_up_sync(0xffffffffu, before_eq, o);
      if (lane >= o) {
        before_gt += ug;
        before_eq += ue;
      }
    }
    const int all_gt = __shfl_sync(0xffffffffu, before_gt, 31), all_eq = __shfl_sync(0xffffffffu, before_eq, 31);
    before_gt -= gt;
    before_eq -= eq;
    gt = all_gt;
    eq = all_eq;
  }
  if (lane == 0) {
    n_gt[warp] = gt;
    n_eq[warp] = eq;
  }
  __syncthreads();
  int g0 = __reduce_add_sync(0xffffffffu, lane < warp ? n_gt[lane] : 0);
  int e0 = __reduce_add_sync(0xffffffffu, lane < warp ? n_eq[lane] : 0);
  if (ctas > 1) {
    if (tid == kThreads - 1) {
      cta_gt = g0 + gt;
      cta_eq = e0 + eq;
    }
    cluster.sync();
    const int other = lane < rank_in ? lane : rank_in;
    g0 += __reduce_add_sync(0xffffffffu, lane < rank_in ? *cluster.map_shared_rank(&cta_gt, other) : 0);
    e0 += __reduce_add_sync(0xffffffffu, lane < rank_in ? *cluster.map_shared_rank(&cta_eq, other) : 0);
  }
  const uint32_t below = (1u << lane) - 1, bit = 1u << lane;
#pragma unroll 2
  for (int v = 0; v < per; ++v) {
    const int i = w_lo + v * 32 + lane;
    uint32_t mg, me;
    int g = g0, e = e0;
    if (kCached) {
      mg = __shfl_sync(0xffffffffu, kept_gt, v);
      me = __shfl_sync(0xffffffffu, kept_eq, v);
      g += __shfl_sync(0xffffffffu, before_gt, v);
      e += __shfl_sync(0xffffffffu, before_eq, v);
    } else {
      classes(w_lo + v * 32, mg, me);
      g0 += __popc(mg);
      e0 += __popc(me);
    }
    if (!(mg | me)) continue;
    if (me) e += __popc(me & below);
    if ((mg & bit) || ((me & bit) && e < ties)) {
      const int at = g + __popc(mg & below) + min(e, ties);
      rows[at] = base + i;
      if (ns) ns[at] = kCached ? score_of(cached[i]) : from[i];
    }
  }
  if (ns)
    for (int i = p.keep + rank_in * kThreads + tid; i < p.new_width; i += ctas * kThreads) ns[i] = 0.f;
  if (ctas > 1) cluster.sync();  // no CTA leaves while another may read its counts
}

// Moves the kept rows: row j of the new table's sequence gets row rows[j] of the old one, K and V.
struct MoveParams {
  View from, to;               // the same pages through two tables
  const int32_t *rows;         // [B][nkv][keep]
  int keep;
};

// A warp takes kMoveRows kept rows of one KV head: a lane each looks one row's two pages up, then the
// rows move in 16-byte pieces, K and V of 2 * D / 8 lanes to a row, all loads before the first store.
// Bound by memory, and at its rate: 16384 rows of 8 x 8 heads, 1.07 GB, in 166 us (6.5 TB/s).
constexpr int kMoveRows = 8, kMoveThreads = 256;

template <int D>
__global__ void __launch_bounds__(kMoveThreads) move_rows_kernel(const __grid_constant__ MoveParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int h = blockIdx.y, b = blockIdx.z, lane = threadIdx.x & 31;
  const int j0 = (blockIdx.x * (kMoveThreads / 32) + threadIdx.x / 32) * kMoveRows;
  if (j0 >= p.keep) return;
  const int j = j0 + lane;
  const int r = lane < kMoveRows && j < p.keep ? p.rows[(static_cast<size_t>(b) * p.from.nkv + h) * p.keep + j] : -1;
  long long src = -1, dst = -1;
  if (r >= 0) {
    const int a = page_of(p.from, b, r), z = page_of(p.to, b, j);
    if (a >= 0 && z >= 0) {
      src = a * p.from.s_page + (r % p.from.page_rows) * p.from.s_row + h * p.from.s_head;
      dst = z * p.to.s_page + (j % p.to.page_rows) * p.to.s_row + h * p.to.s_head;
    } else {
      atomicExch(&g_device_status, RIB_ECAPACITY);
    }
  }
  constexpr int V = D / 8, L = 2 * V, S = 32 / L;  // pieces of a K row; lanes of a row; rows of a step
  const int side = lane / L, piece = lane % L;
  const long long off = (piece >= V ? p.from.s_half : 0) + (piece % V) * 8;
  uint4 x[kMoveRows / S];
#pragma unroll
  for (int i = 0; i < kMoveRows / S; ++i) {
    const long long s = __shfl_sync(0xffffffffu, src, i * S + side);
    if (s >= 0) x[i] = *reinterpret_cast<const uint4 *>(p.from.pages + s + off);
  }
#pragma unroll
  for (int i = 0; i < kMoveRows / S; ++i) {
    const long long d = __shfl_sync(0xffffffffu, dst, i * S + side);
    if (d >= 0) *reinterpret_cast<uint4 *>(p.to.pages + d + off) = x[i];
  }
}

}  // namespace paged
}  // namespace rib
