// Eviction from a paged cache by a score per row: which rows of each KV head stay, and the move of
// those rows to pages of their own.
//
// A sequence of n > keep rows keeps, per KV head, its first `sinks` rows, its last `recent` rows and
// the keep - sinks - recent rows with the highest scores of those between (equal scores: the lower
// row; NaN counts as lowest); a sequence of at most keep rows keeps them all.  The kept rows stay in
// order, so "the last rows" means the same after the next eviction.
#pragma once

#include "paged_cache.cuh"

namespace rib {
namespace paged {

constexpr int kSelThreads = 1024, kSelWarps = kSelThreads / 32;
constexpr int kSelBins = 256;

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
  if (x != x) return 0u;
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// One CTA per (KV head, sequence).  The threshold is found by a radix walk over the keys, 8 bits a
// pass, most significant first: histogram of the candidates that match the prefix so far, then the
// bin that holds the wanted rank.  A last pass writes the kept rows in order; each warp takes a
// consecutive run of rows, so one scan over the warps' counts places them.
__global__ void __launch_bounds__(kSelThreads) select_rows_kernel(const __grid_constant__ SelectParams p) {
  __shared__ uint32_t hist[kSelBins];
  __shared__ int n_gt[kSelWarps], n_eq[kSelWarps];
  __shared__ uint32_t pick_bin, pick_rank;
  pdl_launch_dependents();
  pdl_wait();
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int given = p.lens[b];
  const int n = min(max(given, 0), p.max_len);
  if (tid == 0 && h == 0) {
    p.new_lens[b] = min(n, p.keep);
    if (given < 0 || given > p.max_len) atomicExch(&g_device_status, RIB_ECAPACITY);
  }
  const float *sc = p.scores + b * p.s_seq + h * p.s_head;
  int32_t *rows = p.rows + (static_cast<size_t>(b) * p.nkv + h) * p.keep;
  float *ns = p.new_scores ? p.new_scores + b * p.n_seq + h * p.n_head : nullptr;
  if (n <= p.keep) {
    for (int i = tid; i < p.keep; i += kSelThreads) rows[i] = i < n ? i : -1;
    if (ns)
      for (int i = tid; i < p.new_width; i += kSelThreads) ns[i] = i < n ? sc[i] : 0.f;
    return;
  }
  const int lo = p.sinks, hi = n - p.recent;        // candidates [lo, hi)
  uint32_t rank = p.keep - p.sinks - p.recent;      // of which this many stay
  uint32_t prefix = 0;                              // the key of the last one that stays
  if (rank > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < kSelBins; i += kSelThreads) hist[i] = 0;
      __syncthreads();
      const uint32_t high = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
      for (int i = lo + tid; i < hi; i += kSelThreads) {
        const uint32_t key = order_key(sc[i]);
        if ((key & high) == prefix) atomicAdd(&hist[(key >> shift) & 255u], 1u);
      }
      __syncthreads();
      if (warp == 0) {  // lane holds 8 bins, highest bins in lane 0: counts from the top
        uint32_t c[8], sum = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          c[j] = hist[255 - (8 * lane + j)];
          sum += c[j];
        }
        uint32_t inc = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint32_t up = __shfl_up_sync(0xffffffffu, inc, o);
          if (lane >= o) inc += up;
        }
        uint32_t above = inc - sum;
        if (above < rank && rank <= inc) {
          for (int j = 0; j < 8; ++j) {
            if (rank <= above + c[j]) {
              pick_bin = 255 - (8 * lane + j);
              pick_rank = rank - above;
              break;
            }
            above += c[j];
          }
        }
      }
      __syncthreads();
      prefix |= pick_bin << shift;
      rank = pick_rank;  // rank within the bin; after the last pass: how many equal keys stay
      __syncthreads();
    }
  }
  const bool any = p.keep - p.sinks - p.recent > 0;
  const int ties = any ? static_cast<int>(rank) : 0;
  // ---- ordered write: class 2 stays for certain, class 1 equals the threshold
  const int per = (n + kSelThreads - 1) / kSelThreads * 32;  // rows of a warp
  const int w_lo = min(warp * per, n), w_hi = min(w_lo + per, n);
  auto cls = [&](int i) {
    if (i >= w_hi) return 0;
    if (i < lo || i >= hi) return 2;
    if (!any) return 0;
    const uint32_t key = order_key(sc[i]);
    return key > prefix ? 2 : key == prefix ? 1 : 0;
  };
  int gt = 0, eq = 0;
  for (int i = w_lo; i < w_hi; i += 32) {
    const int k = cls(i + lane);
    gt += __popc(__ballot_sync(0xffffffffu, k == 2));
    eq += __popc(__ballot_sync(0xffffffffu, k == 1));
  }
  if (lane == 0) {
    n_gt[warp] = gt;
    n_eq[warp] = eq;
  }
  __syncthreads();
  int g0 = 0, e0 = 0;
  for (int w = 0; w < warp; ++w) {
    g0 += n_gt[w];
    e0 += n_eq[w];
  }
  const uint32_t below = (1u << lane) - 1;
  for (int i = w_lo; i < w_hi; i += 32) {
    const int k = cls(i + lane);
    const uint32_t mg = __ballot_sync(0xffffffffu, k == 2), me = __ballot_sync(0xffffffffu, k == 1);
    const int e = e0 + __popc(me & below), g = g0 + __popc(mg & below);
    if (k == 2 || (k == 1 && e < ties)) {
      const int at = g + min(e, ties);
      rows[at] = i + lane;
      if (ns) ns[at] = sc[i + lane];
    }
    g0 += __popc(mg);
    e0 += __popc(me);
  }
  if (ns)
    for (int i = p.keep + tid; i < p.new_width; i += kSelThreads) ns[i] = 0.f;
}

// Moves the kept rows: row j of the new table's sequence gets row rows[j] of the old one, K and V.
struct MoveParams {
  View from, to;               // the same pages through two tables
  const int32_t *rows;         // [B][nkv][keep]
  int keep, dim;
};

// A warp takes 32 kept rows of one KV head: each lane looks one row's two pages up, then 16-byte
// pieces move, K and V of 2 * D / 8 lanes to a row.
__global__ void __launch_bounds__(256) move_rows_kernel(const __grid_constant__ MoveParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int h = blockIdx.y, b = blockIdx.z, lane = threadIdx.x & 31;
  const int j0 = (blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32) * 32;
  if (j0 >= p.keep) return;
  const int j = j0 + lane;
  const int r = j < p.keep ? p.rows[(static_cast<size_t>(b) * p.from.nkv + h) * p.keep + j] : -1;
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
  const int vec = p.dim / 8, lanes = 2 * vec;  // 16-byte pieces of a K row; lanes of a row (32, 16)
  const int side = lane / lanes, piece = lane % lanes;
  const long long off = (piece >= vec ? p.from.s_half : 0) + (piece % vec) * 8;
  const int step = 32 / lanes;
#pragma unroll 8
  for (int i = 0; i < 32; i += step) {
    const long long s = __shfl_sync(0xffffffffu, src, i + side), d = __shfl_sync(0xffffffffu, dst, i + side);
    if (s >= 0)
      *reinterpret_cast<uint4 *>(p.to.pages + d + off) = *reinterpret_cast<const uint4 *>(p.from.pages + s + off);
  }
}

}  // namespace paged
}  // namespace rib
