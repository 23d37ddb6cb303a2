// Attention of one new token per sequence over a paged cache, split over the rows and joined.
//
//   o_h = sum_n p_hn v_n,   p_hn = exp(scale q_h.k_n) / sum_m exp(scale q_h.k_m),   n < lens[b],
// with any number of query heads per KV head, head dims 64 and 128, BF16 or FP16.  Optionally the
// weight that each row of each KV head received, w[b][kvh][n] = sum over the head's query heads of
// p_hn, is added to a score per row (what an eviction goes by).
//
// Work split: the unit is (sequence, KV head, 8 query heads).  The tiles of TK rows of all units lie
// on one line, unit after unit, and every CTA of one wave takes an equal run of them, found from the
// lengths on the device: ragged batches and single long sequences fill the GPU alike, and the host
// never needs the lengths.  A CTA writes the units that lie wholly in its run, and one partial
// (m, l, o) for the unit its run begins within and one for the unit it ends within; join_kernel sums
// those in run order.  Nothing in the workspace has to be cleared, and no order depends on timing.
//
// In a CTA each of NW warps takes every NW-th tile and feeds itself: lane 0 copies its next tiles into
// a ring of ST slots of the warp's own by TMA (one 5-D box per 64 dims: 16 rows of K and of V of one
// page), so warps never wait for each other within a unit.  Scores and P.V run on mma.m16n8k16 with
// the heads as the 16 rows.  A decode step reads 2 D bytes per row for 4 D flops per query head, so
// memory bounds it at any group size here; at 8 heads per KV head the tensor pipe is busy for under a
// fifth of the time a tile's copy takes, and a tcgen05 tile (128 rows at least, accumulators in TMEM)
// would add a round trip through TMEM for rows that stay empty.  The upper 8 rows of the A operand are
// free with 8 heads: in P.V they carry p - round(p), so P enters with 16 (BF16) or 22 (FP16) bits and
// its rounding adds nothing to the output's.
#pragma once

#include <cuda.h>

#include "paged_cache.cuh"

namespace rib {
namespace paged {

constexpr int TK = 16;        // rows of a tile: one TMA box, one page at most
constexpr int NW = 4;         // warps of a CTA
constexpr int NT = NW * 32;
constexpr int HU = 8;         // query heads of a unit
constexpr int kCtasPerSm = 2;
constexpr int kMinTiles = 8;  // fewest tiles of a CTA's run while other CTAs idle

template <int D>
struct DecodeCfg {
  static constexpr int ST = 384 / D;              // ring slots of a warp: 24 KB in flight
  static constexpr int HALF = 2 * TK * 128;       // bytes of one box: 64 dims of K and of V rows
  static constexpr int STAGE = HALF * (D / 64);
};

template <int D>
struct DecodeSmem {
  alignas(1024) uint8_t ring[NW][DecodeCfg<D>::ST][DecodeCfg<D>::STAGE];
  alignas(16) float o[NW - 1][HU][D];
  float m[NW][HU], l[NW][HU];
  uint64_t full[NW][DecodeCfg<D>::ST];
  long long start[2];                             // first sequence of the run, tiles before it
};

// A unit that spans CTAs: its first CTA is the record's own, `last` its last one.
struct JoinRecord {
  int b, hu, last;
};

struct DecodeParams {
  CUtensorMap map;              // (D, page_rows, nkv, 2, num_pages), box (64, TK, 1, 2, 1)
  View cache;
  const uint16_t *q;            // [B][nq][D], strides q_seq, q_head
  uint16_t *out;                // [B][nq][D] contiguous
  long long q_seq, q_head;
  const int32_t *lens;          // [B]
  int batch, nq, group, units_per_kv;
  int max_len;                  // rows a sequence may have (host bound)
  float scale2;                 // scale * log2 e
  float *part_o;                // [grid][2][HU][D]
  float *part_ml;               // [grid][2][HU][2]
  JoinRecord *rec;              // [grid]
  float *logits;                // [B][nq][logit_row] scores in log2 units, or null
  float *lse;                   // [B][nq] log2 of the sum, with logits
  long long logit_row;          // max_len rounded up to whole tiles
};

__device__ __forceinline__ void tma_load_5d(void *dst, const void *tmap, int c0, int c1, int c2, int c3, int c4,
                                            uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

template <class T>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<BF16>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9},"
               " {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<F16>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9},"
               " {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Rows of sequence b that are attended: lens[b] within what the table and the caller's bound hold.
__device__ __forceinline__ int seq_rows(const DecodeParams &p, int b) {
  const int n = __ldg(p.lens + b);
  return n < 0 ? 0 : n < p.max_len ? n : p.max_len;
}
__device__ __forceinline__ int seq_tiles(const DecodeParams &p, int b) { return (seq_rows(p, b) + TK - 1) / TK; }

// A place on the line of tiles: tile `tile` of `tiles` of unit hu of sequence b (n rows).
struct Place {
  int b, hu, tile, tiles, n;
};

// Moves to the unit after the current one, past sequences without rows; false behind the last.
__device__ __forceinline__ bool next_unit(const DecodeParams &p, Place &c, int units) {
  c.tile = 0;
  if (++c.hu < units) return true;
  c.hu = 0;
  while (++c.b < p.batch) {
    c.n = seq_rows(p, c.b);
    c.tiles = (c.n + TK - 1) / TK;
    if (c.tiles > 0) return true;
  }
  return false;
}

template <class T, int D, bool kLogits>
__global__ void __launch_bounds__(NT, kCtasPerSm) paged_decode_kernel(const __grid_constant__ DecodeParams p) {
  using Cfg = DecodeCfg<D>;
  constexpr int ST = Cfg::ST;
  extern __shared__ uint8_t smem_raw[];
  DecodeSmem<D> &sm = *reinterpret_cast<DecodeSmem<D> *>(
      smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023));
  __shared__ long long warp_sum[NW];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int units = p.cache.nkv * p.units_per_kv;

  if (lane == 0) {
    for (int i = 0; i < ST; ++i) mbar_init(&sm.full[warp][i], 1);
    fence_mbar_init();
    if (warp == 0) prefetch_tmap(&p.map);
  }
  pdl_launch_dependents();
  pdl_wait();

  // ---- this CTA's run of the line: every thread sums the tiles of a block of sequences
  const int per = (p.batch + NT - 1) / NT;
  const int b_lo = min(tid * per, p.batch), b_hi = min(b_lo + per, p.batch);
  long long mine = 0;
  for (int b = b_lo; b < b_hi; ++b) {
    mine += seq_tiles(p, b);
    if (blockIdx.x == 0 && (p.lens[b] < 0 || p.lens[b] > p.max_len)) atomicExch(&g_device_status, RIB_ECAPACITY);
  }
  long long inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long up = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += up;
  }
  if (lane == 31) warp_sum[warp] = inc;
  __syncthreads();
  long long before = inc - mine, all = 0;
  for (int w = 0; w < NW; ++w) {
    if (w < warp) before += warp_sum[w];
    all += warp_sum[w];
  }
  all *= units;
  // few tiles: fewer CTAs, each with kMinTiles at least
  const long long grid = min(static_cast<long long>(gridDim.x), (all + kMinTiles - 1) / kMinTiles);
  const int cta = blockIdx.x;
  if (cta < grid) {
    const long long s0 = cta * all / grid;
    if (mine > 0 && before * units <= s0 && s0 < (before + mine) * units) {
      long long at = before;
      int b = b_lo;
      for (;; ++b) {
        const int tb = seq_tiles(p, b);
        if (s0 < (at + tb) * units) break;
        at += tb;
      }
      sm.start[0] = b;
      sm.start[1] = at * units;
    }
  }
  __syncthreads();
  // sequences without rows get zeros (and no tiles): spread over the grid
  for (int b = cta; b < p.batch; b += gridDim.x) {
    if (seq_rows(p, b) > 0) continue;
    for (int i = tid; i < p.nq * (D / 2); i += NT)
      reinterpret_cast<uint32_t *>(p.out + static_cast<size_t>(b) * p.nq * D)[i] = 0;
  }
  if (cta >= grid) {
    if (tid == 0 && cta < gridDim.x) p.rec[cta].last = -1;
    return;
  }
  const long long s0 = cta * all / grid, s1 = (cta + 1) * all / grid;
  Place c;
  c.b = static_cast<int>(sm.start[0]);
  c.n = seq_rows(p, c.b);
  c.tiles = (c.n + TK - 1) / TK;
  {
    const long long in_seq = s0 - sm.start[1];
    c.hu = static_cast<int>(in_seq / c.tiles);
    c.tile = static_cast<int>(in_seq % c.tiles);
  }
  const int run = static_cast<int>(s1 - s0);

  // ---- producer side of the warp: lane 0 copies tile after tile of this warp
  Place pc = c;
  int issued = 0, pf = warp;  // tiles issued; run index of the next one
  int page_next = -1;
  // moves pc on by `by` tiles, then reads the next tile's page number
  auto seek = [&](int by) {
    if (pf >= run) return;
    pc.tile += by;
    while (pc.tile >= pc.tiles) {
      const int over = pc.tile - pc.tiles;
      if (!next_unit(p, pc, units)) return;  // cannot happen while pf < run
      pc.tile = over;
    }
    const int i = pc.tile * TK / p.cache.page_rows;
    page_next = i < p.cache.width ? __ldg(p.cache.table + pc.b * p.cache.table_stride + i) : -1;
  };
  auto issue = [&]() {
    if (pf >= run) return;
    const int slot = issued % ST;
    if (page_next < 0 || page_next >= p.cache.num_pages) {
      atomicExch(&g_device_status, RIB_EINVAL);
      page_next = p.cache.num_pages;  // outside the map: the box reads as zeros
    }
    mbar_arrive_expect_tx(&sm.full[warp][slot], Cfg::STAGE);
#pragma unroll
    for (int hf = 0; hf < D / 64; ++hf)
      tma_load_5d(sm.ring[warp][slot] + hf * Cfg::HALF, &p.map, 64 * hf, pc.tile * TK % p.cache.page_rows,
                  pc.hu / p.units_per_kv, 0, page_next, &sm.full[warp][slot]);
    ++issued;
    pf += NW;
    seek(NW);
  };
  if (lane == 0) {
    seek(warp);
#pragma unroll 1
    for (int i = 0; i < ST; ++i) issue();
  }
  __syncwarp();

  const int g = lane >> 2, t4 = lane & 3;
  int it = 0;            // tiles this warp has consumed
  bool dead = false;     // a copy never came: nothing more is read or issued
  for (int f = 0; f < run;) {
    const int seg = min(c.tiles - c.tile, run - f);
    const int kvh = c.hu / p.units_per_kv, g0 = (c.hu % p.units_per_kv) * HU;
    const int heads = min(HU, p.group - g0), h0 = kvh * p.group + g0;
    // A fragments of q: lane row g is head h0 + g, rows 8-15 are zero
    uint32_t qa[D / 16][2];
    {
      const uint16_t *qr = p.q + c.b * p.q_seq + (h0 + g) * p.q_head + 2 * t4;
#pragma unroll
      for (int s = 0; s < D / 16; ++s) {
        qa[s][0] = g < heads ? __ldg(reinterpret_cast<const uint32_t *>(qr + 16 * s)) : 0u;
        qa[s][1] = g < heads ? __ldg(reinterpret_cast<const uint32_t *>(qr + 16 * s + 8)) : 0u;
      }
    }
    float m = -INFINITY, l = 0.f;
    float o[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = 0.f;

    for (int x = f + ((warp - f) & (NW - 1)); x < f + seg; x += NW) {
      const int k0 = (c.tile + x - f) * TK, rows = min(TK, c.n - k0);
      const int slot = it % ST;
      if (!dead && !mbar_wait(&sm.full[warp][slot], (it / ST) & 1)) dead = true;
      dead = __any_sync(0xffffffffu, dead);
      ++it;
      if (dead) continue;
      const uint32_t base = smem_u32(sm.ring[warp][slot]);
      if (rows < TK) {  // rows behind the last one may hold anything: their weight is 0, and 0 * NaN is NaN
        for (int i = lane; i < (TK - rows) * (D / 8); i += 32) {
          const int r = rows + i / (D / 8), ch = i % (D / 8);
          *reinterpret_cast<uint4 *>(sm.ring[warp][slot] + (ch >> 3) * Cfg::HALF + (TK + r) * 128 + (ch & 7) * 16) =
              make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_shared();  // the slot's next copy comes after these writes
        __syncwarp();
      }
      // ---- scores of 16 rows: two n-tiles of 8 rows, each as two chains over the dims
      float s[2][4];
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
        float s_odd[4] = {0.f, 0.f, 0.f, 0.f};
        s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
        const int r = nt * 8 + (lane & 7);
#pragma unroll
        for (int ch = 0; ch < D / 8; ch += 4) {
          const int cc = ch + (lane >> 3);
          uint32_t kb[4];
          ldsm4(base + (cc >> 3) * Cfg::HALF + r * 128 + (((cc & 7) ^ (r & 7)) << 4), kb);
          mma16816<T>(s[nt], qa[ch / 2][0], 0u, qa[ch / 2][1], 0u, kb[0], kb[1]);
          mma16816<T>(s_odd, qa[ch / 2 + 1][0], 0u, qa[ch / 2 + 1][1], 0u, kb[2], kb[3]);
        }
        s[nt][0] += s_odd[0];
        s[nt][1] += s_odd[1];
      }
      // ---- softmax in log2 units; lane holds rows 2 t4, 2 t4 + 1 of both n-tiles for head g
      float sc[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = (e >> 1) * 8 + 2 * t4 + (e & 1);
        sc[e] = r < rows ? s[e >> 1][e & 1] * p.scale2 : -INFINITY;
      }
      if (kLogits && g < heads) {
        float *lg = p.logits + (static_cast<size_t>(c.b) * p.nq + h0 + g) * p.logit_row + k0 + 2 * t4;
        *reinterpret_cast<float2 *>(lg) = make_float2(sc[0], sc[1]);
        *reinterpret_cast<float2 *>(lg + 8) = make_float2(sc[2], sc[3]);
      }
      float mt = fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3]));
      mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 1));
      mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 2));
      const float mn = fmaxf(m, mt);
      const float mz = mn == -INFINITY ? 0.f : mn;  // every score -inf so far: weights 0, not exp(inf - inf)
      if (__any_sync(0xffffffffu, mn != m)) {
        const float al = fast_exp2(m - mz);
        l *= al;
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[i][e] *= al;
        m = mn;
      }
      float pr[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) pr[e] = fast_exp2(sc[e] - mz);
      l += (pr[0] + pr[1]) + (pr[2] + pr[3]);
      // A fragments of P: rows 0-7 the rounded weights, rows 8-15 what the rounding left
      const uint32_t a0 = T::pack(pr[0], pr[1]), a2 = T::pack(pr[2], pr[3]);
      const float2 f0 = T::unpack(a0), f2 = T::unpack(a2);
      const uint32_t a1 = T::pack(pr[0] - f0.x, pr[1] - f0.y), a3 = T::pack(pr[2] - f2.x, pr[3] - f2.y);
#pragma unroll
      for (int ch = 0; ch < D / 8; ch += 2) {
        const int r = lane & 15, cc = ch + (lane >> 4);
        uint32_t vb[4];
        ldsm4_t(base + (cc >> 3) * Cfg::HALF + (TK + r) * 128 + (((cc & 7) ^ (r & 7)) << 4), vb);
        mma16816<T>(o[ch], a0, a1, a2, a3, vb[0], vb[1]);
        mma16816<T>(o[ch + 1], a0, a1, a2, a3, vb[2], vb[3]);
      }
      __syncwarp();  // every lane has read the slot
      if (lane == 0) issue();
    }

    // ---- the warps' results of this unit: scaled to a common maximum, summed in warp order
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    if (t4 == 0) sm.m[warp][g] = m;
    __syncthreads();
    float M = sm.m[0][g];
#pragma unroll
    for (int w = 1; w < NW; ++w) M = fmaxf(M, sm.m[w][g]);
    const float al = M == -INFINITY ? 0.f : fast_exp2(m - M);
    if (t4 == 0) sm.l[warp][g] = l * al;
#pragma unroll
    for (int i = 0; i < D / 8; ++i) {
      o[i][0] = (o[i][0] + o[i][2]) * al;
      o[i][1] = (o[i][1] + o[i][3]) * al;
      if (warp > 0) *reinterpret_cast<float2 *>(&sm.o[warp - 1][g][8 * i + 2 * t4]) = make_float2(o[i][0], o[i][1]);
    }
    __syncthreads();
    if (warp == 0) {
      float L = sm.l[0][g];
#pragma unroll
      for (int w = 1; w < NW; ++w) L += sm.l[w][g];
      const bool whole = c.tile == 0 && seg == c.tiles;
      const int part = c.tile > 0 ? 0 : 1;
      const float inv = whole ? (L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L)) : 1.f;  // a NaN sum stays NaN
      float *po = p.part_o + (static_cast<size_t>(cta) * 2 + part) * HU * D + g * D;
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        float2 v = make_float2(o[i][0], o[i][1]);
#pragma unroll
        for (int w = 0; w < NW - 1; ++w) {
          const float2 u = *reinterpret_cast<const float2 *>(&sm.o[w][g][8 * i + 2 * t4]);
          v.x += u.x;
          v.y += u.y;
        }
        if (g < heads) {
          if (whole)
            *reinterpret_cast<uint32_t *>(p.out + (static_cast<size_t>(c.b) * p.nq + h0 + g) * D + 8 * i + 2 * t4) =
                T::pack(v.x * inv, v.y * inv);
          else
            *reinterpret_cast<float2 *>(po + 8 * i + 2 * t4) = v;
        }
      }
      if (t4 == 0 && g < heads) {
        if (!whole) {
          float *ml = p.part_ml + ((static_cast<size_t>(cta) * 2 + part) * HU + g) * 2;
          ml[0] = M;
          ml[1] = L;
        } else if (kLogits) {
          p.lse[static_cast<size_t>(c.b) * p.nq + h0 + g] = L == 0.f ? INFINITY : M + log2f(L);
        }
      }
      if (lane == 0 && f + seg == run) {  // the run's last unit: does it begin here and end elsewhere?
        JoinRecord r = {c.b, c.hu, -1};
        if (c.tile == 0 && seg < c.tiles) {
          const long long end = s0 + f + c.tiles;  // one behind the unit's last tile
          r.last = static_cast<int>((end * grid - 1) / all);
        }
        p.rec[cta] = r;
      }
    }
    f += seg;
    if (f < run) next_unit(p, c, units);
  }
  if (dead) {  // copies still under way must land before the CTA's shared memory is given up
    const int n_issued = __shfl_sync(0xffffffffu, issued, 0);
    for (int i = max(0, n_issued - ST); i < n_issued; ++i) mbar_wait(&sm.full[warp][i % ST], (i / ST) & 1);
  }
}

// Joins the partials of a unit that spans CTAs, in run order: one CTA per CTA of the split launch.
template <class T, int D>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ DecodeParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const JoinRecord r = p.rec[blockIdx.x];
  if (r.last < 0) return;
  const int first = blockIdx.x, kvh = r.hu / p.units_per_kv, g0 = (r.hu % p.units_per_kv) * HU;
  const int heads = min(HU, p.group - g0), h0 = kvh * p.group + g0;
  for (int i = threadIdx.x; i < heads * (D / 2); i += blockDim.x) {
    const int g = i / (D / 2), d = i % (D / 2) * 2;
    // the first CTA's second partial, then the first partial of those behind it
    auto slot = [&](int c) { return static_cast<size_t>(c) * 2 + (c == first ? 1 : 0); };
    float M = -INFINITY;
    for (int c = first; c <= r.last; ++c) M = fmaxf(M, p.part_ml[(slot(c) * HU + g) * 2]);
    float L = 0.f;
    float2 o = make_float2(0.f, 0.f);
    for (int c = first; c <= r.last; ++c) {
      const float2 ml = *reinterpret_cast<const float2 *>(p.part_ml + (slot(c) * HU + g) * 2);
      const float2 v = *reinterpret_cast<const float2 *>(p.part_o + (slot(c) * HU + g) * D + d);
      const float al = M == -INFINITY ? 0.f : fast_exp2(ml.x - M);
      L = fmaf(ml.y, al, L);
      o.x = fmaf(v.x, al, o.x);
      o.y = fmaf(v.y, al, o.y);
    }
    const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);
    const size_t head = static_cast<size_t>(r.b) * p.nq + h0 + g;
    *reinterpret_cast<uint32_t *>(p.out + head * D + d) = T::pack(o.x * inv, o.y * inv);
    if (p.lse && d == 0) p.lse[head] = L == 0.f ? INFINITY : M + log2f(L);
  }
}

// scores_out[b][kvh][n] = scores[b][kvh][n] + sum over the KV head's query heads of p_hn, n < lens[b].
struct WeightParams {
  const float *logits, *lse, *scores;
  float *scores_out;
  const int32_t *lens;
  long long logit_row, in_seq, in_head, out_seq, out_head;  // strides, elements
  int nq, group, max_len;
};
__global__ void __launch_bounds__(256) row_weight_kernel(const __grid_constant__ WeightParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int h = blockIdx.y, b = blockIdx.z, n = min(p.lens[b], p.max_len);
  for (int k = blockIdx.x * 1024 + threadIdx.x; k < min(n, (static_cast<int>(blockIdx.x) + 1) * 1024); k += 256) {
    float w = 0.f;
    for (int g = 0; g < p.group; ++g) {
      const size_t head = static_cast<size_t>(b) * p.nq + h * p.group + g;
      w += fast_exp2(p.logits[head * p.logit_row + k] - p.lse[head]);
    }
    p.scores_out[b * p.out_seq + h * p.out_head + k] = p.scores[b * p.in_seq + h * p.in_head + k] + w;
  }
}

}  // namespace paged
}  // namespace rib
