// Attention of one new token per sequence over a paged cache, split over the rows and joined.
//
//   o_h = sum_n p_hn v_n,   p_hn = exp(scale q_h.k_n) / sum_m exp(scale q_h.k_m),   n < lens[b],
// with any number of query heads per KV head, head dims 64 and 128, BF16 or FP16.  Optionally the
// weight that each row of each KV head received, w[b][kvh][n] = sum over the head's query heads of
// p_hn, is added to a score per row (what an eviction goes by).
//
// Work split: the unit is (sequence, KV head, HU = 8 or 16 query heads).  The tiles of TK rows of all units lie
// on one line, unit after unit, and every CTA of one wave takes an equal run of them, found from the
// lengths on the device: ragged batches and single long sequences fill the GPU alike, and the host
// never needs the lengths.  A CTA writes the units that lie wholly in its run, and one partial
// (m, l, o) for the unit its run begins within and one for the unit it ends within; join_kernel sums
// those in run order.  (Few tiles: pieces of units instead of runs; short units: whole, with no join.)
// Nothing in the workspace has to be cleared, and no order depends on timing.
//
// In a CTA each of NW warps takes every NW-th tile and feeds itself: lane 0 copies its next tiles into
// a ring of ST slots of the warp's own by TMA (one 5-D box per 64 dims: 16 rows of K and of V of one
// page), so warps never wait for each other within a unit.  Scores and P.V run on mma.m16n8k16 with
// the heads as the 16 rows.  A decode step reads 4 D bytes per row for 4 D flops per query head, so
// memory bounds it up to 16 heads per KV head (8 heads: 52 TFLOP/s at the full memory rate), and
// a tcgen05 tile (128 rows at least, accumulators in TMEM) would add a round trip through TMEM for rows
// that stay empty.  Beyond 16 heads the rows are read once for every 16 (64 x 8-9k rows: 16 heads over one
// 53 us, 32 over one 93).  With 8 heads the upper 8 rows of the A operand are free: in P.V they carry
// p - round(p), so P enters with 16 (BF16) or 22 (FP16) bits.  That rounding is 2^-9 of the output's own; a
// third part of P took 3 to 8 % longer in short calls and with 16 heads, and spilled registers.  FP16 weights
// are lifted by 2^14 (as is their sum; in the exponent, which costs them 2^-21), out of the type's subnormal
// range: many small weights behind one large one add up.  With more than 8 heads per KV head all 16 rows are
// heads, so the rows are still read once, and the rounding's part is a second mma.  Scores, maxima, sums of
// weights and sums over P.V are FP32.
//
// Measured on B200 (one launch pair, state larger than L2): 64 sequences of 30-33k rows, 8 KV heads of
// 64 dims, 600-640 us (6.4-6.9 TB/s); 32 x 8191 rows, 64 heads over 8, FP16, 165-169 us (6.4-6.5 TB/s,
// DRAM reads 1.000 of the rows' bytes); 64 x 512-4096 rows with row weights 108-111 us (of them 13-16 us for
// join and weights); 1 x 32769 rows 30 us, of which the copies take 20.
#pragma once

#include <cuda.h>

#include "paged_cache.cuh"

namespace rib {
namespace paged {

constexpr int TK = 16;        // rows of a tile: one TMA box, one page at most
constexpr int NW = 4;         // warps of a CTA
constexpr int NT = NW * 32;
constexpr int kMaxUnitHeads = 16;  // query heads of a unit at most
// Tiles of a piece where CTAs idle: two for each warp (8 x 512 rows 9.2 us, with 4 tiles 9.9; 1 x 513 rows
// 7.3, with 4 tiles 7.0, with 16 10.1).
constexpr int kMinTiles = 8;
// Where no sequence can have more rows than this, units stay whole and nothing is launched to join them
// (8 x 256 rows: 7.3 us, split and joined 8.4; 64 x 100-200 rows: 13.9, 17.4.  With 512 rows it depends
// on the batch: 64 sequences 25.4 whole, 28.6 split, 8 sequences 11.0 and 9.2).
constexpr int kWholeRows = 256;

template <int D>
struct DecodeCfg {
  // 128 KB (144 KB) of tiles under way on an SM.  More is slower: with 3 slots at D = 128 the 32 x 8191
  // rows above take 182 us instead of 168, with 4 at D = 64 the large batch 662 instead of 630.
  static constexpr int CTAS = D == 128 ? 2 : 3;   // resident per SM
  static constexpr int ST = D == 128 ? 2 : 3;     // ring slots of a warp
  static constexpr int HALF = 2 * TK * 128;       // bytes of one box: 64 dims of K and of V rows
  static constexpr int STAGE = HALF * (D / 64);
};

template <int D, int HU>
struct DecodeSmem {
  alignas(1024) uint8_t ring[NW][DecodeCfg<D>::ST][DecodeCfg<D>::STAGE];
  // [warp that sums][the others][head][its share of the dims], rows padded against bank conflicts
  alignas(16) float o[NW][NW - 1][HU][D / NW + 8];
  float m[NW][HU], l[NW][HU];
  uint64_t full[NW][DecodeCfg<D>::ST];
  long long sum[2][NW];                           // tiles or pieces of each warp's sequences
  long long start_piece;                          // pieces before the run's first sequence
  int start_seq, start_rows;                      // that sequence and its rows
};

// The unit that begins in a CTA's run and ends in CTA `last`'s (-1: there is none).
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
  float *part_o;                // [grid][2][HU][D], HU the query heads of a unit (8 or 16)
  float *part_ml;               // [grid][2][HU][2]
  JoinRecord *rec;              // [grid]
  float *logits;                // [B][nq][logit_row] scores in log2 units, or null
  float2 *norm;                 // [B][nq] (maximum, 1 / sum) of units of one CTA, with logits
  int2 *span;                   // [B][units] first and last CTA of a unit that spans several, or -1
  const float *scores;          // row weights: scores_out = scores + weight, strides below
  float *scores_out;
  long long in_seq, in_head, out_seq, out_head;
  long long logit_row;          // max_len rounded up to whole tiles
  int whole;                    // no unit is split over CTAs, and nothing is left to join
};

__device__ __forceinline__ void tma_load_5d(void *dst, const void *tmap, int c0, int c1, int c2, int c3, int c4,
                                            uint64_t *bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%2, %3, %4, %5, %6}], [%7], %8;" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4), "r"(smem_u32(bar)),
      "l"(policy)
      : "memory");
}

__device__ __forceinline__ uint64_t l2_policy_evict_normal() {
  uint64_t p;
  asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(p));
  return p;
}

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

// d = A B + c.
template <class T>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1, const float (&c)[4]);
template <>
__device__ __forceinline__ void mma16816<BF16>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1, const float (&c)[4]) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9},"
               " {%10, %11, %12, %13};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
template <>
__device__ __forceinline__ void mma16816<F16>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1, const float (&c)[4]) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9},"
               " {%10, %11, %12, %13};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

// a + b, both halves in one instruction.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t &>(d))
      : "l"(reinterpret_cast<uint64_t &>(a)), "l"(reinterpret_cast<uint64_t &>(b)));
  return d;
}

// Rows of sequence b that are attended: lens[b] within what the table and the caller's bound hold.
__device__ __forceinline__ int seq_rows(const DecodeParams &p, int b) {
  const int n = p.lens[b];
  return n < 0 ? 0 : n < p.max_len ? n : p.max_len;
}

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

// Which of a lane's dims, dim + 8 i + e at bit 2 i + e for i < S, hold +infinity, -infinity and NaN among the V
// rows [row, end) of a sequence, 8 of which the warp's lanes of one dim take at a time.
struct OddDims {
  uint32_t pos, neg, nan;
};
template <class T, int S>
__device__ __noinline__ OddDims odd_dims(const View &cache, int b, int kvh, int row, int end, int dim) {
  OddDims x = {0, 0, 0};
  for (row += (threadIdx.x & 31) >> 2; row < end; row += 8) {
    const int page = page_of(cache, b, row);
    if (page < 0) continue;  // counts as zeros
    const uint16_t *v = cache.pages + page * cache.s_page + cache.s_half + kvh * cache.s_head +
                        (row % cache.page_rows) * cache.s_row + dim;
#pragma unroll
    for (int i = 0; i < S; ++i) {
      const uint32_t w = *reinterpret_cast<const uint32_t *>(v + 8 * i);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t u = w >> (16 * e) & 0xffffu, bit = 1u << (2 * i + e);
        if ((u & 0x7fffu) > T::kInf) x.nan |= bit;
        if (u == T::kInf) x.pos |= bit;
        if (u == (T::kInf | 0x8000u)) x.neg |= bit;
      }
    }
  }
#pragma unroll
  for (int o = 4; o <= 16; o <<= 1) {
    x.pos |= __shfl_xor_sync(0xffffffffu, x.pos, o);
    x.neg |= __shfl_xor_sync(0xffffffffu, x.neg, o);
    x.nan |= __shfl_xor_sync(0xffffffffu, x.nan, o);
  }
  return x;
}
// The sum over such a dim, every weight counting as positive; `sum` where there are none.
__device__ __forceinline__ float odd_sum(const OddDims &x, uint32_t bit, float sum) {
  if (!((x.pos | x.neg | x.nan) & bit)) return sum;
  return (x.nan | (x.pos & x.neg)) & bit ? NAN : x.pos & bit ? INFINITY : -INFINITY;
}

// (maximum, factor) such that exp2(score - maximum) * factor is a row's weight.
template <class T>
__device__ __forceinline__ float2 weight_norm(float M, float L) {
  if (L == 0.f) return make_float2(0.f, 0.f);  // every score -inf
  return make_float2(M, static_cast<float>(1 << T::kLift) / L);
}

template <class T, int D, int HU, bool kLogits>
__global__ void __launch_bounds__(NT, DecodeCfg<D>::CTAS) paged_decode_kernel(const __grid_constant__ DecodeParams p) {
  using Cfg = DecodeCfg<D>;
  constexpr int R = HU / 8;  // heads of a lane: rows g and, with 16 heads, g + 8 of the mma tiles
  constexpr int ST = Cfg::ST;
  extern __shared__ uint8_t smem_raw[];
  DecodeSmem<D, HU> &sm = *reinterpret_cast<DecodeSmem<D, HU> *>(
      smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int units = p.cache.nkv * p.units_per_kv;

  if (lane == 0) {
    for (int i = 0; i < ST; ++i) mbar_init(&sm.full[warp][i], 1);
    fence_mbar_init();
    if (warp == 0) prefetch_tmap(&p.map);
  }
  pdl_launch_dependents();
  pdl_wait();

  // ---- this CTA's run of the line.  Every thread sums a block of sequences: their tiles, and their
  // pieces of kMinTiles tiles.
  const int per = (p.batch + NT - 1) / NT;
  const int b_lo = min(tid * per, p.batch), b_hi = min(b_lo + per, p.batch);
  int first_rows = 0;
  long long mine = 0, mine_short = 0;
  for (int b = b_lo; b < b_hi; ++b) {
    const int n = seq_rows(p, b), t = (n + TK - 1) / TK;
    if (b == b_lo) first_rows = n;
    mine += t;
    mine_short += (t + kMinTiles - 1) / kMinTiles;
    if (blockIdx.x == 0 && n != p.lens[b]) atomicExch(&g_device_status, RIB_ECAPACITY);
  }
  auto scan_warp = [&](long long v, long long *sum) {  // sum over the warp's lanes up to this one
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long up = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += up;
    }
    if (lane == 31) sum[warp] = v;
    return v;
  };
  auto scan_cta = [&](long long &v, const long long *sum) {  // adds the warps before; returns the total
    long long total = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      if (w < warp) v += sum[w];
      total += sum[w];
    }
    return total;
  };
  long long before = scan_warp(mine, sm.sum[0]) - mine, before_short = scan_warp(mine_short, sm.sum[1]) - mine_short;
  __syncthreads();
  long long all = scan_cta(before, sm.sum[0]) * units;
  const long long all_short = scan_cta(before_short, sm.sum[1]) * units;
  // Few tiles: pieces of kMinTiles tiles, one to a CTA, each within one unit, so nothing but the join
  // is left behind it (1 x 513 rows, 8 KV heads: 7.3 us, in equal runs that cross units 8.6).  Otherwise
  // (quantum 1) equal runs of tiles, which may begin and end within a unit: pieces would leave CTAs idle.
  int quantum = 1;
  if (!p.whole && all_short <= gridDim.x) {
    quantum = kMinTiles;
    mine = mine_short;
    before = before_short;
    all = all_short;
  }
  // CTA i takes `quot` pieces, the first `rest` one more.
  const int cta = blockIdx.x, grid = static_cast<int>(min(static_cast<long long>(gridDim.x), all));
  const long long quot = !grid ? 0 : all >> 31 ? all / grid : static_cast<int>(all) / grid;
  const int rest = static_cast<int>(all - quot * grid);
  const long long s0 = cta * quot + min(cta, rest);
  int run = cta < grid ? static_cast<int>(quot + (cta < rest)) : 0;
  if (run && before * units <= s0 && s0 < (before + mine) * units) {
    int b = b_lo, n = first_rows;
    while (true) {
      const int t = ((n + TK - 1) / TK + quantum - 1) / quantum;
      if (s0 < (before + t) * units) break;
      before += t;
      n = seq_rows(p, ++b);
    }
    sm.start_seq = b;
    sm.start_rows = n;
    sm.start_piece = before * units;
  }
  __syncthreads();
  if (!run && tid == 0) p.rec[cta].last = -1;
  // sequences without rows have no tiles, and get zeros
  for (int b = cta; b < p.batch; b += gridDim.x) {
    if (seq_rows(p, b) > 0) continue;
    for (int i = tid; i < p.nq * (D / 2); i += NT)
      reinterpret_cast<uint32_t *>(p.out + static_cast<size_t>(b) * p.nq * D)[i] = 0;
  }
  if (!run) return;
  Place c;
  c.b = sm.start_seq;
  c.n = sm.start_rows;
  c.tiles = (c.n + TK - 1) / TK;
  int last_cta = -1;  // with pieces: the CTA that has the last one of this one's unit
  {
    const long long in_seq = s0 - sm.start_piece;
    const int k = (c.tiles + quantum - 1) / quantum;  // pieces of the unit
    c.hu = in_seq >> 31 ? static_cast<int>(in_seq / k) : static_cast<int>(in_seq) / k;
    c.tile = static_cast<int>(in_seq - static_cast<long long>(c.hu) * k);
    if (quantum > 1) {  // piece c.tile of k nearly equal ones
      const int piece = c.tile, q = c.tiles / k, r = c.tiles % k;
      c.tile = piece * q + min(piece, r);
      run = q + (piece < r);
      last_cta = cta - piece + k - 1;
    }
  }
  if (p.whole) {  // short units are not split: the run takes those that begin in it, to their end
    int f = 0;
    if (c.tile > 0) {
      f = c.tiles - c.tile;
      if (f >= run || !next_unit(p, c, units)) {
        if (tid == 0) p.rec[cta].last = -1;
        return;
      }
    }
    int end = f;
    Place w = c;
    do {
      end += w.tiles;
    } while (end < run && next_unit(p, w, units));
    run = end - f;
  }

  // ---- producer side of the warp: tile i of the warp is the run's tile warp + i * NW
  const int count = run > warp ? (run - warp + NW - 1) / NW : 0;
  // Rows are read once: kept out of L2's way (evict first), a sustained large batch runs at a steady
  // 620 us; with the default priority it wandered between 607 and 866.  Units that share rows leave them.
  const uint64_t policy = p.units_per_kv == 1 ? l2_policy_evict_first() : l2_policy_evict_normal();
  // moves `by` tiles along the run
  auto seek = [&](Place &pl, int by) {
    pl.tile += by;
    while (pl.tile >= pl.tiles) {
      const int over = pl.tile - pl.tiles;
      if (!next_unit(p, pl, units)) return;  // never within the run
      pl.tile = over;
    }
  };
  auto page_at = [&](const Place &pl) {
    return p.cache.table[pl.b * p.cache.table_stride + pl.tile * TK / p.cache.page_rows];
  };
  auto copy = [&](const Place &pl, int page, int slot) {
    if (page < 0 || page >= p.cache.num_pages) {
      atomicExch(&g_device_status, RIB_EINVAL);
      page = p.cache.num_pages;  // outside the map: the box reads as zeros
    }
    mbar_arrive_expect_tx(&sm.full[warp][slot], Cfg::STAGE);
#pragma unroll
    for (int hf = 0; hf < D / 64; ++hf)
      tma_load_5d(sm.ring[warp][slot] + hf * Cfg::HALF, &p.map, 64 * hf, pl.tile * TK % p.cache.page_rows,
                  pl.hu / p.units_per_kv, 0, page, &sm.full[warp][slot], policy);
  };
  if (lane < min(ST, count)) {  // the first tiles, a lane each
    Place pl = c;
    seek(pl, warp + lane * NW);
    copy(pl, page_at(pl), lane);
  }
  Place pc = c;  // lane 0: the next tile to copy, its page asked for, and looked at only then
  int issued = min(ST, count), page_next = 0;
  if (lane == 0 && issued < count) {
    seek(pc, warp + issued * NW);
    page_next = page_at(pc);
  }
  auto issue = [&]() {
    copy(pc, page_next, issued % ST);
    if (++issued < count) {
      seek(pc, NW);
      page_next = page_at(pc);
    }
  };
  __syncwarp();

  const int g = lane >> 2, t4 = lane & 3;
  int it = 0;            // tiles this warp has consumed
  bool dead = false;     // a copy never came: nothing more is read or issued
  for (int f = 0; f < run;) {
    const int seg = min(c.tiles - c.tile, run - f);
    const int kvh = c.hu / p.units_per_kv, g0 = (c.hu % p.units_per_kv) * HU;
    const int heads = min(HU, p.group - g0), h0 = kvh * p.group + g0;
    // A fragments of q: rows g (and g + 8) are heads h0 + g (and h0 + g + 8), the others zero
    uint32_t qa[R][D / 16][2];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const uint16_t *qr = p.q + c.b * p.q_seq + (h0 + g + 8 * r) * p.q_head + 2 * t4;
#pragma unroll
      for (int s = 0; s < D / 16; ++s) {
        qa[r][s][0] = g + 8 * r < heads ? *reinterpret_cast<const uint32_t *>(qr + 16 * s) : 0u;
        qa[r][s][1] = g + 8 * r < heads ? *reinterpret_cast<const uint32_t *>(qr + 16 * s + 8) : 0u;
      }
    }
    float m[R], l[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      m[r] = -INFINITY;
      l[r] = 0.f;
    }
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
          const int e = ch / 2;
          mma16816<T>(s[nt], qa[0][e][0], R > 1 ? qa[R - 1][e][0] : 0u, qa[0][e][1], R > 1 ? qa[R - 1][e][1] : 0u, kb[0],
                      kb[1], s[nt]);
          mma16816<T>(s_odd, qa[0][e + 1][0], R > 1 ? qa[R - 1][e + 1][0] : 0u, qa[0][e + 1][1],
                      R > 1 ? qa[R - 1][e + 1][1] : 0u, kb[2], kb[3], s_odd);
        }
#pragma unroll
        for (int e = 0; e < 2 * R; ++e) s[nt][e] += s_odd[e];
      }
      // ---- softmax in log2 units; lane holds rows 2 t4, 2 t4 + 1 of both n-tiles for each of its heads
      float pr[R][4];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float sc[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int row = (e >> 1) * 8 + 2 * t4 + (e & 1);
          sc[e] = row < rows ? s[e >> 1][2 * r + (e & 1)] * p.scale2 : -INFINITY;
        }
        if (kLogits && g + 8 * r < heads) {
          float *lg = p.logits + (static_cast<size_t>(c.b) * p.nq + h0 + g + 8 * r) * p.logit_row + k0 + 2 * t4;
          *reinterpret_cast<float2 *>(lg) = make_float2(sc[0], sc[1]);
          *reinterpret_cast<float2 *>(lg + 8) = make_float2(sc[2], sc[3]);
        }
        float mt = fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3]));
        mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 1));
        mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 2));
        const float mn = fmaxf(m[r], mt);
        const float mz = mn == -INFINITY ? 0.f : mn;  // every score -inf so far: weights 0, not exp(inf - inf)
        if (__any_sync(0xffffffffu, mn != m[r])) {
          const float al = fast_exp2(m[r] - mz);
          l[r] *= al;
#pragma unroll
          for (int i = 0; i < D / 8; ++i)
#pragma unroll
            for (int e = 2 * r; e < (R > 1 ? 2 * r + 2 : 4); ++e) o[i][e] *= al;
          m[r] = mn;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) pr[r][e] = fast_exp2(T::kLift ? sc[e] - mz + T::kLift : sc[e] - mz);
        l[r] += (pr[r][0] + pr[r][1]) + (pr[r][2] + pr[r][3]);
      }
      // A fragments of P: the rounded weights, and what the rounding left (with 8 heads in rows 8-15)
      uint32_t hi[R][2], lo[R][2];
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          hi[r][e] = T::pack(pr[r][2 * e], pr[r][2 * e + 1]);
          const float2 f = T::unpack(hi[r][e]);
          lo[r][e] = T::pack(pr[r][2 * e] - f.x, pr[r][2 * e + 1] - f.y);
        }
#pragma unroll
      for (int ch = 0; ch < D / 8; ch += 2) {
        const int r = lane & 15, cc = ch + (lane >> 4);
        uint32_t vb[4];
        ldsm4_t(base + (cc >> 3) * Cfg::HALF + (TK + r) * 128 + (((cc & 7) ^ (r & 7)) << 4), vb);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          // A tile's products, then added to the sums with a rounding to nearest: as an accumulator of the next
          // mma a sum is cut off toward 0, and over the 16384 tiles that a warp adds of a unit of 2^20 rows it lost
          // 1.1e-4 to 2.4e-4 of the weights' sum (now 1.2e-6).  The additions cost nothing measurable.
          const float zero[4] = {0.f, 0.f, 0.f, 0.f};
          float d[4];
          if (R > 1) {
            mma16816<T>(d, lo[0][0], lo[R - 1][0], lo[0][1], lo[R - 1][1], vb[2 * e], vb[2 * e + 1], zero);
            mma16816<T>(d, hi[0][0], hi[R - 1][0], hi[0][1], hi[R - 1][1], vb[2 * e], vb[2 * e + 1], d);
          } else {
            mma16816<T>(d, hi[0][0], lo[0][0], hi[0][1], lo[0][1], vb[2 * e], vb[2 * e + 1], zero);
          }
#pragma unroll
          for (int j = 0; j < 4; j += 2) {
            const float2 u = add2(make_float2(o[ch + e][j], o[ch + e][j + 1]), make_float2(d[j], d[j + 1]));
            o[ch + e][j] = u.x, o[ch + e][j + 1] = u.y;
          }
        }
      }
      __syncwarp();  // every lane has read the slot
      if (lane == 0 && issued < count) issue();
    }

    // ---- the warps' results of this unit: scaled to a common maximum, summed in warp order
#pragma unroll
    for (int r = 0; r < R; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      if (t4 == 0) sm.m[warp][g + 8 * r] = m[r];
    }
    __syncthreads();
    // every warp sums a share of the dims: it keeps its own part of those and hands out the rest
    constexpr int S = D / 8 / NW;  // n-tiles of a share
    float2 own[R][S];
    float M[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      M[r] = sm.m[0][g + 8 * r];
#pragma unroll
      for (int w = 1; w < NW; ++w) M[r] = fmaxf(M[r], sm.m[w][g + 8 * r]);
      const float al = M[r] == -INFINITY ? 0.f : fast_exp2(m[r] - M[r]);
      if (t4 == 0) sm.l[warp][g + 8 * r] = l[r] * al;
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        const float2 v = R > 1 ? make_float2(o[i][2 * r] * al, o[i][2 * r + 1] * al)
                               : make_float2((o[i][0] + o[i][2]) * al, (o[i][1] + o[i][3]) * al);
        if (i / S == warp)
          own[r][i % S] = v;
        else
          *reinterpret_cast<float2 *>(&sm.o[i / S][warp - (warp > i / S)][g + 8 * r][i % S * 8 + 2 * t4]) = v;
      }
    }
    __syncthreads();
    {
      const bool whole = c.tile == 0 && seg == c.tiles;
      const int part = c.tile > 0 ? 0 : 1;
      const int d0 = warp * (D / NW) + 2 * t4;
      float2 sum[R][S];
      bool odd = false;
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < S; ++i) {
          float2 v = make_float2(0.f, 0.f);  // in warp order
#pragma unroll
          for (int w = 0; w < NW; ++w) {
            const float2 u = w == warp ? own[r][i]
                                       : *reinterpret_cast<const float2 *>(
                                             &sm.o[warp][w - (w > warp)][g + 8 * r][i * 8 + 2 * t4]);
            v.x += u.x;
            v.y += u.y;
          }
          sum[r][i] = v;
          odd |= !(fabsf(v.x) < INFINITY) || !(fabsf(v.y) < INFINITY);
        }
      // Infinite and NaN values: the two parts of a weight times an infinity may make NaN of what the weight itself
      // makes an infinity, so the V rows are asked which dims hold some.
      if (__any_sync(0xffffffffu, odd)) {
        const OddDims x = odd_dims<T, S>(p.cache, c.b, kvh, c.tile * TK, min(c.n, (c.tile + seg) * TK), d0);
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int i = 0; i < S; ++i) {
            sum[r][i].x = odd_sum(x, 1u << (2 * i), sum[r][i].x);
            sum[r][i].y = odd_sum(x, 2u << (2 * i), sum[r][i].y);
          }
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int hd = g + 8 * r;
        float L = sm.l[0][hd];
#pragma unroll
        for (int w = 1; w < NW; ++w) L += sm.l[w][hd];
        const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);  // a NaN sum stays NaN
        uint16_t *out = p.out + (static_cast<size_t>(c.b) * p.nq + h0 + hd) * D + d0;
        float *po = p.part_o + ((static_cast<size_t>(cta) * 2 + part) * HU + hd) * D + d0;
#pragma unroll
        for (int i = 0; i < S; ++i) {
          const float2 v = sum[r][i];
          if (hd < heads) {
            if (whole)
              *reinterpret_cast<uint32_t *>(out + 8 * i) = T::pack(v.x * inv, v.y * inv);
            else
              *reinterpret_cast<float2 *>(po + 8 * i) = v;
          }
        }
        if (warp == 0 && t4 == 0 && hd < heads) {
          if (!whole)
            *reinterpret_cast<float2 *>(p.part_ml + ((static_cast<size_t>(cta) * 2 + part) * HU + hd) * 2) =
                make_float2(M[r], L);
          else if (kLogits)
            p.norm[static_cast<size_t>(c.b) * p.nq + h0 + hd] = weight_norm<T>(M[r], L);
        }
      }
      if (tid == 0) {
        int last = -1;  // the CTA in which a unit that begins here and does not end here ends
        if (c.tile == 0 && !whole) {
          const long long x = s0 + f + c.tiles - 1, big = rest * (quot + 1);  // its last tile
          last = quantum > 1 ? last_cta : static_cast<int>(x < big ? x / (quot + 1) : rest + (x - big) / quot);
        }
        if (f + seg == run) p.rec[cta] = {c.b, c.hu, last};
        if (kLogits && c.tile == 0) p.span[static_cast<size_t>(c.b) * units + c.hu] = make_int2(cta, last);
      }
    }
    f += seg;
    if (f < run) next_unit(p, c, units);
  }
  if (dead) {  // copies still under way must land before the CTA's shared memory is given up
    const int sent = __shfl_sync(0xffffffffu, issued, 0);
    for (int i = max(0, sent - ST); i < sent; ++i) mbar_wait(&sm.full[warp][i % ST], (i / ST) & 1);
  }
}

constexpr int kJoinWarps = 8, kJoinThreads = kJoinWarps * 32;
constexpr int kNormHeads = 128;  // heads whose row weights are summed at once

// Place of CTA c's partial of a unit that begins in CTA `first`: that one's second, the others' first.
__device__ __forceinline__ size_t part_slot(int c, int first) { return static_cast<size_t>(c) * 2 + (c == first); }

// Maximum and sum of head g of a unit over its partials, by a whole warp (in every lane, in CTA order
// within a lane and by a fixed tree over the lanes).
template <int HU>
__device__ __forceinline__ float2 joined_ml(const DecodeParams &p, int first, int last, int g, int lane) {
  float M = -INFINITY, L = 0.f;
  for (int c = first + lane; c <= last; c += 32) {
    const float2 ml = *reinterpret_cast<const float2 *>(p.part_ml + (part_slot(c, first) * HU + g) * 2);
    const float mn = fmaxf(M, ml.x), mz = mn == -INFINITY ? 0.f : mn;
    L = L * fast_exp2(M - mz) + ml.y * fast_exp2(ml.x - mz);
    M = mn;
  }
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, M, o), l2 = __shfl_xor_sync(0xffffffffu, L, o);
    const float mn = fmaxf(M, m2), mz = mn == -INFINITY ? 0.f : mn;
    L = L * fast_exp2(M - mz) + l2 * fast_exp2(m2 - mz);
    M = mn;
  }
  return make_float2(M, L);
}

// Blocks below `grid`: join the unit that begins in that CTA's run and ends in another's.  The warps
// take (head, slice of the partials), so all partials are under way at once; the slices are summed in
// order.  With scores, the blocks behind add the row weights, `rows` rows of one KV head each.
template <class T, int D, int HU>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const __grid_constant__ DecodeParams p, int grid,
                                                            int row_blocks, int rows) {
  constexpr int kSums = HU > kJoinWarps ? HU : kJoinWarps;
  __shared__ float4 acc[kSums][D / 4];  // [head][slice]
  __shared__ float head_sum[HU];
  __shared__ float2 head_norm[kNormHeads];
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (static_cast<int>(blockIdx.x) < grid) {
    const JoinRecord r = p.rec[blockIdx.x];
    if (r.last < 0) return;
    const int first = blockIdx.x, kvh = r.hu / p.units_per_kv, g0 = (r.hu % p.units_per_kv) * HU;
    const int heads = min(HU, p.group - g0), h0 = kvh * p.group + g0;
    const int slices = heads < kJoinWarps ? kJoinWarps / heads : 1, slice = warp % slices;
    constexpr int V = D / 4, R = 32 / V;  // lanes of a row, rows of a load
    constexpr int N = D == 128 ? 6 : 4;   // loads under way at once
    const int v = lane % V, step = slices * R;
    for (int g = warp / slices; g < heads; g += kJoinWarps / slices) {
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      float2 all = make_float2(0.f, 0.f);
      for (int c0 = first + slice * R + lane / V; c0 - lane / V <= r.last; c0 += N * step) {
        float4 u[N];
        float m[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int c = c0 + i * step;
          if (c > r.last) continue;
          const size_t s = part_slot(c, first) * HU + g;
          u[i] = *reinterpret_cast<const float4 *>(p.part_o + s * D + 4 * v);
          m[i] = p.part_ml[2 * s];
        }
        if (c0 - lane / V == first + slice * R) all = joined_ml<HU>(p, first, r.last, g, lane);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          if (c0 + i * step > r.last) continue;
          const float al = all.x == -INFINITY ? 0.f : fast_exp2(m[i] - all.x);
          if (al != 0.f) {
            o = make_float4(fmaf(u[i].x, al, o.x), fmaf(u[i].y, al, o.y), fmaf(u[i].z, al, o.z), fmaf(u[i].w, al, o.w));
          } else {  // infinite and NaN values show whatever their weight
            const float *from = &u[i].x;
            float *to = &o.x;
#pragma unroll
            for (int e = 0; e < 4; ++e) to[e] += fabsf(from[e]) < INFINITY ? 0.f : from[e];
          }
        }
      }
      if (R == 2) {
        o.x += __shfl_xor_sync(0xffffffffu, o.x, 16);
        o.y += __shfl_xor_sync(0xffffffffu, o.y, 16);
        o.z += __shfl_xor_sync(0xffffffffu, o.z, 16);
        o.w += __shfl_xor_sync(0xffffffffu, o.w, 16);
      }
      if (lane < V) acc[g * slices + slice][v] = o;
      if (lane == 0 && slice == 0) head_sum[g] = all.y;
    }
    __syncthreads();
    for (int i = tid; i < heads * V; i += kJoinThreads) {
      const int hg = i / V, d = i % V;
      float4 o = acc[hg * slices][d];
      for (int k = 1; k < slices; ++k) {
        const float4 u = acc[hg * slices + k][d];
        o = make_float4(o.x + u.x, o.y + u.y, o.z + u.z, o.w + u.w);
      }
      const float L = head_sum[hg], inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);
      const size_t head = static_cast<size_t>(r.b) * p.nq + h0 + hg;
      *reinterpret_cast<uint2 *>(p.out + head * D + 4 * d) =
          make_uint2(T::pack(o.x * inv, o.y * inv), T::pack(o.z * inv, o.w * inv));
    }
    return;
  }
  // ---- row weights: scores_out[b][h][n] = scores[b][h][n] + sum over the head's queries of p_hn
  const int id = blockIdx.x - grid, k0 = id % row_blocks * rows;
  const int bh = id / row_blocks, h = bh % p.cache.nkv, b = bh / p.cache.nkv;
  const int n = min(rows, seq_rows(p, b) - k0);
  if (n <= 0) return;
  float *out = p.scores_out + b * p.out_seq + h * p.out_head + k0;
  const size_t first_head = static_cast<size_t>(b) * p.nq + h * p.group;
  // all heads' weights of a row are summed before the score is touched (beyond kNormHeads heads, in parts)
  for (int part = 0; part < p.group; part += kNormHeads) {
    const int heads = min(kNormHeads, p.group - part);
    for (int g = warp; g < heads; g += kJoinWarps) {
      const int u = (part + g) / HU;
      const int2 span = p.span[static_cast<size_t>(bh) * p.units_per_kv + u];
      float2 norm;
      if (span.y < 0) {
        norm = p.norm[first_head + part + g];
      } else {
        const float2 ml = joined_ml<HU>(p, span.x, span.y, part + g - u * HU, lane);
        norm = weight_norm<T>(ml.x, ml.y);
      }
      if (lane == 0) head_norm[g] = norm;
    }
    __syncthreads();
    const float *in = part ? out : p.scores + b * p.in_seq + h * p.in_head + k0;
    const float *logits = p.logits + (first_head + part) * p.logit_row + k0;
    constexpr int R = 4, H = 8;  // rows and heads of a thread under way at once
    for (int k = tid; k < n; k += R * kJoinThreads) {
      float w[R], sum[R];
#pragma unroll
      for (int i = 0; i < R; ++i) {
        w[i] = k + i * kJoinThreads < n ? in[k + i * kJoinThreads] : 0.f;
        sum[i] = 0.f;
      }
      for (int g0 = 0; g0 < heads; g0 += H) {
        float x[H][R];
#pragma unroll
        for (int g = 0; g < H; ++g)
          if (g0 + g < heads) {
            const float *lg = logits + (g0 + g) * p.logit_row + k;
#pragma unroll
            for (int i = 0; i < R; ++i) x[g][i] = k + i * kJoinThreads < n ? lg[i * kJoinThreads] : -INFINITY;
          }
#pragma unroll
        for (int g = 0; g < H; ++g)
          if (g0 + g < heads) {
            const float2 norm = head_norm[g0 + g];
#pragma unroll
            for (int i = 0; i < R; ++i) sum[i] = fmaf(fast_exp2(x[g][i] - norm.x), norm.y, sum[i]);
          }
      }
#pragma unroll
      for (int i = 0; i < R; ++i)
        if (k + i * kJoinThreads < n) out[k + i * kJoinThreads] = w[i] + sum[i];
    }
    __syncthreads();
  }
}

}  // namespace paged
}  // namespace rib
