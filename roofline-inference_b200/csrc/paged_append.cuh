// Rotary positions, and the append of rotated keys and values to a paged cache.
//
// Pair i < r/2 of a head's first r = 2 * pairs dims turns by pos * f_i:
//   (a, b) -> g (a cos - b sin, a sin + b cos),
// with (a, b) = dims (i, i + r/2) (half layout) or (2i, 2i + 1) (interleaved); dims past r pass
// unchanged.  f_i and g carry the scaling for long contexts (a host-made table).  q and k heads may be
// RMS-normalised over all D dims first: x w / sqrt(mean(x^2) + eps).  All in FP32, rounded once.
// The angle is formed in turns, pos * (f_i / 2 pi), in FP64 and reduced to half a turn there: in FP32 a
// position past 2^17 would leave it fewer than 7 bits after the point.
//
// Bound by memory: 4 bytes moved for each value, read once and written once, and about 3 flops.
//
// Work split: D/16 lanes hold one head, 16 dims each as two 16-byte vectors, so both members of a pair
// sit in one lane and no lane exchanges dims with another (the norm's sum of squares is the only
// shuffle).  A lane group keeps one token's cosines for all the heads it takes.  A row is short, so what
// limits the kernel is how many are under way: each lane copies its next heads into a ring of its own
// (cp.async), 5 ahead.  Measured on B200: 32768 tokens of 16 + 16 heads of 128 dims, normalised, in
// 91-95 us (5.7-5.9 TB/s, 0.86-0.89 of the copy rate; loads into registers 119 us); 4093 tokens of 32 + 16 heads,
// interleaved over 64 of 128 dims, 20-21 us (4.9 TB/s; with two chunks of neighbouring dims to a lane,
// half a sector an access, 34 us); one token 2.9 us on the device.
#pragma once

#include "paged_cache.cuh"

namespace rib {
namespace paged {

struct AppendParams {
  View cache;                                        // not read when nkv == 0 (rotation alone)
  const uint16_t *q, *k, *v;
  uint16_t *q_out;
  long long q_token, q_head, k_token, k_head, v_token, v_head, o_token, o_head;  // strides, elements
  const int32_t *pos, *row, *seq;                    // [tokens]; seq null: token t belongs to sequence t
  const double *turns;                               // [pairs] turns per position, f_i / 2 pi
  const uint16_t *qw, *kw;                           // [D] norm weights, or null
  float gain, eps, inv_dim;                          // inv_dim: 1 / dim
  int tokens, nq, nkv, dim, pairs, interleaved;
  int groups;                                        // lane groups of a token
};

// (cosine, sine) of `turns` turns (FP64) times gain.
__device__ __forceinline__ float2 turn_sincos(double turns, float gain) {
  const float part = static_cast<float>(turns - rint(turns));  // [-1/2, 1/2]
  float s, c;
  sincospif(2.0f * part, &s, &c);
  return make_float2(c * gain, s * gain);
}

// A lane's 16 dims <-> the two sides of its 8 pairs, in FP32.
template <class T>
__device__ __forceinline__ void split(uint4 a, uint4 b, int interleaved, float (&xa)[8], float (&xb)[8]) {
  const uint32_t ra[4] = {a.x, a.y, a.z, a.w}, rb[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 u = T::unpack(ra[i]), v = T::unpack(rb[i]);
    if (interleaved) {
      xa[i] = u.x, xb[i] = u.y, xa[4 + i] = v.x, xb[4 + i] = v.y;
    } else {
      xa[2 * i] = u.x, xa[2 * i + 1] = u.y, xb[2 * i] = v.x, xb[2 * i + 1] = v.y;
    }
  }
}
template <class T>
__device__ __forceinline__ void merge(const float (&xa)[8], const float (&xb)[8], int interleaved, uint4 &a, uint4 &b) {
  if (interleaved) {
    a = make_uint4(T::pack(xa[0], xb[0]), T::pack(xa[1], xb[1]), T::pack(xa[2], xb[2]), T::pack(xa[3], xb[3]));
    b = make_uint4(T::pack(xa[4], xb[4]), T::pack(xa[5], xb[5]), T::pack(xa[6], xb[6]), T::pack(xa[7], xb[7]));
  } else {
    a = make_uint4(T::pack(xa[0], xa[1]), T::pack(xa[2], xa[3]), T::pack(xa[4], xa[5]), T::pack(xa[6], xa[7]));
    b = make_uint4(T::pack(xb[0], xb[1]), T::pack(xb[2], xb[3]), T::pack(xb[4], xb[5]), T::pack(xb[6], xb[7]));
  }
}

// Two FP32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<uint64_t &>(d))
      : "l"(reinterpret_cast<uint64_t &>(a)), "l"(reinterpret_cast<uint64_t &>(b)),
        "l"(reinterpret_cast<uint64_t &>(c)));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t &>(d))
      : "l"(reinterpret_cast<uint64_t &>(a)), "l"(reinterpret_cast<uint64_t &>(b)));
  return d;
}

// 32768 tokens: 92.0 us with 5 stages, 91.2 with 6, 90.6 with 9 (which costs short calls); 94.1 with CTAs
// of 128 threads.
constexpr int kAppendThreads = 64;
constexpr int kAppendCtas = 8;      // resident per SM
constexpr int kAppendStages = 6;    // heads of a lane that are under way

__device__ __forceinline__ void cp_async16(void *dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A lane's share of one head: two chunks of 8 dims, which neighbouring lanes continue, so that a load
// or store of a lane group covers whole 32-byte sectors.  Half layout: the two sides of 8 pairs.
// Interleaved: 4 pairs in each chunk.  Past the rotated part: dims that stay put.
struct LaneDims {
  int d0, d1;            // first dim of each chunk
  int p0, p1;            // first pair of the lane's first and last 4 pairs
  bool turn0, turn1;     // those pairs rotate
  bool used;             // the lane holds dims at all
};

// A lane's walk over its group's heads (q, then k, then v) of one token.  It copies its chunks of the
// heads ahead into a ring of its own in shared memory, which no other thread touches.
struct HeadWalk {
  uint4 (*ring)[2][kAppendThreads];
  const uint16_t *q, *k, *v;  // the token's head 0
  int h, ahead, slot, fetch_slot;

  __device__ __forceinline__ void fetch(const AppendParams &p, const LaneDims &l) {
    if (ahead < p.nq + 2 * p.nkv && l.used) {
      const uint16_t *src = ahead < p.nq           ? q + ahead * p.q_head
                            : ahead < p.nq + p.nkv ? k + (ahead - p.nq) * p.k_head
                                                   : v + (ahead - p.nq - p.nkv) * p.v_head;
      cp_async16(&ring[fetch_slot][0][threadIdx.x], src + l.d0);
      cp_async16(&ring[fetch_slot][1][threadIdx.x], src + l.d1);
    }
    cp_async_commit();  // an empty group keeps the count
    ahead += p.groups;
    fetch_slot = fetch_slot + 1 == kAppendStages ? 0 : fetch_slot + 1;
  }
  __device__ __forceinline__ void take(const AppendParams &p, const LaneDims &l, uint4 &a, uint4 &b) {
    cp_async_wait<kAppendStages - 2>();
    a = ring[slot][0][threadIdx.x];
    b = ring[slot][1][threadIdx.x];
    slot = slot + 1 == kAppendStages ? 0 : slot + 1;
    fetch(p, l);
    h += p.groups;
  }
};

// The walk's heads of one kind, [first, end), to `out` (head 0 of the kind).  Folded into the rotation
// are the norm's weights: out_a = aa a + ab b, out_b = ba a + bb b, scaled by the norm's 1 / rms.
template <class T, int LANES, bool kV>
__device__ __forceinline__ void walk_kind(const AppendParams &p, const LaneDims &l, HeadWalk &walk, int first, int end,
                                          uint16_t *out, long long o_head, const uint16_t *w, const float2 *cs,
                                          unsigned mask) {
  if (walk.h >= end) return;
  float2 maa[4], mab[4], mba[4], mbb[4];  // pairs 2 i and 2 i + 1
  if (!kV) {
    float wa[8], wb[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) wa[i] = wb[i] = 1.f;
    if (w && l.used) split<T>(*reinterpret_cast<const uint4 *>(w + l.d0), *reinterpret_cast<const uint4 *>(w + l.d1),
                              p.interleaved, wa, wb);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 t = (i < 4 ? l.turn0 : l.turn1) ? cs[i < 4 ? l.p0 + i : l.p1 + i - 4] : make_float2(1.f, 0.f);
      (i & 1 ? maa[i / 2].y : maa[i / 2].x) = t.x * wa[i];
      (i & 1 ? mab[i / 2].y : mab[i / 2].x) = -t.y * wb[i];
      (i & 1 ? mba[i / 2].y : mba[i / 2].x) = t.y * wa[i];
      (i & 1 ? mbb[i / 2].y : mbb[i / 2].x) = t.x * wb[i];
    }
  }
  uint16_t *dst = out + (walk.h - first) * o_head;
  while (walk.h < end) {
    uint4 a, b;
    walk.take(p, l, a, b);
    if (!kV && (l.turn0 || l.turn1 || w)) {
      if (!l.used) a = b = make_uint4(0, 0, 0, 0);
      const uint4 a0 = a, b0 = b;
      float xa[8], xb[8];
      split<T>(a, b, p.interleaved, xa, xb);
      float inv = 1.f;
      if (w) {
        float2 ss = make_float2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          const float2 u = make_float2(xa[i], xa[i + 1]), v = make_float2(xb[i], xb[i + 1]);
          ss = fma2(u, u, ss);
          ss = fma2(v, v, ss);
        }
        float sum = ss.x + ss.y;
#pragma unroll
        for (int o = LANES / 2; o >= 1; o >>= 1) sum += __shfl_xor_sync(mask, sum, o);
        inv = rsqrtf(sum * p.inv_dim + p.eps);
      }
      const float2 inv2 = make_float2(inv, inv);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 u = mul2(make_float2(xa[2 * i], xa[2 * i + 1]), inv2);
        const float2 v = mul2(make_float2(xb[2 * i], xb[2 * i + 1]), inv2);
        const float2 ou = fma2(maa[i], u, mul2(mab[i], v)), ov = fma2(mba[i], u, mul2(mbb[i], v));
        xa[2 * i] = ou.x, xa[2 * i + 1] = ou.y, xb[2 * i] = ov.x, xb[2 * i + 1] = ov.y;
      }
      merge<T>(xa, xb, p.interleaved, a, b);
      if (!w && !l.turn0) a = a0;  // bit for bit, infinities and NaN too
      if (!w && !l.turn1) b = b0;
    }
    if (l.used) {
      *reinterpret_cast<uint4 *>(dst + l.d0) = a;
      *reinterpret_cast<uint4 *>(dst + l.d1) = b;
    }
    dst += p.groups * o_head;
  }
}

// `groups` lane groups share a token's heads, one after the other over all tokens and CTAs.
// The CTA forms its tokens' cosines and sines together, once, in shared memory, while the first heads
// are under way; a lane keeps those of its 8 pairs for all its heads.
template <class T, int LANES>
__global__ void __launch_bounds__(kAppendThreads, kAppendCtas) append_kernel(const __grid_constant__ AppendParams p) {
  constexpr int P = LANES * 8;  // most pairs
  extern __shared__ __align__(16) uint8_t smem_raw[];
  uint4 (*ring)[2][kAppendThreads] = reinterpret_cast<uint4 (*)[2][kAppendThreads]>(smem_raw);
  float2 (*turn)[P] = reinterpret_cast<float2 (*)[P]>(ring + kAppendStages);
  pdl_launch_dependents();
  pdl_wait();
  constexpr int G = kAppendThreads / LANES;  // lane groups of the CTA
  const long long first = static_cast<long long>(blockIdx.x) * G, mine = first + threadIdx.x / LANES;
  const int t0 = static_cast<int>(first / p.groups), t = static_cast<int>(mine / p.groups);
  const int tokens = min(static_cast<int>((first + G - 1) / p.groups), p.tokens - 1) - t0 + 1;
  const int lane = threadIdx.x % LANES, k = t - t0, g0 = static_cast<int>(mine - static_cast<long long>(t) * p.groups);
  const unsigned mask = ((1u << LANES) - 1) << ((threadIdx.x & 31) / LANES * LANES);
  const int rot = p.pairs / 8;  // lanes that rotate
  const int half = p.dim / 16;  // lanes that hold dims
  LaneDims l;
  l.used = lane < half;
  if (p.interleaved) {
    l.d0 = 8 * lane;
    l.d1 = 8 * (lane + half);
    l.turn0 = l.used && lane < 2 * rot;
    l.turn1 = l.used && lane + half < 2 * rot;
    l.p0 = l.d0 / 2;
    l.p1 = l.d1 / 2;
  } else {
    l.d0 = 8 * (lane < rot ? lane : rot + lane);
    l.d1 = 8 * (lane < rot ? lane + rot : half + lane);
    l.turn0 = l.turn1 = lane < rot;
    l.p0 = 8 * lane;
    l.p1 = 8 * lane + 4;
  }
  HeadWalk walk = {ring, p.q + t * p.q_token, p.k + t * p.k_token, p.v + t * p.v_token, g0, g0, 0, 0};
  if (k < tokens)
    for (int i = 0; i < kAppendStages - 1; ++i) walk.fetch(p, l);
  for (int i = threadIdx.x; i < tokens * p.pairs; i += blockDim.x) {
    const int kk = i / p.pairs, j = i - kk * p.pairs;
    turn[kk][j] = turn_sincos(static_cast<double>(p.pos[t0 + kk]) * p.turns[j], p.gain);
  }
  __syncthreads();
  if (k >= tokens) return;  // whole groups of LANES lanes leave together
  const float2 *cs = turn[k];

  uint16_t *row = nullptr;  // K row of head 0 in the cache
  if (p.nkv > 0) {
    const int r = p.row[t];
    if (r >= 0) {  // a negative row: a padding token, nothing is written for it
      const int page = page_of(p.cache, p.seq ? p.seq[t] : t, r);
      if (page >= 0)
        row = p.cache.pages + page * p.cache.s_page + (r % p.cache.page_rows) * p.cache.s_row;
      else if (lane == 0)
        atomicExch(&g_device_status, RIB_ECAPACITY);
    }
  }
  walk_kind<T, LANES, false>(p, l, walk, 0, p.nq, p.q_out + t * p.o_token, p.o_head, p.qw, cs, mask);
  if (row) {
    walk_kind<T, LANES, false>(p, l, walk, p.nq, p.nq + p.nkv, row, p.cache.s_head, p.kw, cs, mask);
    walk_kind<T, LANES, true>(p, l, walk, p.nq + p.nkv, p.nq + 2 * p.nkv, row + p.cache.s_half, p.cache.s_head,
                              nullptr, cs, mask);
  }
  cp_async_wait<0>();  // nothing may land after the CTA has left
}

}  // namespace paged
}  // namespace rib
