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
// Work split: D/16 lanes hold one head, 16 dims each as two 16-byte vectors, so both members of a pair
// sit in one lane and no lane exchanges dims with another (the norm's sum of squares is the only
// shuffle).  A lane's 8 pairs are the same for every head of a token: it forms their cosines and sines
// once and walks over heads, `groups` lanes groups sharing a token's heads.
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
  float gain, eps;
  int tokens, nq, nkv, dim, pairs, interleaved, groups;
};

// Cosine and sine of `turns` turns (FP64) times gain.
__device__ __forceinline__ void turn_sincos(double turns, float gain, float &c, float &s) {
  const float part = static_cast<float>(turns - rint(turns));  // [-1/2, 1/2]
  sincospif(2.0f * part, &s, &c);
  c *= gain;
  s *= gain;
}

template <class T, int LANES>
__global__ void __launch_bounds__(256) append_kernel(const __grid_constant__ AppendParams p) {
  pdl_wait();
  const int lane = threadIdx.x % LANES;
  const long long id = (static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x) / LANES;
  const int t = static_cast<int>(id / p.groups), g0 = static_cast<int>(id % p.groups);
  if (t >= p.tokens) return;  // whole groups of LANES lanes leave together
  const unsigned mask = LANES == 32 ? 0xffffffffu : ((1u << LANES) - 1) << ((threadIdx.x & 31) / LANES * LANES);
  const int chunks = p.dim / 8, rot = p.pairs / 8;   // 16-byte chunks of a head; lanes that rotate
  const bool turns = lane < rot, used = 2 * lane < chunks;
  // the lane's two chunks
  int c0, c1;
  if (turns && !p.interleaved) {
    c0 = lane;
    c1 = lane + rot;
  } else {  // interleaved pairs, and the dims that pass unchanged, are consecutive
    c0 = 2 * lane;
    c1 = 2 * lane + 1;
  }
  float cs[8], sn[8];
  if (turns) {
    const double pos = static_cast<double>(p.pos[t]);
#pragma unroll
    for (int i = 0; i < 8; ++i) turn_sincos(pos * p.turns[8 * lane + i], p.gain, cs[i], sn[i]);
  }
  uint16_t *dst = nullptr;  // K row of head 0 in the cache
  if (p.nkv > 0) {
    const int r = p.row[t], s = p.seq ? p.seq[t] : t;
    if (r >= 0) {  // a negative row: a padding token, nothing is written for it
      const int page = page_of(p.cache, s, r);
      if (page >= 0) {
        dst = p.cache.pages + page * p.cache.s_page + (r % p.cache.page_rows) * p.cache.s_row;
      } else if (lane == 0) {
        atomicExch(&g_device_status, RIB_ECAPACITY);
      }
    }
  }
  const int items = p.nq + 2 * p.nkv;
  for (int h = g0; h < items; h += p.groups) {
    const bool is_q = h < p.nq, is_v = h >= p.nq + p.nkv;
    const uint16_t *src = is_q ? p.q + t * p.q_token + h * p.q_head
                          : is_v ? p.v + t * p.v_token + (h - p.nq - p.nkv) * p.v_head
                                 : p.k + t * p.k_token + (h - p.nq) * p.k_head;
    uint16_t *out = is_q ? p.q_out + t * p.o_token + h * p.o_head
                    : !dst ? nullptr
                    : is_v ? dst + p.cache.s_half + (h - p.nq - p.nkv) * p.cache.s_head
                           : dst + (h - p.nq) * p.cache.s_head;
    if (!out) continue;  // the same for every lane of the group
    uint4 a = make_uint4(0, 0, 0, 0), b = a;
    if (used) {
      a = *reinterpret_cast<const uint4 *>(src + 8 * c0);
      b = *reinterpret_cast<const uint4 *>(src + 8 * c1);
    }
    const uint16_t *w = is_q ? p.qw : p.kw;
    if (!is_v && (turns || w)) {
      float x[16];
      const uint32_t raw[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 f = T::unpack(raw[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      }
      if (w) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
        for (int o = LANES / 2; o >= 1; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
        const float inv = 1.0f / sqrtf(ss / static_cast<float>(p.dim) + p.eps);
        if (used) {
          const uint4 wa = *reinterpret_cast<const uint4 *>(w + 8 * c0);
          const uint4 wb = *reinterpret_cast<const uint4 *>(w + 8 * c1);
          const uint32_t wr[8] = {wa.x, wa.y, wa.z, wa.w, wb.x, wb.y, wb.z, wb.w};
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float2 f = T::unpack(wr[i]);
            x[2 * i] *= inv * f.x;
            x[2 * i + 1] *= inv * f.y;
          }
        }
      }
      if (turns) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          // constant indices on both sides of the select keep x in registers
          const float u = p.interleaved ? x[2 * i] : x[i], z = p.interleaved ? x[2 * i + 1] : x[8 + i];
          const float ru = u * cs[i] - z * sn[i], rz = u * sn[i] + z * cs[i];
          if (p.interleaved) {
            x[2 * i] = ru;
            x[2 * i + 1] = rz;
          } else {
            x[i] = ru;
            x[8 + i] = rz;
          }
        }
      }
      a = make_uint4(T::pack(x[0], x[1]), T::pack(x[2], x[3]), T::pack(x[4], x[5]), T::pack(x[6], x[7]));
      b = make_uint4(T::pack(x[8], x[9]), T::pack(x[10], x[11]), T::pack(x[12], x[13]), T::pack(x[14], x[15]));
    }
    if (used) {
      *reinterpret_cast<uint4 *>(out + 8 * c0) = a;
      *reinterpret_cast<uint4 *>(out + 8 * c1) = b;
    }
  }
}

}  // namespace paged
}  // namespace rib
