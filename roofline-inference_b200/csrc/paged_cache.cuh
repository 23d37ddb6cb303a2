// Paged KV cache: the device view that the paged kernels share.
//
// Pages are [num_pages][2][nkv][page_rows][D] (K, then V) of BF16 or FP16 values with a stride for
// every dimension but the last; `table` [seqs][width] names the pages of each sequence in order, so
// row r of sequence s lies in page table[s][r / page_rows] at r % page_rows.  A table entry outside
// [0, num_pages) names no page: no kernel reads or writes through it.
//
// Every kernel here waits for the one before it (pdl_wait) before it touches memory, and reads what that
// one may have written with ordinary loads: it may be running while the other still writes, so nothing
// is read-only for its whole life, as the non-coherent path asks.
#pragma once

#include "common.cuh"

namespace rib {
namespace paged {

struct View {
  uint16_t *pages;
  const int32_t *table;
  long long table_stride;                            // entries between two sequences
  long long s_page, s_half, s_head, s_row;           // elements
  int num_pages, nkv, page_rows, seqs, width;
};

// Two packed 16-bit values <-> FP32.
struct BF16 {
  static __device__ __forceinline__ float2 unpack(uint32_t w) { return make_float2(bf16lo(w), bf16hi(w)); }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_bf16x2(lo, hi); }
  static constexpr uint32_t kInf = 0x7f80;
  static constexpr int kLift = 0;   // a weight in (0, 1] keeps its relative precision down to 2^-126
};
struct F16 {
  static __device__ __forceinline__ float2 unpack(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&w));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_f16x2(lo, hi); }
  static constexpr uint32_t kInf = 0x7c00;
  static constexpr int kLift = 14;  // times 2^14, it does down to 2^-28, and below that is off by 2^-39 at most
};

// Page of row `r` of sequence `s`, or -1 where the table names none.
__device__ __forceinline__ int page_of(const View &v, int s, int r) {
  const int i = r / v.page_rows;
  if (s < 0 || s >= v.seqs || r < 0 || i >= v.width) return -1;
  const int page = v.table[s * v.table_stride + i];
  return page >= 0 && page < v.num_pages ? page : -1;
}

}  // namespace paged
}  // namespace rib
