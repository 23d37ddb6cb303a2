// C ABI of the paged cache (include/rib_attention.h): host-side checks, launch geometry and workspace
// layout of paged_append.cuh, paged_decode.cuh and paged_evict.cuh.  Part of the library's one
// translation unit: uses the launch helpers of rib_attention.cu.
#pragma once

#include "paged_append.cuh"
#include "paged_decode.cuh"
#include "paged_evict.cuh"

namespace {

// Rows are 32-bit numbers, and a loop over them steps past its end by up to as many rows as it takes at once.
constexpr long long kMostRows = 0x7f000000;

inline bool aligned4(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }
// Strides of 16-byte vectors (16-bit elements).
template <typename... S>
inline bool strides8(S... s) { return ((s % 8 == 0) && ...); }

// The device view of a cache description; RIB_OK, or what is wrong with it.
int paged_view(const rib_paged_cache *c, rib::paged::View *v) {
  if (!c || !c->pages || !c->table) return RIB_EINVAL;
  if (c->dtype != RIB_DTYPE_BF16 && c->dtype != RIB_DTYPE_F16) return RIB_EINVAL;
  if (c->num_pages < 1 || c->nkv < 1 || c->page_rows < 1 || c->seqs < 1 || c->width < 1 || c->head_dim < 32 ||
      c->head_dim > 256 || c->head_dim % 16 || c->table_stride < 0 || c->stride_page < 0 || c->stride_half < 0 ||
      c->stride_head < 0 || c->stride_row < c->head_dim)
    return RIB_EINVAL;
  if (static_cast<long long>(c->width) * c->page_rows > kMostRows) return RIB_EINVAL;
  if (!aligned16(c->pages) || !aligned4(c->table) ||
      !strides8(c->stride_page, c->stride_half, c->stride_head, c->stride_row))
    return RIB_EALIGN;
  v->pages = static_cast<uint16_t *>(c->pages);
  v->table = c->table;
  v->table_stride = c->table_stride;
  v->s_page = c->stride_page;
  v->s_half = c->stride_half;
  v->s_head = c->stride_head;
  v->s_row = c->stride_row;
  v->num_pages = c->num_pages;
  v->nkv = c->nkv;
  v->page_rows = c->page_rows;
  v->seqs = c->seqs;
  v->width = c->width;
  return RIB_OK;
}

int rotary_ok(const rib_rotary *r, int dim) {
  if (!r || !r->turns || r->pairs < 8 || r->pairs % 8 || 2 * r->pairs > dim || !(r->gain > 0.f)) return RIB_EINVAL;
  return (reinterpret_cast<uintptr_t>(r->turns) & 7u) ? RIB_EALIGN : RIB_OK;
}

bool g_append_smem_done[2][4][kMaxDevices];

template <class T, int LANES>
int append_launch_lanes(rib::paged::AppendParams &p, cudaStream_t st) {
  using namespace rib::paged;
  // the lanes' rings, and (cos, sin) of 8 pairs of every lane
  constexpr int smem = kAppendThreads * (kAppendStages * 32 + 8 * 8);
  constexpr int which = LANES == 2 ? 0 : LANES == 4 ? 1 : LANES == 8 ? 2 : 3;
  if (!set_smem_once(append_kernel<T, LANES>, smem, g_append_smem_done[std::is_same<T, F16>::value][which]))
    return rib::host_fail(RIB_ECUDA, "cudaFuncSetAttribute(append smem)", smem);
  // As many lane groups to a token as one wave holds, a head each at most: few tokens spread over the
  // GPU, many keep their cosines for their heads.  Never fewer than two: the last, partly filled wave is
  // half as long then (20000 tokens of 16 + 16 heads 70 us with one, 63 with two, 67 with four).
  constexpr int in_cta = kAppendThreads / LANES;
  const int items = p.nq + 2 * p.nkv, room = in_cta * kAppendCtas * sm_count();
  p.groups = std::min(items, std::max(2, room / p.tokens));
  p.inv_dim = 1.0f / static_cast<float>(p.dim);
  const long long all = static_cast<long long>(p.tokens) * p.groups;
  return launch_pdl("append_kernel launch", append_kernel<T, LANES>, dim3(ceil_div(all, in_cta)), dim3(kAppendThreads),
                    smem, st, p);
}

template <class T>
int append_launch(rib::paged::AppendParams &p, cudaStream_t st) {
  if (p.dim <= 32) return append_launch_lanes<T, 2>(p, st);
  if (p.dim <= 64) return append_launch_lanes<T, 4>(p, st);
  if (p.dim <= 128) return append_launch_lanes<T, 8>(p, st);
  return append_launch_lanes<T, 16>(p, st);
}

// launch_pdl with thread-block clusters of `ctas` CTAs along x.
template <typename... KArgs, typename... Args>
int launch_cluster(const char *what, void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, int ctas,
                   cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.dynamicSmemBytes = smem;
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ctas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  return e == cudaSuccess ? RIB_OK : rib::host_fail_cuda(what, e);
}

// ------------------------------------------------------------------ paged decode
struct PagedDecodeLayout {
  size_t ml_off, rec_off, norm_off, span_off, logits_off, total;
  long long logit_row;
  int grid;
};

PagedDecodeLayout paged_decode_layout(int batch, int max_len, int nq, int dim, bool scores) {
  using namespace rib::paged;
  PagedDecodeLayout l;
  l.grid = (dim == 128 ? DecodeCfg<128>::CTAS : DecodeCfg<64>::CTAS) * sm_count();
  size_t off = round256(static_cast<size_t>(l.grid) * 2 * kMaxUnitHeads * dim * sizeof(float));
  l.ml_off = off;
  off += round256(static_cast<size_t>(l.grid) * 2 * kMaxUnitHeads * 2 * sizeof(float));
  l.rec_off = off;
  off += round256(static_cast<size_t>(l.grid) * sizeof(JoinRecord));
  l.logit_row = (static_cast<long long>(max_len) + TK - 1) / TK * TK;
  l.norm_off = l.span_off = l.logits_off = off;
  if (scores) {
    off += round256(static_cast<size_t>(batch) * nq * sizeof(float2));
    l.span_off = off;  // at most one unit a query head
    off += round256(static_cast<size_t>(batch) * nq * sizeof(int2));
    l.logits_off = off;
    off += round256(static_cast<size_t>(batch) * nq * l.logit_row * sizeof(float));
  }
  l.total = off;
  return l;
}

// 5-D map (D, page_rows, nkv, 2, num_pages) of the pages, box (64, TK, 1, 2, 1), 128-byte swizzle.
bool paged_map(CUtensorMap *m, const rib_paged_cache *c) {
  rib::prefill::EncodeTiledFn enc = rib::prefill::encode_fn();
  if (!enc) return false;
  cuuint64_t dims[5] = {static_cast<cuuint64_t>(c->head_dim), static_cast<cuuint64_t>(c->page_rows),
                        static_cast<cuuint64_t>(c->nkv), 2, static_cast<cuuint64_t>(c->num_pages)};
  // the stride of a dimension of one element is never used, but has to be a valid one
  const auto bytes = [&](long long stride, cuuint64_t size) {
    return static_cast<cuuint64_t>(size > 1 ? stride : c->stride_row) * 2;
  };
  cuuint64_t strides[4] = {bytes(c->stride_row, 2), bytes(c->stride_head, dims[2]), bytes(c->stride_half, 2),
                           bytes(c->stride_page, dims[4])};
  cuuint32_t box[5] = {64, static_cast<cuuint32_t>(rib::paged::TK), 1, 2, 1};
  cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  const CUresult r =
      enc(m, c->dtype == RIB_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5,
          c->pages, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) rib::host_fail(RIB_ECUDA, "cuTensorMapEncodeTiled (pages)", static_cast<int>(r));
  return r == CUDA_SUCCESS;
}

bool g_paged_smem_done[2][2][2][2][kMaxDevices];
bool g_select_smem_done[2][kMaxDevices];

template <class T, int D, int HU, bool kLogits>
int paged_decode_launch(const rib::paged::DecodeParams &p, int grid, cudaStream_t st) {
  using namespace rib::paged;
  auto kernel = paged_decode_kernel<T, D, HU, kLogits>;
  const int smem = static_cast<int>(sizeof(DecodeSmem<D, HU>)) + 1024;
  if (!set_smem_once(kernel, smem, g_paged_smem_done[std::is_same<T, F16>::value][D == 128][HU == 16][kLogits]))
    return rib::host_fail(RIB_ECUDA, "cudaFuncSetAttribute(paged decode smem)", smem);
  const int s = launch_pdl("paged_decode_kernel launch", kernel, dim3(grid), dim3(NT), smem, st, p);
  if (s != RIB_OK || (p.whole && !kLogits)) return s;
  // blocks of row weights: enough to fill the GPU once, of 1024 rows at least (64 x 512-4096 rows: 120 us;
  // with a block for every 1024 rows of a head 126)
  const long long heads = static_cast<long long>(p.cache.nkv) * p.batch, room = 4LL * sm_count();
  int row_blocks = 0, rows = 0;
  if (kLogits) {
    rows = ceil_div(p.max_len, std::min<long long>(ceil_div(p.max_len, 1024), ceil_div(room, std::min(heads, room))));
    rows = ceil_div(rows, 1024) * 1024;
    row_blocks = ceil_div(p.max_len, rows);
  }
  const long long blocks = grid + row_blocks * heads;
  if (blocks > 0x7fffffffLL) return RIB_EINVAL;
  return launch_pdl("join_kernel launch", join_kernel<T, D, HU>, dim3(static_cast<unsigned>(blocks)), dim3(kJoinThreads), 0,
                    st, p, grid, row_blocks, rows);
}

template <class T, int HU>
int paged_decode_launch(const rib::paged::DecodeParams &p, int dim, int grid, cudaStream_t st) {
  if (dim == 128)
    return p.logits ? paged_decode_launch<T, 128, HU, true>(p, grid, st)
                    : paged_decode_launch<T, 128, HU, false>(p, grid, st);
  return p.logits ? paged_decode_launch<T, 64, HU, true>(p, grid, st) : paged_decode_launch<T, 64, HU, false>(p, grid, st);
}

// Units of 8 query heads, or of 16 where a KV head has more than 8: its rows are read once per unit (64 x
// 8-9k rows, 16 heads over one of 128 dims: 53 us, as two units of 8 88; with 8 heads, 16 would do twice
// the P.V products for nothing).
inline int unit_heads(int group) { return group <= 8 ? 8 : 16; }

template <class T>
int paged_decode_launch(const rib::paged::DecodeParams &p, int dim, int grid, cudaStream_t st) {
  return unit_heads(p.group) == 8 ? paged_decode_launch<T, 8>(p, dim, grid, st)
                                  : paged_decode_launch<T, 16>(p, dim, grid, st);
}

template <int kThreads>
int select_launch(const rib::paged::SelectParams &s, long long units, int batch, cudaStream_t st) {
  using namespace rib::paged;
  // CTAs of a cluster: more while they fit one wave and each still has 4096 rows.  A cluster's barriers cost
  // about 1 us each (one sequence of 4097 rows: 18.6 us with two CTAs a head, 14.6 with one), and a second
  // wave more (8 x 8 heads of 65536 rows: 212 us with four, 204 with two, which fit at once).
  int ctas = 1;
  while (ctas < 8 && 2 * ctas * units <= sm_count() && s.max_len >= 8192 * ctas) ctas *= 2;
  const int part = ceil_div(s.max_len, ctas * kThreads) * kThreads;
  constexpr int most = kSelStepRows * kThreads;
  const bool fits = part <= most;  // always with 512 threads
  if (!set_smem_once(select_rows_kernel<kThreads, true>, most * static_cast<int>(sizeof(float)),
                     g_select_smem_done[kThreads == 1024]))
    return rib::host_fail(RIB_ECUDA, "cudaFuncSetAttribute(select smem)", most);
  auto kernel = select_rows_kernel<kThreads, true>;
  if constexpr (kThreads == 1024)
    if (!fits) kernel = select_rows_kernel<kThreads, false>;
  return launch_cluster("select_rows_kernel launch", kernel, dim3(s.nkv * ctas, batch), dim3(kThreads),
                        fits ? part * sizeof(float) : 0, ctas, st, s);
}

}  // namespace

extern "C" {

int rib_rotary_apply(const rib_rotary *rot, const void *x, long long x_token, long long x_head, void *out,
                     long long out_token, long long out_head, const int32_t *pos, int tokens, int heads, int dim,
                     int dtype, void *stream) {
  if (!x || !out || !pos || tokens < 0 || heads < 1 || dim < 32 || dim > 256 || dim % 16) return RIB_EINVAL;
  if (dtype != RIB_DTYPE_BF16 && dtype != RIB_DTYPE_F16) return RIB_EINVAL;
  const int rs = rotary_ok(rot, dim);
  if (rs != RIB_OK) return rs;
  if (!aligned16(x) || !aligned16(out) || !aligned4(pos) || !strides8(x_token, x_head, out_token, out_head))
    return RIB_EALIGN;
  if (tokens == 0) return RIB_OK;
  if (!bind_stream_device(stream)) return rib::host_fail(RIB_ECUDA, "bind stream device", 0);
  rib::paged::AppendParams p = {};
  p.q = static_cast<const uint16_t *>(x);
  p.q_out = static_cast<uint16_t *>(out);
  p.q_token = x_token;
  p.q_head = x_head;
  p.o_token = out_token;
  p.o_head = out_head;
  p.pos = pos;
  p.turns = rot->turns;
  p.gain = rot->gain;
  p.pairs = rot->pairs;
  p.interleaved = rot->interleaved != 0;
  p.tokens = tokens;
  p.nq = heads;
  p.dim = dim;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == RIB_DTYPE_F16 ? append_launch<rib::paged::F16>(p, st) : append_launch<rib::paged::BF16>(p, st);
}

int rib_paged_append(const rib_paged_cache *cache, const rib_rotary *rot, const void *q, long long q_token,
                     long long q_head, const void *k, long long k_token, long long k_head, const void *v,
                     long long v_token, long long v_head, void *q_out, long long out_token, long long out_head,
                     const int32_t *pos, const int32_t *row, const int32_t *seq, int tokens, int nq, const void *qw,
                     const void *kw, float eps, void *stream) {
  rib::paged::AppendParams p = {};
  const int cs = paged_view(cache, &p.cache);
  if (cs != RIB_OK) return cs;
  if (!q || !k || !v || !q_out || !pos || !row || tokens < 0 || nq < 1) return RIB_EINVAL;
  if (!qw != !kw || (qw && !(eps >= 0.f))) return RIB_EINVAL;
  if (!seq && tokens > cache->seqs) return RIB_EINVAL;
  const int rs = rotary_ok(rot, cache->head_dim);
  if (rs != RIB_OK) return rs;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(q_out) || !aligned16(qw) || !aligned16(kw) ||
      !aligned4(pos) || !aligned4(row) || !aligned4(seq) ||
      !strides8(q_token, q_head, k_token, k_head, v_token, v_head, out_token, out_head))
    return RIB_EALIGN;
  if (tokens == 0) return RIB_OK;
  if (!bind_stream_device(stream)) return rib::host_fail(RIB_ECUDA, "bind stream device", 0);
  p.q = static_cast<const uint16_t *>(q);
  p.k = static_cast<const uint16_t *>(k);
  p.v = static_cast<const uint16_t *>(v);
  p.q_out = static_cast<uint16_t *>(q_out);
  p.q_token = q_token;
  p.q_head = q_head;
  p.k_token = k_token;
  p.k_head = k_head;
  p.v_token = v_token;
  p.v_head = v_head;
  p.o_token = out_token;
  p.o_head = out_head;
  p.pos = pos;
  p.row = row;
  p.seq = seq;
  p.turns = rot->turns;
  p.gain = rot->gain;
  p.pairs = rot->pairs;
  p.interleaved = rot->interleaved != 0;
  p.qw = static_cast<const uint16_t *>(qw);
  p.kw = static_cast<const uint16_t *>(kw);
  p.eps = eps;
  p.tokens = tokens;
  p.nq = nq;
  p.nkv = cache->nkv;
  p.dim = cache->head_dim;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return cache->dtype == RIB_DTYPE_F16 ? append_launch<rib::paged::F16>(p, st) : append_launch<rib::paged::BF16>(p, st);
}

size_t rib_paged_decode_workspace_bytes(int batch, int max_len, int nq, int head_dim, int with_scores) {
  if (batch < 1 || max_len < 1 || nq < 1 || (head_dim != 64 && head_dim != 128)) return 0;
  return paged_decode_layout(batch, max_len, nq, head_dim, with_scores != 0).total;
}

int rib_paged_decode_attention(const rib_paged_cache *cache, const void *q, long long q_seq, long long q_head,
                               const int32_t *lens, int batch, int nq, int max_len, float scale, void *out,
                               const float *scores, long long scores_seq, long long scores_head, float *scores_out,
                               long long out_seq, long long out_head, void *workspace, size_t workspace_bytes,
                               void *stream) {
  using namespace rib::paged;
  DecodeParams p = {};
  const int cs = paged_view(cache, &p.cache);
  if (cs != RIB_OK) return cs;
  const int dim = cache->head_dim;
  if (!q || !lens || !out || batch < 1 || batch > cache->seqs || nq < 1 || nq % cache->nkv || max_len < 1 ||
      max_len > static_cast<long long>(cache->width) * cache->page_rows || !(scale > 0.f) ||
      !(scale * 1.4426950408889634 < 3.4e38) ||  // scores are formed in log2 units
      (dim != 64 && dim != 128) || cache->page_rows % TK || !scores != !scores_out)
    return RIB_EINVAL;
  const PagedDecodeLayout l = paged_decode_layout(batch, max_len, nq, dim, scores != nullptr);
  const int group = nq / cache->nkv, units_per_kv = ceil_div(group, unit_heads(group));
  // a CTA counts the tiles of its run in 32 bits
  if (static_cast<double>(batch) * cache->nkv * units_per_kv * ceil_div(max_len, TK) > static_cast<double>(kMostRows) * l.grid)
    return RIB_EINVAL;
  if (!workspace || workspace_bytes < l.total) return RIB_EINVAL;
  if (!aligned16(q) || !aligned16(out) || !aligned16(workspace) || !aligned4(lens) || !aligned4(scores) ||
      !aligned4(scores_out) || !strides8(q_seq, q_head))
    return RIB_EALIGN;
  if (!bind_stream_device(stream)) return rib::host_fail(RIB_ECUDA, "bind stream device", 0);
  if (!paged_map(&p.map, cache)) return RIB_ECUDA;
  uint8_t *ws = static_cast<uint8_t *>(workspace);
  p.q = static_cast<const uint16_t *>(q);
  p.out = static_cast<uint16_t *>(out);
  p.q_seq = q_seq;
  p.q_head = q_head;
  p.lens = lens;
  p.batch = batch;
  p.nq = nq;
  p.group = group;
  p.units_per_kv = units_per_kv;
  p.max_len = max_len;
  p.scale2 = static_cast<float>(scale * 1.4426950408889634);
  p.whole = max_len <= kWholeRows;
  p.part_o = reinterpret_cast<float *>(ws);
  p.part_ml = reinterpret_cast<float *>(ws + l.ml_off);
  p.rec = reinterpret_cast<JoinRecord *>(ws + l.rec_off);
  p.logit_row = l.logit_row;
  if (scores) {
    p.norm = reinterpret_cast<float2 *>(ws + l.norm_off);
    p.span = reinterpret_cast<int2 *>(ws + l.span_off);
    p.logits = reinterpret_cast<float *>(ws + l.logits_off);
    p.scores = scores;
    p.scores_out = scores_out;
    p.in_seq = scores_seq;
    p.in_head = scores_head;
    p.out_seq = out_seq;
    p.out_head = out_head;
  }
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return cache->dtype == RIB_DTYPE_F16 ? paged_decode_launch<F16>(p, dim, l.grid, st)
                                       : paged_decode_launch<BF16>(p, dim, l.grid, st);
}

int rib_paged_evict(const rib_paged_cache *cache, const int32_t *new_table, long long new_table_stride, int new_width,
                    const int32_t *lens, int batch, int max_len, const float *scores, long long scores_seq,
                    long long scores_head, int keep, int sinks, int recent, int32_t *rows, int32_t *new_lens,
                    float *new_scores, long long new_seq, long long new_head, int new_score_rows, void *stream) {
  using namespace rib::paged;
  MoveParams m;
  const int cs = paged_view(cache, &m.from);
  if (cs != RIB_OK) return cs;
  rib_paged_cache moved = *cache;
  moved.table = new_table;
  moved.table_stride = new_table_stride;
  moved.width = new_width;
  const int ms = paged_view(&moved, &m.to);
  if (ms != RIB_OK) return ms;
  if (!lens || !scores || !rows || !new_lens || batch < 1 || batch > cache->seqs || batch > 65535 ||
      cache->nkv > 65535 || max_len < 1 || max_len > static_cast<long long>(cache->width) * cache->page_rows ||
      keep < 1 || keep > kMostRows || sinks < 0 || recent < 0 || static_cast<long long>(sinks) + recent > keep ||
      std::min(keep, max_len) > static_cast<long long>(new_width) * cache->page_rows ||
      (new_scores && (new_score_rows < keep || new_score_rows > kMostRows)) ||
      (cache->head_dim != 64 && cache->head_dim != 128))
    return RIB_EINVAL;
  if (!aligned4(lens) || !aligned4(scores) || !aligned4(rows) || !aligned4(new_lens) || !aligned4(new_scores))
    return RIB_EALIGN;
  if (!bind_stream_device(stream)) return rib::host_fail(RIB_ECUDA, "bind stream device", 0);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  SelectParams s;
  s.scores = scores;
  s.lens = lens;
  s.rows = rows;
  s.new_lens = new_lens;
  s.new_scores = new_scores;
  s.s_seq = scores_seq;
  s.s_head = scores_head;
  s.n_seq = new_seq;
  s.n_head = new_head;
  s.nkv = cache->nkv;
  s.keep = keep;
  s.sinks = sinks;
  s.recent = recent;
  s.max_len = max_len;
  s.new_width = new_score_rows;
  // CTAs of 512 threads where rows are few, or few for so many heads that the CTAs queue (us for both
  // kernels, 512 against 1024 threads: 90 x 8 heads of 700 rows 27 and 33, 3 x 4 of 700 7.7 and 9.2,
  // 90 x 8 of 2000 76 and 81; but 10 x 4 of 2000 16.5 and 14.2, 30 x 8 of 4000 76 and 71)
  const long long units = static_cast<long long>(batch) * cache->nkv;
  const bool few = max_len <= 1024 || (max_len <= 2048 && units > 2 * sm_count());
  const int e = few ? select_launch<512>(s, units, batch, st) : select_launch<1024>(s, units, batch, st);
  if (e != RIB_OK) return e;
  m.rows = rows;
  m.keep = keep;
  return launch_pdl("move_rows_kernel launch", cache->head_dim == 128 ? move_rows_kernel<128> : move_rows_kernel<64>,
                    dim3(ceil_div(std::min(keep, max_len), kMoveThreads / 32 * kMoveRows), cache->nkv, batch), dim3(kMoveThreads), 0, st, m);
}

}  // extern "C"
