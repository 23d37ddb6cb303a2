// Python binding of the paged-cache entry points (include/rib_attention.h): argument checks, outputs,
// scratch and the launch in one native call.  A decode step makes a few of these calls per layer; as
// ctypes wrappers each spent about 25 us of host time, which the device waited for.
//
// The functions take positional arguments only; paged.py gives them their public names, keywords and
// documentation.  The entry points are handed over by address (bind), so this module links against
// nothing but torch.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <exception>
#include <string>
#include <utility>

#include "../../include/rib_attention.h"

namespace {

decltype(&rib_status_string) status_string;
decltype(&rib_last_error_string) last_error_string;
decltype(&rib_rotary_apply) rotary_apply;
decltype(&rib_paged_append) paged_append_fn;
decltype(&rib_paged_decode_workspace_bytes) decode_workspace_bytes;
decltype(&rib_paged_decode_attention) decode_attention_fn;
decltype(&rib_paged_evict) paged_evict_fn;

constexpr int kMostRows = 0x7f000000;  // as the library has it

struct Refused {};  // a Python exception is set

[[noreturn]] void refuse(const char *fmt, ...) {
  char text[512];
  va_list args;
  va_start(args, fmt);
  vsnprintf(text, sizeof(text), fmt, args);
  va_end(args);
  PyErr_SetString(PyExc_ValueError, text);
  throw Refused{};
}

std::string shape_of(const at::Tensor &t) {
  std::string s = "(";
  for (int64_t n : t.sizes()) s += (s.size() > 1 ? ", " : "") + std::to_string(n);
  return s + ")";
}

const at::Tensor &any_tensor(PyObject *o, const char *name, int dim) {
  if (!THPVariable_Check(o)) refuse("%s must be a torch.Tensor", name);
  const at::Tensor &t = THPVariable_Unpack(o);
  if (!t.is_cuda()) refuse("%s must be a CUDA tensor", name);
  if (t.layout() != at::kStrided) refuse("%s must be a dense tensor", name);
  if (t.dim() != dim) refuse("%s must have %d dimensions, got %s", name, dim, shape_of(t).c_str());
  if (t.stride(dim - 1) != 1 && t.size(dim - 1) != 1) refuse("%s: the last dimension must be contiguous", name);
  if (t.is_neg() || t.is_conj()) refuse("%s must hold its values as they are", name);
  return t;
}

const at::Tensor &tensor(PyObject *o, const char *name, int dim, at::ScalarType type, c10::Device dev) {
  const at::Tensor &t = any_tensor(o, name, dim);
  if (t.scalar_type() != type) refuse("%s must be %s, got %s", name, c10::toString(type), c10::toString(t.scalar_type()));
  if (t.device() != dev)
    refuse("tensors on different devices: %s is on %s, not %s", name, t.device().str().c_str(), dev.str().c_str());
  return t;
}

// A stride as the C ABI takes it: that of a dimension of one element is never used.
int64_t step(const at::Tensor &t, int64_t dim) { return t.size(dim) > 1 ? t.stride(dim) : 0; }

// A tensor that a kernel writes: no two of its elements may share memory by a stride of 0.
const at::Tensor &written(const at::Tensor &t, const char *name) {
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.stride(i) == 0 && t.size(i) > 1) refuse("%s must not be an expanded tensor", name);
  return t;
}

const int32_t *vector(PyObject *o, const char *name, int64_t n, c10::Device dev) {
  const at::Tensor &t = tensor(o, name, 1, at::kInt, dev);
  if (t.size(0) != n) refuse("%s must hold %lld numbers, got %lld", name, (long long)n, (long long)t.size(0));
  return t.const_data_ptr<int32_t>();
}

int dtype_of(const at::Tensor &t, const char *name) {
  if (t.scalar_type() == at::kBFloat16) return RIB_DTYPE_BF16;
  if (t.scalar_type() == at::kHalf) return RIB_DTYPE_F16;
  refuse("%s must be bfloat16 or float16", name);
}

// A number of an argument, within what the C ABI's int holds.
int number(PyObject *o, const char *name) {
  int overflow = 0;
  const long long v = PyLong_AsLongLongAndOverflow(o, &overflow);
  if (v == -1 && PyErr_Occurred()) throw Refused{};
  if (overflow || v > 0x7fffffffLL || v < -0x7fffffffLL) refuse("%s is out of range", name);
  return static_cast<int>(v);
}

double real(PyObject *o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Refused{};
  return v;
}

int size32(int64_t n, const char *name) {
  if (n > 0x7fffffffLL) refuse("%s is too large", name);
  return static_cast<int>(n);
}

rib_paged_cache cache_of(PyObject *pages_o, PyObject *table_o, const at::Tensor **pages_out) {
  const at::Tensor &pages = any_tensor(pages_o, "pages", 5);
  rib_paged_cache c;
  c.dtype = dtype_of(pages, "pages");
  if (pages.size(1) != 2 || pages.numel() == 0)
    refuse("pages must be [num_pages, 2, nkv, page_rows, head_dim], got %s", shape_of(pages).c_str());
  written(pages, "pages");
  const at::Tensor &table = tensor(table_o, "table", 2, at::kInt, pages.device());
  if (table.numel() == 0) refuse("table must be [sequences, width], got %s", shape_of(table).c_str());
  c.pages = pages.data_ptr();
  c.table = table.const_data_ptr<int32_t>();
  c.table_stride = step(table, 0);
  c.stride_page = step(pages, 0);
  c.stride_half = pages.stride(1);
  c.stride_head = step(pages, 2);
  c.stride_row = pages.size(3) > 1 ? pages.stride(3) : pages.size(4);
  c.num_pages = size32(pages.size(0), "pages");
  c.nkv = size32(pages.size(2), "pages");
  c.page_rows = size32(pages.size(3), "pages");
  c.head_dim = size32(pages.size(4), "pages");
  c.seqs = size32(table.size(0), "table");
  c.width = size32(table.size(1), "table");
  *pages_out = &pages;
  return c;
}

// Rotary's handle: (turns, head_dim, pairs, interleaved, gain).
rib_rotary rotary_of(PyObject *o, int64_t dim, c10::Device dev) {
  if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 5) refuse("rot must be a Rotary");
  const int head_dim = number(PyTuple_GET_ITEM(o, 1), "head_dim");
  if (head_dim != dim) refuse("heads have %lld dims, the rotation %d", (long long)dim, head_dim);
  rib_rotary r;
  r.turns = tensor(PyTuple_GET_ITEM(o, 0), "rot", 1, at::kDouble, dev).const_data_ptr<double>();
  r.pairs = number(PyTuple_GET_ITEM(o, 2), "pairs");
  r.interleaved = number(PyTuple_GET_ITEM(o, 3), "interleaved");
  r.gain = static_cast<float>(real(PyTuple_GET_ITEM(o, 4)));
  return r;
}

const at::Tensor &heads(PyObject *o, const char *name, int64_t tokens, int64_t n, const at::Tensor &like) {
  const at::Tensor &t = tensor(o, name, 3, like.scalar_type(), like.device());
  const int64_t dim = like.size(like.dim() - 1);
  if (t.size(0) != tokens || (n >= 0 && t.size(1) != n) || t.size(2) != dim)
    refuse("%s must be [%lld, %s, %lld], got %s", name, (long long)tokens, n < 0 ? "heads" : std::to_string(n).c_str(),
           (long long)dim, shape_of(t).c_str());
  return t;
}

// An uninitialised tensor from torch's CUDA allocator (at::empty without its dispatch, 1 us of 5).
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, c10::Device dev) {
  return at::Tensor(at::detail::empty_cuda(sizes, type, dev, std::nullopt));
}

at::Tensor output(PyObject *o, const at::Tensor &like, const char *name) {
  if (o == Py_None) return fresh(like.sizes(), like.scalar_type(), like.device());
  const at::Tensor &t = tensor(o, name, static_cast<int>(like.dim()), like.scalar_type(), like.device());
  if (t.sizes() != like.sizes()) refuse("%s must be %s, got %s", name, shape_of(like).c_str(), shape_of(t).c_str());
  return written(t, name);
}

void checked(int status, const char *what) {
  if (status == RIB_OK) return;
  if (status == RIB_EINVAL || status == RIB_ECAPACITY || status == RIB_EALIGN)
    refuse("%s: %s", what, status_string(status));
  PyErr_Format(PyExc_RuntimeError, "%s: %s (status %d): %s", what, status_string(status), status, last_error_string());
  throw Refused{};
}

// Runs a body that returns a new reference; C++ exceptions become Python's.
template <class F>
PyObject *guarded(Py_ssize_t given, Py_ssize_t wanted, const char *name, F body) {
  try {
    if (given != wanted) {
      PyErr_Format(PyExc_TypeError, "%s takes %zd arguments, got %zd", name, wanted, given);
      return nullptr;
    }
    if (!paged_evict_fn) {
      PyErr_SetString(PyExc_RuntimeError, "the library is not bound");
      return nullptr;
    }
    return body();
  } catch (const Refused &) {
    return nullptr;
  } catch (...) {
    torch::translate_exception_to_python(std::current_exception());
    return nullptr;
  }
}

void *stream_of(c10::Device dev) { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }

// (x, pos, rot, out)
PyObject *rotary(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded(n, 4, "rotary", [&]() -> PyObject * {
    const at::Tensor &x = any_tensor(a[0], "x", 3);
    const int dtype = dtype_of(x, "x");
    const c10::Device dev = x.device();
    const rib_rotary rot = rotary_of(a[2], x.size(2), dev);
    const int tokens = size32(x.size(0), "x"), nh = size32(x.size(1), "x");
    const int32_t *pos = vector(a[1], "pos", tokens, dev);
    const c10::cuda::CUDAGuard guard(dev);
    const at::Tensor out = output(a[3], x, "out");
    if (x.numel() > 0)
      checked(rotary_apply(&rot, x.const_data_ptr(), step(x, 0), step(x, 1), out.data_ptr(), step(out, 0),
                           step(out, 1), pos, tokens, nh, static_cast<int>(x.size(2)), dtype, stream_of(dev)),
              "rotary");
    return THPVariable_Wrap(out);
  });
}

// (q, k, v, pos, row, pages, table, rot, seq, qw, kw, eps, out)
PyObject *paged_append(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded(n, 13, "paged_append", [&]() -> PyObject * {
    const at::Tensor *pages;
    const rib_paged_cache cache = cache_of(a[5], a[6], &pages);
    const c10::Device dev = pages->device();
    const at::Tensor &q0 = any_tensor(a[0], "q", 3);
    const int tokens = size32(q0.size(0), "q"), nq = size32(q0.size(1), "q");
    const at::Tensor &q = heads(a[0], "q", tokens, -1, *pages), &k = heads(a[1], "k", tokens, cache.nkv, *pages),
                     &v = heads(a[2], "v", tokens, cache.nkv, *pages);
    if (nq < 1) refuse("q has no heads");
    const rib_rotary rot = rotary_of(a[7], cache.head_dim, dev);
    if ((a[9] == Py_None) != (a[10] == Py_None)) refuse("qw and kw come together");
    const void *w[2] = {nullptr, nullptr};
    for (int i = 0; i < 2 && a[9] != Py_None; ++i) {
      const at::Tensor &t = tensor(a[9 + i], i ? "kw" : "qw", 1, pages->scalar_type(), dev);
      if (t.size(0) != cache.head_dim) refuse("%s must hold %d values", i ? "kw" : "qw", cache.head_dim);
      w[i] = t.const_data_ptr();
    }
    const double eps = real(a[11]);
    if (!(eps >= 0.0) || !std::isfinite(eps)) refuse("eps must be finite and not negative");
    if (a[8] == Py_None && tokens > cache.seqs)
      refuse("%d tokens for %d sequences: seq says where each belongs", tokens, cache.seqs);
    const int32_t *pos = vector(a[3], "pos", tokens, dev), *row = vector(a[4], "row", tokens, dev);
    const int32_t *seq = a[8] == Py_None ? nullptr : vector(a[8], "seq", tokens, dev);
    const c10::cuda::CUDAGuard guard(dev);
    const at::Tensor out = output(a[12], q, "out");
    if (tokens > 0)
      checked(paged_append_fn(&cache, &rot, q.const_data_ptr(), step(q, 0), step(q, 1), k.const_data_ptr(),
                              step(k, 0), step(k, 1), v.const_data_ptr(), step(v, 0), step(v, 1), out.data_ptr(),
                              step(out, 0), step(out, 1), pos, row, seq, tokens, nq, w[0], w[1],
                              static_cast<float>(eps), stream_of(dev)),
              "paged_append");
    return THPVariable_Wrap(out);
  });
}

const at::Tensor &scores_of(PyObject *o, const char *name, int64_t batch, int64_t nkv, int64_t least, c10::Device dev) {
  const at::Tensor &t = tensor(o, name, 3, at::kFloat, dev);
  if (t.size(0) != batch || t.size(1) != nkv || t.size(2) < least)
    refuse("%s must be [%lld, %lld, >= %lld], got %s", name, (long long)batch, (long long)nkv, (long long)least,
           shape_of(t).c_str());
  return t;
}

// The rows a sequence may have: what the table holds, or the caller's bound below it.
int max_len_of(PyObject *o, const rib_paged_cache &c) {
  const int64_t room = static_cast<int64_t>(c.width) * c.page_rows;
  if (o == Py_None) return size32(room, "the table's rows");
  const int n = number(o, "max_len");
  if (n < 1) refuse("max_len must be positive");
  if (n > room) refuse("KV capacity exceeded");
  return n;
}

void head_dim_64_128(const rib_paged_cache &c) {
  if (c.head_dim != 64 && c.head_dim != 128) refuse("head_dim must be 64 or 128, got %d", c.head_dim);
}

// First and one past the last byte that a tensor's values lie in.
std::pair<uintptr_t, uintptr_t> span(const at::Tensor &t) {
  int64_t last = 0;
  for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
  const uintptr_t at = reinterpret_cast<uintptr_t>(t.const_data_ptr());
  return {at, at + (last + 1) * t.element_size()};
}

// (q, pages, table, lens, scale, max_len, scores, scores_out, out)
PyObject *paged_decode_attention(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded(n, 9, "paged_decode_attention", [&]() -> PyObject * {
    const at::Tensor *pages;
    const rib_paged_cache cache = cache_of(a[1], a[2], &pages);
    const c10::Device dev = pages->device();
    const at::Tensor &q0 = any_tensor(a[0], "q", 3);
    const int batch = size32(q0.size(0), "q"), nq = size32(q0.size(1), "q");
    const at::Tensor &q = heads(a[0], "q", batch, -1, *pages);
    head_dim_64_128(cache);
    if (cache.page_rows % 16) refuse("page_rows must be a multiple of 16, got %d", cache.page_rows);
    if (batch < 1 || batch > cache.seqs) refuse("%d queries for %d sequences", batch, cache.seqs);
    if (nq < 1 || nq % cache.nkv) refuse("nq (%d) must be a multiple of nkv (%d)", nq, cache.nkv);
    const double scale = real(a[4]);
    if (!(scale > 0.0) || !std::isfinite(scale)) refuse("scale must be positive and finite");
    const int max_len = max_len_of(a[5], cache);
    const int32_t *lens = vector(a[3], "lens", batch, dev);
    const float *in = nullptr;
    float *to = nullptr;
    int64_t in_s[2] = {0, 0}, to_s[2] = {0, 0};
    if (a[6] != Py_None) {
      const at::Tensor &s = scores_of(a[6], "scores", batch, cache.nkv, max_len, dev);
      const at::Tensor &t = a[7] == Py_None ? s : scores_of(a[7], "scores_out", batch, cache.nkv, max_len, dev);
      in = s.const_data_ptr<float>();
      to = written(t, "scores_out").data_ptr<float>();
      in_s[0] = step(s, 0), in_s[1] = step(s, 1), to_s[0] = step(t, 0), to_s[1] = step(t, 1);
      const auto x = span(s), y = span(t);
      if (x.first < y.second && y.first < x.second && (in != to || in_s[0] != to_s[0] || in_s[1] != to_s[1]))
        refuse("scores_out must be scores itself or not overlap it");
    } else if (a[7] != Py_None) {
      refuse("scores_out needs scores");
    }
    const c10::cuda::CUDAGuard guard(dev);
    const at::Tensor out = output(a[8], q, "out");
    if (!out.is_contiguous()) refuse("out must be contiguous");
    const size_t bytes = decode_workspace_bytes(batch, max_len, nq, cache.head_dim, in != nullptr);
    // scratch of this call alone: the allocator hands it on in stream order
    const at::Tensor ws = fresh({static_cast<int64_t>(bytes)}, at::kByte, dev);
    checked(decode_attention_fn(&cache, q.const_data_ptr(), step(q, 0), step(q, 1), lens, batch, nq, max_len,
                                static_cast<float>(scale), out.data_ptr(), in, in_s[0], in_s[1], to, to_s[0], to_s[1],
                                ws.data_ptr(), bytes, stream_of(dev)),
            "paged_decode_attention");
    return THPVariable_Wrap(out);
  });
}

// (pages, table, lens, scores, keep, new_table, sinks, recent, max_len, new_scores)
PyObject *paged_evict(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded(n, 10, "paged_evict", [&]() -> PyObject * {
    const at::Tensor *pages;
    const rib_paged_cache cache = cache_of(a[0], a[1], &pages);
    const c10::Device dev = pages->device();
    head_dim_64_128(cache);
    const int batch = size32(any_tensor(a[2], "lens", 1).size(0), "lens");
    if (batch < 1 || batch > cache.seqs) refuse("%d lengths for %d sequences", batch, cache.seqs);
    const int32_t *lens = vector(a[2], "lens", batch, dev);
    const int max_len = max_len_of(a[8], cache);
    const at::Tensor &scores = scores_of(a[3], "scores", batch, cache.nkv, max_len, dev);
    const at::Tensor &table = tensor(a[5], "new_table", 2, at::kInt, dev);
    const int keep = number(a[4], "keep"), sinks = number(a[6], "sinks"), recent = number(a[7], "recent");
    if (keep < 1 || sinks < 0 || recent < 0 || static_cast<int64_t>(sinks) + recent > keep)
      refuse("need keep >= 1, sinks >= 0, recent >= 0 and sinks + recent <= keep");
    if (keep > kMostRows) refuse("keep must be at most %d", kMostRows);
    const int most = std::min(keep, max_len);
    if (table.size(0) < batch || table.size(1) * cache.page_rows < most)
      refuse("new_table must name pages for %d rows of %d sequences, got %s", most, batch, shape_of(table).c_str());
    float *kept = nullptr;
    int64_t kept_s[2] = {0, 0};
    int kept_rows = 0;
    if (a[9] != Py_None) {
      const at::Tensor &t = scores_of(a[9], "new_scores", batch, cache.nkv, keep, dev);
      const auto x = span(scores), y = span(t);
      if (x.first < y.second && y.first < x.second) refuse("new_scores must not overlap scores");
      kept = written(t, "new_scores").data_ptr<float>();
      kept_s[0] = step(t, 0), kept_s[1] = step(t, 1);
      if (t.size(2) > kMostRows) refuse("new_scores must have at most %d entries a head", kMostRows);
      kept_rows = static_cast<int>(t.size(2));
    }
    const c10::cuda::CUDAGuard guard(dev);
    const at::Tensor rows = fresh({batch, cache.nkv, keep}, at::kInt, dev), new_lens = fresh({batch}, at::kInt, dev);
    checked(paged_evict_fn(&cache, table.const_data_ptr<int32_t>(), step(table, 0),
                           size32(table.size(1), "new_table"), lens, batch, max_len, scores.const_data_ptr<float>(),
                           step(scores, 0), step(scores, 1), keep, sinks, recent, rows.data_ptr<int32_t>(),
                           new_lens.data_ptr<int32_t>(), kept, kept_s[0], kept_s[1], kept_rows, stream_of(dev)),
            "paged_evict");
    PyObject *first = THPVariable_Wrap(rows), *second = THPVariable_Wrap(new_lens);
    PyObject *pair = first && second ? PyTuple_Pack(2, first, second) : nullptr;
    Py_XDECREF(first);
    Py_XDECREF(second);
    return pair;
  });
}

// bind(addresses of the entry points, in the order below)
PyObject *bind(PyObject *, PyObject *const *a, Py_ssize_t n) {
  if (n != 7) {
    PyErr_SetString(PyExc_TypeError, "bind takes 7 addresses");
    return nullptr;
  }
  void *p[7];
  for (int i = 0; i < 7; ++i) {
    p[i] = PyLong_AsVoidPtr(a[i]);
    if (!p[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "no address");
      return nullptr;
    }
  }
  status_string = reinterpret_cast<decltype(status_string)>(p[0]);
  last_error_string = reinterpret_cast<decltype(last_error_string)>(p[1]);
  rotary_apply = reinterpret_cast<decltype(rotary_apply)>(p[2]);
  paged_append_fn = reinterpret_cast<decltype(paged_append_fn)>(p[3]);
  decode_workspace_bytes = reinterpret_cast<decltype(decode_workspace_bytes)>(p[4]);
  decode_attention_fn = reinterpret_cast<decltype(decode_attention_fn)>(p[5]);
  paged_evict_fn = reinterpret_cast<decltype(paged_evict_fn)>(p[6]);
  Py_RETURN_NONE;
}

#define FAST(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(bind), FAST(rotary), FAST(paged_append), FAST(paged_decode_attention), FAST(paged_evict),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_paged_binding", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__paged_binding(void) { return PyModule_Create(&module); }
