// kv_face.cpp -- the Python face of include/vbq_kv.h on torch tensors, as a CPython extension.
//
// A decode step makes these calls once or twice a layer, and through ctypes a call's checks,
// allocations and argument conversion cost 16 us of host time where its kernel takes 9: here they
// are 6 (one sequence of 333 tokens, fp32).  The documented functions are in
// vibeblade_b200/kvcache.py; each passes its arguments on by position.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <map>
#include <stdexcept>
#include <string>
#include <tuple>

#include "vbq_kv.h"

namespace {

// A failed C call: its status, to be raised with the library's own error type and message.
struct Status {
  int code;
};

[[noreturn]] void fail(const char* name, const std::string& what) { throw std::runtime_error(std::string(name) + ": " + what); }
void done(int rc) {
  if (rc != VBQ_OK) throw Status{rc};
}

const at::Tensor& tensor(const char* name, PyObject* o) {
  if (!THPVariable_Check(o)) fail(name, "tensors must be CUDA tensors (the KV cache lives on the GPU only)");
  return THPVariable_Unpack(o);
}
void on(const char* name, const at::Tensor& first, const at::Tensor& t) {
  if (!t.is_cuda() || !first.is_cuda()) fail(name, "tensors must be CUDA tensors (the KV cache lives on the GPU only)");
  if (t.device() != first.device())
    fail(name, "tensors are on different devices (" + t.device().str() + " and " + first.device().str() + ")");
}
long integer(const char* name, const char* what, PyObject* o) {
  const long v = PyLong_AsLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    fail(name, std::string(what) + " must be an integer");
  }
  return v;
}
int32_t int32(const char* name, const char* what, PyObject* o) {
  const long v = integer(name, what, o);
  if (v < INT32_MIN || v > INT32_MAX) fail(name, std::string(what) + " is out of range");
  return (int32_t)v;
}
int32_t dtype_of(const char* name, const char* what, const at::Tensor& t) {
  if (t.scalar_type() == at::kFloat) return VBQ_DTYPE_F32;
  if (t.scalar_type() == at::kBFloat16) return VBQ_DTYPE_BF16;
  fail(name, std::string(what) + " must be float32 or bfloat16");
}
void ints(const char* name, const char* what, const at::Tensor& t, int dim) {
  if (t.scalar_type() != at::kInt || t.dim() != dim || !t.is_contiguous())
    fail(name, std::string(what) + " must be a contiguous int32 tensor of " + std::to_string(dim) +
                   (dim > 1 ? " dimensions" : " dimension"));
}
const int32_t* i32(const at::Tensor& t) { return t.const_data_ptr<int32_t>(); }

struct Pool {
  int64_t pages;
  int32_t layers, heads, page, dim;
  void* codes;
  float* scales;
};
Pool pool_of(const char* name, const at::Tensor& codes, const at::Tensor& scales) {
  if (codes.scalar_type() != at::kChar || codes.dim() != 6 || codes.size(2) != 2 || !codes.is_contiguous())
    fail(name, "codes must be contiguous int8 [pages, layers, 2, kv_heads, page, dim]");
  if (scales.scalar_type() != at::kFloat || scales.sizes() != codes.sizes().slice(0, 4) || !scales.is_contiguous())
    fail(name, "scales must be contiguous float32 [pages, layers, 2, kv_heads], as codes");
  for (int i = 1; i < 6; ++i)
    if (codes.size(i) > INT32_MAX) fail(name, "codes are too large");
  return {codes.size(0), (int32_t)codes.size(1), (int32_t)codes.size(3), (int32_t)codes.size(4), (int32_t)codes.size(5),
          codes.data_ptr(), scales.data_ptr<float>()};
}
struct Batch {
  const int32_t *tables, *lens, *q_start;
  int32_t seqs, max_pages;
};
Batch batch_of(const char* name, const at::Tensor& tables, const at::Tensor& lens, const at::Tensor& q_start) {
  ints(name, "tables", tables, 2);
  ints(name, "lens", lens, 1);
  ints(name, "q_start", q_start, 1);
  const int64_t s = tables.size(0);
  if (s > INT32_MAX - 1 || tables.size(1) > INT32_MAX) fail(name, "tables are too large");
  if (lens.size(0) != s || q_start.size(0) != s + 1)
    fail(name, "lens and q_start must have " + std::to_string(s) + " and " + std::to_string(s + 1) + " entries for " +
                   std::to_string(s) + " table rows");
  return {i32(tables), i32(lens), i32(q_start), (int32_t)s, (int32_t)tables.size(1)};
}
// a [rows, width] tensor with unit column stride; width < 0: any
void rows_of(const char* name, const char* what, const at::Tensor& t, int64_t width) {
  if (t.dim() != 2 || (t.stride(1) != 1 && t.size(1) > 1) || (width >= 0 && t.size(1) != width))
    fail(name, std::string(what) + " must be [rows, " + (width >= 0 ? std::to_string(width) : "heads * dim") +
                   "] with its columns adjacent");
}
// elements between rows; of a single row, whose stride means nothing, its width
int64_t row_stride(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

void* stream_of(const at::Tensor& t) { return at::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

// Workspaces by (device, stream, kind, layout, size), of which the first `zero` bytes are zeroed once; a call
// leaves zero what has to be.  One that was handed out is never replaced or freed, because a captured graph
// may hold its address (and never destroyed: CUDA may be gone by then).  Sizes below 1 MB, which go by a
// call's rows, are rounded up to powers of two, so that there are few.
//
// A call that is captured before its stream has the workspace gets one of the graph's own: memory of the
// graph's pool, whose zeroing is recorded and so runs at each replay.  The capture's later calls share it.
struct Space {
  void* p;
  size_t n;
};
Space workspace(const at::Tensor& like, void* stream, int kind, int64_t layout, size_t need, size_t zero) {
  using Key = std::tuple<int64_t, void*, int, int64_t, size_t>;
  struct Captured {
    unsigned long long capture;
    at::Tensor t;
  };
  static auto& all = *new std::map<Key, at::Tensor>();
  static auto& captured = *new std::map<Key, Captured>();
  size_t size = need;
  if (need < (1 << 20))
    for (size = 256; size < need;) size *= 2;
  const Key key{like.get_device(), stream, kind, layout, size};
  const auto known = all.find(key);
  if (known != all.end()) return {known->second.data_ptr(), size};
  auto made = [&]() {
    const at::Tensor t = at::empty({(int64_t)size}, like.options().dtype(at::kByte));
    t.narrow(0, 0, (int64_t)std::min(size, zero)).zero_();
    return t;
  };
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long capture = 0;
  C10_CUDA_CHECK(cudaStreamGetCaptureInfo(static_cast<cudaStream_t>(stream), &status, &capture));
  if (status == cudaStreamCaptureStatusNone) {
    const at::Tensor t = made();
    all.emplace(key, t);
    return {t.data_ptr(), size};
  }
  Captured& c = captured[key];
  if (!c.t.defined() || c.capture != capture) c = {capture, made()};
  return {c.t.data_ptr(), size};
}

PyObject* wrap(const at::Tensor& t) { return THPVariable_Wrap(t); }
template <typename... T> PyObject* tuple_of(const T&... t) {
  PyObject* r = PyTuple_New(sizeof...(T));
  Py_ssize_t i = 0;
  ((PyTuple_SET_ITEM(r, i++, t)), ...);
  return r;
}

// ---- the calls -------------------------------------------------------------------------

PyObject* append(PyObject* const* a) {
  const char* name = "kv_append";
  const at::Tensor &k = tensor(name, a[0]), &v = tensor(name, a[1]), &codes = tensor(name, a[2]), &scales = tensor(name, a[3]),
                   &tables = tensor(name, a[4]), &lens = tensor(name, a[5]), &q_start = tensor(name, a[6]);
  for (const at::Tensor* t : {&k, &v, &scales, &tables, &lens, &q_start}) on(name, codes, *t);
  const Pool p = pool_of(name, codes, scales);
  const Batch b = batch_of(name, tables, lens, q_start);
  const int32_t d = dtype_of(name, "k", k);
  rows_of(name, "k", k, (int64_t)p.heads * p.dim);
  rows_of(name, "v", v, (int64_t)p.heads * p.dim);
  if (v.scalar_type() != k.scalar_type() || v.size(0) != k.size(0)) fail(name, "k and v must have the same rows and type");
  const int32_t layer = int32(name, "layer", a[7]);
  const c10::cuda::CUDAGuard guard(codes.device());
  done(vbq_kv_append(k.const_data_ptr(), row_stride(k), v.const_data_ptr(), row_stride(v), d, k.size(0), p.codes, p.scales,
                     p.pages, p.layers, layer, p.heads, p.page, p.dim, b.tables, b.max_pages, b.lens, b.q_start, b.seqs,
                     stream_of(codes)));
  Py_RETURN_NONE;
}

PyObject* read(PyObject* const* a) {
  const char* name = "kv_read";
  const at::Tensor &codes = tensor(name, a[0]), &scales = tensor(name, a[1]), &tables = tensor(name, a[2]),
                   &lens = tensor(name, a[3]), &q_start = tensor(name, a[4]);
  for (const at::Tensor* t : {&scales, &tables, &lens, &q_start}) on(name, codes, *t);
  const Pool p = pool_of(name, codes, scales);
  const Batch b = batch_of(name, tables, lens, q_start);
  const long rows = integer(name, "rows", a[5]);
  const int32_t layer = int32(name, "layer", a[6]);
  const bool bf16 = a[7] == Py_True;
  if (rows < 0) fail(name, "rows must not be negative");
  const c10::cuda::CUDAGuard guard(codes.device());
  const auto opt = scales.options().dtype(bf16 ? at::kBFloat16 : at::kFloat);
  const at::Tensor k = at::empty({rows, (int64_t)p.heads * p.dim}, opt), v = at::empty({rows, (int64_t)p.heads * p.dim}, opt);
  done(vbq_kv_read(p.codes, p.scales, p.pages, p.layers, layer, p.heads, p.page, p.dim, b.tables, b.max_pages, b.lens,
                   b.q_start, b.seqs, rows, k.data_ptr(), v.data_ptr(), bf16 ? VBQ_DTYPE_BF16 : VBQ_DTYPE_F32,
                   stream_of(codes)));
  return tuple_of(wrap(k), wrap(v));
}

PyObject* attention(PyObject* const* a) {
  const char* name = "kv_attention";
  const at::Tensor &q = tensor(name, a[0]), &codes = tensor(name, a[1]), &scales = tensor(name, a[2]),
                   &tables = tensor(name, a[3]), &lens = tensor(name, a[4]), &q_start = tensor(name, a[5]);
  for (const at::Tensor* t : {&codes, &scales, &tables, &lens, &q_start}) on(name, q, *t);
  const Pool p = pool_of(name, codes, scales);
  const Batch b = batch_of(name, tables, lens, q_start);
  const int32_t d = dtype_of(name, "q", q);
  rows_of(name, "q", q, -1);
  const int64_t rows = q.size(0), width = q.size(1), per = (int64_t)p.heads * p.dim;
  if (width == 0 || per == 0 || width % per != 0)
    fail(name, "q's width " + std::to_string(width) + " is not a whole number of heads for each of " +
                   std::to_string(p.heads) + " KV heads of " + std::to_string(p.dim));
  const int64_t heads = width / p.dim;
  if (heads > INT32_MAX) fail(name, "too many heads");
  const int32_t layer = int32(name, "layer", a[6]), window = int32(name, "window", a[8]), max_new = int32(name, "max_new", a[9]);
  float scale = 1.0f / std::sqrt((float)p.dim);
  if (a[7] != Py_None) {
    const double s = PyFloat_AsDouble(a[7]);
    if (s == -1.0 && PyErr_Occurred()) {
      PyErr_Clear();
      fail(name, "scale must be a number");
    }
    scale = (float)s;
  }
  const c10::cuda::CUDAGuard guard(q.device());
  at::Tensor out;
  if (a[10] == Py_None) {
    out = at::empty({rows, width}, q.options());
  } else {
    out = tensor(name, a[10]);
    on(name, q, out);
    rows_of(name, "out", out, width);
    if (out.scalar_type() != q.scalar_type() || out.size(0) != rows) fail(name, "out must have q's shape and type");
  }
  const bool with_lse = a[11] == Py_True;
  at::Tensor lse;
  if (with_lse) lse = at::empty({rows, heads}, scales.options());
  size_t need = 0;
  done(vbq_kv_attention_workspace_bytes((int32_t)heads, p.heads, p.dim, d, &need));
  void* st = stream_of(q);
  const Space ws = workspace(q, st, 0, p.dim, need, VBQ_KV_ATTENTION_ZERO_BYTES);  // its layout goes by dim
  done(vbq_kv_attention(q.const_data_ptr(), row_stride(q), out.data_ptr(), row_stride(out),
                        with_lse ? lse.data_ptr<float>() : nullptr, d, rows, (int32_t)heads, p.codes, p.scales, p.pages,
                        p.layers, layer, p.heads, p.page, p.dim, b.tables, b.max_pages, b.lens, b.q_start, b.seqs, scale,
                        window, max_new, ws.p, ws.n, st));
  return with_lse ? tuple_of(wrap(out), wrap(lse)) : wrap(out);
}

struct Rows {
  int64_t pages;
  int32_t rows, width;
};
Rows sequences(const char* name, const at::Tensor& refs, const at::Tensor& tables, const at::Tensor& lens) {
  on(name, refs, tables);
  on(name, refs, lens);
  ints(name, "refs", refs, 1);
  ints(name, "tables", tables, 2);
  ints(name, "lens", lens, 1);
  if (lens.size(0) != tables.size(0)) fail(name, "lens must have an entry for each table row");
  if (tables.size(0) > INT32_MAX || tables.size(1) > INT32_MAX) fail(name, "tables are too large");
  return {refs.size(0), (int32_t)tables.size(0), (int32_t)tables.size(1)};
}
Space pages_space(const at::Tensor& refs, void* st, int64_t pages, int32_t rows) {
  size_t need = 0;
  done(vbq_kv_pages_workspace_bytes(pages, rows, &need));
  return workspace(refs, st, 1, pages, need, need);  // what stays zero is laid out by `pages`
}

PyObject* reserve(PyObject* const* a) {
  const char* name = "kv_reserve";
  const at::Tensor &refs = tensor(name, a[0]), &tables = tensor(name, a[1]), &lens = tensor(name, a[2]),
                   &more = tensor(name, a[3]);
  const Rows r = sequences(name, refs, tables, lens);
  on(name, refs, more);
  ints(name, "new_tokens", more, 1);
  if (more.size(0) != r.rows) fail(name, "new_tokens must have an entry for each table row");
  const int32_t page = int32(name, "page", a[4]);
  const c10::cuda::CUDAGuard guard(refs.device());
  const auto opt = refs.options();
  const at::Tensor refs_out = at::empty({r.pages}, opt), tables_out = at::empty({r.rows, r.width}, opt),
                   lens_out = at::empty({r.rows}, opt), missing = at::empty({1}, opt);
  void* st = stream_of(refs);
  const Space ws = pages_space(refs, st, r.pages, r.rows);
  done(vbq_kv_reserve(i32(refs), i32(tables), i32(lens), i32(more), r.pages, page, r.rows, r.width,
                      refs_out.data_ptr<int32_t>(), tables_out.data_ptr<int32_t>(), lens_out.data_ptr<int32_t>(),
                      missing.data_ptr<int32_t>(), ws.p, ws.n, st));
  return tuple_of(wrap(refs_out), wrap(tables_out), wrap(lens_out), wrap(missing));
}

PyObject* fork(PyObject* const* a) {
  const char* name = "kv_fork";
  const at::Tensor &codes = tensor(name, a[0]), &scales = tensor(name, a[1]), &refs = tensor(name, a[2]),
                   &tables = tensor(name, a[3]), &lens = tensor(name, a[4]), &parents = tensor(name, a[5]);
  for (const at::Tensor* t : {&scales, &refs, &parents}) on(name, codes, *t);
  const Pool p = pool_of(name, codes, scales);
  const Rows r = sequences(name, refs, tables, lens);
  ints(name, "parents", parents, 1);
  if (r.pages != p.pages) fail(name, "refs must have an entry for each page");
  if (parents.size(0) > INT32_MAX) fail(name, "too many rows");
  const int32_t rows = (int32_t)parents.size(0);
  const int64_t blocks = (int64_t)p.layers * 2 * p.heads;
  const c10::cuda::CUDAGuard guard(codes.device());
  const auto opt = refs.options();
  const at::Tensor refs_out = at::empty({r.pages}, opt), tables_out = at::empty({rows, r.width}, opt),
                   lens_out = at::empty({rows}, opt), missing = at::empty({1}, opt);
  void* st = stream_of(refs);
  const Space ws = pages_space(refs, st, r.pages, r.rows > rows ? r.rows : rows);
  done(vbq_kv_fork(p.codes, p.scales, p.pages, blocks * p.page * p.dim, blocks, p.page, i32(refs), i32(tables), i32(lens),
                   r.rows, r.width, i32(parents), rows, refs_out.data_ptr<int32_t>(), tables_out.data_ptr<int32_t>(),
                   lens_out.data_ptr<int32_t>(), missing.data_ptr<int32_t>(), ws.p, ws.n, st));
  return tuple_of(wrap(refs_out), wrap(tables_out), wrap(lens_out), wrap(missing));
}

PyObject* compact(PyObject* const* a) {
  const char* name = "kv_compact";
  const at::Tensor &codes = tensor(name, a[0]), &scales = tensor(name, a[1]), &refs = tensor(name, a[2]),
                   &tables = tensor(name, a[3]), &lens = tensor(name, a[4]);
  for (const at::Tensor* t : {&scales, &refs}) on(name, codes, *t);
  const Pool p = pool_of(name, codes, scales);
  const Rows r = sequences(name, refs, tables, lens);
  if (r.pages != p.pages) fail(name, "refs must have an entry for each page");
  const int64_t blocks = (int64_t)p.layers * 2 * p.heads;
  const c10::cuda::CUDAGuard guard(codes.device());
  const auto opt = refs.options();
  const at::Tensor refs_out = at::empty({r.pages}, opt), tables_out = at::empty({r.rows, r.width}, opt),
                   live = at::empty({1}, opt);
  void* st = stream_of(refs);
  const Space ws = pages_space(refs, st, r.pages, r.rows);
  done(vbq_kv_compact(p.codes, p.scales, p.pages, blocks * p.page * p.dim, blocks, p.page, i32(refs), i32(tables), i32(lens),
                      r.rows, r.width, refs_out.data_ptr<int32_t>(), tables_out.data_ptr<int32_t>(), live.data_ptr<int32_t>(),
                      ws.p, ws.n, st));
  return tuple_of(wrap(refs_out), wrap(tables_out), wrap(live));
}

PyObject* logprobs(PyObject* const* a) {
  const char* name = "token_logprobs";
  const at::Tensor& x = tensor(name, a[0]);
  on(name, x, x);
  const int32_t d = dtype_of(name, "logits", x);
  if (x.dim() != 2 || (x.stride(1) != 1 && x.size(1) > 1)) fail(name, "logits must be [rows, vocab] with its columns adjacent");
  const int64_t rows = x.size(0), vocab = x.size(1);
  const int32_t top = int32(name, "top", a[2]);
  const int32_t* tok = nullptr;
  if (a[1] != Py_None) {
    const at::Tensor& t = tensor(name, a[1]);
    on(name, x, t);
    ints(name, "tokens", t, 1);
    if (t.size(0) != rows) fail(name, "tokens must have an entry for each row of logits");
    tok = i32(t);
  }
  size_t need = 0;
  const c10::cuda::CUDAGuard guard(x.device());
  done(vbq_token_logprobs_workspace_bytes(rows, vocab, top, &need));
  const auto f = x.options().dtype(at::kFloat);
  at::Tensor lp;
  if (tok) lp = at::empty({rows}, f);
  const at::Tensor en = at::empty({rows}, f), tl = at::empty({rows, top}, f), tt = at::empty({rows, top}, f.dtype(at::kInt));
  void* st = stream_of(x);
  const Space ws = need ? workspace(x, st, 2, 0, need, need) : Space{nullptr, 0};
  done(vbq_token_logprobs(x.const_data_ptr(), row_stride(x), d, rows, vocab, tok, top, tok ? lp.data_ptr<float>() : nullptr,
                          en.data_ptr<float>(), tl.data_ptr<float>(), tt.data_ptr<int32_t>(), ws.p, ws.n, st));
  PyObject* first = tok ? wrap(lp) : (Py_INCREF(Py_None), Py_None);
  return tuple_of(first, wrap(en), wrap(tl), wrap(tt));
}

// No C++ exception leaves an entry: each becomes a Python one.
template <PyObject* (*F)(PyObject* const*), Py_ssize_t N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", N, n);
    return nullptr;
  }
  try {
    return F(args);
  } catch (const Status& s) {
    PyObject* m = PyImport_ImportModule("vibeblade_b200._lib");
    PyObject* type = m ? PyObject_GetAttrString(m, "VbqError") : nullptr;
    PyObject* e = type ? PyObject_CallFunction(type, "is", s.code, vbq_last_error()) : nullptr;
    if (e) PyErr_SetObject(type, e);
    Py_XDECREF(e);
    Py_XDECREF(type);
    Py_XDECREF(m);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

#define VBQ_ENTRY(f, n) \
  { #f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<f, n>)), METH_FASTCALL, nullptr }
PyMethodDef kMethods[] = {VBQ_ENTRY(append, 8),  VBQ_ENTRY(read, 8),    VBQ_ENTRY(attention, 12), VBQ_ENTRY(reserve, 5),
                          VBQ_ENTRY(fork, 6),    VBQ_ENTRY(compact, 5), VBQ_ENTRY(logprobs, 3),   {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_kvface", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__kvface(void) { return PyModule_Create(&kModule); }
