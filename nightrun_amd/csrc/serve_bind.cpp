// nightrun_amd._serve: what nightrun_amd/serve.py calls. Takes torch tensors
// apart, checks types, shapes, layouts and devices (ValueError) and calls the C
// ABI (include/nrq_serve.h) on torch's current stream; returns its status. In C++
// because a decode step's calls last a few microseconds each, which is what a dozen
// attribute reads and a ctypes call take in Python.
#include <Python.h>

#include <ATen/ATen.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <initializer_list>
#include <stdexcept>
#include <string>

#include "../../include/nrq_serve.h"

namespace {

#define VALUE_CHECK(cond, ...)                                        \
  do {                                                                \
    if (!(cond)) throw std::invalid_argument(c10::str(__VA_ARGS__)); \
  } while (0)

const at::Tensor& tensor(PyObject* o, const char* what) {
  VALUE_CHECK(THPVariable_Check(o), what, ": expected a tensor");
  return THPVariable_Unpack(o);
}

void* on(const at::Tensor& t, const char* what, long dev) {
  VALUE_CHECK(t.is_cuda() && t.get_device() == dev, what, ": expected a tensor on cuda:", dev, ", got one on ",
              t.device().str());
  return t.data_ptr();
}

int kind(const at::Tensor& t, const char* what) {
  switch (t.scalar_type()) {
    case at::kFloat: return 0;
    case at::kHalf: return NRQ_F16;
    case at::kBFloat16: return NRQ_BF16;
    default: VALUE_CHECK(false, what, ": expected float32, float16 or bfloat16, got ", t.scalar_type());
  }
  return -1;
}

// `dims` dimensions, the last of them contiguous
void rows(const at::Tensor& t, const char* what, int dims) {
  VALUE_CHECK(t.dim() == dims && (t.size(dims - 1) < 2 || t.stride(dims - 1) == 1), what, ": expected ", dims,
              " dimensions, the last contiguous, got shape ", t.sizes(), ", strides ", t.strides());
}

// a contiguous tensor of this type and shape
void* exactly(const at::Tensor& t, const char* what, long dev, at::ScalarType type, at::IntArrayRef shape) {
  VALUE_CHECK(t.scalar_type() == type && t.sizes() == shape && t.is_contiguous(), what, ": expected a contiguous ",
              type, " tensor of shape ", shape, ", got ", t.scalar_type(), " ", t.sizes());
  return on(t, what, dev);
}

const int32_t* ints(const at::Tensor& t, const char* what, long dev, at::IntArrayRef shape) {
  return (const int32_t*)exactly(t, what, dev, at::kInt, shape);
}

void same(const at::Tensor& y, const at::Tensor& x, const char* what) {
  VALUE_CHECK(y.sizes() == x.sizes() && y.scalar_type() == x.scalar_type(), what, ": expected ", x.scalar_type(), " ",
              x.sizes(), ", got ", y.scalar_type(), " ", y.sizes());
}

const float* freqs(const at::Tensor& f, long dev) {
  VALUE_CHECK(f.scalar_type() == at::kFloat && f.dim() == 1 && f.is_contiguous(),
              "freqs: expected a contiguous float32 vector");
  return (const float*)on(f, "freqs", dev);
}

// pools [pages, KV heads, positions of a page, head_dim], any strides but the last
nrq_paged_kv paged(const at::Tensor& k, const at::Tensor& v, long dev) {
  rows(k, "k_pages", 4);
  rows(v, "v_pages", 4);
  VALUE_CHECK(k.scalar_type() == v.scalar_type() && k.sizes() == v.sizes() && k.strides() == v.strides(),
              "k_pages and v_pages differ in type, shape or strides");
  const int type = kind(k, "k_pages");
  VALUE_CHECK(type, "k_pages: expected float16 or bfloat16");
  for (int i = 0; i < 4; i++) VALUE_CHECK(k.size(i) <= INT32_MAX, "k_pages: dimension exceeds 2^31");
  return nrq_paged_kv{on(k, "k_pages", dev), on(v, "v_pages", dev), k.stride(0),         k.stride(1),
                      k.stride(2),           (int32_t)k.size(0),    (int32_t)k.size(2),  (int32_t)k.size(1),
                      (int32_t)k.size(3),    type};
}

nrq_page_table page_table(const at::Tensor& t, long dev) {
  VALUE_CHECK(t.scalar_type() == at::kInt, "table: expected int32, got ", t.scalar_type());
  rows(t, "table", 2);
  VALUE_CHECK(t.size(0) <= INT32_MAX && t.size(1) <= INT32_MAX, "table: dimension exceeds 2^31");
  return nrq_page_table{(const int32_t*)on(t, "table", dev), t.stride(0), (int32_t)t.size(0), (int32_t)t.size(1)};
}

// from torch's allocator, on the current stream: no other stream or captured graph gets the same memory
at::Tensor workspace(size_t n, const at::Tensor& like) { return at::empty({(int64_t)n}, like.options().dtype(at::kByte)); }

struct Mx {
  const void *q, *s;
  size_t rows, cols;
};
Mx mx(const at::Tensor& q, const at::Tensor& s, const char* what, long dev) {
  VALUE_CHECK(q.scalar_type() == at::kByte && s.scalar_type() == at::kByte && q.dim() == 2 && s.dim() == 2 &&
                  q.is_contiguous() && s.is_contiguous() && q.size(0) == s.size(0) && q.size(1) == 16 * s.size(1),
              what, ": expected contiguous uint8 [rows, cols / 2] and [rows, cols / 32], got ", q.sizes(), " and ",
              s.sizes());
  return Mx{on(q, what, dev), on(s, what, dev), (size_t)q.size(0), 2 * (size_t)q.size(1)};
}

double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}
long integer(PyObject* o) {
  const long v = PyLong_AsLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}
void* stream_of(PyObject* o) {
  void* p = PyLong_AsVoidPtr(o);
  if (!p && PyErr_Occurred()) throw python_error();
  return p;
}

// Each function: the positional arguments of serve.py's, then the device and its stream.
#define BIND(name, count)                                                                        \
  int do_##name(PyObject* const* a, long dev, void* stream);                                     \
  PyObject* py_##name(PyObject*, PyObject* const* a, Py_ssize_t n) {                             \
    HANDLE_TH_ERRORS                                                                             \
    if (n != count + 2) {                                                                        \
      PyErr_SetString(PyExc_TypeError, #name ": wrong number of arguments");                     \
      return nullptr;                                                                            \
    }                                                                                            \
    try {                                                                                        \
      return PyLong_FromLong(do_##name(a, integer(a[count]), stream_of(a[count + 1])));          \
    } catch (const std::invalid_argument& e) {                                                   \
      PyErr_SetString(PyExc_ValueError, e.what());                                               \
      return nullptr;                                                                            \
    }                                                                                            \
    END_HANDLE_TH_ERRORS                                                                         \
  }                                                                                              \
  int do_##name(PyObject* const* a, long dev, void* stream)

// y, x, pos, freqs, neox, scale
BIND(rope, 6) {
  const at::Tensor &y = tensor(a[0], "y"), &x = tensor(a[1], "x"), &pos = tensor(a[2], "pos"), &f = tensor(a[3], "freqs");
  rows(x, "x", 3);
  rows(y, "y", 3);
  same(y, x, "y");
  const int64_t s[4] = {x.stride(0), x.stride(1), y.stride(0), y.stride(1)};
  return nrq_dev_rope(on(y, "y", dev), on(x, "x", dev), kind(x, "x"), x.size(0), x.size(1), x.size(2), s,
                      ints(pos, "pos", dev, {x.size(0)}), freqs(f, dev), f.numel(), (int)integer(a[4]),
                      (float)number(a[5]), stream);
}

// y, q, k, v, pos, seq, freqs, k_pages, v_pages, table, neox, scale
BIND(rope_append, 12) {
  const at::Tensor &y = tensor(a[0], "y"), &q = tensor(a[1], "q"), &k = tensor(a[2], "k"), &v = tensor(a[3], "v"),
                   &pos = tensor(a[4], "pos"), &seq = tensor(a[5], "seq"), &f = tensor(a[6], "freqs"),
                   &kp = tensor(a[7], "k_pages"), &vp = tensor(a[8], "v_pages"), &tab = tensor(a[9], "table");
  rows(q, "q", 3);
  rows(k, "k", 3);
  rows(v, "v", 3);
  rows(y, "y", 3);
  same(y, q, "y");
  same(v, k, "v");
  const nrq_paged_kv kv = paged(kp, vp, dev);
  const nrq_page_table t = page_table(tab, dev);
  VALUE_CHECK(k.scalar_type() == q.scalar_type() && k.size(0) == q.size(0) && k.size(1) == kv.n_kv_heads &&
                  k.size(2) == q.size(2) && q.size(2) == kv.head_dim,
              "k: got ", k.scalar_type(), " ", k.sizes(), " with q ", q.scalar_type(), " ", q.sizes(), " and pages ",
              kp.sizes());
  const int64_t s[8] = {q.stride(0), q.stride(1), k.stride(0), k.stride(1), v.stride(0), v.stride(1), y.stride(0), y.stride(1)};
  return nrq_dev_rope_append(on(y, "y", dev), on(q, "q", dev), on(k, "k", dev), on(v, "v", dev), kind(q, "q"),
                             q.size(0), q.size(1), s, ints(pos, "pos", dev, {q.size(0)}),
                             ints(seq, "seq", dev, {q.size(0)}), freqs(f, dev), f.numel(), (int)integer(a[10]),
                             (float)number(a[11]), &kv, &t, stream);
}

// y, q, k_pages, v_pages, table, lens, scale, window, counts or None, lse or None
BIND(paged_attention, 10) {
  const at::Tensor &y = tensor(a[0], "y"), &q = tensor(a[1], "q"), &kp = tensor(a[2], "k_pages"),
                   &vp = tensor(a[3], "v_pages"), &tab = tensor(a[4], "table"), &lens = tensor(a[5], "lens");
  rows(q, "q", 4);
  rows(y, "y", 4);
  same(y, q, "y");
  const nrq_paged_kv kv = paged(kp, vp, dev);
  const nrq_page_table t = page_table(tab, dev);
  VALUE_CHECK(t.seqs == q.size(0) && kv.head_dim == q.size(3), "q ", q.sizes(), " does not go with pages ", kp.sizes(),
              " and table ", tab.sizes());
  const size_t n = q.size(1), heads = q.size(2);
  const int32_t* counts = a[8] == Py_None ? nullptr : ints(tensor(a[8], "counts"), "counts", dev, {q.size(0)});
  float* lse = nullptr;
  if (a[9] != Py_None)
    lse = (float*)exactly(tensor(a[9], "lse"), "lse", dev, at::kFloat, {q.size(0), q.size(1), q.size(2)});
  const int32_t* len = ints(lens, "lens", dev, {q.size(0)});
  const long window = integer(a[7]);
  VALUE_CHECK(window >= 0 && window <= INT32_MAX, "window: ", window);
  void *yp = on(y, "y", dev), *qp = on(q, "q", dev);
  size_t need;
  const int rc = nrq_paged_attention_workspace(q.size(0), n, heads, &kv, &need);
  if (rc) return rc;
  const at::Tensor ws = workspace(need, q);
  const int64_t s[6] = {q.stride(0), q.stride(1), q.stride(2), y.stride(0), y.stride(1), y.stride(2)};
  return nrq_dev_paged_attention(yp, qp, kind(q, "q"), n, heads, s, &kv, &t, len, counts, (float)number(a[6]),
                                 (int32_t)window, lse, ws.data_ptr(), need, stream);
}

// tokens, accepted, target, draft or None, drafted, uniforms, counts or None
BIND(verify_drafts, 7) {
  const at::Tensor &tokens = tensor(a[0], "tokens"), &acc = tensor(a[1], "accepted"), &target = tensor(a[2], "target"),
                   &drafted = tensor(a[4], "drafted"), &u = tensor(a[5], "uniforms");
  rows(target, "target", 3);
  const int64_t b = target.size(0), r = target.size(1), vocab = target.size(2);
  VALUE_CHECK(target.scalar_type() == at::kFloat && r > 0, "target: expected float32 [sequences, new tokens + 1, vocabulary]");
  const float* dp = nullptr;
  int64_t s[4] = {target.stride(0), target.stride(1), 0, 0};
  if (a[3] != Py_None) {
    const at::Tensor& draft = tensor(a[3], "draft");
    rows(draft, "draft", 3);
    VALUE_CHECK(draft.scalar_type() == at::kFloat && draft.size(0) == b && draft.size(1) == r - 1 && draft.size(2) == vocab,
                "draft: got ", draft.scalar_type(), " ", draft.sizes(), " with target ", target.sizes());
    dp = (const float*)on(draft, "draft", dev);
    s[2] = draft.stride(0), s[3] = draft.stride(1);
  }
  const int32_t* counts = a[6] == Py_None ? nullptr : ints(tensor(a[6], "counts"), "counts", dev, {b});
  int32_t* tp = (int32_t*)ints(tokens, "tokens", dev, {b, r});
  int32_t* ap = (int32_t*)ints(acc, "accepted", dev, {b});
  const int32_t* xp = ints(drafted, "drafted", dev, {b, r - 1});
  const float* up = (const float*)exactly(u, "uniforms", dev, at::kFloat, {b, r});
  const float* p = (const float*)on(target, "target", dev);
  size_t need;
  const int rc = nrq_verify_workspace(b, vocab, &need);
  if (rc) return rc;
  const at::Tensor ws = workspace(need, target);
  return nrq_dev_verify_drafts(tp, ap, p, dp, s, xp, up, counts, b, r - 1, vocab, ws.data_ptr(), need, stream);
}

// src, q, scales
BIND(quantize_mxfp4, 3) {
  const at::Tensor& src = tensor(a[0], "src");
  rows(src, "src", 2);
  const Mx m = mx(tensor(a[1], "q"), tensor(a[2], "scales"), "q, scales", dev);
  VALUE_CHECK((size_t)src.size(0) == m.rows && (size_t)src.size(1) == m.cols, "src: expected [", m.rows, ", ", m.cols,
              "], got ", src.sizes());
  return nrq_dev_quantize_mxfp4(on(src, "src", dev), kind(src, "src"), m.rows, m.cols, src.stride(0), (void*)m.q,
                                (void*)m.s, stream);
}

// q, scales, out
BIND(dequantize_mxfp4, 3) {
  const at::Tensor& out = tensor(a[2], "out");
  rows(out, "out", 2);
  const Mx m = mx(tensor(a[0], "q"), tensor(a[1], "scales"), "q, scales", dev);
  VALUE_CHECK((size_t)out.size(0) == m.rows && (size_t)out.size(1) == m.cols, "out: expected [", m.rows, ", ", m.cols,
              "], got ", out.sizes());
  return nrq_dev_dequantize_mxfp4(m.q, m.s, m.rows, m.cols, on(out, "out", dev), kind(out, "out"), out.stride(0), stream);
}

// y, w, w_scales, x, x_scales
BIND(matmul_mxfp4, 5) {
  const at::Tensor& y = tensor(a[0], "y");
  rows(y, "y", 2);
  const Mx w = mx(tensor(a[1], "w"), tensor(a[2], "w_scales"), "w, w_scales", dev);
  const Mx x = mx(tensor(a[3], "x"), tensor(a[4], "x_scales"), "x, x_scales", dev);
  VALUE_CHECK(x.cols == w.cols && (size_t)y.size(0) == x.rows && (size_t)y.size(1) == w.rows, "y ", y.sizes(),
              ": x is [", x.rows, ", ", x.cols, "], w [", w.rows, ", ", w.cols, "]");
  void* yp = on(y, "y", dev);
  const int yk = kind(y, "y");
  size_t need;
  const int rc = nrq_matmul_mxfp4_workspace(w.rows, w.cols, x.rows, &need);
  if (rc) return rc;
  at::Tensor ws;
  if (need) ws = workspace(need, y);
  return nrq_dev_matmul_mxfp4(yp, yk, y.stride(0), w.q, w.s, x.q, x.s, w.rows, w.cols, x.rows,
                              need ? ws.data_ptr() : nullptr, need, stream);
}

// y, w, w_scales, x
BIND(linear_mxfp4, 4) {
  const at::Tensor &y = tensor(a[0], "y"), &x = tensor(a[3], "x");
  rows(y, "y", 2);
  rows(x, "x", 2);
  const Mx w = mx(tensor(a[1], "w"), tensor(a[2], "w_scales"), "w, w_scales", dev);
  const size_t batch = x.size(0);
  VALUE_CHECK((size_t)x.size(1) == w.cols && y.size(0) == x.size(0) && (size_t)y.size(1) == w.rows, "y ", y.sizes(),
              ": x is ", x.sizes(), ", w [", w.rows, ", ", w.cols, "]");
  const int yk = kind(y, "y"), xk = kind(x, "x");
  void *yp = on(y, "y", dev), *xp = on(x, "x", dev);
  size_t need;
  const int rc = nrq_linear_mxfp4_workspace(w.rows, w.cols, batch, &need);
  if (rc) return rc;
  at::Tensor ws;
  if (need) ws = workspace(need, x);
  return nrq_dev_linear_mxfp4(yp, yk, y.stride(0), w.q, w.s, xp, xk, x.stride(0), w.rows, w.cols, batch,
                              need ? ws.data_ptr() : nullptr, need, stream);
}

#define METHOD(name) {#name, (PyCFunction)(void (*)(void))py_##name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(rope),           METHOD(rope_append),      METHOD(paged_attention),
                         METHOD(verify_drafts),  METHOD(quantize_mxfp4),   METHOD(dequantize_mxfp4),
                         METHOD(matmul_mxfp4),   METHOD(linear_mxfp4),     {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_serve", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__serve(void) { return PyModule_Create(&module); }
