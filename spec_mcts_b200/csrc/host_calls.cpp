// The host side of a repeated matmul_q40 or linear_q40 call, and of the calls of a paged cache: checks, the output tensor and the launch in one
// native call.
//
// Through Python's attributes and ctypes a call of matmul_q40 takes 10.7 us of the host and one of linear_q40 13.7, where a kernel of one
// row takes 5.5 (4096 x 4096); here they take 3.7 and 4.1.  Nothing is decided here that kernels.py does not decide: a call that is not the plain repeated one (another
// stream, a written or replaced weight, other types, sizes or devices, a subclass of tensor) is handed back as None, and goes
// the way of a first call, which also words the errors.
#include <Python.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ops/empty.h>

#include <algorithm>
#include <initializer_list>

namespace {

using MatmulTiled = int (*)(const void*, void*, int64_t, const void*, int64_t, int, int, int, int, void*, int, void*);
using GemmNk = int (*)(const void*, int64_t, const void*, const void*, void*, int64_t, int, int, int, int, void*, size_t, void*);
MatmulTiled matmul_tiled = nullptr;
GemmNk gemm_nk = nullptr;

const at::Tensor* tensor(PyObject* o) {
  return THPVariable_CheckExact(o) || Py_TYPE(o) == reinterpret_cast<PyTypeObject*>(ParameterClass) ? &THPVariable_Unpack(o) : nullptr;
}
bool on(const at::Tensor& t, int dev) { return t.is_cuda() && t.get_device() == dev; }
// The two whole numbers of a tuple
bool two(PyObject* t, int64_t& a, int64_t& b) {
  if (!PyTuple_Check(t) || PyTuple_GET_SIZE(t) != 2 || !PyLong_Check(PyTuple_GET_ITEM(t, 0)) || !PyLong_Check(PyTuple_GET_ITEM(t, 1))) return false;
  a = PyLong_AsLongLong(PyTuple_GET_ITEM(t, 0));
  b = PyLong_AsLongLong(PyTuple_GET_ITEM(t, 1));
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}
int64_t version(const at::Tensor& t) { return t.is_inference() ? -1 : (int64_t)t._version(); }
// kernels._workspaces[("gemm", device, stream)] or an undefined tensor
at::Tensor workspace(PyObject* dict, int dev, PyObject* stream) {
  static PyObject* kind = PyUnicode_InternFromString("gemm");
  PyObject* key = Py_BuildValue("(OiO)", kind, dev, stream);
  if (!key) {
    PyErr_Clear();
    return {};
  }
  PyObject* t = PyDict_GetItem(dict, key);
  Py_DECREF(key);
  return t && THPVariable_Check(t) ? THPVariable_Unpack(t) : at::Tensor();
}
// Other Python threads run meanwhile: an allocation may wait for the device, a launch for room in its queue (behind a host function that
// needs the interpreter, say).  What is used in there is owned here
struct WithoutInterpreter {
  PyThreadState* state = PyEval_SaveThread();
  ~WithoutInterpreter() { PyEval_RestoreThread(state); }
};
at::Tensor output(int64_t rows, int64_t cols, int dev) {
  return at::empty({rows, cols}, at::TensorOptions().dtype(at::kHalf).device(at::kCUDA, (c10::DeviceIndex)dev));
}

// matmul(a, b_w, b_s, b_shape, entry of kernels._relayout_cache, kernels._cluster_sizes, kernels._workspaces) -> C or None
PyObject* matmul(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7 || !matmul_tiled) Py_RETURN_NONE;
  const at::Tensor *a = tensor(args[0]), *w = tensor(args[1]), *s = tensor(args[2]);
  PyObject* e = args[4];
  if (!a || !w || !s || !a->is_cuda() || !PyTuple_Check(e) || PyTuple_GET_SIZE(e) != 8) Py_RETURN_NONE;
  const int dev = c10::cuda::current_device();
  if (!on(*a, dev) || !on(*w, dev) || !on(*s, dev)) Py_RETURN_NONE;
  int64_t K, N, k2, n2, vw, vs, pw, ps;
  // the copy is of these tensors, as they are
  if (PyWeakref_GetObject(PyTuple_GET_ITEM(e, 0)) != args[1] || PyWeakref_GetObject(PyTuple_GET_ITEM(e, 1)) != args[2] ||
      !two(PyTuple_GET_ITEM(e, 2), vw, vs) || !two(PyTuple_GET_ITEM(e, 3), K, N) || !two(args[3], k2, n2) || k2 != K || n2 != N ||
      !two(PyTuple_GET_ITEM(e, 4), pw, ps) || vw != version(*w) || vs != version(*s) || pw != (int64_t)(uintptr_t)w->data_ptr() ||
      ps != (int64_t)(uintptr_t)s->data_ptr() || !THPVariable_Check(PyTuple_GET_ITEM(e, 5)))
    Py_RETURN_NONE;
  if (a->scalar_type() != at::kHalf || s->scalar_type() != at::kHalf || a->dim() != 2 || a->size(1) != K || !a->is_contiguous() ||
      !w->is_contiguous() || !s->is_contiguous() || w->numel() * 2 != K * N || s->numel() * 64 != K * N)
    Py_RETURN_NONE;
  const int64_t M = a->size(0);
  if (M < 1 || M > INT32_MAX || (uintptr_t)a->data_ptr() % 16 || (M <= 16 ? K % 16 != 0 || K < 64 : K % 64 != 0)) Py_RETURN_NONE;
  const auto stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream();
  PyObject* st = PyLong_FromVoidPtr(stream);
  if (!st) return nullptr;
  const int known = PySet_Contains(PyTuple_GET_ITEM(e, 7), st);
  const at::Tensor page = known == 1 && M > 8 ? workspace(args[6], dev, st) : at::Tensor();
  Py_DECREF(st);
  if (known != 1) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  int cluster = 16;
  PyObject* d = PyLong_FromLong(dev);
  PyObject* sizes = d ? PyDict_GetItem(args[5], d) : nullptr;
  Py_XDECREF(d);
  if (sizes && PyTuple_Check(sizes) && PyTuple_GET_SIZE(sizes)) cluster = (int)PyLong_AsLong(PyTuple_GET_ITEM(sizes, 0));
  else if (M <= 8) Py_RETURN_NONE;
  if (M > 8 && !page.defined()) Py_RETURN_NONE;
  const at::Tensor copy = THPVariable_Unpack(PyTuple_GET_ITEM(e, 5)), x = *a;
  at::Tensor c;
  int rc;
  {
    WithoutInterpreter w;
    c = output(M, N, dev);
    rc = matmul_tiled(copy.data_ptr(), c.data_ptr(), N, x.data_ptr(), K, (int)M, (int)N, (int)K, cluster,
                      page.defined() ? (char*)page.data_ptr() + 4092 : nullptr, 1, stream);
  }
  if (rc != 0) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(c));
  END_HANDLE_TH_ERRORS
}

// linear(x, w_q, w_s, w_shape, group, kernels._workspaces) -> y or None
PyObject* linear(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6 || !gemm_nk) Py_RETURN_NONE;
  const at::Tensor *x = tensor(args[0]), *w = tensor(args[1]), *s = tensor(args[2]);
  if (!x || !w || !s || !x->is_cuda() || !PyLong_Check(args[4])) Py_RETURN_NONE;
  const int dev = c10::cuda::current_device();
  int64_t N, K;
  if (!on(*x, dev) || !on(*w, dev) || !on(*s, dev) || !two(args[3], N, K) || x->dim() != 2 || x->size(1) != K || K < 1 || N < 1 ||
      K > INT32_MAX || N > INT32_MAX || x->scalar_type() != at::kHalf || !x->is_contiguous() || !w->is_contiguous() || !s->is_contiguous())
    Py_RETURN_NONE;
  const int64_t M = x->size(0);
  if (M < 1 || M > INT32_MAX || (M > 32 && (uintptr_t)x->data_ptr() % 16 == 8)) Py_RETURN_NONE;      // those are copied first
  const auto stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream();
  PyObject* st = PyLong_FromVoidPtr(stream);
  if (!st) return nullptr;
  const at::Tensor ws = workspace(args[5], dev, st);
  Py_DECREF(st);
  if (!ws.defined() || ws.numel() > 64 << 20) Py_RETURN_NONE;        // a large one is noted where a capture uses it
  const int group = (int)PyLong_AsLong(args[4]);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  const at::Tensor in = *x, codes = *w, scales = *s;
  at::Tensor y;
  int rc;
  {
    WithoutInterpreter w;
    y = output(M, N, dev);
    rc = gemm_nk(in.data_ptr(), K, codes.data_ptr(), scales.data_ptr(), y.data_ptr(), N, (int)M, (int)N, (int)K, group, ws.data_ptr(), (size_t)ws.numel(), stream);
  }
  if (rc != 0) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// ---- the paged cache: an append of one token takes 5.3 us of the host this way, 23.2 through Python, attention over 512 keys 5.9 and 23.2
using AttnPages = int (*)(const void*, int, int64_t, const int32_t*, const void*, int64_t, const void*, const void*, const float*, const float*, int, void*,
                          int64_t, int, int, int, int, int, int, int, int, void*, size_t, void*);
using AttnPagesBytes = size_t (*)(int, int, int, int, int, int);
using PageAppend = int (*)(const void*, int, int64_t, int, const int32_t*, const int32_t*, const void*, int64_t, void*, const void*, int64_t, const void*,
                           int64_t, const void*, const void*, int, void*, void*, float*, float*, int, int64_t, int, int, int, int, int, int, void*);
using CausalWindow = int (*)(const void*, int64_t, const void*, int64_t, const void*, int64_t, void*, int64_t, int, int, int, int, int, int, int, void*,
                             size_t, int*, void*);
using CausalWindowBytes = size_t (*)(int, int, int, int, int, int, int);
using AttnPagesScores = int (*)(const void*, int, int64_t, const int32_t*, const void*, int64_t, const void*, const void*, const float*, const float*, int, void*,
                                int64_t, int, int, int, int, int, int, int, int, float, const float*, void*, size_t, void*);
using CausalScores = int (*)(const void*, int64_t, const void*, int64_t, const void*, int64_t, void*, int64_t, int, int, int, int, int, int, int, float, const float*,
                             const int32_t*, int, const int32_t*, int, int, void*, size_t, int*, void*);
using PageFork = int (*)(const int32_t*, int64_t, const int32_t*, const int32_t*, const int32_t*, int32_t*, int64_t, int32_t*, int32_t*, int, int, int, int, void*,
                         size_t, void*);
using PageExtend = int (*)(const int32_t*, int64_t, const int32_t*, const int32_t*, const int32_t*, int32_t*, int64_t, int32_t*, int32_t*, int, int, int, int, void*, void*, float*,
                           float*, int, int64_t, int, void*, size_t, void*);
using PageCompact = int (*)(const int32_t*, int64_t, const int32_t*, const int32_t*, int32_t*, int64_t, int32_t*, int32_t*, int, int, int, int, void*, void*, float*, float*, int,
                            int64_t, int, void*, size_t, void*);
AttnPagesScores attn_pages_scores_fn = nullptr;
CausalScores causal_scores_fn = nullptr;
CausalWindowBytes causal_scores_bytes = nullptr;
PageFork page_fork_fn = nullptr;
PageExtend page_extend_fn = nullptr;
PageCompact page_compact_fn = nullptr;
size_t (*page_fork_bytes)(int, int, int) = nullptr;
size_t (*page_extend_bytes)(int, int, int) = nullptr;
size_t (*page_compact_bytes)(int, int) = nullptr;
AttnPages attn_pages_fn = nullptr;
AttnPagesBytes attn_pages_bytes = nullptr;
PageAppend page_append_fn = nullptr;
CausalWindow causal_window_fn = nullptr;
CausalWindowBytes causal_window_bytes = nullptr;

constexpr int64_t HEAD = 128, MOST = 1 << 30, MOST_PAGE = 1 << 29;

// A whole number of up to MOST; None is `none`
bool whole(PyObject* o, int64_t none, int64_t& x) {
  if (o == Py_None) {
    x = none;
    return true;
  }
  if (!PyLong_CheckExact(o)) return false;
  int over = 0;
  x = PyLong_AsLongLongAndOverflow(o, &over);
  if (over > 0 || x > MOST) x = MOST;
  return over >= 0;
}
// `t` on the device, of a type
bool is(const at::Tensor* t, int dev, at::ScalarType type) { return t && on(*t, dev) && t->scalar_type() == type; }
// ... rows of heads as the kernels read them, and the stride of the rows
bool rows_of(const at::Tensor* t, int dev, int64_t& ld) {
  if (!is(t, dev, at::kHalf) || t->dim() != 3 || t->size(2) != HEAD || t->stride(2) != 1 || t->size(0) < 1 || t->size(0) > INT32_MAX || t->size(1) < 1 ||
      t->size(1) > INT32_MAX / HEAD || (t->size(1) > 1 && t->stride(1) != HEAD) || (uintptr_t)t->data_ptr() % 16)
    return false;
  ld = t->size(0) > 1 ? t->stride(0) : t->size(1) * HEAD;
  return ld % 8 == 0 && ld >= t->size(1) * HEAD;
}
bool vector_of(const at::Tensor* t, int dev, at::ScalarType type, int64_t n) { return is(t, dev, type) && t->dim() == 1 && t->size(0) == n && t->is_contiguous(); }
struct Table { const void* ids; int bytes; int64_t ld, width; };
bool table_of(const at::Tensor* t, int dev, int64_t rows, Table& p) {
  if (!t || !on(*t, dev) || t->dim() != 2 || t->size(0) != rows || t->size(1) < 1 || t->size(1) > INT32_MAX || (t->stride(1) != 1 && t->size(1) > 1)) return false;
  const auto type = t->scalar_type();
  if (type != at::kInt && type != at::kShort) return false;
  p = {t->data_ptr(), type == at::kInt ? 4 : 2, rows > 1 ? t->stride(0) : t->size(1), t->size(1)};
  return p.ld >= p.width;
}
// Two pools and their scales: what they hold, or -1
int pools_of(const at::Tensor* k, const at::Tensor* v, const at::Tensor* ks, const at::Tensor* vs, int dev, int64_t ps) {
  if (!k || !v || !on(*k, dev) || !on(*v, dev) || k->dim() != 3 || k->sizes() != v->sizes() || k->scalar_type() != v->scalar_type() || !k->is_contiguous() ||
      !v->is_contiguous() || k->size(2) != HEAD || k->size(0) < 1 || k->size(0) > INT32_MAX || k->size(1) < 1 || k->size(1) > INT32_MAX)
    return -1;
  const auto type = k->scalar_type();
  if (type == at::kHalf) return ks || vs ? -1 : 0;
  if ((type != at::kChar && type != at::kFloat8_e4m3fn) || k->size(1) % ps) return -1;
  for (const at::Tensor* s : {ks, vs})
    if (!is(s, dev, at::kFloat) || s->dim() != 2 || s->size(0) != k->size(0) || s->size(1) != k->size(1) / ps || !s->is_contiguous()) return -1;
  return type == at::kChar ? 1 : 2;
}
const at::Tensor* tensor_or_none(PyObject* o, bool& fine) {
  if (o == Py_None) return nullptr;
  const at::Tensor* t = tensor(o);
  fine &= t != nullptr;
  return t;
}
void* ptr(const at::Tensor* t) { return t ? t->data_ptr() : nullptr; }
at::Tensor scratch(size_t bytes, int dev) {
  return bytes ? at::empty({(int64_t)bytes}, at::TensorOptions().dtype(at::kByte).device(at::kCUDA, (c10::DeviceIndex)dev)) : at::Tensor();
}
at::Tensor heads(int64_t rows, int64_t n, int dev) {
  return at::empty({rows, n, HEAD}, at::TensorOptions().dtype(at::kHalf).device(at::kCUDA, (c10::DeviceIndex)dev));
}
// Tensors that are used while other Python threads run
at::Tensor held(const at::Tensor* t) { return t ? *t : at::Tensor(); }

// A cap (0: None) and slopes of H heads (nullptr: None)
bool scores_of(PyObject* cap, PyObject* slopes, int dev, int64_t H, float& c, const at::Tensor*& t) {
  c = 0.f;
  if (cap != Py_None) {
    if (PyFloat_CheckExact(cap)) c = (float)PyFloat_AS_DOUBLE(cap);
    if (!(c > 0.f)) return false;
  }
  bool fine = true;
  t = tensor_or_none(slopes, fine);
  return fine && (!t || vector_of(t, dev, at::kFloat, H));
}

// attn_pages(p, q, k, v, k_scale, v_scale, L, page_size, seq_lens, window, sinks, softcap, slopes) -> o or None
PyObject* attn_pages(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 13 || !attn_pages_fn) Py_RETURN_NONE;
  bool fine = true;
  const at::Tensor *p = tensor(args[0]), *q = tensor(args[1]), *k = tensor(args[2]), *v = tensor(args[3]), *ks = tensor_or_none(args[4], fine),
                   *vs = tensor_or_none(args[5], fine), *lens = tensor_or_none(args[8], fine);
  int64_t L, ps, window, sinks, ld;
  Table tbl;
  if (!fine || !whole(args[6], -1, L) || !whole(args[7], -1, ps) || !whole(args[9], 0, window) || !whole(args[10], -1, sinks) || L < 0 || ps < 1 ||
      ps > MOST_PAGE || sinks < 0 || window < (args[9] == Py_None ? 0 : 1))
    Py_RETURN_NONE;
  const int dev = c10::cuda::current_device();
  if (!rows_of(q, dev, ld)) Py_RETURN_NONE;
  const int64_t B = q->size(0), H = q->size(1);
  const int kind = pools_of(k, v, ks, vs, dev, ps);
  if (kind < 0 || !table_of(p, dev, B, tbl) || L > tbl.width * ps || (lens && !vector_of(lens, dev, at::kInt, B))) Py_RETURN_NONE;
  if (args[9] == Py_None) sinks = 0;
  float cap;
  const at::Tensor* slopes;
  if (!scores_of(args[11], args[12], dev, H, cap, slopes)) Py_RETURN_NONE;
  const bool changed = slopes || cap != 0.f;
  if (changed && !attn_pages_scores_fn) Py_RETURN_NONE;
  const int Hkv = (int)k->size(0);
  const auto stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream();
  const at::Tensor own[] = {held(p), held(q), held(k), held(v), held(ks), held(vs), held(lens), held(slopes)};
  at::Tensor o, ws;
  int rc;
  {
    WithoutInterpreter w;
    const size_t bytes = attn_pages_bytes((int)B, (int)H, Hkv, (int)L, (int)window, (int)sinks);
    o = heads(B, H, dev);
    ws = scratch(bytes, dev);
    const auto at = [&](int i) { return own[i].defined() ? own[i].data_ptr() : nullptr; };
    if (changed)
      rc = attn_pages_scores_fn(tbl.ids, tbl.bytes, tbl.ld, (const int32_t*)at(6), at(1), ld, at(2), at(3), (const float*)at(4), (const float*)at(5), kind, o.data_ptr(),
                                own[2].size(1), (int)B, (int)L, (int)H, Hkv, (int)HEAD, (int)ps, (int)window, (int)sinks, cap, (const float*)at(7),
                                bytes ? ws.data_ptr() : nullptr, bytes, stream);
    else
      rc = attn_pages_fn(tbl.ids, tbl.bytes, tbl.ld, (const int32_t*)at(6), at(1), ld, at(2), at(3), (const float*)at(4), (const float*)at(5), kind, o.data_ptr(),
                         own[2].size(1), (int)B, (int)L, (int)H, Hkv, (int)HEAD, (int)ps, (int)window, (int)sinks, bytes ? ws.data_ptr() : nullptr, bytes, stream);
  }
  if (rc != 0) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(o));
  END_HANDLE_TH_ERRORS
}

// page_append(p, k, v, kpool, vpool, pos, page_size, offsets, k_scale, v_scale, q, cos, sin) -> (q rotated or None,) or None
PyObject* page_append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 13 || !page_append_fn) Py_RETURN_NONE;
  bool fine = true;
  const at::Tensor *p = tensor(args[0]), *k = tensor(args[1]), *v = tensor(args[2]), *kp = tensor(args[3]), *vp = tensor(args[4]), *pos = tensor(args[5]),
                   *off = tensor_or_none(args[7], fine), *ks = tensor_or_none(args[8], fine), *vs = tensor_or_none(args[9], fine),
                   *q = tensor_or_none(args[10], fine), *cos = tensor_or_none(args[11], fine), *sin = tensor_or_none(args[12], fine);
  int64_t ps, ldk, ldv, ldq = 0;
  Table tbl;
  if (!fine || !whole(args[6], -1, ps) || ps < 1 || ps > MOST_PAGE) Py_RETURN_NONE;
  const int dev = c10::cuda::current_device();
  const int kind = pools_of(kp, vp, ks, vs, dev, ps);
  if (kind < 0 || !rows_of(k, dev, ldk) || !rows_of(v, dev, ldv) || k->sizes() != v->sizes() || k->size(1) != kp->size(0) || !is(pos, dev, at::kInt) ||
      pos->dim() != 1 || !pos->is_contiguous())
    Py_RETURN_NONE;
  const int64_t T = k->size(0), B = pos->size(0);
  if (B < 1 || B >= INT32_MAX || (off ? !vector_of(off, dev, at::kInt, B + 1) : T != B) || !table_of(p, dev, B, tbl) || !cos != !sin || (q && !cos)) Py_RETURN_NONE;
  if (cos)
    for (const at::Tensor* t : {cos, sin})
      if (!is(t, dev, at::kHalf) || t->dim() != 2 || t->size(1) != HEAD / 2 || t->size(0) != cos->size(0) || t->size(0) < 1 || t->size(0) > INT32_MAX ||
          !t->is_contiguous() || (uintptr_t)t->data_ptr() % 16)
        Py_RETURN_NONE;
  if (q && (!rows_of(q, dev, ldq) || q->size(0) != T)) Py_RETURN_NONE;
  const auto stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream();
  const at::Tensor own[] = {held(p), held(k), held(v), held(kp), held(vp), held(pos), held(off), held(ks), held(vs), held(q), held(cos), held(sin)};
  const int H = q ? (int)q->size(1) : 0, Hkv = (int)kp->size(0), n_pos = cos ? (int)cos->size(0) : 0;
  at::Tensor out;
  int rc;
  {
    WithoutInterpreter w;
    if (H) out = heads(T, H, dev);
    const auto at = [&](int i) { return own[i].defined() ? own[i].data_ptr() : nullptr; };
    rc = page_append_fn(tbl.ids, tbl.bytes, tbl.ld, (int)tbl.width, (const int32_t*)at(5), (const int32_t*)at(6), at(9), ldq, H ? out.data_ptr() : nullptr, at(1),
                        ldk, at(2), ldv, at(10), at(11), n_pos, at(3), at(4), (float*)at(7), (float*)at(8), kind, own[3].size(1), (int)B, (int)T, H, Hkv,
                        (int)HEAD, (int)ps, stream);
  }
  if (rc != 0) Py_RETURN_NONE;
  for (int i : {3, 4, 7, 8})                     // writes that torch did not make itself: counted
    if (own[i].defined() && !own[i].is_inference()) own[i].unsafeGetTensorImpl()->bump_version();
  PyObject* rotated = nullptr;
  if (H) {
    rotated = THPVariable_Wrap(std::move(out));
    if (!rotated) return nullptr;
  } else {
    rotated = Py_NewRef(Py_None);
  }
  PyObject* r = PyTuple_Pack(1, rotated);
  Py_DECREF(rotated);
  return r;
  END_HANDLE_TH_ERRORS
}

// causal_window(q, k, v, window, sinks, offset, kernels._workspaces) -> o or None
PyObject* causal_window(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7 || !causal_window_fn) Py_RETURN_NONE;
  const at::Tensor *q = tensor(args[0]), *k = tensor(args[1]), *v = tensor(args[2]);
  int64_t window, sinks, offset, ldq, ldk, ldv;
  const int dev = c10::cuda::current_device();
  if (!whole(args[3], MOST, window) || !whole(args[4], -1, sinks) || !whole(args[5], -1, offset) || window < 1 || sinks < 0 || offset < 0 ||
      !rows_of(q, dev, ldq) || !rows_of(k, dev, ldk) || !rows_of(v, dev, ldv))
    Py_RETURN_NONE;
  const int64_t S = q->size(0), all = offset + S;
  if (k->size(1) != v->size(1) || k->size(0) < all || v->size(0) < all || all > MOST) Py_RETURN_NONE;
  const auto stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream();
  PyObject* st = PyLong_FromVoidPtr(stream);
  if (!st) return nullptr;
  const at::Tensor page = workspace(args[6], dev, st);
  Py_DECREF(st);
  if (!page.defined()) Py_RETURN_NONE;
  const int H = (int)q->size(1), Hkv = (int)k->size(1), w = (int)std::min(window, all), s = (int)std::min(sinks, all);
  const at::Tensor own[] = {held(q), held(k), held(v)};
  at::Tensor o, ws;
  int rc;
  {
    WithoutInterpreter without;
    const size_t bytes = causal_window_bytes((int)S, H, Hkv, (int)HEAD, (int)offset, w, s);
    o = heads(S, H, dev);
    ws = scratch(bytes, dev);
    rc = causal_window_fn(own[0].data_ptr(), ldq, own[1].data_ptr(), ldk, own[2].data_ptr(), ldv, o.data_ptr(), H * HEAD, (int)S, H, Hkv, (int)HEAD, (int)offset,
                          w, s, bytes ? ws.data_ptr() : nullptr, bytes, (int*)((char*)page.data_ptr() + 4092), stream);
  }
  if (rc != 0) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(o));
  END_HANDLE_TH_ERRORS
}

// causal_scores(q, k, v, window, sinks, offset, softcap, slopes, documents, prefix, kernels._workspaces) -> o or None
PyObject* causal_scores(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 11 || !causal_scores_fn) Py_RETURN_NONE;
  bool fine = true;
  const at::Tensor *q = tensor(args[0]), *k = tensor(args[1]), *v = tensor(args[2]), *docs = tensor_or_none(args[8], fine), *slopes;
  int64_t window, sinks, offset, prefix = 0, ldq, ldk, ldv;
  float cap;
  const int dev = c10::cuda::current_device();
  if (!fine || !whole(args[3], MOST, window) || !whole(args[4], -1, sinks) || !whole(args[5], -1, offset) || window < 1 || sinks < 0 || offset < 0 ||
      !rows_of(q, dev, ldq) || !rows_of(k, dev, ldk) || !rows_of(v, dev, ldv) || !scores_of(args[6], args[7], dev, q->size(1), cap, slopes))
    Py_RETURN_NONE;
  const int64_t S = q->size(0), all = offset + S;
  if (k->size(1) != v->size(1) || k->size(0) < all || v->size(0) < all || all > MOST) Py_RETURN_NONE;
  if (docs && (offset || docs->dim() != 1 || docs->size(0) < 1 || docs->size(0) > MOST || !vector_of(docs, dev, at::kInt, docs->size(0)))) Py_RETURN_NONE;
  const at::Tensor* prefixes = tensor(args[9]);
  if (prefixes ? !docs || !vector_of(prefixes, dev, at::kInt, docs->size(0) - 1) : !whole(args[9], 0, prefix) || prefix < 0) Py_RETURN_NONE;
  const auto stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream();
  PyObject* st = PyLong_FromVoidPtr(stream);
  if (!st) return nullptr;
  const at::Tensor page = workspace(args[10], dev, st);
  Py_DECREF(st);
  if (!page.defined()) Py_RETURN_NONE;
  const int H = (int)q->size(1), Hkv = (int)k->size(1), w = (int)std::min(window, all), s = (int)std::min(sinks, all), n_docs = docs ? (int)docs->size(0) - 1 : 0;
  const at::Tensor own[] = {held(q), held(k), held(v), held(slopes), held(docs), held(prefixes)};
  at::Tensor o, ws;
  int rc;
  {
    WithoutInterpreter without;
    const size_t bytes = causal_scores_bytes((int)S, H, Hkv, (int)HEAD, (int)offset, w, s);
    o = heads(S, H, dev);
    ws = scratch(bytes, dev);
    // (a prefix for each of no documents has no address, and none is looked up)
    const auto at = [&](int i) { return own[i].defined() ? own[i].data_ptr() : nullptr; };
    rc = causal_scores_fn(at(0), ldq, at(1), ldk, at(2), ldv, o.data_ptr(), H * HEAD, (int)S, H, Hkv, (int)HEAD, (int)offset, w, s, cap, (const float*)at(3),
                          (const int32_t*)at(4), n_docs, (const int32_t*)at(5), (int)std::min(prefix, all), 0, bytes ? ws.data_ptr() : nullptr, bytes,
                          (int*)((char*)page.data_ptr() + 4092), stream);
  }
  if (rc != 0) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(o));
  END_HANDLE_TH_ERRORS
}

// The books of a paged cache, where they lie as the library reads them
struct Books {
  at::Tensor table, lens, refs;
  int64_t B, W, n, ld;
};
bool books_of(PyObject* const* args, int dev, Books& b) {
  const at::Tensor *p = tensor(args[0]), *lens = tensor(args[1]), *refs = tensor(args[2]);
  if (!is(p, dev, at::kInt) || p->dim() != 2 || p->size(0) < 1 || p->size(0) > INT32_MAX || p->size(1) < 1 || p->size(1) >= MOST_PAGE || (p->stride(1) != 1 && p->size(1) > 1) ||
      !vector_of(lens, dev, at::kInt, p->size(0)) || !is(refs, dev, at::kInt) || refs->dim() != 1 || refs->size(0) < 1 || refs->size(0) > 1 << 28 || !refs->is_contiguous())
    return false;
  b = {*p, *lens, *refs, p->size(0), p->size(1), refs->size(0), p->size(0) > 1 ? p->stride(0) : p->size(1)};
  return b.ld >= b.W;
}
// Books that are written in place must not overlap, nor `more` them
bool apart(const Books& b, const at::Tensor* more) {
  struct Span { const char *from, *to; };
  const auto span = [](const at::Tensor& t, int64_t n) { return Span{(const char*)t.data_ptr(), (const char*)t.data_ptr() + 4 * n}; };
  const Span x[] = {span(b.table, (b.B - 1) * b.ld + b.W), span(b.lens, b.B), span(b.refs, b.n), span(*more, more->numel())};
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < i; ++j)
      if (x[i].from < x[j].to && x[j].from < x[i].to) return false;
  return true;
}
// Pools [heads, P, 128], or of layers in front, and scales of those
struct BooksPools {
  at::Tensor k, v, ks, vs;
  int kind;
  int64_t heads, P;
};
bool books_pools_of(PyObject* const* args, int dev, const Books& b, int64_t ps, BooksPools& p) {
  bool fine = true;
  const at::Tensor *k = tensor(args[0]), *v = tensor(args[1]), *ks = tensor_or_none(args[2], fine), *vs = tensor_or_none(args[3], fine);
  if (!fine || !k || !v || !on(*k, dev) || !on(*v, dev) || k->dim() < 3 || k->sizes() != v->sizes() || k->scalar_type() != v->scalar_type() || !k->is_contiguous() ||
      !v->is_contiguous() || k->size(-1) != HEAD || k->numel() == 0)
    return false;
  p.P = k->size(-2);
  p.heads = k->numel() / (p.P * HEAD);
  const auto type = k->scalar_type();
  p.kind = type == at::kHalf ? 0 : type == at::kChar ? 1 : type == at::kFloat8_e4m3fn ? 2 : -1;
  if (p.kind < 0 || p.P > INT32_MAX || p.heads > INT32_MAX || b.n * ps > p.P || (p.kind == 0 ? ks || vs : !ks || !vs || p.P % ps != 0)) return false;
  for (const at::Tensor* s : {ks, vs})
    if (s && (!is(s, dev, at::kFloat) || !s->is_contiguous() || s->dim() != k->dim() - 1 || s->size(-1) != p.P / ps || s->sizes().slice(0, s->dim() - 1) != k->sizes().slice(0, k->dim() - 2)))
      return false;
  p.k = *k, p.v = *v, p.ks = held(ks), p.vs = held(vs);
  return true;
}
// New books: a table and two rows of numbers in one piece of memory, each from 16 bytes on (three pieces take 2 us more)
void new_books(int64_t B, int64_t W, int64_t n1, int64_t n2, int dev, at::Tensor& table, at::Tensor& one, at::Tensor& two) {
  const int64_t at1 = (B * W + 3) / 4 * 4, at2 = at1 + (n1 + 3) / 4 * 4;
  const at::Tensor all = at::empty({at2 + n2}, at::TensorOptions().dtype(at::kInt).device(at::kCUDA, (c10::DeviceIndex)dev));
  const auto part = [&](int64_t from, at::IntArrayRef size) {
    at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all.storage()), all.key_set(), all.dtype());
    t.unsafeGetTensorImpl()->set_storage_offset(from);
    t.unsafeGetTensorImpl()->set_sizes_contiguous(size);
    return t;
  };
  table = part(0, {B, W});
  one = part(at1, {n1});
  two = part(at2, {n2});
}
void written(const at::Tensor& t) {
  if (t.defined() && !t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
// `out`: 0 None, 1 a tuple that begins with these objects, -1 something else
int in_place(PyObject* out, std::initializer_list<PyObject*> books) {
  if (out == Py_None) return 0;
  if (!PyTuple_Check(out) || PyTuple_GET_SIZE(out) != 3) return -1;
  Py_ssize_t i = 0;
  for (PyObject* b : books)
    if (PyTuple_GET_ITEM(out, i++) != b) return -1;
  return 1;
}
PyObject* three(at::Tensor a, at::Tensor b, at::Tensor c) {
  PyObject* r = PyTuple_New(3);
  if (!r) return nullptr;
  Py_ssize_t i = 0;
  for (at::Tensor* t : {&a, &b, &c}) {
    PyObject* x = THPVariable_Wrap(std::move(*t));
    if (!x) {
      Py_DECREF(r);
      return nullptr;
    }
    PyTuple_SET_ITEM(r, i++, x);
  }
  return r;
}
int* int_ptr(const at::Tensor& t) { return (int*)t.data_ptr(); }
float* float_ptr(const at::Tensor& t) { return t.defined() ? (float*)t.data_ptr() : nullptr; }

// page_fork(p, lens, refs, parents, page_size, out) -> (p, lens, refs) or None
PyObject* page_fork(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6 || !page_fork_fn) Py_RETURN_NONE;
  const int dev = c10::cuda::current_device(), place = in_place(args[5], {args[0], args[1], args[2]});
  Books b;
  int64_t ps;
  const at::Tensor* parents = tensor(args[3]);
  if (place < 0 || !books_of(args, dev, b) || !vector_of(parents, dev, at::kInt, b.B) || !whole(args[4], -1, ps) || ps < 1 || ps > MOST_PAGE) Py_RETURN_NONE;
  if (place && !apart(b, parents)) Py_RETURN_NONE;
  const auto stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream();
  const at::Tensor from = *parents;
  at::Tensor table, lens, refs, ws;
  int rc;
  {
    WithoutInterpreter without;
    if (place) table = b.table, lens = b.lens, refs = b.refs;
    else new_books(b.B, b.W, b.B, b.n, dev, table, lens, refs);
    const size_t bytes = place ? page_fork_bytes((int)b.B, (int)b.W, (int)b.n) : 0;
    ws = scratch(bytes, dev);
    rc = page_fork_fn(int_ptr(b.table), b.ld, int_ptr(b.lens), int_ptr(b.refs), int_ptr(from), int_ptr(table), place ? b.ld : b.W, int_ptr(lens), int_ptr(refs), (int)b.B,
                      (int)b.W, (int)b.n, (int)ps, bytes ? ws.data_ptr() : nullptr, bytes, stream);
  }
  if (rc != 0) Py_RETURN_NONE;
  if (place)
    for (const at::Tensor* t : {&table, &lens, &refs}) written(*t);
  return three(table, lens, refs);
  END_HANDLE_TH_ERRORS
}

// page_extend(p, lens, refs, kpool, vpool, k_scale, v_scale, add, page_size, out) -> (p, lens, refs) or None
PyObject* page_extend(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 10 || !page_extend_fn) Py_RETURN_NONE;
  const int dev = c10::cuda::current_device(), place = in_place(args[9], {args[0], args[1], args[2]});
  Books b;
  BooksPools p;
  int64_t ps;
  const at::Tensor* add = tensor(args[7]);
  if (place < 0 || !books_of(args, dev, b) || b.B > 16384 || !vector_of(add, dev, at::kInt, b.B) || !whole(args[8], -1, ps) || ps < 1 || ps > MOST_PAGE ||
      !books_pools_of(args + 3, dev, b, ps, p))
    Py_RETURN_NONE;
  if (place && !apart(b, add)) Py_RETURN_NONE;
  const auto stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream();
  const at::Tensor more = *add;
  at::Tensor table, lens, refs, ws;
  int rc;
  {
    WithoutInterpreter without;
    if (place) table = b.table, lens = b.lens, refs = b.refs;
    else new_books(b.B, b.W, b.B, b.n, dev, table, lens, refs);
    const size_t bytes = page_extend_bytes((int)b.B, (int)b.n, place);
    ws = scratch(bytes, dev);
    rc = page_extend_fn(int_ptr(b.table), b.ld, int_ptr(b.lens), int_ptr(b.refs), int_ptr(more), int_ptr(table), place ? b.ld : b.W, int_ptr(lens), int_ptr(refs), (int)b.B,
                        (int)b.W, (int)b.n, (int)ps, p.k.data_ptr(), p.v.data_ptr(), float_ptr(p.ks), float_ptr(p.vs), p.kind, p.P, (int)p.heads, bytes ? ws.data_ptr() : nullptr, bytes, stream);
  }
  if (rc != 0) Py_RETURN_NONE;
  for (const at::Tensor* t : {&p.k, &p.v, &p.ks, &p.vs}) written(*t);
  if (place)
    for (const at::Tensor* t : {&table, &lens, &refs}) written(*t);
  return three(table, lens, refs);
  END_HANDLE_TH_ERRORS
}

// page_compact(p, lens, refs, kpool, vpool, k_scale, v_scale, page_size, out) -> (p, refs, where) or None
PyObject* page_compact(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 9 || !page_compact_fn) Py_RETURN_NONE;
  const int dev = c10::cuda::current_device(), place = in_place(args[8], {args[0], args[2]});
  Books b;
  BooksPools p;
  int64_t ps;
  if (place < 0 || !books_of(args, dev, b) || !whole(args[7], -1, ps) || ps < 1 || ps > MOST_PAGE || !books_pools_of(args + 3, dev, b, ps, p)) Py_RETURN_NONE;
  const auto stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream();
  const at::Tensor* given = place ? tensor(PyTuple_GET_ITEM(args[8], 2)) : nullptr;
  if (place && (!vector_of(given, dev, at::kInt, b.n) || !apart(b, given))) Py_RETURN_NONE;
  at::Tensor table, refs, where = held(given), ws;
  int rc;
  {
    WithoutInterpreter without;
    if (place) table = b.table, refs = b.refs;
    else new_books(b.B, b.W, b.n, b.n, dev, table, refs, where);
    const size_t bytes = page_compact_bytes((int)b.n, place);
    ws = scratch(bytes, dev);
    rc = page_compact_fn(int_ptr(b.table), b.ld, int_ptr(b.lens), int_ptr(b.refs), int_ptr(table), place ? b.ld : b.W, int_ptr(refs), int_ptr(where), (int)b.B, (int)b.W, (int)b.n, (int)ps,
                         p.k.data_ptr(), p.v.data_ptr(), float_ptr(p.ks), float_ptr(p.vs), p.kind, p.P, (int)p.heads, bytes ? ws.data_ptr() : nullptr, bytes, stream);
  }
  if (rc != 0) Py_RETURN_NONE;
  for (const at::Tensor* t : {&p.k, &p.v, &p.ks, &p.vs}) written(*t);
  if (place)
    for (const at::Tensor* t : {&table, &refs, &where}) written(*t);
  return three(table, refs, where);
  END_HANDLE_TH_ERRORS
}

// init_books(addresses of q40_attn_pages_scores, q40_attn_causal_scores, _workspace_bytes, q40_page_fork, _workspace_bytes, q40_page_extend, _workspace_bytes,
// q40_page_compact, _workspace_bytes)
PyObject* init_books(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n == 9) {
    attn_pages_scores_fn = (AttnPagesScores)PyLong_AsVoidPtr(args[0]);
    causal_scores_fn = (CausalScores)PyLong_AsVoidPtr(args[1]);
    causal_scores_bytes = (CausalWindowBytes)PyLong_AsVoidPtr(args[2]);
    page_fork_fn = (PageFork)PyLong_AsVoidPtr(args[3]);
    page_fork_bytes = (size_t (*)(int, int, int))PyLong_AsVoidPtr(args[4]);
    page_extend_fn = (PageExtend)PyLong_AsVoidPtr(args[5]);
    page_extend_bytes = (size_t (*)(int, int, int))PyLong_AsVoidPtr(args[6]);
    page_compact_fn = (PageCompact)PyLong_AsVoidPtr(args[7]);
    page_compact_bytes = (size_t (*)(int, int))PyLong_AsVoidPtr(args[8]);
  }
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
}

// init_pages(addresses of q40_attn_pages, _workspace_bytes, q40_page_append, q40_attn_causal_window, _workspace_bytes)
PyObject* init_pages(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n == 5) {
    attn_pages_fn = (AttnPages)PyLong_AsVoidPtr(args[0]);
    attn_pages_bytes = (AttnPagesBytes)PyLong_AsVoidPtr(args[1]);
    page_append_fn = (PageAppend)PyLong_AsVoidPtr(args[2]);
    causal_window_fn = (CausalWindow)PyLong_AsVoidPtr(args[3]);
    causal_window_bytes = (CausalWindowBytes)PyLong_AsVoidPtr(args[4]);
  }
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
}

// init(address of q40_matmul_tiled, address of q40_gemm_nk)
PyObject* init(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n == 2) {
    matmul_tiled = (MatmulTiled)PyLong_AsVoidPtr(args[0]);
    gemm_nk = (GemmNk)PyLong_AsVoidPtr(args[1]);
  }
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {{"matmul", (PyCFunction)(void*)matmul, METH_FASTCALL, nullptr},
                         {"linear", (PyCFunction)(void*)linear, METH_FASTCALL, nullptr},
                         {"attn_pages", (PyCFunction)(void*)attn_pages, METH_FASTCALL, nullptr},
                         {"page_append", (PyCFunction)(void*)page_append, METH_FASTCALL, nullptr},
                         {"causal_window", (PyCFunction)(void*)causal_window, METH_FASTCALL, nullptr},
                         {"causal_scores", (PyCFunction)(void*)causal_scores, METH_FASTCALL, nullptr},
                         {"page_fork", (PyCFunction)(void*)page_fork, METH_FASTCALL, nullptr},
                         {"page_extend", (PyCFunction)(void*)page_extend, METH_FASTCALL, nullptr},
                         {"page_compact", (PyCFunction)(void*)page_compact, METH_FASTCALL, nullptr},
                         {"init_books", (PyCFunction)(void*)init_books, METH_FASTCALL, nullptr},
                         {"init_pages", (PyCFunction)(void*)init_pages, METH_FASTCALL, nullptr},
                         {"init", (PyCFunction)(void*)init, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host_calls(void) { return PyModule_Create(&module); }
