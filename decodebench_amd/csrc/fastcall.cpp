// fastcall.cpp -- native call path of decodebench_amd.ops (a CPython extension
// module, _fastcall).
//
// One function per op.  It checks the arguments as the Python op does,
// allocates the output, finds the current stream and calls the C ABI entry
// point; whatever it does not take as it is (another device current, a tensor
// subclass, a wrong shape or type, a workspace that has to be made, a non-zero
// status) it answers with None, and the Python op then does the same work, or
// raises, step by step.  In Python those steps took 6.5-7.5 us a call on the
// host of an MI355X, more than the small kernels take on the GPU: F1 [2048,
// 2048] at one row 7.1-7.7 us a call, 5.0 through here; F4 at batch 1, L = 8192
// 10.4 and 8.9.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/EmptyTensor.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>
#include <cmath>
#include <cstdint>

#include "../../include/decodebench_hip.h"

#ifndef DB_BUILT_FOR
#error "build with decodebench_amd.build, which defines DB_BUILT_FOR"
#endif

namespace {

struct Abi {
  decltype(&db_f1_rmsnorm_gemv) f1;
  decltype(&db_f2_gateup_swiglu) f2;
  decltype(&db_f2_rmsnorm_gateup_swiglu) f2n;
  decltype(&db_gemv) gemv;
  decltype(&db_f4_default_splits) f4_default_splits;
  decltype(&db_f4_workspace_bytes) f4_workspace_bytes;
  decltype(&db_f4_splitkv) f4;
  decltype(&db_stream_capture_id) capture_id;
  decltype(&db_gemv_workspace_bytes) gemv_workspace_bytes;
  decltype(&db_gemv_ws) gemv_ws;
  decltype(&db_paged_plan) paged_plan;
  decltype(&db_rope_append) rope_append;
  decltype(&db_paged_attention_workspace_bytes) paged_workspace_bytes;
  decltype(&db_paged_attention) paged_attention;
} abi;

PyObject* raw_stream = nullptr;  // device index -> current stream's handle
PyObject* get_device = nullptr;  // () -> current device
PyObject* workspaces = nullptr;  // dict ([kind,] device, stream, bytes) -> tensor
PyObject* cu_counts = nullptr;   // dict device -> compute units

const at::Tensor* tensor(PyObject* o) {
  return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr;
}

// A contiguous GPU tensor of the type, on device `idx` (any if -1).
bool plain(const at::Tensor* t, at::ScalarType type, int idx) {
  return t && t->is_cuda() && t->scalar_type() == type && t->is_contiguous() &&
         (idx < 0 || t->get_device() == idx);
}

// The current stream of device `idx` if that is the current device.
// 1: found, 0: another device is current, -1: a Python error is set.
int stream_of(int idx, void** stream) {
  PyObject* d = PyObject_CallNoArgs(get_device);
  if (!d) return -1;
  const long cur = PyLong_AsLong(d);
  if (cur == -1 && PyErr_Occurred()) {
    Py_DECREF(d);
    return -1;
  }
  if (cur != idx) {
    Py_DECREF(d);
    return 0;
  }
  PyObject* s = PyObject_CallFunctionObjArgs(raw_stream, d, nullptr);
  Py_DECREF(d);
  if (!s) return -1;
  *stream = PyLong_AsVoidPtr(s);
  Py_DECREF(s);
  return *stream == nullptr && PyErr_Occurred() ? -1 : 1;
}

bool number(PyObject* o, double* v) {
  if (!PyFloat_CheckExact(o)) return false;
  *v = PyFloat_AS_DOUBLE(o);
  return true;
}

// fp16 weights without a scale, or e4m3 bytes with one fp32 scale per row.
bool weights(const at::Tensor* w, PyObject* scale, int64_t N, int idx, int* dtype,
             const float** sp) {
  *sp = nullptr;
  if (plain(w, at::kHalf, idx)) {
    *dtype = DB_DTYPE_F16;
    return scale == Py_None;
  }
  if (!plain(w, at::kFloat8_e4m3fn, idx) && !plain(w, at::kByte, idx)) return false;
  const at::Tensor* s = tensor(scale);
  if (!plain(s, at::kFloat, idx) || s->dim() != 1 || s->size(0) != N) return false;
  *dtype = DB_DTYPE_FP8_E4M3;
  *sp = static_cast<const float*>(s->data_ptr());
  return true;
}

// A GEMV op of x [B, K] or [K] on w0 (and w1) [N, K]; g and eps in the norm
// modes.  New reference, Py_None where the Python op has to take over.
PyObject* gemv_op(PyObject* xo, PyObject* go, PyObject* w0o, PyObject* w1o, PyObject* epso,
                  PyObject* s0o, PyObject* s1o) {
  const at::Tensor* x = tensor(xo);
  if (!plain(x, at::kHalf, -1)) Py_RETURN_NONE;
  const int64_t dim = x->dim();
  if (dim != 1 && dim != 2) Py_RETURN_NONE;
  const int idx = x->get_device();
  const int64_t B = dim == 2 ? x->size(0) : 1, K = x->size(dim - 1);
  const at::Tensor* w0 = tensor(w0o);
  const at::Tensor* w1 = w1o ? tensor(w1o) : nullptr;
  if (!w0 || w0->dim() != 2 || w0->size(1) != K) Py_RETURN_NONE;
  const int64_t N = w0->size(0);
  if (B > INT_MAX || K > INT_MAX || N > INT_MAX) Py_RETURN_NONE;
  int dtype = 0, dtype1 = 0;
  const float *s0 = nullptr, *s1 = nullptr;
  if (!weights(w0, s0o, N, idx, &dtype, &s0)) Py_RETURN_NONE;
  if (w1o && (!w1 || w1->sizes() != w0->sizes() || w1->scalar_type() != w0->scalar_type() ||
              !weights(w1, s1o, N, idx, &dtype1, &s1)))
    Py_RETURN_NONE;
  const at::Tensor* g = nullptr;
  double eps = 0.0;
  if (go) {
    g = tensor(go);
    if (!plain(g, at::kHalf, idx) || g->dim() != 1 || g->size(0) != K || !number(epso, &eps))
      Py_RETURN_NONE;
  }
  void* stream = nullptr;
  const int found = stream_of(idx, &stream);
  if (found < 0) return nullptr;
  if (found == 0) Py_RETURN_NONE;
  at::Tensor y = at::empty({B, N}, at::TensorOptions().dtype(at::kHalf).device(
                                       at::Device(at::kCUDA, (c10::DeviceIndex)idx)));
  const void* xp = x->data_ptr();
  const void* gp = g ? g->data_ptr() : nullptr;
  const void* w0p = w0->data_ptr();
  const void* w1p = w1 ? w1->data_ptr() : nullptr;
  void* yp = y.data_ptr();
  const int b = (int)B, k = (int)K, n = (int)N;
  // K split over workgroups, in a workspace that the allocator takes back in
  // stream order after this call; one launch where there is no room for it.
  at::Tensor ws;
  size_t bytes = b > 8 ? abi.gemv_workspace_bytes(g != nullptr, w1 != nullptr, b, k, n, dtype) : 0;
  if (bytes > 0) {
    try {
      ws = at::empty({(int64_t)bytes}, at::TensorOptions().dtype(at::kByte).device(y.device()));
    } catch (const c10::OutOfMemoryError&) {
      bytes = 0;
    }
  }
  void* wsp = bytes > 0 ? ws.data_ptr() : nullptr;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  if (bytes > 0)
    rc = abi.gemv_ws(xp, gp, w0p, w1p, s0, s1, yp, wsp, bytes, b, k, n, (float)eps, dtype, stream);
  else if (w1)
    rc = g ? abi.f2n(xp, gp, w0p, w1p, s0, s1, yp, b, k, n, (float)eps, dtype, stream)
           : abi.f2(xp, w0p, w1p, s0, s1, yp, b, k, n, dtype, stream);
  else
    rc = g ? abi.f1(xp, gp, w0p, s0, yp, b, k, n, (float)eps, dtype, stream)
           : abi.gemv(xp, w0p, s0, yp, b, k, n, dtype, stream);
  Py_END_ALLOW_THREADS
  if (rc != DB_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(dim == 1 ? y.select(0, 0) : y);
}

// (x, g, W, eps, w_scale)
PyObject* f1(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 5) Py_RETURN_NONE;
  return gemv_op(a[0], a[1], a[2], nullptr, a[3], a[4], nullptr);
  END_HANDLE_TH_ERRORS
}

// (x, W, w_scale)
PyObject* gemv(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 3) Py_RETURN_NONE;
  return gemv_op(a[0], nullptr, a[1], nullptr, nullptr, a[2], nullptr);
  END_HANDLE_TH_ERRORS
}

// (x, Wg, Wu, sg, su)
PyObject* f2(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 5) Py_RETURN_NONE;
  return gemv_op(a[0], nullptr, a[1], a[2], nullptr, a[3], a[4]);
  END_HANDLE_TH_ERRORS
}

// (x, g, Wg, Wu, eps, sg, su)
PyObject* f2n(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7) Py_RETURN_NONE;
  return gemv_op(a[0], a[1], a[2], a[3], a[4], a[5], a[6]);
  END_HANDLE_TH_ERRORS
}

// (q, K, V, scale or None, n_splits or None): outside capture, with a
// workspace of its size already in the cache.
PyObject* f4(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 5) Py_RETURN_NONE;
  const at::Tensor *q = tensor(a[0]), *k = tensor(a[1]), *v = tensor(a[2]);
  if (!plain(q, at::kHalf, -1) || q->dim() != 3) Py_RETURN_NONE;
  const int idx = q->get_device();
  if (!plain(k, at::kHalf, idx) || !plain(v, at::kHalf, idx) || k->dim() != 4 ||
      k->sizes() != v->sizes())
    Py_RETURN_NONE;
  const int64_t B = q->size(0), Hq = q->size(1), D = q->size(2);
  const int64_t Hkv = k->size(1), L = k->size(2);
  if (k->size(0) != B || k->size(3) != D || D < 1 || B > INT_MAX || Hq > INT_MAX ||
      Hkv > INT_MAX || L > INT_MAX || D > INT_MAX)
    Py_RETURN_NONE;
  double scale = 1.0 / std::sqrt((double)D);
  if (a[3] != Py_None && !number(a[3], &scale)) Py_RETURN_NONE;
  void* stream = nullptr;
  const int found = stream_of(idx, &stream);
  if (found < 0) return nullptr;
  if (found == 0) Py_RETURN_NONE;
  PyObject* dev = PyLong_FromLong(idx);
  if (!dev) return nullptr;
  long S = 0;
  if (a[4] == Py_None) {
    PyObject* cu = PyDict_GetItemWithError(cu_counts, dev);  // borrowed
    const long cus = cu ? PyLong_AsLong(cu) : 0;
    if (cus > 0) S = abi.f4_default_splits((int)B, (int)Hkv, (int)L, (int)cus);
  } else if (PyLong_CheckExact(a[4])) {
    S = PyLong_AsLong(a[4]);
  }
  if (PyErr_Occurred() || S < 1 || S > 256) {
    PyErr_Clear();
    Py_DECREF(dev);
    Py_RETURN_NONE;
  }
  const size_t bytes =
      abi.f4_workspace_bytes((int)B, (int)Hq, (int)Hkv, (int)L, (int)D, (int)S);
  at::Tensor ws;  // keeps the workspace alive through the call
  if (bytes > 0) {
    unsigned long long capture = 0;
    if (abi.capture_id(stream, &capture) != DB_OK || capture != 0) {
      Py_DECREF(dev);
      Py_RETURN_NONE;
    }
    PyObject* key = Py_BuildValue("(OKn)", dev, (unsigned long long)(uintptr_t)stream,
                                  (Py_ssize_t)bytes);
    PyObject* hit = key ? PyDict_GetItemWithError(workspaces, key) : nullptr;  // borrowed
    Py_XDECREF(key);
    const at::Tensor* t = hit ? tensor(hit) : nullptr;
    if (!t) {
      Py_DECREF(dev);
      if (PyErr_Occurred()) return nullptr;
      Py_RETURN_NONE;
    }
    ws = *t;
  }
  Py_DECREF(dev);
  at::Tensor o = at::empty({B, Hq, D}, at::TensorOptions().dtype(at::kHalf).device(
                                           at::Device(at::kCUDA, (c10::DeviceIndex)idx)));
  const void *qp = q->data_ptr(), *kp = k->data_ptr(), *vp = v->data_ptr();
  void *op = o.data_ptr(), *wp = bytes ? ws.data_ptr() : nullptr;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = abi.f4(qp, kp, vp, op, wp, bytes, (int)B, (int)Hq, (int)Hkv, (int)L, (int)D, (int)S,
              (float)scale, stream);
  Py_END_ALLOW_THREADS
  if (rc != DB_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(o);
  END_HANDLE_TH_ERRORS
}

// ------------------------------------------------ a step over a paged KV cache
// A GPU tensor of the type and number of dimensions, its last one contiguous.
bool strided(const at::Tensor* t, at::ScalarType type, int64_t dim, int idx) {
  return t && t->is_cuda() && t->scalar_type() == type && t->dim() == dim &&
         (idx < 0 || t->get_device() == idx) && (t->size(dim - 1) <= 1 || t->stride(dim - 1) == 1);
}

// Whether the sizes fit the C ABI's ints.
bool ints(const at::Tensor* t) {
  for (const int64_t n : t->sizes())
    if (n > INT_MAX) return false;
  return true;
}

long long stride_of(const at::Tensor* t, int64_t d) { return t->size(d) > 1 ? t->stride(d) : 0; }

int activation(at::ScalarType t) {
  return t == at::kHalf ? DB_DTYPE_F16 : t == at::kBFloat16 ? DB_DTYPE_BF16 : -1;
}

bool paged_cache(PyObject* ko, PyObject* vo, PyObject* kso, PyObject* vso, at::ScalarType act,
                 int idx, db_paged_cache* c) {
  const at::Tensor *k = tensor(ko), *v = tensor(vo);
  if (!k) return false;
  const at::ScalarType type = k->scalar_type();
  if (!strided(k, type, 4, idx) || !strided(v, type, 4, idx) || k->sizes() != v->sizes() ||
      !ints(k))
    return false;
  *c = {};
  if (type == at::kFloat8_e4m3fn) {
    const at::Tensor *ks = tensor(kso), *vs = tensor(vso);
    for (const at::Tensor* s : {ks, vs})
      if (!plain(s, at::kFloat, idx) || s->dim() != 1 || s->size(0) != k->size(1)) return false;
    c->k_scale = static_cast<const float*>(ks->data_ptr());
    c->v_scale = static_cast<const float*>(vs->data_ptr());
    c->dtype = DB_DTYPE_FP8_E4M3;
  } else {
    if (type != act || kso != Py_None || vso != Py_None) return false;
    c->dtype = activation(type);
  }
  c->k = k->data_ptr();
  c->v = v->data_ptr();
  c->k_page_stride = stride_of(k, 0);
  c->k_head_stride = stride_of(k, 1);
  c->k_token_stride = stride_of(k, 2);
  c->v_page_stride = stride_of(v, 0);
  c->v_head_stride = stride_of(v, 1);
  c->v_token_stride = stride_of(v, 2);
  c->pages = (int)k->size(0);
  c->Hkv = (int)k->size(1);
  c->page_size = (int)k->size(2);
  c->D = (int)k->size(3);
  return true;
}

at::Tensor empty_on(at::IntArrayRef sizes, at::ScalarType type, int idx) {
  return at::empty(sizes, at::TensorOptions().dtype(type).device(
                              at::Device(at::kCUDA, (c10::DeviceIndex)idx)));
}

// The same for `n` elements on the current device, without at::empty's dispatch: from
// torch's allocator, as the storage of an empty tensor names it.
at::Tensor empty_here(int64_t n, at::ScalarType type, int idx) {
  static c10::Allocator* const allocator = empty_on({0}, type, idx).storage().allocator();
  if (!allocator) return empty_on({n}, type, idx);
  return at::Tensor(at::detail::empty_generic(
      {n}, allocator, c10::DispatchKeySet(c10::DispatchKey::CUDA), type, std::nullopt));
}

bool integer(PyObject* o, long* v) {
  if (!PyLong_CheckExact(o)) return false;
  *v = PyLong_AsLong(o);
  if (*v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return *v >= 0 && *v <= INT_MAX;
}

// (past_len, new_len, block_table, free_pages, page_size, n_tokens, free_start or None):
// (q_start, kv_len, position, slot, free_next)
PyObject* plan(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7) Py_RETURN_NONE;
  const at::Tensor *past = tensor(a[0]), *fresh = tensor(a[1]), *table = tensor(a[2]),
                   *pages = tensor(a[3]);
  long page = 0, T = 0;
  if (!plain(past, at::kInt, -1) || !integer(a[4], &page) || !integer(a[5], &T)) Py_RETURN_NONE;
  const int idx = past->get_device();
  if (!plain(fresh, at::kInt, idx) || !plain(pages, at::kInt, idx) ||
      !strided(table, at::kInt, 2, idx) || !ints(table) || pages->dim() != 1 || !ints(pages))
    Py_RETURN_NONE;
  const int64_t R = table->size(0), width = table->size(1);
  if (past->dim() != 1 || past->size(0) != R || fresh->dim() != 1 || fresh->size(0) != R ||
      (R > 1 && table->stride(0) < width))
    Py_RETURN_NONE;
  const int* start = nullptr;
  if (a[6] != Py_None) {
    const at::Tensor* t = tensor(a[6]);
    if (!plain(t, at::kInt, idx) || t->numel() != 1) Py_RETURN_NONE;
    start = static_cast<const int*>(t->data_ptr());
  }
  void* stream = nullptr;
  const int found = stream_of(idx, &stream);
  if (found < 0) return nullptr;
  if (found == 0) Py_RETURN_NONE;
  // Storage of its own for each: torch saves no two types of one storage, and with a
  // part of one all of it.
  at::Tensor out[5] = {
      empty_here(R + 1, at::kInt, idx), empty_here(R, at::kInt, idx), empty_here(T, at::kInt, idx),
      empty_here(T, at::kLong, idx), empty_here(1, at::kInt, idx)};
  const int *pp = static_cast<const int*>(past->data_ptr()),
            *np = static_cast<const int*>(fresh->data_ptr()),
            *fp = static_cast<const int*>(pages->data_ptr());
  int* tp = static_cast<int*>(table->data_ptr());
  const long long row = R > 1 ? table->stride(0) : width;
  const int count = (int)pages->numel();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = abi.paged_plan(pp, np, tp, row, (int)width, fp, count, start, (int)page, (int)R, (int)T,
                      static_cast<int*>(out[0].data_ptr()), static_cast<int*>(out[1].data_ptr()),
                      static_cast<int*>(out[2].data_ptr()),
                      static_cast<long long*>(out[3].data_ptr()),
                      static_cast<int*>(out[4].data_ptr()), stream);
  Py_END_ALLOW_THREADS
  if (rc != DB_OK) Py_RETURN_NONE;
  PyObject* result = PyTuple_New(5);
  if (!result) return nullptr;
  for (int i = 0; i < 5; ++i) PyTuple_SET_ITEM(result, i, THPVariable_Wrap(out[i]));
  return result;
  END_HANDLE_TH_ERRORS
}

// (qkv, position, slot, K, V, inv_freq, axes as bytes or None, interleaved, k_scale, v_scale)
PyObject* rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 10) Py_RETURN_NONE;
  const at::Tensor *qkv = tensor(a[0]), *pos = tensor(a[1]), *slot = tensor(a[2]),
                   *freq = tensor(a[5]);
  if (!qkv || activation(qkv->scalar_type()) < 0 || !PyBool_Check(a[7])) Py_RETURN_NONE;
  const at::ScalarType type = qkv->scalar_type();
  if (!strided(qkv, type, 2, -1) || !ints(qkv)) Py_RETURN_NONE;
  const int idx = qkv->get_device();
  db_paged_cache cache;
  if (!paged_cache(a[3], a[4], a[8], a[9], type, idx, &cache) || cache.D < 1) Py_RETURN_NONE;
  const int64_t T = qkv->size(0), Hq = qkv->size(1) / cache.D - 2ll * cache.Hkv;
  if (Hq < 1 || (Hq + 2ll * cache.Hkv) * cache.D != qkv->size(1) || !plain(pos, at::kInt, idx) ||
      !plain(slot, at::kLong, idx) || !plain(freq, at::kFloat, idx) || pos->dim() < 1 ||
      pos->dim() > 2 || pos->size(pos->dim() - 1) != T || slot->dim() != 1 || slot->size(0) != T ||
      freq->dim() != 1 || freq->size(0) > 128)
    Py_RETURN_NONE;
  const int64_t axes = pos->dim() == 1 ? 1 : pos->size(0);
  if (axes < 1 || axes > 4) Py_RETURN_NONE;
  const unsigned char* map = nullptr;
  if (a[6] != Py_None) {
    if (!PyBytes_CheckExact(a[6]) || PyBytes_GET_SIZE(a[6]) != freq->size(0)) Py_RETURN_NONE;
    map = reinterpret_cast<const unsigned char*>(PyBytes_AS_STRING(a[6]));
  } else if (axes != 1) {
    Py_RETURN_NONE;
  }
  void* stream = nullptr;
  const int found = stream_of(idx, &stream);
  if (found < 0) return nullptr;
  if (found == 0) Py_RETURN_NONE;
  at::Tensor q = empty_on({T, Hq, cache.D}, type, idx);
  const void* xp = qkv->data_ptr();
  const long long row = T > 1 ? qkv->stride(0) : qkv->size(1);
  const int* pp = static_cast<const int*>(pos->data_ptr());
  const long long* sp = static_cast<const long long*>(slot->data_ptr());
  const float* fp = static_cast<const float*>(freq->data_ptr());
  const int rot = 2 * (int)freq->size(0), inter = a[7] == Py_True;
  void* qp = q.data_ptr();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = abi.rope_append(xp, row, pp, (int)axes, map, sp, fp, rot, inter, &cache, qp, (int)T,
                       (int)Hq, activation(type), stream);
  Py_END_ALLOW_THREADS
  if (rc != DB_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(q);
  END_HANDLE_TH_ERRORS
}

// (q, K, V, block_table, q_start, kv_len, scale or None, causal, window or None,
//  max_new or None, k_scale, v_scale): with a workspace that needs tickets outside
// capture only, and already in the cache.
PyObject* paged(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 12) Py_RETURN_NONE;
  const at::Tensor *q = tensor(a[0]), *table = tensor(a[3]), *start = tensor(a[4]),
                   *len = tensor(a[5]);
  if (!q || activation(q->scalar_type()) < 0 || !PyBool_Check(a[7])) Py_RETURN_NONE;
  const at::ScalarType type = q->scalar_type();
  if (!strided(q, type, 3, -1) || !ints(q)) Py_RETURN_NONE;
  const int idx = q->get_device();
  db_paged_cache cache;
  if (!paged_cache(a[1], a[2], a[10], a[11], type, idx, &cache)) Py_RETURN_NONE;
  const int64_t T = q->size(0), Hq = q->size(1), D = q->size(2);
  if (D != cache.D || D < 1 || !strided(table, at::kInt, 2, idx) || !ints(table) ||
      !plain(start, at::kInt, idx) || !plain(len, at::kInt, idx))
    Py_RETURN_NONE;
  const int64_t R = table->size(0), width = table->size(1);
  if (start->dim() != 1 || start->size(0) != R + 1 || len->dim() != 1 || len->size(0) != R)
    Py_RETURN_NONE;
  double scale = 1.0 / std::sqrt((double)D);
  long window = 0, most = T;
  if ((a[6] != Py_None && !number(a[6], &scale)) ||
      (a[8] != Py_None && (!integer(a[8], &window) || window < 1)) ||
      (a[9] != Py_None && (!integer(a[9], &most) || most < 1)))
    Py_RETURN_NONE;
  if (most > T) most = T;
  void* stream = nullptr;
  const int found = stream_of(idx, &stream);
  if (found < 0) return nullptr;
  if (found == 0) Py_RETURN_NONE;
  size_t zeroed = 0;
  const size_t bytes = abi.paged_workspace_bytes((int)T, (int)Hq, cache.Hkv, (int)D, (int)R,
                                                 (int)most, &zeroed);
  if (bytes == 0) Py_RETURN_NONE;
  at::Tensor ws;  // keeps the workspace alive through the call
  if (zeroed > 0) {
    unsigned long long capture = 0;
    if (abi.capture_id(stream, &capture) != DB_OK || capture != 0) Py_RETURN_NONE;
    PyObject* key = Py_BuildValue("(sKiKn)", "paged", (unsigned long long)zeroed, idx, (unsigned long long)(uintptr_t)stream,
                                  (Py_ssize_t)bytes);
    PyObject* hit = key ? PyDict_GetItemWithError(workspaces, key) : nullptr;  // borrowed
    Py_XDECREF(key);
    const at::Tensor* t = hit ? tensor(hit) : nullptr;
    if (!t) {
      if (PyErr_Occurred()) return nullptr;
      Py_RETURN_NONE;
    }
    ws = *t;
  } else {
    ws = empty_on({(int64_t)bytes}, at::kByte, idx);
  }
  at::Tensor o = empty_on({T, Hq, D}, type, idx);
  const void* qp = q->data_ptr();
  const long long qt = stride_of(q, 0), qh = stride_of(q, 1), row = stride_of(table, 0);
  const int *tp = static_cast<const int*>(table->data_ptr()),
            *sp = static_cast<const int*>(start->data_ptr()),
            *lp = static_cast<const int*>(len->data_ptr());
  void *op = o.data_ptr(), *wp = ws.data_ptr();
  const int causal = a[7] == Py_True;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = abi.paged_attention(qp, qt, qh, op, &cache, tp, row, (int)width, sp, lp, (int)T, (int)R,
                           (int)Hq, (int)most, (float)scale, causal, (int)window,
                           activation(type), wp, bytes, stream);
  Py_END_ALLOW_THREADS
  if (rc != DB_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(o);
  END_HANDLE_TH_ERRORS
}

// (entry point addresses, raw_stream, get_device, workspaces, cu_counts)
PyObject* init(PyObject*, PyObject* args) {
  unsigned long long p[14];
  PyObject *rs, *gd, *ws, *cu;
  if (!PyArg_ParseTuple(args, "(KKKKKKKKKKKKKK)OOO!O!", &p[0], &p[1], &p[2], &p[3], &p[4], &p[5],
                        &p[6], &p[7], &p[8], &p[9], &p[10], &p[11], &p[12], &p[13], &rs, &gd,
                        &PyDict_Type, &ws, &PyDict_Type, &cu))
    return nullptr;
  abi.f1 = reinterpret_cast<decltype(abi.f1)>((uintptr_t)p[0]);
  abi.f2 = reinterpret_cast<decltype(abi.f2)>((uintptr_t)p[1]);
  abi.f2n = reinterpret_cast<decltype(abi.f2n)>((uintptr_t)p[2]);
  abi.gemv = reinterpret_cast<decltype(abi.gemv)>((uintptr_t)p[3]);
  abi.f4_default_splits = reinterpret_cast<decltype(abi.f4_default_splits)>((uintptr_t)p[4]);
  abi.f4_workspace_bytes = reinterpret_cast<decltype(abi.f4_workspace_bytes)>((uintptr_t)p[5]);
  abi.f4 = reinterpret_cast<decltype(abi.f4)>((uintptr_t)p[6]);
  abi.capture_id = reinterpret_cast<decltype(abi.capture_id)>((uintptr_t)p[7]);
  abi.gemv_workspace_bytes = reinterpret_cast<decltype(abi.gemv_workspace_bytes)>((uintptr_t)p[8]);
  abi.gemv_ws = reinterpret_cast<decltype(abi.gemv_ws)>((uintptr_t)p[9]);
  abi.paged_plan = reinterpret_cast<decltype(abi.paged_plan)>((uintptr_t)p[10]);
  abi.rope_append = reinterpret_cast<decltype(abi.rope_append)>((uintptr_t)p[11]);
  abi.paged_workspace_bytes =
      reinterpret_cast<decltype(abi.paged_workspace_bytes)>((uintptr_t)p[12]);
  abi.paged_attention = reinterpret_cast<decltype(abi.paged_attention)>((uintptr_t)p[13]);
  Py_INCREF(rs);
  Py_INCREF(gd);
  Py_INCREF(ws);
  Py_INCREF(cu);
  Py_XSETREF(raw_stream, rs);
  Py_XSETREF(get_device, gd);
  Py_XSETREF(workspaces, ws);
  Py_XSETREF(cu_counts, cu);
  Py_RETURN_NONE;
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyCFunction fast() {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F));
}

PyMethodDef methods[] = {
    {"init", init, METH_VARARGS, nullptr},
    {"f1", fast<f1>(), METH_FASTCALL, nullptr},
    {"gemv", fast<gemv>(), METH_FASTCALL, nullptr},
    {"f2", fast<f2>(), METH_FASTCALL, nullptr},
    {"f2n", fast<f2n>(), METH_FASTCALL, nullptr},
    {"f4", fast<f4>(), METH_FASTCALL, nullptr},
    {"plan", fast<plan>(), METH_FASTCALL, nullptr},
    {"rope", fast<rope>(), METH_FASTCALL, nullptr},
    {"paged", fast<paged>(), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fastcall", nullptr, -1, methods,
                      nullptr,               nullptr,     nullptr, nullptr};

}  // namespace

// built_for names the torch and the Python whose object layouts this module
// holds; its functions are only called where both are the running ones.
PyMODINIT_FUNC PyInit__fastcall(void) {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "built_for", DB_BUILT_FOR) < 0) Py_CLEAR(m);
  return m;
}
