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
#include <torch/csrc/Dtype.h>
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
  decltype(&db_quantize_blocks) quantize_blocks;
  decltype(&db_gemm_blocks_workspace_bytes) gemm_blocks_workspace_bytes;
  decltype(&db_gemm_blocks) gemm_blocks;
  decltype(&db_moe_route_workspace_bytes) moe_route_workspace_bytes;
  decltype(&db_moe_route) moe_route;
  decltype(&db_moe_experts_workspace_bytes) moe_experts_workspace_bytes;
  decltype(&db_moe_experts) moe_experts;
  decltype(&db_moe_layer_workspace_bytes) moe_layer_workspace_bytes;
  decltype(&db_moe_layer) moe_layer;
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

// ------------------------------------- block-scaled e4m3, mixture of experts
int64_t blocks128(int64_t n) { return (n + 127) / 128; }

long long row_stride(const at::Tensor* t) { return t->size(0) > 1 ? t->stride(0) : t->size(1); }

bool codes(const at::Tensor* t, int idx) {
  return plain(t, at::kFloat8_e4m3fn, idx) || plain(t, at::kByte, idx);
}

// Rows of 16-bit activations [T, K].
const at::Tensor* rows16(PyObject* o, int* idx) {
  const at::Tensor* x = tensor(o);
  if (!x || activation(x->scalar_type()) < 0 || !strided(x, x->scalar_type(), 2, -1) || !ints(x))
    return nullptr;
  *idx = x->get_device();
  return x;
}

// (x): (q, scale)
PyObject* quantize_blocks(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  int idx = -1;
  const at::Tensor* x = n == 1 ? rows16(a[0], &idx) : nullptr;
  if (!x) Py_RETURN_NONE;
  void* stream = nullptr;
  const int found = stream_of(idx, &stream);
  if (found < 0) return nullptr;
  if (found == 0) Py_RETURN_NONE;
  const int64_t T = x->size(0), K = x->size(1);
  at::Tensor q = empty_on({T, K}, at::kFloat8_e4m3fn, idx);
  at::Tensor scale = empty_on({blocks128(K), T}, at::kFloat, idx).t();
  const void* xp = x->data_ptr();
  const long long row = row_stride(x);
  const int dtype = activation(x->scalar_type());
  void* qp = q.data_ptr();
  float* sp = static_cast<float*>(scale.data_ptr());
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = abi.quantize_blocks(xp, row, qp, sp, 1, T, (int)T, (int)K, dtype, stream);
  Py_END_ALLOW_THREADS
  if (rc != DB_OK) Py_RETURN_NONE;
  PyObject* result = PyTuple_New(2);
  if (!result) return nullptr;
  PyTuple_SET_ITEM(result, 0, THPVariable_Wrap(q));
  PyTuple_SET_ITEM(result, 1, THPVariable_Wrap(scale));
  return result;
  END_HANDLE_TH_ERRORS
}

// (x, W, w_scale, x_scale or None, dtype or None): x [T, K]
PyObject* gemm_blocks(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 5) Py_RETURN_NONE;
  const at::Tensor *x = tensor(a[0]), *w = tensor(a[1]), *ws = tensor(a[2]);
  if (!x || x->dim() != 2 || !x->is_cuda() || !ints(x)) Py_RETURN_NONE;
  const at::ScalarType type = x->scalar_type();
  const int idx = x->get_device();
  const bool fp8 = type == at::kFloat8_e4m3fn;
  if (!strided(x, type, 2, idx) || (!fp8 && activation(type) < 0)) Py_RETURN_NONE;
  const int64_t T = x->size(0), K = x->size(1);
  at::ScalarType out = fp8 ? at::kHalf : type;
  if (a[4] != Py_None) {
    if (!THPDtype_Check(a[4])) Py_RETURN_NONE;
    const at::ScalarType want = reinterpret_cast<THPDtype*>(a[4])->scalar_type;
    if (activation(want) < 0 || (!fp8 && want != type)) Py_RETURN_NONE;
    out = want;
  }
  const float* xs = nullptr;
  long long xs_t = 0, xs_b = 0;
  if (fp8) {
    const at::Tensor* s = tensor(a[3]);
    if (!s || !s->is_cuda() || s->get_device() != idx || s->scalar_type() != at::kFloat ||
        s->dim() != 2 || s->size(0) != T || s->size(1) != blocks128(K))
      Py_RETURN_NONE;
    xs = static_cast<const float*>(s->data_ptr());
    xs_t = stride_of(s, 0);
    xs_b = stride_of(s, 1);
  } else if (a[3] != Py_None) {
    Py_RETURN_NONE;
  }
  if (!codes(w, idx) || w->dim() != 2 || w->size(1) != K || !ints(w)) Py_RETURN_NONE;
  const int64_t N = w->size(0);
  if (!plain(ws, at::kFloat, idx) || ws->dim() != 2 || ws->size(0) != blocks128(N) ||
      ws->size(1) != blocks128(K))
    Py_RETURN_NONE;
  void* stream = nullptr;
  const int found = stream_of(idx, &stream);
  if (found < 0) return nullptr;
  if (found == 0) Py_RETURN_NONE;
  const int xdt = fp8 ? DB_DTYPE_FP8_E4M3 : activation(type), ydt = activation(out);
  at::Tensor y = empty_on({T, N}, out, idx);
  const size_t bytes = abi.gemm_blocks_workspace_bytes((int)T, (int)K, (int)N, xdt);
  at::Tensor work;
  if (bytes > 0) work = empty_here((int64_t)bytes, at::kByte, idx);
  const void *xp = x->data_ptr(), *wp = w->data_ptr();
  const float* wsp = static_cast<const float*>(ws->data_ptr());
  const long long row = row_stride(x);
  void *yp = y.data_ptr(), *kp = bytes > 0 ? work.data_ptr() : nullptr;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = abi.gemm_blocks(xp, row, xs, xs_t, xs_b, wp, wsp, yp, (int)T, (int)K, (int)N, xdt, ydt, kp,
                       bytes, stream);
  Py_END_ALLOW_THREADS
  if (rc != DB_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(y);
  END_HANDLE_TH_ERRORS
}

// (x, Wr, top_k, renormalize): (experts, weights)
PyObject* moe_route(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  int idx = -1;
  long k = 0;
  const at::Tensor* x = n == 4 ? rows16(a[0], &idx) : nullptr;
  if (!x || !integer(a[2], &k) || !PyBool_Check(a[3])) Py_RETURN_NONE;
  const at::Tensor* wr = tensor(a[1]);
  const int64_t T = x->size(0), H = x->size(1);
  if (!plain(wr, x->scalar_type(), idx) || wr->dim() != 2 || wr->size(1) != H || !ints(wr))
    Py_RETURN_NONE;
  void* stream = nullptr;
  const int found = stream_of(idx, &stream);
  if (found < 0) return nullptr;
  if (found == 0) Py_RETURN_NONE;
  const int E = (int)wr->size(0);
  if (k < 1 || k > E || k > 64) Py_RETURN_NONE;
  at::Tensor experts = empty_on({T, k}, at::kInt, idx), weights = empty_on({T, k}, at::kFloat, idx);
  const size_t bytes = abi.moe_route_workspace_bytes((int)T, (int)H, E);
  at::Tensor work;
  if (bytes > 0) work = empty_here((int64_t)bytes, at::kByte, idx);
  const void *xp = x->data_ptr(), *wp = wr->data_ptr();
  const long long row = row_stride(x);
  int* ep = static_cast<int*>(experts.data_ptr());
  float* sp = static_cast<float*>(weights.data_ptr());
  void* kp = bytes > 0 ? work.data_ptr() : nullptr;
  const int renormalize = a[3] == Py_True, dtype = activation(x->scalar_type());
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = abi.moe_route(xp, row, wp, ep, sp, (int)T, (int)H, E, (int)k, renormalize, dtype, kp, bytes,
                     stream);
  Py_END_ALLOW_THREADS
  if (rc != DB_OK) Py_RETURN_NONE;
  PyObject* result = PyTuple_New(2);
  if (!result) return nullptr;
  PyTuple_SET_ITEM(result, 0, THPVariable_Wrap(experts));
  PyTuple_SET_ITEM(result, 1, THPVariable_Wrap(weights));
  return result;
  END_HANDLE_TH_ERRORS
}

// The experts' weights (Wg, Wu, Wd) and scales (sg, su, sd) for activations of x's
// type and width.
bool experts_of(PyObject* const* w, PyObject* const* s, const at::Tensor* x, int idx, db_moe* m) {
  const at::Tensor *wg = tensor(w[0]), *wu = tensor(w[1]), *wd = tensor(w[2]);
  if (!wg) return false;
  const at::ScalarType type = wg->scalar_type();
  const int64_t H = x->size(1);
  if (!plain(wg, type, idx) || !plain(wu, type, idx) || !plain(wd, type, idx) || wg->dim() != 3 ||
      wg->size(2) != H || wu->sizes() != wg->sizes() || wd->dim() != 3 || !ints(wg))
    return false;
  const int64_t E = wg->size(0), I = wg->size(1);
  if (wd->size(0) != E || wd->size(1) != H || wd->size(2) != I) return false;
  *m = {};
  m->dtype = m->w_dtype = activation(x->scalar_type());
  if (type == at::kFloat8_e4m3fn || type == at::kByte) {
    m->w_dtype = DB_DTYPE_FP8_E4M3;
    const float** to[3] = {&m->sg, &m->su, &m->sd};
    for (int i = 0; i < 3; ++i) {
      const at::Tensor* t = tensor(s[i]);
      if (!plain(t, at::kFloat, idx) || t->dim() != 3 || t->size(0) != E ||
          t->size(1) != blocks128(i < 2 ? I : H) || t->size(2) != blocks128(i < 2 ? H : I))
        return false;
      *to[i] = static_cast<const float*>(t->data_ptr());
    }
  } else if (type != x->scalar_type() || s[0] != Py_None || s[1] != Py_None || s[2] != Py_None) {
    return false;
  }
  m->wg = wg->data_ptr();
  m->wu = wu->data_ptr();
  m->wd = wd->data_ptr();
  m->E = (int)E;
  m->H = (int)H;
  m->I = (int)I;
  return true;
}

// (x, experts, weights, Wg, Wu, Wd, sg, su, sd)
PyObject* moe_experts(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  int idx = -1;
  const at::Tensor* x = n == 9 ? rows16(a[0], &idx) : nullptr;
  if (!x) Py_RETURN_NONE;
  const at::Tensor *e = tensor(a[1]), *w = tensor(a[2]);
  const int64_t T = x->size(0);
  if (!plain(e, at::kInt, idx) || !plain(w, at::kFloat, idx) || e->dim() != 2 || e->size(0) != T ||
      w->sizes() != e->sizes() || !ints(e))
    Py_RETURN_NONE;
  db_moe m;
  if (!experts_of(a + 3, a + 6, x, idx, &m)) Py_RETURN_NONE;
  void* stream = nullptr;
  const int found = stream_of(idx, &stream);
  if (found < 0) return nullptr;
  if (found == 0) Py_RETURN_NONE;
  const int k = (int)e->size(1);
  const size_t bytes = abi.moe_experts_workspace_bytes(&m, (int)T, k);
  if (bytes == 0) Py_RETURN_NONE;
  at::Tensor y = empty_on({T, x->size(1)}, x->scalar_type(), idx);
  at::Tensor work = empty_here((int64_t)bytes, at::kByte, idx);
  const void* xp = x->data_ptr();
  const long long row = row_stride(x);
  const int* ep = static_cast<const int*>(e->data_ptr());
  const float* sp = static_cast<const float*>(w->data_ptr());
  void *yp = y.data_ptr(), *kp = work.data_ptr();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = abi.moe_experts(xp, row, ep, sp, &m, yp, (int)T, k, kp, bytes, stream);
  Py_END_ALLOW_THREADS
  if (rc != DB_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(y);
  END_HANDLE_TH_ERRORS
}

// (x, Wr, Wg, Wu, Wd, top_k, renormalize, sg, su, sd)
PyObject* moe_layer(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  int idx = -1;
  long k = 0;
  const at::Tensor* x = n == 10 ? rows16(a[0], &idx) : nullptr;
  if (!x || !integer(a[5], &k) || k < 1 || !PyBool_Check(a[6])) Py_RETURN_NONE;
  const at::Tensor* wr = tensor(a[1]);
  const int64_t T = x->size(0);
  db_moe m;
  if (!experts_of(a + 2, a + 7, x, idx, &m) || !plain(wr, x->scalar_type(), idx) ||
      wr->dim() != 2 || wr->size(0) != m.E || wr->size(1) != m.H || k > m.E)
    Py_RETURN_NONE;
  void* stream = nullptr;
  const int found = stream_of(idx, &stream);
  if (found < 0) return nullptr;
  if (found == 0) Py_RETURN_NONE;
  const size_t bytes = abi.moe_layer_workspace_bytes(&m, (int)T, (int)k);
  if (bytes == 0) Py_RETURN_NONE;
  at::Tensor y = empty_on({T, x->size(1)}, x->scalar_type(), idx);
  at::Tensor work = empty_here((int64_t)bytes, at::kByte, idx);
  const void *xp = x->data_ptr(), *wp = wr->data_ptr();
  const long long row = row_stride(x);
  const int renormalize = a[6] == Py_True;
  void *yp = y.data_ptr(), *kp = work.data_ptr();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = abi.moe_layer(xp, row, wp, &m, yp, (int)T, (int)k, renormalize, kp, bytes, stream);
  Py_END_ALLOW_THREADS
  if (rc != DB_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(y);
  END_HANDLE_TH_ERRORS
}

// Entry point i of the list that init is given.
template <class F>
bool entry(PyObject* list, Py_ssize_t i, F* to) {
  const unsigned long long p = PyLong_AsUnsignedLongLong(PyTuple_GET_ITEM(list, i));
  if (p == (unsigned long long)-1 && PyErr_Occurred()) return false;
  *to = reinterpret_cast<F>((uintptr_t)p);
  return true;
}

// (entry point addresses in the order of Abi, raw_stream, get_device, workspaces, cu_counts)
PyObject* init(PyObject*, PyObject* args) {
  PyObject *list, *rs, *gd, *ws, *cu;
  if (!PyArg_ParseTuple(args, "O!OOO!O!", &PyTuple_Type, &list, &rs, &gd, &PyDict_Type, &ws,
                        &PyDict_Type, &cu))
    return nullptr;
  if (PyTuple_GET_SIZE(list) != 23) {
    PyErr_SetString(PyExc_ValueError, "init takes 23 entry points");
    return nullptr;
  }
  Abi e;
  if (!entry(list, 0, &e.f1) || !entry(list, 1, &e.f2) || !entry(list, 2, &e.f2n) ||
      !entry(list, 3, &e.gemv) || !entry(list, 4, &e.f4_default_splits) ||
      !entry(list, 5, &e.f4_workspace_bytes) || !entry(list, 6, &e.f4) ||
      !entry(list, 7, &e.capture_id) || !entry(list, 8, &e.gemv_workspace_bytes) ||
      !entry(list, 9, &e.gemv_ws) || !entry(list, 10, &e.paged_plan) ||
      !entry(list, 11, &e.rope_append) || !entry(list, 12, &e.paged_workspace_bytes) ||
      !entry(list, 13, &e.paged_attention) || !entry(list, 14, &e.quantize_blocks) ||
      !entry(list, 15, &e.gemm_blocks_workspace_bytes) || !entry(list, 16, &e.gemm_blocks) ||
      !entry(list, 17, &e.moe_route_workspace_bytes) || !entry(list, 18, &e.moe_route) ||
      !entry(list, 19, &e.moe_experts_workspace_bytes) || !entry(list, 20, &e.moe_experts) ||
      !entry(list, 21, &e.moe_layer_workspace_bytes) || !entry(list, 22, &e.moe_layer))
    return nullptr;
  abi = e;
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
    {"quantize_blocks", fast<quantize_blocks>(), METH_FASTCALL, nullptr},
    {"gemm_blocks", fast<gemm_blocks>(), METH_FASTCALL, nullptr},
    {"moe_route", fast<moe_route>(), METH_FASTCALL, nullptr},
    {"moe_experts", fast<moe_experts>(), METH_FASTCALL, nullptr},
    {"moe_layer", fast<moe_layer>(), METH_FASTCALL, nullptr},
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
