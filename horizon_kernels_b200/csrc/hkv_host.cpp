// Native side of kernels.write, kernels.decode_ragged, kernels.prefill, their window forms, kernels.accumulate_weights,
// kernels.evict, the writes with a rotation, the calls of the 8-bit cache, and of the backend's cache update and decode: takes the callers' Python arguments as they are, checks them and calls the C ABI (include/hkv.h). What the wrappers do per call in
// Python (about forty attribute reads and checks, a device context, the conversion of 25 ctypes arguments) costs 20 to 25
// microseconds, longer than a small decode step runs on the GPU; here it costs two.
//
// Each function answers None when an argument is not of the plain form it knows (wrong type, shape or device, a tensor
// subclass, anything that throws): nothing has been launched then, and the Python path checks, raises or serves the
// call. Otherwise it answers the status of the C call. No state is kept between calls.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/Functions.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <type_traits>
#include <utility>
#include <vector>

#include "../../include/hkv.h"

namespace {

struct Abi {                       // entry points of the loaded libhkv.so, handed over by bind()
  decltype(&hkv_write) write = nullptr;
  decltype(&hkv_write_rot) write_rot = nullptr;
  decltype(&hkv_write_k8) write_k8 = nullptr;
  decltype(&hkv_decode) decode = nullptr;
  decltype(&hkv_decode_rot) decode_rot = nullptr;
  decltype(&hkv_decode_k8) decode_k8 = nullptr;
  decltype(&hkv_prefill_scratch_bytes) prefill_scratch_bytes = nullptr;
  decltype(&hkv_prefill) prefill = nullptr;
  decltype(&hkv_decode_window) decode_window = nullptr;
  decltype(&hkv_prefill_window_scratch_bytes) prefill_window_scratch_bytes = nullptr;
  decltype(&hkv_prefill_window) prefill_window = nullptr;
  decltype(&hkv_accumulate_weights) accumulate_weights = nullptr;
  decltype(&hkv_evict) evict = nullptr;
  decltype(&hkv_write_rotary) write_rotary = nullptr;
  decltype(&hkv_write_b8) write_b8 = nullptr;
  decltype(&hkv_decode_b8) decode_b8 = nullptr;
  decltype(&hkv_prefill_b8) prefill_b8 = nullptr;
} abi;

const at::Tensor* tensor(PyObject* o) { return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr; }

bool integer(PyObject* o, long long* v) {
  if (!PyLong_CheckExact(o)) return false;
  *v = PyLong_AsLongLong(o);
  if (*v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}
bool number(PyObject* o, double* v) {
  if (!PyFloat_CheckExact(o)) return false;
  *v = PyFloat_AS_DOUBLE(o);
  return true;
}
bool boolean(PyObject* o, bool* v) {
  if (!PyBool_Check(o)) return false;
  *v = o == Py_True;
  return true;
}
bool on(const at::Tensor& t, int dev) { return t.is_cuda() && t.device().index() == dev; }

struct Cache {
  void* part[4];
  int64_t strides[6];
};
bool cache_of(PyObject* flat, PyObject* strides, int dev, Cache* c) {
  if (!PyTuple_CheckExact(flat) || PyTuple_GET_SIZE(flat) != 4 || !PyTuple_CheckExact(strides) || PyTuple_GET_SIZE(strides) != 6)
    return false;
  for (int i = 0; i < 4; ++i) {
    const at::Tensor* t = tensor(PyTuple_GET_ITEM(flat, i));
    if (!t || !on(*t, dev)) return false;
    c->part[i] = t->data_ptr();
  }
  for (int i = 0; i < 6; ++i) {
    long long v;
    if (!integer(PyTuple_GET_ITEM(strides, i), &v)) return false;
    c->strides[i] = v;
  }
  return true;
}
// per-head scales and, with rotated keys, the sign vector
bool scales(const at::Tensor* gk, const at::Tensor* gv, int64_t KVH, int dev) {
  for (const at::Tensor* t : {gk, gv})
    if (!t || !on(*t, dev) || t->scalar_type() != at::kFloat || t->dim() != 1 || t->size(0) != KVH || !t->is_contiguous()) return false;
  return true;
}
bool sign_vector(PyObject* o, int64_t D, int dev, const float** p) {
  *p = nullptr;
  if (o == Py_None) return true;
  const at::Tensor* t = tensor(o);
  if (!t || !on(*t, dev) || t->scalar_type() != at::kFloat || t->dim() != 1 || t->size(0) != D || !t->is_contiguous()) return false;
  *p = static_cast<const float*>(t->data_ptr());
  return true;
}

// a sliding window, the tokens that stay visible before it, and where the log-sum-exps go
struct Window {
  int window, sinks;
  float* lse;
};
bool lse_rows(const at::Tensor* t, int64_t NT, int64_t HQ, int dev) {
  return t && on(*t, dev) && t->scalar_type() == at::kFloat && t->dim() == 2 && t->size(0) >= NT && t->size(1) == HQ && t->is_contiguous();
}
bool window_of(PyObject* window, PyObject* sinks, PyObject* lse, int64_t NT, int64_t HQ, int dev, Window* w) {
  long long a, b;
  if (!integer(window, &a) || !integer(sinks, &b) || a < 0 || b < 0 || a > INT32_MAX || b > INT32_MAX) return false;
  w->window = (int)a;
  w->sinks = (int)b;
  w->lse = nullptr;
  if (lse == Py_None) return true;
  const at::Tensor* t = tensor(lse);
  if (!lse_rows(t, NT, HQ, dev)) return false;
  w->lse = static_cast<float*>(t->data_ptr());
  return true;
}
// (B, KVH, W) fp32 rows that do not overlap
bool weight_rows(const at::Tensor* t, int64_t B, int64_t KVH, int dev) {
  if (!t || !on(*t, dev) || t->scalar_type() != at::kFloat || t->dim() != 3 || t->size(0) != B || t->size(1) != KVH || t->size(2) > INT32_MAX)
    return false;
  const int64_t W = t->size(2), sb = t->stride(0), sh = t->stride(1);
  if (sb < 0 || sh < 0 || (t->stride(2) != 1 && W > 1)) return false;
  return ((KVH <= 1 || (sh > 0 && sh >= W)) && (B <= 1 || (sb > 0 && sb >= (KVH - 1) * sh + W))) ||
         ((B <= 1 || (sb > 0 && sb >= W)) && (KVH <= 1 || (sh > 0 && sh >= (B - 1) * sb + W)));
}

// the 8-bit cache: key tiles and value tiles, strides (page, head)
struct Tiles {
  void *k, *v;
  int64_t strides[2];
};
bool tiles_of(PyObject* flat, PyObject* strides, int dev, Tiles* c) {
  if (!PyTuple_CheckExact(flat) || PyTuple_GET_SIZE(flat) != 2 || !PyTuple_CheckExact(strides) || PyTuple_GET_SIZE(strides) != 2) return false;
  const at::Tensor *k = tensor(PyTuple_GET_ITEM(flat, 0)), *v = tensor(PyTuple_GET_ITEM(flat, 1));
  if (!k || !v || !on(*k, dev) || !on(*v, dev)) return false;
  c->k = k->data_ptr();
  c->v = v->data_ptr();
  for (int i = 0; i < 2; ++i) {
    long long s;
    if (!integer(PyTuple_GET_ITEM(strides, i), &s)) return false;
    c->strides[i] = s;
  }
  return true;
}
bool format_of(PyObject* o, int* fmt) {
  if (!PyUnicode_CheckExact(o)) return false;
  *fmt = PyUnicode_CompareWithASCIIString(o, "e4m3") == 0 ? HKV_B8_E4M3 : PyUnicode_CompareWithASCIIString(o, "int8") == 0 ? HKV_B8_INT8 : -1;
  return *fmt >= 0;
}
// keys and values of a write, and their slots
bool new_rows(const at::Tensor* k, const at::Tensor* v, const at::Tensor* slots, int dev) {
  return k && v && slots && on(*k, dev) && on(*v, dev) && on(*slots, dev) && k->scalar_type() == at::kBFloat16 &&
         v->scalar_type() == at::kBFloat16 && k->dim() == 3 && v->sizes() == k->sizes() && k->stride(2) == 1 && v->stride(2) == 1 &&
         slots->scalar_type() == at::kLong && slots->dim() == 1 && slots->is_contiguous() && slots->size(0) <= k->size(0) &&
         k->size(1) <= INT32_MAX && k->size(2) <= INT32_MAX;
}
// query, positions, table and where the turned queries go (the C call refuses rows that overlap)
bool rotary_of(const at::Tensor* q, const at::Tensor* k, const at::Tensor* slots, PyObject* positions, PyObject* table, PyObject* out,
               PyObject* interleaved, int dev, hkv_rotary* r) {
  const at::Tensor *pos = tensor(positions), *t = tensor(table), *o = tensor(out);
  bool pairs;
  if (!q || !pos || !t || !o || !on(*q, dev) || !on(*pos, dev) || !on(*t, dev) || !on(*o, dev) || !boolean(interleaved, &pairs) ||
      q->scalar_type() != at::kBFloat16 || o->scalar_type() != at::kBFloat16 || q->dim() != 3 || o->sizes() != q->sizes() ||
      q->size(2) != k->size(2) || q->stride(2) != 1 || o->stride(2) != 1 || pos->scalar_type() != at::kLong || pos->dim() != 1 ||
      !pos->is_contiguous() || pos->size(0) != q->size(0) || slots->size(0) > q->size(0) || t->dim() != 2 || !t->is_contiguous() ||
      (t->scalar_type() != at::kFloat && t->scalar_type() != at::kBFloat16) || t->size(1) % 16 || t->size(1) < 16 ||
      t->size(1) > k->size(2) || q->size(1) > INT32_MAX)
    return false;
  *r = hkv_rotary{q->data_ptr(), q->stride(0), q->stride(1), o->data_ptr(), o->stride(0), o->stride(1), q->size(0),
                  static_cast<const int64_t*>(pos->data_ptr()), t->data_ptr(), t->size(0), (int)q->size(1), (int)t->size(1),
                  t->scalar_type() == at::kBFloat16, pairs};
  return true;
}

// The launches behind the checks. Cache parts and strides as in include/hkv.h.
struct Rows {                      // new keys and values
  const void *k, *v;
  int64_t k0, k1, v0, v1, KVH, D;
};
PyObject* run_write(const Rows& r, const Cache& c, int PS, const at::Tensor& slots, const at::Tensor& gk, const at::Tensor& gv, bool search,
                    const float* signs, bool k8, int dev) {
  const int64_t *sl = static_cast<const int64_t*>(slots.data_ptr()), n_slots = slots.size(0);
  const float *gkp = static_cast<const float*>(gk.data_ptr()), *gvp = static_cast<const float*>(gv.data_ptr());
  void* st = c10::cuda::getCurrentCUDAStream(dev).stream();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  if (k8)
    rc = abi.write_k8(r.k, r.v, r.k0, r.k1, r.v0, r.v1, c.part[0], c.part[2], c.part[3], c.strides, PS, sl, n_slots, gkp, gvp,
                      (int)r.KVH, (int)r.D, search, st);
  else if (signs)
    rc = abi.write_rot(r.k, r.v, r.k0, r.k1, r.v0, r.v1, c.part[0], c.part[1], c.part[2], c.part[3], c.strides, PS, sl, n_slots, gkp,
                       gvp, (int)r.KVH, (int)r.D, search, signs, st);
  else
    rc = abi.write(r.k, r.v, r.k0, r.k1, r.v0, r.v1, c.part[0], c.part[1], c.part[2], c.part[3], c.strides, PS, sl, n_slots, gkp, gvp,
                   (int)r.KVH, (int)r.D, search, st);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}
PyObject* run_decode(const void* q, const Cache& c, int PS, const at::Tensor& bt, const at::Tensor& lens, const at::Tensor& qsl, int64_t HQ,
                     int64_t D, double s1, double s2, const at::Tensor& gk, const at::Tensor& gv, int qlmax, void* out,
                     const at::Tensor& ws, int splits, const float* signs, bool k8, int dev, const Window* win = nullptr) {
  const int32_t *btp = static_cast<const int32_t*>(bt.data_ptr()), *lp = static_cast<const int32_t*>(lens.data_ptr()),
                *sp = static_cast<const int32_t*>(qsl.data_ptr());
  const float *gkp = static_cast<const float*>(gk.data_ptr()), *gvp = static_cast<const float*>(gv.data_ptr());
  void* wp = ws.data_ptr();
  const size_t wsb = ws.nbytes();
  const int B = (int)bt.size(0), MP = (int)bt.size(1), KVH = (int)gk.size(0), G = (int)(HQ / KVH);
  void* st = c10::cuda::getCurrentCUDAStream(dev).stream();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  if (win)
    rc = abi.decode_window(q, c.part[0], c.part[1], c.part[2], c.part[3], c.strides, PS, btp, MP, lp, sp, B, KVH, G, (int)D, qlmax,
                           (float)s1, (float)s2, gkp, gvp, wp, wsb, splits, signs, k8, win->window, win->sinks, win->lse, out, st);
  else if (k8)
    rc = abi.decode_k8(q, c.part[0], c.part[2], c.part[3], c.strides, PS, btp, MP, lp, sp, B, KVH, G, (int)D, qlmax, (float)s1,
                       (float)s2, gkp, gvp, wp, wsb, splits, out, st);
  else if (signs)
    rc = abi.decode_rot(q, c.part[0], c.part[1], c.part[2], c.part[3], c.strides, PS, btp, MP, lp, sp, B, KVH, G, (int)D, qlmax,
                        (float)s1, (float)s2, gkp, gvp, wp, wsb, splits, signs, out, st);
  else
    rc = abi.decode(q, c.part[0], c.part[1], c.part[2], c.part[3], c.strides, PS, btp, MP, lp, sp, B, KVH, G, (int)D, qlmax, (float)s1,
                    (float)s2, gkp, gvp, wp, wsb, splits, out, st);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}
// parts and strides of the logical (pages, heads, positions, slot) cache that the engine holds, as layout.slot_views /
// flat_views (K8: k8_views / k8_flat_views) give them
bool cache_of_slots(PyObject* o, int64_t KVH, int64_t D, bool k8, int dev, Cache* c, int* PS) {
  const at::Tensor* t = tensor(o);
  if (!t || !on(*t, dev) || t->scalar_type() != at::kByte || t->dim() != 4 || (D != 128 && D != 256)) return false;
  const int64_t slot = (k8 ? D : 0) + D / 2 + D / 16;
  if (t->size(1) != (k8 ? KVH : 2 * KVH) || t->size(3) != slot || t->stride(3) != 1 || t->size(2) > INT32_MAX) return false;
  uint8_t* p = static_cast<uint8_t*>(t->data_ptr());
  uint8_t* v = k8 ? p + D : p + KVH * t->stride(1);
  c->part[0] = p;
  c->part[1] = k8 ? v + D / 2 : p + D / 2;
  c->part[2] = v;
  c->part[3] = v + D / 2;
  for (int i = 0; i < 6; i += 3) {
    c->strides[i] = t->stride(0);
    c->strides[i + 1] = t->stride(2);
    c->strides[i + 2] = t->stride(1);
  }
  *PS = (int)t->size(2);
  return true;
}
// (tokens, heads * D) or (tokens, heads, D) bf16
bool token_rows(const at::Tensor& t, int64_t heads, int64_t D) {
  return t.scalar_type() == at::kBFloat16 && ((t.dim() == 2 && t.size(1) == heads * D) || (t.dim() == 3 && t.size(1) == heads && t.size(2) == D));
}

// write(key, value, flat, strides, PS, slot_mapping, gk, gv, search, signs, k8)
PyObject* write(PyObject*, PyObject* const* a, Py_ssize_t n) {
  try {
    if (n != 11 || !abi.write) Py_RETURN_NONE;
    const at::Tensor *k = tensor(a[0]), *v = tensor(a[1]), *slots = tensor(a[5]), *gk = tensor(a[6]), *gv = tensor(a[7]);
    if (!k || !v || !slots || !k->is_cuda()) Py_RETURN_NONE;
    const int dev = k->device().index();
    long long PS;
    bool search, k8;
    const float* signs;
    Cache c;
    if (dev != c10::cuda::current_device() || !on(*v, dev) || !on(*slots, dev) || k->scalar_type() != at::kBFloat16 ||
        v->scalar_type() != at::kBFloat16 || k->dim() != 3 || v->sizes() != k->sizes() || k->stride(2) != 1 || v->stride(2) != 1 ||
        slots->scalar_type() != at::kLong || slots->dim() != 1 || !slots->is_contiguous() || slots->size(0) > k->size(0) ||
        !integer(a[4], &PS) || PS != (int)PS || !boolean(a[8], &search) || !boolean(a[10], &k8))
      Py_RETURN_NONE;
    const int64_t KVH = k->size(1), D = k->size(2);
    if (KVH > INT32_MAX || D > INT32_MAX || !scales(gk, gv, KVH, dev) || !sign_vector(a[9], D, dev, &signs) || (k8 && signs) ||
        !cache_of(a[2], a[3], dev, &c))
      Py_RETURN_NONE;
    return run_write({k->data_ptr(), v->data_ptr(), k->stride(0), k->stride(1), v->stride(0), v->stride(1), KVH, D}, c, (int)PS, *slots, *gk,
                     *gv, search, signs, k8, dev);
  } catch (...) {
    Py_RETURN_NONE;
  }
}

// decode(query, flat, strides, PS, block_tables, seq_lens, query_start_loc, bmm1_scale, bmm2_scale, gk, gv, qlmax, out,
//        workspace, splits, signs, k8); decode_window: .., window, sinks, lse
template <bool WIN>
PyObject* decode_any(PyObject*, PyObject* const* a, Py_ssize_t n) {
  try {
    if (n != (WIN ? 20 : 17) || !abi.decode) Py_RETURN_NONE;
    const at::Tensor *q = tensor(a[0]), *bt = tensor(a[4]), *lens = tensor(a[5]), *qsl = tensor(a[6]), *gk = tensor(a[9]),
                     *gv = tensor(a[10]), *out = tensor(a[12]), *ws = tensor(a[13]);
    if (!q || !bt || !lens || !qsl || !gk || !out || !ws || !q->is_cuda() || gk->dim() != 1) Py_RETURN_NONE;
    const int dev = q->device().index();
    long long PS, qlmax, splits = 0;
    double s1, s2;
    bool k8;
    const float* signs;
    Cache c;
    if (dev != c10::cuda::current_device() || !integer(a[3], &PS) || PS != (int)PS || !number(a[7], &s1) || !number(a[8], &s2) ||
        !integer(a[11], &qlmax) || qlmax != (int)qlmax || (a[14] != Py_None && (!integer(a[14], &splits) || splits != (int)splits)) ||
        !boolean(a[16], &k8))
      Py_RETURN_NONE;
    if (q->scalar_type() != at::kBFloat16 || out->scalar_type() != at::kBFloat16 || q->dim() != 3 || out->dim() != 3 ||
        out->size(1) != q->size(1) || out->size(2) != q->size(2) || out->size(0) < q->size(0) || !q->is_contiguous() ||
        !out->is_contiguous() || bt->dim() != 2 || lens->dim() != 1 || qsl->dim() != 1 || lens->size(0) != bt->size(0) ||
        qsl->size(0) != bt->size(0) + 1 || !on(*out, dev) || !on(*ws, dev))
      Py_RETURN_NONE;
    for (const at::Tensor* t : {bt, lens, qsl})
      if (!on(*t, dev) || t->scalar_type() != at::kInt || !t->is_contiguous()) Py_RETURN_NONE;
    const int64_t B = bt->size(0), MP = bt->size(1), KVH = gk->size(0), HQ = q->size(1), D = q->size(2);
    if (KVH < 1 || HQ % KVH || B > INT32_MAX || MP > INT32_MAX || HQ > INT32_MAX || D > INT32_MAX || !scales(gk, gv, KVH, dev) ||
        !sign_vector(a[15], D, dev, &signs) || (k8 && signs) || !cache_of(a[1], a[2], dev, &c))
      Py_RETURN_NONE;
    Window w;
    if (WIN && !window_of(a[17], a[18], a[19], q->size(0), HQ, dev, &w)) Py_RETURN_NONE;
    return run_decode(q->data_ptr(), c, (int)PS, *bt, *lens, *qsl, HQ, D, s1, s2, *gk, *gv, (int)qlmax, out->data_ptr(), *ws, (int)splits, signs,
                      k8, dev, WIN ? &w : nullptr);
  } catch (...) {
    Py_RETURN_NONE;
  }
}

// write_rotary(query, key, value, flat, strides, PS, slot_mapping, positions, cos_sin, gk, gv, query_out, interleaved, search, signs, k8)
PyObject* write_rotary(PyObject*, PyObject* const* a, Py_ssize_t n) {
  try {
    if (n != 16 || !abi.write_rotary) Py_RETURN_NONE;
    const at::Tensor *q = tensor(a[0]), *k = tensor(a[1]), *v = tensor(a[2]), *slots = tensor(a[6]), *gk = tensor(a[9]), *gv = tensor(a[10]);
    if (!k || !k->is_cuda()) Py_RETURN_NONE;
    const int dev = k->device().index();
    long long PS;
    bool search, k8;
    const float* signs;
    Cache c;
    hkv_rotary r;
    if (dev != c10::cuda::current_device() || !new_rows(k, v, slots, dev) || !integer(a[5], &PS) || PS != (int)PS || !boolean(a[13], &search) ||
        !boolean(a[15], &k8) || !scales(gk, gv, k->size(1), dev) || !sign_vector(a[14], k->size(2), dev, &signs) || (k8 && signs) ||
        !cache_of(a[3], a[4], dev, &c) || !rotary_of(q, k, slots, a[7], a[8], a[11], a[12], dev, &r))
      Py_RETURN_NONE;
    const void *kp = k->data_ptr(), *vp = v->data_ptr();
    const int64_t k0 = k->stride(0), k1 = k->stride(1), v0 = v->stride(0), v1 = v->stride(1), n_slots = slots->size(0);
    const int64_t* sl = static_cast<const int64_t*>(slots->data_ptr());
    const float *gkp = static_cast<const float*>(gk->data_ptr()), *gvp = static_cast<const float*>(gv->data_ptr());
    const int KVH = (int)k->size(1), D = (int)k->size(2);
    void* st = c10::cuda::getCurrentCUDAStream(dev).stream();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = abi.write_rotary(kp, vp, k0, k1, v0, v1, c.part[0], c.part[1], c.part[2], c.part[3], c.strides, (int)PS, sl, n_slots, gkp, gvp,
                          KVH, D, search, signs, k8, &r, st);
    Py_END_ALLOW_THREADS
    if (rc == HKV_ERR_RANGE) Py_RETURN_NONE;          // (the Python path says which rows overlap)
    return PyLong_FromLong(rc);
  } catch (...) {
    Py_RETURN_NONE;
  }
}

// write_b8(key, value, flat, strides, PS, slot_mapping, gk, gv, fmt)
// write_rotary_b8(query, key, value, flat, strides, PS, slot_mapping, positions, cos_sin, gk, gv, query_out, interleaved, fmt)
template <bool ROT>
PyObject* write_b8_any(PyObject*, PyObject* const* a, Py_ssize_t n) {
  try {
    if (n != (ROT ? 14 : 9) || !abi.write_b8) Py_RETURN_NONE;
    PyObject* const* b = a + (ROT ? 1 : 0);            // key, value, flat, strides, PS, slot_mapping
    PyObject* const* s = ROT ? a + 9 : a + 6;          // gk, gv
    const at::Tensor *k = tensor(b[0]), *v = tensor(b[1]), *slots = tensor(b[5]), *gk = tensor(s[0]), *gv = tensor(s[1]);
    if (!k || !k->is_cuda()) Py_RETURN_NONE;
    const int dev = k->device().index();
    long long PS;
    int fmt;
    Tiles c;
    hkv_rotary r;
    if (dev != c10::cuda::current_device() || !new_rows(k, v, slots, dev) || !integer(b[4], &PS) || PS != (int)PS ||
        !format_of(a[n - 1], &fmt) || !scales(gk, gv, k->size(1), dev) || !tiles_of(b[2], b[3], dev, &c) ||
        (ROT && !rotary_of(tensor(a[0]), k, slots, a[7], a[8], a[11], a[12], dev, &r)))
      Py_RETURN_NONE;
    const void *kp = k->data_ptr(), *vp = v->data_ptr();
    const int64_t k0 = k->stride(0), k1 = k->stride(1), v0 = v->stride(0), v1 = v->stride(1), n_slots = slots->size(0);
    const int64_t* sl = static_cast<const int64_t*>(slots->data_ptr());
    const float *gkp = static_cast<const float*>(gk->data_ptr()), *gvp = static_cast<const float*>(gv->data_ptr());
    const int KVH = (int)k->size(1), D = (int)k->size(2);
    void* st = c10::cuda::getCurrentCUDAStream(dev).stream();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = abi.write_b8(kp, vp, k0, k1, v0, v1, c.k, c.v, c.strides, (int)PS, sl, n_slots, gkp, gvp, KVH, D, fmt, ROT ? &r : nullptr, st);
    Py_END_ALLOW_THREADS
    if (ROT && rc == HKV_ERR_RANGE) Py_RETURN_NONE;    // (as above)
    return PyLong_FromLong(rc);
  } catch (...) {
    Py_RETURN_NONE;
  }
}

// decode_b8(query, flat, strides, PS, block_tables, seq_lens, query_start_loc, bmm1_scale, bmm2_scale, gk, gv, qlmax, out, workspace, fmt,
//           window, sinks, splits, lse)
PyObject* decode_b8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  try {
    if (n != 19 || !abi.decode_b8) Py_RETURN_NONE;
    const at::Tensor *q = tensor(a[0]), *bt = tensor(a[4]), *lens = tensor(a[5]), *qsl = tensor(a[6]), *gk = tensor(a[9]),
                     *gv = tensor(a[10]), *out = tensor(a[12]), *ws = tensor(a[13]);
    if (!q || !bt || !lens || !qsl || !gk || !out || !ws || !q->is_cuda() || gk->dim() != 1) Py_RETURN_NONE;
    const int dev = q->device().index();
    long long PS, qlmax, splits = 0;
    double s1, s2;
    int fmt;
    Tiles c;
    Window w;
    if (dev != c10::cuda::current_device() || !integer(a[3], &PS) || PS != (int)PS || !number(a[7], &s1) || !number(a[8], &s2) ||
        !integer(a[11], &qlmax) || qlmax != (int)qlmax || !format_of(a[14], &fmt) ||
        (a[17] != Py_None && (!integer(a[17], &splits) || splits != (int)splits)))
      Py_RETURN_NONE;
    if (q->scalar_type() != at::kBFloat16 || out->scalar_type() != at::kBFloat16 || q->dim() != 3 || out->dim() != 3 ||
        out->size(1) != q->size(1) || out->size(2) != q->size(2) || out->size(0) < q->size(0) || !q->is_contiguous() ||
        !out->is_contiguous() || bt->dim() != 2 || lens->dim() != 1 || qsl->dim() != 1 || lens->size(0) != bt->size(0) ||
        qsl->size(0) != bt->size(0) + 1 || !on(*out, dev) || !on(*ws, dev))
      Py_RETURN_NONE;
    for (const at::Tensor* t : {bt, lens, qsl})
      if (!on(*t, dev) || t->scalar_type() != at::kInt || !t->is_contiguous()) Py_RETURN_NONE;
    const int64_t B = bt->size(0), MP = bt->size(1), KVH = gk->size(0), HQ = q->size(1), D = q->size(2);
    if (KVH < 1 || HQ % KVH || B > INT32_MAX || MP > INT32_MAX || HQ > INT32_MAX || D > INT32_MAX || !scales(gk, gv, KVH, dev) ||
        !tiles_of(a[1], a[2], dev, &c) || !window_of(a[15], a[16], a[18], q->size(0), HQ, dev, &w))
      Py_RETURN_NONE;
    const void* qp = q->data_ptr();
    const int32_t *btp = static_cast<const int32_t*>(bt->data_ptr()), *lp = static_cast<const int32_t*>(lens->data_ptr()),
                  *sp = static_cast<const int32_t*>(qsl->data_ptr());
    const float *gkp = static_cast<const float*>(gk->data_ptr()), *gvp = static_cast<const float*>(gv->data_ptr());
    void *op = out->data_ptr(), *wp = ws->data_ptr(), *st = c10::cuda::getCurrentCUDAStream(dev).stream();
    const size_t wsb = ws->nbytes();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = abi.decode_b8(qp, c.k, c.v, c.strides, (int)PS, btp, (int)MP, lp, sp, (int)B, (int)KVH, (int)(HQ / KVH), (int)D, (int)qlmax,
                       (float)s1, (float)s2, gkp, gvp, wp, wsb, (int)splits, fmt, w.window, w.sinks, w.lse, op, st);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
  } catch (...) {
    Py_RETURN_NONE;
  }
}

// accumulate_weights(query, flat, strides, PS, block_tables, seq_lens, query_start_loc, bmm1_scale, gk, qlmax, lse, weights, window,
//                    sinks, signs, k8, workspace)
PyObject* accumulate_weights(PyObject*, PyObject* const* a, Py_ssize_t n) {
  try {
    if (n != 17 || !abi.accumulate_weights) Py_RETURN_NONE;
    const at::Tensor *q = tensor(a[0]), *bt = tensor(a[4]), *lens = tensor(a[5]), *qsl = tensor(a[6]), *gk = tensor(a[8]),
                     *wt = tensor(a[11]), *ws = a[16] == Py_None ? nullptr : tensor(a[16]);
    if (!q || !bt || !lens || !qsl || !gk || !wt || (!ws && a[16] != Py_None) || !q->is_cuda() || gk->dim() != 1) Py_RETURN_NONE;
    const int dev = q->device().index();
    long long PS, qlmax;
    double s1;
    bool k8;
    const float* signs;
    Cache c;
    Window w;
    if (dev != c10::cuda::current_device() || !integer(a[3], &PS) || PS != (int)PS || !number(a[7], &s1) || !integer(a[9], &qlmax) ||
        qlmax != (int)qlmax || !boolean(a[15], &k8) || q->scalar_type() != at::kBFloat16 || q->dim() != 3 || !q->is_contiguous() ||
        bt->dim() != 2 || lens->dim() != 1 || qsl->dim() != 1 || lens->size(0) != bt->size(0) || qsl->size(0) != bt->size(0) + 1 ||
        (ws && (!on(*ws, dev) || ws->nbytes() < 64)))
      Py_RETURN_NONE;
    for (const at::Tensor* t : {bt, lens, qsl})
      if (!on(*t, dev) || t->scalar_type() != at::kInt || !t->is_contiguous()) Py_RETURN_NONE;
    const int64_t B = bt->size(0), MP = bt->size(1), KVH = gk->size(0), HQ = q->size(1), D = q->size(2);
    if (KVH < 1 || HQ % KVH || B > INT32_MAX || MP > INT32_MAX || HQ > INT32_MAX || D > INT32_MAX || !scales(gk, gk, KVH, dev) ||
        !sign_vector(a[14], D, dev, &signs) || (k8 && signs) || !cache_of(a[1], a[2], dev, &c) || a[10] == Py_None ||
        !window_of(a[12], a[13], a[10], q->size(0), HQ, dev, &w) || !weight_rows(wt, B, KVH, dev))
      Py_RETURN_NONE;
    const void* qp = q->data_ptr();
    const int32_t *btp = static_cast<const int32_t*>(bt->data_ptr()), *lp = static_cast<const int32_t*>(lens->data_ptr()),
                  *sp = static_cast<const int32_t*>(qsl->data_ptr());
    const float* gkp = static_cast<const float*>(gk->data_ptr());
    float* wtp = static_cast<float*>(wt->data_ptr());
    const int64_t wb = wt->stride(0), wh = wt->stride(1);
    const int W = (int)wt->size(2);
    void *wp = ws ? ws->data_ptr() : nullptr, *st = c10::cuda::getCurrentCUDAStream(dev).stream();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = abi.accumulate_weights(qp, c.part[0], c.part[1], c.strides, (int)PS, btp, (int)MP, lp, sp, (int)B, (int)KVH, (int)(HQ / KVH),
                                (int)D, (int)qlmax, (float)s1, gkp, w.lse, wtp, wb, wh, W, w.window, w.sinks, signs, k8, wp, st);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
  } catch (...) {
    Py_RETURN_NONE;
  }
}

// addresses of a tensor's elements: [first, last)
std::pair<uintptr_t, uintptr_t> extent(const at::Tensor& t) {
  int64_t n = t.numel() ? 1 : 0;
  for (int64_t i = 0; n && i < t.dim(); ++i) n += (t.size(i) - 1) * t.stride(i);
  const uintptr_t p = reinterpret_cast<uintptr_t>(t.data_ptr());
  return {p, p + n * t.element_size()};
}
bool overlap(const at::Tensor& x, const at::Tensor& y) {
  const auto a = extent(x), b = extent(y);
  return a.first < b.second && b.first < a.second;
}

// evict(flat, strides, PS, D, block_tables, seq_lens, weights, keep, sinks, recent, kept, out_lens, out_tables, out_weights, k8)
PyObject* evict(PyObject*, PyObject* const* a, Py_ssize_t n) {
  try {
    if (n != 15 || !abi.evict) Py_RETURN_NONE;
    const at::Tensor *bt = tensor(a[4]), *lens = tensor(a[5]), *wt = tensor(a[6]), *kept = tensor(a[10]), *ol = tensor(a[11]),
                     *ot = a[12] == Py_None ? bt : tensor(a[12]), *ow = a[13] == Py_None ? wt : tensor(a[13]);
    if (!bt || !lens || !wt || !kept || !ol || !ot || !ow || !wt->is_cuda() || bt->dim() != 2 || ot->dim() != 2 || wt->dim() != 3) Py_RETURN_NONE;
    const int dev = wt->device().index();
    long long PS, D, keep, sinks, recent;
    bool k8;
    Cache c;
    if (dev != c10::cuda::current_device() || !integer(a[2], &PS) || PS != (int)PS || PS < 1 || !integer(a[3], &D) || D != (int)D ||
        !integer(a[7], &keep) || keep != (int)keep || !integer(a[8], &sinks) || sinks != (int)sinks || !integer(a[9], &recent) ||
        recent != (int)recent || !boolean(a[14], &k8) || keep < 1 || sinks < 0 || recent < 0 || sinks + recent > keep ||
        !cache_of(a[0], a[1], dev, &c))
      Py_RETURN_NONE;
    for (const at::Tensor* t : {bt, lens, kept, ol, ot})
      if (!on(*t, dev) || t->scalar_type() != at::kInt || !t->is_contiguous()) Py_RETURN_NONE;
    const int64_t B = bt->size(0), MP = bt->size(1), KVH = wt->size(1), OMP = ot->size(1);
    if (B > INT32_MAX || MP > INT32_MAX || OMP > INT32_MAX || KVH > INT32_MAX || !weight_rows(wt, B, KVH, dev) ||
        !weight_rows(ow, B, KVH, dev) || ow->size(2) < keep || ot->size(0) != B || lens->dim() != 1 || lens->size(0) != B || ol->dim() != 1 ||
        ol->size(0) != B || kept->dim() != 3 || kept->size(0) != B || kept->size(1) != KVH || kept->size(2) != keep || keep > OMP * PS ||
        overlap(*lens, *ol) || ((ow->data_ptr() != wt->data_ptr() || ow->strides() != wt->strides()) && overlap(*wt, *ow)))
      Py_RETURN_NONE;
    const int32_t *btp = static_cast<const int32_t*>(bt->data_ptr()), *lp = static_cast<const int32_t*>(lens->data_ptr()),
                  *otp = static_cast<const int32_t*>(ot->data_ptr());
    int32_t *kp = static_cast<int32_t*>(kept->data_ptr()), *olp = static_cast<int32_t*>(ol->data_ptr());
    const float* wtp = static_cast<const float*>(wt->data_ptr());
    float* owp = static_cast<float*>(ow->data_ptr());
    const int64_t wb = wt->stride(0), wh = wt->stride(1), ob = ow->stride(0), oh = ow->stride(1);
    const int W = (int)wt->size(2), OW = (int)ow->size(2);
    void* st = c10::cuda::getCurrentCUDAStream(dev).stream();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = abi.evict(c.part[0], c.part[1], c.part[2], c.part[3], c.strides, (int)PS, btp, (int)MP, lp, (int)B, (int)KVH, (int)D, k8, wtp, wb,
                   wh, W, (int)keep, (int)sinks, (int)recent, otp, (int)OMP, kp, olp, owp, ob, oh, OW, st);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
  } catch (...) {
    Py_RETURN_NONE;
  }
}

// layer_write(key, value, kv_cache, slot_mapping, gk, gv, D, search, signs, k8)
PyObject* layer_write(PyObject*, PyObject* const* a, Py_ssize_t n) {
  try {
    if (n != 10 || !abi.write) Py_RETURN_NONE;
    const at::Tensor *k = tensor(a[0]), *v = tensor(a[1]), *slots = tensor(a[3]), *gk = tensor(a[4]), *gv = tensor(a[5]);
    if (!k || !v || !slots || !gk || !k->is_cuda() || gk->dim() != 1) Py_RETURN_NONE;
    const int dev = k->device().index();
    const int64_t KVH = gk->size(0);
    long long D;
    bool search, k8;
    const float* signs;
    int PS;
    Cache c;
    if (dev != c10::cuda::current_device() || !on(*v, dev) || !on(*slots, dev) || !integer(a[6], &D) || !boolean(a[7], &search) ||
        !boolean(a[9], &k8) || KVH < 1 || KVH > 65536 || !cache_of_slots(a[2], KVH, D, k8, dev, &c, &PS) || !token_rows(*k, KVH, D) ||
        !token_rows(*v, KVH, D) || k->dim() != v->dim() || k->size(0) != v->size(0) || k->stride(-1) != 1 || v->stride(-1) != 1 ||
        slots->scalar_type() != at::kLong || slots->dim() != 1 || !slots->is_contiguous() || slots->size(0) > k->size(0) ||
        !scales(gk, gv, KVH, dev) || !sign_vector(a[8], D, dev, &signs) || (k8 && signs))
      Py_RETURN_NONE;
    const bool flat = k->dim() == 2;
    return run_write({k->data_ptr(), v->data_ptr(), k->stride(0), flat ? D : k->stride(1), v->stride(0), flat ? D : v->stride(1), KVH, D}, c, PS,
                     *slots, *gk, *gv, search, signs, k8, dev);
  } catch (...) {
    Py_RETURN_NONE;
  }
}

// layer_decode(query, kv_cache, block_table, seq_lens, query_start_loc, tokens, scale, v_scale, gk, gv, qlmax, output, workspace,
//              splits, heads, D, signs, k8); the first `tokens` rows of query belong to the step
PyObject* layer_decode(PyObject*, PyObject* const* a, Py_ssize_t n) {
  try {
    if (n != 18 || !abi.decode) Py_RETURN_NONE;
    const at::Tensor *q = tensor(a[0]), *bt = tensor(a[2]), *lens = tensor(a[3]), *qsl = tensor(a[4]), *gk = tensor(a[8]),
                     *gv = tensor(a[9]), *out = tensor(a[11]), *ws = tensor(a[12]);
    if (!q || !bt || !lens || !qsl || !gk || !out || !ws || !q->is_cuda() || gk->dim() != 1) Py_RETURN_NONE;
    const int dev = q->device().index();
    const int64_t KVH = gk->size(0);
    long long T, qlmax, splits, HQ, D;
    double s1, s2;
    bool k8;
    const float* signs;
    int PS;
    Cache c;
    if (dev != c10::cuda::current_device() || !integer(a[5], &T) || !number(a[6], &s1) || !number(a[7], &s2) || !integer(a[10], &qlmax) ||
        qlmax != (int)qlmax || !integer(a[13], &splits) || splits != (int)splits || !integer(a[14], &HQ) || HQ != (int)HQ ||
        !integer(a[15], &D) || !boolean(a[17], &k8) || KVH < 1 || KVH > 65536 || HQ < 1 || HQ % KVH)
      Py_RETURN_NONE;
    if (!cache_of_slots(a[1], KVH, D, k8, dev, &c, &PS) || !token_rows(*q, HQ, D) || !token_rows(*out, HQ, D) || !q->is_contiguous() ||
        !out->is_contiguous() || T < 0 || q->size(0) < T || out->size(0) < T || bt->dim() != 2 || lens->dim() != 1 || qsl->dim() != 1 ||
        lens->size(0) != bt->size(0) || qsl->size(0) != bt->size(0) + 1 || !on(*out, dev) || !on(*ws, dev) || bt->size(0) > INT32_MAX ||
        bt->size(1) > INT32_MAX || !scales(gk, gv, KVH, dev) || !sign_vector(a[16], D, dev, &signs) || (k8 && signs))
      Py_RETURN_NONE;
    for (const at::Tensor* t : {bt, lens, qsl})
      if (!on(*t, dev) || t->scalar_type() != at::kInt || !t->is_contiguous()) Py_RETURN_NONE;
    return run_decode(q->data_ptr(), c, PS, *bt, *lens, *qsl, HQ, D, s1, s2, *gk, *gv, (int)qlmax, out->data_ptr(), *ws, (int)splits, signs,
                      k8, dev);
  } catch (...) {
    Py_RETURN_NONE;
  }
}

// [(table row, q0, q1, L)] within B requests, NT query tokens and a table's reach
bool prefill_rows(PyObject* list, int64_t B, int64_t reach, int64_t NT, std::vector<int32_t>* rows) {
  if (!PyList_CheckExact(list) || PyList_GET_SIZE(list) > INT32_MAX) return false;
  const Py_ssize_t n = PyList_GET_SIZE(list);
  rows->resize(4 * n);
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* t = PyList_GET_ITEM(list, i);
    long long v[4];
    if (!PyTuple_CheckExact(t) || PyTuple_GET_SIZE(t) != 4) return false;
    for (int k = 0; k < 4; ++k)
      if (!integer(PyTuple_GET_ITEM(t, k), &v[k])) return false;
    if (v[3] > reach || v[0] < 0 || v[0] >= B || v[1] < 0 || v[1] >= v[2] || v[2] > NT || v[3] < 1 || v[3] > INT32_MAX) return false;
    for (int k = 0; k < 4; ++k) (*rows)[4 * i + k] = (int32_t)v[k];
  }
  return true;
}

// prefill(query, flat, strides, PS, block_tables, rows, qk_scale, out_scale, KVH, out, chunk, signs, k8, workspace);
// prefill_window: .., window, sinks, lse
template <bool WIN>
PyObject* prefill_any(PyObject*, PyObject* const* a, Py_ssize_t n) {
  try {
    if (n != (WIN ? 17 : 14) || !abi.prefill) Py_RETURN_NONE;
    const at::Tensor *q = tensor(a[0]), *bt = tensor(a[4]), *out = tensor(a[9]), *ws = a[13] == Py_None ? nullptr : tensor(a[13]);
    if (!q || !bt || !out || (!ws && a[13] != Py_None) || !q->is_cuda() || !PyList_CheckExact(a[5])) Py_RETURN_NONE;
    const int dev = q->device().index();
    long long PS, KVH, chunk;
    double s1, s2;
    bool k8;
    const float* signs;
    Cache c;
    if (dev != c10::cuda::current_device() || !integer(a[3], &PS) || PS < 1 || PS != (int)PS || !number(a[6], &s1) ||
        !number(a[7], &s2) || !integer(a[8], &KVH) || KVH < 1 || KVH != (int)KVH || !integer(a[10], &chunk) ||
        !boolean(a[12], &k8))
      Py_RETURN_NONE;
    const bool out_f32 = out->scalar_type() == at::kFloat;
    if (q->scalar_type() != at::kBFloat16 || (out->scalar_type() != at::kBFloat16 && !out_f32) || q->dim() != 3 || out->dim() != 3 ||
        out->size(1) != q->size(1) || out->size(2) != q->size(2) || out->size(0) < q->size(0) || !q->is_contiguous() ||
        !out->is_contiguous() || !on(*out, dev) || !on(*bt, dev) || bt->scalar_type() != at::kInt || bt->dim() != 2 ||
        !bt->is_contiguous() || (ws && (!on(*ws, dev) || ws->nbytes() < 64)))
      Py_RETURN_NONE;
    const int64_t B = bt->size(0), MP = bt->size(1), NT = q->size(0), HQ = q->size(1), D = q->size(2);
    if (HQ % KVH || B > INT32_MAX || MP > INT32_MAX || NT > INT32_MAX || HQ > INT32_MAX || D > INT32_MAX ||
        !sign_vector(a[11], D, dev, &signs) || (k8 && signs) || !cache_of(a[1], a[2], dev, &c))
      Py_RETURN_NONE;
    std::vector<int32_t> rows;
    if (!prefill_rows(a[5], B, MP * PS, NT, &rows)) Py_RETURN_NONE;
    const Py_ssize_t n_rows = (Py_ssize_t)(rows.size() / 4);
    const int G = (int)(HQ / KVH);
    Window w;
    if (WIN && !window_of(a[14], a[15], a[16], NT, HQ, dev, &w)) Py_RETURN_NONE;
    const size_t nb = WIN ? abi.prefill_window_scratch_bytes(rows.data(), (int)n_rows, (int)NT, (int)KVH, G, (int)D, chunk,
                                                             signs != nullptr, w.window, w.sinks)
                          : abi.prefill_scratch_bytes(rows.data(), (int)n_rows, (int)NT, (int)KVH, G, (int)D, chunk, signs != nullptr);
    const void* qp = q->data_ptr();
    const int32_t* btp = static_cast<const int32_t*>(bt->data_ptr());
    void *op = out->data_ptr(), *wp = ws ? ws->data_ptr() : nullptr;
    const at::Tensor scratch = at::empty({(int64_t)(nb ? nb : 1)}, q->options().dtype(at::kByte));
    void* sp = scratch.data_ptr();
    void* st = c10::cuda::getCurrentCUDAStream(dev).stream();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    if (WIN)
      rc = abi.prefill_window(qp, 0, c.part[0], c.part[1], c.part[2], c.part[3], c.strides, (int)PS, btp, (int)B, (int)MP,
                              rows.data(), (int)n_rows, (int)NT, (int)KVH, G, (int)D, (float)s1, (float)s2, signs, k8, chunk, w.window,
                              w.sinks, w.lse, sp, nb, op, out_f32, wp, st);
    else
      rc = abi.prefill(qp, 0, c.part[0], c.part[1], c.part[2], c.part[3], c.strides, (int)PS, btp, (int)B, (int)MP,
                       rows.data(), (int)n_rows, (int)NT, (int)KVH, G, (int)D, (float)s1, (float)s2, signs, k8, chunk, sp, nb, op,
                       out_f32, wp, st);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
  } catch (...) {
    Py_RETURN_NONE;
  }
}

// prefill_b8(query, flat, strides, PS, block_tables, rows, qk_scale, out_scale, KVH, out, fmt, window, sinks, chunk, workspace, lse)
PyObject* prefill_b8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  try {
    if (n != 16 || !abi.prefill_b8) Py_RETURN_NONE;
    const at::Tensor *q = tensor(a[0]), *bt = tensor(a[4]), *out = tensor(a[9]), *ws = a[14] == Py_None ? nullptr : tensor(a[14]);
    if (!q || !bt || !out || (!ws && a[14] != Py_None) || !q->is_cuda()) Py_RETURN_NONE;
    const int dev = q->device().index();
    long long PS, KVH, chunk;
    double s1, s2;
    int fmt;
    Tiles c;
    Window w;
    if (dev != c10::cuda::current_device() || !integer(a[3], &PS) || PS < 1 || PS != (int)PS || !number(a[6], &s1) || !number(a[7], &s2) ||
        !integer(a[8], &KVH) || KVH < 1 || KVH != (int)KVH || !format_of(a[10], &fmt) || !integer(a[13], &chunk))
      Py_RETURN_NONE;
    const bool out_f32 = out->scalar_type() == at::kFloat;
    if (q->scalar_type() != at::kBFloat16 || (out->scalar_type() != at::kBFloat16 && !out_f32) || q->dim() != 3 || out->dim() != 3 ||
        out->size(1) != q->size(1) || out->size(2) != q->size(2) || out->size(0) < q->size(0) || !q->is_contiguous() ||
        !out->is_contiguous() || !on(*out, dev) || !on(*bt, dev) || bt->scalar_type() != at::kInt || bt->dim() != 2 ||
        !bt->is_contiguous() || (ws && (!on(*ws, dev) || ws->nbytes() < 64)))
      Py_RETURN_NONE;
    const int64_t B = bt->size(0), MP = bt->size(1), NT = q->size(0), HQ = q->size(1), D = q->size(2);
    std::vector<int32_t> rows;
    if (HQ % KVH || B > INT32_MAX || MP > INT32_MAX || NT > INT32_MAX || HQ > INT32_MAX || D > INT32_MAX || !tiles_of(a[1], a[2], dev, &c) ||
        !prefill_rows(a[5], B, MP * PS, NT, &rows) || !window_of(a[11], a[12], a[15], NT, HQ, dev, &w))
      Py_RETURN_NONE;
    const int G = (int)(HQ / KVH), n_rows = (int)(rows.size() / 4);
    const size_t nb = abi.prefill_window_scratch_bytes(rows.data(), n_rows, (int)NT, (int)KVH, G, (int)D, chunk, 0, w.window, w.sinks);
    const void* qp = q->data_ptr();
    const int32_t* btp = static_cast<const int32_t*>(bt->data_ptr());
    void *op = out->data_ptr(), *wp = ws ? ws->data_ptr() : nullptr;
    const at::Tensor scratch = at::empty({(int64_t)(nb ? nb : 1)}, q->options().dtype(at::kByte));
    void *sp = scratch.data_ptr(), *st = c10::cuda::getCurrentCUDAStream(dev).stream();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = abi.prefill_b8(qp, 0, c.k, c.v, c.strides, (int)PS, btp, (int)B, (int)MP, rows.data(), n_rows, (int)NT, (int)KVH, G, (int)D,
                        (float)s1, (float)s2, chunk, fmt, w.window, w.sinks, w.lse, sp, nb, op, out_f32, wp, st);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
  } catch (...) {
    Py_RETURN_NONE;
  }
}

// bind(addresses of the entry points in the order of Abi)
PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long p[17];
  if (!PyArg_ParseTuple(args, "KKKKKKKKKKKKKKKKK", &p[0], &p[1], &p[2], &p[3], &p[4], &p[5], &p[6], &p[7], &p[8], &p[9], &p[10], &p[11],
                        &p[12], &p[13], &p[14], &p[15], &p[16]))
    return nullptr;
  int i = 0;
  auto take = [&](auto& f) { f = reinterpret_cast<std::remove_reference_t<decltype(f)>>(p[i++]); };
  take(abi.write);
  take(abi.write_rot);
  take(abi.write_k8);
  take(abi.decode);
  take(abi.decode_rot);
  take(abi.decode_k8);
  take(abi.prefill_scratch_bytes);
  take(abi.prefill);
  take(abi.decode_window);
  take(abi.prefill_window_scratch_bytes);
  take(abi.prefill_window);
  take(abi.accumulate_weights);
  take(abi.evict);
  take(abi.write_rotary);
  take(abi.write_b8);
  take(abi.decode_b8);
  take(abi.prefill_b8);
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", bind, METH_VARARGS, "hands over the addresses of the C entry points"},
    {"write", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(write)), METH_FASTCALL, "status, or None: not the plain form"},
    {"decode", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(decode_any<false>)), METH_FASTCALL, "status, or None: not the plain form"},
    {"layer_write", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(layer_write)), METH_FASTCALL, "status, or None: not the plain form"},
    {"layer_decode", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(layer_decode)), METH_FASTCALL, "status, or None: not the plain form"},
    {"prefill", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(prefill_any<false>)), METH_FASTCALL, "status, or None: not the plain form"},
    {"decode_window", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(decode_any<true>)), METH_FASTCALL, "status, or None: not the plain form"},
    {"prefill_window", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(prefill_any<true>)), METH_FASTCALL, "status, or None: not the plain form"},
    {"accumulate_weights", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(accumulate_weights)), METH_FASTCALL, "status, or None: not the plain form"},
    {"evict", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(evict)), METH_FASTCALL, "status, or None: not the plain form"},
    {"write_rotary", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(write_rotary)), METH_FASTCALL, "status, or None: not the plain form"},
    {"write_b8", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(write_b8_any<false>)), METH_FASTCALL, "status, or None: not the plain form"},
    {"write_rotary_b8", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(write_b8_any<true>)), METH_FASTCALL, "status, or None: not the plain form"},
    {"decode_b8", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(decode_b8)), METH_FASTCALL, "status, or None: not the plain form"},
    {"prefill_b8", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(prefill_b8)), METH_FASTCALL, "status, or None: not the plain form"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "hkv_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_hkv_host(void) {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "torch_version", HKV_TORCH_VERSION) != 0) {   // the torch it is compiled against
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
