// Native host path of the Python layer: one call per operator that checks the
// tensors' layout, allocates outputs and workspace through torch's caching
// allocator and enqueues the C-ABI call on the caller's stream. What it covers
// is the ordinary case (plain tensors on one device, aligned layouts); anything
// else returns None and the Python layer takes its general path, so a call
// accepts, refuses and returns the same either way.
//
// Why: the same steps in Python (strides, data pointers, some thirty ctypes
// arguments) took as long as a small kernel: a flash_attention forward 15 us of
// host time, a decode step of append, rotation and attention 64 us, forward and
// backward 75 us (an idle box; busy ones up to twice that).
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdint>

#include "mpx_attn.h"
#include "mpx_attn_sched.h"
#include "mpx_cache8.h"
#include "mpx_norm.h"

namespace {

// Entries of the loaded library, by address (init).
#define MPX_ENTRIES(X)                                                                      \
  X(mpx_attn_fwd_lse)                                                                       \
  X(mpx_attn_fwd_dropout)                                                                   \
  X(mpx_attn_fwd_workspace_bytes)                                                           \
  X(mpx_attn_bwd)                                                                           \
  X(mpx_attn_bwd_dropout)                                                                   \
  X(mpx_attn_bwd_grouped)                                                                   \
  X(mpx_attn_bwd_workspace_bytes)                                                           \
  X(mpx_attn_bwd_grouped_workspace_bytes)                                                   \
  X(mpx_attn_bwd_ds_preferred)                                                              \
  X(mpx_paged_decode_gqa)                                                                   \
  X(mpx_paged_decode_workspace_bytes)                                                       \
  X(mpx_paged_prefill_gqa)                                                                  \
  X(mpx_paged_prefill_workspace_bytes)                                                      \
  X(mpx_kv_append)                                                                          \
  X(mpx_kv_append_rope)                                                                     \
  X(mpx_rope_at)                                                                            \
  X(mpx_kv_append8)                                                                         \
  X(mpx_kv_load8)                                                                           \
  X(mpx_paged_attend8)                                                                      \
  X(mpx_paged_attend8_call_workspace_bytes)                                                      \
  X(mpx_qk_norm_rope)                                                                       \
  X(mpx_qk_norm_rope_bwd)                                                                   \
  X(mpx_qk_norm_rope_bwd_workspace_bytes)                                                   \
  X(mpx_last_error)
struct Api {
#define X(name) decltype(&::name) name = nullptr;
  MPX_ENTRIES(X)
#undef X
} api;

// A plain torch tensor on a device (no subclass, no functorch or dispatch
// wrapper, storage present), or nullptr.
const at::Tensor* plain(PyObject* obj) {
  if (!THPVariable_CheckExact(obj) && Py_TYPE(obj) != (PyTypeObject*)ParameterClass) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(obj);
  static const c10::DispatchKeySet wrapped({c10::DispatchKey::Python,
                                            c10::DispatchKey::FuncTorchGradWrapper,
                                            c10::DispatchKey::FuncTorchBatched,
                                            c10::DispatchKey::Functionalize});
  if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || !t.has_storage() ||
      t.key_set().has_any(wrapped))
    return nullptr;
  return &t;
}

int dtype_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return MPX_F32;
    case at::kHalf: return MPX_F16;
    case at::kBFloat16: return MPX_BF16;
    default: return -1;
  }
}

// The kernels' layout: last dimension contiguous, other strides multiples of
// 16 bytes, 16-byte aligned.
bool aligned_rows(const at::Tensor& t, int vec) {
  const int64_t n = t.dim();
  if (t.stride(n - 1) != 1 || ((uintptr_t)t.data_ptr() & 15u) != 0) return false;
  for (int64_t i = 0; i + 1 < n; ++i)
    if (t.stride(i) % vec != 0) return false;
  return true;
}

bool int32_contiguous(const at::Tensor& t) {
  return t.scalar_type() == at::kInt && t.is_contiguous();
}

struct Strides {
  int64_t s[3];
  // (batch, head, seq) of a 4-D tensor in BSHD or BHSD order
  Strides(const at::Tensor& t, bool bshd)
      : s{t.stride(0), t.stride(bshd ? 2 : 1), t.stride(bshd ? 1 : 2)} {}
};

at::Tensor bytes(size_t n, const at::Tensor& like) {
  return at::empty({(int64_t)(n < 16 ? 16 : n)}, like.options().dtype(at::kByte));
}

// f() without the GIL, which is taken back also when f throws (data_ptr() of
// some tensors does).
template <class F>
int call(F&& f) {
  struct Released {
    PyThreadState* const state = PyEval_SaveThread();
    ~Released() { PyEval_RestoreThread(state); }
  } released;
  return f();
}

// An argument as the general path's int(...) and ctypes read it: what has
// __int__, __index__ or __trunc__ (masks and windows come as the user gave
// them: floats, numpy scalars), of which the low bits count.
int64_t as_int(PyObject* o) {
  if (PyLong_Check(o)) return (int64_t)PyLong_AsUnsignedLongLongMask(o);
  PyObject* const x = PyNumber_Long(o);
  if (!x) return -1;
  const int64_t v = (int64_t)PyLong_AsUnsignedLongLongMask(x);
  Py_DECREF(x);
  return v;
}
double as_float(PyObject* o) { return PyFloat_AsDouble(o); }

bool wrong_count(Py_ssize_t n, Py_ssize_t want) {
  if (n == want) return false;
  PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, n);
  return true;
}

// attn_fwd(q, k, v, bshd, D, scale, causal, wl, wr, want_lse, drop_p, seed, stream)
//   -> o, (o, lse), an error code, or None
PyObject* attn_fwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (wrong_count(n, 13)) return nullptr;
  const at::Tensor *q = plain(a[0]), *k = plain(a[1]), *v = plain(a[2]);
  if (!q || !k || !v || q->device() != k->device() || q->device() != v->device()) Py_RETURN_NONE;
  const int code = dtype_code(*q);
  const bool bshd = as_int(a[3]) != 0;
  const int D = (int)as_int(a[4]);
  const int vec = code == MPX_F32 ? 4 : 8;
  for (const at::Tensor* t : {q, k, v})
    if (t->dim() != 4 || t->size(3) != D || dtype_code(*t) != code || code < 0 ||
        !aligned_rows(*t, vec))
      Py_RETURN_NONE;
  const double scale = as_float(a[5]), drop_p = as_float(a[10]);
  const int causal = (int)as_int(a[6]), wl = (int)as_int(a[7]), wr = (int)as_int(a[8]);
  const bool want_lse = as_int(a[9]) != 0;
  const uint64_t seed = PyLong_AsUnsignedLongLongMask(a[11]);
  void* stream = PyLong_AsVoidPtr(a[12]);
  if (PyErr_Occurred()) return nullptr;
  const int hd = bshd ? 2 : 1, sd = bshd ? 1 : 2;
  const int B = (int)q->size(0), H = (int)q->size(hd), Sq = (int)q->size(sd);
  const int H_kv = (int)k->size(hd), Sk = (int)k->size(sd);
  at::Tensor o = at::empty(q->sizes(), q->options()), lse, ws;
  if (want_lse) lse = at::empty({B, H, Sq}, q->options().dtype(at::kFloat));
  const size_t need = api.mpx_attn_fwd_workspace_bytes(B, H, Sq, Sk, D, causal, wl, wr, code);
  if (need) ws = bytes(need, *q);
  const Strides qs(*q, bshd), ks(*k, bshd), vs(*v, bshd), os(o, bshd);
  float* const lp = want_lse ? lse.data_ptr<float>() : nullptr;
  void* const wp = need ? ws.data_ptr() : nullptr;
  const int rc = call([&] {
    if (drop_p >= 0)
      return api.mpx_attn_fwd_dropout(q->data_ptr(), k->data_ptr(), v->data_ptr(), o.data_ptr(), lp,
                                      qs.s, ks.s, vs.s, os.s, B, H, H_kv, Sq, Sk, D, (float)scale,
                                      causal, wl, wr, code, (float)drop_p, seed, wp, need, stream);
    return api.mpx_attn_fwd_lse(q->data_ptr(), k->data_ptr(), v->data_ptr(), o.data_ptr(), lp,
                                qs.s, ks.s, vs.s, os.s, B, H, H_kv, Sq, Sk, D, (float)scale,
                                causal, wl, wr, code, wp, need, stream);
  });
  if (rc != MPX_OK) return PyLong_FromLong(rc);
  if (!want_lse) return THPVariable_Wrap(std::move(o));
  PyObject* out = PyTuple_New(2);
  if (!out) return nullptr;
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(o)));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(lse)));
  return out;
  END_HANDLE_TH_ERRORS
}

// attn_bwd(q, k, v, o, dout, lse, bshd, scale, causal, wl, wr, drop_p, seed,
//   may_store_ds, stream) -> (dq, dk, dv), an error code, or None (also where
// the stored-dS schedule is the better one, or memory for parts is short)
PyObject* attn_bwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (wrong_count(n, 15)) return nullptr;
  const at::Tensor* t[6];
  for (int i = 0; i < 6; ++i) {
    t[i] = plain(a[i]);
    if (!t[i] || t[i]->device() != t[0]->device()) Py_RETURN_NONE;
  }
  const at::Tensor &q = *t[0], &k = *t[1], &v = *t[2], &o = *t[3], &dout = *t[4], &lse = *t[5];
  const int code = dtype_code(q);
  if (code < 0 || q.dim() != 4) Py_RETURN_NONE;
  const int vec = code == MPX_F32 ? 4 : 8, D = (int)q.size(3);
  for (int i = 0; i < 5; ++i)
    if (t[i]->dim() != 4 || t[i]->size(3) != D || dtype_code(*t[i]) != code ||
        !aligned_rows(*t[i], vec))
      Py_RETURN_NONE;
  if (lse.scalar_type() != at::kFloat || !lse.is_contiguous() || dout.sizes() != q.sizes() ||
      o.sizes() != q.sizes())
    Py_RETURN_NONE;
  const bool bshd = as_int(a[6]) != 0;
  const double scale = as_float(a[7]), drop_p = as_float(a[11]);
  const int causal = (int)as_int(a[8]), wl = (int)as_int(a[9]), wr = (int)as_int(a[10]);
  const uint64_t seed = PyLong_AsUnsignedLongLongMask(a[12]);
  const bool may_store = as_int(a[13]) != 0;
  void* stream = PyLong_AsVoidPtr(a[14]);
  if (PyErr_Occurred()) return nullptr;
  const int hd = bshd ? 2 : 1, sd = bshd ? 1 : 2;
  const int B = (int)q.size(0), H = (int)q.size(hd), Sq = (int)q.size(sd);
  const int H_kv = (int)k.size(hd), Sk = (int)k.size(sd);
  if (may_store && drop_p >= 0 &&
      api.mpx_attn_bwd_ds_preferred(B, H, H_kv, Sq, Sk, D, code, wl))
    Py_RETURN_NONE;
  const bool grouped = H != H_kv;
  const size_t need =
      grouped ? api.mpx_attn_bwd_grouped_workspace_bytes(B, H, H_kv, Sq, Sk, D, code, wl)
              : api.mpx_attn_bwd_workspace_bytes(B, H, Sq);
  at::Tensor ws;
  try {
    ws = bytes(need, q);
  } catch (const c10::OutOfMemoryError&) {
    Py_RETURN_NONE;
  }
  at::Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()),
             dv = at::empty(v.sizes(), v.options());
  const Strides s[8] = {{q, bshd}, {k, bshd}, {v, bshd}, {o, bshd},
                        {dout, bshd}, {dq, bshd}, {dk, bshd}, {dv, bshd}};
  const float* const lp = lse.data_ptr<float>();
  const int rc = call([&] {
#define MPX_BWD_ARGS                                                                          \
  q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), dout.data_ptr(), lp, dq.data_ptr(), \
      dk.data_ptr(), dv.data_ptr(), s[0].s, s[1].s, s[2].s, s[3].s, s[4].s, s[5].s, s[6].s,   \
      s[7].s, B, H, H_kv, Sq, Sk, D, (float)scale, causal, wl, wr, code
    if (grouped)
      return api.mpx_attn_bwd_grouped(MPX_BWD_ARGS, drop_p >= 0 ? (float)drop_p : 0.f, seed,
                                      ws.data_ptr(), need, stream);
    if (drop_p >= 0)
      return api.mpx_attn_bwd_dropout(MPX_BWD_ARGS, (float)drop_p, seed, ws.data_ptr(), need,
                                      stream);
    return api.mpx_attn_bwd(MPX_BWD_ARGS, ws.data_ptr(), need, stream);
#undef MPX_BWD_ARGS
  });
  if (rc != MPX_OK) return PyLong_FromLong(rc);
  PyObject* out = PyTuple_New(3);
  if (!out) return nullptr;
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(dq)));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(dk)));
  PyTuple_SET_ITEM(out, 2, THPVariable_Wrap(std::move(dv)));
  return out;
  END_HANDLE_TH_ERRORS
}

// paged_attend(q, k_pool, v_pool, tables, lens, slopes or None, scale, causal,
//   stream) -> o, an error code, or None; the caller has checked the shapes.
// Decode for one query per sequence, else prefill (head dims of the kernels).
PyObject* paged_attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (wrong_count(n, 9)) return nullptr;
  const at::Tensor* t[6];
  for (int i = 0; i < 6; ++i) {
    t[i] = nullptr;
    if (i == 5 && a[5] == Py_None) break;
    t[i] = plain(a[i]);
    if (!t[i] || t[i]->device() != t[0]->device()) Py_RETURN_NONE;
  }
  const at::Tensor &q = *t[0], &kp = *t[1], &vp = *t[2], &bt = *t[3], &cl = *t[4];
  const int code = dtype_code(q);
  const int vec = code == MPX_F32 ? 4 : 8;
  if (code < 0 || q.dim() != 4 || kp.dim() != 4 || q.size(3) % vec != 0 || !aligned_rows(q, vec) ||
      !kp.is_contiguous() || !vp.is_contiguous() || !int32_contiguous(bt) ||
      !int32_contiguous(cl) ||
      (t[5] && (t[5]->scalar_type() != at::kFloat || !t[5]->is_contiguous())))
    Py_RETURN_NONE;
  const double scale = as_float(a[6]);
  const int B = (int)q.size(0), Sq = (int)q.size(1), H = (int)q.size(2), D = (int)q.size(3);
  const int causal = Sq == 1 ? 0 : (int)as_int(a[7]);  // (decode takes no mask)
  void* stream = PyLong_AsVoidPtr(a[8]);
  if (PyErr_Occurred()) return nullptr;
  const int nb = (int)kp.size(0), bs = (int)kp.size(1), H_kv = (int)kp.size(2);
  const int mb = (int)bt.size(1);
  at::Tensor o = at::empty(q.sizes(), q.options());
  const size_t need =
      Sq == 1 ? api.mpx_paged_decode_workspace_bytes(B, H, D, bs, mb)
              : api.mpx_paged_prefill_workspace_bytes(B, Sq, H, D, bs, mb, causal, code);
  at::Tensor ws = bytes(need, q);
  const int64_t qs[3] = {q.stride(0), q.stride(2), q.stride(1)};
  const int64_t os[3] = {o.stride(0), o.stride(2), o.stride(1)};
  const float* const sl = t[5] ? t[5]->data_ptr<float>() : nullptr;
  const int rc = call([&] {
    if (Sq != 1)
      return api.mpx_paged_prefill_gqa(q.data_ptr(), kp.data_ptr(), vp.data_ptr(),
                                       bt.data_ptr<int32_t>(), cl.data_ptr<int32_t>(), sl,
                                       o.data_ptr(), qs, os, B, Sq, H, H_kv, D, nb, bs, mb,
                                       (float)scale, causal, code, ws.data_ptr(),
                                       (size_t)ws.numel(), stream);
    return api.mpx_paged_decode_gqa(q.data_ptr(), kp.data_ptr(), vp.data_ptr(),
                                    bt.data_ptr<int32_t>(), cl.data_ptr<int32_t>(), sl,
                                    o.data_ptr(), qs, os, B, H, H_kv, D, nb, bs, mb, (float)scale,
                                    code, ws.data_ptr(), (size_t)ws.numel(), stream);
  });
  if (rc != MPX_OK) return PyLong_FromLong(rc);
  return THPVariable_Wrap(std::move(o));
  END_HANDLE_TH_ERRORS
}

// kv_append(k, v, k_pool, v_pool, tables, starts, counts, errors, cos or None,
//   sin or None, stream) -> an error code, or None; clears errors first; the
// caller has checked the shapes
PyObject* kv_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (wrong_count(n, 11)) return nullptr;
  const bool rope = a[8] != Py_None;
  const at::Tensor* t[10];
  for (int i = 0; i < (rope ? 10 : 8); ++i) {
    t[i] = plain(a[i]);
    if (!t[i] || t[i]->device() != t[0]->device()) Py_RETURN_NONE;
  }
  const at::Tensor &k = *t[0], &v = *t[1], &kp = *t[2], &vp = *t[3], &bt = *t[4];
  const int code = dtype_code(kp);
  const int vec = code == MPX_F32 ? 4 : 8;
  if (code < 0 || k.dim() != 4 || v.dim() != 4 || !aligned_rows(k, vec) || !aligned_rows(v, vec) ||
      !int32_contiguous(bt) || !int32_contiguous(*t[5]) || !int32_contiguous(*t[6]) ||
      !int32_contiguous(*t[7]))
    Py_RETURN_NONE;
  if (rope && (!t[8]->is_contiguous() || !t[9]->is_contiguous() || dtype_code(*t[8]) < 0))
    Py_RETURN_NONE;
  void* stream = PyLong_AsVoidPtr(a[10]);
  if (PyErr_Occurred()) return nullptr;
  t[7]->zero_();
  const int B = (int)k.size(0), T = (int)k.size(1), H = (int)k.size(2), D = (int)k.size(3);
  const int nb = (int)kp.size(0), bs = (int)kp.size(1), mb = (int)bt.size(1);
  const int64_t ks[3] = {k.stride(0), k.stride(1), k.stride(2)};
  const int64_t vs[3] = {v.stride(0), v.stride(1), v.stride(2)};
  const int rc = call([&] {
    if (rope)
      return api.mpx_kv_append_rope(
          k.data_ptr(), v.data_ptr(), kp.data_ptr(), vp.data_ptr(), bt.data_ptr<int32_t>(),
          t[5]->data_ptr<int32_t>(), t[6]->data_ptr<int32_t>(), ks, vs, B, T, H, D, nb, bs, mb,
          code, t[8]->data_ptr(), t[9]->data_ptr(), (int)t[8]->size(0), dtype_code(*t[8]),
          t[7]->data_ptr<int32_t>(), stream);
    return api.mpx_kv_append(k.data_ptr(), v.data_ptr(), kp.data_ptr(), vp.data_ptr(),
                             bt.data_ptr<int32_t>(), t[5]->data_ptr<int32_t>(),
                             t[6]->data_ptr<int32_t>(), ks, vs, B, T, H, D, nb, bs, mb, code,
                             t[7]->data_ptr<int32_t>(), stream);
  });
  return PyLong_FromLong(rc);
  END_HANDLE_TH_ERRORS
}

// rope_at(x, cos, sin, positions, errors, stream) -> out, an error code, or
// None; clears errors first; the caller has checked the shapes
PyObject* rope_at(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (wrong_count(n, 6)) return nullptr;
  const at::Tensor* t[5];
  for (int i = 0; i < 5; ++i) {
    t[i] = plain(a[i]);
    if (!t[i] || t[i]->device() != t[0]->device()) Py_RETURN_NONE;
  }
  const at::Tensor& x = *t[0];
  const int code = dtype_code(x), cdt = dtype_code(*t[1]);
  if (code < 0 || cdt < 0 || x.dim() != 4 || !aligned_rows(x, code == MPX_F32 ? 4 : 8) ||
      !t[1]->is_contiguous() || !t[2]->is_contiguous() || !int32_contiguous(*t[3]) ||
      !int32_contiguous(*t[4]))
    Py_RETURN_NONE;
  void* stream = PyLong_AsVoidPtr(a[5]);
  if (PyErr_Occurred()) return nullptr;
  at::Tensor out = at::empty(x.sizes(), x.options());
  t[4]->zero_();
  const int64_t xs[3] = {x.stride(0), x.stride(1), x.stride(2)};
  const int64_t os[3] = {out.stride(0), out.stride(1), out.stride(2)};
  const int rc = call([&] {
    return api.mpx_rope_at(x.data_ptr(), out.data_ptr(), t[1]->data_ptr(), t[2]->data_ptr(), xs, os,
                           (int)x.size(0), (int)x.size(1), (int)x.size(2), (int)x.size(3),
                           t[3]->data_ptr<int32_t>(), (int)t[1]->size(0), code, cdt,
                           t[4]->data_ptr<int32_t>(), stream);
  });
  if (rc != MPX_OK) return PyLong_FromLong(rc);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// ---- the 8-bit cache and the query/key norm ---------------------------------------
// These check everything that the Python layer checks, so that it calls them
// first: what is not exactly the ordinary case is left to it, refusals too.

void* stream_of(const at::Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

bool tracked(std::initializer_list<const at::Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const at::Tensor* t : ts)
    if (t && t->requires_grad()) return true;
  return false;
}

// Whether one is a dual tensor of forward-mode differentiation (which the general
// path refuses).
bool dual(std::initializer_list<const at::Tensor*> ts) {
  for (const at::Tensor* t : ts)
    if (t && t->_fw_grad(0).defined()) return true;
  return false;
}

// A plain tensor on `dev`, or nullptr.
const at::Tensor* plain_on(PyObject* o, c10::Device dev) {
  const at::Tensor* t = plain(o);
  return t && t->device() == dev ? t : nullptr;
}

bool aligned(const at::Tensor& t) { return ((uintptr_t)t.data_ptr() & 15u) == 0; }

// An int32 vector of n entries.
bool int32_vector(const at::Tensor& t, int64_t n) {
  return t.dim() == 1 && t.size(0) == n && int32_contiguous(t);
}

// Pools of 8-bit codes, their scales and int32 tables, checked.
struct Cache8 {
  const at::Tensor *kp, *vp, *bt, *ks, *vs;
  int code, nb, bs, H, D, mb;
  bool ok = false;
  Cache8(PyObject* k_pool, PyObject* v_pool, PyObject* tables, PyObject* scales) {
    if (!(kp = plain(k_pool)) || !PyTuple_CheckExact(scales) || PyTuple_GET_SIZE(scales) != 2) return;
    const c10::Device dev = kp->device();
    if (!(vp = plain_on(v_pool, dev)) || !(bt = plain_on(tables, dev)) ||
        !(ks = plain_on(PyTuple_GET_ITEM(scales, 0), dev)) ||
        !(vs = plain_on(PyTuple_GET_ITEM(scales, 1), dev)))
      return;
    code = kp->scalar_type() == at::kFloat8_e4m3fn ? MPX8_E4M3
           : kp->scalar_type() == at::kChar        ? MPX8_INT8
                                                   : -1;
    if (code < 0 || vp->scalar_type() != kp->scalar_type() || kp->dim() != 4 ||
        vp->sizes() != kp->sizes() || !kp->is_contiguous() || !vp->is_contiguous() ||
        !aligned(*kp) || !aligned(*vp) || bt->dim() != 2 || !int32_contiguous(*bt))
      return;
    if (kp->size(0) >= INT32_MAX || kp->size(1) > MPX8_MAX_BLOCK_SIZE || kp->size(1) == 0 ||
        kp->size(3) % 16 != 0 || kp->size(3) > 256 || kp->size(3) == 0)
      return;
    nb = (int)kp->size(0); bs = (int)kp->size(1); H = (int)kp->size(2); D = (int)kp->size(3);
    mb = (int)bt->size(1);
    for (const at::Tensor* s : {ks, vs})
      if (s->scalar_type() != at::kFloat || s->dim() != 2 || s->size(0) != nb || s->size(1) != H ||
          !s->is_contiguous())
        return;
    ok = true;
  }
};

// cos and sin tables (rows, D / 2) of one of the kernels' types.
bool table_pair(const at::Tensor* c, const at::Tensor* s, int D) {
  return c && s && c->dim() == 2 && c->sizes() == s->sizes() && c->size(1) * 2 == D &&
         c->size(0) <= INT32_MAX && dtype_code(*c) >= 0 && dtype_code(*s) == dtype_code(*c) &&
         c->is_contiguous() && s->is_contiguous() && aligned(*c) && aligned(*s);
}

// store8(k_pool, v_pool, tables, k, v, starts, counts or None, errors or None,
//   rope or None, scales) -> errors, an error code, or None
PyObject* store8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (wrong_count(n, 10)) return nullptr;
  const Cache8 c(a[0], a[1], a[2], a[9]);
  if (!c.ok) Py_RETURN_NONE;
  const c10::Device dev = c.kp->device();
  const at::Tensor *k = plain_on(a[3], dev), *v = plain_on(a[4], dev), *start = plain_on(a[5], dev);
  const at::Tensor* count = a[6] == Py_None ? nullptr : plain_on(a[6], dev);
  const at::Tensor* err = a[7] == Py_None ? nullptr : plain_on(a[7], dev);
  if (!k || !v || !start || (!count && a[6] != Py_None) || (!err && a[7] != Py_None)) Py_RETURN_NONE;
  const int code = dtype_code(*k);
  if (code < 0 || dtype_code(*v) != code || k->dim() != 4 || v->sizes() != k->sizes() ||
      k->size(2) != c.H || k->size(3) != c.D || k->numel() == 0 ||
      !aligned_rows(*k, code == MPX_F32 ? 4 : 8) || !aligned_rows(*v, code == MPX_F32 ? 4 : 8) ||
      c.bt->size(0) != k->size(0) || tracked({k, v}) || dual({k, v, c.ks, c.vs}))
    Py_RETURN_NONE;
  const int64_t B = k->size(0), T = k->size(1);
  if (B >= 65535 || T >= INT32_MAX || !int32_vector(*start, B) || (count && !int32_vector(*count, B)))
    Py_RETURN_NONE;
  const at::Tensor *cos = nullptr, *sin = nullptr;
  if (a[8] != Py_None) {
    if (!PyTuple_CheckExact(a[8]) || PyTuple_GET_SIZE(a[8]) != 2) Py_RETURN_NONE;
    cos = plain_on(PyTuple_GET_ITEM(a[8], 0), dev);
    sin = plain_on(PyTuple_GET_ITEM(a[8], 1), dev);
    if (!table_pair(cos, sin, c.D) || dual({cos, sin})) Py_RETURN_NONE;
  }
  const int words = cos ? 4 : 3;
  if (err && (err->scalar_type() != at::kInt || err->numel() != words || !err->is_contiguous()))
    Py_RETURN_NONE;
  const c10::DeviceGuard guard(dev);
  at::Tensor made;
  if (!err) {
    made = at::empty({words}, start->options());
    err = &made;
  }
  const int64_t ks[3] = {k->stride(0), k->stride(1), k->stride(2)};
  const int64_t vs[3] = {v->stride(0), v->stride(1), v->stride(2)};
  const int rc = call([&] {
    return api.mpx_kv_append8(
        k->data_ptr(), v->data_ptr(), c.kp->data_ptr(), c.vp->data_ptr(), c.ks->data_ptr<float>(),
        c.vs->data_ptr<float>(), c.bt->data_ptr<int32_t>(), start->data_ptr<int32_t>(),
        count ? count->data_ptr<int32_t>() : nullptr, ks, vs, (int)B, (int)T, c.H, c.D, c.nb, c.bs,
        c.mb, code, c.code, cos ? cos->data_ptr() : nullptr, sin ? sin->data_ptr() : nullptr,
        cos ? (int)cos->size(0) : 0, cos ? dtype_code(*cos) : 0, err->data_ptr<int32_t>(),
        stream_of(*k));
  });
  if (rc != MPX_OK) return PyLong_FromLong(rc);
  if (made.defined()) return THPVariable_Wrap(std::move(made));
  Py_INCREF(a[7]);
  return a[7];
  END_HANDLE_TH_ERRORS
}

// load8(k_pool, v_pool, tables, starts, counts, T, scales, dtype code) -> (k, v), an
//   error code, or None
PyObject* load8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (wrong_count(n, 8)) return nullptr;
  const Cache8 c(a[0], a[1], a[2], a[6]);
  if (!c.ok || !PyLong_CheckExact(a[5]) || !PyLong_CheckExact(a[7])) Py_RETURN_NONE;
  const c10::Device dev = c.kp->device();
  const at::Tensor *start = plain_on(a[3], dev), *count = plain_on(a[4], dev);
  const int64_t B = c.bt->size(0), T = PyLong_AsLongLong(a[5]);
  const int64_t dt = PyLong_AsLongLong(a[7]);
  if (PyErr_Occurred()) return nullptr;
  if (!start || !count || T <= 0 || T >= INT32_MAX || B == 0 || c.H == 0 || dt < 0 || dt > 2 ||
      !int32_vector(*start, B) || !int32_vector(*count, B) || dual({c.ks, c.vs}))
    Py_RETURN_NONE;
  const c10::DeviceGuard guard(dev);
  const auto opts = c.ks->options().dtype(dt == MPX_F32   ? at::kFloat
                                          : dt == MPX_F16 ? at::kHalf
                                                          : at::kBFloat16);
  at::Tensor k = at::empty({B, T, c.H, c.D}, opts), v = at::empty({B, T, c.H, c.D}, opts);
  const int rc = call([&] {
    return api.mpx_kv_load8(c.kp->data_ptr(), c.vp->data_ptr(), c.ks->data_ptr<float>(),
                            c.vs->data_ptr<float>(), c.bt->data_ptr<int32_t>(),
                            start->data_ptr<int32_t>(), count->data_ptr<int32_t>(), k.data_ptr(),
                            v.data_ptr(), (int)B, (int)T, c.H, c.D, c.nb, c.bs, c.mb, (int)dt,
                            c.code, stream_of(k));
  });
  if (rc != MPX_OK) return PyLong_FromLong(rc);
  PyObject* out = PyTuple_New(2);
  if (!out) return nullptr;
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(k)));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(v)));
  return out;
  END_HANDLE_TH_ERRORS
}

// attend8(q, k_pool, v_pool, tables, lens, scale or None, block_size, causal,
//   slopes or None, gqa, scales, query_start or None) -> o, an error code, or None
PyObject* attend8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (wrong_count(n, 12)) return nullptr;
  const Cache8 c(a[1], a[2], a[3], a[10]);
  if (!c.ok) Py_RETURN_NONE;
  const c10::Device dev = c.kp->device();
  const at::Tensor *q = plain_on(a[0], dev), *cl = plain_on(a[4], dev);
  const at::Tensor* sl = a[8] == Py_None ? nullptr : plain_on(a[8], dev);
  const at::Tensor* qs = a[11] == Py_None ? nullptr : plain_on(a[11], dev);
  if (!q || !cl || (!sl && a[8] != Py_None) || (!qs && a[11] != Py_None) ||
      !(a[5] == Py_None || PyFloat_CheckExact(a[5])) || !PyLong_CheckExact(a[6]) ||
      !PyBool_Check(a[7]) || !PyBool_Check(a[9]) || PyLong_AsLongLong(a[6]) != c.bs)
    Py_RETURN_NONE;
  const int code = dtype_code(*q);
  if (code < 0 || q->dim() != 4 || q->size(3) != c.D || q->numel() == 0 ||
      !aligned_rows(*q, code == MPX_F32 ? 4 : 8) || tracked({q, sl, c.ks, c.vs}) ||
      dual({q, sl, c.ks, c.vs}))
    Py_RETURN_NONE;
  const int64_t B = q->size(0), Sq = q->size(1), H = q->size(2);
  if (B > 65535 || Sq * H >= (1 << 30) || c.H == 0 ||
      (a[9] == Py_True ? H % c.H != 0 : H != c.H) || c.bt->size(0) != B || !int32_vector(*cl, B) ||
      (qs && !int32_vector(*qs, B)) ||
      (sl && (sl->scalar_type() != at::kFloat || sl->numel() != H || !sl->is_contiguous())))
    Py_RETURN_NONE;
  const double scale = a[5] == Py_None ? 1.0 / std::sqrt((double)c.D) : PyFloat_AsDouble(a[5]);
  const c10::DeviceGuard guard(dev);
  at::Tensor o = at::empty(q->sizes(), q->options()), ws;
  const size_t need = api.mpx_paged_attend8_call_workspace_bytes(
      (int)B, (int)Sq, (int)H, c.H, c.D, c.bs, c.mb, code, a[7] == Py_True, qs != nullptr);
  if (need) ws = bytes(need, *q);
  const int64_t qst[3] = {q->stride(0), q->stride(2), q->stride(1)};
  const int64_t ost[3] = {o.stride(0), o.stride(2), o.stride(1)};
  const int rc = call([&] {
    return api.mpx_paged_attend8(
        q->data_ptr(), c.kp->data_ptr(), c.vp->data_ptr(), c.ks->data_ptr<float>(),
        c.vs->data_ptr<float>(), c.bt->data_ptr<int32_t>(), cl->data_ptr<int32_t>(),
        qs ? qs->data_ptr<int32_t>() : nullptr, sl ? sl->data_ptr<float>() : nullptr, o.data_ptr(),
        qst, ost, (int)B, (int)Sq, (int)H, c.H, c.D, c.nb, c.bs, c.mb, (float)scale,
        a[7] == Py_True, code, c.code, need ? ws.data_ptr() : nullptr, need, stream_of(*q));
  });
  if (rc != MPX_OK) return PyLong_FromLong(rc);
  return THPVariable_Wrap(std::move(o));
  END_HANDLE_TH_ERRORS
}

// q, k, weights and tables of one call, and the call's numbers.
struct NormCall {
  at::Tensor q, k, wq, wk, cos, sin, pos, err;  // pos, err: undefined where an offset is given
  int64_t offset;
  double eps;
};

int norm_forward(const NormCall& c, at::Tensor& oq, at::Tensor& ok) {
  oq = at::empty(c.q.sizes(), c.q.options());
  ok = at::empty(c.k.sizes(), c.k.options());
  const int64_t qs[3] = {c.q.stride(0), c.q.stride(1), c.q.stride(2)};
  const int64_t ks[3] = {c.k.stride(0), c.k.stride(1), c.k.stride(2)};
  return api.mpx_qk_norm_rope(
      c.q.data_ptr(), c.k.data_ptr(), c.wq.data_ptr(), c.wk.data_ptr(), c.cos.data_ptr(),
      c.sin.data_ptr(), oq.data_ptr(), ok.data_ptr(), qs, ks, (int)c.q.size(0), (int)c.q.size(1),
      (int)c.q.size(2), (int)c.k.size(2), (int)c.q.size(3), (int)c.offset,
      c.pos.defined() ? c.pos.data_ptr<int32_t>() : nullptr, (int)c.cos.size(0), (float)c.eps,
      dtype_code(c.q), dtype_code(c.wq), dtype_code(c.cos),
      c.err.defined() ? c.err.data_ptr<int32_t>() : nullptr, stream_of(c.q));
}

using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

// The differentiable call: saves its inputs, whose norms the backward computes
// again, and refuses to be differentiated twice.
struct NormFunction : torch::autograd::Function<NormFunction> {
  static variable_list forward(AutogradContext* ctx, const Variable& q, const Variable& k,
                               const Variable& wq, const Variable& wk, const NormCall& c) {
    at::Tensor oq, ok;
    const int rc = norm_forward(c, oq, ok);
    TORCH_CHECK(rc == MPX_OK, api.mpx_last_error());
    ctx->save_for_backward({q, k, wq, wk, c.cos, c.sin, c.pos});
    ctx->saved_data["offset"] = c.offset;
    ctx->saved_data["eps"] = c.eps;
    return {oq, ok};
  }

  static variable_list backward(AutogradContext* ctx, variable_list dy) {
    const variable_list s = ctx->get_saved_variables();
    const at::Tensor &q = s[0], &k = s[1], &wq = s[2], &wk = s[3], &cos = s[4], &sin = s[5];
    const at::Tensor& pos = s[6];
    const bool again = at::GradMode::is_enabled();
    variable_list out(5);  // (one for each argument of forward)
    {
      const at::NoGradGuard none;
      const c10::DeviceGuard guard(q.device());
      const int code = dtype_code(q);
      auto rows = [&](const at::Tensor& t) {
        if (aligned_rows(t, code == MPX_F32 ? 4 : 8)) return t;
        const at::Tensor u = t.contiguous();
        return aligned(u) ? u : u.clone();
      };
      const at::Tensor gq = rows(dy[0]), gk = rows(dy[1]);
      at::Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options());
      at::Tensor dwq = at::empty(wq.sizes(), wq.options()), dwk = at::empty(wk.sizes(), wk.options());
      const int B = (int)q.size(0), S = (int)q.size(1), H = (int)q.size(2), D = (int)q.size(3);
      const int H_kv = (int)k.size(2);
      const size_t need = api.mpx_qk_norm_rope_bwd_workspace_bytes(B, S, H, H_kv, D);
      const at::Tensor ws = bytes(need, q);
      int64_t st[4][3];
      const at::Tensor* t[4] = {&q, &k, &gq, &gk};
      for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 3; ++j) st[i][j] = t[i]->stride(j);
      const int rc = api.mpx_qk_norm_rope_bwd(
          q.data_ptr(), k.data_ptr(), wq.data_ptr(), wk.data_ptr(), cos.data_ptr(), sin.data_ptr(),
          gq.data_ptr(), gk.data_ptr(), dq.data_ptr(), dk.data_ptr(), dwq.data_ptr(),
          dwk.data_ptr(), st[0], st[1], st[2], st[3], B, S, H, H_kv, D,
          (int)ctx->saved_data["offset"].toInt(), pos.defined() ? pos.data_ptr<int32_t>() : nullptr,
          (int)cos.size(0), (float)ctx->saved_data["eps"].toDouble(), code, dtype_code(wq),
          dtype_code(cos), ws.data_ptr(), need, stream_of(q));
      TORCH_CHECK(rc == MPX_OK, api.mpx_last_error());
      out[0] = std::move(dq);
      out[1] = std::move(dk);
      out[2] = std::move(dwq);
      out[3] = std::move(dwk);
    }
    if (again) {  // (create_graph: what is made of these gradients cannot be differentiated)
      variable_list grads(out.begin(), out.begin() + 4);
      for (Variable& g : grads) g.requires_grad_(true);
      auto error = std::make_shared<torch::autograd::DelayedError>(
          "trying to differentiate twice a function that was marked with @once_differentiable", 4);
      grads = (*error)(std::move(grads));
      std::move(grads.begin(), grads.end(), out.begin());
    }
    return out;
  }
};

// A backward pass that is being captured cannot end in a leaf whose gradient node
// was made on the default stream, by an eager graph that is still alive: the node
// keeps its stream, and work of a capture that waits on the default stream ends the
// process. So the forward refuses such leaves.
bool has_live_leaf(std::initializer_list<const at::Tensor*> tensors) {
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return false;
  for (const at::Tensor* t : tensors) {
    if (!t->requires_grad() || !t->is_leaf()) continue;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
    const auto stream = node ? node->stream() : std::nullopt;
    if (stream && stream->id() == 0) return true;
  }
  return false;
}

// live_leaf(tensors...) -> bool
PyObject* live_leaf(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  for (Py_ssize_t i = 0; i < n; ++i) {
    const at::Tensor* t = plain(a[i]);
    if (t && has_live_leaf({t})) Py_RETURN_TRUE;
  }
  Py_RETURN_FALSE;
  END_HANDLE_TH_ERRORS
}

// qk_norm_rope(q, k, q_weight, k_weight, cos, sin, offset, eps, positions or None,
//   errors or None) -> (q_out, k_out), an error code, or None
PyObject* qk_norm_rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (wrong_count(n, 10)) return nullptr;
  const at::Tensor* t[6];
  for (int i = 0; i < 6; ++i)
    if (!(t[i] = i ? plain_on(a[i], t[0]->device()) : plain(a[0]))) Py_RETURN_NONE;
  const at::Tensor &q = *t[0], &k = *t[1], &wq = *t[2], &wk = *t[3];
  const int code = dtype_code(q), wcode = dtype_code(wq);
  if (code < 0 || wcode < 0 || dtype_code(k) != code || dtype_code(wk) != wcode || q.dim() != 4 ||
      k.dim() != 4 || q.numel() == 0 || k.numel() == 0)
    Py_RETURN_NONE;
  const int64_t B = q.size(0), S = q.size(1), D = q.size(3);
  const int vec = code == MPX_F32 ? 4 : 8;
  if (k.size(0) != B || k.size(1) != S || k.size(3) != D || D % 16 != 0 || D > 256 ||
      B * S * (q.size(2) + k.size(2)) >= INT32_MAX || !aligned_rows(q, vec) ||
      !aligned_rows(k, vec) || wq.dim() != 1 || wq.size(0) != D || wk.sizes() != wq.sizes() ||
      !wq.is_contiguous() || !wk.is_contiguous() || !aligned(wq) || !aligned(wk) ||
      !table_pair(t[4], t[5], (int)D) || tracked({t[4], t[5]}) ||
      dual({t[0], t[1], t[2], t[3], t[4], t[5]}) || !PyLong_CheckExact(a[6]) ||
      !PyFloat_CheckExact(a[7]))
    Py_RETURN_NONE;
  NormCall c{q, k, wq, wk, *t[4], *t[5], {}, {}, PyLong_AsLongLong(a[6]), PyFloat_AsDouble(a[7])};
  if (PyErr_Occurred()) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  if (!(c.eps >= 0.0 && c.eps < INFINITY)) Py_RETURN_NONE;
  if (a[8] == Py_None) {
    if (a[9] != Py_None || c.offset < 0 || c.offset + S > c.cos.size(0)) Py_RETURN_NONE;
  } else {
    const at::Tensor* pos = plain_on(a[8], q.device());
    const at::Tensor* e = a[9] == Py_None ? nullptr : plain_on(a[9], q.device());
    if (!pos || !int32_vector(*pos, B) || c.offset != 0 || (!e && a[9] != Py_None)) Py_RETURN_NONE;
    if (e && (e->scalar_type() != at::kInt || e->numel() != 1)) Py_RETURN_NONE;
    c.pos = *pos;
    if (e) c.err = *e;
  }
  const c10::DeviceGuard guard(q.device());
  if (c.pos.defined() && !c.err.defined()) c.err = at::empty({1}, c.pos.options());
  at::Tensor oq, ok;
  int rc = MPX_OK;
  if (tracked({&q, &k, &wq, &wk})) {
    if (has_live_leaf({&q, &k, &wq, &wk})) Py_RETURN_NONE;  // (refused there)
    variable_list out;
    call([&] {
      out = NormFunction::apply(q, k, wq, wk, c);
      return 0;
    });
    oq = std::move(out[0]);
    ok = std::move(out[1]);
  } else {
    rc = call([&] { return norm_forward(c, oq, ok); });
  }
  if (rc != MPX_OK) return PyLong_FromLong(rc);
  PyObject* out = PyTuple_New(2);
  if (!out) return nullptr;
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(oq)));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(ok)));
  return out;
  END_HANDLE_TH_ERRORS
}

// init({entry name: address}): the library that the calls go to.
PyObject* init(PyObject*, PyObject* dict) {
#define X(name)                                                                       \
  {                                                                                   \
    PyObject* p = PyDict_GetItemString(dict, #name);                                  \
    if (!p) {                                                                         \
      PyErr_SetString(PyExc_KeyError, #name);                                         \
      return nullptr;                                                                 \
    }                                                                                 \
    api.name = reinterpret_cast<decltype(&::name)>(PyLong_AsVoidPtr(p));              \
    if (PyErr_Occurred()) return nullptr;                                             \
  }
  MPX_ENTRIES(X)
#undef X
  Py_RETURN_NONE;
}

// entries(): the names that init needs.
PyObject* entries(PyObject*, PyObject*) {
  PyObject* out = PyList_New(0);
  if (!out) return nullptr;
#define X(name)                                             \
  {                                                         \
    PyObject* s = PyUnicode_FromString(#name);              \
    if (!s || PyList_Append(out, s) != 0) {                 \
      Py_XDECREF(s);                                        \
      Py_DECREF(out);                                       \
      return nullptr;                                       \
    }                                                       \
    Py_DECREF(s);                                           \
  }
  MPX_ENTRIES(X)
#undef X
  return out;
}

#define FAST(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(attn_fwd),  FAST(attn_bwd), FAST(paged_attend),
                         FAST(kv_append), FAST(rope_at),  FAST(store8),
                         FAST(load8),     FAST(attend8),  FAST(qk_norm_rope),
                         FAST(live_leaf),
                         {"init", init, METH_O, nullptr},
                         {"entries", entries, METH_NOARGS, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_mpx_host", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__mpx_host() { return PyModule_Create(&module); }
