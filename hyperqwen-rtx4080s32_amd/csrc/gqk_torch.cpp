// gqk_torch.cpp - the eager way from torch to the C ABI for the calls of a decode step (host code, a CPython module).
//
// A step's small calls take 3 to 10 us on the GPU; checked and bound in Python they took 14 to 29 us of the host.  Each
// function here takes the arguments of its Python counterpart, makes the same checks, allocates the outputs, launches
// and returns the result - or returns None, with nothing done, wherever a call is not plainly all right: an argument of
// another type, layout, device or shape, a subclass, autograd, a mode or a profiler that wants to see the op, a device that
// is not current or has no workspace yet.  The Python path then raises its errors, or goes through the op.
#include <Python.h>
#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/record_function.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <math.h>
#include <vector>
#include "gguf_hip.h"

namespace {

using at::Tensor;

constexpr int kDevices = 64;
Tensor* g_workspace[kDevices];

// What the dispatcher would look at besides the backend: nothing of it is on.
bool plain_world() {
  using c10::DispatchKey;
  const c10::impl::LocalDispatchKeySet tls = c10::impl::tls_local_dispatch_key_set();
  const c10::DispatchKeySet usual({DispatchKey::BackendSelect, DispatchKey::ADInplaceOrView});
  return !(tls.included_.raw_repr() & ~usual.raw_repr()) && !c10::impl::TorchDispatchModeTLS::any_modes_set() &&
         !at::impl::torch_function_mode_enabled() && !at::hasCallbacks();
}

// A tensor as it is in memory: no subclass, no lazy negation, no autograd.
bool plain(PyObject* o, const Tensor** out) {
  if (!THPVariable_CheckExact(o)) return false;
  const Tensor& t = THPVariable_Unpack(o);
  using c10::DispatchKey;
  static const c10::DispatchKeySet usual({DispatchKey::CUDA, DispatchKey::ADInplaceOrView, DispatchKey::AutogradCUDA,
                                          DispatchKey::AutocastCUDA});   // autocast has no rule for these ops
  if (!t.defined() || (t.key_set().raw_repr() & ~usual.raw_repr()) || !t.is_cuda()) return false;
  if (t.requires_grad() && c10::GradMode::is_enabled()) return false;
  *out = &t;
  return true;
}
// the same or None
bool plain_or_none(PyObject* o, const Tensor** out) {
  *out = nullptr;
  return o == Py_None || plain(o, out);
}

bool same_device(const Tensor& a, const Tensor* b) { return !b || b->get_device() == a.get_device(); }
bool aligned(const Tensor& t, size_t n) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & (n - 1)) == 0; }

int heads_type(at::ScalarType t) {
  return t == at::kBFloat16 ? GQK_DTYPE_BF16 : t == at::kHalf ? GQK_DTYPE_F16 : -1;
}

// [tokens, heads, dim] as the kernels read them
bool heads_of(const Tensor* t, gqk_heads* h) {
  if (t->dim() != 3 || t->size(2) > 0x7fffffff) return false;
  const int64_t row = t->size(0) > 1 ? t->stride(0) : 0, head = t->size(1) > 1 ? t->stride(1) : 0;
  if (t->stride(2) != 1 || ((row | head) & 7) || row < 0 || head < 0 || !aligned(*t, 16)) return false;
  *h = gqk_heads{t->data_ptr(), row, head, static_cast<int32_t>(t->size(1))};
  return true;
}

bool like(const Tensor& a, const Tensor& b) {
  return a.scalar_type() == b.scalar_type() && a.get_device() == b.get_device() && a.sizes() == b.sizes();
}

bool scale_of(const Tensor* s, int64_t heads, const Tensor& ref) {
  return !s || (s->scalar_type() == at::kFloat && s->dim() == 1 && s->size(0) == heads && s->is_contiguous() && same_device(ref, s));
}

bool pages_of(const Tensor& k, const Tensor& v, const Tensor* ks, const Tensor* vs, const Tensor& ref, gqk_pages* p) {
  if (k.dim() != 4 || k.sizes() != v.sizes() || k.scalar_type() != v.scalar_type()) return false;
  const int type = k.scalar_type() == at::kFloat8_e4m3fn ? GQK_DTYPE_FP8 : heads_type(k.scalar_type());
  if (type < 0 || (type != GQK_DTYPE_FP8 && k.scalar_type() != ref.scalar_type())) return false;
  if (k.stride(3) != 1 || v.stride(3) != 1 || k.size(3) != ref.size(2) || !same_device(ref, &k) || !same_device(ref, &v)) return false;
  if (!scale_of(ks, k.size(2), ref) || !scale_of(vs, k.size(2), ref)) return false;
  for (int i = 0; i < 3; ++i)
    if (k.size(i) < 1 || k.size(i) > 0x7fffffff) return false;
  auto stride = [](const Tensor& t, int i) { return t.size(i) > 1 ? t.stride(i) : 0; };
  *p = gqk_pages{k.data_ptr(), v.data_ptr(), stride(k, 0), stride(k, 1), stride(k, 2), stride(v, 0), stride(v, 1), stride(v, 2),
                 ks ? ks->data_ptr<float>() : nullptr, vs ? vs->data_ptr<float>() : nullptr, type, static_cast<int32_t>(k.size(0)),
                 static_cast<int32_t>(k.size(1)), static_cast<int32_t>(k.size(2)), static_cast<int32_t>(k.size(3))};
  return true;
}

bool index_of(const Tensor& t, int64_t n, const Tensor& ref) {
  return (t.scalar_type() == at::kInt || t.scalar_type() == at::kLong) && t.dim() == 1 && t.size(0) == n && t.is_contiguous() &&
         same_device(ref, &t);
}

bool here(const Tensor& t) { return t.get_device() < kDevices && c10::hip::current_device() == t.get_device(); }
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

// the call's workspace: its own, or the device's
bool workspace_of(const Tensor* own, const Tensor& ref, void** at, int64_t* bytes) {
  const Tensor* t = own ? own : g_workspace[ref.get_device()];
  if (!t || !same_device(ref, t) || !t->is_contiguous()) return false;
  *at = t->data_ptr();
  *bytes = t->numel() * t->element_size();
  return true;
}

void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

PyObject* none() { Py_RETURN_NONE; }

// paged_attention(q, k_pages, v_pages, block_table, lengths, scale, window, k_scale, v_scale, max_length, out, return_lse, workspace)
PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Tensor *q, *k, *v, *table, *lengths, *ks, *vs, *out, *ws;
  if (n != 13 || !plain_world() || !plain(a[0], &q) || !plain(a[1], &k) || !plain(a[2], &v) || !plain(a[3], &table) ||
      !plain(a[4], &lengths) || !plain_or_none(a[7], &ks) || !plain_or_none(a[8], &vs) || !plain_or_none(a[10], &out) ||
      !plain_or_none(a[12], &ws))
    return none();
  gqk_heads qh, oh;
  gqk_pages p;
  const int type = heads_type(q->scalar_type());
  if (type < 0 || !here(*q) || !heads_of(q, &qh) || !pages_of(*k, *v, ks, vs, *q, &p)) return none();
  const int64_t batch = q->size(0), heads = q->size(1), dim = q->size(2);
  if (batch < 1 || batch > 65535 || heads < 1 || heads % p.heads) return none();
  if (table->scalar_type() != at::kInt || table->dim() != 2 || table->size(0) != batch || !same_device(*q, table) ||
      (table->size(1) > 1 && table->stride(1) != 1) || table->size(1) > 0x7fffffff || lengths->scalar_type() != at::kInt ||
      lengths->dim() != 1 || lengths->size(0) != batch || !lengths->is_contiguous() || !same_device(*q, lengths))
    return none();
  const int64_t room = std::min<int64_t>(table->size(1) * p.page_size, GQK_MAX_KEYS);
  int64_t window = 0, most = room;
  double scale = 1.0 / sqrt(static_cast<double>(dim));
  if (!PyLong_CheckExact(a[6])) return none();
  window = PyLong_AsLongLong(a[6]);
  if (a[9] != Py_None) {
    if (!PyLong_CheckExact(a[9])) return none();
    most = PyLong_AsLongLong(a[9]);
  }
  if (a[5] != Py_None) {
    if (!PyFloat_CheckExact(a[5])) return none();
    scale = PyFloat_AS_DOUBLE(a[5]);
  }
  if (PyErr_Occurred()) {   // an integer beyond 64 bits
    PyErr_Clear();
    return none();
  }
  if (window < 0 || window > 0x7fffffff || most < 0 || most > room) return none();
  void* space;
  int64_t bytes;
  if (!workspace_of(ws, *q, &space, &bytes) || (out && (!like(*out, *q) || !heads_of(out, &oh)))) return none();
  Tensor made, lse;
  if (!out) {
    made = at::empty({batch, heads, dim}, q->options());
    heads_of(&made, &oh);
  }
  const bool with_lse = a[11] == Py_True;
  if (with_lse) lse = at::empty({batch, heads}, q->options().dtype(at::kFloat));
  const int rc = gqk_paged_attention(qh.data, qh.row, qh.head, type, static_cast<int>(batch), static_cast<int>(heads), &p,
                                     table->data_ptr<int>(), table->stride(0), static_cast<int>(table->size(1)),
                                     lengths->data_ptr<int>(), static_cast<int>(most), static_cast<int>(window),
                                     static_cast<float>(scale), oh.data, oh.row, oh.head, with_lse ? lse.data_ptr<float>() : nullptr,
                                     space, bytes, stream_of(*q));
  if (rc) return none();   // nothing was launched: the Python path says why
  PyObject* result = out ? (Py_INCREF(a[10]), a[10]) : THPVariable_Wrap(made);
  written(out ? *out : made);
  if (!with_lse) return result;
  return Py_BuildValue("(NN)", result, THPVariable_Wrap(lse));
  END_HANDLE_TH_ERRORS
}

// qk_norm_rope(q, k, positions, table, q_weight, k_weight, eps, flags, v, k_pages, v_pages, slots, k_scale, v_scale, out_q, out_k)
PyObject* rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Tensor *q, *k, *pos, *table, *wq, *wk, *v, *kp, *vp, *slots, *ks, *vs, *oq, *ok;
  if (n != 16 || !plain_world() || !plain(a[0], &q) || !plain_or_none(a[1], &k) || !plain(a[2], &pos) || !plain(a[3], &table) ||
      !plain_or_none(a[4], &wq) || !plain_or_none(a[5], &wk) || !plain_or_none(a[8], &v) || !plain_or_none(a[9], &kp) ||
      !plain_or_none(a[10], &vp) || !plain_or_none(a[11], &slots) || !plain_or_none(a[12], &ks) || !plain_or_none(a[13], &vs) ||
      !plain_or_none(a[14], &oq) || !plain_or_none(a[15], &ok) || !PyFloat_CheckExact(a[6]) || !PyLong_CheckExact(a[7]))
    return none();
  gqk_heads qh, kh, vh, oqh, okh;
  gqk_pages p;
  const int type = heads_type(q->scalar_type());
  if (type < 0 || !here(*q) || !heads_of(q, &qh)) return none();
  const int64_t tokens = q->size(0), dim = q->size(2);
  if (tokens < 1 || q->size(1) < 1) return none();
  for (const Tensor* t : {k, v})
    if (t && (t->dim() != 3 || t->size(0) != tokens || t->size(1) < 1 || t->size(2) != dim || t->scalar_type() != q->scalar_type() ||
              !same_device(*q, t)))
      return none();
  if ((k && !heads_of(k, &kh)) || (v && !heads_of(v, &vh)) || (!k && (wk || ok))) return none();
  for (const Tensor* w : {wq, wk})
    if (w && (w->dim() != 1 || w->size(0) != dim || (w->scalar_type() != q->scalar_type() && w->scalar_type() != at::kFloat) ||
              !w->is_contiguous() || !same_device(*q, w)))
      return none();
  if (wq && wk && wq->scalar_type() != wk->scalar_type()) return none();
  if (!index_of(*pos, tokens, *q) || table->scalar_type() != at::kFloat || table->dim() != 2 || table->size(1) % 2 ||
      table->size(1) > dim || !table->is_contiguous() || !same_device(*q, table))
    return none();
  if (kp) {
    if (!vp || !k || !v || !slots || !pages_of(*kp, *vp, ks, vs, *k, &p) || k->size(1) != p.heads || v->size(1) != p.heads ||
        !index_of(*slots, tokens, *q))
      return none();
  } else if (v || vp || slots || ks || vs) {
    return none();
  }
  if ((oq && (!like(*oq, *q) || !heads_of(oq, &oqh))) || (ok && (!like(*ok, *k) || !heads_of(ok, &okh)))) return none();
  Tensor made_q, made_k;
  if (!oq) {
    made_q = at::empty(q->sizes(), q->options());
    heads_of(&made_q, &oqh);
  }
  const bool new_k = !ok && k && !kp;
  if (new_k) {
    made_k = at::empty(k->sizes(), k->options());
    heads_of(&made_k, &okh);
  }
  const Tensor* w = wq ? wq : wk;
  const int rc = gqk_qk_norm_rope(&qh, k ? &kh : nullptr, v ? &vh : nullptr, type, tokens, static_cast<int>(dim), pos->data_ptr(),
                                  pos->scalar_type() == at::kLong, table->data_ptr<float>(), table->size(0),
                                  static_cast<int>(table->size(1)), wq ? wq->data_ptr() : nullptr, wk ? wk->data_ptr() : nullptr,
                                  w && w->scalar_type() == at::kFloat ? GQK_DTYPE_F32 : type,
                                  static_cast<float>(PyFloat_AS_DOUBLE(a[6])), static_cast<int>(PyLong_AsLong(a[7])), &oqh,
                                  ok || new_k ? &okh : nullptr, kp ? &p : nullptr, slots ? slots->data_ptr() : nullptr,
                                  slots && slots->scalar_type() == at::kLong, stream_of(*q));
  if (rc) return none();
  for (const Tensor* t : {oq, ok, kp, vp})
    if (t) written(*t);
  PyObject* first = oq ? (Py_INCREF(a[14]), a[14]) : THPVariable_Wrap(made_q);
  PyObject* second = ok ? (Py_INCREF(a[15]), a[15]) : new_k ? THPVariable_Wrap(made_k) : none();
  return Py_BuildValue("(NN)", first, second);
  END_HANDLE_TH_ERRORS
}

// lora_add(y, x, a, b, ids, scales, n_outs, out, workspace)
PyObject* lora(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Tensor *y, *x, *A, *B, *ids, *scales, *out, *ws;
  if (n != 9 || !plain_world() || !plain(a[0], &y) || !plain(a[1], &x) || !plain(a[2], &A) || !plain(a[3], &B) || !plain(a[4], &ids) ||
      !plain_or_none(a[5], &scales) || !plain_or_none(a[7], &out) || !plain_or_none(a[8], &ws))
    return none();
  const bool tuple = PyTuple_CheckExact(a[6]);
  if (!tuple && !PyList_CheckExact(a[6])) return none();
  const Py_ssize_t parts = tuple ? PyTuple_GET_SIZE(a[6]) : PyList_GET_SIZE(a[6]);
  if (parts < 1 || parts > 8) return none();
  int64_t outs[8], N = 0;
  for (Py_ssize_t i = 0; i < parts; ++i) {
    PyObject* o = tuple ? PyTuple_GET_ITEM(a[6], i) : PyList_GET_ITEM(a[6], i);
    if (!PyLong_CheckExact(o)) return none();
    outs[i] = PyLong_AsLongLong(o);
    if (outs[i] < 1 || outs[i] > 0x7fffffff) {
      PyErr_Clear();
      return none();
    }
    N += outs[i];
  }
  const int type = heads_type(x->scalar_type());
  if (type < 0 || !here(*x) || x->dim() != 2) return none();
  const int64_t M = x->size(0), K = x->size(1);
  if (M < 1 || M > 0x7fffffff || K < 8) return none();
  if (A->dim() != 4 || A->size(1) != parts || A->size(3) != K || B->dim() != 3 || B->size(0) != A->size(0) || B->size(1) != N ||
      B->size(2) != A->size(2) || A->size(0) > 0x7fffffff || A->size(2) > 256)
    return none();
  for (const Tensor* t : {A, B})
    if (t->scalar_type() != x->scalar_type() || !t->is_contiguous() || !same_device(*x, t)) return none();
  for (const Tensor* t : {y, out})
    if (t && (t->dim() != 2 || t->size(0) != M || t->size(1) != N || t->scalar_type() != x->scalar_type() || !same_device(*x, t) ||
              (N > 1 && t->stride(1) != 1) || (M > 1 && t->stride(0) < N)))
      return none();
  if ((x->stride(1) != 1) || (M > 1 && (x->stride(0) < K || x->stride(0) % 8 || x->stride(0) > GQK_LORA_MAX_K))) return none();
  if (!index_of(*ids, M, *x) || (scales && (scales->scalar_type() != at::kFloat || scales->dim() != 1 ||
                                            scales->size(0) != A->size(0) || !scales->is_contiguous() || !same_device(*x, scales))))
    return none();
  void* space;
  int64_t bytes;
  if (!workspace_of(ws, *x, &space, &bytes)) return none();
  const int64_t need = gqk_lora_workspace_bytes(static_cast<int>(M), K, static_cast<int>(parts), static_cast<int>(A->size(2)));
  if (need < 0 || need > bytes) return none();   // rows in turns: the Python path
  Tensor made;
  if (!out) made = at::empty({M, N}, x->options());
  const Tensor& to = out ? *out : made;
  auto row = [&](const Tensor& t) { return M > 1 ? t.stride(0) : t.size(1); };
  const int rc = gqk_lora_add(y->data_ptr(), row(*y), x->data_ptr(), row(*x), static_cast<int>(M), K, A->data_ptr(), B->data_ptr(),
                              static_cast<int>(A->size(0)), static_cast<int>(parts), outs, static_cast<int>(A->size(2)),
                              ids->data_ptr(), ids->scalar_type() == at::kLong, scales ? scales->data_ptr<float>() : nullptr, type,
                              to.data_ptr(), row(to), space, bytes, stream_of(*x));
  if (rc) return none();
  written(to);
  if (!out) return THPVariable_Wrap(made);
  Py_INCREF(a[7]);
  return a[7];
  END_HANDLE_TH_ERRORS
}

// page numbers of a list or a contiguous CPU tensor
bool numbers(PyObject* o, std::vector<int32_t>& to) {
  if (THPVariable_CheckExact(o)) {
    const Tensor& t = THPVariable_Unpack(o);
    if (!t.defined() || !t.device().is_cpu() || t.layout() != at::kStrided || t.dim() != 1 || !t.is_contiguous() || t.is_neg()) return false;
    to.resize(t.numel());
    if (t.scalar_type() == at::kInt) {
      std::copy_n(t.data_ptr<int>(), t.numel(), to.data());
    } else if (t.scalar_type() == at::kLong) {
      const int64_t* from = t.data_ptr<int64_t>();
      for (int64_t i = 0; i < t.numel(); ++i) {
        if (from[i] < 0 || from[i] > 0x7fffffff) return false;
        to[i] = static_cast<int32_t>(from[i]);
      }
    } else {
      return false;
    }
    return true;
  }
  if (!PyList_CheckExact(o)) return false;
  to.resize(PyList_GET_SIZE(o));
  for (size_t i = 0; i < to.size(); ++i) {
    PyObject* x = PyList_GET_ITEM(o, i);
    if (!PyLong_CheckExact(x)) return false;
    const long long p = PyLong_AsLongLong(x);
    if (p < 0 || p > 0x7fffffff) {
      PyErr_Clear();
      return false;
    }
    to[i] = static_cast<int32_t>(p);
  }
  return true;
}

// copy_pages(pages, src, dst, dim): True when done
PyObject* copy(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Tensor* t;
  if (n != 4 || !plain_world() || !plain(a[0], &t) || !here(*t) || !PyLong_CheckExact(a[3])) return none();
  int64_t dim = PyLong_AsLongLong(a[3]);
  if (PyErr_Occurred()) PyErr_Clear();
  if (dim < 0) dim += t->dim();
  if (dim < 0 || dim >= t->dim() || t->numel() == 0) return none();
  std::vector<int32_t> src, dst;
  if (!numbers(a[1], src) || !numbers(a[2], dst) || src.size() != dst.size()) return none();
  int64_t own = 1, planes = 1, plane = 0;
  for (int64_t i = t->dim() - 1; i > dim; --i) {
    if (t->size(i) != 1 && t->stride(i) != own) return none();
    own *= t->size(i);
  }
  for (int64_t i = dim - 1; i >= 0; --i) {
    if (t->size(i) == 1) continue;
    if (planes > 1 && t->stride(i) != plane * planes) return none();
    if (planes == 1) plane = t->stride(i);
    planes *= t->size(i);
  }
  const int64_t size = t->element_size(), page = t->size(dim) > 1 ? t->stride(dim) : own;
  if (gqk_copy_pages(t->data_ptr(), planes, plane * size, t->size(dim), page * size, own * size, src.data(), dst.data(),
                     static_cast<int64_t>(src.size()), stream_of(*t)))
    return none();
  written(*t);
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// set_workspace(device index, tensor): what a call without a workspace of its own uses
PyObject* set_workspace(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Tensor* t;
  const long i = n == 2 ? PyLong_AsLong(a[0]) : -1;
  if (i < 0 || i >= kDevices || !plain(a[1], &t)) {
    PyErr_Clear();
    return none();
  }
  delete g_workspace[i];
  g_workspace[i] = new Tensor(*t);
  return none();
  END_HANDLE_TH_ERRORS
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f))
PyMethodDef methods[] = {{"paged_attention", FAST(attention), METH_FASTCALL, nullptr},
                         {"qk_norm_rope", FAST(rope), METH_FASTCALL, nullptr},
                         {"lora_add", FAST(lora), METH_FASTCALL, nullptr},
                         {"copy_pages", FAST(copy), METH_FASTCALL, nullptr},
                         {"set_workspace", FAST(set_workspace), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fast", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fast() { return PyModule_Create(&module); }
