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

// contiguous int32 [n]
bool i32_of(const Tensor& t, int64_t n, const Tensor& ref) {
  return t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == n && t.is_contiguous() && same_device(ref, &t);
}

// a page table of so many dimensions: int32, its columns side by side
bool table_of(const Tensor& t, int64_t dims, int64_t batch, const Tensor& ref) {
  return t.scalar_type() == at::kInt && t.dim() == dims && t.size(0) == batch && same_device(ref, &t) && t.size(-1) <= 0x7fffffff &&
         (t.size(-1) <= 1 || t.stride(-1) == 1);
}

// a Python integer of 0 .. 2^31 - 1
bool int_of(PyObject* o, int64_t* to) {
  if (!PyLong_CheckExact(o)) return false;
  *to = PyLong_AsLongLong(o);
  if (PyErr_Occurred()) {   // beyond 64 bits
    PyErr_Clear();
    return false;
  }
  return *to >= 0 && *to <= 0x7fffffff;
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
  const bool by_head = table->dim() == 3;   // a table for each of the pages' heads
  if (by_head && table->size(1) != p.heads) return none();
  if (!table_of(*table, by_head ? 3 : 2, batch, *q) || !i32_of(*lengths, batch, *q)) return none();
  const int64_t width = table->size(-1), room = std::min<int64_t>(width * p.page_size, GQK_MAX_KEYS);
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
  const int rc = gqk_paged_attention_heads(
      qh.data, qh.row, qh.head, type, static_cast<int>(batch), static_cast<int>(heads), &p, table->data_ptr<int>(), table->stride(0),
      by_head ? table->stride(1) : 0, static_cast<int>(width), lengths->data_ptr<int>(), static_cast<int>(most), static_cast<int>(window),
      static_cast<float>(scale), oh.data, oh.row, oh.head, with_lse ? lse.data_ptr<float>() : nullptr, space, bytes, stream_of(*q));
  if (rc) return none();   // nothing was launched: the Python path says why
  PyObject* result = out ? (Py_INCREF(a[10]), a[10]) : THPVariable_Wrap(made);
  written(out ? *out : made);
  if (!with_lse) return result;
  return Py_BuildValue("(NN)", result, THPVariable_Wrap(lse));
  END_HANDLE_TH_ERRORS
}

// tree_attention(q, k_pages, v_pages, block_table, lengths, starts, mask, scale, window, k_scale, v_scale, max_length, max_tokens, out,
// return_lse, workspace)
PyObject* tree(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Tensor *q, *k, *v, *table, *lengths, *starts, *mask, *ks, *vs, *out, *ws;
  if (n != 16 || !plain_world() || !plain(a[0], &q) || !plain(a[1], &k) || !plain(a[2], &v) || !plain(a[3], &table) ||
      !plain(a[4], &lengths) || !plain(a[5], &starts) || !plain_or_none(a[6], &mask) || !plain_or_none(a[9], &ks) ||
      !plain_or_none(a[10], &vs) || !plain_or_none(a[13], &out) || !plain_or_none(a[15], &ws))
    return none();
  gqk_heads qh, oh;
  gqk_pages p;
  const int type = heads_type(q->scalar_type());
  if (type < 0 || !here(*q) || !heads_of(q, &qh) || !pages_of(*k, *v, ks, vs, *q, &p) || lengths->dim() != 1) return none();
  const int64_t tokens = q->size(0), heads = q->size(1), dim = q->size(2), batch = lengths->size(0);
  if (batch < 1 || batch > 65535 || tokens < 1 || tokens > GQK_MAX_TOKENS || heads < 1 || heads % p.heads || heads / p.heads > GQK_MAX_GROUP)
    return none();
  if (!table_of(*table, 2, batch, *q) || !i32_of(*lengths, batch, *q) || !i32_of(*starts, batch + 1, *q)) return none();
  if (mask && (mask->scalar_type() != at::kInt || mask->dim() != 2 || mask->size(0) != tokens || mask->size(1) < 1 ||
               mask->size(1) > 0x7fffffff || !mask->is_contiguous() || !same_device(*q, mask)))
    return none();
  const int64_t room = std::min<int64_t>(table->size(1) * p.page_size, GQK_MAX_KEYS);
  int64_t window, most = room, most_tokens = tokens;
  double scale = 1.0 / sqrt(static_cast<double>(dim));
  if (!int_of(a[8], &window) || (a[11] != Py_None && !int_of(a[11], &most)) || most > room ||
      (a[12] != Py_None && !int_of(a[12], &most_tokens)))
    return none();
  most_tokens = std::min(most_tokens, tokens);
  if (a[7] != Py_None) {
    if (!PyFloat_CheckExact(a[7])) return none();
    scale = PyFloat_AS_DOUBLE(a[7]);
  }
  void* space;
  int64_t bytes;
  if (!workspace_of(ws, *q, &space, &bytes) || (out && (!like(*out, *q) || !heads_of(out, &oh)))) return none();
  if (out && out->storage().data() == q->storage().data() && (out->data_ptr() != q->data_ptr() || out->strides() != q->strides()))
    return none();   // q is copied
  Tensor made, lse;
  if (!out) {
    made = at::empty({tokens, heads, dim}, q->options());
    heads_of(&made, &oh);
  }
  const bool with_lse = a[14] == Py_True;
  if (with_lse) lse = at::empty({tokens, heads}, q->options().dtype(at::kFloat));
  const int rc = gqk_tree_attention(
      qh.data, qh.row, qh.head, type, static_cast<int>(tokens), static_cast<int>(batch), static_cast<int>(heads), &p, table->data_ptr<int>(),
      table->stride(0), static_cast<int>(table->size(1)), lengths->data_ptr<int>(), starts->data_ptr<int>(),
      mask ? mask->data_ptr<int>() : nullptr, mask ? static_cast<int>(mask->size(1)) : 0, static_cast<int>(most),
      static_cast<int>(most_tokens), static_cast<int>(window), static_cast<float>(scale), oh.data, oh.row, oh.head,
      with_lse ? lse.data_ptr<float>() : nullptr, space, bytes, stream_of(*q));
  if (rc) return none();
  PyObject* result = out ? (Py_INCREF(a[13]), a[13]) : THPVariable_Wrap(made);
  written(out ? *out : made);
  if (!with_lse) return result;
  return Py_BuildValue("(NN)", result, THPVariable_Wrap(lse));
  END_HANDLE_TH_ERRORS
}

// add_rms_norm(x, residual, weight, eps, flags, f8, group, out, out_residual): (out, residual), or with f8 (out, scale, residual)
PyObject* norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Tensor *x, *r, *w, *out, *rout;
  int64_t group;
  if (n != 9 || !plain_world() || !plain(a[0], &x) || !plain_or_none(a[1], &r) || !plain_or_none(a[2], &w) || !PyFloat_CheckExact(a[3]) ||
      !PyLong_CheckExact(a[4]) || !int_of(a[6], &group) || !plain_or_none(a[7], &out) || !plain_or_none(a[8], &rout))
    return none();
  const int type = heads_type(x->scalar_type());
  const bool f8 = a[5] == Py_True;
  if (type < 0 || !here(*x) || x->dim() != 2 || (f8 && out)) return none();   // (an 8-bit out may share memory: the Python path looks)
  const int64_t rows = x->size(0), dim = x->size(1);
  if (rows < 1 || rows > 0x7fffffff || dim < 1 || dim > GQK_NORM_MAX_DIM || (group && dim % group) || (!r && rout)) return none();
  for (const Tensor* t : {x, r, out, rout})
    if (t && (!like(*t, *x) || (dim > 1 && t->stride(1) != 1) || (rows > 1 && t->stride(0) < dim))) return none();
  if (w && (w->dim() != 1 || w->size(0) != dim || (w->scalar_type() != x->scalar_type() && w->scalar_type() != at::kFloat) ||
            !w->is_contiguous() || !same_device(*x, w)))
    return none();
  // outputs that share memory with another tensor, unless row by row the same as an input: the Python path looks
  if (out && rout && out->storage().data() == rout->storage().data()) return none();
  for (const Tensor* o : {out, rout})
    for (const Tensor* t : {x, r, w})
      if (o && t && o->storage().data() == t->storage().data() &&
          (t == w || o->data_ptr() != t->data_ptr() || (rows > 1 && o->stride(0) != t->stride(0))))
        return none();
  Tensor made, scale, made_r;
  if (!out) made = at::empty({rows, dim}, f8 ? x->options().dtype(at::kFloat8_e4m3fn) : x->options());
  if (f8) scale = at::empty({rows, group ? dim / group : 1}, x->options().dtype(at::kFloat));
  if (r && !rout) made_r = at::empty({rows, dim}, x->options());
  auto row = [&](const Tensor* t) { return rows > 1 ? t->stride(0) : dim; };
  const Tensor *to = out ? out : &made, *to_r = rout ? rout : r ? &made_r : nullptr;
  const int rc = gqk_add_rms_norm(x->data_ptr(), row(x), r ? r->data_ptr() : nullptr, r ? row(r) : 0, type, rows, static_cast<int>(dim),
                                  w ? w->data_ptr() : nullptr, w && w->scalar_type() == at::kFloat ? GQK_DTYPE_F32 : type,
                                  static_cast<float>(PyFloat_AS_DOUBLE(a[3])), static_cast<int>(PyLong_AsLong(a[4])), to->data_ptr(),
                                  row(to), f8 ? GQK_DTYPE_FP8 : type, f8 ? scale.data_ptr<float>() : nullptr, static_cast<int>(group),
                                  to_r ? to_r->data_ptr() : nullptr, to_r ? row(to_r) : 0, stream_of(*x));
  if (rc) return none();
  for (const Tensor* t : {out, rout})
    if (t) written(*t);
  PyObject* first = out ? (Py_INCREF(a[7]), a[7]) : THPVariable_Wrap(made);
  PyObject* last = rout ? (Py_INCREF(a[8]), a[8]) : r ? THPVariable_Wrap(made_r) : none();
  if (!f8) return Py_BuildValue("(NN)", first, last);
  return Py_BuildValue("(NNN)", first, THPVariable_Wrap(scale), last);
  END_HANDLE_TH_ERRORS
}

// step_tables(page_lists, requests, lengths, counts, tokens, page_size, parents, tree): StepTables' fields
PyObject* tables(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Tensor *lists, *requests, *lengths, *counts, *parents;
  int64_t tokens, page_size, tree;
  if (n != 8 || !plain_world() || !plain(a[0], &lists) || !plain(a[1], &requests) || !plain(a[2], &lengths) || !plain(a[3], &counts) ||
      !int_of(a[4], &tokens) || !int_of(a[5], &page_size) || !plain_or_none(a[6], &parents) || !int_of(a[7], &tree))
    return none();
  if (!here(*lists) || lists->scalar_type() != at::kInt || lists->dim() != 2 || lists->size(0) > 0x7fffffff || lists->size(1) > 0x7fffffff ||
      (lists->size(1) > 1 && lists->stride(1) != 1) || (lists->size(0) > 1 && lists->stride(0) < lists->size(1)) || requests->dim() != 1)
    return none();
  const int64_t batch = requests->size(0), width = lists->size(1);
  if (batch > 65535 || !index_of(*requests, batch, *lists) || !i32_of(*lengths, batch, *lists) || !i32_of(*counts, batch, *lists) ||
      (parents && !i32_of(*parents, tokens, *lists)) || (parents != nullptr) != (tree > 0) || tree > GQK_MAX_TREE)
    return none();
  const auto i32 = lists->options();
  Tensor table = at::empty({batch, width}, i32), totals = at::empty({batch}, i32), starts = at::empty({batch + 1}, i32),
         sequences = at::empty({tokens}, i32), positions = at::empty({tokens}, i32), slots = at::empty({tokens}, i32.dtype(at::kLong)), mask;
  if (tree) mask = at::empty({tokens, (tree + 31) / 32}, i32);
  const int rc = gqk_step_tables(lists->data_ptr<int>(), lists->size(0) > 1 ? lists->stride(0) : width, static_cast<int>(lists->size(0)),
                                 static_cast<int>(width), requests->data_ptr(), requests->scalar_type() == at::kLong,
                                 lengths->data_ptr<int>(), counts->data_ptr<int>(), static_cast<int>(batch), static_cast<int>(tokens),
                                 static_cast<int>(page_size), parents ? parents->data_ptr<int>() : nullptr, static_cast<int>(tree),
                                 table.data_ptr<int>(), totals.data_ptr<int>(), starts.data_ptr<int>(), sequences.data_ptr<int>(),
                                 positions.data_ptr<int>(), slots.data_ptr<int64_t>(), tree ? mask.data_ptr<int>() : nullptr,
                                 stream_of(*lists));
  if (rc) return none();
  return Py_BuildValue("(NNNNNNN)", THPVariable_Wrap(table), THPVariable_Wrap(totals), THPVariable_Wrap(starts), THPVariable_Wrap(sequences),
                       THPVariable_Wrap(positions), THPVariable_Wrap(slots), tree ? THPVariable_Wrap(mask) : none());
  END_HANDLE_TH_ERRORS
}

// page_bounds(k_pages, block_table, lengths, bounds, count): True when done
PyObject* bounds(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Tensor *k, *table, *lengths, *to;
  int64_t count;
  if (n != 5 || !plain_world() || !plain(a[0], &k) || !plain(a[1], &table) || !plain(a[2], &lengths) || !plain(a[3], &to) ||
      !int_of(a[4], &count) || !here(*k) || k->dim() != 4 || k->numel() == 0 || k->stride(3) != 1 || lengths->dim() != 1)
    return none();
  const int type = k->scalar_type() == at::kFloat8_e4m3fn ? GQK_DTYPE_FP8 : heads_type(k->scalar_type());
  const int64_t batch = lengths->size(0);
  if (type < 0 || batch > 65535 || !table_of(*table, 2, batch, *k) || !i32_of(*lengths, batch, *k) || to->scalar_type() != k->scalar_type() ||
      !same_device(*k, to) || !to->is_contiguous() || to->dim() != 4 || to->size(0) != k->size(0) || to->size(1) != 2 ||
      to->size(2) != k->size(2) || to->size(3) != k->size(3))
    return none();
  for (int i = 0; i < 4; ++i)
    if (k->size(i) > 0x7fffffff) return none();
  auto stride = [&](int i) { return k->size(i) > 1 ? k->stride(i) : 0; };
  gqk_pages p{};
  p.k = k->data_ptr();
  p.k_page = stride(0);
  p.k_token = stride(1);
  p.k_head = stride(2);
  p.dtype = type;
  p.pages = static_cast<int32_t>(k->size(0));
  p.page_size = static_cast<int32_t>(k->size(1));
  p.heads = static_cast<int32_t>(k->size(2));
  p.dim = static_cast<int32_t>(k->size(3));
  if (gqk_page_bounds(&p, table->data_ptr<int>(), table->stride(0), static_cast<int>(table->size(1)), lengths->data_ptr<int>(),
                      static_cast<int>(batch), static_cast<int>(count), to->data_ptr(), stream_of(*k)))
    return none();
  written(*to);
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// select_pages(q, bounds, block_table, lengths, keep, page_size, sink, recent, max_length, workspace): (table, lengths)
PyObject* select(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Tensor *q, *from, *table, *lengths, *ws;
  int64_t keep, page_size, sink, recent, most = 0;
  if (n != 10 || !plain_world() || !plain(a[0], &q) || !plain(a[1], &from) || !plain(a[2], &table) || !plain(a[3], &lengths) ||
      !int_of(a[4], &keep) || !int_of(a[5], &page_size) || !int_of(a[6], &sink) || !int_of(a[7], &recent) ||
      (a[8] != Py_None && !int_of(a[8], &most)) || !plain_or_none(a[9], &ws))
    return none();
  gqk_heads qh;
  const int type = heads_type(q->scalar_type());
  if (type < 0 || !here(*q) || !heads_of(q, &qh)) return none();
  const int64_t batch = q->size(0), heads = q->size(1), dim = q->size(2);
  if (from->dim() != 4 || from->size(1) != 2 || from->size(3) != dim || from->size(0) < 1 || from->size(0) > 0x7fffffff ||
      from->size(2) < 1 || from->size(2) > heads || (from->scalar_type() != q->scalar_type() && from->scalar_type() != at::kFloat8_e4m3fn) ||
      !from->is_contiguous() || !same_device(*q, from))
    return none();
  if (batch < 1 || batch > 65535 || keep < 1 || page_size < 1 || !table_of(*table, 2, batch, *q) || !i32_of(*lengths, batch, *q)) return none();
  const int64_t room = std::min<int64_t>(table->size(1) * page_size, GQK_MAX_KEYS);
  if (a[8] == Py_None) most = room;
  if (most > room) return none();
  void* space;
  int64_t bytes;
  if (!workspace_of(ws, *q, &space, &bytes)) return none();
  Tensor chosen = at::empty({batch, from->size(2), keep}, table->options()), kept = at::empty({batch}, table->options());
  if (gqk_select_pages(qh.data, qh.row, qh.head, type, static_cast<int>(batch), static_cast<int>(heads), from->data_ptr(),
                       from->scalar_type() == at::kFloat8_e4m3fn ? GQK_DTYPE_FP8 : type, static_cast<int>(from->size(0)),
                       static_cast<int>(from->size(2)), static_cast<int>(dim), table->data_ptr<int>(), table->stride(0),
                       static_cast<int>(table->size(1)), lengths->data_ptr<int>(), static_cast<int>(most), static_cast<int>(page_size),
                       static_cast<int>(keep), static_cast<int>(sink), static_cast<int>(recent), chosen.data_ptr<int>(),
                       kept.data_ptr<int>(), space, bytes, stream_of(*q)))
    return none();
  return Py_BuildValue("(NN)", THPVariable_Wrap(chosen), THPVariable_Wrap(kept));
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
                         {"tree_attention", FAST(tree), METH_FASTCALL, nullptr},
                         {"add_rms_norm", FAST(norm), METH_FASTCALL, nullptr},
                         {"step_tables", FAST(tables), METH_FASTCALL, nullptr},
                         {"page_bounds", FAST(bounds), METH_FASTCALL, nullptr},
                         {"select_pages", FAST(select), METH_FASTCALL, nullptr},
                         {"lora_add", FAST(lora), METH_FASTCALL, nullptr},
                         {"copy_pages", FAST(copy), METH_FASTCALL, nullptr},
                         {"set_workspace", FAST(set_workspace), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fast", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fast() { return PyModule_Create(&module); }
