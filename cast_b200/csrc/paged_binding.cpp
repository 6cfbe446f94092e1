// Direct calls of the paged entry points from Python, for arguments that need no conversion.
//
// A one-token step is a few microseconds on the GPU; reading some sixty tensor attributes from Python and passing
// thirty arguments through ctypes took twice that. The functions here read the tensors themselves, check them as
// cast_b200/paged.py does, and call the C ABI on the current stream. Whatever is not exactly as the C ABI takes it
// (another type, device or layout, a list of integers) returns NotImplemented, and paged.py goes on with its own
// checks and conversions; so does an error code, which paged.py's call of the same entry point then raises.
#define PY_SSIZE_T_CLEAN
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>

#include <climits>
#include <vector>

#include "../../include/cast_b200.h"

namespace {

decltype(&cast_paged_append) g_append = nullptr;
decltype(&cast_paged_decode_attn) g_decode = nullptr;
decltype(&cast_paged_decode_workspace_size) g_decode_ws = nullptr;
decltype(&cast_tree_attn_paged_fwd) g_tree = nullptr;
decltype(&cast_tree_attn_paged_workspace_size) g_tree_ws = nullptr;

PyObject* not_here() { Py_RETURN_NOTIMPLEMENTED; }

const at::Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

int dtype_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return CAST_F32;
    case at::kBFloat16: return CAST_BF16;
    case at::kHalf: return CAST_F16;
    default: return -1;
  }
}

// Pages [num_pages, H_kv, page_size, D] on a CUDA device, dim stride 1. Sizes above the C ABI's int go to paged.py.
bool pages_ok(const at::Tensor* t) {
  return t && t->is_cuda() && t->dim() == 4 && t->stride(3) == 1 && dtype_code(*t) >= 0 && t->size(0) <= INT_MAX &&
         t->size(1) <= INT_MAX && t->size(2) <= INT_MAX;
}
bool alike(const at::Tensor* t, const at::Tensor& o) {
  return t && t->sizes() == o.sizes() && t->strides() == o.strides() && t->scalar_type() == o.scalar_type() &&
         t->device() == o.device();
}
// [n, heads, D] of the pages' type and device, dim stride 1.
bool rows_ok(const at::Tensor* t, const at::Tensor& pages, int64_t n, int64_t heads) {
  return t && t->dim() == 3 && t->size(0) == n && (heads < 0 || t->size(1) == heads) && t->size(2) == pages.size(3) &&
         t->stride(2) == 1 && t->scalar_type() == pages.scalar_type() && t->device() == pages.device();
}
// As the attention kernels take it without a copy.
bool aligned_rows(const at::Tensor& t) {
  return t.stride(0) > 0 && t.stride(1) > 0 && t.stride(0) % 4 == 0 && t.stride(1) % 4 == 0 &&
         reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
}
bool ints_ok(const at::Tensor* t, const at::Tensor& on, int64_t n, at::ScalarType type = at::kInt) {
  return t && t->scalar_type() == type && t->device() == on.device() && t->is_contiguous() && (n < 0 || t->numel() == n);
}
bool table_ok(const at::Tensor* t, const at::Tensor& on) {
  return t && t->dim() == 2 && t->scalar_type() == at::kInt && t->device() == on.device() && t->stride(1) == 1 &&
         t->size(0) <= INT_MAX && t->size(1) <= INT_MAX;
}
bool device_current(const at::Tensor& t) { return c10::cuda::current_device() == t.get_device(); }
const int32_t* ints(const at::Tensor* t) { return t ? static_cast<const int32_t*>(t->data_ptr()) : nullptr; }

// An optional tensor argument: absent (None), present, or neither (false).
bool optional(PyObject* o, const at::Tensor*& t) {
  t = nullptr;
  if (o == Py_None) return true;
  t = tensor(o);
  return t != nullptr;
}
bool number(PyObject* o, double& x) {
  if (!PyFloat_Check(o) && !PyLong_Check(o)) return false;
  x = PyFloat_AsDouble(o);
  if (x == -1.0 && PyErr_Occurred()) { PyErr_Clear(); return false; }
  return true;
}
// A scale: None (0, the C ABI's default) or a positive number.
bool scale_ok(PyObject* o, double& x) {
  x = 0.0;
  return o == Py_None || (number(o, x) && x >= 1e-30 && x <= 1e30);
}
bool integer(PyObject* o, int& x) {
  if (!PyLong_Check(o)) return false;
  int over = 0;
  const long v = PyLong_AsLongAndOverflow(o, &over);
  if (over || v < INT_MIN || v > INT_MAX) return false;
  x = static_cast<int>(v);
  return true;
}

// The caller's workspace where it is large enough and one piece, else a new one (kept in `own`).
void* workspace(const at::Tensor* given, size_t n, const at::Tensor& on, at::Tensor& own) {
  if (n == 0) return nullptr;
  if (given && given->device() == on.device() && given->nbytes() >= n && given->is_contiguous() &&
      reinterpret_cast<uintptr_t>(given->data_ptr()) % 256 == 0)
    return given->data_ptr();
  own = at::empty({static_cast<int64_t>(n)}, on.options().dtype(at::kByte));
  return own.data_ptr();
}

// Layers of an argument: a tensor, or a list or tuple of them.
bool layers(PyObject* o, std::vector<const at::Tensor*>& out) {
  out.clear();
  if (const at::Tensor* t = tensor(o)) {
    out.push_back(t);
    return true;
  }
  if (!PyList_Check(o) && !PyTuple_Check(o)) return false;
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(o);
  for (Py_ssize_t i = 0; i < n; ++i) {
    const at::Tensor* t = tensor(PySequence_Fast_GET_ITEM(o, i));
    if (!t) return false;
    out.push_back(t);
  }
  return n > 0;
}

// append(k_pages, v_pages, page_table, seq_len, k, v, cu_q, keep, accepted, inv_freq, positions, interleaved,
//        rope_scale, q, q_out)
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  if (n_args != 15 || !g_append) return not_here();
  std::vector<const at::Tensor*> kp, vp, k, v;
  if (!layers(a[0], kp) || !layers(a[1], vp) || !layers(a[4], k) || !layers(a[5], v)) return not_here();
  const size_t n = kp.size();
  if (vp.size() != n || k.size() != n || v.size() != n || !pages_ok(kp[0])) return not_here();
  const at::Tensor& p0 = *kp[0];
  const at::Tensor &k0 = *k[0], &v0 = *v[0];
  if (k0.dim() != 3) return not_here();
  const int64_t total = k0.size(0), heads = p0.size(1), D = p0.size(3);
  if (!rows_ok(&k0, p0, total, heads) || !rows_ok(&v0, p0, total, heads)) return not_here();
  std::vector<void*> pages(2 * n);
  std::vector<const void*> rows(2 * n);
  for (size_t i = 0; i < n; ++i) {
    if (!alike(kp[i], p0) || !alike(vp[i], p0) || !alike(k[i], k0) || !alike(v[i], v0)) return not_here();
    pages[2 * i] = kp[i]->data_ptr();
    pages[2 * i + 1] = vp[i]->data_ptr();
    rows[2 * i] = k[i]->data_ptr();
    rows[2 * i + 1] = v[i]->data_ptr();
  }
  const at::Tensor *table = tensor(a[2]), *len = tensor(a[3]), *cu, *keep, *acc, *freq, *pos, *q, *q_out;
  if (!table_ok(table, p0) || !optional(a[6], cu) || !optional(a[7], keep) || !optional(a[8], acc) ||
      !optional(a[9], freq) || !optional(a[10], pos) || !optional(a[13], q) || !optional(a[14], q_out))
    return not_here();
  const int64_t B = table->size(0);
  if (!ints_ok(len, p0, B) || (cu && !ints_ok(cu, p0, B + 1)) || (pos && !ints_ok(pos, p0, total))) return not_here();
  if (!keep != !acc || (keep && (!cu || keep->dim() != 2 || keep->size(0) != B || !ints_ok(keep, p0, -1) || !ints_ok(acc, p0, B))))
    return not_here();
  if (freq && (!ints_ok(freq, p0, -1, at::kFloat) || 2 * freq->numel() > D)) return not_here();
  const int64_t n_freq = freq ? freq->numel() : 0;
  if ((q_out && !q) || (q && (n > 1 || keep || n_freq == 0 || q->dim() != 3 || !rows_ok(q, p0, total, -1))))
    return not_here();
  double scale;
  if (!PyBool_Check(a[11]) || !number(a[12], scale) || !device_current(p0)) return not_here();
  at::Tensor fresh;
  const at::Tensor* out = q_out;
  if (q) {
    if (!q_out) {
      fresh = at::empty_like(*q);
      out = &fresh;
    }
    if (!rows_ok(out, p0, total, q->size(1)) || (out->stride(0) == 0 && total > 1) ||
        (out->stride(1) == 0 && out->size(1) > 1))      // rows or heads that fall on one another
      return not_here();
  }
  const int64_t ps[6] = {p0.stride(0), p0.stride(1), p0.stride(2), p0.stride(0), p0.stride(1), p0.stride(2)};
  const int64_t ns[4] = {k0.stride(0), k0.stride(1), v0.stride(0), v0.stride(1)};
  int64_t qs[4] = {0, 0, 0, 0};
  if (q) {
    qs[0] = q->stride(0); qs[1] = q->stride(1); qs[2] = out->stride(0); qs[3] = out->stride(1);
  }
  const int code = g_append(
      static_cast<int>(n), pages.data(), rows.data(), dtype_code(p0), static_cast<int>(heads), static_cast<int>(D),
      static_cast<int>(p0.size(0)), static_cast<int>(p0.size(2)), ps, total, ns, ints(table), table->stride(0),
      static_cast<int>(table->size(1)), ints(len), static_cast<int>(B), ints(cu), ints(keep),
      keep ? static_cast<int>(keep->size(1)) : 0, ints(acc), ints(pos),
      n_freq ? static_cast<const float*>(freq->data_ptr()) : nullptr, static_cast<int>(n_freq), a[11] == Py_True,
      static_cast<float>(scale), q ? q->data_ptr() : nullptr, q ? out->data_ptr() : nullptr,
      q ? static_cast<int>(q->size(1)) : 0, q ? qs : nullptr,
      c10::cuda::getCurrentCUDAStream(p0.get_device()).stream());
  if (code != CAST_OK) return not_here();
  if (!q) Py_RETURN_NONE;
  if (!q_out) return THPVariable_Wrap(fresh);
  Py_INCREF(a[14]);
  return a[14];
}

// decode(q, k_pages, v_pages, page_table, seq_len, sm_scale, softcap, window, alibi_slopes, out, lse, workspace)
PyObject* decode(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  if (n_args != 12 || !g_decode) return not_here();
  const at::Tensor *q = tensor(a[0]), *kp = tensor(a[1]), *vp = tensor(a[2]), *table = tensor(a[3]), *len = tensor(a[4]);
  const at::Tensor *slopes, *out, *lse, *ws;
  if (!q || q->dim() != 3 || !pages_ok(kp) || !alike(vp, *kp) || !rows_ok(q, *kp, q->size(0), -1) || !aligned_rows(*q) ||
      !table_ok(table, *kp) || !optional(a[8], slopes) || !optional(a[9], out) || !optional(a[10], lse) ||
      !optional(a[11], ws))
    return not_here();
  const int64_t B = q->size(0), heads = q->size(1), kv = kp->size(1), D = kp->size(3);
  if (kv < 1 || heads % kv != 0 || table->size(0) != B || !ints_ok(len, *kp, B)) return not_here();
  double scale, cap;
  int window;
  if (!scale_ok(a[5], scale) || !number(a[6], cap) || !integer(a[7], window)) return not_here();
  if (slopes && (!ints_ok(slopes, *kp, heads, at::kFloat) || slopes->dim() != 1)) return not_here();
  if (lse && (!ints_ok(lse, *kp, B * heads, at::kFloat) || lse->dim() != 2 || lse->size(1) != heads)) return not_here();
  if (out && (!rows_ok(out, *kp, B, heads) || !aligned_rows(*out))) return not_here();
  if (!device_current(*kp)) return not_here();
  const int code = dtype_code(*kp);
  const size_t n = g_decode_ws(code, static_cast<int>(B), static_cast<int>(heads), static_cast<int>(kv), static_cast<int>(D));
  if (n == 0) return not_here();
  at::Tensor fresh, own;
  if (!out) fresh = at::empty_like(*q);
  const at::Tensor& o = out ? *out : fresh;
  void* w = workspace(ws, n, *kp, own);
  const int64_t st[7] = {q->stride(0), q->stride(1), kp->stride(0), kp->stride(1), kp->stride(2), o.stride(0), o.stride(1)};
  const int rc = g_decode(q->data_ptr(), kp->data_ptr(), vp->data_ptr(), o.data_ptr(),
                          lse ? static_cast<float*>(lse->data_ptr()) : nullptr, code, st, ints(table), table->stride(0),
                          static_cast<int>(table->size(1)), ints(len), static_cast<int>(B), static_cast<int>(heads),
                          static_cast<int>(kv), static_cast<int>(D), static_cast<int>(kp->size(0)),
                          static_cast<int>(kp->size(2)), static_cast<float>(scale), static_cast<float>(cap), window,
                          slopes ? static_cast<const float*>(slopes->data_ptr()) : nullptr, w, n,
                          c10::cuda::getCurrentCUDAStream(kp->get_device()).stream());
  if (rc != CAST_OK) return not_here();
  if (!out) return THPVariable_Wrap(fresh);
  Py_INCREF(a[9]);
  return a[9];
}

// tree(q, k_pages, v_pages, page_table, k_pack, v_pack, cu_q, prefix_len, pack_len, ancestor_mask, sm_scale, parent,
//      max_pack, max_prefix, out, workspace)
PyObject* tree(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  if (n_args != 16 || !g_tree) return not_here();
  const at::Tensor *q = tensor(a[0]), *kp = tensor(a[1]), *vp = tensor(a[2]), *table = tensor(a[3]), *k = tensor(a[4]),
                   *v = tensor(a[5]), *cu = tensor(a[6]), *pre = tensor(a[7]), *pack = tensor(a[8]);
  const at::Tensor *anc, *par, *out, *ws;
  if (!q || q->dim() != 3 || !pages_ok(kp) || !alike(vp, *kp) || !table_ok(table, *kp) || !optional(a[9], anc) ||
      !optional(a[11], par) || !optional(a[14], out) || !optional(a[15], ws))
    return not_here();
  const int64_t total = q->size(0), heads = q->size(1), kv = kp->size(1), D = kp->size(3), B = table->size(0);
  if (kv < 1 || heads % kv != 0 || !rows_ok(q, *kp, total, -1) || !rows_ok(k, *kp, total, kv) || !rows_ok(v, *kp, total, kv) ||
      !aligned_rows(*q) || !aligned_rows(*k) || !aligned_rows(*v) || !ints_ok(cu, *kp, B + 1) || !ints_ok(pre, *kp, B) ||
      !ints_ok(pack, *kp, B))
    return not_here();
  if (total < 1 || total > INT_MAX || !anc == !par || (par && !ints_ok(par, *kp, total)) ||
      (anc && (!ints_ok(anc, *kp, -1, at::kLong) || anc->numel() % total != 0)))
    return not_here();
  if (out && (!rows_ok(out, *kp, total, heads) || !aligned_rows(*out))) return not_here();
  double scale;
  int max_pack, max_prefix;
  if (!scale_ok(a[10], scale) || !integer(a[12], max_pack) || !integer(a[13], max_prefix) ||
      max_pack < 0 || max_prefix < 0 || !device_current(*kp))
    return not_here();
  const int code = dtype_code(*kp);
  const size_t n = g_tree_ws(code, static_cast<int>(B), static_cast<int>(total), static_cast<int>(heads),
                             static_cast<int>(kv), static_cast<int>(D), max_pack, max_prefix);
  at::Tensor fresh, own;
  if (!out) fresh = at::empty_like(*q);
  const at::Tensor& o = out ? *out : fresh;
  void* w = workspace(ws, n, *kp, own);
  const int64_t st[11] = {q->stride(0), q->stride(1), kp->stride(0), kp->stride(1), kp->stride(2), k->stride(0),
                          k->stride(1), v->stride(0), v->stride(1), o.stride(0), o.stride(1)};
  const int rc = g_tree(q->data_ptr(), kp->data_ptr(), vp->data_ptr(), k->data_ptr(), v->data_ptr(), o.data_ptr(), code, st,
                        ints(table), table->stride(0), static_cast<int>(table->size(1)), ints(cu), ints(pre), ints(pack),
                        anc ? static_cast<const int64_t*>(anc->data_ptr()) : nullptr,
                        anc ? static_cast<int>(anc->numel() / total) : 0, ints(par), static_cast<int>(B),
                        static_cast<int>(total), static_cast<int>(kp->size(0)), static_cast<int>(kp->size(2)),
                        static_cast<int>(heads), static_cast<int>(kv), static_cast<int>(D), static_cast<float>(scale),
                        max_pack, max_prefix, w, n, c10::cuda::getCurrentCUDAStream(kp->get_device()).stream());
  if (rc != CAST_OK) return not_here();
  if (!out) return THPVariable_Wrap(fresh);
  Py_INCREF(a[14]);
  return a[14];
}

// bind(addresses of cast_paged_append, cast_paged_decode_attn, cast_paged_decode_workspace_size,
//      cast_tree_attn_paged_fwd, cast_tree_attn_paged_workspace_size)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  void* p[5];
  if (n != 5) {
    PyErr_SetString(PyExc_TypeError, "bind takes five addresses");
    return nullptr;
  }
  for (int i = 0; i < 5; ++i) {
    p[i] = PyLong_AsVoidPtr(a[i]);
    if (PyErr_Occurred()) return nullptr;
  }
  g_append = reinterpret_cast<decltype(g_append)>(p[0]);
  g_decode = reinterpret_cast<decltype(g_decode)>(p[1]);
  g_decode_ws = reinterpret_cast<decltype(g_decode_ws)>(p[2]);
  g_tree = reinterpret_cast<decltype(g_tree)>(p[3]);
  g_tree_ws = reinterpret_cast<decltype(g_tree_ws)>(p[4]);
  Py_RETURN_NONE;
}

// A C++ exception (an allocation that fails, say) becomes a Python one.
template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  return F(self, a, n);
  END_HANDLE_TH_ERRORS
}

#define CAST_METHOD(name) \
  {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&guarded<&name>)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {CAST_METHOD(append), CAST_METHOD(decode), CAST_METHOD(tree), CAST_METHOD(bind),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_paged_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__paged_binding() { return PyModule_Create(&module); }
