// The ordinary call of the dense block's operators straight from torch tensors: is everything as it should be, the argument
// block, the op's own buffers, the C entry.  Anything else (another stream, another allocator, an argument that is not as it
// should be) is left to ops.py, which says what is wrong or takes the long way: each function here returns None for that,
// the result, or the entry's status as an int.
//
// Why: a single token's append takes the GPU 3 us, and its arguments cost 11 us in Python (a tensor's attribute is 60 to 200 ns,
// and the op looks at sixty); here they cost 1.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>

#include "wsvd_b200.h"

namespace {

using at::Tensor;

struct Entries {
  int (*append)(const WsvdKvRopeAppendParams*, void*);
  size_t (*paged_bytes)(const WsvdPagedDecodeParams*);
  int (*paged)(const WsvdPagedDecodeParams*, void*, size_t, void*);
  size_t (*adapter_bytes)(const WsvdAdapterAddParams*);
  int (*adapter)(const WsvdAdapterAddParams*, void*, size_t, void*);
} entries;

// A tensor argument, or null for None; `bad` where it is neither (or a subclass, which may not have memory).
const Tensor* tensor(PyObject* o, bool* bad) {
  if (o == Py_None) return nullptr;
  if (!THPVariable_CheckExact(o)) {
    *bad = true;
    return nullptr;
  }
  return &THPVariable_Unpack(o);
}

// strided memory of `dims` dims, the last one contiguous
bool rows(const Tensor* t, int64_t dims, at::ScalarType type, const at::Device& device) {
  return t && t->layout() == at::kStrided && t->dim() == dims && t->scalar_type() == type && t->device() == device && t->stride(dims - 1) == 1;
}
bool vector(const Tensor* t, int64_t n, at::ScalarType type, const at::Device& device) {
  return rows(t, 1, type, device) && t->size(0) == n;
}
bool scales(const Tensor* t, const Tensor& cache) {
  return t && t->layout() == at::kStrided && t->dim() == 2 && t->scalar_type() == at::kHalf && t->device() == cache.device() &&
         t->size(0) == cache.size(0) && t->size(1) == cache.size(1);
}
// sizes that the C entries take as 32-bit numbers
bool countable(std::initializer_list<int64_t> sizes) { return std::max(sizes) <= INT32_MAX; }
// a gradient is wanted of one of them, or one carries a tangent (which torch.no_grad() does not switch off)
bool differentiated(std::initializer_list<const Tensor*> ts) {
  const bool backward = c10::GradMode::is_enabled();
  for (const Tensor* t : ts)
    if (t && ((backward && t->requires_grad()) || t->_fw_grad(0).defined())) return true;
  return false;
}
// an output's elements have a place in memory each
bool apart(const Tensor* t) {
  if (!t || t->numel() == 0) return true;
  int64_t order[3], dims = t->dim(), reach = 1;
  for (int64_t i = 0; i < dims; ++i) {
    int64_t j = i;
    for (; j > 0 && t->stride(order[j - 1]) > t->stride(i); --j) order[j] = order[j - 1];
    order[j] = i;
  }
  for (int64_t i = 0; i < dims; ++i) {
    const int64_t size = t->size(order[i]), stride = t->stride(order[i]);
    if (size > 1 && stride < reach) return false;
    reach += stride * (size - 1);
  }
  return true;
}
// Whether two tensors have a byte of memory in common, as ops.py's _meet: apart = sum of i stride over a's dims - the same over b's.
struct Terms {
  int n = 0, budget = 256;
  int64_t size, stride[6], first[6], last[6];
  void add(const Tensor& t, bool minus) {
    for (int64_t d = 0; d < t.dim(); ++d) {
      const int64_t s = t.stride(d) * t.element_size(), most = t.size(d) - 1;
      if (most < 1 || s == 0) continue;
      int i = 0;
      while (i < n && stride[i] > s) ++i;
      if (i == n || stride[i] != s) {
        for (int j = n++; j > i; --j) stride[j] = stride[j - 1], first[j] = first[j - 1], last[j] = last[j - 1];
        stride[i] = s, first[i] = last[i] = 0;
      }
      (minus ? first[i] : last[i]) += minus ? -most : most;
    }
  }
  static int64_t below(int64_t a, int64_t b) { return a / b - (a % b != 0 && a < 0); }  // b > 0
  bool reach(int at, int64_t left) {
    int64_t low = 0, high = 0;
    for (int i = at; i < n; ++i) low += stride[i] * first[i], high += stride[i] * last[i];
    if (left <= low - size || left >= high + size) return false;
    if (at == n) return true;
    const int64_t s = stride[at];
    low -= s * first[at], high -= s * last[at];
    const int64_t from = std::max(first[at], -below(high + size - 1 - left, s)), to = std::min(last[at], below(left - low + size - 1, s));
    for (int64_t i = from; i <= to; ++i)
      if (--budget < 0 || reach(at + 1, left - i * s)) return true;
    return false;
  }
};
bool meet(const Tensor& a, const Tensor& b) {
  if (a.numel() == 0 || b.numel() == 0) return false;
  Terms t;
  t.size = std::max(a.element_size(), b.element_size());
  t.add(a, false);
  t.add(b, true);
  return t.reach(0, static_cast<const char*>(b.data_ptr()) - static_cast<const char*>(a.data_ptr()));
}
// an output may be the input `in_place` itself (one shape), and has no memory of any input otherwise
bool no_overlap(const Tensor* out, const Tensor& in_place, std::initializer_list<const Tensor*> others) {
  if (!out) return true;
  bool same = out->data_ptr() == in_place.data_ptr();
  for (int64_t d = 0; same && d < out->dim(); ++d) same = out->size(d) < 2 || out->stride(d) == in_place.stride(d);
  if (!same && meet(*out, in_place)) return false;
  for (const Tensor* t : others)
    if (meet(*out, *t)) return false;
  return true;
}
int code(at::ScalarType t) { return t == at::kChar ? WSVD_I8 : t == at::kHalf ? WSVD_F16 : WSVD_BF16; }
bool half(at::ScalarType t) { return t == at::kHalf || t == at::kBFloat16; }
void* at_of(const Tensor* t) { return t ? t->data_ptr() : nullptr; }
bool same_shape(const Tensor& a, const Tensor& b) { return a.sizes() == b.sizes(); }

PyObject* none() { Py_RETURN_NONE; }

bool cache_fits(const Tensor* k, const Tensor* v, const Tensor* ks, const Tensor* vs, at::ScalarType type, int64_t heads, int64_t dim,
                const at::Device& device) {
  if (!k || !v) return false;
  const at::ScalarType held = k->scalar_type();
  if (held != type && held != at::kChar) return false;
  if (!rows(k, 3, held, device) || !rows(v, 3, held, device) || k->size(1) != heads || k->size(2) != dim || !same_shape(*k, *v)) return false;
  return held == at::kChar ? scales(ks, *k) && scales(vs, *k) : !ks && !vs;
}
bool metadata_fits(const Tensor* lens, const Tensor* idx, const Tensor* table, int64_t batch, const at::Device& device) {
  return vector(lens, batch, at::kInt, device) && vector(idx, batch, at::kInt, device) && rows(table, 2, at::kInt, device) &&
         countable({batch, table->size(0), table->size(1)});
}

// ---- kv_rope_append(k, v, lens, idx, table, cache_k, cache_v, inv_freq, k_scale, v_scale, q, q_out, cu_new, pos_offset, layout)

struct Append {
  const Tensor *k, *v, *lens, *idx, *table, *ck, *cv, *inv, *ks, *vs, *q, *q_out, *cu, *off;
  int layout;
  int64_t batch;

  bool fits(PyObject* const* a, Py_ssize_t n) {
    if (n != 15) return false;
    bool bad = false;
    const Tensor** to[] = {&k, &v, &lens, &idx, &table, &ck, &cv, &inv, &ks, &vs, &q, &q_out, &cu, &off};
    for (int i = 0; i < 14; ++i) *to[i] = tensor(a[i], &bad);
    if (bad || !k || k->dim() != 3 || !half(k->scalar_type())) return false;
    layout = (int)PyLong_AsLong(a[14]);
    const at::ScalarType type = k->scalar_type();
    const at::Device device = k->device();
    const int64_t N = k->size(0), H = k->size(1), D = k->size(2);
    batch = cu ? cu->dim() == 1 ? cu->size(0) - 1 : -1 : N;
    return batch >= 0 && countable({N, H, q && q->dim() == 3 ? q->size(1) : 0}) && rows(k, 3, type, device) && rows(v, 3, type, device) &&
           same_shape(*k, *v) && H > 0 && D >= 2 && D % 2 == 0 && D <= 256 &&
           inv && inv->dim() == 1 && vector(inv, inv->size(0), at::kFloat, device) && 2 * inv->size(0) <= D &&
           cache_fits(ck, cv, ks, vs, type, H, D, device) && metadata_fits(lens, idx, table, batch, device) &&
           (!cu || vector(cu, batch + 1, at::kInt, device)) && (!off || vector(off, batch, at::kInt, device)) &&
           (q ? rows(q, 3, type, device) && q->size(0) == N && q->size(2) == D : !q_out) &&
           (!q_out || (rows(q_out, 3, type, device) && same_shape(*q, *q_out) && no_overlap(q_out, *q, {k, v}))) &&
           apart(q_out) && apart(ck) && apart(cv) && apart(ks) && apart(vs) && !meet(*ck, *cv) &&
           !(q_out && (meet(*q_out, *ck) || meet(*q_out, *cv))) && !differentiated({k, v, q, q_out, ck, cv, ks, vs, inv});
  }
};

PyObject* append_fits(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Append x;
  return PyBool_FromLong(x.fits(a, n));
  END_HANDLE_TH_ERRORS
}

PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Append x;
  if (!x.fits(a, n) || !x.k->is_cuda()) return none();
  const c10::cuda::CUDAGuard guard(x.k->device());
  Tensor made;
  const bool own = x.q && !x.q_out;
  if (own) {
    made = at::empty(x.q->sizes(), x.q->options().requires_grad(false));
    x.q_out = &made;
  }
  WsvdKvRopeAppendParams p = {};
  p.k = at_of(x.k), p.k_stride_n = x.k->stride(0), p.k_stride_h = x.k->stride(1);
  p.v = at_of(x.v), p.v_stride_n = x.v->stride(0), p.v_stride_h = x.v->stride(1);
  if (x.q) {
    p.q = at_of(x.q), p.q_stride_n = x.q->stride(0), p.q_stride_h = x.q->stride(1);
    p.q_out = at_of(x.q_out), p.qo_stride_n = x.q_out->stride(0), p.qo_stride_h = x.q_out->stride(1);
    p.n_q_heads = (int32_t)x.q->size(1);
  }
  p.cache_k = at_of(x.ck), p.ck_stride_t = x.ck->stride(0), p.ck_stride_h = x.ck->stride(1);
  p.cache_v = at_of(x.cv), p.cv_stride_t = x.cv->stride(0), p.cv_stride_h = x.cv->stride(1);
  if (x.ks) {
    p.k_scale = at_of(x.ks), p.ks_stride_t = x.ks->stride(0), p.ks_stride_h = x.ks->stride(1);
    p.v_scale = at_of(x.vs), p.vs_stride_t = x.vs->stride(0), p.vs_stride_h = x.vs->stride(1);
  }
  p.inv_freq = static_cast<const float*>(at_of(x.inv));
  p.req_to_token = static_cast<const int32_t*>(at_of(x.table)), p.rtt_stride = x.table->stride(0);
  p.b_req_idx = static_cast<const int32_t*>(at_of(x.idx)), p.b_seq_len = static_cast<const int32_t*>(at_of(x.lens));
  p.cu_new = static_cast<const int32_t*>(at_of(x.cu)), p.pos_offset = static_cast<const int32_t*>(at_of(x.off));
  p.n_token_slots = x.ck->size(0);
  p.rows = (int32_t)x.k->size(0), p.batch = (int32_t)x.batch, p.n_kv_heads = (int32_t)x.k->size(1), p.head_dim = (int32_t)x.k->size(2);
  p.rot_dim = (int32_t)(2 * x.inv->size(0)), p.max_len = (int32_t)x.table->size(1), p.n_req = (int32_t)x.table->size(0);
  p.dtype = code(x.k->scalar_type()), p.cache_dtype = code(x.ck->scalar_type()), p.rope_layout = x.layout, p.clear_tail = own;
  const int status = entries.append(&p, c10::cuda::getCurrentCUDAStream(x.k->get_device()).stream());
  if (status != 0) return PyLong_FromLong(status);
  if (own) return THPVariable_Wrap(made);
  if (!x.q) Py_RETURN_TRUE;
  PyObject* given = a[11];
  Py_INCREF(given);
  return given;
  END_HANDLE_TH_ERRORS
}

// ---- paged_decode(q, lens, idx, table, cache_k, cache_v, k_scale, v_scale, out, workspace, return_lse, window, sm_scale)

struct Paged {
  const Tensor *q, *lens, *idx, *table, *ck, *cv, *ks, *vs, *out, *workspace;
  bool want_lse;
  int64_t window;
  double sm_scale;

  bool fits(PyObject* const* a, Py_ssize_t n) {
    if (n != 13) return false;
    bool bad = false;
    const Tensor** to[] = {&q, &lens, &idx, &table, &ck, &cv, &ks, &vs, &out, &workspace};
    for (int i = 0; i < 10; ++i) *to[i] = tensor(a[i], &bad);
    if (bad || !q || q->dim() != 3 || !half(q->scalar_type()) || !ck || ck->dim() != 3) return false;
    want_lse = PyObject_IsTrue(a[10]) == 1;
    window = PyLong_AsLongLong(a[11]);
    sm_scale = PyFloat_AsDouble(a[12]);
    if (PyErr_Occurred()) {
      PyErr_Clear();
      return false;
    }
    const at::ScalarType type = q->scalar_type();
    const at::Device device = q->device();
    const int64_t H = q->size(1), D = q->size(2), K = ck->size(1);
    return countable({H, K}) && rows(q, 3, type, device) && D >= 1 && D <= 256 && K > 0 && H > 0 && H % K == 0 && window >= 0 &&
           cache_fits(ck, cv, ks, vs, type, K, D, device) && metadata_fits(lens, idx, table, q->size(0), device) &&
           (!out || (rows(out, 3, type, device) && same_shape(*out, *q) && no_overlap(out, *q, {ck, cv}))) &&
           (!workspace || (workspace->device() == device && workspace->is_contiguous())) && apart(out) && !differentiated({q, ck, cv, ks, vs, out});
  }
};

PyObject* paged_fits(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Paged x;
  return PyBool_FromLong(x.fits(a, n));
  END_HANDLE_TH_ERRORS
}

PyObject* paged(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Paged x;
  if (!x.fits(a, n) || !x.q->is_cuda()) return none();
  const c10::cuda::CUDAGuard guard(x.q->device());
  const int64_t B = x.q->size(0), H = x.q->size(1);
  const auto options = x.q->options().requires_grad(false);
  const Tensor out = x.out ? *x.out : at::empty(x.q->sizes(), options);
  Tensor lse, scratch;
  if (x.want_lse) lse = at::empty({B, H}, options.dtype(at::kFloat));
  WsvdPagedDecodeParams p = {};
  p.q = at_of(x.q), p.q_stride_b = x.q->stride(0), p.q_stride_h = x.q->stride(1);
  p.k = at_of(x.ck), p.k_stride_t = x.ck->stride(0), p.k_stride_h = x.ck->stride(1);
  p.v = at_of(x.cv), p.v_stride_t = x.cv->stride(0), p.v_stride_h = x.cv->stride(1);
  if (x.ks) {
    p.k_scale = at_of(x.ks), p.ks_stride_t = x.ks->stride(0), p.ks_stride_h = x.ks->stride(1);
    p.v_scale = at_of(x.vs), p.vs_stride_t = x.vs->stride(0), p.vs_stride_h = x.vs->stride(1);
  }
  p.req_to_token = static_cast<const int32_t*>(at_of(x.table)), p.rtt_stride = x.table->stride(0);
  p.b_req_idx = static_cast<const int32_t*>(at_of(x.idx)), p.b_seq_len = static_cast<const int32_t*>(at_of(x.lens));
  p.out = at_of(&out), p.out_stride_b = out.stride(0), p.out_stride_h = out.stride(1);
  p.lse = x.want_lse ? static_cast<float*>(at_of(&lse)) : nullptr;
  p.n_token_slots = x.ck->size(0);
  p.batch = (int32_t)B, p.n_q_heads = (int32_t)H, p.n_kv_heads = (int32_t)x.ck->size(1), p.head_dim = (int32_t)x.q->size(2);
  p.max_len = (int32_t)x.table->size(1), p.n_req = (int32_t)x.table->size(0);
  p.dtype = code(x.q->scalar_type()), p.cache_dtype = code(x.ck->scalar_type());
  p.window = (int32_t)std::min<int64_t>(x.window, INT32_MAX), p.sm_scale = (float)x.sm_scale;
  if (!x.workspace) {
    scratch = at::empty({(int64_t)entries.paged_bytes(&p)}, options.dtype(at::kByte));
    x.workspace = &scratch;
  }
  const int status = entries.paged(&p, at_of(x.workspace), x.workspace->nbytes(), c10::cuda::getCurrentCUDAStream(x.q->get_device()).stream());
  if (status != 0) return PyLong_FromLong(status);
  PyObject* result = x.out ? a[8] : THPVariable_Wrap(out);
  if (x.out) Py_INCREF(result);
  if (!x.want_lse) return result;
  PyObject* second = THPVariable_Wrap(lse);
  PyObject* pair = PyTuple_Pack(2, result, second);
  Py_DECREF(result);
  Py_DECREF(second);
  return pair;
  END_HANDLE_TH_ERRORS
}

// ---- adapter_add(y, x, a, b, adapter, scale, cu_new, out, workspace)

struct Adapters {
  const Tensor *y, *x, *a, *b, *adapter, *scale, *cu, *out, *workspace;

  bool fits(PyObject* const* o, Py_ssize_t n) {
    if (n != 9) return false;
    bool bad = false;
    const Tensor** to[] = {&y, &x, &a, &b, &adapter, &scale, &cu, &out, &workspace};
    for (int i = 0; i < 9; ++i) *to[i] = tensor(o[i], &bad);
    if (bad || !x || x->dim() != 2 || !half(x->scalar_type()) || !y || y->dim() != 2 || !a || a->dim() != 3 || !adapter || adapter->dim() != 1)
      return false;
    const at::ScalarType type = x->scalar_type();
    const at::Device device = x->device();
    const int64_t N = x->size(0), in = x->size(1), columns = y->size(1), count = a->size(0), rank = a->size(2), B = adapter->size(0);
    return countable({N, in, columns, count, B}) && rows(x, 2, type, device) && rows(y, 2, type, device) && rows(a, 3, type, device) &&
           rows(b, 3, type, device) && y->size(0) == N &&
           a->size(1) == in && b->size(0) == count && b->size(1) == rank && b->size(2) == columns && rank >= 1 && rank <= 256 && in > 0 &&
           columns > 0 && vector(adapter, B, at::kInt, device) && (!scale || vector(scale, count, at::kFloat, device)) &&
           (cu ? vector(cu, B + 1, at::kInt, device) : B == N) &&
           (!out || (rows(out, 2, type, device) && same_shape(*out, *y) && no_overlap(out, *y, {x, a, b}))) &&
           (!workspace || (workspace->device() == device && workspace->is_contiguous())) && apart(out) && !differentiated({x, y, a, b, scale, out});
  }
};

PyObject* adapter_fits(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Adapters t;
  return PyBool_FromLong(t.fits(o, n));
  END_HANDLE_TH_ERRORS
}

PyObject* adapter(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Adapters t;
  if (!t.fits(o, n) || !t.x->is_cuda()) return none();
  const c10::cuda::CUDAGuard guard(t.x->device());
  const auto options = t.x->options().requires_grad(false);
  const Tensor out = t.out ? *t.out : at::empty(t.y->sizes(), options);
  Tensor scratch;
  WsvdAdapterAddParams p = {};
  p.y = at_of(t.y), p.y_stride = t.y->stride(0);
  p.x = at_of(t.x), p.x_stride = t.x->stride(0);
  p.a = at_of(t.a), p.a_stride_i = t.a->stride(0), p.a_stride_k = t.a->stride(1);
  p.b = at_of(t.b), p.b_stride_i = t.b->stride(0), p.b_stride_r = t.b->stride(1);
  p.out = at_of(&out), p.out_stride = out.stride(0);
  p.adapter = static_cast<const int32_t*>(at_of(t.adapter)), p.scale = static_cast<const float*>(at_of(t.scale));
  p.cu_new = static_cast<const int32_t*>(at_of(t.cu));
  p.rows = (int32_t)t.x->size(0), p.batch = (int32_t)t.adapter->size(0), p.n_in = (int32_t)t.x->size(1), p.n_out = (int32_t)t.y->size(1);
  p.rank = (int32_t)t.a->size(2), p.n_adapters = (int32_t)t.a->size(0), p.dtype = code(t.x->scalar_type()), p.copy_tail = !t.out;
  if (!t.workspace) {
    scratch = at::empty({(int64_t)entries.adapter_bytes(&p)}, options.dtype(at::kByte));
    t.workspace = &scratch;
  }
  const int status = entries.adapter(&p, at_of(t.workspace), t.workspace->nbytes(), c10::cuda::getCurrentCUDAStream(t.x->get_device()).stream());
  if (status != 0) return PyLong_FromLong(status);
  if (!t.out) return THPVariable_Wrap(out);
  Py_INCREF(o[7]);
  return o[7];
  END_HANDLE_TH_ERRORS
}

// ---- the addresses of the C entries

PyObject* connect(PyObject*, PyObject* args) {
  unsigned long long f[5];
  if (!PyArg_ParseTuple(args, "KKKKK", f, f + 1, f + 2, f + 3, f + 4)) return nullptr;
  entries.append = reinterpret_cast<decltype(entries.append)>(f[0]);
  entries.paged_bytes = reinterpret_cast<decltype(entries.paged_bytes)>(f[1]);
  entries.paged = reinterpret_cast<decltype(entries.paged)>(f[2]);
  entries.adapter_bytes = reinterpret_cast<decltype(entries.adapter_bytes)>(f[3]);
  entries.adapter = reinterpret_cast<decltype(entries.adapter)>(f[4]);
  Py_RETURN_NONE;
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr
PyMethodDef methods[] = {{"connect", connect, METH_VARARGS, nullptr},
                         {"append", FAST(append)},
                         {"append_fits", FAST(append_fits)},
                         {"paged", FAST(paged)},
                         {"paged_fits", FAST(paged_fits)},
                         {"adapter", FAST(adapter)},
                         {"adapter_fits", FAST(adapter_fits)},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_bind", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__bind() { return PyModule_Create(&module); }
