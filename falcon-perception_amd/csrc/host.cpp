// The calls an eager layer or step makes (append, decode step, prefill attention; tables, page copies and attention of shared
// prefixes; trees of drafts, their attention and verification, their rows) from PyTorch tensors to the C ABI of include/fp_paged_kv.h, as a Python module.
//
// Bound by the host: a layer of a small eager step is shorter on the GPU than its calls are in Python, where every pointer, size
// and stride is an attribute look-up and the foreign call converts forty arguments one by one.  Here they are read from the tensors in C++:
// four short fp32 sequences, 28 layers, without graphs 818 -> 380 us a step (29 -> 13.5 us a layer, of which the GPU works 7), one prompt
// of 613 rows 911 -> 700 us (33 -> 25 us a layer, now the GPU's).
//
// The functions take the tensors as ops.py would hand them to the library.  What they do not recognise at once (a tensor
// subclass, another device or type, rows that are not dense, shapes that do not match) they leave alone and return None: ops.py
// then converts the arguments or says what is wrong with them.  Nothing is kept from one call to the next.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/version.h>

#include <exception>
#include <initializer_list>

#include "fp_paged_kv.h"

namespace {

// The tensor behind a Python object, or null: not a plain tensor on the GPU.
const at::Tensor* gpu_tensor(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.is_cuda() && t.layout() == at::kStrided ? &t : nullptr;
}

int dtype_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return FP_DTYPE_F32;
    case at::kBFloat16: return FP_DTYPE_BF16;
    case at::kHalf: return FP_DTYPE_F16;
    default: return -1;
  }
}

int index_code(const at::Tensor& t) {
  return t.scalar_type() == at::kInt ? FP_INDEX_I32 : t.scalar_type() == at::kLong ? FP_INDEX_I64 : -1;
}

bool is_table(const at::Tensor& t) { return t.dim() == 2 && t.scalar_type() == at::kLong && t.stride(1) == 1; }
bool is_indices(const at::Tensor& t, int64_t n) { return t.scalar_type() == at::kLong && t.is_contiguous() && t.numel() == n; }
bool is_bytes(const at::Tensor& t) { return t.scalar_type() == at::kByte && t.is_contiguous(); }
bool dense_rows(const at::Tensor& t) { return t.stride(t.dim() - 1) == 1; }

// All of them (null: not given) lie on the device of this index, which the caller says is current.
bool on_device(int64_t device, std::initializer_list<const at::Tensor*> tensors) {
  for (const at::Tensor* t : tensors)
    if (t && t->get_device() != device) return false;
  return true;
}

// Each is a number that the C ABI takes as int32_t.
bool fits(std::initializer_list<int64_t> sizes) {
  for (const int64_t n : sizes)
    if (n != static_cast<int32_t>(n)) return false;
  return true;
}

// Other Python threads run while this one allocates and launches, which may wait (for a full queue, or for memory).
struct Unlocked {
  PyThreadState* const thread = PyEval_SaveThread();
  Unlocked() = default;
  Unlocked(const Unlocked&) = delete;
  ~Unlocked() { PyEval_RestoreThread(thread); }
};

PyObject* fail(const char* what, int rc) {
  PyErr_Format(PyExc_RuntimeError, "%s failed (%d): %s", what, rc, fp_last_error());
  return nullptr;
}

// One call's arguments, taken in order.  `ok` turns false at the first that is not what was asked for.
struct Args {
  PyObject* const* at;
  bool ok = true;
  const at::Tensor* tensor() {
    const at::Tensor* t = gpu_tensor(*at++);
    if (!t) ok = false;
    return t;
  }
  const at::Tensor* maybe_tensor() {  // null for None
    if (*at == Py_None) {
      ++at;
      return nullptr;
    }
    return tensor();
  }
  int64_t integer() {
    const long long v = PyLong_AsLongLong(*at++);
    if (v == -1 && PyErr_Occurred()) {
      PyErr_Clear();
      ok = false;
    }
    return v;
  }
  double number() {
    const double v = PyFloat_AsDouble(*at++);
    if (v == -1.0 && PyErr_Occurred()) {
      PyErr_Clear();
      ok = false;
    }
    return v;
  }
};

PyObject* pair(const at::Tensor& a, const at::Tensor& b) {
  PyObject* t = PyTuple_New(2);
  if (!t) return nullptr;
  PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(a));
  PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(b));
  return t;
}

// pool_k, pool_v, k, v, page_table, batch_idx, input_pos, page_size, clamp_negative, packed, stream -> True
PyObject* append_unguarded(PyObject* const* args) {
  Args a{args};
  const at::Tensor *pk = a.tensor(), *pv = a.tensor(), *k = a.tensor(), *v = a.tensor(), *table = a.tensor(), *bidx = a.tensor(),
                   *pos = a.tensor();
  const int64_t page_size = a.integer(), clamp = a.integer(), packed = a.integer(), stream = a.integer();
  if (!a.ok) Py_RETURN_NONE;
  const int dt = dtype_code(*k), it = index_code(*pos);
  if (dt < 0 || it < 0 || k->dim() != 4 || k->sizes() != v->sizes() || v->scalar_type() != k->scalar_type() ||
      pk->scalar_type() != k->scalar_type() || pv->scalar_type() != k->scalar_type() || pk->dim() != 3 || !pk->is_contiguous() ||
      !pv->is_contiguous() || !dense_rows(*k) || !dense_rows(*v) || !is_table(*table) || !pos->is_contiguous())
    Py_RETURN_NONE;
  int64_t T, H, S, ks[3], vs[3];
  const int64_t D = k->size(3);
  if (packed) {
    T = k->size(2), H = k->size(1), S = 1;
    if (k->size(0) != 1 || pos->numel() != T) Py_RETURN_NONE;
    ks[0] = k->stride(2), ks[1] = k->stride(1), ks[2] = 0;
    vs[0] = v->stride(2), vs[1] = v->stride(1), vs[2] = 0;
  } else {
    T = k->size(0), H = k->size(1), S = k->size(2);
    if (pos->numel() != T * S) Py_RETURN_NONE;
    for (int i = 0; i < 3; ++i) ks[i] = k->stride(i), vs[i] = v->stride(i);
  }
  if (!is_indices(*bidx, T)) Py_RETURN_NONE;
  int rc;
  {
    const Unlocked others;
    rc = fp_kv_append(pk->data_ptr(), pv->data_ptr(), k->data_ptr(), v->data_ptr(), ks[0], ks[1], ks[2], vs[0], vs[1], vs[2],
                      static_cast<const int64_t*>(table->data_ptr()), table->stride(0),
                      static_cast<const int64_t*>(bidx->data_ptr()), pos->data_ptr(), it, T, H, S, D, page_size,
                      table->size(1), table->size(0), pk->size(1), dt, clamp ? 1 : 0, reinterpret_cast<void*>(stream));
  }
  if (rc < 0) return fail("fp_kv_append", rc);
  Py_RETURN_TRUE;
}

// q, pool_k, pool_v, page_table, batch_idx, input_pos, page_size, max_context, scale, split_tokens, workspace, sinks, kv_rep,
// k_new, v_new, plan, arrivals, next_arrivals, stream -> (out, lse)
PyObject* decode_unguarded(PyObject* const* args) {
  Args a{args};
  const at::Tensor *q = a.tensor(), *pk = a.tensor(), *pv = a.tensor(), *table = a.tensor(), *bidx = a.tensor(), *pos = a.tensor();
  const int64_t page_size = a.integer(), max_context = a.integer();
  const double scale = a.number();
  const int64_t split_tokens = a.integer();
  const at::Tensor *ws = a.maybe_tensor(), *sinks = a.maybe_tensor();
  const int64_t kv_rep = a.integer();
  const at::Tensor *kn = a.maybe_tensor(), *vn = a.maybe_tensor(), *plan = a.maybe_tensor(), *arrivals = a.tensor(),
                   *after = a.maybe_tensor();
  const int64_t stream = a.integer();
  if (!a.ok) Py_RETURN_NONE;
  const int dt = dtype_code(*q), it = index_code(*pos);
  if (dt < 0 || it < 0 || q->dim() != 4 || q->size(2) != 1 || pk->dim() != 3 || pk->sizes() != pv->sizes() ||
      pk->size(2) != q->size(3) || pk->scalar_type() != q->scalar_type() || pv->scalar_type() != q->scalar_type() ||
      !pk->is_contiguous() || !pv->is_contiguous() || !dense_rows(*q) || !is_table(*table) || split_tokens <= 0 || kv_rep < 1)
    Py_RETURN_NONE;
  const int64_t B = q->size(0), Hq = q->size(1), D = q->size(3), Hc = pk->size(0);
  if (!is_indices(*bidx, B) || pos->numel() != B || !pos->is_contiguous() || (ws && !is_bytes(*ws)) || (plan && !is_bytes(*plan)) ||
      arrivals->scalar_type() != at::kInt || !arrivals->is_contiguous() ||
      (after && (after->scalar_type() != at::kInt || !after->is_contiguous() || after->numel() != arrivals->numel())) ||
      (sinks && (sinks->scalar_type() != at::kFloat || sinks->dim() != 1 || sinks->size(0) != Hq || !sinks->is_contiguous() ||
                 sinks->device() != q->device())))
    Py_RETURN_NONE;
  if (!kn != !vn) Py_RETURN_NONE;
  if (kn) {
    const int64_t fresh[4] = {B, Hc, 1, D};
    if (kn->sizes() != at::IntArrayRef(fresh, 4) || vn->sizes() != at::IntArrayRef(fresh, 4) || kn->scalar_type() != q->scalar_type() ||
        vn->scalar_type() != q->scalar_type() || !dense_rows(*kn) || !dense_rows(*vn))
      Py_RETURN_NONE;
  }
  at::Tensor out, lse;
  int rc;
  {
    const Unlocked others;
    out = at::empty({B, Hq, 1, D}, q->options());
    lse = at::empty({B, Hq, 1}, q->options().dtype(at::kFloat));
    rc = fp_paged_decode_step(
        static_cast<int32_t*>(arrivals->data_ptr()), after ? static_cast<int32_t*>(after->data_ptr()) : nullptr,
        arrivals->numel() * 4, kn ? kn->data_ptr() : nullptr, vn ? vn->data_ptr() : nullptr,
        kn ? kn->stride(0) : 0, kn ? kn->stride(1) : 0, vn ? vn->stride(0) : 0, vn ? vn->stride(1) : 0, q->data_ptr(), q->stride(0),
        q->stride(1), pk->data_ptr(), pv->data_ptr(), static_cast<const int64_t*>(table->data_ptr()), table->stride(0),
        static_cast<const int64_t*>(bidx->data_ptr()), pos->data_ptr(), it, out.data_ptr(), out.stride(0), out.stride(1),
        static_cast<float*>(lse.data_ptr()), sinks ? static_cast<const float*>(sinks->data_ptr()) : nullptr, ws ? ws->data_ptr() : nullptr,
        ws ? ws->numel() : 0, B, Hq, Hc, kv_rep, D, page_size, table->size(1), table->size(0), pk->size(1), max_context, split_tokens,
        static_cast<float>(scale), dt, plan ? plan->data_ptr() : nullptr, plan ? plan->numel() : 0, reinterpret_cast<void*>(stream));
  }
  if (rc < 0) return fail("fp_paged_decode_step", rc);
  return pair(out, lse);
}

// q, pool_k, pool_v, page_table, batch_idx, row_limit, page_size, scale, sinks, workspace, score_bound, tile_order, order_rows,
// stream -> (out, lse)
PyObject* prefill_unguarded(PyObject* const* args) {
  Args a{args};
  const at::Tensor *q = a.tensor(), *pk = a.tensor(), *pv = a.tensor(), *table = a.tensor(), *bidx = a.tensor(), *limit = a.tensor();
  const int64_t page_size = a.integer();
  const double scale = a.number();
  const at::Tensor *sinks = a.maybe_tensor(), *ws = a.maybe_tensor();
  const double bound = a.number();
  const at::Tensor* order = a.maybe_tensor();
  const int64_t order_rows = a.integer(), stream = a.integer();
  if (!a.ok) Py_RETURN_NONE;
  const int dt = dtype_code(*q);
  if (dt < 0 || q->dim() != 4 || q->size(0) != 1 || pk->dim() != 3 || pk->sizes() != pv->sizes() || pk->size(2) != q->size(3) ||
      pk->scalar_type() != q->scalar_type() || pv->scalar_type() != q->scalar_type() || !pk->is_contiguous() || !pv->is_contiguous() ||
      !dense_rows(*q) || !is_table(*table))
    Py_RETURN_NONE;
  const int64_t Hq = q->size(1), Lq = q->size(2), D = q->size(3), Hc = pk->size(0);
  if (!is_indices(*bidx, Lq) || limit->scalar_type() != at::kInt || !limit->is_contiguous() || limit->numel() != Lq ||
      (ws && !is_bytes(*ws)) ||
      (sinks && (sinks->scalar_type() != at::kFloat || sinks->dim() != 1 || sinks->size(0) != Hq || !sinks->is_contiguous() ||
                 sinks->device() != q->device())) ||
      (order && (order_rows <= 0 || order->scalar_type() != at::kInt || !order->is_contiguous() ||
                 order->numel() != (Lq + order_rows - 1) / order_rows)))
    Py_RETURN_NONE;
  at::Tensor out, lse;
  int rc = FP_OK;
  {
    const Unlocked others;
    out = at::empty_like(*q);
    lse = at::empty({1, Hq, Lq}, q->options().dtype(at::kFloat));
    if (dense_rows(out))
      rc = fp_paged_prefill(
          q->data_ptr(), q->stride(2), q->stride(1), pk->data_ptr(), pv->data_ptr(), static_cast<const int64_t*>(table->data_ptr()),
          table->stride(0), static_cast<const int64_t*>(bidx->data_ptr()), static_cast<const int32_t*>(limit->data_ptr()), out.data_ptr(),
          out.stride(2), out.stride(1), static_cast<float*>(lse.data_ptr()), sinks ? static_cast<const float*>(sinks->data_ptr()) : nullptr,
          Lq, Hq, Hc, D, page_size, table->size(1), table->size(0), pk->size(1), static_cast<float>(scale), static_cast<float>(bound), dt,
          ws ? ws->data_ptr() : nullptr, ws ? ws->numel() : 0, order ? static_cast<const int32_t*>(order->data_ptr()) : nullptr,
          order ? order_rows : 0, reinterpret_cast<void*>(stream));
  }
  if (!dense_rows(out)) Py_RETURN_NONE;
  if (rc < 0) return fail("fp_paged_prefill", rc);
  return pair(out, lse);
}

bool is_vector(const at::Tensor& t, at::ScalarType type, int64_t n) {
  return t.dim() == 1 && t.scalar_type() == type && t.is_contiguous() && t.size(0) == n;
}

// batch_idx, input_pos, prefix_ids, prefix_lens: the step of an attention over shared prefixes
bool is_shared_step(const at::Tensor& bidx, const at::Tensor& pos, const at::Tensor& ids, const at::Tensor& lens) {
  return bidx.dim() == 1 && is_indices(bidx, bidx.size(0)) && index_code(pos) >= 0 && pos.is_contiguous() &&
         (pos.dim() == 1 || pos.dim() == 2) && pos.size(0) == bidx.size(0) && ids.dim() == 1 &&
         is_vector(ids, at::kInt, ids.size(0)) && is_vector(lens, at::kInt, ids.size(0));
}

// batch_idx, input_pos, prefix_ids, prefix_lens, q_heads, cached_heads, head_dim, max_context, plan, device, stream -> True
PyObject* shared_plan_unguarded(PyObject* const* args) {
  Args a{args};
  const at::Tensor *bidx = a.tensor(), *pos = a.tensor(), *ids = a.tensor(), *lens = a.tensor();
  const int64_t Hq = a.integer(), Hc = a.integer(), D = a.integer(), max_context = a.integer();
  const at::Tensor* plan = a.tensor();
  const int64_t device = a.integer(), stream = a.integer();
  if (!a.ok || !is_shared_step(*bidx, *pos, *ids, *lens) || !is_bytes(*plan) || !on_device(device, {bidx, pos, ids, lens, plan}) ||
      !fits({bidx->size(0), pos->size(pos->dim() - 1), Hq, Hc, D, ids->size(0), max_context}))
    Py_RETURN_NONE;
  int rc;
  {
    const Unlocked others;
    rc = fp_shared_decode_plan(static_cast<const int64_t*>(bidx->data_ptr()), pos->data_ptr(), index_code(*pos),
                               static_cast<const int32_t*>(ids->data_ptr()), static_cast<const int32_t*>(lens->data_ptr()),
                               bidx->size(0), pos->dim() == 2 ? pos->size(1) : 1, Hq, Hc, D, ids->size(0), max_context,
                               plan->data_ptr(), plan->numel(), reinterpret_cast<void*>(stream));
  }
  if (rc < 0) return fail("fp_shared_decode_plan", rc);
  Py_RETURN_TRUE;
}

// q, pool_k, pool_v, page_table, batch_idx, input_pos, prefix_ids, prefix_lens, page_size, max_context, scale, sinks, plan, workspace,
// device, stream -> (out, lse)
PyObject* shared_unguarded(PyObject* const* args) {
  Args a{args};
  const at::Tensor *q = a.tensor(), *pk = a.tensor(), *pv = a.tensor(), *table = a.tensor(), *bidx = a.tensor(), *pos = a.tensor(),
                   *ids = a.tensor(), *lens = a.tensor();
  const int64_t page_size = a.integer(), max_context = a.integer();
  const double scale = a.number();
  const at::Tensor *sinks = a.maybe_tensor(), *plan = a.tensor(), *ws = a.tensor();
  const int64_t device = a.integer(), stream = a.integer();
  if (!a.ok) Py_RETURN_NONE;
  const int dt = dtype_code(*q);
  if (dt < 0 || q->dim() != 4 || pk->dim() != 3 || pk->sizes() != pv->sizes() || pk->size(2) != q->size(3) ||
      pk->scalar_type() != q->scalar_type() || pv->scalar_type() != q->scalar_type() || !pk->is_contiguous() || !pv->is_contiguous() ||
      !q->is_contiguous() || !is_table(*table) || !is_shared_step(*bidx, *pos, *ids, *lens) || !is_bytes(*plan) || !is_bytes(*ws))
    Py_RETURN_NONE;
  const int64_t B = q->size(0), Hq = q->size(1), S = q->size(2), D = q->size(3), Hc = pk->size(0);
  if (bidx->size(0) != B || (pos->dim() == 2 ? pos->size(1) : 1) != S || ids->size(0) != table->size(0) ||
      (sinks && !is_vector(*sinks, at::kFloat, Hq)) || !fits({B, S, Hq, Hc, D, page_size, table->size(0), table->size(1), max_context}) ||
      !on_device(device, {q, pk, pv, table, bidx, pos, ids, lens, sinks, plan, ws}))
    Py_RETURN_NONE;
  at::Tensor out, lse;
  int rc;
  {
    const Unlocked others;
    out = at::empty({B, Hq, S, D}, q->options());
    lse = at::empty({B, Hq, S}, q->options().dtype(at::kFloat));
    rc = fp_paged_decode_shared(
        q->data_ptr(), q->stride(0), q->stride(1), q->stride(2), pk->data_ptr(), pv->data_ptr(),
        static_cast<const int64_t*>(table->data_ptr()), table->stride(0), static_cast<const int64_t*>(bidx->data_ptr()), pos->data_ptr(),
        index_code(*pos), out.data_ptr(), out.stride(0), out.stride(1), out.stride(2), static_cast<float*>(lse.data_ptr()),
        sinks ? static_cast<const float*>(sinks->data_ptr()) : nullptr, ws->data_ptr(), ws->numel(), plan->data_ptr(), plan->numel(), B,
        S, Hq, Hc, D, page_size, table->size(1), table->size(0), pk->size(1), max_context, static_cast<float>(scale), dt,
        reinterpret_cast<void*>(stream));
  }
  if (rc < 0) return fail("fp_paged_decode_shared", rc);
  return pair(out, lse);
}

// Elements of a byte buffer's memory, from `offset` bytes on, as a tensor of these sizes that shares it
at::Tensor part(const at::Tensor& buffer, int64_t offset, at::IntArrayRef sizes, at::ScalarType type) {
  at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(buffer.storage()), buffer.key_set(), c10::scalarTypeToTypeMeta(type));
  t.unsafeGetTensorImpl()->set_storage_offset(buffer.storage_offset() + offset / static_cast<int64_t>(c10::elementSize(type)));
  t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
  return t;
}

PyObject* tuple_of(const at::Tensor* t, int n) {
  PyObject* const made = PyTuple_New(n);
  if (!made) return nullptr;
  for (int i = 0; i < n; ++i) PyTuple_SET_ITEM(made, i, THPVariable_Wrap(t[i]));
  return made;
}

// slots, old_lens, new_lens, free_pages, free_count, page_table, page_size, max_rows, parents, row_multiple, inverse, device, stream ->
// the nine tensors of StepTables
PyObject* tables_unguarded(PyObject* const* args) {
  Args a{args};
  const at::Tensor *slots = a.tensor(), *before = a.tensor(), *after = a.tensor(), *pages = a.tensor(), *count = a.tensor(),
                   *table = a.tensor();
  const int64_t page_size = a.integer(), rows = a.integer();
  const at::Tensor* parents = a.maybe_tensor();
  const int64_t multiple = a.integer();
  const at::Tensor* inverse = a.maybe_tensor();
  const int64_t device = a.integer(), stream = a.integer();
  if (!a.ok || slots->dim() != 1 || pages->dim() != 1 || rows < 0 || multiple < 1) Py_RETURN_NONE;
  const int64_t B = slots->size(0);
  if (!is_vector(*slots, at::kLong, B) || index_code(*before) < 0 || !is_vector(*before, before->scalar_type(), B) ||
      !is_vector(*after, before->scalar_type(), B) || !is_vector(*pages, at::kLong, pages->size(0)) || !is_vector(*count, at::kInt, 1) ||
      !is_table(*table) || (parents && !is_vector(*parents, at::kLong, B)) ||
      (inverse && (!is_table(*inverse) || inverse->size(0) != table->size(0))) ||
      !fits({pages->size(0), B, rows, multiple, page_size, table->size(0), table->size(1)}) ||
      !on_device(device, {slots, before, after, pages, count, table, parents, inverse}))
    Py_RETURN_NONE;
  at::Tensor made[9];
  int rc;
  {
    const Unlocked others;
    // two allocations, the rows and the rest: with nine a call is 13.6 us of the host, with two 8.1
    const auto bytes = slots->options().dtype(at::kByte);
    const int64_t wide = (rows + 3) / 4 * 4;
    const at::Tensor big = at::empty({20 * wide}, bytes), small = at::empty({16 * B + 4 * (2 * B + 3)}, bytes);
    made[0] = part(big, 0, {rows}, at::kLong);
    made[2] = part(big, 8 * wide, {rows}, at::kLong);
    made[1] = part(big, 16 * wide, {rows}, at::kInt);
    made[5] = part(small, 0, {B}, at::kLong);
    made[6] = part(small, 8 * B, {B}, at::kLong);
    made[3] = part(small, 16 * B, {B + 1}, at::kInt);
    made[7] = part(small, 20 * B + 4, {B}, at::kInt);
    made[4] = part(small, 24 * B + 4, {1}, at::kInt);
    made[8] = part(small, 24 * B + 8, {1}, at::kInt);
    const auto at = [&](int i) { return made[i].data_ptr(); };
    rc = fp_step_tables(static_cast<const int64_t*>(slots->data_ptr()), before->data_ptr(), after->data_ptr(), index_code(*before),
                        parents ? static_cast<const int64_t*>(parents->data_ptr()) : nullptr, static_cast<const int64_t*>(pages->data_ptr()),
                        static_cast<const int32_t*>(count->data_ptr()), pages->size(0), static_cast<int64_t*>(table->data_ptr()),
                        table->stride(0), inverse ? static_cast<int64_t*>(inverse->data_ptr()) : nullptr, inverse ? inverse->stride(0) : 0,
                        inverse ? inverse->size(1) : 0, static_cast<int64_t*>(at(0)), static_cast<int32_t*>(at(1)),
                        static_cast<int64_t*>(at(2)), static_cast<int32_t*>(at(3)), static_cast<int32_t*>(at(4)),
                        static_cast<int64_t*>(at(5)), static_cast<int64_t*>(at(6)), static_cast<int32_t*>(at(7)),
                        static_cast<int32_t*>(at(8)), B, rows, multiple, page_size, table->size(1), table->size(0),
                        reinterpret_cast<void*>(stream));
  }
  if (rc < 0) return fail("fp_step_tables", rc);
  return tuple_of(made, 9);
}

// pool, src, dst, rows, page_size, device, stream -> True
PyObject* copy_unguarded(PyObject* const* args) {
  Args a{args};
  const at::Tensor *pool = a.tensor(), *src = a.tensor(), *dst = a.tensor(), *rows = a.tensor();
  const int64_t page_size = a.integer(), device = a.integer(), stream = a.integer();
  if (!a.ok || dtype_code(*pool) < 0 || pool->dim() < 2 || !pool->is_contiguous() || pool->numel() == 0 || src->dim() != 1 ||
      !is_vector(*src, at::kLong, src->size(0)) || !is_vector(*dst, at::kLong, src->size(0)) ||
      !is_vector(*rows, at::kInt, src->size(0)) || page_size < 1 || !fits({src->size(0), pool->size(-1), page_size}) ||
      !on_device(device, {pool, src, dst, rows}))
    Py_RETURN_NONE;
  const int64_t D = pool->size(-1), n_slots = pool->size(-2);
  int rc;
  {
    const Unlocked others;
    rc = fp_copy_pages(pool->data_ptr(), static_cast<const int64_t*>(src->data_ptr()), static_cast<const int64_t*>(dst->data_ptr()),
                       static_cast<const int32_t*>(rows->data_ptr()), src->size(0), pool->numel() / (n_slots * D), n_slots, D, page_size,
                       dtype_code(*pool), reinterpret_cast<void*>(stream));
  }
  if (rc < 0) return fail("fp_copy_pages", rc);
  Py_RETURN_TRUE;
}

// [B, S] of this type
bool is_matrix(const at::Tensor& t, at::ScalarType type, int64_t B, int64_t S) {
  return t.dim() == 2 && t.scalar_type() == type && t.is_contiguous() && t.size(0) == B && t.size(1) == S;
}
bool is_lengths(const at::Tensor& t, int64_t n) { return index_code(t) >= 0 && is_vector(t, t.scalar_type(), n); }
bool is_tree(const at::Tensor& masks, const at::Tensor& pos) {
  return masks.dim() == 2 && is_matrix(masks, at::kLong, masks.size(0), masks.size(1)) && index_code(pos) >= 0 &&
         is_matrix(pos, pos.scalar_type(), masks.size(0), masks.size(1));
}

// parents, cached, device, stream -> masks, input_pos, rope_pos
PyObject* draft_tree_unguarded(PyObject* const* args) {
  Args a{args};
  const at::Tensor *parents = a.tensor(), *cached = a.tensor();
  const int64_t device = a.integer(), stream = a.integer();
  if (!a.ok || parents->dim() != 2) Py_RETURN_NONE;
  const int64_t B = parents->size(0), S = parents->size(1);
  if (!is_matrix(*parents, at::kInt, B, S) || !is_lengths(*cached, B) || !fits({B, S}) || S < 1 || S > 64 || !on_device(device, {parents, cached}))
    Py_RETURN_NONE;
  at::Tensor made[3];
  int rc;
  {
    const Unlocked others;
    const at::Tensor all = at::empty({16 * B * S}, parents->options().dtype(at::kByte));
    made[0] = part(all, 0, {B, S}, at::kLong);
    made[1] = part(all, 8 * B * S, {B, S}, at::kInt);
    made[2] = part(all, 12 * B * S, {B, S}, at::kInt);
    rc = fp_draft_tree(static_cast<const int32_t*>(parents->data_ptr()), cached->data_ptr(), index_code(*cached), B, S,
                       static_cast<int64_t*>(made[0].data_ptr()), static_cast<int32_t*>(made[1].data_ptr()),
                       static_cast<int32_t*>(made[2].data_ptr()), reinterpret_cast<void*>(stream));
  }
  if (rc < 0) return fail("fp_draft_tree", rc);
  return tuple_of(made, 3);
}

// batch_idx, masks, input_pos, page_table, q_heads, cached_heads, head_dim, max_context, prefix_ids, prefix_lens, plan, device, stream -> True
PyObject* tree_plan_unguarded(PyObject* const* args) {
  Args a{args};
  const at::Tensor *bidx = a.tensor(), *masks = a.tensor(), *pos = a.tensor(), *table = a.tensor();
  const int64_t Hq = a.integer(), Hc = a.integer(), D = a.integer(), max_context = a.integer();
  const at::Tensor *ids = a.maybe_tensor(), *lens = a.maybe_tensor(), *plan = a.tensor();
  const int64_t device = a.integer(), stream = a.integer();
  if (!a.ok || !is_tree(*masks, *pos) || !is_vector(*bidx, at::kLong, masks->size(0)) || !is_table(*table) || !ids != !lens ||
      (ids && (!is_vector(*ids, at::kInt, table->size(0)) || !is_vector(*lens, at::kInt, table->size(0)))) || !is_bytes(*plan) ||
      !on_device(device, {bidx, masks, pos, table, ids, lens, plan}) || !fits({masks->size(0), masks->size(1), Hq, Hc, D, table->size(0), max_context}))
    Py_RETURN_NONE;
  int rc;
  {
    const Unlocked others;
    rc = fp_tree_decode_plan(static_cast<const int64_t*>(bidx->data_ptr()), pos->data_ptr(), index_code(*pos),
                             ids ? static_cast<const int32_t*>(ids->data_ptr()) : nullptr,
                             ids ? static_cast<const int32_t*>(lens->data_ptr()) : nullptr, masks->size(0), masks->size(1), Hq, Hc, D,
                             table->size(0), max_context, plan->data_ptr(), plan->numel(), reinterpret_cast<void*>(stream));
  }
  if (rc < 0) return fail("fp_tree_decode_plan", rc);
  Py_RETURN_TRUE;
}

// q, pool_k, pool_v, page_table, batch_idx, masks, input_pos, page_size, max_context, scale, sinks, plan, workspace, device, stream -> (out, lse)
PyObject* tree_unguarded(PyObject* const* args) {
  Args a{args};
  const at::Tensor *q = a.tensor(), *pk = a.tensor(), *pv = a.tensor(), *table = a.tensor(), *bidx = a.tensor(), *masks = a.tensor(),
                   *pos = a.tensor();
  const int64_t page_size = a.integer(), max_context = a.integer();
  const double scale = a.number();
  const at::Tensor *sinks = a.maybe_tensor(), *plan = a.tensor(), *ws = a.tensor();
  const int64_t device = a.integer(), stream = a.integer();
  if (!a.ok) Py_RETURN_NONE;
  const int dt = dtype_code(*q);
  if (dt < 0 || q->dim() != 4 || pk->dim() != 3 || pk->sizes() != pv->sizes() || pk->size(2) != q->size(3) ||
      pk->scalar_type() != q->scalar_type() || pv->scalar_type() != q->scalar_type() || !pk->is_contiguous() || !pv->is_contiguous() ||
      !q->is_contiguous() || reinterpret_cast<uintptr_t>(q->data_ptr()) % 16 != 0 || !is_table(*table) || !is_tree(*masks, *pos) ||
      !is_bytes(*plan) || !is_bytes(*ws))
    Py_RETURN_NONE;
  const int64_t B = q->size(0), Hq = q->size(1), S = q->size(2), D = q->size(3), Hc = pk->size(0);
  if (!is_vector(*bidx, at::kLong, B) || masks->size(0) != B || masks->size(1) != S || (sinks && !is_vector(*sinks, at::kFloat, Hq)) ||
      !fits({B, S, Hq, Hc, D, page_size, table->size(0), table->size(1), max_context}) ||
      !on_device(device, {q, pk, pv, table, bidx, masks, pos, sinks, plan, ws}))
    Py_RETURN_NONE;
  at::Tensor out, lse;
  int rc;
  {
    const Unlocked others;
    out = at::empty({B, Hq, S, D}, q->options());
    lse = at::empty({B, Hq, S}, q->options().dtype(at::kFloat));
    rc = fp_paged_decode_tree(
        static_cast<const int64_t*>(masks->data_ptr()), q->data_ptr(), q->stride(0), q->stride(1), q->stride(2), pk->data_ptr(), pv->data_ptr(),
        static_cast<const int64_t*>(table->data_ptr()), table->stride(0), static_cast<const int64_t*>(bidx->data_ptr()), pos->data_ptr(),
        index_code(*pos), out.data_ptr(), out.stride(0), out.stride(1), out.stride(2), static_cast<float*>(lse.data_ptr()),
        sinks ? static_cast<const float*>(sinks->data_ptr()) : nullptr, ws->data_ptr(), ws->numel(), plan->data_ptr(), plan->numel(), B,
        S, Hq, Hc, D, page_size, table->size(1), table->size(0), pk->size(1), max_context, static_cast<float>(scale), dt,
        reinterpret_cast<void*>(stream));
  }
  if (rc < 0) return fail("fp_paged_decode_tree", rc);
  return pair(out, lse);
}

// logits, tokens, parents, uniforms, temperatures, draft_probs, workspace, device, stream -> accepted, path, tokens, logprobs
PyObject* verify_unguarded(PyObject* const* args) {
  Args a{args};
  const at::Tensor *logits = a.tensor(), *tokens = a.tensor(), *parents = a.tensor(), *uniforms = a.tensor(), *heat = a.maybe_tensor(),
                   *probs = a.maybe_tensor(), *ws = a.tensor();
  const int64_t device = a.integer(), stream = a.integer();
  if (!a.ok) Py_RETURN_NONE;
  const int dt = dtype_code(*logits), pt = probs ? dtype_code(*probs) : 0;
  if (dt < 0 || pt < 0 || logits->dim() != 3 || !dense_rows(*logits) || (probs && (probs->sizes() != logits->sizes() || !dense_rows(*probs))))
    Py_RETURN_NONE;
  const int64_t B = logits->size(0), S = logits->size(1), V = logits->size(2);
  if (S < 1 || S > 64 || V < 1 || !is_matrix(*tokens, at::kLong, B, S) || !is_matrix(*parents, at::kInt, B, S) || !is_matrix(*uniforms, at::kFloat, B, S) ||
      (heat && !is_vector(*heat, at::kFloat, B)) || !is_bytes(*ws) || !fits({B, S, V}) ||
      !on_device(device, {logits, tokens, parents, uniforms, heat, probs, ws}))
    Py_RETURN_NONE;
  at::Tensor made[4];
  int rc;
  {
    const Unlocked others;
    const at::Tensor all = at::empty({B * (16 * S + 4)}, logits->options().dtype(at::kByte));
    made[2] = part(all, 0, {B, S}, at::kLong);
    made[1] = part(all, 8 * B * S, {B, S}, at::kInt);
    made[3] = part(all, 12 * B * S, {B, S}, at::kFloat);
    made[0] = part(all, 16 * B * S, {B}, at::kInt);
    rc = fp_verify_drafts(logits->data_ptr(), logits->stride(0), logits->stride(1), dt, static_cast<const int64_t*>(tokens->data_ptr()),
                          static_cast<const int32_t*>(parents->data_ptr()), static_cast<const float*>(uniforms->data_ptr()),
                          heat ? static_cast<const float*>(heat->data_ptr()) : nullptr, probs ? probs->data_ptr() : nullptr,
                          probs ? probs->stride(0) : 0, probs ? probs->stride(1) : 0, pt, static_cast<int32_t*>(made[0].data_ptr()),
                          static_cast<int32_t*>(made[1].data_ptr()), static_cast<int64_t*>(made[2].data_ptr()),
                          static_cast<float*>(made[3].data_ptr()), ws->data_ptr(), ws->numel(), B, S, V, reinterpret_cast<void*>(stream));
  }
  if (rc < 0) return fail("fp_verify_drafts", rc);
  return tuple_of(made, 4);
}

// pool, page_table, batch_idx, cached, path, page_size, device, stream -> True
PyObject* keep_unguarded(PyObject* const* args) {
  Args a{args};
  const at::Tensor *pool = a.tensor(), *table = a.tensor(), *bidx = a.tensor(), *cached = a.tensor(), *path = a.tensor();
  const int64_t page_size = a.integer(), device = a.integer(), stream = a.integer();
  if (!a.ok || dtype_code(*pool) < 0 || pool->dim() < 2 || !pool->is_contiguous() || pool->numel() == 0 || path->dim() != 2) Py_RETURN_NONE;
  const int64_t B = path->size(0), S = path->size(1), D = pool->size(-1), n_slots = pool->size(-2);
  if (S < 1 || S > 64 || !is_matrix(*path, at::kInt, B, S) || !is_table(*table) || !is_vector(*bidx, at::kLong, B) || !is_lengths(*cached, B) ||
      page_size < 1 || !fits({B, S, D, page_size, table->size(0), table->size(1)}) || !on_device(device, {pool, table, bidx, cached, path}))
    Py_RETURN_NONE;
  int rc;
  {
    const Unlocked others;
    rc = fp_keep_rows(pool->data_ptr(), static_cast<const int64_t*>(table->data_ptr()), table->stride(0),
                      static_cast<const int64_t*>(bidx->data_ptr()), cached->data_ptr(), index_code(*cached),
                      static_cast<const int32_t*>(path->data_ptr()), B, S, pool->numel() / (n_slots * D), n_slots, D, page_size, table->size(1),
                      table->size(0), dtype_code(*pool), reinterpret_cast<void*>(stream));
  }
  if (rc < 0) return fail("fp_keep_rows", rc);
  Py_RETURN_TRUE;
}

// A C++ exception (an allocation that failed) becomes a Python one.
template <PyObject* (*kCall)(PyObject* const*), Py_ssize_t kArgs>
PyObject* guarded(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != kArgs) {
    PyErr_Format(PyExc_TypeError, "%zd arguments expected, %zd given", kArgs, n);
    return nullptr;
  }
  HANDLE_TH_ERRORS
  return kCall(args);
  END_HANDLE_TH_ERRORS
}

#define FP_METHOD(name, call, n) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<call, n>)), METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {FP_METHOD("append", append_unguarded, 11), FP_METHOD("decode", decode_unguarded, 19),
                          FP_METHOD("prefill", prefill_unguarded, 14),
                          FP_METHOD("shared_plan", shared_plan_unguarded, 11), FP_METHOD("shared", shared_unguarded, 16),
                          FP_METHOD("tables", tables_unguarded, 13), FP_METHOD("copy_pages", copy_unguarded, 7),
                          FP_METHOD("draft_tree", draft_tree_unguarded, 4), FP_METHOD("tree_plan", tree_plan_unguarded, 13),
                          FP_METHOD("tree", tree_unguarded, 15), FP_METHOD("verify", verify_unguarded, 9), FP_METHOD("keep", keep_unguarded, 8),
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "fp_host", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_fp_host() {
  if (fp_abi_version() != FP_ABI_VERSION) {
    PyErr_Format(PyExc_RuntimeError, "libfp_paged_kv.so has ABI %d, fp_host was built for %d", fp_abi_version(), FP_ABI_VERSION);
    return nullptr;
  }
  PyObject* const module = PyModule_Create(&kModule);
  if (module) PyModule_AddStringConstant(module, "torch_version", TORCH_VERSION);
  return module;
}
