// The host's part of a decode step and of a token through the model, as calls of one Python module
// (_host): the operands' checks, the outputs' allocation and the library's entry point in one
// native call each.  Nothing is kept from call to call: every operand is looked at every time.
//
// Bound: the interpreter.  A check of a tensor costs 0.1 us an attribute from Python, 17 tensors
// of 4 to 8 attributes a step, which made a step of a small layer wait for its caller.  us of a host
// thread, from Python / from here: a paged layer's step 29 / 22, a static one's 26 / 12, a token of a
// 4-layer model 331 / 218, of which 3 us a launch are the runtime's.
//
// A call that finds an operand other than the kernels take it returns None (or false): the
// caller then goes the general way, which takes or refuses it.  The calls of a batch of sequences
// (rotate, paged_append, paged_attention) are the only way and refuse it themselves.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/TracerMode.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <c10/util/SmallVector.h>
#include <torch/csrc/Exceptions.h>
#include <hip/hip_runtime_api.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <initializer_list>
#include <string>
#include <vector>

#include "../../include/dram_attention_amd.h"

namespace {

PyObject *parameter_class;   // torch.nn.Parameter

// Plain tensors only: what a subclass does when it is read is its own.
const at::Tensor *tensor_of(PyObject *o) {
  if (Py_TYPE(o) != (PyTypeObject *)THPVariableClass && (PyObject *)Py_TYPE(o) != parameter_class) return nullptr;
  const at::Tensor &t = THPVariable_Unpack(o);
  return t.layout() == at::kStrided ? &t : nullptr;
}

int dtype_code(const at::Tensor &t) {
  switch (t.scalar_type()) {
    case at::kFloat: return DA_F32;
    case at::kHalf: return DA_F16;
    case at::kBFloat16: return DA_BF16;
    default: return -1;
  }
}

bool like(const at::Tensor &t, const at::Tensor &x) {
  return t.scalar_type() == x.scalar_type() && t.device() == x.device() && t.is_contiguous();
}
bool aligned(const at::Tensor &t) { return (uintptr_t)t.data_ptr() % 16 == 0; }
bool is_shape(const at::Tensor &t, at::IntArrayRef want) { return t.sizes() == want; }

// A whole number of any kind (numpy's too); `ok` is left false by anything else.
int64_t whole_number(PyObject *o, bool &ok) {
  PyObject *n = PyNumber_Index(o);
  const long long v = n ? PyLong_AsLongLong(n) : -1;
  Py_XDECREF(n);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    ok = false;
  }
  return v;
}

// Positional arguments, read in order; what is not what it should be leaves `ok` false.
struct Args {
  PyObject *const *at;
  Py_ssize_t left;
  bool ok = true;
  PyObject *next() {
    if (left <= 0) {
      ok = false;
      return Py_None;
    }
    --left;
    return *at++;
  }
  const at::Tensor *tensor() {
    const at::Tensor *t = tensor_of(next());
    ok = ok && t != nullptr;
    return t;
  }
  const at::Tensor *tensor_or_none() {
    PyObject *o = next();
    if (o == Py_None) return nullptr;
    const at::Tensor *t = tensor_of(o);
    ok = ok && t != nullptr;
    return t;
  }
  int64_t integer() { return whole_number(next(), ok); }
  double number() {
    PyObject *o = next();
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) {
      PyErr_Clear();
      ok = false;
    }
    return v;
  }
  void *pointer() {
    PyObject *o = next();
    if (!PyLong_Check(o)) {
      ok = false;
      return nullptr;
    }
    void *p = PyLong_AsVoidPtr(o);
    if (p == nullptr && PyErr_Occurred()) {
      PyErr_Clear();
      ok = false;
    }
    return p;
  }
};

PyObject *raise(int rc, const char *what) {
  PyErr_Format(PyExc_RuntimeError, "%s failed (code %d): %s", what, rc, da_last_error_string());
  return nullptr;
}
// Other Python threads run while this one allocates or launches: either may wait, an allocation for
// another thread that holds the allocator, a launch for room in its queue.
// (autograd's threads call without holding the interpreter)
struct Released {
  PyThreadState *state = PyGILState_Check() ? PyEval_SaveThread() : nullptr;
  ~Released() {
    if (state) PyEval_RestoreThread(state);
  }
};
template <typename F>
int unlocked(F call) {
  const Released others;
  return call();
}
at::Tensor empty_like(at::IntArrayRef sizes, const at::Tensor &x) {
  const Released others;
  return at::empty(sizes, x.options().requires_grad(false));
}
PyObject *wrap(at::Tensor t) { return THPVariable_Wrap(std::move(t)); }
// A tuple that takes these over; null, with the error that is set, if one is.
PyObject *tuple_of(std::initializer_list<PyObject *> items) {
  PyObject *result = PyTuple_New((Py_ssize_t)items.size());
  bool whole = result != nullptr;
  Py_ssize_t n = 0;
  for (PyObject *o : items) {
    whole = whole && o != nullptr;
    if (result)
      PyTuple_SET_ITEM(result, n++, o);
    else
      Py_XDECREF(o);
  }
  if (!whole) Py_CLEAR(result);
  return result;
}

// The position of the token: a Python int, or one int32 on the device.
struct Position {
  int64_t len;
  const int32_t *len_dev;
};
bool position(PyObject *o, int64_t paged, const at::Tensor &x, Position &p) {
  if (PyLong_CheckExact(o)) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) {
      PyErr_Clear();
      return false;
    }
    p = {v - paged, nullptr};
    return true;
  }
  const at::Tensor *t = tensor_of(o);
  if (!t || t->scalar_type() != at::kInt || t->device() != x.device() || t->numel() < 1) return false;
  p = {-paged, (const int32_t *)t->data_ptr()};
  return true;
}

// step_args(xq, xk, xv, start_pos, minmax, dram, hbm, times, d2h, h2d, counter, cache_k, cache_v, n_slots,
// page, top_k, paged, dram_ptr, stream_blocks, score_flags, link_gbps, block_gbps, scratch, idx, scores, topk_ws,
// workspace) -> (argument block of da_decode_step, output); None: not a step for one call; an
// int, the query rows of a kv head: the operands are, but the last five are not there yet.
PyObject *step_args(PyObject *, PyObject *const *argv, Py_ssize_t argc) {
  HANDLE_TH_ERRORS
  Args in{argv, argc};
  const at::Tensor *xq = in.tensor(), *xk = in.tensor(), *xv = in.tensor();
  PyObject *start = in.next();
  const at::Tensor *minmax = in.tensor(), *dram = in.tensor(), *hbm = in.tensor(), *times = in.tensor(),
                   *d2h = in.tensor(), *h2d = in.tensor(), *counter = in.tensor(), *cache_k = in.tensor(),
                   *cache_v = in.tensor();
  const int64_t N = in.integer(), page = in.integer(), top_k = in.integer(), paged = in.integer();
  void *dram_ptr = in.pointer();
  const int64_t stream_blocks = in.integer(), flags = in.integer();
  const double link = in.number(), block = in.number();
  PyObject *scratch = in.next();
  if (!in.ok) Py_RETURN_NONE;
  const int dtype = dtype_code(*xq);
  if (dtype < 0 || !xq->is_cuda() || xq->dim() != 4 || minmax->dim() != 4) Py_RETURN_NONE;
  const int64_t H = minmax->size(0), P = minmax->size(1), D = minmax->size(3), Hq = xq->size(2);
  if (H < 1 || cache_k->dim() != 4) Py_RETURN_NONE;
  const int64_t rep = Hq / H, kp = top_k < P ? top_k : P, capacity = cache_k->size(1), page_dim = page * 2 * D;
  if (!(is_shape(*xq, {1, 1, rep * H, D}) && is_shape(*xk, {1, 1, H, D}) && is_shape(*xv, {1, 1, H, D}) && kp > 0 &&
        N > 0 && minmax->size(2) == 2 && is_shape(*hbm, {H, N, page_dim}) && is_shape(*dram, {H, P, page_dim}) &&
        is_shape(*times, {H, N}) && is_shape(*h2d, {H, N}) && is_shape(*d2h, {H, P}) &&
        is_shape(*cache_k, {1, capacity, H, D}) && is_shape(*cache_v, {1, capacity, H, D}) &&
        times->scalar_type() == at::kFloat && d2h->scalar_type() == at::kLong && h2d->scalar_type() == at::kLong &&
        counter->scalar_type() == at::kInt && counter->numel() == 1))
    Py_RETURN_NONE;
  // (what the attending page stream takes)
  const int64_t row = D * xq->element_size();
  if (!((row == 64 || row == 128 || row == 256 || row == 512) && rep >= 1 && rep <= 8 && page * 2 * row <= 16384 &&
        H <= 64))
    Py_RETURN_NONE;
  for (const at::Tensor *t : {xq, xk, xv, minmax, hbm, cache_k, cache_v})
    if (!like(*t, *xq)) Py_RETURN_NONE;
  for (const at::Tensor *t : {times, d2h, h2d, counter})
    if (t->device() != xq->device() || !t->is_contiguous()) Py_RETURN_NONE;
  if (dram->scalar_type() != xq->scalar_type() || !dram->is_contiguous()) Py_RETURN_NONE;
  Position pos;
  if (!position(start, paged, *xq, pos)) Py_RETURN_NONE;
  if (!pos.len_dev && (pos.len < 0 || pos.len >= capacity)) Py_RETURN_NONE;

  // (the room is looked at like the operands: the kernels write to all of it)
  const int64_t total = rep * kp;
  auto fits = [&](const at::Tensor *t, at::IntArrayRef shape, at::ScalarType type) {
    return t && t->scalar_type() == type && t->device() == xq->device() && t->is_contiguous() && is_shape(*t, shape);
  };
  const at::Tensor *idx = in.tensor_or_none(), *scores = in.tensor_or_none(), *topk_ws = in.tensor_or_none(),
                   *workspace = in.tensor_or_none();
  if (!in.ok) Py_RETURN_NONE;
  const size_t topk_need = da_topk_pages_workspace_bytes((int)rep, (int)H, P, (int)kp);
  if (!PyTuple_Check(scratch) || PyTuple_GET_SIZE(scratch) != 7 || !fits(idx, {H, total}, at::kLong) ||
      !fits(scores, {rep, H, P}, at::kFloat) || !workspace || !fits(workspace, workspace->sizes(), at::kFloat) ||
      (topk_need && (!topk_ws || !fits(topk_ws, topk_ws->sizes(), at::kByte) ||
                     (size_t)topk_ws->nbytes() < topk_need)))
    return PyLong_FromLongLong(rep);
  const at::Tensor *room[7];   // miss_page, miss_slot, miss_count, hit_mask, workspace, slot_epoch, candidates
  for (int i = 0; i < 7; ++i)
    if (!(room[i] = tensor_of(PyTuple_GET_ITEM(scratch, i)))) Py_RETURN_NONE;
  if (room[0]->dim() != 2 || room[0]->size(1) != total) return PyLong_FromLongLong(rep);
  const at::Tensor &list = *room[6];
  if (list.dim() != 2 || list.size(1) < 1) Py_RETURN_NONE;
  const int64_t stamps_end = list.storage_offset() + H * (list.size(1) + 1);   // (a word per head behind the lists)
  if (!(fits(room[0], {H, total}, at::kInt) && fits(room[1], {H, total}, at::kInt) && fits(room[2], {H}, at::kInt) &&
        fits(room[3], {H, total}, at::kByte) && fits(room[4], room[4]->sizes(), at::kByte) &&
        fits(room[5], {H, N}, at::kInt) && fits(&list, {H, list.size(1)}, at::kInt) &&
        (int64_t)list.storage().nbytes() >= stamps_end * 4))
    Py_RETURN_NONE;

  at::Tensor out = empty_like({1, 1, Hq, D}, *xq);
  da_decode_step_args a = {};
  a.q = xq->data_ptr();
  a.new_k = xk->data_ptr();
  a.new_v = xv->data_ptr();
  a.out = out.data_ptr();
  a.minmax = minmax->data_ptr();
  a.scores = (float *)scores->data_ptr();
  a.idx = (int64_t *)idx->data_ptr();
  if (topk_need) {
    a.topk_workspace = topk_ws->data_ptr();
    a.topk_workspace_bytes = (int64_t)topk_ws->nbytes();
  }
  a.access_time = (float *)times->data_ptr();
  a.candidates = (int32_t *)room[6]->data_ptr();
  a.step = (int32_t *)counter->data_ptr();
  a.d2h = (int64_t *)d2h->data_ptr();
  a.h2d = (int64_t *)h2d->data_ptr();
  a.miss_page = (int32_t *)room[0]->data_ptr();
  a.miss_slot = (int32_t *)room[1]->data_ptr();
  a.miss_count = (int32_t *)room[2]->data_ptr();
  a.hit_mask = (uint8_t *)room[3]->data_ptr();
  a.lru_workspace = room[4]->data_ptr();
  a.lru_workspace_bytes = (int64_t)room[4]->nbytes();
  a.slot_epoch = (int32_t *)room[5]->data_ptr();
  a.dram = dram_ptr;
  a.hbm = hbm->data_ptr();
  a.cache_k = cache_k->data_ptr();
  a.cache_v = cache_v->data_ptr();
  a.cache_len_dev = pos.len_dev;
  a.workspace = workspace->data_ptr();
  a.workspace_bytes = (int64_t)workspace->nbytes();
  a.q_head_stride = D;
  a.n_pages = P;
  a.cache_rows = capacity;
  a.cache_len = pos.len;
  a.n_q_heads = (int32_t)Hq;
  a.n_kv_heads = (int32_t)H;
  a.head_dim = (int32_t)D;
  a.dtype = dtype;
  a.page_size = (int32_t)page;
  a.kp = (int32_t)kp;
  a.n_slots = (int32_t)N;
  a.k_cand = (int32_t)room[6]->size(1);
  a.score_flags = (int32_t)flags;
  const int64_t blocks = stream_blocks / H < total ? stream_blocks / H : total;
  a.gather_blocks = (int32_t)(blocks > 1 ? blocks : 1);
  a.scale = (float)(1.0 / std::sqrt((double)D));
  a.link_gbps = (float)link;
  a.block_gbps = (float)block;
  return tuple_of({PyBytes_FromStringAndSize((const char *)&a, sizeof(a)), wrap(std::move(out))});
  END_HANDLE_TH_ERRORS
}

// static_step(xq, xk, xv, start_pos, prefix_k, prefix_v, cache_k, cache_v, paged, workspace, stream) -> output of
// a step over a static prefix, or None.
PyObject *static_step(PyObject *, PyObject *const *argv, Py_ssize_t argc) {
  HANDLE_TH_ERRORS
  Args in{argv, argc};
  const at::Tensor *xq = in.tensor(), *xk = in.tensor(), *xv = in.tensor();
  PyObject *start = in.next();
  const at::Tensor *pk = in.tensor(), *pv = in.tensor(), *ck = in.tensor(), *cv = in.tensor();
  const int64_t paged = in.integer();
  const at::Tensor *workspace = in.tensor_or_none();
  void *stream = in.pointer();
  if (!in.ok || !workspace) Py_RETURN_NONE;
  const int dtype = dtype_code(*xq);
  if (dtype < 0 || !xq->is_cuda() || xq->dim() != 4 || pk->dim() != 3 || ck->dim() != 4) Py_RETURN_NONE;
  const int64_t Hq = xq->size(2), D = xq->size(3), H = ck->size(2), capacity = ck->size(1), T = pk->size(1);
  if (!(is_shape(*xq, {1, 1, Hq, D}) && is_shape(*xk, {1, 1, H, D}) && is_shape(*xv, {1, 1, H, D}) &&
        is_shape(*pk, {H, T, D}) && is_shape(*pv, {H, T, D}) && is_shape(*ck, {1, capacity, H, D}) &&
        is_shape(*cv, {1, capacity, H, D}) && T > 0 && capacity > 0 && pk->strides() == pv->strides() &&
        ck->strides() == cv->strides() && xk->strides() == xv->strides() && workspace->is_contiguous()))
    Py_RETURN_NONE;
  for (const at::Tensor *t : {xq, xk, xv, pk, pv, ck, cv})
    if (t->scalar_type() != xq->scalar_type() || t->device() != xq->device() || t->stride(-1) != 1) Py_RETURN_NONE;
  if (workspace->device() != xq->device()) Py_RETURN_NONE;
  Position pos;
  if (!position(start, paged, *xq, pos)) Py_RETURN_NONE;
  at::Tensor out = empty_like({1, 1, Hq, D}, *xq);
  const int rc = unlocked([&] {
    return da_decode_attention(
        xq->data_ptr(), xq->stride(2), (int)Hq, (int)H, (int)D, dtype, pk->data_ptr(), pv->data_ptr(), pk->stride(1),
        pk->stride(0), T, ck->data_ptr(), cv->data_ptr(), ck->stride(1), ck->stride(2), capacity, pos.len, pos.len_dev,
        xk->data_ptr(), xv->data_ptr(), xk->stride(2), (float)(1.0 / std::sqrt((double)D)), out.data_ptr(), D, nullptr,
        workspace->data_ptr(), workspace->nbytes(), stream);
  });
  if (rc) return raise(rc, "da_decode_attention");
  return wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// alike(x, ...) -> whether all are plain, contiguous, aligned GPU tensors of x's type and device.
PyObject *alike(PyObject *, PyObject *const *argv, Py_ssize_t argc) {
  HANDLE_TH_ERRORS
  Args in{argv, argc};
  const at::Tensor *x = in.tensor();
  if (!in.ok || !x->is_cuda() || dtype_code(*x) < 0 || !like(*x, *x) || !aligned(*x)) Py_RETURN_FALSE;
  while (in.left > 0) {
    const at::Tensor *t = in.tensor();
    if (!in.ok || !like(*t, *x) || !aligned(*t)) Py_RETURN_FALSE;
  }
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// linears(x, nn.Linear, longest_row, module, out, in, module, out, in, ...) -> the modules' weights as a tuple, or
// None: each is an nn.Linear (no kind of its own) without bias, that nobody hooked and whose forward
// nobody exchanged, its weight a plain contiguous aligned tensor of x's type and device, of shape
// (out, in) (-1: whatever the module says) and with rows that the one-token layers hold.
PyObject *linears(PyObject *, PyObject *const *argv, Py_ssize_t argc) {
  HANDLE_TH_ERRORS
  static PyObject *hooks = PyUnicode_InternFromString("_forward_hooks");
  static PyObject *pre_hooks = PyUnicode_InternFromString("_forward_pre_hooks");
  static PyObject *forward = PyUnicode_InternFromString("forward");
  static PyObject *parameters = PyUnicode_InternFromString("_parameters");
  static PyObject *weight_name = PyUnicode_InternFromString("weight");
  static PyObject *bias_name = PyUnicode_InternFromString("bias");
  static PyObject *out_name = PyUnicode_InternFromString("out_features");
  static PyObject *in_name = PyUnicode_InternFromString("in_features");
  Args in{argv, argc};
  const at::Tensor *x = in.tensor();
  PyObject *linear = in.next();
  const int64_t longest = in.integer();
  if (!in.ok || in.left % 3) Py_RETURN_NONE;
  const Py_ssize_t n = in.left / 3;
  PyObject *weights = PyTuple_New(n);
  if (!weights) return nullptr;
  auto item = [](PyObject *dict, PyObject *name) -> PyObject * {
    PyObject *o = dict && PyDict_Check(dict) ? PyDict_GetItemWithError(dict, name) : nullptr;
    if (!o) PyErr_Clear();
    return o;
  };
  auto features = [&](PyObject *dict, PyObject *name) -> int64_t {
    PyObject *o = item(dict, name);
    bool ok = o != nullptr;
    const int64_t n = ok ? whole_number(o, ok) : 0;
    return ok ? n : -2;
  };
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject *m = in.next();
    const int64_t want_out = in.integer(), want_in = in.integer();
    bool fits = in.ok && (PyObject *)Py_TYPE(m) == linear;
    PyObject **dict_at = fits ? _PyObject_GetDictPtr(m) : nullptr;
    PyObject *dict = dict_at ? *dict_at : nullptr;
    PyObject *h = item(dict, hooks), *p = item(dict, pre_hooks), *params = item(dict, parameters);
    PyObject *w = item(params, weight_name), *b = item(params, bias_name);
    fits = fits && h && p && PyDict_Check(h) && PyDict_Check(p) && PyDict_Size(h) == 0 && PyDict_Size(p) == 0 &&
           !item(dict, forward) && w && b == Py_None;
    const at::Tensor *t = fits ? tensor_of(w) : nullptr;
    if (t) {
      const int64_t rows = features(dict, out_name), cols = features(dict, in_name);
      const int64_t row_bytes = cols * (int64_t)x->element_size();
      fits = like(*t, *x) && aligned(*t) && is_shape(*t, {rows, cols}) && (want_out < 0 || want_out == rows) &&
             (want_in < 0 || want_in == cols) && row_bytes % 16 == 0 && row_bytes <= longest;
    }
    if (!t || !fits) {
      Py_DECREF(weights);
      Py_RETURN_NONE;
    }
    Py_INCREF(w);
    PyTuple_SET_ITEM(weights, i, w);
  }
  return weights;
  END_HANDLE_TH_ERRORS
}

// qkv_rope(x, norm_weight, eps, wq, wk, wv, n_heads, n_kv_heads, head_dim, rope_row, stream) -> (q, k, v); the
// operands are checked.
PyObject *qkv_rope(PyObject *, PyObject *const *argv, Py_ssize_t argc) {
  HANDLE_TH_ERRORS
  Args in{argv, argc};
  const at::Tensor *x = in.tensor(), *norm = in.tensor();
  const double eps = in.number();
  const at::Tensor *wq = in.tensor(), *wk = in.tensor(), *wv = in.tensor();
  const int64_t Hq = in.integer(), H = in.integer(), D = in.integer();
  const at::Tensor *rope = in.tensor();
  void *stream = in.pointer();
  if (!in.ok) return PyErr_Format(PyExc_TypeError, "qkv_rope: bad argument");
  at::Tensor q = empty_like({1, 1, Hq, D}, *x), k = empty_like({1, 1, H, D}, *x), v = empty_like({1, 1, H, D}, *x);
  const int rc = unlocked([&] {
    return da_linear_qkv_rope(x->data_ptr(), norm->data_ptr(), (float)eps, (int)x->size(-1), wq->data_ptr(),
                              wk->data_ptr(), wv->data_ptr(), (int)Hq, (int)H, (int)D,
                              (const float *)rope->data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                              dtype_code(*x), stream);
  });
  if (rc) return raise(rc, "da_linear_qkv_rope");
  return tuple_of({wrap(std::move(q)), wrap(std::move(k)), wrap(std::move(v))});
  END_HANDLE_TH_ERRORS
}

// block_tail(attended, wo, x, norm_weight, eps, w1, w3, w2, stream) -> the block's output; the operands
// are checked.
PyObject *block_tail(PyObject *, PyObject *const *argv, Py_ssize_t argc) {
  HANDLE_TH_ERRORS
  Args in{argv, argc};
  const at::Tensor *attended = in.tensor(), *wo = in.tensor(), *x = in.tensor(), *norm = in.tensor();
  const double eps = in.number();
  const at::Tensor *w1 = in.tensor(), *w3 = in.tensor(), *w2 = in.tensor();
  void *stream = in.pointer();
  if (!in.ok) return PyErr_Format(PyExc_TypeError, "block_tail: bad argument");
  const int64_t dim = w2->size(0), hidden = w2->size(1);
  at::Tensor room = empty_like({dim + hidden}, *x), out = empty_like(x->sizes(), *x);
  char *h = (char *)room.data_ptr();
  const int rc = unlocked([&] {
    return da_linear_block_tail(attended->data_ptr(), (int)wo->size(1), wo->data_ptr(), x->data_ptr(), (int)dim,
                                norm->data_ptr(), (float)eps, w1->data_ptr(), w3->data_ptr(), (int)hidden,
                                w2->data_ptr(), h, h + dim * x->element_size(), out.data_ptr(), dtype_code(*x),
                                stream);
  });
  if (rc) return raise(rc, "da_linear_block_tail");
  return wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// ---- a batch of sequences in HBM --------------------------------------------------------------

const at::Tensor &plain(PyObject *o, const char *name) {
  const at::Tensor *t = tensor_of(o);
  TORCH_CHECK_TYPE(t != nullptr, name, " must be a plain torch.Tensor (got ", Py_TYPE(o)->tp_name, ")");
  TORCH_CHECK_VALUE(!t->is_neg() && !t->_is_zerotensor(), name, " is a lazy view: resolve it first");
  // (the kernels count heads, channels and pages in 32 bits; tokens in 64 or refused by them)
  for (int64_t d = t->dim() - 2; d < t->dim(); ++d)
    TORCH_CHECK_VALUE(d < 0 || t->size(d) <= 0x7fffffff, name, " of ", t->sizes(), " is too large");
  return *t;
}
const at::Tensor *plain_or_none(PyObject *o, const char *name) { return o == Py_None ? nullptr : &plain(o, name); }

int float_type(const at::Tensor &t, const char *name) {
  const int code = dtype_code(t);
  TORCH_CHECK_TYPE(code >= 0, name, " must be float32, float16 or bfloat16 (got ", t.scalar_type(), ")");
  return code;
}
int page_type(const at::Tensor &pages, const at::Tensor &x) {
  if (pages.scalar_type() == at::kFloat8_e4m3fn) {
    TORCH_CHECK_TYPE(x.scalar_type() != at::kFloat, "8-bit pages go with 16-bit queries and keys (got float32)");
    return DA_E4M3;
  }
  TORCH_CHECK_TYPE(pages.scalar_type() == x.scalar_type(), "pages of ", pages.scalar_type(), " do not go with ",
                   x.scalar_type(), " (the same type, or float8_e4m3fn)");
  return dtype_code(pages);
}
int whole_type(const at::Tensor &t, const char *name) {
  TORCH_CHECK_TYPE(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong, name, " must be int32 or int64 (got ",
                   t.scalar_type(), ")");
  return t.scalar_type() == at::kLong ? DA_I64 : DA_I32;
}
void on_device_of(const at::Tensor &x, std::initializer_list<std::pair<const at::Tensor *, const char *>> others) {
  for (const auto &o : others)
    if (o.first)
      TORCH_CHECK(o.first->device() == x.device(), o.second, " is on ", o.first->device(), ", the rows on ", x.device());
  TORCH_CHECK(x.is_cuda(), "the operands must live on a GPU: the HIP kernels are the only implementation (got device ",
              x.device(), ")");
}
void not_for_gradients(std::initializer_list<const at::Tensor *> all, const char *what) {
  if (at::GradMode::is_enabled())
    for (const at::Tensor *t : all)
      TORCH_CHECK(!t || !t->requires_grad(), what, " has no gradient: call it under torch.no_grad()");
}
// A dual tensor's tangent is no operand of the kernels: refused where forward mode is on, under torch.no_grad too.
void not_forward_mode(const char *what) {
  TORCH_CHECK(!torch::autograd::ForwardADLevel::try_get_by_idx(0), what, " has no forward-mode derivative");
}
// A tracer would write down the outputs' allocation and nothing else: its program would return memory as it was.
// (Dispatch modes that count, log or keep operators are no tracers: what a call returns under them is right.)
void not_traced(const char *what) {
  using namespace c10::impl;
  TORCH_CHECK(!at::tracer::impl::is_dispatch_enabled() &&                              // torch.jit.trace
                  !TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::PROXY) &&      // make_fx
                  !tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch),        // make_fx ahead of autograd
              what, " cannot be traced: a tracer sees none of its kernels");
}
// What a call writes into, autograd knows as changed.
void changed(const at::Tensor &t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
int64_t stride_of(const at::Tensor &t, int64_t d) { return t.size(d) > 1 ? t.stride(d) : 0; }
bool dense_rows(const at::Tensor &t) { return t.size(-1) <= 1 || t.stride(-1) == 1; }
// What indices add to an address, axis by axis from the longest stride to the shortest, in bytes.
struct Axis {
  int64_t stride, least, most;   // least and largest index, or difference of two tensors' indices
};
using Axes = c10::SmallVector<Axis, 8>;
constexpr int kMostLookedAt = 4096;
void longest_first(Axes &axes) {
  std::sort(axes.begin(), axes.end(), [](const Axis &x, const Axis &y) { return x.stride > y.stride; });
}
// Whether differences of indices make up for `apart` bytes, up to less than an element (`moved`: one of them is not 0).
// One or two an axis are looked at, those that the shorter strides can still make up for, or more where strides are
// shorter than what lies within them: `budget` at the most, behind which tensors are taken to be apart.
bool made_up(const Axis *axes, size_t n, int64_t apart, int64_t element, bool moved, int &budget) {
  if (n == 0) return moved && std::abs(apart) < element;
  int64_t low = 1 - element, high = element - 1;
  for (size_t i = 1; i < n; ++i) low -= axes[i].stride * axes[i].most, high -= axes[i].stride * axes[i].least;
  auto floored = [](int64_t x, int64_t d) { return x / d - (x % d < 0); };
  const int64_t s = axes[0].stride, first = std::max(axes[0].least, -floored(apart - low, s)),
                last = std::min(axes[0].most, floored(high - apart, s));
  for (int64_t by = first; by <= last && --budget >= 0; ++by)
    if (made_up(axes + 1, n - 1, apart + by * s, element, moved || by != 0, budget)) return true;
  return false;
}
// Whether two tensors of one type and number of axes have a byte in common, at other indices if not `anywhere`.
bool meet(const at::Tensor &a, const at::Tensor &b, bool anywhere = true) {
  if (a.numel() == 0 || b.numel() == 0 || a.is_meta() || b.is_meta()) return false;
  const int64_t e = a.element_size();
  Axes axes;
  for (int64_t d = 0; d < a.dim(); ++d) {
    const int64_t as = a.size(d) > 1 ? a.stride(d) * e : 0, bs = b.size(d) > 1 ? b.stride(d) * e : 0;
    if (as == bs || as == 0 || bs == 0) {
      if (as + bs > 0) axes.push_back({std::max(as, bs), as ? 1 - a.size(d) : 0, bs ? b.size(d) - 1 : 0});
    } else {
      axes.push_back({as, 1 - a.size(d), 0});
      axes.push_back({bs, 0, b.size(d) - 1});
    }
  }
  longest_first(axes);
  int budget = kMostLookedAt;
  return made_up(axes.data(), axes.size(), (const char *)b.data_ptr() - (const char *)a.data_ptr(), e, anywhere, budget);
}
// Whether elements of a tensor share memory.
bool folds(const at::Tensor &t) { return at::has_internal_overlap(t) == at::MemOverlap::Yes || meet(t, t, false); }
// Whether a tensor has a byte in memory of `length` bytes that its first element is `at` bytes behind, in the same way.
bool reached(const Axis *axes, size_t n, int64_t at, int64_t element, int64_t length, int &budget) {
  int64_t within = element - 1;   // (to the last byte, behind the axes from the second on)
  for (size_t i = 1; i < n; ++i) within += axes[i].stride * axes[i].most;
  const int64_t end = at + within + (n ? axes[0].stride * axes[0].most : 0);
  if (end < 0 || at >= length) return false;
  if (n == 0 || at >= 0 || end < length) return true;   // (its first or last byte is there)
  const int64_t s = axes[0].stride, first = std::max<int64_t>(0, (-within - at + s - 1) / s),
                last = std::min(axes[0].most, (length - 1 - at) / s);
  for (int64_t by = first; by <= last && --budget >= 0; ++by)
    if (reached(axes + 1, n - 1, at + by * s, element, length, budget)) return true;
  return false;
}
bool reaches(const at::Tensor &t, const at::Tensor &memory) {   // (`memory` is contiguous)
  if (t.numel() == 0 || memory.numel() == 0 || t.is_meta() || memory.is_meta()) return false;
  const int64_t at = (const char *)t.data_ptr() - (const char *)memory.data_ptr(), length = memory.nbytes();
  int64_t extent = t.element_size();
  for (int64_t d = 0; d < t.dim(); ++d) extent += (t.size(d) - 1) * t.stride(d) * (int64_t)t.element_size();
  if (at >= length || at + extent <= 0) return false;
  Axes axes;
  for (int64_t d = 0; d < t.dim(); ++d)
    if (t.size(d) > 1 && t.stride(d) > 0) axes.push_back({t.stride(d) * (int64_t)t.element_size(), 0, t.size(d) - 1});
  longest_first(axes);
  int budget = kMostLookedAt;
  return reached(axes.data(), axes.size(), at, t.element_size(), length, budget);
}
// Rows as the kernels read them: the last axis dense, and where `vectors` 16-byte aligned.  (A gradient may be a lazy
// view of what its memory holds.)
at::Tensor rows_of(const at::Tensor &t, bool vectors) {
  if (t.is_neg() || t._is_zerotensor()) {
    const Released others;
    return t.is_neg() ? t.resolve_neg().contiguous() : at::zeros(t.sizes(), t.options().requires_grad(false));
  }
  bool fits = dense_rows(t);
  if (vectors) {
    fits = fits && aligned(t);
    for (int64_t d = 0; d + 1 < t.dim(); ++d) fits = fits && stride_of(t, d) * (int64_t)t.element_size() % 16 == 0;
  }
  if (fits) return t;
  const Released others;
  return t.clone(at::MemoryFormat::Contiguous);
}
at::Tensor in_line(const at::Tensor &t) {   // a one-dimensional operand
  if (t.is_contiguous()) return t;
  const Released others;
  return t.contiguous();
}

void *stream_of(const at::Tensor &t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

// A leaf that an eager graph holds has the place where its gradient arrives on that graph's stream: a backward pass
// that is captured would lead there, out of the capture, and take the process down.  Refused while it is harmless.
void no_eager_graph_of(const at::Tensor &t) {
  if (!t.defined() || !t.requires_grad() || !t.is_leaf()) return;
  const auto arrival = torch::autograd::impl::try_get_grad_accumulator(t);
  // (By number: torch's graphs call the device cuda, c10::hip calls it hip.)
  if (!arrival || !arrival->stream() || arrival->stream()->id() == c10::hip::getCurrentHIPStream(t.device().index()).id())
    return;
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  const hipError_t rc = hipStreamIsCapturing((hipStream_t)stream_of(t), &status);
  TORCH_CHECK(rc == hipSuccess && status == hipStreamCaptureStatusNone,
              "a leaf of this captured call is still held by an eager graph: drop that graph's results first, or capture "
              "under torch.no_grad()");
}

// How a call turns channels: frequencies (or none), layout, factor.
struct Turn {
  const at::Tensor *freqs;
  bool half;
  double factor;
};
Turn read_turn(Args &in, int64_t head_dim) {
  Turn t = {plain_or_none(in.next(), "freqs"), in.integer() != 0, in.number()};
  TORCH_CHECK_TYPE(in.ok, "factor must be a number");
  if (t.freqs) {
    TORCH_CHECK_TYPE(t.freqs->scalar_type() == at::kDouble, "freqs must be float64 (got ", t.freqs->scalar_type(), ")");
    TORCH_CHECK_VALUE(t.freqs->dim() == 1 && t.freqs->is_contiguous(), "freqs must be one contiguous row");
    TORCH_CHECK_VALUE(2 * t.freqs->numel() <= head_dim, t.freqs->numel(), " frequencies turn ", 2 * t.freqs->numel(),
                      " channels, but heads have ", head_dim);
    TORCH_CHECK_VALUE(t.freqs->numel() <= 256, "up to 256 frequencies (got ", t.freqs->numel(), ")");
    TORCH_CHECK(!at::GradMode::is_enabled() || !t.freqs->requires_grad(), "frequencies have no gradient");
  }
  return t;
}

// xq and, if defined, xk turned by their positions: new tensors, or the same ones `in_place`.
struct Pair {
  at::Tensor q, k;
};
Pair turn_rows(const at::Tensor &xq, const at::Tensor &xk, const at::Tensor &positions, const Turn &turn, bool inverse,
               bool in_place) {
  const bool both = xk.defined();
  const int64_t dims = xq.dim(), tok = dims - 3, D = xq.size(-1), S = xq.size(tok), B = dims == 4 ? xq.size(0) : 1;
  const bool shared = positions.dim() == 1;
  const c10::DeviceGuard guard(xq.device());
  const at::Tensor q = in_place ? xq : rows_of(xq, false), k = !both || in_place ? xk : rows_of(xk, false);
  at::Tensor yq = in_place ? xq : empty_like(xq.sizes(), xq), yk;
  if (both) yk = in_place ? xk : empty_like(xk.sizes(), xk);
  da_rotate_args a = {};
  auto strides = [&](const at::Tensor &t, int64_t *to) {
    to[0] = dims == 4 ? stride_of(t, 0) : 0;
    to[1] = stride_of(t, tok);
    to[2] = stride_of(t, tok + 1);
  };
  a.q = q.data_ptr();
  a.q_out = yq.data_ptr();
  strides(q, a.q_strides);
  strides(yq, a.q_out_strides);
  a.n_q_heads = (int32_t)q.size(tok + 1);
  if (both) {
    a.k = k.data_ptr();
    a.k_out = yk.data_ptr();
    strides(k, a.k_strides);
    strides(yk, a.k_out_strides);
    a.n_k_heads = (int32_t)k.size(tok + 1);
  }
  a.freqs = (const double *)turn.freqs->data_ptr();
  a.positions = positions.data_ptr();
  a.position_strides[0] = shared ? 0 : stride_of(positions, 0);
  a.position_strides[1] = stride_of(positions, positions.dim() - 1);
  a.batch = B;
  a.tokens = S;
  a.head_dim = (int32_t)D;
  a.rotary_dim = (int32_t)(2 * turn.freqs->numel());
  a.layout = turn.half ? DA_ROTARY_HALF : DA_ROTARY_INTERLEAVED;
  a.inverse = inverse;
  a.dtype = dtype_code(q);
  a.position_type = whole_type(positions, "positions");
  a.factor = (float)turn.factor;
  void *stream = stream_of(xq);
  const int rc = unlocked([&] { return da_rotate(&a, sizeof(a), stream); });
  TORCH_CHECK(rc == 0, "da_rotate failed (code ", rc, "): ", da_last_error_string());
  if (in_place) {
    changed(yq);
    if (both) changed(yk);
  }
  return {std::move(yq), std::move(yk)};
}

// The gradient of a turn is the turn back of the gradient (the matrix is orthogonal but for the factor, which stays),
// by the same function, so that it has a gradient itself.  As a function of C++ a call costs the host 20 us less
// than as one of Python.
struct Turned : torch::autograd::Function<Turned> {
  using Context = torch::autograd::AutogradContext;
  using Variables = torch::autograd::variable_list;

  static Variables forward(Context *ctx, const at::Tensor &q, const std::optional<at::Tensor> &k,
                           const at::Tensor &positions, const at::Tensor &freqs, bool half, double factor,
                           bool inverse) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({positions, freqs});
    ctx->saved_data["how"] = (int64_t)(half | inverse << 1 | (int)k.has_value() << 2);
    ctx->saved_data["factor"] = factor;
    Pair y = turn_rows(q, k ? *k : at::Tensor(), positions, {&freqs, half, factor}, inverse, false);
    // (each output wants a gradient if its own input does)
    if (k && !q.requires_grad()) ctx->mark_non_differentiable({y.q});
    if (k && !k->requires_grad()) ctx->mark_non_differentiable({y.k});
    return k ? Variables{y.q, y.k} : Variables{y.q};
  }

  static Variables backward(Context *ctx, Variables grads) {
    // (gradients without a tangent are taken where forward mode is on for something else)
    for (const at::Tensor &g : grads)
      TORCH_CHECK(!g.defined() || !g._fw_grad(0).defined(), "rotate's gradient has no forward-mode derivative");
    not_traced("rotate's gradient");
    const Variables saved = ctx->get_saved_variables();
    const int64_t how = ctx->saved_data["how"].toInt();
    const double factor = ctx->saved_data["factor"].toDouble();
    const bool half = how & 1, inverse = !(how & 2);
    at::Tensor g[2];
    for (size_t i = 0; i < grads.size(); ++i)
      if (ctx->needs_input_grad(i)) g[i] = grads[i];
    auto turn = [&](const at::Tensor &q, const at::Tensor &k) -> Pair {
      if (!at::GradMode::is_enabled()) return turn_rows(q, k, saved[0], {&saved[1], half, factor}, inverse, false);
      Variables y = apply(q, k.defined() ? std::optional<at::Tensor>(k) : std::nullopt, saved[0], saved[1], half, factor,
                          inverse);
      return {y[0], y.size() > 1 ? y[1] : at::Tensor()};
    };
    Pair d;
    if (g[0].defined())
      d = turn(g[0], g[1]);
    else if (g[1].defined())
      d.k = turn(g[1], at::Tensor()).q;
    return {d.q, d.k, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

// rotate(xq, xk, positions, freqs, half, factor, in_place) -> (yq, yk), with gradients unless in place; xk and yk may
// be None.
PyObject *rotate(PyObject *, PyObject *const *argv, Py_ssize_t argc) {
  HANDLE_TH_ERRORS
  Args in{argv, argc};
  const at::Tensor &xq = plain(in.next(), "xq"), *xk = plain_or_none(in.next(), "xk");
  const at::Tensor &positions = plain(in.next(), "positions");
  float_type(xq, "xq");
  const int64_t dims = xq.dim();
  TORCH_CHECK_VALUE(dims == 3 || dims == 4, "xq must be (tokens, heads, head_dim) or (batch, tokens, heads, head_dim)");
  const int64_t D = xq.size(-1), S = xq.size(dims - 3), B = dims == 4 ? xq.size(0) : 1;
  TORCH_CHECK_VALUE(D > 0, "heads without channels");
  const Turn turn = read_turn(in, D);
  TORCH_CHECK_TYPE(turn.freqs != nullptr, "freqs must be a tensor");
  const bool in_place = in.integer() != 0;
  TORCH_CHECK_TYPE(in.ok, "rotate: bad argument");
  not_forward_mode(in_place ? "rotate_" : "rotate");
  not_traced(in_place ? "rotate_" : "rotate");
  if (xk) {
    TORCH_CHECK_TYPE(xk->scalar_type() == xq.scalar_type(), "xk is ", xk->scalar_type(), " but xq is ", xq.scalar_type());
    TORCH_CHECK_VALUE(xk->dim() == dims && xk->size(-1) == D && xk->size(dims - 3) == S && (dims == 3 || xk->size(0) == B),
                      "xk ", xk->sizes(), " does not go with xq ", xq.sizes());
  }
  whole_type(positions, "positions");
  TORCH_CHECK_VALUE(positions.dim() == 1 ? positions.size(0) == S
                                         : dims == 4 && positions.dim() == 2 && positions.size(0) == B &&
                                               positions.size(1) == S,
                    "positions ", positions.sizes(), " do not go with xq ", xq.sizes());
  on_device_of(xq, {{xk, "xk"}, {&positions, "positions"}, {turn.freqs, "freqs"}});
  Pair y;
  if (in_place) {
    not_for_gradients({&xq, xk}, "rotate_");
    for (const at::Tensor *t : {&xq, xk}) {
      if (!t) continue;
      TORCH_CHECK_VALUE(dense_rows(*t) && !folds(*t),
                        "what is turned in place must have dense rows that do not share memory");
    }
    TORCH_CHECK_VALUE(!xk || !meet(xq, *xk), "xq and xk share memory");
    y = turn_rows(xq, xk ? *xk : at::Tensor(), positions, turn, false, true);
  } else if (at::GradMode::is_enabled() && (xq.requires_grad() || (xk && xk->requires_grad()))) {
    no_eager_graph_of(xq);
    if (xk) no_eager_graph_of(*xk);
    auto out = Turned::apply(xq, xk ? std::optional<at::Tensor>(*xk) : std::nullopt, positions, *turn.freqs, turn.half,
                             turn.factor, false);
    y = {out[0], xk ? out[1] : at::Tensor()};
  } else {
    y = turn_rows(xq, xk ? *xk : at::Tensor(), positions, turn, false, false);
  }
  PyObject *second = Py_None;
  if (xk)
    second = wrap(std::move(y.k));
  else
    Py_INCREF(second);
  return tuple_of({wrap(std::move(y.q)), second});
  END_HANDLE_TH_ERRORS
}

// What both calls on a paged cache look at: the pools and the table.
struct Pages {
  const at::Tensor &k, &v, &table;
  int type;
};
Pages read_pages(Args &in, const at::Tensor &x) {
  const at::Tensor &k = plain(in.next(), "k_pages"), &v = plain(in.next(), "v_pages"), &table = plain(in.next(), "page_table");
  TORCH_CHECK_VALUE(k.dim() == 4 && k.sizes() == v.sizes(), "k_pages ", k.sizes(), " and v_pages ", v.sizes(),
                    " must both be (pages, page_size, kv heads, head_dim)");
  TORCH_CHECK_TYPE(k.scalar_type() == v.scalar_type(), "k_pages is ", k.scalar_type(), " but v_pages is ", v.scalar_type());
  const int type = page_type(k, x);
  TORCH_CHECK_VALUE(k.size(1) > 0 && k.size(2) > 0, "pages without tokens or heads");
  TORCH_CHECK_VALUE(dense_rows(k) && dense_rows(v), "head_dim must be the dense axis of the pages");
  for (int64_t d = 0; d < 3; ++d)
    TORCH_CHECK_VALUE(stride_of(k, d) == stride_of(v, d), "k_pages and v_pages must have the same strides");
  for (int64_t d = 0; d < 4; ++d) TORCH_CHECK_VALUE(k.size(d) <= 0x7fffffff, "pages ", k.sizes(), " are too many");
  whole_type(table, "page_table");
  TORCH_CHECK_VALUE(table.dim() == 2 && dense_rows(table) && table.size(0) <= 0x7fffffff && table.size(1) <= 0x7fffffff,
                    "page_table must be (sequences, pages) with dense rows");
  return {k, v, table, type};
}
template <typename A>
void give_pages(A &a, const Pages &p) {
  for (int d = 0; d < 3; ++d) a.page_strides[d] = stride_of(p.k, d);
  a.page_table = p.table.data_ptr();
  a.table_stride = stride_of(p.table, 0);
  a.table_type = whole_type(p.table, "page_table");
  a.n_pages = (int32_t)p.k.size(0);
  a.page_size = (int32_t)p.k.size(1);
  a.n_sequences = (int32_t)p.table.size(0);
  a.pages_per_sequence = (int32_t)p.table.size(1);
  a.n_kv_heads = (int32_t)p.k.size(2);
  a.head_dim = (int32_t)p.k.size(3);
  a.page_dtype = p.type;
}
const at::Tensor *read_scale(PyObject *o, const char *name, const Pages &p) {
  const at::Tensor *t = plain_or_none(o, name);
  if (t) {
    TORCH_CHECK_VALUE(p.type == DA_E4M3, name, " is for 8-bit pages (these are ", p.k.scalar_type(), ")");
    TORCH_CHECK_TYPE(t->scalar_type() == at::kFloat, name, " must be float32 (got ", t->scalar_type(), ")");
    TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == p.k.size(2) && t->is_contiguous(), name,
                      " must hold one number per kv head");
  }
  return t;
}
const float *numbers(const at::Tensor *t) { return t ? (const float *)t->data_ptr() : nullptr; }

// paged_append(xk, xv, k_pages, v_pages, page_table, positions, sequences, xq, freqs, half, factor, k_scale, v_scale) ->
// the turned queries, or None without any.
PyObject *paged_append(PyObject *, PyObject *const *argv, Py_ssize_t argc) {
  HANDLE_TH_ERRORS
  Args in{argv, argc};
  const at::Tensor &xk = plain(in.next(), "xk"), &xv = plain(in.next(), "xv");
  const int dtype = float_type(xk, "xk");
  const Pages pages = read_pages(in, xk);
  const at::Tensor &positions = plain(in.next(), "positions"), *sequences = plain_or_none(in.next(), "sequences");
  const at::Tensor *xq = plain_or_none(in.next(), "xq");
  const int64_t H = pages.k.size(2), D = pages.k.size(3);
  const Turn turn = read_turn(in, D);
  const at::Tensor *k_scale = read_scale(in.next(), "k_scale", pages), *v_scale = read_scale(in.next(), "v_scale", pages);
  TORCH_CHECK_TYPE(in.ok, "append_kv_pages_: bad argument");
  not_forward_mode("append_kv_pages_");
  not_traced("append_kv_pages_");
  TORCH_CHECK_VALUE(xk.dim() == 3 && xk.size(1) == H && xk.size(2) == D && xv.sizes() == xk.sizes(), "xk ", xk.sizes(),
                    " and xv ", xv.sizes(), " must both be (tokens, ", H, ", ", D, ") as the pages are");
  const int64_t T = xk.size(0);
  TORCH_CHECK_TYPE(xv.scalar_type() == xk.scalar_type(), "xv is ", xv.scalar_type(), " but xk is ", xk.scalar_type());
  if (xq) {
    TORCH_CHECK_TYPE(xq->scalar_type() == xk.scalar_type(), "xq is ", xq->scalar_type(), " but xk is ", xk.scalar_type());
    TORCH_CHECK_VALUE(xq->dim() == 3 && xq->size(0) == T && xq->size(2) == D, "xq ", xq->sizes(), " does not go with xk ",
                      xk.sizes());
  }
  const int position_type = whole_type(positions, "positions");
  const int sequence_type = sequences ? whole_type(*sequences, "sequences") : DA_I32;
  TORCH_CHECK_VALUE(positions.dim() == 1 && positions.size(0) == T, "positions ", positions.sizes(), " do not go with ", T,
                    " tokens");
  TORCH_CHECK_VALUE(!sequences || (sequences->dim() == 1 && sequences->size(0) == T), "sequences must name one for each of ",
                    T, " tokens");
  TORCH_CHECK_VALUE(sequences || T == pages.table.size(0), T, " tokens for the ", pages.table.size(0),
                    " sequences of the table: say which with sequences=");
  not_for_gradients({&xk, &xv, xq, &pages.k, &pages.v, k_scale, v_scale}, "append_kv_pages_");
  for (const at::Tensor *t : {&pages.k, &pages.v})
    TORCH_CHECK_VALUE(!folds(*t), "pages must not share memory");
  TORCH_CHECK_VALUE(!meet(pages.k, pages.v), "k_pages and v_pages share memory");
  on_device_of(xk, {{&xv, "xv"}, {&pages.k, "k_pages"}, {&pages.v, "v_pages"}, {&pages.table, "page_table"},
                    {&positions, "positions"}, {sequences, "sequences"}, {xq, "xq"}, {turn.freqs, "freqs"},
                    {k_scale, "k_scale"}, {v_scale, "v_scale"}});
  const c10::DeviceGuard guard(xk.device());
  const at::Tensor k = rows_of(xk, false), v = rows_of(xv, false), q = xq ? rows_of(*xq, false) : at::Tensor();
  const at::Tensor at_positions = in_line(positions), of = sequences ? in_line(*sequences) : at::Tensor();
  at::Tensor out;
  if (xq) out = empty_like(xq->sizes(), *xq);
  da_paged_append_args a = {};
  give_pages(a, pages);
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.k_pages = pages.k.data_ptr();
  a.v_pages = pages.v.data_ptr();
  a.positions = at_positions.data_ptr();
  a.sequences = sequences ? of.data_ptr() : nullptr;
  a.k_scale = numbers(k_scale);
  a.v_scale = numbers(v_scale);
  for (int d = 0; d < 2; ++d) {
    a.k_strides[d] = stride_of(k, d);
    a.v_strides[d] = stride_of(v, d);
    if (xq) {
      a.q_strides[d] = stride_of(q, d);
      a.q_out_strides[d] = stride_of(out, d);
    }
  }
  if (xq) {
    a.q = q.data_ptr();
    a.q_out = out.data_ptr();
    a.n_q_heads = (int32_t)q.size(1);
  }
  if (turn.freqs) {
    a.freqs = (const double *)turn.freqs->data_ptr();
    a.rotary_dim = (int32_t)(2 * turn.freqs->numel());
  }
  a.n_tokens = T;
  a.layout = turn.half ? DA_ROTARY_HALF : DA_ROTARY_INTERLEAVED;
  a.dtype = dtype;
  a.position_type = position_type;
  a.sequence_type = sequence_type;
  a.factor = (float)turn.factor;
  void *stream = stream_of(xk);
  const int rc = unlocked([&] { return da_paged_append(&a, sizeof(a), stream); });
  if (rc) return raise(rc, "da_paged_append");
  changed(pages.k);
  changed(pages.v);
  if (!xq) Py_RETURN_NONE;
  return wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// paged_attention(xq, k_pages, v_pages, page_table, lengths, scale, k_scale, v_scale, out, lse) -> output; scale, scales,
// out and lse may be None.
PyObject *paged_attention(PyObject *, PyObject *const *argv, Py_ssize_t argc) {
  HANDLE_TH_ERRORS
  Args in{argv, argc};
  const at::Tensor &xq = plain(in.next(), "xq");
  const int dtype = float_type(xq, "xq");
  const Pages pages = read_pages(in, xq);
  const at::Tensor &lengths = plain(in.next(), "lengths");
  const int64_t B = pages.table.size(0), H = pages.k.size(2), D = pages.k.size(3);
  PyObject *scale_at = in.next();
  double scale = 1.0 / std::sqrt((double)D);
  if (scale_at != Py_None) {
    scale = PyFloat_AsDouble(scale_at);
    if (scale == -1.0 && PyErr_Occurred()) return nullptr;
    // (the kernels have it in fp32, times log2 e)
    TORCH_CHECK_VALUE(std::isfinite((float)scale * 1.4426950408889634f), "scale must be finite in fp32 (got ", scale, ")");
  }
  const at::Tensor *k_scale = read_scale(in.next(), "k_scale", pages), *v_scale = read_scale(in.next(), "v_scale", pages);
  const at::Tensor *out_given = plain_or_none(in.next(), "out"), *lse = plain_or_none(in.next(), "lse");
  TORCH_CHECK_TYPE(in.ok, "paged_decode_attention: bad argument");
  not_forward_mode("paged_decode_attention");
  not_traced("paged_decode_attention");
  TORCH_CHECK_VALUE(xq.dim() == 3 && xq.size(0) == B && xq.size(2) == D && xq.size(1) > 0 && xq.size(1) % H == 0, "xq ",
                    xq.sizes(), " must be (", B, " sequences, a multiple of ", H, " heads, ", D, ")");
  const int64_t Hq = xq.size(1);
  const int length_type = whole_type(lengths, "lengths");
  TORCH_CHECK_VALUE(lengths.dim() == 1 && lengths.size(0) == B, "lengths must hold one for each of ", B, " sequences");
  if (out_given)
    TORCH_CHECK_VALUE(out_given->sizes() == xq.sizes() && out_given->scalar_type() == xq.scalar_type() &&
                          out_given->is_contiguous() && aligned(*out_given),
                      "out must be contiguous, 16-byte aligned and of xq's shape and type");
  if (lse)
    TORCH_CHECK_VALUE(lse->scalar_type() == at::kFloat && is_shape(*lse, {B, Hq}) && lse->is_contiguous(),
                      "lse must be contiguous float32 of shape (sequences, heads)");
  not_for_gradients({&xq, &pages.k, &pages.v, k_scale, v_scale, out_given, lse}, "paged_decode_attention");
  // (a workgroup has a sequence's queries before it writes there, or the launch behind writes: out may be xq itself)
  for (const at::Tensor *to : {out_given, lse})
    for (const at::Tensor *from : {&xq, &pages.k, &pages.v, &pages.table, &lengths, k_scale, v_scale, lse})
      TORCH_CHECK_VALUE(!to || !from || from == to || !reaches(*from, *to) ||
                            (to == out_given && from == &xq && xq.data_ptr() == to->data_ptr() && xq.is_contiguous()),
                        to == lse ? "lse" : "out", " shares memory with another operand");
  on_device_of(xq, {{&pages.k, "k_pages"}, {&pages.v, "v_pages"}, {&pages.table, "page_table"}, {&lengths, "lengths"},
                    {k_scale, "k_scale"}, {v_scale, "v_scale"}, {out_given, "out"}, {lse, "lse"}});
  const c10::DeviceGuard guard(xq.device());
  const at::Tensor q = rows_of(xq, true), lens = in_line(lengths);
  at::Tensor out = out_given ? *out_given : empty_like(xq.sizes(), xq), room;
  da_paged_attention_args a = {};
  give_pages(a, pages);
  a.q = q.data_ptr();
  a.k_pages = pages.k.data_ptr();
  a.v_pages = pages.v.data_ptr();
  a.lengths = lens.data_ptr();
  a.k_scale = numbers(k_scale);
  a.v_scale = numbers(v_scale);
  a.out = out.data_ptr();
  a.lse = lse ? (float *)lse->data_ptr() : nullptr;
  a.q_strides[0] = stride_of(q, 0);
  a.q_strides[1] = stride_of(q, 1);
  a.n_q_heads = (int32_t)Hq;
  a.dtype = dtype;
  a.length_type = length_type;
  a.scale = (float)scale;
  const size_t need = da_paged_attention_workspace_bytes(&a, sizeof(a));
  if (need) {   // (the call's own: freed at its end, which the caching allocator orders behind the launches)
    const Released others;
    room = at::empty({(int64_t)need}, xq.options().dtype(at::kByte).requires_grad(false));
    a.workspace = room.data_ptr();
    a.workspace_bytes = (int64_t)need;
  }
  void *stream = stream_of(xq);
  const int rc = unlocked([&] { return da_paged_attention(&a, sizeof(a), stream); });
  if (rc) return raise(rc, "da_paged_attention");
  if (out_given) changed(out);
  if (lse) changed(*lse);
  return wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

#define DA_CALL(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {DA_CALL(step_args), DA_CALL(static_step), DA_CALL(alike), DA_CALL(linears),
                         DA_CALL(qkv_rope),  DA_CALL(block_tail),  DA_CALL(rotate), DA_CALL(paged_append),
                         DA_CALL(paged_attention), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__host() {
  PyObject *nn = PyImport_ImportModule("torch.nn");
  if (!nn) return nullptr;
  parameter_class = PyObject_GetAttrString(nn, "Parameter");
  Py_DECREF(nn);
  return parameter_class ? PyModule_Create(&module) : nullptr;
}
