// device_ops_torch.cpp -- the operators on device tensors for torch: checks a call's tensors, fills the argument struct of the C ABI, allocates
// what was not given, and calls.  In C++ because a step's calls are shorter than the same checks in Python take (20 to 40 us a call there, 3 to 7
// here).  What each function takes and returns is described in linmt_b200/device_ops.py, which passes its arguments on in order.
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <string>
#include <vector>

#include "../../include/linmt_decoder.h"

namespace {

using at::Tensor;
PyObject* g_error = nullptr;       // linmt_b200.decoder.LinmtError

#define NEED(ok, ...) TORCH_CHECK_VALUE(ok, __VA_ARGS__)

const Tensor& tensor(PyObject* o, const char* name) {
  NEED(THPVariable_Check(o), name, " has to be a CUDA tensor");
  return THPVariable_Unpack(o);
}
const Tensor& on_cuda(PyObject* o, const char* name) {
  const Tensor& t = tensor(o, name);
  NEED(t.is_cuda() && t.layout() == at::kStrided && !t.is_neg(), name, " has to be a CUDA tensor");
  NEED(!t.requires_grad() || !at::GradMode::is_enabled(), name, " requires a gradient, and there is no backward pass: call under torch.no_grad()");
  NEED(!c10::AutogradState::get_tls_state().get_fw_grad_mode() || !t._fw_grad(0).defined(), name, " has a tangent, and there is no derivative: call with the primal (forward_ad.unpack_dual)");
  return t;
}
const Tensor& on_device(PyObject* o, const char* name, int dev) {
  const Tensor& t = on_cuda(o, name);
  NEED(t.get_device() == dev, name, " has to be a tensor on CUDA device ", dev);
  return t;
}
// A contiguous tensor of the given type and shape on the call's device.
const Tensor& dense(PyObject* o, const char* name, int dev, at::ScalarType type, at::IntArrayRef shape) {
  const Tensor& t = on_device(o, name, dev);
  NEED(t.scalar_type() == type, name, " has to be ", type, ", not ", t.scalar_type());
  NEED(t.sizes() == shape, name, " has to have the shape ", shape, ", not ", t.sizes());
  NEED(t.is_contiguous(), name, " has to be contiguous");
  return t;
}
uint8_t* flags(PyObject* o, const char* name, int dev, at::IntArrayRef shape) {
  const Tensor& t = on_device(o, name, dev);
  NEED(t.scalar_type() == at::kBool || t.scalar_type() == at::kByte, name, " has to be a bool or uint8 tensor");
  return static_cast<uint8_t*>(dense(o, name, dev, t.scalar_type(), shape).data_ptr());
}
int dtype_of(const Tensor& t) { return t.scalar_type() == at::kFloat ? LINMT_F32 : t.scalar_type() == at::kBFloat16 ? LINMT_BF16 : t.scalar_type() == at::kHalf ? LINMT_F16 : -1; }
int int32_of(int64_t v, const char* name) {
  NEED(v >= INT32_MIN && v <= INT32_MAX, name, " = ", v, " is too large");
  return (int)v;
}
int64_t integer(PyObject* o, const char* name) {
  PyObject* i = PyNumber_Index(o);
  if (!i) throw python_error();
  const long long v = PyLong_AsLongLong(i);
  Py_DECREF(i);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    NEED(false, name, " is too large");
  }
  return v;
}
double real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}
Tensor make(at::IntArrayRef shape, at::ScalarType type, int dev) { return Tensor(at::detail::empty_cuda(shape, type, c10::Device(at::kCUDA, (c10::DeviceIndex)dev), std::nullopt)); }
void* stream_of(int dev) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream(); }
void done_or_raise(int rc) {
  if (rc == LINMT_OK) return;
  NEED(rc != LINMT_EINVAL && rc != LINMT_ELIMIT, linmt_op_error());
  PyErr_Format(g_error, "%s (%d)", linmt_op_error(), rc);
  throw python_error();
}
void arguments(Py_ssize_t got, Py_ssize_t want) { TORCH_CHECK_TYPE(got == want, "takes ", want, " arguments, got ", got); }
// Two places of a tensor that is written share no memory, as far as strides of 0 say.
bool apart(const Tensor& t) {
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.size(i) > 1 && t.stride(i) == 0) return false;
  return true;
}

// A caller's tensor has been written: autograd finds one that it has saved for a backward pass changed.  (Tensors of the inference mode keep no count.)
void was_written(PyObject* o) {
  const Tensor& t = THPVariable_Unpack(o);
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
// The bytes from a tensor's first to its last.
struct Span { const char *p, *end; };
Span span_of(const Tensor& t) {
  const char* const p = static_cast<const char*>(t.data_ptr());
  if (t.numel() == 0) return {p, p};
  int64_t last = 0;
  for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
  return {p, p + (last + 1) * (int64_t)t.element_size()};
}
// Whether the bytes p .. end - 1 meet elements of `bytes` bytes at `base` and `dims` strides from it, the widest first.
bool meets(const char* base, const int64_t* size, const int64_t* stride, int dims, int64_t bytes, const char* p, const char* end) {
  int64_t extent = bytes;
  for (int i = 0; i < dims; ++i) extent += (size[i] - 1) * stride[i];
  if (end <= base || p >= base + extent) return false;
  if (dims == 0) return true;
  if (extent - (size[0] - 1) * stride[0] > stride[0]) return true;      // (strides that do not nest: as far as can be told)
  const int64_t first = p <= base ? 0 : (p - base) / stride[0], last = std::min((end - 1 - base) / stride[0], size[0] - 1);
  for (int64_t i = first; i <= last; ++i)
    if (i > first && i < last) return true;
    else if (meets(base + i * stride[0], size + 1, stride + 1, dims - 1, bytes, p, end)) return true;
  return false;
}
bool meets(const Tensor& t, const Span& s) {
  const Span all = span_of(t);
  if (t.numel() == 0 || s.p == s.end || all.end <= s.p || s.end <= all.p) return false;
  int64_t size[8], stride[8];
  int dims = 0;
  for (int64_t i = 0; i < t.dim(); ++i) {
    if (t.size(i) == 1) continue;
    if (dims == 8) return true;
    const int64_t by = t.stride(i) * (int64_t)t.element_size();
    int j = dims++;
    for (; j > 0 && stride[j - 1] < by; --j) { size[j] = size[j - 1]; stride[j] = stride[j - 1]; }
    size[j] = t.size(i);
    stride[j] = by;
  }
  return meets(all.p, size, stride, dims, (int64_t)t.element_size(), s.p, s.end);
}
// A tensor that is written while `read` is still read has to lie apart from it, or in the gaps between its places.
void lie_apart(const Tensor& written, const char* name, PyObject* read, const char* of) {
  if (read == Py_None) return;
  const Tensor& r = THPVariable_Unpack(read);
  NEED(!meets(written, span_of(r)) || !meets(r, span_of(written)), name, " overlaps ", of);
}

PyObject* beam_select(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  arguments(n_args, 6);
  const Tensor& logits = on_cuda(a[0], "logits");
  const int dev = logits.get_device();
  NEED(logits.dim() == 3 && dtype_of(logits) >= 0, "logits have to be [n, k, vocab] in float32, bfloat16 or float16");
  const int64_t n = logits.size(0), k = logits.size(1), v = logits.size(2);
  NEED(v >= 1 && (logits.stride(2) == 1 || v == 1), "the words of a row of logits have to be contiguous");
  const int64_t shape[2] = {n, k};
  linmt_beam_select_args g{};
  g.size = sizeof(g);
  g.device = dev;
  g.logits = logits.data_ptr();
  g.stride_n = logits.stride(0);
  g.stride_k = logits.stride(1);
  g.scores = static_cast<const float*>(dense(a[1], "scores", dev, at::kFloat, shape).data_ptr());
  if (a[2] != Py_None) g.done = flags(a[2], "done", dev, shape);
  if (a[3] != Py_None) {
    const Tensor& allowed = on_device(a[3], "allowed", dev);
    const int64_t words = (v + 31) / 32;
    NEED(allowed.dim() == 2 && (allowed.size(0) == 1 || allowed.size(0) == n), "allowed has to be [1 or n, ceil(vocab / 32)]");
    const int64_t want[2] = {allowed.size(0), words};
    g.allowed = static_cast<const uint32_t*>(dense(a[3], "allowed", dev, at::kInt, want).data_ptr());
    g.allowed_stride = allowed.size(0) == 1 ? 0 : words;
  }
  g.n = int32_of(n, "n");
  g.k = int32_of(k, "k");
  g.vocab = int32_of(v, "vocab");
  g.eos = int32_of(integer(a[4], "eos"), "eos");
  g.dtype = dtype_of(logits);
  Tensor t[4];
  if (a[5] == Py_None) {
    t[0] = make(shape, at::kInt, dev);
    t[1] = make(shape, at::kInt, dev);
    t[2] = make(shape, at::kFloat, dev);
    t[3] = make(shape, at::kBool, dev);
  } else {
    NEED(PyTuple_Check(a[5]) && PyTuple_GET_SIZE(a[5]) == 4, "out has to be (tokens, parents, scores, done)");
    t[0] = dense(PyTuple_GET_ITEM(a[5], 0), "out[0]", dev, at::kInt, shape);
    t[1] = dense(PyTuple_GET_ITEM(a[5], 1), "out[1]", dev, at::kInt, shape);
    t[2] = dense(PyTuple_GET_ITEM(a[5], 2), "out[2]", dev, at::kFloat, shape);
    flags(PyTuple_GET_ITEM(a[5], 3), "out[3]", dev, shape);
    t[3] = THPVariable_Unpack(PyTuple_GET_ITEM(a[5], 3));
    // A sentence's results are written while others are still read: each has to lie apart from all that is read, or be it, place for place.
    auto span = [](const void* p, int64_t bytes) { return Span{static_cast<const char*>(p), static_cast<const char*>(p) + bytes}; };
    auto meet = [](const Span& x, const Span& y) { return x.p < y.end && y.p < x.end; };
    const Span outs[4] = {span(t[0].data_ptr(), n * k * 4), span(t[1].data_ptr(), n * k * 4), span(t[2].data_ptr(), n * k * 4), span(t[3].data_ptr(), n * k)};
    const Span reads[4] = {span(g.scores, n * k * 4), span(g.done, g.done ? n * k : 0), span(g.allowed, g.allowed ? (g.allowed_stride ? n : 1) * ((v + 31) / 32) * 4 : 0),
                           span(g.logits, n * k ? ((n - 1) * g.stride_n + (k - 1) * g.stride_k + v) * (int64_t)logits.element_size() : 0)};
    for (int i = 0; i < 4 && n * k; ++i) {
      for (int j = 0; j < i; ++j) NEED(!meet(outs[i], outs[j]), "out[", j, "] and out[", i, "] overlap");
      for (int j = 0; j < 4; ++j) NEED(!meet(outs[i], reads[j]) || (i == j + 2 && outs[i].p == reads[j].p), "out[", i, "] overlaps what the call reads");
    }
  }
  g.out_tokens = static_cast<int32_t*>(t[0].data_ptr());
  g.out_parents = static_cast<int32_t*>(t[1].data_ptr());
  g.out_scores = static_cast<float*>(t[2].data_ptr());
  g.out_done = static_cast<uint8_t*>(t[3].data_ptr());
  if (n) {
    g.stream = stream_of(dev);
    done_or_raise(linmt_beam_select(&g));
  }
  if (a[5] != Py_None) {
    for (int i = 0; i < 4; ++i) was_written(PyTuple_GET_ITEM(a[5], i));
    Py_INCREF(a[5]);
    return a[5];
  }
  PyObject* r = PyTuple_New(4);
  if (!r) throw python_error();
  for (int i = 0; i < 4; ++i) PyTuple_SET_ITEM(r, i, THPVariable_Wrap(std::move(t[i])));
  return r;
  END_HANDLE_TH_ERRORS
}

struct Strides {
  int64_t layers, l, n, k, row;      // in bytes; row: bytes of one
  const char* p;
  const char* end;                   // behind the last byte
};

Strides strides_of(const Tensor& x, int64_t n, int64_t k, const char* what, Py_ssize_t i) {
  const int64_t d = x.dim(), size = x.element_size();
  NEED(d >= 2 && d <= 4, what, "[", i, "] has to be [n, k], [n, k, width] or [layers, n, k, width]");
  const int f = d == 4;
  NEED(x.size(f) == n && x.size(f + 1) == k, what, "[", i, "] has to have the sentences and beams of parents, not ", x.sizes());
  const int64_t width = d == 2 ? 1 : x.size(d - 1);
  NEED(d == 2 || width <= 1 || x.stride(d - 1) == 1, "the rows of ", what, "[", i, "] have to be contiguous");
  Strides s{f ? x.size(0) : 1, f ? x.stride(0) * size : 0, x.stride(f) * size, x.stride(f + 1) * size, width * size, static_cast<const char*>(x.data_ptr()), nullptr};
  s.end = s.p + (s.layers - 1) * s.l + (n - 1) * s.n + (k - 1) * s.k + s.row;
  return s;
}
// Whether two states share no byte, as far as can be told: one lies behind the other, or they are columns of the same rows, whose strides nest.
bool disjoint(const Strides& a, const Strides& b, int64_t n, int64_t k) {
  if (a.end <= b.p || b.end <= a.p) return true;
  const Strides &x = a.p <= b.p ? a : b, &y = a.p <= b.p ? b : a;
  struct Dim { int64_t stride, size; } dims[3];
  int m = 0;
  if (x.layers > 1 || y.layers > 1) {
    if (x.layers != y.layers || x.l != y.l) return false;
    dims[m++] = {x.l, x.layers};
  }
  if (n > 1) {
    if (x.n != y.n) return false;
    dims[m++] = {x.n, n};
  }
  if (k > 1) {
    if (x.k != y.k) return false;
    dims[m++] = {x.k, k};
  }
  std::sort(dims, dims + m, [](const Dim& p, const Dim& q) { return p.stride < q.stride; });
  int64_t room = INT64_MAX, inner = 0;      // the least distance of two rows
  for (int i = 0; i < m; ++i) {
    room = std::min(room, dims[i].stride - inner);
    inner += (dims[i].size - 1) * dims[i].stride;
  }
  const int64_t d = y.p - x.p;
  return d >= x.row && d + y.row <= room;
}

PyObject* beam_reorder(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  arguments(n_args, 3);
  const Tensor& parents = on_cuda(a[1], "parents");
  const int dev = parents.get_device();
  NEED(parents.dim() == 2, "parents have to be [n, k]");
  const int64_t n = parents.size(0), k = parents.size(1);
  dense(a[1], "parents", dev, at::kInt, parents.sizes());
  NEED(PyList_Check(a[0]) && PyList_Check(a[2]) && PyList_GET_SIZE(a[0]) == PyList_GET_SIZE(a[2]), "out has to have a tensor for every state");
  linmt_beam_reorder_args g;
  g.size = sizeof(g);
  g.device = dev;
  g.stream = stream_of(dev);
  g.parents = static_cast<const int32_t*>(parents.data_ptr());
  g.n = int32_of(n, "n");
  g.k = int32_of(k, "k");
  g.reserved = 0;
  const Py_ssize_t all = PyList_GET_SIZE(a[0]);
  std::vector<linmt_beam_state> states;
  std::vector<Strides> from, to;
  states.reserve((size_t)all);
  from.reserve((size_t)all);
  to.reserve((size_t)all);
  Strides by{};
  by.p = static_cast<const char*>(parents.data_ptr());
  by.end = by.p + n * k * 4;
  for (Py_ssize_t i = 0; i < all; ++i) {
    PyObject *ox = PyList_GET_ITEM(a[0], i), *oy = PyList_GET_ITEM(a[2], i);
    const Tensor &x = on_device(ox, "states", dev), &y = on_device(oy, "out", dev);
    const Strides s = strides_of(x, n, k, "states", i);
    Strides d = s;
    if (oy != ox) {
      NEED(y.scalar_type() == x.scalar_type() && y.sizes() == x.sizes(), "out[", i, "] has to be like states[", i, "]");
      NEED(y.is_conj() == x.is_conj(), "out[", i, "] has to be like states[", i, "]: one of the two is a conjugate view");
      d = strides_of(y, n, k, "out", i);
    }
    if (x.numel() == 0) continue;
    NEED(apart(y), "out[", i, "] has rows that share memory");
    const bool in_place = s.p == d.p && s.l == d.l && s.n == d.n && s.k == d.k;
    NEED(in_place || disjoint(s, d, n, k), "out[", i, "] overlaps states[", i, "]");
    NEED(d.end <= by.p || by.end <= d.p, "out[", i, "] overlaps parents");
    for (size_t j = 0; j < states.size(); ++j)
      NEED(disjoint(d, to[j], n, k) && disjoint(d, from[j], n, k) && disjoint(s, to[j], n, k), "out[", i, "] or an out before it overlaps another state");
    states.push_back({x.data_ptr(), y.data_ptr(), s.l, s.n, s.k, d.l, d.n, d.k, s.row, s.layers});
    from.push_back(s);
    to.push_back(d);
  }
  for (size_t i = 0; i < states.size(); i += 16) {
    g.n_states = (int)std::min<size_t>(16, states.size() - i);
    std::copy(states.begin() + i, states.begin() + i + g.n_states, g.state);
    done_or_raise(linmt_beam_reorder(&g));
  }
  for (Py_ssize_t i = 0; i < all; ++i) was_written(PyList_GET_ITEM(a[2], i));
  Py_INCREF(a[2]);
  return a[2];
  END_HANDLE_TH_ERRORS
}

// A table [n][width] of int32 with contiguous rows.
const Tensor& table_of(PyObject* o, int dev, int64_t n) {
  const Tensor& t = on_device(o, "table", dev);
  NEED(t.scalar_type() == at::kInt && t.dim() == 2 && t.size(0) == n, "table has to be [n, width] int32");
  NEED(t.size(1) <= 1 || t.stride(1) == 1, "the rows of table have to be contiguous");
  return t;
}

PyObject* plan_pages(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  arguments(n_args, 7);
  const Tensor& now = on_cuda(a[1], "new");
  const int dev = now.get_device();
  NEED(now.dim() == 1, "new has to be [n]");
  const int64_t n = now.size(0), shape[1] = {n}, one[1] = {1}, total = integer(a[6], "total");
  linmt_plan_pages_args g{};
  g.size = sizeof(g);
  g.device = dev;
  g.stream = stream_of(dev);
  g.new_len = static_cast<const int32_t*>(dense(a[1], "new", dev, at::kInt, shape).data_ptr());
  if (a[0] != Py_None) g.old_len = static_cast<const int32_t*>(dense(a[0], "old", dev, at::kInt, shape).data_ptr());
  const Tensor& table = table_of(a[2], dev, n);
  NEED(table.stride(0) >= table.size(1) || n <= 1, "the rows of table share memory");
  g.table = static_cast<int32_t*>(table.data_ptr());
  g.table_stride = table.stride(0);
  const Tensor& free = on_device(a[3], "free", dev);
  NEED(free.dim() == 1, "free has to be [n_free]");
  g.free_pages = static_cast<const int32_t*>(dense(a[3], "free", dev, at::kInt, free.sizes()).data_ptr());
  g.used = static_cast<const int32_t*>(dense(a[4], "used", dev, at::kInt, one).data_ptr());
  // Every CTA reads the lengths and the free pages for itself, while others write the table.
  lie_apart(table, "table", a[0], "old");
  lie_apart(table, "table", a[1], "new");
  lie_apart(table, "table", a[3], "free");
  lie_apart(table, "table", a[4], "used");
  NEED(total >= 0, "total is negative");
  g.n = int32_of(n, "n");
  g.width = int32_of(table.size(1), "width");
  g.page = int32_of(integer(a[5], "page"), "page");
  g.n_free = int32_of(free.size(0), "n_free");
  g.total = total;
  Tensor slots = make({total}, at::kLong, dev), starts = make({n + 1}, at::kInt, dev), used = make(one, at::kInt, dev);
  g.out_slots = static_cast<int64_t*>(slots.data_ptr());
  g.out_starts = static_cast<int32_t*>(starts.data_ptr());
  g.out_used = static_cast<int32_t*>(used.data_ptr());
  done_or_raise(linmt_plan_pages(&g));
  was_written(a[2]);
  PyObject* r = PyTuple_New(3);
  if (!r) throw python_error();
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(slots)));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(starts)));
  PyTuple_SET_ITEM(r, 2, THPVariable_Wrap(std::move(used)));
  return r;
  END_HANDLE_TH_ERRORS
}

linmt_pages4 pool_of(PyObject* o, int dev) {
  const Tensor& p = on_device(o, "pages", dev);
  NEED(p.scalar_type() == at::kByte && p.dim() == 4 && p.size(3) % 18 == 0, "pages have to be uint8 [n_pages, heads, page / 16, 18 * dim]");
  NEED(p.stride(3) == 1 && (p.stride(2) == p.size(3) || p.size(2) == 1), "the tiles of a page's head have to be contiguous");
  return {p.data_ptr(), p.stride(0), p.stride(1), int32_of(p.size(0), "n_pages"), int32_of(p.size(1), "heads"), int32_of(p.size(2) * 16, "page"), int32_of(p.size(3) / 18, "dim")};
}

int64_t slots_of(PyObject* o, int dev, linmt_pages4_rows_args& g) {
  const Tensor& slots = on_cuda(o, "slots");
  NEED(slots.dim() == 1, "slots have to be [t]");
  g.slots = static_cast<const int64_t*>(dense(o, "slots", dev, at::kLong, slots.sizes()).data_ptr());
  g.t = int32_of(slots.size(0), "t");
  return slots.size(0);
}
void rows_of(const Tensor& x, const char* name, const linmt_pages4_rows_args& g, void*& p, int64_t& t, int64_t& h) {
  const int64_t want[3] = {g.t, g.pages.heads, g.pages.dim};
  NEED(dtype_of(x) == g.dtype && g.dtype >= 0, name, " has to be float32, bfloat16 or float16, k and v alike");
  NEED(x.sizes() == at::IntArrayRef(want), name, " has to have the shape ", at::IntArrayRef(want), ", not ", x.sizes());
  NEED(x.stride(2) == 1 || x.numel() == 0, "the components of ", name, " have to be contiguous");
  p = x.data_ptr();
  t = x.stride(0);
  h = x.stride(1);
}

PyObject* write_pages4(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  arguments(n_args, 4);
  const int dev = on_cuda(a[1], "slots").get_device();
  linmt_pages4_rows_args g{};
  g.size = sizeof(g);
  g.device = dev;
  g.stream = stream_of(dev);
  g.pages = pool_of(a[0], dev);
  NEED(apart(THPVariable_Unpack(a[0])), "pages have places that share memory");
  slots_of(a[1], dev, g);
  const Tensor &k = on_device(a[2], "k", dev), &v = on_device(a[3], "v", dev);
  g.dtype = dtype_of(k);
  rows_of(k, "k", g, g.k, g.k_stride_t, g.k_stride_h);
  rows_of(v, "v", g, g.v, g.v_stride_t, g.v_stride_h);
  lie_apart(THPVariable_Unpack(a[0]), "pages", a[1], "slots");
  lie_apart(THPVariable_Unpack(a[0]), "pages", a[2], "k");
  lie_apart(THPVariable_Unpack(a[0]), "pages", a[3], "v");
  done_or_raise(linmt_write_pages4(&g));
  was_written(a[0]);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyObject* read_pages4(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  arguments(n_args, 3);
  const int dev = on_cuda(a[1], "slots").get_device();
  linmt_pages4_rows_args g{};
  g.size = sizeof(g);
  g.device = dev;
  g.stream = stream_of(dev);
  g.pages = pool_of(a[0], dev);
  const int64_t shape[3] = {slots_of(a[1], dev, g), g.pages.heads, g.pages.dim};
  const int64_t type = integer(a[2], "dtype");
  NEED(type >= 0 && type <= 2, "dtype has to be float32, bfloat16 or float16");
  const at::ScalarType st = type == LINMT_F32 ? at::kFloat : type == LINMT_BF16 ? at::kBFloat16 : at::kHalf;
  Tensor k = make(shape, st, dev), v = make(shape, st, dev);
  g.dtype = (int)type;
  rows_of(k, "k", g, g.k, g.k_stride_t, g.k_stride_h);
  rows_of(v, "v", g, g.v, g.v_stride_t, g.v_stride_h);
  done_or_raise(linmt_read_pages4(&g));
  PyObject* r = PyTuple_New(2);
  if (!r) throw python_error();
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(k)));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(v)));
  return r;
  END_HANDLE_TH_ERRORS
}

PyObject* attend_pages4(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  arguments(n_args, 12);
  const Tensor& q = on_cuda(a[0], "q");
  const int dev = q.get_device();
  linmt_attend_pages4_args g{};
  g.size = sizeof(g);
  g.device = dev;
  g.stream = stream_of(dev);
  g.pages = pool_of(a[1], dev);
  g.dtype = dtype_of(q);
  NEED(q.dim() == 4 && g.dtype >= 0 && q.size(3) == g.pages.dim, "q has to be [n, g, heads, ", g.pages.dim, "] in float32, bfloat16 or float16");
  NEED(q.stride(3) == 1 || q.numel() == 0, "the components of q have to be contiguous");
  const int64_t n = q.size(0), rows = q.size(1), heads = q.size(2), by_n[1] = {n}, by_head[1] = {heads}, by_row[2] = {n, rows}, by_all[3] = {n, rows, heads};
  g.n = int32_of(n, "n");
  g.g = int32_of(rows, "g");
  g.heads = int32_of(heads, "heads");
  g.q = q.data_ptr();
  g.q_stride_n = q.stride(0);
  g.q_stride_g = q.stride(1);
  g.q_stride_h = q.stride(2);
  const Tensor& table = table_of(a[2], dev, n);
  g.table = static_cast<const int32_t*>(table.data_ptr());
  g.table_stride = table.stride(0);
  g.width = int32_of(table.size(1), "width");
  g.len = static_cast<const int32_t*>(dense(a[3], "lens", dev, at::kInt, by_n).data_ptr());
  g.scale = a[4] == Py_None ? 1.f / std::sqrt((float)g.pages.dim) : (float)real(a[4]);
  g.cap = (float)real(a[5]);
  NEED((a[6] == Py_None) == (a[7] == Py_None), "slope goes with centre");
  NEED((a[8] == Py_None) == (a[9] == Py_None), "first goes with last");
  if (a[6] != Py_None) {
    g.slope = static_cast<const float*>(dense(a[6], "slope", dev, at::kFloat, by_head).data_ptr());
    g.centre = static_cast<const float*>(dense(a[7], "centre", dev, at::kFloat, by_row).data_ptr());
  }
  if (a[8] != Py_None) {
    g.first = static_cast<const int32_t*>(dense(a[8], "first", dev, at::kInt, by_row).data_ptr());
    g.last = static_cast<const int32_t*>(dense(a[9], "last", dev, at::kInt, by_row).data_ptr());
  }
  Tensor out, lse;
  if (a[10] == Py_None) {
    out = make(q.sizes(), q.scalar_type(), dev);
  } else {
    out = on_device(a[10], "out", dev);
    NEED(out.scalar_type() == q.scalar_type() && out.sizes() == q.sizes() && out.stride(3) == 1, "out has to be like q, its components contiguous");
    NEED(apart(out), "out has rows that share memory");
    const bool flat = q.stride(2) == q.size(3) && out.stride(2) == q.size(3);      // heads one behind the other: a row of all of them
    auto places = [&](const Tensor& x) {
      const int64_t e = x.element_size();
      Strides s{n, x.stride(0) * e, x.stride(1) * e, x.stride(2) * e, (flat ? heads : 1) * x.size(3) * e, static_cast<const char*>(x.data_ptr()), nullptr};
      s.end = s.p + (n - 1) * s.l + (rows - 1) * s.n + (flat ? 0 : heads - 1) * s.k + s.row;
      return s;
    };
    const Strides from = places(q), to = places(out);
    const bool same = from.p == to.p && from.l == to.l && from.n == to.n && from.k == to.k;
    NEED(q.numel() == 0 || same || disjoint(from, to, rows, flat ? 1 : heads), "out overlaps q");
    static const char* const read[] = {nullptr, "pages", "table", "lens", nullptr, nullptr, "slope", "centre", "first", "last"};
    for (int i = 1; i < 10; ++i)
      if (read[i]) lie_apart(out, "out", a[i], read[i]);
  }
  g.out = out.data_ptr();
  g.out_stride_n = out.stride(0);
  g.out_stride_g = out.stride(1);
  g.out_stride_h = out.stride(2);
  const int want_lse = PyObject_IsTrue(a[11]);
  if (want_lse < 0) throw python_error();
  if (want_lse) {
    lse = make(by_all, at::kFloat, dev);
    g.lse = static_cast<float*>(lse.data_ptr());
  }
  Tensor ws;
  if (q.numel()) {
    const int64_t need = linmt_attend_pages4_workspace(&g);
    NEED(need >= 0, linmt_op_error());
    if (need) {
      ws = make({need}, at::kByte, dev);     // goes back to torch's pool of this stream behind the call's kernels
      g.workspace = ws.data_ptr();
      g.workspace_bytes = need;
    }
    done_or_raise(linmt_attend_pages4(&g));
  }
  PyObject* o = a[10];
  if (o == Py_None) o = THPVariable_Wrap(std::move(out));
  else {
    was_written(o);
    Py_INCREF(o);
  }
  if (!want_lse) return o;
  PyObject* r = PyTuple_New(2);
  if (!r) { Py_DECREF(o); throw python_error(); }
  PyTuple_SET_ITEM(r, 0, o);
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(lse)));
  return r;
  END_HANDLE_TH_ERRORS
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyCFunction fast() { return reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(F)); }

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__device_ops() {
  static PyMethodDef methods[] = {{"beam_select", fast<beam_select>(), METH_FASTCALL, nullptr}, {"beam_reorder", fast<beam_reorder>(), METH_FASTCALL, nullptr},
                                  {"plan_pages", fast<plan_pages>(), METH_FASTCALL, nullptr},   {"write_pages4", fast<write_pages4>(), METH_FASTCALL, nullptr},
                                  {"read_pages4", fast<read_pages4>(), METH_FASTCALL, nullptr}, {"attend_pages4", fast<attend_pages4>(), METH_FASTCALL, nullptr},
                                  {nullptr, nullptr, 0, nullptr}};
  static PyModuleDef module = {PyModuleDef_HEAD_INIT, "_device_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};
  PyObject* decoder = PyImport_ImportModule("linmt_b200.decoder");
  if (!decoder) return nullptr;
  g_error = PyObject_GetAttrString(decoder, "LinmtError");
  Py_DECREF(decoder);
  return g_error ? PyModule_Create(&module) : nullptr;
}
