// Host side of calls whose time is the host's: a CPython module against torch's
// headers.  From Python each property of a tensor costs about 70 ns.
//
// Calls over many tensors: it reads what a launch needs from a list of tensors
// (pointer, count, dtype, layout, device) in one pass, and says whether the
// written ones share memory (a dozen properties of 768 gradients and their
// targets took 650 us, here 15 us).
// Calls over small batches, whose kernels take 10 us: the checks of a call's
// arguments, its outputs and workspace, the call of the C entry and its record
// for autograd in one function each (in Python a forward took 21 to 25 us of
// host time, now 8 to 12, a training call 123 to 134, now 82 to 88).
// The Python callers keep the checks' messages: a check here only says whether
// there is anything to look at.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>

#include <algorithm>
#include <cstdint>
#include <exception>
#include <memory>
#include <mutex>
#include <string>
#include <vector>

#include "../../include/esa_hip.h"

namespace {

constexpr int kF32 = ESA_F32, kBf16 = ESA_BF16;

// C++ exceptions (torch's errors among them) end here as Python's.
template <class F>
PyObject* guarded(F f) {
  try {
    return f();
  } catch (const c10::OutOfMemoryError& e) {
    if (!PyErr_Occurred()) {
      PyObject* torch = PyImport_ImportModule("torch");
      PyObject* type = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
      if (type) PyErr_SetString(type, e.what_without_backtrace());
      Py_XDECREF(type);
      Py_XDECREF(torch);
    }
    return nullptr;
  } catch (const std::exception& e) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// What the C ABI takes of a list of tensors.
struct Listed {
  std::vector<void*> ptrs;
  std::vector<int64_t> counts;
  std::vector<int32_t> codes;
  int device = 0;   // the tensors' GPU, -1 if one is on the host, -2 if they are on several
  bool contiguous = true;
  size_t n = 0;
};

// False with Python's error set: not a list of dense float32 and bfloat16 tensors.
bool read(PyObject* list, Listed& x) {
  if (!PyList_Check(list)) {
    PyErr_SetString(PyExc_TypeError, "a list of tensors is expected");
    return false;
  }
  x.n = PyList_GET_SIZE(list);
  x.ptrs.resize(x.n + 1);   // (an empty array has an address, too)
  x.counts.resize(x.n + 1);
  x.codes.resize(x.n + 1);
  for (size_t i = 0; i < x.n; ++i) {
    PyObject* o = PyList_GET_ITEM(list, i);
    if (!THPVariable_Check(o)) {
      PyErr_Format(PyExc_TypeError, "tensors are expected (got %s)", Py_TYPE(o)->tp_name);
      return false;
    }
    const at::Tensor& t = THPVariable_Unpack(o);
    if (t.scalar_type() != at::kFloat && t.scalar_type() != at::kBFloat16) {
      PyErr_Format(PyExc_TypeError, "tensors must be float32 or bfloat16 (got %s)", at::toString(t.scalar_type()));
      return false;
    }
    if (t.layout() != at::kStrided) {
      PyErr_SetString(PyExc_TypeError, "tensors must be dense");
      return false;
    }
    const int at = t.is_cuda() ? t.get_device() : -1;
    if (i == 0 || at == -1) x.device = at == -1 ? -1 : at;
    else if (x.device >= 0 && at != x.device) x.device = -2;
    x.contiguous = x.contiguous && t.is_contiguous() && !t.is_neg();
    x.codes[i] = t.scalar_type() == at::kFloat ? kF32 : kBf16;
    x.counts[i] = t.numel();
    x.ptrs[i] = t.data_ptr();
  }
  return true;
}

// describe(list) -> (pointers, counts, codes, device, contiguous): bytes of n void*, n int64 and n int32, and whether all
// tensors are contiguous.  A dtype other than float32 and bfloat16 raises TypeError.
PyObject* describe(PyObject*, PyObject* list) {
  return guarded([&]() -> PyObject* {
    Listed x;
    if (!read(list, x)) return nullptr;
    return Py_BuildValue("(y#y#y#iO)", reinterpret_cast<const char*>(x.ptrs.data()), (Py_ssize_t)(x.n * sizeof(void*)),
                         reinterpret_cast<const char*>(x.counts.data()), (Py_ssize_t)(x.n * sizeof(int64_t)),
                         reinterpret_cast<const char*>(x.codes.data()), (Py_ssize_t)(x.n * sizeof(int32_t)), x.device,
                         x.contiguous ? Py_True : Py_False);
  });
}

// What keeps a target from taking its tensor: "shapes", or "dtypes" (a target has its tensor's dtype or is float32); null:
// nothing.  Both are lists of tensors.
const char* misfit_of(PyObject* a, PyObject* b) {
  if (PyList_GET_SIZE(a) != PyList_GET_SIZE(b)) return "shapes";
  for (Py_ssize_t i = 0; i < PyList_GET_SIZE(a); ++i) {
    const at::Tensor &t = THPVariable_Unpack(PyList_GET_ITEM(a, i)), &u = THPVariable_Unpack(PyList_GET_ITEM(b, i));
    if (t.sizes() != u.sizes()) return "shapes";
    if (u.scalar_type() != t.scalar_type() && u.scalar_type() != at::kFloat) return "dtypes";
  }
  return nullptr;
}

// misfit(tensors, targets) -> None or misfit_of's word
PyObject* misfit(PyObject*, PyObject* args) {
  return guarded([&]() -> PyObject* {
    PyObject *a, *b;
    if (!PyArg_ParseTuple(args, "O!O!", &PyList_Type, &a, &PyList_Type, &b)) return nullptr;
    for (PyObject* list : {a, b})
      for (Py_ssize_t i = 0; i < PyList_GET_SIZE(list); ++i)
        if (!THPVariable_Check(PyList_GET_ITEM(list, i))) {
          PyErr_SetString(PyExc_TypeError, "tensors are expected");
          return nullptr;
        }
    const char* word = misfit_of(a, b);
    if (!word) Py_RETURN_NONE;
    return PyUnicode_FromString(word);
  });
}

struct Span {
  uint64_t first, end;
  int64_t owner;
};

bool spans_of(PyObject* tuple, std::vector<Span>& out) {
  const char *ptrs, *counts, *codes;
  Py_ssize_t np, nc, nd;
  if (!PyArg_ParseTuple(tuple, "y#y#y#", &ptrs, &np, &counts, &nc, &codes, &nd)) return false;
  const size_t n = np / sizeof(void*);
  if (nc != (Py_ssize_t)(n * 8) || nd != (Py_ssize_t)(n * 4)) {
    PyErr_SetString(PyExc_ValueError, "pointers, counts and codes of different lengths");
    return false;
  }
  for (size_t i = 0; i < n; ++i) {
    const uint64_t first = reinterpret_cast<const uint64_t*>(ptrs)[i];
    const uint64_t bytes = (uint64_t)reinterpret_cast<const int64_t*>(counts)[i] *
                           (reinterpret_cast<const int32_t*>(codes)[i] == kF32 ? 4 : 2);
    out.push_back({first, first + bytes, (int64_t)i});
  }
  return true;
}

// Whether every written tensor keeps to itself: no byte of it is another written tensor's, nor of another position's read
// tensor; its own read tensor may lie exactly there.
bool apart(std::vector<Span> w, const std::vector<Span>& r) {
  w.erase(std::remove_if(w.begin(), w.end(), [](const Span& s) { return s.end <= s.first; }), w.end());
  auto before = [](const Span& a, const Span& b) { return a.first < b.first; };
  if (!std::is_sorted(w.begin(), w.end(), before)) std::sort(w.begin(), w.end(), before);   // in a flat buffer they are
  for (size_t i = 1; i < w.size(); ++i)
    if (w[i].first < w[i - 1].end) return false;
  for (const Span& s : r) {
    if (s.end <= s.first || w.empty() || s.end <= w.front().first || s.first >= w.back().end) continue;
    // written spans are disjoint and in order: those that end behind s.first, up to the first beyond s.end
    auto it = std::upper_bound(w.begin(), w.end(), s.first, [](uint64_t at, const Span& b) { return at < b.end; });
    for (; it != w.end() && it->first < s.end; ++it)
      if (it->owner != s.owner || it->first != s.first || it->end != s.end) return false;
  }
  return true;
}

// separate(written, read or None) -> apart's answer, both (pointers, counts, codes) of describe
PyObject* separate(PyObject*, PyObject* args) {
  return guarded([&]() -> PyObject* {
    PyObject *written, *read;
    if (!PyArg_ParseTuple(args, "OO", &written, &read)) return nullptr;
    std::vector<Span> w, r;
    if (!spans_of(written, w) || (read != Py_None && !spans_of(read, r))) return nullptr;
    return PyBool_FromLong(apart(std::move(w), r));
  });
}

std::vector<Span> spans_of(const Listed& x) {
  std::vector<Span> out;
  out.reserve(x.n);
  for (size_t i = 0; i < x.n; ++i) {
    const uint64_t first = reinterpret_cast<uint64_t>(x.ptrs[i]);
    out.push_back({first, first + (uint64_t)x.counts[i] * (x.codes[i] == kF32 ? 4 : 2), (int64_t)i});
  }
  return out;
}

void count_change(PyObject* list) {
  for (Py_ssize_t i = 0; i < PyList_GET_SIZE(list); ++i) {
    PyObject* o = PyList_GET_ITEM(list, i);
    if (!THPVariable_Check(o)) continue;
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  }
}

// changed(list): the tensors' memory was written outside torch (what torch's own in-place operations count).
PyObject* changed(PyObject*, PyObject* list) {
  return guarded([&]() -> PyObject* {
    if (!PyList_Check(list)) {
      PyErr_SetString(PyExc_TypeError, "a list of tensors is expected");
      return nullptr;
    }
    count_change(list);
    Py_RETURN_NONE;
  });
}

// ---- calls of small batches

// What the checks say of a call: its arguments fit, all tensors are of torch's own types.
constexpr long kFits = 1, kExact = 2;

int code_of(const at::Tensor& t) { return t.scalar_type() == at::kFloat ? kF32 : t.scalar_type() == at::kBFloat16 ? kBf16 : -1; }
bool head_dim_ok(int64_t d) { return d == 16 || d == 24 || d == 32 || d == 64; }

// The tensors of a call; args[i] None where optional.
struct Args {
  long flags = kFits | kExact;
  const at::Tensor* first = nullptr;
  const at::Tensor* get(PyObject* o) {
    if (!THPVariable_Check(o)) {
      flags = 0;
      return nullptr;
    }
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!THPVariable_CheckTypeExact(Py_TYPE(o))) flags &= ~kExact;
    if (!first) first = &t;
    if (t.layout() != at::kStrided || t.is_neg() || !t.is_cuda() || t.get_device() != first->get_device()) flags &= ~kFits;
    return &t;
  }
  void want(bool ok) { flags = ok ? flags : flags & ~kFits; }
};

bool index_fits(const at::Tensor& t, int64_t n) {
  return t.scalar_type() == at::kInt && t.dim() == 1 && t.is_contiguous() && (n < 0 || t.numel() == n);
}

// relative_fits(q, k, v, bias, cu_q, cu_k, q_start) -> flags
PyObject* relative_fits(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 7) return PyLong_FromLong(0);
    Args a;
    const at::Tensor* t[7] = {};
    for (int i = 0; i < 7; ++i)
      if (i < 6 || args[i] != Py_None)
        if (!(t[i] = a.get(args[i]))) return PyLong_FromLong(0);
    const at::Tensor &q = *t[0], &k = *t[1], &v = *t[2], &bias = *t[3], &cu_q = *t[4], &cu_k = *t[5];
    a.want(q.dim() == 3 && k.dim() == 3 && v.dim() == 3 && bias.dim() == 2 && code_of(q) >= 0 && code_of(bias) >= 0);
    if (!(a.flags & kFits)) return PyLong_FromLong(a.flags);
    a.want(q.is_contiguous() && k.is_contiguous() && v.is_contiguous() && code_of(k) == code_of(q) && code_of(v) == code_of(q));
    a.want(head_dim_ok(q.size(2)) && k.size(1) == q.size(1) && k.size(2) == q.size(2) && v.sizes() == k.sizes());
    a.want(bias.size(1) == q.size(1) && index_fits(cu_q, -1) && cu_q.numel() >= 2 && index_fits(cu_k, cu_q.numel()));
    if (t[6]) a.want(index_fits(*t[6], cu_q.numel() - 1));
    return PyLong_FromLong(a.flags);
  });
}

const at::Tensor& tensor_of(PyObject* o) {
  TORCH_CHECK(THPVariable_Check(o), "a tensor is expected");
  return THPVariable_Unpack(o);
}
void* pointer_of(PyObject* o) { return o == Py_None ? nullptr : tensor_of(o).data_ptr(); }
PyObject* wrapped(const at::Tensor& t) { return t.defined() ? THPVariable_Wrap(t) : Py_NewRef(Py_None); }

// Owned references as a tuple.
template <size_t N>
PyObject* tuple_of(PyObject* const (&items)[N]) {
  PyObject* r = PyTuple_New(N);
  for (size_t i = 0; i < N; ++i) {
    if (!r || !items[i]) {
      for (size_t j = r ? i : 0; j < N; ++j) Py_XDECREF(items[j]);
      Py_XDECREF(r);
      return nullptr;
    }
    PyTuple_SET_ITEM(r, i, items[i]);
  }
  return r;
}

// f() without the interpreter's lock, which is held again whether f returns or throws.
template <class F>
int without_gil(F f) {
  struct Released {
    PyThreadState* state = PyEval_SaveThread();
    ~Released() { PyEval_RestoreThread(state); }
  } released;
  return f();
}

at::Tensor bytes_on(const at::Tensor& like, size_t bytes) {
  return at::empty({(int64_t)std::max<size_t>(bytes, 256)}, like.options().dtype(at::kByte));
}

// A relative attention call besides its tensors.
struct RelCall {
  decltype(&esa_rel_attn_fwd) fwd;
  decltype(&esa_rel_attn_bwd) bwd;
  decltype(&esa_rel_attn_workspace_size) size;
  std::string starts;   // int32 values
  float scale, dropout;
  unsigned long long seed;
  const int* first() const { return reinterpret_cast<const int*>(starts.data()); }
  int side() const { return (int)(starts.size() / sizeof(int)); }
  // (addresses of forward, backward and size query, starts (bytes of int32), scale, dropout_p, seed)
  explicit RelCall(PyObject* const* a)
      : fwd(reinterpret_cast<decltype(fwd)>(PyLong_AsVoidPtr(a[0]))),
        bwd(reinterpret_cast<decltype(bwd)>(PyLong_AsVoidPtr(a[1]))),
        size(reinterpret_cast<decltype(size)>(PyLong_AsVoidPtr(a[2]))),
        starts(PyBytes_AsString(a[3]), PyBytes_Size(a[3])),
        scale((float)PyFloat_AsDouble(a[4])),
        dropout((float)PyFloat_AsDouble(a[5])),
        seed(PyLong_AsUnsignedLongLong(a[6])) {}
};

struct RelTensors {
  at::Tensor q, k, v, table, cu_q, cu_k, q_start, out, low, lse;   // q_start, low: or undefined
};

void* stream_of(const at::Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
const void* data_or_null(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// out, low (where kept) and lse of t's inputs; the C entry's status.
int relative_run(const RelCall& c, RelTensors& t, bool keep) {
  const at::Tensor &q = t.q, &k = t.k;
  TORCH_CHECK(q.size(0) <= INT32_MAX && k.size(0) <= INT32_MAX && q.size(1) <= INT32_MAX && t.cu_q.numel() <= INT32_MAX,
              "sizes beyond 32 bits");
  const int batch = (int)t.cu_q.numel() - 1, tq = (int)q.size(0), tk = (int)k.size(0), heads = (int)q.size(1), hd = (int)q.size(2);
  const int buckets = (int)t.table.size(0);
  const c10::DeviceGuard on(q.device());
  size_t bytes = 0;
  if (const int rc = c.size(batch, tq, tk, heads, hd, code_of(q), buckets, c.first(), c.side(), 0, &bytes)) return rc;
  t.out = at::empty(q.sizes(), q.options());
  if (keep && q.scalar_type() == at::kBFloat16) t.low = at::empty(q.sizes(), q.options());
  t.lse = at::empty({heads, tq}, q.options().dtype(at::kFloat));
  const at::Tensor ws = bytes_on(q, bytes);
  return c.fwd(q.data_ptr(), k.data_ptr(), t.v.data_ptr(), t.table.data_ptr(), code_of(t.table), buckets, c.first(), c.side(),
               static_cast<const int*>(data_or_null(t.q_start)), t.cu_q.data_ptr<int>(), t.cu_k.data_ptr<int>(), batch, tq, tk,
               heads, hd, code_of(q), c.scale, c.dropout, c.seed, t.out.data_ptr(), t.low.defined() ? t.low.data_ptr() : nullptr,
               t.lse.data_ptr<float>(), ws.data_ptr(), (size_t)ws.numel(), stream_of(q));
}

// A gradient as the kernels take it: dense, by value, on a 16-byte boundary.
at::Tensor gradient_of(const at::Tensor& grad) {
  const at::Tensor g = grad.resolve_neg().contiguous();
  return reinterpret_cast<uintptr_t>(g.data_ptr()) % 16 ? g.clone() : g;
}

// d: dq, dk, dv and the table's gradient in the table's type; the C entry's status.
int relative_back(const RelCall& c, const RelTensors& t, const at::Tensor& grad, at::Tensor (&d)[4]) {
  const at::Tensor &q = t.q, &k = t.k;
  const int batch = (int)t.cu_q.numel() - 1, tq = (int)q.size(0), tk = (int)k.size(0), heads = (int)q.size(1), hd = (int)q.size(2);
  const int buckets = (int)t.table.size(0);
  const c10::DeviceGuard on(q.device());
  const at::Tensor g = gradient_of(grad);
  size_t bytes = 0;
  int rc = c.size(batch, tq, tk, heads, hd, code_of(q), buckets, c.first(), c.side(), 1, &bytes);
  if (rc) return rc;
  d[0] = at::empty(q.sizes(), q.options());
  d[1] = at::empty(k.sizes(), k.options());
  d[2] = at::empty(k.sizes(), k.options());
  d[3] = at::empty(t.table.sizes(), t.table.options().dtype(at::kFloat));
  const at::Tensor ws = bytes_on(q, bytes);
  rc = c.bwd(g.data_ptr(), q.data_ptr(), k.data_ptr(), t.v.data_ptr(), t.out.data_ptr(), data_or_null(t.low),
             t.lse.data_ptr<float>(), t.table.data_ptr(), code_of(t.table), buckets, c.first(), c.side(),
             static_cast<const int*>(data_or_null(t.q_start)), t.cu_q.data_ptr<int>(), t.cu_k.data_ptr<int>(), batch, tq, tk, heads,
             hd, code_of(q), c.scale, c.dropout, c.seed, d[0].data_ptr(), d[1].data_ptr(), d[2].data_ptr(), d[3].data_ptr<float>(),
             ws.data_ptr(), (size_t)ws.numel(), stream_of(q));
  if (rc == ESA_OK && t.table.scalar_type() != at::kFloat) d[3] = d[3].to(t.table.scalar_type());
  return rc;
}

at::Tensor optional(PyObject* o) { return o == Py_None ? at::Tensor() : tensor_of(o); }

// (q, k, v, bias, q_start, cu_q, cu_k)
RelTensors relative_inputs(PyObject* const* a) {
  RelTensors t;
  t.q = tensor_of(a[0]);
  t.k = tensor_of(a[1]);
  t.v = tensor_of(a[2]);
  t.table = tensor_of(a[3]).contiguous();
  t.q_start = optional(a[4]);
  t.cu_q = tensor_of(a[5]);
  t.cu_k = tensor_of(a[6]);
  return t;
}

// relative_forward(RelCall's seven, relative_inputs' seven, keep) -> (status, out, out_low or None, lse, the table)
PyObject* relative_forward(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    TORCH_CHECK(n == 15 && PyBytes_Check(args[3]), "relative_forward: arguments");
    const RelCall c(args);
    RelTensors t = relative_inputs(args + 7);
    const bool keep = PyObject_IsTrue(args[14]);
    if (PyErr_Occurred()) return nullptr;
    const int rc = without_gil([&] { return relative_run(c, t, keep); });
    return tuple_of({PyLong_FromLong(rc), wrapped(t.out), wrapped(t.low), wrapped(t.lse), wrapped(t.table)});
  });
}

// relative_backward(RelCall's seven, relative_inputs' seven, out, out_low, lse, dout) -> (status, dq, dk, dv, dtable)
PyObject* relative_backward(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    TORCH_CHECK(n == 18 && PyBytes_Check(args[3]), "relative_backward: arguments");
    const RelCall c(args);
    RelTensors t = relative_inputs(args + 7);
    t.out = tensor_of(args[14]);
    t.low = optional(args[15]);
    t.lse = tensor_of(args[16]);
    const at::Tensor& g = tensor_of(args[17]);
    if (PyErr_Occurred()) return nullptr;
    at::Tensor d[4];
    const int rc = without_gil([&] { return relative_back(c, t, g, d); });
    return tuple_of({PyLong_FromLong(rc), wrapped(d[0]), wrapped(d[1]), wrapped(d[2]), wrapped(d[3])});
  });
}

// ---- the same as autograd nodes, for ordinary eager calls

// Results of a backward that is itself recorded: differentiating them again is refused.
torch::autograd::variable_list only_once(torch::autograd::variable_list&& grads, bool recorded) {
  if (!recorded) return std::move(grads);
  for (at::Tensor& g : grads)
    if (g.defined()) {
      g = g.detach();
      g.requires_grad_(true);
    }
  const auto refuse = std::make_shared<torch::autograd::DelayedError>(
      "these gradients cannot be differentiated again", (int64_t)grads.size());
  return (*refuse)(std::move(grads));
}

using torch::autograd::SavedVariable;

struct RelativeAttentionBackward : torch::autograd::Node {
  RelCall call;
  SavedVariable q, k, v, table, cu_q, cu_k, q_start, out, low, lse;
  std::mutex mutex;
  explicit RelativeAttentionBackward(const RelCall& c) : call(c) {}
  std::string name() const override { return "RelativeAttentionBackward"; }
  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex);
    for (SavedVariable* x : {&q, &k, &v, &table, &cu_q, &cu_k, &q_start, &out, &low, &lse}) x->reset_data();
  }
  torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
    const std::lock_guard<std::mutex> lock(mutex);
    torch::autograd::variable_list result(4);
    if (!grads[0].defined()) return result;
    const bool recorded = at::GradMode::is_enabled();
    const at::AutoGradMode none(false);
    RelTensors t;
    t.q = q.unpack();
    t.k = k.unpack();
    t.v = v.unpack();
    t.table = table.unpack();
    t.cu_q = cu_q.unpack();
    t.cu_k = cu_k.unpack();
    t.q_start = q_start.unpack();
    t.out = out.unpack(getptr());
    t.low = low.unpack();
    t.lse = lse.unpack();
    at::Tensor d[4];
    const int rc = relative_back(call, t, grads[0], d);
    TORCH_CHECK(rc == ESA_OK, "esa_rel_attn_bwd: status ", rc);
    for (int i = 0; i < 4; ++i) result[i] = d[i];
    return only_once(std::move(result), recorded);
  }
};

bool wants_grad(const at::Tensor& t) { return t.defined() && t.requires_grad(); }

// relative(RelCall's seven, relative_inputs' seven) -> (status, out, lse), recorded where torch would
PyObject* relative(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    TORCH_CHECK(n == 14 && PyBytes_Check(args[3]), "relative: arguments");
    const RelCall c(args);
    RelTensors t = relative_inputs(args + 7);
    const at::Tensor& bias = tensor_of(args[10]);
    if (PyErr_Occurred()) return nullptr;
    const bool record = at::GradMode::is_enabled() && (wants_grad(t.q) || wants_grad(t.k) || wants_grad(t.v) || wants_grad(bias));
    int rc;
    {
      const at::AutoGradMode none(false);
      if (record) t.table = t.table.detach();
      rc = without_gil([&] { return relative_run(c, t, record); });
    }
    if (rc == ESA_OK && record) {
      std::shared_ptr<RelativeAttentionBackward> node(new RelativeAttentionBackward(c), torch::autograd::deleteNode);
      node->set_next_edges(torch::autograd::collect_next_edges(t.q, t.k, t.v, bias));
      torch::autograd::set_history(t.out, node);
      node->q = SavedVariable(t.q, false);
      node->k = SavedVariable(t.k, false);
      node->v = SavedVariable(t.v, false);
      // the bias itself where it was read as it lies, for the check that it has not been written since
      node->table = SavedVariable(bias.is_contiguous() ? bias : t.table, false);
      node->cu_q = SavedVariable(t.cu_q, false);
      node->cu_k = SavedVariable(t.cu_k, false);
      node->q_start = SavedVariable(t.q_start, false);
      node->out = SavedVariable(t.out, true);
      node->low = SavedVariable(t.low, false);
      node->lse = SavedVariable(t.lse, false);
    }
    return tuple_of({PyLong_FromLong(rc), wrapped(t.out), wrapped(t.lse)});
  });
}

// clip(address of esa_grad_clip, of its size query, stream, gradients, targets, infinity, max_norm) -> (status, the norm),
// or None, and nothing done, where the lists are not contiguous tensors of one GPU that fit and keep apart.
PyObject* clip(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    TORCH_CHECK(n == 7 && PyList_Check(args[3]) && PyList_Check(args[4]), "clip: arguments");
    const auto fn = reinterpret_cast<decltype(&esa_grad_clip)>(PyLong_AsVoidPtr(args[0]));
    const auto size_of = reinterpret_cast<decltype(&esa_grad_workspace_size)>(PyLong_AsVoidPtr(args[1]));
    void* stream = PyLong_AsVoidPtr(args[2]);
    const int infinity = PyObject_IsTrue(args[5]);
    const float max_norm = (float)PyFloat_AsDouble(args[6]);
    if (PyErr_Occurred()) return nullptr;
    Listed in, other;
    if (!read(args[3], in)) return nullptr;
    const bool in_place = args[3] == args[4];
    if (!in_place && !read(args[4], other)) return nullptr;
    const Listed& out = in_place ? in : other;
    if (in.n == 0 || in.device < 0 || out.device != in.device || !in.contiguous || !out.contiguous || in.n > INT32_MAX) Py_RETURN_NONE;
    if (!in_place && misfit_of(args[3], args[4])) Py_RETURN_NONE;
    if (!apart(spans_of(out), in_place ? std::vector<Span>() : spans_of(in))) Py_RETURN_NONE;
    const auto like = at::TensorOptions().device(at::Device(at::kCUDA, (at::DeviceIndex)in.device));
    const c10::DeviceGuard on(like.device());
    const auto counts = reinterpret_cast<const long long*>(in.counts.data());
    size_t bytes = 0;
    at::Tensor norm, ws;
    int rc = size_of((int)in.n, counts, 1, &bytes);
    if (rc == ESA_OK) {
      norm = at::empty({}, like.dtype(at::kFloat));
      ws = at::empty({(int64_t)std::max<size_t>(bytes, 256)}, like.dtype(at::kByte));
      rc = without_gil([&] {
        return fn((int)in.n, in.ptrs.data(), out.ptrs.data(), counts, in.codes.data(), out.codes.data(), infinity, max_norm,
                  norm.data_ptr<float>(), ws.data_ptr(), (size_t)ws.numel(), stream);
      });
      count_change(args[4]);
    }
    return tuple_of({PyLong_FromLong(rc), wrapped(norm)});
  });
}

// qk_norm_fits(q, k, q_weight, k_weight, positions, frequencies) -> flags; all but q may be None
PyObject* qk_norm_fits(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 6) return PyLong_FromLong(0);
    Args a;
    const at::Tensor* t[6] = {};
    for (int i = 0; i < 6; ++i)
      if (i == 0 || args[i] != Py_None)
        if (!(t[i] = a.get(args[i]))) return PyLong_FromLong(0);
    const at::Tensor& q = *t[0];
    a.want(q.dim() == 3 && code_of(q) >= 0);
    if (!(a.flags & kFits)) return PyLong_FromLong(a.flags);
    const int64_t hd = q.size(2), most = 2048;
    a.want(head_dim_ok(hd) && q.size(1) >= 1 && q.size(1) <= most);
    if (t[1]) {
      const at::Tensor& k = *t[1];
      a.want(k.dim() == 3 && code_of(k) == code_of(q) && k.size(0) == q.size(0) && k.size(1) >= 1 && k.size(1) <= most &&
             k.size(2) == hd);
    } else {
      a.want(!t[3]);
    }
    for (int i = 2; i < 4; ++i)
      if (t[i]) a.want(t[i]->dim() == 1 && t[i]->size(0) == hd && code_of(*t[i]) >= 0);
    a.want(!t[4] == !t[5]);
    if (t[4] && t[5]) {
      const at::Tensor &p = *t[4], &f = *t[5];
      a.want((p.scalar_type() == at::kInt || p.scalar_type() == at::kLong) && p.dim() == 1 && p.is_contiguous() &&
             p.numel() == q.size(0));
      a.want(f.scalar_type() == at::kDouble && f.dim() == 1 && f.is_contiguous());
      const int64_t r = 2 * f.numel();
      a.want(r % 8 == 0 && r >= 8 && r <= hd);
    }
    return PyLong_FromLong(a.flags);
  });
}

// The rows where they lie, or their copy where they are no 16-byte aligned runs.
at::Tensor rows_of(const at::Tensor& x) {
  const int64_t size = x.element_size();
  if (x.stride(2) == 1 && reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0 && x.stride(0) * size % 16 == 0 &&
      x.stride(1) * size % 16 == 0)
    return x;
  return x.clone(at::MemoryFormat::Contiguous);
}

// A call of the norms with rotation besides its tensors.
struct NormCall {
  decltype(&esa_qk_norm_fwd) fwd;
  decltype(&esa_qk_norm_bwd) bwd;
  decltype(&esa_qk_norm_bwd_workspace_size) size;
  float eps;
  int interleaved;
  // (addresses of forward, backward and the backward's size query, eps, interleaved)
  explicit NormCall(PyObject* const* a)
      : fwd(reinterpret_cast<decltype(fwd)>(PyLong_AsVoidPtr(a[0]))),
        bwd(reinterpret_cast<decltype(bwd)>(PyLong_AsVoidPtr(a[1]))),
        size(reinterpret_cast<decltype(size)>(PyLong_AsVoidPtr(a[2]))),
        eps((float)PyFloat_AsDouble(a[3])),
        interleaved(PyObject_IsTrue(a[4])) {}
};

struct NormTensors {
  at::Tensor q, k, wq, wk, positions, frequencies;   // rows where they are read; weights in float32; all but q may be undefined
  bool keys() const { return k.defined(); }
  int heads_k() const { return keys() ? (int)k.size(1) : 0; }
  int rotary() const { return frequencies.defined() ? 2 * (int)frequencies.numel() : 0; }
  int positions_bytes() const { return positions.defined() ? (int)positions.element_size() : 0; }
  const float* weight(const at::Tensor& w) const { return static_cast<const float*>(data_or_null(w)); }
  void strides(long long (&x)[4]) const {
    x[0] = q.stride(0);
    x[1] = q.stride(1);
    x[2] = keys() ? k.stride(0) : 0;
    x[3] = keys() ? k.stride(1) : 0;
  }
};

at::Tensor f32_of(const at::Tensor& w) { return w.defined() ? w.detach().to(at::kFloat).contiguous() : w; }

// (q, k, q_weight, k_weight, positions, frequencies)
NormTensors norm_inputs(PyObject* const* a) {
  NormTensors t;
  t.q = rows_of(tensor_of(a[0]));
  if (a[1] != Py_None) t.k = rows_of(tensor_of(a[1]));
  t.wq = f32_of(optional(a[2]));
  t.wk = f32_of(optional(a[3]));
  t.positions = optional(a[4]);
  t.frequencies = optional(a[5]);
  return t;
}

int norm_run(const NormCall& c, const NormTensors& t, at::Tensor& q_out, at::Tensor& k_out) {
  TORCH_CHECK(t.q.size(0) <= INT32_MAX, "sizes beyond 32 bits");
  long long strides[4];
  t.strides(strides);
  const c10::DeviceGuard on(t.q.device());
  q_out = at::empty(t.q.sizes(), t.q.options());
  if (t.keys()) k_out = at::empty(t.k.sizes(), t.k.options());
  return c.fwd(t.q.data_ptr(), data_or_null(t.k), strides, (int)t.q.size(0), (int)t.q.size(1), t.heads_k(), (int)t.q.size(2),
               code_of(t.q), t.weight(t.wq), t.weight(t.wk), data_or_null(t.positions), t.positions_bytes(),
               static_cast<const double*>(data_or_null(t.frequencies)), t.rotary(), c.interleaved, c.eps, q_out.data_ptr(),
               k_out.defined() ? k_out.data_ptr() : nullptr, stream_of(t.q));
}

// d: dq, dk and where their types (c10::ScalarType) are given, the weights' gradients.
int norm_back(const NormCall& c, const NormTensors& t, const at::Tensor& grad_q, const at::Tensor& grad_k,
              const std::optional<at::ScalarType> (&types)[2], at::Tensor (&d)[4]) {
  long long strides[4];
  t.strides(strides);
  const int total = (int)t.q.size(0), hd = (int)t.q.size(2);
  const c10::DeviceGuard on(t.q.device());
  auto given = [](const at::Tensor& g, const at::Tensor& like) {
    return gradient_of(g.defined() ? g : at::zeros(like.sizes(), like.options()));
  };
  const at::Tensor gq = given(grad_q, t.q), gk = t.keys() ? given(grad_k, t.k) : at::Tensor();
  d[0] = at::empty(t.q.sizes(), t.q.options());
  if (t.keys()) d[1] = at::empty(t.k.sizes(), t.k.options());
  at::Tensor ws;
  for (int i = 0; i < 2; ++i)
    if (types[i]) d[2 + i] = at::empty({hd}, t.q.options().dtype(at::kFloat));
  if (types[0] || types[1]) {
    size_t bytes = 0;
    if (const int rc = c.size(total, hd, &bytes)) return rc;
    ws = bytes_on(t.q, bytes);
  }
  auto floats = [](const at::Tensor& x) { return x.defined() ? x.data_ptr<float>() : nullptr; };
  const int rc = c.bwd(gq.data_ptr(), data_or_null(gk), t.q.data_ptr(), data_or_null(t.k), strides, total, (int)t.q.size(1),
                       t.heads_k(), hd, code_of(t.q), t.weight(t.wq), t.weight(t.wk), data_or_null(t.positions),
                       t.positions_bytes(), static_cast<const double*>(data_or_null(t.frequencies)), t.rotary(), c.interleaved,
                       c.eps, d[0].data_ptr(), t.keys() ? d[1].data_ptr() : nullptr, floats(d[2]), floats(d[3]),
                       ws.defined() ? ws.data_ptr() : nullptr, ws.defined() ? (size_t)ws.numel() : 0, stream_of(t.q));
  for (int i = 0; i < 2; ++i)
    if (rc == ESA_OK && types[i]) d[2 + i] = d[2 + i].to(*types[i]);
  return rc;
}

// qk_norm_forward(NormCall's five, norm_inputs' six) -> (status, q_out, k_out or None, q's rows, k's rows or None)
PyObject* qk_norm_forward(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    TORCH_CHECK(n == 11, "qk_norm_forward: arguments");
    const NormCall c(args);
    const NormTensors t = norm_inputs(args + 5);
    if (PyErr_Occurred()) return nullptr;
    at::Tensor q_out, k_out;
    const int rc = without_gil([&] { return norm_run(c, t, q_out, k_out); });
    return tuple_of({PyLong_FromLong(rc), wrapped(q_out), wrapped(k_out), wrapped(t.q), wrapped(t.k)});
  });
}

// qk_norm_backward(NormCall's five, norm_inputs' six (the forward's rows; the weights themselves), gq, gk or None, whether
// the weights' gradients are wanted) -> (status, dq, dk or None, dwq or None, dwk or None)
PyObject* qk_norm_backward(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    TORCH_CHECK(n == 15, "qk_norm_backward: arguments");
    const NormCall c(args);
    const NormTensors t = norm_inputs(args + 5);
    const at::Tensor gq = optional(args[11]), gk = optional(args[12]);
    std::optional<at::ScalarType> types[2];
    for (int i = 0; i < 2; ++i)
      if (args[7 + i] != Py_None && PyObject_IsTrue(args[13 + i])) types[i] = tensor_of(args[7 + i]).scalar_type();
    if (PyErr_Occurred()) return nullptr;
    at::Tensor d[4];
    const int rc = without_gil([&] { return norm_back(c, t, gq, gk, types, d); });
    return tuple_of({PyLong_FromLong(rc), wrapped(d[0]), wrapped(d[1]), wrapped(d[2]), wrapped(d[3])});
  });
}

struct QkNormBackward : torch::autograd::Node {
  NormCall call;
  std::optional<at::ScalarType> types[2];
  SavedVariable q, k, wq, wk, positions, frequencies;
  std::mutex mutex;
  explicit QkNormBackward(const NormCall& c) : call(c) {}
  std::string name() const override { return "QkNormBackward"; }
  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex);
    for (SavedVariable* x : {&q, &k, &wq, &wk, &positions, &frequencies}) x->reset_data();
  }
  torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
    const std::lock_guard<std::mutex> lock(mutex);
    const bool recorded = at::GradMode::is_enabled();
    const at::AutoGradMode none(false);
    NormTensors t;
    t.q = q.unpack();
    t.k = k.unpack();
    t.wq = f32_of(wq.unpack());
    t.wk = f32_of(wk.unpack());
    t.positions = positions.unpack();
    t.frequencies = frequencies.unpack();
    at::Tensor d[4];
    const int rc = norm_back(call, t, grads[0], grads.size() > 1 ? grads[1] : at::Tensor(), types, d);
    TORCH_CHECK(rc == ESA_OK, "esa_qk_norm_bwd: status ", rc);
    return only_once({d[0], d[1], d[2], d[3]}, recorded);
  }
};

// qk_norm(NormCall's five, norm_inputs' six) -> (status, q_out, k_out or None), recorded where torch would
PyObject* qk_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    TORCH_CHECK(n == 11, "qk_norm: arguments");
    const NormCall c(args);
    const at::Tensor q = tensor_of(args[5]), k = optional(args[6]), wq = optional(args[7]), wk = optional(args[8]);
    if (PyErr_Occurred()) return nullptr;
    const bool record = at::GradMode::is_enabled() && (wants_grad(q) || wants_grad(k) || wants_grad(wq) || wants_grad(wk));
    at::Tensor q_out, k_out;
    NormTensors t;
    int rc;
    {
      const at::AutoGradMode none(false);
      t = norm_inputs(args + 5);
      rc = without_gil([&] { return norm_run(c, t, q_out, k_out); });
    }
    if (rc == ESA_OK && record) {
      std::shared_ptr<QkNormBackward> node(new QkNormBackward(c), torch::autograd::deleteNode);
      node->set_next_edges(torch::autograd::collect_next_edges(q, k, wq, wk));
      if (wants_grad(wq)) node->types[0] = wq.scalar_type();
      if (wants_grad(wk)) node->types[1] = wk.scalar_type();
      torch::autograd::set_history(q_out, node);
      if (k_out.defined()) torch::autograd::set_history(k_out, node);
      node->q = SavedVariable(t.q, false);
      node->k = SavedVariable(t.k, false);
      node->wq = SavedVariable(wq, false);
      node->wk = SavedVariable(wk, false);
      node->positions = SavedVariable(t.positions, false);
      node->frequencies = SavedVariable(t.frequencies, false);
    }
    return tuple_of({PyLong_FromLong(rc), wrapped(q_out), wrapped(k_out)});
  });
}

PyCFunction fast(PyObject* (*f)(PyObject*, PyObject* const*, Py_ssize_t)) { return reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(f)); }

PyMethodDef methods[] = {{"relative_fits", fast(relative_fits), METH_FASTCALL, nullptr},
                         {"relative", fast(relative), METH_FASTCALL, nullptr},
                         {"relative_forward", fast(relative_forward), METH_FASTCALL, nullptr},
                         {"relative_backward", fast(relative_backward), METH_FASTCALL, nullptr},
                         {"qk_norm_backward", fast(qk_norm_backward), METH_FASTCALL, nullptr},
                         {"qk_norm_fits", fast(qk_norm_fits), METH_FASTCALL, nullptr},
                         {"qk_norm", fast(qk_norm), METH_FASTCALL, nullptr},
                         {"qk_norm_forward", fast(qk_norm_forward), METH_FASTCALL, nullptr},
                         {"clip", fast(clip), METH_FASTCALL, nullptr},
                         {"describe", describe, METH_O, nullptr},
                         {"misfit", misfit, METH_VARARGS, nullptr},
                         {"separate", separate, METH_VARARGS, nullptr},
                         {"changed", changed, METH_O, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "esa_tensors", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_esa_tensors() { return PyModule_Create(&module); }
