// Host side of calls whose time is the host's: a CPython module against torch's
// headers.  From Python each property of a tensor costs about 70 ns.
//
// Calls over many tensors: it reads what a launch needs from a list of tensors
// (pointer, count, dtype, layout, device) in one pass, and says whether the
// written ones share memory (a dozen properties of 768 gradients and their
// targets took 650 us, here 15 us).
// Calls over small batches, whose kernels take 10 us: the checks of a call's
// arguments, its outputs and workspace and the call of the C entry in one
// function each (with their Python form a forward took 21 to 25 us of
// host time, now 8 to 12; the body of a small backward 46, now 30).
// The Python callers keep the checks' messages: a check here only says whether
// there is anything to look at.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstdint>
#include <exception>
#include <vector>

#include "../../include/esa_hip.h"

namespace {

constexpr int kF32 = ESA_F32, kBf16 = ESA_BF16;

// C++ exceptions (torch's errors among them) end here as Python's.
template <class F>
PyObject* guarded(F f) {
  try {
    return f();
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

// What the checks say of a call: its arguments fit, all tensors are of torch's own types, one wants a gradient.
constexpr long kFits = 1, kExact = 2, kGrad = 4;

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
    if (t.requires_grad()) flags |= kGrad;
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

template <class F>
int without_gil(F f) {
  int rc;
  Py_BEGIN_ALLOW_THREADS rc = f();
  Py_END_ALLOW_THREADS return rc;
}

at::Tensor bytes_on(const at::Tensor& like, size_t bytes) {
  return at::empty({(int64_t)std::max<size_t>(bytes, 256)}, like.options().dtype(at::kByte));
}

// relative_forward(address of esa_rel_attn_fwd, of its size query, stream, q, k, v, bias, starts (bytes of int32), q_start,
// cu_q, cu_k, scale, dropout_p, seed, keep) -> (status, out, out_low or None, lse, the table); keep: out_low is wanted.
PyObject* relative_forward(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    TORCH_CHECK(n == 15 && PyBytes_Check(args[7]), "relative_forward: arguments");
    const auto fn = reinterpret_cast<decltype(&esa_rel_attn_fwd)>(PyLong_AsVoidPtr(args[0]));
    const auto size_of = reinterpret_cast<decltype(&esa_rel_attn_workspace_size)>(PyLong_AsVoidPtr(args[1]));
    void* stream = PyLong_AsVoidPtr(args[2]);
    const at::Tensor &q = tensor_of(args[3]), &k = tensor_of(args[4]), &v = tensor_of(args[5]);
    const at::Tensor table = tensor_of(args[6]).contiguous();
    const int* starts = reinterpret_cast<const int*>(PyBytes_AS_STRING(args[7]));
    const int side = (int)(PyBytes_GET_SIZE(args[7]) / sizeof(int)), buckets = (int)table.size(0);
    const int* q_start = static_cast<const int*>(pointer_of(args[8]));
    const at::Tensor &cu_q = tensor_of(args[9]), &cu_k = tensor_of(args[10]);
    const float scale = (float)PyFloat_AsDouble(args[11]), dropout = (float)PyFloat_AsDouble(args[12]);
    const unsigned long long seed = PyLong_AsUnsignedLongLong(args[13]);
    const bool keep = PyObject_IsTrue(args[14]) && q.scalar_type() == at::kBFloat16;
    if (PyErr_Occurred()) return nullptr;
    TORCH_CHECK(q.size(0) <= INT32_MAX && k.size(0) <= INT32_MAX && q.size(1) <= INT32_MAX && cu_q.numel() <= INT32_MAX,
                "sizes beyond 32 bits");
    const int batch = (int)cu_q.numel() - 1, tq = (int)q.size(0), tk = (int)k.size(0), heads = (int)q.size(1), hd = (int)q.size(2);
    const c10::DeviceGuard on(q.device());
    at::Tensor out, low, lse, ws;
    size_t bytes = 0;
    int rc = size_of(batch, tq, tk, heads, hd, code_of(q), buckets, starts, side, 0, &bytes);
    if (rc == ESA_OK) {
      out = at::empty(q.sizes(), q.options());
      if (keep) low = at::empty(q.sizes(), q.options());
      lse = at::empty({heads, tq}, q.options().dtype(at::kFloat));
      ws = bytes_on(q, bytes);
      rc = without_gil([&] {
        return fn(q.data_ptr(), k.data_ptr(), v.data_ptr(), table.data_ptr(), code_of(table), buckets, starts, side, q_start,
                  cu_q.data_ptr<int>(), cu_k.data_ptr<int>(), batch, tq, tk, heads, hd, code_of(q), scale, dropout, seed,
                  out.data_ptr(), keep ? low.data_ptr() : nullptr, lse.data_ptr<float>(), ws.data_ptr(), (size_t)ws.numel(),
                  stream);
      });
    }
    return tuple_of({PyLong_FromLong(rc), wrapped(out), wrapped(low), wrapped(lse), wrapped(table)});
  });
}

// A gradient as the kernels take it: dense, by value, on a 16-byte boundary.
at::Tensor gradient_of(PyObject* o) {
  const at::Tensor g = tensor_of(o).resolve_neg().contiguous();
  return reinterpret_cast<uintptr_t>(g.data_ptr()) % 16 ? g.clone() : g;
}

// relative_backward(address of esa_rel_attn_bwd, of its size query, stream, dout, q, k, v, out, out_low, lse, table, starts,
// q_start, cu_q, cu_k, scale, dropout_p, seed) -> (status, dq, dk, dv, dtable in the table's type); arguments as the
// forward's and its results
PyObject* relative_backward(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    TORCH_CHECK(n == 18 && PyBytes_Check(args[11]), "relative_backward: arguments");
    const auto fn = reinterpret_cast<decltype(&esa_rel_attn_bwd)>(PyLong_AsVoidPtr(args[0]));
    const auto size_of = reinterpret_cast<decltype(&esa_rel_attn_workspace_size)>(PyLong_AsVoidPtr(args[1]));
    void* stream = PyLong_AsVoidPtr(args[2]);
    const at::Tensor &q = tensor_of(args[4]), &k = tensor_of(args[5]), &v = tensor_of(args[6]), &out = tensor_of(args[7]);
    const void* low = pointer_of(args[8]);
    const at::Tensor &lse = tensor_of(args[9]), &table = tensor_of(args[10]);
    const int* starts = reinterpret_cast<const int*>(PyBytes_AS_STRING(args[11]));
    const int side = (int)(PyBytes_GET_SIZE(args[11]) / sizeof(int)), buckets = (int)table.size(0);
    const int* q_start = static_cast<const int*>(pointer_of(args[12]));
    const at::Tensor &cu_q = tensor_of(args[13]), &cu_k = tensor_of(args[14]);
    const float scale = (float)PyFloat_AsDouble(args[15]), dropout = (float)PyFloat_AsDouble(args[16]);
    const unsigned long long seed = PyLong_AsUnsignedLongLong(args[17]);
    if (PyErr_Occurred()) return nullptr;
    const int batch = (int)cu_q.numel() - 1, tq = (int)q.size(0), tk = (int)k.size(0), heads = (int)q.size(1), hd = (int)q.size(2);
    const c10::DeviceGuard on(q.device());
    const at::Tensor g = gradient_of(args[3]);
    at::Tensor dq, dk, dv, dtable;
    size_t bytes = 0;
    int rc = size_of(batch, tq, tk, heads, hd, code_of(q), buckets, starts, side, 1, &bytes);
    if (rc == ESA_OK) {
      dq = at::empty(q.sizes(), q.options());
      dk = at::empty(k.sizes(), k.options());
      dv = at::empty(v.sizes(), v.options());
      dtable = at::empty(table.sizes(), table.options().dtype(at::kFloat));
      const at::Tensor ws = bytes_on(q, bytes);
      rc = without_gil([&] {
        return fn(g.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), low, lse.data_ptr<float>(),
                  table.data_ptr(), code_of(table), buckets, starts, side, q_start, cu_q.data_ptr<int>(), cu_k.data_ptr<int>(),
                  batch, tq, tk, heads, hd, code_of(q), scale, dropout, seed, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                  dtable.data_ptr<float>(), ws.data_ptr(), (size_t)ws.numel(), stream);
      });
      if (rc == ESA_OK && table.scalar_type() != at::kFloat) dtable = dtable.to(table.scalar_type());
    }
    return tuple_of({PyLong_FromLong(rc), wrapped(dq), wrapped(dk), wrapped(dv), wrapped(dtable)});
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

// qk_norm_forward(address of esa_qk_norm_fwd, stream, q, k, wq, wk (float32), positions, frequencies, eps, interleaved) ->
// (status, q_out, k_out or None, q's rows, k's rows or None)
PyObject* qk_norm_forward(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    TORCH_CHECK(n == 10, "qk_norm_forward: arguments");
    const auto fn = reinterpret_cast<decltype(&esa_qk_norm_fwd)>(PyLong_AsVoidPtr(args[0]));
    void* stream = PyLong_AsVoidPtr(args[1]);
    const at::Tensor q = rows_of(tensor_of(args[2]));
    at::Tensor k;
    if (args[3] != Py_None) k = rows_of(tensor_of(args[3]));
    const float *wq = static_cast<const float*>(pointer_of(args[4])), *wk = static_cast<const float*>(pointer_of(args[5]));
    const void* positions = pointer_of(args[6]);
    const int positions_bytes = positions || args[6] != Py_None ? (int)tensor_of(args[6]).element_size() : 0;
    const double* frequencies = static_cast<const double*>(pointer_of(args[7]));
    const int rotary = args[7] != Py_None ? 2 * (int)tensor_of(args[7]).numel() : 0;
    const float eps = (float)PyFloat_AsDouble(args[8]);
    const int interleaved = PyObject_IsTrue(args[9]);
    if (PyErr_Occurred()) return nullptr;
    TORCH_CHECK(q.size(0) <= INT32_MAX, "sizes beyond 32 bits");
    const long long strides[4] = {q.stride(0), q.stride(1), k.defined() ? k.stride(0) : 0, k.defined() ? k.stride(1) : 0};
    const c10::DeviceGuard on(q.device());
    const at::Tensor q_out = at::empty(q.sizes(), q.options());
    at::Tensor k_out;
    if (k.defined()) k_out = at::empty(k.sizes(), k.options());
    const int rc = without_gil([&] {
      return fn(q.data_ptr(), k.defined() ? k.data_ptr() : nullptr, strides, (int)q.size(0), (int)q.size(1),
                k.defined() ? (int)k.size(1) : 0, (int)q.size(2), code_of(q), wq, wk, positions, positions_bytes, frequencies,
                rotary, interleaved, eps, q_out.data_ptr(), k_out.defined() ? k_out.data_ptr() : nullptr, stream);
    });
    return tuple_of({PyLong_FromLong(rc), wrapped(q_out), wrapped(k_out), wrapped(q), wrapped(k)});
  });
}

// qk_norm_backward(address of esa_qk_norm_bwd, of its size query, stream, gq, gk, q, k, wq, wk, positions, frequencies, eps,
// interleaved, type code of dwq or None, of dwk) -> (status, dq, dk or None, dwq or None, dwk or None); q and k the rows
// that the forward returned; type codes: ESA_F32, ESA_BF16
PyObject* qk_norm_backward(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    TORCH_CHECK(n == 15, "qk_norm_backward: arguments");
    const auto fn = reinterpret_cast<decltype(&esa_qk_norm_bwd)>(PyLong_AsVoidPtr(args[0]));
    const auto size_of = reinterpret_cast<decltype(&esa_qk_norm_bwd_workspace_size)>(PyLong_AsVoidPtr(args[1]));
    void* stream = PyLong_AsVoidPtr(args[2]);
    const at::Tensor& q = tensor_of(args[5]);
    const bool keys = args[6] != Py_None;
    const at::Tensor& k = keys ? tensor_of(args[6]) : q;
    const float *wq = static_cast<const float*>(pointer_of(args[7])), *wk = static_cast<const float*>(pointer_of(args[8]));
    const void* positions = pointer_of(args[9]);
    const int positions_bytes = args[9] != Py_None ? (int)tensor_of(args[9]).element_size() : 0;
    const double* frequencies = static_cast<const double*>(pointer_of(args[10]));
    const int rotary = args[10] != Py_None ? 2 * (int)tensor_of(args[10]).numel() : 0;
    const float eps = (float)PyFloat_AsDouble(args[11]);
    const int interleaved = PyObject_IsTrue(args[12]);
    const long code[2] = {args[13] == Py_None ? -1 : PyLong_AsLong(args[13]), args[14] == Py_None ? -1 : PyLong_AsLong(args[14])};
    if (PyErr_Occurred()) return nullptr;
    const long long strides[4] = {q.stride(0), q.stride(1), keys ? k.stride(0) : 0, keys ? k.stride(1) : 0};
    const int total = (int)q.size(0), hd = (int)q.size(2);
    const c10::DeviceGuard on(q.device());
    const at::Tensor gq = gradient_of(args[3]), dq = at::empty(q.sizes(), q.options());
    at::Tensor gk, dk, dw[2], ws;
    if (keys) {
      gk = gradient_of(args[4]);
      dk = at::empty(k.sizes(), k.options());
    }
    int rc = ESA_OK;
    for (int i = 0; i < 2; ++i)
      if (code[i] >= 0) dw[i] = at::empty({hd}, q.options().dtype(at::kFloat));
    if (dw[0].defined() || dw[1].defined()) {
      size_t bytes = 0;
      rc = size_of(total, hd, &bytes);
      if (rc == ESA_OK) ws = bytes_on(q, bytes);
    }
    if (rc == ESA_OK)
      rc = without_gil([&] {
        return fn(gq.data_ptr(), keys ? gk.data_ptr() : nullptr, q.data_ptr(), keys ? k.data_ptr() : nullptr, strides, total,
                  (int)q.size(1), keys ? (int)k.size(1) : 0, hd, code_of(q), wq, wk, positions, positions_bytes, frequencies,
                  rotary, interleaved, eps, dq.data_ptr(), keys ? dk.data_ptr() : nullptr,
                  dw[0].defined() ? dw[0].data_ptr<float>() : nullptr, dw[1].defined() ? dw[1].data_ptr<float>() : nullptr,
                  ws.defined() ? ws.data_ptr() : nullptr, ws.defined() ? (size_t)ws.numel() : 0, stream);
      });
    for (int i = 0; i < 2; ++i)
      if (rc == ESA_OK && code[i] == kBf16) dw[i] = dw[i].to(at::kBFloat16);
    return tuple_of({PyLong_FromLong(rc), wrapped(dq), wrapped(dk), wrapped(dw[0]), wrapped(dw[1])});
  });
}

PyCFunction fast(PyObject* (*f)(PyObject*, PyObject* const*, Py_ssize_t)) { return reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(f)); }

PyMethodDef methods[] = {{"relative_fits", fast(relative_fits), METH_FASTCALL, nullptr},
                         {"relative_forward", fast(relative_forward), METH_FASTCALL, nullptr},
                         {"relative_backward", fast(relative_backward), METH_FASTCALL, nullptr},
                         {"qk_norm_backward", fast(qk_norm_backward), METH_FASTCALL, nullptr},
                         {"qk_norm_fits", fast(qk_norm_fits), METH_FASTCALL, nullptr},
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
