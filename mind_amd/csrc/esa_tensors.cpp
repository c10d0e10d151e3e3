// Host side of calls over many tensors: a CPython module that reads what a
// launch needs from a list of torch tensors (pointer, count, dtype, layout,
// device) in one pass, and says whether the written ones share memory.  From
// Python each property of each tensor costs about 70 ns: a dozen of them for
// 768 gradients and their targets took 650 us, here 15 us.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstdint>
#include <exception>
#include <vector>

namespace {

constexpr int kF32 = 0, kBf16 = 1;   // ESA_F32, ESA_BF16

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

// describe(list) -> (pointers, counts, codes, device, contiguous): bytes of n void*, n int64 and n int32; device is the
// tensors' GPU, -1 if one is on the host, -2 if they are on several; contiguous tells whether all are.  A dtype other than
// float32 and bfloat16 raises TypeError.
PyObject* describe(PyObject*, PyObject* list) {
  return guarded([&]() -> PyObject* {
    if (!PyList_Check(list)) {
      PyErr_SetString(PyExc_TypeError, "a list of tensors is expected");
      return nullptr;
    }
    const Py_ssize_t n = PyList_GET_SIZE(list);
    std::vector<void*> ptrs(n + 1);   // (an empty array has an address, too)
    std::vector<int64_t> counts(n + 1);
    std::vector<int32_t> codes(n + 1);
    int device = 0;
    bool contiguous = true;
    for (Py_ssize_t i = 0; i < n; ++i) {
      PyObject* o = PyList_GET_ITEM(list, i);
      if (!THPVariable_Check(o)) {
        PyErr_Format(PyExc_TypeError, "tensors are expected (got %s)", Py_TYPE(o)->tp_name);
        return nullptr;
      }
      const at::Tensor& t = THPVariable_Unpack(o);
      if (t.scalar_type() != at::kFloat && t.scalar_type() != at::kBFloat16) {
        PyErr_Format(PyExc_TypeError, "tensors must be float32 or bfloat16 (got %s)", at::toString(t.scalar_type()));
        return nullptr;
      }
      if (t.layout() != at::kStrided) {
        PyErr_SetString(PyExc_TypeError, "tensors must be dense");
        return nullptr;
      }
      const int at = t.is_cuda() ? t.get_device() : -1;
      if (i == 0 || at == -1) device = at == -1 ? -1 : at;
      else if (device >= 0 && at != device) device = -2;
      contiguous = contiguous && t.is_contiguous() && !t.is_neg();
      codes[i] = t.scalar_type() == at::kFloat ? kF32 : kBf16;
      counts[i] = t.numel();
      ptrs[i] = t.data_ptr();
    }
    return Py_BuildValue("(y#y#y#iO)", reinterpret_cast<const char*>(ptrs.data()), (Py_ssize_t)(n * sizeof(void*)),
                         reinterpret_cast<const char*>(counts.data()), (Py_ssize_t)(n * sizeof(int64_t)),
                         reinterpret_cast<const char*>(codes.data()), (Py_ssize_t)(n * sizeof(int32_t)), device,
                         contiguous ? Py_True : Py_False);
  });
}

// misfit(tensors, targets) -> None, or what keeps a target from taking its tensor: "shapes", or "dtypes" (a target has
// its tensor's dtype or is float32).
PyObject* misfit(PyObject*, PyObject* args) {
  return guarded([&]() -> PyObject* {
    PyObject *a, *b;
    if (!PyArg_ParseTuple(args, "O!O!", &PyList_Type, &a, &PyList_Type, &b)) return nullptr;
    if (PyList_GET_SIZE(a) != PyList_GET_SIZE(b)) return PyUnicode_FromString("shapes");
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(a); ++i) {
      PyObject *x = PyList_GET_ITEM(a, i), *y = PyList_GET_ITEM(b, i);
      if (!THPVariable_Check(x) || !THPVariable_Check(y)) {
        PyErr_SetString(PyExc_TypeError, "tensors are expected");
        return nullptr;
      }
      const at::Tensor &t = THPVariable_Unpack(x), &u = THPVariable_Unpack(y);
      if (t.sizes() != u.sizes()) return PyUnicode_FromString("shapes");
      if (u.scalar_type() != t.scalar_type() && u.scalar_type() != at::kFloat) return PyUnicode_FromString("dtypes");
    }
    Py_RETURN_NONE;
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

// separate(written, read or None) -> bool, both (pointers, counts, codes) of describe: whether every written tensor keeps
// to itself.  No byte of it is another written tensor's, nor of another position's read tensor; its own read tensor may
// lie exactly there.
PyObject* separate(PyObject*, PyObject* args) {
  return guarded([&]() -> PyObject* {
    PyObject *written, *read;
    if (!PyArg_ParseTuple(args, "OO", &written, &read)) return nullptr;
    std::vector<Span> w, r;
    if (!spans_of(written, w) || (read != Py_None && !spans_of(read, r))) return nullptr;
    w.erase(std::remove_if(w.begin(), w.end(), [](const Span& s) { return s.end <= s.first; }), w.end());
    auto before = [](const Span& a, const Span& b) { return a.first < b.first; };
    if (!std::is_sorted(w.begin(), w.end(), before)) std::sort(w.begin(), w.end(), before);   // in a flat buffer they are
    for (size_t i = 1; i < w.size(); ++i)
      if (w[i].first < w[i - 1].end) Py_RETURN_FALSE;
    for (const Span& s : r) {
      if (s.end <= s.first || w.empty() || s.end <= w.front().first || s.first >= w.back().end) continue;
      // written spans are disjoint and in order: those that end behind s.first, up to the first beyond s.end
      auto it = std::upper_bound(w.begin(), w.end(), s.first, [](uint64_t at, const Span& b) { return at < b.end; });
      for (; it != w.end() && it->first < s.end; ++it)
        if (it->owner != s.owner || it->first != s.first || it->end != s.end) Py_RETURN_FALSE;
    }
    Py_RETURN_TRUE;
  });
}

// changed(list): the tensors' memory was written outside torch (what torch's own in-place operations count).
PyObject* changed(PyObject*, PyObject* list) {
  return guarded([&]() -> PyObject* {
    if (!PyList_Check(list)) {
      PyErr_SetString(PyExc_TypeError, "a list of tensors is expected");
      return nullptr;
    }
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(list); ++i) {
      PyObject* o = PyList_GET_ITEM(list, i);
      if (!THPVariable_Check(o)) continue;
      const at::Tensor& t = THPVariable_Unpack(o);
      if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
    }
    Py_RETURN_NONE;
  });
}

PyMethodDef methods[] = {{"describe", describe, METH_O, nullptr},
                         {"misfit", misfit, METH_VARARGS, nullptr},
                         {"separate", separate, METH_VARARGS, nullptr},
                         {"changed", changed, METH_O, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "esa_tensors", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_esa_tensors() { return PyModule_Create(&module); }
