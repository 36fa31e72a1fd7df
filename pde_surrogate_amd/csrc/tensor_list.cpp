// Host side of the list operators: reads a Python list of parameters -- their gradients, addresses, types, sizes, orders --
// in one call.  Through Python's own attribute look-ups the same takes about 0.1 us per tensor and question, 80 us for the 82
// parameters of the default DenseED and ten questions each; the kernels of such a step take under 10 us.
//
// A CPython module against the installed torch's headers (the only file here that knows torch's C++ types; the kernels' library
// does not link to it).  No function launches anything or keeps a reference; errors come back as numbers that adamw.py turns
// into messages, and no C++ exception leaves a function.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <algorithm>
#include <utility>
#include <vector>
#include <torch/csrc/autograd/python_variable.h>

namespace {

int code_of(at::ScalarType t) { return t == at::kFloat ? 0 : t == at::kBFloat16 ? 1 : t == at::kHalf ? 2 : -1; }

bool same_strides(const at::Tensor& a, const at::Tensor& b) {
  if (a.dim() != b.dim()) return false;
  for (int64_t d = 0; d < a.dim(); ++d)
    if (a.size(d) != 1 && a.stride(d) != b.stride(d)) return false;
  return true;
}
// element k of a's memory is element k of b's and of `like`'s, all of them dense
bool same_dense_order(const at::Tensor& a, const at::Tensor& b, const at::Tensor& like) {
  if (a.is_neg() || b.is_neg()) return false;          // (a lazy negation: the memory holds something else)
  if (a.is_contiguous() && b.is_contiguous() && like.is_contiguous()) return true;
  return a.is_non_overlapping_and_dense() && b.is_non_overlapping_and_dense() && same_strides(a, b) && same_strides(a, like);
}

bool as_list(PyObject* o) {
  if (PyList_Check(o)) return true;
  PyErr_SetString(PyExc_TypeError, "expected a list of tensors");
  return false;
}

template <class F>
PyObject* guarded(F&& f) {
  try {
    return f();
  } catch (const std::exception& e) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

unsigned long long* words(PyObject* o) { return static_cast<unsigned long long*>(PyLong_AsVoidPtr(o)); }

// gather(params, like, dtype, device, sizes, param_out, grad_out) -> place of the first parameter that is not a dense tensor of
// that element type on that device with that many elements, the memory order of its entry of `like` (the order of its state) and
// a gradient of the same kind and order; -1: all are, and the addresses have been written.  sizes, param_out, grad_out: addresses
// of arrays as long as the lists
PyObject* gather(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject* {
    if (nargs != 7 || !as_list(args[0]) || !as_list(args[1]) || PyList_GET_SIZE(args[0]) != PyList_GET_SIZE(args[1])) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "gather takes seven arguments, the first two of one length");
      return nullptr;
    }
    const long dtype = PyLong_AsLong(args[2]), device = PyLong_AsLong(args[3]);
    const unsigned long long *sizes = words(args[4]);
    unsigned long long *pout = words(args[5]), *gout = words(args[6]);
    if (PyErr_Occurred()) return nullptr;
    const Py_ssize_t n = PyList_GET_SIZE(args[0]);
    for (Py_ssize_t k = 0; k < n; ++k) {
      PyObject *o = PyList_GET_ITEM(args[0], k), *l = PyList_GET_ITEM(args[1], k);
      if (!THPVariable_Check(o) || !THPVariable_Check(l)) return PyLong_FromSsize_t(k);
      const at::Tensor& p = THPVariable_Unpack(o);
      const at::Tensor& g = p.grad();
      if (!g.defined() || p.layout() != at::kStrided || g.layout() != at::kStrided || !p.is_cuda() || !g.is_cuda() ||
          p.get_device() != device || g.get_device() != device || code_of(p.scalar_type()) != dtype || code_of(g.scalar_type()) != dtype ||
          (unsigned long long)p.numel() != sizes[k] || (unsigned long long)g.numel() != sizes[k] || 
          !same_dense_order(p, g, THPVariable_Unpack(l)))
        return PyLong_FromSsize_t(k);
      pout[k] = reinterpret_cast<unsigned long long>(p.data_ptr());
      gout[k] = reinterpret_cast<unsigned long long>(g.data_ptr());
    }
    return PyLong_FromLong(-1);
  });
}

// gradients(params, out, sizes) -> (count of float32, of bfloat16, of float16 gradients, their device, place of the first
// parameter whose gradient is not a dense device tensor of one of these types on one device, or -1, whether two gradients have
// memory in common).  out, sizes: addresses of arrays of three times the list's length, one third for each type
PyObject* gradients(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject* {
    if (nargs != 3 || !as_list(args[0])) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "gradients takes three arguments");
      return nullptr;
    }
    unsigned long long *out = words(args[1]), *sizes = words(args[2]);
    if (PyErr_Occurred()) return nullptr;
    const Py_ssize_t n = PyList_GET_SIZE(args[0]);
    Py_ssize_t count[3] = {0, 0, 0}, bad = -1;
    int device = -1;
    for (Py_ssize_t k = 0; k < n && bad < 0; ++k) {
      PyObject* o = PyList_GET_ITEM(args[0], k);
      if (!THPVariable_Check(o)) { bad = k; break; }
      const at::Tensor& g = THPVariable_Unpack(o).grad();
      if (!g.defined()) continue;
      const int c = code_of(g.scalar_type());
      if (g.layout() != at::kStrided || !g.is_cuda() || c < 0 || (device >= 0 && g.get_device() != device) ||
          !(g.is_contiguous() || g.is_non_overlapping_and_dense())) { bad = k; break; }
      device = g.get_device();
      out[c * n + count[c]] = reinterpret_cast<unsigned long long>(g.data_ptr());
      sizes[c * n + count[c]++] = (unsigned long long)g.numel();
    }
    std::vector<std::pair<unsigned long long, unsigned long long>> used;         // first byte, byte behind the last
    used.reserve(n);
    for (int c = 0; c < 3; ++c)
      for (Py_ssize_t k = 0; k < count[c]; ++k)
        if (sizes[c * n + k]) used.emplace_back(out[c * n + k], out[c * n + k] + sizes[c * n + k] * (c == 0 ? 4 : 2));
    std::sort(used.begin(), used.end());
    bool shared = false;
    for (size_t k = 1; k < used.size(); ++k) shared |= used[k].first < used[k - 1].second;
    return Py_BuildValue("nnnini", count[0], count[1], count[2], device, bad, (int)shared);
  });
}

// overlap(lists) -> whether two stretches of memory have bytes in common.  lists: tuples (address of an array of addresses, of one
// of numbers of elements, how many, bytes of an element)
PyObject* overlap(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject* {
    if (nargs != 1 || !as_list(args[0])) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "overlap takes a list");
      return nullptr;
    }
    struct List {
      const unsigned long long *at, *size;
      Py_ssize_t count;
      unsigned long long item;
    };
    std::vector<List> lists;
    unsigned long long end = 0;
    size_t many = 0;
    bool apart = true;                     // each stretch behind the one before, as they mostly are: nothing to sort
    for (Py_ssize_t j = 0; j < PyList_GET_SIZE(args[0]); ++j) {
      unsigned long long a, b;
      List x;
      if (!PyTuple_Check(PyList_GET_ITEM(args[0], j))) {
        PyErr_SetString(PyExc_TypeError, "overlap takes a list of tuples");
        return nullptr;
      }
      if (!PyArg_ParseTuple(PyList_GET_ITEM(args[0], j), "KKnK", &a, &b, &x.count, &x.item)) return nullptr;
      x.at = reinterpret_cast<const unsigned long long*>(a);
      x.size = reinterpret_cast<const unsigned long long*>(b);
      for (Py_ssize_t k = 0; apart && k < x.count; ++k)
        if (x.size[k]) {
          apart = x.at[k] >= end;
          end = x.at[k] + x.size[k] * x.item;
        }
      many += x.count;
      lists.push_back(x);
    }
    if (apart) Py_RETURN_FALSE;
    std::vector<std::pair<unsigned long long, unsigned long long>> used;         // first byte, byte behind the last
    used.reserve(many);
    for (const List& x : lists)
      for (Py_ssize_t k = 0; k < x.count; ++k)
        if (x.size[k]) used.emplace_back(x.at[k], x.at[k] + x.size[k] * x.item);
    std::sort(used.begin(), used.end());
    for (size_t k = 1; k < used.size(); ++k)
      if (used[k].first < used[k - 1].second) Py_RETURN_TRUE;
    Py_RETURN_FALSE;
  });
}

// fits(groups, params, mask) -> whether the lists of parameters in `groups` are, one behind the other, these very objects, and
// those with a gradient are the ones that `mask` (bytes) marks
// fits(groups, params, mask, known) -> the same of an optimiser's groups: they are the very dictionaries in `known` (a list of each
// and its number of parameters), and whether the marked parameters still have a gradient is left to gather, which looks at them
PyObject* fits(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject* {
    static PyObject* const name = PyUnicode_InternFromString("params");
    PyObject* const known = nargs == 4 ? args[3] : nullptr;
    if (nargs < 3 || nargs > 4 || !as_list(args[0]) || !as_list(args[1]) || !PyBytes_Check(args[2]) ||
        PyBytes_GET_SIZE(args[2]) != PyList_GET_SIZE(args[1]) || (known && !as_list(known))) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "fits takes a list of lists, a list and as many bytes");
      return nullptr;
    }
    const char* mask = PyBytes_AS_STRING(args[2]);
    const Py_ssize_t n = PyList_GET_SIZE(args[1]);
    Py_ssize_t at = 0;
    if (known && PyList_GET_SIZE(known) != 2 * PyList_GET_SIZE(args[0])) Py_RETURN_FALSE;
    for (Py_ssize_t j = 0; j < PyList_GET_SIZE(args[0]); ++j) {
      PyObject* group = PyList_GET_ITEM(args[0], j);
      if (known) {
        if (group != PyList_GET_ITEM(known, 2 * j) || !PyDict_Check(group) || !(group = PyDict_GetItemWithError(group, name))) Py_RETURN_FALSE;
        if (!PyList_Check(group) || PyList_GET_SIZE(group) != PyLong_AsSsize_t(PyList_GET_ITEM(known, 2 * j + 1))) Py_RETURN_FALSE;
      }
      if (!as_list(group)) return nullptr;
      for (Py_ssize_t k = 0; k < PyList_GET_SIZE(group); ++k, ++at) {
        PyObject* o = PyList_GET_ITEM(group, k);
        if (at >= n || o != PyList_GET_ITEM(args[1], at)) Py_RETURN_FALSE;
        if (known && mask[at]) continue;
        if (!THPVariable_Check(o) || THPVariable_Unpack(o).grad().defined() != (mask[at] != 0)) Py_RETURN_FALSE;
      }
    }
    if (at != n) Py_RETURN_FALSE;
    Py_RETURN_TRUE;
  });
}

// ---- the states of an optimiser, compared with what they were
// `known`: for each parameter the parameter, the dictionary of its state, pairs of a name and a tensor, and None, in the order of
// the dictionaries; `dicts`: those dictionaries; `tensors`: those tensors, each once.  A note is an array of 1 + len(dicts) + 2
// len(tensors) numbers: the version of `state`, of each dictionary, and where each tensor's memory is

// changes with every change of a dictionary and is never the same for two (0: this Python has none, and every dictionary is read)
uint64_t version_of(PyObject* dict) {
#if PY_VERSION_HEX < 0x030C0000
  return reinterpret_cast<PyDictObject*>(dict)->ma_version_tag;
#else
  return 0;
#endif
}
// a tensor's storage, which views of one buffer share (0: it has none), and its place there
struct Place {
  unsigned long long storage, offset;
};
inline Place place_of(const at::Tensor& t) {
  const c10::TensorImpl* impl = t.unsafeGetTensorImpl();
  return {reinterpret_cast<unsigned long long>(impl->unsafe_storage().unsafeGetStorageImpl()), static_cast<unsigned long long>(impl->storage_offset())};
}
void note_versions(PyObject* state, PyObject* dicts, unsigned long long* note) {
  *note++ = version_of(state);
  for (Py_ssize_t k = 0; k < PyList_GET_SIZE(dicts); ++k) *note++ = version_of(PyList_GET_ITEM(dicts, k));
}
// whether the dictionaries hold what `known` lists; what else they hold is the program's own
bool as_known(PyObject* dict, PyObject* known) {
  const Py_ssize_t n = PyList_GET_SIZE(known);
  Py_ssize_t k = 0, i = 0;
  PyObject *p, *state, *name, *value;
  while (k < n && PyDict_Next(dict, &i, &p, &state)) {
    if (p != PyList_GET_ITEM(known, k)) continue;
    if (++k >= n || state != PyList_GET_ITEM(known, k)) return false;
    ++k;
    Py_ssize_t j = 0;
    while (k + 1 < n && PyList_GET_ITEM(known, k) != Py_None && PyDict_Next(state, &j, &name, &value)) {
      if (name != PyList_GET_ITEM(known, k)) continue;
      if (value != PyList_GET_ITEM(known, k + 1)) return false;
      k += 2;
    }
    if (k >= n || PyList_GET_ITEM(known, k) != Py_None) return false;
    ++k;
  }
  return k == n;
}
bool all_dicts(PyObject* list) {
  for (Py_ssize_t k = 0; k < PyList_GET_SIZE(list); ++k)
    if (!PyDict_Check(PyList_GET_ITEM(list, k))) return false;
  return true;
}

// note(state, dicts, tensors, out)
PyObject* note(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject* {
    if (nargs != 4 || !PyDict_Check(args[0]) || !as_list(args[1]) || !as_list(args[2]) || !all_dicts(args[1])) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "note takes a dictionary, a list of them, a list of tensors and an address");
      return nullptr;
    }
    unsigned long long* out = words(args[3]);
    if (PyErr_Occurred()) return nullptr;
    note_versions(args[0], args[1], out);
    out += 1 + PyList_GET_SIZE(args[1]);
    for (Py_ssize_t k = 0; k < PyList_GET_SIZE(args[2]); ++k) {
      if (!THPVariable_Check(PyList_GET_ITEM(args[2], k))) {
        PyErr_SetString(PyExc_TypeError, "note takes a list of tensors");
        return nullptr;
      }
      const Place place = place_of(THPVariable_Unpack(PyList_GET_ITEM(args[2], k)));
      *out++ = place.storage;
      *out++ = place.offset;
    }
    Py_RETURN_NONE;
  });
}

// held(state, known, dicts, tensors, note) -> whether nothing of it has been replaced since the note was made
PyObject* held(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject* {
    if (nargs != 5 || !PyDict_Check(args[0]) || !as_list(args[1]) || !as_list(args[2]) || !as_list(args[3])) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "held takes a dictionary, three lists and an address");
      return nullptr;
    }
    unsigned long long* noted = words(args[4]);
    if (PyErr_Occurred()) return nullptr;
    const Py_ssize_t n = PyList_GET_SIZE(args[2]);
    bool same = noted[0] != 0 && version_of(args[0]) == noted[0];
    for (Py_ssize_t k = 0; same && k < n; ++k) same = version_of(PyList_GET_ITEM(args[2], k)) == noted[1 + k];
    if (!same) {
      if (!as_known(args[0], args[1])) Py_RETURN_FALSE;
      note_versions(args[0], args[2], noted);
    }
    const unsigned long long* at = noted + 1 + n;
    const Py_ssize_t m = PyList_GET_SIZE(args[3]);             // (all of them tensors: note has made sure)
    for (Py_ssize_t k = 0; k < m; ++k, at += 2) {
      const Place place = place_of(THPVariable_Unpack(PyList_GET_ITEM(args[3], k)));
      if (place.storage != at[0] || place.offset != at[1]) Py_RETURN_FALSE;
    }
    Py_RETURN_TRUE;
  });
}

// changed(params, gradients): autograd's version counters move, as after any in-place change, of the tensors or their gradients
PyObject* changed(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject* {
    if (nargs != 2 || !as_list(args[0])) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "changed takes two arguments");
      return nullptr;
    }
    const bool grads = PyObject_IsTrue(args[1]) == 1;
    for (Py_ssize_t k = 0; k < PyList_GET_SIZE(args[0]); ++k) {
      PyObject* o = PyList_GET_ITEM(args[0], k);
      if (!THPVariable_Check(o)) continue;
      const at::Tensor& p = THPVariable_Unpack(o);
      const at::Tensor& t = grads ? p.grad() : p;
      if (t.defined() && !t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
    }
    Py_RETURN_NONE;
  });
}

PyMethodDef methods[] = {
    {"gather", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(gather)), METH_FASTCALL, nullptr},
    {"gradients", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(gradients)), METH_FASTCALL, nullptr},
    {"overlap", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(overlap)), METH_FASTCALL, nullptr},
    {"fits", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(fits)), METH_FASTCALL, nullptr},
    {"note", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(note)), METH_FASTCALL, nullptr},
    {"held", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(held)), METH_FASTCALL, nullptr},
    {"changed", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(changed)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensor_list", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensor_list(void) { return PyModule_Create(&module); }
