// Calls of the cached-decoding kernels from torch tensors (Python module
// hackathon_b200._torch_call, built where torch is installed).
//
// A decode step makes these calls once for each layer, on buffers whose shapes
// repeat, and its kernels take a few microseconds: the time to describe eight
// tensors in Python would be most of a call.  Here a call's signature (types,
// shapes, device, attributes) is looked up among those already checked; the
// checks themselves, and the records of a new signature, are made in Python
// (kernel_registry.py).  Only what follows from the signature is kept.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>
#include <string>
#include <unordered_map>
#include <utility>
#include <vector>

#include "c3b200.h"

namespace {

typedef int (*LaunchFn)(int, const c3b_tensor*, int, const c3b_tensor*, int, const void*, size_t, void*);
typedef const char* (*ErrorFn)();
LaunchFn g_launch = nullptr;
ErrorFn g_error = nullptr;

struct Ready {
  int kid = 0, n_in = 0;
  std::vector<c3b_tensor> records;  // inputs, then outputs; addresses are filled in for each call
  std::string params;
  int64_t workspace = 0;            // bytes of a last output that the caller did not bring
  std::vector<std::pair<Py_ssize_t, PyObject*>> shapes;  // outputs given in another shape than their logical one
};

struct State {
  PyObject_HEAD
  std::string* name;
  std::unordered_map<std::string, Ready>* kept;
};

void release(Ready& r) {
  for (auto& s : r.shapes) Py_DECREF(s.second);
}

void forget(State* s) {
  for (auto& e : *s->kept) release(e.second);
  s->kept->clear();
}

template <typename T>
void put(std::string& key, T v) {
  key.append(reinterpret_cast<const char*>(&v), sizeof(T));
}

// Adds the tensors of a sequence to the key.  0: done, 1: not torch tensors, -1: an error is set.
int describe(PyObject* items, std::string& key, std::vector<const at::Tensor*>& tensors, int& device) {
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(items);
  PyObject** at_ = PySequence_Fast_ITEMS(items);
  put(key, (int32_t)n);
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* o = at_[i];
    if (o == Py_None) {
      put(key, (int16_t)-1);
      continue;
    }
    if (!THPVariable_Check(o)) return 1;
    const at::Tensor& t = THPVariable_Unpack(o);
    if (t.layout() != at::kStrided) return 1;
    if (!t.is_cuda()) {
      PyErr_SetString(PyExc_TypeError, "kernel arrays must live on the GPU");
      return -1;
    }
    if (!t.is_contiguous()) {
      PyErr_SetString(PyExc_ValueError, "kernel arrays must be C-contiguous");
      return -1;
    }
    const int d = t.get_device();
    if (device >= 0 && d != device) {
      PyErr_SetString(PyExc_ValueError, "kernel arrays on different devices");
      return -1;
    }
    device = d;
    put(key, (int16_t)t.scalar_type());
    put(key, (int16_t)t.dim());
    for (int64_t s : t.sizes()) put(key, s);
    tensors.push_back(&t);
  }
  return 0;
}

// Adds the attributes to the key: names and numbers.  1: something else is among them.
int attributes(PyObject* params, std::string& key) {
  if (params == Py_None) return 0;
  if (!PyDict_Check(params)) return 1;
  PyObject *k, *v;
  Py_ssize_t pos = 0;
  while (PyDict_Next(params, &pos, &k, &v)) {
    Py_ssize_t len;
    const char* name = PyUnicode_Check(k) ? PyUnicode_AsUTF8AndSize(k, &len) : nullptr;
    if (!name) {
      PyErr_Clear();
      return 1;
    }
    put(key, (int32_t)len);
    key.append(name, (size_t)len);
    if (v == Py_None) {
      key.push_back('n');
    } else if (PyFloat_Check(v)) {
      key.push_back('f');
      put(key, PyFloat_AS_DOUBLE(v));
    } else if (PyLong_Check(v)) {
      const long long x = PyLong_AsLongLong(v);
      if (x == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        return 1;
      }
      key.push_back('i');
      put(key, x);
    } else {
      return 1;
    }
  }
  return 0;
}

// call(inputs, outputs, params) -> None when launched, the signature (bytes) when it is new,
// NotImplemented for arrays or attributes that the general path takes.
PyObject* state_call(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  State* s = reinterpret_cast<State*>(self);
  if (nargs != 3 || !PyList_Check(args[1]) || !(PyList_Check(args[0]) || PyTuple_Check(args[0]))) Py_RETURN_NOTIMPLEMENTED;
  try {
    std::string key;
    key.reserve(512);
    std::vector<const at::Tensor*> tensors;
    tensors.reserve(16);
    int device = -1;
    for (int i = 0; i < 2; ++i) {
      const int rc = describe(args[i], key, tensors, device);
      if (rc < 0) return nullptr;
      if (rc > 0) Py_RETURN_NOTIMPLEMENTED;
    }
    if (device < 0 || attributes(args[2], key)) Py_RETURN_NOTIMPLEMENTED;
    put(key, (int32_t)device);
    const auto found = s->kept->find(key);
    if (found == s->kept->end()) return PyBytes_FromStringAndSize(key.data(), (Py_ssize_t)key.size());
    const Ready& r = found->second;
    const c10::cuda::OptionalCUDAGuard guard(c10::Device(c10::DeviceType::CUDA, (c10::DeviceIndex)device));
    c3b_tensor rec[24];
    const size_t n = r.records.size();
    memcpy(rec, r.records.data(), n * sizeof(c3b_tensor));
    for (size_t i = 0; i < tensors.size(); ++i) rec[i].ptr = tensors[i]->data_ptr();
    c10::DataPtr scratch;
    if (r.workspace) {
      scratch = c10::cuda::CUDACachingAllocator::get()->allocate((size_t)r.workspace);
      rec[n - 1].ptr = scratch.get();
    }
    const int rc = g_launch(r.kid, rec, r.n_in, rec + r.n_in, (int)n - r.n_in, r.params.data(), r.params.size(),
                            c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream());
    if (rc < 0) {
      PyErr_Format(PyExc_RuntimeError, "%s failed (%d): %s", s->name->c_str(), rc, g_error());
      return nullptr;
    }
    if (r.shapes.empty()) Py_RETURN_NONE;
    // `view` is Python's: hold the shapes, since what it runs may make calls of its own
    std::vector<std::pair<Py_ssize_t, PyObject*>> shapes(r.shapes);
    for (auto& v : shapes) Py_INCREF(v.second);
    bool ok = true;
    for (auto& v : shapes) {
      PyObject* view = ok ? PyObject_CallMethod(PyList_GET_ITEM(args[1], v.first), "view", "O", v.second) : nullptr;
      ok = ok && view && PyList_SetItem(args[1], v.first, view) == 0;
      Py_DECREF(v.second);
    }
    if (!ok) return nullptr;
    Py_RETURN_NONE;
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// add(signature, kid, n_in, records, params, workspace, shapes): what a signature's launches need.
PyObject* state_add(PyObject* self, PyObject* args) {
  State* s = reinterpret_cast<State*>(self);
  const char *sig, *rec, *par;
  Py_ssize_t nsig, nrec, npar;
  int kid, n_in;
  long long workspace;
  PyObject* shapes;
  if (!PyArg_ParseTuple(args, "y#iiy#y#LO!", &sig, &nsig, &kid, &n_in, &rec, &nrec, &par, &npar, &workspace, &PyList_Type,
                        &shapes))
    return nullptr;
  const size_t n = (size_t)nrec / sizeof(c3b_tensor);
  if ((size_t)nrec % sizeof(c3b_tensor) || n > 24 || n_in < 0 || (size_t)n_in > n) {
    PyErr_SetString(PyExc_ValueError, "bad records");
    return nullptr;
  }
  if (s->kept->size() >= 512) forget(s);
  Ready r;
  r.kid = kid, r.n_in = n_in, r.workspace = workspace;
  r.records.resize(n);
  memcpy(r.records.data(), rec, (size_t)nrec);
  r.params.assign(par, (size_t)npar);
  for (Py_ssize_t i = 0; i < PyList_GET_SIZE(shapes); ++i) {
    Py_ssize_t at_;
    PyObject* shape;
    if (!PyArg_ParseTuple(PyList_GET_ITEM(shapes, i), "nO!", &at_, &PyTuple_Type, &shape)) {
      release(r);
      return nullptr;
    }
    Py_INCREF(shape);
    r.shapes.emplace_back(at_, shape);
  }
  std::string key(sig, (size_t)nsig);
  const auto old = s->kept->find(key);
  if (old != s->kept->end()) {
    release(old->second);
    s->kept->erase(old);
  }
  s->kept->emplace(std::move(key), std::move(r));
  Py_RETURN_NONE;
}

PyObject* state_new(PyTypeObject* type, PyObject* args, PyObject*) {
  const char* name;
  if (!PyArg_ParseTuple(args, "s", &name)) return nullptr;
  State* s = reinterpret_cast<State*>(type->tp_alloc(type, 0));
  if (s) {
    s->name = new std::string(name);
    s->kept = new std::unordered_map<std::string, Ready>();
  }
  return reinterpret_cast<PyObject*>(s);
}

void state_free(PyObject* self) {
  State* s = reinterpret_cast<State*>(self);
  if (s->kept) forget(s);
  delete s->kept;
  delete s->name;
  Py_TYPE(self)->tp_free(self);
}

PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long launch, error;
  if (!PyArg_ParseTuple(args, "KK", &launch, &error)) return nullptr;
  g_launch = reinterpret_cast<LaunchFn>(launch);
  g_error = reinterpret_cast<ErrorFn>(error);
  Py_RETURN_NONE;
}

PyMethodDef state_methods[] = {
    {"call", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(state_call)), METH_FASTCALL, nullptr},
    {"add", state_add, METH_VARARGS, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyMethodDef module_methods[] = {{"bind", bind, METH_VARARGS, "Addresses of c3b_launch and c3b_last_error."},
                                {nullptr, nullptr, 0, nullptr}};
PyTypeObject state_type = {PyVarObject_HEAD_INIT(nullptr, 0)};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_torch_call", nullptr, -1, module_methods};

}  // namespace

PyMODINIT_FUNC PyInit__torch_call(void) {
  state_type.tp_name = "hackathon_b200._torch_call.State";
  state_type.tp_basicsize = sizeof(State);
  state_type.tp_flags = Py_TPFLAGS_DEFAULT;
  state_type.tp_new = state_new;
  state_type.tp_dealloc = state_free;
  state_type.tp_methods = state_methods;
  if (PyType_Ready(&state_type) < 0) return nullptr;
  PyObject* m = PyModule_Create(&module_def);
  if (!m) return nullptr;
  Py_INCREF(&state_type);
  if (PyModule_AddObject(m, "State", reinterpret_cast<PyObject*>(&state_type)) < 0) {
    Py_DECREF(&state_type);
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
