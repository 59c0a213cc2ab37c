// Python module _calls: repeated calls of the 8-bit linear path's operators.
//
// An operator's first call with tensors of some layout checks them, fills a
// descriptor and knows its outputs' layouts (ops.py).  A Plan keeps that, and
// run() makes the next call with the same layouts from it: compares the layouts,
// allocates the outputs and calls the C entry.  The host's share of a call: 5.9 us
// (norm with residual and e4m3 output, three outputs), 4.9 (quantise), 4.4 (product);
// through ctypes and torch's Python functions 10.8, 7.3 and 8.6.  The launch itself is
// 2.3 of them, each output 0.5.  With 64 layouts in turn the plans are searched: 7.0, 5.1
// and 5.2 to 6.4 us; a layout's first call costs 44, 30 and 35.
//
// A Plan holds no tensor and no address of one.  What it cannot serve (other
// layouts, another current device, a handle on another stream than torch's)
// run() answers with None, and the operator goes the long way.  The module belongs to
// the Python and torch that it was built with (CALLS_PYTHON, CALLS_TORCH): another
// Python cannot import it, for another torch the operators leave it alone.
#include <Python.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>
#include <vector>

namespace {

constexpr int kMaxSlots = 6;  // pointers behind (handle, descriptor) of the longest entry
constexpr int kMaxInputs = 5;

// An owned reference.
struct Ref {
  PyObject* p;
  explicit Ref(PyObject* o) : p(o) {}
  Ref(const Ref&) = delete;
  Ref& operator=(const Ref&) = delete;
  ~Ref() { Py_XDECREF(p); }
  PyObject* release() {
    PyObject* o = p;
    p = nullptr;
    return o;
  }
};

struct Layout {
  bool absent = false;
  std::vector<int64_t> sizes, strides;
  at::ScalarType type{};
};

struct Plan {
  PyObject_HEAD
  PyObject* keep;  // owner of the descriptor
  void *entry, *get_stream, *desc;
  int device;
  std::vector<Layout>*in, *out;
  std::vector<int>* slots;  // of each pointer: an input (>= 0), output -1 - slot, or kNull
};
constexpr int kNull = 1000;

void plan_dealloc(PyObject* self) {
  Plan* p = reinterpret_cast<Plan*>(self);
  delete p->in;
  delete p->out;
  delete p->slots;
  Py_XDECREF(p->keep);
  Py_TYPE(self)->tp_free(self);
}

bool read_ints(PyObject* o, std::vector<int64_t>& v) {
  PyObject* f = PySequence_Fast(o, "expected a sequence of ints");
  if (!f) return false;
  for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(f); ++i) v.push_back(PyLong_AsLongLong(PySequence_Fast_GET_ITEM(f, i)));
  Py_DECREF(f);
  return !PyErr_Occurred();
}

// Plan(entry, get_stream, descriptor address, its owner, device, inputs, outputs, slots)
PyObject* plan_new(PyTypeObject* type, PyObject* args, PyObject*) {
  HANDLE_TH_ERRORS
  unsigned long long entry, get_stream, desc;
  PyObject *keep, *inputs, *outputs, *slots;
  int device;
  if (!PyArg_ParseTuple(args, "KKKOiO!O!O!", &entry, &get_stream, &desc, &keep, &device, &PyTuple_Type, &inputs,
                        &PyTuple_Type, &outputs, &PyTuple_Type, &slots))
    return nullptr;
  Plan* p = reinterpret_cast<Plan*>(type->tp_alloc(type, 0));
  if (!p) return nullptr;
  p->entry = reinterpret_cast<void*>(entry);
  p->get_stream = reinterpret_cast<void*>(get_stream);
  p->desc = reinterpret_cast<void*>(desc);
  p->device = device;
  Py_INCREF(keep);
  p->keep = keep;
  auto bad = [&](const char* what) -> PyObject* {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, what);
    Py_DECREF(p);
    return nullptr;
  };
  p->in = new std::vector<Layout>;
  p->out = new std::vector<Layout>;
  p->slots = new std::vector<int>;
  const Py_ssize_t n_in = PyTuple_GET_SIZE(inputs), n_out = PyTuple_GET_SIZE(outputs), n = PyTuple_GET_SIZE(slots);
  if (n_in > kMaxInputs || (n != 3 && n != kMaxSlots)) return bad("Plan: wrong number of inputs or pointers");
  for (Py_ssize_t i = 0; i < n_in; ++i) {
    PyObject* o = PyTuple_GET_ITEM(inputs, i);
    Layout l;
    if (o == Py_None) {
      l.absent = true;
    } else {
      if (!THPVariable_Check(o)) return bad("Plan: expected tensors");
      const at::Tensor& t = THPVariable_Unpack(o);
      l.sizes = t.sizes().vec();
      l.strides = t.strides().vec();
      l.type = t.scalar_type();
    }
    p->in->push_back(std::move(l));
  }
  for (Py_ssize_t i = 0; i < n_out; ++i) {
    PyObject *sizes, *strides, *dtype;
    Layout l;
    if (!PyArg_ParseTuple(PyTuple_GET_ITEM(outputs, i), "OOO", &sizes, &strides, &dtype)) return bad("");
    if (!THPDtype_Check(dtype) || !read_ints(sizes, l.sizes) || !read_ints(strides, l.strides) ||
        l.sizes.size() != l.strides.size())
      return bad("Plan: expected (sizes, strides, dtype)");
    l.type = reinterpret_cast<THPDtype*>(dtype)->scalar_type;
    p->out->push_back(std::move(l));
  }
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* o = PyTuple_GET_ITEM(slots, i);
    const long v = o == Py_None ? kNull : PyLong_AsLong(o);
    if (v != kNull && (v >= n_in || v < -n_out || PyErr_Occurred())) return bad("Plan: wrong slot");
    p->slots->push_back((int)v);
  }
  return reinterpret_cast<PyObject*>(p);
  END_HANDLE_TH_ERRORS
}

PyTypeObject plan_type = {PyVarObject_HEAD_INIT(nullptr, 0)};

bool fits(const Layout& l, PyObject* o, int device) {
  if (o == Py_None || l.absent) return l.absent && o == Py_None;
  if (!THPVariable_Check(o)) return false;
  const at::Tensor& t = THPVariable_Unpack(o);
  // only plain tensors: a subclass may stand for something else than its memory
  return t.is_cuda() && t.get_device() == device && t.scalar_type() == l.type && t.layout() == at::kStrided &&
         !t.key_set().has(c10::DispatchKey::Python) && t.sizes() == at::IntArrayRef(l.sizes) &&
         t.strides() == at::IntArrayRef(l.strides);
}

// run(plans, handle, its device, own_stream, *tensors): the outputs (a list) of the first plan that
// fits, an error code of its C entry, or None.
PyObject* run(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs < 4 || !PyList_Check(args[0])) {
    PyErr_SetString(PyExc_TypeError, "run(plans, handle, device, own_stream, *tensors)");
    return nullptr;
  }
  void* handle = PyLong_AsVoidPtr(args[1]);
  const long device = PyLong_AsLong(args[2]);
  void* own = PyLong_AsVoidPtr(args[3]);
  if (PyErr_Occurred()) return nullptr;
  if (!handle) Py_RETURN_NONE;
  PyObject* const* ins = args + 4;
  const Py_ssize_t n_in = nargs - 4;
  Plan* p = nullptr;
  for (Py_ssize_t i = 0; i < PyList_GET_SIZE(args[0]) && !p; ++i) {
    PyObject* o = PyList_GET_ITEM(args[0], i);
    if (!PyObject_TypeCheck(o, &plan_type)) continue;
    Plan* c = reinterpret_cast<Plan*>(o);
    bool ok = c->device == device && (Py_ssize_t)c->in->size() == n_in;
    for (Py_ssize_t j = 0; ok && j < n_in; ++j) ok = fits((*c->in)[j], ins[j], c->device);
    if (ok) p = c;
  }
  if (!p || c10::cuda::current_device() != p->device) Py_RETURN_NONE;
  // in order with torch's current stream: the handle runs on it, or on its own stream,
  // a blocking one, which is ordered with the legacy default stream
  void* cur = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)p->device).stream();
  void* runs_on = reinterpret_cast<void* (*)(void*)>(p->get_stream)(handle);
  if (cur != runs_on && !(cur == nullptr && runs_on == own)) Py_RETURN_NONE;

  Ref guard(Py_NewRef(reinterpret_cast<PyObject*>(p)));
  std::vector<at::Tensor> outs;
  outs.reserve(p->out->size());
  for (const Layout& l : *p->out)
    outs.push_back(at::detail::empty_strided_cuda(l.sizes, l.strides, l.type,
                                                  c10::Device(c10::kCUDA, (c10::DeviceIndex)p->device)));
  void* ptr[kMaxSlots] = {};
  for (size_t i = 0; i < p->slots->size(); ++i) {
    const int s = (*p->slots)[i];
    if (s == kNull) continue;
    ptr[i] = s >= 0 ? const_cast<void*>(THPVariable_Unpack(ins[s]).const_data_ptr()) : outs[-1 - s].mutable_data_ptr();
  }
  int rc;
  Py_BEGIN_ALLOW_THREADS;
  if (p->slots->size() == 3)
    rc = reinterpret_cast<int (*)(void*, const void*, void*, void*, void*)>(p->entry)(handle, p->desc, ptr[0], ptr[1], ptr[2]);
  else
    rc = reinterpret_cast<int (*)(void*, const void*, void*, void*, void*, void*, void*, void*)>(p->entry)(
        handle, p->desc, ptr[0], ptr[1], ptr[2], ptr[3], ptr[4], ptr[5]);
  Py_END_ALLOW_THREADS;
  if (rc) return PyLong_FromLong(rc);
  Ref list(PyList_New((Py_ssize_t)outs.size()));
  if (!list.p) return nullptr;
  for (size_t i = 0; i < outs.size(); ++i) {
    PyObject* o = THPVariable_Wrap(std::move(outs[i]));
    if (!o) return nullptr;
    PyList_SET_ITEM(list.p, (Py_ssize_t)i, o);
  }
  return list.release();
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {{"run", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(run)), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods};

}  // namespace

#define CALLS_TEXT_OF(x) #x
#define CALLS_TEXT(x) CALLS_TEXT_OF(x)

// The version that Python reports begins with `built`, its major and minor numbers.
static bool same_python(const char* built) {
  const size_t n = strlen(built);
  const char* v = Py_GetVersion();
  return strncmp(v, built, n) == 0 && (v[n] < '0' || v[n] > '9');
}

PyMODINIT_FUNC PyInit__calls() {
  // before anything whose layout belongs to a version of Python
  if (!same_python(CALLS_TEXT(CALLS_PYTHON))) {
    PyErr_SetString(PyExc_ImportError, "built for Python " CALLS_TEXT(CALLS_PYTHON));
    return nullptr;
  }
  plan_type.tp_name = "_calls.Plan";
  plan_type.tp_basicsize = sizeof(Plan);
  plan_type.tp_flags = Py_TPFLAGS_DEFAULT;
  plan_type.tp_new = plan_new;
  plan_type.tp_dealloc = plan_dealloc;
  if (PyType_Ready(&plan_type) < 0) return nullptr;
  PyObject* m = PyModule_Create(&module);
  if (!m) return nullptr;
  if (PyModule_AddObjectRef(m, "Plan", reinterpret_cast<PyObject*>(&plan_type)) < 0 ||
      PyModule_AddStringConstant(m, "torch_version", CALLS_TEXT(CALLS_TORCH)) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
