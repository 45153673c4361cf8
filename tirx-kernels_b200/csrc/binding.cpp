// The operators' calls from Python: argument checks and the C entry point in one step.
//
// A decode-sized operator takes 5 to 12 us on the GPU; checking eight tensors in Python and calling through ctypes took
// the host 8.5 us, which then was the time of the call.  Here a call is bound once to an entry point of b200_nvfp4.h,
// the types and shapes of its tensors and its sizes, and takes 3 us, of which the launch is 2.
//
//   launch = bind(symbol, address, specs, sizes)
//     specs  (name, torch dtype, shape as a tuple or a number of elements, may be None) per pointer argument
//     sizes  the other arguments, in order; None: given with each call, behind the tensors
//   launch(*tensors, *given) -> 0, the entry point's status, or -1: a tensor is not what its spec says, is not contiguous
//     or not on the current CUDA device (nothing was called; the caller says which)
//   check = bind(None, 0, specs, ()): the tensors' check alone
//
// The stream is the current one of the current device.  The interpreter's lock is released around the entry point.
#include <Python.h>

#include <array>
#include <cstddef>
#include <exception>
#include <new>
#include <string>
#include <tuple>
#include <utility>
#include <vector>

#include <ATen/core/Tensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include "b200_nvfp4.h"

namespace {

struct Spec {
  at::ScalarType type;
  bool optional;
  bool shaped;                 // shape, else numel
  std::vector<int64_t> shape;
  int64_t numel;               // -1: any
};
struct Value {
  long long i;
  double d;
};

constexpr size_t kMostTensors = 16, kMostValues = 12;

// The entry point's arguments from `pointers` (the stream is the last) and `values`, each in order.
template <typename Function>
struct Entry;
template <typename... A>
struct Entry<int (*)(A...)> {
  static constexpr size_t kPointers = (0 + ... + (std::is_pointer_v<A> ? 1 : 0));
  static constexpr size_t kValues = sizeof...(A) - kPointers;
  static_assert(kPointers <= kMostTensors + 1 && kValues <= kMostValues);
  template <typename T>
  static T next(void* const*& pointers, const Value*& values) {
    if constexpr (std::is_pointer_v<T>) return static_cast<T>(*pointers++);
    else if constexpr (std::is_floating_point_v<T>) return static_cast<T>(values++->d);
    else return static_cast<T>(values++->i);
  }
  static int run(void* address, void* const* pointers, const Value* values) {
    const std::tuple<A...> arguments{next<A>(pointers, values)...};  // braces: in order
    return std::apply(reinterpret_cast<int (*)(A...)>(address), arguments);
  }
};

struct Symbol {
  const char* name;
  int (*run)(void*, void* const*, const Value*);
  size_t pointers, values;
};
#define B2_SYMBOL(f) {#f, &Entry<decltype(&f)>::run, Entry<decltype(&f)>::kPointers, Entry<decltype(&f)>::kValues}
const Symbol kSymbols[] = {B2_SYMBOL(b2_nvfp4_gemm_epilogue), B2_SYMBOL(b2_nvfp4_grouped_gemm), B2_SYMBOL(b2_nvfp4_quantize_grouped),
                           B2_SYMBOL(b2_moe_expert_ffn), B2_SYMBOL(b2_gated_add_rmsnorm_fp4quant)};

struct Launch {
  PyObject_HEAD
  vectorcallfunc vectorcall;
  const Symbol* symbol;  // null: a check alone
  void* address;
  std::vector<Spec> specs;
  std::vector<Value> values;
  std::vector<size_t> given;  // which of them come with the call
};

bool matches(const Spec& spec, const at::Tensor& t) {
  if (t.scalar_type() != spec.type || !t.is_cuda() || !t.is_contiguous()) return false;
  return spec.shaped ? t.sizes() == at::IntArrayRef(spec.shape) : spec.numel < 0 || t.numel() == spec.numel;
}

// Returns -1 where a tensor is refused.  With `run` false the entry point is not called.
long launch_or_check(Launch* self, PyObject* const* args) {
  void* pointers[kMostTensors + 1];
  Value values[kMostValues];
  int device = -1;
  const size_t tensors = self->specs.size();
  for (size_t n = 0; n < tensors; ++n) {
    const Spec& spec = self->specs[n];
    if (args[n] == Py_None && spec.optional) {
      pointers[n] = nullptr;
      continue;
    }
    if (!THPVariable_Check(args[n])) return -1;
    const at::Tensor& t = THPVariable_Unpack(args[n]);
    if (!matches(spec, t)) return -1;
    if (device < 0) device = c10::cuda::current_device();
    if (t.get_device() != device) return -1;
    pointers[n] = const_cast<void*>(t.const_data_ptr());
  }
  if (!self->symbol) return 0;
  if (device < 0) return -1;
  pointers[tensors] = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream();
  for (size_t n = 0; n < self->values.size(); ++n) values[n] = self->values[n];
  for (size_t n = 0; n < self->given.size(); ++n) {
    Value& v = values[self->given[n]];
    PyObject* arg = args[tensors + n];
    v.d = PyFloat_AsDouble(arg);
    if (v.d == -1.0 && PyErr_Occurred()) return -2;
    v.i = 0;
    if (PyLong_Check(arg)) {
      v.i = PyLong_AsLongLong(arg);
      if (v.i == -1 && PyErr_Occurred()) return -2;
    }
  }
  int status = 0;
  Py_BEGIN_ALLOW_THREADS
  status = self->symbol->run(self->address, pointers, values);
  Py_END_ALLOW_THREADS
  return status;
}

PyObject* launch_call(PyObject* object, PyObject* const* args, size_t nargsf, PyObject* names) {
  Launch* self = reinterpret_cast<Launch*>(object);
  const size_t want = self->specs.size() + self->given.size();
  if ((names && PyTuple_GET_SIZE(names)) || static_cast<size_t>(PyVectorcall_NARGS(nargsf)) != want) {
    PyErr_Format(PyExc_TypeError, "%zu positional arguments expected", want);
    return nullptr;
  }
  try {
    const long status = launch_or_check(self, args);
    return status == -2 ? nullptr : PyLong_FromLong(status);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

void launch_free(PyObject* object) {
  Launch* self = reinterpret_cast<Launch*>(object);
  self->specs.~vector();
  self->values.~vector();
  self->given.~vector();
  Py_TYPE(object)->tp_free(object);
}

PyTypeObject launch_type = {PyVarObject_HEAD_INIT(nullptr, 0)};

bool read_spec(PyObject* item, Spec* spec) {
  if (!PyTuple_Check(item) || PyTuple_GET_SIZE(item) != 4 || !THPDtype_Check(PyTuple_GET_ITEM(item, 1))) {
    PyErr_SetString(PyExc_TypeError, "a spec is (name, dtype, shape, optional)");
    return false;
  }
  spec->type = reinterpret_cast<THPDtype*>(PyTuple_GET_ITEM(item, 1))->scalar_type;
  spec->optional = PyObject_IsTrue(PyTuple_GET_ITEM(item, 3)) == 1;
  PyObject* shape = PyTuple_GET_ITEM(item, 2);
  spec->shaped = PyTuple_Check(shape);
  spec->numel = 0;
  if (!spec->shaped) {
    spec->numel = PyLong_AsLongLong(shape);
    return !PyErr_Occurred();
  }
  for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(shape); ++i) {
    spec->shape.push_back(PyLong_AsLongLong(PyTuple_GET_ITEM(shape, i)));
    if (PyErr_Occurred()) return false;
  }
  return true;
}

PyObject* bind(PyObject*, PyObject* args) {
  const char* name = nullptr;
  unsigned long long address = 0;
  PyObject *specs = nullptr, *sizes = nullptr;
  if (!PyArg_ParseTuple(args, "zKO!O!", &name, &address, &PyTuple_Type, &specs, &PyTuple_Type, &sizes)) return nullptr;
  const size_t tensors = static_cast<size_t>(PyTuple_GET_SIZE(specs)), values = static_cast<size_t>(PyTuple_GET_SIZE(sizes));
  const Symbol* symbol = nullptr;
  if (name) {
    for (const Symbol& s : kSymbols)
      if (std::string(s.name) == name) symbol = &s;
    if (!symbol || !address || symbol->pointers != tensors + 1 || symbol->values != values) {
      PyErr_Format(PyExc_TypeError, "%s is not bound with %zu tensors and %zu sizes", name, tensors, values);
      return nullptr;
    }
  } else if (tensors > kMostTensors || values) {
    PyErr_SetString(PyExc_TypeError, "a check has at most 16 tensors and no sizes");
    return nullptr;
  }
  try {
    std::vector<Spec> read(tensors);
    for (size_t n = 0; n < tensors; ++n)
      if (!read_spec(PyTuple_GET_ITEM(specs, static_cast<Py_ssize_t>(n)), &read[n])) return nullptr;
    std::vector<Value> fixed(values, Value{0, 0.0});
    std::vector<size_t> given;
    for (size_t n = 0; n < values; ++n) {
      PyObject* item = PyTuple_GET_ITEM(sizes, static_cast<Py_ssize_t>(n));
      if (item == Py_None) {
        given.push_back(n);
      } else if (PyLong_Check(item)) {
        fixed[n].i = PyLong_AsLongLong(item);
        fixed[n].d = static_cast<double>(fixed[n].i);
        if (PyErr_Occurred()) return nullptr;
      } else {
        PyErr_SetString(PyExc_TypeError, "sizes are integers, or None for what comes with the call");
        return nullptr;
      }
    }
    Launch* self = reinterpret_cast<Launch*>(launch_type.tp_alloc(&launch_type, 0));
    if (!self) return nullptr;
    self->vectorcall = launch_call;
    self->symbol = symbol;
    self->address = reinterpret_cast<void*>(static_cast<uintptr_t>(address));
    new (&self->specs) std::vector<Spec>(std::move(read));
    new (&self->values) std::vector<Value>(std::move(fixed));
    new (&self->given) std::vector<size_t>(std::move(given));
    return reinterpret_cast<PyObject*>(self);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

PyMethodDef methods[] = {{"bind", bind, METH_VARARGS, "bind(symbol, address, specs, sizes) -> launch"}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "b200nvfp4_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_b200nvfp4_binding() {
  launch_type.tp_name = "b200nvfp4_binding.Launch";
  launch_type.tp_basicsize = sizeof(Launch);
  launch_type.tp_flags = Py_TPFLAGS_DEFAULT | Py_TPFLAGS_HAVE_VECTORCALL;
  launch_type.tp_vectorcall_offset = offsetof(Launch, vectorcall);
  launch_type.tp_call = PyVectorcall_Call;
  launch_type.tp_dealloc = launch_free;
  if (PyType_Ready(&launch_type) < 0) return nullptr;
  return PyModule_Create(&module);
}
