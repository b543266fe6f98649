// pycall.cpp - the Python side's short way into the C entry points (module ftb._pycall).
//
// A call on a few rows spends its time on the host: what its checks look at (shape, strides, dtype
// and device of up to eight tensors) costs more to gather attribute by attribute than the launch.
//   key(a, b, ...)    these properties of all arguments in one bytes object (None has its mark)
//   call(fn, template, offsets, stream, a, b, ...)
//                     copies an argument struct, writes the tensors' data pointers at the given
//                     offsets and calls int fn(const void* args, void* stream), without the
//                     interpreter's lock; calls of one stream take turns, since one may be several
//                     launches over the stream's workspace
//   empty(a, b)       the output: a's shape and device, b's dtype, contiguous
// On one host, per call: 2.5 -> 0.3 us for the key and its look-up, 1.7 -> 0.2 us for the struct and
// the call, 1.4 to 2.7 -> 0.6 to 1.2 us for an output. A norm of one row went from 10.5 to 6.2 us, the
// rotary positions of 64 tokens from 11.9 to 5.4 (0.3 more for the turns of a stream's calls and the
// look at the current device).
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <ATen/ops/empty.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/version.h>

#include <cstdint>
#include <cstring>
#include <exception>
#include <map>
#include <mutex>
#include <utility>

namespace {

constexpr size_t kMaxArgs = 1024;  // bytes of an argument struct

// The lock of a stream's calls, found under the interpreter's lock and taken without it. One each:
// a launch may wait for its stream, and that for a peer whose stream another thread has to feed.
std::mutex& lock_of(int device, void* stream) {
  static std::map<std::pair<int, void*>, std::mutex> locks;  // (nodes stay where they are)
  return locks[{device, stream}];
}

PyObject* key(PyObject*, PyObject* const* args, Py_ssize_t n) {
  int64_t buf[256];
  size_t at = 0;
  try {
    for (Py_ssize_t i = 0; i < n; ++i) {
      if (args[i] == Py_None) {
        if (at + 1 > 256) {
          PyErr_SetString(PyExc_ValueError, "too many arguments");
          return nullptr;
        }
        buf[at++] = -1;
        continue;
      }
      if (!THPVariable_Check(args[i])) {
        PyErr_SetString(PyExc_TypeError, "expected tensors");
        return nullptr;
      }
      const at::Tensor& t = THPVariable_Unpack(args[i]);
      const auto sizes = t.sizes();
      const auto strides = t.strides();  // (throws where a layout has none)
      if (at + 1 + 2 * sizes.size() > 256) {
        PyErr_SetString(PyExc_ValueError, "too many dimensions");
        return nullptr;
      }
      const c10::Device d = t.device();
      buf[at++] = (int64_t)t.scalar_type() | (int64_t)d.type() << 16 |
                  (int64_t)(uint8_t)d.index() << 32 | (int64_t)sizes.size() << 48;
      for (int64_t s : sizes) buf[at++] = s;
      for (int64_t s : strides) buf[at++] = s;
    }
  } catch (const std::exception&) {  // (as torch raises it: out of memory is its own kind)
    torch::translate_exception_to_python(std::current_exception());
    return nullptr;
  }
  return PyBytes_FromStringAndSize(reinterpret_cast<const char*>(buf), (Py_ssize_t)(at * 8));
}

PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n < 4 || !PyBytes_Check(args[1]) || !PyTuple_Check(args[2]) ||
      PyTuple_GET_SIZE(args[2]) != n - 4) {
    PyErr_SetString(PyExc_TypeError, "call(fn, template, offsets, stream, a tensor per offset)");
    return nullptr;
  }
  void* fn = PyLong_AsVoidPtr(args[0]);
  void* stream = PyLong_AsVoidPtr(args[3]);
  if (PyErr_Occurred()) return nullptr;
  alignas(16) char buf[kMaxArgs];
  const size_t size = (size_t)PyBytes_GET_SIZE(args[1]);
  if (!fn || size > kMaxArgs) {
    PyErr_SetString(PyExc_ValueError, "no function, or a struct that is too large");
    return nullptr;
  }
  std::memcpy(buf, PyBytes_AS_STRING(args[1]), size);
  int device = -1;  // the tensors'
  std::mutex* turn = nullptr;
  try {
    for (Py_ssize_t i = 4; i < n; ++i) {
      if (args[i] == Py_None) continue;
      const size_t off = PyLong_AsSize_t(PyTuple_GET_ITEM(args[2], i - 4));
      if (PyErr_Occurred()) return nullptr;
      if (!THPVariable_Check(args[i]) || size < sizeof(void*) || off > size - sizeof(void*)) {
        PyErr_SetString(PyExc_TypeError, "expected tensors, and offsets inside the struct");
        return nullptr;
      }
      const at::Tensor& t = THPVariable_Unpack(args[i]);
      void* p = t.data_ptr();
      std::memcpy(buf + off, &p, sizeof(p));
      device = t.device().index();
    }
    turn = &lock_of(device, stream);
  } catch (const std::exception&) {  // (as torch raises it: out of memory is its own kind)
    torch::translate_exception_to_python(std::current_exception());
    return nullptr;
  }
  int st;
  Py_BEGIN_ALLOW_THREADS;
  {
    const std::lock_guard<std::mutex> held(*turn);
    st = reinterpret_cast<int (*)(const void*, void*)>(fn)(buf, stream);
  }
  Py_END_ALLOW_THREADS;
  return PyLong_FromLong(st);
}

// empty(a, b): an uninitialised contiguous tensor of a's shape and device and b's dtype
PyObject* empty(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 2 || !THPVariable_Check(args[0]) || !THPVariable_Check(args[1])) {
    PyErr_SetString(PyExc_TypeError, "empty(shape and device of, dtype of)");
    return nullptr;
  }
  try {
    const at::Tensor& a = THPVariable_Unpack(args[0]);
    return THPVariable_Wrap(
        at::empty(a.sizes(), a.options().dtype(THPVariable_Unpack(args[1]).scalar_type())));
  } catch (const std::exception&) {  // (as torch raises it: out of memory is its own kind)
    torch::translate_exception_to_python(std::current_exception());
    return nullptr;
  }
}

PyMethodDef methods[] = {
    {"key", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(key)), METH_FASTCALL,
     "shape, strides, dtype and device of tensors, as bytes"},
    {"call", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(call)), METH_FASTCALL,
     "calls a C entry point with tensors' pointers written into an argument struct"},
    {"empty", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(empty)), METH_FASTCALL,
     "an uninitialised contiguous tensor of one tensor's shape and another's dtype"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_pycall", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__pycall() {
  PyObject* m = PyModule_Create(&module);
  // (its calls go into torch's libraries, whose C++ interface changes from version to version)
  if (m && PyModule_AddStringConstant(m, "torch_version", TORCH_VERSION) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
