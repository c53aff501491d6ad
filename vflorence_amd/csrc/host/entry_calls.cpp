// Python callables over entries of libvflorence_amd.so whose calls are as short as their Python
// argument handling: a ctypes call converts 15 to 24 arguments in 1.7 to 2.4 us, these in 0.2 to
// 0.3.  Arguments go by position, an address as an int or None; the result is the entry's status.
// An argument of another type or out of its C type's range raises before the entry is called.
// (The package does without this module where it is not built, through ctypes.)
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <limits>
#include <tuple>
#include <type_traits>
#include <utility>

#include "../../../include/vflorence_amd.h"

namespace {

template <typename T> bool convert(PyObject *o, T &to) {
  if constexpr (std::is_pointer_v<T>) {
    if (o == Py_None) {
      to = nullptr;
      return true;
    }
    const unsigned long long v = PyLong_AsUnsignedLongLong(o);
    if (v == (unsigned long long)-1 && PyErr_Occurred()) return false;
    to = reinterpret_cast<T>(static_cast<uintptr_t>(v));
  } else if constexpr (std::is_floating_point_v<T>) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) return false;
    to = static_cast<T>(v);
  } else {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) return false;
    if (v < std::numeric_limits<T>::min() || v > std::numeric_limits<T>::max()) {
      PyErr_Format(PyExc_OverflowError, "%lld does not fit the entry's argument", v);
      return false;
    }
    to = static_cast<T>(v);
  }
  return true;
}

template <typename... A, std::size_t... I>
PyObject *call_with(int (*entry)(A...), PyObject *const *args, std::index_sequence<I...>) {
  std::tuple<A...> values;
  if (!(convert(args[I], std::get<I>(values)) && ...)) return nullptr;
  int status;
  Py_BEGIN_ALLOW_THREADS  // (a launch may wait for room in its queue)
  status = entry(std::get<I>(values)...);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(status);
}

template <typename... A> PyObject *call(int (*entry)(A...), PyObject *const *args, Py_ssize_t n) {
  if (n != (Py_ssize_t)sizeof...(A)) {
    PyErr_Format(PyExc_TypeError, "%zu arguments expected, got %zd", sizeof...(A), n);
    return nullptr;
  }
  return call_with(entry, args, std::index_sequence_for<A...>{});
}

#define VFL_CALLS(X)               \
  X(vfl_reshape_and_cache_4bit)    \
  X(vfl_gather_cache_4bit)         \
  X(vfl_attention_with_kv_cache_4bit) \
  X(vfl_packed_cross_attention)

#define VFL_FUNCTION(name)                                                          \
  PyObject *py_##name(PyObject *, PyObject *const *args, Py_ssize_t n) {            \
    return call(&name, args, n);                                                    \
  }
VFL_CALLS(VFL_FUNCTION)
#undef VFL_FUNCTION

#define VFL_METHOD(name)                                                             \
  {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&py_##name)),   \
   METH_FASTCALL, nullptr},
PyMethodDef methods[] = {VFL_CALLS(VFL_METHOD){nullptr, nullptr, 0, nullptr}};
#undef VFL_METHOD

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", "Entries of libvflorence_amd.so", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls() { return PyModule_Create(&module); }
