// CPython entry points of the serving operators: the functions of the C ABI taken positionally,
// tensors by their data_ptr(), None as a null pointer, the status returned. A call through ctypes
// converts ~20 arguments in ~3 us, as long as a small launch takes; this is ~1 us. (_lib.call uses
// it where it has the name, ctypes otherwise.)
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <cstddef>
#include <cstdint>
#include <tuple>
#include <type_traits>
#include <utility>

#include "orchard_b200.h"

namespace {

PyObject* g_data_ptr = nullptr;  // "data_ptr"

// Conversions. `ok` turns false with a Python error set; from then on nothing more is asked of the
// arguments (a call into Python with an error set would replace it by a SystemError).
unsigned long long whole(PyObject* o, bool& ok) {
  if (PyLong_Check(o)) return PyLong_AsUnsignedLongLongMask(o);
  PyObject* i = PyNumber_Index(o);
  ok = i != nullptr;
  if (!ok) return 0;
  const unsigned long long v = PyLong_AsUnsignedLongLongMask(i);
  Py_DECREF(i);
  return v;
}

unsigned long long address(PyObject* o, bool& ok) {
  if (o == Py_None) return 0;
  if (PyLong_Check(o)) return PyLong_AsUnsignedLongLongMask(o);
  PyObject* p = PyObject_CallMethodNoArgs(o, g_data_ptr);
  ok = p != nullptr;
  if (!ok) return 0;
  const unsigned long long v = whole(p, ok);
  Py_DECREF(p);
  return v;
}

template <typename T>
T convert(PyObject* o, bool& ok) {
  if (!ok) return T{};
  if constexpr (std::is_pointer_v<T>) {
    return reinterpret_cast<T>(static_cast<uintptr_t>(address(o, ok)));
  } else if constexpr (std::is_floating_point_v<T>) {
    const double v = PyFloat_AsDouble(o);
    ok = v != -1.0 || PyErr_Occurred() == nullptr;
    return static_cast<T>(v);
  } else {
    return static_cast<T>(whole(o, ok));
  }
}

template <typename... A, size_t... I>
PyObject* invoke(int (*fn)(A...), PyObject* const* args, std::index_sequence<I...>) {
  bool ok = true;
  const std::tuple<A...> v{convert<A>(args[I], ok)...};  // braces: converted in order
  if (!ok) return nullptr;
  int status = 0;
  Py_BEGIN_ALLOW_THREADS;
  status = fn(std::get<I>(v)...);
  Py_END_ALLOW_THREADS;
  return PyLong_FromLong(status);
}

template <typename... A>
PyObject* take(int (*fn)(A...), PyObject* const* args, Py_ssize_t n) {
  if (n != (Py_ssize_t)sizeof...(A)) {
    PyErr_Format(PyExc_TypeError, "%zd arguments given, %zu taken", n, sizeof...(A));
    return nullptr;
  }
  return invoke(fn, args, std::index_sequence_for<A...>{});
}

template <auto Fn>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return take(Fn, args, n);
}

#define ENTRY(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(entry<&name>)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {ENTRY(orch_attention_prefix),    ENTRY(orch_cache_evict),
                           ENTRY(orch_logits_process),      ENTRY(orch_q4t_qkv_rope_at),
                           ENTRY(orch_q4t_rms_qkv_rope_at), {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_entry", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__entry(void) {
  g_data_ptr = PyUnicode_InternFromString("data_ptr");
  return g_data_ptr ? PyModule_Create(&g_module) : nullptr;
}
