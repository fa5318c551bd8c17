// _tmlayer: CPython calls of the entry points that a forward makes once or more per
// layer (norm, rotary positions, attention of prompts and branches) and per step
// (sampling).  Each
// function takes the entry point's arguments in order, addresses as integers, and
// returns its status; conversions follow the C parameter types.  ctypes spends
// ~3.5 us on a call of twenty arguments, this ~0.5 us.  The interpreter lock is
// released during the call, whose launch waits when the stream's queue is full.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <stdint.h>

#include <tuple>
#include <type_traits>
#include <utility>

#include "../../include/treemoe_amd.h"

namespace {

template <typename T>
T convert(PyObject* o) {
  if constexpr (std::is_pointer_v<T>)
    return (T)PyLong_AsVoidPtr(o);
  else if constexpr (std::is_floating_point_v<T>)
    return (T)PyFloat_AsDouble(o);
  else if constexpr (sizeof(T) == 8)
    return (T)PyLong_AsLongLong(o);
  else
    return (T)PyLong_AsLong(o);
}

template <auto F, typename... A, size_t... I>
PyObject* invoke(int (*)(A...), PyObject* const* args, Py_ssize_t n, std::index_sequence<I...>) {
  if (n != (Py_ssize_t)sizeof...(A)) {
    PyErr_Format(PyExc_TypeError, "expected %d arguments, got %d", (int)sizeof...(A), (int)n);
    return nullptr;
  }
  std::tuple<A...> a{convert<A>(args[I])...};
  if (PyErr_Occurred()) return nullptr;
  int rc = 0;
  Py_BEGIN_ALLOW_THREADS
  rc = F(std::get<I>(a)...);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

template <typename... A>
constexpr std::index_sequence_for<A...> indexes(int (*)(A...)) {
  return {};
}

template <auto F>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return invoke<F>(F, args, n, indexes(F));
}

// prompt_cached_workspace(T, seq_len, Hq, kvh, hd) -> (status, bytes)
PyObject* cached_workspace(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 5) {
    PyErr_SetString(PyExc_TypeError, "expected 5 arguments");
    return nullptr;
  }
  int64_t a[5], bytes = 0;
  for (int i = 0; i < 5; ++i) a[i] = convert<int64_t>(args[i]);
  if (PyErr_Occurred()) return nullptr;
  const int rc = tm_prompt_cached_workspace(a[0], a[1], a[2], a[3], a[4], &bytes);
  return Py_BuildValue("iL", rc, (long long)bytes);
}

// mass_workspace(T, seq_len, Hq, kvh, hd) -> (status, bytes)
PyObject* mass_workspace(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 5) {
    PyErr_SetString(PyExc_TypeError, "expected 5 arguments");
    return nullptr;
  }
  int64_t a[5], bytes = 0;
  for (int i = 0; i < 5; ++i) a[i] = convert<int64_t>(args[i]);
  if (PyErr_Occurred()) return nullptr;
  const int rc = tm_mass_workspace(a[0], a[1], a[2], a[3], a[4], &bytes);
  return Py_BuildValue("iL", rc, (long long)bytes);
}

// branch_workspace(T, units, max_count, seq_len, longest, Hq, kvh, hd) -> (status, bytes)
PyObject* branch_workspace(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 8) {
    PyErr_SetString(PyExc_TypeError, "expected 8 arguments");
    return nullptr;
  }
  int64_t a[8], bytes = 0;
  for (int i = 0; i < 8; ++i) a[i] = convert<int64_t>(args[i]);
  if (PyErr_Occurred()) return nullptr;
  const int rc = tm_branch_workspace(a[0], a[1], a[2], a[3], a[4], a[5], a[6], a[7], &bytes);
  return Py_BuildValue("iL", rc, (long long)bytes);
}

#define TM_ENTRY(name) \
  {#name, (PyCFunction)(void (*)(void))entry<name>, METH_FASTCALL, nullptr}

PyMethodDef kMethods[] = {
    TM_ENTRY(tm_rms_norm),
    TM_ENTRY(tm_rms_norm_fp8),
    TM_ENTRY(tm_rotary),
    TM_ENTRY(tm_rotary_append),
    TM_ENTRY(tm_sample_tokens),
    TM_ENTRY(tm_prompt_attention),
    {"prompt_cached_workspace", (PyCFunction)(void (*)(void))cached_workspace, METH_FASTCALL,
     nullptr},
    TM_ENTRY(tm_prompt_attention_cached),
    {"branch_workspace", (PyCFunction)(void (*)(void))branch_workspace, METH_FASTCALL, nullptr},
    TM_ENTRY(tm_branch_attention),
    TM_ENTRY(tm_branch_advance),
    TM_ENTRY(tm_beam_select),
    TM_ENTRY(tm_reorder_rows),
    {"mass_workspace", (PyCFunction)(void (*)(void))mass_workspace, METH_FASTCALL, nullptr},
    TM_ENTRY(tm_attention_mass),
    TM_ENTRY(tm_evict),
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_tmlayer", "CPython calls of libtreemoe_amd.so",
                       -1, kMethods};

}  // namespace

PyMODINIT_FUNC PyInit__tmlayer(void) { return PyModule_Create(&kModule); }
