// _tmlayer: CPython calls of the entry points that a forward makes once or more per
// layer (norm, rotary positions, attention of prompts and branches, attention mass) and per
// step (sampling, beams, eviction).  Each function takes the entry point's arguments in order,
// addresses as integers, and returns its status, a size query its status and the bytes;
// conversions follow the C parameter types.  ctypes spends
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

// A size query: its arguments without the last, which takes the bytes -> (status, bytes).
template <auto F, typename... A, size_t... I>
PyObject* query(int (*)(A...), PyObject* const* args, Py_ssize_t n, std::index_sequence<I...>) {
  if (n != (Py_ssize_t)sizeof...(I)) {
    PyErr_Format(PyExc_TypeError, "expected %d arguments, got %d", (int)sizeof...(I), (int)n);
    return nullptr;
  }
  const int64_t a[] = {convert<int64_t>(args[I])...};
  if (PyErr_Occurred()) return nullptr;
  int64_t bytes = 0;
  const int rc = F(a[I]..., &bytes);
  return Py_BuildValue("iL", rc, (long long)bytes);
}
template <typename... A>
constexpr std::make_index_sequence<sizeof...(A) - 1> sizes(int (*)(A...)) {
  return {};
}
template <auto F>
PyObject* bytes_of(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return query<F>(F, args, n, sizes(F));
}

#define TM_ENTRY(name) \
  {#name, (PyCFunction)(void (*)(void))entry<name>, METH_FASTCALL, nullptr}

#define TM_BYTES(name, entry) \
  {name, (PyCFunction)(void (*)(void))bytes_of<entry>, METH_FASTCALL, nullptr}

PyMethodDef kMethods[] = {
    TM_ENTRY(tm_rms_norm),
    TM_ENTRY(tm_rms_norm_fp8),
    TM_ENTRY(tm_rotary),
    TM_ENTRY(tm_rotary_append),
    TM_ENTRY(tm_sample_tokens),
    TM_ENTRY(tm_prompt_attention),
    TM_BYTES("prompt_cached_workspace", tm_prompt_cached_workspace),
    TM_ENTRY(tm_prompt_attention_cached),
    TM_BYTES("branch_workspace", tm_branch_workspace),
    TM_ENTRY(tm_branch_attention),
    TM_ENTRY(tm_branch_advance),
    TM_ENTRY(tm_beam_select),
    TM_ENTRY(tm_reorder_rows),
    TM_BYTES("beam_workspace", tm_beam_workspace),
    TM_BYTES("mass_workspace", tm_mass_workspace),
    TM_BYTES("evict_workspace", tm_evict_workspace),
    TM_ENTRY(tm_attention_mass),
    TM_ENTRY(tm_evict),
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_tmlayer", "CPython calls of libtreemoe_amd.so",
                       -1, kMethods};

}  // namespace

PyMODINIT_FUNC PyInit__tmlayer(void) { return PyModule_Create(&kModule); }
