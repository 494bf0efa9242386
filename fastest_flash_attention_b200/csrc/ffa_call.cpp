// Direct calls of the C ABI from CPython, for the entry points whose time is
// the call itself: ctypes spends 0.1 us on every argument of a call (2.4 us of
// the 6 of a windowed decode; 0.3 here), and needs an array object for every tuple of
// strides.  The signatures come from include/ffa_b200.h, so an argument list
// that does not fit it does not compile, and a Python value that does not fit
// its parameter raises.  The library itself stays free of Python: the module is
// given the addresses of the functions that ctypes loaded (bind).
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <limits.h>
#include <string.h>

#include <tuple>
#include <utility>

#include "ffa_b200.h"

namespace {

// One Python argument as a C parameter.
template <typename T>
struct Arg;

template <>
struct Arg<int> {
  int v;
  bool set(PyObject* o) {
    const long x = PyLong_AsLong(o);
    if (x == -1 && PyErr_Occurred()) return false;
    if (x < INT_MIN || x > INT_MAX) {
      PyErr_SetString(PyExc_OverflowError, "argument does not fit a 32-bit int");
      return false;
    }
    v = (int)x;
    return true;
  }
  int get() { return v; }
};

template <>
struct Arg<int64_t> {
  int64_t v;
  bool set(PyObject* o) {
    v = PyLong_AsLongLong(o);
    return !(v == -1 && PyErr_Occurred());
  }
  int64_t get() { return v; }
};

template <>
struct Arg<size_t> {
  size_t v;
  bool set(PyObject* o) {
    v = PyLong_AsSize_t(o);
    return !(v == (size_t)-1 && PyErr_Occurred());
  }
  size_t get() { return v; }
};

template <>
struct Arg<float> {
  float v;
  bool set(PyObject* o) {
    const double x = PyFloat_AsDouble(o);
    v = (float)x;
    return !(x == -1.0 && PyErr_Occurred());
  }
  float get() { return v; }
};

// An address (int) or None.
template <typename T>
struct Arg<T*> {
  void* v;
  bool set(PyObject* o) {
    if (o == Py_None) {
      v = nullptr;
      return true;
    }
    v = PyLong_AsVoidPtr(o);
    return !(v == nullptr && PyErr_Occurred());
  }
  T* get() { return static_cast<T*>(v); }
};

// Strides: a tuple of up to four ints, or None.
template <>
struct Arg<const int64_t*> {
  int64_t v[4];
  bool none;
  bool set(PyObject* o) {
    none = o == Py_None;
    if (none) return true;
    if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) > 4) {
      PyErr_SetString(PyExc_TypeError, "strides must be a tuple of at most four ints");
      return false;
    }
    for (Py_ssize_t i = 0; i < 4; ++i) v[i] = 0;
    for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(o); ++i) {
      v[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(o, i));
      if (v[i] == -1 && PyErr_Occurred()) return false;
    }
    return true;
  }
  const int64_t* get() { return none ? nullptr : v; }
};

// The entry points, in the order of their slots.
enum Slot {
  FWD_SINK, BWD_SINK, WINDOW_DECODE, ROTARY, ROTARY_APPEND, PAGE_COPY, TOKEN_MOVE, ASSIGN_SLOTS,
  RELEASE_PAGES, PAGED_PREFILL, PREFIX_DECODE, SLOTS
};
const char* const kNames[SLOTS] = {"ffa_fwd_sink",      "ffa_bwd_sink",  "ffa_window_decode", "ffa_rotary",
                                   "ffa_rotary_append", "ffa_page_copy", "ffa_token_move",    "ffa_assign_slots",
                                   "ffa_release_pages", "ffa_paged_prefill", "ffa_prefix_decode"};
void* g_fn[SLOTS];

template <int ID, typename F>
struct Call;

template <int ID, typename... A>
struct Call<ID, int(A...)> {
  template <size_t... I>
  static PyObject* run(PyObject* const* args, std::index_sequence<I...>) {
    std::tuple<Arg<A>...> a;
    if (!(std::get<I>(a).set(args[I]) && ...)) return nullptr;
    int status;
    Py_BEGIN_ALLOW_THREADS;
    status = reinterpret_cast<int (*)(A...)>(g_fn[ID])(std::get<I>(a).get()...);
    Py_END_ALLOW_THREADS;
    return PyLong_FromLong(status);
  }
  static PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != (Py_ssize_t)sizeof...(A)) {
      PyErr_Format(PyExc_TypeError, "%s takes %zd arguments, got %zd", kNames[ID], (Py_ssize_t)sizeof...(A), n);
      return nullptr;
    }
    if (!g_fn[ID]) {
      PyErr_Format(PyExc_RuntimeError, "%s has no address yet", kNames[ID]);
      return nullptr;
    }
    return run(args, std::index_sequence_for<A...>{});
  }
};

PyObject* bind(PyObject*, PyObject* args) {
  const char* name;
  unsigned long long address;
  if (!PyArg_ParseTuple(args, "sK", &name, &address)) return nullptr;
  for (int i = 0; i < SLOTS; ++i)
    if (!strcmp(name, kNames[i])) {
      g_fn[i] = reinterpret_cast<void*>(address);
      Py_RETURN_NONE;
    }
  PyErr_Format(PyExc_KeyError, "no entry point %s", name);
  return nullptr;
}

#define FFA_ENTRY(id, fn) \
  { #fn, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(Call<id, decltype(fn)>::call)), METH_FASTCALL, nullptr }
PyMethodDef kMethods[] = {FFA_ENTRY(FWD_SINK, ffa_fwd_sink),
                          FFA_ENTRY(BWD_SINK, ffa_bwd_sink),
                          FFA_ENTRY(WINDOW_DECODE, ffa_window_decode),
                          FFA_ENTRY(ROTARY, ffa_rotary),
                          FFA_ENTRY(ROTARY_APPEND, ffa_rotary_append),
                          FFA_ENTRY(PAGE_COPY, ffa_page_copy),
                          FFA_ENTRY(TOKEN_MOVE, ffa_token_move),
                          FFA_ENTRY(ASSIGN_SLOTS, ffa_assign_slots),
                          FFA_ENTRY(RELEASE_PAGES, ffa_release_pages),
                          FFA_ENTRY(PAGED_PREFILL, ffa_paged_prefill),
                          FFA_ENTRY(PREFIX_DECODE, ffa_prefix_decode),
                          {"bind", bind, METH_VARARGS, "bind(name, address)"},
                          {nullptr, nullptr, 0, nullptr}};
#undef FFA_ENTRY

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_ffa_call", "Direct calls of the kernel library.", -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ffa_call(void) {
  PyObject* m = PyModule_Create(&kModule);
  if (!m) return nullptr;
  PyObject* names = PyTuple_New(SLOTS);
  if (!names) {
    Py_DECREF(m);
    return nullptr;
  }
  for (int i = 0; i < SLOTS; ++i) PyTuple_SET_ITEM(names, i, PyUnicode_FromString(kNames[i]));
  if (PyModule_AddObject(m, "NAMES", names) < 0) {
    Py_DECREF(names);
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
