// _tx_calls: what a call through the C-ABI costs on the host besides its launch.
//
// A Python caller of a launch looks at ten tensors or so: their shapes, strides, types and devices
// decide the plan, their addresses go to the launch.  Asked one attribute at a time that takes 5 us
// of a call of 8, more than a small kernel; here it takes well under 1.
//   form(*objects) -> bytes    the shapes, strides, types and devices of tensors, the values of
//                              numbers and strings, of tuples and lists element by element: equal
//                              exactly where all of these are
//   call(function, *objects) -> int
//                              function (an address) of up to 20 pointer-sized arguments: tensors
//                              and bytes give their address, None 0, numbers themselves
//   addresses(tensors) -> bytes  their addresses, as an array
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <string>

namespace {

template <class T> void put(std::string &s, T v) {
  s.append(reinterpret_cast<const char *>(&v), sizeof v);
}

// False with a Python error set.
bool putForm(std::string &s, PyObject *o) {
  if (o == Py_None) {
    s.push_back('-');
  } else if (THPVariable_Check(o)) {
    const at::Tensor &t = THPVariable_Unpack(o);
    if (t.layout() != c10::kStrided) {
      PyErr_SetString(PyExc_TypeError, "a tensor with strides is needed");
      return false;
    }
    s.push_back('t');
    s.push_back((char)t.dim());
    s.push_back((char)t.scalar_type());
    s.push_back((char)t.device().type());
    s.push_back((char)t.device().index());
    for (int64_t x : t.sizes())
      put(s, x);
    for (int64_t x : t.strides())
      put(s, x);
  } else if (PyBool_Check(o)) {
    s.push_back(o == Py_True ? 'T' : 'F');
  } else if (PyFloat_Check(o)) {
    s.push_back('f');
    put(s, PyFloat_AS_DOUBLE(o));
  } else if (PyLong_Check(o)) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred())
      return false;
    s.push_back('i');
    put(s, (int64_t)v);
  } else if (PyUnicode_Check(o)) {
    Py_ssize_t n;
    const char *c = PyUnicode_AsUTF8AndSize(o, &n);
    if (!c)
      return false;
    s.push_back('s');
    put(s, (int64_t)n);
    s.append(c, n);
  } else if (PyTuple_Check(o) || PyList_Check(o)) {
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(o);
    s.push_back('(');
    put(s, (int64_t)n);
    for (Py_ssize_t i = 0; i < n; ++i)
      if (!putForm(s, PySequence_Fast_GET_ITEM(o, i)))
        return false;
  } else {
    PyErr_Format(PyExc_TypeError, "a tensor or a number is needed, not %s", Py_TYPE(o)->tp_name);
    return false;
  }
  return true;
}

// The C++ exceptions of torch's accessors become Python's.
template <class F> PyObject *guarded(F f) {
  try {
    return f();
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

PyObject *form(PyObject *, PyObject *const *args, Py_ssize_t n) {
  return guarded([&]() -> PyObject * {
    std::string s;
    s.reserve(1024);
    for (Py_ssize_t i = 0; i < n; ++i)
      if (!putForm(s, args[i]))
        return nullptr;
    return PyBytes_FromStringAndSize(s.data(), (Py_ssize_t)s.size());
  });
}

bool word(PyObject *o, uintptr_t &v) {
  if (o == Py_None) {
    v = 0;
  } else if (THPVariable_Check(o)) {
    v = reinterpret_cast<uintptr_t>(THPVariable_Unpack(o).data_ptr());
  } else if (PyBytes_Check(o)) {
    v = reinterpret_cast<uintptr_t>(PyBytes_AS_STRING(o));
  } else if (PyLong_Check(o)) {
    v = (uintptr_t)PyLong_AsUnsignedLongLong(o);
    return !PyErr_Occurred();
  } else {
    PyErr_Format(PyExc_TypeError, "a tensor, bytes, an int or None is needed, not %s",
                 Py_TYPE(o)->tp_name);
    return false;
  }
  return true;
}

// Every argument is one integer register or stack slot, and a callee of fewer leaves the rest
// alone, so one function type of 20 serves all.
constexpr int kMost = 20;
typedef uintptr_t W;
typedef int (*Fn)(W, W, W, W, W, W, W, W, W, W, W, W, W, W, W, W, W, W, W, W);

PyObject *call(PyObject *, PyObject *const *args, Py_ssize_t n) {
  if (n < 1 || n - 1 > kMost) {
    PyErr_Format(PyExc_TypeError, "a function and at most %d arguments are needed", kMost);
    return nullptr;
  }
  return guarded([&]() -> PyObject * {
    W f = 0, a[kMost] = {};
    for (Py_ssize_t i = 0; i < n; ++i)
      if (!word(args[i], i ? a[i - 1] : f))
        return nullptr;
    if (!f) {
      PyErr_SetString(PyExc_ValueError, "no function");
      return nullptr;
    }
    int rc;
    Py_BEGIN_ALLOW_THREADS;
    rc = reinterpret_cast<Fn>(f)(a[0], a[1], a[2], a[3], a[4], a[5], a[6], a[7], a[8], a[9], a[10],
                                 a[11], a[12], a[13], a[14], a[15], a[16], a[17], a[18], a[19]);
    Py_END_ALLOW_THREADS;
    return PyLong_FromLong(rc);
  });
}

PyObject *addresses(PyObject *, PyObject *list) {
  if (!PyTuple_Check(list) && !PyList_Check(list)) {
    PyErr_SetString(PyExc_TypeError, "a tuple or list of tensors is needed");
    return nullptr;
  }
  return guarded([&]() -> PyObject * {
    std::string s;
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(list);
    for (Py_ssize_t i = 0; i < n; ++i) {
      W v;
      if (!word(PySequence_Fast_GET_ITEM(list, i), v))
        return nullptr;
      put(s, v);
    }
    return PyBytes_FromStringAndSize(s.data(), (Py_ssize_t)s.size());
  });
}

PyMethodDef methods[] = {
    {"form", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(form)), METH_FASTCALL,
     "What a plan depends on, of these arguments, as bytes."},
    {"call", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(call)), METH_FASTCALL,
     "Calls a C function by its address."},
    {"addresses", addresses, METH_O, "The addresses of tensors, as an array."},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tx_calls", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

} // namespace

PyMODINIT_FUNC PyInit__tx_calls(void) { return PyModule_Create(&module); }
