// The calls of the decode step in 4 bits for Python, without ctypes: arguments go from Python objects to the C ABI's types here, tensors by their
// data_ptr(). A decode step in eager mode is as fast as its calls are made: ctypes and the conversions in Python take 2.5 us of the 4.9 of a call with
// thirteen arguments, this 0.8.
//
// The functions' addresses come from the library that the package has loaded (bind), so that there is one library, whichever it is.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <cstdint>
#include <tuple>
#include <utility>

#include "w8a8.h"

namespace {

PyObject* data_ptr_name;

// None, a number, or what has a data_ptr().
bool to_c(PyObject* o, void** out) {
    if (o == Py_None) {
        *out = nullptr;
        return true;
    }
    if (PyLong_Check(o)) {
        *out = PyLong_AsVoidPtr(o);
    } else {
        PyObject* address = PyObject_CallMethodNoArgs(o, data_ptr_name);
        if (!address) return false;
        *out = PyLong_AsVoidPtr(address);
        Py_DECREF(address);
    }
    return *out || !PyErr_Occurred();
}
bool to_c(PyObject* o, int* out) {
    const long v = PyLong_AsLong(o);
    if (v == -1 && PyErr_Occurred()) return false;
    if (v < INT32_MIN || v > INT32_MAX) {
        PyErr_Format(PyExc_OverflowError, "%ld does not fit an int", v);
        return false;
    }
    *out = static_cast<int>(v);
    return true;
}
bool to_c(PyObject* o, float* out) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) return false;
    *out = static_cast<float>(v);
    return true;
}
template <class T>
bool to_c(PyObject* o, T** out) {
    void* p;
    if (!to_c(o, &p)) return false;
    *out = static_cast<T*>(p);
    return true;
}

template <class... A, size_t... I>
PyObject* call(int (*fn)(A...), PyObject* const* args, Py_ssize_t n, std::index_sequence<I...>) {
    if (!fn || n != static_cast<Py_ssize_t>(sizeof...(A))) {
        PyErr_Format(PyExc_TypeError, fn ? "%zd arguments for %zd" : "not bound", n, static_cast<Py_ssize_t>(sizeof...(A)));
        return nullptr;
    }
    std::tuple<A...> values;
    if (!(to_c(args[I], &std::get<I>(values)) && ...)) return nullptr;
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = fn(std::get<I>(values)...);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(status);
}
template <class... A>
PyObject* call(int (*fn)(A...), PyObject* const* args, Py_ssize_t n) {
    return call(fn, args, n, std::index_sequence_for<A...>());
}

#define CALLS(X)                                                                                                                          \
    X(w8a8_plan_blocks) X(w8a8_kv4_write) X(w8a8_kv4_read) X(w8a8_kv4_attention_decode) X(w8a8_kv4_attention_decode_ahead) X(w8a8_linear4_q)
#define DEFINE(name)                                                                       \
    decltype(&::name) at_##name;                                                           \
    PyObject* py_##name(PyObject*, PyObject* const* args, Py_ssize_t n) { return call(at_##name, args, n); }
CALLS(DEFINE)

struct Bound {
    const char* name;
    void** at;
};
#define BOUND(name) {#name, reinterpret_cast<void**>(&at_##name)},
const Bound bound[] = {CALLS(BOUND)};

PyObject* bind(PyObject*, PyObject* addresses) {  // {name: address}
    for (const Bound& b : bound) {
        PyObject* address = PyMapping_GetItemString(addresses, b.name);
        if (!address) return nullptr;
        *b.at = PyLong_AsVoidPtr(address);
        Py_DECREF(address);
        if (PyErr_Occurred()) return nullptr;
    }
    Py_RETURN_NONE;
}

#define METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_##name)), METH_FASTCALL, nullptr},
PyMethodDef methods[] = {CALLS(METHOD){"bind", bind, METH_O, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "w8a8_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_w8a8_calls() {
    data_ptr_name = PyUnicode_InternFromString("data_ptr");
    return data_ptr_name ? PyModule_Create(&module) : nullptr;
}
