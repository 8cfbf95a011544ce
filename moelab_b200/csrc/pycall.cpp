// CPython module over the calls that a decode step makes for every layer (moeb_kv_write, moeb_kv_read, moeb_kv_attention). They
// last 3 us on the host with their launch; ctypes needs 2 us more for the 22 arguments of an attention call, this module
// 0.4 (call from Python 10.0 -> 7.8 us, kv_write 7.5 -> 5.8). Arguments come in the order of include/moelab_b200.h, pointers as integers or None; the status comes back. The functions'
// addresses are those of the loaded library (bind), so nothing is linked here. The GIL is released during a call.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <limits.h>

#include "../../include/moelab_b200.h"

namespace {

decltype(&moeb_kv_write) write_fn;
decltype(&moeb_kv_read) read_fn;
decltype(&moeb_kv_attention) attention_fn;

// Converts arguments one after the other; after the first that does not convert, `bad` is set with a Python exception.
struct Args {
    PyObject *const *at;
    bool bad = false;
    template <typename T>
    operator T *() {  // a pointer: None or an integer
        PyObject *o = *at++;
        if (bad || o == Py_None) return nullptr;
        void *p = PyLong_AsVoidPtr(o);
        if (!p && PyErr_Occurred()) bad = true;
        return static_cast<T *>(p);
    }
    operator long() {
        PyObject *o = *at++;
        if (bad) return 0;
        const long v = PyLong_AsLong(o);
        if (v == -1 && PyErr_Occurred()) bad = true;
        return v;
    }
    operator int() {
        const long v = *this;
        if (v >= INT_MIN && v <= INT_MAX) return (int)v;
        if (!bad) PyErr_SetString(PyExc_OverflowError, "an argument does not fit 32 bits");
        bad = true;
        return 0;
    }
    operator size_t() { return (size_t) static_cast<long>(*this); }
    operator float() {
        PyObject *o = *at++;
        if (bad) return 0.f;
        const double v = PyFloat_AsDouble(o);
        if (v == -1.0 && PyErr_Occurred()) bad = true;
        return (float)v;
    }
};

// The values are converted left to right: a braced list is evaluated in order.
template <typename... T>
struct Values;
template <>
struct Values<> {
    explicit Values(Args &) {}
    template <typename F, typename... V>
    int call(F f, V... v) { return f(v...); }
};
template <typename H, typename... T>
struct Values<H, T...> {
    H head;
    Values<T...> tail;
    explicit Values(Args &a) : head(a), tail(a) {}
    template <typename F, typename... V>
    int call(F f, V... v) { return tail.call(f, v..., head); }
};

template <typename... T>
PyObject *forward(int (*f)(T...), PyObject *const *args, Py_ssize_t n) {
    if (n != (Py_ssize_t)sizeof...(T)) return PyErr_Format(PyExc_TypeError, "%d arguments, %zd given", (int)sizeof...(T), n);
    if (!f) return PyErr_Format(PyExc_RuntimeError, "bind() has not been called");
    Args a{args};
    Values<T...> v(a);
    if (a.bad) return nullptr;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = v.call(f);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}

PyObject *kv_write(PyObject *, PyObject *const *args, Py_ssize_t n) { return forward(write_fn, args, n); }
PyObject *kv_read(PyObject *, PyObject *const *args, Py_ssize_t n) { return forward(read_fn, args, n); }
PyObject *kv_attention(PyObject *, PyObject *const *args, Py_ssize_t n) { return forward(attention_fn, args, n); }

PyObject *bind(PyObject *, PyObject *args) {
    unsigned long long w, r, a;
    if (!PyArg_ParseTuple(args, "KKK", &w, &r, &a)) return nullptr;
    write_fn = reinterpret_cast<decltype(write_fn)>(w);
    read_fn = reinterpret_cast<decltype(read_fn)>(r);
    attention_fn = reinterpret_cast<decltype(attention_fn)>(a);
    Py_RETURN_NONE;
}

template <typename F>
PyCFunction fast(F f) {
    return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f));
}

PyMethodDef methods[] = {{"bind", bind, METH_VARARGS, "addresses of moeb_kv_write, moeb_kv_read, moeb_kv_attention"},
                         {"moeb_kv_write", fast(kv_write), METH_FASTCALL, nullptr},
                         {"moeb_kv_read", fast(kv_read), METH_FASTCALL, nullptr},
                         {"moeb_kv_attention", fast(kv_attention), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "moelab_b200_pycall", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_moelab_b200_pycall() { return PyModule_Create(&module); }
