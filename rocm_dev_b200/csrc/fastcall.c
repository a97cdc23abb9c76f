/* CPython entry to the short calls of the library: the same functions that ctypes reaches, with their arguments converted
 * in C.  A 4-bit product of one token takes 6 us on the device; ctypes spends 1.2 us on a call with its 14
 * arguments.  Optional: without it (no Python headers) the package calls through ctypes.
 *   bind(quantize, dequantize, dense, skinny)   addresses of the library's functions, once
 *   quantize(...), dequantize(...), dense(...), skinny(...)   their arguments in order, None for NULL; returns the status */
#define PY_SSIZE_T_CLEAN
#define Py_LIMITED_API 0x030A0000
#include <Python.h>

#include "../../include/rocm_dev_b200.h"

static __typeof__(&rdb_quantize_fp4) g_quantize;
static __typeof__(&rdb_dequantize_fp4) g_dequantize;
static __typeof__(&rdb_dense_gemm_fp4_tuned) g_dense;
static __typeof__(&rdb_skinny_gemm_fp4) g_skinny;

/* Integers and addresses of up to 16 arguments; false with an exception set. */
static int numbers(PyObject *const *args, Py_ssize_t n, Py_ssize_t want, long long *v) {
    if (n != want) {
        PyErr_Format(PyExc_TypeError, "%zd arguments expected, got %zd", want, n);
        return 0;
    }
    for (Py_ssize_t i = 0; i < n; i++) {
        if (args[i] == Py_None) {
            v[i] = 0;
            continue;
        }
        v[i] = (long long)PyLong_AsUnsignedLongLongMask(args[i]);
        if (v[i] == -1 && PyErr_Occurred()) return 0;
    }
    return 1;
}
#define P(i) ((void *)(uintptr_t)v[i])
#define I(i) ((int)v[i])
#define FUNCTION(name, count, ...)                                                       \
    static PyObject *name(PyObject *self, PyObject *const *args, Py_ssize_t n) {         \
        long long v[count];                                                              \
        int status;                                                                      \
        (void)self;                                                                      \
        if (!numbers(args, n, count, v)) return NULL;                                    \
        if (!g_##name) {                                                                 \
            PyErr_SetString(PyExc_RuntimeError, "bind() first");                         \
            return NULL;                                                                 \
        }                                                                                \
        Py_BEGIN_ALLOW_THREADS                                                           \
        status = g_##name(__VA_ARGS__);                                                  \
        Py_END_ALLOW_THREADS                                                             \
        return PyLong_FromLong(status);                                                  \
    }

FUNCTION(quantize, 14, P(0), I(1), v[2], I(3), I(4), I(5), P(6), P(7), P(8), P(9), P(10), P(11), P(12), P(13))
FUNCTION(dequantize, 9, P(0), P(1), P(2), I(3), I(4), I(5), P(6), I(7), P(8))
FUNCTION(dense, 15, P(0), P(1), P(2), P(3), P(4), P(5), P(6), I(7), I(8), I(9), I(10), I(11), I(12), I(13), P(14))
FUNCTION(skinny, 14, P(0), P(1), P(2), P(3), P(4), P(5), P(6), I(7), I(8), I(9), I(10), I(11), (unsigned)v[12], P(13))

static PyObject *bind(PyObject *self, PyObject *const *args, Py_ssize_t n) {
    long long v[4];
    (void)self;
    if (!numbers(args, n, 4, v)) return NULL;
    g_quantize = (__typeof__(g_quantize))(uintptr_t)v[0];
    g_dequantize = (__typeof__(g_dequantize))(uintptr_t)v[1];
    g_dense = (__typeof__(g_dense))(uintptr_t)v[2];
    g_skinny = (__typeof__(g_skinny))(uintptr_t)v[3];
    Py_INCREF(Py_None);
    return Py_None;
}

#define METHOD(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, NULL}
static PyMethodDef methods[] = {METHOD(bind), METHOD(quantize), METHOD(dequantize), METHOD(dense), METHOD(skinny), {NULL, NULL, 0, NULL}};
static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fastcall", NULL, -1, methods, NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__fastcall(void) { return PyModule_Create(&module); }
