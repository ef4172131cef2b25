/*
 * Python callables for the entry points whose smallest calls are bound by the host: the grouped products and the 8-bit ones.
 * A ctypes call converts 11 to 16 arguments through Python objects (about 1.3 us); these take integers (or None for a null
 * pointer) by the vector-call protocol and hand them to the C ABI (0.2 us).  Same arguments, same status code as through
 * ctypes, which serves where this module has not been built.
 */
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include "../../include/maize_gemm.h"

/* Integers 0 .. count-1 of `args`, None as 0; returns 0 with a Python error set if one is neither. */
static int take(const char *name, PyObject *const *args, Py_ssize_t given, Py_ssize_t count, unsigned long long *to)
{
    if (given != count) {
        PyErr_Format(PyExc_TypeError, "%s takes %zd arguments, got %zd", name, count, given);
        return 0;
    }
    for (Py_ssize_t i = 0; i < count; ++i) {
        if (args[i] == Py_None) {
            to[i] = 0;
            continue;
        }
        to[i] = PyLong_AsUnsignedLongLongMask(args[i]);
        if (to[i] == (unsigned long long)-1 && PyErr_Occurred())
            return 0;
    }
    return 1;
}

#define PTR(i) ((void *)(uintptr_t)v[i])
#define U64(i) ((uint64_t)v[i])
#define U32(i) ((uint32_t)v[i])

#define ENTRY(name, count, call)                                                       \
    static PyObject *py_##name(PyObject *self, PyObject *const *args, Py_ssize_t nargs) \
    {                                                                                  \
        unsigned long long v[count];                                                   \
        int status;                                                                    \
        (void)self;                                                                    \
        if (!take(#name, args, nargs, count, v))                                       \
            return NULL;                                                               \
        Py_BEGIN_ALLOW_THREADS status = (int)call;                                     \
        Py_END_ALLOW_THREADS return PyLong_FromLong(status);                           \
    }

ENTRY(maize_grouped_gemm_bf16, 14,
      maize_grouped_gemm_bf16(PTR(0), PTR(1), U64(2), PTR(3), U64(4), U64(5), PTR(6), U64(7), PTR(8), U32(9), U32(10), U32(11),
                              U32(12), PTR(13)))
ENTRY(maize_grouped_gemm_bf16_kn, 14,
      maize_grouped_gemm_bf16_kn(PTR(0), PTR(1), U64(2), PTR(3), U64(4), U64(5), PTR(6), U64(7), PTR(8), U32(9), U32(10), U32(11),
                                 U32(12), PTR(13)))
ENTRY(maize_grouped_gemm_bf16_wgrad, 14,
      maize_grouped_gemm_bf16_wgrad(PTR(0), PTR(1), U64(2), PTR(3), U64(4), PTR(5), U64(6), U64(7), PTR(8), U32(9), U32(10),
                                    U32(11), U32(12), PTR(13)))
ENTRY(maize_quantize_e4m3, 11,
      maize_quantize_e4m3(PTR(0), PTR(1), U64(2), U32(3), U32(4), U32(5), PTR(6), U64(7), PTR(8), U64(9), PTR(10)))
ENTRY(maize_gemm_e4m3, 15,
      maize_gemm_e4m3(PTR(0), PTR(1), U64(2), PTR(3), U64(4), PTR(5), U64(6), PTR(7), U64(8), PTR(9), U64(10), U32(11), U32(12),
                      U32(13), PTR(14)))

#define METHOD(name) {#name, (PyCFunction)(void (*)(void))py_##name, METH_FASTCALL, NULL}
static PyMethodDef methods[] = {
    METHOD(maize_grouped_gemm_bf16), METHOD(maize_grouped_gemm_bf16_kn), METHOD(maize_grouped_gemm_bf16_wgrad),
    METHOD(maize_quantize_e4m3),     METHOD(maize_gemm_e4m3),            {NULL, NULL, 0, NULL}};

static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "maize_calls", NULL, -1, methods, NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit_maize_calls(void) { return PyModule_Create(&module); }
