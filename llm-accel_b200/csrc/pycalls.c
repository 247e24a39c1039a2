/* Calls of the C ABI from Python for what a serving loop calls at every step: the operators that take
 * device pointers and a stream.  Through ctypes a call of 17 arguments costs 4 us, more than its
 * launches; here it costs a tenth of that.  llmx.py binds the addresses of the library that it
 * has loaded and uses ctypes for all else, and for these too where this module was not built.
 *
 * Arguments are whole numbers, longer ones cut to the parameter's size.  Pointers are too, or None for NULL, but nothing
 * that merely has an __index__: a tensor of one element has, and its value is not its address.  A call with anything
 * else (a ctypes pointer, say, or None in a number's place) goes through ctypes after all, which takes it or says
 * what is wrong.  The result is the status code. */
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <stdint.h>

#include "llmx.h"

static PyObject *integral; /* numbers.Integral */

/* kinds: a letter per argument, P where it is a pointer. */
static int arguments(const char *name, const char *kinds, PyObject *const *args, Py_ssize_t got, Py_ssize_t want, unsigned long long *out) {
    if (got != want) {
        PyErr_Format(PyExc_TypeError, "%s takes %zd arguments, got %zd", name, want, got);
        return 0;
    }
    for (Py_ssize_t i = 0; i < want; i++) {
        if (args[i] == Py_None && kinds[i] == 'P') {
            out[i] = 0;
            continue;
        }
        if (kinds[i] == 'P' && !PyLong_Check(args[i])) {
            const int is = PyObject_IsInstance(args[i], integral);
            if (is == 0) PyErr_Format(PyExc_TypeError, "%s: argument %zd is not an address", name, i + 1);
            if (is <= 0) return 0;
        }
        out[i] = PyLong_AsUnsignedLongLongMask(args[i]);
        if (out[i] == (unsigned long long)-1 && PyErr_Occurred()) return 0;
    }
    return 1;
}

#define P(type, i) ((type)(uintptr_t)a[i])
#define U(i) ((uint32_t)a[i])
#define Z(i) ((size_t)a[i])
/* A function of this module: the bound address, and the call with its arguments a[0], a[1] and on, one for each letter
 * of kinds (P, U and Z, as below; I: int). */
#define CALL(fn, kinds, ...)                                                          \
    static __typeof__(&fn) p_##fn;                                                    \
    static PyObject *o_##fn; /* the same function through ctypes */                   \
    static PyObject *c_##fn(PyObject *self, PyObject *const *args, Py_ssize_t got) {  \
        unsigned long long a[sizeof(kinds) - 1];                                      \
        int rc;                                                                       \
        (void)self;                                                                   \
        if (!p_##fn) {                                                                \
            PyErr_SetString(PyExc_RuntimeError, #fn " is not bound");                 \
            return NULL;                                                              \
        }                                                                             \
        if (!arguments(#fn, kinds, args, got, (Py_ssize_t)sizeof(kinds) - 1, a)) {    \
            if (!PyErr_ExceptionMatches(PyExc_TypeError)) return NULL;                \
            PyErr_Clear();                                                            \
            return PyObject_Vectorcall(o_##fn, args, (size_t)got, NULL);              \
        }                                                                             \
        Py_BEGIN_ALLOW_THREADS rc = p_##fn(__VA_ARGS__);                              \
        Py_END_ALLOW_THREADS return PyLong_FromLong(rc);                              \
    }

CALL(llmx_adapters_project, "PPUZPPIZP", P(llmx_adapters *, 0), P(const int16_t *, 1), U(2), Z(3), P(const int32_t *, 4), P(void *, 5), (int)a[6], Z(7),
     P(void *, 8))
CALL(llmx_verify_drafts, "PZPZUPPUUUPPPPPPPZP", P(const int32_t *, 0), Z(1), P(const int32_t *, 2), Z(3), U(4), P(const uint32_t *, 5), P(const uint32_t *, 6), U(7),
     U(8), U(9), P(const float *, 10), P(const uint32_t *, 11), P(const uint32_t *, 12), P(uint32_t *, 13), P(uint32_t *, 14), P(uint64_t *, 15),
     P(void *, 16), Z(17), P(void *, 18))
CALL(llmx_token_logprobs, "PZUUPPUPPPPPPZP", P(const int32_t *, 0), Z(1), U(2), U(3), P(const uint32_t *, 4), P(const float *, 5), U(6), P(float *, 7),
     P(uint32_t *, 8), P(float *, 9), P(uint32_t *, 10), P(float *, 11), P(void *, 12), Z(13), P(void *, 14))
CALL(llmx_paged_append, "PPUZPPUPUPZPPUPZP", P(llmx_paged *, 0), P(const int16_t *, 1), U(2), Z(3), P(const uint32_t *, 4), P(const uint32_t *, 5), U(6),
     P(const int16_t *, 7), U(8), P(const int32_t *, 9), Z(10), P(int16_t *, 11), P(int16_t *, 12), U(13), P(int16_t *, 14), Z(15), P(void *, 16))
CALL(llmx_paged_attention, "PPUZPPUUPZPPUPZP", P(llmx_paged *, 0), P(const int16_t *, 1), U(2), Z(3), P(const uint32_t *, 4), P(const uint32_t *, 5), U(6), U(7),
     P(const int32_t *, 8), Z(9), P(const int16_t *, 10), P(const int16_t *, 11), U(12), P(int16_t *, 13), Z(14), P(void *, 15))

/* bind(name, address, function): where the library's function of that name is, and the same through ctypes. */
static PyObject *bind(PyObject *self, PyObject *args) {
    const char *name;
    unsigned long long address;
    PyObject *function;
    (void)self;
    if (!PyArg_ParseTuple(args, "sKO", &name, &address, &function)) return NULL;
#define BIND(fn)                                                     \
    if (strcmp(name, #fn) == 0) {                                    \
        p_##fn = (__typeof__(&fn))(uintptr_t)address;                \
        Py_INCREF(function);                                         \
        Py_XSETREF(o_##fn, function);                                \
        Py_RETURN_NONE;                                              \
    }
    BIND(llmx_adapters_project)
    BIND(llmx_verify_drafts)
    BIND(llmx_token_logprobs)
    BIND(llmx_paged_append)
    BIND(llmx_paged_attention)
#undef BIND
    PyErr_Format(PyExc_KeyError, "%s", name);
    return NULL;
}

#define ENTRY(fn) {#fn, (PyCFunction)(void (*)(void))c_##fn, METH_FASTCALL, NULL}
static PyMethodDef methods[] = {ENTRY(llmx_adapters_project), ENTRY(llmx_verify_drafts),   ENTRY(llmx_token_logprobs), ENTRY(llmx_paged_append),
                                ENTRY(llmx_paged_attention),  {"bind", bind, METH_VARARGS, NULL}, {NULL, NULL, 0, NULL}};
static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_llmxcalls", NULL, -1, methods, NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__llmxcalls(void) {
    PyObject *numbers = PyImport_ImportModule("numbers");
    if (!numbers) return NULL;
    Py_XSETREF(integral, PyObject_GetAttrString(numbers, "Integral"));
    Py_DECREF(numbers);
    return integral ? PyModule_Create(&module) : NULL;
}
