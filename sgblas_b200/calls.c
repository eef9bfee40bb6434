/* The entry points around the language-model products (sgblas_lm.h) as functions of
 * Python, for calls whose own time is a few microseconds: ctypes spends two of them on
 * converting fifteen arguments, this a quarter of one. The same arguments in the
 * same order as the C functions; device pointers are tensors (anything with data_ptr()),
 * integer addresses or None, *beta a number or None. Returns the status.
 *
 * The functions' addresses are given by bind(), so that this module and ctypes call one
 * and the same library. */
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <limits.h>

#include <sgblas/sgblas_lm.h>

#define MAX_ARGS 24

typedef union Value {
  void *p;
  int i;
  long long l;
  float f;
  const float *scalar;
} Value;

static PyObject *data_ptr_name;

static int toPointer(PyObject *o, void **out) {
  if (o == Py_None) {
    *out = NULL;
    return 0;
  }
  if (PyLong_Check(o)) {
    *out = PyLong_AsVoidPtr(o);
    return *out == NULL && PyErr_Occurred() ? -1 : 0;
  }
  PyObject *address = PyObject_CallMethodNoArgs(o, data_ptr_name);
  if (address == NULL) return -1;
  *out = PyLong_AsVoidPtr(address);
  Py_DECREF(address);
  return *out == NULL && PyErr_Occurred() ? -1 : 0;
}

static int toLong(PyObject *o, long long low, long long high, long long *out) {
  PyObject *index = PyLong_Check(o) ? Py_NewRef(o) : PyNumber_Index(o);
  if (index == NULL) return -1;
  *out = PyLong_AsLongLong(index);
  Py_DECREF(index);
  if (*out == -1 && PyErr_Occurred()) return -1;
  if (*out < low || *out > high) {
    PyErr_SetString(PyExc_OverflowError, "an argument does not fit its C type");
    return -1;
  }
  return 0;
}

/* Converts the arguments by `signature`, a letter each: p a pointer, i an int, l a long long,
 * f a float, s a pointer to one (held in `scalars`). */
static int convert(const char *name, const char *signature, PyObject *const *args, Py_ssize_t count,
                   Value *out, float *scalars) {
  const Py_ssize_t wanted = (Py_ssize_t)strlen(signature);
  if (count != wanted) {
    PyErr_Format(PyExc_TypeError, "%s takes %zd arguments (%zd given)", name, wanted, count);
    return -1;
  }
  for (Py_ssize_t k = 0; k < count; ++k) {
    long long v = 0;
    double d = 0.0;
    switch (signature[k]) {
      case 'p':
        if (toPointer(args[k], &out[k].p) != 0) return -1;
        break;
      case 'i':
        if (toLong(args[k], INT_MIN, INT_MAX, &v) != 0) return -1;
        out[k].i = (int)v;
        break;
      case 'l':
        if (toLong(args[k], LLONG_MIN, LLONG_MAX, &out[k].l) != 0) return -1;
        break;
      default:
        if (signature[k] == 's' && args[k] == Py_None) {
          out[k].scalar = NULL;
          break;
        }
        d = PyFloat_AsDouble(args[k]);
        if (d == -1.0 && PyErr_Occurred()) return -1;
        scalars[k] = (float)d;
        if (signature[k] == 's') out[k].scalar = &scalars[k];
        else out[k].f = scalars[k];
    }
  }
  return 0;
}

/* A method NAME of the C function FUNCTION: its signature, and the call with converted
 * arguments v. */
#define METHOD(NAME, FUNCTION, SIGNATURE, ...)                                                  \
  static __typeof__(FUNCTION) *NAME##_at;                                                       \
  static PyObject *NAME(PyObject *self, PyObject *const *args, Py_ssize_t count) {              \
    (void)self;                                                                                 \
    Value v[MAX_ARGS];                                                                          \
    float scalars[MAX_ARGS];                                                                    \
    _Static_assert(sizeof(SIGNATURE) - 1 <= MAX_ARGS, "arguments");                             \
    if (NAME##_at == NULL) {                                                                    \
      PyErr_SetString(PyExc_RuntimeError, #NAME " is not bound to a library");                  \
      return NULL;                                                                              \
    }                                                                                           \
    if (convert(#NAME, SIGNATURE, args, count, v, scalars) != 0) return NULL;                   \
    int status;                                                                                 \
    Py_BEGIN_ALLOW_THREADS                                                                      \
    status = NAME##_at(__VA_ARGS__);                                                            \
    Py_END_ALLOW_THREADS                                                                        \
    return PyLong_FromLong(status);                                                             \
  }

METHOD(rms_norm, sgblasRmsNorm, "piiipipipfpipipipi", v[0].p, v[1].i, v[2].i, v[3].i, v[4].p, v[5].i, v[6].p, v[7].i,
       v[8].p, v[9].f, v[10].p, v[11].i, v[12].p, v[13].i, v[14].p, v[15].i, v[16].p, v[17].i)
METHOD(rms_norm_backward, sgblasRmsNormBackward, "piiipipipfpipisp", v[0].p, v[1].i, v[2].i, v[3].i, v[4].p, v[5].i,
       v[6].p, v[7].i, v[8].p, v[9].f, v[10].p, v[11].i, v[12].p, v[13].i, v[14].scalar, v[15].p)
METHOD(sort_tokens, sgblasSortTokens, "piiippp", v[0].p, v[1].i, v[2].i, v[3].i, v[4].p, v[5].p, v[6].p)
METHOD(scatter_tokens, sgblasScatterTokens, "piiiipppiipi", v[0].p, v[1].i, v[2].i, v[3].i, v[4].i, v[5].p, v[6].p,
       v[7].p, v[8].i, v[9].i, v[10].p, v[11].i)
METHOD(gather_tokens, sgblasGatherTokens, "piiiipppiipi", v[0].p, v[1].i, v[2].i, v[3].i, v[4].i, v[5].p, v[6].p,
       v[7].p, v[8].i, v[9].i, v[10].p, v[11].i)
METHOD(gather_tokens_backward, sgblasGatherTokensBackward, "piiiipppiipipip", v[0].p, v[1].i, v[2].i, v[3].i, v[4].i,
       v[5].p, v[6].p, v[7].p, v[8].i, v[9].i, v[10].p, v[11].i, v[12].p, v[13].i, v[14].p)
METHOD(quantize_fp4, sgblasQuantizeFp4, "piiipiilpilpil", v[0].p, v[1].i, v[2].i, v[3].i, v[4].p, v[5].i, v[6].i,
       v[7].l, v[8].p, v[9].i, v[10].l, v[11].p, v[12].i, v[13].l)
METHOD(gemm_fp4, sgblasGemmFp4, "piiipipipipipii", v[0].p, v[1].i, v[2].i, v[3].i, v[4].p, v[5].i, v[6].p, v[7].i,
       v[8].p, v[9].i, v[10].p, v[11].i, v[12].p, v[13].i, v[14].i)
METHOD(grouped_gemm_fp4, sgblasGroupedGemmFp4, "piiiippilpilpipipii", v[0].p, v[1].i, v[2].i, v[3].i, v[4].i, v[5].p,
       v[6].p, v[7].i, v[8].l, v[9].p, v[10].i, v[11].l, v[12].p, v[13].i, v[14].p, v[15].i, v[16].p, v[17].i, v[18].i)

/* bind(name, address): the function that name's method calls. */
static PyObject *bind(PyObject *self, PyObject *const *args, Py_ssize_t count) {
  (void)self;
  if (count != 2) {
    PyErr_SetString(PyExc_TypeError, "bind takes a name and an address");
    return NULL;
  }
  const char *name = PyUnicode_AsUTF8(args[0]);
  if (name == NULL) return NULL;
  void *at = PyLong_AsVoidPtr(args[1]);
  if (at == NULL && PyErr_Occurred()) return NULL;
#define BIND(NAME)                     \
  if (strcmp(name, #NAME) == 0) {      \
    *(void **)(&NAME##_at) = at;       \
    Py_RETURN_NONE;                    \
  }
  BIND(rms_norm)
  BIND(rms_norm_backward)
  BIND(sort_tokens)
  BIND(scatter_tokens)
  BIND(gather_tokens)
  BIND(gather_tokens_backward)
  BIND(quantize_fp4)
  BIND(gemm_fp4)
  BIND(grouped_gemm_fp4)
  PyErr_Format(PyExc_ValueError, "no method %s", name);
  return NULL;
}

#define ENTRY(NAME) {#NAME, (PyCFunction)(void (*)(void))NAME, METH_FASTCALL, NULL}
static PyMethodDef methods[] = {ENTRY(rms_norm), ENTRY(rms_norm_backward), ENTRY(sort_tokens), ENTRY(scatter_tokens),
                                ENTRY(gather_tokens), ENTRY(gather_tokens_backward), ENTRY(quantize_fp4),
                                ENTRY(gemm_fp4), ENTRY(grouped_gemm_fp4), ENTRY(bind), {NULL, NULL, 0, NULL}};

static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", NULL, -1, methods, NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__calls(void) {
  data_ptr_name = PyUnicode_InternFromString("data_ptr");
  if (data_ptr_name == NULL) return NULL;
  return PyModule_Create(&module);
}
