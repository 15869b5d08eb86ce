/* pyaddr.c -- the Python binding's pointer marshalling.
 *
 * The ctypes binding hands numpy buffers to the C ABI as plain addresses.
 * numpy's own route (ndarray.ctypes.data_as) builds several Python objects per
 * array and costs microseconds; for the small one-shot calls that is a large
 * share of the call.  addr(obj) reads the address through the buffer protocol
 * instead (C-contiguous buffers only; None -> None).  Host code only: no HIP.
 *
 * invoke(function, spec, args...) calls an entry point on torch tensors: it reads
 * data_ptr() and stride() itself and calls through a plain pointer, without a
 * ctypes object per argument (cross attention of one token 11.0 -> 8.2 us a
 * call, its gradient 21.0 -> 16.5, layer norm 9.3 -> 8.1).  spec has a letter for each argument: 't' a tensor
 * [batch, heads, rows, d] as lcDeviceTensor*, 'p' a tensor's address or None,
 * 'i' an integer or an address.  Every argument travels as a 64-bit integer, as
 * the x86-64 ABI passes pointers, sizes, strides and enums alike; unused ones
 * are ignored by the callee.  Returns the status, or -1 - k when tensor argument
 * k's last dimension is not contiguous (nothing is called then).
 */
#define PY_SSIZE_T_CLEAN
#include <Python.h>

static PyObject* lc_addr(PyObject* self, PyObject* obj) {
  (void)self;
  if (obj == Py_None) {
    Py_RETURN_NONE;
  }
  Py_buffer view;
  if (PyObject_GetBuffer(obj, &view, PyBUF_C_CONTIGUOUS) != 0) {
    return NULL;
  }
  /* The caller keeps obj alive for the duration of the C call. */
  PyObject* r = PyLong_FromVoidPtr(view.buf);
  PyBuffer_Release(&view);
  return r;
}

#define LC_MOST_ARGS 16
typedef int (*lc_entry)(long long, long long, long long, long long, long long, long long, long long, long long, long long,
                        long long, long long, long long, long long, long long, long long, long long);

static PyObject* kDataPtr;
static PyObject* kStride;
static PyObject* kShape;

struct lc_tensor { /* lcDeviceTensor */
  long long data, sb, sh, ss;
};

static int lc_address(PyObject* tensor, long long* out) {
  PyObject* r = PyObject_CallMethodObjArgs(tensor, kDataPtr, NULL);
  if (r == NULL) {
    return -1;
  }
  *out = (long long)PyLong_AsUnsignedLongLong(r);
  Py_DECREF(r);
  return PyErr_Occurred() ? -1 : 0;
}

/* 1: the last dimension is not contiguous. */
static int lc_view(PyObject* tensor, struct lc_tensor* out) {
  PyObject* st;
  long long last;
  if (lc_address(tensor, &out->data) != 0 || (st = PyObject_CallMethodObjArgs(tensor, kStride, NULL)) == NULL) {
    return -1;
  }
  if (!PyTuple_Check(st) || PyTuple_GET_SIZE(st) != 4) {
    Py_DECREF(st);
    PyErr_SetString(PyExc_ValueError, "a tensor of four dimensions is needed");
    return -1;
  }
  out->sb = PyLong_AsLongLong(PyTuple_GET_ITEM(st, 0));
  out->sh = PyLong_AsLongLong(PyTuple_GET_ITEM(st, 1));
  out->ss = PyLong_AsLongLong(PyTuple_GET_ITEM(st, 2));
  last = PyLong_AsLongLong(PyTuple_GET_ITEM(st, 3));
  Py_DECREF(st);
  if (PyErr_Occurred()) {
    return -1;
  }
  if (last != 1) { /* the stride of a dimension of one value means nothing */
    PyObject* shape = PyObject_GetAttr(tensor, kShape);
    PyObject* d = shape != NULL ? PySequence_GetItem(shape, 3) : NULL;
    const long long n = d != NULL ? PyLong_AsLongLong(d) : 0;
    Py_XDECREF(shape);
    Py_XDECREF(d);
    if (PyErr_Occurred()) {
      return -1;
    }
    return n > 1 ? 1 : 0;
  }
  return 0;
}

static PyObject* lc_invoke(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  struct lc_tensor views[LC_MOST_ARGS];
  long long a[LC_MOST_ARGS] = {0};
  int tensors = 0, status;
  Py_ssize_t len, i;
  const char* spec;
  lc_entry entry;
  (void)self;
  if (n < 2 || (spec = PyUnicode_AsUTF8AndSize(args[1], &len)) == NULL) {
    if (!PyErr_Occurred()) {
      PyErr_SetString(PyExc_TypeError, "invoke(function, spec, args...)");
    }
    return NULL;
  }
  if (len != n - 2 || len > LC_MOST_ARGS) {
    PyErr_SetString(PyExc_TypeError, "invoke: the arguments do not match the spec");
    return NULL;
  }
  entry = (lc_entry)(size_t)PyLong_AsUnsignedLongLong(args[0]);
  if (PyErr_Occurred()) {
    return NULL;
  }
  for (i = 0; i < len; ++i) {
    PyObject* x = args[i + 2];
    if (spec[i] == 't') {
      const int r = lc_view(x, &views[tensors]);
      if (r < 0) {
        return NULL;
      }
      if (r > 0) {
        return PyLong_FromLong(-1 - tensors);
      }
      a[i] = (long long)(size_t)&views[tensors++];
    } else if (spec[i] == 'p') {
      if (x != Py_None && lc_address(x, &a[i]) != 0) {
        return NULL;
      }
    } else {
      a[i] = PyLong_AsLongLong(x);
      if (a[i] == -1 && PyErr_Occurred()) { /* addresses and sizes past 2^63 */
        PyErr_Clear();
        a[i] = (long long)PyLong_AsUnsignedLongLong(x);
        if (PyErr_Occurred()) {
          return NULL;
        }
      }
    }
  }
  Py_BEGIN_ALLOW_THREADS
  status = entry(a[0], a[1], a[2], a[3], a[4], a[5], a[6], a[7], a[8], a[9], a[10], a[11], a[12], a[13], a[14], a[15]);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(status);
}

static PyMethodDef kMethods[] = {
    {"invoke", (PyCFunction)(void (*)(void))lc_invoke, METH_FASTCALL, "Calls an entry point on torch tensors."},
    {"addr", lc_addr, METH_O, "Address of a C-contiguous buffer (None -> None)."},
    {NULL, NULL, 0, NULL},
};

static struct PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_addr", NULL, -1, kMethods, NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__addr(void) {
  kDataPtr = PyUnicode_InternFromString("data_ptr");
  kStride = PyUnicode_InternFromString("stride");
  kShape = PyUnicode_InternFromString("shape");
  if (kDataPtr == NULL || kStride == NULL || kShape == NULL) {
    return NULL;
  }
  return PyModule_Create(&kModule);
}
