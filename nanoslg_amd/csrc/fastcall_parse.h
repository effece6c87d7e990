/* Conversion of a fast call's Python arguments by the codes of its signature: p pointer (an int; None for
 * NULL), q int64, i int32, z size_t, f float. */
#ifndef NSLG_FASTCALL_PARSE_H
#define NSLG_FASTCALL_PARSE_H

#include <Python.h>
#include <stdint.h>
#include <string.h>

typedef union {
  void* p;
  int64_t q;
  int32_t i;
  size_t z;
  float f;
} arg_t;

#define MAX_ARGS 40

/* Convert args[0..n) by the codes of sig into out; 0, or -1 with a Python error. */
static int parse(const char* name, const char* sig, PyObject* const* args, Py_ssize_t n, arg_t* out) {
  const Py_ssize_t want = (Py_ssize_t)strlen(sig);
  if (n != want) {
    PyErr_Format(PyExc_TypeError, "%s takes %zd arguments (%zd given)", name, want, n);
    return -1;
  }
  for (Py_ssize_t k = 0; k < n; ++k) {
    PyObject* o = args[k];
    switch (sig[k]) {
      case 'p':
        if (o == Py_None) {
          out[k].p = NULL;
        } else {
          out[k].p = PyLong_AsVoidPtr(o);
          if (out[k].p == NULL && PyErr_Occurred()) return -1;
        }
        break;
      case 'q': {
        long long v = PyLong_AsLongLong(o);
        if (v == -1 && PyErr_Occurred()) return -1;
        out[k].q = (int64_t)v;
        break;
      }
      case 'z': {
        unsigned long long v = PyLong_AsUnsignedLongLong(o);
        if (v == (unsigned long long)-1 && PyErr_Occurred()) return -1;
        out[k].z = (size_t)v;
        break;
      }
      case 'i': {
        long v = PyLong_AsLong(o);
        if (v == -1 && PyErr_Occurred()) return -1;
        if (v < INT32_MIN || v > INT32_MAX) {
          PyErr_Format(PyExc_OverflowError, "%s: argument %zd out of int32 range", name, k);
          return -1;
        }
        out[k].i = (int32_t)v;
        break;
      }
      case 'f': {
        double v = PyFloat_AsDouble(o);
        if (v == -1.0 && PyErr_Occurred()) return -1;
        out[k].f = (float)v;
        break;
      }
      default:
        PyErr_Format(PyExc_SystemError, "%s: bad signature code", name);
        return -1;
    }
  }
  return 0;
}

#endif
