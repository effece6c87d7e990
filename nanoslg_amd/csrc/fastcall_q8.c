/*
 * _nslg_fast_q8: a CPython binding of the 8-bit cache's entry points (nslg_q8_* of nslg_kv.h), as _nslg_fast is of
 * the others': the entry point's arguments in order, as Python ints (pointers, sizes) and a float (the softmax
 * scale); returns its status. Small decode batches are paced by the host's Python: ctypes converts the
 * 38 arguments of a decode call in about 4 us, this in under 1.
 */
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include "../../include/nslg_kv.h"
#include "fastcall_parse.h"

static PyObject* append_kv(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  (void)self;
  arg_t a[MAX_ARGS];
  if (parse("q8_append_kv", "pqpqppiqppppqipppiiiiip", args, n, a)) return NULL;
  const int rc = nslg_q8_append_kv(
      a[0].p, a[1].q, a[2].p, a[3].q, a[4].p, a[5].p, a[6].i, a[7].q, a[8].p, a[9].p, a[10].p, a[11].p,
      a[12].q, a[13].i, a[14].p, a[15].p, a[16].p, a[17].i, a[18].i, a[19].i, a[20].i, a[21].i,
      a[22].p);
  return PyLong_FromLong(rc);
}

static PyObject* gather_kv(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  (void)self;
  arg_t a[MAX_ARGS];
  if (parse("q8_gather_kv", "ppppqipppiiiiiippp", args, n, a)) return NULL;
  const int rc = nslg_q8_gather_kv(
      a[0].p, a[1].p, a[2].p, a[3].p, a[4].q, a[5].i, a[6].p, a[7].p, a[8].p, a[9].i, a[10].i, a[11].i,
      a[12].i, a[13].i, a[14].i, a[15].p, a[16].p, a[17].p);
  return PyLong_FromLong(rc);
}

static PyObject* paged_decode(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  (void)self;
  arg_t a[MAX_ARGS];
  if (parse("q8_paged_decode", "pqpqpqpppqqppppqipppqiiiifiipipppqpzqp", args, n, a)) return NULL;
  const int rc = nslg_q8_paged_decode(
      a[0].p, a[1].q, a[2].p, a[3].q, a[4].p, a[5].q, a[6].p, a[7].p, a[8].p, a[9].q, a[10].q, a[11].p,
      a[12].p, a[13].p, a[14].p, a[15].q, a[16].i, a[17].p, a[18].p, a[19].p, a[20].q, a[21].i,
      a[22].i, a[23].i, a[24].i, a[25].f, a[26].i, a[27].i, a[28].p, a[29].i, a[30].p, a[31].p,
      a[32].p, a[33].q, a[34].p, a[35].z, a[36].q, a[37].p);
  return PyLong_FromLong(rc);
}

static PyObject* paged_prefill(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  (void)self;
  arg_t a[MAX_ARGS];
  if (parse("q8_paged_prefill", "pqppiqippppqipppiiiifiipqpzp", args, n, a)) return NULL;
  const int rc = nslg_q8_paged_prefill(
      a[0].p, a[1].q, a[2].p, a[3].p, a[4].i, a[5].q, a[6].i, a[7].p, a[8].p, a[9].p, a[10].p, a[11].q,
      a[12].i, a[13].p, a[14].p, a[15].p, a[16].i, a[17].i, a[18].i, a[19].i, a[20].f, a[21].i,
      a[22].i, a[23].p, a[24].q, a[25].p, a[26].z, a[27].p);
  return PyLong_FromLong(rc);
}

static PyMethodDef methods[] = {
    {"append_kv", (PyCFunction)(void (*)(void))append_kv, METH_FASTCALL,
     "nslg_q8_append_kv: the entry point's arguments in order; returns its status"},
    {"gather_kv", (PyCFunction)(void (*)(void))gather_kv, METH_FASTCALL,
     "nslg_q8_gather_kv: the entry point's arguments in order; returns its status"},
    {"paged_decode", (PyCFunction)(void (*)(void))paged_decode, METH_FASTCALL,
     "nslg_q8_paged_decode: the entry point's arguments in order; returns its status"},
    {"paged_prefill", (PyCFunction)(void (*)(void))paged_prefill, METH_FASTCALL,
     "nslg_q8_paged_prefill: the entry point's arguments in order; returns its status"},
    {NULL, NULL, 0, NULL}};

static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_nslg_fast_q8",
                                    "Fast-call binding of the 8-bit cache's entry points of libnslg_kv", -1, methods,
                                    NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__nslg_fast_q8(void) { return PyModule_Create(&module); }
