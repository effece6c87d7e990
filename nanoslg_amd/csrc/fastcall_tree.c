/*
 * _nslg_fast_tree: a CPython binding of the entry points for trees of drafted tokens, as _nslg_fast is of the cache's:
 * the entry point's arguments in order, as Python ints (pointers, sizes) and a float (the softmax scale); returns
 * its status.
 */
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include "../../include/nslg_kv.h"
#include "fastcall_parse.h"

static PyObject* tree_plan(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  (void)self;
  arg_t a[MAX_ARGS];
  if (parse("tree_plan", "ppppiqiipipp", args, n, a)) return NULL;
  const int rc = nslg_tree_plan(
      a[0].p, a[1].p, a[2].p, a[3].p, a[4].i, a[5].q, a[6].i, a[7].i, a[8].p, a[9].i, a[10].p, a[11].p);
  return PyLong_FromLong(rc);
}

static PyObject* paged_tree_attention(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  (void)self;
  arg_t a[MAX_ARGS];
  if (parse("paged_tree_attention", "pqpippiqipqpqppqipppqiiiifipqpzp", args, n, a)) return NULL;
  const int rc = nslg_paged_tree_attention(
      a[0].p, a[1].q, a[2].p, a[3].i, a[4].p, a[5].p, a[6].i, a[7].q, a[8].i, a[9].p, a[10].q, a[11].p, a[12].q,
      a[13].p, a[14].p, a[15].q, a[16].i, a[17].p, a[18].p, a[19].p, a[20].q, a[21].i, a[22].i, a[23].i, a[24].i,
      a[25].f, a[26].i, a[27].p, a[28].q, a[29].p, a[30].z, a[31].p);
  return PyLong_FromLong(rc);
}

static PyObject* verify_tree(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  (void)self;
  arg_t a[MAX_ARGS];
  if (parse("verify_tree", "ppppqiipqpqqiippppppzp", args, n, a)) return NULL;
  const int rc = nslg_verify_tree(
      a[0].p, a[1].p, a[2].p, a[3].p, a[4].q, a[5].i, a[6].i, a[7].p, a[8].q, a[9].p, a[10].q, a[11].q, a[12].i,
      a[13].i, a[14].p, a[15].p, a[16].p, a[17].p, a[18].p, a[19].p, a[20].z, a[21].p);
  return PyLong_FromLong(rc);
}

static PyObject* move_accepted(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  (void)self;
  arg_t a[MAX_ARGS];
  if (parse("move_accepted", "ppiqiiiipipppppip", args, n, a)) return NULL;
  const int rc = nslg_move_accepted(
      a[0].p, a[1].p, a[2].i, a[3].q, a[4].i, a[5].i, a[6].i, a[7].i, a[8].p, a[9].i, a[10].p, a[11].p, a[12].p,
      a[13].p, a[14].p, a[15].i, a[16].p);
  return PyLong_FromLong(rc);
}

static PyMethodDef methods[] = {
    {"tree_plan", (PyCFunction)(void (*)(void))tree_plan, METH_FASTCALL,
     "nslg_tree_plan: the entry point's arguments in order; returns its status"},
    {"paged_tree_attention", (PyCFunction)(void (*)(void))paged_tree_attention, METH_FASTCALL,
     "nslg_paged_tree_attention: the entry point's arguments in order; returns its status"},
    {"verify_tree", (PyCFunction)(void (*)(void))verify_tree, METH_FASTCALL,
     "nslg_verify_tree: the entry point's arguments in order; returns its status"},
    {"move_accepted", (PyCFunction)(void (*)(void))move_accepted, METH_FASTCALL,
     "nslg_move_accepted: the entry point's arguments in order; returns its status"},
    {NULL, NULL, 0, NULL}};

static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_nslg_fast_tree",
                                    "Fast-call binding of libnslg_kv's entry points for trees of drafted tokens", -1, methods,
                                    NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__nslg_fast_tree(void) { return PyModule_Create(&module); }
