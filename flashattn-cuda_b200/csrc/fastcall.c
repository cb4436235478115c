/* fastcall.c -- a CPython binding of the entry points of libb200attn.so whose
 * calls are short: prefill and the quantised paged KV cache.
 *
 * b200attn calls the C-ABI through ctypes; converting fifteen to twenty-five
 * arguments costs a few microseconds per call, which is as much as the kernel
 * launch itself and dominates small calls.  This module converts the same
 * arguments itself and calls the same exported functions, so both routes run
 * identical library code.
 */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <stdint.h>

#include "../../include/b200attn.h"

/* prefill_fwd_kv(q, k, v, o, lse, B, H, Hkv, N, Nk, D, dtype, causal, scale, stream) -> status
 * pointers and the stream are integers (lse may be 0 for the O-only path). */
static PyObject* prefill_fwd_kv(PyObject* self, PyObject* args) {
  unsigned long long q, k, v, o, lse, stream;
  int B, H, Hkv, N, Nk, D, dtype, causal;
  float scale;
  (void)self;
  if (!PyArg_ParseTuple(args, "KKKKKiiiiiiiifK", &q, &k, &v, &o, &lse, &B, &H, &Hkv, &N, &Nk, &D,
                        &dtype, &causal, &scale, &stream))
    return NULL;
  const int rc = b2a_prefill_fwd_kv((const void*)(uintptr_t)q, (const void*)(uintptr_t)k,
                                    (const void*)(uintptr_t)v, (void*)(uintptr_t)o,
                                    (float*)(uintptr_t)lse, B, H, Hkv, N, Nk, D, dtype, causal,
                                    scale, (void*)(uintptr_t)stream);
  return PyLong_FromLong(rc);
}

/* The quantised cache's entry points take n integers and, decode, one float last.
 * `wide` has a bit for each of 64 bits: pointers (0 for a null one), the stream and
 * strides.  The others are ints: a value that does not fit one is refused. */
static int parse_ints(PyObject* const* args, Py_ssize_t nargs, Py_ssize_t n, unsigned wide,
                      long long* v) {
  if (nargs < n) {
    PyErr_Format(PyExc_TypeError, "expected at least %zd arguments, got %zd", n, nargs);
    return -1;
  }
  for (Py_ssize_t i = 0; i < n; ++i) {
    if (args[i] == Py_None) {
      v[i] = 0;
      continue;
    }
    v[i] = PyLong_AsLongLong(args[i]);
    if (v[i] == -1 && PyErr_Occurred()) return -1;
    if (!(wide >> i & 1u) && v[i] != (int)v[i]) {
      PyErr_Format(PyExc_RuntimeError, "%lld does not fit in 32 bits", v[i]);
      return -1;
    }
  }
  return 0;
}
#define PTR(i) ((void*)(uintptr_t)v[i])
#define INT(i) ((int)v[i])
#define BITS(from, to) ((1u << (to)) - (1u << (from))) /* from .. to - 1 */

/* kvq_append(k, v, data, index, index_scale, table, lens, B, Hkv, T, D, page, max_pages,
 * num_pages, bits, dtype, advance, stream, k strides x 3, v strides x 3) -> status */
static PyObject* kvq_append(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  long long v[24];
  (void)self;
  if (parse_ints(args, nargs, 24, BITS(0, 7) | BITS(17, 24), v) != 0) return NULL;
  const int64_t ks[3] = {v[18], v[19], v[20]}, vs[3] = {v[21], v[22], v[23]};
  return PyLong_FromLong(b2a_kvq_append_paged(
      PTR(0), PTR(1), ks, vs, PTR(2), (int8_t*)PTR(3), (float*)PTR(4), (const int32_t*)PTR(5),
      (int32_t*)PTR(6), INT(7), INT(8), INT(9), INT(10), INT(11), INT(12), INT(13), INT(14),
      INT(15), INT(16), PTR(17)));
}

/* kvq_read(data, table, start, cu, k_out, v_out, B, Hkv, D, page, max_pages, num_pages, total,
 * max_len, bits, dtype, stream) -> status */
static PyObject* kvq_read(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  long long v[17];
  (void)self;
  if (parse_ints(args, nargs, 17, BITS(0, 6) | BITS(16, 17), v) != 0) return NULL;
  return PyLong_FromLong(b2a_kvq_read_paged(
      PTR(0), (const int32_t*)PTR(1), (const int32_t*)PTR(2), (const int32_t*)PTR(3), PTR(4),
      PTR(5), INT(6), INT(7), INT(8), INT(9), INT(10), INT(11), INT(12), INT(13), INT(14),
      INT(15), PTR(16)));
}

/* kvq_select(q, index, index_scale, table, lens, keys, pages, B, H, Hkv, D, page, max_pages,
 * num_pages, top_k, dtype, stream, q strides x 2) -> status */
static PyObject* kvq_select(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  long long v[19];
  (void)self;
  if (parse_ints(args, nargs, 19, BITS(0, 7) | BITS(16, 19), v) != 0) return NULL;
  const int64_t qs[2] = {v[17], v[18]};
  return PyLong_FromLong(b2a_kvq_select_pages(
      PTR(0), qs, (const int8_t*)PTR(1), (const float*)PTR(2), (const int32_t*)PTR(3),
      (const int32_t*)PTR(4), (uint32_t*)PTR(5), (int32_t*)PTR(6), INT(7), INT(8), INT(9),
      INT(10), INT(11), INT(12), INT(13), INT(14), INT(15), PTR(16)));
}

/* kvq_decode(q, data, table, lens, pages, n_pages, workspace, o, lse, B, H, Hkv, D, page,
 * max_pages, num_pages, workers, bits, dtype, stream, q strides x 2, scale) -> status */
static PyObject* kvq_decode(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  long long v[22];
  (void)self;
  if (nargs != 23) {
    PyErr_Format(PyExc_TypeError, "expected 23 arguments, got %zd", nargs);
    return NULL;
  }
  if (parse_ints(args, nargs, 22, BITS(0, 5) | BITS(6, 9) | BITS(19, 22), v) != 0) return NULL;
  const double scale = PyFloat_AsDouble(args[22]);
  if (scale == -1.0 && PyErr_Occurred()) return NULL;
  const int64_t qs[2] = {v[20], v[21]};
  return PyLong_FromLong(b2a_kvq_decode_paged(
      PTR(0), qs, PTR(1), (const int32_t*)PTR(2), (const int32_t*)PTR(3), (const int32_t*)PTR(4),
      INT(5), (float*)PTR(6), PTR(7), (float*)PTR(8), INT(9), INT(10), INT(11), INT(12), INT(13),
      INT(14), INT(15), INT(16), INT(17), INT(18), (float)scale, PTR(19)));
}

static PyMethodDef kMethods[] = {
    {"prefill_fwd_kv", prefill_fwd_kv, METH_VARARGS,
     "b2a_prefill_fwd_kv(q, k, v, o, lse, B, H, Hkv, N, Nk, D, dtype, causal, scale, stream)"},
    {"kvq_append", (PyCFunction)(void (*)(void))kvq_append, METH_FASTCALL, "b2a_kvq_append_paged"},
    {"kvq_read", (PyCFunction)(void (*)(void))kvq_read, METH_FASTCALL, "b2a_kvq_read_paged"},
    {"kvq_select", (PyCFunction)(void (*)(void))kvq_select, METH_FASTCALL, "b2a_kvq_select_pages"},
    {"kvq_decode", (PyCFunction)(void (*)(void))kvq_decode, METH_FASTCALL, "b2a_kvq_decode_paged"},
    {NULL, NULL, 0, NULL}};

static struct PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_fastcall",
                                     "CPython binding of libb200attn.so's short calls", -1, kMethods};

PyMODINIT_FUNC PyInit__fastcall(void) { return PyModule_Create(&kModule); }
