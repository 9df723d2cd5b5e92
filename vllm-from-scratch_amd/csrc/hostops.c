// Host-side work of calls that are short on the device, as a CPython extension module
// (mvsd._hostops):
//   penalty_entries  what the penalties need to know of each request's history, gathered without
//                    converting every list to an array first.  32 requests of 650 tokens: 4.0 ms with
//                    numpy (np.unique per request), 0.17 here.
//   tensor_table, state_table  the checks of a call's tensors and their addresses, by the tensors'
//                    public attributes.  Host time of a beam step (16 tensors and a structure of 33
//                    words): 29.2 us in Python alone, 19.7 so; of reordering 16 tensors 30.8 and 12.5.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <stdint.h>
#include <stdlib.h>
#include <string.h>

static uint64_t mix(uint64_t x) {
  x ^= x >> 31;
  x *= 0x9e3779b97f4a7c15ull;
  return x ^ (x >> 29);
}

// The place of token t among this request's entries [0, *n), added when it is new: an
// open-addressing table of mask + 1 slots (a power of two) that hold a place + 1, or 0.
static int32_t place_of(int32_t* slots, size_t mask, int64_t* keys, int32_t* n, int64_t t) {
  size_t i = (size_t)mix((uint64_t)t) & mask;
  while (slots[i]) {
    const int32_t at = slots[i] - 1;
    if (keys[at] == t) return at;
    i = (i + 1) & mask;
  }
  keys[*n] = t;
  slots[i] = *n + 1;
  return (*n)++;
}

// Adds the first `len` tokens of a fast sequence to the request's entries: of its prompt (kind 0),
// output (1) or drafts (2).  0 where a token is no integer (the exception is set).
static int add_tokens(PyObject* seq, Py_ssize_t len, int kind, int32_t* slots, size_t mask,
                      int64_t* keys, int32_t* info, int32_t* n) {
  // a list can change while __index__ of an element runs: look at it afresh each time
  for (Py_ssize_t i = 0; i < len && i < PySequence_Fast_GET_SIZE(seq); ++i) {
    PyObject* item = PySequence_Fast_GET_ITEM(seq, i);
    int64_t t;
    if (PyLong_CheckExact(item)) {
      t = PyLong_AsLongLong(item);
    } else {
      Py_INCREF(item);
      PyObject* whole = PyNumber_Index(item);
      t = whole ? PyLong_AsLongLong(whole) : -1;
      Py_XDECREF(whole);
      Py_DECREF(item);
    }
    if (t == -1 && PyErr_Occurred()) return 0;
    const int32_t before = *n;
    const int32_t at = place_of(slots, mask, keys, n, t);
    if (at == before) info[at] = 0;
    if (kind == 0) info[at] |= (int32_t)0x80000000u;
    if (kind == 1) ++info[at];
  }
  return 1;
}

// penalty_entries(prompts, outputs, specs, buffer) -> number of entries E
//
// prompts, outputs: sequences of token sequences (missing tail requests count as empty); specs: one
// token sequence per request.  For request r the distinct tokens of its prompt, output and drafts
// are entries [off[r], off[r + 1]); buffer (writable int32) receives off [B + 1], then the tokens
// [E], then, per entry, the token's count in the output | (in the prompt) << 31.  The buffer has
// room for B + 1 + 2 * (all tokens).  TypeError where a token is no integer.
static PyObject* penalty_entries(PyObject* self, PyObject* args) {
  PyObject* lists[3];
  Py_buffer buf;
  if (!PyArg_ParseTuple(args, "OOOw*", &lists[0], &lists[1], &lists[2], &buf)) return NULL;
  PyObject* outer[3] = {NULL, NULL, NULL};
  PyObject* result = NULL;
  int64_t* keys = NULL;
  int32_t* info = NULL;
  int32_t* slots = NULL;
  size_t slots_room = 0, keys_cap = 0;
  for (int s = 0; s < 3; ++s) {
    outer[s] = PySequence_Fast(lists[s], "a sequence of token sequences is expected");
    if (!outer[s]) goto out;
  }
  {
    const Py_ssize_t B = PySequence_Fast_GET_SIZE(outer[2]);
    const int64_t room = (int64_t)(buf.len / 4);
    int32_t* off = (int32_t*)buf.buf;
    int32_t* tok = off + B + 1;  // tokens, then (moved behind them at the end) the infos
    int64_t total = 0;           // entries so far
    if (room < B + 1) {
      PyErr_SetString(PyExc_ValueError, "buffer too small");
      goto out;
    }
    // infos are collected here, since their place follows the last token
    size_t info_cap = (size_t)((room - B - 1) / 2);
    info = (int32_t*)malloc((info_cap ? info_cap : 1) * sizeof(int32_t));
    if (!info) {
      PyErr_NoMemory();
      goto out;
    }
    off[0] = 0;
    for (Py_ssize_t r = 0; r < B; ++r) {
      PyObject* inner[3] = {NULL, NULL, NULL};
      Py_ssize_t len[3] = {0, 0, 0};
      size_t all = 0;
      int ok = 1;
      for (int s = 0; s < 3 && ok; ++s) {
        if (r >= PySequence_Fast_GET_SIZE(outer[s])) continue;
        inner[s] = PySequence_Fast(PySequence_Fast_GET_ITEM(outer[s], r),
                                   "a token sequence is expected");
        if (!inner[s]) ok = 0;
        else all += (size_t)(len[s] = PySequence_Fast_GET_SIZE(inner[s]));
      }
      if (ok && (total + (int64_t)all) > (int64_t)info_cap) {
        PyErr_SetString(PyExc_ValueError, "buffer too small");
        ok = 0;
      }
      // The table has this request's own size, so that a short history after a long one clears a
      // small one; at most a quarter full (half full: 0.20 ms instead of 0.17 for 32 requests).
      size_t cap = 16;
      while (cap < 4 * all) cap *= 2;
      if (ok && cap > slots_room) {
        free(slots);
        slots = (int32_t*)malloc(cap * sizeof(int32_t));
        slots_room = slots ? cap : 0;
      }
      if (ok && all > keys_cap) {
        free(keys);
        keys_cap = all;
        keys = (int64_t*)malloc(keys_cap * sizeof(int64_t));
      }
      if (ok && (!slots || (all && !keys))) {
        PyErr_NoMemory();
        ok = 0;
      }
      if (ok) {
        memset(slots, 0, cap * sizeof(int32_t));
        int32_t n = 0;
        for (int s = 0; s < 3 && ok; ++s)
          ok = !inner[s] || add_tokens(inner[s], len[s], s, slots, cap - 1, keys, info + total, &n);
        for (int32_t e = 0; ok && e < n; ++e) tok[total + e] = (int32_t)keys[e];
        total += ok ? n : 0;
        off[r + 1] = (int32_t)total;
      }
      for (int s = 0; s < 3; ++s) Py_XDECREF(inner[s]);
      if (!ok) goto out;
    }
    memcpy(tok + total, info, (size_t)total * sizeof(int32_t));
    result = PyLong_FromLongLong(total);
  }
out:
  for (int s = 0; s < 3; ++s) Py_XDECREF(outer[s]);
  free(slots);
  free(keys);
  free(info);
  PyBuffer_Release(&buf);
  return result;
}

// ------------------------------------------------------------------ tensors ----------

static PyObject *s_dtype, *s_shape, *s_device, *s_is_contiguous, *s_data_ptr, *s_stride,
    *s_element_size;

// A method without arguments that gives an integer.  -1 and an exception where it does not.
static int64_t call_int(PyObject* o, PyObject* name) {
  PyObject* v = PyObject_CallMethodNoArgs(o, name);
  if (!v) return -1;
  const int64_t n = PyLong_AsLongLong(v);
  Py_DECREF(v);
  return n;
}

// Whether o.name equals `want`; -1 and an exception where that cannot be said.
static int attr_equals(PyObject* o, PyObject* name, PyObject* want) {
  PyObject* v = PyObject_GetAttr(o, name);
  if (!v) return -1;
  const int same = v == want ? 1 : PyObject_RichCompareBool(v, want, Py_EQ);
  Py_DECREF(v);
  return same;
}

// tensor_table(buffer, at, tensors, dtypes, shapes, device) -> -1, or the first that fails
//
// Tensor k has dtype dtypes[k], shape shapes[k], the device, and is contiguous: its address becomes
// element at + k of the buffer (writable int64).  The caller finds out what is wrong with one that
// fails.
static PyObject* tensor_table(PyObject* self, PyObject* args) {
  Py_buffer buf;
  Py_ssize_t at;
  PyObject *tensors, *dtypes, *shapes, *device;
  if (!PyArg_ParseTuple(args, "w*nO!O!O!O", &buf, &at, &PyTuple_Type, &tensors, &PyTuple_Type,
                        &dtypes, &PyTuple_Type, &shapes, &device))
    return NULL;
  const Py_ssize_t n = PyTuple_GET_SIZE(tensors);
  Py_ssize_t k = 0;
  if (PyTuple_GET_SIZE(dtypes) != n || PyTuple_GET_SIZE(shapes) != n || at < 0 ||
      at + n > buf.len / (Py_ssize_t)sizeof(int64_t)) {
    PyBuffer_Release(&buf);
    PyErr_SetString(PyExc_ValueError, "tensor_table: sizes do not agree");
    return NULL;
  }
  for (; k < n; ++k) {
    PyObject* t = PyTuple_GET_ITEM(tensors, k);
    // a step in place has its state's tensors twice: checked once (4.4 us for 16 tensors, 2.8 so)
    Py_ssize_t same = 0;
    while (same < k && (PyTuple_GET_ITEM(tensors, same) != t ||
                        PyTuple_GET_ITEM(dtypes, same) != PyTuple_GET_ITEM(dtypes, k) ||
                        PyTuple_GET_ITEM(shapes, same) != PyTuple_GET_ITEM(shapes, k)))
      ++same;
    if (same < k) {
      ((int64_t*)buf.buf)[at + k] = ((int64_t*)buf.buf)[at + same];
      continue;
    }
    if (attr_equals(t, s_dtype, PyTuple_GET_ITEM(dtypes, k)) != 1) break;
    if (attr_equals(t, s_shape, PyTuple_GET_ITEM(shapes, k)) != 1) break;
    if (attr_equals(t, s_device, device) != 1) break;
    PyObject* c = PyObject_CallMethodNoArgs(t, s_is_contiguous);
    Py_XDECREF(c);  // Py_True and Py_False outlive it
    if (c != Py_True) break;
    const int64_t p = call_int(t, s_data_ptr);
    if (p == -1) break;
    ((int64_t*)buf.buf)[at + k] = p;
  }
  PyErr_Clear();
  PyBuffer_Release(&buf);
  return PyLong_FromSsize_t(k < n ? k : -1);
}

typedef struct {
  int64_t address, stride, rows, outer, length, inner;
} StateRows;

// A state tensor [rows, ..., length, ...], contiguous within a row, on the device: 1, or 0 where it
// is none (an exception may be set).
static int state_rows(PyObject* t, Py_ssize_t dim, PyObject* device, StateRows* s) {
  if (attr_equals(t, s_device, device) != 1) return 0;
  PyObject* shape = PyObject_GetAttr(t, s_shape);
  PyObject* stride = shape ? PyObject_CallMethodNoArgs(t, s_stride) : NULL;
  int ok = 0;
  if (shape && stride && PyTuple_Check(shape) && PyTuple_Check(stride) &&
      PyTuple_GET_SIZE(shape) == PyTuple_GET_SIZE(stride) && dim >= 1 &&
      dim < PyTuple_GET_SIZE(shape)) {
    const Py_ssize_t nd = PyTuple_GET_SIZE(shape);
    int64_t expect = 1, outer = 1, inner = 1, length = 0;
    ok = 1;
    for (Py_ssize_t d = nd - 1; d > 0 && ok; --d) {
      const int64_t n = PyLong_AsLongLong(PyTuple_GET_ITEM(shape, d));
      const int64_t st = PyLong_AsLongLong(PyTuple_GET_ITEM(stride, d));
      if (n < 0 || (st != expect && n > 1 && expect != 0)) ok = 0;
      expect *= n;
      if (d == dim) length = n;
      else if (d > dim) inner *= n;
      else outer *= n;
    }
    const int64_t size = ok ? call_int(t, s_element_size) : -1;
    s->rows = PyLong_AsLongLong(PyTuple_GET_ITEM(shape, 0));
    s->stride = PyLong_AsLongLong(PyTuple_GET_ITEM(stride, 0)) * size;
    s->outer = outer;
    s->length = length;
    s->inner = inner * size;
    if (size < 1 || s->rows < 0 || (s->rows > 1 && s->stride < expect * size)) ok = 0;
    s->address = ok ? call_int(t, s_data_ptr) : -1;
    if (s->address == -1) ok = 0;
  }
  Py_XDECREF(shape);
  Py_XDECREF(stride);
  return ok && !PyErr_Occurred();
}

// state_table(buffer, states, outs, length_dim, device, least_rows) -> entries written, or -1
//
// states and outs (the same tuple: in place): tensors as state_rows takes them, outs[k] of the shape
// and dtype of states[k], with at least least_rows rows.  Eight int64 an entry (mvsd_beam_state);
// empty tensors have none.  -1 where a tensor is something else.
static PyObject* state_table(PyObject* self, PyObject* args) {
  Py_buffer buf;
  PyObject *states, *outs, *device;
  Py_ssize_t dim;
  long long least;
  if (!PyArg_ParseTuple(args, "w*O!O!nOL", &buf, &PyTuple_Type, &states, &PyTuple_Type, &outs,
                        &dim, &device, &least))
    return NULL;
  const Py_ssize_t n = PyTuple_GET_SIZE(states);
  int64_t* out = (int64_t*)buf.buf;
  Py_ssize_t m = 0;
  int ok = PyTuple_GET_SIZE(outs) == n && buf.len >= n * 8 * (Py_ssize_t)sizeof(int64_t);
  for (Py_ssize_t k = 0; k < n && ok; ++k) {
    PyObject *x = PyTuple_GET_ITEM(states, k), *to = PyTuple_GET_ITEM(outs, k);
    StateRows a, b;
    ok = state_rows(x, dim, device, &a) && a.rows >= least;
    b = a;
    if (ok && to != x) {
      PyObject* dtype = PyObject_GetAttr(x, s_dtype);
      PyObject* shape = PyObject_GetAttr(x, s_shape);
      ok = dtype && shape && attr_equals(to, s_dtype, dtype) == 1 &&
           attr_equals(to, s_shape, shape) == 1 && state_rows(to, dim, device, &b);
      Py_XDECREF(dtype);
      Py_XDECREF(shape);
    }
    if (!ok || a.rows == 0 || a.outer == 0 || a.length == 0 || a.inner == 0) continue;
    const int64_t row[8] = {a.address, b.address, a.stride, b.stride,
                            a.rows,    a.outer,   a.length, a.inner};
    memcpy(out + 8 * m++, row, sizeof(row));
  }
  PyErr_Clear();
  PyBuffer_Release(&buf);
  return PyLong_FromSsize_t(ok ? m : -1);
}

static PyMethodDef methods[] = {
    {"tensor_table", tensor_table, METH_VARARGS,
     "tensor_table(buffer, at, tensors, dtypes, shapes, device) -> -1 or the first that fails"},
    {"state_table", state_table, METH_VARARGS,
     "state_table(buffer, states, outs, length_dim, device, least_rows) -> entries or -1"},
    {"penalty_entries", penalty_entries, METH_VARARGS,
     "penalty_entries(prompts, outputs, specs, buffer) -> number of entries"},
    {NULL, NULL, 0, NULL}};

static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_hostops", NULL, -1, methods,
                                    NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__hostops(void) {
  if (!(s_dtype = PyUnicode_InternFromString("dtype")) ||
      !(s_shape = PyUnicode_InternFromString("shape")) ||
      !(s_device = PyUnicode_InternFromString("device")) ||
      !(s_is_contiguous = PyUnicode_InternFromString("is_contiguous")) ||
      !(s_data_ptr = PyUnicode_InternFromString("data_ptr")) ||
      !(s_stride = PyUnicode_InternFromString("stride")) ||
      !(s_element_size = PyUnicode_InternFromString("element_size")))
    return NULL;
  return PyModule_Create(&module);
}
