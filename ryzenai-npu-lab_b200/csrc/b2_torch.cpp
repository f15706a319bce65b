// Native binding of the entry points whose smallest calls are bound by the
// host (module _b2torch): the checks of a call's tensors and the library call in
// one go (a decode step 8 us per call, through Python and ctypes 16).  Each
// function takes the arguments of its Python wrapper in a fixed order and returns
// the library's status, or None when an argument is not what the wrapper accepts:
// the wrapper then repeats its checks in Python, which word the refusal (or
// accept what this path does not know, a tensor subclass for instance).
//
// The library's functions come by address (bind), so this module links neither
// against it nor against CUDA; their types come from the headers.  The module is
// of use to the torch and the Python it was compiled against alone, whose names
// it carries (stamp): build.py and attention_kv8.py look for them before it is
// loaded.

#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <torch/csrc/autograd/python_variable.h>

#include <initializer_list>

#include "b2_kv8.h"
#include "b2_tables.h"

namespace {

constexpr char kStamp[] = B2_TORCH_STAMP;

constexpr int64_t kHq = 16, kHkv = 8, kDim = 64, kBlock = 64, kWidth = 2048;
constexpr int kNorm = 1, kRope = 2, kStore = 4;

using StepFn = decltype(&b2_kv8_decode_step);
using AppendFn = decltype(&b2_kv8_append);
using PrefillFn = decltype(&b2_kv8_prefill_attn);
using ExtendFn = decltype(&b2_tables_extend);
StepFn g_step = nullptr;
AppendFn g_append = nullptr;
PrefillFn g_prefill = nullptr;
ExtendFn g_extend = nullptr;

// A tensor's address, for a parameter of any pointer type.
struct Address {
  void *p = nullptr;
  template <class T>
  operator T *() const {
    return static_cast<T *>(p);
  }
};

// The checks of one call: `ok` stays true while every argument is as expected.
struct Args {
  PyObject *const *at;
  int64_t index = -1;  // device of the call's tensors
  bool ok = true;

  explicit Args(PyObject *const *args) : at(args) {}

  const at::Tensor *tensor(PyObject *o) {
    if (!THPVariable_CheckExact(o)) {
      ok = false;
      return nullptr;
    }
    return &THPVariable_Unpack(o);
  }
  // contiguous tensor i of this type on the call's device
  const at::Tensor *plain(int i, at::ScalarType type) {
    const at::Tensor *t = tensor(at[i]);
    if (t && (t->scalar_type() != type || !t->is_cuda() || t->get_device() != index || !t->is_contiguous())) ok = false;
    return ok ? t : nullptr;
  }
  Address ptr(int i, at::ScalarType type, std::initializer_list<int64_t> sizes) {
    const at::Tensor *t = plain(i, type);
    if (!t || !t->sizes().equals(at::IntArrayRef(sizes.begin(), sizes.size()))) {
      ok = false;
      return {};
    }
    return {t->data_ptr()};
  }
  Address ptr_or_null(int i, at::ScalarType type, std::initializer_list<int64_t> sizes) {
    return at[i] == Py_None ? Address{} : ptr(i, type, sizes);
  }
  int64_t whole(int i) {
    const int64_t v = PyLong_Check(at[i]) ? PyLong_AsLongLong(at[i]) : -1;
    if (v == -1 || PyErr_Occurred()) {
      PyErr_Clear();
      ok = false;
    }
    return v;
  }
  float number(int i) {
    const double v = PyFloat_Check(at[i]) ? PyFloat_AS_DOUBLE(at[i]) : (ok = false, 0.0);
    return static_cast<float>(v);
  }
};

constexpr auto kI32 = at::kInt;
constexpr auto kBf16 = at::kBFloat16;
constexpr auto kF32 = at::kFloat;
constexpr auto kE4m3 = at::kFloat8_e4m3fn;

struct Cache {
  Address k, v, ks, vs;
  int64_t blocks;
};

Cache cache_args(Args &a, int i) {
  Cache c{};
  const at::Tensor *k = a.plain(i, kE4m3);
  if (!k || k->dim() != 4) {
    a.ok = false;
    return c;
  }
  c.blocks = k->size(0);
  c.k = a.ptr(i, kE4m3, {c.blocks, kHkv, kBlock, kDim});
  c.v = a.ptr(i + 1, kE4m3, {c.blocks, kHkv, kDim, kBlock});
  c.ks = a.ptr(i + 2, kF32, {c.blocks, kHkv});
  c.vs = a.ptr(i + 3, kF32, {c.blocks, kHkv});
  return c;
}

struct QkArgs {
  Address gq, gk, cos, sin;
  int64_t rows = 0;
};

QkArgs qk_args(Args &a, int i, int64_t mode) {
  QkArgs q;
  if (mode & kNorm) {
    q.gq = a.ptr(i, kBf16, {kDim});
    q.gk = a.ptr(i + 1, kBf16, {kDim});
  }
  if (mode & kRope) {
    const at::Tensor *c = a.plain(i + 2, kBf16);
    if (c && c->dim() == 2 && c->size(0) > 0) {
      q.rows = c->size(0);
      q.cos = a.ptr(i + 2, kBf16, {q.rows, kDim});
      q.sin = a.ptr(i + 3, kBf16, {q.rows, kDim});
    } else {
      a.ok = false;
    }
  }
  return q;
}

bool small(std::initializer_list<int64_t> values) {
  for (const int64_t v : values)
    if (v > 0x7fffffff) return false;
  return true;
}

PyObject *not_here() { Py_RETURN_NONE; }

// qkv, past_lens, k, v, k_scale, v_scale, block_tables, out, workspace, dev_err, chunk_lens, gamma_q, gamma_k, cos,
// sin, mode, eps, scale, stream, row_start, max_tokens
PyObject *step(PyObject *, PyObject *const *args, Py_ssize_t n) {
  if (n != 21 || !g_step) return not_here();
  Args a(args);
  const at::Tensor *qkv = a.tensor(args[0]);
  if (!qkv || (qkv->dim() != 2 && qkv->dim() != 3) || !qkv->is_cuda()) return not_here();
  a.index = qkv->get_device();
  const bool padded = qkv->dim() == 3;
  const at::Tensor *tables = a.plain(6, kI32);
  if (!tables || tables->dim() != 2 || !a.plain(0, kBf16) || (args[19] == Py_None) != padded ||
      (args[20] == Py_None) != padded)
    return not_here();
  const int64_t b = tables->size(0), cols = tables->size(1), mode = a.whole(15);
  const int64_t t = padded ? qkv->size(1) : a.whole(20), width = qkv->size(-1);
  const int64_t rows = padded ? b * t : qkv->size(0);
  if (t < 1 || t > 4 || width < kWidth || (padded && qkv->size(0) != b)) return not_here();
  const Address q{qkv->data_ptr()}, past = a.ptr(1, kI32, {b}), table = a.ptr(6, kI32, {b, cols});
  const Address start = a.ptr_or_null(19, kI32, {b});
  const Cache c = cache_args(a, 2);
  const Address out = padded ? a.ptr(7, kBf16, {b, t, kHq, kDim}) : a.ptr(7, kBf16, {rows, kHq, kDim});
  const at::Tensor *work = a.plain(8, at::kByte);
  const Address err = a.ptr(9, kI32, {1}), chunk = a.ptr_or_null(10, kI32, {b});
  const QkArgs qk = qk_args(a, 11, mode);
  const float eps = a.number(16), scale = a.number(17);
  const int64_t stream = PyLong_AsLongLong(args[18]);
  if (!a.ok || !small({b, rows, width, cols, c.blocks, qk.rows})) return not_here();
  return PyLong_FromLong(g_step(q, width, static_cast<int32_t>(rows), start, static_cast<int32_t>(t), chunk, qk.gq,
                                qk.gk, eps, qk.cos, qk.sin, static_cast<int32_t>(qk.rows), past, table,
                                static_cast<int32_t>(cols), c.k, c.v, c.ks, c.vs, static_cast<int32_t>(c.blocks),
                                static_cast<int32_t>(b), scale, static_cast<int32_t>(mode), out, work->data_ptr(),
                                work->numel(), err, reinterpret_cast<void *>(stream)));
}

// qkv, past_lens, k, v, k_scale, v_scale, block_tables, out, workspace, dev_err, chunk_lens, gamma_q, gamma_k, cos,
// sin, mode, eps, scale, stream, row_start, max_tokens, slots, positions, q buffer
PyObject *prefill(PyObject *, PyObject *const *args, Py_ssize_t n) {
  if (n != 24 || !g_prefill || !g_append) return not_here();
  Args a(args);
  const at::Tensor *qkv = a.tensor(args[0]);
  if (!qkv || (qkv->dim() != 2 && qkv->dim() != 3) || !qkv->is_cuda()) return not_here();
  a.index = qkv->get_device();
  const bool padded = qkv->dim() == 3;
  const int64_t width = qkv->size(-1);
  const at::Tensor *tables = a.plain(6, kI32);
  if (width < kWidth || !tables || tables->dim() != 2 || !a.plain(0, kBf16)) return not_here();
  const int64_t rows = qkv->numel() / width, b = tables->size(0), cols = tables->size(1), mode = a.whole(15);
  const Address past = a.ptr(1, kI32, {b}), table = a.ptr(6, kI32, {b, cols});
  const Cache c = cache_args(a, 2);
  int64_t tokens;
  Address out, start;
  if (padded) {
    tokens = qkv->size(1);
    if (qkv->size(0) != b || args[19] != Py_None) return not_here();
    out = a.ptr(7, kBf16, {b, tokens, kHq, kDim});
  } else {
    tokens = a.whole(20);
    start = a.ptr(19, kI32, {b});
    out = a.ptr(7, kBf16, {rows, kHq, kDim});
    if (args[21] == Py_None) return not_here();
  }
  const at::Tensor *work = a.plain(8, at::kByte);
  const Address err = a.ptr(9, kI32, {1}), chunk = a.ptr_or_null(10, kI32, {b});
  const QkArgs qk = qk_args(a, 11, mode);
  const float eps = a.number(16), scale = a.number(17);
  const int64_t stream = PyLong_AsLongLong(args[18]);
  const Address slots = a.ptr_or_null(21, kI32, {rows}), positions = a.ptr_or_null(22, kI32, {rows});
  const Address q_buf = a.ptr_or_null(23, kBf16, {rows, kHq, kDim});
  if (!a.ok || !small({b, width, cols, c.blocks, qk.rows, rows, tokens}) ||
      ((mode & (kNorm | kRope)) != 0) != (q_buf.p != nullptr))
    return not_here();
  void *st = reinterpret_cast<void *>(stream);
  const Address x{qkv->data_ptr()};
  if (mode) {
    const int rc = g_append(x, width, static_cast<int32_t>(rows), slots, positions, past, chunk,
                            static_cast<int32_t>(tokens), table, static_cast<int32_t>(cols), qk.gq, qk.gk, eps, qk.cos,
                            qk.sin, static_cast<int32_t>(qk.rows), c.k, c.v, c.ks, c.vs,
                            static_cast<int32_t>(c.blocks), q_buf, static_cast<int32_t>(mode), err, st);
    if (rc) return PyLong_FromLong(rc);
  }
  return PyLong_FromLong(g_prefill(q_buf.p ? q_buf : x, q_buf.p ? kHq * kDim : width, static_cast<int32_t>(rows), start,
                                   past, chunk, static_cast<int32_t>(tokens), table, static_cast<int32_t>(cols), c.k,
                                   c.v, c.ks, c.vs, static_cast<int32_t>(c.blocks), static_cast<int32_t>(b), scale, out,
                                   work->data_ptr(), work->numel(), err, st));
}

// block_tables, held, free_list, free_count, past_lens, new_lens, held_out, free_count_out, granted, row_start, slots,
// positions, tokens_per_seq, dev_err, stream
PyObject *extend(PyObject *, PyObject *const *args, Py_ssize_t n) {
  if (n != 15 || !g_extend) return not_here();
  Args a(args);
  const at::Tensor *tables = a.tensor(args[0]);
  if (!tables || tables->dim() != 2 || !tables->is_cuda()) return not_here();
  a.index = tables->get_device();
  const int64_t b = tables->size(0), cols = tables->size(1);
  const at::Tensor *list = a.plain(2, kI32), *slot_rows = a.plain(10, kI32);
  if (!list || !slot_rows) return not_here();
  const int64_t blocks = list->numel(), rows = slot_rows->numel(), tokens = a.whole(12);
  const Address table = a.ptr(0, kI32, {b, cols}), held = a.ptr(1, kI32, {b}), free_list = a.ptr(2, kI32, {blocks});
  const Address count = a.ptr(3, kI32, {1}), past = a.ptr(4, kI32, {b}), fresh = a.ptr(5, kI32, {b});
  const Address held_out = a.ptr_or_null(6, kI32, {b}), count_out = a.ptr_or_null(7, kI32, {1});
  const Address granted = a.ptr(8, kI32, {b}), start = a.ptr(9, kI32, {b}), slots = a.ptr(10, kI32, {rows});
  const Address positions = a.ptr(11, kI32, {rows}), err = a.ptr(13, kI32, {1});
  const int64_t stream = PyLong_AsLongLong(args[14]);
  if (!a.ok || !small({b, cols, blocks, rows, tokens})) return not_here();
  return PyLong_FromLong(g_extend(table, static_cast<int32_t>(cols), held, free_list, static_cast<int32_t>(blocks), count,
                                  past, fresh, static_cast<int32_t>(b), held_out.p ? held_out : held,
                                  count_out.p ? count_out : count, granted, start, slots, positions,
                                  static_cast<int32_t>(rows), static_cast<int32_t>(tokens), err,
                                  reinterpret_cast<void *>(stream)));
}

// bind(step, append, prefill, extend): the library functions' addresses
PyObject *bind(PyObject *, PyObject *const *args, Py_ssize_t n) {
  if (n != 4) {
    PyErr_SetString(PyExc_TypeError, "bind takes four addresses");
    return nullptr;
  }
  void *p[4];
  for (int i = 0; i < 4; ++i) {
    p[i] = PyLong_AsVoidPtr(args[i]);
    if (PyErr_Occurred()) return nullptr;
  }
  g_step = reinterpret_cast<StepFn>(p[0]);
  g_append = reinterpret_cast<AppendFn>(p[1]);
  g_prefill = reinterpret_cast<PrefillFn>(p[2]);
  g_extend = reinterpret_cast<ExtendFn>(p[3]);
  Py_RETURN_NONE;
}

template <PyObject *(*fn)(PyObject *, PyObject *const *, Py_ssize_t)>
PyObject *guarded(PyObject *self, PyObject *const *args, Py_ssize_t n) noexcept {
  try {
    return fn(self, args, n);
  } catch (...) {  // a tensor without storage, say: the Python path words it
    PyErr_Clear();
    return not_here();
  }
}

#define ENTRY(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(guarded<name>)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {ENTRY(bind), ENTRY(step), ENTRY(prefill), ENTRY(extend), {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_b2torch", "native binding of libb2attn.so's smallest calls", -1, g_methods,
                        nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__b2torch(void) {
  PyObject *m = PyModule_Create(&g_module);
  if (m && PyModule_AddStringConstant(m, "stamp", kStamp) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
