// CPython extension `tileccl_amd._host`, second part: the training operators' host side.
//
// An operator on a few rows takes as long as the host needs to issue it: checks, outputs, a descriptor and the launch are
// 12 to 16 us in Python beside the 2.5 us of the launch itself, and 4 to 6 us here.  Each function takes the
// operator's arguments in order, checks them, allocates the outputs and the workspace, and calls the C entry point.  It
// returns None if there is something about the arguments that it does not take; ops_training.py says what that is.
//
// mean and rstd, and the two sums of the backward pass, share an allocation each: they live as long as each other.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/hip/EmptyTensor.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <cstring>
#include <exception>

#include "../../include/tileccl_hip.h"
#include "tccl_host_ops.h"

namespace {

// What bind() is given: callables, types and the addresses of the entry points.
PyObject *current_stream, *report, *device0;
PyObject *norm_result, *norm_gradients, *checkpoint_type;
PyObject *f16, *bf16, *f32;  // torch.float16, torch.bfloat16, torch.float32
int (*entry_norm)(const tccl_norm_desc*, void*);
int (*entry_norm_grad)(const tccl_norm_grad_desc*, void*);
int64_t (*entry_norm_grad_workspace)(int32_t, int32_t, int32_t, int32_t);
int (*entry_hold)(const tccl_held_desc*, void*);
int (*entry_restore)(const tccl_held_desc*, void*);
int (*entry_weight)(const tccl_weight_gradient_desc*, void*);
int64_t (*entry_weight_workspace)(int32_t, int32_t, int32_t);

template <typename Body>
PyObject* guarded(Body body) {
  try {
    return body();
  } catch (const std::exception& e) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

PyObject* none() { Py_RETURN_NONE; }

int code_of(at::ScalarType t) {
  return t == at::kHalf ? TCCL_F16 : t == at::kBFloat16 ? TCCL_BF16 : t == at::kFloat ? TCCL_F32 : -1;
}

// A matrix with contiguous rows: where it lies and its pitch.
struct Matrix {
  const at::Tensor* t = nullptr;
  char* at = nullptr;
  int64_t rows = 0, cols = 0, pitch = 0;

  bool open(PyObject* o) {
    if (!THPVariable_Check(o)) return false;
    t = &THPVariable_Unpack(o);
    if (!t->is_cuda() || t->layout() != at::kStrided || t->dim() != 2) return false;
    rows = t->size(0), cols = t->size(1);
    if (cols < 1 || rows > TCCL_TRAINING_MAX_ROWS || cols > INT32_MAX || (cols > 1 && t->stride(1) != 1)) return false;
    pitch = rows > 1 ? t->stride(0) : cols;
    at = (char*)t->data_ptr();
    return pitch >= cols;
  }
  bool like(const Matrix& m) const { return rows == m.rows && cols == m.cols && t->scalar_type() == m.t->scalar_type() && t->device() == m.t->device(); }
  char* end() const { return rows ? at + ((rows - 1) * pitch + cols) * t->element_size() : at; }
  // No memory in common (rows between rows count as the matrix's).
  bool elsewhere(const Matrix& m) const { return !(at < m.end() && m.at < end()); }
  // No byte of the matrix's rows lies in a contiguous tensor.
  bool clear_of(const at::Tensor& o) const {
    if (!rows || !o.numel()) return true;
    const int64_t step = pitch * (int64_t)t->element_size(), width = cols * (int64_t)t->element_size();
    const int64_t from = (char*)o.data_ptr() - at, to = from + (int64_t)o.nbytes();  // seen from the first row
    const int64_t row = from < width ? 0 : (from - width) / step + 1;               // the first one that ends behind `from`
    return row >= rows || row * step >= to;
  }
  bool clear_of(const at::Tensor* o) const { return !o || clear_of(*o); }
  // The same elements in the same places, or none in common.
  bool apart(const Matrix& m) const { return !m.t || elsewhere(m) || (at == m.at && pitch == m.pitch && t->scalar_type() == m.t->scalar_type()); }
};

bool vector_of(PyObject* o, int64_t n, const at::Device& device, const at::Tensor*& t) {
  if (!THPVariable_Check(o)) return false;
  t = &THPVariable_Unpack(o);
  return t->is_cuda() && t->layout() == at::kStrided && t->dim() == 1 && t->size(0) == n && t->device() == device && (n <= 1 || t->stride(0) == 1);
}

struct Held {
  const at::Tensor *values = nullptr, *scales = nullptr;
  int64_t rows = 0, cols = 0;
  at::ScalarType type;
};

bool bytes_of(const at::Tensor& t, const at::Device& device) {
  return t.is_cuda() && t.layout() == at::kStrided && t.scalar_type() == at::kByte && t.device() == device && t.is_contiguous();
}

int64_t row_blocks(int64_t rows) { return (rows + TCCL_HELD_ROWS - 1) / TCCL_HELD_ROWS; }
int64_t col_blocks(int64_t cols) { return (cols + TCCL_HELD_COLS - 1) / TCCL_HELD_COLS; }

bool open_held(PyObject* o, Held& h) {
  if ((PyObject*)Py_TYPE(o) != checkpoint_type || PyTuple_GET_SIZE(o) != 5) return false;
  PyObject *v = PyTuple_GET_ITEM(o, 0), *s = PyTuple_GET_ITEM(o, 1), *d = PyTuple_GET_ITEM(o, 4);
  if (!THPVariable_Check(v) || !THPVariable_Check(s) || (d != f16 && d != bf16)) return false;
  h.values = &THPVariable_Unpack(v), h.scales = &THPVariable_Unpack(s);
  h.rows = PyLong_AsLongLong(PyTuple_GET_ITEM(o, 2)), h.cols = PyLong_AsLongLong(PyTuple_GET_ITEM(o, 3));
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  h.type = d == f16 ? at::kHalf : at::kBFloat16;
  if (h.rows < 0 || h.cols < 1 || h.rows > TCCL_TRAINING_MAX_ROWS || h.cols > INT32_MAX) return false;
  const at::Device device = h.values->device();
  const int64_t rb = row_blocks(h.rows), cb = col_blocks(h.cols);
  return bytes_of(*h.values, device) && bytes_of(*h.scales, device) && h.values->dim() == 3 && h.values->size(0) == rb && h.values->size(1) == cb * TCCL_HELD_COLS &&
         h.values->size(2) == TCCL_HELD_ROWS && h.scales->dim() == 2 && h.scales->size(0) == cb && h.scales->size(1) == (rb + 15) / 16 * 16;
}

at::Tensor empty(at::IntArrayRef sizes, at::ScalarType type, const at::Device& device) {
  return at::Tensor(at::detail::empty_cuda(sizes, type, device, std::nullopt));
}

// n elements of `base` from `offset` on, as a tensor of their own in the same memory.
at::Tensor part(const at::Tensor& base, int64_t offset, int64_t n) {
  at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(base.storage()), base.key_set(), base.dtype());
  t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
  t.unsafeGetTensorImpl()->set_storage_offset(offset);
  return t;
}

struct Owned {
  PyObject* o = nullptr;
  ~Owned() { Py_XDECREF(o); }
};

// An instance of a named tuple from its fields; takes the references over.
PyObject* named(PyObject* type, PyObject* const* fields, int n) {
  Owned tuple, args;
  bool whole = true;
  for (int i = 0; i < n; ++i) whole = whole && fields[i];
  if (whole) tuple.o = PyTuple_New(n);
  if (!tuple.o) {
    for (int i = 0; i < n; ++i) Py_XDECREF(fields[i]);
    return nullptr;
  }
  for (int i = 0; i < n; ++i) PyTuple_SET_ITEM(tuple.o, i, fields[i]);
  args.o = PyTuple_Pack(1, tuple.o);
  return args.o ? PyTuple_Type.tp_new((PyTypeObject*)type, args.o, nullptr) : nullptr;
}

PyObject* optional(const at::Tensor& t) { return t.defined() ? THPVariable_Wrap(t) : none(); }

bool stream_now(void*& stream) {
  PyObject* index[1] = {device0};
  Owned s;
  s.o = PyObject_Vectorcall(current_stream, index, 1, nullptr);
  if (!s.o) return false;
  stream = (void*)(uintptr_t)PyLong_AsUnsignedLongLong(s.o);
  return !PyErr_Occurred();
}

// The entry point has refused or failed: raises what `report` makes of it.
bool failed(int rc, const char* what) {
  if (!rc) return false;
  Owned r;
  r.o = PyObject_CallFunction(report, "is", rc, what);
  if (r.o) PyErr_SetString(PyExc_RuntimeError, what);
  return true;
}

struct HeldOut {
  at::Tensor values, scales;
  void make(int64_t rows, int64_t cols, const at::Device& device) {
    const int64_t rb = row_blocks(rows), cb = col_blocks(cols);
    values = empty({rb, cb * TCCL_HELD_COLS, TCCL_HELD_ROWS}, at::kByte, device);
    scales = empty({cb, (rb + 15) / 16 * 16}, at::kByte, device);
  }
  PyObject* wrapped(int64_t rows, int64_t cols, at::ScalarType type) const {
    PyObject* dtype = type == at::kHalf ? f16 : bf16;
    Py_INCREF(dtype);
    PyObject* fields[5] = {THPVariable_Wrap(values), THPVariable_Wrap(scales), PyLong_FromLongLong(rows), PyLong_FromLongLong(cols), dtype};
    return named(checkpoint_type, fields, 5);
  }
};

// layer_norm(x, weight, bias, eps, residual, checkpoint, out)
PyObject* layer_norm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 7) return none();
  return guarded([&]() -> PyObject* {
    Matrix x, residual, out;
    tccl_norm_desc d;
    memset(&d, 0, sizeof d);
    if (!x.open(args[0])) return none();
    const at::ScalarType type = x.t->scalar_type();
    const at::Device device = x.t->device();
    const int code = code_of(type);
    if (code < 0 || x.cols > TCCL_NORM_MAX_COLS) return none();
    d.dtype = d.affine_dtype = code;
    const at::Tensor* affine[2] = {nullptr, nullptr};
    for (int i = 1; i <= 2; ++i) {
      if (args[i] == Py_None) continue;
      const at::Tensor*& t = affine[i - 1];
      if (!vector_of(args[i], x.cols, device, t) || (t->scalar_type() != type && t->scalar_type() != at::kFloat)) return none();
      if (i == 2 && d.weight && d.affine_dtype != code_of(t->scalar_type())) return none();
      d.affine_dtype = code_of(t->scalar_type());
      (i == 1 ? d.weight : d.bias) = t->data_ptr();
    }
    d.eps = (float)PyFloat_AsDouble(args[3]);
    const int wanted = PyObject_IsTrue(args[5]);
    if (PyErr_Occurred()) return nullptr;
    if (wanted && type == at::kFloat) return none();
    if (args[4] != Py_None && (!residual.open(args[4]) || !residual.like(x))) return none();
    if (args[6] != Py_None && (!out.open(args[6]) || !out.like(x) || !out.apart(x) || !out.apart(residual) || !out.clear_of(affine[0]) || !out.clear_of(affine[1])))
      return none();
    at::Tensor made, summed, stats = empty({2 * x.rows}, at::kFloat, device);
    HeldOut held;
    d.x = x.at, d.ld_x = x.pitch, d.rows = (int32_t)x.rows, d.cols = (int32_t)x.cols;
    if (!out.t) {
      made = empty({x.rows, x.cols}, type, device);
      d.out = made.data_ptr(), d.ld_out = x.cols;
    } else {
      d.out = out.at, d.ld_out = out.pitch;
    }
    if (residual.t) {
      summed = empty({x.rows, x.cols}, type, device);
      d.residual = residual.at, d.ld_residual = residual.pitch, d.summed = summed.data_ptr(), d.ld_summed = x.cols;
    }
    if (wanted) {
      held.make(x.rows, x.cols, device);
      d.values = held.values.data_ptr(), d.scales = held.scales.data_ptr();
    }
    d.mean = (float*)stats.data_ptr(), d.rstd = d.mean + x.rows;
    void* stream;
    if (!stream_now(stream)) return nullptr;
    if (failed(entry_norm(&d, stream), "tccl_layer_norm")) return nullptr;
    PyObject* result = args[6];
    if (out.t)
      Py_INCREF(result);
    else
      result = THPVariable_Wrap(made);
    PyObject* fields[5] = {result, THPVariable_Wrap(part(stats, 0, x.rows)), THPVariable_Wrap(part(stats, x.rows, x.rows)), optional(summed),
                           wanted ? held.wrapped(x.rows, x.cols, type) : none()};
    return named(norm_result, fields, 5);
  });
}

// layer_norm_backward(grad, x, mean, rstd, weight, grad_summed, affine, out)
PyObject* layer_norm_backward(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 8) return none();
  return guarded([&]() -> PyObject* {
    Matrix grad, x, more, out;
    Held held;
    tccl_norm_grad_desc d;
    memset(&d, 0, sizeof d);
    if (!grad.open(args[0])) return none();
    const at::ScalarType type = grad.t->scalar_type();
    const at::Device device = grad.t->device();
    const int code = code_of(type);
    if (code < 0 || grad.cols > TCCL_NORM_MAX_COLS) return none();
    const bool full = THPVariable_Check(args[1]);
    if (full) {
      if (!x.open(args[1]) || !x.like(grad)) return none();
      d.x = x.at, d.ld_x = x.pitch;
    } else {
      if (!open_held(args[1], held) || held.rows != grad.rows || held.cols != grad.cols || held.type != type || held.values->device() != device) return none();
      d.values = held.values->data_ptr(), d.scales = held.scales->data_ptr();
    }
    const at::Tensor *mean, *rstd, *weight = nullptr;
    if (!vector_of(args[2], grad.rows, device, mean) || mean->scalar_type() != at::kFloat) return none();
    if (!vector_of(args[3], grad.rows, device, rstd) || rstd->scalar_type() != at::kFloat) return none();
    d.mean = (const float*)mean->data_ptr(), d.rstd = (const float*)rstd->data_ptr();
    d.dtype = d.affine_dtype = code;
    if (args[4] != Py_None) {
      if (!vector_of(args[4], grad.cols, device, weight) || (weight->scalar_type() != type && weight->scalar_type() != at::kFloat)) return none();
      d.weight = weight->data_ptr(), d.affine_dtype = code_of(weight->scalar_type());
    }
    if (args[5] != Py_None) {
      if (!more.open(args[5]) || !more.like(grad)) return none();
      d.grad_summed = more.at, d.ld_grad_summed = more.pitch;
    }
    const int affine = PyObject_IsTrue(args[6]);
    if (affine < 0) return nullptr;
    if (args[7] != Py_None && (!out.open(args[7]) || !out.like(grad) || !out.apart(grad) || !out.apart(more) || !out.apart(x) || !out.clear_of(held.values) ||
                               !out.clear_of(held.scales) || !out.clear_of(mean) || !out.clear_of(rstd) || !out.clear_of(weight)))
      return none();
    at::Tensor made, sums;
    d.grad = grad.at, d.ld_grad = grad.pitch, d.rows = (int32_t)grad.rows, d.cols = (int32_t)grad.cols;
    if (!out.t) {
      made = empty({grad.rows, grad.cols}, type, device);
      d.dx = made.data_ptr(), d.ld_dx = grad.cols;
    } else {
      d.dx = out.at, d.ld_dx = out.pitch;
    }
    if (affine) {
      sums = empty({2 * grad.cols}, at::kFloat, device);
      d.dweight = (float*)sums.data_ptr(), d.dbias = d.dweight + grad.cols;
    }
    d.workspace_bytes = entry_norm_grad_workspace(d.rows, d.cols, code, !full);
    if (d.workspace_bytes < 0) return failed((int)TCCL_ERR_UNSUPPORTED, "tccl_layer_norm_grad"), nullptr;
    const at::Tensor workspace = empty({d.workspace_bytes}, at::kByte, device);
    d.workspace = workspace.data_ptr();
    void* stream;
    if (!stream_now(stream)) return nullptr;
    if (failed(entry_norm_grad(&d, stream), "tccl_layer_norm_grad")) return nullptr;
    PyObject* result = args[7];
    if (out.t)
      Py_INCREF(result);
    else
      result = THPVariable_Wrap(made);
    PyObject* fields[3] = {result, affine ? THPVariable_Wrap(part(sums, 0, grad.cols)) : none(), affine ? THPVariable_Wrap(part(sums, grad.cols, grad.cols)) : none()};
    return named(norm_gradients, fields, 3);
  });
}

// checkpoint_activation(x)
PyObject* checkpoint_activation(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 1) return none();
  return guarded([&]() -> PyObject* {
    Matrix x;
    if (!x.open(args[0])) return none();
    const at::ScalarType type = x.t->scalar_type();
    if (type != at::kHalf && type != at::kBFloat16) return none();
    HeldOut held;
    held.make(x.rows, x.cols, x.t->device());
    const tccl_held_desc d = {x.at, held.values.data_ptr(), held.scales.data_ptr(), x.pitch, (int32_t)x.rows, (int32_t)x.cols, code_of(type)};
    void* stream;
    if (!stream_now(stream)) return nullptr;
    if (failed(entry_hold(&d, stream), "tccl_hold")) return nullptr;
    return held.wrapped(x.rows, x.cols, type);
  });
}

// restore_activation(held, out)
PyObject* restore_activation(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 2) return none();
  return guarded([&]() -> PyObject* {
    Held held;
    Matrix out;
    at::Tensor made;
    if (!open_held(args[0], held)) return none();
    tccl_held_desc d = {nullptr, held.values->data_ptr(), held.scales->data_ptr(), held.cols, (int32_t)held.rows, (int32_t)held.cols, code_of(held.type)};
    if (args[1] != Py_None) {
      if (!out.open(args[1]) || out.rows != held.rows || out.cols != held.cols || out.t->scalar_type() != held.type || out.t->device() != held.values->device() ||
          !out.clear_of(held.values) || !out.clear_of(held.scales))
        return none();
      d.x = out.at, d.ld = out.pitch;
    } else {
      made = empty({held.rows, held.cols}, held.type, held.values->device());
      d.x = made.data_ptr();
    }
    void* stream;
    if (!stream_now(stream)) return nullptr;
    if (failed(entry_restore(&d, stream), "tccl_restore")) return nullptr;
    if (made.defined()) return THPVariable_Wrap(made);
    Py_INCREF(args[1]);
    return args[1];
  });
}

// weight_gradient(held, grad, outputs, transposed, out_dtype, add, out): outputs is None, or how many of the columns of grad
// have a part (its rows have been filled up to whole vectors).
PyObject* weight_gradient(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 7) return none();
  return guarded([&]() -> PyObject* {
    Held held;
    Matrix grad, add, out;
    if (!open_held(args[0], held) || !grad.open(args[1])) return none();
    const at::ScalarType type = grad.t->scalar_type();
    const at::Device device = grad.t->device();
    if (held.type != type || held.rows != grad.rows || held.values->device() != device) return none();
    // Rows that are no whole 16-byte vectors are copied first (ops_training.py).
    if (grad.rows && (grad.cols % 8 || (grad.rows > 1 && grad.pitch % 8) || (uintptr_t)grad.at % 16)) return none();
    const int64_t outputs = args[2] == Py_None ? grad.cols : PyLong_AsLongLong(args[2]);
    const int transposed = PyObject_IsTrue(args[3]);
    if (PyErr_Occurred()) return nullptr;
    if (outputs < 1 || outputs > grad.cols) return none();
    if (args[4] != f32 && args[4] != (type == at::kHalf ? f16 : bf16)) return none();
    const at::ScalarType result = args[4] == f32 ? at::kFloat : type;
    const int64_t rows = transposed ? outputs : held.cols, cols = transposed ? held.cols : outputs;
    tccl_weight_gradient_desc d;
    memset(&d, 0, sizeof d);
    if (args[5] != Py_None) {
      if (!add.open(args[5]) || add.rows != rows || add.cols != cols || add.t->scalar_type() != result || add.t->device() != device) return none();
      d.add = add.at, d.ld_add = add.pitch;
    }
    at::Tensor made;
    if (args[6] != Py_None) {
      if (!out.open(args[6]) || out.rows != rows || out.cols != cols || out.t->scalar_type() != result || out.t->device() != device || !out.apart(add) || !out.elsewhere(grad) ||
          !out.clear_of(held.values) || !out.clear_of(held.scales))
        return none();
      d.out = out.at, d.ld_out = out.pitch;
    } else {
      made = empty({rows, cols}, result, device);
      d.out = made.data_ptr(), d.ld_out = cols;
    }
    d.values = held.values->data_ptr(), d.scales = held.scales->data_ptr();
    d.grad = grad.at, d.ld_grad = grad.pitch;
    d.rows = (int32_t)grad.rows, d.cols = (int32_t)held.cols, d.outputs = (int32_t)outputs;
    d.dtype = code_of(type), d.out_dtype = code_of(result), d.transposed = transposed;
    d.workspace_bytes = entry_weight_workspace(d.rows, d.cols, d.outputs);
    if (d.workspace_bytes < 0) return failed((int)TCCL_ERR_INVALID, "tccl_weight_gradient"), nullptr;
    at::Tensor workspace;
    if (d.workspace_bytes) {
      workspace = empty({d.workspace_bytes}, at::kByte, device);
      d.workspace = workspace.data_ptr();
    }
    void* stream;
    if (!stream_now(stream)) return nullptr;
    if (failed(entry_weight(&d, stream), "tccl_weight_gradient")) return nullptr;
    if (made.defined()) return THPVariable_Wrap(made);
    Py_INCREF(args[6]);
    return args[6];
  });
}

// bind_operators(stream, report, (LayerNormResult, LayerNormGradients, ActivationCheckpoint), (float16, bfloat16, float32), entries):
// entries are the addresses of the entry points, in the order below.
PyObject* bind_operators(PyObject*, PyObject* args) {
  PyObject *stream, *rep, *result, *gradients, *checkpoint, *half, *bfloat, *full;
  unsigned long long e[7];
  if (!PyArg_ParseTuple(args, "OO(OOO)(OOO)(KKKKKKK)", &stream, &rep, &result, &gradients, &checkpoint, &half, &bfloat, &full, e, e + 1, e + 2, e + 3, e + 4, e + 5, e + 6))
    return nullptr;
  for (PyObject* type : {result, gradients, checkpoint})
    if (!PyType_Check(type) || !PyType_IsSubtype((PyTypeObject*)type, &PyTuple_Type)) {
      PyErr_SetString(PyExc_TypeError, "results are named tuples");
      return nullptr;
    }
  PyObject** slots[] = {&current_stream, &report, &norm_result, &norm_gradients, &checkpoint_type, &f16, &bf16, &f32};
  PyObject* values[] = {stream, rep, result, gradients, checkpoint, half, bfloat, full};
  for (int i = 0; i < 8; ++i) {
    Py_INCREF(values[i]);
    Py_XSETREF(*slots[i], values[i]);
  }
  if (!device0) device0 = PyLong_FromLong(0);  // every rank lives on device 0
  entry_norm = (decltype(entry_norm))(uintptr_t)e[0];
  entry_norm_grad = (decltype(entry_norm_grad))(uintptr_t)e[1];
  entry_norm_grad_workspace = (decltype(entry_norm_grad_workspace))(uintptr_t)e[2];
  entry_hold = (decltype(entry_hold))(uintptr_t)e[3];
  entry_restore = (decltype(entry_restore))(uintptr_t)e[4];
  entry_weight = (decltype(entry_weight))(uintptr_t)e[5];
  entry_weight_workspace = (decltype(entry_weight_workspace))(uintptr_t)e[6];
  Py_RETURN_NONE;
}

#define FAST(f) (PyCFunction)(void (*)())f, METH_FASTCALL, nullptr
PyMethodDef methods[] = {{"bind_operators", bind_operators, METH_VARARGS, nullptr},
                         {"layer_norm", FAST(layer_norm)},
                         {"layer_norm_backward", FAST(layer_norm_backward)},
                         {"checkpoint_activation", FAST(checkpoint_activation)},
                         {"restore_activation", FAST(restore_activation)},
                         {"weight_gradient", FAST(weight_gradient)},
                         {nullptr, nullptr, 0, nullptr}};

}  // namespace

PyMethodDef* operator_methods() { return methods; }
