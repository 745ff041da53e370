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

#include <algorithm>
#include <cstdint>
#include <cstring>
#include <exception>
#include <utility>
#include <vector>

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
// What bind_layers() is given.
PyObject* gated_result;
int (*entry_weight_full)(const tccl_weight_gradient_full_desc*, void*);
int64_t (*entry_weight_full_workspace)(const tccl_weight_gradient_full_desc*);
int (*entry_gated)(const tccl_gated_desc*, void*);
int64_t (*entry_gated_workspace)(const tccl_gated_desc*);
int64_t (*entry_gated_grad_workspace)(const tccl_gated_grad_desc*);
int (*entry_gated_grad)(const tccl_gated_grad_desc*, void*);
int (*entry_gemm)(const tccl_gemm_desc*, void*);
int64_t (*entry_input_grad_workspace)(const tccl_gated_input_grad_desc*);
int (*entry_input_grad_cut)(int32_t, int32_t, int32_t, int32_t, int32_t*);
int (*entry_input_grad)(const tccl_gated_input_grad_desc*, void*);
int (*entry_pack)(const tccl_pack_desc*, int32_t, int32_t, void*);
int (*entry_adamw)(const tccl_adamw_desc*, void*);
int (*entry_moments)(const tccl_adamw_moments_desc*, void*);

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

  // turned: the transposed view.
  bool open(PyObject* o, bool turned = false) {
    if (!THPVariable_Check(o)) return false;
    t = &THPVariable_Unpack(o);
    if (!t->is_cuda() || t->layout() != at::kStrided || t->dim() != 2 || t->is_neg()) return false;
    rows = t->size(turned), cols = t->size(!turned);
    if (cols < 1 || rows > TCCL_TRAINING_MAX_ROWS || cols > INT32_MAX || (cols > 1 && t->stride(!turned) != 1)) return false;
    pitch = rows > 1 ? t->stride(turned) : cols;
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
  // No byte of either's rows lies in the other's; rows of one pitch may lie beside each other.
  bool clear_of(const Matrix& m) const {
    if (elsewhere(m)) return true;
    const int64_t step = pitch * (int64_t)t->element_size(), width = cols * (int64_t)t->element_size(), other = m.cols * (int64_t)m.t->element_size();
    if (rows < 2 || m.rows < 2 || step != m.pitch * (int64_t)m.t->element_size()) return false;
    const int64_t ahead = ((m.at - at) % step + step) % step;
    return ahead >= width && ahead + other <= step;
  }
  // The same elements in the same places, or none in common.
  bool apart(const Matrix& m) const { return !m.t || elsewhere(m) || (at == m.at && pitch == m.pitch && t->scalar_type() == m.t->scalar_type()); }
};

bool vector_of(PyObject* o, int64_t n, const at::Device& device, const at::Tensor*& t) {
  if (!THPVariable_Check(o)) return false;
  t = &THPVariable_Unpack(o);
  return t->is_cuda() && t->layout() == at::kStrided && t->dim() == 1 && t->size(0) == n && t->device() == device && (n <= 1 || t->stride(0) == 1) && !t->is_neg();
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

// ---- the gated layer, weight gradients from an input in full, AdamW ---------------------------------

bool on_device0(const at::Tensor& t) { return t.is_cuda() && t.device().index() == 0; }  // where the ranks live

constexpr int64_t kMostPitch = 1 << 24;  // of what weight gradients read

bool sixteen_bits(at::ScalarType t) { return t == at::kHalf || t == at::kBFloat16; }

// The workspace that a call asks for; false: an error is set.
template <typename Desc>
bool with_workspace(Desc& d, int64_t (*entry)(const Desc*), const char* what, const at::Device& device, at::Tensor& workspace) {
  d.workspace_bytes = entry(&d);
  if (d.workspace_bytes < 0) return failed((int)TCCL_ERR_INVALID, what), false;
  if (d.workspace_bytes) {
    workspace = empty({d.workspace_bytes}, at::kByte, device);
    d.workspace = workspace.data_ptr();
  }
  return true;
}

// A weight (inputs x 2 outputs) as its memory lies: by rows, or (k-major) as 2 outputs rows of inputs.
struct GatedWeight {
  const at::Tensor* t = nullptr;
  char* at = nullptr;
  int64_t inputs = 0, outputs = 0, pitch = 0, up = 0;
  bool kmajor = false;

  bool open(PyObject* o) {
    if (!THPVariable_Check(o)) return false;
    t = &THPVariable_Unpack(o);
    if (!on_device0(*t) || t->layout() != at::kStrided || t->dim() != 2 || t->is_neg()) return false;
    inputs = t->size(0), outputs = t->size(1) / 2;
    if (inputs < 1 || outputs < 1 || t->size(1) % 2 || inputs > TCCL_GATED_MAX_COLS || outputs > TCCL_GATED_MAX_COLS || !sixteen_bits(t->scalar_type())) return false;
    at = (char*)t->data_ptr();
    if (t->stride(1) == 1 && (inputs == 1 || t->stride(0) >= 2 * outputs)) {
      pitch = inputs > 1 ? t->stride(0) : 2 * outputs;
      up = outputs;
      return true;
    }
    kmajor = true;
    pitch = t->stride(1), up = outputs * pitch;
    return (inputs == 1 || t->stride(0) == 1) && pitch >= inputs;
  }
  bool clear_of(const Matrix& m) const {
    const char* end = at + ((kmajor ? 2 * outputs - 1 : inputs - 1) * pitch + (kmajor ? inputs : 2 * outputs)) * 2;
    return !(at < m.end() && m.at < end);
  }
};

// gated_linear(x, weight, activation, keep, out)
PyObject* gated_linear(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 5) return none();
  return guarded([&]() -> PyObject* {
    Matrix x, out;
    GatedWeight w;
    if (!x.open(args[0]) || !on_device0(*x.t) || !w.open(args[1])) return none();
    const at::ScalarType type = x.t->scalar_type();
    const at::Device device = x.t->device();
    if (type != w.t->scalar_type() || x.cols != w.inputs) return none();
    tccl_gated_desc d;
    memset(&d, 0, sizeof d);
    d.activation = (int32_t)PyLong_AsLong(args[2]);
    const int keep = PyObject_IsTrue(args[3]);
    if (PyErr_Occurred()) return nullptr;
    at::Tensor made, kept;
    if (args[4] != Py_None) {
      if (!out.open(args[4]) || out.rows != x.rows || out.cols != w.outputs || out.t->scalar_type() != type || out.t->device() != device || !out.elsewhere(x) || !w.clear_of(out))
        return none();
      d.out = out.at, d.ld_out = out.pitch;
    } else {
      made = empty({x.rows, w.outputs}, type, device);
      d.out = made.data_ptr(), d.ld_out = w.outputs;
    }
    if (keep) {
      kept = empty({x.rows, 2 * w.outputs}, type, device);
      d.kept = kept.data_ptr(), d.ld_kept = 2 * w.outputs;
    }
    d.x = x.at, d.weight = w.at, d.ld_x = x.pitch, d.ld_weight = w.pitch, d.up = w.up;
    d.rows = (int32_t)x.rows, d.inputs = (int32_t)w.inputs, d.outputs = (int32_t)w.outputs;
    d.dtype = code_of(type), d.kmajor = w.kmajor;
    at::Tensor workspace;
    if (!with_workspace(d, entry_gated_workspace, "tccl_gated", device, workspace)) return nullptr;
    void* stream;
    if (!stream_now(stream)) return nullptr;
    if (failed(entry_gated(&d, stream), "tccl_gated")) return nullptr;
    PyObject* result = args[4];
    if (out.t)
      Py_INCREF(result);
    else
      result = THPVariable_Wrap(made);
    PyObject* fields[2] = {result, optional(kept)};
    return named(gated_result, fields, 2);
  });
}

// What weight_gradient() will be given beside `inner` (t NULL: memory of its own): x, a tensor or its checkpoint, the result's type or what is added.
// All that it refuses is refused ahead of the launch that writes inner, perhaps over what this is made of.
struct WeightGradientWanted {
  Matrix x, add;
  Held held;

  bool takes(PyObject* o, const GatedWeight& w, int64_t rows, at::ScalarType type, const at::Device& device, const Matrix& inner, PyObject* out_dtype, PyObject* added) {
    const bool on_vectors = inner.cols % 8 == 0 && (inner.rows <= 1 || inner.pitch % 8 == 0) && (uintptr_t)inner.at % 16 == 0;
    if (THPVariable_Check(o)) {
      if (!x.open(o) || x.t->scalar_type() != type || x.t->device() != device || x.rows != rows || x.cols != w.inputs || x.pitch > kMostPitch) return false;
      if (inner.t && inner.pitch > kMostPitch) return false;
    } else {
      if (!open_held(o, held) || held.type != type || held.values->device() != device || held.rows != rows || held.cols != w.inputs || (uintptr_t)held.values->data_ptr() % 16) return false;
      if (inner.t && on_vectors && inner.pitch > kMostPitch) return false;  // (else it is copied)
    }
    if (added == Py_None) return out_dtype == f32 || out_dtype == (type == at::kHalf ? f16 : bf16);
    return add.open(added, w.kmajor) && add.rows == (w.kmajor ? 2 * w.outputs : w.inputs) && add.cols == (w.kmajor ? w.inputs : 2 * w.outputs) &&
           (add.t->scalar_type() == at::kFloat || add.t->scalar_type() == type) && add.t->device() == device;
  }
  // Nothing of it lies where inner goes.
  bool clear_of(const Matrix& inner) const {
    return (!x.t || inner.clear_of(x)) && inner.clear_of(held.values) && inner.clear_of(held.scales) && (!add.t || inner.clear_of(add));
  }
};

// gated_gradient(grad, kept, x, weight, activation, out, weights, out_dtype, add): of the projections.  With kept, weight is not read.  `weights`: weight_gradient()
// of x, out_dtype and add follows.
PyObject* gated_gradient(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 9) return none();
  return guarded([&]() -> PyObject* {
    Matrix grad, kept, x, out;
    GatedWeight w;
    WeightGradientWanted wanted;
    if (!grad.open(args[0]) || !on_device0(*grad.t) || !w.open(args[3])) return none();
    const at::ScalarType type = grad.t->scalar_type();
    const at::Device device = grad.t->device();
    if (!sixteen_bits(type) || w.t->scalar_type() != type || grad.cols != w.outputs) return none();
    const bool computed = args[1] == Py_None;
    if (computed) {
      if (!x.open(args[2]) || x.t->scalar_type() != type || x.t->device() != device || x.cols != w.inputs || x.rows != grad.rows) return none();
    } else if (!kept.open(args[1]) || kept.rows != grad.rows || kept.cols != 2 * w.outputs || kept.t->scalar_type() != type || kept.t->device() != device) {
      return none();
    }
    tccl_gated_grad_desc d;
    memset(&d, 0, sizeof d);
    d.activation = (int32_t)PyLong_AsLong(args[4]);
    const int weights = PyObject_IsTrue(args[6]);
    if (PyErr_Occurred()) return nullptr;
    at::Tensor made;
    if (args[5] != Py_None) {
      if (!out.open(args[5]) || out.rows != grad.rows || out.cols != 2 * w.outputs || out.t->scalar_type() != type || out.t->device() != device || !out.elsewhere(grad) ||
          !out.apart(kept) || (x.t && !out.elsewhere(x)) || !w.clear_of(out))
        return none();
      d.inner = out.at, d.ld_inner = out.pitch;
    } else {
      made = empty({grad.rows, 2 * w.outputs}, type, device);
      d.inner = made.data_ptr(), d.ld_inner = 2 * w.outputs;
    }
    if (weights && (!wanted.takes(args[2], w, grad.rows, type, device, out, args[7], args[8]) || (out.t && !wanted.clear_of(out)))) return none();
    d.grad = grad.at, d.ld_grad = grad.pitch;
    if (computed)
      d.x = x.at, d.ld_x = x.pitch, d.weight = w.at, d.ld_weight = w.pitch, d.up = w.up;
    else
      d.kept = kept.at, d.ld_kept = kept.pitch;
    d.rows = (int32_t)grad.rows, d.inputs = (int32_t)w.inputs, d.outputs = (int32_t)w.outputs;
    d.dtype = code_of(type), d.kmajor = w.kmajor;
    at::Tensor workspace;
    if (!with_workspace(d, entry_gated_grad_workspace, "tccl_gated_grad", device, workspace)) return nullptr;
    void* stream;
    if (!stream_now(stream)) return nullptr;
    if (failed(entry_gated_grad(&d, stream), "tccl_gated_grad")) return nullptr;
    if (made.defined()) return THPVariable_Wrap(made);
    Py_INCREF(args[5]);
    return args[5];
  });
}

// The same by tccl_gated_input_grad, whose tiles start anew from a 64-bit address in every step.
PyObject* input_gradient_in_tiles(const Matrix& inner, const GatedWeight& w) {
  const at::ScalarType type = inner.t->scalar_type();
  const at::Tensor dx = empty({inner.rows, w.inputs}, type, inner.t->device());
  tccl_gated_input_grad_desc d;
  memset(&d, 0, sizeof d);
  d.inner = inner.at, d.weight = w.at, d.dx = dx.data_ptr();
  d.ld_inner = inner.pitch, d.ld_weight = w.pitch, d.ld_dx = w.inputs;
  d.rows = (int32_t)inner.rows, d.inputs = (int32_t)w.inputs, d.outputs = (int32_t)w.outputs, d.dtype = code_of(type), d.kmajor = w.kmajor;
  at::Tensor workspace;
  if (!with_workspace(d, entry_input_grad_workspace, "tccl_gated_input_grad", inner.t->device(), workspace)) return nullptr;
  void* stream;
  if (!stream_now(stream)) return nullptr;
  if (failed(entry_input_grad(&d, stream), "tccl_gated_input_grad")) return nullptr;
  return THPVariable_Wrap(dx);
}

// input_gradient(inner, weight): inner @ weight.t(), by the kernel that splits the sum where it is the quicker one; else by the library's GEMM, which reads
// whole 16-byte vectors (an operand that does not lie in these is copied first, both in one launch), writes them and reaches 4 GiB far from a tile's
// base: the rows of a tile, and all of a k-major weight, the last step's 64 of its rows in full.  What is longer, and rows of a result that are no
// whole vectors, are left to the former.
PyObject* input_gradient(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 2) return none();
  return guarded([&]() -> PyObject* {
    Matrix inner;
    GatedWeight w;
    if (!inner.open(args[0]) || !on_device0(*inner.t) || !w.open(args[1])) return none();
    const at::ScalarType type = inner.t->scalar_type();
    if (w.t->scalar_type() != type || inner.cols != 2 * w.outputs) return none();
    int32_t splits = 0;
    if (failed(entry_input_grad_cut((int32_t)inner.rows, (int32_t)w.inputs, (int32_t)w.outputs, 0, &splits), "tccl_gated_input_grad_cut")) return nullptr;
    const int64_t N = w.inputs, K = inner.cols, depth = (K + 7) / 8 * 8;
    if (splits || N % 8) return input_gradient_in_tiles(inner, w);
    const bool copy_a = K != depth || inner.pitch % 8 || (uintptr_t)inner.at % 16, copy_b = K != depth || w.pitch % 8 || (uintptr_t)w.at % 16;
    auto on_64_bytes = [](int64_t cols) { return (cols + 31) / 32 * 32; };  // as the GEMM fetches rows
    const int64_t lda = copy_a ? on_64_bytes(depth) : inner.pitch, ldb = copy_b ? on_64_bytes(w.kmajor ? N : depth) : w.pitch;
    const int64_t span_a = 255 * lda + depth, span_b = w.kmajor ? ((depth + 63) / 64 * 64 - 1) * ldb + N : 255 * ldb + depth;
    if (std::max(span_a, span_b) * 2 > 0xfffffff0ll) return input_gradient_in_tiles(inner, w);
    const at::Tensor dx = empty({inner.rows, N}, type, inner.t->device());
    if (!inner.rows) return THPVariable_Wrap(dx);
    void* stream;
    if (!stream_now(stream)) return nullptr;
    tccl_gemm_desc d;
    memset(&d, 0, sizeof d);
    d.A = inner.at, d.B = w.at, d.C = dx.data_ptr();
    d.M = (int32_t)inner.rows, d.N = (int32_t)N, d.K = (int32_t)depth;
    d.lda = lda, d.ldb = ldb, d.ldc = N;
    d.in_dtype = d.out_dtype = code_of(type);
    d.alpha = 1.f, d.block_m = d.block_n = 128, d.group_m = 8;
    d.flags = w.kmajor ? 0 : TCCL_GEMM_B_KMAJOR;  // of weight.t(): its columns are the weight's rows
    tccl_pack_desc jobs[2];
    int n = 0;
    at::Tensor a, b;
    auto copied = [&](at::Tensor& to, const char* from, int64_t pitch, int64_t rows, int64_t cols, int64_t to_rows, int64_t to_cols, int64_t to_pitch) {
      to = empty({to_rows, to_pitch}, type, inner.t->device());
      jobs[n++] = {from, to.data_ptr(), pitch, 1, to_pitch, (int32_t)rows, (int32_t)cols, (int32_t)to_rows, (int32_t)to_cols};
      return to.data_ptr();
    };
    if (copy_a) d.A = copied(a, inner.at, inner.pitch, inner.rows, K, inner.rows, depth, lda);
    if (copy_b) d.B = w.kmajor ? copied(b, w.at, w.pitch, K, N, depth, N, ldb) : copied(b, w.at, w.pitch, N, K, N, depth, ldb);
    if (n && failed(entry_pack(jobs, n, 2, stream), "tccl_pack_matrices")) return nullptr;
    if (failed(entry_gemm(&d, stream), "tccl_gemm")) return nullptr;
    return THPVariable_Wrap(dx);
  });
}

// weight_gradient_full(x, grad, transposed, out_dtype, add, out)
PyObject* weight_gradient_full(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 6) return none();
  return guarded([&]() -> PyObject* {
    Matrix x, grad, add, out;
    if (!x.open(args[0]) || !on_device0(*x.t) || !grad.open(args[1])) return none();
    const at::ScalarType type = grad.t->scalar_type();
    const at::Device device = grad.t->device();
    if (!sixteen_bits(type) || x.t->scalar_type() != type || x.t->device() != device || x.rows != grad.rows) return none();
    if (x.cols > kMostPitch || grad.cols > kMostPitch || x.pitch > kMostPitch || grad.pitch > kMostPitch) return none();
    const int64_t inputs = x.cols, outputs = grad.cols;
    const int transposed = PyObject_IsTrue(args[2]);
    if (PyErr_Occurred()) return nullptr;
    if (args[3] != f32 && args[3] != (type == at::kHalf ? f16 : bf16)) return none();
    const at::ScalarType result = args[3] == f32 ? at::kFloat : type;
    const int64_t rows = transposed ? outputs : inputs, cols = transposed ? inputs : outputs;
    tccl_weight_gradient_full_desc d;
    memset(&d, 0, sizeof d);
    if (args[4] != Py_None) {
      if (!add.open(args[4]) || add.rows != rows || add.cols != cols || add.t->scalar_type() != result || add.t->device() != device) return none();
      d.add = add.at, d.ld_add = add.pitch;
    }
    at::Tensor made;
    if (args[5] != Py_None) {
      if (!out.open(args[5]) || out.rows != rows || out.cols != cols || out.t->scalar_type() != result || out.t->device() != device || !out.apart(add) || !out.elsewhere(grad) || !out.elsewhere(x))
        return none();
      d.out = out.at, d.ld_out = out.pitch;
    } else {
      made = empty({rows, cols}, result, device);
      d.out = made.data_ptr(), d.ld_out = cols;
    }
    d.x = x.at, d.ld_x = x.pitch, d.grad = grad.at, d.ld_grad = grad.pitch;
    d.rows = (int32_t)grad.rows, d.cols = (int32_t)inputs, d.outputs = (int32_t)outputs;
    d.dtype = code_of(type), d.out_dtype = code_of(result), d.transposed = transposed;
    at::Tensor workspace;
    if (!with_workspace(d, entry_weight_full_workspace, "tccl_weight_gradient_full", device, workspace)) return nullptr;
    void* stream;
    if (!stream_now(stream)) return nullptr;
    if (failed(entry_weight_full(&d, stream), "tccl_weight_gradient_full")) return nullptr;
    if (made.defined()) return THPVariable_Wrap(made);
    Py_INCREF(args[5]);
    return args[5];
  });
}

bool flat_of(PyObject* o, at::ScalarType type, int64_t least, const at::Tensor*& t) {
  if (!THPVariable_Check(o)) return false;
  t = &THPVariable_Unpack(o);
  return on_device0(*t) && t->layout() == at::kStrided && t->dim() == 1 && t->scalar_type() == type && t->numel() >= least && (t->numel() <= 1 || t->stride(0) == 1) &&
         !t->is_neg() && !((uintptr_t)t->data_ptr() % 16 && type != at::kByte);
}

// A number, or a device tensor of one element that holds it.
bool number_or_word(PyObject* o, at::ScalarType type, const void*& at) {
  if (!THPVariable_Check(o)) return true;
  const at::Tensor& t = THPVariable_Unpack(o);
  at = t.data_ptr();
  return on_device0(t) && t.scalar_type() == type && t.numel() == 1 && !t.is_neg() && !((uintptr_t)at % 4);
}

typedef std::pair<const char*, const char*> Span;

// adamw_step(params, grads, (first, second, first_scales, second_scales, master, sizes), step, lr, beta1, beta2, eps, weight_decay, grad_scale):
// True, or None for arguments that it does not take.  params and grads are tuples.
PyObject* adamw_step(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 10) return none();
  return guarded([&]() -> PyObject* {
    if (!PyTuple_Check(args[0]) || !PyTuple_Check(args[1]) || !PyTuple_Check(args[2]) || PyTuple_GET_SIZE(args[2]) != 6) return none();
    const Py_ssize_t n = PyTuple_GET_SIZE(args[0]);
    PyObject* state[6];
    for (int i = 0; i < 6; ++i) state[i] = PyTuple_GET_ITEM(args[2], i);
    if (PyTuple_GET_SIZE(args[1]) != n || !PyTuple_Check(state[5]) || PyTuple_GET_SIZE(state[5]) != n || n > INT32_MAX) return none();
    tccl_adamw_desc d;
    memset(&d, 0, sizeof d);
    std::vector<void*> params(n), grads(n);
    std::vector<int64_t> sizes(n);
    std::vector<const at::Tensor*> tensors(n);
    std::vector<Span> written, read;
    int64_t blocks = 0;
    at::ScalarType type = at::kFloat, grad_type = at::kFloat;
    for (Py_ssize_t i = 0; i < n; ++i) {
      PyObject *po = PyTuple_GET_ITEM(args[0], i), *go = PyTuple_GET_ITEM(args[1], i);
      if (!THPVariable_Check(po) || !THPVariable_Check(go)) return none();
      const at::Tensor &p = THPVariable_Unpack(po), &g = THPVariable_Unpack(go);
      if (!i) type = p.scalar_type(), grad_type = g.scalar_type();
      if (!on_device0(p) || !on_device0(g) || p.scalar_type() != type || g.scalar_type() != grad_type || !p.sizes().equals(g.sizes()) || !p.is_contiguous() || !g.is_contiguous() || g.is_neg() ||
          p.is_neg())
        return none();
      sizes[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(state[5], i));
      if (PyErr_Occurred()) return nullptr;
      if (sizes[i] != p.numel()) return none();
      params[i] = p.data_ptr(), grads[i] = g.data_ptr(), tensors[i] = &p;
      blocks += (sizes[i] + TCCL_MOMENT_BLOCK - 1) / TCCL_MOMENT_BLOCK;
      if (sizes[i]) {
        written.emplace_back((const char*)p.data_ptr(), (const char*)p.data_ptr() + p.nbytes());
        read.emplace_back((const char*)g.data_ptr(), (const char*)g.data_ptr() + g.nbytes());
      }
    }
    d.dtype = code_of(type), d.grad_dtype = code_of(grad_type);
    if (d.dtype < 0 || d.grad_dtype < 0 || (grad_type != type && grad_type != at::kFloat)) return none();
    d.bits = state[2] == Py_None ? 32 : 8;
    const at::ScalarType moment = d.bits == 8 ? at::kByte : at::kFloat;
    const at::Tensor* flat[5] = {};
    for (int i = 0; i < 5; ++i) {
      if (i == 4 ? state[4] == Py_None : i >= 2 && d.bits == 32) {
        if (state[i] != Py_None) return none();
        continue;
      }
      const bool scales = i == 2 || i == 3;
      if (!flat_of(state[i], i == 4 ? at::kFloat : scales ? at::kByte : moment, scales ? blocks : blocks * TCCL_MOMENT_BLOCK, flat[i])) return none();
      if (!scales && (uintptr_t)flat[i]->data_ptr() % 16) return none();
      if (flat[i]->numel()) written.emplace_back((const char*)flat[i]->data_ptr(), (const char*)flat[i]->data_ptr() + flat[i]->nbytes());
    }
    if (flat[4] && type == at::kFloat) return none();
    // Nothing that is written shares memory with anything else.
    std::sort(written.begin(), written.end());
    for (size_t i = 1; i < written.size(); ++i)
      if (written[i].first < written[i - 1].second) return none();
    const void *step_at = nullptr, *lr_at = nullptr, *scale_at = nullptr;
    if (!number_or_word(args[3], at::kInt, step_at) || !number_or_word(args[4], at::kFloat, lr_at) || !number_or_word(args[9], at::kFloat, scale_at)) return none();
    for (const void* word : {step_at, lr_at, scale_at})
      if (word) read.emplace_back((const char*)word, (const char*)word + 4);
    for (const Span& g : read) {
      auto after = std::lower_bound(written.begin(), written.end(), Span(g.second, nullptr));
      if (after != written.begin() && (after - 1)->second > g.first) return none();
    }
    d.step_at = (const int32_t*)step_at, d.lr_at = (const float*)lr_at, d.grad_scale_at = (const float*)scale_at;
    const long long step = step_at ? 1 : PyLong_AsLongLong(args[3]);
    if (!lr_at) d.lr = PyFloat_AsDouble(args[4]);
    if (!scale_at) d.grad_scale = PyFloat_AsDouble(args[9]);
    d.beta1 = PyFloat_AsDouble(args[5]), d.beta2 = PyFloat_AsDouble(args[6]), d.eps = PyFloat_AsDouble(args[7]), d.weight_decay = PyFloat_AsDouble(args[8]);
    if (PyErr_Occurred()) return nullptr;
    if (step < 1 || step > INT32_MAX) return none();
    d.step = (int32_t)step;
    d.params = params.data(), d.grads = grads.data(), d.sizes = sizes.data(), d.tensors = (int32_t)n;
    d.first = flat[0]->data_ptr(), d.second = flat[1]->data_ptr();
    if (flat[2]) d.first_scales = flat[2]->data_ptr(), d.second_scales = flat[3]->data_ptr();
    if (flat[4]) d.master = flat[4]->data_ptr();
    void* stream;
    if (!stream_now(stream)) return nullptr;
    if (failed(entry_adamw(&d, stream), "tccl_adamw")) return nullptr;
    for (const at::Tensor* t : tensors)
      if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();  // what autograd has saved of them is no longer there
    Py_RETURN_TRUE;
  });
}

// adamw_moments(first, second, first_scales, second_scales)
PyObject* adamw_moments(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 4) return none();
  return guarded([&]() -> PyObject* {
    const at::Tensor *first, *second, *fs, *ss;
    if (!flat_of(args[0], at::kByte, 0, first)) return none();
    const int64_t n = first->numel(), blocks = n / TCCL_MOMENT_BLOCK;
    if (n % TCCL_MOMENT_BLOCK || !flat_of(args[1], at::kByte, n, second) || second->numel() != n || !flat_of(args[2], at::kByte, blocks, fs) || !flat_of(args[3], at::kByte, blocks, ss) ||
        ((uintptr_t)first->data_ptr() | (uintptr_t)second->data_ptr()) % 16)
      return none();
    const at::Tensor m = empty({n}, at::kBFloat16, first->device()), v = empty({n}, at::kBFloat16, first->device());
    const tccl_adamw_moments_desc d = {first->data_ptr(), second->data_ptr(), fs->data_ptr(), ss->data_ptr(), m.data_ptr(), v.data_ptr(), blocks};
    void* stream;
    if (!stream_now(stream)) return nullptr;
    if (failed(entry_moments(&d, stream), "tccl_adamw_moments")) return nullptr;
    Owned a, b;
    a.o = THPVariable_Wrap(m), b.o = THPVariable_Wrap(v);
    return a.o && b.o ? PyTuple_Pack(2, a.o, b.o) : nullptr;
  });
}

// bind_layers(GatedLinearResult, entries): the entry points in the order below.
PyObject* bind_layers(PyObject*, PyObject* args) {
  PyObject* result;
  unsigned long long e[13];
  if (!PyArg_ParseTuple(args, "O(KKKKKKKKKKKKK)", &result, e, e + 1, e + 2, e + 3, e + 4, e + 5, e + 6, e + 7, e + 8, e + 9, e + 10, e + 11, e + 12)) return nullptr;
  if (!PyType_Check(result) || !PyType_IsSubtype((PyTypeObject*)result, &PyTuple_Type)) {
    PyErr_SetString(PyExc_TypeError, "results are named tuples");
    return nullptr;
  }
  Py_INCREF(result);
  Py_XSETREF(gated_result, result);
  entry_weight_full = (decltype(entry_weight_full))(uintptr_t)e[0];
  entry_weight_full_workspace = (decltype(entry_weight_full_workspace))(uintptr_t)e[1];
  entry_gated = (decltype(entry_gated))(uintptr_t)e[2];
  entry_gated_grad = (decltype(entry_gated_grad))(uintptr_t)e[3];
  entry_adamw = (decltype(entry_adamw))(uintptr_t)e[4];
  entry_moments = (decltype(entry_moments))(uintptr_t)e[5];
  entry_gated_workspace = (decltype(entry_gated_workspace))(uintptr_t)e[6];
  entry_gated_grad_workspace = (decltype(entry_gated_grad_workspace))(uintptr_t)e[7];
  entry_gemm = (decltype(entry_gemm))(uintptr_t)e[8];
  entry_pack = (decltype(entry_pack))(uintptr_t)e[9];
  entry_input_grad_workspace = (decltype(entry_input_grad_workspace))(uintptr_t)e[10];
  entry_input_grad_cut = (decltype(entry_input_grad_cut))(uintptr_t)e[11];
  entry_input_grad = (decltype(entry_input_grad))(uintptr_t)e[12];
  Py_RETURN_NONE;
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
                         {"bind_layers", bind_layers, METH_VARARGS, nullptr},
                         {"gated_linear", FAST(gated_linear)},
                         {"gated_gradient", FAST(gated_gradient)},
                         {"input_gradient", FAST(input_gradient)},
                         {"weight_gradient_full", FAST(weight_gradient_full)},
                         {"adamw_step", FAST(adamw_step)},
                         {"adamw_moments", FAST(adamw_moments)},
                         {nullptr, nullptr, 0, nullptr}};

}  // namespace

PyMethodDef* operator_methods() { return methods; }
