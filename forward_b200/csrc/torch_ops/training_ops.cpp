// Python face of the training operators' C entry points (include/fwd_eb_train.h): argument checks, output and
// scratch tensors from torch's allocator, the call.  Written against the CPython API because the
// small calls of a training step take a few microseconds on the GPU, less than the same
// work costs in the interpreter (layer norm of 32 rows: 13.9 us a call through ctypes, 6.5 here).
//
// The entry points come as addresses (bind), so that the module runs with whichever build of the
// library the process loaded.  A call that the library refuses gives its status back as an int.
#include <ATen/ATen.h>
#include <Python.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <optional>
#include <string>

#include "fwd_eb_train.h"

namespace {

decltype(&fwd_eb_layer_norm_forward) g_norm_forward;
decltype(&fwd_eb_layer_norm_backward) g_norm_backward;
decltype(&fwd_eb_layer_norm_workspace_size) g_norm_workspace;
decltype(&fwd_eb_backward) g_backward;
decltype(&fwd_eb_backward_workspace_size) g_backward_workspace;

struct Refused {   // a Python exception to raise
  PyObject* type;
  std::string text;
};
[[noreturn]] void value_error(const std::string& text) { throw Refused{PyExc_ValueError, text}; }
[[noreturn]] void type_error(const std::string& text) { throw Refused{PyExc_TypeError, text}; }

using Maybe = const at::Tensor*;   // null: None was given

Maybe maybe(PyObject* o, const char* name) {
  if (o == Py_None) return nullptr;
  if (!THPVariable_Check(o)) type_error(std::string(name) + " must be a tensor");
  return &THPVariable_Unpack(o);
}
const at::Tensor& tensor(PyObject* o, const char* name) {
  Maybe t = maybe(o, name);
  if (!t) type_error(std::string(name) + " must be a tensor");
  return *t;
}
long long integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw python_error();
  return v != 0;
}

int code_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return FWD_EB_F32;
    case at::kHalf: return FWD_EB_F16;
    case at::kBFloat16: return FWD_EB_BF16;
    default: return -1;
  }
}
int dtype_of(const at::Tensor& t, const char* name) {
  const int code = code_of(t.scalar_type());
  if (code < 0) type_error(std::string(name) + ": unsupported dtype " + c10::toString(t.scalar_type()));
  return code;
}
at::ScalarType type_of(int code) {
  return code == FWD_EB_F32 ? at::kFloat : code == FWD_EB_F16 ? at::kHalf : at::kBFloat16;
}

struct Named {
  const char* name;
  Maybe t;
};
// Ordinal of the one CUDA device of the tensors; the first is there.
c10::DeviceIndex device_of(std::initializer_list<Named> all) {
  const c10::Device device = all.begin()->t->device();
  for (const Named& n : all) {
    if (!n.t) continue;
    if (!n.t->is_cuda()) value_error(std::string(n.name) + " must be a CUDA tensor; there is no CPU path");
    if (n.t->device() != device)
      value_error(std::string(n.name) + " is on " + n.t->device().str() + ", " + all.begin()->name + " on " + device.str());
  }
  return device.index();
}

// Row stride of a 2-D tensor with unit column stride (0, that is `cols`, when it has at most one row); refuses
// anything but [rows, cols] (rows < 0: any).
int64_t rows_of(const at::Tensor& t, const char* name, int64_t cols, int64_t rows) {
  if (t.dim() != 2 || t.size(1) != cols || (rows >= 0 && t.size(0) != rows))
    value_error(std::string(name) + " must be [" + (rows < 0 ? "n" : std::to_string(rows)) + ", " + std::to_string(cols) + "]");
  if (t.size(0) == 0) return 0;
  if (cols > 1 && t.stride(1) != 1) value_error(std::string(name) + " must have unit column stride");
  if (t.size(0) == 1) return 0;
  if (t.stride(0) < cols) value_error(std::string(name) + ": rows overlap");
  return t.stride(0);
}
void vector_of(const at::Tensor& t, const char* name, int64_t cols) {
  if (t.dim() != 1 || t.size(0) != cols || (cols > 1 && t.stride(0) != 1))
    value_error(std::string(name) + " must be contiguous [" + std::to_string(cols) + "]");
}
void stats_of(const at::Tensor& t, const char* name, int64_t rows) {
  if (t.scalar_type() != at::kFloat || t.dim() != 1 || t.size(0) != rows || !t.is_contiguous())
    value_error(std::string(name) + " must be contiguous fp32 [" + std::to_string(rows) + "]");
}
void* pointer(Maybe t) { return t ? t->data_ptr() : nullptr; }

// A given tensor was written: what autograd saved of it before counts as changed, as after torch's own in-place calls.
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

PyObject* wrapped(const std::optional<at::Tensor>& t) {
  if (!t) Py_RETURN_NONE;
  return THPVariable_Wrap(*t);
}

void want(Py_ssize_t n, Py_ssize_t given) {
  if (n != given) type_error("wrong number of arguments");
}

// layer_norm(x, weight, bias, eps, out, return_stats) -> y, or (y, mean, rstd)
PyObject* layer_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  try {
    want(6, n);
    const at::Tensor& x = tensor(a[0], "x");
    Maybe weight = maybe(a[1], "weight"), bias = maybe(a[2], "bias"), out = maybe(a[4], "out");
    const double eps = PyFloat_AsDouble(a[3]);
    if (eps == -1.0 && PyErr_Occurred()) throw python_error();
    const bool stats = truth(a[5]);
    const auto device = device_of({{"x", &x}, {"weight", weight}, {"bias", bias}, {"out", out}});
    if (x.dim() != 2) value_error("x must be [rows, cols]");
    const int64_t rows = x.size(0), cols = x.size(1);
    fwd_eb_layer_norm_params p = {};
    p.dtype = dtype_of(x, "x");
    p.x_stride = rows_of(x, "x", cols, -1);
    if (weight) {
      vector_of(*weight, "weight", cols);
      p.weight_dtype = dtype_of(*weight, "weight");
    }
    if (bias) {
      vector_of(*bias, "bias", cols);
      const int code = dtype_of(*bias, "bias");
      if (weight && code != p.weight_dtype) type_error("bias must have the weight's dtype");
      p.weight_dtype = code;
    }
    if (out) {
      if (out->scalar_type() != x.scalar_type()) type_error("out must have x's dtype");
      p.y_stride = rows_of(*out, "out", cols, rows);
    }
    c10::cuda::CUDAGuard guard(device);
    at::Tensor y = out ? *out : at::empty({rows, cols}, x.options());
    std::optional<at::Tensor> mean, rstd;
    if (stats) {
      const auto options = x.options().dtype(at::kFloat);
      mean = at::empty({rows}, options);
      rstd = at::empty({rows}, options);
      p.mean = static_cast<float*>(mean->data_ptr());
      p.rstd = static_cast<float*>(rstd->data_ptr());
    }
    p.x = x.data_ptr();
    p.rows = rows;
    p.cols = cols;
    p.weight = pointer(weight);
    p.bias = pointer(bias);
    p.eps = eps;
    p.y = y.data_ptr();
    const int rc = g_norm_forward(&p, c10::cuda::getCurrentCUDAStream(device).stream());
    if (rc) return PyLong_FromLong(rc);
    if (out) written(*out);
    PyObject* result = out ? Py_NewRef(a[4]) : THPVariable_Wrap(y);
    if (!stats) return result;
    return Py_BuildValue("(NNN)", result, wrapped(mean), wrapped(rstd));
  } catch (const Refused& r) {
    PyErr_SetString(r.type, r.text.c_str());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// layer_norm_backward(grad_y, x, mean, rstd, weight, grad_x, need_x, need_params, param dtype code or -1)
PyObject* layer_norm_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  try {
    want(9, n);
    const at::Tensor &gy = tensor(a[0], "grad_y"), &x = tensor(a[1], "x"), &mean = tensor(a[2], "mean"),
                     &rstd = tensor(a[3], "rstd");
    Maybe weight = maybe(a[4], "weight"), given = maybe(a[5], "grad_x");
    const bool need_x = truth(a[6]), need_params = truth(a[7]);
    const auto device = device_of({{"x", &x}, {"grad_y", &gy}, {"mean", &mean}, {"rstd", &rstd}, {"weight", weight},
                                   {"grad_x", given}});
    if (x.dim() != 2) value_error("x must be [rows, cols]");
    const int64_t rows = x.size(0), cols = x.size(1);
    fwd_eb_layer_norm_params p = {};
    p.dtype = dtype_of(x, "x");
    if (gy.scalar_type() != x.scalar_type() || (given && given->scalar_type() != x.scalar_type()))
      type_error("grad_y and grad_x must have x's dtype");
    if (given && !need_x) value_error("grad_x is given but need_x is False");
    p.x_stride = rows_of(x, "x", cols, -1);
    p.grad_y_stride = rows_of(gy, "grad_y", cols, rows);
    stats_of(mean, "mean", rows);
    stats_of(rstd, "rstd", rows);
    const int asked = (int)integer(a[8]);
    p.weight_dtype = asked < 0 ? FWD_EB_F32 : asked;
    if (weight) {
      vector_of(*weight, "weight", cols);
      p.weight_dtype = dtype_of(*weight, "weight");
    }
    if (given) p.grad_x_stride = rows_of(*given, "grad_x", cols, rows);
    c10::cuda::CUDAGuard guard(device);
    std::optional<at::Tensor> gx, gw, gb;
    if (need_x) gx = given ? *given : at::empty({rows, cols}, x.options());
    if (need_params) {
      const auto options = x.options().dtype(type_of(p.weight_dtype));
      gw = at::empty({cols}, options);
      gb = at::empty({cols}, options);
    }
    p.x = x.data_ptr();
    p.rows = rows;
    p.cols = cols;
    p.weight = pointer(weight);
    p.mean = static_cast<float*>(mean.data_ptr());
    p.rstd = static_cast<float*>(rstd.data_ptr());
    p.grad_y = gy.data_ptr();
    p.grad_x = gx ? gx->data_ptr() : nullptr;
    p.grad_weight = gw ? gw->data_ptr() : nullptr;
    p.grad_bias = gb ? gb->data_ptr() : nullptr;
    at::Tensor scratch;
    p.workspace_bytes = g_norm_workspace(&p);
    if (p.workspace_bytes) {
      scratch = at::empty({(int64_t)p.workspace_bytes}, x.options().dtype(at::kByte));
      p.workspace = scratch.data_ptr();
    }
    const int rc = g_norm_backward(&p, c10::cuda::getCurrentCUDAStream(device).stream());
    if (rc) return PyLong_FromLong(rc);
    if (given) written(*given);
    return Py_BuildValue("(NNN)", given ? Py_NewRef(a[5]) : wrapped(gx), wrapped(gw), wrapped(gb));
  } catch (const Refused& r) {
    PyErr_SetString(r.type, r.text.c_str());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// embedding_bag_backward(grad_out, table, indices, offsets, mode, fixed_len, per_sample_weights, include_last_offset,
//   padding_idx, row_lo, flags, winners, grad_table, grad dtype code or -1, accumulate, need_table, need_weights)
PyObject* embedding_bag_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  try {
    want(17, n);
    const at::Tensor &go = tensor(a[0], "grad_out"), &table = tensor(a[1], "table"), &indices = tensor(a[2], "indices");
    Maybe offsets = maybe(a[3], "offsets"), psw = maybe(a[6], "per_sample_weights"), winners = maybe(a[11], "winners"),
          given = maybe(a[12], "grad_table");
    const int mode = (int)integer(a[4]);
    const long long fixed = integer(a[5]);
    const bool last = truth(a[7]), accumulate = truth(a[14]), need_table = truth(a[15]), need_weights = truth(a[16]);
    const auto device = device_of({{"grad_out", &go}, {"table", &table}, {"indices", &indices}, {"offsets", offsets},
                                   {"per_sample_weights", psw}, {"winners", winners}, {"grad_table", given}});
    if (table.dim() != 2 || (table.size(1) > 1 && table.size(0) > 0 && table.stride(1) != 1))
      value_error("table must be 2-D with unit column stride");
    const int64_t rows = table.size(0), dim = table.size(1);
    if (dim > INT32_MAX) value_error("table has too many columns");
    if (!indices.is_contiguous()) value_error("indices must be contiguous");
    const int64_t count = indices.numel();
    const bool gather = mode == FWD_EB_MODE_GATHER;
    if (fixed < 0 || fixed > INT32_MAX) value_error("fixed_len must be a 32-bit number and not negative");
    int64_t bags = 0;
    if (gather) {
      bags = count;
      offsets = nullptr;
    } else if (fixed > 0) {
      bags = count / fixed;
      offsets = nullptr;
    } else {
      if (!offsets) value_error("offsets is None and fixed_len is 0");
      if (offsets->scalar_type() != indices.scalar_type() || !offsets->is_contiguous())
        value_error("offsets must be a contiguous tensor of the indices' dtype");
      bags = offsets->numel() - (last ? 1 : 0);
    }
    if (bags < 0) value_error("offsets is empty, include_last_offset wants an entry");
    if (accumulate && !given) value_error("accumulate=True adds to a grad_table that the caller gives");
    if (!need_table && !need_weights) value_error("neither gradient is asked for");
    if (given && !need_table) value_error("grad_table is given but need_table is False");
    const int go_code = dtype_of(go, "grad_out"), table_code = dtype_of(table, "table");
    if (go_code == FWD_EB_BF16) type_error("grad_out: unsupported dtype BFloat16");
    if (table_code == FWD_EB_BF16) type_error("table: unsupported dtype BFloat16");
    if (indices.scalar_type() != at::kInt && indices.scalar_type() != at::kLong)
      type_error(std::string("indices: unsupported dtype ") + c10::toString(indices.scalar_type()));
    if (psw && (psw->scalar_type() != at::kFloat || !psw->is_contiguous() || psw->numel() != count))
      value_error("per_sample_weights must be contiguous fp32, one per index");
    int64_t win_stride = 0;
    if (winners) {
      if (winners->scalar_type() != at::kFloat || winners->dim() != 3 || winners->size(0) != bags ||
          winners->size(1) != dim || winners->size(2) != 2)
        value_error("winners must be fp32 [" + std::to_string(bags) + ", " + std::to_string(dim) + ", 2]");
      if (bags > 0 && dim > 0 &&
          (winners->stride(2) != 1 || (dim > 1 && winners->stride(1) != 2) ||
           (bags > 1 && (winners->stride(0) % 2 != 0 || winners->stride(0) < 2 * dim))))
        value_error("winners must be rows of adjacent pairs");
      win_stride = bags > 1 ? winners->stride(0) / 2 : 0;
    }
    const int64_t go_stride = rows_of(go, "grad_out", dim, bags);
    const int asked = (int)integer(a[13]);
    int gt_code = asked < 0 ? table_code : asked;
    int64_t gt_stride = 0;
    if (given) {
      gt_code = dtype_of(*given, "grad_table");
      gt_stride = rows_of(*given, "grad_table", dim, rows);
    }
    if (need_table && gt_code == FWD_EB_BF16) type_error("grad_table: unsupported dtype BFloat16");

    c10::cuda::CUDAGuard guard(device);
    std::optional<at::Tensor> gt, gw;
    if (need_table) gt = given ? *given : at::empty({rows, dim}, table.options().dtype(type_of(gt_code)));
    if (need_weights) gw = at::empty({count}, table.options().dtype(at::kFloat));
    // where nothing is to be computed an empty tensor has no address to hand over
    if ((rows > 0 && need_table) || (count > 0 && need_weights)) {
      fwd_eb_backward_params p = {};
      fwd_eb_params& f = p.fwd;
      f.table = table.data_ptr();
      f.table_dtype = table_code;
      f.dim = (int32_t)dim;
      f.num_rows = rows;
      f.row_lo = integer(a[9]);
      f.table_stride = rows > 1 ? table.stride(0) : 0;
      f.indices = indices.data_ptr();
      f.offsets = pointer(offsets);
      f.index_dtype = indices.scalar_type() == at::kLong ? FWD_EB_I64 : FWD_EB_I32;
      f.fixed_len = gather ? 0 : (int32_t)fixed;
      f.num_indices = count;
      f.num_bags = gather ? 0 : bags;
      f.per_sample_weights = static_cast<const float*>(pointer(psw));
      f.mode = mode;
      f.include_last_offset = last;
      f.padding_idx = integer(a[8]);
      f.flags = (uint32_t)integer(a[10]);
      p.grad_out = go.data_ptr();
      p.grad_out_dtype = go_code;
      p.grad_table_dtype = need_table ? gt_code : FWD_EB_F32;
      p.grad_out_stride = go_stride;
      p.grad_table = gt ? gt->data_ptr() : nullptr;
      p.grad_table_stride = gt_stride;
      p.grad_weights = gw ? static_cast<float*>(gw->data_ptr()) : nullptr;
      p.winners = pointer(winners);
      p.winners_stride = win_stride;
      p.flags = accumulate ? FWD_EB_BACKWARD_ACCUMULATE : 0;
      at::Tensor scratch;
      p.workspace_bytes = g_backward_workspace(&p);
      if (p.workspace_bytes) {
        scratch = at::empty({(int64_t)p.workspace_bytes}, table.options().dtype(at::kByte));
        p.workspace = scratch.data_ptr();
      }
      const int rc = g_backward(&p, c10::cuda::getCurrentCUDAStream(device).stream());
      if (rc) return PyLong_FromLong(rc);
    }
    if (given) written(*given);
    return Py_BuildValue("(NN)", given ? Py_NewRef(a[12]) : wrapped(gt), wrapped(gw));
  } catch (const Refused& r) {
    PyErr_SetString(r.type, r.text.c_str());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// current_stream(device ordinal, refuse a capture) -> the stream's address
PyObject* current_stream(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  try {
    want(2, n);
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)integer(a[0])).stream();
    if (truth(a[1])) {
      cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
      if (cudaStreamIsCapturing(stream, &status) != cudaSuccess || status != cudaStreamCaptureStatusNone)
        throw Refused{PyExc_RuntimeError, "a step that is captured needs capturable=True"};
    }
    return PyLong_FromVoidPtr(stream);
  } catch (const Refused& r) {
    PyErr_SetString(r.type, r.text.c_str());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// touched(list of tensors): each was written
PyObject* touched(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  try {
    want(1, n);
    if (!PyList_Check(a[0])) type_error("touched takes a list");
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(a[0]); ++i) written(tensor(PyList_GET_ITEM(a[0], i), "a tensor"));
    Py_RETURN_NONE;
  } catch (const Refused& r) {
    PyErr_SetString(r.type, r.text.c_str());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// bind(addresses of the five entry points above, in their order)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 5) {
    PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
    return nullptr;
  }
  void* at[5];
  for (int i = 0; i < 5; ++i) {
    at[i] = PyLong_AsVoidPtr(a[i]);
    if (!at[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null address");
      return nullptr;
    }
  }
  g_norm_forward = reinterpret_cast<decltype(g_norm_forward)>(at[0]);
  g_norm_backward = reinterpret_cast<decltype(g_norm_backward)>(at[1]);
  g_norm_workspace = reinterpret_cast<decltype(g_norm_workspace)>(at[2]);
  g_backward = reinterpret_cast<decltype(g_backward)>(at[3]);
  g_backward_workspace = reinterpret_cast<decltype(g_backward_workspace)>(at[4]);
  Py_RETURN_NONE;
}

#define FWD_EB_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&name)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {
    FWD_EB_METHOD(layer_norm), FWD_EB_METHOD(layer_norm_backward), FWD_EB_METHOD(embedding_bag_backward),
    FWD_EB_METHOD(current_stream), FWD_EB_METHOD(touched), FWD_EB_METHOD(bind), {nullptr, nullptr, 0, nullptr},
};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_training_ops", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__training_ops() { return PyModule_Create(&g_module); }
