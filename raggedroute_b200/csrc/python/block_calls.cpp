// The short way from Python to the expert-block entry points. A call for one
// token is a few microseconds of GPU work, less than the checks of up to a dozen
// tensors in Python and the conversions of ctypes take (host time of a call:
// unpermute_norm 12.5 us that way, 4.2 this way; grouped_gemm_int8 10.7 and 3.2).
// Each function here takes the tensors of the Python function of the same name
// (expert_block.py), makes the same checks on them and calls the entry point on
// the current stream. It returns True when the call is launched, raises when the
// entry point refuses it, and returns False, having done nothing, when a check
// fails or the tensors are on another device than the current one: the Python
// function then makes the call itself, or names what is wrong.
#include <Python.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <initializer_list>
#include <utility>

#include "../../../include/raggedroute_b200.h"

namespace {

PyObject* error_class = nullptr;  // RaggedRouteError(code, cuda_error, message, op)

PyObject* finish(rr_status s, const char* op) {
  if (s.code == RR_SUCCESS) Py_RETURN_TRUE;
  if (error_class == nullptr) Py_RETURN_FALSE;
  PyObject* e = PyObject_CallFunction(error_class, "iiss", s.code, s.cuda_error,
                                      s.message != nullptr ? s.message : "error", op);
  if (e != nullptr) {
    PyErr_SetObject(error_class, e);
    Py_DECREF(e);
  }
  return nullptr;
}

// The arguments of one call. A failed check clears `ok`; nothing is launched then.
class Args {
 public:
  Args(PyObject* const* args, Py_ssize_t count, Py_ssize_t expected)
      : args_(args), ok_(count == expected) {}

  bool ok() const { return ok_; }

  // Argument i as a CUDA tensor of `dims` dimensions: its sizes and device
  // become the call's.
  const at::Tensor* tensor(int i, int dims) {
    if (!ok_ || !THPVariable_Check(args_[i])) return fail();
    const at::Tensor& t = THPVariable_Unpack(args_[i]);
    if (t.dim() != dims || !t.is_cuda()) return fail();
    for (const int64_t n : t.sizes()) {
      if (n > INT32_MAX) return fail();
    }
    if (device_ < 0) device_ = t.device().index();
    return &t;
  }

  // The data type of the rows: RR_DTYPE_*.
  int dtype(const at::Tensor* t) {
    if (t != nullptr && t->scalar_type() == at::kFloat) return RR_DTYPE_FP32;
    if (t != nullptr && t->scalar_type() == at::kBFloat16) return RR_DTYPE_BF16;
    ok_ = false;
    return RR_DTYPE_FP32;
  }

  // The address of argument i: a contiguous tensor of this type and shape on the
  // call's device, or None.
  void* data(int i, at::ScalarType type, std::initializer_list<int64_t> shape) {
    if (!ok_ || args_[i] == Py_None) return nullptr;
    if (!THPVariable_Check(args_[i])) return ok_ = false, nullptr;
    const at::Tensor& t = THPVariable_Unpack(args_[i]);
    if (t.scalar_type() != type || !t.is_cuda() || t.device().index() != device_ ||
        t.sizes() != at::IntArrayRef(shape) || !t.is_contiguous()) {
      return ok_ = false, nullptr;
    }
    return t.data_ptr();
  }
  template <typename P>
  P* data_as(int i, at::ScalarType type, std::initializer_list<int64_t> shape) {
    return static_cast<P*>(data(i, type, shape));
  }

  int integer(int i) {
    const long v = ok_ ? PyLong_AsLong(args_[i]) : 0;
    if (v < INT32_MIN || v > INT32_MAX || (v == -1 && PyErr_Occurred())) ok_ = false;
    return static_cast<int>(v);
  }
  float real(int i) {
    const double v = ok_ ? PyFloat_AsDouble(args_[i]) : 0.0;
    if (v == -1.0 && PyErr_Occurred()) ok_ = false;
    return static_cast<float>(v);
  }

  // Adds argument i, None or any contiguous tensor, as the workspace.
  void workspace(int i) {
    if (!ok_ || args_[i] == Py_None) return;
    if (!THPVariable_Check(args_[i])) {
      ok_ = false;
      return;
    }
    const at::Tensor& t = THPVariable_Unpack(args_[i]);
    if (!t.is_cuda() || t.device().index() != device_ || !t.is_contiguous()) {
      ok_ = false;
      return;
    }
    context_.workspace = t.data_ptr();
    context_.workspace_bytes = t.nbytes();
  }

  // Runs call(context) on the current stream, without the interpreter's lock.
  template <typename Call>
  PyObject* run(const char* op, Call&& call) {
    int current = -1;
    if (ok_ && (cudaGetDevice(&current) != cudaSuccess || current != device_)) ok_ = false;
    if (!ok_) {
      PyErr_Clear();
      Py_RETURN_FALSE;
    }
    context_.stream =
        c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device_)).stream();
    rr_status s;
    Py_BEGIN_ALLOW_THREADS
    s = call(&context_);
    Py_END_ALLOW_THREADS
    return finish(s, op);
  }

 private:
  std::nullptr_t fail() {
    ok_ = false;
    return nullptr;
  }

  PyObject* const* args_;
  bool ok_;
  int device_ = -1;
  rr_context context_{};
};

// Sizes of the gated operators from x [R, K] (argument 0) and Wg [E, K, N].
struct Gated {
  int dtype = 0, rows = 0, hidden = 0, experts = 0, output = 0;
  at::ScalarType type = at::kFloat;
  void *x = nullptr, *wg = nullptr, *wu = nullptr;
  int32_t* offsets = nullptr;

  explicit Gated(Args& in) {
    const at::Tensor *tx = in.tensor(0, 2), *tw = in.tensor(1, 3);
    if (!in.ok()) return;
    dtype = in.dtype(tx);
    type = tx->scalar_type();
    rows = static_cast<int>(tx->size(0));
    hidden = static_cast<int>(tx->size(1));
    experts = static_cast<int>(tw->size(0));
    output = static_cast<int>(tw->size(2));
    x = in.data(0, type, {rows, hidden});
    wg = in.data(1, type, {experts, hidden, output});
    wu = in.data(2, type, {experts, hidden, output});
    offsets = in.data_as<int32_t>(3, at::kInt, {experts + 1});
  }
};

// Inputs of the combine: y_permuted, route_pos, route_weights, residual,
// post_gamma, gate, pre_gamma are arguments 0 to 6.
struct Norm {
  int dtype = 0, tokens = 0, top_k = 0, output = 0;
  int64_t routes = 0;
  at::ScalarType type = at::kFloat;
  void *y = nullptr, *residual = nullptr;
  int32_t* pos = nullptr;
  float *weights = nullptr, *post = nullptr, *gate = nullptr, *pre = nullptr;

  explicit Norm(Args& in) {
    const at::Tensor *tr = in.tensor(3, 2), *tp = in.tensor(1, 2);
    if (!in.ok()) return;
    dtype = in.dtype(tr);
    type = tr->scalar_type();
    tokens = static_cast<int>(tr->size(0));
    output = static_cast<int>(tr->size(1));
    top_k = static_cast<int>(tp->size(1));
    routes = static_cast<int64_t>(tokens) * top_k;
    y = in.data(0, type, {routes, output});
    pos = in.data_as<int32_t>(1, at::kInt, {tokens, top_k});
    weights = in.data_as<float>(2, at::kFloat, {tokens, top_k});
    residual = in.data(3, type, {tokens, output});
    post = in.data_as<float>(4, at::kFloat, {output});
    gate = in.data_as<float>(5, at::kFloat, {output});
    pre = in.data_as<float>(6, at::kFloat, {output});
  }
};

PyObject* grouped_gated_gemm(Args& in) {
  const Gated g(in);
  void* h = in.data(4, g.type, {g.rows, g.output});
  float* gate_up = in.data_as<float>(5, at::kFloat, {g.rows, 2LL * g.output});
  const int act = in.integer(6);
  in.workspace(7);
  return in.run("grouped_gated_gemm", [&](const rr_context* ctx) {
    return rr_grouped_gated_gemm(g.x, g.wg, g.wu, g.offsets, h, gate_up, g.rows, g.experts,
                                 g.hidden, g.output, act, g.dtype, ctx);
  });
}

PyObject* grouped_gated_gemm_backward(Args& in) {
  const Gated g(in);
  float* gate_up = in.data_as<float>(4, at::kFloat, {g.rows, 2LL * g.output});
  void* dh = in.data(5, g.type, {g.rows, g.output});
  void* dx = in.data(6, g.type, {g.rows, g.hidden});
  void* dwg = in.data(7, g.type, {g.experts, g.hidden, g.output});
  void* dwu = in.data(8, g.type, {g.experts, g.hidden, g.output});
  const int act = in.integer(9);
  in.workspace(10);
  return in.run("grouped_gated_gemm_backward", [&](const rr_context* ctx) {
    return rr_grouped_gated_gemm_backward(g.x, g.wg, g.wu, g.offsets, gate_up, dh, dx, dwg, dwu,
                                          g.rows, g.experts, g.hidden, g.output, act, g.dtype, ctx);
  });
}

PyObject* quantize_rows_int8(Args& in) {
  const at::Tensor* t = in.tensor(0, 2);
  const int dtype = in.dtype(t);
  const int rows = in.ok() ? static_cast<int>(t->size(0)) : 0;
  const int hidden = in.ok() ? static_cast<int>(t->size(1)) : 0;
  void* x = in.ok() ? in.data(0, t->scalar_type(), {rows, hidden}) : nullptr;
  int8_t* xq = in.data_as<int8_t>(1, at::kChar, {rows, rr_int8_row_stride(hidden)});
  float* scale = in.data_as<float>(2, at::kFloat, {rows});
  return in.run("quantize_rows_int8", [&](const rr_context* ctx) {
    return rr_quantize_rows_int8(x, xq, scale, rows, hidden, dtype, ctx);
  });
}

PyObject* grouped_gemm_int8(Args& in) {
  const at::Tensor *tx = in.tensor(0, 2), *tw = in.tensor(2, 3), *ty = in.tensor(5, 2);
  const int dtype = in.dtype(ty);
  const int rows = in.ok() ? static_cast<int>(tx->size(0)) : 0;
  const int stride = in.ok() ? static_cast<int>(tx->size(1)) : 0;
  const int experts = in.ok() ? static_cast<int>(tw->size(0)) : 0;
  const int output = in.ok() ? static_cast<int>(tw->size(1)) : 0;
  // A row has to be a row stride long; -1 fits no tensor.
  const int row = rr_int8_row_stride(stride) == stride ? stride : -1;
  int8_t* xq = in.data_as<int8_t>(0, at::kChar, {rows, row});
  float* x_scale = in.data_as<float>(1, at::kFloat, {rows});
  int8_t* wq = in.data_as<int8_t>(2, at::kChar, {experts, output, row});
  float* w_scale = in.data_as<float>(3, at::kFloat, {experts, output});
  int32_t* offsets = in.data_as<int32_t>(4, at::kInt, {experts + 1});
  void* y = in.ok() ? in.data(5, ty->scalar_type(), {rows, output}) : nullptr;
  return in.run("grouped_gemm_int8", [&](const rr_context* ctx) {
    return rr_grouped_gemm_int8(xq, x_scale, wq, w_scale, offsets, y, rows, experts, stride, output,
                                dtype, ctx);
  });
}

PyObject* unpermute_norm(Args& in) {
  const Norm n(in);
  void* out = in.data(7, n.type, {n.tokens, n.output});
  void* normed = in.data(8, n.type, {n.tokens, n.output});
  float* inv_rms = in.data_as<float>(9, at::kFloat, {n.tokens, 2});
  const float eps = in.real(10), scale = in.real(11);
  return in.run("unpermute_norm", [&](const rr_context* ctx) {
    return rr_unpermute_norm(n.y, n.pos, n.weights, n.residual, n.post, n.gate, n.pre, out, normed,
                             inv_rms, eps, scale, n.tokens, n.top_k, n.output, n.dtype, ctx);
  });
}

PyObject* unpermute_norm_backward(Args& in) {
  const Norm n(in);
  float* inv_rms = in.data_as<float>(7, at::kFloat, {n.tokens, 2});
  void* d_out = in.data(8, n.type, {n.tokens, n.output});
  void* d_normed = in.data(9, n.type, {n.tokens, n.output});
  void* d_residual = in.data(10, n.type, {n.tokens, n.output});
  void* d_y = in.data(11, n.type, {n.routes, n.output});
  float* d_weights = in.data_as<float>(12, at::kFloat, {n.tokens, n.top_k});
  float* d_post = in.data_as<float>(13, at::kFloat, {n.output});
  float* d_gate = in.data_as<float>(14, at::kFloat, {n.output});
  float* d_pre = in.data_as<float>(15, at::kFloat, {n.output});
  const float scale = in.real(16);
  in.workspace(17);
  return in.run("unpermute_norm_backward", [&](const rr_context* ctx) {
    return rr_unpermute_norm_backward(n.y, n.pos, n.weights, n.residual, n.post, n.gate, n.pre,
                                      inv_rms, d_out, d_normed, d_residual, d_y, d_weights, d_post,
                                      d_gate, d_pre, scale, n.tokens, n.top_k, n.output, n.dtype,
                                      ctx);
  });
}

// A function of `count` arguments as a Python one. An exception of the tensor
// library (a tensor without storage, say) is a failed check like the others.
template <auto kFunction, int kCount>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t count) {
  try {
    Args in(args, count, kCount);
    if (!in.ok()) Py_RETURN_FALSE;
    return kFunction(in);
  } catch (...) {
    PyErr_Clear();
    Py_RETURN_FALSE;
  }
}

PyObject* set_error(PyObject*, PyObject* cls) {
  Py_INCREF(cls);
  Py_XSETREF(error_class, cls);
  Py_RETURN_NONE;
}

template <auto kFunction, int kCount>
PyCFunction fast() {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(entry<kFunction, kCount>));
}

PyMethodDef methods[] = {
    {"grouped_gated_gemm", fast<grouped_gated_gemm, 8>(), METH_FASTCALL, nullptr},
    {"grouped_gated_gemm_backward", fast<grouped_gated_gemm_backward, 11>(), METH_FASTCALL,
     nullptr},
    {"quantize_rows_int8", fast<quantize_rows_int8, 3>(), METH_FASTCALL, nullptr},
    {"grouped_gemm_int8", fast<grouped_gemm_int8, 6>(), METH_FASTCALL, nullptr},
    {"unpermute_norm", fast<unpermute_norm, 12>(), METH_FASTCALL, nullptr},
    {"unpermute_norm_backward", fast<unpermute_norm_backward, 18>(), METH_FASTCALL, nullptr},
    {"set_error", set_error, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_block_calls", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__block_calls() { return PyModule_Create(&module); }
