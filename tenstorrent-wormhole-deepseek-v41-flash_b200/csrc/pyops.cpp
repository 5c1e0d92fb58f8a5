// Native half of dsmoe/ops.py: argument checks, output allocation and the C ABI call of each operator in one
// step (module dsmoe._ops). A small call of these operators takes 2 to 4 us on the GPU; checks and allocations
// written in Python cost 10 to 17 us a call, here 4 to 6. The compute is libdsmoe.so's, through include/dsmoe.h.
//
// Errors: ValueError / TypeError for arguments (the messages name the operator), dsmoe.DsmoeError for a failing
// entry point, torch's own exceptions (out of memory) as they are. No C++ exception leaves a function. The gradients
// of dispatch and combine are autograd functions of their own here: backward runs without Python.
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/utils/tensor_dtypes.h>

#include <ATen/cuda/EmptyTensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <c10/core/DefaultDtype.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <optional>
#include <sstream>
#include <string>
#include <unordered_set>
#include <vector>

#include "../../include/dsmoe.h"

namespace {

using at::Tensor;

constexpr int64_t kBlock = 128;
constexpr int64_t kMaxExperts = 1024, kMaxTopk = 64, kMaxRow = 16384, kMaxK = 131071;

PyObject* g_error = nullptr;  // dsmoe._lib.DsmoeError

// A refusal, caught at the entry points and raised in Python. type: nullptr with code DSMOE_OK where the Python
// error is set already, nullptr with another code for a failing entry point.
struct Refused {
  PyObject* type;
  std::string what;
  int code = DSMOE_OK;
};

template <typename... A>
[[noreturn]] void refuse(PyObject* type, const char* name, const A&... a) {
  std::ostringstream s;
  s << name << ": ";
  (s << ... << a);
  throw Refused{type, s.str()};
}
template <typename... A>
void value_check(bool ok, const char* name, const A&... a) {
  if (!ok) refuse(PyExc_ValueError, name, a...);
}
template <typename... A>
void type_check(bool ok, const char* name, const A&... a) {
  if (!ok) refuse(PyExc_TypeError, name, a...);
}

const Tensor& tensor(const char* name, PyObject* o) {
  type_check(THPVariable_Check(o), name, "expected a tensor, got ", Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}
// None -> an undefined tensor
Tensor maybe(const char* name, PyObject* o) { return o == Py_None ? Tensor() : tensor(name, o); }

// All on one GPU, and none with a forward-mode tangent, which a kernel would lose without a word.
void same_device(const char* name, std::initializer_list<const Tensor*> ts) {
  const Tensor& a = **ts.begin();
  if (c10::AutogradState::get_tls_state().get_fw_grad_mode())
    for (const Tensor* t : ts)
      value_check(!t->defined() || !t->_fw_grad(0).defined(), name, "has no forward-mode derivative: pass primals without tangents");
  for (const Tensor* t : ts) {
    if (!t->defined()) continue;
    value_check(t->is_cuda(), name, "dsmoe kernels take CUDA tensors only, got ", t->sizes(), " on ", t->device());
    value_check(t->get_device() == a.get_device(), name, "tensors on ", a.device(), " and ", t->device());
  }
}
void no_grad(const char* name, std::initializer_list<const Tensor*> ts) {
  if (!c10::GradMode::is_enabled()) return;
  for (const Tensor* t : ts)
    value_check(!t->defined() || !t->requires_grad(), name,
                "has no gradient: detach its inputs or call it under torch.no_grad()");
}
void want(const char* name, const Tensor& t, const char* what, at::ScalarType dtype, at::IntArrayRef shape) {
  type_check(t.scalar_type() == dtype, name, what, " must be ", dtype, ", got ", t.scalar_type());
  value_check(t.sizes() == shape, name, what, " must be ", shape, ", got ", t.sizes());
}

int float_code(const char* name, const Tensor& t, const char* what) {
  if (t.scalar_type() == at::kBFloat16) return DSMOE_DTYPE_BF16;
  if (t.scalar_type() == at::kFloat) return DSMOE_DTYPE_F32;
  refuse(PyExc_TypeError, name, what, " must be bfloat16 or float32, got ", t.scalar_type());
}

Tensor empty(const Tensor& like, at::IntArrayRef shape, at::ScalarType dtype) {
  return Tensor(at::detail::empty_cuda(shape, dtype, like.device(), std::nullopt));
}
// Whether the memory does not hold the values: views that are conjugated or negated when they are read (or zeros
// without memory), which are contiguous all the same.
bool lazy(const Tensor& t) {
  return t.key_set().has_any(
      c10::DispatchKeySet({c10::DispatchKey::Conjugate, c10::DispatchKey::Negative, c10::DispatchKey::ZeroTensor}));
}
// contiguous, its values in memory and 16-byte aligned; aligned: whether the kernel wants the alignment
Tensor dense(const Tensor& t, bool aligned = true) {
  if (lazy(t)) {
    const Tensor r = t._is_zerotensor() ? at::zeros(t.sizes(), t.options()) : t.resolve_conj().resolve_neg();
    return r.is_contiguous() ? r : r.contiguous();
  }
  Tensor c = t.is_contiguous() ? t : t.contiguous();
  return aligned && reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 ? c.clone() : c;
}
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
// A caller's tensor that a kernel writes: autograd refuses a backward pass that saved what stood there.
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// The call on t's device and that device's current stream.
template <typename F>
void run(const Tensor& t, F call) {
  const auto i = static_cast<c10::DeviceIndex>(t.get_device());
  std::optional<c10::cuda::CUDAGuard> guard;
  if (c10::cuda::current_device() != i) guard.emplace(i);
  const int rc = call(static_cast<void*>(c10::cuda::getCurrentCUDAStream(i).stream()));
  if (rc != DSMOE_OK) throw Refused{nullptr, dsmoe_last_error(), rc};
}

PyObject* wrap(const Tensor& t) {
  if (t.defined()) return THPVariable_Wrap(t);
  Py_RETURN_NONE;
}
PyObject* tuple(std::initializer_list<const Tensor*> ts) {
  PyObject* r = PyTuple_New(static_cast<Py_ssize_t>(ts.size()));
  Py_ssize_t i = 0;
  for (const Tensor* t : ts) PyTuple_SET_ITEM(r, i++, wrap(*t));
  return r;
}

// f(args) with refusals turned into Python errors
template <typename F>
PyObject* guarded(PyObject* const* args, Py_ssize_t n, Py_ssize_t expected, F f) {
  HANDLE_TH_ERRORS
  if (n != expected) {
    PyErr_Format(PyExc_TypeError, "dsmoe._ops: %zd arguments, expected %zd", n, expected);
    return nullptr;
  }
  try {
    return f(args);
  } catch (const Refused& r) {
    if (r.type) {
      PyErr_SetString(r.type, r.what.c_str());
    } else if (r.code != DSMOE_OK) {
      PyObject* e = PyObject_CallFunction(g_error ? g_error : PyExc_RuntimeError, "is", r.code, r.what.c_str());
      if (e) {
        PyErr_SetObject(reinterpret_cast<PyObject*>(Py_TYPE(e)), e);
        Py_DECREF(e);
      }
    }
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// fmt -> dtype code, and the outputs [..., n] in 8 bits with their scales
int quant_out(const char* name, PyObject* fmt, bool pow2, const Tensor& like, int64_t n, Tensor& q, Tensor& s) {
  Py_ssize_t len = 0;
  const char* f = PyUnicode_Check(fmt) ? PyUnicode_AsUTF8AndSize(fmt, &len) : "";
  const bool fp8 = f && std::string_view(f, len) == "fp8", int8 = f && std::string_view(f, len) == "int8";
  PyErr_Clear();
  value_check(fp8 || int8, name, "fmt must be one of ['fp8', 'int8']");
  value_check(!pow2 || fp8, name, "power-of-2 scales (scale_fmt) are for fmt 'fp8'");
  value_check(n > 0 && n <= kMaxRow, name, "rows of ", n, " values (1..", kMaxRow, ")");
  value_check(int8 || n % kBlock == 0, name, "fmt 'fp8' needs rows of a multiple of ", kBlock, " values, got ", n);
  c10::SmallVector<int64_t, 6> shape(like.sizes().begin(), like.sizes().end() - 1);
  if (fp8) shape.push_back(n / kBlock);
  s = empty(like, shape, at::kFloat);
  if (fp8) shape.back() = n;
  else shape.push_back(n);
  q = empty(like, shape, fp8 ? at::kFloat8_e4m3fn : at::kChar);
  return fp8 ? DSMOE_DTYPE_E4M3 : DSMOE_DTYPE_I8;
}

// x, weight, residual, eps, fmt, pow2, normed, inplace -> (q, s, residual, normed)
PyObject* rms_norm_quant(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(args, n, 8, [](PyObject* const* args) -> PyObject* {
    const char* name = "rms_norm_quant";
    const Tensor &x0 = tensor(name, args[0]), &w0 = tensor(name, args[1]);
    const Tensor r0 = maybe(name, args[2]);
    const double eps = PyFloat_AsDouble(args[3]);
    if (PyErr_Occurred()) throw Refused{nullptr, ""};
    const bool pow2 = args[5] == Py_True, normed = args[6] == Py_True, inplace = args[7] == Py_True;
    same_device(name, {&x0, &w0, &r0});
    no_grad(name, {&x0, &w0, &r0});
    const int dt = float_code(name, x0, "x"), wdt = float_code(name, w0, "weight");
    value_check(x0.dim() >= 1, name, "x must be [..., hidden]");
    const int64_t h = x0.size(-1);
    want(name, w0, "weight", w0.scalar_type(), {h});
    if (r0.defined()) want(name, r0, "residual", x0.scalar_type(), x0.sizes());
    value_check(!inplace || (r0.defined() && r0.is_contiguous() && !lazy(r0)), name,
                "inplace needs a contiguous residual that is no conjugate or negative view");
    Tensor q, s, out, y;
    const int code = quant_out(name, args[4], pow2, x0, h, q, s);
    const Tensor x = dense(x0), w = dense(w0), r = r0.defined() ? dense(r0) : r0;
    if (r.defined()) out = inplace ? r : empty(x0, x0.sizes(), x0.scalar_type());
    if (normed) y = empty(x0, x0.sizes(), x0.scalar_type());
    if (x.numel()) {
      run(x, [&](void* st) {
        return dsmoe_rms_norm_quant(ptr(x), dt, ptr(r), ptr(w), wdt, x.numel() / h, h, static_cast<float>(eps), code, pow2,
                                    ptr(q), static_cast<float*>(ptr(s)), ptr(out), ptr(y), st);
      });
      if (inplace && out.data_ptr() == r0.data_ptr()) written(r0);
      else if (inplace) r0.copy_(out);  // it was not 16-byte aligned
    }
    return tuple({&q, &s, inplace ? &r0 : &out, &y});
  });
}

// gu, row_weight, limit, fmt, pow2 -> (q, s)
PyObject* swiglu_quant(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(args, n, 5, [](PyObject* const* args) -> PyObject* {
    const char* name = "swiglu_quant";
    const Tensor& g0 = tensor(name, args[0]);
    Tensor wr = maybe(name, args[1]);
    const double limit = PyFloat_AsDouble(args[2]);
    if (PyErr_Occurred()) throw Refused{nullptr, ""};
    const bool pow2 = args[4] == Py_True;
    same_device(name, {&g0, &wr});
    no_grad(name, {&g0, &wr});
    const int dt = float_code(name, g0, "gu");
    value_check(g0.dim() >= 1 && g0.size(-1) % 2 == 0, name, "gu must be [..., 2 * inter], got ", g0.sizes());
    value_check(limit > 0, name, "limit must be positive, got ", limit);
    if (wr.defined()) {
      want(name, wr, "row_weight", at::kFloat, g0.sizes().slice(0, g0.dim() - 1));
      wr = dense(wr, false);
    }
    const int64_t inter = g0.size(-1) / 2;
    Tensor q, s;
    const int code = quant_out(name, args[3], pow2, g0, inter, q, s);
    const Tensor g = dense(g0);
    if (g.numel())
      run(g, [&](void* st) {
        return dsmoe_swiglu_quant(ptr(g), dt, static_cast<float*>(ptr(wr)), g.numel() / (2 * inter), inter,
                                  static_cast<float>(limit), code, pow2, ptr(q), static_cast<float*>(ptr(s)), st);
      });
    return tuple({&q, &s});
  });
}

// a, a_s, b, b_s, offsets (None: one product), out_dtype, out -> out
PyObject* int8_product(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(args, n, 7, [](PyObject* const* args) -> PyObject* {
    const bool grouped = args[4] != Py_None;
    const char* name = grouped ? "int8_grouped_gemm" : "int8_gemm";
    const Tensor &a0 = tensor(name, args[0]), &as0 = tensor(name, args[1]), &b0 = tensor(name, args[2]),
                 &bs0 = tensor(name, args[3]);
    Tensor off = maybe(name, args[4]), out = maybe(name, args[6]);
    same_device(name, {&a0, &as0, &b0, &bs0, &off, &out});
    no_grad(name, {&as0, &bs0, &out});
    type_check(a0.scalar_type() == at::kChar && b0.scalar_type() == at::kChar, name, "a and b must be int8, got ",
               a0.scalar_type(), ", ", b0.scalar_type());
    if (grouped) {
      value_check(b0.dim() == 3 && a0.dim() == 2, name, "a must be [rows, K] and b [E, N, K], got ", a0.sizes(), ", ", b0.sizes());
      value_check(b0.size(0) > 0 && b0.size(0) <= kMaxExperts, name, b0.size(0), " experts (1..", kMaxExperts, ")");
      want(name, off, "offsets", at::kInt, {b0.size(0) + 1});
      off = dense(off, false);
    } else {
      value_check(b0.dim() == 2 && a0.dim() >= 1, name, "b must be [N, K], got ", b0.sizes());
    }
    const int64_t K = a0.size(-1), N = b0.size(-2);
    value_check(b0.size(-1) == K && K > 0 && K <= kMaxK && K % 16 == 0, name, "a ", a0.sizes(), " and b ", b0.sizes(),
                " need one K, a multiple of 16, at most ", kMaxK);
    want(name, as0, "a_s", at::kFloat, a0.sizes().slice(0, a0.dim() - 1));
    want(name, bs0, "b_s", at::kFloat, b0.sizes().slice(0, b0.dim() - 1));
    type_check(args[5] == Py_None || THPDtype_Check(args[5]), name, "out_dtype must be a torch.dtype");
    c10::SmallVector<int64_t, 6> shape(a0.sizes().begin(), a0.sizes().end());
    shape.back() = N;
    at::ScalarType dt = args[5] == Py_None ? c10::get_default_dtype_as_scalartype()
                                           : reinterpret_cast<THPDtype*>(args[5])->scalar_type;
    if (out.defined()) {
      type_check(args[5] == Py_None || dt == out.scalar_type(), name, "out is ", out.scalar_type(), ", out_dtype ", dt);
      dt = out.scalar_type();
      value_check(out.sizes() == at::IntArrayRef(shape) && out.is_contiguous() && !lazy(out), name, "out must be a contiguous ",
                  at::IntArrayRef(shape), " tensor and no conjugate or negative view");
    }
    type_check(dt == at::kFloat || dt == at::kBFloat16, name, "output dtype must be bfloat16 or float32, got ", dt);
    if (!out.defined()) out = empty(a0, shape, dt);
    const int64_t M = a0.numel() / K;
    if (M && N) {
      if (args[6] != Py_None) written(out);
      const Tensor a = dense(a0), b = dense(b0), as = dense(as0, false), bs = dense(bs0, false);
      const int code = dt == at::kFloat ? DSMOE_DTYPE_F32 : DSMOE_DTYPE_BF16;
      run(a, [&](void* st) {
        const auto* pa = static_cast<const int8_t*>(ptr(a));
        const auto* pb = static_cast<const int8_t*>(ptr(b));
        const auto* sa = static_cast<const float*>(ptr(as));
        const auto* sb = static_cast<const float*>(ptr(bs));
        if (!grouped) return dsmoe_int8_gemm(pa, sa, M, K, pb, sb, N, ptr(out), code, st);
        return dsmoe_int8_grouped_gemm(pa, sa, M, K, pb, sb, static_cast<int>(b.size(0)), N, static_cast<const int*>(ptr(off)),
                                       ptr(out), code, st);
      });
    }
    return wrap(out);
  });
}

// idx, n_experts -> (pos, src, offsets)
PyObject* sort_tokens(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(args, n, 2, [](PyObject* const* args) -> PyObject* {
    const char* name = "sort_tokens";
    const Tensor& i0 = tensor(name, args[0]);
    const long long E = PyLong_AsLongLong(args[1]);
    if (PyErr_Occurred()) throw Refused{nullptr, ""};
    same_device(name, {&i0});
    type_check(i0.scalar_type() == at::kLong && i0.dim() == 2, name, "idx must be [tokens, k] int64, got ", i0.sizes(), " ",
               i0.scalar_type());
    const int64_t P = i0.size(0), k = i0.size(1);
    value_check(k > 0 && k <= kMaxTopk, name, k, " choices per token (1..", kMaxTopk, ")");
    value_check(E > 0 && E <= kMaxExperts, name, E, " experts (1..", kMaxExperts, ")");
    const Tensor idx = dense(i0, false);
    Tensor pos = empty(idx, {P, k}, at::kInt), src = empty(idx, {P * k}, at::kInt);
    Tensor off = P ? empty(idx, {E + 1}, at::kInt) : at::zeros({E + 1}, idx.options().dtype(at::kInt));
    if (P)
      run(idx, [&](void* st) {
        return dsmoe_sort_tokens(static_cast<const int64_t*>(ptr(idx)), P, static_cast<int>(k), static_cast<int>(E),
                                 static_cast<int*>(ptr(pos)), static_cast<int*>(ptr(src)), static_cast<int*>(ptr(off)), st);
      });
    return tuple({&pos, &src, &off});
  });
}

void check_order(const char* name, const Tensor& pos, const Tensor& off) {
  value_check(pos.scalar_type() == at::kInt && off.scalar_type() == at::kInt && pos.dim() == 2 && off.dim() == 1 &&
                  pos.is_contiguous() && off.is_contiguous() && !lazy(pos) && !lazy(off) && pos.size(1) >= 1 && pos.size(1) <= kMaxTopk &&
                  off.size(0) >= 2 && off.size(0) <= kMaxExperts + 1,
              name, "order must come from sort_tokens");
}

// xs, and the scales of xs where s is defined
std::pair<Tensor, Tensor> dispatch(const char* name, const Tensor& x0, const Tensor& pos, const Tensor& off, Tensor s) {
  same_device(name, {&x0, &pos, &off, &s});
  check_order(name, pos, off);
  const int64_t P = pos.size(0), k = pos.size(1);
  value_check(x0.dim() == 2 && x0.size(0) == P && x0.size(1) > 0, name, "x must be [", P, ", width], got ", x0.sizes());
  if (s.defined()) {
    want(name, s, "scales", at::kFloat, {P});
    no_grad(name, {&x0, &s});
    s = dense(s, false);
  }
  const Tensor x = dense(x0, false);
  Tensor xs = empty(x, {P * k, x.size(1)}, x.scalar_type()), ss = s.defined() ? empty(x, {P * k}, at::kFloat) : Tensor();
  if (P)
    run(x, [&](void* st) {
      return dsmoe_dispatch_rows(ptr(x), static_cast<const float*>(ptr(s)), static_cast<const int*>(ptr(pos)),
                                 static_cast<const int*>(ptr(off)), static_cast<int>(off.size(0) - 1), P, static_cast<int>(k),
                                 x.size(1) * static_cast<int64_t>(x.element_size()), ptr(xs), static_cast<float*>(ptr(ss)), st);
    });
  return {xs, ss};
}

Tensor combine(const char* name, const Tensor& y0, const Tensor& pos, const Tensor& off, Tensor wt) {
  same_device(name, {&y0, &pos, &off, &wt});
  check_order(name, pos, off);
  const int dt = float_code(name, y0, "ys");
  const int64_t P = pos.size(0), k = pos.size(1);
  value_check(y0.dim() == 2 && y0.size(0) == P * k && y0.size(1) > 0, name, "ys must be [", P * k, ", width], got ", y0.sizes());
  if (wt.defined()) {
    want(name, wt, "wt", at::kFloat, pos.sizes());
    wt = dense(wt, false);
  }
  const Tensor ys = dense(y0, false);
  Tensor y = empty(ys, {P, ys.size(1)}, ys.scalar_type());
  if (P)
    run(ys, [&](void* st) {
      return dsmoe_combine_rows(ptr(ys), dt, static_cast<const int*>(ptr(pos)), static_cast<const float*>(ptr(wt)), P,
                                static_cast<int>(k), ys.size(1), ptr(y), st);
    });
  return y;
}

// ------------------------------------------------------------------ gradients

// A gradient captured into a CUDA graph must not reach a leaf whose accumulation node was made outside the capture
// (a live eager graph holds it): autograd would run that node on the stream it was made on and break the capture.
void check_capture(const char* name, std::initializer_list<const Tensor*> ts) {
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return;
  std::vector<std::shared_ptr<torch::autograd::Node>> todo;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) todo.push_back(torch::autograd::impl::gradient_edge(*t).function);
  std::unordered_set<torch::autograd::Node*> seen;
  while (!todo.empty()) {
    const auto node = todo.back();
    todo.pop_back();
    if (!node || !seen.insert(node.get()).second) continue;
    if (dynamic_cast<torch::autograd::AccumulateGrad*>(node.get())) {
      const auto stream = node->stream();
      cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
      bool inside = true;
      if (stream) {
        // an error is the legacy stream's answer while another stream is being captured
        inside = cudaStreamIsCapturing(c10::cuda::CUDAStream(*stream).stream(), &status) == cudaSuccess &&
                 status != cudaStreamCaptureStatusNone;
        if (!inside) cudaGetLastError();
      }
      if (!inside)
        refuse(PyExc_RuntimeError, name,
               "a gradient cannot be captured while an eager graph of the same leaf is alive; delete its outputs first");
    }
    for (const auto& e : node->next_edges()) todo.push_back(e.function);
  }
}

// f() on an autograd thread, where a refusal is a torch error; differentiable once
template <typename F>
auto in_backward(const char* name, std::initializer_list<const Tensor*> ts, F f) {
  if (c10::GradMode::is_enabled())
    for (const Tensor* t : ts)
      TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->requires_grad(), name, ": differentiable once (create_graph is not supported)");
  try {
    return f();
  } catch (const Refused& r) {
    TORCH_CHECK(false, name, ": ", r.what);
  }
}

struct Dispatch : torch::autograd::Function<Dispatch> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& pos, const Tensor& off) {
    ctx->save_for_backward({pos, off});
    return dispatch("dispatch_tokens", x, pos, off, Tensor()).first;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list g) {
    const auto saved = ctx->get_saved_variables();
    const char* name = "dispatch_tokens (gradient)";
    const Tensor dx = in_backward(name, {&g[0]}, [&] { return combine(name, g[0], saved[0], saved[1], Tensor()); });
    return {dx, Tensor(), Tensor()};
  }
};

struct Combine : torch::autograd::Function<Combine> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& ys, const std::optional<Tensor>& weights,
                        const Tensor& pos, const Tensor& off) {
    const Tensor wt = weights ? *weights : Tensor();
    // the rows are needed for the weights' gradient alone
    ctx->save_for_backward({wt.defined() && wt.requires_grad() ? ys : Tensor(), wt, pos, off});
    return combine("combine_tokens", ys, pos, off, wt);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list g) {
    const auto saved = ctx->get_saved_variables();
    const char* name = "combine_tokens (gradient)";
    const Tensor &ys0 = saved[0], &wt0 = saved[1], &pos = saved[2], &off = saved[3];
    const bool need_ys = ctx->needs_input_grad(0), need_wt = wt0.defined() && ctx->needs_input_grad(1);
    Tensor dys, dwt;
    in_backward(name, {&g[0], &ys0, &wt0}, [&] {
      const Tensor dy = dense(g[0], false), ys = need_wt ? dense(ys0, false) : Tensor(), wt = wt0.defined() ? dense(wt0, false) : wt0;
      const int64_t P = pos.size(0), k = pos.size(1), H = dy.size(1);
      if (need_ys) dys = empty(dy, {P * k, H}, dy.scalar_type());
      if (need_wt) dwt = empty(dy, {P, k}, at::kFloat);
      if (P && (need_ys || need_wt))
        run(dy, [&](void* st) {
          return dsmoe_combine_grad(ptr(dy), ptr(ys), float_code(name, dy, "dy"), static_cast<const int*>(ptr(pos)),
                                    static_cast<const float*>(ptr(wt)), static_cast<const int*>(ptr(off)),
                                    static_cast<int>(off.size(0) - 1), P, static_cast<int>(k), H, ptr(dys),
                                    static_cast<float*>(ptr(dwt)), st);
        });
      return 0;
    });
    return {dys, dwt, Tensor(), Tensor()};
  }
};

bool wants_grad(const Tensor& t) { return c10::GradMode::is_enabled() && t.defined() && t.requires_grad(); }

// x, pos, offsets, scales -> xs, or (xs, ss)
PyObject* dispatch_tokens(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(args, n, 4, [](PyObject* const* args) -> PyObject* {
    const char* name = "dispatch_tokens";
    const Tensor &x = tensor(name, args[0]), &pos = tensor(name, args[1]), &off = tensor(name, args[2]);
    const Tensor s = maybe(name, args[3]);
    if (s.defined()) {
      const auto r = dispatch(name, x, pos, off, s);
      return tuple({&r.first, &r.second});
    }
    if (!wants_grad(x)) return wrap(dispatch(name, x, pos, off, s).first);
    type_check(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kFloat, name,
               "a gradient needs bfloat16 or float32, got ", x.scalar_type());
    same_device(name, {&x, &pos, &off});
    check_capture(name, {&x});
    return wrap(Dispatch::apply(x, pos, off));
  });
}

// ys, pos, offsets, wt -> y
PyObject* combine_tokens(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(args, n, 4, [](PyObject* const* args) -> PyObject* {
    const char* name = "combine_tokens";
    const Tensor &ys = tensor(name, args[0]), &pos = tensor(name, args[1]), &off = tensor(name, args[2]);
    const Tensor wt = maybe(name, args[3]);
    if (!wants_grad(ys) && !wants_grad(wt)) return wrap(combine(name, ys, pos, off, wt));
    same_device(name, {&ys, &pos, &off, &wt});
    check_capture(name, {&ys, &wt});
    return wrap(Combine::apply(ys, wt.defined() ? std::optional<Tensor>(wt) : std::nullopt, pos, off));
  });
}

PyObject* set_error_type(PyObject*, PyObject* type) {
  Py_INCREF(type);
  Py_XDECREF(g_error);
  g_error = type;
  Py_RETURN_NONE;
}

#define DSMOE_FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(f)), METH_FASTCALL, nullptr
PyMethodDef kMethods[] = {{"rms_norm_quant", DSMOE_FAST(rms_norm_quant)},
                          {"swiglu_quant", DSMOE_FAST(swiglu_quant)},
                          {"int8_product", DSMOE_FAST(int8_product)},
                          {"sort_tokens", DSMOE_FAST(sort_tokens)},
                          {"dispatch_tokens", DSMOE_FAST(dispatch_tokens)},
                          {"combine_tokens", DSMOE_FAST(combine_tokens)},
                          {"set_error_type", set_error_type, METH_O, nullptr},
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_ops", "Native half of dsmoe.ops.", -1, kMethods};

}  // namespace

PyMODINIT_FUNC PyInit__ops() { return PyModule_Create(&kModule); }
