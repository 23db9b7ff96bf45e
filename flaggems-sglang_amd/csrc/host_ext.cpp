// Python module `flaggems_sglang._host`: the host side of the dense operators
// (flaggems_sglang.ops.dense) and of the routed layer's steps (host_steps.h) --
// argument checks, output allocation, the current stream, the call into
// libfgs_moe.so's C ABI. A decode step's kernels
// take 2 to 8 us and a launch 3.3; the same steps in Python took 9.6 to 13 us a
// call (a norm with four outputs 13.2, here 5.8; the dispatcher's empty() 7.2),
// so at one token the host was what a layer waited for.
//
// The library's entries come in by address (bind), from the handle that
// flaggems_sglang._capi has loaded. No C++ exception leaves this file.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/EmptyTensor.h>
#include <ATen/core/Tensor.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPFunctions.h>
#include <ATen/hip/EmptyTensor.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include <array>
#include <initializer_list>
#include <string>

#include "fgs_moe.h"

namespace {

constexpr int64_t kGroup = 128;  // columns of an e4m3 scale
// Largest row strides of the product's operands and activation scales.
constexpr int64_t kMaxStride = int64_t{1} << 22, kMaxScaleStride = int64_t{1} << 20;

struct Library {
  decltype(&fgs_moe_last_error) last_error;
  decltype(&fgs_moe_rms_norm) rms_norm;
  decltype(&fgs_moe_silu_and_mul_quant) silu_and_mul_quant;
  decltype(&fgs_moe_fp8_block_matmul) fp8_block_matmul;
};
Library g_lib{};

// A refusal: the Python exception to raise.
struct Refusal {
  PyObject* type;
  std::string text;
};
struct Raised {};  // ... of a Python call that has set one
[[noreturn]] void refuse(PyObject* type, std::string text) {
  throw Refusal{type, std::move(text)};
}
void require(bool ok, const char* text) {
  if (!ok) refuse(PyExc_AssertionError, text);
}

struct Arg {
  const char* name;
  const at::Tensor* t;  // null: not given
};

Arg tensor_arg(PyObject* o, const char* name, bool optional = false) {
  if (optional && o == Py_None) return {name, nullptr};
  if (!THPVariable_Check(o)) refuse(PyExc_TypeError, std::string(name) + " must be a tensor");
  return {name, &THPVariable_Unpack(o)};
}

// Whether all of a tensor's values lie inside its storage. (A freed one's have
// no address, or only an offset for one, and the library takes a null residual
// or bias for none.)
bool in_memory(const at::Tensor& t) {
  return !t._is_zerotensor() &&
         t.storage().nbytes() >= at::detail::computeStorageNbytes(t.sizes(), t.strides(),
                                                                  t.element_size(),
                                                                  t.storage_offset());
}

// Every tensor given is on one GPU, holds its values and needs no gradient; that
// GPU's index.
int check_inputs(std::initializer_list<Arg> args) {
  const at::Tensor* first = args.begin()->t;
  if (!first->is_cuda())
    refuse(PyExc_RuntimeError, std::string(args.begin()->name) +
                                   " must be a GPU tensor: the fused-MoE kernels run only on the "
                                   "MI355X (no CPU path)");
  const bool grad = c10::GradMode::is_enabled();
  const bool tangents = c10::AutogradState::get_tls_state().get_fw_grad_mode();
  for (const Arg& a : args) {
    if (!a.t) continue;
    if (a.t->device() != first->device())
      refuse(PyExc_RuntimeError, std::string(a.name) + " is on " + a.t->device().str() +
                                     ", not on " + first->device().str());
    if (!a.t->has_storage())  // (sparse, or inside a transformation)
      refuse(PyExc_NotImplementedError, std::string(a.name) + " has no storage: this operator takes "
                                                              "dense tensors, outside torch.func");
    if (!in_memory(*a.t))
      refuse(PyExc_RuntimeError,
             std::string(a.name) + " has no memory for its values (a zero tensor, or freed)");
    if (a.t->is_neg())  // (its memory holds the values' negatives)
      refuse(PyExc_NotImplementedError, std::string(a.name) + " is a lazily negated view");
    if (grad && a.t->requires_grad())
      refuse(PyExc_RuntimeError, std::string(a.name) +
                                     " requires a gradient: this operator has no backward pass "
                                     "(call it under torch.no_grad())");
    if (tangents && a.t->_fw_grad(0).defined())
      refuse(PyExc_RuntimeError, std::string(a.name) +
                                     " has a forward-mode tangent: this operator has no "
                                     "forward-mode derivative (give it the primal)");
  }
  return first->get_device();
}

int type_code(const at::Tensor& t) {  // FGS_DTYPE_*, -1: none of them
  switch (t.scalar_type()) {
    case at::kBFloat16: return FGS_DTYPE_BF16;
    case at::kHalf: return FGS_DTYPE_FP16;
    case at::kFloat: return FGS_DTYPE_FP32;
    default: return -1;
  }
}

at::Tensor make(at::IntArrayRef shape, at::ScalarType type, const at::Tensor& like) {
  return at::Tensor(at::detail::empty_cuda(shape, type, like.device(), std::nullopt));
}

// The rows of a tensor's last dimension: where they are if they lie evenly
// spaced (as a slice of a wider tensor), else copied.
struct Rows {
  at::Tensor t;
  int64_t stride;
};
Rows rows_of(const at::Tensor& x, int64_t cols) {
  if (x.is_contiguous()) return {x, cols};
  if (x.dim() == 2 && (x.stride(1) == 1 || cols == 1)) return {x, x.stride(0)};
  return {x.contiguous(), cols};
}

struct Scales {
  at::Tensor t;
  int64_t row, col;
};
Scales make_scales(const at::Tensor& x, int64_t rows, int64_t cols, int mode, bool column_major) {
  at::DimVector lead(x.sizes().begin(), x.sizes().end() - 1);
  if (mode == FGS_QUANT_INT8_TOKEN) return {make(lead, at::kFloat, x), 1, 0};
  const int64_t groups = (cols + kGroup - 1) / kGroup;
  at::DimVector shape = lead;
  shape.push_back(groups);
  if (!column_major) return {make(shape, at::kFloat, x), groups, 1};
  at::Tensor t = make({groups, rows}, at::kFloat, x).t();
  return {x.dim() == 2 ? t : t.view(shape), 1, rows};
}

void* stream_of(int index) {
  return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(static_cast<c10::DeviceIndex>(index))
      .stream();
}

// The GPU `index` as the current one, and the interpreter's lock given away, for
// a scope, however it is left.
struct OnGpu {
  explicit OnGpu(int index) : was(c10::hip::current_device()), moved(was != index) {
    if (moved) c10::hip::set_device(static_cast<c10::DeviceIndex>(index));
  }
  ~OnGpu() {
    if (moved) static_cast<void>(c10::hip::SetDevice(static_cast<c10::DeviceIndex>(was)));
  }
  OnGpu(const OnGpu&) = delete;
  const int was;
  const bool moved;
};
// (A backward pass comes without the lock.)
struct Unlocked {
  Unlocked() : state(PyGILState_Check() ? PyEval_SaveThread() : nullptr) {}
  ~Unlocked() {
    if (state) PyEval_RestoreThread(state);
  }
  Unlocked(const Unlocked&) = delete;
  PyThreadState* const state;
};

// Runs a library entry with its GPU current and without the interpreter lock,
// and raises what it returns. (The arguments are values by then: what asks a
// tensor for its memory, which may raise, is the caller's expression.)
template <class... P, class... A>
void call(int index, const char* what, int32_t (*entry)(P...), A... args) {
  int32_t rc;
  {
    const OnGpu gpu(index);
    const Unlocked unlocked;
    rc = entry(args...);
  }
  if (rc == FGS_OK) return;
  refuse(rc == FGS_EINVAL ? PyExc_ValueError
                          : rc == FGS_EUNSUPPORTED ? PyExc_NotImplementedError : PyExc_RuntimeError,
         std::string(what) + ": " + g_lib.last_error());
}

// Tells autograd that the library has written a caller's tensor.
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

PyObject* wrap(const at::Tensor& t) {
  if (!t.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(t);
}
template <size_t N>
PyObject* wrap_all(const std::array<at::Tensor, N>& ts) {
  PyObject* out = PyTuple_New(N);
  if (!out) throw Raised{};
  for (size_t i = 0; i < N; ++i) {
    PyObject* o = wrap(ts[i]);
    if (!o) {
      Py_DECREF(out);
      throw Raised{};
    }
    PyTuple_SET_ITEM(out, i, o);
  }
  return out;
}

bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Raised{};
  return v != 0;
}
int64_t whole(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Raised{};
  return v;
}
float real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Raised{};
  return static_cast<float>(v);
}
void* ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* floats(const at::Tensor& t) { return static_cast<float*>(ptr(t)); }

// Rows in memory, in bytes.
struct Span {
  const char* at;
  int64_t rows, stride, bytes;
  const char* end() const { return at + (rows - 1) * stride + bytes; }
};
Span span(const at::Tensor& t, int64_t rows, int64_t cols, int64_t stride) {
  const int64_t e = t.element_size();
  return {static_cast<const char*>(ptr(t)), rows, stride * e, cols * e};
}
// Whether a value of one may be one of the other. (Columns of one wider tensor,
// rows the same stride apart, are not; other strides whose ranges cross count as
// shared.)
bool shared(const Span& a, const Span& b) {
  if (a.rows == 0 || b.rows == 0 || a.end() <= b.at || b.end() <= a.at) return false;
  const int64_t stride = a.rows == 1 ? b.stride : a.stride;
  if ((a.rows > 1 && b.rows > 1 && a.stride != b.stride) || stride <= 0) return true;
  const int64_t between = ((b.at - a.at) % stride + stride) % stride;
  return between < a.bytes || between + b.bytes > stride;
}

// rms_norm(x, weight, eps, residual, weight_offset, quantisation, return_norm,
// column_major, inplace) -> (norm, residual, q, scales)
PyObject* rms_norm(PyObject* const* args) {
  const Arg xa = tensor_arg(args[0], "x"), wa = tensor_arg(args[1], "weight"),
            ra = tensor_arg(args[3], "residual", true);
  const int index = check_inputs({xa, wa, ra});
  const float eps = real(args[2]), offset = real(args[4]);
  const int mode = static_cast<int>(whole(args[5]));
  const bool with_norm = args[6] == Py_None ? mode == FGS_QUANT_NONE : truth(args[6]);
  const bool column_major = truth(args[7]), inplace = truth(args[8]);
  const at::Tensor& x = *xa.t;
  const int type = type_code(x);
  require(type >= 0, "x must be bfloat16, float16 or float32");
  require(x.dim() >= 1 && x.size(-1) > 0, "x must have columns");
  const int64_t cols = x.size(-1), rows = x.numel() / cols;
  require(wa.t->dim() == 1 && wa.t->size(0) == cols, "weight must be [cols]");
  const int weight_type = type_code(*wa.t);
  require(weight_type == type || weight_type == FGS_DTYPE_FP32,
          "weight must be of x's type or float32");
  require(with_norm || mode != FGS_QUANT_NONE || ra.t, "no output was asked for");
  require(!inplace || ra.t, "inplace needs a residual");

  const Rows xr = rows_of(x, cols);
  Rows rr{{}, 0};
  at::Tensor res_out;
  int64_t out_stride = 0;
  if (ra.t) {
    require(ra.t->sizes() == x.sizes() && ra.t->scalar_type() == x.scalar_type(),
            "residual must be of x's shape and type");
    rr = rows_of(*ra.t, cols);
    if (inplace) {
      if (!rr.t.is_same(*ra.t) || (rows > 1 && rr.stride < cols))
        refuse(PyExc_ValueError, "fused_rms_norm: an inplace residual must have evenly spaced rows "
                                 "that do not overlap");
      res_out = *ra.t;
      out_stride = rr.stride;
    } else {
      res_out = make(x.sizes(), x.scalar_type(), x);
      out_stride = cols;
    }
  }
  at::Tensor norm, q;
  Scales scales{{}, 0, 0};
  if (with_norm) norm = make(x.sizes(), x.scalar_type(), x);
  if (mode != FGS_QUANT_NONE) {
    q = make(x.sizes(), mode == FGS_QUANT_INT8_TOKEN ? at::kChar : at::kFloat8_e4m3fn, x);
    scales = make_scales(x, rows, cols, mode, column_major);
  }
  const at::Tensor weight = wa.t->is_contiguous() ? *wa.t : wa.t->contiguous();
  if (inplace) {
    const Span to = span(res_out, rows, cols, out_stride), from = span(xr.t, rows, cols, xr.stride);
    const bool same = to.at == from.at && (rows <= 1 || to.stride == from.stride);
    if ((!same && shared(to, from)) || shared(to, span(weight, 1, cols, cols)))
      refuse(PyExc_ValueError, "fused_rms_norm: an inplace residual may be x itself, but share no "
                               "part of x's or the weight's memory otherwise");
  }
  void* stream = stream_of(index);
  call(index, "fused_rms_norm", g_lib.rms_norm, ptr(xr.t), xr.stride, ptr(rr.t), rr.stride,
       ptr(weight), type, weight_type, eps, offset, rows, cols, ptr(norm), ptr(res_out), out_stride,
       mode, ptr(q), floats(scales.t), scales.row, scales.col, stream);
  if (inplace) written(res_out);
  return wrap_all<4>({norm, res_out, q, scales.t});
}

// silu_and_mul_quant(x, quantisation, gelu, column_major) -> (q, scales)
PyObject* silu_and_mul_quant(PyObject* const* args) {
  const Arg xa = tensor_arg(args[0], "x");
  const int index = check_inputs({xa});
  const int mode = static_cast<int>(whole(args[1]));
  const bool gelu = truth(args[2]), column_major = truth(args[3]);
  const at::Tensor& x = *xa.t;
  const int type = type_code(x);
  require(type >= 0, "x must be bfloat16, float16 or float32");
  require(x.dim() >= 1 && x.size(-1) > 0 && x.size(-1) % 2 == 0,
          "x must hold a gate half and an up half");
  const int64_t n = x.size(-1) / 2, rows = x.numel() / (2 * n);
  const Rows xr = rows_of(x, 2 * n);
  at::DimVector shape(x.sizes().begin(), x.sizes().end());
  shape.back() = n;
  const at::Tensor q =
      make(shape, mode == FGS_QUANT_INT8_TOKEN ? at::kChar : at::kFloat8_e4m3fn, x);
  const Scales scales = make_scales(x, rows, n, mode, column_major);
  void* stream = stream_of(index);
  call(index, "silu_and_mul_quant", g_lib.silu_and_mul_quant, ptr(xr.t), xr.stride, type, rows, n,
       gelu, mode, ptr(q), floats(scales.t), scales.row, scales.col, stream);
  return wrap_all<2>({q, scales.t});
}

// An e4m3 matrix with adjacent columns and 16-byte aligned rows: where it is,
// or copied.
Rows byte_rows(const at::Tensor& t, int64_t cols) {
  if (reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0) {
    if (t.is_contiguous() && cols % 16 == 0) return {t, cols};
    if (t.stride(1) == 1 &&
        (t.size(0) <= 1 || (t.stride(0) % 16 == 0 && t.stride(0) <= kMaxStride)))
      return {t, t.stride(0)};
  }
  return {t.clone(at::MemoryFormat::Contiguous), cols};
}

// fp8_block_matmul(a, a_scale, w, w_scale, bias, out dtype's code, out, flags)
PyObject* fp8_block_matmul(PyObject* const* args) {
  const Arg aa = tensor_arg(args[0], "a"), sa = tensor_arg(args[1], "a_scale"),
            wa = tensor_arg(args[2], "w"), swa = tensor_arg(args[3], "w_scale"),
            ba = tensor_arg(args[4], "bias", true), oa = tensor_arg(args[6], "out", true);
  const int index = check_inputs({aa, sa, wa, swa, ba, oa});
  const int flags = static_cast<int>(whole(args[7]));
  at::Tensor a = *aa.t, a_scale = *sa.t;
  const at::Tensor& w = *wa.t;
  require(a.scalar_type() == at::kFloat8_e4m3fn && w.scalar_type() == at::kFloat8_e4m3fn,
          "a and w must be float8_e4m3fn");
  require(w.dim() == 2 && a.dim() >= 1 && a.size(-1) == w.size(1),
          "a must be [..., k] and w [n, k]");
  const int64_t n = w.size(0), k = w.size(1), kb = (k + kGroup - 1) / kGroup;
  at::DimVector shape(a.sizes().begin(), a.sizes().end());
  shape.back() = kb;
  require(a_scale.sizes() == shape, "a_scale must be [..., ceil(k / 128)]");
  require(swa.t->dim() == 2 && swa.t->size(0) == (n + kGroup - 1) / kGroup &&
              swa.t->size(1) == kb,
          "w_scale must be [ceil(n / 128), ceil(k / 128)]");
  require(a_scale.scalar_type() == at::kFloat && swa.t->scalar_type() == at::kFloat,
          "scales must be float32");
  shape.back() = n;
  int out_type = static_cast<int>(whole(args[5]));
  if (oa.t) {
    out_type = type_code(*oa.t);
    require(oa.t->sizes() == shape, "out must be [..., n]");
    if (oa.t->dim() == 2 ? oa.t->stride(1) != 1 && n > 1 : !oa.t->is_contiguous())
      refuse(PyExc_ValueError, "fp8_block_matmul: the columns of out must be adjacent");
  }
  require(out_type == FGS_DTYPE_BF16 || out_type == FGS_DTYPE_FP16,
          "the output must be bfloat16 or float16");
  at::Tensor bias;
  if (ba.t) {
    require(ba.t->dim() == 1 && ba.t->size(0) == n && type_code(*ba.t) >= 0,
            "bias must be [n], bfloat16, float16 or float32");
    bias = ba.t->is_contiguous() ? *ba.t : ba.t->contiguous();
  }
  const int64_t m = k ? a.numel() / k : 0;
  if (a.dim() != 2) {
    a = a.reshape({m, k});
    a_scale = a_scale.reshape({m, kb});
  }
  const Rows ar = byte_rows(a, k), wr = byte_rows(w, k);
  if (m > 1 && a_scale.stride(0) > kMaxScaleStride) a_scale = a_scale.contiguous();
  const at::Tensor w_scale = swa.t->is_contiguous() ? *swa.t : swa.t->contiguous();
  const at::Tensor out =
      oa.t ? *oa.t : make(shape, out_type == FGS_DTYPE_BF16 ? at::kBFloat16 : at::kHalf, a);
  const int64_t ldo = oa.t && out.dim() == 2 ? out.stride(0) : n;
  if (oa.t) {
    const Span to = span(out, m, n, ldo);
    if (shared(to, span(ar.t, m, k, ar.stride)) || shared(to, span(wr.t, n, k, wr.stride)) ||
        shared(to, span(a_scale, m, (kb - 1) * a_scale.stride(1) + 1, a_scale.stride(0))) ||
        shared(to, span(w_scale, 1, w_scale.numel(), w_scale.numel())) ||
        (bias.defined() && shared(to, span(bias, 1, n, n))))
      refuse(PyExc_ValueError, "fp8_block_matmul: out shares memory with an input");
  }
  void* stream = stream_of(index);
  call(index, "fp8_block_matmul", g_lib.fp8_block_matmul, ptr(ar.t), ar.stride, floats(a_scale),
       a_scale.stride(0), a_scale.stride(1), ptr(wr.t), wr.stride, floats(w_scale), ptr(bias),
       bias.defined() ? type_code(bias) : FGS_DTYPE_FP32, m, n, k, out_type, flags, ptr(out), ldo,
       stream);
  if (oa.t) {
    written(out);
    Py_INCREF(args[6]);
    return args[6];
  }
  return wrap(out);
}

#include "host_steps.h"

// bind(addresses of fgs_moe_last_error, _rms_norm, _silu_and_mul_quant,
// _fp8_block_matmul)
PyObject* bind(PyObject* const* args) {
  auto address = [&](int i) { return reinterpret_cast<void*>(whole(args[i])); };
  g_lib.last_error = reinterpret_cast<decltype(g_lib.last_error)>(address(0));
  g_lib.rms_norm = reinterpret_cast<decltype(g_lib.rms_norm)>(address(1));
  g_lib.silu_and_mul_quant = reinterpret_cast<decltype(g_lib.silu_and_mul_quant)>(address(2));
  g_lib.fp8_block_matmul = reinterpret_cast<decltype(g_lib.fp8_block_matmul)>(address(3));
  Py_RETURN_NONE;
}

// A module function of N positional arguments around `f`.
template <PyObject* (*F)(PyObject* const*), Py_ssize_t N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "%zd arguments expected, got %zd", N, n);
    return nullptr;
  }
  try {
    if (F != bind && F != bind_steps && !g_lib.last_error) refuse(PyExc_RuntimeError, "the library is not bound");
    return F(args);
  } catch (const Refusal& r) {
    PyErr_SetString(r.type, r.text.c_str());
  } catch (const Raised&) {  // a Python error is set
  } catch (...) {            // torch's, as the Python errors they stand for
    torch::translate_exception_to_python(std::current_exception());
  }
  return nullptr;
}
template <PyObject* (*F)(PyObject* const*), Py_ssize_t N>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<F, N>)),
          METH_FASTCALL, nullptr};
}

PyMethodDef g_methods[] = {
    method<bind, 4>("bind"),
    method<rms_norm, 9>("rms_norm"),
    method<silu_and_mul_quant, 4>("silu_and_mul_quant"),
    method<fp8_block_matmul, 8>("fp8_block_matmul"),
    method<bind_steps, 13>("bind_steps"),
    method<permute, 4>("permute"),
    method<permute_rows, 4>("permute_rows"),
    method<unpermute, 5>("unpermute"),
    method<topk_gating, 4>("topk_gating"),
    method<linear, 9>("linear"),
    method<foreign_leaf, 1>("foreign_leaf"),
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, g_methods,
                        nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&g_module); }
