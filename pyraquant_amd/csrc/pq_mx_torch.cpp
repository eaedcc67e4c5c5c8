// The Mxfp4Linear call and its backward pass without Python between the module and the kernels: pyraquant_amd._mx.
//
//   layer(x, codes, scales, lr_A, lr_B, bias, out_features, laid_out) -> y
//   quant(x, checkpoint) -> (codes, scales, q8 or None)
//   values(codes, scales, bits, rows, cols, dtype) -> [rows, cols]
//
// lr_A [K, R] and lr_B [R, N], or in the kernels' order (laid_out: lr_A's fragments [ceil(K / 128) 128, P], lr_B's rows [N, P]);
// None without a low-rank branch. Three
// allocations a forward pass that a backward pass follows (y, what the backward pass keeps, and scratch), two otherwise; the
// backward pass runs on autograd's thread without the interpreter. Work goes to the current stream of x's device.
#include <Python.h>

#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/pyraquant_amd.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Refused {
  int status;
  std::string text;
};

void check(int status, const char* what) {
  if (status != PQ_OK) throw Refused{status, std::string(what) + ": " + pq_last_error()};
}

int64_t up(int64_t bytes) { return (bytes + 255) & ~int64_t(255); }
int64_t units(int64_t M, int64_t K) { return (M + 15) / 16 * ((K + 127) / 128); }
int32_t code_of(const Tensor& x) { return x.scalar_type() == at::kBFloat16 ? PQ_BF16 : PQ_F16; }
template <typename T>
T* data(const Tensor& t) { return t.defined() ? static_cast<T*>(const_cast<void*>(t.const_data_ptr())) : nullptr; }

// Rows as the kernels read them: consecutive elements, 16-byte aligned, none over another, no further apart than `most` (a copy
// where not).
Tensor rows_of(const Tensor& t, int64_t most = INT64_MAX) {
  Tensor x = t.is_neg() ? t.resolve_neg() : t;
  const int64_t M = x.size(0), K = x.size(1);
  if ((K > 1 && x.stride(1) != 1) || (M > 1 && (x.stride(0) < K || x.stride(0) % 8 || x.stride(0) > most)) || (uintptr_t)x.const_data_ptr() % 16)
    x = x.clone(at::MemoryFormat::Contiguous);
  return x;
}
int64_t stride_of(const Tensor& x) { return x.size(0) > 1 ? x.stride(0) : x.size(1); }

int64_t padded(int64_t C) { return (C + 127) / 128 * 128; }   // columns of a factor's fragments

// What the backward pass keeps, slices of one allocation: offsets, in bytes.
struct Kept {
  int64_t q8 = 0, scales, t, ap, bp, total;   // ap: lr_A's rows [K, P], bp: lr_B's fragments
  Kept(int64_t M, int64_t K, int64_t N, int64_t P, bool x, bool down, bool factors) {
    scales = x ? up(M * K) : 0;
    t = scales + (x ? up(units(M, K) * 64) : 0);
    ap = t + (down ? up(4 * M * P) : 0);   // (t: fp32)
    bp = ap + (factors ? up(2 * K * P) : 0);
    total = bp + (factors ? up(2 * P * padded(N)) : 0);
  }
};

// What a call needs: gradients of x, lr_A, lr_B and the bias.
struct Wanted {
  bool x, A, B, b;
  bool any() const { return x || A || B || b; }
};

Tensor bytes(int64_t n, const Tensor& like) { return at::empty({n}, like.options().dtype(at::kByte).requires_grad(false)); }

// y; `kept` is filled where something is wanted.
Tensor forward(const Tensor& x0, const Tensor& codes, const Tensor& scales, const Tensor& A, const Tensor& B, const Tensor& bias,
               int64_t N, bool laid_out, Wanted w, Tensor& kept) {
  const Tensor x = rows_of(x0);
  const c10::DeviceGuard guard(x.device());
  const hipStream_t stream = c10::hip::getCurrentHIPStream(x.device().index()).stream();
  const int64_t M = x.size(0), K = x.size(1), R = !A.defined() ? 0 : A.size(1), P = R == 0 ? 0 : R <= 32 ? 32 : 64;
  const Kept k(M, K, N, P, w.A, w.B, P && w.any());
  // scratch: the codes, and what is not kept of scales and t; the forward pass's order of the factors where they come in theirs
  const int64_t s_scales = up(units(M, K) * 1024), s_t = s_scales + (w.A ? 0 : up(units(M, K) * 64));
  const int64_t s_at = s_t + (w.B ? 0 : up(4 * M * P)), s_bt = s_at + (P && !laid_out ? up(2 * P * padded(K)) : 0);
  const int64_t s_ws = s_bt + (P && !laid_out ? up(2 * N * P) : 0), ws = P && M ? pq_mx_lowrank_workspace_size(M, K, P) : 0;
  const Tensor scratch = bytes(s_ws + ws, x);
  if (w.any()) kept = bytes(k.total, x);
  const Tensor y = at::empty({M, N}, x.options().requires_grad(false));
  uint8_t *const s = data<uint8_t>(scratch), *const h = data<uint8_t>(kept);
  const void *at = nullptr, *bt = nullptr;
  if (P && laid_out) {
    at = A.const_data_ptr(), bt = B.const_data_ptr();
    if (w.any())   // the orders of the backward pass from those of the forward pass
      check(pq_mx_factors(at, 0, PQ_MX_FRAGMENTS, bt, P, PQ_MX_BY_COLUMN, K, N, P, P, nullptr, h + k.ap, nullptr, h + k.bp, stream),
            "mxfp4 factors");
  } else if (P) {
    const Tensor a = (R > 1 && A.stride(1) != 1) || A.stride(0) < R || A.is_neg() ? A.resolve_neg().clone(at::MemoryFormat::Contiguous) : A;
    const Tensor b = B.stride(1) != 1 || B.stride(0) < N || B.is_neg() ? B.resolve_neg().clone(at::MemoryFormat::Contiguous) : B;
    at = s + s_at, bt = s + s_bt;
    check(pq_mx_factors(a.const_data_ptr(), a.stride(0), PQ_MX_BY_COLUMN, b.const_data_ptr(), b.stride(0), PQ_MX_BY_RANK, K, N, R, P,
                        s + s_at, w.any() ? h + k.ap : nullptr, s + s_bt, w.any() ? h + k.bp : nullptr, stream),
          "mxfp4 factors");
  }
  check(pq_mx_linear(x.const_data_ptr(), code_of(x), M, K, stride_of(x), data<uint8_t>(codes), data<uint8_t>(scales),
                     data<float>(bias), at, bt, P, y.data_ptr(), N, N, s, w.A ? h + k.scales : s + s_scales,
                     w.A ? reinterpret_cast<int8_t*>(h + k.q8) : nullptr, P ? reinterpret_cast<float*>(w.B ? h + k.t : s + s_t) : nullptr,
                     ws ? s + s_ws : nullptr, ws, stream),
        "mxfp4 layer");
  return y;
}

struct Layer : torch::autograd::Function<Layer> {
  using Maybe = std::optional<Tensor>;   // (an argument that is not there is no input of the graph's node)
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Maybe& lr_A, const Maybe& lr_B, const Maybe& b, const Tensor& codes,
                        const Tensor& scales, int64_t N, bool laid_out) {
    const Tensor A = lr_A.value_or(Tensor()), B = lr_B.value_or(Tensor()), bias = b.value_or(Tensor());
    const Wanted w{x.requires_grad(), A.defined() && A.requires_grad(), B.defined() && B.requires_grad(),
                   bias.defined() && bias.requires_grad()};
    Tensor kept;
    const Tensor y = ::forward(x, codes, scales, A, B, bias, N, laid_out, w, kept);
    ctx->save_for_backward({kept, codes, scales});
    ctx->saved_data["sizes"] = std::vector<int64_t>{x.size(0), x.size(1), N, A.defined() ? A.size(1) : 0,
                                                    (int64_t)w.x | (int64_t)w.A << 1 | (int64_t)w.B << 2 | (int64_t)w.b << 3};
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &kept = saved[0], &codes = saved[1], &scales = saved[2];
    const std::vector<int64_t> z = ctx->saved_data["sizes"].toIntVector();
    const int64_t M = z[0], K = z[1], N = z[2], R = z[3], P = R == 0 ? 0 : R <= 32 ? 32 : 64;
    const Wanted had{(z[4] & 1) != 0, (z[4] & 2) != 0, (z[4] & 4) != 0, (z[4] & 8) != 0};
    const Kept k(M, K, N, P, had.A, had.B, P && had.any());
    variable_list out(8);
    if (!grads[0].defined()) return out;
    // (needs_input_grad counts the inputs that are there)
    const Wanted w{had.x && ctx->needs_input_grad(0), had.A && ctx->needs_input_grad(1), had.B && ctx->needs_input_grad(2),
                   had.b && ctx->needs_input_grad(P ? 3 : 1)};
    try {
      const Tensor dy = rows_of(grads[0], 1 << 21);   // (pq_mx_grad_input's limit)
      const c10::DeviceGuard guard(dy.device());
      const hipStream_t stream = c10::hip::getCurrentHIPStream(dy.device().index()).stream();
      const auto opt = dy.options().requires_grad(false);
      const int32_t code = code_of(dy);
      uint8_t* const h = data<uint8_t>(kept);
      if (w.x) out[0] = at::empty({M, K}, opt);
      if (M == 0) {
        if (w.A) out[1] = at::zeros({K, R}, opt);
        if (w.B) out[2] = at::zeros({R, N}, opt);
        if (w.b) out[3] = at::zeros({N}, opt.dtype(at::kFloat));
        return out;
      }
      if (w.A) out[1] = at::empty({K, R}, opt);
      if (w.B) out[2] = at::empty({R, N}, opt);
      if (w.b) out[3] = at::empty({N}, opt.dtype(at::kFloat));
      const bool sums = w.A || w.B || w.b, need_dt = P && (w.x || w.A);
      const int64_t P_sums = P ? P : 32;   // (the bias's gradient has no rank)
      const int64_t s_dt = need_dt ? up(4 * M * P) : 0;
      const int64_t ws_sums = sums ? pq_mx_grad_factors_workspace_size(M, K, N, P_sums) : 0;
      const int64_t ws_dx = w.x ? pq_mx_grad_input_workspace_size(M, N, K) : 0;
      const int64_t ws_dt = need_dt ? pq_mx_lowrank_workspace_size(M, N, P) : 0;
      const Tensor scratch = bytes(s_dt + std::max({ws_sums, ws_dx, ws_dt}), dy);   // (one after the other on the stream)
      uint8_t* const s = data<uint8_t>(scratch);
      float* const dt = reinterpret_cast<float*>(s);
      if (need_dt)
        check(pq_mx_lowrank_down(dy.const_data_ptr(), code, M, N, stride_of(dy), h + k.bp, P, dt, ws_dt ? s + s_dt : nullptr, ws_dt, stream),
              "mxfp4 dt");
      if (sums)
        check(pq_mx_grad_factors(dy.const_data_ptr(), code, stride_of(dy), w.B ? reinterpret_cast<float*>(h + k.t) : nullptr, dt,
                                 reinterpret_cast<int8_t*>(h + k.q8), h + k.scales, M, K, N, P ? R : 1, P_sums, data<void>(out[1]),
                                 data<void>(out[2]), data<float>(out[3]), s + s_dt, ws_sums, stream),
              "mxfp4 factor gradients");
      if (w.x)
        check(pq_mx_grad_input(dy.const_data_ptr(), code, stride_of(dy), data<uint8_t>(codes), data<uint8_t>(scales),
                               P ? dt : nullptr, P ? h + k.ap : nullptr, P, out[0].data_ptr(), K, M, N, K,
                               ws_dx ? s + s_dt : nullptr, ws_dx, stream),
              "mxfp4 input gradient");
    } catch (const Refused& r) {
      throw std::runtime_error(r.text);
    }
    if (at::GradMode::is_enabled()) once(out, grads[0], P != 0);
    return out;
  }

  // The gradients of a pass with create_graph: each gets edges to what it depends on by the formulas, through a node that raises. (What
  // the kernels write has no history: without this it would count as a constant wherever it is differentiated.)
  static void once(variable_list& out, const Tensor& dy, bool branch) {
    const torch::autograd::edge_list& inputs = torch::autograd::get_current_node()->next_edges();   // x, lr_A and lr_B, bias
    const torch::autograd::Edge none, x = inputs[0], A = branch ? inputs[1] : none, B = branch ? inputs[2] : none;
    const torch::autograd::Edge back = dy.requires_grad() ? torch::autograd::impl::gradient_edge(dy) : none;
    const torch::autograd::edge_list on[4] = {{back, A, B}, {back, B, x}, {back, A, x}, {back}};   // dx, dlr_A, dlr_B, dbias
    for (int i = 0; i < 4; ++i) {
      torch::autograd::edge_list edges;
      for (const auto& e : on[i])
        if (e.is_valid()) edges.push_back(e);
      if (out[i].defined() && !edges.empty())
        torch::autograd::set_history(out[i], std::make_shared<torch::autograd::Error>("the 4-bit layers have no second derivatives", std::move(edges)));
    }
  }
};

// An argument that is a tensor or None; false with a Python error set.
bool tensor_arg(PyObject* o, bool optional, const char* name, Tensor& t) {
  if (optional && o == Py_None) return true;
  if (!THPVariable_Check(o)) {
    PyErr_Format(PyExc_TypeError, "%s is no tensor", name);
    return false;
  }
  t = THPVariable_Unpack(o);
  return true;
}

// The state the kernels need, as AssertionError (ValueError for a type).
const char* wrong(const Tensor& x, const Tensor& codes, const Tensor& scales, const Tensor& A, const Tensor& B, const Tensor& bias,
                  int64_t N, bool laid_out) {
  if (!x.is_cuda()) return "the 4-bit layers run on the GPU only (got a CPU tensor)";
  if (x.dim() < 1) return "x has no dimension";
  const int64_t K = x.size(-1);
  for (const Tensor* t : {&codes, &scales, &A, &B, &bias})
    if (t->defined() && t->device() != x.device()) return "operands on different devices";
  if (K < 32 || K % 32 || N < 16 || N % 16) return "in_features must be a multiple of 32 and out_features of 16";
  if (codes.scalar_type() != at::kByte || scales.scalar_type() != at::kByte || !codes.is_contiguous() || !scales.is_contiguous() ||
      codes.numel() != units(N, K) * 1024 || scales.numel() != units(N, K) * 64)
    return "the weight's codes and scales are not those of a weight of this layer's sizes (x has another in_features?)";
  if (bias.defined() && (bias.scalar_type() != at::kFloat || !bias.is_contiguous() || bias.numel() != N || (uintptr_t)bias.const_data_ptr() % 16))
    return "bias must be contiguous fp32 [out_features]";
  if (A.defined() != B.defined()) return "lr_A and lr_B go together";
  if (A.defined()) {
    if (A.dim() != 2 || B.dim() != 2 || A.scalar_type() != x.scalar_type() || B.scalar_type() != x.scalar_type())
      return "lr_A and lr_B must be matrices of x's type";
    const int64_t R = A.size(1);
    if (laid_out ? A.size(0) != padded(K) || B.size(0) != N || B.size(1) != R || !A.is_contiguous() || !B.is_contiguous() ||
                       (R != 32 && R != 64) || (uintptr_t)A.const_data_ptr() % 16 || (uintptr_t)B.const_data_ptr() % 16
                 : A.size(0) != K || B.size(0) != R || B.size(1) != N || R < 1 || R > 64)
      return "lr_A and lr_B do not fit the layer";
  }
  return nullptr;
}

PyObject* layer(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 8) {
    PyErr_SetString(PyExc_TypeError, "layer(x, codes, scales, lr_A, lr_B, bias, out_features, laid_out)");
    return nullptr;
  }
  Tensor x, codes, scales, A, B, bias;
  if (!tensor_arg(args[0], false, "x", x) || !tensor_arg(args[1], false, "codes", codes) ||
      !tensor_arg(args[2], false, "scales", scales) || !tensor_arg(args[3], true, "lr_A", A) || !tensor_arg(args[4], true, "lr_B", B) ||
      !tensor_arg(args[5], true, "bias", bias))
    return nullptr;
  const int64_t N = PyLong_AsLongLong(args[6]);
  const int laid_out = PyObject_IsTrue(args[7]);
  if ((N == -1 && PyErr_Occurred()) || laid_out < 0) return nullptr;
  if (x.is_cuda() && x.scalar_type() != at::kBFloat16 && x.scalar_type() != at::kHalf) {
    PyErr_SetString(PyExc_ValueError, "x must be bfloat16 or float16");
    return nullptr;
  }
  if (const char* const text = wrong(x, codes, scales, A, B, bias, N, laid_out != 0)) {
    PyErr_SetString(PyExc_AssertionError, text);
    return nullptr;
  }
  for (const Tensor* t : {&x, &A, &B, &bias})
    if (t->defined() && t->_fw_grad(0).defined()) {
      PyErr_SetString(PyExc_RuntimeError, "the 4-bit layers have no forward-mode derivatives");
      return nullptr;
    }
  if (laid_out && at::GradMode::is_enabled() && A.defined() && (A.requires_grad() || B.requires_grad())) {
    PyErr_SetString(PyExc_AssertionError, "a frozen layer's factors, in the kernels' order, have no gradients (trainable=True tunes them)");
    return nullptr;
  }
  Tensor y;
  int status = PQ_OK;
  std::string text;
  {
    pybind11::gil_scoped_release release;
    try {
      const Tensor x2 = x.dim() == 2 ? x : x.reshape({-1, x.size(-1)});
      const bool any = at::GradMode::is_enabled() && (x2.requires_grad() || (A.defined() && (A.requires_grad() || B.requires_grad())) ||
                                                      (bias.defined() && bias.requires_grad()));
      if (any) {
        auto maybe = [](const Tensor& t) { return t.defined() ? Layer::Maybe(t) : std::nullopt; };
        y = Layer::apply(x2, maybe(A), maybe(B), maybe(bias), codes, scales, N, laid_out != 0);
      } else {
        Tensor kept;
        y = ::forward(x2, codes, scales, A, B, bias, N, laid_out != 0, {false, false, false, false}, kept);
      }
      if (x.dim() != 2) {
        std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
        shape.back() = N;
        y = y.reshape(shape);
      }
    } catch (const Refused& r) {
      status = r.status;
      text = r.text;
    }
  }
  if (status != PQ_OK) {
    PyErr_SetString(status == PQ_EDTYPE ? PyExc_ValueError : status == PQ_ELAUNCH ? PyExc_RuntimeError : PyExc_AssertionError, text.c_str());
    return nullptr;
  }
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

PyObject* raise(int status, const char* what) {
  PyErr_Format(status == PQ_EDTYPE ? PyExc_ValueError : status == PQ_ELAUNCH ? PyExc_RuntimeError : PyExc_AssertionError, "%s: %s", what,
               pq_last_error());
  return nullptr;
}
// PQ_BF16, PQ_F16 or PQ_F32; -1 with a Python error set.
int32_t float_code(at::ScalarType t) {
  if (t == at::kBFloat16) return PQ_BF16;
  if (t == at::kHalf) return PQ_F16;
  if (t == at::kFloat) return PQ_F32;
  PyErr_SetString(PyExc_ValueError, "unsupported dtype (expected bfloat16, float16 or float32)");
  return -1;
}

PyObject* quant(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Tensor x;
  if (nargs != 2 || !tensor_arg(args[0], false, "x", x)) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "quant(x, checkpoint)");
    return nullptr;
  }
  const int checkpoint = PyObject_IsTrue(args[1]);
  if (checkpoint < 0) return nullptr;
  if (!x.is_cuda() || x.dim() != 2 || x.size(1) < 32 || x.size(1) % 32) {
    PyErr_SetString(PyExc_AssertionError, !x.is_cuda() ? "the 4-bit layers run on the GPU only (got a CPU tensor)"
                                                       : "x must be a matrix whose rows are a multiple of 32 values");
    return nullptr;
  }
  const int32_t code = float_code(x.scalar_type());
  if (code < 0) return nullptr;
  Tensor codes, scales, q8;
  int st;
  {
    pybind11::gil_scoped_release release;
    const int64_t M = x.size(0), K = x.size(1);
    Tensor r = (x.is_neg() ? x.resolve_neg() : x).detach();
    if (r.stride(1) != 1 || (M > 1 && r.stride(0) < K)) r = r.clone(at::MemoryFormat::Contiguous);
    const c10::DeviceGuard guard(x.device());
    codes = bytes(units(M, K) * 1024, r);
    scales = bytes(units(M, K) * 64, r);
    if (checkpoint) q8 = at::empty({M, K}, codes.options().dtype(at::kChar));
    st = pq_mx_quant(r.const_data_ptr(), code, M, K, stride_of(r), data<uint8_t>(codes), data<uint8_t>(scales), data<int8_t>(q8),
                     c10::hip::getCurrentHIPStream(x.device().index()).stream());
  }
  if (st != PQ_OK) return raise(st, "quant_mxfp4");
  PyObject* const none = Py_None;
  if (!checkpoint) Py_INCREF(none);
  return Py_BuildValue("(NNN)", THPVariable_Wrap(codes), THPVariable_Wrap(scales), checkpoint ? THPVariable_Wrap(q8) : none);
  END_HANDLE_TH_ERRORS
}

PyObject* values(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Tensor codes, scales;
  if (nargs != 6 || !tensor_arg(args[0], false, "codes", codes) || !tensor_arg(args[1], false, "scales", scales) ||
      !THPDtype_Check(args[5])) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "values(codes, scales, bits, rows, cols, dtype)");
    return nullptr;
  }
  const int64_t bits = PyLong_AsLongLong(args[2]), M = PyLong_AsLongLong(args[3]), K = PyLong_AsLongLong(args[4]);
  if (PyErr_Occurred()) return nullptr;
  const at::ScalarType type = reinterpret_cast<THPDtype*>(args[5])->scalar_type;
  const int32_t code = float_code(type);
  if (code < 0) return nullptr;
  const bool eight = bits == 8;
  if (!codes.is_cuda() || !scales.is_cuda() || codes.device() != scales.device() || M < 0 || K < 32 || K % 32 || (bits != 4 && !eight) ||
      codes.scalar_type() != (eight ? at::kChar : at::kByte) || scales.scalar_type() != at::kByte || !codes.is_contiguous() ||
      !scales.is_contiguous() || codes.numel() < (eight ? M * K : units(M, K) * 1024) || scales.numel() < units(M, K) * 64) {
    PyErr_SetString(PyExc_AssertionError, "codes and scales are not those of a matrix of this size on the GPU");
    return nullptr;
  }
  Tensor out;
  int st;
  {
    pybind11::gil_scoped_release release;
    const c10::DeviceGuard guard(codes.device());
    out = at::empty({M, K}, codes.options().dtype(type));
    st = pq_mx_values(codes.const_data_ptr(), data<uint8_t>(scales), (int32_t)bits, M, K, out.data_ptr(), code, K,
                      c10::hip::getCurrentHIPStream(codes.device().index()).stream());
  }
  if (st != PQ_OK) return raise(st, "mxfp4 values");
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

template <typename F>
PyCFunction fast(F* f) { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(f)); }
PyMethodDef kMethods[] = {
    {"layer", fast(layer), METH_FASTCALL,
     "layer(x, codes, scales, lr_A, lr_B, bias, out_features, laid_out): the Mxfp4Linear call, differentiable"},
    {"quant", fast(quant), METH_FASTCALL, "quant(x, checkpoint): (codes, scales, q8 or None), pq_mx_quant"},
    {"values", fast(values), METH_FASTCALL, "values(codes, scales, bits, rows, cols, dtype): [rows, cols], pq_mx_values"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_mx", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__mx() { return PyModule_Create(&kModule); }
