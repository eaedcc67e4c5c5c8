// The call of low-rank adapters and its backward pass without Python between the module and the kernels: pyraquant_amd._adapt.
//
//   adapt(x, y, ids, lr_A, lr_B, scale, rank, laid_out, out or None) -> y + scale[id] (x lr_A[id]) lr_B[id]
//
// lr_A [slots, K, R] and lr_B [slots, R, N], or (laid_out) lr_A in PQ_ADAPTER_DOWN and lr_B in PQ_ADAPTER_UP, [slots, C, P] with C rounded up to 128. Work goes to the current stream of x's device.
#include <Python.h>

#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>

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
int32_t code_of(const Tensor& x) { return x.scalar_type() == at::kBFloat16 ? PQ_BF16 : PQ_F16; }
int64_t padded(int64_t R) { return R <= 16 ? 16 : R <= 32 ? 32 : 64; }
template <typename T>
T* data(const Tensor& t) { return t.defined() ? static_cast<T*>(const_cast<void*>(t.const_data_ptr())) : nullptr; }
Tensor bytes(int64_t n, const Tensor& like) { return at::empty({n}, like.options().dtype(at::kByte).requires_grad(false)); }

// A matrix of rows as the kernels read it: consecutive elements, 16-byte aligned, none over another (a copy where not).
Tensor rows_of(const Tensor& t) {
  Tensor x = t.is_neg() ? t.resolve_neg() : t;
  const int64_t M = x.size(0), K = x.size(1);
  if ((K > 1 && x.stride(1) != 1) || (M > 1 && (x.stride(0) < K || x.stride(0) % 8 || x.stride(0) > (1 << 30))) || (uintptr_t)x.const_data_ptr() % 16)
    x = x.clone(at::MemoryFormat::Contiguous);
  return x;
}
int64_t stride_of(const Tensor& x) { return x.size(0) > 1 ? x.stride(0) : x.size(1); }
Tensor dense(const Tensor& t) {   // contiguous and aligned
  const Tensor x = t.is_neg() ? t.resolve_neg() : t;
  return x.is_contiguous() && (uintptr_t)x.const_data_ptr() % 16 == 0 ? x : x.clone(at::MemoryFormat::Contiguous);
}

struct Sizes {
  int64_t M, K, N, slots, R, P, each;
  int32_t id_bits;
};
// (K to C: one launch makes both products)
bool few_rows(const Sizes& z, int64_t K, int64_t C) { return pq_adapter_rows_fit(z.M, K, C, z.P, z.each); }
struct Factors {   // in the orders that a pass reads
  const void *down, *up;
};

// out [M, N] from x [M, K] and y [M, N]; parts: scratch; joined: t with its scale [M, P], kept for the backward pass, or NULL.
void forward(const Tensor& x, const Tensor& y, const Tensor& ids, const Tensor& scale, Factors f, const Sizes& z, const Tensor& out,
             float* parts, float* joined, hipStream_t stream) {
  if (few_rows(z, z.K, z.N)) {
    check(pq_adapter_rows(x.const_data_ptr(), code_of(x), z.M, z.K, stride_of(x), f.down, data<float>(scale), f.up, z.slots, z.N, z.R, z.P,
                          ids.const_data_ptr(), z.id_bits, z.each, y.const_data_ptr(), stride_of(y), out.data_ptr(), stride_of(out), joined, stream),
          "adapters");
    return;
  }
  check(pq_adapter_down(x.const_data_ptr(), code_of(x), z.M, z.K, stride_of(x), f.down, z.slots, z.P, ids.const_data_ptr(), z.id_bits,
                        z.each, parts, stream),
        "adapters");
  check(pq_adapter_up(parts, pq_adapter_slices(z.M, z.K), data<float>(scale), f.up, z.slots, z.N, z.R, z.P, ids.const_data_ptr(), z.id_bits,
                      z.each, y.const_data_ptr(), stride_of(y), out.data_ptr(), stride_of(out), joined, code_of(x), z.M, stream),
        "adapters");
}
int64_t factor_bytes(const Sizes& z, int64_t C) { return up(2 * z.slots * pq_adapter_factor_size(C, z.P)); }
int64_t parts_bytes(const Sizes& z, int64_t C) { return up(4 * pq_adapter_slices(z.M, C) * z.M * z.P); }

// What the backward pass keeps of a call: t with its scale, and the factors in the orders that it reads (those of a laid out call are
// turned there).
struct Kept {
  Tensor t, a_up, b_down;
};
struct Wanted {
  bool x, A, B;
};
Tensor order(const Sizes& z, int64_t C, const Tensor& like) {
  return at::empty({z.slots * pq_adapter_factor_size(C, z.P)}, like.options().requires_grad(false));
}

// The whole call; `kept` is filled with what is wanted.
Tensor run(const Tensor& x0, const Tensor& y0, const Tensor& ids, const Tensor& A, const Tensor& B, const Tensor& scale, const Sizes& z,
           bool laid_out, Tensor out, Wanted w, Kept& kept) {
  const c10::DeviceGuard guard(x0.device());
  const hipStream_t stream = c10::hip::getCurrentHIPStream(x0.device().index()).stream();
  const bool in_place = out.defined() && out.const_data_ptr() == y0.const_data_ptr();
  const Tensor x = rows_of(x0), y = in_place ? y0 : rows_of(y0);
  if (!out.defined()) out = at::empty({z.M, z.N}, x.options().requires_grad(false));
  const int64_t parts = few_rows(z, z.K, z.N) ? 0 : parts_bytes(z, z.K), at = laid_out ? 0 : factor_bytes(z, z.K), bt = laid_out ? 0 : factor_bytes(z, z.N);
  if (w.B) kept.t = at::empty({z.M, z.P}, x.options().dtype(at::kFloat).requires_grad(false));
  if (!laid_out && w.x) kept.a_up = order(z, z.K, x);
  if (!laid_out && (w.x || w.A)) kept.b_down = order(z, z.N, x);
  const Tensor scratch = parts + at + bt ? bytes(parts + at + bt, x) : Tensor();
  uint8_t* const s = data<uint8_t>(scratch);
  Factors f{A.const_data_ptr(), B.const_data_ptr()};
  if (!laid_out) {
    const Tensor a = dense(A), b = dense(B);
    f = {s, s + at};
    check(pq_adapter_factors(a.const_data_ptr(), PQ_ADAPTER_BY_COLUMN, b.const_data_ptr(), PQ_ADAPTER_BY_RANK, z.slots, z.K, z.N, z.R, z.P, s,
                             data<void>(kept.a_up), data<void>(kept.b_down), s + at, stream),
          "adapters");
  }
  forward(x, y, ids, scale, f, z, out, reinterpret_cast<float*>(s + at + bt), data<float>(kept.t), stream);
  return out;
}

struct Adapt : torch::autograd::Function<Adapt> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& y, const Tensor& ids, const Tensor& A, const Tensor& B,
                        const Tensor& scale, std::vector<int64_t> sizes, bool laid_out) {
    const Sizes z{sizes[0], sizes[1], sizes[2], sizes[3], sizes[4], sizes[5], sizes[6], (int32_t)sizes[7]};
    Kept kept;
    const Tensor out = run(x, y, ids, A, B, scale, z, laid_out, Tensor(), {x.requires_grad(), A.requires_grad(), B.requires_grad()}, kept);
    ctx->save_for_backward({A.requires_grad() ? x : Tensor(), ids, A, B, scale, kept.t, kept.a_up, kept.b_down});
    ctx->saved_data["sizes"] = sizes;
    ctx->saved_data["laid_out"] = laid_out;
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &ids = saved[1], &A = saved[2], &B = saved[3], &scale = saved[4], &kept = saved[5], &a_up = saved[6], &b_down = saved[7];
    const std::vector<int64_t> sizes = ctx->saved_data["sizes"].toIntVector();
    const Sizes z{sizes[0], sizes[1], sizes[2], sizes[3], sizes[4], sizes[5], sizes[6], (int32_t)sizes[7]};
    const bool laid_out = ctx->saved_data["laid_out"].toBool();
    variable_list out(8);
    if (!grads[0].defined()) return out;
    const bool want_x = ctx->needs_input_grad(0), want_A = ctx->needs_input_grad(3), want_B = ctx->needs_input_grad(4);
    if (ctx->needs_input_grad(1)) out[1] = grads[0];
    if (!want_x && !want_A && !want_B) return out;
    try {
      const Tensor dy = rows_of(grads[0]), x = want_A ? rows_of(saved[0]) : Tensor();
      const c10::DeviceGuard guard(dy.device());
      const hipStream_t stream = c10::hip::getCurrentHIPStream(dy.device().index()).stream();
      const auto opt = dy.options().requires_grad(false);
      const int32_t code = code_of(dy);
      if (want_x) out[0] = at::empty({z.M, z.K}, opt);
      if (want_A) out[3] = at::empty({z.slots, z.K, z.R}, opt);
      if (want_B) out[4] = at::empty({z.slots, z.R, z.N}, opt);
      const bool need_dt = want_x || want_A, few = few_rows(z, z.N, z.K);
      const int64_t joined = want_A ? up(4 * z.M * z.P) : 0, parts = joined + (need_dt && !few ? parts_bytes(z, z.N) : 0);
      const int64_t ap = need_dt && laid_out ? factor_bytes(z, z.K) : 0, bp = need_dt && laid_out ? factor_bytes(z, z.N) : 0;
      const int64_t ws = want_A || want_B ? pq_adapter_grads_workspace_size(z.M, z.K, z.N, z.slots, z.P, z.each) : 0;
      const Tensor scratch = parts + ap + bp + ws ? bytes(parts + ap + bp + ws, dy) : Tensor();
      uint8_t* const s = data<uint8_t>(scratch);
      float* const dt = want_A ? reinterpret_cast<float*>(s) : nullptr;   // with its scale
      float* const dt_parts = reinterpret_cast<float*>(s + joined);
      if (need_dt) {
        const void *g = data<void>(a_up), *f = data<void>(b_down);
        if (laid_out) {
          g = s + parts, f = s + parts + ap;
          check(pq_adapter_factors(A.const_data_ptr(), PQ_ADAPTER_DOWN, B.const_data_ptr(), PQ_ADAPTER_UP, z.slots, z.K, z.N, z.P, z.P, nullptr,
                                   want_x ? s + parts : nullptr, s + parts + ap, nullptr, stream),
                "adapters");
        }
        if (few) {
          check(pq_adapter_rows(dy.const_data_ptr(), code, z.M, z.N, stride_of(dy), f, data<float>(scale), g, z.slots, z.K, z.R, z.P,
                                ids.const_data_ptr(), z.id_bits, z.each, nullptr, 0, data<void>(out[0]), z.K, dt, stream),
                "adapters' input gradient");
        } else {
          check(pq_adapter_down(dy.const_data_ptr(), code, z.M, z.N, stride_of(dy), f, z.slots, z.P, ids.const_data_ptr(), z.id_bits, z.each, dt_parts, stream),
                "adapters' dt");
          check(pq_adapter_up(dt_parts, pq_adapter_slices(z.M, z.N), data<float>(scale), g, z.slots, z.K, z.R, z.P, ids.const_data_ptr(), z.id_bits,
                              z.each, nullptr, 0, data<void>(out[0]), z.K, dt, code, z.M, stream),
                "adapters' input gradient");
        }
      }
      if (want_A || want_B)
        check(pq_adapter_grads(x.defined() ? x.const_data_ptr() : nullptr, x.defined() ? stride_of(x) : z.K, dy.const_data_ptr(), stride_of(dy), code,
                               data<float>(kept), dt, ids.const_data_ptr(), z.id_bits, z.each, z.M, z.K, z.N, z.slots, z.R, z.P,
                               data<void>(out[3]), data<void>(out[4]), s + parts + ap + bp, ws, stream),
              "adapters' factor gradients");
    } catch (const Refused& r) {
      throw std::runtime_error(r.text);
    }
    if (at::GradMode::is_enabled()) once(out, grads[0]);
    return out;
  }

  // The gradients of a pass with create_graph: each gets edges to what it depends on, through a node that raises. (What the kernels write
  // has no history: without this it would count as a constant wherever it is differentiated.)
  static void once(variable_list& out, const Tensor& dy) {
    const torch::autograd::edge_list& in = torch::autograd::get_current_node()->next_edges();   // x, y, ids, lr_A, lr_B, scale
    const torch::autograd::Edge back = dy.requires_grad() ? torch::autograd::impl::gradient_edge(dy) : torch::autograd::Edge();
    const std::pair<int, torch::autograd::edge_list> on[3] = {{0, {back, in[3], in[4]}}, {3, {back, in[4], in[0]}}, {4, {back, in[3], in[0]}}};
    for (const auto& [i, list] : on) {
      torch::autograd::edge_list edges;
      for (const auto& e : list)
        if (e.is_valid()) edges.push_back(e);
      if (out[i].defined() && !edges.empty())
        torch::autograd::set_history(out[i], std::make_shared<torch::autograd::Error>("adapters have no second derivatives", std::move(edges)));
    }
  }
};

bool tensor_arg(PyObject* o, bool optional, const char* name, Tensor& t) {
  if (optional && o == Py_None) return true;
  if (!THPVariable_Check(o)) {
    PyErr_Format(PyExc_TypeError, "%s is no tensor", name);
    return false;
  }
  t = THPVariable_Unpack(o);
  return true;
}

std::pair<uintptr_t, uintptr_t> span(const Tensor& t) {
  int64_t last = 0;
  for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
  const uintptr_t at = (uintptr_t)t.const_data_ptr();
  return {at, t.numel() ? at + (last + 1) * t.element_size() : at};
}
bool meet(const Tensor& a, const Tensor& b) {
  const auto s = span(a), t = span(b);
  return s.first < t.second && t.first < s.second;
}

// Whether the gradient of t's leaf (t, or what t is a view or a cast of) would be accumulated on another stream than the current one: a graph that
// was made there lives.
bool elsewhere(const Tensor& t) {
  if (!t.defined() || !t.requires_grad()) return false;
  std::shared_ptr<torch::autograd::Node> node = t.grad_fn();
  if (!node) node = torch::autograd::impl::try_get_grad_accumulator(t);
  for (int i = 0; i < 8 && node; ++i) {
    if (dynamic_cast<torch::autograd::AccumulateGrad*>(node.get())) {
      const std::optional<c10::Stream> at = node->stream();
      return at && *at != c10::impl::VirtualGuardImpl(t.device().type()).getStream(t.device());
    }
    if (node->num_outputs() != 1) return false;
    node = node->next_edge(0).function;
  }
  return false;
}

// What the kernels need, as AssertionError.
const char* wrong(const Tensor& x, const Tensor& y, const Tensor& ids, const Tensor& A, const Tensor& B, const Tensor& scale, int64_t R,
                  bool laid_out, const Tensor& out) {
  if (!x.is_cuda()) return "adapters run on the GPU only (got a CPU tensor)";
  for (const Tensor* t : {&y, &ids, &A, &B, &scale, &out})
    if (t->defined() && t->device() != x.device()) return "operands on different devices";
  if (x.dim() < 1 || y.dim() != x.dim() || A.dim() != 3 || B.dim() != 3) return "x and y have the same leading dimensions, lr_A and lr_B three";
  for (int64_t d = 0; d + 1 < x.dim(); ++d)
    if (y.size(d) != x.size(d)) return "x and y have the same leading dimensions";
  const int64_t K = x.size(-1), N = y.size(-1), slots = A.size(0);
  if (K < 8 || K % 8 || N < 8 || N % 8) return "in_features and out_features are multiples of 8";
  if (R < 1 || R > 64) return "adapters have ranks of 1 to 64";
  if (slots < 1 || slots > 65535 || B.size(0) != slots) return "lr_A and lr_B hold the same adapters, 1 to 65535";
  const int64_t P = padded(R);
  if (laid_out ? A.size(1) != (K + 127) / 128 * 128 || A.size(2) != P || B.size(1) != (N + 127) / 128 * 128 || B.size(2) != P || !A.is_contiguous() || !B.is_contiguous() ||
                     (uintptr_t)A.const_data_ptr() % 16 || (uintptr_t)B.const_data_ptr() % 16
               : A.size(1) != K || A.size(2) != R || B.size(1) != R || B.size(2) != N)
    return "lr_A and lr_B do not fit x and y";
  if (scale.scalar_type() != at::kFloat || scale.dim() != 1 || scale.size(0) != slots || !scale.is_contiguous()) return "scale is contiguous fp32 [slots]";
  if (ids.dim() > x.dim() - 1) return "ids have some of x's leading dimensions";
  if (x.dim() == 2 && ids.dim() == 1) {   // rows, or requests of equally many rows end to end
    if (ids.size(0) != x.size(0) && (!ids.size(0) || !x.size(0) || x.size(0) % ids.size(0))) return "ids are one for each row, or for each request of as many rows";
  } else {
    for (int64_t d = 0; d < ids.dim(); ++d)
      if (ids.size(d) != x.size(d)) return "ids have some of x's leading dimensions";
  }
  if (out.defined()) {
    if (out.sizes() != y.sizes()) return "out has another shape than y";
    if (!out.is_contiguous()) return "out must be contiguous";
    if ((uintptr_t)out.const_data_ptr() % 16) return "out must be 16-byte aligned";
    const bool same = out.const_data_ptr() == y.const_data_ptr() && y.is_contiguous() && !y.is_neg();
    if (out.is_neg() || meet(out, x) || (meet(out, y) && !same) || meet(out, A) || meet(out, B) || meet(out, ids) || meet(out, scale))
      return "out shares memory with an operand (it may be y itself)";
  }
  return nullptr;
}

PyObject* adapt(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 9) {
    PyErr_SetString(PyExc_TypeError, "adapt(x, y, ids, lr_A, lr_B, scale, rank, laid_out, out)");
    return nullptr;
  }
  Tensor x, y, ids, A, B, scale, out;
  if (!tensor_arg(args[0], false, "x", x) || !tensor_arg(args[1], false, "y", y) || !tensor_arg(args[2], false, "ids", ids) ||
      !tensor_arg(args[3], false, "lr_A", A) || !tensor_arg(args[4], false, "lr_B", B) || !tensor_arg(args[5], false, "scale", scale) ||
      !tensor_arg(args[8], true, "out", out))
    return nullptr;
  const int64_t R = PyLong_AsLongLong(args[6]);
  const int laid_out = PyObject_IsTrue(args[7]);
  if ((R == -1 && PyErr_Occurred()) || laid_out < 0) return nullptr;
  if (x.is_cuda() && x.scalar_type() != at::kBFloat16 && x.scalar_type() != at::kHalf) {
    PyErr_SetString(PyExc_ValueError, "x must be bfloat16 or float16");
    return nullptr;
  }
  for (const Tensor* t : {&y, &A, &B, &out})
    if (x.is_cuda() && t->defined() && t->scalar_type() != x.scalar_type()) {
      PyErr_SetString(PyExc_ValueError, "x, y and the factors must be of one type");
      return nullptr;
    }
  if (ids.scalar_type() != at::kInt && ids.scalar_type() != at::kLong) {
    PyErr_SetString(PyExc_ValueError, "ids must be int32 or int64");
    return nullptr;
  }
  if (const char* const text = wrong(x, y, ids, A, B, scale, R, laid_out != 0, out)) {
    PyErr_SetString(PyExc_AssertionError, text);
    return nullptr;
  }
  for (const Tensor* t : {&x, &y, &A, &B, &scale, &out})
    if (t->defined() && t->_fw_grad(0).defined()) {
      PyErr_SetString(PyExc_RuntimeError, "adapters have no forward-mode derivatives");
      return nullptr;
    }
  const bool any = at::GradMode::is_enabled() && (x.requires_grad() || y.requires_grad() || A.requires_grad() || B.requires_grad());
  const char* refused = nullptr;
  if (at::GradMode::is_enabled() && scale.requires_grad()) refused = "scale has no gradient";
  else if (at::GradMode::is_enabled() && laid_out && (A.requires_grad() || B.requires_grad()))
    refused = "frozen adapters, in the kernels' order, have no gradients (trainable=True tunes them)";
  else if (out.defined() && (any || (at::GradMode::is_enabled() && out.requires_grad())))
    refused = "out is for calls without gradients";
  if (refused) {
    PyErr_SetString(PyExc_AssertionError, refused);
    return nullptr;
  }
  // A captured backward pass would wait for that stream, which is not captured, in autograd's own thread: the process would end there.
  if (any && c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None &&
      (elsewhere(x) || elsewhere(y) || elsewhere(A) || elsewhere(B))) {
    PyErr_SetString(PyExc_RuntimeError, "a graph of the same leaves that was made outside the capture lives: drop its results before a step is captured");
    return nullptr;
  }
  Tensor result;
  int status = PQ_OK;
  std::string text;
  {
    pybind11::gil_scoped_release release;
    try {
      const c10::DeviceGuard guard(x.device());
      const int64_t K = x.size(-1), N = y.size(-1), M = x.numel() / K;
      const Tensor x2 = x.dim() == 2 ? x : x.reshape({M, K}), y2 = y.dim() == 2 ? y : y.reshape({M, N});
      const Tensor i2 = ids.is_contiguous() ? ids : ids.contiguous();
      const Tensor o2 = !out.defined() || out.dim() == 2 ? out : out.view({M, N});
      const Sizes z{M, K, N, A.size(0), R, padded(R), std::max<int64_t>(M / std::max<int64_t>(ids.numel(), 1), 1), ids.scalar_type() == at::kLong ? 64 : 32};
      if (any) {
        result = Adapt::apply(x2, y2, i2, A, B, scale, std::vector<int64_t>{z.M, z.K, z.N, z.slots, z.R, z.P, z.each, z.id_bits}, laid_out != 0);
      } else {
        Kept kept;
        result = run(x2, y2, i2, A, B, scale, z, laid_out != 0, o2, {false, false, false}, kept);
      }
      if (out.defined()) {
        if (!out.is_inference()) out.unsafeGetTensorImpl()->bump_version();
        result = out;
      } else if (y.dim() != 2) {
        result = result.reshape(y.sizes());
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
  return THPVariable_Wrap(std::move(result));
  END_HANDLE_TH_ERRORS
}

template <typename F>
PyCFunction fast(F* f) { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(f)); }
PyMethodDef kMethods[] = {
    {"adapt", fast(adapt), METH_FASTCALL,
     "adapt(x, y, ids, lr_A, lr_B, scale, rank, laid_out, out): y + scale[id] (x lr_A[id]) lr_B[id], differentiable"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_adapt", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__adapt() { return PyModule_Create(&kModule); }
