// The optimizer's side of tuning without Python between a step and the kernels: pyraquant_amd._tune.
//
//   Plan(params, bits)                      the states of a parameter group, and the list of its tensors in device memory
//   step([(plan, lr, b1, b2, eps, wd, seed), ...], max_norm) -> the gradients' norm, or None (max_norm 0: no limit)
//
// Gradients are collected anew each step; the list is built again where a parameter has moved. Work goes to the current stream of
// the parameters' device.
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/utils/pybind.h>

#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <ATen/ops/zeros.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/StreamGuard.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>
#include <optional>

#include "../../include/pyraquant_amd.h"

namespace {

namespace py = pybind11;
using at::Tensor;

[[noreturn]] void refuse(PyObject* type, const std::string& text) {
  PyErr_SetString(type, text.c_str());
  throw py::error_already_set();
}
void need(bool ok, const std::string& text) {
  if (!ok) refuse(PyExc_AssertionError, text);
}
void check(int status, const char* what) {
  if (status == PQ_OK) return;
  refuse(status == PQ_EDTYPE ? PyExc_ValueError : status == PQ_ELAUNCH ? PyExc_RuntimeError : PyExc_AssertionError,
         std::string(what) + ": " + pq_last_error());
}
int32_t code_of(at::ScalarType t) {
  if (t == at::kBFloat16) return PQ_BF16;
  if (t == at::kHalf) return PQ_F16;
  if (t == at::kFloat) return PQ_F32;
  refuse(PyExc_ValueError, "unsupported dtype (expected bfloat16, float16 or float32)");
}
hipStream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
c10::Stream current(at::Device d) { return c10::impl::VirtualGuardImpl(d.type()).getStream(d); }
bool capturing() { return c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None; }
template <typename T>
T* data(const Tensor& t) { return t.defined() ? static_cast<T*>(const_cast<void*>(t.const_data_ptr())) : nullptr; }

class Plan {
 public:
  Plan(const std::vector<Tensor>& params, int bits) : params_(params), bits_(bits), device_(params.empty() ? at::Device(at::kCPU) : params[0].device()) {
    need(bits == 8 || bits == 32, "states have 8 or 32 bits (got " + std::to_string(bits) + ")");
    need(!params.empty(), "a parameter group without parameters");
    first_.push_back(0);
    if (device_.is_cuda()) home_ = current(device_);
    for (const Tensor& p : params) {
      need(p.is_cuda(), "the optimizer runs on the GPU only (got a CPU tensor)");
      need(p.device() == params[0].device(), "a parameter group lies on one device");
      need(p.layout() == at::kStrided && p.is_non_overlapping_and_dense(), "parameters must be dense");
      need(!p.is_neg() && !p.is_conj(), "parameters must hold their values");
      code_of(p.scalar_type());
      offsets_.push_back(n_);
      sizes_.push_back(p.numel());
      n_ += (p.numel() + PQ_ADAMW_BLOCK - 1) / PQ_ADAMW_BLOCK * PQ_ADAMW_BLOCK;
      first_.push_back(first_.back() + (p.numel() + PQ_ADAMW_CHUNK - 1) / PQ_ADAMW_CHUNK);
    }
    need(first_.back() < (1 << 30), "a parameter group holds at most 2^40 values");
    list();
    const c10::DeviceGuard guard(params[0].device());
    const c10::StreamGuard stream(*home_);
    const auto opt = at::TensorOptions().device(params[0].device());
    m_ = at::zeros({n_}, opt.dtype(bits == 8 ? at::kByte : at::kFloat));
    v_ = at::zeros({n_}, m_.options());
    if (bits == 8) exps_ = at::zeros({n_ / PQ_ADAMW_BLOCK, 2}, opt.dtype(at::kByte));
    steps_ = at::zeros({first_.back()}, opt.dtype(at::kInt));
  }

  // Whether this is the plan of these parameters (the objects; where they lie may change), and `state` still holds what was given out for each: in
  // their order, as give() and its caller put them there.
  bool holds(py::handle params, int bits, py::handle state) const {
    if (!PyList_Check(params.ptr()) || PyList_GET_SIZE(params.ptr()) != (Py_ssize_t)params_.size() || bits != bits_) return false;
    for (size_t i = 0; i < params_.size(); ++i) {
      PyObject* const o = PyList_GET_ITEM(params.ptr(), i);
      if (!THPVariable_Check(o) || THPVariable_Unpack(o).unsafeGetTensorImpl() != params_[i].unsafeGetTensorImpl()) return false;
    }
    if (!PyDict_Check(state.ptr()) || given_.size() != params_.size()) return false;
    size_t k = 0;
    Py_ssize_t at = 0;
    for (PyObject *key, *value; k < given_.size() && PyDict_Next(state.ptr(), &at, &key, &value);)
      k += key == PyList_GET_ITEM(params.ptr(), k) && value == given_[k].ptr();
    return k == given_.size();
  }
  // What the caller puts into the optimizer's state for each parameter.
  void give(std::vector<py::object> given) { given_ = std::move(given); }

  // This step's gradients; copies of those that lie in another order than their parameter.
  void collect() {
    grads_.assign(params_.size(), nullptr);
    copies_.clear();
    bool moved = false;
    for (size_t i = 0; i < params_.size(); ++i) {
      const Tensor& p = params_[i];
      moved |= p.const_data_ptr() != at_[i] || p.numel() != sizes_[i] || p.scalar_type() != types_[i] || p.device() != device_ ||
               !p.is_non_overlapping_and_dense();
      const Tensor& g = p.grad();
      if (!g.defined()) continue;
      if (g.layout() != at::kStrided) refuse(PyExc_RuntimeError, "sparse gradients are not supported");
      if (g.scalar_type() != p.scalar_type()) refuse(PyExc_ValueError, "a gradient of another type than its parameter");
      need(g.device() == p.device() && g.sizes() == p.sizes(), "a gradient of another shape or on another device than its parameter");
      Tensor d = g;
      if (g.is_neg() || !((p.is_contiguous() && g.is_contiguous()) || g.strides() == p.strides())) {
        const c10::DeviceGuard guard(p.device());
        d = at::empty_like(p, p.options().requires_grad(false)).copy_(g.detach());
        copies_.push_back(d);
      }
      grads_[i] = d.const_data_ptr();
    }
    if (moved) list();   // (after the checks: a step that is refused changes nothing)
  }

  pq_adamw_list c_list() const {
    return {data<pq_adamw_tensor>(tensors_), data<int32_t>(chunks_), first_.data(), grads_.data(), (int64_t)params_.size()};
  }
  pq_adamw_states c_states() const { return {m_.data_ptr(), v_.data_ptr(), data<uint8_t>(exps_), data<int32_t>(steps_), n_, bits_}; }
  // Autograd learns that the parameters have changed.
  void changed() {
    for (size_t i = 0; i < params_.size(); ++i)
      if (grads_[i] && !params_[i].is_inference()) params_[i].unsafeGetTensorImpl()->bump_version();
    copies_.clear();
  }

  // What is the plan's own is on the current stream until the work there is done, and in a captured graph for good: a list that such
  // a graph reads stays, with the memory of the parameters that it names and of the rate.
  void used(const Tensor& rate = Tensor()) {
    if (capturing()) {
      captured_ = true;
      auto hold = [&](const Tensor& t) {
        if (held_.empty() || held_.back().unsafeGetStorageImpl() != t.storage().unsafeGetStorageImpl()) held_.push_back(t.storage());
      };
      if (!holds_params_) std::for_each(params_.begin(), params_.end(), hold);
      holds_params_ = true;
      if (rate.defined()) hold(rate);
      return;
    }
    const c10::Stream now = current(device_);
    if (now != *home_)
      for (const Tensor* t : {&tensors_, &chunks_, &m_, &v_, &exps_, &steps_})
        if (t->defined()) t->record_stream(now);
  }
  bool captured() const { return captured_; }

  std::pair<Tensor, Tensor> moments(at::ScalarType type) {
    const int32_t code = code_of(type);
    const c10::DeviceGuard guard(m_.device());
    const Tensor m = at::empty({n_}, m_.options().dtype(type)), r = at::empty({n_}, m_.options().dtype(type));
    const pq_adamw_states s = c_states();
    check(pq_adamw_moments(&s, m.data_ptr(), r.data_ptr(), code, stream_of(m_)), "moments");
    used();
    return {m, r};
  }
  void load(const Tensor& mean, const Tensor& root, int64_t steps) {
    for (const Tensor* t : {&mean, &root}) {
      need(t->device() == m_.device() && t->dim() == 1 && t->numel() == n_, "moments are flat tensors of " + std::to_string(n_) +
                                                                           " values on the parameters' device");
      code_of(t->scalar_type());
    }
    need(steps >= 0 && steps < INT32_MAX, "steps must be 0 or more");
    const c10::DeviceGuard guard(m_.device());
    auto plain = [](const Tensor& t) {
      Tensor f = t.detach().to(at::kFloat).resolve_neg().contiguous();
      return (uintptr_t)f.const_data_ptr() % 16 ? f.clone() : f;
    };
    const Tensor a = plain(mean), b = plain(root);
    const pq_adamw_states s = c_states();
    check(pq_adamw_load(&s, data<float>(a), data<float>(b), stream_of(m_)), "load_moments");
    steps_.fill_(steps);
    used();
  }

  const Tensor& like() const { return m_; }
  py::tuple states() const { return bits_ == 8 ? py::make_tuple(m_, v_, exps_) : py::make_tuple(m_, v_); }
  // What belongs to parameter i: its counts, its values of m and v, and its blocks' exponents (or None)
  py::tuple of(int64_t i) const {
    need(i >= 0 && i < (int64_t)params_.size(), "no such parameter");
    const int64_t at = offsets_[i], n = sizes_[i];
    const py::object exps = exps_.defined() ? py::cast(exps_.slice(0, at / PQ_ADAMW_BLOCK, (at + n + PQ_ADAMW_BLOCK - 1) / PQ_ADAMW_BLOCK))
                                            : py::object(py::none());
    return py::make_tuple(steps_.slice(0, first_[i], first_[i + 1]), m_.slice(0, at, at + n), v_.slice(0, at, at + n), exps);
  }
  const std::vector<int64_t>& offsets() const { return offsets_; }

 private:
  // The list of tensors and chunks in device memory, from where the parameters lie now and what they are. (at_ and types_ are those of the
  // list: they change with it, or where anything is refused neither does.)
  void list() {
    if (capturing())
      refuse(PyExc_RuntimeError, "the optimizer's first step, and the first after its parameters moved, cannot be captured: take one before");
    std::vector<pq_adamw_tensor> t(params_.size());
    std::vector<int32_t> chunks((size_t)first_.back());
    std::vector<std::pair<uintptr_t, uintptr_t>> spans;
    std::vector<const void*> places(params_.size());
    std::vector<at::ScalarType> types(params_.size());
    for (size_t i = 0; i < params_.size(); ++i) {
      const Tensor& p = params_[i];
      need(p.numel() == sizes_[i] && p.is_non_overlapping_and_dense(), "a parameter has changed its size, or is not dense any more");
      need(p.device() == device_, "a parameter has left the device that its states are on");
      places[i] = p.const_data_ptr();
      types[i] = p.scalar_type();
      t[i] = {const_cast<void*>(places[i]), sizes_[i], offsets_[i], code_of(types[i]), (int32_t)first_[i]};
      std::fill(chunks.begin() + first_[i], chunks.begin() + first_[i + 1], (int32_t)i);
      if (sizes_[i]) spans.emplace_back((uintptr_t)places[i], (uintptr_t)places[i] + p.numel() * p.element_size());
    }
    std::sort(spans.begin(), spans.end());
    for (size_t i = 1; i < spans.size(); ++i) need(spans[i].first >= spans[i - 1].second, "two parameters of a group share memory");
    const c10::DeviceGuard guard(params_[0].device());
    const c10::StreamGuard stream(*home_);
    auto up = [&](const void* from, int64_t bytes) {
      Tensor host = at::empty({std::max<int64_t>(bytes, 1)}, at::TensorOptions().dtype(at::kByte));
      std::copy_n(static_cast<const uint8_t*>(from), bytes, data<uint8_t>(host));
      return host.to(params_[0].device());   // (waits: the host's copy goes away)
    };
    const Tensor tensors = up(t.data(), (int64_t)(t.size() * sizeof(pq_adamw_tensor)));
    const Tensor its_chunks = up(chunks.data(), (int64_t)(chunks.size() * sizeof(int32_t)));
    if (captured_) kept_.insert(kept_.end(), {tensors_, chunks_});
    holds_params_ = false;
    tensors_ = tensors, chunks_ = its_chunks, at_ = std::move(places), types_ = std::move(types);
  }

  std::vector<Tensor> params_, copies_, kept_;
  std::vector<c10::Storage> held_;    // what graphs go on with beside kept_
  std::optional<c10::Stream> home_;   // where all that is the plan's own was allocated
  bool captured_ = false, holds_params_ = false;   // (the parameters of this list)
  int bits_;
  at::Device device_;
  int64_t n_ = 0;
  std::vector<int64_t> offsets_, sizes_, first_;
  std::vector<const void*> at_, grads_;
  std::vector<at::ScalarType> types_;
  Tensor tensors_, chunks_, m_, v_, exps_, steps_;
  std::vector<py::object> given_;
};

py::object step(const py::list& groups, double max_norm) {
  need(max_norm >= 0, "max_norm must be above 0");
  struct Group {
    Plan* plan;
    pq_adamw_rates rates;
    Tensor rate;   // in device memory, or none
  };
  std::vector<Group> all;
  for (const py::handle h : groups) {
    const py::tuple t = py::reinterpret_borrow<py::tuple>(h);
    Group g{t[0].cast<Plan*>(), {}, {}};
    if (THPVariable_Check(t[1].ptr())) {
      const Tensor lr = THPVariable_Unpack(t[1].ptr());
      need(lr.numel() == 1, "lr is one number");
      if (lr.is_cuda() && lr.scalar_type() == at::kFloat && lr.device() == g.plan->like().device()) g.rate = lr, g.rates.lr_at = data<float>(lr);
      else g.rates.lr = lr.item().toDouble();
    } else {
      g.rates.lr = t[1].cast<double>();
    }
    g.rates.beta1 = t[2].cast<double>(), g.rates.beta2 = t[3].cast<double>();
    g.rates.eps = t[4].cast<double>(), g.rates.weight_decay = t[5].cast<double>();
    g.rates.seed = (uint32_t)t[6].cast<int64_t>();
    g.rates.max_norm = max_norm;
    const pq_adamw_rates& r = g.rates;   // (checked for all groups before any is stepped)
    need((r.lr_at || r.lr >= 0) && r.beta1 >= 0 && r.beta1 < 1 && r.beta2 >= 0 && r.beta2 < 1 && r.eps >= 0 && r.weight_decay >= 0,
         "lr, eps and weight_decay must be 0 or more, betas in [0, 1)");
    need(!max_norm || all.empty() || all[0].plan->like().device() == g.plan->like().device(),
         "a limit on the norm of gradients on several devices is not supported");
    g.plan->collect();
    all.push_back(g);
  }
  Tensor norm, partials;
  std::vector<int64_t> sums;
  int64_t n_partials = 0;
  if (max_norm && !all.empty()) {
    const c10::DeviceGuard guard(all[0].plan->like().device());
    int64_t total = 0;
    for (const Group& g : all) {
      const pq_adamw_list l = g.plan->c_list();
      sums.push_back(pq_grad_squares_partials(&l));
      total += sums.back();
    }
    norm = at::empty({}, all[0].plan->like().options().dtype(at::kFloat));
    if (total) {
      const bool join = total > 512;   // a place for their sum, in front
      partials = at::empty({total + join}, norm.options().dtype(at::kDouble));
      double* to = data<double>(partials) + join;
      for (size_t i = 0; i < all.size(); to += sums[i++]) {
        const pq_adamw_list l = all[i].plan->c_list();
        check(pq_grad_squares(&l, to, sums[i], stream_of(norm)), "AdamW");
      }
      n_partials = total;
      if (join) {
        check(pq_grad_squares_join(data<double>(partials) + 1, total, data<double>(partials), stream_of(norm)), "AdamW");
        n_partials = 1;
      }
    }
  }
  if (norm.defined() && !n_partials) norm.zero_();   // no gradient at all
  for (const Group& g : all) {
    const c10::DeviceGuard guard(g.plan->like().device());
    const pq_adamw_list l = g.plan->c_list();
    const pq_adamw_states s = g.plan->c_states();
    check(pq_adamw_step(&l, &s, &g.rates, data<double>(partials), n_partials, data<float>(norm),
                        stream_of(g.plan->like())),
          "AdamW");
    g.plan->used(g.rate);
    g.plan->changed();
  }
  return norm.defined() ? py::cast(norm) : py::object(py::none());
}

}  // namespace

PYBIND11_MODULE(_tune, m) {
  py::class_<Plan>(m, "Plan")
      .def(py::init<const std::vector<Tensor>&, int>())
      .def("holds", &Plan::holds)
      .def("give", &Plan::give)
      .def("captured", &Plan::captured)
      .def("states", &Plan::states)
      .def("of", &Plan::of)
      .def("offsets", &Plan::offsets)
      .def("moments", [](Plan& p, py::handle dtype) {
        if (!THPDtype_Check(dtype.ptr())) refuse(PyExc_TypeError, "moments(dtype)");
        return p.moments(reinterpret_cast<THPDtype*>(dtype.ptr())->scalar_type);
      })
      .def("load", &Plan::load);
  m.def("step", &step);
}
