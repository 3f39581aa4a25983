// Torch binding of the optimizer kernels (csrc/kernels/adamw.hip): collects
// the tensors' pointers, checks what the kernels assume of them, and launches
// on the current stream of the tensors' own device.
#include <torch/extension.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPException.h>
#include <c10/hip/HIPStream.h>
#include <algorithm>
#include <memory>
#include <numeric>
#include <unordered_set>
#include <vector>

#include "kernels/train_api.h"

namespace {

hipStream_t stream_now() {
  return c10::hip::getCurrentHIPStream().stream();
}

int code_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return 0;
    case at::kBFloat16: return 1;
    case at::kHalf: return 2;
    default:
      TORCH_CHECK(false, "expected float32, bfloat16 or float16, got ", t);
  }
}

bool dense(const at::Tensor& t) {
  return t.unsafeGetTensorImpl()->is_non_overlapping_and_dense();
}

// The same place of every element in memory (strides of sides of length one
// say nothing).
bool same_layout(const at::Tensor& a, const at::Tensor& b) {
  if (a.sizes() != b.sizes()) return false;
  for (int64_t d = 0; d < a.dim(); ++d)
    if (a.size(d) > 1 && a.stride(d) != b.stride(d)) return false;
  return true;
}

// What a kernel wrote: autograd's saved tensors are told, as of torch's own
// updates.
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// False for a tensor whose storage was freed, and for autograd's zeros that
// were never made: a kernel would read from address 0.
bool has_memory(const at::Tensor& t) {
  return t.numel() == 0 || t.storage().data() != nullptr;
}

void check_grad(const at::Tensor& g) {
  TORCH_CHECK(g.layout() == at::kStrided,
              "sparse gradients are not supported");
  TORCH_CHECK(has_memory(g), "a gradient has no memory");
}

// The parameters of one group that share a device and a dtype, with their
// states.  An undefined state tensor marks a parameter that had no gradient
// yet.
class AdamWPlan {
 public:
  using Tensors = std::vector<at::Tensor>;
  using Maybe = std::vector<c10::optional<at::Tensor>>;

  AdamWPlan(Tensors params, Maybe masters, Maybe m, Maybe v, Maybe ms,
            Maybe vs, Maybe steps, std::vector<int64_t> indices, int64_t bits)
      : params_(std::move(params)), indices_(std::move(indices)),
        bits_((int)bits) {
    const size_t n = params_.size();
    TORCH_CHECK(n > 0, "no parameters");
    TORCH_CHECK(masters.size() == n && m.size() == n && v.size() == n &&
                    ms.size() == n && vs.size() == n && steps.size() == n &&
                    indices_.size() == n,
                "one state entry a parameter");
    TORCH_CHECK(bits_ == 8 || bits_ == 32, "state_bits is 8 or 32");
    device_ = params_[0].device();
    dtype_ = params_[0].scalar_type();
    const bool wants_master = code_of(dtype_) != 0;
    std::unordered_set<const void*> seen;
    for (size_t i = 0; i < n; ++i) {
      const at::Tensor& p = params_[i];
      TORCH_CHECK(p.is_cuda(), "parameters of a plan are on a GPU");
      TORCH_CHECK(p.device() == device_ && p.scalar_type() == dtype_,
                  "parameters of a plan share a device and a dtype");
      TORCH_CHECK(dense(p), "parameter ", indices_[i],
                  " is not dense in memory: the update runs over storage");
      TORCH_CHECK(p.numel() == 0 || seen.insert(p.unsafeGetTensorImpl()).second,
                  "parameter ", indices_[i], " appears twice in its group");
      State s;
      if (steps[i].has_value()) {
        const auto kind = bits_ == 8 ? at::kByte : at::kFloat;
        s.step = checked(*steps[i], at::kFloat, "step");
        TORCH_CHECK(s.step.numel() == 1, "step holds one number");
        s.m = state(m[i], p, kind, "exp_avg");
        s.v = state(v[i], p, kind, "exp_avg_sq");
        if (wants_master)
          s.master = state(masters[i], p, at::kFloat, "master");
        if (bits_ == 8) {
          const int64_t blocks =
              (p.numel() + DDL_MOMENT_BLOCK - 1) / DDL_MOMENT_BLOCK;
          s.ms = scales(ms[i], blocks, "exp_avg_scale");
          s.vs = scales(vs[i], blocks, "exp_avg_sq_scale");
        }
      }
      states_.push_back(std::move(s));
    }
    settle();
    // A launch takes so many tensors: the largest come first, so that all
    // launches but one are short.
    order_.resize(n);
    std::iota(order_.begin(), order_.end(), 0);
    std::stable_sort(order_.begin(), order_.end(), [&](int64_t a, int64_t b) {
      return params_[a].numel() > params_[b].numel();
    });
  }

  // Reads the gradients as they are now.  Lazily negated ones, and those laid
  // out unlike their parameter, are copied first.  Returns the places (in this
  // plan) of parameters with a gradient and no state.
  std::vector<int64_t> collect() {
    c10::DeviceGuard guard(device_);
    forget();
    moved_ = false;
    std::vector<int64_t> missing;
    for (const int64_t i : order_) {
      const at::Tensor& p = params_[i];
      const at::Tensor& grad = p.grad();
      if (!grad.defined()) continue;
      const State& s = states_[i];
      if (!s.step.defined()) missing.push_back(i);
      if (!s.step.defined() || p.numel() == 0) continue;
      check_grad(grad);
      at::Tensor g = grad.is_neg() ? grad.resolve_neg() : grad;
      TORCH_CHECK(p.device() == device_ && p.scalar_type() == dtype_ &&
                      same_layout(p, s.m),
                  "parameter ", indices_[i],
                  " changed its device, dtype, shape or layout");
      TORCH_CHECK(has_memory(p), "parameter ", indices_[i], " has no memory");
      TORCH_CHECK(g.device() == device_ && g.scalar_type() == dtype_,
                  "the gradient of parameter ", indices_[i],
                  " differs from it in device or dtype");
      if (!same_layout(p, g)) {
        at::NoGradGuard no_grad;
        at::Tensor copy = at::empty_like(p);
        copy.copy_(g);
        g = copy;
      }
      DdlAdamTensor r{};
      const bool master = s.master.defined();
      r.p = master ? p.data_ptr() : nullptr;
      r.g = g.const_data_ptr();
      r.w = master ? s.master.data_ptr<float>() : (float*)p.data_ptr();
      r.m = s.m.data_ptr();
      r.v = s.v.data_ptr();
      r.ms = bits_ == 8 ? s.ms.data_ptr<float>() : nullptr;
      r.vs = bits_ == 8 ? s.vs.data_ptr<float>() : nullptr;
      if ((r.p ? r.p : r.w) != begins_[i]) moved_ = true;
      r.n = p.numel();
      r.step = s.step.data_ptr<float>();
      r.index = (uint32_t)indices_[i];
      rows_.push_back(r);
      places_.push_back(i);
      grads_.push_back(std::move(g));
    }
    return missing;
  }

  // Whether collect() saw a parameter at another place in memory than
  // settle() did, or the constructor.
  bool moved() const { return moved_; }

  void settle() {
    begins_.clear();
    for (const auto& p : params_) begins_.push_back(p.const_data_ptr());
  }

  std::vector<DdlGradTensor> grad_rows() const {
    std::vector<DdlGradTensor> out;
    for (const auto& r : rows_)
      out.push_back(DdlGradTensor{const_cast<void*>(r.g), r.n});
    return out;
  }

  // The update for what collect() saw; forgets the gradients afterwards.
  void step(const DdlAdamScalars& c, const DdlNormFold* fold,
            const float* coef) {
    c10::DeviceGuard guard(device_);
    const auto s = stream_now();
    const int64_t n = (int64_t)rows_.size();
    if (n) {
      at::Tensor ws = at::empty(
          {ddl_adamw_ws_bytes(n)},
          at::TensorOptions().dtype(at::kByte).device(device_));
      ddl_adamw_prepare(rows_.data(), n, &c, ws.data_ptr(), fold, s);
      ddl_adamw(rows_.data(), n, &c, code_of(dtype_), bits_, ws.data_ptr(),
                coef, s);
    } else if (fold) {
      ddl_grad_norm_fold(fold, s);
    }
    C10_HIP_KERNEL_LAUNCH_CHECK();
    for (const int64_t i : places_) written(params_[i]);
    forget();
  }

  c10::Device device() const { return device_; }
  int dtype() const { return code_of(dtype_); }

 private:
  struct State {
    at::Tensor master, m, v, ms, vs, step;
  };

  void forget() {
    rows_.clear();
    places_.clear();
    grads_.clear();
  }

  at::Tensor checked(const at::Tensor& t, at::ScalarType kind,
                     const char* name) const {
    TORCH_CHECK(t.device() == device_ && t.scalar_type() == kind, name,
                " is ", kind, " on the parameter's device");
    return t;
  }

  at::Tensor state(const c10::optional<at::Tensor>& t, const at::Tensor& p,
                   at::ScalarType kind, const char* name) const {
    TORCH_CHECK(t.has_value(), name, " is missing");
    TORCH_CHECK(same_layout(*t, p), name,
                " has another shape or layout than its parameter");
    return checked(*t, kind, name);
  }

  at::Tensor scales(const c10::optional<at::Tensor>& t, int64_t blocks,
                    const char* name) const {
    TORCH_CHECK(t.has_value(), name, " is missing");
    TORCH_CHECK(t->numel() == blocks && t->is_contiguous(), name, " holds ",
                blocks, " contiguous scales");
    return checked(*t, at::kFloat, name);
  }

  Tensors params_;
  std::vector<int64_t> indices_;
  int bits_;
  c10::Device device_{c10::kCPU};
  at::ScalarType dtype_;
  std::vector<State> states_;
  std::vector<int64_t> order_;  // places, the largest parameter first
  std::vector<const void*> begins_;  // of the parameters in memory
  bool moved_ = false;
  std::vector<int64_t> places_;  // of what collect() saw, as are these
  std::vector<DdlAdamTensor> rows_;
  Tensors grads_;
};

struct NormList {
  std::vector<DdlGradTensor> rows;
  int dtype;
};

// Partial sums of these lists, and where norm and coefficient go (0-dim
// float32 tensors); the fold is still to be launched.
struct Norm {
  at::Tensor partials, norm;  // the coefficient lies behind the partial sums
  DdlNormFold fold;
};

Norm norm_of(const std::vector<NormList>& lists, c10::Device device,
             double mul, double max_norm) {
  const auto s = stream_now();
  const auto opts = at::TensorOptions().device(device);
  Norm out;
  int64_t blocks = 0;
  for (const auto& l : lists)
    blocks += ddl_grad_norm_blocks(l.rows.data(), (int64_t)l.rows.size());
  out.partials =
      at::empty({blocks + 1}, opts.dtype(at::kDouble));
  out.norm = at::empty({}, opts.dtype(at::kFloat));
  double* at = out.partials.data_ptr<double>();
  for (const auto& l : lists) {
    const int64_t n = (int64_t)l.rows.size();
    ddl_grad_norm_partials(l.rows.data(), n, l.dtype, at, s);
    at += ddl_grad_norm_blocks(l.rows.data(), n);
  }
  out.fold = DdlNormFold{out.partials.data_ptr<double>(), blocks, mul,
                         max_norm, out.norm.data_ptr<float>(),
                         reinterpret_cast<float*>(
                             out.partials.data_ptr<double>() + blocks)};
  return out;
}

// (lr, beta1, beta2, eps, weight_decay, seed) of a plan's group
using Hyper = std::tuple<double, double, double, double, double, int64_t>;

// One step of all plans, which have collected their gradients.  max_norm 0:
// no clipping; otherwise returns the gradients' norm.
c10::optional<at::Tensor> adamw_step(
    const std::vector<std::shared_ptr<AdamWPlan>>& plans,
    const std::vector<Hyper>& hyper, double grad_mul, double max_norm) {
  TORCH_CHECK(plans.size() == hyper.size(), "numbers for each plan");
  Norm norm;
  const bool clip = max_norm != 0 && !plans.empty();
  if (clip) {
    std::vector<NormList> lists;
    for (const auto& p : plans) {
      TORCH_CHECK(p->device() == plans[0]->device(),
                  "clipping needs all parameters on one device");
      lists.push_back(NormList{p->grad_rows(), p->dtype()});
    }
    c10::DeviceGuard guard(plans[0]->device());
    norm = norm_of(lists, plans[0]->device(), grad_mul, max_norm);
  }
  for (size_t i = 0; i < plans.size(); ++i) {
    const auto& [lr, beta1, beta2, eps, decay, seed] = hyper[i];
    plans[i]->step(DdlAdamScalars{lr, beta1, beta2, eps, decay,
                                  (float)grad_mul, (uint32_t)seed},
                   clip && i == 0 ? &norm.fold : nullptr,
                   clip ? norm.fold.coef : nullptr);
  }
  if (!clip) return c10::nullopt;
  return norm.norm;
}

// The gradients of these parameters.
at::Tensor clip_grads(const std::vector<at::Tensor>& params, double grad_mul,
                      double max_norm) {
  std::vector<NormList> lists(3);
  for (int i = 0; i < 3; ++i) lists[i].dtype = i;
  std::vector<std::pair<const char*, const char*>> places;
  places.reserve(params.size());
  std::vector<const at::Tensor*> grads;
  grads.reserve(params.size());
  c10::optional<c10::Device> device;
  for (const auto& p : params) {
    const at::Tensor& g = p.grad();
    if (!g.defined()) continue;
    check_grad(g);
    if (!device.has_value()) device = g.device();
    TORCH_CHECK(g.is_cuda() && g.device() == *device,
                "all gradients are on one GPU");
    TORCH_CHECK(dense(g), "a gradient is not dense in memory");
    const int dtype = code_of(g.scalar_type());
    if (g.numel() == 0) continue;
    lists[dtype].rows.push_back(DdlGradTensor{g.data_ptr(), g.numel()});
    grads.push_back(&g);
    const char* start = static_cast<const char*>(g.const_data_ptr());
    places.emplace_back(start, start + g.nbytes());
  }
  std::sort(places.begin(), places.end());
  for (size_t i = 1; i < places.size(); ++i)
    TORCH_CHECK(places[i - 1].second <= places[i].first,
                "a gradient appears twice, or two share memory");
  TORCH_CHECK(device.has_value(), "no gradients");
  c10::DeviceGuard guard(*device);
  Norm norm = norm_of(lists, *device, grad_mul, max_norm);
  const bool fold =
      norm.fold.blocks > 0 && norm.fold.blocks <= DDL_FOLD_IN_SCALE;
  if (!fold) ddl_grad_norm_fold(&norm.fold, stream_now());
  for (const auto& l : lists)
    ddl_grad_scale(l.rows.data(), (int64_t)l.rows.size(), l.dtype, &norm.fold,
                   fold, stream_now());
  C10_HIP_KERNEL_LAUNCH_CHECK();
  for (const at::Tensor* g : grads) written(*g);
  return norm.norm;
}

}  // namespace

void bind_adamw(pybind11::module& m) {
  pybind11::class_<AdamWPlan, std::shared_ptr<AdamWPlan>>(m, "AdamWPlan")
      .def(pybind11::init<AdamWPlan::Tensors, AdamWPlan::Maybe,
                          AdamWPlan::Maybe, AdamWPlan::Maybe, AdamWPlan::Maybe,
                          AdamWPlan::Maybe, AdamWPlan::Maybe,
                          std::vector<int64_t>, int64_t>())
      .def("collect", &AdamWPlan::collect)
      .def("moved", &AdamWPlan::moved)
      .def("settle", &AdamWPlan::settle);
  m.def("adamw_step", &adamw_step);
  m.def("clip_grads", &clip_grads);
}
