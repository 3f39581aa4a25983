// Torch binding of the dense layer (csrc/kernels/linear*.hip): checks, packs
// operands whose rows do not begin at 4 bytes, allocates outputs and
// workspaces, and launches on the current stream of the tensors' device.  The
// autograd function is here too: in Python it would cost a small layer more
// time than its kernels.
#include <torch/extension.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPException.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/variable.h>

#include "kernels/linear_api.h"

namespace {

using Maybe = c10::optional<at::Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

hipStream_t stream_now() {
  return c10::hip::getCurrentHIPStream().stream();
}

int code_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return 0;
    case at::kBFloat16: return 1;
    case at::kHalf: return 2;
    default:
      TORCH_CHECK_TYPE(false, "x is float32, bfloat16 or float16, not ", t);
  }
}

// False for a tensor whose storage was freed, and for autograd's zeros that
// were never made: a kernel would read from address 0.
bool has_memory(const at::Tensor& t) {
  return t.numel() == 0 || t.storage().data() != nullptr;
}

constexpr int64_t LIMIT = (int64_t)1 << 29;

int64_t round_up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// A matrix whose columns are neighbours in memory; its rows may lie anywhere.
at::Tensor inner_contiguous(const at::Tensor& t) {
  return t.size(1) <= 1 || t.stride(1) == 1 ? t : t.contiguous();
}

// Elements from one row to the next; a single row has no say.
int64_t row_stride(const at::Tensor& t) {
  return t.size(0) > 1 ? t.stride(0) : t.size(1);
}

// Rows that the tiled kernel reads as they are: they begin at 4 bytes, and are
// no further apart than its 32-bit offsets inside a tile reach.
int64_t reach(const at::Tensor& t) {
  return ((int64_t)1 << 31) / 256 / t.element_size();
}

bool fits(const at::Tensor& t) {
  return (t.size(1) <= 1 || t.stride(1) == 1) &&
         (t.size(0) <= 1 || t.stride(0) * t.element_size() % 4 == 0) &&
         row_stride(t) < reach(t) && ((uintptr_t)t.const_data_ptr() & 3) == 0;
}

// The same matrices with rows padded by zeros to 16 bytes where they do not
// fit, in one launch.
void pack(at::Tensor* a, at::Tensor* b) {
  DdlPack todo[2];
  at::Tensor from[2];
  int count = 0, dtype = 0;
  for (at::Tensor* t : {a, b}) {
    if (t == nullptr || fits(*t)) continue;
    from[count] = inner_contiguous(*t);
    const at::Tensor& src = from[count];
    const int64_t wide = round_up(src.size(1), 8);
    TORCH_CHECK(wide < reach(src), "a matrix has ", src.size(1),
                " columns, the kernel's offsets reach ", reach(src));
    at::Tensor dst = at::empty({src.size(0), wide}, src.options());
    todo[count++] = DdlPack{src.const_data_ptr(), dst.data_ptr(),
                            row_stride(src), wide, src.size(0), src.size(1)};
    dtype = code_of(src.scalar_type());
    *t = dst;
  }
  if (count) ddl_pack_rows(todo, count, dtype, stream_now());
}

// out = epilogue(a b^T) with its workspace; `p` is planned, and holds something.
void product(DdlProduct& p, int64_t floats, const at::Tensor& like) {
  at::Tensor slabs;
  if (floats) {
    slabs = at::empty({floats}, like.options().dtype(at::kFloat));
    p.slabs = slabs.data_ptr<float>();
  }
  ddl_product(&p, stream_now());
}

// y = act(x w^T + bias) + residual, and z = x w^T + bias if asked for.  x and
// w are replaced by what the kernel read.
at::Tensor forward_of(at::Tensor& x, at::Tensor& w, const Maybe& bias,
                      const Maybe& residual, int64_t act, at::Tensor* z) {
  c10::DeviceGuard guard(x.device());
  const int64_t m = x.size(0), k = x.size(1), n = w.size(0);
  at::Tensor y = at::empty({m, n}, x.options());
  at::Tensor b, res;
  DdlProduct p{};
  p.dtype = code_of(x.scalar_type());
  p.act = (int)act;
  p.m = m;
  p.n = n;
  p.r = k;
  p.out = y.data_ptr();
  p.ldo = n;
  if (z) {
    // float32: z rounded to 16 bits would cost the gradients a third rounding
    // beside dz's and their own
    *z = at::empty({m, n}, x.options().dtype(at::kFloat));
    p.z = z->data_ptr<float>();
  }
  if (bias.has_value()) {
    b = bias->contiguous();
    p.bias = b.const_data_ptr();
  }
  if (residual.has_value()) {
    res = inner_contiguous(*residual);
    p.residual = res.const_data_ptr();
    p.ldres = row_stride(res);
  }
  if (m == 0 || n == 0) return y;
  const int64_t floats = ddl_product_plan(&p);
  const bool few = ddl_few_rows_pay(&p, fits(x) && fits(w));
  if (few) {
    x = inner_contiguous(x);
    w = inner_contiguous(w);
  } else {
    pack(&x, &w);
  }
  p.a = x.const_data_ptr();
  p.lda = row_stride(x);
  p.b = w.const_data_ptr();
  p.ldb = row_stride(w);
  if (few)
    ddl_product_few(&p, stream_now());
  else
    product(p, floats, x);
  C10_HIP_KERNEL_LAUNCH_CHECK();
  return y;
}

struct Grads {
  at::Tensor dx, dw, db;
};

// z: what the activation took, in float32 (its output, in x's dtype, does for
// ReLU); not looked at without an activation.  x and w may be padded copies of
// matrices with k columns.
// dy may be a lazy negation (autograd leaves them behind conjugates).
Grads backward_of(const at::Tensor& dy, at::Tensor x, at::Tensor w,
                  const at::Tensor& z, int64_t k, int64_t act, bool want_dx,
                  bool want_dw, bool want_db) {
  c10::DeviceGuard guard(x.device());
  const auto s = stream_now();
  const int64_t m = x.size(0), n = w.size(0);
  const int dtype = code_of(x.scalar_type());
  Grads out;
  if (want_dx) out.dx = at::empty({m, k}, x.options());
  if (want_dw) out.dw = at::empty({n, k}, x.options());
  if (want_db) out.db = at::empty({n}, x.options());
  if (m == 0 || n == 0 || k == 0) {  // sums over nothing
    for (auto* t : {&out.dx, &out.dw})
      if (t->defined()) t->zero_();
    if (want_db && m == 0) out.db.zero_();
  }
  if (m == 0 || n == 0) return out;

  at::Tensor d = inner_contiguous(dy.resolve_neg()), dz, zc;
  const bool products = k > 0 && (want_dx || want_dw);
  if (act) {
    zc = inner_contiguous(z);
    if (products) {
      TORCH_CHECK(round_up(n, 8) < reach(x), "the backward pass of ", n,
                  " outputs: the kernel's offsets reach ", reach(x));
      dz = at::empty({m, round_up(n, 8)}, x.options());
    }
  }
  DdlProduct px{}, pw{};
  int64_t fx = 0, fw = 0;
  bool small = false;
  if (products) {
    px.dtype = dtype;
    px.b_col = 1;
    px.n = k;
    px.ldo = k;
    pw = px;
    pw.a_col = 1;
    px.m = pw.r = m;
    px.r = pw.m = n;
    if (want_dx) fx = ddl_product_plan(&px);
    if (want_dw) fw = ddl_product_plan(&pw);
    small = want_dx && want_dw && ddl_small_backward(&px, &pw);
  }
  DdlBiasFold fold{};
  at::Tensor partials;
  if (want_db) {
    fold.n = n;
    fold.dbias = out.db.data_ptr();
    if (act || !small) {
      fold.chunks = ddl_bias_chunks(m, n);
      partials = at::empty({fold.chunks * n}, x.options().dtype(at::kFloat));
      fold.partials = partials.data_ptr<float>();
    }
  }
  if (fold.partials || dz.defined())
    ddl_act_bwd(d.const_data_ptr(), row_stride(d),
                act ? zc.const_data_ptr() : nullptr,
                act && zc.scalar_type() == at::kFloat,
                act ? row_stride(zc) : 0,
                dz.defined() ? dz.data_ptr() : nullptr,
                dz.defined() ? dz.size(1) : 0, m, n, (int)act, dtype,
                fold.partials ? partials.data_ptr<float>() : nullptr, s);
  if (products) {
    if (!act) {
      dz = d;
      pack(&dz, want_dx ? &w : nullptr);
      if (want_dw) pack(&x, nullptr);
    } else {
      pack(want_dx ? &w : nullptr, want_dw ? &x : nullptr);
    }
    px.a = pw.a = dz.const_data_ptr();
    px.lda = pw.lda = row_stride(dz);
    px.b = w.const_data_ptr();
    px.ldb = row_stride(w);
    pw.b = x.const_data_ptr();
    pw.ldb = row_stride(x);
    if (want_dx) px.out = out.dx.data_ptr();
    if (want_dw) pw.out = out.dw.data_ptr();
    if (small) {
      ddl_backward_small(&px, &pw, &fold, s);
      fold.n = 0;
    } else {
      if (want_dx) product(px, fx, x);
      if (want_dw) product(pw, fw, x);
    }
  }
  if (fold.n) ddl_fold_bias(&fold, dtype, s);
  C10_HIP_KERNEL_LAUNCH_CHECK();
  return out;
}

// Gradients that raise when they are differentiated again.
variable_list differentiable_once(variable_list grads) {
  for (auto& g : grads)
    if (g.defined()) g = g.detach().requires_grad_(true);
  auto error = std::make_shared<torch::autograd::DelayedError>(
      "linear_act is differentiable once", (int64_t)grads.size());
  return (*error)(std::move(grads));
}

class LinearAct : public torch::autograd::Function<LinearAct> {
 public:
  static at::Tensor forward(AutogradContext* ctx, at::Tensor x, at::Tensor w,
                            const Maybe& bias, const Maybe& residual,
                            int64_t act, bool wants_products) {
    // ReLU's output tells where its input was positive; with a residual on
    // top, and for the smooth activations, the input itself is kept
    const bool by_output = act == 1 && !residual.has_value();
    const bool want_z = act != 0 && !by_output && wants_products;
    ctx->saved_data["act"] = act;
    ctx->saved_data["k"] = x.size(1);
    ctx->saved_data["bias"] = bias.has_value();
    ctx->saved_data["residual"] = residual.has_value();
    at::Tensor z;
    at::Tensor y = forward_of(x, w, bias, residual, act, want_z ? &z : nullptr);
    ctx->save_for_backward({x, w, by_output ? y : z});
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list dys) {
    const auto saved = ctx->get_saved_variables();
    const at::Tensor& dy = dys[0];
    variable_list out(6);
    if (!dy.defined()) return out;
    const bool want_x = ctx->needs_input_grad(0);
    const bool want_w = ctx->needs_input_grad(1);
    // tensors that are not there are not counted
    const bool bias = ctx->saved_data["bias"].toBool();
    const bool residual = ctx->saved_data["residual"].toBool();
    const bool want_b = bias && ctx->needs_input_grad(2);
    const bool want_r = residual && ctx->needs_input_grad(bias ? 3 : 2);
    {
      at::AutoDispatchBelowADInplaceOrView below;
      if (want_x || want_w || want_b) {
        for (const auto* t : {&dy, &saved[0], &saved[1], &saved[2]})
          TORCH_CHECK_VALUE(!t->defined() || has_memory(*t),
                            "a tensor of the backward pass has no memory");
        Grads g = backward_of(dy, saved[0], saved[1], saved[2],
                              ctx->saved_data["k"].toInt(),
                              ctx->saved_data["act"].toInt(), want_x, want_w,
                              want_b);
        out[0] = g.dx;
        out[1] = g.dw;
        out[2] = g.db;
      }
    }
    if (want_r) out[3] = dy;
    return c10::GradMode::is_enabled() ? differentiable_once(std::move(out))
                                       : out;
  }
};

// A leaf whose gradient an eager graph of the default stream still waits for
// ties a captured backward pass to that stream, which cannot be captured: the
// engine's thread would end the process.
void check_capture(const at::Tensor& t, const char* name) {
  if (!t.defined() || !t.requires_grad() || !t.is_leaf()) return;
  const auto node = torch::autograd::impl::try_get_grad_accumulator(t);
  if (!node) return;
  const auto stream = node->stream();
  TORCH_CHECK(!stream.has_value() ||
                  stream->id() != c10::hip::getDefaultHIPStream(
                                      t.device().index()).id(),
              "captured while an eager graph that ", name,
              " is a leaf of lives on the default stream: drop its outputs "
              "before the capture, or run it on another stream");
}

// functional.linear_act on a GPU.
at::Tensor linear_act(const at::Tensor& x, const at::Tensor& w,
                      const Maybe& bias, int64_t act, Maybe residual) {
  TORCH_CHECK(x.is_cuda(), "x is on a GPU");
  TORCH_CHECK_VALUE(act >= 0 && act <= 4, "unknown activation ", act);
  TORCH_CHECK_VALUE(w.dim() == 2, "weight has shape (out, in), not ",
                    w.sizes());
  const int64_t n = w.size(0), k = w.size(1);
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) == k, "x ends in ", k,
                    " features, its shape is ", x.sizes());
  code_of(x.scalar_type());
  const bool dual = torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr;
  auto plain = [&](const at::Tensor& t, const char* name) {
    TORCH_CHECK_VALUE(!t.is_neg(), name, " is a lazy negation: call "
                      "resolve_neg() first");
    TORCH_CHECK_VALUE(has_memory(t), name, " has no memory");
    TORCH_CHECK_NOT_IMPLEMENTED(!dual || !t._fw_grad(0).defined(), name,
                                " carries a tangent: linear_act has no "
                                "forward-mode derivative");
  };
  plain(x, "x");
  auto like = [&](const at::Tensor& t, const char* name) {
    TORCH_CHECK_TYPE(t.scalar_type() == x.scalar_type() &&
                         t.device() == x.device(),
                     name, " is ", t.scalar_type(), " on ", t.device(),
                     ", x is ", x.scalar_type(), " on ", x.device());
    plain(t, name);
  };
  like(w, "weight");
  if (bias.has_value()) {
    TORCH_CHECK_VALUE(bias->dim() == 1 && bias->size(0) == n,
                      "bias has shape (", n, "), not ", bias->sizes());
    like(*bias, "bias");
  }
  auto shape = x.sizes().vec();
  shape.back() = n;
  const at::Tensor given = residual.value_or(at::Tensor());
  if (residual.has_value()) {
    like(*residual, "residual");
    bool ok = residual->dim() <= (int64_t)shape.size();
    for (int64_t d = 1; ok && d <= residual->dim(); ++d)
      ok = residual->size(-d) == 1 ||
           residual->size(-d) == shape[shape.size() - d];
    TORCH_CHECK_VALUE(ok, "residual of shape ", residual->sizes(),
                      " does not broadcast to ", at::IntArrayRef(shape));
    if (residual->sizes() != at::IntArrayRef(shape))
      residual = residual->expand(shape);
  }
  const bool matrix = x.dim() == 2;
  int64_t rows = 1;
  for (size_t d = 0; d + 1 < shape.size(); ++d) rows *= shape[d];
  // a grid holds below 2^32 threads, 256 of them take 64 rows or outputs
  TORCH_CHECK_VALUE(rows < LIMIT && n < LIMIT, "x of ", rows,
                    " rows and weight of ", n, " outputs: below ", LIMIT,
                    " of each are supported");
  at::Tensor x2 = matrix ? x : x.reshape({rows, k});
  if (!matrix && residual.has_value()) residual = residual->reshape({rows, n});
  const bool products =
      x2.requires_grad() || w.requires_grad() ||
      (bias.has_value() && bias->requires_grad());
  const bool any =
      products || (residual.has_value() && residual->requires_grad());
  at::Tensor y;
  if (any && c10::GradMode::is_enabled()) {
    c10::DeviceGuard guard(x.device());
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() !=
        c10::hip::CaptureStatus::None) {
      check_capture(x, "x");
      check_capture(w, "weight");
      if (bias.has_value()) check_capture(*bias, "bias");
      check_capture(given, "residual");
    }
    y = LinearAct::apply(x2, w, bias, residual, act, products);
  } else {
    at::AutoDispatchBelowADInplaceOrView below;
    at::Tensor w2 = w;
    y = forward_of(x2, w2, bias, residual, act, nullptr);
  }
  return matrix ? y : y.view(shape);
}

// (bm, bn, stages, parts of r) that a product of this size takes.
std::tuple<int, int, int, int> linear_plan(int64_t m, int64_t n, int64_t r,
                                           int dtype) {
  DdlProduct p{};
  p.m = m;
  p.n = n;
  p.r = r;
  p.dtype = dtype;
  ddl_product_plan(&p);
  return {p.bm, p.bn, p.stages, p.splits};
}

}  // namespace

void bind_linear(pybind11::module& m) {
  m.def("linear_act", &linear_act);
  m.def("linear_plan", &linear_plan);
}
