// Torch binding of the dense layer (csrc/kernels/linear.hip): checks, packs
// operands whose rows do not lie on 16-byte boundaries, allocates outputs and
// workspaces, and launches on the current stream of the tensors' device.
#include <torch/extension.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPException.h>
#include <c10/hip/HIPStream.h>

#include "kernels/linear_api.h"

namespace {

using Maybe = c10::optional<at::Tensor>;

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

void check_like(const at::Tensor& t, const at::Tensor& x, const char* name) {
  TORCH_CHECK(t.device() == x.device(), name, " is on another device than x");
  TORCH_CHECK(t.scalar_type() == x.scalar_type(), name,
              " has another dtype than x");
}

void check_matrix(const at::Tensor& t, int64_t rows, int64_t cols,
                  const char* name) {
  TORCH_CHECK(t.dim() == 2 && t.size(0) == rows && t.size(1) == cols, name,
              " has shape ", t.sizes(), ", expected (", rows, ", ", cols, ")");
}

int64_t round_up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// A matrix whose columns are neighbours in memory; its rows may lie anywhere.
at::Tensor inner_contiguous(const at::Tensor& t) {
  return t.stride(1) == 1 || t.size(1) <= 1 ? t : t.contiguous();
}

// Elements from one row to the next; a single row has no say.
int64_t row_stride(const at::Tensor& t) {
  return t.size(0) > 1 ? t.stride(0) : t.size(1);
}

// What the kernel reads: rows that begin and end at 16 bytes, no further
// apart than its 32-bit offsets inside a tile reach.
struct Operand {
  at::Tensor keep;
  const void* data;
  int64_t ld;
};

Operand operand(const at::Tensor& matrix) {
  const at::Tensor t = inner_contiguous(matrix);
  const int64_t per = 16 / t.element_size();
  const int64_t reach = ((int64_t)1 << 31) / 256 / t.element_size();
  const int64_t ld = row_stride(t);
  if (ld % per == 0 && t.size(1) % per == 0 && ld < reach &&
      ((uintptr_t)t.const_data_ptr() & 15) == 0)
    return {t, t.const_data_ptr(), ld};
  const int64_t wide = round_up(t.size(1), per);
  TORCH_CHECK(wide < reach, "a matrix has ", t.size(1),
              " columns, more than the kernel's offsets reach (", reach, ")");
  at::Tensor packed = at::empty({t.size(0), wide}, t.options());
  if (packed.numel())
    ddl_pack_rows(t.const_data_ptr(), ld, packed.data_ptr(), wide, t.size(0),
                  t.size(1), code_of(t.scalar_type()), stream_now());
  return {packed, packed.const_data_ptr(), wide};
}

// out = epilogue(a b^T) with its workspace.
void product(DdlProduct& p, const at::Tensor& like) {
  if (p.m == 0 || p.n == 0) return;
  at::Tensor slabs;
  if (const int64_t floats = ddl_product_ws_floats(&p)) {
    slabs = at::empty({floats}, like.options().dtype(at::kFloat));
    p.slabs = slabs.data_ptr<float>();
  }
  ddl_product(&p, stream_now());
  C10_HIP_KERNEL_LAUNCH_CHECK();
}

// y = act(x w^T + bias) + residual, and z = x w^T + bias if asked for.
std::tuple<at::Tensor, at::Tensor> linear_fwd(at::Tensor x, at::Tensor w,
                                              Maybe bias, Maybe residual,
                                              int64_t act, bool want_z) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2 && w.dim() == 2,
              "x and weight are matrices on a GPU");
  TORCH_CHECK(act >= 0 && act <= 4, "unknown activation ", act);
  const int64_t m = x.size(0), k = x.size(1), n = w.size(0);
  const int dtype = code_of(x.scalar_type());
  check_like(w, x, "weight");
  check_matrix(w, n, k, "weight");
  c10::DeviceGuard guard(x.device());
  at::Tensor y = at::empty({m, n}, x.options());
  at::Tensor z = want_z ? at::empty({m, n}, x.options()) : at::Tensor();
  at::Tensor b, res;
  DdlProduct p{};
  if (bias.has_value()) {
    check_like(*bias, x, "bias");
    TORCH_CHECK(bias->dim() == 1 && bias->size(0) == n, "bias has shape ",
                bias->sizes(), ", expected (", n, ")");
    b = bias->contiguous();
    p.bias = b.const_data_ptr();
  }
  if (residual.has_value()) {
    check_like(*residual, x, "residual");
    check_matrix(*residual, m, n, "residual");
    res = inner_contiguous(*residual);
    p.residual = res.const_data_ptr();
    p.ldres = row_stride(res);
  }
  const Operand a = operand(x), c = operand(w);
  p.a = a.data;
  p.lda = a.ld;
  p.b = c.data;
  p.ldb = c.ld;
  p.m = m;
  p.n = n;
  p.r = k;
  p.out = y.data_ptr();
  p.ldo = n;
  p.z = want_z ? z.data_ptr() : nullptr;
  p.act = (int)act;
  p.dtype = dtype;
  product(p, x);
  return {y, z};
}

// The gradients of linear_fwd that are asked for.  z: what the activation
// took (its output does for ReLU); not looked at without an activation.
std::tuple<at::Tensor, at::Tensor, at::Tensor> linear_bwd(
    at::Tensor dy, at::Tensor x, at::Tensor w, Maybe z, int64_t act,
    bool want_dx, bool want_dw, bool want_db) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2 && w.dim() == 2,
              "x and weight are matrices on a GPU");
  TORCH_CHECK(act >= 0 && act <= 4, "unknown activation ", act);
  const int64_t m = x.size(0), k = x.size(1), n = w.size(0);
  const int dtype = code_of(x.scalar_type());
  check_like(w, x, "weight");
  check_like(dy, x, "dy");
  check_matrix(w, n, k, "weight");
  check_matrix(dy, m, n, "dy");
  c10::DeviceGuard guard(x.device());
  const auto s = stream_now();
  at::Tensor dx, dw, db, zc;
  if (want_dx) dx = at::empty({m, k}, x.options());
  if (want_dw) dw = at::empty({n, k}, x.options());
  if (want_db) db = at::empty({n}, x.options());
  if (m == 0 || n == 0 || k == 0) {  // sums over nothing
    for (auto* t : {&dx, &dw})
      if (t->defined()) t->zero_();
    if (want_db && m == 0) db.zero_();
  }
  if (m == 0 || n == 0) return {dx, dw, db};

  const at::Tensor d = inner_contiguous(dy);
  if (act) {
    TORCH_CHECK(z.has_value(), "the activation's input is missing");
    check_like(*z, x, "z");
    check_matrix(*z, m, n, "z");
    zc = inner_contiguous(*z);
  }
  Operand dz{};
  const bool products = k > 0 && (want_dx || want_dw);
  if (act && products) {
    const int64_t wide = round_up(n, 16 / x.element_size());
    dz.keep = at::empty({m, wide}, x.options());
    dz.data = dz.keep.const_data_ptr();
    dz.ld = wide;
  }
  if (want_db || dz.keep.defined()) {
    at::Tensor partials;
    if (want_db)
      partials = at::empty({ddl_act_bwd_ws_floats(m, n)},
                           x.options().dtype(at::kFloat));
    ddl_act_bwd(d.const_data_ptr(), row_stride(d),
                act ? zc.const_data_ptr() : nullptr, act ? row_stride(zc) : 0,
                dz.keep.defined() ? dz.keep.data_ptr() : nullptr, dz.ld, m, n,
                (int)act, dtype,
                want_db ? partials.data_ptr<float>() : nullptr,
                want_db ? db.data_ptr() : nullptr, s);
    C10_HIP_KERNEL_LAUNCH_CHECK();
  }
  if (!products) return {dx, dw, db};
  if (!act) dz = operand(d);

  DdlProduct p{};
  p.dtype = dtype;
  p.a = dz.data;
  p.lda = dz.ld;
  p.b_col = 1;
  p.n = k;
  p.ldo = k;
  if (want_dx) {
    const Operand b = operand(w);
    p.b = b.data;
    p.ldb = b.ld;
    p.m = m;
    p.r = n;
    p.out = dx.data_ptr();
    product(p, x);
  }
  if (want_dw) {
    const Operand b = operand(x);
    p.b = b.data;
    p.ldb = b.ld;
    p.a_col = 1;
    p.m = n;
    p.r = m;
    p.out = dw.data_ptr();
    product(p, x);
  }
  return {dx, dw, db};
}

}  // namespace

void bind_linear(pybind11::module& m) {
  m.def("linear_fwd", &linear_fwd);
  m.def("linear_bwd", &linear_bwd);
}
