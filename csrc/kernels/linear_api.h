// C ABI of the dense-layer kernels in linear.hip (host binding:
// csrc/bind/linear_binding.cpp).  dtype codes as in api.h; act: 0 none,
// 1 ReLU, 2 GELU (erf), 3 GELU (tanh), 4 SiLU.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

extern "C" {

// out[i][j] = epilogue(sum_r a(i, r) b(j, r)).  An operand is stored with r
// contiguous (`*_col` 0: a(i, r) = a[i * lda + r]) or with the output's index
// contiguous (`*_col` 1: a(i, r) = a[r * lda + i]).  Rows begin at 4 bytes and
// end anywhere; what lies between them does not count.
struct DdlProduct {
  const void* a;
  const void* b;
  int64_t lda, ldb;     // elements
  int64_t m, n, r;
  int a_col, b_col;
  void* out;            // [m][ldo]
  int64_t ldo;
  // epilogue: z = sum + bias[j]; out = act(z) + residual[i][j]
  const void* bias;
  const void* residual;
  int64_t ldres;
  float* z;             // [m][ldo], or null
  int act;
  int dtype;
  // filled in by ddl_product_plan
  int kind, bm, bn, stages, splits;
  float us;             // its estimate
  int64_t steps, steps_per_split;
  float* slabs;         // as many floats as the plan says
};

// Chooses tile and split; returns the floats that slabs has to hold.
int64_t ddl_product_plan(DdlProduct* p);
void ddl_product(const DdlProduct* p, hipStream_t s);

// The same for at most 16 rows, both operands with r contiguous and rows
// anywhere (any lda, ldb, r and alignment); needs no slabs.  Whether that is
// estimated to be faster than the planned product; `aligned`: its operands
// would not have to be packed.
bool ddl_few_rows_pay(const DdlProduct* p, bool aligned);
void ddl_product_few(const DdlProduct* p, hipStream_t s);

// dz[i][j] = dy[i][j] act'(z[i][j]), zeros in columns n..lddz (a multiple of
// 8), and the column sums of dz before its rounding, of some rows each: partials
// holds ddl_bias_chunks(m, n) * n floats.  z is float32 (z_f32), or for act 1 the
// output in the tensors' dtype.  dz or partials may be null.
int64_t ddl_bias_chunks(int64_t m, int64_t n);
void ddl_act_bwd(const void* dy, int64_t lddy, const void* z, int z_f32,
                 int64_t ldz, void* dz, int64_t lddz, int64_t m, int64_t n,
                 int act, int dtype, float* partials, hipStream_t s);

// dbias[j] = sum of partials[c][j]; nothing for n = 0.
struct DdlBiasFold {
  const float* partials;
  void* dbias;
  int64_t chunks, n;
};
void ddl_fold_bias(const DdlBiasFold* f, int dtype, hipStream_t s);

// dx and dw, planned, and the fold in one launch, where that is estimated to
// be faster than a launch each.  Without partials the bias gradient is summed
// from dw's a: 64 x 64 -> 96 bf16 takes 8.4 us so, 11.0 with partial sums made
// first, 2048 x 64 -> 64 18.8 (21.3).
bool ddl_small_backward(const DdlProduct* dx, const DdlProduct* dw);
void ddl_backward_small(const DdlProduct* dx, const DdlProduct* dw,
                        const DdlBiasFold* bias, hipStream_t s);

// dst[i][0..ldd) = src[i][0..n), then zeros, for one or two matrices; ldd is a
// multiple of 8, dst of 16 bytes.
struct DdlPack {
  const void* src;
  void* dst;
  int64_t lds, ldd, m, n;
};
void ddl_pack_rows(const DdlPack* matrices, int count, int dtype,
                   hipStream_t s);

}  // extern "C"
