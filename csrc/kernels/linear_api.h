// C ABI of the dense-layer kernels in linear.hip (host binding:
// csrc/bind/linear_binding.cpp).  dtype codes as in api.h; act: 0 none,
// 1 ReLU, 2 GELU (erf), 3 GELU (tanh), 4 SiLU.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

extern "C" {

// out[i][j] = epilogue(sum_r a(i, r) b(j, r)).  An operand is stored with r
// contiguous (`*_col` 0: a(i, r) = a[i * lda + r]) or with the output's index
// contiguous (`*_col` 1: a(i, r) = a[r * lda + i]).  What is contiguous is a
// multiple of 16 bytes long (zeros behind the end of r), rows begin at
// 16-byte boundaries.
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
  void* z;              // [m][ldo], z rounded, or null
  int act;
  int dtype;
  float* slabs;         // ddl_product_ws_floats floats
};

int64_t ddl_product_ws_floats(const DdlProduct* p);
void ddl_product(const DdlProduct* p, hipStream_t s);

// dz[i][j] = dy[i][j] act'(z[i][j]), zeros in columns n..lddz, and the column
// sums of the rounded dz: partial sums (ddl_act_bwd_ws_floats floats), then
// their fold into dbias.  act 1 may take y in the place of z.  dz or dbias
// may be null.
int64_t ddl_act_bwd_ws_floats(int64_t m, int64_t n);
void ddl_act_bwd(const void* dy, int64_t lddy, const void* z, int64_t ldz,
                 void* dz, int64_t lddz, int64_t m, int64_t n, int act,
                 int dtype, float* partials, void* dbias, hipStream_t s);

// dst[i][0..ldd) = src[i][0..n), then zeros.
void ddl_pack_rows(const void* src, int64_t lds, void* dst, int64_t ldd,
                   int64_t m, int64_t n, int dtype, hipStream_t s);

}  // extern "C"
