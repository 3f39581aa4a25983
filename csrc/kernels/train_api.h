// C ABI of the optimizer kernels in adamw.hip (host binding:
// csrc/bind/adamw_binding.cpp).  dtype codes as in api.h.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

extern "C" {

// One tensor of an AdamW step.  `w` is the float32 master, or the parameter
// itself where that is float32 (then `p` is null).  `ms`/`vs` are the scales
// of 8-bit moments, one a block of DDL_MOMENT_BLOCK elements; unused where
// the moments are float32.
struct DdlAdamTensor {
  void* p;
  const void* g;
  float* w;
  void* m;
  void* v;
  float* ms;
  float* vs;
  int64_t n;
  float* step;     // the tensor's own step count, on the device
  uint32_t index;  // its place in the optimizer: seeds the random rounding
};

struct DdlAdamScalars {
  double lr, beta1, beta2, eps, weight_decay;
  float grad_mul;   // 1 / grad_scale
  uint32_t seed;
};

struct DdlGradTensor {
  void* g;
  int64_t n;
};

#define DDL_MOMENT_BLOCK 256

// Partial sums of squares -> norm = sqrt(sum) * mul and
// coef = min(1, max_norm / (norm + 1e-6)).
struct DdlNormFold {
  const double* partials;
  int64_t blocks;
  double mul, max_norm;
  float* norm;
  float* coef;
};

// Step counts += 1, and the numbers that follow from them for each tensor;
// the fold, where there is one, in the same launch.
// ws: ddl_adamw_ws_bytes(count) bytes.
int64_t ddl_adamw_ws_bytes(int64_t count);
void ddl_adamw_prepare(const DdlAdamTensor* t, int64_t count,
                       const DdlAdamScalars* c, void* ws,
                       const DdlNormFold* fold, hipStream_t s);
// The update of all tensors.  coef: device scalar that multiplies every
// gradient (clipping), or null.
void ddl_adamw(const DdlAdamTensor* t, int64_t count,
               const DdlAdamScalars* c, int dtype, int bits, const void* ws,
               const float* coef, hipStream_t s);

// Global gradient norm: partial sums of one list, ddl_grad_norm_blocks()
// doubles, to be folded together with those of other lists.
int64_t ddl_grad_norm_blocks(const DdlGradTensor* t, int64_t count);
void ddl_grad_norm_partials(const DdlGradTensor* t, int64_t count, int dtype,
                            double* partials, hipStream_t s);
void ddl_grad_norm_fold(const DdlNormFold* f, hipStream_t s);
// g *= coef, which is read from f->coef, or with `fold` made from the partial
// sums on the way (ddl_grad_norm_fold is not needed then); nothing is read or
// written where it is 1.
void ddl_grad_scale(const DdlGradTensor* t, int64_t count, int dtype,
                    const DdlNormFold* f, int fold, hipStream_t s);
// Partial sums up to which the fold is better off in the scaling launch, whose
// blocks each add up all of them: clipping 4 million elements (1956 sums) takes
// 13 us so and 16 with a launch for the fold, 8 million (3908) 17 and 16.
#define DDL_FOLD_IN_SCALE 2048

}  // extern "C"
