// The tiled products of linear_tile.h for one type (a file each, so that they
// are compiled side by side).
#include "linear_tile.h"

void ddl_product_f32(const DdlProduct* p, hipStream_t s) {
  run_product<float>(p, s);
}

void ddl_backward_small_f32(const DdlProduct* dx, const DdlProduct* dw,
                           const DdlBiasFold* bias, hipStream_t s) {
  run_backward_small<float>(*dx, *dw, *bias, s);
}
