// The tiled products of linear_tile.h for one type (a file each, so that they
// are compiled side by side).
#include "linear_tile.h"

void ddl_product_f16(const DdlProduct* p, hipStream_t s) {
  run_product<f16>(p, s);
}

void ddl_backward_small_f16(const DdlProduct* dx, const DdlProduct* dw,
                           const DdlBiasFold* bias, hipStream_t s) {
  run_backward_small<f16>(*dx, *dw, *bias, s);
}
