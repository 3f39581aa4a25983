// Dense layer: the forward product for few rows, the backward of the
// activation with the bias gradient, and the C ABI.  The tiled products are
// in linear_tile.h.
#include "linear_tile.h"

#define DDL_TYPE(NAME)                                                    \
  void ddl_product_##NAME(const DdlProduct* p, hipStream_t s);            \
  void ddl_backward_small_##NAME(const DdlProduct* dx,                    \
                                 const DdlProduct* dw,                    \
                                 const DdlBiasFold* bias, hipStream_t s);
DDL_TYPE(f32)
DDL_TYPE(bf16)
DDL_TYPE(f16)
#undef DDL_TYPE

namespace {

// ---- forward for few rows ----------------------------------------------------

// Up to 16 rows of x: what counts is one pass over W.  A block takes 16
// outputs; its waves take turns along the inputs and read W straight into
// fragments (16 lines of 64 bytes an instruction, a whole line in two), four
// lines ahead; their sums meet in LDS, in the waves' order.  No slabs and no
// second launch.  Rows may begin and end anywhere.  bf16, 1 x 4096 -> 4096:
// 9.1 us with the launch, where W alone takes 6.6 at 5.07 TB/s.
constexpr int FEW_UNROLL = 4;

// 16 bytes of a row; WHOLE: they end before r.
template <typename T, bool WHOLE>
__device__ __forceinline__ typename Frag<T>::type piece(const T* row,
                                                        int64_t k, int64_t r) {
  constexpr int E = 16 / (int)sizeof(T);
  union { typename Frag<T>::type f; T t[E]; uint4 u; } v;
  if (WHOLE || k + E <= r) {
    __builtin_memcpy(&v.u, row + k, 16);
  } else {
    v.u = uint4{0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (k + e < r) v.t[e] = row[k + e];
  }
  return v.f;
}

template <typename T, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void few_rows_k(
    const T* __restrict__ x, int64_t ldx, const T* __restrict__ w, int64_t ldw,
    int64_t r, Epilogue e) {
  constexpr int E = 16 / (int)sizeof(T);
  constexpr int CHUNK = LINE / (int)sizeof(T);  // elements of r a line holds
  __shared__ float sums[WAVES][16][16 + 4];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  // rows past the end repeat the last one; nothing of them is stored
  const T* wrow = w + min(n0 + c, e.n - 1) * ldw;
  const T* xrow = x + min((int64_t)c, e.m - 1) * ldx;

  f32x4 acc[1][1] = {};
  using F = typename Frag<T>::type;
  auto take = [&](int64_t chunk, auto lines, auto whole) {
    constexpr int N = decltype(lines)::value;
    constexpr bool WHOLE = decltype(whole)::value;
    F wf[N][2][1], xf[N][2][1];
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t k =
            (chunk + u * WAVES) * CHUNK + h * (CHUNK / 2) + g * E;
        wf[u][h][0] = piece<T, WHOLE>(wrow, k, r);
        xf[u][h][0] = piece<T, WHOLE>(xrow, k, r);
      }
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) multiply(acc, xf[u][h], wf[u][h]);
  };
  const int64_t whole = r / CHUNK;
  int64_t k0 = wave;
  for (; k0 + (FEW_UNROLL - 1) * WAVES < whole; k0 += FEW_UNROLL * WAVES)
    take(k0, std::integral_constant<int, FEW_UNROLL>{}, std::true_type{});
  for (; k0 < whole; k0 += WAVES)
    take(k0, std::integral_constant<int, 1>{}, std::true_type{});
  if (k0 * CHUNK < r)
    take(k0, std::integral_constant<int, 1>{}, std::false_type{});

#pragma unroll
  for (int q = 0; q < 4; ++q) sums[wave][c][g * 4 + q] = acc[0][0][q];
  __syncthreads();
  const int t = threadIdx.x;
  if (t < 32) {
    const int64_t i = t >> 1, j = n0 + (t & 1) * 8;
    if (i < e.m && j < e.n) {
      float sum[8] = {}, bias[8];
#pragma unroll 2
      for (int s = 0; s < WAVES; ++s)
#pragma unroll
        for (int k = 0; k < 8; ++k) sum[k] += sums[s][i][(t & 1) * 8 + k];
      load_bias8<T>(e, j, bias);
      finish8<T>(e, i, j, sum, bias);
    }
  }
}

template <typename T>
void run_few(const DdlProduct* p, hipStream_t s) {
  few_rows_k<T, 16><<<(unsigned)cdiv(p->n, 16), 1024, 0, s>>>(
      (const T*)p->a, p->lda, (const T*)p->b, p->ldb, p->r, epilogue_of(p));
}

// ---- backward of the activation, bias gradient ------------------------------

// 256 threads take 8 columns each: LANES of them a row, all rows of a turn
// twice.  64 columns a block where there are no more, 256 otherwise.  A block
// adds its rows of a column in float32, the fold adds the blocks in 64 bits.
constexpr int BWD_NARROW = 8, BWD_WIDE = 32;

// Rows that a block sums: one turn where there are few, as many turns as leave
// four blocks to a compute unit where there are many, since the bias
// gradient's fold reads a number a column of each block.  1048576 x 64 -> 8
// with its gradients takes 359 us so; 1056 with 16 rows a block and 32 lanes a
// row at all sizes.
inline int64_t bwd_rows(int64_t m, int64_t n) {
  const int64_t lanes = n <= BWD_NARROW * 8 ? BWD_NARROW : BWD_WIDE;
  const int64_t turn = 2 * (256 / lanes);
  const int64_t blocks = cdiv(n, lanes * 8) * cdiv(m, turn);
  return turn * std::max<int64_t>(1, cdiv(blocks, 4 * compute_units()));
}

// Elements j..j+7 of a row of n, zeros behind its end; it may begin anywhere.
template <typename T>
__device__ __forceinline__ void row8(const T* row, int64_t j, int64_t n,
                                     float* out) {
  T r[8];
  if (j + 8 <= n) {
    __builtin_memcpy(r, row + j, sizeof(r));
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      r[k] = j + k < n ? row[j + k] : from_f32<T>(0.f);
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) out[k] = to_f32(r[k]);
}

template <typename T, typename Z, int LANES>
__global__ __launch_bounds__(256) void act_bwd_k(
    const T* __restrict__ dy, int64_t lddy, const Z* __restrict__ z,
    int64_t ldz, T* __restrict__ dz, int64_t lddz, int64_t m, int64_t n,
    int64_t rows, int act, float* __restrict__ partials) {
  constexpr int GROUPS = 256 / LANES, COLS = LANES * 8;
  __shared__ float part[GROUPS][COLS];
  const int cg = threadIdx.x % LANES, rg = threadIdx.x / LANES;
  const int64_t col_blocks = cdiv(n, COLS);
  const int64_t cb = blockIdx.x % col_blocks, rb = blockIdx.x / col_blocks;
  const int64_t j = cb * COLS + cg * 8;
  const int64_t end_row = min(m, (rb + 1) * rows);
  float sum[8] = {};
  for (int64_t i0 = rb * rows + rg; i0 < end_row; i0 += 2 * GROUPS) {
    float v[2][8], q[2][8];
#pragma unroll
    for (int t = 0; t < 2; ++t) {  // all loads first
      const int64_t i = i0 + t * GROUPS;
      const int64_t end = i < end_row ? n : 0;  // rows past the end are empty
      row8(dy + (i < end_row ? i * lddy : 0), j, end, v[t]);
      if (act) row8(z + (i < end_row ? i * ldz : 0), j, end, q[t]);
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      if (act) activate_grad8<sizeof(T) == 2>(v[t], q[t], act);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        // a gradient of NaN behind the row's end would enter the products
        if (j + k >= n) v[t][k] = 0.f;
        sum[k] += v[t][k];
      }
      const int64_t i = i0 + t * GROUPS;
      if (dz && i < end_row && j < lddz) {  // lddz is a multiple of 8
        Vec8<T> o;
#pragma unroll
        for (int k = 0; k < 8; ++k) o.v[k] = from_f32<T>(v[t][k]);
        store8(dz + i * lddz + j, o);
      }
    }
  }
  if (!partials) return;
#pragma unroll
  for (int k = 0; k < 8; ++k) part[rg][cg * 8 + k] = sum[k];
  __syncthreads();
  const int64_t col = cb * COLS + threadIdx.x;
  if (threadIdx.x < COLS && col < n) {
    float total = 0.f;
#pragma unroll
    for (int k = 0; k < GROUPS; ++k) total += part[k][threadIdx.x];
    partials[rb * n + col] = total;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void fold_bias_k(DdlBiasFold f,
                                                   int64_t first) {
  __shared__ __align__(16) char smem[256 * sizeof(double)];
  fold_bias(f.partials, f.n, f.chunks, (T*)f.dbias, f.n, first + blockIdx.x,
            smem);
}

// ---- rows that do not begin at 4 bytes --------------------------------------

struct PackArgs {
  DdlPack m[2];
  int64_t pieces[2];  // of 8 elements of dst
};

template <typename T>
__global__ __launch_bounds__(256) void pack_rows_k(PackArgs a) {
  for (int64_t at = global_tid(); at < a.pieces[0] + a.pieces[1];
       at += grid_stride()) {
    const bool second = at >= a.pieces[0];
    const DdlPack& m = a.m[second];
    const int64_t piece = at - (second ? a.pieces[0] : 0);
    const int64_t per = m.ldd / 8;
    const int64_t i = piece / per, j = (piece % per) * 8;
    const T* src = (const T*)m.src + i * m.lds + j;
    Vec8<T> v;
    if (j + 8 <= m.n) {
      __builtin_memcpy(v.v, src, sizeof(v.v));
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        v.v[k] = j + k < m.n ? src[k] : from_f32<T>(0.f);
    }
    store8((T*)m.dst + i * m.ldd + j, v);
  }
}

// ---- host ------------------------------------------------------------------

template <typename T, typename Z>
void run_act_bwd(const void* dy, int64_t lddy, const void* z, int64_t ldz,
                 void* dz, int64_t lddz, int64_t m, int64_t n, int act,
                 float* partials, hipStream_t s) {
  const int64_t rows = bwd_rows(m, n), chunks = cdiv(m, rows);
  auto launch = [&](auto kernel, int lanes) {
    kernel<<<(unsigned)(chunks * cdiv(n, lanes * 8)), 256, 0, s>>>(
        (const T*)dy, lddy, (const Z*)z, ldz, (T*)dz, lddz, m, n, rows, act,
        partials);
  };
  if (n <= BWD_NARROW * 8)
    launch(act_bwd_k<T, Z, BWD_NARROW>, BWD_NARROW);
  else
    launch(act_bwd_k<T, Z, BWD_WIDE>, BWD_WIDE);
}

}  // namespace

extern "C" {

int64_t ddl_product_plan(DdlProduct* p) {
  plan_product(p);
  return p->splits > 1 ? p->splits * p->m * cdiv(p->n, 8) * 8 : 0;
}

void ddl_product(const DdlProduct* p, hipStream_t s) {
  switch (p->dtype) {
    case 0: ddl_product_f32(p, s); break;
    case 1: ddl_product_bf16(p, s); break;
    case 2: ddl_product_f16(p, s); break;
  }
}

bool ddl_small_backward(const DdlProduct* dx, const DdlProduct* dw) {
  return small_backward(dx, dw);
}

void ddl_backward_small(const DdlProduct* dx, const DdlProduct* dw,
                        const DdlBiasFold* bias, hipStream_t s) {
  switch (dx->dtype) {
    case 0: ddl_backward_small_f32(dx, dw, bias, s); break;
    case 1: ddl_backward_small_bf16(dx, dw, bias, s); break;
    case 2: ddl_backward_small_f16(dx, dw, bias, s); break;
  }
}

// The few-row kernel, and the tiled one with what comes before it, in us.  A
// block of the former reads its part of W at 28 KB a us, less with more rows
// of x beside it, and a third of that where 2-byte rows begin anywhere: 16 x
// 25088 -> 4096 takes 46 us (tiled 34), 1 x 16384 -> 128 20 (10), 16 x 4096 ->
// 4096 10.9 (12.5), 1 x 2047 -> 1001 10.7 (13.6, of which packing 5), 1 x 4098
// -> 4096 8.1 (11.8); float32, 16 x 14242 -> 2853 45 (71).
bool ddl_few_rows_pay(const DdlProduct* p, bool aligned) {
  // its grid: below 2^32 threads, 1024 of them for 16 outputs
  if (p->m > 16 || cdiv(p->n, 16) >= ((int64_t)1 << 22)) return false;
  const float size = p->dtype == 0 ? 4.f : 2.f;
  const float row = p->r * size, all = row * p->n;
  float rate = 28e3f / (1.f + (p->dtype == 0 ? 0.4f : 0.8f) * p->m / 16.f);
  if (!aligned && p->dtype != 0) rate /= 3.f;
  const float rounds = std::ceil(p->n / (16.f * compute_units()));
  const float few = 1.f + std::max(all / 5.5e6f, rounds * 16.f * row / rate);
  const float tiled = p->us + (aligned ? 0.f : 5.f + all / 2e6f);
  return few <= tiled;
}

void ddl_product_few(const DdlProduct* p, hipStream_t s) {
  switch (p->dtype) {
    case 0: run_few<float>(p, s); break;
    case 1: run_few<bf16>(p, s); break;
    case 2: run_few<f16>(p, s); break;
  }
}

int64_t ddl_bias_chunks(int64_t m, int64_t n) {
  return cdiv(m, bwd_rows(m, n));
}

void ddl_act_bwd(const void* dy, int64_t lddy, const void* z, int z_f32,
                 int64_t ldz, void* dz, int64_t lddz, int64_t m, int64_t n,
                 int act, int dtype, float* partials, hipStream_t s) {
#define RUN(T, Z) \
  run_act_bwd<T, Z>(dy, lddy, z, ldz, dz, lddz, m, n, act, partials, s)
  switch (dtype * 2 + (z_f32 ? 1 : 0)) {
    case 0:
    case 1: RUN(float, float); break;
    case 2: RUN(bf16, bf16); break;
    case 3: RUN(bf16, float); break;
    case 4: RUN(f16, f16); break;
    case 5: RUN(f16, float); break;
  }
#undef RUN
}

void ddl_fold_bias(const DdlBiasFold* f, int dtype, hipStream_t s) {
  const int64_t blocks = cdiv(f->n, FOLD_COLS);
  constexpr int64_t MOST = (int64_t)1 << 23;  // a grid: below 2^32 threads
  for (int64_t at = 0; at < blocks; at += MOST) {
    const unsigned grid = (unsigned)std::min(MOST, blocks - at);
    switch (dtype) {
      case 0: fold_bias_k<float><<<grid, 256, 0, s>>>(*f, at); break;
      case 1: fold_bias_k<bf16><<<grid, 256, 0, s>>>(*f, at); break;
      case 2: fold_bias_k<f16><<<grid, 256, 0, s>>>(*f, at); break;
    }
  }
}

void ddl_pack_rows(const DdlPack* matrices, int count, int dtype,
                   hipStream_t s) {
  PackArgs a{};
  for (int i = 0; i < count; ++i) {
    a.m[i] = matrices[i];
    a.pieces[i] = matrices[i].m * (matrices[i].ldd / 8);
  }
  const int64_t all = a.pieces[0] + a.pieces[1];
  if (all == 0) return;
  const unsigned blocks = (unsigned)std::min<int64_t>(cdiv(all, 256), 1 << 14);
  if (dtype == 0)
    pack_rows_k<float><<<blocks, 256, 0, s>>>(a);
  else  // the two 16-bit types are copied alike
    pack_rows_k<f16><<<blocks, 256, 0, s>>>(a);
}

}  // extern "C"
