// Dense layer: the forward product for few rows, the backward of the
// activation with the bias gradient, and the C ABI.  The tiled products are
// in linear_tile.h.
#include "linear_tile.h"

void ddl_product_bf16(const DdlProduct* p, hipStream_t s);
void ddl_product_f16(const DdlProduct* p, hipStream_t s);
void ddl_product_f32(const DdlProduct* p, hipStream_t s);

namespace {

// ---- forward for few rows ----------------------------------------------------

// Up to 16 MT rows of x: what counts is one pass over W.  A block takes 16
// outputs; its waves take turns along the inputs and read W straight into
// fragments (16 lines of 64 bytes an instruction, a whole line in two), many
// loads ahead; their sums meet in LDS, in the waves' order.  No slabs and no
// second launch.  Rows may begin and end anywhere.
constexpr int FEW_UNROLL = 4;  // lines of W a lane has under way

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

template <typename T, int MT, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void few_rows_k(
    const T* __restrict__ x, int64_t ldx, const T* __restrict__ w, int64_t ldw,
    int64_t r, Epilogue e) {
  constexpr int E = 16 / (int)sizeof(T);
  constexpr int CHUNK = LINE / (int)sizeof(T);  // elements of r a line holds
  __shared__ float sums[WAVES][MT][16][16 + 4];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  // rows past the end repeat the last one; nothing of them is stored
  const T* wrow = w + min(n0 + c, e.n - 1) * ldw;
  const T* xrow[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
    xrow[i] = x + min((int64_t)i * 16 + c, e.m - 1) * ldx;

  f32x4 acc[MT] = {};
  using F = typename Frag<T>::type;
  auto take = [&](int64_t chunk, auto lines, auto whole) {
    constexpr int N = decltype(lines)::value;
    constexpr bool WHOLE = decltype(whole)::value;
    F wf[N][2], xf[N][2][MT];
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t k =
            (chunk + u * WAVES) * CHUNK + h * (CHUNK / 2) + g * E;
        wf[u][h] = piece<T, WHOLE>(wrow, k, r);
#pragma unroll
        for (int i = 0; i < MT; ++i)
          xf[u][h][i] = piece<T, WHOLE>(xrow[i], k, r);
      }
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < MT; ++i)
          acc[i] = mma(wf[u][h], xf[u][h][i], acc[i]);
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
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int q = 0; q < 4; ++q) sums[wave][i][c][g * 4 + q] = acc[i][q];
  __syncthreads();
  const int t = threadIdx.x;
  if (t < MT * 32) {
    const int64_t i = t >> 1, j = n0 + (t & 1) * 8;
    if (i < e.m && j < e.n) {
      float sum[8] = {}, bias[8];
#pragma unroll 2
      for (int s = 0; s < WAVES; ++s)
#pragma unroll
        for (int k = 0; k < 8; ++k)
          sum[k] += sums[s][i >> 4][i & 15][(t & 1) * 8 + k];
      load_bias8<T>(e, j, bias);
      finish8<T>(e, i, j, sum, bias);
    }
  }
}

template <typename T, int MT>
void launch_few(const DdlProduct* p, hipStream_t s) {
  few_rows_k<T, MT, 16><<<(unsigned)cdiv(p->n, 16), 1024, 0, s>>>(
      (const T*)p->a, p->lda, (const T*)p->b, p->ldb, p->r, epilogue_of<T>(p));
}

template <typename T>
void run_few(const DdlProduct* p, hipStream_t s) {
  if (p->m <= 16) launch_few<T, 1>(p, s);
  else launch_few<T, 2>(p, s);
}

// ---- backward of the activation, bias gradient ------------------------------

constexpr int BWD_ROWS = 32;   // rows a block sums
constexpr int BWD_COLS = 256;  // 32 threads of 8 columns

// Elements j..j+7 of a row of n, zeros behind its end.
template <typename T>
__device__ __forceinline__ Vec8<T> row8(const T* row, int64_t j, int64_t n,
                                        bool wide) {
  if (wide && j + 8 <= n) return load8(row + j);
  Vec8<T> r;
#pragma unroll
  for (int k = 0; k < 8; ++k)
    r.v[k] = j + k < n ? row[j + k] : from_f32<T>(0.f);
  return r;
}

template <typename T, typename Z>
__global__ __launch_bounds__(256) void act_bwd_k(
    const T* __restrict__ dy, int64_t lddy, const Z* __restrict__ z,
    int64_t ldz, T* __restrict__ dz, int64_t lddz, int64_t m, int64_t n,
    int act, int wide, float* __restrict__ partials) {
  __shared__ float part[8][BWD_COLS];
  const int cg = threadIdx.x & 31, rg = threadIdx.x >> 5;
  const int64_t col_blocks = cdiv(n, BWD_COLS);
  const int64_t cb = blockIdx.x % col_blocks, rb = blockIdx.x / col_blocks;
  const int64_t j = cb * BWD_COLS + cg * 8;
  float sum[8] = {};
  for (int64_t i = rb * BWD_ROWS + rg;
       i < min(m, (rb + 1) * (int64_t)BWD_ROWS) && j < n; i += 8) {
    const Vec8<T> d = row8(dy + i * lddy, j, n, wide & 1);
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = to_f32(d.v[k]);
    if (act) {
      const Vec8<Z> q = row8(z + i * ldz, j, n, wide & 2);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] *= activate_grad(to_f32(q.v[k]), act);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (j + k >= n) v[k] = 0.f;
      sum[k] += v[k];
    }
    if (dz) {  // rows of dz are padded to 16 bytes
      Vec8<T> o;
#pragma unroll
      for (int k = 0; k < 8; ++k) o.v[k] = from_f32<T>(v[k]);
      T* row = dz + i * lddz + j;
      if (j + 8 <= lddz) {
        store8(row, o);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (j + k < lddz) row[k] = o.v[k];
      }
    }
  }
  if (!partials) return;
#pragma unroll
  for (int k = 0; k < 8; ++k) part[rg][cg * 8 + k] = sum[k];
  __syncthreads();
  const int64_t col = cb * BWD_COLS + threadIdx.x;
  if (col < n) {
    float total = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) total += part[k][threadIdx.x];
    partials[rb * n + col] = total;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void fold_bias_k(const float* partials,
                                                   int64_t chunks, int64_t n,
                                                   T* dbias) {
  const int64_t j = global_tid();
  if (j >= n) return;
  double sum = 0.0;  // as many chunks as there are rows / 32
  for (int64_t c = 0; c < chunks; ++c) sum += partials[c * n + j];
  dbias[j] = from_f32<T>((float)sum);
}

// ---- rows that do not begin or end at 16 bytes -------------------------------

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
                 float* partials, void* dbias, hipStream_t s) {
  const int64_t chunks = cdiv(m, BWD_ROWS);
  const unsigned blocks = (unsigned)(chunks * cdiv(n, BWD_COLS));
  const int wide =
      (lddy % (16 / (int)sizeof(T)) == 0 && takes16(dy) ? 1 : 0) |
      (ldz % (16 / (int)sizeof(Z)) == 0 && takes16(z) ? 2 : 0);
  act_bwd_k<T, Z><<<blocks, 256, 0, s>>>(
      (const T*)dy, lddy, (const Z*)z, ldz, (T*)dz, lddz, m, n, act, wide,
      dbias ? partials : nullptr);
  if (dbias)
    fold_bias_k<T><<<(unsigned)cdiv(n, 256), 256, 0, s>>>(partials, chunks, n,
                                                          (T*)dbias);
}

}  // namespace

extern "C" {

int64_t ddl_product_ws_floats(const DdlProduct* p) {
  const Plan plan = plan_of(p);
  return plan.splits > 1 ? plan.splits * p->m * cdiv(p->n, 8) * 8 : 0;
}

void ddl_product(const DdlProduct* p, hipStream_t s) {
  switch (p->dtype) {
    case 0: ddl_product_f32(p, s); break;
    case 1: ddl_product_bf16(p, s); break;
    case 2: ddl_product_f16(p, s); break;
  }
}

int ddl_few_rows(void) { return 32; }

void ddl_product_few(const DdlProduct* p, hipStream_t s) {
  switch (p->dtype) {
    case 0: run_few<float>(p, s); break;
    case 1: run_few<bf16>(p, s); break;
    case 2: run_few<f16>(p, s); break;
  }
}

int64_t ddl_act_bwd_ws_floats(int64_t m, int64_t n) {
  return cdiv(m, BWD_ROWS) * n;
}

void ddl_act_bwd(const void* dy, int64_t lddy, const void* z, int z_f32,
                 int64_t ldz, void* dz, int64_t lddz, int64_t m, int64_t n,
                 int act, int dtype, float* partials, void* dbias,
                 hipStream_t s) {
  switch (dtype * 2 + (z_f32 ? 1 : 0)) {
    case 0:
    case 1:
      run_act_bwd<float, float>(dy, lddy, z, ldz, dz, lddz, m, n, act,
                                partials, dbias, s);
      break;
    case 2:
      run_act_bwd<bf16, bf16>(dy, lddy, z, ldz, dz, lddz, m, n, act, partials,
                              dbias, s);
      break;
    case 3:
      run_act_bwd<bf16, float>(dy, lddy, z, ldz, dz, lddz, m, n, act,
                               partials, dbias, s);
      break;
    case 4:
      run_act_bwd<f16, f16>(dy, lddy, z, ldz, dz, lddz, m, n, act, partials,
                            dbias, s);
      break;
    case 5:
      run_act_bwd<f16, float>(dy, lddy, z, ldz, dz, lddz, m, n, act, partials,
                              dbias, s);
      break;
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
