// Dense layer: out = act(x W^T + bias) + residual, and the products of its
// backward pass, on matrix instructions.
//
// All three products are out[i][j] = sum_r a(i, r) b(j, r):
//   forward  i = row,     j = output, r = input:  x and W contiguous in r
//   dx       i = row,     j = input,  r = output: dz in r, W in j
//   dW       i = output,  j = input,  r = row:    dz in i, x in j
// so an operand lies with r contiguous ("row") or with its output index
// contiguous ("col"), and nothing is transposed in memory.
//
// Tiles go from memory to LDS by buffer loads (16 B a lane, no registers in
// between), double buffered: the loads of step t+1 are issued before the
// products of step t.  Reads past an operand's end return zeros by the
// buffer's own bounds check; r's ragged end is cut by moving a lane's offset
// out of bounds.
//
// LDS images (16-byte units, one 128-byte line of a row operand or one line
// of a col operand after the other).  A wave's loads fill LDS in lane order,
// so units are exchanged on the source side: unit u of line l is stored at
// place u ^ f(l), with f chosen such that the 16 lanes of a fragment read
// touch all banks.  Fragments of 2-byte col operands come out of
// ds_read_b64_tr_b16, which transposes 4 x 16 elements among 16 lanes.
//
// The b fragment is the first operand of the matrix instruction and its rows
// are dealt so that a lane ends up with 16 consecutive j of one row i: the
// epilogue and the stores work on whole 16-byte pieces without another pass
// through LDS.
//
// Compiled without fast-math: infinities and NaN keep their meaning.
#include "common.h"
#include "linear_api.h"

namespace {

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((address_space(3))) unsigned int lds_u32;
typedef __attribute__((address_space(3))) s16x4* lds_s16x4;

constexpr int LINE = 128;            // bytes of r a step takes of a row
constexpr uint32_t OUTSIDE = 0x80000000u;  // past every buffer's end

struct Epilogue {
  const void* bias;
  const void* residual;
  void* out;
  void* z;
  int64_t ldo, ldres, m, n;
  int act;
  int wide;  // rows of out, z and residual take 16-byte accesses
};

struct Product {
  const char* a;
  const char* b;
  int64_t lda, ldb;  // bytes
  int64_t r;         // reduction length, padded to 16 bytes for row operands
  int64_t steps;     // r in steps of LINE bytes
  int64_t steps_per_split;
  int splits, tiles_m, tiles_n;
  float* slabs;
  int64_t ldslab;
  Epilogue e;
};

// ---- activations -----------------------------------------------------------

__device__ __forceinline__ float sigmoid(float z) {
  return 1.f / (1.f + __expf(-z));
}

__device__ __forceinline__ float activate(float z, int act) {
  switch (act) {
    case 1: return z < 0.f ? 0.f : z;  // NaN passes
    case 2: return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
    case 3: {
      // 0.5 (1 + tanh(u)) = sigmoid(2 u)
      const float u = 1.5957691216057308f * (z + 0.044715f * z * z * z);
      return z * sigmoid(u);
    }
    case 4: return z * sigmoid(z);
    default: return z;
  }
}

__device__ __forceinline__ float activate_grad(float z, int act) {
  switch (act) {
    case 1: return z <= 0.f ? 0.f : 1.f;
    case 2:
      return 0.5f * (1.f + erff(z * 0.70710678118654752f)) +
             z * 0.3989422804014327f * __expf(-0.5f * z * z);
    case 3: {
      const float u = 1.5957691216057308f * (z + 0.044715f * z * z * z);
      const float s = sigmoid(u);
      return s + z * s * (1.f - s) *
                     (1.5957691216057308f * (1.f + 0.134145f * z * z));
    }
    case 4: {
      const float s = sigmoid(z);
      return s * (1.f + z * (1.f - s));
    }
    default: return 1.f;
  }
}

// ---- matrix instructions ---------------------------------------------------

// A fragment is 16 bytes a lane: of row (lane & 15), elements
// (lane >> 4) * E + 0..E-1 of 4 E consecutive r, E = 16 / sizeof(T).
template <typename T> struct Frag;
template <> struct Frag<bf16> { using type = bf16x8; };
template <> struct Frag<f16> { using type = f16x8; };
template <> struct Frag<float> { using type = f32x4; };

__device__ __forceinline__ f32x4 mma(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(f32x4 a, f32x4 b, f32x4 c) {
#pragma unroll
  for (int e = 0; e < 4; ++e)
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
  return c;
}

// ---- epilogue --------------------------------------------------------------

// COUNT consecutive j of row i, from column j on.
template <typename T, int COUNT>
__device__ __forceinline__ void finish(const Epilogue& e, int64_t i, int64_t j,
                                       const float* sum, const float* bias) {
  constexpr int PIECE = 16 / (int)sizeof(T);
  float z[COUNT], y[COUNT];
#pragma unroll
  for (int k = 0; k < COUNT; ++k) {
    z[k] = sum[k] + bias[k];
    y[k] = activate(z[k], e.act);
  }
  T* out = (T*)e.out + i * e.ldo + j;
  T* zout = e.z ? (T*)e.z + i * e.ldo + j : nullptr;
  const T* res =
      e.residual ? (const T*)e.residual + i * e.ldres + j : nullptr;
#pragma unroll
  for (int k0 = 0; k0 < COUNT; k0 += PIECE) {
    if (e.wide && j + k0 + PIECE <= e.n) {
      union { uint4 u; T t[PIECE]; } o, r, p;
      if (res) {
        r.u = *reinterpret_cast<const uint4*>(res + k0);
#pragma unroll
        for (int k = 0; k < PIECE; ++k) y[k0 + k] += to_f32(r.t[k]);
      }
#pragma unroll
      for (int k = 0; k < PIECE; ++k) {
        o.t[k] = from_f32<T>(y[k0 + k]);
        p.t[k] = from_f32<T>(z[k0 + k]);
      }
      *reinterpret_cast<uint4*>(out + k0) = o.u;
      if (zout) *reinterpret_cast<uint4*>(zout + k0) = p.u;
    } else {
#pragma unroll
      for (int k = k0; k < k0 + PIECE; ++k) {
        if (j + k < e.n) {
          const float r = res ? to_f32(res[k]) : 0.f;
          out[k] = from_f32<T>(res ? y[k] + r : y[k]);
          if (zout) zout[k] = from_f32<T>(z[k]);
        }
      }
    }
  }
}

template <typename T, int COUNT>
__device__ __forceinline__ void load_bias(const Epilogue& e, int64_t j,
                                          float* bias) {
#pragma unroll
  for (int k = 0; k < COUNT; ++k)
    bias[k] = e.bias && j + k < e.n ? to_f32(((const T*)e.bias)[j + k]) : 0.f;
}

// ---- the tiled product -----------------------------------------------------

// Place of unit u of line l is u ^ swizzle(l).
template <typename T, bool COL, bool IS_B>
__device__ __forceinline__ int swizzle(int l) {
  if constexpr (!COL) {
    // a reads lines x = 0..15 at one unit, b lines (x >> 2) * 16 + (x & 3)
    return IS_B ? (l & 3) | (((l >> 4) & 1) << 2) : l & 7;
  } else if constexpr (sizeof(T) == 2) {
    // 4 lines a 16-lane group; a: 2 neighbouring units, b: 4 units, 2 apart
    return IS_B ? (l & 1) | (((l >> 1) & 1) << 3)
                : ((l & 3) << 1) | (((l >> 3) & 1) << 3);
  } else {
    return IS_B ? (l >> 2) & 3 : ((l >> 2) & 3) << 2;
  }
}

// One operand's tile of W output indexes: ROWS lines in memory and in LDS.
template <typename T, bool COL, bool IS_B, int W, int WAVES>
struct Tile {
  static constexpr int BYTES = W * LINE;
  static constexpr int LOADS = BYTES / (WAVES * 1024);
  static constexpr int UNITS = COL ? W * (int)sizeof(T) / 16 : LINE / 16;
  static constexpr int STEP = LINE / (int)sizeof(T);  // elements of r
  static_assert(BYTES % (WAVES * 1024) == 0, "whole loads");

  uint32_t offset[LOADS];   // of this lane's 16 bytes from the tile's start
  uint32_t along[LOADS];    // its place in r: bytes (row) or lines (col)

  __device__ __forceinline__ void init(int wave, int lane, int64_t ld,
                                       int64_t indexes) {
#pragma unroll
    for (int q = 0; q < LOADS; ++q) {
      const int u = (q * WAVES + wave) * 64 + lane;
      const int line = u / UNITS;
      const int unit = (u % UNITS) ^ swizzle<T, COL, IS_B>(line);
      const int64_t index = COL ? unit * (16 / (int)sizeof(T)) : line;
      along[q] = COL ? line : unit * 16;
      offset[q] = index < indexes ? (uint32_t)(line * ld) + unit * 16 : OUTSIDE;
    }
  }

  // Loads the tile at `base`; `end`: bytes from there to the operand's end;
  // `left`: what is left of r, in `along`'s measure, where it ends inside.
  template <bool CUT>
  __device__ __forceinline__ void load(char* lds, int wave, const char* base,
                                       int64_t end, uint32_t left) const {
    const int records = (int)min(end, (int64_t)0x7FFFFFFF);
    __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<char*>(base), 0, records, 0x00020000);
#pragma unroll
    for (int q = 0; q < LOADS; ++q) {
      uint32_t o = offset[q];
      if (CUT && along[q] >= left) o = OUTSIDE;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rsrc, (lds_u32*)(lds + (q * WAVES + wave) * 1024), 16, o, 0, 0, 0);
    }
  }

  // Fragment number f (16 indexes) of the wave's part that starts at index w;
  // half kk of the step.
  __device__ __forceinline__ typename Frag<T>::type read(const char* lds,
                                                         int lane, int w,
                                                         int f, int kk) const {
    const int x = lane & 15, g = lane >> 4;
    // b's rows: 16 consecutive j of a lane are spread over 4 fragments
    auto index = [&](int y) {
      return IS_B ? w + (f >> 2) * 64 + (y >> 2) * 16 + (f & 3) * 4 + (y & 3)
                  : w + f * 16 + y;
    };
    if constexpr (!COL) {
      const int line = index(x);
      const int unit = (kk * 4 + g) ^ swizzle<T, COL, IS_B>(line);
      return *reinterpret_cast<const typename Frag<T>::type*>(
          lds + line * LINE + unit * 16);
    } else if constexpr (sizeof(T) == 2) {
      typename Frag<T>::type out;
      s16x4* half = reinterpret_cast<s16x4*>(&out);
      const int first = index((x & 3) * 4);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int line = kk * 32 + g * 8 + h * 4 + (x >> 2);
        const int unit = (first >> 3) ^ swizzle<T, COL, IS_B>(line);
        half[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(
            lds + line * (W * 2) + unit * 16 + (first & 7) * 2));
      }
      return out;
    } else {
      typename Frag<T>::type out;
      const int i = index(x);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int line = kk * 16 + g * 4 + e;
        const int unit = (i >> 2) ^ swizzle<T, COL, IS_B>(line);
        out[e] = *reinterpret_cast<const float*>(lds + line * (W * 4) +
                                                 unit * 16 + (i & 3) * 4);
      }
      return out;
    }
  }
};

template <typename T, int BM, int BN, int WM, int WN, bool A_COL, bool B_COL>
__global__ __launch_bounds__(WM * WN * 64) void product_k(Product p) {
  constexpr int WAVES = WM * WN;
  constexpr int MI = BM / WM / 16, NI = BN / WN / 16;
  static_assert(NI % 4 == 0, "a lane's 16 columns are 4 fragments");
  using TA = Tile<T, A_COL, false, BM, WAVES>;
  using TB = Tile<T, B_COL, true, BN, WAVES>;
  constexpr int STAGE = TA::BYTES + TB::BYTES;
  __shared__ __align__(16) char smem[2 * STAGE];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tiles = p.tiles_m * p.tiles_n;
  const unsigned id = xcd_swizzle(blockIdx.x, gridDim.x);
  const int split = id / tiles;
  const int tile = id % tiles;
  // i runs fastest: neighbours on an XCD share the b tile
  const int64_t i0 = (int64_t)(tile % p.tiles_m) * BM;
  const int64_t j0 = (int64_t)(tile / p.tiles_m) * BN;

  TA ta;
  TB tb;
  ta.init(wave, lane, p.lda, p.e.m - i0);
  tb.init(wave, lane, p.ldb, p.e.n - j0);

  const int64_t t0 = split * p.steps_per_split;
  const int64_t t1 = min(p.steps, t0 + p.steps_per_split);
  constexpr int64_t STEP = TA::STEP;
  // bytes from a tile's start to the operand's end
  const char* a = p.a + (A_COL ? i0 * (int64_t)sizeof(T) : i0 * p.lda);
  const char* b = p.b + (B_COL ? j0 * (int64_t)sizeof(T) : j0 * p.ldb);
  const int64_t a_all = A_COL
      ? (p.r - 1) * p.lda + (p.e.m - i0) * (int64_t)sizeof(T)
      : (p.e.m - i0 - 1) * p.lda + p.r * (int64_t)sizeof(T);
  const int64_t b_all = B_COL
      ? (p.r - 1) * p.ldb + (p.e.n - j0) * (int64_t)sizeof(T)
      : (p.e.n - j0 - 1) * p.ldb + p.r * (int64_t)sizeof(T);
  // what is contiguous is a multiple of 16 bytes long
  const int64_t a_end = (a_all + 15) & ~(int64_t)15;
  const int64_t b_end = (b_all + 15) & ~(int64_t)15;

  auto load = [&](int64_t t, int stage) {
    char* l = smem + stage * STAGE;
    const int64_t ao = A_COL ? t * STEP * p.lda : t * LINE;
    const int64_t bo = B_COL ? t * STEP * p.ldb : t * LINE;
    const int64_t left = p.r - t * STEP;
    if (left >= STEP) {
      ta.template load<false>(l, wave, a + ao, a_end - ao, 0);
      tb.template load<false>(l + TA::BYTES, wave, b + bo, b_end - bo, 0);
    } else {
      const uint32_t bytes = (uint32_t)(left * (int)sizeof(T));
      ta.template load<true>(l, wave, a + ao, a_end - ao,
                             A_COL ? (uint32_t)left : bytes);
      tb.template load<true>(l + TA::BYTES, wave, b + bo, b_end - bo,
                             B_COL ? (uint32_t)left : bytes);
    }
  };

  f32x4 acc[MI][NI] = {};
  const int wm = (wave / WN) * (BM / WM), wn = (wave % WN) * (BN / WN);

  if (t0 < t1) load(t0, 0);
  for (int64_t t = t0; t < t1; ++t) {
    const int stage = (int)(t - t0) & 1;
    // This step's tile has landed, and this wave's reads of the other stage
    // have returned; past the barrier both hold for all waves.
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (t + 1 < t1) load(t + 1, stage ^ 1);
    const char* la = smem + stage * STAGE;
    const char* lb = la + TA::BYTES;
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      typename Frag<T>::type af[MI], bf[NI];
#pragma unroll
      for (int f = 0; f < NI; ++f) bf[f] = tb.read(lb, lane, wn, f, kk);
#pragma unroll
      for (int f = 0; f < MI; ++f) af[f] = ta.read(la, lane, wm, f, kk);
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) acc[i][j] = mma(bf[j], af[i], acc[i][j]);
    }
  }

  const int x = lane & 15, g = lane >> 4;
#pragma unroll
  for (int h = 0; h < NI / 4; ++h) {
    const int64_t j = j0 + wn + h * 64 + g * 16;
    float bias[16];
    if (p.splits == 1) load_bias<T, 16>(p.e, j, bias);
#pragma unroll
    for (int f = 0; f < MI; ++f) {
      const int64_t i = i0 + wm + f * 16 + x;
      if (i >= p.e.m || j >= p.e.n) continue;
      float sum[16];
#pragma unroll
      for (int k = 0; k < 16; ++k) sum[k] = acc[f][h * 4 + (k >> 2)][k & 3];
      if (p.splits > 1) {
        // rows of a slab are padded to 16 numbers
        float* s = p.slabs + (split * p.e.m + i) * p.ldslab + j;
#pragma unroll
        for (int k = 0; k < 16; k += 4)
          *reinterpret_cast<float4*>(s + k) =
              float4{sum[k], sum[k + 1], sum[k + 2], sum[k + 3]};
      } else {
        finish<T, 16>(p.e, i, j, sum, bias);
      }
    }
  }
}

// Adds the slabs in order (no atomics: the result does not depend on which
// block ends first) and applies the epilogue; 8 columns a thread.
template <typename T>
__global__ __launch_bounds__(256) void join_k(const float* slabs, int splits,
                                              int64_t ldslab, Epilogue e) {
  const int64_t groups = ldslab / 8;
  const int64_t at = global_tid();
  if (at >= groups * e.m) return;
  const int64_t i = at / groups, j = (at % groups) * 8;
  if (j >= e.n) return;
  float sum[8] = {};
  for (int s = 0; s < splits; ++s) {
    const float* q = slabs + (s * e.m + i) * ldslab + j;
    const float4 lo = *reinterpret_cast<const float4*>(q);
    const float4 hi = *reinterpret_cast<const float4*>(q + 4);
    sum[0] += lo.x; sum[1] += lo.y; sum[2] += lo.z; sum[3] += lo.w;
    sum[4] += hi.x; sum[5] += hi.y; sum[6] += hi.z; sum[7] += hi.w;
  }
  float bias[8];
  load_bias<T, 8>(e, j, bias);
  finish<T, 8>(e, i, j, sum, bias);
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

template <typename T>
__global__ __launch_bounds__(256) void act_bwd_k(
    const T* __restrict__ dy, int64_t lddy, const T* __restrict__ z,
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
      const Vec8<T> q = row8(z + i * ldz, j, n, wide & 2);
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

template <typename T>
__global__ __launch_bounds__(256) void pack_rows_k(const T* __restrict__ src,
                                                   int64_t lds_, T* dst,
                                                   int64_t ldd, int64_t m,
                                                   int64_t n) {
  const int64_t per = cdiv(ldd, 256);
  for (int64_t b = blockIdx.x; b < m * per; b += gridDim.x) {
    const int64_t i = b / per;
    const int64_t j = (b % per) * 256 + threadIdx.x;
    if (j < ldd)
      dst[i * ldd + j] = j < n ? src[i * lds_ + j] : from_f32<T>(0.f);
  }
}

// ---- host ------------------------------------------------------------------

int compute_units() {
  static const int n = [] {
    hipDeviceProp_t prop;
    return hipGetDeviceProperties(&prop, 0) == hipSuccess
               ? prop.multiProcessorCount : 256;
  }();
  return n;
}

struct Plan {
  int bm, bn, splits;
  int64_t steps, steps_per_split;
};

Plan plan_of(const DdlProduct* p) {
  const int size = p->dtype == 0 ? 4 : 2;
  Plan best{};
  best.steps = cdiv(p->r * size, LINE);
  const int64_t big = cdiv(p->m, 256) * cdiv(p->n, 256);
  best.bm = best.bn = big * 4 >= compute_units() * 3 ? 256 : 128;
  if (p->dtype == 0) best.bm = best.bn = 128;
  const int64_t tiles = cdiv(p->m, best.bm) * cdiv(p->n, best.bn);
  int64_t splits = std::max<int64_t>(1, compute_units() / tiles);
  splits = std::min(splits, std::max<int64_t>(1, best.steps / 8));
  best.steps_per_split = std::max<int64_t>(1, cdiv(best.steps, splits));
  best.splits = (int)std::max<int64_t>(1, cdiv(best.steps,
                                                best.steps_per_split));
  return best;
}

template <typename T, int BM, int BN, int WM, int WN>
void launch_product(const Product& p, int a_col, int b_col, hipStream_t s) {
  const int blocks = p.tiles_m * p.tiles_n * p.splits;
  const dim3 grid(blocks), block(WM * WN * 64);
  if (a_col && b_col)
    product_k<T, BM, BN, WM, WN, true, true><<<grid, block, 0, s>>>(p);
  else if (b_col)
    product_k<T, BM, BN, WM, WN, false, true><<<grid, block, 0, s>>>(p);
  else
    product_k<T, BM, BN, WM, WN, false, false><<<grid, block, 0, s>>>(p);
}

bool takes16(const void* p) { return ((uintptr_t)p & 15) == 0; }

template <typename T>
void run_product(const DdlProduct* d, hipStream_t s) {
  const Plan plan = plan_of(d);
  const int64_t per = 16 / (int)sizeof(T);
  Product p{};
  p.a = (const char*)d->a;
  p.b = (const char*)d->b;
  p.lda = d->lda * (int64_t)sizeof(T);
  p.ldb = d->ldb * (int64_t)sizeof(T);
  p.r = d->r;
  p.steps = plan.steps;
  p.steps_per_split = plan.steps_per_split;
  p.splits = plan.splits;
  p.tiles_m = (int)cdiv(d->m, plan.bm);
  p.tiles_n = (int)cdiv(d->n, plan.bn);
  p.slabs = d->slabs;
  p.ldslab = cdiv(d->n, 16) * 16;
  p.e = Epilogue{d->bias, d->residual, d->out, d->z, d->ldo, d->ldres, d->m,
                 d->n, d->act,
                 d->ldo % per == 0 && takes16(d->out) && takes16(d->z) &&
                     (!d->residual ||
                      (d->ldres % per == 0 && takes16(d->residual)))};
  if (sizeof(T) == 2 && plan.bm == 256) {
    if constexpr (sizeof(T) == 2)
      launch_product<T, 256, 256, 2, 4>(p, d->a_col, d->b_col, s);
  } else {
    launch_product<T, 128, 128, 2, 2>(p, d->a_col, d->b_col, s);
  }
  if (p.splits > 1) {
    const int64_t threads = p.ldslab / 8 * d->m;
    join_k<T><<<(unsigned)cdiv(threads, 256), 256, 0, s>>>(
        p.slabs, p.splits, p.ldslab, p.e);
  }
}

}  // namespace

extern "C" {

int64_t ddl_product_ws_floats(const DdlProduct* p) {
  const Plan plan = plan_of(p);
  return plan.splits > 1 ? plan.splits * p->m * cdiv(p->n, 16) * 16 : 0;
}

void ddl_product(const DdlProduct* p, hipStream_t s) {
  switch (p->dtype) {
    case 0: run_product<float>(p, s); break;
    case 1: run_product<bf16>(p, s); break;
    case 2: run_product<f16>(p, s); break;
  }
}

int64_t ddl_act_bwd_ws_floats(int64_t m, int64_t n) {
  return cdiv(m, BWD_ROWS) * n;
}

void ddl_act_bwd(const void* dy, int64_t lddy, const void* z, int64_t ldz,
                 void* dz, int64_t lddz, int64_t m, int64_t n, int act,
                 int dtype, float* partials, void* dbias, hipStream_t s) {
  const int64_t chunks = cdiv(m, BWD_ROWS);
  const unsigned blocks = (unsigned)(chunks * cdiv(n, BWD_COLS));
  const int per = dtype == 0 ? 4 : 8;
  const int wide = (lddy % per == 0 && takes16(dy) ? 1 : 0) |
                   (ldz % per == 0 && takes16(z) ? 2 : 0);
#define RUN(T)                                                                \
  act_bwd_k<T><<<blocks, 256, 0, s>>>((const T*)dy, lddy, (const T*)z, ldz,   \
                                      (T*)dz, lddz, m, n, act, wide,          \
                                      dbias ? partials : nullptr);            \
  if (dbias)                                                                  \
    fold_bias_k<T><<<(unsigned)cdiv(n, 256), 256, 0, s>>>(partials, chunks,   \
                                                          n, (T*)dbias)
  switch (dtype) {
    case 0: RUN(float); break;
    case 1: RUN(bf16); break;
    case 2: RUN(f16); break;
  }
#undef RUN
}

void ddl_pack_rows(const void* src, int64_t lds, void* dst, int64_t ldd,
                   int64_t m, int64_t n, int dtype, hipStream_t s) {
  const unsigned blocks =
      (unsigned)std::min<int64_t>(m * cdiv(ldd, 256), 1 << 20);
  switch (dtype) {
    case 0:
      pack_rows_k<float><<<blocks, 256, 0, s>>>((const float*)src, lds,
                                                (float*)dst, ldd, m, n);
      break;
    default:  // the two 16-bit types are copied alike
      pack_rows_k<f16><<<blocks, 256, 0, s>>>((const f16*)src, lds, (f16*)dst,
                                              ldd, m, n);
  }
}

}  // extern "C"
