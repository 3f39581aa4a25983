// Products of the dense layer, out = act(x W^T + bias) + residual, and of its
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
// between) into a ring of stages.  Reads past an operand's end return zeros by the
// buffer's own bounds check, 4 bytes at a time; r's ragged end is cut by moving
// a lane's offset out of bounds, and inside of 16 bytes by clearing the rest in
// LDS.  So rows may begin at any 4 bytes: 256 x 25090 -> 4098 forward takes 94
// us, 226 if both operands are first copied to rows that begin at 16.
//
// LDS images (16-byte units, one 128-byte line of a row operand or one line
// of a col operand after the other).  A wave's loads fill LDS in lane order,
// so units are exchanged on the source side: unit u of line l is stored at
// place u ^ f(l), with f chosen such that the 16 lanes of a fragment read
// touch all banks.  Fragments of 2-byte col operands come out of
// ds_read_b64_tr_b16, which transposes 4 x 16 elements among 16 lanes.
//
// The b fragment is the first operand of the matrix instruction and its rows
// are dealt so that a lane ends up with 16 consecutive j of one row i.
//
// Compiled without fast-math: infinities and NaN keep their meaning.
#pragma once
#include "common.h"
#include "linear_api.h"

#include <cmath>
#include <type_traits>

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
  float* z;
  int64_t ldo, ldres, m, n;
  int act;
  int stream;  // out is stored past the caches
};

struct Product {
  const char* a;
  const char* b;
  int64_t lda, ldb;  // bytes
  int64_t r;         // reduction length
  int64_t steps;     // r in steps of LINE bytes
  int64_t steps_per_split;
  int splits, tiles_m, tiles_n;
  float* slabs;
  int64_t ldslab;
  Epilogue e;
};

// ---- activations -----------------------------------------------------------

// Functions of the activations.  FAST, for 16-bit types: the hardware's
// reciprocal and power, off by one part in 2^22 of themselves (the power's
// argument is rounded besides, |z| 2^-24 of the result), and a fit of the normal
// distribution, where float32 takes an IEEE division, expf and erff.  GELU's
// backward over 1024 x 4096 f16 takes 9.3 us so and 11.8 with the latter two and
// the hardware's power.
template <bool FAST>
__device__ __forceinline__ float sigmoid(float z) {
  if constexpr (FAST)
    return __builtin_amdgcn_rcpf(
        1.f + __builtin_amdgcn_exp2f(z * -1.4426950408889634f));
  return 1.f / (1.f + expf(-z));
}

// The standard normal distribution at z, and e = exp(-z^2 / 2).  FAST: below 0
// it is e t P(t), t = 1 / (1 + 0.42 |z| / sqrt 2), Hastings' form of the error
// function (Abramowitz and Stegun 7.1.26); P, of degree 5, is a least-maximum fit
// of exp(x^2) erfc(x) / 2t at x = |z| / sqrt 2, made for this kernel.  Off by
// 1.7e-7, and in the tail by 1.7e-5 of the value.
template <bool FAST>
__device__ __forceinline__ float normal(float z, float& e) {
  if constexpr (FAST) {
    const float t = __builtin_amdgcn_rcpf(1.f + 0.29698484809835f * fabsf(z));
    e = __builtin_amdgcn_exp2f(z * z * -0.72134752044448f);
    float q = -0.08244086f;
    q = q * t + 0.24082047f;
    q = q * t - 0.04314515f;
    q = q * t + 0.15598618f;
    q = q * t + 0.10966496f;
    q = q * t + 0.11911423f;
    q *= t * e;
    return z < 0.f ? q : 1.f - q;
  }
  e = expf(-0.5f * z * z);
  return 0.5f * (1.f + erff(z * 0.70710678118654752f));
}

template <bool FAST>
__device__ __forceinline__ float activate(float z, int act) {
  switch (act) {
    case 1: return z < 0.f ? 0.f : z;  // NaN passes
    case 2: {
      float e;
      return z * normal<FAST>(z, e);
    }
    case 3: {
      // 0.5 (1 + tanh(u)) = sigmoid(2 u)
      const float u = 1.5957691216057308f * (z + 0.044715f * z * z * z);
      return z * sigmoid<FAST>(u);
    }
    case 4: return z * sigmoid<FAST>(z);
    default: return z;
  }
}

template <bool FAST>
__device__ __forceinline__ float activate_grad(float z, int act) {
  switch (act) {
    case 2: {
      float e;
      const float phi = normal<FAST>(z, e);
      return phi + z * 0.3989422804014327f * e;
    }
    case 3: {
      const float u = 1.5957691216057308f * (z + 0.044715f * z * z * z);
      const float s = sigmoid<FAST>(u);
      return s + z * s * (1.f - s) *
                     (1.5957691216057308f * (1.f + 0.134145f * z * z));
    }
    case 4: {
      const float s = sigmoid<FAST>(z);
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
// Of the four instructions that a float32 fragment pair takes, number e.
__device__ __forceinline__ f32x4 mma(float a, float b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// acc[i][j] += b[j] a[i].  For float32 the four instructions of a pair depend
// on one another: they are spread over the pairs.
template <int MI, int NI>
__device__ __forceinline__ void multiply(f32x4 (&acc)[MI][NI],
                                         const f32x4 (&a)[MI],
                                         const f32x4 (&b)[NI]) {
#pragma unroll
  for (int e = 0; e < 4; ++e)
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j)
        acc[i][j] = mma(b[j][e], a[i][e], acc[i][j]);
}

template <typename F, int MI, int NI>
__device__ __forceinline__ void multiply(f32x4 (&acc)[MI][NI],
                                         const F (&a)[MI], const F (&b)[NI]) {
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j) acc[i][j] = mma(b[j], a[i], acc[i][j]);
}

// ---- epilogue --------------------------------------------------------------

// `fn` on 8 values; the switch stands outside, so that the code of one
// activation is run through without a branch an element.
template <bool FAST>
__device__ __forceinline__ void activate8(float* y, int act) {
  auto all = [&](auto which) {
#pragma unroll
    for (int k = 0; k < 8; ++k) y[k] = activate<FAST>(y[k], which.value);
  };
  switch (act) {
    case 1: all(std::integral_constant<int, 1>{}); break;
    case 2: all(std::integral_constant<int, 2>{}); break;
    case 3: all(std::integral_constant<int, 3>{}); break;
    case 4: all(std::integral_constant<int, 4>{}); break;
  }
}

// v[k] *= act'(z[k]).  ReLU's is a choice, no product: what arrives where it
// is shut is dropped, also an infinity or NaN.
template <bool FAST>
__device__ __forceinline__ void activate_grad8(float* v, const float* z,
                                               int act) {
  auto all = [&](auto which) {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] *= activate_grad<FAST>(z[k], which.value);
  };
  switch (act) {
    case 1:
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = z[k] <= 0.f ? 0.f : v[k];
      break;
    case 2: all(std::integral_constant<int, 2>{}); break;
    case 3: all(std::integral_constant<int, 3>{}); break;
    case 4: all(std::integral_constant<int, 4>{}); break;
  }
}

template <typename T>
__device__ __forceinline__ void store_out(T* out, const T (&o)[8],
                                          int stream) {
  if (!stream) {
    __builtin_memcpy(out, o, sizeof(o));
    return;
  }
  typedef __attribute__((ext_vector_type(4))) unsigned int u32x4;
  typedef u32x4 anywhere __attribute__((aligned(2)));
  constexpr int PIECE = 16 / (int)sizeof(T);
#pragma unroll
  for (int k = 0; k < 8; k += PIECE) {
    u32x4 v;
    __builtin_memcpy(&v, o + k, 16);
    // The compiler would make one plain store of this and the other one.
    asm volatile("");
    __builtin_nontemporal_store(v, reinterpret_cast<anywhere*>(out + k));
    asm volatile("");
  }
}

// Columns j..j+7 of row i; `sum` is the product.
template <typename T>
__device__ __forceinline__ void finish8(const Epilogue& e, int64_t i,
                                        int64_t j, const float* sum,
                                        const float* bias) {
  float z[8], y[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) y[k] = z[k] = sum[k] + bias[k];
  activate8<sizeof(T) == 2>(y, e.act);
  T* out = (T*)e.out + i * e.ldo + j;
  float* zout = e.z ? e.z + i * e.ldo + j : nullptr;
  const T* res =
      e.residual ? (const T*)e.residual + i * e.ldres + j : nullptr;
  if (j + 8 <= e.n) {
    // rows begin anywhere: 16-byte accesses do not need their alignment
    T o[8];
    if (res) {
      T r[8];
      __builtin_memcpy(r, res, sizeof(r));
#pragma unroll
      for (int k = 0; k < 8; ++k) y[k] += to_f32(r[k]);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) o[k] = from_f32<T>(y[k]);
    store_out(out, o, e.stream);
    if (zout) __builtin_memcpy(zout, z, sizeof(z));
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (j + k < e.n) {
        out[k] = from_f32<T>(res ? y[k] + to_f32(res[k]) : y[k]);
        if (zout) zout[k] = z[k];
      }
    }
  }
}

template <typename T>
__device__ __forceinline__ void load_bias8(const Epilogue& e, int64_t j,
                                           float* bias) {
#pragma unroll
  for (int k = 0; k < 8; ++k)
    bias[k] = e.bias && j + k < e.n ? to_f32(((const T*)e.bias)[j + k]) : 0.f;
}

// A large output would push the operands that the next product reads out of
// the last level cache (256 MB): a training pass of 512 x 25088 -> 4096, with
// 205 MB each of W and dW, takes 368 us so and 389 otherwise.  Small ones stay
// for who reads them next.
inline Epilogue epilogue_of(const DdlProduct* d) {
  const int64_t bytes = d->m * d->n * (d->dtype == 0 ? 4 : 2);
  return Epilogue{d->bias,  d->residual, d->out, d->z, d->ldo, d->ldres,
                  d->m, d->n, d->act, bytes >= ((int64_t)64 << 20)};
}

// ---- the tiled product -----------------------------------------------------

// Place of unit u of line l is u ^ swizzle(l); UNITS: units of a line.
template <typename T, bool COL, bool IS_B, int UNITS>
__device__ __forceinline__ int swizzle(int l) {
  if constexpr (!COL) {
    // a reads lines x = 0..15 at one unit, b lines (x >> 2) * 16 + (x & 3)
    return IS_B ? (l & 3) | (((l >> 4) & 1) << 2) : l & 7;
  } else if constexpr (sizeof(T) == 2 && UNITS >= 16) {
    // 4 lines a 16-lane group; a: 2 neighbouring units, b: 4 units, 2 apart
    return IS_B ? (l & 1) | (((l >> 1) & 1) << 3)
                : ((l & 3) << 1) | (((l >> 3) & 1) << 3);
  } else if constexpr (sizeof(T) == 2) {
    // two lines of 8 units lie side by side over the banks
    static_assert(UNITS == 8, "a line is 128 bytes or more");
    return IS_B ? (l >> 1) & 1
                : (((l >> 1) & 1) << 1) | (((l >> 3) & 1) << 2);
  } else {
    static_assert(UNITS >= 16, "a line is 256 bytes or more");
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

  // LDS instructions a fragment
  static constexpr int READS = !COL ? 1 : sizeof(T) == 2 ? 2 : 4;

  uint32_t offset[LOADS];   // of this lane's 16 bytes from the tile's start
  uint32_t along[LOADS];    // its place in r: bytes (row) or lines (col)

  __device__ __forceinline__ void init(int wave, int lane, int64_t ld,
                                       int64_t indexes) {
#pragma unroll
    for (int q = 0; q < LOADS; ++q) {
      const int u = (q * WAVES + wave) * 64 + lane;
      const int line = u / UNITS;
      const int unit = (u % UNITS) ^ swizzle<T, COL, IS_B, UNITS>(line);
      const int64_t index = COL ? unit * (16 / (int)sizeof(T)) : line;
      along[q] = COL ? line : unit * 16;
      offset[q] = index < indexes ? (uint32_t)(line * ld) + unit * 16 : OUTSIDE;
    }
  }

  // Loads the tile at `base`; `end`: bytes from there to the operand's end;
  // `left`: what is left of r, in `along`'s measure (0: zeros are loaded).
  __device__ __forceinline__ void load(char* __restrict lds, int wave, const char* base,
                                       int64_t end, uint32_t left) const {
    const int records = (int)max(min(end, (int64_t)0x7FFFFFFF), (int64_t)0);
    __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<char*>(base), 0, records, 0x00020000);
#pragma unroll
    for (int q = 0; q < LOADS; ++q) {
      const uint32_t o = along[q] < left ? offset[q] : OUTSIDE;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rsrc, (lds_u32*)(lds + (q * WAVES + wave) * 1024), 16, o, 0, 0, 0);
    }
  }

  // Zeros the rest of the 16 bytes that a row operand's r ends inside of, in
  // all lines; `keep`: bytes of r in this tile.
  __device__ __forceinline__ void clear_rest(char* lds, int keep) const {
    for (int line = threadIdx.x; line < W; line += WAVES * 64) {
      const int unit = (keep >> 4) ^ swizzle<T, COL, IS_B, UNITS>(line);
      uint32_t* word = reinterpret_cast<uint32_t*>(lds + line * LINE) + unit * 4;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int left = (keep & 15) - q * 4;
        if (left < 4) word[q] = left == 2 ? word[q] & 0xFFFFu : 0u;
      }
    }
  }

  // Fragment number f (16 indexes) of the wave's part that starts at index w;
  // half kk of the step.
  __device__ __forceinline__ typename Frag<T>::type read(const char* __restrict lds,
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
      const int unit = (kk * 4 + g) ^ swizzle<T, COL, IS_B, UNITS>(line);
      return *reinterpret_cast<const typename Frag<T>::type*>(
          lds + line * LINE + unit * 16);
    } else if constexpr (sizeof(T) == 2) {
      typename Frag<T>::type out;
      s16x4* half = reinterpret_cast<s16x4*>(&out);
      const int first = index((x & 3) * 4);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int line = kk * 32 + g * 8 + h * 4 + (x >> 2);
        const int unit = (first >> 3) ^ swizzle<T, COL, IS_B, UNITS>(line);
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
        const int unit = (i >> 2) ^ swizzle<T, COL, IS_B, UNITS>(line);
        out[e] = *reinterpret_cast<const float*>(lds + line * (W * 4) +
                                                 unit * 16 + (i & 3) * 4);
      }
      return out;
    }
  }
};

// Waits until at most LOADS of this wave's loads are under way and its LDS
// reads have returned, then for the block's other waves to say the same.
template <int LOADS>
__device__ __forceinline__ void meet() {
  static_assert(LOADS < 64, "the counter's range");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(LOADS) : "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Lets the scheduler spread LDS reads and loads evenly among the matrix
// instructions of a block: issued in one go, they fill the LDS queue and hold
// the matrix instructions back.
template <int READS, int MATRIX, int LOADS>
__device__ __forceinline__ void interleave() {
  constexpr int PAIRS = READS > MATRIX / 2 ? 2 : 1;  // reads a matrix instr.
#pragma unroll
  for (int i = 0; i < READS / PAIRS; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    if (i < LOADS) __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, PAIRS, 0);
  }
  __builtin_amdgcn_sched_group_barrier(0x008, MATRIX - READS / PAIRS, 0);
}

// The epilogue of a block: each wave lays its sums into its own part of LDS,
// 64 columns a line, and takes them back 8 columns a lane: whole lines go to
// memory, and the epilogue's code is there once (unrolled over the registers
// it was so long that fetching it cost 40 us a tile).  16-byte units are
// exchanged within a line by its row, which spreads both accesses over the
// banks.  `smem` holds BYTES that no wave uses any more.
template <typename T, int MI, int NI, int WAVES, int BYTES>
__device__ __forceinline__ void write_out(const Product& p, char* smem,
                                          const f32x4 (&acc)[MI][NI],
                                          int wave, int lane, int split,
                                          int64_t i0, int64_t j0) {
  constexpr int PASS = WAVES * MI * 16 * 256 <= BYTES ? MI : MI / 2;
  constexpr int ROWS = PASS * 16;
  static_assert(WAVES * ROWS * 256 <= BYTES, "sums fit the tiles' LDS");
  float* sums = reinterpret_cast<float*>(smem) + wave * ROWS * 64;
  const int x = lane & 15, g = lane >> 4;
  const int row = lane >> 3, unit = (lane & 7) * 2;
#pragma unroll
  for (int h = 0; h < NI / 4; ++h) {
    const int64_t j = j0 + h * 64 + (lane & 7) * 8;
    float bias[8];
    if (p.splits == 1) load_bias8<T>(p.e, j, bias);
#pragma unroll
    for (int f0 = 0; f0 < MI; f0 += PASS) {
#pragma unroll
      for (int f = 0; f < PASS; ++f)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<f32x4*>(sums + (f * 16 + x) * 64 +
                                    ((g * 4 + q) ^ x) * 4) =
              acc[f0 + f][h * 4 + q];
      // A wave's LDS accesses are done in order: no barrier within a wave.
#pragma unroll 1
      for (int r = row; r < ROWS; r += 8) {
        const int64_t i = i0 + f0 * 16 + r;
        union { f32x4 v[2]; float f[8]; } sum;
#pragma unroll
        for (int q = 0; q < 2; ++q)
          sum.v[q] = *reinterpret_cast<const f32x4*>(
              sums + r * 64 + ((unit + q) ^ (r & 15)) * 4);
        if (i >= p.e.m || j >= p.e.n) continue;
        if (p.splits > 1) {
          // rows of a slab are padded to 8 numbers
          float* s = p.slabs + (split * p.e.m + i) * p.ldslab + j;
          *reinterpret_cast<f32x4*>(s) = sum.v[0];
          *reinterpret_cast<f32x4*>(s + 4) = sum.v[1];
        } else {
          finish8<T>(p.e, i, j, sum.f, bias);
        }
      }
    }
  }
}

template <typename T, int BM, int BN, int STAGES>
constexpr int lds_bytes() { return STAGES * (BM + BN) * LINE; }

// Block `id` of the product, with lds_bytes of LDS.
template <typename T, int BM, int BN, int WM, int WN, int STAGES, bool A_COL,
          bool B_COL>
__device__ __forceinline__ void product_block(const Product& p, unsigned id,
                                              char* smem) {
  constexpr int WAVES = WM * WN;
  constexpr int MI = BM / WM / 16, NI = BN / WN / 16;
  static_assert(NI % 4 == 0, "a lane's 16 columns are 4 fragments");
  using TA = Tile<T, A_COL, false, BM, WAVES>;
  using TB = Tile<T, B_COL, true, BN, WAVES>;
  constexpr int STAGE = TA::BYTES + TB::BYTES;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tiles = p.tiles_m * p.tiles_n;
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
  // The hardware checks 4 bytes at a time; the last 2 of them may lie behind
  // an operand of 16-bit numbers.
  const int64_t a_end = (a_all + 3) & ~(int64_t)3;
  const int64_t b_end = (b_all + 3) & ~(int64_t)3;

  auto load = [&](int64_t t, int stage) {
    char* l = smem + stage * STAGE;
    const int64_t ao = A_COL ? t * STEP * p.lda : t * LINE;
    const int64_t bo = B_COL ? t * STEP * p.ldb : t * LINE;
    // past this block's part of r nothing is read
    const int64_t left =
        t < t1 ? min(p.r - t * STEP, (int64_t)STEP) : (int64_t)0;
    const uint32_t lines = (uint32_t)left;
    const uint32_t bytes = (uint32_t)(left * (int)sizeof(T));
    ta.load(l, wave, a + ao, a_end - ao, A_COL ? lines : bytes);
    tb.load(l + TA::BYTES, wave, b + bo, b_end - bo, B_COL ? lines : bytes);
  };

  f32x4 acc[MI][NI] = {};
  const int wm = (wave / WN) * (BM / WM), wn = (wave % WN) * (BN / WN);

  // Half a step's fragments are read while the other half's products run.
  // Once a step, in its middle: the next tile has landed and this wave's reads
  // of the present one have returned; past the barrier both hold for all
  // waves, so the present stage is loaded anew, STAGES - 1 steps ahead.  Loads
  // past the end are issued too, and read nothing: their number is the same
  // in every step.
  using F = typename Frag<T>::type;
  F a0[MI], b0[NI], a1[MI], b1[NI];
  // Where r does not end at 16 bytes, what a row operand's last load of a line
  // brings from behind it (the next row) is cleared before the step is read.
  const int keep = (int)(p.r * (int)sizeof(T) - (p.steps - 1) * LINE);
  const bool ragged =
      !(A_COL && B_COL) && (keep & 15) != 0 && t1 == p.steps;
  auto settle = [&](int stage) {
    char* l = smem + stage * STAGE;
    if constexpr (!A_COL) ta.clear_rest(l, keep);
    if constexpr (!B_COL) tb.clear_rest(l + TA::BYTES, keep);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  auto read = [&](F (&af)[MI], F (&bf)[NI], int stage, int kk) {
    const char* la = smem + stage * STAGE;
#pragma unroll
    for (int f = 0; f < NI; ++f)
      bf[f] = tb.read(la + TA::BYTES, lane, wn, f, kk);
#pragma unroll
    for (int f = 0; f < MI; ++f) af[f] = ta.read(la, lane, wm, f, kk);
  };
  constexpr int PER = sizeof(T) == 4 ? 4 : 1;  // instructions a fragment pair
  constexpr int READS = MI * TA::READS + NI * TB::READS;
  constexpr int LOADS = TA::LOADS + TB::LOADS;
  if (t0 < t1) {
#pragma unroll
    for (int q = 0; q < STAGES; ++q) load(t0 + q, q);
    meet<(STAGES - 1) * LOADS>();
    int stage = 0;
    int64_t t = t0;
    if (ragged && t + 1 == t1) settle(stage);
    read(a0, b0, stage, 0);
    auto turn = [&](auto last) {
      const int next = stage + 1 < STAGES ? stage + 1 : 0;
      read(a1, b1, stage, 1);
      multiply(acc, a0, b0);
      interleave<READS, MI * NI * PER, 0>();
      meet<(STAGES - 2) * LOADS>();
      if constexpr (decltype(last)::value) settle(next);
      load(t + STAGES, stage);
      read(a0, b0, next, 0);
      multiply(acc, a1, b1);
      interleave<READS, MI * NI * PER, LOADS>();
      stage = next;
      ++t;
    };
    // the turn that clears stands apart: a branch in the loop costs 2 %
    while (t + 1 + ragged < t1) turn(std::false_type{});
    if (t + 1 < t1) turn(std::true_type{});
    read(a1, b1, stage, 1);
    multiply(acc, a0, b0);
    multiply(acc, a1, b1);
  }

  meet<0>();
  write_out<T, MI, NI, WAVES, STAGES * STAGE>(p, smem, acc, wave, lane, split,
                                              i0 + wm, j0 + wn);
}

template <typename T, int BM, int BN, int WM, int WN, int STAGES, bool A_COL,
          bool B_COL>
__global__ __launch_bounds__(WM * WN * 64, 2) void product_k(Product p) {
  __shared__ __align__(16) char smem[lds_bytes<T, BM, BN, STAGES>()];
  product_block<T, BM, BN, WM, WN, STAGES, A_COL, B_COL>(
      p, xcd_swizzle(blockIdx.x, gridDim.x), smem);
}

// The bias gradient from partial sums of act_bwd_k (T: float), or from dz
// itself where the small backward pass has it anyway: FOLD_COLS columns a block
// of 256 threads.
constexpr int FOLD_COLS = 16;

template <typename From, typename T>
__device__ __forceinline__ void fold_bias(const From* rows, int64_t ld,
                                          int64_t count, T* dbias, int64_t n,
                                          int64_t block, char* smem) {
  constexpr int LANES = 256 / FOLD_COLS;
  double* part = reinterpret_cast<double*>(smem);
  const int col = threadIdx.x % FOLD_COLS, lane = threadIdx.x / FOLD_COLS;
  const int64_t j = block * FOLD_COLS + col;
  double sum = 0.0;
  if (j < n)
#pragma unroll 8
    for (int64_t c = lane; c < count; c += LANES) sum += to_f32(rows[c * ld + j]);
  part[threadIdx.x] = sum;
  __syncthreads();
  if (lane == 0 && j < n) {
    for (int k = 1; k < LANES; ++k) sum += part[k * FOLD_COLS + col];
    dbias[j] = from_f32<T>((float)sum);
  }
}

// Both products of a small layer's backward pass and the fold of its bias
// gradient, side by side in one launch: each alone leaves most of the GPU
// idle, and a launch costs the host 4 us.
template <typename T>
__global__ __launch_bounds__(256, 2) void backward_small_k(
    Product dx, Product dw, DdlBiasFold bias) {
  __shared__ __align__(16) char smem[lds_bytes<T, 64, 64, 4>()];
  unsigned id = blockIdx.x;
  const unsigned nx = dx.tiles_m * dx.tiles_n, nw = dw.tiles_m * dw.tiles_n;
  if (id < nx) {
    product_block<T, 64, 64, 4, 1, 4, false, true>(dx, id, smem);
  } else if (id < nx + nw) {
    product_block<T, 64, 64, 4, 1, 4, true, true>(dw, id - nx, smem);
  } else {
    id -= nx + nw;
    if (bias.partials)
      fold_bias(bias.partials, bias.n, bias.chunks, (T*)bias.dbias, bias.n, id,
                smem);
    else
      fold_bias((const T*)dw.a, dw.lda / (int64_t)sizeof(T), dw.r,
                (T*)bias.dbias, bias.n, id, smem);
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
  const float* first = slabs + i * ldslab + j;
  const int64_t slab = e.m * ldslab;
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    const Vec8<float> q = load8(first + s * slab);
#pragma unroll
    for (int k = 0; k < 8; ++k) sum[k] += q.v[k];
  }
  float bias[8];
  load_bias8<T>(e, j, bias);
  finish8<T>(e, i, j, sum, bias);
}

// ---- host ------------------------------------------------------------------

inline int compute_units() {
  static const int n = [] {
    hipDeviceProp_t prop;
    return hipGetDeviceProperties(&prop, 0) == hipSuccess
               ? prop.multiProcessorCount : 256;
  }();
  return n;
}

// A tile of bm x bn, blocks a compute unit holds, and measured times in us: of
// a step (128 bytes of r) where half of the room is taken and where all is, and
// of a block's beginning and end.
struct TileKind {
  int bm, bn, stages, per_unit;
  float alone, full, ends;
};

// bf16 and f16.  Each is fastest somewhere (us, the kernel alone; next best):
//   256 x 256     4096^3 104, 128 x 128 122; dx of 512 x 25088 -> 4096 94, 120
//   256 x 128     its forward, split in four, 97, 256 x 256 in eight 100
//   128 x 128, 4  2048^3 24, 128 x 64 27; 1024 x 4096 -> 4096 42, 45
//   128 x 128, 2  dW of 256 x 25088 -> 4096 93, 256 x 256 121
//   128 x 64      512 x 4096 -> 4096 29, 64 x 64 31
//   64 x 64       512^3 6.2, 128 x 64 7.5
constexpr TileKind KINDS16[] = {{256, 256, 2, 1, 1.25f, 1.6f, 12.f},
                                {256, 128, 3, 1, 0.8f, 0.88f, 9.f},
                                {128, 128, 4, 1, 0.45f, 0.54f, 6.f},
                                {128, 128, 2, 2, 0.75f, 1.f, 5.f},
                                {128, 64, 3, 2, 0.39f, 0.64f, 4.5f},
                                {64, 64, 4, 2, 0.27f, 0.45f, 3.f}};
// float32: 4096^3 980 (128 x 128), 1016, 1127; dx of 512 x 25088 -> 4096 977,
// 934 (128 x 64), 968; 256 x 2048 -> 1000 26, 21, 19 (64 x 64).
constexpr TileKind KINDS32[] = {{128, 128, 2, 2, 2.f, 3.75f, 5.f},
                                {128, 64, 3, 2, 1.05f, 2.f, 5.f},
                                {64, 64, 4, 2, 0.64f, 1.1f, 4.f}};

// The tile and the split of r with the smallest estimate: rounds of blocks
// over the compute units, and for a split the launch that joins its slabs
// (3 us and 0.2 us a MB of them).
inline void plan_product(DdlProduct* p) {
  constexpr int SPLITS[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32};
  const float units = (float)compute_units();
  p->steps = cdiv(p->r * (p->dtype == 0 ? 4 : 2), LINE);
  p->kind = -1;
  // what any of them has to move, at 5.5 TB/s
  const float memory = (p->dtype == 0 ? 4.f : 2.f) / 5.5e6f *
                       ((float)p->m * p->r + (float)p->n * p->r +
                        (float)p->m * p->n);
  auto consider = [&](const TileKind& k, int kind) {
    const float tiles = (float)(cdiv(p->m, k.bm) * cdiv(p->n, k.bn));
    for (const int s : SPLITS) {
      if (s > 1 && p->steps < 2 * s) break;
      const float per = std::ceil((float)p->steps / s);
      const float blocks = tiles * s;
      float rounds = blocks / (units * k.per_unit);
      // up to half of the units' room, then towards all of it
      const float share = std::min(std::max(2.f * rounds - 1.f, 0.f), 1.f);
      const float step = k.alone + share * (k.full - k.alone);
      // many rounds do not end together
      rounds = rounds <= 3.f ? std::ceil(rounds) : rounds + 0.5f;
      float us = rounds * (k.ends + per * step);
      us = std::max(us, memory);
      if (s > 1) us += 3.f + s * (float)p->m * (float)p->n * 8e-7f;
      if (p->kind < 0 || us < p->us) {
        p->us = us;
        p->kind = kind;
        p->bm = k.bm;
        p->bn = k.bn;
        p->stages = k.stages;
        p->splits = s;
      }
    }
  };
  int kind = 0;
  if (p->dtype == 0)
    for (const auto& k : KINDS32) consider(k, kind++);
  else
    for (const auto& k : KINDS16) consider(k, kind++);
  p->steps_per_split = std::max<int64_t>(1, cdiv(p->steps, p->splits));
  p->splits = (int)std::max<int64_t>(1, cdiv(p->steps, p->steps_per_split));
}

// Whether dx and dw, both planned, are better off in backward_small_k: its
// blocks go through the units two at a time, and the longest one is waited
// for; a launch of their own costs each 4 us.
inline bool small_backward(const DdlProduct* dx, const DdlProduct* dw) {
  const TileKind k = dx->dtype == 0 ? KINDS32[2] : KINDS16[5];
  float work = 0.f, longest = 0.f;
  for (const auto* p : {dx, dw}) {
    const float tiles = (float)(cdiv(p->m, k.bm) * cdiv(p->n, k.bn));
    work += tiles * (k.ends + p->steps * k.full);
    longest = std::max(longest, k.ends + p->steps * k.alone);
  }
  return std::max(work / (compute_units() * k.per_unit), longest) <
         dx->us + dw->us + 4.f;
}

template <typename T> Product product_of(const DdlProduct* d) {
  Product p{};
  p.a = (const char*)d->a;
  p.b = (const char*)d->b;
  p.lda = d->lda * (int64_t)sizeof(T);
  p.ldb = d->ldb * (int64_t)sizeof(T);
  p.r = d->r;
  p.steps = d->steps;
  p.steps_per_split = d->steps_per_split;
  p.splits = d->splits;
  p.tiles_m = (int)cdiv(d->m, d->bm);
  p.tiles_n = (int)cdiv(d->n, d->bn);
  p.slabs = d->slabs;
  p.ldslab = cdiv(d->n, 8) * 8;
  p.e = epilogue_of(d);
  return p;
}

template <typename T, int BM, int BN, int WM, int WN, int STAGES>
void launch_product(const Product& p, int a_col, int b_col, hipStream_t s) {
  const dim3 grid(p.tiles_m * p.tiles_n * p.splits), block(WM * WN * 64);
  if (a_col && b_col)
    product_k<T, BM, BN, WM, WN, STAGES, true, true><<<grid, block, 0, s>>>(p);
  else if (b_col)
    product_k<T, BM, BN, WM, WN, STAGES, false, true>
        <<<grid, block, 0, s>>>(p);
  else
    product_k<T, BM, BN, WM, WN, STAGES, false, false>
        <<<grid, block, 0, s>>>(p);
}

template <typename T>
void run_product(const DdlProduct* d, hipStream_t s) {
  const Product p = product_of<T>(d);
  if constexpr (sizeof(T) == 2) {
    switch (d->kind) {
      case 0:
        launch_product<T, 256, 256, 2, 4, 2>(p, d->a_col, d->b_col, s);
        break;
      case 1:
        launch_product<T, 256, 128, 4, 2, 3>(p, d->a_col, d->b_col, s);
        break;
      case 2:
        launch_product<T, 128, 128, 4, 2, 4>(p, d->a_col, d->b_col, s);
        break;
      case 3:
        launch_product<T, 128, 128, 4, 2, 2>(p, d->a_col, d->b_col, s);
        break;
      case 4:
        launch_product<T, 128, 64, 4, 1, 3>(p, d->a_col, d->b_col, s);
        break;
      case 5:
        launch_product<T, 64, 64, 4, 1, 4>(p, d->a_col, d->b_col, s);
        break;
    }
  } else {
    switch (d->kind) {
      case 0:
        launch_product<T, 128, 128, 4, 2, 2>(p, d->a_col, d->b_col, s);
        break;
      case 1:
        launch_product<T, 128, 64, 4, 1, 3>(p, d->a_col, d->b_col, s);
        break;
      case 2:
        launch_product<T, 64, 64, 4, 1, 4>(p, d->a_col, d->b_col, s);
        break;
    }
  }
  if (p.splits > 1) {
    const int64_t threads = p.ldslab / 8 * d->m;
    join_k<T><<<(unsigned)cdiv(threads, 256), 256, 0, s>>>(
        p.slabs, p.splits, p.ldslab, p.e);
  }
}

template <typename T>
void run_backward_small(DdlProduct dx, DdlProduct dw, const DdlBiasFold& bias,
                        hipStream_t s) {
  for (auto* p : {&dx, &dw}) {
    p->kind = sizeof(T) == 4 ? 2 : 5;
    p->bm = p->bn = 64;
    p->splits = 1;
    p->steps_per_split = std::max<int64_t>(1, p->steps);
  }
  const Product x = product_of<T>(&dx), w = product_of<T>(&dw);
  const int64_t blocks = (int64_t)x.tiles_m * x.tiles_n +
                         (int64_t)w.tiles_m * w.tiles_n +
                         cdiv(bias.n, FOLD_COLS);
  backward_small_k<T><<<(unsigned)blocks, 256, 0, s>>>(x, w, bias);
}

}  // namespace
