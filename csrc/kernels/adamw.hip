// Multi-tensor AdamW (float32 or 8-bit moments), global gradient norm, and
// gradient scaling.
//
// For every element, with c1 = 1 - beta1^t, c2 = 1 - beta2^t in 64 bits:
//   g = grad * grad_mul * coef
//   m = beta1 m + (1 - beta1) g;   v = beta2 v + (1 - beta2) g^2
//   w = w (1 - lr wd) - (lr / c1) m / (sqrt(v) / sqrt(c2) + eps)
// One pass; the bound is memory.  A 16-bit parameter moves 28 B with float32
// moments (gradient 2, master 8, moments 16, parameter 2) and 16 B with
// 8-bit ones.
//
// The tensors' pointers travel as kernel arguments, read anew from the
// tensors at every step: there is no table on the device that could go
// stale, nothing is copied from the host, and a captured step replays.
//
// 8-bit moments: m and r = sqrt(v) are e4m3 codes times one float32 scale
// (largest magnitude / 448) for each 256 consecutive elements; r rather than
// v, because e4m3 spans 2^18 and v twice the octaves of r.  beta2 = 0.999
// moves v by about 0.1 % a step and a code is 6 to 12 % wide: to nearest, v
// would never move.  So a code is rounded up with the probability of the part
// that rounding down drops, by 16 bits of a hash of (seed, step, tensor,
// element): the expected code is the value, and a run can be repeated bit
// for bit.  One exception: a positive r takes at least the smallest code,
// 2^-9 of a scale.  Rounded to zero, r would leave the next step without its
// denominator while m, drawn by other bits, may have been rounded up: with
// gradients at 1e-6 of their block's largest, steps of the first twenty reached
// 364 times lr; they reach 1.5 times so (float32 moments: 1.0).
//
// This file is compiled without fast-math: infinities and NaN keep their
// meaning, divisions and roots are correctly rounded.  Products and sums of
// the moments are rounded one by one, so that the codes are the same as
// those of the CPU path.
#include "common.h"
#include "train_api.h"

#include <cmath>

#pragma clang fp contract(off)

namespace {

constexpr int THREADS = 256;
constexpr int MOMENT_BLOCK = DDL_MOMENT_BLOCK;
static_assert(MOMENT_BLOCK == 32 * 8, "half a wave holds a block");

// Kernel arguments hold at most 4 KiB.  A tensor's length is told by its
// blocks and by what its last block lacks.
constexpr int MAX_T32 = 84;
constexpr int MAX_T8 = 62;
constexpr int MAX_NORM = 266;
constexpr int MAX_PREP = 192;

struct Scalars {  // per tensor, written by prepare_k
  float step_size;     // lr / c1
  float inv_sqrt_c2;   // 1 / sqrt(c2)
  uint32_t key;
  uint32_t pad;
};

struct T32 {
  void* p;
  const void* g;
  float* w;
  float* m;
  float* v;
};

struct T8 : T32 {
  float* ms;
  float* vs;
};

struct TG {
  void* g;
};

template <typename Row, int MAX> struct Args {
  Row t[MAX];
  int first[MAX + 1];   // first block of each tensor, and the end
  uint16_t lacks[MAX];  // elements that the last block is short of a chunk
  uint8_t aligned[MAX]; // every pointer of the tensor takes 16-byte accesses
  int count;
  int chunk;            // elements a block

  // Elements of this block of tensor i.
  __device__ __forceinline__ void range(int i, int64_t& begin,
                                        int64_t& end) const {
    const int block = (int)blockIdx.x - first[i];
    begin = (int64_t)block * chunk;
    end = begin + chunk -
          ((int)blockIdx.x + 1 == first[i + 1] ? lacks[i] : 0);
  }
};
using NormArgs = Args<TG, MAX_NORM>;
static_assert(sizeof(Args<T32, MAX_T32>) < 4000, "kernel argument limit");
static_assert(sizeof(Args<T8, MAX_T8>) < 4000, "kernel argument limit");
static_assert(sizeof(NormArgs) + sizeof(DdlNormFold) < 4080, "kernel argument limit");

struct PrepArgs {
  float* step[MAX_PREP];
  uint32_t index[MAX_PREP];
  int count;
};

struct Consts {
  float beta1, one_minus_beta1, beta2, one_minus_beta2, eps, decay, grad_mul;
};

// The tensor whose blocks hold `block`: the last whose first is not past it.
__device__ __forceinline__ int find_tensor(const int* first, int count,
                                           int block) {
  int lo = 0, hi = count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first[mid] <= block) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__host__ __device__ __forceinline__ uint32_t mix(uint32_t x) {
  x ^= x >> 16;
  x *= 0x6A09E667u;
  x ^= x >> 15;
  x *= 0x5DB3D743u;
  x ^= x >> 16;
  return x;
}

// Sum of up to 1024 threads, in the same order every time, to all of them.
__device__ __forceinline__ double block_sum(double v) {
  __shared__ double part[16];
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_down(v, off, WAVE);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  double total = 0.0;
  for (int i = 0; i < (int)blockDim.x / WAVE; ++i) total += part[i];
  return total;
}

// norm = sqrt(sum of the partial sums) * mul; the coefficient that brings it
// to max_norm, which one thread stores.  NaN stays NaN, as in torch's
// clip_grad_norm_.
__device__ __forceinline__ float fold_norm(const DdlNormFold& f, bool store) {
  double sum = 0.0;
#pragma unroll 4
  for (int64_t i = threadIdx.x; i < f.blocks; i += blockDim.x)
    sum += f.partials[i];
  sum = block_sum(sum);
  const float n = (float)(sqrt(sum) * f.mul);
  float k = (float)f.max_norm / (n + 1e-6f);
  k = k >= 1.f ? 1.f : k;
  if (store && threadIdx.x == 0) {
    *f.norm = n;
    *f.coef = k;
  }
  return k;
}

constexpr int FOLD_THREADS = 1024;

__global__ __launch_bounds__(FOLD_THREADS) void fold_norm_k(DdlNormFold f) {
  fold_norm(f, true);
}

// One thread a tensor; the fold of the norm rides along.  beta^t is
// exp(t log beta) in 64 bits, good to 2^-45 for the steps that matter.
__global__ __launch_bounds__(FOLD_THREADS) void prepare_k(
    PrepArgs a, double lr, double log_beta1, double log_beta2, uint32_t seed,
    Scalars* out, DdlNormFold f) {
  if (f.partials) fold_norm(f, true);
  const int i = threadIdx.x;
  if (i >= a.count) return;
  const float t = *a.step[i] + 1.f;
  *a.step[i] = t;
  Scalars s;
  s.step_size = (float)(lr / -expm1((double)t * log_beta1));
  s.inv_sqrt_c2 = (float)(1.0 / sqrt(-expm1((double)t * log_beta2)));
  const uint32_t stream = mix(seed + 0x9E3779B9u * (a.index[i] + 1u));
  s.key = mix(stream + (uint32_t)t);
  s.pad = 0;
  out[i] = s;
}

struct Update {
  Consts c;
  float mul, step_size, inv_sqrt_c2;
  __device__ __forceinline__ void operator()(float g, float& w, float& m,
                                             float& v, float& root) const {
    g *= mul;
    m = c.beta1 * m + c.one_minus_beta1 * g;
    v = c.beta2 * v + c.one_minus_beta2 * (g * g);
    root = sqrtf(v);
    w = w * c.decay - (step_size * m) / (root * inv_sqrt_c2 + c.eps);
  }
};

template <typename T, bool MASTER>
__global__ __launch_bounds__(THREADS) void adamw32_k(
    Args<T32, MAX_T32> a, Consts c, const Scalars* __restrict__ ws,
    const float* __restrict__ coef) {
  const int ti = find_tensor(a.first, a.count, blockIdx.x);
  const T32 t = a.t[ti];
  const Scalars s = ws[ti];
  Update up{c, coef ? c.grad_mul * *coef : c.grad_mul, s.step_size,
            s.inv_sqrt_c2};
  int64_t begin, end;
  a.range(ti, begin, end);
  T* p = (T*)t.p;
  const T* grad = (const T*)t.g;
  if (a.aligned[ti]) {
    for (int64_t i = begin + threadIdx.x * 8; i + 8 <= end;
         i += THREADS * 8) {
      Vec8<T> g = load8(grad + i);
      Vec8<float> w = load8(t.w + i), m = load8(t.m + i), v = load8(t.v + i);
      Vec8<T> out;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float root;
        up(to_f32(g.v[j]), w.v[j], m.v[j], v.v[j], root);
        if constexpr (MASTER) out.v[j] = from_f32<T>(w.v[j]);
      }
      store8(t.w + i, w);
      store8(t.m + i, m);
      store8(t.v + i, v);
      if constexpr (MASTER) store8(p + i, out);
    }
  }
  const int64_t done = a.aligned[ti] ? begin + ((end - begin) & ~7) : begin;
  for (int64_t i = done + threadIdx.x; i < end; i += THREADS) {
    float w = t.w[i], m = t.m[i], v = t.v[i], root;
    up(to_f32(grad[i]), w, m, v, root);
    t.w[i] = w;
    t.m[i] = m;
    t.v[i] = v;
    if constexpr (MASTER) p[i] = from_f32<T>(w);
  }
}

// ---- 8-bit moments ---------------------------------------------------------

// A code of y >= 0 (at most 448, or NaN), rounded up by chance `r` of 2^16.
// At and above 2^-6 a code keeps 3 bits of the mantissa; below, codes are
// 2^-9 apart.  Both arms give a value that e4m3 holds, so the conversion
// that follows does not round.
__device__ __forceinline__ float round_by_chance(float y, uint32_t r) {
  const float normal =
      __uint_as_float((__float_as_uint(y) + (r << 4)) & ~0xFFFFFu);
  const float small =
      floorf(y * 512.f + (float)r * 0x1p-16f) * (1.f / 512.f);
  return y < 0x1p-6f ? small : normal;
}

__device__ __forceinline__ bool finite(float x) {
  return (__float_as_uint(x) & 0x7F800000u) != 0x7F800000u;
}

__device__ __forceinline__ uint32_t pack4(const float* q) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], r, true);
}

__device__ __forceinline__ void unpack4(uint32_t c, float* q) {
  auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false);
  auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
  q[0] = lo[0]; q[1] = lo[1]; q[2] = hi[0]; q[3] = hi[1];
}

// Largest of 32 lanes.
__device__ __forceinline__ float half_wave_max(float x) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) x = fmaxf(x, __shfl_xor(x, off, WAVE));
  return x;
}

// Codes of 8 values of a lane, whose block's largest finite magnitude is
// `top`.  An infinite or NaN value becomes a NaN code and leaves its block's
// scale alone; a block whose values are all below 2^-100 becomes zeros.
// LEAST: no value is below zero, and a positive one of another block takes at
// least the smallest code.
template <bool LEAST>
__device__ __forceinline__ uint2 encode8(const float* x, float top,
                                         const uint32_t* r, int shift,
                                         float& scale) {
  const bool tiny = top < 0x1p-100f;
  scale = tiny ? 0.f : top * (1.f / 448.f);
  const float inv = tiny ? 0.f : (1.f / top) * 448.f;
  float q[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float y = fminf(fabsf(x[j]) * inv, 448.f);
    const float code = round_by_chance(y, (r[j] >> shift) & 0xFFFFu);
    const float e = LEAST ? fmaxf(code, y > 0.f ? 0x1p-9f : 0.f)
                          : copysignf(code, x[j]);
    q[j] = finite(x[j]) ? e : __uint_as_float(0x7FC00000u);
  }
  return uint2{pack4(q), pack4(q + 4)};
}

// Half a wave takes one block of 256 elements, 8 a lane.
template <typename T, bool MASTER>
__global__ __launch_bounds__(THREADS) void adamw8_k(
    Args<T8, MAX_T8> a, Consts c, const Scalars* __restrict__ ws,
    const float* __restrict__ coef) {
  const int ti = find_tensor(a.first, a.count, blockIdx.x);
  const T8 t = a.t[ti];
  const Scalars s = ws[ti];
  Update up{c, coef ? c.grad_mul * *coef : c.grad_mul, s.step_size,
            s.inv_sqrt_c2};
  int64_t begin, end;
  a.range(ti, begin, end);
  T* p = (T*)t.p;
  const T* grad = (const T*)t.g;
  uint8_t* mc = (uint8_t*)t.m;
  uint8_t* vc = (uint8_t*)t.v;
  const bool aligned = a.aligned[ti];
  // The trip count is the same for every lane of a half wave, which the
  // shuffles need: it depends on the half wave's first element alone.
  const int64_t lane = threadIdx.x & 31;
  for (int64_t b = begin + (threadIdx.x >> 5) * MOMENT_BLOCK; b < end;
       b += THREADS * 8) {
    const int64_t i = b + lane * 8;
    const int64_t block = b / MOMENT_BLOCK;
    const bool whole = aligned && i + 8 <= end;
    float g[8], w[8], m[8], v[8], root[8];
    if (whole) {
      const Vec8<T> gv = load8(grad + i);
      const Vec8<float> wv = load8(t.w + i);
      const uint2 mv = *reinterpret_cast<const uint2*>(mc + i);
      const uint2 vv = *reinterpret_cast<const uint2*>(vc + i);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        g[j] = to_f32(gv.v[j]);
        w[j] = wv.v[j];
      }
      unpack4(mv.x, m); unpack4(mv.y, m + 4);
      unpack4(vv.x, v); unpack4(vv.y, v + 4);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        g[j] = w[j] = m[j] = v[j] = 0.f;
        if (i + j < end) {
          g[j] = to_f32(grad[i + j]);
          w[j] = t.w[i + j];
          m[j] = __builtin_amdgcn_cvt_f32_fp8((int)mc[i + j], 0);
          v[j] = __builtin_amdgcn_cvt_f32_fp8((int)vc[i + j], 0);
        }
      }
    }
    const float ms = t.ms[block], vs = t.vs[block];
    float mtop = 0.f, vtop = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      m[j] *= ms;
      const float r = v[j] * vs;
      v[j] = r * r;
      up(g[j], w[j], m[j], v[j], root[j]);
      if (finite(m[j])) mtop = fmaxf(mtop, fabsf(m[j]));
      if (finite(root[j])) vtop = fmaxf(vtop, root[j]);
    }
    mtop = half_wave_max(mtop);
    vtop = half_wave_max(vtop);
    uint32_t r[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = mix((uint32_t)(i + j) ^ s.key);
    float ms_new, vs_new;
    const uint2 mq = encode8<false>(m, mtop, r, 0, ms_new);
    const uint2 vq = encode8<true>(root, vtop, r, 16, vs_new);
    if (lane == 0) {
      t.ms[block] = ms_new;
      t.vs[block] = vs_new;
    }
    if (whole) {
      Vec8<float> wv;
      Vec8<T> out;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        wv.v[j] = w[j];
        if constexpr (MASTER) out.v[j] = from_f32<T>(w[j]);
      }
      store8(t.w + i, wv);
      if constexpr (MASTER) store8(p + i, out);
      *reinterpret_cast<uint2*>(mc + i) = mq;
      *reinterpret_cast<uint2*>(vc + i) = vq;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (i + j < end) {
          t.w[i + j] = w[j];
          if constexpr (MASTER) p[i + j] = from_f32<T>(w[j]);
          mc[i + j] = (uint8_t)((j < 4 ? mq.x : mq.y) >> (8 * (j & 3)));
          vc[i + j] = (uint8_t)((j < 4 ? vq.x : vq.y) >> (8 * (j & 3)));
        }
      }
    }
  }
}

// ---- gradient norm and scaling --------------------------------------------

// Squares are summed in 64 bits: a float32 gradient of 2e19 has a square
// that 32 bits do not hold, and the sum's order does not matter to 32 bits.
template <typename T>
__global__ __launch_bounds__(THREADS) void grad_norm_k(NormArgs a,
                                                       double* partials) {
  const int ti = find_tensor(a.first, a.count, blockIdx.x);
  const T* g = (const T*)a.t[ti].g;
  int64_t begin, end;
  a.range(ti, begin, end);
  const bool aligned = a.aligned[ti];
  double sum = 0.0;
  auto add = [&](const Vec8<T>& x) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const double d = (double)to_f32(x.v[j]);
      sum += d * d;
    }
  };
  if (aligned) {
    constexpr int TURN = THREADS * 8;
    int64_t i = begin + threadIdx.x * 8;
    for (; i + TURN + 8 <= end; i += 2 * TURN) {
      const Vec8<T> x = load8(g + i), y = load8(g + i + TURN);
      add(x);
      add(y);
    }
    for (; i + 8 <= end; i += TURN) add(load8(g + i));
  }
  const int64_t done = aligned ? begin + ((end - begin) & ~7) : begin;
  for (int64_t i = done + threadIdx.x; i < end; i += THREADS) {
    const double d = (double)to_f32(g[i]);
    sum += d * d;
  }
  sum = block_sum(sum);
  if (threadIdx.x == 0) partials[blockIdx.x] = sum;
}

// FOLD: the coefficient comes from the partial sums, which every block adds up.
template <typename T, bool FOLD>
__global__ __launch_bounds__(THREADS) void grad_scale_k(NormArgs a,
                                                        DdlNormFold f) {
  const float k = FOLD ? fold_norm(f, blockIdx.x == 0) : *f.coef;
  if (k == 1.f) return;
  const int ti = find_tensor(a.first, a.count, blockIdx.x);
  T* g = (T*)a.t[ti].g;
  int64_t begin, end;
  a.range(ti, begin, end);
  const bool aligned = a.aligned[ti];
  if (aligned) {
    for (int64_t i = begin + threadIdx.x * 8; i + 8 <= end;
         i += THREADS * 8) {
      Vec8<T> x = load8(g + i);
#pragma unroll
      for (int j = 0; j < 8; ++j) x.v[j] = from_f32<T>(to_f32(x.v[j]) * k);
      store8(g + i, x);
    }
  }
  const int64_t done = aligned ? begin + ((end - begin) & ~7) : begin;
  for (int64_t i = done + threadIdx.x; i < end; i += THREADS)
    g[i] = from_f32<T>(to_f32(g[i]) * k);
}

// ---- host ------------------------------------------------------------------

constexpr int64_t MAX_BLOCKS = 1 << 23;  // a grid holds below 2^32 threads

// Elements a block takes: two turns of its threads.  ResNet-50's step takes
// 141 us so, 146 with four turns; few elements are spread over more blocks:
// 2 million take 10.4 us in single turns, 12.4 in four.
int chunk_of(int64_t total) {
  constexpr int TURN = THREADS * 8;
  static_assert(TURN % MOMENT_BLOCK == 0, "a chunk holds whole blocks");
  return total >= ((int64_t)1 << 23) ? 2 * TURN : TURN;
}

template <typename Row> int64_t total_of(const Row* t, int64_t count) {
  int64_t total = 0;
  for (int64_t i = 0; i < count; ++i) total += t[i].n;
  return total;
}

bool takes16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Hands `launch` the tensors in groups of at most MAX, with the blocks that
// each group needs and the place of its first tensor.
template <typename Row, int MAX, typename Tensor, typename Fill,
          typename Launch>
void in_groups(const Tensor* t, int64_t count, Fill fill, Launch launch) {
  Args<Row, MAX> a;
  a.count = 0;
  a.chunk = chunk_of(total_of(t, count));
  int64_t blocks = 0, start = 0;
  auto flush = [&](int64_t next) {
    a.first[a.count] = (int)blocks;
    if (blocks) launch(a, (int)blocks, start);
    a.count = 0;
    blocks = 0;
    start = next;
  };
  for (int64_t i = 0; i < count; ++i) {
    const int64_t more = cdiv(t[i].n, a.chunk);
    if (a.count == MAX || blocks + more > MAX_BLOCKS) flush(i);
    a.first[a.count] = (int)blocks;
    a.lacks[a.count] = (uint16_t)(more * a.chunk - t[i].n);
    a.aligned[a.count] = fill(a.t[a.count], t[i]);
    ++a.count;
    blocks += more;
  }
  flush(count);
}

Consts consts_of(const DdlAdamScalars* c) {
  return Consts{(float)c->beta1, (float)(1.0 - c->beta1),
                (float)c->beta2, (float)(1.0 - c->beta2),
                (float)c->eps,   (float)(1.0 - c->lr * c->weight_decay),
                c->grad_mul};
}

template <typename T, bool MASTER>
void run_adamw(const DdlAdamTensor* t, int64_t count, const Consts& c,
               int bits, const Scalars* ws, const float* coef,
               hipStream_t s) {
  auto common = [](T32& r, const DdlAdamTensor& t) {
    r.p = t.p;
    r.g = t.g;
    r.w = t.w;
    r.m = (float*)t.m;
    r.v = (float*)t.v;
    return (!MASTER || takes16(t.p)) && takes16(t.g) && takes16(t.w);
  };
  if (bits == 32) {
    in_groups<T32, MAX_T32>(
        t, count,
        [&](T32& r, const DdlAdamTensor& t) {
          return common(r, t) && takes16(t.m) && takes16(t.v);
        },
        [&](const auto& a, int blocks, int64_t at) {
          adamw32_k<T, MASTER><<<blocks, THREADS, 0, s>>>(a, c, ws + at, coef);
        });
  } else {
    in_groups<T8, MAX_T8>(
        t, count,
        [&](T8& r, const DdlAdamTensor& t) {
          r.ms = t.ms;
          r.vs = t.vs;
          return common(r, t) && ((uintptr_t)t.m & 7) == 0 &&
                 ((uintptr_t)t.v & 7) == 0;
        },
        [&](const auto& a, int blocks, int64_t at) {
          adamw8_k<T, MASTER><<<blocks, THREADS, 0, s>>>(a, c, ws + at, coef);
        });
  }
}

template <typename Launch>
void norm_groups(const DdlGradTensor* t, int64_t count, Launch launch) {
  in_groups<TG, MAX_NORM>(
      t, count,
      [](TG& r, const DdlGradTensor& t) {
        r.g = t.g;
        return takes16(t.g);
      },
      launch);
}

}  // namespace

extern "C" {

int64_t ddl_adamw_ws_bytes(int64_t count) {
  return count * (int64_t)sizeof(Scalars);
}

void ddl_adamw_prepare(const DdlAdamTensor* t, int64_t count,
                       const DdlAdamScalars* c, void* ws,
                       const DdlNormFold* fold, hipStream_t s) {
  DdlNormFold f{};
  if (fold) f = *fold;
  for (int64_t at = 0; at < count; at += MAX_PREP) {
    PrepArgs a;
    a.count = (int)std::min<int64_t>(MAX_PREP, count - at);
    for (int k = 0; k < a.count; ++k) {
      a.step[k] = t[at + k].step;
      a.index[k] = t[at + k].index;
    }
    const int threads = f.partials ? FOLD_THREADS : MAX_PREP;
    prepare_k<<<1, threads, 0, s>>>(a, c->lr, std::log(c->beta1),
                                    std::log(c->beta2), c->seed,
                                    (Scalars*)ws + at, f);
    f = DdlNormFold{};
  }
}

void ddl_adamw(const DdlAdamTensor* t, int64_t count,
               const DdlAdamScalars* c, int dtype, int bits, const void* ws,
               const float* coef, hipStream_t s) {
  const Consts k = consts_of(c);
  const Scalars* sc = (const Scalars*)ws;
  switch (dtype) {
    case 0: run_adamw<float, false>(t, count, k, bits, sc, coef, s); break;
    case 1: run_adamw<bf16, true>(t, count, k, bits, sc, coef, s); break;
    case 2: run_adamw<f16, true>(t, count, k, bits, sc, coef, s); break;
  }
}

int64_t ddl_grad_norm_blocks(const DdlGradTensor* t, int64_t count) {
  const int chunk = chunk_of(total_of(t, count));
  int64_t blocks = 0;
  for (int64_t i = 0; i < count; ++i) blocks += cdiv(t[i].n, chunk);
  return blocks;
}

void ddl_grad_norm_partials(const DdlGradTensor* t, int64_t count, int dtype,
                            double* partials, hipStream_t s) {
  norm_groups(t, count, [&](const NormArgs& a, int blocks, int64_t) {
    switch (dtype) {
      case 0: grad_norm_k<float><<<blocks, THREADS, 0, s>>>(a, partials); break;
      case 1: grad_norm_k<bf16><<<blocks, THREADS, 0, s>>>(a, partials); break;
      case 2: grad_norm_k<f16><<<blocks, THREADS, 0, s>>>(a, partials); break;
    }
    partials += blocks;
  });
}

void ddl_grad_norm_fold(const DdlNormFold* f, hipStream_t s) {
  fold_norm_k<<<1, FOLD_THREADS, 0, s>>>(*f);
}

void ddl_grad_scale(const DdlGradTensor* t, int64_t count, int dtype,
                    const DdlNormFold* f, int fold, hipStream_t s) {
  norm_groups(t, count, [&](const NormArgs& a, int blocks, int64_t) {
#define RUN(T)                                                \
  if (fold)                                                   \
    grad_scale_k<T, true><<<blocks, THREADS, 0, s>>>(a, *f);  \
  else                                                        \
    grad_scale_k<T, false><<<blocks, THREADS, 0, s>>>(a, *f)
    switch (dtype) {
      case 0: RUN(float); break;
      case 1: RUN(bf16); break;
      case 2: RUN(f16); break;
    }
#undef RUN
  });
}

}  // extern "C"
