// Newton-Schulz orthogonalisation and the Muon server step for MI355X
// (gfx950).
//
// For a matrix U of m x n values, with s = min(m, n) and L = max(m, n):
//     X = U / (|U|_F + eps),  then `steps` times
//     G = X X^T (on the side of length s),  X <- (a I + b G + c G^2) X.
//
// Two ways to the same result, both f32-exact to a few last places:
//
// thin   G is taken once, in f64 over the long axis; the steps are then taken
//        on s x s matrices alone (each multiplies X by Q = a I + b G + c G^2
//        and G by Q^2), and one product applies P = Q_1 ... Q_k to U.  Two
//        passes over the values instead of two a step.  G has to be f64: an
//        error in it grows by a^2 = 12 with every step.
// wide   the chain as written, with every operand held as two f16 planes,
//        hi + lo (22 bits): a b = hi hi + hi lo + lo hi on the f16 matrix
//        units, accumulated in f32.  Three f16 products cost 3 / 16 of one
//        f32 product at this card's matrix rates.

#include <ATen/ATen.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include "ops.h"

namespace {

constexpr int WAVE = 64;
constexpr int PAD = 128;      // rows and columns of the wide planes
constexpr float UP = 4096.0f; // planes hold 2^12 times the value

using half4 = __attribute__((ext_vector_type(4))) _Float16;
using half8 = __attribute__((ext_vector_type(8))) _Float16;
using f32x4 = __attribute__((ext_vector_type(4))) float;
using f64x4 = __attribute__((ext_vector_type(4))) double;

template <typename T>
__device__ inline float to_f32(T v);
template <>
__device__ inline float to_f32(float v) { return v; }
template <>
__device__ inline float to_f32(__half v) { return __half2float(v); }
template <>
__device__ inline float to_f32(__hip_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ inline T from_f32(float v);
template <>
__device__ inline float from_f32(float v) { return v; }
template <>
__device__ inline __half from_f32(float v) { return __float2half_rn(v); }
template <>
__device__ inline __hip_bfloat16 from_f32(float v) {
  return __float2bfloat16(v);
}

struct Coeffs { double a, b, c; };

// What a product ends in: the values of `out` (T), or the weights' step
// W <- W keep - rate O.
struct Result {
  void* out;      // orthogonalize: T; Muon: the f32 table
  float keep, rate;
  bool step;
};

template <typename T>
__device__ inline void finish(const Result& r, int64_t at, float o) {
  if (r.step) {
    float* w = (float*)r.out + at;
    *w = *w * r.keep - r.rate * o;
  } else {
    ((T*)r.out)[at] = from_f32<T>(o);
  }
}

// ---------------------------------------------------------------------
// Muon: which matrices a push touches, momentum
// ---------------------------------------------------------------------

__device__ inline int64_t lower_bound(const int64_t* v, int64_t n,
                                      int64_t x) {
  int64_t lo = 0;
  while (n > 0) {
    int64_t h = n / 2;
    if (v[lo + h] < x) { lo += h + 1; n -= h + 1; } else { n = h; }
  }
  return lo;
}

__global__ __launch_bounds__(256) void k_touched(
    int* __restrict__ touched, const int64_t* __restrict__ rows, int64_t n,
    int64_t batch, int64_t m) {
  int64_t b = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (b >= batch) return;
  int64_t lo = lower_bound(rows, n, b * m);
  touched[b] = lo < n && rows[lo] < (b + 1) * m;
}

// M <- mu M + g and U = g + mu M (nesterov) or M, a wave a row.  g is the sum
// of the row's gradients in the order of the push: rows are sorted, order[j]
// is the place of the j-th in `grads`.
__global__ __launch_bounds__(256) void k_momentum(
    float* __restrict__ u, float* __restrict__ momentum,
    const float* __restrict__ grads, const int64_t* __restrict__ rows,
    const int64_t* __restrict__ order, const int* __restrict__ touched,
    int64_t n, int64_t total, int64_t m, int64_t dim, float mu,
    bool nesterov) {
  const int lane = threadIdx.x % WAVE;
  const int64_t waves = (int64_t)gridDim.x * (256 / WAVE);
  for (int64_t r = (int64_t)blockIdx.x * (256 / WAVE) + threadIdx.x / WAVE;
       r < total; r += waves) {
    if (!touched[r / m]) continue;
    const int64_t lo = lower_bound(rows, n, r);
    for (int64_t c = lane; c < dim; c += WAVE) {
      float g = 0.0f;
      for (int64_t j = lo; j < n && rows[j] == r; ++j)
        g += grads[(order ? order[j] : j) * dim + c];
      float v = mu * momentum[r * dim + c] + g;
      momentum[r * dim + c] = v;
      u[r * dim + c] = nesterov ? g + mu * v : v;
    }
  }
}

// ---------------------------------------------------------------------
// thin: G in f64, the chain on s x s, one product
// ---------------------------------------------------------------------

constexpr int THIN_MAX = 320;  // the largest short side
constexpr int SUPER = 128;     // a block's square of G
constexpr int KC = 32;         // long-axis places a block stages at a time
constexpr int PITCH = SUPER + 16;

// Partial sums of G over one chunk of the long axis: part[b][chunk][sp][sp],
// tiles on and under the diagonal.  f64 matrix instructions: 16x16x4, a lane
// holds row (or column) lane % 16 at place lane / 16.  They bound it: 64
// cycles a tile and 4 places.
template <typename T, bool TALL>
__global__ __launch_bounds__(256) void k_gram64(
    double* __restrict__ part, const T* __restrict__ u,
    const int* __restrict__ touched, int64_t long_, int s, int sp,
    int64_t chunk) {
  __shared__ float rows_[KC][PITCH], cols_[KC][PITCH];
  const int64_t b = blockIdx.z;
  if (touched && !touched[b]) return;
  // blockIdx.y counts the pairs of super-tiles (si >= sj)
  int si = 0, sj = blockIdx.y;
  while (sj > si) { sj -= si + 1; ++si; }
  const bool diagonal = si == sj;
  const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE;
  const T* x = u + b * long_ * s;
  const int64_t k0 = blockIdx.x * chunk;
  const int64_t k1 = k0 + chunk < long_ ? k0 + chunk : long_;
  const int pair[2] = {wave, 7 - wave};  // this wave's rows of tiles

  f64x4 acc[2][8];
#pragma unroll
  for (int p = 0; p < 2; ++p)
#pragma unroll
    for (int t = 0; t < 8; ++t) acc[p][t] = (f64x4){0, 0, 0, 0};

  auto stage = [&](float (*to)[PITCH], int base, int64_t k) {
    for (int e = threadIdx.x; e < KC * SUPER; e += 256) {
      // neighbours in memory are neighbours in threads
      int kk = TALL ? e / SUPER : e % KC, c = TALL ? e % SUPER : e / KC;
      int col = base + c;
      float v = 0.0f;
      if (col < s && k + kk < k1)
        v = to_f32(TALL ? x[(k + kk) * s + col] : x[col * long_ + k + kk]);
      to[kk][c] = v;
    }
  };

  for (int64_t k = k0; k < k1; k += KC) {
    __syncthreads();
    stage(rows_, si * SUPER, k);
    if (!diagonal) stage(cols_, sj * SUPER, k);
    __syncthreads();
    const float (*cols)[PITCH] = diagonal ? rows_ : cols_;
    for (int q = 0; q < KC; q += 4) {
      const int kk = q + lane / 16;
      double av[2];
#pragma unroll
      for (int p = 0; p < 2; ++p) av[p] = rows_[kk][pair[p] * 16 + lane % 16];
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        double bv = cols[kk][t * 16 + lane % 16];
#pragma unroll
        for (int p = 0; p < 2; ++p)
          if ((!diagonal || t <= pair[p]) && si * SUPER + pair[p] * 16 < sp &&
              sj * SUPER + t * 16 < sp)
            acc[p][t] = __builtin_amdgcn_mfma_f64_16x16x4f64(av[p], bv,
                                                             acc[p][t], 0, 0,
                                                             0);
      }
    }
  }
  double* out = part + (b * gridDim.x + blockIdx.x) * (int64_t)sp * sp;
#pragma unroll
  for (int p = 0; p < 2; ++p)
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      int i0 = si * SUPER + pair[p] * 16, j0 = sj * SUPER + t * 16;
      if ((diagonal && t > pair[p]) || i0 >= sp || j0 >= sp) continue;
#pragma unroll
      for (int r = 0; r < 4; ++r)
        out[(int64_t)(i0 + lane / 16 + 4 * r) * sp + j0 + lane % 16] =
            acc[p][t][r];
    }
}

// G = the sum of the parts, in their order; the upper half by symmetry.
__global__ __launch_bounds__(256) void k_gram_sum(
    double* __restrict__ g, const double* __restrict__ part,
    const int* __restrict__ touched, int chunks, int sp) {
  const int64_t b = blockIdx.y;
  if (touched && !touched[b]) return;
  const int64_t size = (int64_t)sp * sp;
  int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= size) return;
  int i = e / sp, j = e % sp;
  if (i < j) return;
  const double* p = part + b * chunks * size + e;
  double sum = 0;
  for (int k = 0; k < chunks; ++k) sum += p[k * size];
  g[b * size + e] = sum;
  g[b * size + (int64_t)j * sp + i] = sum;
}

// X = U / n with n = |U|_F + eps as (u x) y: the power of two x keeps y and
// the products normal for values near the ends of f32's range.  NaN for a
// matrix that is not finite.
__device__ inline double2 norm_factors(double sumsq, double eps) {
  if (!(sumsq < INFINITY)) return make_double2(1.0, NAN);
  const double n = sqrt(sumsq) + eps;
  const double x = n > 0x1p60 ? 0x1p-60 : (n < 0x1p-60 ? 0x1p60 : 1.0);
  return make_double2(x, 1.0 / (n * x));
}

// |U|_F^2 is G's trace; G becomes X's.  One block a matrix.
__global__ __launch_bounds__(256) void k_gram_norm(
    double* __restrict__ g, double2* __restrict__ nu,
    const int* __restrict__ touched, int sp, double eps) {
  __shared__ double lds[256];
  const int64_t b = blockIdx.x;
  if (touched && !touched[b]) return;
  double* m = g + b * (int64_t)sp * sp;
  double t = 0;
  for (int i = threadIdx.x; i < sp; i += 256) t += m[(int64_t)i * sp + i];
  lds[threadIdx.x] = t;
  __syncthreads();
  for (int o = 128; o; o >>= 1) {
    if (threadIdx.x < o) lds[threadIdx.x] += lds[threadIdx.x + o];
    __syncthreads();
  }
  const double2 f = norm_factors(lds[0], eps);
  const double v = f.x * f.y;
  if (threadIdx.x == 0) nu[b] = f;
  for (int64_t e = threadIdx.x; e < (int64_t)sp * sp; e += 256) m[e] *= v * v;
}

// out = x y for commuting symmetric matrices (so out is symmetric): a wave a
// tile on or under the diagonal, mirrored.  q, if given, becomes
// a I + b x + c out (used with y = x).
__global__ __launch_bounds__(64) void k_small_mul(
    double* __restrict__ out, double* __restrict__ q,
    const double* __restrict__ x, const double* __restrict__ y,
    const int* __restrict__ touched, int s, int sp, Coeffs k) {
  const int64_t b = blockIdx.y;
  if (touched && !touched[b]) return;
  int ti = 0, tj = blockIdx.x;
  while (tj > ti) { tj -= ti + 1; ++ti; }
  const int64_t base = b * (int64_t)sp * sp;
  const int lane = threadIdx.x;
  const double* xr = x + base + (int64_t)(ti * 16 + lane % 16) * sp;
  const double* yr = y + base + (int64_t)(tj * 16 + lane % 16) * sp;
  f64x4 acc = (f64x4){0, 0, 0, 0};
  for (int kk = lane / 16; kk < sp; kk += 4)
    acc = __builtin_amdgcn_mfma_f64_16x16x4f64(xr[kk], yr[kk], acc, 0, 0, 0);
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    int i = ti * 16 + lane / 16 + 4 * r, j = tj * 16 + lane % 16;
    if (i < j) continue;  // a tile on the diagonal
    int64_t at = base + (int64_t)i * sp + j, ta = base + (int64_t)j * sp + i;
    if (q) {
      double v = k.b * x[at] + k.c * acc[r] + (i == j && i < s ? k.a : 0.0);
      q[at] = v;
      q[ta] = v;
    } else {
      out[at] = acc[r];
      out[ta] = acc[r];
    }
  }
}

// P with the norm's second factor, in f32
__global__ __launch_bounds__(256) void k_small_out(
    float* __restrict__ pf, const double* __restrict__ p,
    const double2* __restrict__ nu, const int* __restrict__ touched, int sp) {
  const int64_t b = blockIdx.y;
  if (touched && !touched[b]) return;
  int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e < (int64_t)sp * sp)
    pf[b * (int64_t)sp * sp + e] = (float)(p[b * (int64_t)sp * sp + e] *
                                           nu[b].y);
}

// O = U P (TALL) or P U: a wave 16 places of the long axis by 64 of the short
// one, f32 matrix instructions 16x16x4.
template <typename T, bool TALL>
__global__ __launch_bounds__(256) void k_thin_apply(
    Result res, const T* __restrict__ u, const float* __restrict__ pf,
    const double2* __restrict__ nu, const int* __restrict__ touched,
    int64_t long_, int s, int sp) {
  const int64_t b = blockIdx.z;
  if (touched && !touched[b]) return;
  const float pre = (float)nu[b].x;
  const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE;
  const int64_t r = ((int64_t)blockIdx.x * 4 + wave) * 16 + lane % 16;
  const int j0 = blockIdx.y * 64;
  const T* x = u + b * long_ * s;
  const float* p = pf + b * (int64_t)sp * sp;
  f32x4 acc[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) acc[t] = (f32x4){0, 0, 0, 0};
  for (int k = lane / 16; k < sp; k += 4) {
    float v = 0.0f;
    if (k < s && r < long_) v = to_f32(TALL ? x[r * s + k] : x[k * long_ + r]) * pre;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      int j = j0 + t * 16 + lane % 16;
      float w = j < sp ? p[(int64_t)k * sp + j] : 0.0f;
      // D[short][long]
      acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(w, v, acc[t], 0, 0, 0);
    }
  }
  if (r >= long_) return;
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      int j = j0 + t * 16 + (lane / 16) * 4 + i;
      if (j < s)
        finish<T>(res, b * long_ * s + (TALL ? r * s + j : j * long_ + r),
                  acc[t][i]);
    }
}

// ---------------------------------------------------------------------
// wide: planes of f16 hi + lo
// ---------------------------------------------------------------------

// A matrix in two planes: hi at p, lo at p + plane; rows `pitch` apart.
struct Planes {
  _Float16* p;
  int64_t plane, pitch, batch;  // batch: from one matrix to the next
};

__device__ inline void split(float v, _Float16& hi, _Float16& lo) {
  hi = (_Float16)v;
  lo = (_Float16)(v - (float)hi);
}

template <typename T>
__global__ __launch_bounds__(256) void k_sumsq(
    double* __restrict__ part, const T* __restrict__ u,
    const int* __restrict__ touched, int64_t size) {
  __shared__ double lds[256];
  const int64_t b = blockIdx.y;
  if (touched && !touched[b]) return;
  double t = 0;
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < size;
       e += (int64_t)gridDim.x * 256) {
    double v = to_f32(u[b * size + e]);
    t += v * v;
  }
  lds[threadIdx.x] = t;
  __syncthreads();
  for (int o = 128; o; o >>= 1) {
    if (threadIdx.x < o) lds[threadIdx.x] += lds[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) part[b * gridDim.x + blockIdx.x] = lds[0];
}

__global__ __launch_bounds__(256) void k_norm(
    float2* __restrict__ scale, const double* __restrict__ part, int parts,
    int64_t batch, double eps) {
  int64_t b = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (b >= batch) return;
  double t = 0;
  for (int k = 0; k < parts; ++k) t += part[b * parts + k];
  const double2 f = norm_factors(t, eps);
  scale[b] = make_float2((float)f.x, (float)f.y);
}

// The planes of X as it lies in memory (m x n) and transposed, 64 x 64 values
// a block, zeros around them.
template <typename T>
__global__ __launch_bounds__(256) void k_planes(
    Planes nat, Planes trn, const T* __restrict__ u,
    const float2* __restrict__ scale, const int* __restrict__ touched,
    int64_t m, int64_t n) {
  __shared__ float lds[64][65];
  const int64_t b = blockIdx.z;
  if (touched && !touched[b]) return;
  const float2 sc = scale[b];
  const int64_t wide = nat.pitch / 64;
  const int64_t r0 = blockIdx.x / wide * 64, c0 = blockIdx.x % wide * 64;
  for (int e = threadIdx.x; e < 64 * 64; e += 256) {
    int r = e / 64, c = e % 64;
    float v = 0.0f;
    if (r0 + r < m && c0 + c < n)
      v = to_f32(u[(b * m + r0 + r) * n + c0 + c]) * sc.x * sc.y * UP;
    lds[r][c] = v;
    _Float16* to = nat.p + b * nat.batch + (r0 + r) * nat.pitch + c0 + c;
    split(v, to[0], to[nat.plane]);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < 64 * 64; e += 256) {
    int c = e / 64, r = e % 64;
    _Float16* to = trn.p + b * trn.batch + (c0 + c) * trn.pitch + r0 + r;
    split(lds[r][c], to[0], to[trn.plane]);
  }
}

enum Ending { GRAM, POLY, UPDATE, FINAL };

struct Product {
  Planes a, b;       // rows of K values each: D[i][j] = sum_k a[i][k] b[j][k]
  int k;             // a multiple of 32
  Planes d, dt;      // D and D transposed (GRAM, POLY: d alone, symmetric)
  float ca, cb, cc;  // POLY: a I + b a + c D
  int s;             // POLY: I ends here
  int64_t rows, cols;  // FINAL: D's own size
  bool tall;           // FINAL: D transposed is what lies in memory
  Result res;
};

// One block an NT x NT tile of D, four waves a quarter each, 32 places of K
// at a time through LDS.  LDS rows are four 16-byte pieces; piece c of row r
// lies at c ^ (r / 2 % 4), so that eight lanes that read one piece of eight
// rows hit different banks.
template <int NT, Ending E, typename T>
__global__ __launch_bounds__(256) void k_product(
    Product pr, const int* __restrict__ touched) {
  constexpr int W = NT / 32;               // 16-tiles a wave on each side
  constexpr int LOADS = NT * 4 / 256;      // 16-byte pieces a thread and plane
  __shared__ half8 lds[2][2][NT * 4];      // operand, plane
  const int64_t b = blockIdx.z;
  if (touched && !touched[b]) return;
  int bi = blockIdx.y, bj = blockIdx.x;
  if (E == GRAM || E == POLY) {
    bi = 0;
    while (bj > bi) { bj -= bi + 1; ++bi; }
  }
  const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE;
  const int wi = wave / 2 * (NT / 2), wj = wave % 2 * (NT / 2);

  const _Float16* src[2] = {
      pr.a.p + b * pr.a.batch + (int64_t)bi * NT * pr.a.pitch,
      pr.b.p + b * pr.b.batch + (int64_t)bj * NT * pr.b.pitch};
  const int64_t pitch[2] = {pr.a.pitch, pr.b.pitch};
  const int64_t plane[2] = {pr.a.plane, pr.b.plane};

  half8 next[2][2][LOADS];
  auto fetch = [&](int k) {
#pragma unroll
    for (int o = 0; o < 2; ++o)
#pragma unroll
      for (int l = 0; l < LOADS; ++l) {
        int e = threadIdx.x + l * 256, r = e / 4, c = e % 4;
        const _Float16* at = src[o] + r * pitch[o] + k + c * 8;
        next[o][0][l] = *(const half8*)at;
        next[o][1][l] = *(const half8*)(at + plane[o]);
      }
  };

  f32x4 acc[W][W];
#pragma unroll
  for (int i = 0; i < W; ++i)
#pragma unroll
    for (int j = 0; j < W; ++j) acc[i][j] = (f32x4){0, 0, 0, 0};

  fetch(0);
  for (int k = 0; k < pr.k; k += 32) {
    __syncthreads();
#pragma unroll
    for (int o = 0; o < 2; ++o)
#pragma unroll
      for (int l = 0; l < LOADS; ++l) {
        int e = threadIdx.x + l * 256, r = e / 4, c = e % 4;
        lds[o][0][r * 4 + (c ^ (r / 2 % 4))] = next[o][0][l];
        lds[o][1][r * 4 + (c ^ (r / 2 % 4))] = next[o][1][l];
      }
    __syncthreads();
    if (k + 32 < pr.k) fetch(k + 32);
    half8 av[W][2], bv[W][2];
#pragma unroll
    for (int t = 0; t < W; ++t)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        int ra = wi + t * 16 + lane % 16, rb = wj + t * 16 + lane % 16;
        av[t][h] = lds[0][h][ra * 4 + (lane / 16 ^ (ra / 2 % 4))];
        bv[t][h] = lds[1][h][rb * 4 + (lane / 16 ^ (rb / 2 % 4))];
      }
#pragma unroll
    for (int i = 0; i < W; ++i)
#pragma unroll
      for (int j = 0; j < W; ++j) {
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
            av[i][0], bv[j][1], acc[i][j], 0, 0, 0);
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
            av[i][1], bv[j][0], acc[i][j], 0, 0, 0);
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
            av[i][0], bv[j][0], acc[i][j], 0, 0, 0);
      }
  }

  // a lane holds D[i .. i + 3][j] of each tile
#pragma unroll
  for (int ti = 0; ti < W; ++ti)
#pragma unroll
    for (int tj = 0; tj < W; ++tj) {
      const int64_t i = (int64_t)bi * NT + wi + ti * 16 + lane / 16 * 4;
      const int64_t j = (int64_t)bj * NT + wj + tj * 16 + lane % 16;
      if (E == FINAL) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (i + r < pr.rows && j < pr.cols)
            finish<T>(pr.res,
                      b * pr.rows * pr.cols +
                          (pr.tall ? j * pr.rows + i + r
                                   : (i + r) * pr.cols + j),
                      acc[ti][tj][r] * (1.0f / (UP * UP)));
        continue;
      }
      half4 hi, lo;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float v = acc[ti][tj][r] * (1.0f / UP);
        if (E == POLY) {
          const _Float16* g = pr.a.p + b * pr.a.batch +
                              (i + r) * pr.a.pitch + j;
          v = pr.cc * v + pr.cb * ((float)g[0] + (float)g[pr.a.plane]);
          if (i + r == j && j < pr.s) v += pr.ca * UP;
        }
        _Float16 h, l;
        split(v, h, l);
        hi[r] = h;
        lo[r] = l;
        _Float16* to = pr.d.p + b * pr.d.batch + (i + r) * pr.d.pitch + j;
        to[0] = h;
        to[pr.d.plane] = l;
      }
      if (E == UPDATE || bi != bj) {
        const Planes& t = E == UPDATE ? pr.dt : pr.d;
        _Float16* to = t.p + b * t.batch + j * t.pitch + i;
        *(half4*)to = hi;
        *(half4*)(to + t.plane) = lo;
      }
    }
}

// ---------------------------------------------------------------------
// host
// ---------------------------------------------------------------------

struct Chain {
  const void* u;
  at::ScalarType type;
  int64_t batch, m, n;
  const int* touched;
  int steps;
  Coeffs k;
  double eps;
  Result res;
  at::TensorOptions options;
  hipStream_t stream;
};

int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

template <typename T, bool TALL>
void run_thin(const Chain& c) {
  const int s = std::min(c.m, c.n);
  const int64_t long_ = std::max(c.m, c.n);
  const int sp = round_up(s, 16), nt = sp / 16;
  const int super = (s + SUPER - 1) / SUPER, pairs = super * (super + 1) / 2;
  // chunks of 256 places at least, about two blocks a CU
  int64_t chunks = std::min<int64_t>((long_ + 255) / 256,
                                     std::max<int64_t>(1, 512 / (c.batch *
                                                                 pairs)));
  const int64_t chunk = round_up((long_ + chunks - 1) / chunks, KC);
  chunks = (long_ + chunk - 1) / chunk;
  const int64_t size = (int64_t)sp * sp;
  auto f64 = c.options.dtype(at::kDouble);
  auto part = at::empty({c.batch * chunks * size}, f64);
  auto work = at::empty({6, c.batch * size}, f64);
  auto nu = at::empty({2 * c.batch}, f64);
  double2* nus = (double2*)nu.data_ptr<double>();
  auto pf = at::empty({c.batch * size}, c.options.dtype(at::kFloat));
  double* w[6];
  for (int i = 0; i < 6; ++i) w[i] = work.data_ptr<double>() + i * c.batch * size;
  hipLaunchKernelGGL((k_gram64<T, TALL>), dim3(chunks, pairs, c.batch),
                     dim3(256), 0, c.stream, part.data_ptr<double>(),
                     (const T*)c.u, c.touched, long_, s, sp, chunk);
  const dim3 all((size + 255) / 256, c.batch);
  double *g = w[0], *q = w[1], *p = w[2], *t = w[3], *g2 = w[4], *p2 = w[5];
  hipLaunchKernelGGL(k_gram_sum, all, dim3(256), 0, c.stream, g,
                     part.data_ptr<double>(), c.touched, (int)chunks, sp);
  hipLaunchKernelGGL(k_gram_norm, dim3(c.batch), dim3(256), 0, c.stream, g,
                     nus, c.touched, sp, c.eps);
  const dim3 tiles(nt * (nt + 1) / 2, c.batch);
  auto mul = [&](double* out, double* poly, const double* x, const double* y) {
    hipLaunchKernelGGL(k_small_mul, tiles, dim3(64), 0, c.stream, out, poly, x,
                       y, c.touched, s, sp, c.k);
  };
  for (int i = 0; i < c.steps; ++i) {
    // Q from G; P <- P Q (the first P is Q); G <- Q (G Q)
    double* qi = i == 0 ? p : q;
    mul(nullptr, qi, g, g);
    if (i > 0) { mul(p2, nullptr, p, q); std::swap(p, p2); }
    if (i + 1 < c.steps) {
      mul(t, nullptr, g, qi);
      mul(g2, nullptr, qi, t);
      std::swap(g, g2);
    }
  }
  hipLaunchKernelGGL(k_small_out, all, dim3(256), 0, c.stream,
                     pf.data_ptr<float>(), p, nus, c.touched, sp);
  hipLaunchKernelGGL((k_thin_apply<T, TALL>),
                     dim3((long_ + 63) / 64, (s + 63) / 64, c.batch),
                     dim3(256), 0, c.stream, c.res, (const T*)c.u,
                     pf.data_ptr<float>(), nus, c.touched, long_, s, sp);
}

template <int NT, typename T>
void run_products(const Chain& c, Planes x, Planes xt, Planes xt2, Planes g,
                  Planes q) {
  const int64_t s = std::min(c.m, c.n), long_ = std::max(c.m, c.n);
  const int ns = (s + NT - 1) / NT, nl = (long_ + NT - 1) / NT;
  const dim3 half(ns * (ns + 1) / 2, 1, c.batch), full(nl, ns, c.batch);
  Product pr{};
  pr.ca = (float)c.k.a;
  pr.cb = (float)c.k.b;
  pr.cc = (float)c.k.c;
  pr.s = s;
  pr.rows = s;
  pr.cols = long_;
  pr.tall = c.m > c.n;
  pr.res = c.res;
  const int ks = round_up(s, 32), kl = round_up(long_, 32);
  for (int i = 0; i < c.steps; ++i) {
    pr.a = pr.b = x;
    pr.k = kl;
    pr.d = g;
    hipLaunchKernelGGL((k_product<NT, GRAM, T>), half, dim3(256), 0, c.stream,
                       pr, c.touched);
    pr.a = pr.b = g;
    pr.k = ks;
    pr.d = q;
    hipLaunchKernelGGL((k_product<NT, POLY, T>), half, dim3(256), 0, c.stream,
                       pr, c.touched);
    pr.a = q;
    pr.b = xt;
    pr.d = x;
    pr.dt = xt2;
    if (i + 1 < c.steps)
      hipLaunchKernelGGL((k_product<NT, UPDATE, T>), full, dim3(256), 0,
                         c.stream, pr, c.touched);
    else
      hipLaunchKernelGGL((k_product<NT, FINAL, T>), full, dim3(256), 0,
                         c.stream, pr, c.touched);
    std::swap(xt, xt2);
  }
}

template <typename T>
void run_wide(const Chain& c) {
  const int64_t mp = round_up(c.m, PAD), np = round_up(c.n, PAD);
  const int64_t s = std::min(c.m, c.n), sp = round_up(s, PAD);
  const bool tall = c.m > c.n;
  auto f16 = c.options.dtype(at::kHalf);
  std::vector<at::Tensor> keep;
  auto planes = [&](int64_t rows, int64_t cols) {
    keep.push_back(at::empty({2 * c.batch * rows * cols}, f16));
    return Planes{(_Float16*)keep.back().data_ptr(), c.batch * rows * cols,
                  cols, rows * cols};
  };
  Planes nat = planes(mp, np), trn = planes(np, mp);
  Planes x = tall ? trn : nat, xt = tall ? nat : trn;
  Planes xt2 = tall ? planes(mp, np) : planes(np, mp);
  Planes g = planes(sp, sp), q = planes(sp, sp);
  const int parts = (int)std::min<int64_t>(
      256, (c.m * c.n + 4095) / 4096);
  auto part = at::empty({c.batch * parts}, c.options.dtype(at::kDouble));
  auto scale = at::empty({2 * c.batch}, c.options.dtype(at::kFloat));
  hipLaunchKernelGGL(k_sumsq<T>, dim3(parts, c.batch), dim3(256), 0, c.stream,
                     part.data_ptr<double>(), (const T*)c.u, c.touched,
                     c.m * c.n);
  hipLaunchKernelGGL(k_norm, dim3((c.batch + 255) / 256), dim3(256), 0,
                     c.stream, (float2*)scale.data_ptr<float>(),
                     part.data_ptr<double>(), parts, c.batch, c.eps);
  hipLaunchKernelGGL(k_planes<T>, dim3(np / 64 * (mp / 64), 1, c.batch),
                     dim3(256), 0, c.stream, nat, trn, (const T*)c.u,
                     (const float2*)scale.data_ptr<float>(), c.touched, c.m,
                     c.n);
  run_products<64, T>(c, x, xt, xt2, g, q);
}

template <typename T>
void run(const Chain& c) {
  const int64_t s = std::min(c.m, c.n), long_ = std::max(c.m, c.n);
  if (s <= 64 || (s <= THIN_MAX && long_ >= 32 * s)) {
    if (c.m >= c.n) run_thin<T, true>(c); else run_thin<T, false>(c);
  } else {
    run_wide<T>(c);
  }
}

void dispatch(const Chain& whole) {
  // grids hold 65535 matrices
  for (int64_t b = 0; b < whole.batch; b += 32768) {
    Chain c = whole;
    const int64_t size = c.m * c.n * b;
    c.batch = std::min<int64_t>(32768, whole.batch - b);
    c.u = (const char*)c.u + size * c10::elementSize(c.type);
    c.res.out = (char*)c.res.out +
                size * (c.res.step ? 4 : c10::elementSize(c.type));
    if (c.touched) c.touched += b;
    if (c.type == at::kFloat) run<float>(c);
    else if (c.type == at::kHalf) run<__half>(c);
    else run<__hip_bfloat16>(c);
  }
}

void check_chain(int64_t m, int64_t n, int64_t steps) {
  TORCH_CHECK(steps >= 1 && steps <= 100, "steps must be 1 to 100");
  TORCH_CHECK(m < (int64_t{1} << 31) - 256 && n < (int64_t{1} << 31) - 256 &&
                  std::min(m, n) <= 65536,
              "matrices of ", m, " x ", n, " are too large");
}

}  // namespace

at::Tensor orthogonalize(at::Tensor x, int64_t steps, double a, double b,
                         double c, double eps) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 3 && x.is_contiguous(),
              "x must be a contiguous 3-D device tensor");
  const auto type = x.scalar_type();
  TORCH_CHECK(type == at::kFloat || type == at::kHalf || type == at::kBFloat16,
              "x must be float32, bfloat16 or float16");
  check_chain(x.size(1), x.size(2), steps);
  c10::DeviceGuard guard(x.device());
  auto out = at::empty_like(x);
  if (!x.numel()) return out;
  dispatch(Chain{x.data_ptr(), type, x.size(0), x.size(1), x.size(2), nullptr,
                 (int)steps, {a, b, c}, eps, {out.data_ptr(), 0, 0, false},
                 x.options(), at::hip::getCurrentHIPStream().stream()});
  return out;
}

void apply_muon(at::Tensor table, at::Tensor momentum, at::Tensor rows,
                c10::optional<at::Tensor> order, at::Tensor grads, double lr,
                double mu, bool nesterov, double weight_decay, int64_t steps,
                int64_t matrix_rows, double a, double b, double c,
                double eps) {
  for (const auto& t : {table, momentum, rows, grads})
    TORCH_CHECK(t.is_cuda() && t.is_contiguous() &&
                    t.device() == table.device(),
                "operands must be contiguous on the table's device");
  TORCH_CHECK(table.dim() == 2 && table.scalar_type() == at::kFloat &&
                  momentum.sizes() == table.sizes() &&
                  momentum.scalar_type() == at::kFloat,
              "table and momentum must be float32 of one 2-D shape");
  const int64_t n = rows.numel(), dim = table.size(1);
  TORCH_CHECK(rows.scalar_type() == at::kLong &&
                  grads.scalar_type() == at::kFloat && grads.dim() == 2 &&
                  grads.size(0) == n && grads.size(1) == dim,
              "grads must be float32, one row for each int64 of rows");
  TORCH_CHECK(!order || (order->scalar_type() == at::kLong &&
                         order->numel() == n && order->is_contiguous() &&
                         order->device() == table.device()),
              "order must be int64, one for each row");
  TORCH_CHECK(matrix_rows >= 1 && table.size(0) % matrix_rows == 0,
              "the table is not a whole number of matrices of ", matrix_rows,
              " rows");
  check_chain(matrix_rows, dim, steps);
  const int64_t batch = table.size(0) / matrix_rows;
  if (!n || !table.numel()) return;
  c10::DeviceGuard guard(table.device());
  hipStream_t stream = at::hip::getCurrentHIPStream().stream();
  auto touched = at::empty({batch}, table.options().dtype(at::kInt));
  hipLaunchKernelGGL(k_touched, dim3((batch + 255) / 256), dim3(256), 0,
                     stream, touched.data_ptr<int>(),
                     rows.data_ptr<int64_t>(), n, batch, matrix_rows);
  auto u = at::empty_like(table);
  const int64_t total = table.size(0);
  hipLaunchKernelGGL(k_momentum,
                     dim3(std::min<int64_t>((total + 3) / 4, 4096)), dim3(256),
                     0, stream, u.data_ptr<float>(),
                     momentum.data_ptr<float>(), grads.data_ptr<float>(),
                     rows.data_ptr<int64_t>(),
                     order ? order->data_ptr<int64_t>() : nullptr,
                     touched.data_ptr<int>(), n, total, matrix_rows, dim,
                     (float)mu, nesterov);
  const double rate = lr * std::sqrt(std::max(1.0, (double)matrix_rows / dim));
  dispatch(Chain{u.data_ptr(), at::kFloat, batch, matrix_rows, dim,
                 touched.data_ptr<int>(), (int)steps, {a, b, c}, eps,
                 {table.data_ptr(), (float)(1.0 - lr * weight_decay),
                  (float)rate, true},
                 table.options(), stream});
}
