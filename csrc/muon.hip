// Newton-Schulz orthogonalisation and the Muon server step for MI355X
// (gfx950).
//
// For a matrix U of m x n values, with s = min(m, n) and L = max(m, n):
//     X = U / (|U|_F + eps),  then `steps` times
//     G = X X^T (on the side of length s),  X <- (a I + b G + c G^2) X.
//
// Two ways to the same result.  Both hold the operands of their large products
// in two f16 planes, hi + lo, and add in f32: 22 to 24 bits of a value and down
// to 2^-37 of its matrix's norm, and the product of two lows is left out.  That
// is three f16 products in place of one f32 product, which costs 16 / 3 as much
// at this card's matrix rates.  Off the chain in 64 bits by 1e-7 to 4e-6 of the
// result's norm where singular values are alike (steps in f32: 2e-6 to 4e-6).
// What lies along a singular value near zero is multiplied by a^steps = 485,
// roundings too: where all but a few are zero the result is up to 4e-4 off (as
// steps in f32 are, though not for the same matrices: a 300 x 900 matrix of
// equal values is 3.5e-4 off on the thin route, 1e-5 in f32; random ones of
// rank 1 are 1e-4 to 2e-4 off on the wide route, 2e-4 to 4e-4 in f32).
//
// thin   G is taken once, in f64 over the long axis; the steps are then taken
//        on s x s matrices alone (each multiplies X by Q = a I + b G + c G^2
//        and G by Q^2), and one product applies P = Q_1 ... Q_k to U.  Two
//        passes over the values instead of two a step.  G has to be f64: an
//        error in it grows by a^2 = 12 with every step.
// wide   the chain as written, with every operand in planes:
//        a b = hi hi + hi lo + lo hi on the f16 matrix units.

#include <ATen/ATen.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <tuple>
#include <type_traits>
#include <vector>

#include "ops.h"
#include "quads.h"

namespace {

constexpr int WAVE = 64;
constexpr int PAD = 128;      // rows and columns of the wide planes
constexpr float UP = 4096.0f; // planes hold 2^12 times the value

using half4 = __attribute__((ext_vector_type(4))) _Float16;
using half8 = __attribute__((ext_vector_type(8))) _Float16;
using f32x4 = __attribute__((ext_vector_type(4))) float;
using f64x4 = __attribute__((ext_vector_type(4))) double;

struct Coeffs { double a, b, c; };

template <typename I>
__host__ __device__ inline I round_up(I v, int to) {
  return (v + to - 1) / to * to;
}

// What a product ends in: the values of `out` (T), or the weights' step
// W <- W keep - rate O.
struct Result {
  void* out;      // orthogonalize: T; Muon: the f32 table
  float keep, rate;
  bool step;
};

// The wave's number in a scalar register: branches on it cost nothing.
__device__ inline int this_wave() {
  return __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
}

template <typename T>
__device__ inline void finish(const Result& r, int64_t at, float o) {
  if (r.step) {
    float* w = (float*)r.out + at;
    *w = *w * r.keep - r.rate * o;
  } else {
    ((T*)r.out)[at] = from_f32<T>(o);
  }
}

// The same for four neighbours, `held` of them (any number).
template <typename T>
__device__ inline void finish_quad(const Result& r, int64_t at, float4 o,
                                   int64_t held) {
  if (r.step) {
    float* w = (float*)r.out + at;
    float4 v = load_quad(w, held);
    v.x = v.x * r.keep - r.rate * o.x;
    v.y = v.y * r.keep - r.rate * o.y;
    v.z = v.z * r.keep - r.rate * o.z;
    v.w = v.w * r.keep - r.rate * o.w;
    store_quad(w, v, held);
  } else {
    store_quad((T*)r.out + at, o, held);
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

struct Momentum {
  float* u;
  float* m;
  const float* grads;
  const int64_t* rows;   // sorted
  const int64_t* order;  // place of the j-th in grads, or null: j
  const float* sums;     // place n is the first of k_long_runs' sums
  int64_t n;
  float mu;
  bool nesterov;
};

// Where a row's gradient is: its place in grads (>= 0), nowhere (-1), or, for
// several, -2 - j with j the first of them in the sorted push.  Said before
// the values are wanted, so that no load of those waits for a comparison.
__device__ inline int64_t several(int64_t j) { return -2 - j; }

// The sum of a row's gradients (at columns c .. c + 3) in the order of the
// push.
__device__ inline float4 row_gradient(const Momentum& q, int64_t place,
                                      int64_t row, int dim, int c, int held) {
  const float* from = place < q.n ? q.grads : q.sums;
  float4 g = load_quad(from + place * dim + c, place >= 0 ? held : 0);
  if (place < -1)
    for (int64_t j = several(place); j < q.n && q.rows[j] == row; ++j) {
      const float4 h = load_quad(
          q.grads + (q.order ? q.order[j] : j) * dim + c, held);
      g.x += h.x;
      g.y += h.y;
      g.z += h.z;
      g.w += h.w;
    }
  return g;
}

// M's new value from its old one; u gets U's.
__device__ inline float4 next_momentum(const Momentum& q, float4 v, float4 g,
                                       float4* u) {
  v.x = q.mu * v.x + g.x;
  v.y = q.mu * v.y + g.y;
  v.z = q.mu * v.z + g.z;
  v.w = q.mu * v.w + g.w;
  *u = q.nesterov ? make_float4(g.x + q.mu * v.x, g.y + q.mu * v.y,
                                g.z + q.mu * v.z, g.w + q.mu * v.w)
                  : v;
  return v;
}

// place[r] (see several()) for up to 256 rows of one matrix at a time, of a
// sorted push; touched[b] = whether the push names a row of matrix b.
__global__ __launch_bounds__(256) void k_places(
    int64_t* __restrict__ place, int* __restrict__ touched,
    const int64_t* __restrict__ rows, const int64_t* __restrict__ order,
    int64_t n, int64_t m, int64_t windows) {
  __shared__ int64_t mine[256];
  __shared__ int64_t ends[2];
  const int64_t chunks = (m + 255) / 256;
  for (int64_t w = blockIdx.x; w < windows; w += gridDim.x) {
    const int64_t b = w / chunks, chunk = w % chunks;
    const int64_t r0 = b * m + chunk * 256;
    const int64_t count = min(m - chunk * 256, (int64_t)256);
    mine[threadIdx.x] = -1;
    if (threadIdx.x % WAVE == 0 && threadIdx.x < 2 * WAVE) {
      // a push of every row has row r at place r
      const int64_t x = threadIdx.x == 0 ? r0 : r0 + count;
      const bool direct = x < n && rows[x] == x && (x == 0 || rows[x - 1] < x);
      ends[threadIdx.x / WAVE] = direct ? x : lower_bound(rows, n, x);
    }
    __syncthreads();
    const int64_t lo = ends[0], hi = ends[1];
    if (chunk == 0 && threadIdx.x == 0) {
      bool some = hi > lo;
      if (!some) {
        const int64_t at = lower_bound(rows, n, b * m);
        some = at < n && rows[at] < (b + 1) * m;
      }
      touched[b] = some;
    }
    for (int64_t j = lo + threadIdx.x; j < hi; j += 256) {
      const int64_t at = rows[j] - r0;  // within, unless rows are not sorted
      if (at >= 0 && at < count && (j == lo || rows[j - 1] != rows[j]))
        mine[at] = j + 1 < hi && rows[j + 1] == rows[j]
                       ? several(j)
                       : (order ? order[j] : j);
    }
    __syncthreads();
    if (threadIdx.x < count) place[r0 + threadIdx.x] = mine[threadIdx.x];
    __syncthreads();
  }
}

// The same of a push in any order, of up to SHORT places, with the rows and
// their places in `sorted` and `order`.  A block reads the whole push and keeps
// what names its 256 rows, each wave a quarter of the push, so that equal rows
// stay in the order that they came in.  Rows outside the table are in nobody's
// window; the sorted rows end with -1 then.
constexpr int SHORT = 16384;

__global__ __launch_bounds__(256) void k_places_any(
    int64_t* __restrict__ place, int* __restrict__ touched,
    int64_t* __restrict__ sorted, int64_t* __restrict__ order,
    const int64_t* __restrict__ rows, int n, int64_t m, int64_t total) {
  __shared__ uint32_t list[SHORT + 3];  // row in the window, place in the push
  __shared__ int next[4][256];          // a row's: how many, then where to
  __shared__ int only[256], ends[4][2], sums[4];
  const int64_t chunks = (m + 255) / 256;
  const int64_t b = blockIdx.x / chunks, chunk = blockIdx.x % chunks;
  const int64_t r0 = b * m + chunk * 256;
  const int count = min(m - chunk * 256, (int64_t)256);
  const int lane = threadIdx.x % WAVE, wave = this_wave(), t = threadIdx.x;
  const uint64_t under = (1ull << lane) - 1;
  const int share = (n + 3) / 4, from = min(wave * share, n);
  const int to = min(from + share, n);
  uint32_t* mine = list + wave * share;
  int held = 0, before = 0, here = 0;
  for (int w = 0; w < 4; ++w) next[w][t] = 0;
  __syncthreads();
  for (int j0 = from; j0 < to; j0 += 4 * WAVE) {
    int64_t r[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int j = j0 + q * WAVE + lane;
      r[q] = j < to ? rows[j] : -1;
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int64_t at = r[q] - r0;
      const bool in = at >= 0 && at < count;
      const uint64_t votes = __ballot(in);
      before += __popcll(__ballot(r[q] >= 0 && r[q] < r0));
      here |= __ballot(r[q] >= b * m && r[q] < (b + 1) * m) != 0;
      if (in) {
        atomicAdd(&next[wave][at], 1);
        mine[held + __popcll(votes & under)] =
            (uint32_t)at << 16 | (j0 + q * WAVE + lane);
      }
      held += __popcll(votes);
    }
  }
  if (lane == 0) {
    ends[wave][0] = before;
    ends[wave][1] = here;
  }
  __syncthreads();
  // where row t's run begins among the sorted ones, and each wave's share of it
  int named = 0;
  for (int w = 0; w < 4; ++w) named += next[w][t];
  int run = named;
#pragma unroll
  for (int o = 1; o < WAVE; o *= 2) {
    const int left = __shfl_up(run, o);
    if (lane >= o) run += left;
  }
  if (lane == WAVE - 1) sums[wave] = run;
  __syncthreads();
  for (int w = 0; w < 4; ++w) run += ends[w][0] + (w < wave ? sums[w] : 0);
  const int first = run - named;
  for (int w = 0, at = first; w < 4; ++w) {
    const int more = next[w][t];
    next[w][t] = at;
    at += more;
  }
  __syncthreads();
  // 64 of a wave's at a time: a row's place moves on by those that name it
  for (int e = 0; e < held; e += WAVE) {
    const bool some = e + lane < held;
    const uint32_t v = some ? mine[e + lane] : 0;
    const int r = v >> 16, j = v & 0xffff;
    uint64_t same = __ballot(some);
#pragma unroll
    for (int bit = 0; bit < 8; ++bit) {
      const uint64_t set = __ballot(r >> bit & 1);
      same &= r >> bit & 1 ? set : ~set;
    }
    const int at = next[wave][r];
    __builtin_amdgcn_wave_barrier();
    if (some) {
      const int mine_at = at + __popcll(same & under);
      sorted[mine_at] = r0 + r;
      order[mine_at] = j;
      only[r] = j;
      if (!(same >> lane >> 1)) next[wave][r] = mine_at + 1;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
  if (t < count)
    place[r0 + t] = named > 1 ? several(first) : named ? only[t] : -1;
  if (r0 + count == total) {  // the last window: no row from here on
    if (t == 255) sums[0] = run;
    __syncthreads();
    for (int j = sums[0] + t; j < n; j += 256) sorted[j] = -1;
  }
  if (t == 0 && chunk == 0)
    touched[b] = ends[0][1] | ends[1][1] | ends[2][1] | ends[3][1];
}

// Rows that a push names more than LONG times (a frequent word of a batch):
// sums[x] is the sum of the one whose run begins in the x-th LONG places of the
// sorted push, in the push's order, and the row's place is n + x.  A block
// takes WIDTH columns: all its threads load, 128 gradients at a time, and a
// thread a column adds.  Bound by those additions and the latency of a turn's
// loads: 16 to 30 ns a gradient, where row_gradient, whose loads wait for each
// other, takes 0.3 to 0.9 us (3952 x 32, 16,000 gradients, half of them of one
// row: 222 us a step, 2468 without; 2048 x 512, 100,000: 1755, 43483).  A push
// without such rows pays the launch, 2 us.
constexpr int LONG = 64;

template <int WIDTH>
__global__ __launch_bounds__(256) void k_long_runs(
    float* __restrict__ sums, int64_t* __restrict__ place, Momentum q,
    int64_t total, int64_t dim) {
  constexpr int TURN = 128, EACH = TURN * WIDTH / 256;
  __shared__ float tile[TURN * WIDTH];
  __shared__ int64_t from[2][TURN];  // places in grads
  __shared__ int counts[2][TURN / WAVE];
  __shared__ int64_t first;
  const int t = threadIdx.x;
  for (int64_t x = blockIdx.x; x * LONG < q.n; x += gridDim.x) {
    __syncthreads();  // of the run before
    if (t < LONG) {  // one wave; runs this long begin once in LONG places
      const int64_t j = x * LONG + t;
      bool begins = false;
      if (j + LONG < q.n) {
        const int64_t r = q.rows[j];
        begins = r >= 0 && r < total && q.rows[j + LONG] == r &&
                 (j == 0 || q.rows[j - 1] != r);
      }
      const uint64_t votes = __ballot(begins);
      if (t == 0) first = votes ? j + __builtin_ctzll(votes) : -1;
    }
    __syncthreads();
    if (first < 0) continue;
    const int64_t row = q.rows[first];
    auto look = [&](int64_t j, int buffer) {
      if (t >= TURN) return;
      const bool same = j + t < q.n && q.rows[j + t] == row;
      from[buffer][t] = !same ? -1 : q.order ? q.order[j + t] : j + t;
      const uint64_t votes = __ballot(same);
      if (t % WAVE == 0) counts[buffer][t / WAVE] = __popcll(votes);
    };
    for (int64_t c0 = (int64_t)blockIdx.y * WIDTH; c0 < dim;
         c0 += (int64_t)gridDim.y * WIDTH) {
      float v[EACH], sum = 0.0f;
      auto fetch = [&](int buffer) {
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
          const int64_t g = from[buffer][(t + e * 256) / WIDTH];
          const int64_t c = c0 + t % WIDTH;
          v[e] = g >= 0 && c < dim ? q.grads[g * dim + c] : 0.0f;
        }
      };
      __syncthreads();  // of the columns before
      look(first, 0);
      look(first + TURN, 1);
      __syncthreads();
      fetch(0);
      int64_t j = first;
      for (int buffer = 0;; buffer ^= 1) {
#pragma unroll
        for (int e = 0; e < EACH; ++e) tile[t + e * 256] = v[e];
        const int count = counts[buffer][0] + counts[buffer][1];
        const bool more = counts[buffer ^ 1][0] != 0;
        __syncthreads();
        if (more) {
          fetch(buffer ^ 1);
          look(j + 2 * TURN, buffer);
        }
        if (t < WIDTH) {
#pragma unroll 16
          for (int k = 0; k < count; ++k) sum += tile[k * WIDTH + t];
        }
        __syncthreads();
        if (!more) break;
        j += TURN;
      }
      if (t < WIDTH && c0 + t < dim) sums[x * dim + c0 + t] = sum;
    }
    if (blockIdx.y == 0 && t == 0) place[row] = q.n + x;
  }
}

// active[0] = how many of up to 32768 matrices are touched, then which.
__global__ __launch_bounds__(1024) void k_active(
    int* __restrict__ active, const int* __restrict__ touched, int batch) {
  __shared__ int counts[16];
  int before = 0;
  for (int b0 = 0; b0 < batch; b0 += 1024) {
    const int b = b0 + threadIdx.x;
    const bool mine = b < batch && touched[b];
    const uint64_t votes = __ballot(mine);
    const int wave = threadIdx.x / WAVE, lane = threadIdx.x % WAVE;
    if (lane == 0) counts[wave] = __popcll(votes);
    __syncthreads();
    int at = before;
    for (int w = 0; w < 16; ++w) {
      if (w < wave) at += counts[w];
      before += counts[w];
    }
    if (mine) active[1 + at + __popcll(votes & ((1ull << lane) - 1))] = b;
    __syncthreads();
  }
  if (threadIdx.x == 0) active[0] = before;
}

// M <- mu M + g and U = g + mu M (nesterov) or M, `group` lanes a row.  Bound
// by memory: 16 bytes a value.
__global__ __launch_bounds__(256) void k_momentum(
    Momentum q, const int64_t* __restrict__ place,
    const int* __restrict__ touched, int64_t total, int64_t m, int dim,
    int group) {
  const int lane = threadIdx.x & (group - 1);
  for (int64_t row = ((int64_t)blockIdx.x * 256 + threadIdx.x) / group;
       row < total; row += (int64_t)gridDim.x * (256 / group)) {
    if (!touched[row / m]) continue;
    const int64_t j = place[row];
    for (int c = lane * 4; c < dim; c += group * 4) {
      const int64_t at = row * dim + c;
      const int held = dim - c;
      float4 v = load_quad(q.m + at, held), u;
      v = next_momentum(q, v, row_gradient(q, j, row, dim, c, held), &u);
      store_quad(q.m + at, v, held);
      store_quad(q.u + at, u, held);
    }
  }
}

// ---------------------------------------------------------------------
// thin: G in f64, the chain on s x s, one product
// ---------------------------------------------------------------------

constexpr int THIN_MAX = 320;  // the largest short side
constexpr int NARROW = 64;     // up to here one block takes the whole chain
constexpr int SUPER = 128;     // a block's square of G
constexpr int KC = 32;         // long-axis places a block stages at a time
constexpr int PITCH = SUPER + 16;

// X = (u x) y t, what the product that applies P needs of the norm.
struct Norm { float x, y, t; };

// X = U / n with n = |U|_F + eps as (u x) y 2^e, with (u x) y of a norm between
// 1/4 and 1, so that f16 planes of it hold their bits also where U is small
// beside eps; e is 0 from |U|_F = eps up.  The power of two x keeps y and the
// products normal for values near the ends of f32's range.  NaN for a matrix
// that is not finite; zeros stay zeros whatever eps, whose reciprocal may be
// more than an f32 holds.
// eps < 0: U is X already.
struct Unit {
  double x, y;
  int e;
  __device__ inline double all() const { return ldexp(x * y, e); }
  __device__ inline Norm norm() const {
    return Norm{(float)x, (float)y, (float)ldexp(1.0, e)};
  }
};

__device__ inline Unit unit_of(double sumsq, double eps) {
  if (!(sumsq < INFINITY)) return {1.0, NAN, 0};
  if (sumsq == 0) return {1.0, 1.0, 0};
  const double u = sqrt(sumsq), n = eps < 0 ? 1.0 : u + eps;
  const int e = min(0, ilogb(u) - ilogb(n) + 1);
  const double own = ldexp(n, e);  // |U|_F to 4 |U|_F (eps < 0: no more than 1)
  const double x = own > 0x1p60 ? 0x1p-60 : (own < 0x1p-60 ? 0x1p60 : 1.0);
  return {x, 1.0 / (own * x), e};
}

__device__ inline void split(float v, _Float16& hi, _Float16& lo) {
  // v as it is: a product that the compiler fuses with one of the conversions
  // and not with the other gives them two values of hi, once in 2^14
  asm("" : "+v"(v));
  hi = (_Float16)v;
  lo = (_Float16)(v - (float)hi);
}

// The sum of a block's values, the same for every thread and run.
__device__ inline double block_sum(double v, double* lds) {
#pragma unroll
  for (int o = WAVE / 2; o; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if (threadIdx.x % WAVE == 0) lds[threadIdx.x / WAVE] = v;
  __syncthreads();
  v = 0;
  for (int w = 0; w < (int)blockDim.x / WAVE; ++w) v += lds[w];
  return v;
}

// NT neighbours, those before `held` (any number), zeros after them
template <int NT, typename T>
__device__ inline void load_some(float (&v)[NT], const T* at, int64_t held) {
  if (NT == 4) {
    const float4 f = load_quad(at, held);
    v[0] = f.x;
    v[1 % NT] = f.y;
    v[2 % NT] = f.z;
    v[3 % NT] = f.w;
  } else if (NT == 2 && held >= 2) {
    Pair<T> p;
    p.load(at);
    v[0] = to_f32(p.get(0));
    v[1 % NT] = to_f32(p.get(1));
  } else {
    v[0] = held > 0 ? to_f32(at[0]) : 0.0f;
    if (NT == 2) v[1 % NT] = 0.0f;
  }
}

// Partial sums of G over one chunk of the long axis, short side up to
// 16 NT <= 64.  f64 matrix instructions 16x16x4: a lane holds row (or column)
// lane % 16 of a tile at place lane / 16.  Both orders are free: tile t takes
// columns NT c + t, so that a lane's values lie side by side, and four
// neighbouring places serve four instructions.  No LDS on the way: a wave reads
// its own places, the next ones while it multiplies, and four waves' sums are
// joined at the end.  part[b][chunk][tile (i, j <= i)][16][16].
template <typename T, bool TALL, int NT>
__global__ __launch_bounds__(256) void k_gram_narrow(
    double* __restrict__ part, const T* __restrict__ u,
    const int* __restrict__ touched, int64_t long_, int s, int64_t chunk) {
  constexpr int TILES = NT * (NT + 1) / 2;
  __shared__ double lds[TILES * 256];
  const int64_t b = blockIdx.y;
  if (touched && !touched[b]) return;
  const int lane = threadIdx.x % WAVE, wave = this_wave();
  const T* x = u + b * long_ * s;
  const int64_t k0 = blockIdx.x * chunk + wave * (chunk / 4);
  const int64_t k1 = min(k0 + chunk / 4, long_);
  f64x4 acc[TILES];
#pragma unroll
  for (int t = 0; t < TILES; ++t) acc[t] = (f64x4){0, 0, 0, 0};
  constexpr int TURNS = NT > 2 ? 1 : 2;  // 16 places each, loaded together
  float v[TURNS][4][NT];
  auto fetch = [&](int64_t k) {
#pragma unroll
    for (int h = 0; h < TURNS; ++h) {
      if (TALL) {
        const int col = lane % 16 * NT;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int64_t kk = k + h * 16 + 4 * c + lane / 16;
          load_some<NT>(v[h][c], x + kk * s + col, kk < k1 ? s - col : 0);
        }
      } else {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const int col = lane % 16 * NT + t;
          const int64_t kk = k + h * 16 + lane / 16 * 4;
          const float4 f = load_quad(x + col * long_ + kk,
                                     col < s ? k1 - kk : 0);
          v[h][0][t] = f.x;
          v[h][1][t] = f.y;
          v[h][2][t] = f.z;
          v[h][3][t] = f.w;
        }
      }
    }
  };
  fetch(k0);
  for (int64_t k = k0; k < k1; k += 16 * TURNS) {
    double w[TURNS][4][NT];
#pragma unroll
    for (int h = 0; h < TURNS; ++h)
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int t = 0; t < NT; ++t) w[h][c][t] = v[h][c][t];
    fetch(k + 16 * TURNS);
#pragma unroll
    for (int h = 0; h < TURNS; ++h)
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int j = 0; j <= i; ++j)
            acc[i * (i + 1) / 2 + j] = __builtin_amdgcn_mfma_f64_16x16x4f64(
                w[h][c][i], w[h][c][j], acc[i * (i + 1) / 2 + j], 0, 0, 0);
  }
  for (int w = 0; w < 4; ++w) {
    if (wave == w) {
#pragma unroll
      for (int t = 0; t < TILES; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          double* to = lds + t * 256 + (lane / 16 + 4 * r) * 16 + lane % 16;
          *to = w ? *to + acc[t][r] : acc[t][r];
        }
    }
    __syncthreads();
  }
  double* out = part + (b * gridDim.x + blockIdx.x) * (int64_t)(TILES * 256);
#pragma unroll
  for (int t = 0; t < TILES; ++t)
    out[t * 256 + threadIdx.x] = lds[t * 256 + threadIdx.x];
}

// sum[b][size] = the chunks' sum, in an order of its own that does not change:
// 16 values a block, 16 threads a value.
__global__ __launch_bounds__(256) void k_part_sum(
    double* __restrict__ sum, const double* __restrict__ part,
    const int* __restrict__ touched, int chunks, int64_t size) {
  __shared__ double slices[16][17];
  const int64_t b = blockIdx.y;
  if (touched && !touched[b]) return;
  const int64_t e = (int64_t)blockIdx.x * 16 + threadIdx.x % 16;
  const double* p = part + b * chunks * size + e;
  double v[4] = {0, 0, 0, 0};
  int k = threadIdx.x / 16;
  for (; k + 48 < chunks; k += 64)
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] += p[(k + q * 16) * size];
  for (; k < chunks; k += 16) v[0] += p[k * size];
  slices[threadIdx.x / 16][threadIdx.x % 16] = (v[0] + v[1]) + (v[2] + v[3]);
  __syncthreads();
  if (threadIdx.x >= 16) return;
  double t = 0;
  for (int q = 0; q < 16; ++q) t += slices[q][threadIdx.x];
  sum[b * size + e] = t;
}

// KC places of a diagonal square of G, 8 x 8 tiles of which nt x nt exist:
// wave W takes tile rows W and 7 - W up to the diagonal, nine tiles.
template <int W, int N>
__device__ inline void diagonal_places(f64x4 (&acc)[N],
                                       const float (*rows)[PITCH], int lane,
                                       int nt) {
#pragma unroll
  for (int q = 0; q < KC; q += 4) {
    const float* at = rows[q + lane / 16] + lane % 16;
    double v[8 - W];
#pragma unroll
    for (int t = 0; t < 8 - W; ++t) v[t] = at[t * 16];
    if (W < nt) {
#pragma unroll
      for (int t = 0; t <= W; ++t)
        acc[t] = __builtin_amdgcn_mfma_f64_16x16x4f64(v[W], v[t], acc[t], 0,
                                                      0, 0);
    }
    if (7 - W < nt) {
#pragma unroll
      for (int t = 0; t <= 7 - W; ++t)
        acc[W + 1 + t] = __builtin_amdgcn_mfma_f64_16x16x4f64(
            v[7 - W], v[t], acc[W + 1 + t], 0, 0, 0);
    }
  }
}

// f(tile row, tile column, sum) for each of the nine
template <int W, int N, typename F>
__device__ inline void diagonal_tiles(const f64x4 (&acc)[N], F f) {
#pragma unroll
  for (int t = 0; t <= W; ++t) f(W, t, acc[t]);
#pragma unroll
  for (int t = 0; t <= 7 - W; ++t) f(7 - W, t, acc[W + 1 + t]);
}

#define BY_WAVE(wave, call)        \
  switch (wave) {                  \
    case 0: { constexpr int W = 0; call; } break; \
    case 1: { constexpr int W = 1; call; } break; \
    case 2: { constexpr int W = 2; call; } break; \
    default: { constexpr int W = 3; call; } break; \
  }

// The same for short sides up to THIN_MAX: a block takes the places of one
// chunk for a SUPER x SUPER square of G on the diagonal, or for half of one under
// it, through LDS (two buffers, one barrier a turn), nine or eight tiles a wave.
// The matrix instructions bound it: 64 cycles a tile and 4 places.
// part[b][chunk][sp][sp].
//
// With STEP (tall, one square) the values are those of U as the momentum
// makes it: M and the gradients come in, M and U go out on the way.
template <typename T, bool TALL, bool STEP>
__global__ __launch_bounds__(256, 2) void k_gram64(
    double* __restrict__ part, double* __restrict__ traces,
    const T* __restrict__ u, Momentum mom, const int64_t* __restrict__ place,
    const int* __restrict__ touched, int64_t long_, int s, int sp,
    int64_t chunk) {
  constexpr int HALF = SUPER / 2, HPITCH = HALF + 16;
  __shared__ float lds[2][KC][PITCH];
  __shared__ float other[STEP ? 1 : 2][KC][HPITCH];  // the half's rows
  __shared__ double sums[4];
  const int64_t b = blockIdx.z;
  if (touched && !touched[b]) return;
  // blockIdx.y: of each row of squares first the halves, then the diagonal one
  int si = 0, y = STEP ? 0 : blockIdx.y;
  while (y > 2 * si) { y -= 2 * si + 1; ++si; }
  const int sj = y / 2;
  const bool diagonal = STEP || si == sj;
  const int row0 = si * SUPER + (diagonal ? 0 : y % 2 * HALF);
  const int col0 = sj * SUPER;
  const int nt = min(8, (sp - col0) / 16);  // tiles of its columns
  if (row0 >= sp) return;                   // no such half
  const int lane = threadIdx.x % WAVE, wave = this_wave();
  const T* x = u + b * long_ * s;
  const int64_t k0 = blockIdx.x * chunk;
  const int64_t k1 = min(k0 + chunk, long_);

  f64x4 acc[9];
#pragma unroll
  for (int t = 0; t < 9; ++t) acc[t] = (f64x4){0, 0, 0, 0};

  // STEP: the places are known a turn ahead of the values
  int64_t at_[4];
  auto look = [&](int64_t k) {
#pragma unroll
    for (int l = 0; l < 4; ++l) {
      const int64_t kk = k + (threadIdx.x + l * 256) / 32;
      at_[l] = STEP && kk < k1 ? place[b * long_ + kk] : -1;
    }
  };

  // Quads along the columns (TALL) or along the places: four of the square's
  // columns a thread, and two of the half's rows (STEP: four gradients).
  float4 next[4], more[STEP ? 4 : 2];
  auto some = [&](int64_t k, int kk, int col) {
    return load_quad(TALL ? x + (k + kk) * s + col
                          : x + (int64_t)col * long_ + k + kk,
                     TALL ? (k + kk < k1 ? (int64_t)s - col : 0)
                          : (col < s ? k1 - k - kk : 0));
  };
  auto fetch = [&](int64_t k) {
#pragma unroll
    for (int l = 0; l < 4; ++l) {
      const int e = threadIdx.x + l * 256;
      const int kk = TALL ? e / 32 : e % 8 * 4, c = TALL ? e % 32 * 4 : e / 8;
      if (STEP) {
        const int held = k + kk < k1 ? s - c : 0;
        const int64_t row = b * long_ + k + kk;
        next[l] = load_quad(mom.m + row * s + c, held);
        more[l % (STEP ? 4 : 2)] = row_gradient(mom, at_[l], row, s, c, held);
      } else {
        next[l] = some(k, kk, col0 + c);
      }
    }
    if (!STEP && !diagonal) {
#pragma unroll
      for (int l = 0; l < 2; ++l) {
        const int e = threadIdx.x + l * 256;
        more[l] = some(k, TALL ? e / 16 : e % 8 * 4,
                       row0 + (TALL ? e % 16 * 4 : e / 8));
      }
    }
  };
  auto put_some = [&](float* to, int pitch, float4 f) {
    if (TALL) {
      *(float4*)to = f;
    } else {
      to[0] = f.x;
      to[pitch] = f.y;
      to[2 * pitch] = f.z;
      to[3 * pitch] = f.w;
    }
  };
  auto put = [&](int64_t k, int buffer) {
#pragma unroll
    for (int l = 0; l < 4; ++l) {
      const int e = threadIdx.x + l * 256;
      const int kk = TALL ? e / 32 : e % 8 * 4, c = TALL ? e % 32 * 4 : e / 8;
      float4 v = next[l];
      if (STEP) {
        const int held = k + kk < k1 ? s - c : 0;
        const int64_t at = (b * long_ + k + kk) * s + c;
        const float4 m = next_momentum(mom, next[l],
                                       more[l % (STEP ? 4 : 2)], &v);
        store_quad(mom.m + at, m, held);
        store_quad(mom.u + at, v, held);
      }
      put_some(&lds[buffer][kk][c], PITCH, v);
    }
    if (!STEP && !diagonal) {
#pragma unroll
      for (int l = 0; l < 2; ++l) {
        const int e = threadIdx.x + l * 256;
        put_some(&other[STEP ? 0 : buffer][TALL ? e / 16 : e % 8 * 4]
                       [TALL ? e % 16 * 4 : e / 8],
                 HPITCH, more[l]);
      }
    }
  };

  look(k0);
  fetch(k0);
  look(k0 + KC);
  put(k0, 0);
  int buffer = 0;
  for (int64_t k = k0; k < k1; k += KC) {
    __syncthreads();
    const bool again = k + KC < k1;
    if (again) {
      fetch(k + KC);
      look(k + 2 * KC);
    }
    const float (*cols)[PITCH] = lds[buffer];
    if (diagonal) {
      BY_WAVE(wave, diagonal_places<W>(acc, cols, lane, nt))
    } else if (row0 + wave * 16 < sp) {
      const float (*rows)[HPITCH] = other[STEP ? 0 : buffer];
#pragma unroll
      for (int q = 0; q < KC; q += 4) {
        const int kk = q + lane / 16;
        const double av = rows[kk][wave * 16 + lane % 16];
        double bv[8];
#pragma unroll
        for (int t = 0; t < 8; ++t) bv[t] = cols[kk][t * 16 + lane % 16];
#pragma unroll
        for (int t = 0; t < 8; ++t)  // all of them exist left of the diagonal
          acc[t] = __builtin_amdgcn_mfma_f64_16x16x4f64(av, bv[t], acc[t], 0,
                                                        0, 0);
      }
    }
    if (again) put(k + KC, buffer ^ 1);
    buffer ^= 1;
  }
  double* out = part + (b * gridDim.x + blockIdx.x) * (int64_t)sp * sp;
  double trace = 0;
  auto keep = [&](int ti, int tj, const f64x4& v) {
    const int i0 = row0 + ti * 16, j0 = col0 + tj * 16;
    if (i0 >= sp || j0 >= sp) return;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = i0 + lane / 16 + 4 * r, j = j0 + lane % 16;
      out[(int64_t)i * sp + j] = v[r];
      if (i == j) trace += v[r];
    }
  };
  if (diagonal) {
    BY_WAVE(wave, diagonal_tiles<W>(acc, keep))
    trace = block_sum(trace, sums);
    if (threadIdx.x == 0)
      traces[(b * gridDim.x + blockIdx.x) * ((sp + SUPER - 1) / SUPER) + si] =
          trace;
  } else {
#pragma unroll
    for (int t = 0; t < 8; ++t) keep(wave, t, acc[t]);
  }
}

// G = nu^2 times the sum of the parts, in their order; the upper half by
// symmetry.  nu from the trace, |U|_F^2.
__global__ __launch_bounds__(256) void k_gram_sum(
    double* __restrict__ g, Norm* __restrict__ norm,
    const double* __restrict__ part, const double* __restrict__ traces,
    const int* __restrict__ touched, int chunks, int sp, double eps) {
  __shared__ double sums[4];
  const int64_t b = blockIdx.y;
  if (touched && !touched[b]) return;
  const int count = chunks * ((sp + SUPER - 1) / SUPER);
  double t = 0;
  for (int k = threadIdx.x; k < count; k += 256) t += traces[b * count + k];
  const Unit f = unit_of(block_sum(t, sums), eps);
  const double nu = f.all();
  if (blockIdx.x == 0 && threadIdx.x == 0) norm[b] = f.norm();
  // 16 values a block, 16 threads a value
  __shared__ double slices[16][17];
  const int64_t size = (int64_t)sp * sp;
  const int64_t e = (int64_t)blockIdx.x * 16 + threadIdx.x % 16;
  const int i = e / sp, j = e % sp;
  const double* p = part + b * chunks * size + e;
  double sum[4] = {0, 0, 0, 0};
  if (i >= j) {
    int k = threadIdx.x / 16;
    for (; k + 48 < chunks; k += 64)
#pragma unroll
      for (int q = 0; q < 4; ++q) sum[q] += p[(k + q * 16) * size];
    for (; k < chunks; k += 16) sum[0] += p[k * size];
  }
  slices[threadIdx.x / 16][threadIdx.x % 16] =
      (sum[0] + sum[1]) + (sum[2] + sum[3]);
  __syncthreads();
  if (threadIdx.x >= 16 || i < j) return;
  double v = 0;
  for (int q = 0; q < 16; ++q) v += slices[q][threadIdx.x];
  v *= nu * nu;
  g[b * size + e] = v;
  g[b * size + (int64_t)j * sp + i] = v;
}

// One product of commuting symmetric matrices (so it is symmetric too):
// out = x y, or, if `poly`, a I + b x + c (x y).
struct SmallMul {
  double* out;
  const double *x, *y;
  bool poly;
};

// A block a tile on or under the diagonal, mirrored; the four waves share the
// places of the sum.  blockIdx.z counts the products.
__global__ __launch_bounds__(256) void k_small_mul(
    SmallMul j0, SmallMul j1, const int* __restrict__ touched, int s, int sp,
    Coeffs k) {
  __shared__ double lds[4][256];
  const int64_t b = blockIdx.y;
  if (touched && !touched[b]) return;
  const SmallMul job = blockIdx.z ? j1 : j0;
  int ti = 0, tj = blockIdx.x;
  while (tj > ti) { tj -= ti + 1; ++ti; }
  const int64_t base = b * (int64_t)sp * sp;
  const int lane = threadIdx.x % WAVE, wave = this_wave();
  const double* xr = job.x + base + (int64_t)(ti * 16 + lane % 16) * sp;
  const double* yr = job.y + base + (int64_t)(tj * 16 + lane % 16) * sp;
  f64x4 acc = (f64x4){0, 0, 0, 0};
  for (int kk = wave * 16; kk < sp; kk += 64) {
    const f64x4 xv = *(const f64x4*)(xr + kk + lane / 16 * 4);
    const f64x4 yv = *(const f64x4*)(yr + kk + lane / 16 * 4);
#pragma unroll
    for (int c = 0; c < 4; ++c)
      acc = __builtin_amdgcn_mfma_f64_16x16x4f64(xv[c], yv[c], acc, 0, 0, 0);
  }
#pragma unroll
  for (int r = 0; r < 4; ++r)
    lds[wave][(lane / 16 + 4 * r) * 16 + lane % 16] = acc[r];
  __syncthreads();
  const int e = threadIdx.x;
  double v = (lds[0][e] + lds[1][e]) + (lds[2][e] + lds[3][e]);
  const int i = ti * 16 + e / 16, j = tj * 16 + e % 16;
  if (i < j) return;  // a tile on the diagonal
  const int64_t at = base + (int64_t)i * sp + j, ta = base + (int64_t)j * sp + i;
  if (job.poly) v = k.b * job.x[at] + k.c * v + (i == j && i < s ? k.a : 0.0);
  job.out[at] = v;
  job.out[ta] = v;
}

// `by` P in two f16 planes of jp x kp places, zeros around it
__global__ __launch_bounds__(256) void k_small_out(
    _Float16* __restrict__ planes, const double* __restrict__ p,
    const int* __restrict__ touched, int s, int sp, int jp, int kp,
    double by) {
  const int64_t b = blockIdx.y;
  if (touched && !touched[b]) return;
  const int e = blockIdx.x * 256 + threadIdx.x;
  if (e >= jp * kp) return;
  const int i = e / kp, j = e % kp;
  const int64_t plane = gridDim.y * (int64_t)jp * kp;
  _Float16* to = planes + b * (int64_t)jp * kp + e;
  split(i < s && j < s ? (float)(p[(b * sp + i) * sp + j] * by) : 0.0f, to[0],
        to[plane]);
}

// The chain for short sides up to 64: one block a matrix, G, Q, P and G Q in
// LDS; a wave a tile on or under the diagonal.  What bounds it is the length
// of the chain: 14 products that wait for each other at five steps.
template <int NT, int WAVES>
__global__ __launch_bounds__(WAVES * WAVE) void k_chain(
    _Float16* __restrict__ planes, Norm* __restrict__ norm,
    const double* __restrict__ part, const int* __restrict__ touched,
    int chunks, int s, int steps, Coeffs k, double eps, int jp, int kp,
    double by) {
  constexpr int SP = NT * 16, LP = SP + 2, TILES = NT * (NT + 1) / 2;
  // tiles of two products at a time
  constexpr int MINE = (2 * TILES + WAVES - 1) / WAVES;
  __shared__ double g[SP * LP], q[SP * LP], p[SP * LP], t[SP * LP];
  __shared__ double sums[WAVES];
  const int64_t b = blockIdx.x;
  if (touched && !touched[b]) return;
  const int lane = threadIdx.x % WAVE, wave = this_wave();
  const double* from = part + b * chunks * (int64_t)(TILES * 256);

  // the sum of the parts: 256 threads take a value of every tile each, and
  // every (WAVES / 4)-th part
  const int slice = wave / 4, e = threadIdx.x % 256;
  double sum[TILES] = {};
#pragma unroll 8
  for (int c = slice; c < chunks; c += WAVES / 4)
#pragma unroll
    for (int o = 0; o < TILES; ++o)
      sum[o] += from[((int64_t)c * TILES + o) * 256 + e];
  for (int w = 0; w < WAVES / 4; ++w) {
    if (slice == w) {
      int ti = 0, tj = 0;
#pragma unroll
      for (int o = 0; o < TILES; ++o) {
        // as k_gram_narrow orders them
        const int i = e / 16 * NT + ti, j = e % 16 * NT + tj;
        double v = sum[o];
        if (w) v += g[i * LP + j];
        g[i * LP + j] = v;
        if (ti != tj) g[j * LP + i] = v;
        if (++tj > ti) { tj = 0; ++ti; }
      }
    }
    __syncthreads();
  }
  const double trace = threadIdx.x < SP ? g[threadIdx.x * (LP + 1)] : 0.0;
  const Unit f = unit_of(block_sum(trace, sums), eps);
  const double nu = f.all();
  if (threadIdx.x == 0) norm[b] = f.norm();
  for (int o = threadIdx.x; o < SP * LP; o += WAVES * WAVE)
    if (o % LP < SP) g[o] *= nu * nu;
  __syncthreads();

  // One or two products: out = x y, or a I + b x + c x y; `out` may be one of
  // the operands.
  struct Job { double* out; const double *x, *y; };
  auto mul = [&](Job j0, Job j1, bool poly) {
    f64x4 acc[MINE];
#pragma unroll
    for (int o = 0; o < MINE; ++o) {
      acc[o] = (f64x4){0, 0, 0, 0};
      int tj = wave + o * WAVES, ti = 0;
      const bool second = tj >= TILES;
      if (second) tj -= TILES;
      const Job job = second ? j1 : j0;
      if (!job.out || tj >= TILES) continue;
      while (tj > ti) { tj -= ti + 1; ++ti; }
      const double* xr = job.x + (ti * 16 + lane % 16) * LP + lane / 16;
      const double* yr = job.y + (tj * 16 + lane % 16) * LP + lane / 16;
#pragma unroll
      for (int kk = 0; kk < SP; kk += 4)
        acc[o] = __builtin_amdgcn_mfma_f64_16x16x4f64(xr[kk], yr[kk], acc[o],
                                                      0, 0, 0);
      if (poly) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = ti * 16 + lane / 16 + 4 * r;
          const int j = tj * 16 + lane % 16;
          acc[o][r] = k.b * job.x[i * LP + j] + k.c * acc[o][r] +
                      (i == j && i < s ? k.a : 0.0);
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int o = 0; o < MINE; ++o) {
      int tj = wave + o * WAVES, ti = 0;
      const bool second = tj >= TILES;
      if (second) tj -= TILES;
      double* out = second ? j1.out : j0.out;
      if (!out || tj >= TILES) continue;
      while (tj > ti) { tj -= ti + 1; ++ti; }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = ti * 16 + lane / 16 + 4 * r;
        const int j = tj * 16 + lane % 16;
        if (i < j) continue;
        out[i * LP + j] = acc[o][r];
        out[j * LP + i] = acc[o][r];
      }
    }
    __syncthreads();
  };
  const Job none{nullptr, nullptr, nullptr};
  for (int step = 0; step < steps; ++step) {
    double* qi = step ? q : p;  // the first Q is P
    mul({qi, g, g}, none, true);
    const Job grow{t, g, qi}, more{p, p, q};
    const bool last = step + 1 == steps;
    if (step) mul(more, last ? none : grow, false);
    else if (!last) mul(grow, none, false);
    if (!last) mul({g, qi, t}, none, false);
  }
  const int64_t plane = gridDim.x * (int64_t)jp * kp;
  for (int o = threadIdx.x; o < jp * kp; o += WAVES * WAVE) {
    const int i = o / kp, j = o % kp;
    _Float16* to = planes + b * (int64_t)jp * kp + o;
    split(i < s && j < s ? (float)(p[i * LP + j] * by) : 0.0f, to[0],
          to[plane]);
  }
}

// O = U P (TALL) or P U: 16 JT of P's rows, up to KS places long, in LDS; a wave
// takes its values from memory to the matrix instructions by itself, split in
// two planes on the way, CH places of the sum at a time.  A lane holds eight
// places of long-axis row lane % 16, or (wide) of four neighbouring ones, which
// lie in four tiles.  Of 32 places of the sum, lane group g = lane / 16 takes
// 4 g .. 4 g + 3 and 16 + 4 g .. 16 + 4 g + 3, so that a load of four groups is
// 64 bytes of a row; P lies in LDS in that order.  Bound by memory.
template <typename T, bool TALL, int JT, int KS, int WAVES>
__global__ __launch_bounds__(WAVES * WAVE) void k_thin_apply(
    Result res, const T* __restrict__ u, const _Float16* __restrict__ planes,
    const Norm* __restrict__ norm, const int* __restrict__ touched,
    int64_t long_, int s, int jp, int kp, float down) {
  constexpr int LP = KS + 8;  // rows of eight lanes' pieces in other banks
  constexpr int RT = TALL ? 2 : 4;         // tiles of the long axis a wave
  constexpr int TURN = WAVES * 16 * RT;    // places of it a block and turn
  constexpr int CH = KS < 64 ? 32 : TALL && KS == 128 ? 128 : 64;
  __shared__ _Float16 lds[2][JT * 16 * LP];
  const int64_t b = blockIdx.z;
  if (touched && !touched[b]) return;
  const int lane = threadIdx.x % WAVE, wave = this_wave();
  const int j0 = blockIdx.y * JT * 16;
  const Norm nm = norm[b];
  const float up = nm.y * UP;
  auto result = [&](float v) { return v * down * nm.t; };
  const T* x = u + b * long_ * s;
  const _Float16* p = planes + (b * jp + j0) * (int64_t)kp;
  const int64_t plane = gridDim.z * (int64_t)jp * kp;
  for (int e = threadIdx.x; e < 2 * JT * 16 * (KS / 8); e += WAVES * WAVE) {
    const int h = e / (JT * 16 * (KS / 8)), r = e / (KS / 8) % (JT * 16);
    const int c = e % (KS / 8) * 8;
    half8 v = {};
    if (c < kp) v = *(const half8*)(p + h * plane + (int64_t)r * kp + c);
    // places c .. c + 3 are those of group c % 16 / 4, the next four the next's
    _Float16* to = &lds[h][r * LP + c / 32 * 32 + c % 16 * 2 + c % 32 / 16 * 4];
    *(half4*)to = __builtin_shufflevector(v, v, 0, 1, 2, 3);
    *(half4*)(to + 8) = __builtin_shufflevector(v, v, 4, 5, 6, 7);
  }
  __syncthreads();

  for (int64_t base = (int64_t)blockIdx.x * TURN + wave * (16 * RT);
       base < long_; base += (int64_t)gridDim.x * TURN) {
    // the long-axis place of the lane's row in tile w
    const int64_t r0 = base + (TALL ? lane % 16 : lane % 16 * 4);
    auto at = [&](int w) { return r0 + w * (TALL ? 16 : 1); };
    f32x4 acc[JT][RT];
#pragma unroll
    for (int t = 0; t < JT; ++t)
#pragma unroll
      for (int w = 0; w < RT; ++w) acc[t][w] = (f32x4){0, 0, 0, 0};
    for (int kc = 0; kc < kp; kc += CH) {
      float raw[CH / 32][RT][8];
#pragma unroll
      for (int ks = 0; ks < CH / 32; ++ks) {
        const int k = kc + ks * 32 + lane / 16 * 4;
        if (TALL) {
#pragma unroll
          for (int w = 0; w < RT; ++w)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float4 f = load_quad(x + at(w) * s + k + h * 16,
                                         at(w) < long_ ? s - k - h * 16 : 0);
              raw[ks][w][h * 4] = f.x;
              raw[ks][w][h * 4 + 1] = f.y;
              raw[ks][w][h * 4 + 2] = f.z;
              raw[ks][w][h * 4 + 3] = f.w;
            }
        } else {
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            const int kk = k + c % 4 + c / 4 * 16;
            const float4 f = load_quad(x + kk * long_ + r0,
                                       kk < s ? long_ - r0 : 0);
            raw[ks][0][c] = f.x;
            raw[ks][1][c] = f.y;
            raw[ks][2 % RT][c] = f.z;
            raw[ks][3 % RT][c] = f.w;
          }
        }
      }
#pragma unroll
      for (int ks = 0; ks < CH / 32; ++ks) {
        if (KS > 128 && kc + ks * 32 >= kp) continue;
        half8 hi[RT], lo[RT];
#pragma unroll
        for (int w = 0; w < RT; ++w)
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            _Float16 h, l;
            split(raw[ks][w][c] * nm.x * up, h, l);
            hi[w][c] = h;
            lo[w][c] = l;
          }
#pragma unroll
        for (int t = 0; t < JT; ++t) {
          const int from = (t * 16 + lane % 16) * LP + kc + ks * 32 +
                           lane / 16 * 8;
          const half8 ph = *(const half8*)&lds[0][from];
          const half8 pl = *(const half8*)&lds[1][from];
#pragma unroll
          for (int w = 0; w < RT; ++w) {
            acc[t][w] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                pl, hi[w], acc[t][w], 0, 0, 0);
            acc[t][w] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                ph, lo[w], acc[t][w], 0, 0, 0);
            acc[t][w] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                ph, hi[w], acc[t][w], 0, 0, 0);
          }
        }
      }
    }
    const int64_t mine = b * long_ * s;
#pragma unroll
    for (int t = 0; t < JT; ++t) {
      const int j = j0 + t * 16 + lane / 16 * 4;
      if (TALL) {
#pragma unroll
        for (int w = 0; w < RT; ++w)
          finish_quad<T>(res, mine + at(w) * s + j,
                         make_float4(result(acc[t][w][0]), result(acc[t][w][1]),
                                     result(acc[t][w][2]),
                                     result(acc[t][w][3])),
                         at(w) < long_ ? s - j : 0);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          finish_quad<T>(res, mine + (int64_t)(j + i) * long_ + r0,
                         make_float4(result(acc[t][0][i]), result(acc[t][1][i]),
                                     result(acc[t][2 % RT][i]),
                                     result(acc[t][3 % RT][i])),
                         j + i < s ? long_ - r0 : 0);
      }
    }
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

template <typename T>
__global__ __launch_bounds__(256) void k_sumsq(
    double* __restrict__ part, const T* __restrict__ u,
    const int* __restrict__ touched, int64_t size) {
  __shared__ double lds[4];
  const int64_t b = blockIdx.y;
  if (touched && !touched[b]) return;
  const T* x = u + b * size;
  double t = 0;
#pragma unroll 4
  for (int64_t e = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; e < size;
       e += (int64_t)gridDim.x * 1024) {
    const float4 f = load_quad(x + e, size - e);
    t += ((double)f.x * f.x + (double)f.y * f.y) +
         ((double)f.z * f.z + (double)f.w * f.w);
  }
  t = block_sum(t, lds);
  if (threadIdx.x == 0) part[b * gridDim.x + blockIdx.x] = t;
}

// The planes of X as it lies in memory (m x n) and transposed, 64 x 64 values
// a block, zeros around them, as 2^-e X (see unit_of); e goes to `small`.  The
// values are on their way while the norm is summed, and go out four at a time.
template <typename T>
__global__ __launch_bounds__(256) void k_planes(
    Planes nat, Planes trn, int* __restrict__ small, const T* __restrict__ u,
    const double* __restrict__ part, int parts,
    const int* __restrict__ touched, int64_t m, int64_t n, double eps) {
  __shared__ float lds[64][65];
  __shared__ double sums[4];
  const int64_t b = blockIdx.z;
  if (touched && !touched[b]) return;
  const int64_t wide = nat.pitch / 64;
  const int64_t r0 = blockIdx.x / wide * 64, c0 = blockIdx.x % wide * 64;
  float4 v[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int64_t r = r0 + threadIdx.x / 16 + k * 16;
    const int64_t c = c0 + threadIdx.x % 16 * 4;
    v[k] = load_quad(u + (b * m + r) * n + c, r < m ? n - c : 0);
  }
  double t = 0;
  for (int k = threadIdx.x; k < parts; k += 256) t += part[b * parts + k];
  const Unit f = unit_of(block_sum(t, sums), eps);
  const float2 sc = make_float2((float)f.x, (float)f.y);
  if (blockIdx.x == 0 && threadIdx.x == 0) small[b] = f.e;
  auto put = [](const Planes& to, int64_t at, const float (&x)[4]) {
    half4 hi, lo;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      _Float16 h, l;
      split(x[i], h, l);
      hi[i] = h;
      lo[i] = l;
    }
    *(half4*)(to.p + at) = hi;
    *(half4*)(to.p + at + to.plane) = lo;
  };
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int r = threadIdx.x / 16 + k * 16, c = threadIdx.x % 16 * 4;
    const float x[4] = {v[k].x * sc.x * sc.y * UP, v[k].y * sc.x * sc.y * UP,
                        v[k].z * sc.x * sc.y * UP, v[k].w * sc.x * sc.y * UP};
#pragma unroll
    for (int i = 0; i < 4; ++i) lds[r][c + i] = x[i];
    put(nat, b * nat.batch + (r0 + r) * nat.pitch + c0 + c, x);
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int c = threadIdx.x / 16 + k * 16, r = threadIdx.x % 16 * 4;
    const float x[4] = {lds[r][c], lds[r + 1][c], lds[r + 2][c],
                        lds[r + 3][c]};
    put(trn, b * trn.batch + (c0 + c) * trn.pitch + r0 + r, x);
  }
}

enum Ending { GRAM, POLY, UPDATE, FINAL };

// D[i][j] = scale sum_k a[i][k] b[j][k], of the values that the planes hold.
struct Factors {
  Planes a, b, d;
  float scale;
};

// Planes of X hold 2^-e X with e = min(0, small[b] + grown), where the steps so
// far multiply by 2^grown at most: a matrix that is small beside eps (see
// unit_of) keeps its bits while it grows.
struct Exponents {
  const int* small;
  int grown;  // of the X that the product takes
  int times;  // how often it takes X
  int next;   // UPDATE: `grown` of the X that it makes

  __device__ inline int of(int64_t b, int g) const {
    return min(0, small[b] + g);
  }
};

struct Product {
  Factors f[2];      // blockIdx.y says which
  Exponents e;
  int k;             // a multiple of 32
  Planes dt;         // UPDATE: D transposed (GRAM, POLY: D is symmetric)
  float ca, cb, cc;  // POLY: a I + b a + c D
  int s;             // POLY: I ends here
  int64_t rows, cols;  // FINAL: D's own size
  bool tall;           // FINAL: D transposed is what lies in memory
  Result res;
  // the work: tiles of one matrix (ns rows of them, nl columns), matrices;
  // of all tiles the first `whole` are a block's each, the others have their
  // sum shared out to `splits` blocks, which leave it in `parts`
  int ns, nl, tiles, splits;
  uint32_t all, whole;
  float* parts;
};

constexpr int XCDS = 8;   // block b runs on XCD b % 8, each with its own L2
constexpr int STRIP = 8;  // tiles are taken in strips of eight columns

// Tile t of the ns x nl tiles, or (HALF) of those on and under the diagonal
// of ns x ns: strips of STRIP columns, a strip's rows one after the other, so
// that neighbours in t share their operands' rows.
template <bool HALF>
__device__ inline void tile_of(int t, int ns, int nl, int* bi, int* bj) {
  if (!HALF) {
    const int strip = t / (ns * STRIP), rest = t - strip * ns * STRIP;
    const int wide = min(STRIP, nl - strip * STRIP);
    *bi = rest / wide;
    *bj = strip * STRIP + rest % wide;
    return;
  }
  int c0 = 0;
  for (;;) {
    const int wide = min(STRIP, ns - c0), head = wide * (wide + 1) / 2;
    const int size = head + max(0, ns - c0 - STRIP) * STRIP;
    if (t < size) {
      if (t >= head) {
        *bi = c0 + STRIP + (t - head) / STRIP;
        *bj = c0 + (t - head) % STRIP;
      } else {
        int i = 0;
        while (t > i) { t -= i + 1; ++i; }
        *bi = c0 + i;
        *bj = c0 + t;
      }
      return;
    }
    t -= size;
    c0 += STRIP;
  }
}

// a's values (both planes) that POLY adds, as a lane holds D's.
template <int NT>
struct Old {
  half4 v[NT / 32][NT / 32][2];

  __device__ inline void load(const Planes& a, int64_t b, int bi, int bj) {
    const int lane = threadIdx.x % WAVE, wave = this_wave();
    // a is symmetric: its row j has a lane's four values side by side
    const _Float16* g =
        a.p + b * a.batch +
        ((int64_t)bj * NT + wave % 2 * (NT / 2) + lane % 16) * a.pitch +
        (int64_t)bi * NT + wave / 2 * (NT / 2) + lane / 16 * 4;
#pragma unroll
    for (int ti = 0; ti < NT / 32; ++ti)
#pragma unroll
      for (int tj = 0; tj < NT / 32; ++tj)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          v[ti][tj][h] =
              *(const half4*)(g + h * a.plane + tj * 16 * a.pitch + ti * 16);
  }
};

// Halves of LDS that end_product needs.
template <int NT>
constexpr int end_size() { return 2 * NT * (NT + 8); }

// What one block leaves of its tile: a lane holds D[i .. i + 3][j] of each
// 16 x 16 tile of its wave's quarter.  `lds` is free to be written once
// everybody is here.
template <int NT, Ending E, typename T>
__device__ inline void end_product(const Product& pr, const Factors& f,
                                   int64_t b, int bi, int bj,
                                   f32x4 (&acc)[NT / 32][NT / 32],
                                   const Old<NT>& old, _Float16* lds) {
  constexpr int W = NT / 32;
  const int lane = threadIdx.x % WAVE, wave = this_wave();
  const int wi = wave / 2 * (NT / 2), wj = wave % 2 * (NT / 2);
  // what D has to be multiplied by for the exponents of its X
  float by = 1.0f;
  if (E != POLY)
    by = ldexpf(1.0f, pr.e.times * pr.e.of(b, pr.e.grown) -
                          (E == UPDATE ? pr.e.of(b, pr.e.next) : 0));
  if (E == FINAL) {
#pragma unroll
    for (int ti = 0; ti < W; ++ti)
#pragma unroll
      for (int tj = 0; tj < W; ++tj) {
        const int64_t i = (int64_t)bi * NT + wi + ti * 16 + lane / 16 * 4;
        const int64_t j = (int64_t)bj * NT + wj + tj * 16 + lane % 16;
        if (j >= pr.cols) continue;
        const f32x4 v = acc[ti][tj] * f.scale * by;
        const int64_t base = b * pr.rows * pr.cols;
        if (pr.tall) {
          finish_quad<T>(pr.res, base + j * pr.rows + i,
                         make_float4(v[0], v[1], v[2], v[3]), pr.rows - i);
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (i + r < pr.rows)
              finish<T>(pr.res, base + (i + r) * pr.cols + j, v[r]);
        }
      }
    return;
  }
  // D as it is goes out through LDS, in 16-byte pieces; D transposed, four
  // values a lane, from the registers.
  constexpr int ROW = NT + 8;
  const bool both = E == UPDATE || bi != bj;
  const Planes& t = E == UPDATE ? pr.dt : f.d;
  const float scale = f.scale * by;
  __syncthreads();
#pragma unroll
  for (int ti = 0; ti < W; ++ti)
#pragma unroll
    for (int tj = 0; tj < W; ++tj) {
      const int li = wi + ti * 16 + lane / 16 * 4;
      const int lj = wj + tj * 16 + lane % 16;
      const int64_t i = (int64_t)bi * NT + li, j = (int64_t)bj * NT + lj;
      const f32x4 v = acc[ti][tj] * scale;
      half4 hi, lo;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float x = v[r];
        if (E == POLY) {
          x = pr.cc * x + pr.cb * ((float)old.v[ti][tj][0][r] +
                                   (float)old.v[ti][tj][1][r]);
          if (i + r == j && j < pr.s) x += pr.ca * UP;
        }
        _Float16 xh, xl;
        split(x, xh, xl);
        hi[r] = xh;
        lo[r] = xl;
        lds[(li + r) * ROW + lj] = xh;
        lds[(NT + li + r) * ROW + lj] = xl;
      }
      if (both) {
        _Float16* to = t.p + b * t.batch + j * t.pitch + i;
        *(half4*)to = hi;
        *(half4*)(to + t.plane) = lo;
      }
    }
  __syncthreads();
#pragma unroll
  for (int e = threadIdx.x; e < NT * NT / 4; e += 256) {
    const int r = e / (NT / 8), c = e % (NT / 8) * 8;  // rows of both planes
    const int h = r >= NT;
    *(half8*)(f.d.p + h * f.d.plane + b * f.d.batch +
              ((int64_t)bi * NT + r - h * NT) * f.d.pitch + (int64_t)bj * NT +
              c) = *(const half8*)(lds + r * ROW + c);
  }
}

// A block an NT x NT tile of D (or its share of the sum): while the matrix
// instructions work on one of the LDS buffers, the places that follow go from
// memory to the others without a stop in registers.  KH = 1: a wave takes a
// quarter of the tile, 32 places at a time.  KH = 2: 64 places at a time, whole
// lines; a wave takes half of the tile's columns and half of the places, which
// are a quarter fewer LDS reads, and then two waves add their halves.  A row of
// a buffer is PER 16-byte pieces, turned so that eight lanes that read one
// piece of eight rows hit different banks.  Three products of 16 cycles for
// each pair of 16 x 16 x 32 operands.
template <int NT, int KH, int BUFFERS, Ending E, typename T>
__global__ __launch_bounds__(256, 2) void k_product(
    Product pr, const int* __restrict__ active) {
  constexpr bool HALF = E == GRAM || E == POLY;
  constexpr int PLACES = 32 * KH, PER = PLACES / 8;
  constexpr int W = NT / 32, R = W * KH;  // a wave's 16-tiles: R rows of W
  constexpr int PIECES = NT * PER;        // of an operand's plane
  constexpr int LOADS = PIECES / 256;     // a thread's
  constexpr int STAGE = BUFFERS * 4 * PIECES, LAST = end_size<NT>() / 8;
  __shared__ half8 lds[STAGE > LAST ? STAGE : LAST];
  auto stage = [&](int buffer, int operand, int h) {
    return lds + ((buffer * 2 + operand) * 2 + h) * PIECES;
  };

  const Factors f = HALF && blockIdx.y ? pr.f[1] : pr.f[0];

  // each XCD takes one run of the whole tiles of the matrices there are to do,
  // and one of the shares (32 bits: divisions by 64 cost as much as a step)
  uint32_t id = blockIdx.x, count = pr.whole, splits = 1;
  const uint32_t shares = round_up((uint32_t)pr.whole, XCDS);
  const bool shared = id >= shares;
  if (shared) {
    id -= shares;
    splits = pr.splits;
    count = (pr.all - pr.whole) * splits;
  } else if (active) {
    count = min(count, (uint32_t)(active[0] * pr.tiles));
  }
  const uint32_t each = (count + XCDS - 1) / XCDS;
  if (id / XCDS >= each) return;
  id = id % XCDS * each + id / XCDS;
  if (id >= count) return;
  float* parts = pr.parts + (blockIdx.y * (int64_t)(pr.all - pr.whole) *
                                 pr.splits + id) * (NT * NT);
  uint32_t tile = id, part = 0;
  if (shared) {
    tile = id / splits;
    part = id - tile * splits;
    tile += pr.whole;
  }
  const uint32_t matrix = tile / (uint32_t)pr.tiles;
  if (active && matrix >= (uint32_t)active[0]) return;
  const int64_t b = active ? active[1 + matrix] : matrix;
  int bi, bj;
  tile_of<HALF>(tile - matrix * pr.tiles, pr.ns, pr.nl, &bi, &bj);

  const int lane = threadIdx.x % WAVE, wave = this_wave();
  const int kh = KH == 2 ? wave / 2 : 0;
  const int wi = KH == 2 ? 0 : wave / 2 * (NT / 2), wj = wave % 2 * (NT / 2);
  auto turned = [](int r, int c) { return c ^ (r * PER / 8 % PER); };
  int first = 0, steps = (pr.k + PLACES - 1) / PLACES;
  if (shared) {
    const uint32_t share = steps / splits, more = steps - share * splits;
    first = part * share + min(part, more);
    steps = share + (part < more);
  }

  const _Float16* src[2] = {
      f.a.p + b * f.a.batch + (int64_t)bi * NT * f.a.pitch + first * PLACES,
      f.b.p + b * f.b.batch + (int64_t)bj * NT * f.b.pitch + first * PLACES};
  const int64_t plane[2] = {f.a.plane, f.b.plane};
  int64_t from[2][LOADS];
#pragma unroll
  for (int l = 0; l < LOADS; ++l) {
    const int e = (l * 4 + wave) * WAVE + lane, r = e / PER;
    const int c = turned(r, e % PER) * 8;
    from[0][l] = r * f.a.pitch + c;
    from[1][l] = r * f.b.pitch + c;
  }
  auto fetch = [&](int step, int buffer) {
#pragma unroll
    for (int o = 0; o < 2; ++o)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int l = 0; l < LOADS; ++l)
          __builtin_amdgcn_global_load_lds(
              (const __attribute__((address_space(1))) void*)(
                  src[o] + h * plane[o] + from[o][l] + step * PLACES),
              (__attribute__((address_space(3))) void*)(
                  stage(buffer, o, h) + (l * 4 + wave) * WAVE),
              16, 0, 0);
  };

  f32x4 acc[R][W];
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < W; ++j) acc[i][j] = (f32x4){0, 0, 0, 0};

  // Small tiles have the registers to bring in POLY's a before the loop: the
  // ending of a block, 1.2 us of a product's 7 at 200 x 300, took 2.2 with it.
  Old<NT> old;
  if (E == POLY && NT == 64 && !shared) old.load(f.a, b, bi, bj);
#pragma unroll
  for (int p = 0; p < BUFFERS - 1; ++p)
    if (p < steps) fetch(p, p);
  int buffer = 0;
  for (int step = 0; step < steps; ++step) {
    // This step's pieces have come (a wave's loads come in order, 4 LOADS a
    // step, and those of BUFFERS - 2 later steps may still be under way), this
    // wave's reads of the step before are done, and so are everybody's.
    if (step + BUFFERS - 1 <= steps)
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier"
                   :: "n"((BUFFERS - 2) * 4 * LOADS) : "memory");
    else
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    half8 av[R][2], bv[W][2];
#pragma unroll
    for (int t = 0; t < R; ++t)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int ra = wi + t * 16 + lane % 16, rb = wj + t * 16 + lane % 16;
        const int c = kh * 4 + lane / 16;
        av[t][h] = stage(buffer, 0, h)[ra * PER + turned(ra, c)];
        if (t < W)
          bv[t % W][h] = stage(buffer, 1, h)[rb * PER + turned(rb, c)];
      }
    if (step + BUFFERS - 1 < steps)
      fetch(step + BUFFERS - 1,
            buffer ? buffer - 1 : BUFFERS - 1);
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < W; ++j) {
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
            av[i][0], bv[j][1], acc[i][j], 0, 0, 0);
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
            av[i][1], bv[j][0], acc[i][j], 0, 0, 0);
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
            av[i][0], bv[j][0], acc[i][j], 0, 0, 0);
      }
    buffer = buffer + 1 == BUFFERS ? 0 : buffer + 1;
  }

  // a wave keeps the quarter of the tile that is its number's
  f32x4 sum[W][W];
  if (KH == 2) {
    f32x4* sent = (f32x4*)lds;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < W; ++i)
#pragma unroll
      for (int j = 0; j < W; ++j) {
        sent[(wave * W + i) * W * WAVE + j * WAVE + lane] =
            kh ? acc[i][j] : acc[(W + i) % R][j];
        sum[i][j] = kh ? acc[(W + i) % R][j] : acc[i][j];
      }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < W; ++i)
#pragma unroll
      for (int j = 0; j < W; ++j)
        sum[i][j] += sent[((wave ^ 2) * W + i) * W * WAVE + j * WAVE + lane];
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i)
#pragma unroll
      for (int j = 0; j < W; ++j) sum[i][j] = acc[i][j];
  }

  if (shared) {
#pragma unroll
    for (int i = 0; i < W; ++i)
#pragma unroll
      for (int j = 0; j < W; ++j)
        ((f32x4*)parts)[(i * W + j) * 256 + threadIdx.x] = sum[i][j];
    return;
  }
  if (E == POLY && NT != 64) old.load(f.a, b, bi, bj);
  end_product<NT, E, T>(pr, f, b, bi, bj, sum, old, (_Float16*)lds);
}

// The tiles whose sum was shared out: its parts, in their order.
template <int NT, Ending E, typename T>
__global__ __launch_bounds__(256) void k_join(
    Product pr, const int* __restrict__ active) {
  constexpr int W = NT / 32;
  __shared__ half8 lds[end_size<NT>() / 8];
  const uint32_t tile = pr.whole + blockIdx.x;
  const uint32_t matrix = tile / (uint32_t)pr.tiles;
  if (active && matrix >= (uint32_t)active[0]) return;
  const int64_t b = active ? active[1 + matrix] : matrix;
  int bi, bj;
  tile_of<E == GRAM || E == POLY>(tile - matrix * pr.tiles, pr.ns, pr.nl, &bi,
                                  &bj);
  const Factors& f = pr.f[blockIdx.y];
  const f32x4* parts = (const f32x4*)pr.parts +
                       ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) *
                           pr.splits * (W * W * 256);
  f32x4 acc[W][W];
#pragma unroll
  for (int i = 0; i < W; ++i)
#pragma unroll
    for (int j = 0; j < W; ++j) acc[i][j] = parts[(i * W + j) * 256 +
                                                  threadIdx.x];
  for (int q = 1; q < pr.splits; ++q)
#pragma unroll
    for (int i = 0; i < W; ++i)
#pragma unroll
      for (int j = 0; j < W; ++j)
        acc[i][j] += parts[((q * W + i) * W + j) * 256 + threadIdx.x];
  Old<NT> old;
  if (E == POLY) old.load(f.a, b, bi, bj);
  end_product<NT, E, T>(pr, f, b, bi, bj, acc, old, (_Float16*)lds);
}

// ---------------------------------------------------------------------
// host
// ---------------------------------------------------------------------

struct Chain {
  const void* u;
  at::ScalarType type;
  int64_t batch, m, n;
  const int* touched;
  const int* active;  // how many are touched, and which
  int steps;
  Coeffs k;
  double eps;
  Result res;
  at::TensorOptions options;
  hipStream_t stream;
  bool thin = false;
  // Muon: U comes from these; with `fused` the pass that sums G makes it,
  // without it is there
  bool fused = false;
  Momentum momentum{};
  const int64_t* place = nullptr;
};

// Thin touches the values twice and takes some 14 small products in f64, which
// wait for each other: their time is that of their launches while batch * s is
// small and that of the f64 units, batch * s^3, above.  Wide takes three
// products over the values a step, batch * s^2 * long.  So thin is the faster
// one from a ratio long / s that is small (3) while the products fill few CUs
// and large (16) where they fill the card; s * s in f64 has to fit its kernels
// (THIN_MAX).  Measured, thin against wide.  f32: 1 x 128 x 512 82 us, 98; 1 x 200 x 600
// 104, 118; 1 x 256 x 512 115, 111; 1 x 320 x 1280 137, 162; of many matrices
// the small products take longer: 4 x 200 x 800 147, 130; 16 x 128 x 1024 158,
// 141; 8 x 200 x 3200 225, 246; 16 x 128 x 2048 164, 193.  bfloat16, whose wide
// chain takes steps on G too: 1 x 200 x 600 108, 116; 2 x 200 x 1600 133, 137;
// 1 x 256 x 1024 133, 123; 1 x 256 x 4096 134, 140; 1 x 320 x 5120 172, 158;
// 2 x 256 x 4096 168, 146; 16 x 200 x 6400 553, 402
bool is_thin(at::ScalarType type, int64_t batch, int64_t m, int64_t n) {
  const int64_t s = std::min(m, n), long_ = std::max(m, n);
  if (s <= NARROW) return true;
  if (type == at::kBFloat16)
    return s <= 256 && batch * s <= 448 && long_ >= (s <= 224 ? 3 : 8) * s;
  return s <= THIN_MAX && long_ >= (batch * s <= 512 ? 3 : 16) * s;
}

// How far P's values can reach: its value at singular values from 0 to 1.
struct Reach {
  double x[257], p[257];
  Reach() {
    for (int i = 0; i < 257; ++i) x[i] = i / 256.0;
    start();
  }
  void start() {
    for (double& v : p) v = 1.0;
  }
  // a step; how much it multiplies by at most
  double step(const Coeffs& k) {
    double top = 0;
    for (int i = 0; i < 257; ++i) {
      const double y = x[i] * x[i], q = k.a + k.b * y + k.c * y * y;
      p[i] *= q;
      x[i] *= q;
      top = std::max(top, std::abs(q));
    }
    return top;
  }
  // the power of two that keeps P under 4, up to what lies between the points
  float hold() const {
    double top = 0;
    for (double v : p) top = std::max(top, std::abs(v));
    return top > 4 ? (float)std::exp2(-std::ceil(std::log2(top / 4))) : 1.0f;
  }
};

// By how many powers of two the first i steps multiply a value at most.
std::vector<int> growth(const Coeffs& k, int steps) {
  Reach reach;
  std::vector<int> g{0};
  double power = 0;
  for (int i = 0; i < steps; ++i) {
    power += std::log2(std::max(reach.step(k), 0x1p-20));
    g.push_back((int)std::ceil(power));
  }
  return g;
}

template <typename T, bool TALL>
void run_thin(const Chain& c) {
  const int s = std::min(c.m, c.n);
  const int64_t long_ = std::max(c.m, c.n);
  const bool narrow = s <= NARROW;
  const int nt = !narrow ? (s + 15) / 16 : s <= 16 ? 1 : s <= 32 ? 2 : 4;
  const int sp = nt * 16;
  // blocks of G's squares: one on the diagonal, two under it
  const int super = (s + SUPER - 1) / SUPER, squares = super * super;
  // chunks: about two blocks a CU (four where a block needs little), of at
  // least 64 places (16 a wave) or KC
  const int64_t least = narrow ? 64 : KC;
  int64_t chunks = std::min<int64_t>(
      (long_ + least - 1) / least,
      std::max<int64_t>(1, narrow ? 1024 / c.batch
                                  : 512 / (c.batch * squares)));
  const int64_t chunk = round_up((long_ + chunks - 1) / chunks, least);
  chunks = (long_ + chunk - 1) / chunk;
  const int64_t size = narrow ? nt * (nt + 1) / 2 * 256 : (int64_t)sp * sp;
  // the planes of P: JT * 16 rows a block
  const int jt = s <= 32 ? 2 : s <= 64 || s > 128 ? 4 : 8;
  const int jp = round_up(s, jt * 16), kp = round_up(s, 32);
  Reach reach;
  for (int i = 0; i < c.steps; ++i) reach.step(c.k);
  const double by = UP * reach.hold();
  auto f64 = c.options.dtype(at::kDouble);
  auto part = at::empty({c.batch * chunks * size}, f64);
  auto pl = at::empty({2 * c.batch * jp * kp}, c.options.dtype(at::kHalf));
  auto nm = at::empty({c.batch * 3}, c.options.dtype(at::kFloat));
  _Float16* planes = (_Float16*)pl.data_ptr();
  Norm* norm = (Norm*)nm.data_ptr();
  double* parts = part.data_ptr<double>();
  at::Tensor work;
  if (narrow) {
    auto go = [&](auto* gram, auto* chain, int threads) {
      hipLaunchKernelGGL(gram, dim3(chunks, c.batch), dim3(256), 0, c.stream,
                         parts, (const T*)c.u, c.touched, long_, s, chunk);
      // one block would take longer over many parts than another kernel does
      if (chunks * size > 131072) {
        work = at::empty({c.batch * size}, f64);
        hipLaunchKernelGGL(k_part_sum, dim3(size / 16, c.batch), dim3(256), 0,
                           c.stream, work.data_ptr<double>(), parts,
                           c.touched, (int)chunks, size);
        parts = work.data_ptr<double>();
        chunks = 1;
      }
      hipLaunchKernelGGL(chain, dim3(c.batch), dim3(threads), 0, c.stream,
                         planes, norm, parts, c.touched, (int)chunks, s,
                         c.steps, c.k, c.eps, jp, kp, by);
    };
    if (nt == 1) go(k_gram_narrow<T, TALL, 1>, k_chain<1, 4>, 256);
    else if (nt == 2) go(k_gram_narrow<T, TALL, 2>, k_chain<2, 16>, 1024);
    else go(k_gram_narrow<T, TALL, 4>, k_chain<4, 16>, 1024);
  } else {
    auto tr = at::empty({c.batch * chunks * super}, f64);
    work = at::empty({6, c.batch * size}, f64);
    double* w[6];
    for (int i = 0; i < 6; ++i)
      w[i] = work.data_ptr<double>() + i * c.batch * size;
    auto gram = [&](auto* kfn, const Momentum& q, const int64_t* place) {
      hipLaunchKernelGGL(kfn, dim3(chunks, squares, c.batch), dim3(256), 0,
                         c.stream, parts, tr.data_ptr<double>(),
                         (const T*)c.u, q, place, c.touched, long_, s, sp,
                         chunk);
    };
    if constexpr (TALL && std::is_same_v<T, float>) {
      if (c.fused) gram(k_gram64<T, TALL, true>, c.momentum, c.place);
      else gram(k_gram64<T, TALL, false>, {}, nullptr);
    } else {
      gram(k_gram64<T, TALL, false>, {}, nullptr);
    }
    double *g = w[0], *q = w[1], *p = w[2], *t = w[3], *g2 = w[4], *p2 = w[5];
    hipLaunchKernelGGL(k_gram_sum, dim3(size / 16, c.batch),
                       dim3(256), 0, c.stream, g, norm, parts,
                       tr.data_ptr<double>(), c.touched, (int)chunks, sp,
                       c.eps);
    auto mul = [&](SmallMul j0, SmallMul j1, int jobs) {
      hipLaunchKernelGGL(k_small_mul, dim3(nt * (nt + 1) / 2, c.batch, jobs),
                         dim3(256), 0, c.stream, j0, j1, c.touched, s, sp,
                         c.k);
    };
    for (int i = 0; i < c.steps; ++i) {
      // Q from G; P <- P Q (the first P is Q); G <- Q (G Q)
      const bool last = i + 1 == c.steps;
      double* qi = i == 0 ? p : q;
      mul({qi, g, g, true}, {}, 1);
      if (i == 0 && !last) mul({t, g, qi, false}, {}, 1);
      if (i > 0) mul({p2, p, q, false}, {t, g, qi, false}, last ? 1 : 2);
      if (!last) {
        mul({g2, qi, t, false}, {}, 1);
        std::swap(g, g2);
      }
      if (i > 0) std::swap(p, p2);
    }
    hipLaunchKernelGGL(k_small_out, dim3((jp * kp + 255) / 256, c.batch),
                       dim3(256), 0, c.stream, planes, p, c.touched, s, sp, jp,
                       kp, by);
  }
  // a few turns a block, so that P's planes come in once for them
  auto apply = [&](auto* kfn, int waves, int most) {
    const int turn = waves * 16 * (TALL ? 2 : 4);
    const dim3 grid(std::min<int64_t>((long_ + turn - 1) / turn, most),
                    jp / (jt * 16), c.batch);
    hipLaunchKernelGGL(kfn, grid, dim3(waves * WAVE), 0, c.stream, c.res,
                       (const T*)c.u, planes, norm, c.touched, long_, s, jp,
                       kp, (float)(1.0 / (UP * by)));
  };
  if (s <= 32) apply(k_thin_apply<T, TALL, 2, 32, 4>, 4, 2048);
  else if (s <= 64) apply(k_thin_apply<T, TALL, 4, 64, 4>, 4, 2048);
  else if (s <= 128) apply(k_thin_apply<T, TALL, 8, 128, 4>, 4, 2048);
  else apply(k_thin_apply<T, TALL, 4, 320, 8>, 8, 256);
}

// Tiles of one product, and how many blocks share the sum of those after the
// first `whole`.
struct Cut {
  int tile, ns, nl, tiles, splits;
  int64_t all, whole;
};

// 128 x 128 tiles where they give every CU one, else 64 x 64.  Two blocks fit
// a CU: tiles that are left over after a number of full rounds would keep the
// card for a round of their own, so their sums are shared out, as are those of
// all tiles where there are too few.  A share is `least` steps of 32 places:
// what the join costs is about that.
Cut cut_of(int64_t rows, int64_t cols, bool half, int64_t batch, int64_t k) {
  constexpr int64_t ROUND = 512;
  Cut c{};
  for (c.tile = 128;; c.tile = 64) {
    c.ns = (rows + c.tile - 1) / c.tile;
    c.nl = (cols + c.tile - 1) / c.tile;
    c.tiles = half ? c.ns * (c.ns + 1) / 2 : c.ns * c.nl;
    c.all = c.tiles * batch;
    if (c.tile == 64 || c.all >= ROUND / 2) break;
  }
  const int64_t least = c.tile == 128 ? 16 : 32;
  const int64_t rest = c.all % ROUND, steps = round_up(k, 32) / 32;
  c.splits = 1;
  c.whole = c.all;
  if (rest && rest <= ROUND / 2 && c.all < 8 * ROUND && steps >= 2 * least) {
    c.splits = std::min(ROUND / rest, steps / least);
    c.whole = c.all - rest;
  }
  return c;
}

template <Ending E, typename T>
void run_product(const Chain& c, Product pr, const Cut& cut, int jobs = 1) {
  pr.ns = cut.ns;
  pr.nl = cut.nl;
  pr.tiles = cut.tiles;
  pr.all = cut.all;
  pr.whole = cut.whole;
  pr.splits = cut.splits;
  const int64_t rest = cut.all - cut.whole;
  const dim3 grid(round_up(cut.whole, XCDS) +
                      round_up(rest * cut.splits, XCDS),
                  jobs);
  auto go = [&](auto* kfn, auto* join) {
    hipLaunchKernelGGL(kfn, grid, dim3(256), 0, c.stream, pr, c.active);
    if (rest)
      hipLaunchKernelGGL(join, dim3(rest, jobs), dim3(256), 0, c.stream, pr,
                         c.active);
  };
  // Of small tiles, two blocks on a CU wait for LDS and one for its loads: it
  // needs them further ahead than buffers of 64 places reach.  Measured, KH = 2
  // against 1: 12 x 512 x 1024 340 us, 362; 1500 x 2048 477, 544; 3 x 300 x
  // 1001 178, 159; 200 x 300 116, 104
  const int64_t blocks = (cut.whole + rest * cut.splits) * jobs;
  if (cut.tile == 128) go(k_product<128, 1, 2, E, T>, k_join<128, E, T>);
  else if (blocks > 256) go(k_product<64, 2, 2, E, T>, k_join<64, E, T>);
  else go(k_product<64, 1, 4, E, T>, k_join<64, E, T>);
}

// How many steps in a row are taken on the Gram matrix before P is applied to
// X; 1 for none.  With L = r s a step costs 3 r + 1 products of s^3 on X, and n
// in a row cost 3 r + 4 n - 3.  What G is off grows by q^2 with every step: n is
// bounded so that it does so by 200 in all (three of Muon's).  Before it is
// rounded the result of five is then 3e-6 (singular values alike) to 2e-4 off
// (all values equal), where steps on X leave 2e-6 and 1e-5: at most an eighth of
// bfloat16's rounding, which is 1.7e-3, but too much for the other types.
// Measured: 8 x 512 x 2048 303 us, on X 424.
template <typename T>
int steps_on_gram(const Chain& c, int64_t s, int64_t long_) {
  if (!std::is_same_v<T, __hip_bfloat16> || long_ * 2 < s * 3) return 1;
  Reach reach;
  int n = 0;
  for (double power = 1.0, sum = 0.0; n < c.steps; ++n) {
    if ((sum += power) > 200.0) break;
    const double q = reach.step(c.k);
    power *= q * q;
  }
  return std::max(n, 1);
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
  const int parts = (int)std::min<int64_t>(
      std::max<int64_t>(1, 1024 / c.batch), (c.m * c.n + 4095) / 4096);
  auto part = at::empty({c.batch * parts}, c.options.dtype(at::kDouble));
  auto small = at::empty({c.batch}, c.options.dtype(at::kInt));
  hipLaunchKernelGGL(k_sumsq<T>, dim3(parts, c.batch), dim3(256), 0, c.stream,
                     part.data_ptr<double>(), (const T*)c.u, c.touched,
                     c.m * c.n);
  hipLaunchKernelGGL(k_planes<T>, dim3(np / 64 * (mp / 64), 1, c.batch),
                     dim3(256), 0, c.stream, nat, trn, small.data_ptr<int>(),
                     (const T*)c.u, part.data_ptr<double>(), parts, c.touched, c.m, c.n,
                     c.eps);
  const int64_t long_ = std::max(c.m, c.n);
  const Cut gram = cut_of(s, s, true, c.batch, long_);
  const Cut poly = cut_of(s, s, true, c.batch, s);
  const Cut full = cut_of(s, long_, false, c.batch, s);
  int64_t shared = 0;
  for (const Cut& cut : {gram, poly, full})
    shared = std::max(shared, (cut.all - cut.whole) * cut.splits * cut.tile *
                                  cut.tile);
  auto sums = at::empty({2 * shared}, c.options.dtype(at::kFloat));
  Product pr{};
  pr.e.small = small.data_ptr<int>();
  const std::vector<int> grown = growth(c.k, c.steps);
  pr.ca = (float)c.k.a;
  pr.cb = (float)c.k.b;
  pr.cc = (float)c.k.c;
  pr.s = s;
  pr.rows = s;
  pr.cols = long_;
  pr.tall = tall;
  pr.res = c.res;
  pr.parts = sums.data_ptr<float>();
  const int ks = round_up(s, 32), kl = round_up(long_, 32);
  const float down = 1.0f / UP;
  auto square = [&] { return planes(sp, sp); };
  auto again = [&] { return tall ? planes(mp, np) : planes(np, mp); };
  Planes g = square(), q = square(), xt2{};

  auto new_gram = [&](int done) {
    pr.f[0] = {x, x, g, down};
    pr.k = kl;
    pr.e.grown = grown[done];
    pr.e.times = 2;
    run_product<GRAM, T>(c, pr, gram);
    pr.e.times = 0;
    pr.k = ks;
  };
  auto new_poly = [&](Planes to) {
    pr.f[0] = {g, g, to, down};
    run_product<POLY, T>(c, pr, poly);
  };
  // X <- (by / held) X, after `to` steps, the last time as the result
  auto apply = [&](Planes by, float held, int to) {
    pr.e.times = 1;
    if (to == c.steps) {
      pr.f[0] = {by, xt, x, down * down / held};
      run_product<FINAL, T>(c, pr, full);
      return;
    }
    if (!xt2.p) xt2 = again();
    pr.f[0] = {by, xt, x, down / held};
    pr.dt = xt2;
    pr.e.next = grown[to];
    run_product<UPDATE, T>(c, pr, full);
    std::swap(xt, xt2);
  };

  const int row = steps_on_gram<T>(c, s, long_);
  if (row == 1) {
    for (int i = 0; i < c.steps; ++i) {
      new_gram(i);
      new_poly(q);
      apply(q, 1.0f, i + 1);
    }
    return;
  }
  // Q from G; P <- P Q (the first P is Q); G <- Q (G Q)
  Planes p = square(), p2 = square(), t = square(), g2 = square();
  Reach reach;
  for (int done = 0; done < c.steps;) {
    const int todo = std::min(row, c.steps - done);
    float held = 1.0f;  // P's planes hold P times this
    reach.start();
    new_gram(done);
    for (int i = 0; i < todo; ++i) {
      const bool last = i + 1 == todo;
      const Planes qi = i ? q : p;
      new_poly(qi);
      reach.step(c.k);
      if (i) {
        const float to = reach.hold();
        pr.f[0] = {p, q, p2, down * (to / held)};
        held = to;
        pr.f[1] = {g, q, t, down};
        run_product<GRAM, T>(c, pr, poly, last ? 1 : 2);
        std::swap(p, p2);
      } else if (!last) {
        pr.f[0] = {g, qi, t, down};
        run_product<GRAM, T>(c, pr, poly);
      }
      if (!last) {
        pr.f[0] = {qi, t, g2, down};
        run_product<GRAM, T>(c, pr, poly);
        std::swap(g, g2);
      }
    }
    done += todo;
    apply(p, held, done);
  }
}

template <typename T>
void thin(const Chain& c) {
  if (c.m >= c.n) run_thin<T, true>(c); else run_thin<T, false>(c);
}

// P's planes hold 40 bits from its largest value down, and the values that
// matter are near one: steps are taken in one round while P does not reach
// beyond 2^11 (six of Muon's).
int thin_round(const Coeffs& k, int steps) {
  Reach reach;
  int n = 0;
  while (n < steps) {
    reach.step(k);
    if (n && reach.hold() < 0x1p-9f) break;
    ++n;
  }
  return n;
}

template <typename T>
void run(const Chain& c) {
  if (!c.thin) {
    run_wide<T>(c);
    return;
  }
  const int most = thin_round(c.k, c.steps);
  if (most == c.steps) {
    thin<T>(c);
    return;
  }
  // several rounds, with X in f32 between
  TORCH_CHECK((std::is_same_v<T, float>), "rounds are taken in f32");
  Chain round = c;
  at::Tensor x, next;
  for (int done = 0; done < c.steps; done += most) {
    round.steps = std::min(most, c.steps - done);
    next = at::Tensor();
    if (done + most < c.steps) {
      next = at::empty({c.batch * c.m * c.n}, c.options.dtype(at::kFloat));
      round.res = {next.data_ptr(), 0, 0, false};
    } else {
      round.res = c.res;
    }
    thin<T>(round);
    x = next;
    if (x.defined()) round.u = x.data_ptr();
    round.fused = false;
    round.eps = -1.0;  // U is X already
  }
}

void dispatch(const Chain& whole) {
  // grids hold 65535 matrices; all of them take the same route
  const bool thin = is_thin(whole.type, whole.batch, whole.m, whole.n);
  for (int64_t b = 0; b < whole.batch; b += 32768) {
    Chain c = whole;
    c.thin = thin;
    const int64_t size = c.m * c.n * b;
    c.batch = std::min<int64_t>(32768, whole.batch - b);
    c.u = (const char*)c.u + size * c10::elementSize(c.type);
    c.res.out = (char*)c.res.out +
                size * (c.res.step ? 4 : c10::elementSize(c.type));
    at::Tensor active;
    if (c.touched) {
      c.touched += b;
      if (!c.thin) {
        active = at::empty({c.batch + 1}, c.options.dtype(at::kInt));
        c.active = active.data_ptr<int>();
        hipLaunchKernelGGL(k_active, dim3(1), dim3(1024), 0, c.stream,
                           active.data_ptr<int>(), c.touched, (int)c.batch);
      }
    }
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
  if (type != at::kFloat && is_thin(type, x.size(0), x.size(1), x.size(2)) &&
      thin_round({a, b, c}, steps) < steps)
    return orthogonalize(x.to(at::kFloat), steps, a, b, c, eps).to(type);
  dispatch(Chain{x.data_ptr(), type, x.size(0), x.size(1), x.size(2), nullptr,
                 nullptr, (int)steps, {a, b, c}, eps, {out.data_ptr(), 0, 0, false},
                 x.options(), at::hip::getCurrentHIPStream().stream()});
  return out;
}

void apply_muon(at::Tensor table, at::Tensor momentum, at::Tensor rows,
                bool sorted_unique, at::Tensor grads, double lr,
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
  TORCH_CHECK(matrix_rows >= 1 && table.size(0) % matrix_rows == 0,
              "the table is not a whole number of matrices of ", matrix_rows,
              " rows");
  check_chain(matrix_rows, dim, steps);
  const int64_t batch = table.size(0) / matrix_rows;
  if (!n || !table.numel()) return;
  const int64_t total = table.size(0);
  c10::DeviceGuard guard(table.device());
  hipStream_t stream = at::hip::getCurrentHIPStream().stream();
  // Blocks that each read the whole push, against a sort and k_places (the
  // whole step): 5000 places and 16 windows 41 us, 78; 9000 and 48 417, 441;
  // 16000 and 1 (all of them in it) 97, 153; 16000 and 1024 65, 85.  A sort
  // clears memory in ways that a graph does not repeat: none is captured.
  const int64_t windows = batch * ((matrix_rows + 255) / 256);
  hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
  TORCH_CHECK(hipStreamIsCapturing(stream, &capture) == hipSuccess,
              "the stream cannot be asked whether it is captured");
  const bool captured = capture != hipStreamCaptureStatusNone;
  const bool any = !sorted_unique && n <= SHORT &&
                   (windows <= 1024 || (captured && windows <= 1 << 20));
  TORCH_CHECK(sorted_unique || any || !captured, "a push in any order of "
              "more than ", SHORT, " rows, or into a table of more than ",
              1 << 20, " windows (256 rows of a matrix or what is left of "
              "one), cannot be captured");
  auto touched = at::empty({batch}, table.options().dtype(at::kInt));
  auto u = at::empty_like(table);
  auto place = at::empty({total}, rows.options());
  at::Tensor order;
  int64_t* at_ = place.data_ptr<int64_t>();
  if (any) {
    const auto push = rows;
    rows = at::empty_like(push);
    order = at::empty_like(push);
    hipLaunchKernelGGL(k_places_any, dim3(windows), dim3(256), 0, stream, at_,
                       touched.data_ptr<int>(), rows.data_ptr<int64_t>(),
                       order.data_ptr<int64_t>(), push.data_ptr<int64_t>(),
                       (int)n, matrix_rows, total);
  } else {
    if (!sorted_unique)
      std::tie(rows, order) = at::sort(rows, /*stable=*/true, 0, false);
    hipLaunchKernelGGL(k_places, dim3(std::min<int64_t>(windows, 1 << 20)),
                       dim3(256), 0, stream, at_, touched.data_ptr<int>(),
                       rows.data_ptr<int64_t>(),
                       order.defined() ? order.data_ptr<int64_t>() : nullptr,
                       n, matrix_rows, windows);
  }
  Momentum q{u.data_ptr<float>(),       momentum.data_ptr<float>(),
             grads.data_ptr<float>(),   rows.data_ptr<int64_t>(),
             order.defined() ? order.data_ptr<int64_t>() : nullptr,
             nullptr,                   n,
             (float)mu,                 nesterov};
  at::Tensor sums;
  if (!sorted_unique && n > LONG) {
    const int64_t chunks = (n + LONG - 1) / LONG;
    sums = at::empty({chunks * dim}, table.options());
    q.sums = (const float*)((uintptr_t)sums.data_ptr<float>() -
                            (uintptr_t)(n * dim) * sizeof(float));
    auto go = [&](auto* kfn, int width) {
      const dim3 grid(std::min<int64_t>(chunks, 1 << 20),
                      std::min<int64_t>((dim + width - 1) / width, 65535));
      hipLaunchKernelGGL(kfn, grid, dim3(256), 0, stream,
                         sums.data_ptr<float>(), at_, q, total, dim);
    };
    if (dim <= 16) go(k_long_runs<16>, 16);
    else if (dim <= 32) go(k_long_runs<32>, 32);
    else go(k_long_runs<64>, 64);
  }
  // one pass makes U and sums G where a block holds a row and a square of G
  const bool fused = is_thin(at::kFloat, batch, matrix_rows, dim) && dim > NARROW &&
                     dim <= SUPER && matrix_rows >= dim && batch <= 32768;
  if (!fused) {
    int group = 1;
    while (group < 64 && group * 4 < dim) group *= 2;
    const int64_t blocks = (total * group + 255) / 256;
    hipLaunchKernelGGL(k_momentum, dim3(std::min<int64_t>(blocks, 8192)),
                       dim3(256), 0, stream, q, place.data_ptr<int64_t>(),
                       touched.data_ptr<int>(), total, matrix_rows, (int)dim,
                       group);
  }
  const double rate = lr * std::sqrt(std::max(1.0, (double)matrix_rows / dim));
  Chain chain{u.data_ptr(), at::kFloat, batch, matrix_rows, dim,
              touched.data_ptr<int>(), nullptr, (int)steps, {a, b, c}, eps,
              {table.data_ptr(), (float)(1.0 - lr * weight_decay),
               (float)rate, true},
              table.options(), stream};
  chain.fused = fused;
  chain.momentum = q;
  chain.place = place.data_ptr<int64_t>();
  dispatch(chain);
}
