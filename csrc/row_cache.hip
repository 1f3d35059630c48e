// 8-bit row records for MI355X (gfx950): rows are quantised as they are
// written into a cache and read back as values.
//
// A record of a row x of dim values is
//     [code: 1 byte x dim][zeros to a multiple of 4][scale: f32]
// and stands for code * scale.  With amax = max |x_j|:
//   int8  scale = RN(amax / 127) between 2^-126 and INT8_TOP,
//         code = RNE(x / scale)
//   fp8   scale = the smallest power of two >= 2^-126 with
//         amax <= 448 * scale,  code = e4m3(x / scale), nearest even,
//         |x| counted as FP8_TOP at most
// Both codes are the exact quotient's, so any two implementations agree on
// every byte.  A row that holds an infinity or NaN gets a NaN scale and zero
// codes: it reads back as NaN throughout and never as finite values.
//
// Slots outside [0, rows) are padding: not written, read back as zeros.

#include <ATen/ATen.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <type_traits>

#include "ops.h"
#include "quads.h"

namespace {

constexpr int WAVE = 64;
constexpr float TINY = 0x1p-126f;  // the smallest normal f32
constexpr float FP8_TOP = 0x1.ep+127f;  // 240 * 2^120: the next code is 2^128
// The largest scale whose code 127 is finite; RN(FLT_MAX / 127) is one ulp up.
constexpr float INT8_TOP = 0x1.020406p+121f;

// int64, int32 or no slots (row j's is j)
struct Slots {
  const void* at;
  bool wide;
  __device__ inline int64_t operator[](int64_t j) const {
    if (!at) return j;
    return wide ? ((const int64_t*)at)[j] : ((const int32_t*)at)[j];
  }
};

// |x| as an ordered integer: finite < inf < NaN, so the largest one of a
// row also says whether the row is finite.
__device__ inline uint32_t magnitude(float x) {
  return __float_as_uint(x) & 0x7fffffffu;
}

struct Scale { float s, inv; };  // inv is 1 / s: fp8 exactly, int8 nearly

template <bool FP8>
__device__ inline Scale scale_of(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return {__uint_as_float(0x7fc00000u), 0.0f};
  const float amax = __uint_as_float(amax_bits);
  if (!FP8) {
    // amax / 127: the product with the rounded reciprocal is off by an ulp at
    // most, its remainder is exact, and one fma rounds the sum correctly
    constexpr float y = 1.0f / 127.0f;
    const float q = amax * y;
    const float s = fminf(fmaxf(fmaf(fmaf(-127.0f, q, amax), y, q), TINY),
                          INT8_TOP);
    return {s, __builtin_amdgcn_rcpf(s)};
  }
  // 448 = 1.75 * 2^8: with amax = m * 2^e, 1 <= m < 2, the exponent is
  // e - 8 while m <= 1.75 and e - 7 above.  (Subnormal: the 2^-126 floor.)
  int e = (int)(amax_bits >> 23) - 127;
  int k = (amax_bits & 0x7fffffu) <= 0x600000u ? e - 8 : e - 7;
  if (k < -126) k = -126;
  return {__uint_as_float((uint32_t)(k + 127) << 23),
          __uint_as_float((uint32_t)(127 - k) << 23)};
}

// Nearest integer to the exact quotient x / s, ties to even, from q, which is
// off by one at most: the remainder x - q s is exact in one fma (a multiple of
// ulp(s) / 2 no larger than s) and says which way.
__device__ inline float nearest(float q, float x, float s) {
  const float r = fmaf(-q, s, x), twice = 2.0f * fabsf(r);
  const bool odd = ((int)q) & 1;
  return twice > s || (twice == s && odd) ? q + copysignf(1.0f, r) : q;
}

// x * inv is off the quotient by 2^-15 at most (inv by an ulp, the product by
// half of one, 2^7 steps), so only values that near to a half need the
// remainder.
__device__ inline uint32_t codes_int8(float4 f, float s, float inv) {
  float4 y = make_float4(f.x * inv, f.y * inv, f.z * inv, f.w * inv);
  float4 q = make_float4(rintf(y.x), rintf(y.y), rintf(y.z), rintf(y.w));
  const float off = fmaxf(fmaxf(fabsf(y.x - q.x), fabsf(y.y - q.y)),
                          fmaxf(fabsf(y.z - q.z), fabsf(y.w - q.w)));
  if (off > 0.4999f)
    q = make_float4(nearest(q.x, f.x, s), nearest(q.y, f.y, s),
                    nearest(q.z, f.z, s), nearest(q.w, f.w, s));
  return (uint32_t)((int)q.x & 255) | (uint32_t)((int)q.y & 255) << 8 |
         (uint32_t)((int)q.z & 255) << 16 | (uint32_t)(int)q.w << 24;
}

__device__ inline uint32_t quad_magnitude(float4 f) {
  return max(max(magnitude(f.x), magnitude(f.y)),
             max(magnitude(f.z), magnitude(f.w)));
}

__device__ inline uint32_t group_max(uint32_t v, int group) {
  for (int o = group / 2; o; o >>= 1)
    v = max(v, (uint32_t)__shfl_xor((int)v, o));
  return v;
}

template <bool FP8>
__device__ inline uint32_t encode(float4 f, Scale sc) {
  const float s = sc.s, inv = sc.inv;
  if (s != s) return 0;  // the row is not finite
  if (FP8) {
    auto part = [&](float x) {
      return __builtin_amdgcn_fmed3f(x, -FP8_TOP, FP8_TOP) * inv;
    };
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(part(f.x), part(f.y), 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(part(f.z), part(f.w), w,
                                                     true);
  }
  return codes_int8(f, s, inv);
}

template <bool FP8>
__device__ inline float4 decode(uint32_t w, float s) {
  if (FP8)
    return make_float4(__builtin_amdgcn_cvt_f32_fp8((int)w, 0) * s,
                       __builtin_amdgcn_cvt_f32_fp8((int)w, 1) * s,
                       __builtin_amdgcn_cvt_f32_fp8((int)w, 2) * s,
                       __builtin_amdgcn_cvt_f32_fp8((int)w, 3) * s);
  return make_float4((float)(int8_t)w * s, (float)(int8_t)(w >> 8) * s,
                     (float)(int8_t)(w >> 16) * s,
                     (float)(int8_t)(w >> 24) * s);
}

// The last of the writes to a slot wins, whatever the order that they run in.
__global__ __launch_bounds__(256) void k_cache_owner(int* __restrict__ owner,
                                                     Slots slots, int64_t n,
                                                     int64_t rows) {
  for (int64_t j = (int64_t)blockIdx.x * 256 + threadIdx.x; j < n;
       j += (int64_t)gridDim.x * 256) {
    int64_t s = slots[j];
    if (s >= 0 && s < rows) atomicMax(owner + s, (int)j);
  }
}

// `group` lanes (a power of two) take ROWS rows at a time; a lane holds QUADS
// quads of each in registers, so that the values are read once, and all the
// loads of a turn are under way before the first is used.
template <typename T, bool FP8, int QUADS, int ROWS>
__global__ __launch_bounds__(256) void k_cache_write(
    uint8_t* __restrict__ cache, int64_t cache_stride,
    const T* __restrict__ values, int64_t value_stride, Slots slots,
    const int* __restrict__ owner, int64_t n, int dim, int64_t rows,
    int group) {
  const int lane = threadIdx.x & (group - 1);
  const int per_block = 256 / group;
  const int quads = (dim + 3) / 4;
  for (int64_t j0 = ((int64_t)blockIdx.x * per_block + threadIdx.x / group) *
                    ROWS;
       j0 < n; j0 += (int64_t)gridDim.x * per_block * ROWS) {
    int64_t slot[ROWS];
    float4 x[ROWS][QUADS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      slot[r] = j0 + r < n ? slots[j0 + r] : -1;
      if (slot[r] >= rows) slot[r] = -1;
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      if (owner && slot[r] >= 0 && owner[slot[r]] != (int)(j0 + r))
        slot[r] = -1;
#pragma unroll
      for (int i = 0; i < QUADS; ++i) {
        const int q = lane + i * group;
        x[r][i] = load_quad(values + (j0 + r) * value_stride + q * 4,
                            slot[r] < 0 ? 0 : dim - q * 4);
      }
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < QUADS; ++i) top = max(top, quad_magnitude(x[r][i]));
      const Scale s = scale_of<FP8>(group_max(top, group));
      if (slot[r] < 0) continue;
      uint32_t* out = (uint32_t*)(cache + slot[r] * cache_stride);
#pragma unroll
      for (int i = 0; i < QUADS; ++i) {
        const int q = lane + i * group;
        if (q < quads) out[q] = encode<FP8>(x[r][i], s);
      }
      if (lane == 0) out[quads] = __float_as_uint(s.s);
    }
  }
}

// Rows too long for registers: a wave a row, which it reads twice.
template <typename T, bool FP8>
__global__ __launch_bounds__(256) void k_cache_write_long(
    uint8_t* __restrict__ cache, int64_t cache_stride,
    const T* __restrict__ values, int64_t value_stride, Slots slots,
    const int* __restrict__ owner, int64_t n, int64_t dim, int64_t rows) {
  const int lane = threadIdx.x % WAVE;
  const int64_t quads = (dim + 3) / 4;
  for (int64_t j = (int64_t)blockIdx.x * 4 + threadIdx.x / WAVE; j < n;
       j += (int64_t)gridDim.x * 4) {
    const int64_t slot = slots[j];
    if (slot < 0 || slot >= rows) continue;
    if (owner && owner[slot] != (int)j) continue;
    const T* x = values + j * value_stride;
    uint32_t* out = (uint32_t*)(cache + slot * cache_stride);
    uint32_t top = 0;
    for (int64_t q = lane; q < quads; q += WAVE)
      top = max(top, quad_magnitude(load_quad(x + q * 4, dim - q * 4)));
    const Scale s = scale_of<FP8>(group_max(top, WAVE));
    for (int64_t q = lane; q < quads; q += WAVE)
      out[q] = encode<FP8>(load_quad(x + q * 4, dim - q * 4), s);
    if (lane == 0) out[quads] = __float_as_uint(s.s);
  }
}

template <typename T, bool FP8, int QUADS, int ROWS>
__global__ __launch_bounds__(256) void k_cache_read(
    T* __restrict__ out, const uint8_t* __restrict__ cache,
    int64_t cache_stride, Slots slots, int64_t n, int dim, int64_t rows,
    int group) {
  const int lane = threadIdx.x & (group - 1);
  const int per_block = 256 / group;
  const int quads = (dim + 3) / 4;
  for (int64_t j0 = ((int64_t)blockIdx.x * per_block + threadIdx.x / group) *
                    ROWS;
       j0 < n; j0 += (int64_t)gridDim.x * per_block * ROWS) {
    int64_t slot[ROWS];
    uint32_t w[ROWS][QUADS];
    float s[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      slot[r] = j0 + r < n ? slots[j0 + r] : -1;
      if (slot[r] >= rows) slot[r] = -1;
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      // zeros for padding
      const uint32_t* rec = (const uint32_t*)(cache + slot[r] * cache_stride);
#pragma unroll
      for (int i = 0; i < QUADS; ++i) {
        const int q = lane + i * group;
        w[r][i] = slot[r] >= 0 && q < quads ? rec[q] : 0;
      }
      s[r] = slot[r] >= 0 ? __uint_as_float(rec[quads]) : 0.0f;
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      if (j0 + r >= n) continue;
#pragma unroll
      for (int i = 0; i < QUADS; ++i) {
        const int q = lane + i * group;
        store_quad(out + (j0 + r) * dim + q * 4, decode<FP8>(w[r][i], s[r]),
                   dim - q * 4);
      }
    }
  }
}

template <typename T, bool FP8>
__global__ __launch_bounds__(256) void k_cache_read_long(
    T* __restrict__ out, const uint8_t* __restrict__ cache,
    int64_t cache_stride, Slots slots, int64_t n, int64_t dim, int64_t rows) {
  const int lane = threadIdx.x % WAVE;
  const int64_t quads = (dim + 3) / 4;
  for (int64_t j = (int64_t)blockIdx.x * 4 + threadIdx.x / WAVE; j < n;
       j += (int64_t)gridDim.x * 4) {
    const int64_t slot = slots[j];
    const bool held = slot >= 0 && slot < rows;
    const uint32_t* rec = (const uint32_t*)(cache + (held ? slot : 0) *
                                                        cache_stride);
    const float s = held ? __uint_as_float(rec[quads]) : 0.0f;
    for (int64_t q = lane; q < quads; q += WAVE)
      store_quad(out + j * dim + q * 4, decode<FP8>(held ? rec[q] : 0, s),
                 dim - q * 4);
  }
}

int grid_of(int64_t blocks) {
  return (int)std::max<int64_t>(1, std::min<int64_t>(blocks, 4096));
}

// How lanes share a row: `group` lanes of `quads` quads each, 0 quads for a
// row too long for registers.  The pair that leaves the fewest places of it
// empty, under 32 lanes only if it saves a fifth; of several, up to four quads
// and lanes near to 32 (500,000 x 256 bf16 as fp8: 32 x 2 4.6 TB/s, 64 x 1 3.8;
// 1,000,000 x 300 f32 as int8: 16 x 5 4% slower than 32 x 3; 100,003 x 77 f16:
// 8 x 3 10 us, 32 x 1 16.5).
struct Share { int group, quads; };

Share share_of(int64_t dim) {
  const int64_t need = (dim + 3) / 4;
  if (need > WAVE * 8) return {WAVE, 0};
  Share best{0, 0};
  int least = INT_MAX;
  for (int group : {32, 64, 16, 8, 4, 2, 1}) {
    if (group < 8 && need > 4) break;
    const int64_t q = (need + group - 1) / group;
    const int quads = q == 7 ? 8 : (int)q;
    const int cost = group * quads * (group < 32 ? 5 : 4);
    if (quads <= 8 && (cost < least ||
                       (cost == least && best.quads > 4 && quads <= 4))) {
      best = {group, quads};
      least = cost;
    }
  }
  return best;
}

// f(std::integral_constant<QUADS>{}, std::integral_constant<ROWS>{})
template <typename F>
void by_share(int quads, F f) {
  using std::integral_constant;
  if (quads == 1) f(integral_constant<int, 1>{}, integral_constant<int, 4>{});
  else if (quads == 2)
    f(integral_constant<int, 2>{}, integral_constant<int, 2>{});
  else if (quads == 3)
    f(integral_constant<int, 3>{}, integral_constant<int, 2>{});
  else if (quads == 4)
    f(integral_constant<int, 4>{}, integral_constant<int, 1>{});
  else if (quads == 5)
    f(integral_constant<int, 5>{}, integral_constant<int, 1>{});
  else if (quads == 6)
    f(integral_constant<int, 6>{}, integral_constant<int, 1>{});
  else f(integral_constant<int, 8>{}, integral_constant<int, 1>{});
}

template <typename T, bool FP8>
void launch_write(at::Tensor& cache, const at::Tensor& values, Slots slots,
                  const int* owner, hipStream_t stream) {
  const int64_t n = values.size(0), dim = values.size(1);
  const Share sh = share_of(dim);
  const T* x = (const T*)values.data_ptr();
  uint8_t* out = cache.data_ptr<uint8_t>();
  auto go = [&](auto* kfn, int rows) {
    const int64_t per = (int64_t)(256 / sh.group) * rows;
    hipLaunchKernelGGL(kfn, dim3(grid_of((n + per - 1) / per)), dim3(256), 0,
                       stream, out, cache.stride(0), x, values.stride(0),
                       slots, owner, n, (int)dim, cache.size(0), sh.group);
  };
  if (sh.quads)
    by_share(sh.quads, [&](auto q, auto r) {
      constexpr int Q = decltype(q)::value, R = decltype(r)::value;
      go(k_cache_write<T, FP8, Q, R>, R);
    });
  else
    hipLaunchKernelGGL((k_cache_write_long<T, FP8>), dim3(grid_of((n + 3) / 4)),
                       dim3(256), 0, stream, out, cache.stride(0), x,
                       values.stride(0), slots, owner, n, dim, cache.size(0));
}

template <typename T, bool FP8>
void launch_read(at::Tensor& out, const at::Tensor& cache, Slots slots,
                 hipStream_t stream) {
  const int64_t n = out.size(0), dim = out.size(1);
  const Share sh = share_of(dim);
  T* to = (T*)out.data_ptr();
  const uint8_t* from = cache.data_ptr<uint8_t>();
  auto go = [&](auto* kfn, int rows) {
    const int64_t per = (int64_t)(256 / sh.group) * rows;
    hipLaunchKernelGGL(kfn, dim3(grid_of((n + per - 1) / per)), dim3(256), 0,
                       stream, to, from, cache.stride(0), slots, n, (int)dim,
                       cache.size(0), sh.group);
  };
  if (sh.quads)
    by_share(sh.quads, [&](auto q, auto r) {
      constexpr int Q = decltype(q)::value, R = decltype(r)::value;
      go(k_cache_read<T, FP8, Q, R>, R);
    });
  else
    hipLaunchKernelGGL((k_cache_read_long<T, FP8>), dim3(grid_of((n + 3) / 4)),
                       dim3(256), 0, stream, to, from, cache.stride(0), slots,
                       n, dim, cache.size(0));
}

// f(T{}, std::bool_constant<FP8>{}) for the value type and the format
template <typename F>
void by_types(at::ScalarType t, bool fp8, F f) {
  auto formats = [&](auto v) {
    if (fp8) f(v, std::true_type{}); else f(v, std::false_type{});
  };
  if (t == at::kFloat) formats(float{});
  else if (t == at::kHalf) formats(__half{});
  else if (t == at::kBFloat16) formats(__hip_bfloat16{});
  else TORCH_CHECK(false, "values must be float32, bfloat16 or float16");
}

Slots slots_of(const c10::optional<at::Tensor>& slots) {
  if (!slots) return {nullptr, false};
  return {slots->data_ptr(), slots->scalar_type() == at::kLong};
}

bool is_fp8(const std::string& fmt) {
  TORCH_CHECK_VALUE(fmt == "int8" || fmt == "fp8", "unknown row format '",
                    fmt, "'");
  return fmt == "fp8";
}

bool is_value_type(at::ScalarType t) {
  return t == at::kFloat || t == at::kBFloat16 || t == at::kHalf;
}

// ops/reference.py refuses the same on the CPU.
void check_records(const char* name, const at::Tensor& cache, int64_t dim,
                   const c10::optional<at::Tensor>& slots) {
  TORCH_CHECK_VALUE(
      dim >= 1 && cache.scalar_type() == at::kByte && cache.dim() == 2 &&
          cache.size(1) == (dim + 3) / 4 * 4 + 4,
      name, ": the cache of rows of ", dim,
      " values is uint8 of shape (rows, record_bytes(", dim, ")), got ",
      cache.scalar_type(), " of ", cache.sizes());
  TORCH_CHECK_VALUE(!cache.size(0) ||
                        (cache.stride(1) == 1 && cache.stride(0) % 4 == 0 &&
                         (uintptr_t)cache.data_ptr() % 4 == 0),
                    name,
                    ": cache records must be contiguous and 4-byte aligned");
  if (slots)
    TORCH_CHECK_VALUE((slots->scalar_type() == at::kLong ||
                       slots->scalar_type() == at::kInt) &&
                          slots->dim() == 1 &&
                          slots->device() == cache.device(),
                      name, ": slots must be 1-D int64 or int32 on the "
                      "cache's device, got ", slots->scalar_type(), " of ",
                      slots->sizes(), " on ", slots->device());
}

}  // namespace

void cache_write(at::Tensor cache, at::Tensor values,
                 c10::optional<at::Tensor> slots, const std::string& fmt,
                 bool unique) {
  const bool fp8 = is_fp8(fmt);
  TORCH_CHECK_VALUE(values.dim() == 2 && is_value_type(values.scalar_type()) &&
                        values.device() == cache.device(),
                    "cache_write: values must be 2-D float32, bfloat16 or "
                    "float16 on the cache's device, got ",
                    values.scalar_type(), " of ", values.sizes(), " on ",
                    values.device());
  check_records("cache_write", cache, values.size(1), slots);
  const int64_t n = values.size(0);
  TORCH_CHECK_VALUE(n == (slots ? slots->numel() : cache.size(0)),
                    "cache_write: ", n, " rows of values for ",
                    slots ? slots->numel() : cache.size(0),
                    slots ? " slots" : " records");
  TORCH_CHECK_VALUE(cache.size(0) < 2 || cache.stride(0) >= cache.size(1),
                    "cache_write: cache records must not overlap");
  TORCH_CHECK_VALUE(n < (int64_t{1} << 31),
                    "cache_write: 2^31 rows or more in one write");
  TORCH_CHECK(!(values.requires_grad() && c10::GradMode::is_enabled()),
              "cache_write has no gradient: pass values.detach()");
  TORCH_CHECK(!values._fw_grad(0).defined(),
              "cache_write has no gradient: an operand carries a tangent");
  if (!n) return;
  c10::DeviceGuard guard(cache.device());
  hipStream_t stream = at::hip::getCurrentHIPStream().stream();
  if (values.stride(1) != 1) values = values.contiguous();
  if (slots) slots = slots->contiguous();
  at::Tensor owner;
  if (slots && !unique)
    owner = at::full({cache.size(0)}, -1, cache.options().dtype(at::kInt));
  const Slots at_ = slots_of(slots);
  int* own = owner.defined() ? owner.data_ptr<int>() : nullptr;
  if (own)
    hipLaunchKernelGGL(k_cache_owner, dim3(grid_of((n + 255) / 256)),
                       dim3(256), 0, stream, own, at_, n, cache.size(0));
  by_types(values.scalar_type(), fp8, [&](auto t, auto f) {
    launch_write<decltype(t), decltype(f)::value>(cache, values, at_, own,
                                                  stream);
  });
}

at::Tensor cache_read(at::Tensor cache, int64_t dim,
                      c10::optional<at::Tensor> slots, const std::string& fmt,
                      at::ScalarType dtype) {
  const bool fp8 = is_fp8(fmt);
  check_records("cache_read", cache, dim, slots);
  TORCH_CHECK_VALUE(is_value_type(dtype), "cache_read: dtype must be float32, "
                    "bfloat16 or float16, got ", dtype);
  const int64_t n = slots ? slots->numel() : cache.size(0);
  c10::DeviceGuard guard(cache.device());
  if (slots) slots = slots->contiguous();
  auto out = at::empty({n, dim}, cache.options().dtype(dtype));
  if (!n) return out;
  if (!cache.size(0)) return out.zero_();
  hipStream_t stream = at::hip::getCurrentHIPStream().stream();
  by_types(dtype, fp8, [&](auto t, auto f) {
    launch_read<decltype(t), decltype(f)::value>(out, cache, slots_of(slots),
                                                 stream);
  });
  return out;
}
