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
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include "ops.h"

namespace {

constexpr int WAVE = 64;
constexpr float TINY = 0x1p-126f;  // the smallest normal f32
constexpr float FP8_TOP = 0x1.ep+127f;  // 240 * 2^120: the next code is 2^128
// The largest scale whose code 127 is finite; RN(FLT_MAX / 127) is one ulp up.
constexpr float INT8_TOP = 0x1.020406p+121f;

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
__device__ inline __half from_f32(float v) {
  // Keeps the product's own rounding to f32: fused with the conversion it
  // would round once, and differ from every other path in a last place.
  asm volatile("" : "+v"(v));
  return __float2half_rn(v);
}
template <>
__device__ inline __hip_bfloat16 from_f32(float v) {
  return __float2bfloat16(v);
}

template <typename S>
__device__ inline int64_t slot_of(const S* slots, int64_t j) {
  return slots ? (int64_t)slots[j] : j;
}

// |x| as an ordered integer: finite < inf < NaN, so the largest one of a
// row also says whether the row is finite.
__device__ inline uint32_t magnitude(float x) {
  return __float_as_uint(x) & 0x7fffffffu;
}

template <bool FP8>
__device__ inline float scale_of(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  float amax = __uint_as_float(amax_bits);
  if (!FP8) return fminf(fmaxf(amax / 127.0f, TINY), INT8_TOP);
  // 448 = 1.75 * 2^8: with amax = m * 2^e, 1 <= m < 2, the exponent is
  // e - 8 while m <= 1.75 and e - 7 above.  (Subnormal: the 2^-126 floor.)
  int e = (int)(amax_bits >> 23) - 127;
  int k = (amax_bits & 0x7fffffu) <= 0x600000u ? e - 8 : e - 7;
  if (k < -126) k = -126;
  return __uint_as_float((uint32_t)(k + 127) << 23);
}

// Nearest integer to the exact quotient x / s, ties to even.  x * inv is off
// by at most one step next to a half; the remainder x - q s is exact in one
// fma (a multiple of ulp(s) / 2 no larger than s) and says which way.
__device__ inline int code_int8(float x, float s, float inv) {
  float q = rintf(x * inv);
  float r = fmaf(-q, s, x);
  float twice = 2.0f * fabsf(r);
  bool odd = ((int)q) & 1;
  if (twice > s || (twice == s && odd)) q += copysignf(1.0f, r);
  return (int)q;
}

__device__ inline uint32_t wave_max(uint32_t v) {
#pragma unroll
  for (int o = WAVE / 2; o; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o));
  return v;
}

// The last of the writes to a slot wins, whatever the order that they run in.
template <typename S>
__global__ __launch_bounds__(256) void k_cache_owner(
    int* __restrict__ owner, const S* __restrict__ slots, int64_t n,
    int64_t rows) {
  for (int64_t j = (int64_t)blockIdx.x * 256 + threadIdx.x; j < n;
       j += (int64_t)gridDim.x * 256) {
    int64_t s = (int64_t)slots[j];
    if (s >= 0 && s < rows) atomicMax(owner + s, (int)j);
  }
}

// One wave a row: the row's largest magnitude, then its codes.
template <typename T, typename S, bool FP8>
__global__ __launch_bounds__(256) void k_cache_write(
    uint8_t* __restrict__ cache, int64_t cache_stride,
    const T* __restrict__ values, int64_t value_stride,
    const S* __restrict__ slots, const int* __restrict__ owner, int64_t n,
    int64_t dim, int64_t rows) {
  const int lane = threadIdx.x % WAVE;
  const int64_t waves = (int64_t)gridDim.x * (256 / WAVE);
  const int64_t padded = (dim + 3) / 4 * 4;
  for (int64_t j = (int64_t)blockIdx.x * (256 / WAVE) + threadIdx.x / WAVE;
       j < n; j += waves) {
    int64_t slot = slot_of(slots, j);
    if (slot < 0 || slot >= rows) continue;
    if (owner && owner[slot] != (int)j) continue;
    const T* x = values + j * value_stride;
    uint8_t* out = cache + slot * cache_stride;
    uint32_t top = 0;
    for (int64_t c = lane; c < dim; c += WAVE)
      top = max(top, magnitude(to_f32(x[c])));
    const float s = scale_of<FP8>(wave_max(top));
    const bool finite = s == s;
    const float inv = 1.0f / s;
    for (int64_t c = lane; c < padded; c += WAVE) {
      uint8_t code = 0;
      if (c < dim && finite) {
        float v = to_f32(x[c]);
        if (FP8)
          code = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(
              __builtin_amdgcn_fmed3f(v, -FP8_TOP, FP8_TOP) * inv, 0.0f, 0,
              false);
        else
          code = (uint8_t)code_int8(v, s, inv);
      }
      out[c] = code;
    }
    if (lane == 0) *(float*)(out + padded) = s;
  }
}

template <typename T, typename S, bool FP8>
__global__ __launch_bounds__(256) void k_cache_read(
    T* __restrict__ out, const uint8_t* __restrict__ cache,
    int64_t cache_stride, const S* __restrict__ slots, int64_t n, int64_t dim,
    int64_t rows) {
  const int lane = threadIdx.x % WAVE;
  const int64_t waves = (int64_t)gridDim.x * (256 / WAVE);
  const int64_t padded = (dim + 3) / 4 * 4;
  for (int64_t j = (int64_t)blockIdx.x * (256 / WAVE) + threadIdx.x / WAVE;
       j < n; j += waves) {
    int64_t slot = slot_of(slots, j);
    const bool held = slot >= 0 && slot < rows;
    const uint8_t* rec = cache + (held ? slot : 0) * cache_stride;
    const float s = held ? *(const float*)(rec + padded) : 0.0f;
    for (int64_t c = lane; c < dim; c += WAVE) {
      float v = 0.0f;
      if (held) {
        uint8_t code = rec[c];
        v = (FP8 ? __builtin_amdgcn_cvt_f32_fp8((int)code, 0)
                 : (float)(int8_t)code) * s;
      }
      out[j * dim + c] = from_f32<T>(v);
    }
  }
}

int grid_of(int64_t waves) {
  int64_t g = (waves + 3) / 4;
  return (int)(g < 1 ? 1 : (g > 4096 ? 4096 : g));
}

template <typename T, typename S>
void launch_write(at::Tensor& cache, const at::Tensor& values, const S* slots,
                  const int* owner, bool fp8, hipStream_t stream) {
  int64_t n = values.size(0), dim = values.size(1);
  auto* kfn = fp8 ? k_cache_write<T, S, true> : k_cache_write<T, S, false>;
  hipLaunchKernelGGL(kfn, dim3(grid_of(n)), dim3(256), 0, stream,
                     cache.data_ptr<uint8_t>(), cache.stride(0),
                     (const T*)values.data_ptr(), values.stride(0), slots,
                     owner, n, dim, cache.size(0));
}

template <typename T, typename S>
void launch_read(at::Tensor& out, const at::Tensor& cache, const S* slots,
                 bool fp8, hipStream_t stream) {
  int64_t n = out.size(0), dim = out.size(1);
  auto* kfn = fp8 ? k_cache_read<T, S, true> : k_cache_read<T, S, false>;
  hipLaunchKernelGGL(kfn, dim3(grid_of(n)), dim3(256), 0, stream,
                     (T*)out.data_ptr(), cache.data_ptr<uint8_t>(),
                     cache.stride(0), slots, n, dim, cache.size(0));
}

// f(T{}, S{}) for the value type and the slot type
template <typename F>
void by_types(at::ScalarType t, bool wide, F f) {
  auto slots = [&](auto v) {
    if (wide) f(v, int64_t{}); else f(v, int32_t{});
  };
  if (t == at::kFloat) slots(float{});
  else if (t == at::kHalf) slots(__half{});
  else if (t == at::kBFloat16) slots(__hip_bfloat16{});
  else TORCH_CHECK(false, "values must be float32, bfloat16 or float16");
}

bool is_fp8(const std::string& fmt) {
  TORCH_CHECK(fmt == "int8" || fmt == "fp8", "unknown row format ", fmt);
  return fmt == "fp8";
}

void check_cache(const at::Tensor& cache, int64_t dim) {
  TORCH_CHECK(cache.is_cuda(), "cache must be a device tensor");
  TORCH_CHECK(cache.dim() == 2 && cache.scalar_type() == at::kByte,
              "cache must be a 2-D uint8 tensor");
  TORCH_CHECK(dim >= 1 && cache.size(1) == (dim + 3) / 4 * 4 + 4,
              "cache records do not hold rows of ", dim, " values");
  TORCH_CHECK(cache.stride(1) == 1 && cache.stride(0) % 4 == 0 &&
                  (uintptr_t)cache.data_ptr() % 4 == 0,
              "cache records must be contiguous and 4-byte aligned");
}

void check_slots(const c10::optional<at::Tensor>& slots, int64_t n,
                 const at::Tensor& cache) {
  if (!slots) return;
  TORCH_CHECK(slots->device() == cache.device() && slots->is_contiguous() &&
                  slots->numel() == n &&
                  (slots->scalar_type() == at::kLong ||
                   slots->scalar_type() == at::kInt),
              "slots must be n contiguous int64 or int32 on the cache's "
              "device");
}

}  // namespace

void cache_write(at::Tensor cache, at::Tensor values,
                 c10::optional<at::Tensor> slots, const std::string& fmt,
                 bool unique) {
  const bool fp8 = is_fp8(fmt);
  TORCH_CHECK(values.dim() == 2 && values.device() == cache.device(),
              "values must be 2-D on the cache's device");
  const int64_t n = values.size(0);
  check_cache(cache, values.size(1));
  check_slots(slots, n, cache);
  TORCH_CHECK(values.stride(1) == 1 || values.size(1) == 1,
              "rows of values must be contiguous");
  TORCH_CHECK(slots || n == cache.size(0), "without slots there is one "
              "record for each row of values");
  TORCH_CHECK(cache.size(0) < 2 || cache.stride(0) >= cache.size(1),
              "cache records must not overlap");
  TORCH_CHECK(n < (int64_t{1} << 31), "too many rows in one write");
  if (!n) return;
  c10::DeviceGuard guard(cache.device());
  hipStream_t stream = at::hip::getCurrentHIPStream().stream();
  at::Tensor owner;
  if (slots && !unique)
    owner = at::full({cache.size(0)}, -1, cache.options().dtype(at::kInt));
  by_types(values.scalar_type(),
           slots && slots->scalar_type() == at::kLong, [&](auto t, auto s) {
    using T = decltype(t);
    using S = decltype(s);
    const S* at_ = slots ? (const S*)slots->data_ptr() : nullptr;
    if (owner.defined())
      hipLaunchKernelGGL(k_cache_owner<S>, dim3(grid_of(n / WAVE + 1)),
                         dim3(256), 0, stream, owner.data_ptr<int>(), at_, n,
                         cache.size(0));
    launch_write<T, S>(cache, values, at_,
                       owner.defined() ? owner.data_ptr<int>() : nullptr, fp8,
                       stream);
  });
}

at::Tensor cache_read(at::Tensor cache, int64_t dim,
                      c10::optional<at::Tensor> slots, const std::string& fmt,
                      at::ScalarType dtype) {
  const bool fp8 = is_fp8(fmt);
  check_cache(cache, dim);
  const int64_t n = slots ? slots->numel() : cache.size(0);
  check_slots(slots, n, cache);
  c10::DeviceGuard guard(cache.device());
  auto out = at::empty({n, dim}, cache.options().dtype(dtype));
  if (!n) return out;
  if (!cache.size(0)) return out.zero_();
  hipStream_t stream = at::hip::getCurrentHIPStream().stream();
  by_types(dtype, slots && slots->scalar_type() == at::kLong,
           [&](auto t, auto s) {
    using T = decltype(t);
    using S = decltype(s);
    launch_read<T, S>(out, cache,
                      slots ? (const S*)slots->data_ptr() : nullptr, fp8,
                      stream);
  });
  return out;
}
