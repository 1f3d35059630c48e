// Value types and vectors of four of them, shared by the device sources.
#pragma once

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

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
  // Keeps the value's own rounding to f32: a product that is fused with the
  // conversion would round once, and differ from every other path in a last
  // place.
  asm volatile("" : "+v"(v));
  return __float2half_rn(v);
}
template <>
__device__ inline __hip_bfloat16 from_f32(float v) {
  return __float2bfloat16(v);
}

// Four neighbouring values at any address that a T may have: the memory path
// takes vectors that are aligned to their elements.
template <typename T>
struct Bits;
template <>
struct Bits<float> { using Raw = float; };
template <>
struct Bits<__half> { using Raw = uint16_t; };
template <>
struct Bits<__hip_bfloat16> { using Raw = uint16_t; };

template <typename T>
struct Quad {
  using Raw = typename Bits<T>::Raw;
  typedef Raw Vec __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  Vec v;
  __device__ inline void load(const T* at) { v = *(const Vec*)at; }
  __device__ inline void store(T* at) const { *(Vec*)at = v; }
  __device__ inline T get(int i) const {
    Raw r = v[i];
    return *(T*)&r;
  }
  __device__ inline void set(int i, T t) { v[i] = *(Raw*)&t; }
};

// The same of two
template <typename T>
struct Pair {
  using Raw = typename Bits<T>::Raw;
  typedef Raw Vec __attribute__((ext_vector_type(2), aligned(sizeof(T))));
  Vec v;
  __device__ inline void load(const T* at) { v = *(const Vec*)at; }
  __device__ inline T get(int i) const {
    Raw r = v[i];
    return *(T*)&r;
  }
};

// The first `held` (any number) of four values, zeros after them.
template <typename T>
__device__ inline float4 load_quad(const T* at, int64_t held) {
  float4 f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (held >= 4) {
    Quad<T> q;
    q.load(at);
    f = make_float4(to_f32(q.get(0)), to_f32(q.get(1)), to_f32(q.get(2)),
                    to_f32(q.get(3)));
  } else {
    if (held > 0) f.x = to_f32(at[0]);
    if (held > 1) f.y = to_f32(at[1]);
    if (held > 2) f.z = to_f32(at[2]);
  }
  return f;
}

template <typename T>
__device__ inline void store_quad(T* at, float4 f, int64_t held) {
  Quad<T> q;
  q.set(0, from_f32<T>(f.x));
  q.set(1, from_f32<T>(f.y));
  q.set(2, from_f32<T>(f.z));
  q.set(3, from_f32<T>(f.w));
  if (held >= 4) {
    q.store(at);
  } else {
    if (held > 0) at[0] = q.get(0);
    if (held > 1) at[1] = q.get(1);
    if (held > 2) at[2] = q.get(2);
  }
}
