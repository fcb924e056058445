// Vector loads and stores of N contiguous bf16 / fp16 / fp32 values as fp32
// registers.  N * sizeof(T) is 4, 8, 16 or 32 bytes and the address is aligned
// to min(16, N * sizeof(T)).  Stores round to nearest even.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace tb {

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }

template <int BYTES>
struct RawOf;
template <>
struct RawOf<2> { using type = unsigned short; };
template <>
struct RawOf<4> { using type = uint32_t; };
template <>
struct RawOf<8> { using type = uint2; };
template <>
struct RawOf<16> { using type = uint4; };

template <typename T, int N>
__device__ __forceinline__ void load_vec(const T* p, float (&f)[N]) {
  constexpr int kPer = N * sizeof(T) > 16 ? 16 / static_cast<int>(sizeof(T)) : N;
  using Raw = typename RawOf<kPer * sizeof(T)>::type;
#pragma unroll
  for (int j = 0; j < N / kPer; ++j) {
    const Raw r = *reinterpret_cast<const Raw*>(p + j * kPer);
    const T* e = reinterpret_cast<const T*>(&r);
#pragma unroll
    for (int i = 0; i < kPer; ++i) f[j * kPer + i] = to_f32(e[i]);
  }
}

template <typename T, int N>
__device__ __forceinline__ void store_vec(T* p, const float (&f)[N]) {
  constexpr int kPer = N * sizeof(T) > 16 ? 16 / static_cast<int>(sizeof(T)) : N;
  using Raw = typename RawOf<kPer * sizeof(T)>::type;
#pragma unroll
  for (int j = 0; j < N / kPer; ++j) {
    Raw r;
    T* e = reinterpret_cast<T*>(&r);
#pragma unroll
    for (int i = 0; i < kPer; ++i) e[i] = from_f32<T>(f[j * kPer + i]);
    *reinterpret_cast<Raw*>(p + j * kPer) = r;
  }
}

// N values as they lie in memory (N * sizeof(T) at most 16 bytes), so that loads
// can be kept in flight in few registers.
template <typename T, int N>
struct Packed {
  typename RawOf<N * sizeof(T)>::type raw;
  __device__ __forceinline__ void load(const T* p) { raw = *reinterpret_cast<const decltype(raw)*>(p); }
  __device__ __forceinline__ void unpack(float (&f)[N]) const {
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = to_f32(e[i]);
  }
};

}  // namespace tb
