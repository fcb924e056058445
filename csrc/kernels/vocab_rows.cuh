// Rows of logits [R, V] walked in vectors of 16 bytes, whatever the row's alignment,
// by a thread-block cluster, and the running maximum and sum of a softmax over them.
//
// Vector v of a row lies on a 16-byte boundary and holds the elements v E - mis ..
// v E - mis + E - 1, where mis is the number of elements between the boundary below
// the row's start and that start; elements outside the row are never touched (the
// first and the last vector are read element by element where they reach out).
// CTA c of the cluster walks the vectors [v0, v1).  Eight vectors (128 bytes) are a
// group, 32 groups a chunk: a warp takes a chunk at a time, lane l its vectors l,
// 32 + l, ..., 224 + l, so that every load of the warp is 512 consecutive bytes.
#pragma once

#include <cooperative_groups.h>
#include <math.h>

#include <type_traits>

#include "device_common.cuh"
#include "vec_io.cuh"

namespace tb {

constexpr double kLog2e = 1.4426950408889634;
constexpr float kLn2 = 0.69314718f;
constexpr int kChunk = 256;  // vectors of a chunk

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// log of a positive finite number as the sum of two, off by 2^-25 or so: the exponent's
// share exactly (its factor ln 2 in two parts, the first of 12 bits).
__device__ __forceinline__ float2 log_of(float x) {
  int e;
  float f = frexpf(x, &e);  // [0.5, 1)
  if (f < 0.70710678f) {
    f *= 2.f;
    --e;
  }
  constexpr float kHigh = 0.693115234375f, kLow = 3.19461846e-5f;  // ln 2
  return make_float2(e * kHigh, fmaf(static_cast<float>(e), kLow, logf(f)));
}
// 1 / T, and log p of a logit.
struct Scaled {
  float inv_t;
  __device__ __forceinline__ float operator()(float z, float top, float2 lns) const {
    return fmaf(z - top, inv_t, -lns.x) - lns.y;
  }
};

// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n.reg .b64 a, b, c, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nmov.b64 c, {%6, %7};\n"
      "fma.rn.f32x2 d, a, b, c;\nmov.b64 {%0, %1}, d;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n.reg .b64 a, b, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nadd.rn.f32x2 d, a, b;\nmov.b64 {%0, %1}, d;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n.reg .b64 a, b, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nmul.rn.f32x2 d, a, b;\nmov.b64 {%0, %1}, d;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// A vector as it lies in memory: its values in pairs, its maximum (NaN is left out), and
// -inf put in the place of one element.
template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr uint32_t kLowest = 0xff800000u;
  using Max = float;
  __device__ __forceinline__ static float2 pair(const uint4& p, int i) {
    return i == 0 ? make_float2(__uint_as_float(p.x), __uint_as_float(p.y)) : make_float2(__uint_as_float(p.z), __uint_as_float(p.w));
  }
  __device__ __forceinline__ static Max max(Max a, Max b) { return fmaxf(a, b); }
  __device__ __forceinline__ static Max top(const uint4& p) {
    return fmaxf(fmaxf(__uint_as_float(p.x), __uint_as_float(p.y)), fmaxf(__uint_as_float(p.z), __uint_as_float(p.w)));
  }
  __device__ __forceinline__ static float value(Max m) { return fmaxf(m, -INFINITY); }
};
template <>
struct Vec<__nv_bfloat16> {
  static constexpr uint32_t kLowest = 0xff80ff80u;
  using Max = uint32_t;
  __device__ __forceinline__ static uint32_t word(const uint4& p, int i) { return i == 0 ? p.x : i == 1 ? p.y : i == 2 ? p.z : p.w; }
  __device__ __forceinline__ static float2 pair(const uint4& p, int i) {
    const uint32_t w = word(p, i);
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  __device__ __forceinline__ static Max max(Max a, Max b) {
    const __nv_bfloat162 m = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
  }
  __device__ __forceinline__ static Max top(const uint4& p) { return max(max(p.x, p.y), max(p.z, p.w)); }
  __device__ __forceinline__ static float value(Max m) {
    return fmaxf(fmaxf(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u)), -INFINITY);
  }
};
template <>
struct Vec<__half> {
  static constexpr uint32_t kLowest = 0xfc00fc00u;
  using Max = uint32_t;
  __device__ __forceinline__ static float2 pair(const uint4& p, int i) {
    const uint32_t w = Vec<__nv_bfloat16>::word(p, i);
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  }
  __device__ __forceinline__ static Max max(Max a, Max b) {
    const __half2 m = __hmax2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
  }
  __device__ __forceinline__ static Max top(const uint4& p) { return max(max(p.x, p.y), max(p.z, p.w)); }
  __device__ __forceinline__ static float value(Max m) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&m));
    return fmaxf(fmaxf(f.x, f.y), -INFINITY);
  }
};

template <typename T>
struct Row {
  static constexpr int E = 16 / sizeof(T);
  static constexpr int kPairs = E / 2;
  const T* row;   // the row's first element
  const T* base;  // the 16-byte boundary at or below it
  int mis, V, NV;
  int v0, v1;
  __device__ __forceinline__ Row(const T* r, int V_, int rank, int ranks) : row(r), V(V_) {
    mis = static_cast<int>((reinterpret_cast<uintptr_t>(r) & 15) / sizeof(T));
    base = r - mis;
    NV = (V + mis + E - 1) / E;
    const int groups = (NV + 7) / 8, per = (groups + ranks - 1) / ranks;
    v0 = min(rank * per, groups) * 8;
    v1 = min(min(rank * per + per, groups) * 8, NV);
  }
  // Whether every element of the vectors [a, b) is the row's.
  __device__ __forceinline__ bool inside(int a, int b) const { return (a > 0 || mis == 0) && b * E - mis <= V; }
  __device__ __forceinline__ uint4 load_inside(int v) const {
    uint4 p;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(p.x), "=r"(p.y), "=r"(p.z), "=r"(p.w)
                 : "l"(base + static_cast<long long>(v) * E)
                 : "memory");
    return p;
  }
  // With a policy for the L2 cache.
  __device__ __forceinline__ uint4 load_inside(int v, uint64_t policy) const {
    uint4 p;
    asm volatile("ld.global.L1::no_allocate.L2::cache_hint.v4.u32 {%0, %1, %2, %3}, [%4], %5;"
                 : "=r"(p.x), "=r"(p.y), "=r"(p.z), "=r"(p.w)
                 : "l"(base + static_cast<long long>(v) * E), "l"(policy)
                 : "memory");
    return p;
  }
  __device__ __forceinline__ static uint4 lowest() {
    return make_uint4(Vec<T>::kLowest, Vec<T>::kLowest, Vec<T>::kLowest, Vec<T>::kLowest);
  }
  // A vector of [v0, v1) or behind it: -inf outside the row.
  __device__ uint4 load(int v) const {
    if (v < v1 && inside(v, v + 1)) return load_inside(v);
    union {
      uint4 p;
      T x[E];
    } u;
    u.p = lowest();
    if (v < v1) {
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const int i = v * E - mis + j;
        if (i >= 0 && i < V) u.x[j] = row[i];
      }
    }
    return u.p;
  }
  // A lane's vectors of the chunk that begins at vector c.
  __device__ __forceinline__ void load_chunk(int c, uint4 (&p)[8]) const {
    const int lane = threadIdx.x & 31;
    if (c + kChunk <= v1 && inside(c, c + kChunk)) {
#pragma unroll
      for (int i = 0; i < 8; ++i) p[i] = load_inside(c + i * 32 + lane);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) p[i] = load(c + i * 32 + lane);
    }
  }
  // The same for N vectors of a lane, with a policy.
  template <int N>
  __device__ __forceinline__ void load_some(int c, uint4 (&p)[N], uint64_t policy) const {
    const int lane = threadIdx.x & 31;
    if (c + N * 32 <= v1 && inside(c, c + N * 32)) {
#pragma unroll
      for (int i = 0; i < N; ++i) p[i] = load_inside(c + i * 32 + lane, policy);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) p[i] = load(c + i * 32 + lane);
    }
  }
};

// What is read again soon stays in the L2 cache before all else; what is not goes first.
__device__ __forceinline__ uint64_t read_again() {
  uint64_t p;
  asm("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(p));
  return p;
}
__device__ __forceinline__ uint64_t read_once() {
  uint64_t p;
  asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
  return p;
}

// A maximum m and the sum s of 2^((x - m) k1), in fp32 (a row's sum is off by 1e-7 or so: each
// of 1,024 partial sums adds V / 1,024 terms); an infinite m counts as 0 in the exponent
// (s is then 0, inf or NaN).
struct SoftSum {
  float m = -INFINITY, s = 0.f;
  __device__ __forceinline__ void merge(float om, float os, float k1) {
    const float top = fmaxf(m, om);
    s = (m == top ? s : s * ex2((m - top) * k1)) + (om == top ? os : os * ex2((om - top) * k1));
    m = top;
  }
  __device__ __forceinline__ void merge_lanes(float k1) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float om = __shfl_xor_sync(0xffffffffu, m, o), os = __shfl_xor_sync(0xffffffffu, s, o);
      merge(om, os, k1);
    }
  }
};

// The exponent x k1 + c of 2^((x - m) k1) in one operation: c = -m k1 rounded, whose
// rounding d `fix` takes out of a sum of such powers, as 1 - d ln 2 (below 2^11, where d is
// at most 2^-14, off by 2^-29).  Where that product is larger (up to masks of the type's
// lowest value as the only values of a row), the difference is formed first.
struct Exponent {
  float m, k1, c, fix;
  bool near;
  __device__ __forceinline__ Exponent(float m_, float k1_) : k1(k1_) {
    m = isinf(m_) ? 0.f : m_;
    c = -(m * k1);
    near = fabsf(c) < 2048.f;
    fix = near ? 1.f - fmaf(m, k1, c) * kLn2 : 1.f;
  }
  __device__ __forceinline__ float2 powers(float2 x) const {
    const float2 a = near ? fma2(x, make_float2(k1, k1), make_float2(c, c)) : make_float2((x.x - m) * k1, (x.y - m) * k1);
    return make_float2(ex2(a.x), ex2(a.y));
  }
  __device__ __forceinline__ float power(float x) const { return ex2(near ? fmaf(x, k1, c) : (x - m) * k1); }
};

// -inf in the place of the elements whose bits are set in `in`.
template <typename T>
__device__ __forceinline__ uint4 without(uint4 p, uint32_t in) {
  constexpr int E = Row<T>::E;
  uint32_t w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (E == 4) {
      if (in >> i & 1) w[i] = Vec<T>::kLowest;
    } else {
      const uint32_t m = (in >> (2 * i) & 1 ? 0xffffu : 0u) | (in >> (2 * i + 1) & 1 ? 0xffff0000u : 0u);
      w[i] = (w[i] & ~m) | (Vec<T>::kLowest & m);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// factor x 2^((x - m) k1) of a vector's elements, rounded to their type.
template <typename T>
__device__ __forceinline__ uint4 scaled_powers(const uint4& p, const Exponent& e, float2 factor) {
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < Row<T>::kPairs; ++j) {
    const float2 y = mul2(e.powers(Vec<T>::pair(p, j)), factor);
    if constexpr (sizeof(T) == 4) {
      w[2 * j] = __float_as_uint(y.x);
      w[2 * j + 1] = __float_as_uint(y.y);
    } else if constexpr (std::is_same<T, __half>::value) {
      const __half2 h = __floats2half2_rn(y.x, y.y);
      w[j] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(y.x, y.y);
      w[j] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// The running form, a chunk's vectors of a lane at a time.
template <typename T>
struct RunningSum {
  float m = -INFINITY;
  float2 s0 = {0.f, 0.f}, s1 = {0.f, 0.f};
  template <int N>
  __device__ __forceinline__ void add(const uint4 (&p)[N], float top, float k1) {
    if (top > m) {  // (what is there gets the new maximum's rounding, which done() takes out)
      const float f = m == -INFINITY ? 0.f : Exponent(m, k1).fix * (2.f - Exponent(top, k1).fix) * ex2((m - top) * k1);
      s0 = mul2(s0, make_float2(f, f));
      s1 = mul2(s1, make_float2(f, f));
      m = top;
    }
    const Exponent e(m, k1);
    if (e.near) {
      const float2 k2 = make_float2(k1, k1), c2 = make_float2(e.c, e.c);
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < Row<T>::kPairs; ++j) {
          const float2 a = fma2(Vec<T>::pair(p[i], j), k2, c2);
          float2& s = j & 1 ? s1 : s0;
          s = add2(s, make_float2(ex2(a.x), ex2(a.y)));
        }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < Row<T>::kPairs; ++j) s0 = add2(s0, e.powers(Vec<T>::pair(p[i], j)));
    }
  }
  __device__ __forceinline__ SoftSum done(float k1) const {
    SoftSum r;
    r.m = m;
    r.s = ((s0.x + s0.y) + (s1.x + s1.y)) * Exponent(m, k1).fix;
    return r;
  }
};

}  // namespace tb
