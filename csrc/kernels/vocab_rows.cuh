// Rows of logits [R, V] walked in vectors of 16 bytes, whatever the row's alignment,
// by a thread-block cluster, and the running maximum and sum of a softmax over them.
//
// Vector v of a row lies on a 16-byte boundary and holds the elements v E - mis ..
// v E - mis + E - 1, where mis is the number of elements between the boundary below
// the row's start and that start; elements outside the row are never touched (the
// first and the last vector are read element by element where they reach out).
// CTA c of the cluster walks the vectors [v0, v1).  Eight vectors (128 bytes) are a group.
#pragma once

#include <cooperative_groups.h>
#include <math.h>

#include "device_common.cuh"
#include "vec_io.cuh"

namespace tb {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
struct Row {
  static constexpr int E = 16 / sizeof(T);
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
  __device__ __forceinline__ void load(int v, float (&x)[E]) const {  // -inf outside the row
    if (inside(v, v + 1)) {
      load_vec<T, E>(base + static_cast<long long>(v) * E, x);
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const int i = v * E - mis + j;
        x[j] = i >= 0 && i < V ? to_f32(row[i]) : -INFINITY;
      }
    }
  }
};

// Running maximum m and sum s of 2^((x - m) k1).  The difference is formed before it
// is scaled, so that the type's lowest value neither overflows nor loses its ties; an
// infinite maximum counts as 0 there (s is then 0, inf or NaN).
struct SoftSum {
  float m = -INFINITY, s = 0.f;
  __device__ __forceinline__ static float origin(float m) { return isinf(m) ? 0.f : m; }
  template <int N>
  __device__ __forceinline__ void add(const float (&x)[N], float top, float k1) {  // top: the largest of x
    if (top > m) {
      s *= m == -INFINITY ? 0.f : ex2((m - top) * k1);
      m = top;
    }
    const float o = origin(m);
#pragma unroll
    for (int j = 0; j < N; ++j) s += ex2((x[j] - o) * k1);
  }
  __device__ __forceinline__ void merge(float om, float os, float k1) {
    const float top = fmaxf(m, om);
    s = (m == top ? s : s * ex2((m - top) * k1)) + (om == top ? os : os * ex2((om - top) * k1));
    m = top;
  }
};

// Merges every thread's sum; the result is valid in all threads.  `buf` holds 2 x 32 floats.
__device__ __forceinline__ SoftSum block_merge(SoftSum a, float k1, float* buf) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float om = __shfl_xor_sync(0xffffffffu, a.m, o), os = __shfl_xor_sync(0xffffffffu, a.s, o);
    a.merge(om, os, k1);
  }
  __syncthreads();
  if (lane == 0) {
    buf[w] = a.m;
    buf[32 + w] = a.s;
  }
  __syncthreads();
  a.m = lane < nw ? buf[lane] : -INFINITY;
  a.s = lane < nw ? buf[32 + lane] : 0.f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float om = __shfl_xor_sync(0xffffffffu, a.m, o), os = __shfl_xor_sync(0xffffffffu, a.s, o);
    a.merge(om, os, k1);
  }
  return a;
}

// The same over a cluster (`mine`: two floats of shared memory).
__device__ __forceinline__ SoftSum cluster_merge(SoftSum a, float k1, float* mine) {
  cooperative_groups::cluster_group cl = cooperative_groups::this_cluster();
  const unsigned n = cl.num_blocks();
  if (n == 1) return a;
  if (threadIdx.x == 0) {
    mine[0] = a.m;
    mine[1] = a.s;
  }
  cl.sync();
  SoftSum all;
  for (unsigned r = 0; r < n; ++r) {
    const float* o = cl.map_shared_rank(mine, r);
    all.merge(o[0], o[1], k1);
  }
  return all;
}

}  // namespace tb
