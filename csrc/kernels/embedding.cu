// Embedding lookup with a scale, and its gradient:
//
//   y_t = s W[id_t],      dW[v] += s sum_{t: id_t = v} dy_t.
//
// The sum of a row is formed in fp32 in a fixed order, so the same inputs give the same bits.
#include "kernels.h"
#include "vec_io.cuh"

#include <math.h>

namespace {

template <typename I>
__device__ __forceinline__ long long id_at(const void* ids, int t) {
  return static_cast<long long>(static_cast<const I*>(ids)[t]);
}
__device__ __forceinline__ long long id_of(const void* ids, int ids64, long long t) {
  return ids64 ? static_cast<const long long*>(ids)[t] : static_cast<const int*>(ids)[t];
}

// A thread for every N elements of the output.
template <typename T, int N>
__global__ void __launch_bounds__(256) lookup_kernel(TbEmbeddingArgs a) {
  const int per = a.H / N;
  const long long total = static_cast<long long>(a.N) * per;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    const long long t = i / per;
    const int h = static_cast<int>(i % per) * N;
    const long long id = id_of(a.ids, a.ids64, t);
    float x[N];
    if (id >= 0 && id < a.V) {
      tb::load_vec<T, N>(static_cast<const T*>(a.weight) + id * a.ld_w + h, x);
#pragma unroll
      for (int j = 0; j < N; ++j) x[j] *= a.scale;
    } else {
      if (id >= 0 && a.err) *a.err = 1;
#pragma unroll
      for (int j = 0; j < N; ++j) x[j] = id < 0 ? 0.f : NAN;
    }
    tb::store_vec<T, N>(static_cast<T*>(a.out) + t * a.ld_out + h, x);
  }
}

// One CTA per token: the first token of an id sums the rows of all of its tokens.
template <typename T, typename G>
__global__ void __launch_bounds__(128) grad_kernel(TbEmbeddingGradArgs a) {
  const int t = blockIdx.x;
  const long long id = id_of(a.ids, a.ids64, t);
  if (id < 0) return;
  if (id >= a.V) {
    if (a.err && threadIdx.x == 0) *a.err = 1;
    return;
  }
  for (int u0 = 0; u0 < t; u0 += 4096) {
    int earlier = 0;
    for (int u = u0 + threadIdx.x; u < min(t, u0 + 4096); u += 128) earlier |= id_of(a.ids, a.ids64, u) == id;
    if (__syncthreads_or(earlier)) return;
  }
  for (int h0 = 0; h0 < a.H; h0 += 512) {
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    for (int u = t; u < a.N; ++u) {
      if (id_of(a.ids, a.ids64, u) != id) continue;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int h = h0 + j * 128 + threadIdx.x;
        if (h < a.H) sum[j] += tb::to_f32(static_cast<const T*>(a.dy)[u * a.ld_dy + h]);
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int h = h0 + j * 128 + threadIdx.x;
      G* p = static_cast<G*>(a.grad) + id * a.ld_grad + h;
      if (h < a.H) *p = tb::from_f32<G>(fmaf(sum[j], a.scale, a.zero ? 0.f : tb::to_f32(*p)));
    }
  }
}

template <typename T>
cudaError_t lookup(const TbEmbeddingArgs& a, cudaStream_t s) {
  constexpr int E = 16 / sizeof(T);
  const uintptr_t at = reinterpret_cast<uintptr_t>(a.weight) | reinterpret_cast<uintptr_t>(a.out) |
                       static_cast<uintptr_t>(a.ld_w * sizeof(T)) | static_cast<uintptr_t>(a.ld_out * sizeof(T)) |
                       static_cast<uintptr_t>(a.H * sizeof(T));
  const long long threads = static_cast<long long>(a.N) * (at % 16 == 0 ? a.H / E : a.H);
  const unsigned grid = static_cast<unsigned>(min((threads + 255) / 256, 1ll << 20));
  if (at % 16 == 0) {
    lookup_kernel<T, E><<<grid, 256, 0, s>>>(a);
  } else {
    lookup_kernel<T, 1><<<grid, 256, 0, s>>>(a);
  }
  return cudaGetLastError();
}

template <typename T, typename G>
cudaError_t grad(const TbEmbeddingGradArgs& a, cudaStream_t s) {
  if (a.zero) {
    const cudaError_t e = cudaMemset2DAsync(a.grad, a.ld_grad * sizeof(G), 0, a.H * sizeof(G), a.V, s);
    if (e != cudaSuccess) return e;
  }
  if (a.N == 0) return cudaSuccess;
  grad_kernel<T, G><<<a.N, 128, 0, s>>>(a);
  return cudaGetLastError();
}

template <typename T>
cudaError_t grad_of(const TbEmbeddingGradArgs& a, cudaStream_t s) {
  switch (a.grad_dtype) {
    case TB_BF16: return grad<T, __nv_bfloat16>(a, s);
    case TB_F16: return grad<T, __half>(a, s);
    case TB_F32: return grad<T, float>(a, s);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace

extern "C" int tb_embedding(const TbEmbeddingArgs* args, cudaStream_t s) {
  const TbEmbeddingArgs& a = *args;
  if (a.N < 0 || a.H < 1 || a.V < 1) return static_cast<int>(cudaErrorInvalidValue);
  if (a.N == 0) return 0;
  switch (a.dtype) {
    case TB_BF16: return static_cast<int>(lookup<__nv_bfloat16>(a, s));
    case TB_F16: return static_cast<int>(lookup<__half>(a, s));
    case TB_F32: return static_cast<int>(lookup<float>(a, s));
    default: return static_cast<int>(cudaErrorInvalidValue);
  }
}

extern "C" size_t tb_embedding_grad_ws_bytes(int N, int H, int V) { return 0; }

extern "C" int tb_embedding_grad(const TbEmbeddingGradArgs* args, cudaStream_t s) {
  const TbEmbeddingGradArgs& a = *args;
  if (a.N < 0 || a.H < 1 || a.V < 1) return static_cast<int>(cudaErrorInvalidValue);
  switch (a.dtype) {
    case TB_BF16: return static_cast<int>(grad_of<__nv_bfloat16>(a, s));
    case TB_F16: return static_cast<int>(grad_of<__half>(a, s));
    case TB_F32: return static_cast<int>(grad_of<float>(a, s));
    default: return static_cast<int>(cudaErrorInvalidValue);
  }
}
