// Attention of one new token per sequence over the 8-bit paged KV cache:
//
//   a_j = scale * ks_j * (q . k_j),   out = sum_j softmax(a)_j * vs_j * v_j
//
// with k_j, v_j the e4m3 codes and ks_j, vs_j the scales of token j.  One pass
// over the context with the running maximum and sum of the softmax in fp32.
#include <math.h>

#include "device_common.cuh"
#include "kernels.h"
#include "vec_io.cuh"

namespace {

__device__ __forceinline__ float code_value(uint8_t c) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(c)));
  return __half2float(__ushort_as_half(static_cast<unsigned short>(r & 0xffff)));
}

// One CTA per (sequence, query head): each of its four warps takes every
// fourth token, a lane D / 32 dimensions; the warps' partials are joined in
// shared memory.
template <typename T, int D>
__global__ void decode_attn_quant_kernel(TbDecodeAttnQuantArgs a) {
  constexpr int E = D / 32;
  __shared__ float sm[4], sl[4], so[4][D];
  const int b = blockIdx.x / a.Hq, h = blockIdx.x % a.Hq, kh = h / (a.Hq / a.cache.Hk);
  const int w = threadIdx.x / 32, lane = threadIdx.x % 32;
  const TbQuantCache& c = a.cache;
  const T* q = static_cast<const T*>(a.q) + b * a.qs_b + h * a.qs_h;
  float qf[E], acc[E] = {};
#pragma unroll
  for (int i = 0; i < E; ++i) qf[i] = tb::to_f32(q[lane + 32 * i]) * a.scale;
  float m = -INFINITY, l = 0.f;
  const long long cap = static_cast<long long>(c.max_blocks) * c.bs, want = a.ctx_len[b];
  if (want > cap && a.err && threadIdx.x == 0) atomicCAS(a.err, 0, 1);
  const long long ctx = want < cap ? want : cap;
  for (long long j = w; j < ctx; j += 4) {
    const int pb = static_cast<int>(j / c.bs);
    const int blk = c.block_table[static_cast<long long>(b) * c.max_blocks + pb];
    if (blk < 0 || blk >= c.num_blocks) {
      if (a.err && lane == 0) atomicCAS(a.err, 0, 1);
      continue;
    }
    const long long row = (static_cast<long long>(blk) * c.Hk + kh) * c.bs + (j - static_cast<long long>(pb) * c.bs);
    const uint8_t* kr = static_cast<const uint8_t*>(c.kc) + row * D;
    const uint8_t* vr = static_cast<const uint8_t*>(c.vc) + row * D;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) s += qf[i] * code_value(kr[lane + 32 * i]);
    s = tb::warp_sum(s) * c.ks[row];
    const float mn = fmaxf(m, s), mr = mn == -INFINITY ? 0.f : mn;
    const float cor = __expf(m - mr), p = __expf(s - mr);
    l = l * cor + p;
    const float pv = p * c.vs[row];
#pragma unroll
    for (int i = 0; i < E; ++i) acc[i] = acc[i] * cor + pv * code_value(vr[lane + 32 * i]);
    m = mn;
  }
  if (lane == 0) {
    sm[w] = m;
    sl[w] = l;
  }
#pragma unroll
  for (int i = 0; i < E; ++i) so[w][lane + 32 * i] = acc[i];
  __syncthreads();
  float M = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  if (M == -INFINITY) M = 0.f;
  float L = 0.f;
  for (int i = 0; i < 4; ++i) L += sl[i] * __expf(sm[i] - M);
  T* o = static_cast<T*>(a.out) + b * a.os_b + h * a.os_h;
  for (int d = threadIdx.x; d < D; d += blockDim.x) {
    float v = 0.f;
    for (int i = 0; i < 4; ++i) v += so[i][d] * __expf(sm[i] - M);
    o[d] = tb::from_f32<T>(L == 0.f ? 0.f : v / L);
  }
}

template <typename T>
int launch(const TbDecodeAttnQuantArgs& a, cudaStream_t s) {
  const int grid = a.B * a.Hq;
  switch (a.cache.D) {
    case 64: decode_attn_quant_kernel<T, 64><<<grid, 128, 0, s>>>(a); break;
    case 128: decode_attn_quant_kernel<T, 128><<<grid, 128, 0, s>>>(a); break;
    case 256: decode_attn_quant_kernel<T, 256><<<grid, 128, 0, s>>>(a); break;
    default: return static_cast<int>(cudaErrorInvalidValue);
  }
  return static_cast<int>(cudaGetLastError());
}

}  // namespace

extern "C" size_t tb_decode_attention_quant_ws_bytes(int, int, int, int, int) { return 0; }

extern "C" int tb_decode_attention_quant(const TbDecodeAttnQuantArgs* args, cudaStream_t s) {
  const TbDecodeAttnQuantArgs& a = *args;
  if (a.B <= 0 || a.Hq <= 0) return 0;
  if (a.cache.Hk <= 0 || a.Hq % a.cache.Hk || a.cache.bs <= 0) return static_cast<int>(cudaErrorInvalidValue);
  if (a.dtype == TB_BF16) return launch<__nv_bfloat16>(a, s);
  if (a.dtype == TB_F16) return launch<__half>(a, s);
  return static_cast<int>(cudaErrorInvalidValue);
}
