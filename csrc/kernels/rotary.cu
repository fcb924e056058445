// Rotary positions in their general form: the half layout (pairs (i, i + R/2))
// and the interleaved one (pairs (2i, 2i + 1)), the first R of D dimensions of
// a head, any row and head strides, bf16 / fp16 / fp32.  For the pair (a, b)
// and its table entry (c, s) of the row's position
//
//   y_a = c a - s b,   y_b = c b + s a        (backward: s -> -s),
//
// in fp32 with one rounding at the store; scaling for long contexts lives in
// the table.  Dimensions behind R are copied (in place: left alone).
//
// The kernel moves every element once in and once out and does 3 flops per
// element, so memory bounds it.
#include <math.h>

#include "device_common.cuh"
#include "kernels.h"
#include "vec_io.cuh"

namespace {

// One thread: one unit of one head, two vectors of NP elements.  Rotated units
// hold NP pairs (half layout: NP elements of each half; interleaved: 2 NP
// neighbours), the others 2 NP copied elements.
template <typename T, int NP, bool INTER>
__global__ void rotary_kernel(TbRotaryArgs a, int rot_units, int units) {
  const long long total = static_cast<long long>(a.T) * a.H * units;
  const T* x = static_cast<const T*>(a.x);
  T* y = static_cast<T*>(a.y);
  const float2* table = reinterpret_cast<const float2*>(a.table);
  const int half = a.R / 2;
  const float sgn = a.transpose ? -1.f : 1.f;
  for (long long e = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x; e < total;
       e += static_cast<long long>(gridDim.x) * blockDim.x) {
    const int u = static_cast<int>(e % units);
    const long long r = e / units;
    const int h = static_cast<int>(r % a.H);
    const long long t = r / a.H;
    const int p = a.pos[t];
    const bool bad = p >= a.max_pos;
    if (bad && a.err && u == 0 && h == 0) atomicCAS(a.err, 0, 1);
    const int o1 = INTER || u >= rot_units ? u * 2 * NP : u * NP;
    const int o2 = INTER || u >= rot_units ? o1 + NP : o1 + half;
    const T* xr = x + t * a.xs_t + static_cast<long long>(h) * a.xs_h;
    T* yr = y + t * a.ys_t + static_cast<long long>(h) * a.ys_h;
    float f[NP], g[NP];
    tb::load_vec<T, NP>(xr + o1, f);
    tb::load_vec<T, NP>(xr + o2, g);
    if (bad) {
#pragma unroll
      for (int i = 0; i < NP; ++i) f[i] = g[i] = NAN;
    } else if (u < rot_units && p >= 0) {
      const float2* tab = table + static_cast<long long>(p) * half + u * NP;
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const float2 cs = tab[i];
        const float sn = sgn * cs.y;
        float& v = INTER ? (2 * i < NP ? f[2 * i % NP] : g[2 * i % NP]) : f[i];
        float& w = INTER ? (2 * i + 1 < NP ? f[(2 * i + 1) % NP] : g[(2 * i + 1) % NP]) : g[i];
        const float nv = v * cs.x - w * sn;
        w = w * cs.x + v * sn;
        v = nv;
      }
    }
    tb::store_vec<T, NP>(yr + o1, f);
    tb::store_vec<T, NP>(yr + o2, g);
  }
}

template <typename T, int NP, bool INTER>
int launch_vec(const TbRotaryArgs& a, cudaStream_t s) {
  const int rot_units = a.R / 2 / NP;
  const int units = rot_units + (a.x == a.y ? 0 : (a.D - a.R) / (2 * NP));
  const long long total = static_cast<long long>(a.T) * a.H * units;
  const long long blocks = (total + 255) / 256;
  rotary_kernel<T, NP, INTER><<<static_cast<int>(blocks < 1184 ? blocks : 1184), 256, 0, s>>>(a, rot_units, units);
  return static_cast<int>(cudaGetLastError());
}

// Whether vectors of NP elements fit the sizes, the strides and the addresses.
template <typename T, int NP>
bool fits(const TbRotaryArgs& a) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.y);
  return a.R / 2 % NP == 0 && (a.D - a.R) % (2 * NP) == 0 && a.xs_t % NP == 0 && a.xs_h % NP == 0 &&
         a.ys_t % NP == 0 && a.ys_h % NP == 0 && at % (NP * sizeof(T)) == 0;
}

template <typename T, int NP>
int launch_layout(const TbRotaryArgs& a, cudaStream_t s) {
  return a.interleaved ? launch_vec<T, NP, true>(a, s) : launch_vec<T, NP, false>(a, s);
}

// The widest vectors that fit: 16 bytes, 8 bytes, or single elements.
template <typename T>
int launch_type(const TbRotaryArgs& a, cudaStream_t s) {
  constexpr int kWide = 16 / static_cast<int>(sizeof(T));
  if (fits<T, kWide>(a)) return launch_layout<T, kWide>(a, s);
  if (fits<T, kWide / 2>(a)) return launch_layout<T, kWide / 2>(a, s);
  return launch_layout<T, 1>(a, s);
}

}  // namespace

extern "C" int tb_rotary(const TbRotaryArgs* args, cudaStream_t s) {
  const TbRotaryArgs& a = *args;
  if (a.T <= 0 || a.H <= 0) return 0;
  if (a.R <= 0 || a.R % 2 || a.D % 2 || a.R > a.D || a.max_pos <= 0) return static_cast<int>(cudaErrorInvalidValue);
  switch (a.dtype) {
    case TB_BF16: return launch_type<__nv_bfloat16>(a, s);
    case TB_F16: return launch_type<__half>(a, s);
    case TB_F32: return launch_type<float>(a, s);
  }
  return static_cast<int>(cudaErrorInvalidValue);
}
