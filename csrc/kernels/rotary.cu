// Rotary positions in their general form: the half layout (pairs (i, i + R/2))
// and the interleaved one (pairs (2i, 2i + 1)), the first R of D dimensions of
// a head, any row and head strides, bf16 / fp16 / fp32.  For the pair (a, b)
// and its table entry (c, s) of the row's position
//
//   y_a = c a - s b,   y_b = c b + s a        (backward: s -> -s),
//
// in fp32 with one rounding at the store; scaling for long contexts lives in
// the table.  Dimensions behind R are copied (in place: left alone, but NaN like the
// others in rows whose position is past the table).
//
// The kernel moves every element once in and once out and does 3 flops per
// element, so memory bounds it: 16,383 rows x 40 heads x 128 in bf16 take 53 us on
// one B200, 6.3 TB/s (97% of its copy rate).
#include <math.h>

#include "device_common.cuh"
#include "kernels.h"
#include "vec_io.cuh"

namespace {

// Threads of a block, and the blocks of an SM that the registers have to allow.
constexpr int threads_of(int hu) { return hu == 8 ? 128 : 256; }
constexpr int blocks_of(int hu) { return hu == 4 ? 3 : 4; }

// A thread holds one unit, two vectors of NP elements, of HU heads of a token
// (every HS-th), so it reads its table entries once: read anew for each head they
// are twice the bytes of a bf16 row, out of L1 (88 us with HU = 1, 58 with 4, 53
// with 8 at the size above).  Rotated units hold NP pairs (half layout: NP elements
// of each half; interleaved: 2 NP neighbours), the others 2 NP copied elements.  All loads are issued before the first product.
template <typename T, int NP, int HU, bool INTER>
__global__ void __launch_bounds__(threads_of(HU), blocks_of(HU))
    rotary_kernel(TbRotaryArgs a, int rot_units, int units, int HS, int tokens) {
  const T* x = static_cast<const T*>(a.x);
  T* y = static_cast<T*>(a.y);
  const int half = a.R / 2, per = units * HS;
  const int tk = threadIdx.x / per;
  const long long t = blockIdx.x * static_cast<long long>(tokens) + tk;
  if (tk >= tokens || t >= a.T) return;
  const int p = a.pos[t];
  const bool bad = p >= a.max_pos;
  const float sgn = a.transpose ? -1.f : 1.f;
  for (int i = threadIdx.x - tk * per; i < per; i += blockDim.x) {  // (more than one round only where per > blockDim.x)
    const int u = i % units, h0 = i / units;
    const bool turn = u < rot_units && p >= 0 && !bad;
    const int o1 = INTER || u >= rot_units ? u * 2 * NP : u * NP;
    const int o2 = INTER || u >= rot_units ? o1 + NP : o1 + half;
    const T* xr = x + t * a.xs_t;
    T* yr = y + t * a.ys_t;
    tb::Packed<T, NP> lo[HU], hi[HU];
    float cs[2 * NP];
    if (turn) tb::load_vec<float, 2 * NP>(a.table + (static_cast<long long>(p) * half + u * NP) * 2, cs);
#pragma unroll
    for (int k = 0; k < HU; ++k)
      if (h0 + k * HS < a.H) {
        lo[k].load(xr + (h0 + k * HS) * a.xs_h + o1);
        hi[k].load(xr + (h0 + k * HS) * a.xs_h + o2);
      }
    if (bad) break;  // (here, so that the loads do not wait for the position)
#pragma unroll
    for (int k = 0; k < HU; ++k)
      if (h0 + k * HS < a.H) {
        float f[NP], g[NP];
        lo[k].unpack(f);
        hi[k].unpack(g);
        if (turn) {
#pragma unroll
          for (int j = 0; j < NP; ++j) {
            const float c = cs[2 * j], sn = sgn * cs[2 * j + 1];
            float& v = INTER ? (2 * j < NP ? f[2 * j % NP] : g[2 * j % NP]) : f[j];
            float& w = INTER ? (2 * j + 1 < NP ? f[(2 * j + 1) % NP] : g[(2 * j + 1) % NP]) : g[j];
            const float nv = v * c - w * sn;
            w = w * c + v * sn;
            v = nv;
          }
        }
        tb::store_vec<T, NP>(yr + (h0 + k * HS) * a.ys_h + o1, f);
        tb::store_vec<T, NP>(yr + (h0 + k * HS) * a.ys_h + o2, g);
      }
  }
  if (bad) {  // the whole row becomes NaN, with the dimensions that have no unit in place
    if (a.err && threadIdx.x == tk * per) atomicCAS(a.err, 0, 1);
    float f[NP];
#pragma unroll
    for (int j = 0; j < NP; ++j) f[j] = NAN;
    const int row = a.D / NP, step = min(per, static_cast<int>(blockDim.x));
    for (int i = threadIdx.x - tk * per; i < a.H * row; i += step)
      tb::store_vec<T, NP>(y + t * a.ys_t + i / row * a.ys_h + i % row * NP, f);
  }
}

template <typename T, int NP, int HU, bool INTER>
int launch_vec(const TbRotaryArgs& a, cudaStream_t s) {
  const int rot_units = a.R / 2 / NP;
  const int units = rot_units + (a.x == a.y ? 0 : (a.D - a.R) / (2 * NP));
  const int HS = (a.H + HU - 1) / HU;
  const long long per = static_cast<long long>(units) * HS;
  constexpr int kThreads = threads_of(HU);
  const int tokens = per >= kThreads ? 1 : static_cast<int>(kThreads / per);
  const int grid = static_cast<int>((a.T + (tokens - 1ll)) / tokens);  // (T + tokens can pass 31 bits)
  rotary_kernel<T, NP, HU, INTER><<<grid, kThreads, 0, s>>>(a, rot_units, units, HS, tokens);
  return static_cast<int>(cudaGetLastError());
}

// Whether vectors of NP elements fit the sizes, the strides and the addresses.
template <typename T, int NP>
bool fits(const TbRotaryArgs& a) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.y);
  return a.R / 2 % NP == 0 && (a.D - a.R) % (2 * NP) == 0 && a.xs_t % NP == 0 && a.xs_h % NP == 0 &&
         a.ys_t % NP == 0 && a.ys_h % NP == 0 && at % (NP * sizeof(T)) == 0 &&
         reinterpret_cast<uintptr_t>(a.table) % 16 == 0;
}

// Heads per thread.  One where more would leave an SM (of 148) fewer than 1,024
// threads (64 rows x 14 heads take 2.2 us so, mostly launch, with four 2.9) or find no
// heads to hold (100,000 rows x 1 head x 128: 15.4 us, with four 20.4).  Else four, and
// eight in smaller blocks for 8 or more heads in vectors of 16 bytes: 53 against 58 us
// at the size above, 40 against 46 for 60,000 rows x 8 heads x 128, and 20 either way for
// 16,000 rows x 16 heads x 80 (40 rotated), which are in vectors of 8 bytes.
template <typename T, int NP, bool INTER>
int launch_heads(const TbRotaryArgs& a, cudaStream_t s) {
  const bool few = static_cast<long long>(a.T) * a.H * (a.D / (2 * NP)) < 4ll * 148 * 1024;
  if (few || a.H == 1) return launch_vec<T, NP, 1, INTER>(a, s);
  if constexpr (NP * sizeof(T) == 16)
    if (a.H >= 8) return launch_vec<T, NP, 8, INTER>(a, s);
  return launch_vec<T, NP, 4, INTER>(a, s);
}

template <typename T, int NP>
int launch_layout(const TbRotaryArgs& a, cudaStream_t s) {
  return a.interleaved ? launch_heads<T, NP, true>(a, s) : launch_heads<T, NP, false>(a, s);
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
  if (a.R <= 0 || a.R % 2 || a.D % 2 || a.R > a.D || a.H > 0x7fffffff / a.D || a.max_pos <= 0)
    return static_cast<int>(cudaErrorInvalidValue);
  switch (a.dtype) {
    case TB_BF16: return launch_type<__nv_bfloat16>(a, s);
    case TB_F16: return launch_type<__half>(a, s);
    case TB_F32: return launch_type<float>(a, s);
  }
  return static_cast<int>(cudaErrorInvalidValue);
}
