// The 8-bit paged KV cache: rows quantised as they are written and read back.
//
// A row (one token, one KV head, D values) gets its own scale, so the largest
// value of the row maps to the largest code:
//
//   a = max(max_i |x_i|, 2^-90),   s = a / 448,   code_i = e4m3(x_i * (448 / a)).
//
// The floor keeps 448 / a finite for a row of zeros (and of denormals).  Two
// fp32 roundings come before the one to e4m3, so a code can differ from the
// exactly scaled one only where that lies within 2^-23 of a rounding border.  A
// NaN anywhere in a row makes its scale NaN, an infinity makes it infinite and
// the row read back NaN or infinite: nothing is silently clipped.
//
// Reads and writes are one pass over the rows and a few operations per
// element: memory bounds both directions, launch latency the decode step.
#include <math.h>

#include "device_common.cuh"
#include "kernels.h"
#include "vec_io.cuh"

namespace {

constexpr float kMaxCode = 448.f;
constexpr uint32_t kMinAmaxBits = 0x12800000u;  // 2^-90

// The cache row (in rows of D codes) of KV head 0 of a token's slot, or -1:
// padding, or (with *err set) a sequence, position or block out of range.
// Head h is bs rows further per head.
__device__ __forceinline__ long long slot_row(const TbQuantCache& c, int seq, int pos, int* err) {
  if (seq < 0 || pos < 0) return -1;
  const int b = pos / c.bs;
  int blk = -1;
  if (seq < c.num_seqs && b < c.max_blocks) blk = c.block_table[static_cast<long long>(seq) * c.max_blocks + b];
  if (blk < 0 || blk >= c.num_blocks) {
    if (err) atomicCAS(err, 0, 1);
    return -1;
  }
  return static_cast<long long>(blk) * c.Hk * c.bs + (pos - b * c.bs);
}

// e4m3 codes of four floats, the first in the low byte; saturates, keeps NaN.
__device__ __forceinline__ uint32_t to_e4m3x4(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return static_cast<uint32_t>(lo) | static_cast<uint32_t>(hi) << 16;
}

// Four floats from codes (exact: every e4m3 value is an fp16 value).
__device__ __forceinline__ void from_e4m3x4(uint32_t w, float (&f)[4]) {
  uint32_t lo, hi;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(lo) : "h"(static_cast<uint16_t>(w)));
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(hi) : "h"(static_cast<uint16_t>(w >> 16)));
  const float2 a = __half22float2(*reinterpret_cast<__half2*>(&lo));
  const float2 b = __half22float2(*reinterpret_cast<__half2*>(&hi));
  f[0] = a.x;
  f[1] = a.y;
  f[2] = b.x;
  f[3] = b.y;
}

template <typename T>
__device__ __forceinline__ void load4(const T* p, bool aligned, float (&f)[4]) {
  if (aligned) {
    tb::load_vec<T, 4>(p, f);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = tb::to_f32(p[i]);
  }
}
template <typename T>
__device__ __forceinline__ void store4(T* p, bool aligned, const float (&f)[4]) {
  if (aligned) {
    tb::store_vec<T, 4>(p, f);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = tb::from_f32<T>(f[i]);
  }
}

// D / 8 lanes per row; a lane holds two vectors of four elements: both members
// of its pairs where the row is rotated in the half layout, else 8 neighbours.
// Rows of a token: Hk of k, Hk of v, then (rotated calls) Hq of q.
template <typename T, int D>
__global__ void kv_quant_write_kernel(TbKvQuantWriteArgs a, int slots, bool aligned) {
  constexpr int L = D / 8;
  const int l = threadIdx.x % L;
  const int Hk = a.cache.Hk, R = a.rot.R;
  const long long rows = static_cast<long long>(a.T) * slots;
  const long long per = static_cast<long long>(gridDim.x) * (blockDim.x / L);
  // every lane of a warp runs the same number of rounds: the shuffles need all of them
  for (long long r0 = blockIdx.x * static_cast<long long>(blockDim.x / L); r0 < rows; r0 += per) {
    const long long r = r0 + threadIdx.x / L;
    const bool live = r < rows;
    const long long t = live ? r / slots : 0;
    const int slot = live ? static_cast<int>(r - t * slots) : 0;
    const int kind = slot < Hk ? 0 : slot < 2 * Hk ? 1 : 2;  // k, v, q
    const int h = slot - (kind == 0 ? 0 : kind == 1 ? Hk : 2 * Hk);
    const int p = a.pos[t], seq = a.seq[t];
    const bool turn = R > 0 && kind != 1 && 8 * l < R;
    const bool half = turn && !a.rot.interleaved;
    const int o1 = half ? 4 * l : 8 * l, o2 = half ? 4 * l + R / 2 : 8 * l + 4;
    const bool past = R > 0 && p >= a.rot.max_pos;
    const T* x = kind == 0   ? static_cast<const T*>(a.k) + t * a.ks_t + h * a.ks_h
                 : kind == 1 ? static_cast<const T*>(a.v) + t * a.vs_t + h * a.vs_h
                             : static_cast<const T*>(a.rot.x) + t * a.rot.xs_t + h * a.rot.xs_h;
    float f[4] = {}, g[4] = {};
    if (live) {
      load4<T>(x + o1, aligned, f);
      load4<T>(x + o2, aligned, g);
    }
    if (turn && p >= 0 && !past) {
      const float2* tab = reinterpret_cast<const float2*>(a.rot.table) + static_cast<long long>(p) * (R / 2) + 4 * l;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 cs = tab[i];
        float& v = half ? f[i] : i < 2 ? f[2 * i] : g[2 * i - 4];
        float& w = half ? g[i] : i < 2 ? f[2 * i + 1] : g[2 * i - 3];
        const float nv = v * cs.x - w * cs.y;
        w = w * cs.x + v * cs.y;
        v = nv;
      }
    }
    // absolute values compare like their bits, and NaN is above infinity
    uint32_t m = kMinAmaxBits;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = max(m, max(__float_as_uint(f[i]) & 0x7fffffffu, __float_as_uint(g[i]) & 0x7fffffffu));
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (!live) continue;
    if (past && l == 0 && a.rot.err) atomicCAS(a.rot.err, 0, 1);
    if (kind == 2) {
      T* y = static_cast<T*>(a.rot.y) + t * a.rot.ys_t + h * a.rot.ys_h;
      if (past) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = g[i] = NAN;
      }
      store4<T>(y + o1, aligned, f);
      store4<T>(y + o2, aligned, g);
      continue;
    }
    long long row = past ? -1 : slot_row(a.cache, seq, p, a.rot.err);
    if (row < 0) continue;
    row += static_cast<long long>(h) * a.cache.bs;
    const float amax = __uint_as_float(m), inv = __fdiv_rn(kMaxCode, amax);
    uint8_t* c = static_cast<uint8_t*>(kind == 0 ? a.cache.kc : a.cache.vc) + row * D;
    *reinterpret_cast<uint32_t*>(c + o1) = to_e4m3x4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv);
    *reinterpret_cast<uint32_t*>(c + o2) = to_e4m3x4(g[0] * inv, g[1] * inv, g[2] * inv, g[3] * inv);
    if (l == 0) (kind == 0 ? a.cache.ks : a.cache.vs)[row] = __fdiv_rn(amax, kMaxCode);
  }
}

template <typename T, int D>
__global__ void kv_quant_read_kernel(TbKvQuantReadArgs a, bool aligned) {
  constexpr int L = D / 8;
  const int Hk = a.cache.Hk;
  const long long total = static_cast<long long>(a.T) * 2 * Hk * L;
  for (long long e = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x; e < total;
       e += static_cast<long long>(gridDim.x) * blockDim.x) {
    const int l = static_cast<int>(e % L);
    const long long r = e / L, t = r / (2 * Hk);
    const int slot = static_cast<int>(r - t * (2 * Hk)), h = slot % Hk;
    const bool is_v = slot >= Hk;
    long long row = slot_row(a.cache, a.seq[t], a.pos[t], l == 0 ? a.err : nullptr);
    if (row < 0) continue;
    row += static_cast<long long>(h) * a.cache.bs;
    const uint2 w = *reinterpret_cast<const uint2*>(
        static_cast<const uint8_t*>(is_v ? a.cache.vc : a.cache.kc) + row * D + 8 * l);
    const float s = (is_v ? a.cache.vs : a.cache.ks)[row];
    float f[4], g[4];
    from_e4m3x4(w.x, f);
    from_e4m3x4(w.y, g);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[i] *= s;
      g[i] *= s;
    }
    T* y = is_v ? static_cast<T*>(a.v) + t * a.vs_t + h * a.vs_h : static_cast<T*>(a.k) + t * a.ks_t + h * a.ks_h;
    store4<T>(y + 8 * l, aligned, f);
    store4<T>(y + 8 * l + 4, aligned, g);
  }
}

// Whether every row of a [T, H, D] view starts on a vector of four elements.
bool rows_aligned(const void* p, long long st, long long sh, int dtype) {
  const int bytes = dtype == TB_F32 ? 16 : 8;
  return reinterpret_cast<uintptr_t>(p) % bytes == 0 && st % 4 == 0 && sh % 4 == 0;
}

int grid_of(long long threads) {
  const long long b = (threads + 255) / 256;
  return static_cast<int>(b < 1184 ? b : 1184);
}

template <typename T, int D>
int write_as(const TbKvQuantWriteArgs& a, cudaStream_t s) {
  const int slots = 2 * a.cache.Hk + (a.rot.x ? a.rot.H : 0);
  bool al = rows_aligned(a.k, a.ks_t, a.ks_h, a.rot.dtype) && rows_aligned(a.v, a.vs_t, a.vs_h, a.rot.dtype);
  if (a.rot.x)
    al = al && rows_aligned(a.rot.x, a.rot.xs_t, a.rot.xs_h, a.rot.dtype) &&
         rows_aligned(a.rot.y, a.rot.ys_t, a.rot.ys_h, a.rot.dtype);
  kv_quant_write_kernel<T, D>
      <<<grid_of(static_cast<long long>(a.T) * slots * (D / 8)), 256, 0, s>>>(a, slots, al);
  return static_cast<int>(cudaGetLastError());
}

template <typename T, int D>
int read_as(const TbKvQuantReadArgs& a, cudaStream_t s) {
  const bool al = rows_aligned(a.k, a.ks_t, a.ks_h, a.dtype) && rows_aligned(a.v, a.vs_t, a.vs_h, a.dtype);
  kv_quant_read_kernel<T, D>
      <<<grid_of(static_cast<long long>(a.T) * 2 * a.cache.Hk * (D / 8)), 256, 0, s>>>(a, al);
  return static_cast<int>(cudaGetLastError());
}

bool cache_ok(const TbQuantCache& c) {
  return c.Hk > 0 && c.bs > 0 && c.num_blocks >= 0 && (c.D == 64 || c.D == 128 || c.D == 256);
}

template <typename T>
int write_d(const TbKvQuantWriteArgs& a, cudaStream_t s) {
  return a.cache.D == 64 ? write_as<T, 64>(a, s) : a.cache.D == 128 ? write_as<T, 128>(a, s) : write_as<T, 256>(a, s);
}
template <typename T>
int read_d(const TbKvQuantReadArgs& a, cudaStream_t s) {
  return a.cache.D == 64 ? read_as<T, 64>(a, s) : a.cache.D == 128 ? read_as<T, 128>(a, s) : read_as<T, 256>(a, s);
}

}  // namespace

extern "C" int tb_kv_quant_write(const TbKvQuantWriteArgs* args, cudaStream_t s) {
  const TbKvQuantWriteArgs& a = *args;
  if (a.T <= 0) return 0;
  if (!cache_ok(a.cache) || a.rot.R < 0 || a.rot.R % 8 || a.rot.R > a.cache.D || (a.rot.R > 0) != (a.rot.max_pos > 0))
    return static_cast<int>(cudaErrorInvalidValue);
  switch (a.rot.dtype) {
    case TB_BF16: return write_d<__nv_bfloat16>(a, s);
    case TB_F16: return write_d<__half>(a, s);
    case TB_F32: return write_d<float>(a, s);
  }
  return static_cast<int>(cudaErrorInvalidValue);
}

extern "C" int tb_kv_quant_read(const TbKvQuantReadArgs* args, cudaStream_t s) {
  const TbKvQuantReadArgs& a = *args;
  if (a.T <= 0) return 0;
  if (!cache_ok(a.cache)) return static_cast<int>(cudaErrorInvalidValue);
  switch (a.dtype) {
    case TB_BF16: return read_d<__nv_bfloat16>(a, s);
    case TB_F16: return read_d<__half>(a, s);
    case TB_F32: return read_d<float>(a, s);
  }
  return static_cast<int>(cudaErrorInvalidValue);
}
