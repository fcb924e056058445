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
__device__ __forceinline__ void store4(T* p, bool aligned, const float (&f)[4]) {
  if (aligned) {
    tb::store_vec<T, 4>(p, f);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = tb::from_f32<T>(f[i]);
  }
}

// One pass over the rows: D / 8 lanes per row, eight elements each, U rows per
// lane (all loaded before the first is reduced).  ROT: q and k rows are rotated; a
// lane then holds both members of its pairs (half layout: two vectors of four),
// else eight neighbours.  Rows of a token: Hk of k, Hk of v, then Hq of q.
template <typename T, int D, int U, bool ROT>
__global__ void __launch_bounds__(256) kv_quant_write_kernel(TbKvQuantWriteArgs a, int slots, bool aligned) {
  constexpr int L = D / 8, kRows = 256 / L;  // lanes per row, rows per block and round
  const int l = threadIdx.x % L;
  const int Hk = a.cache.Hk, R = ROT ? a.rot.R : 0;
  const long long rows = static_cast<long long>(a.T) * slots;
  const long long r0 = blockIdx.x * static_cast<long long>(U * kRows) + threadIdx.x / L;
  int p[U], seq[U], slot[U];
  long long t[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const long long r = r0 + u * kRows;
    t[u] = r >> 32 ? r / slots : static_cast<uint32_t>(r) / static_cast<uint32_t>(slots);
    slot[u] = static_cast<int>(r - t[u] * slots);
    p[u] = seq[u] = -1;
    if (r < rows) {
      p[u] = a.pos[t[u]];
      seq[u] = a.seq[t[u]];
    } else {
      t[u] = -1;
    }
  }
  tb::Packed<T, 4> x0[U], x1[U];
  long long row[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int kind = slot[u] < Hk ? 0 : slot[u] < 2 * Hk ? 1 : 2, h = slot[u] - kind * Hk;  // k, v, q
    const bool turn = ROT && kind != 1 && 8 * l < R, half = turn && !a.rot.interleaved;
    const int o1 = half ? 4 * l : 8 * l, o2 = half ? 4 * l + R / 2 : 8 * l + 4;
    const bool past = ROT && p[u] >= a.rot.max_pos;
    const T* x = kind == 0   ? static_cast<const T*>(a.k) + t[u] * a.ks_t + h * a.ks_h
                 : kind == 1 ? static_cast<const T*>(a.v) + t[u] * a.vs_t + h * a.vs_h
                             : static_cast<const T*>(a.rot.x) + t[u] * a.rot.xs_t + h * a.rot.xs_h;
    const bool need = t[u] >= 0 && (kind == 2 || (p[u] >= 0 && seq[u] >= 0));
    if (need && aligned) {
      x0[u].load(x + o1);
      x1[u].load(x + o2);
    } else if (need) {
      T* e0 = reinterpret_cast<T*>(&x0[u].raw);
      T* e1 = reinterpret_cast<T*>(&x1[u].raw);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        e0[i] = x[o1 + i];
        e1[i] = x[o2 + i];
      }
    } else {
      x0[u].raw = x1[u].raw = {};
    }
    row[u] = -1;
    if (need && kind < 2 && !past) row[u] = slot_row(a.cache, seq[u], p[u], l == 0 ? a.rot.err : nullptr);
    if (row[u] >= 0) row[u] += static_cast<long long>(h) * a.cache.bs;
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int kind = slot[u] < Hk ? 0 : slot[u] < 2 * Hk ? 1 : 2, h = slot[u] - kind * Hk;
    const bool turn = ROT && kind != 1 && 8 * l < R, half = turn && !a.rot.interleaved;
    const int o1 = half ? 4 * l : 8 * l, o2 = half ? 4 * l + R / 2 : 8 * l + 4;
    const bool past = ROT && p[u] >= a.rot.max_pos;
    float f[4], g[4];
    x0[u].unpack(f);
    x1[u].unpack(g);
    if (turn && p[u] >= 0 && !past) {
      const float2* tab = reinterpret_cast<const float2*>(a.rot.table) + static_cast<long long>(p[u]) * (R / 2) + 4 * l;
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
    if (ROT && t[u] >= 0 && past && l == 0 && a.rot.err) atomicCAS(a.rot.err, 0, 1);
    if (ROT && t[u] >= 0 && kind == 2) {
      T* y = static_cast<T*>(a.rot.y) + t[u] * a.rot.ys_t + h * a.rot.ys_h;
      if (past) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = g[i] = NAN;
      }
      store4<T>(y + o1, aligned, f);
      store4<T>(y + o2, aligned, g);
    }
    if (row[u] < 0) continue;
    const float amax = __uint_as_float(m), inv = __fdiv_rn(kMaxCode, amax);
    uint8_t* c = static_cast<uint8_t*>(kind == 0 ? a.cache.kc : a.cache.vc) + row[u] * D;
    const uint32_t c0 = to_e4m3x4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv);
    const uint32_t c1 = to_e4m3x4(g[0] * inv, g[1] * inv, g[2] * inv, g[3] * inv);
    if (ROT) {
      *reinterpret_cast<uint32_t*>(c + o1) = c0;
      *reinterpret_cast<uint32_t*>(c + o2) = c1;
    } else {
      *reinterpret_cast<uint2*>(c + o1) = make_uint2(c0, c1);
    }
    if (l == 0) (kind == 0 ? a.cache.ks : a.cache.vs)[row[u]] = __fdiv_rn(amax, kMaxCode);
  }
}

// D / 16 lanes per row, sixteen codes each, U rows per lane.
template <typename T, int D, int U>
__global__ void __launch_bounds__(256) kv_quant_read_kernel(TbKvQuantReadArgs a, bool aligned) {
  constexpr int L = D / 16, kRows = 256 / L;
  const int l = threadIdx.x % L, Hk = a.cache.Hk, slots = 2 * Hk;
  const long long rows = static_cast<long long>(a.T) * slots;
  const long long r0 = blockIdx.x * static_cast<long long>(U * kRows) + threadIdx.x / L;
  long long t[U], row[U];
  int slot[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const long long r = r0 + u * kRows;
    t[u] = r >> 32 ? r / slots : static_cast<uint32_t>(r) / static_cast<uint32_t>(slots);
    slot[u] = static_cast<int>(r - t[u] * slots);
    row[u] = -1;
    if (r < rows) row[u] = slot_row(a.cache, a.seq[t[u]], a.pos[t[u]], l == 0 ? a.err : nullptr);
    if (row[u] >= 0) row[u] += static_cast<long long>(slot[u] < Hk ? slot[u] : slot[u] - Hk) * a.cache.bs;
  }
  uint4 w[U];
  float s[U];
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (row[u] >= 0) {
      w[u] = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(slot[u] < Hk ? a.cache.kc : a.cache.vc) +
                                             row[u] * D + 16 * l);
      s[u] = (slot[u] < Hk ? a.cache.ks : a.cache.vs)[row[u]];
    }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (row[u] < 0) continue;
    T* y = (slot[u] < Hk ? static_cast<T*>(a.k) + t[u] * a.ks_t + slot[u] * a.ks_h
                         : static_cast<T*>(a.v) + t[u] * a.vs_t + (slot[u] - Hk) * a.vs_h) +
           16 * l;
    const uint32_t ww[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
    float f[16];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float q[4];
      from_e4m3x4(ww[i], q);
#pragma unroll
      for (int e = 0; e < 4; ++e) f[4 * i + e] = q[e] * s[u];
    }
    if (aligned) {
      tb::store_vec<T, 16>(y, f);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) y[i] = tb::from_f32<T>(f[i]);
    }
  }
}

// Whether every row of a [T, H, D] view starts on a multiple of `bytes`.
bool rows_aligned(const void* p, long long st, long long sh, int dtype, int bytes) {
  const int e = dtype == TB_F32 ? 4 : 2;
  return reinterpret_cast<uintptr_t>(p) % bytes == 0 && st * e % bytes == 0 && sh * e % bytes == 0;
}

// Rows per lane: as many as leave every SM 2,048 threads, at most four.
constexpr long long kFullMachine = 148 * 2048;

template <typename T, int D, bool ROT>
int write_rot(const TbKvQuantWriteArgs& a, cudaStream_t s) {
  constexpr int kRows = 256 / (D / 8);
  const int slots = 2 * a.cache.Hk + (a.rot.x ? a.rot.H : 0), v = 4 * (a.rot.dtype == TB_F32 ? 4 : 2);
  bool al = rows_aligned(a.k, a.ks_t, a.ks_h, a.rot.dtype, v) && rows_aligned(a.v, a.vs_t, a.vs_h, a.rot.dtype, v);
  if (a.rot.x)
    al = al && rows_aligned(a.rot.x, a.rot.xs_t, a.rot.xs_h, a.rot.dtype, v) &&
         rows_aligned(a.rot.y, a.rot.ys_t, a.rot.ys_h, a.rot.dtype, v);
  const long long rows = static_cast<long long>(a.T) * slots;
  const int u = rows * (D / 8) >= 4 * kFullMachine ? 4 : 1;
  const long long grid = (rows + u * kRows - 1) / (u * kRows);
  if (grid > 0x7fffffff) return static_cast<int>(cudaErrorInvalidValue);
  if (u == 4)
    kv_quant_write_kernel<T, D, 4, ROT><<<static_cast<int>(grid), 256, 0, s>>>(a, slots, al);
  else
    kv_quant_write_kernel<T, D, 1, ROT><<<static_cast<int>(grid), 256, 0, s>>>(a, slots, al);
  return static_cast<int>(cudaGetLastError());
}

template <typename T, int D>
int write_as(const TbKvQuantWriteArgs& a, cudaStream_t s) {
  return a.rot.R > 0 ? write_rot<T, D, true>(a, s) : write_rot<T, D, false>(a, s);
}

template <typename T, int D>
int read_as(const TbKvQuantReadArgs& a, cudaStream_t s) {
  constexpr int kRows = 256 / (D / 16);
  const bool al = rows_aligned(a.k, a.ks_t, a.ks_h, a.dtype, 16) && rows_aligned(a.v, a.vs_t, a.vs_h, a.dtype, 16);
  const long long rows = static_cast<long long>(a.T) * 2 * a.cache.Hk;
  const int u = rows * (D / 16) >= 4 * kFullMachine ? 4 : 1;
  const long long grid = (rows + u * kRows - 1) / (u * kRows);
  if (grid > 0x7fffffff) return static_cast<int>(cudaErrorInvalidValue);
  if (u == 4)
    kv_quant_read_kernel<T, D, 4><<<static_cast<int>(grid), 256, 0, s>>>(a, al);
  else
    kv_quant_read_kernel<T, D, 1><<<static_cast<int>(grid), 256, 0, s>>>(a, al);
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
