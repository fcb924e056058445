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
// Reads and writes are one pass over the rows and a few operations per element.
// On one B200 at D = 128 in bf16: read of 84 K tokens x 8 KV heads (522 MB) 86 us,
// 6.0 TB/s; write of 23 K tokens among 49 K rows x 8 KV heads (143 MB) 28 us, 5.1 TB/s;
// a decode step of 512 tokens with rotary 4 us, launch and one chain of loads.
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

// A warp takes G tokens side by side, a row of each per round, and of their
// slots (k heads, v heads, then q heads) the rounds [part, part + 1) / parts: the
// head is the same for the whole warp, and a row costs an addition.
struct Split {
  int parts, slots;
};

// Word j of an array that starts anywhere, and element j of such words.
__device__ __forceinline__ uint32_t word_at(const float* p, int j) { return __float_as_uint(p[j]); }
template <typename T>
__device__ __forceinline__ uint32_t word_at(const T* p, int j) {
  const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
  return h[2 * j] | static_cast<uint32_t>(h[2 * j + 1]) << 16;
}
__device__ __forceinline__ float element(const float*, const uint32_t (&w)[8], int j) { return __uint_as_float(w[j]); }
__device__ __forceinline__ float element(const __nv_bfloat16*, const uint32_t (&w)[8], int j) {
  return __uint_as_float(j % 2 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
}
__device__ __forceinline__ float element(const __half*, const uint32_t (&w)[8], int j) {
  return __half2float(__ushort_as_half(static_cast<unsigned short>(w[j / 2] >> (j % 2 * 16))));
}

// The largest |x| of a lane's values, two at a time where they have 16 bits; a
// NaN wins.
__device__ __forceinline__ uint32_t max_two(const float*, uint32_t a, uint32_t b) {
  return max(a, b);  // absolute values compare like their bits, and NaN is above infinity
}
__device__ __forceinline__ uint32_t max_two(const __nv_bfloat16*, uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t max_two(const __half*, uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
template <typename T, int W>
__device__ __forceinline__ uint32_t top_of(const T* tag, const uint32_t (&w)[W]) {
  constexpr uint32_t kAbs = sizeof(T) == 4 ? 0x7fffffffu : 0x7fff7fffu;
  uint32_t m = w[0] & kAbs;
#pragma unroll
  for (int i = 1; i < W; ++i) m = max_two(tag, m, w[i] & kAbs);
  return m;
}
// ... as the bits of an fp32 number
__device__ __forceinline__ uint32_t top_bits(const float*, uint32_t m) { return m; }
template <typename T>
__device__ __forceinline__ uint32_t top_bits(const T*, uint32_t m) {
  const unsigned short h = static_cast<unsigned short>(max(m & 0xffffu, m >> 16));
  return __float_as_uint(tb::to_f32(*reinterpret_cast<const T*>(&h)));
}

// 32 bytes from a multiple of 32.
__device__ __forceinline__ void load_sector(const void* p, uint32_t (&w)[8]) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
               : "l"(p));
}

// Rows as they come: a lane holds 32 neighbouring bytes of a row (with 16, 16,384
// tokens x 2 KV heads x 128 in bf16 took 7.3 us for 5.7), and four heads of it are in
// flight.  The four rows are reduced together (4 shuffles at D = 128 in 16 bits, 12
// apart), and the two divisions of a row are done once per lane.  align: what rows
// start on a multiple of, 32, 16 or fewer bytes.
template <typename T, int D>
__global__ void __launch_bounds__(128, 8)  // (64 registers: all of a round's loads are in flight)
    kv_quant_write_kernel(TbKvQuantWriteArgs a, Split sp, int align) {
  constexpr int E = 32 / sizeof(T), L = D / E, G = 32 / L;  // elements of a lane, lanes per row, tokens
  constexpr int U = 4, W = 8;                               // heads in flight, words of a lane
  const T* tag = nullptr;
  const int lane = threadIdx.x % 32, l = lane % L, Hk = a.cache.Hk;
  const long long item = blockIdx.x * (blockDim.x / 32ll) + threadIdx.x / 32, group = item / sp.parts, t = group * G + lane / L;
  const int p = t < a.T ? a.pos[t] : -1, seq = t < a.T ? a.seq[t] : -1;
  const bool need = p >= 0 && seq >= 0;  // (the rows are loaded while their slots are still looked up)
  if (!__any_sync(0xffffffffu, need)) return;
  const int row0 = static_cast<int>(slot_row(a.cache, seq, p, l == 0 ? a.rot.err : nullptr));
  const int part = static_cast<int>(item - group * sp.parts), hi_slot = (part + 1) * sp.slots / sp.parts;
  const int lo_slot = part * sp.slots / sp.parts;
  // where the next row is read and its codes go; both jump to v behind the last k head
  const T* vp = static_cast<const T*>(a.v) + t * a.vs_t + E * l;
  uint8_t* vc = static_cast<uint8_t*>(a.cache.vc) + static_cast<long long>(row0) * D + E * l;
  const long long head = static_cast<long long>(a.cache.bs) * D;
  const T* from = lo_slot < Hk ? static_cast<const T*>(a.k) + t * a.ks_t + lo_slot * a.ks_h + E * l
                               : vp + (lo_slot - Hk) * a.vs_h;
  uint8_t* to = lo_slot < Hk
                    ? static_cast<uint8_t*>(a.cache.kc) + static_cast<long long>(row0) * D + lo_slot * head + E * l
                    : vc + (lo_slot - Hk) * head;
  for (int s0 = lo_slot; s0 < hi_slot; s0 += U) {
    uint32_t x[U][W], m[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int slot = s0 + u;
#pragma unroll
      for (int j = 0; j < W; ++j) x[u][j] = 0;
      if (slot == Hk) from = vp;
      const T* row = from;
      from += slot < Hk ? a.ks_h : a.vs_h;
      if (slot < hi_slot && need) {
        if (align == 32) {
          load_sector(row, x[u]);
        } else if (align == 16) {
#pragma unroll
          for (int j = 0; j < W; j += 4) {
            const uint4 y = reinterpret_cast<const uint4*>(row)[j / 4];
            x[u][j] = y.x;
            x[u][j + 1] = y.y;
            x[u][j + 2] = y.z;
            x[u][j + 3] = y.w;
          }
        } else {
#pragma unroll
          for (int j = 0; j < W; ++j) x[u][j] = word_at(row, j);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) m[u] = top_of(tag, x[u]);
    // reduce and deal out: a quarter of a row's lanes ends with the maximum of one of the four rows each
    const bool hi = l & L / 2, mid = l & L / 4;
    uint32_t m0 = hi ? m[2] : m[0], m1 = hi ? m[3] : m[1];
    m0 = max_two(tag, m0, __shfl_xor_sync(0xffffffffu, hi ? m[0] : m[2], L / 2));
    m1 = max_two(tag, m1, __shfl_xor_sync(0xffffffffu, hi ? m[1] : m[3], L / 2));
    uint32_t top = max_two(tag, mid ? m1 : m0, __shfl_xor_sync(0xffffffffu, mid ? m0 : m1, L / 4));
#pragma unroll
    for (int o = L / 8; o > 0; o >>= 1) top = max_two(tag, top, __shfl_xor_sync(0xffffffffu, top, o));
    const float amax = __uint_as_float(max(top_bits(tag, top), kMinAmaxBits)), inv = __fdiv_rn(kMaxCode, amax);
    const int own = s0 + (hi ? 2 : 0) + (mid ? 1 : 0);  // the slot of this lane's maximum
    if (l % (L / 4) == 0 && own < hi_slot && row0 >= 0)
      (own < Hk ? a.cache.ks + own * a.cache.bs : a.cache.vs + (own - Hk) * a.cache.bs)[row0] = __fdiv_rn(amax, kMaxCode);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int slot = s0 + u;
      const float f = __shfl_sync(0xffffffffu, inv, (lane & ~(L - 1)) + (u / 2) * (L / 2) + (u % 2) * (L / 4));
      if (slot == Hk) to = vc;
      uint8_t* c = to;
      to += head;
      if (slot >= hi_slot || row0 < 0) continue;
      uint32_t code[E / 4];
#pragma unroll
      for (int j = 0; j < E; j += 4)
        code[j / 4] = to_e4m3x4(element(tag, x[u], j) * f, element(tag, x[u], j + 1) * f, element(tag, x[u], j + 2) * f,
                                element(tag, x[u], j + 3) * f);
      if constexpr (E == 16)
        *reinterpret_cast<uint4*>(c) = make_uint4(code[0], code[1], code[2], code[3]);
      else
        *reinterpret_cast<uint2*>(c) = make_uint2(code[0], code[1]);
    }
  }
}

// One token's q and k rows rotated first: G heads of it per round, its table
// entries in registers for all of them.  A lane holds both members of its pairs
// (half layout: two vectors of four), else eight neighbours.  wide_table: the table
// starts on a multiple of 16 bytes (it may start on any multiple of 8; its rows are
// multiples of 32 long).
template <typename T, int D>
__global__ void __launch_bounds__(128)
    kv_quant_write_rot_kernel(TbKvQuantWriteArgs a, Split sp, bool aligned, bool wide_table) {
  constexpr int L = D / 8, G = 32 / L, U = 2;
  const int lane = threadIdx.x % 32, l = lane % L, Hk = a.cache.Hk, R = a.rot.R;
  const long long item = blockIdx.x * (blockDim.x / 32ll) + threadIdx.x / 32, t = item / sp.parts;
  if (t >= a.T) return;
  const int part = static_cast<int>(item - t * sp.parts), rounds = (sp.slots + G - 1) / G;
  const int lo = part * rounds / sp.parts, hi = (part + 1) * rounds / sp.parts;
  const int seq = a.seq[t], p = seq < 0 ? -1 : a.pos[t];  // (padding, whatever its position)
  const bool past = p >= a.rot.max_pos, turn = 8 * l < R, half = turn && !a.rot.interleaved;
  float cs[8];
  if (turn && p >= 0 && !past) {
    const float* entry = a.rot.table + (static_cast<long long>(p) * (R / 2) + 4 * l) * 2;
    if (wide_table) {
      tb::load_vec<float, 8>(entry, cs);
    } else {
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const float2 e = *reinterpret_cast<const float2*>(entry + j);
        cs[j] = e.x;
        cs[j + 1] = e.y;
      }
    }
  }
  int base = -1;
  if (past) {
    if (a.rot.err && lane == 0) atomicCAS(a.rot.err, 0, 1);
  } else {
    base = static_cast<int>(slot_row(a.cache, seq, p, lane == 0 ? a.rot.err : nullptr));
  }
  for (int i = lo; i < hi; i += U) {
    tb::Packed<T, 4> x0[U], x1[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int slot = (i + u) * G + lane / L, kind = slot < Hk ? 0 : slot < 2 * Hk ? 1 : 2, h = slot - kind * Hk;
      const bool pairs = half && kind != 1;
      const T* x = kind == 0   ? static_cast<const T*>(a.k) + t * a.ks_t + h * a.ks_h
                   : kind == 1 ? static_cast<const T*>(a.v) + t * a.vs_t + h * a.vs_h
                               : static_cast<const T*>(a.rot.x) + t * a.rot.xs_t + h * a.rot.xs_h;
      const int o1 = pairs ? 4 * l : 8 * l, o2 = pairs ? 4 * l + R / 2 : 8 * l + 4;
      x0[u].raw = x1[u].raw = {};
      if (i + u < hi && slot < sp.slots && (kind == 2 || (p >= 0 && seq >= 0))) {
        if (aligned) {
          x0[u].load(x + o1);
          x1[u].load(x + o2);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            reinterpret_cast<T*>(&x0[u].raw)[j] = x[o1 + j];
            reinterpret_cast<T*>(&x1[u].raw)[j] = x[o2 + j];
          }
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int slot = (i + u) * G + lane / L, kind = slot < Hk ? 0 : slot < 2 * Hk ? 1 : 2, h = slot - kind * Hk;
      const bool live = i + u < hi && slot < sp.slots, pairs = half && kind != 1;
      const int o1 = pairs ? 4 * l : 8 * l, o2 = pairs ? 4 * l + R / 2 : 8 * l + 4;
      float f[4], g[4];
      x0[u].unpack(f);
      x1[u].unpack(g);
      if (turn && kind != 1 && p >= 0 && !past) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float& v = pairs ? f[j] : j < 2 ? f[2 * j] : g[2 * j - 4];
          float& w = pairs ? g[j] : j < 2 ? f[2 * j + 1] : g[2 * j - 3];
          const float nv = v * cs[2 * j] - w * cs[2 * j + 1];
          w = w * cs[2 * j] + v * cs[2 * j + 1];
          v = nv;
        }
      }
      uint32_t m = kMinAmaxBits;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        m = max(m, max(__float_as_uint(f[j]) & 0x7fffffffu, __float_as_uint(g[j]) & 0x7fffffffu));
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
      if (live && kind == 2) {
        T* y = static_cast<T*>(a.rot.y) + t * a.rot.ys_t + h * a.rot.ys_h;
        if (past) {
#pragma unroll
          for (int j = 0; j < 4; ++j) f[j] = g[j] = NAN;
        }
        store4<T>(y + o1, aligned, f);
        store4<T>(y + o2, aligned, g);
      } else if (live && base >= 0) {
        const long long row = base + static_cast<long long>(h) * a.cache.bs;
        const float amax = __uint_as_float(m), inv = __fdiv_rn(kMaxCode, amax);
        uint8_t* c = static_cast<uint8_t*>(kind == 0 ? a.cache.kc : a.cache.vc) + row * D;
        *reinterpret_cast<uint32_t*>(c + o1) = to_e4m3x4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv);
        *reinterpret_cast<uint32_t*>(c + o2) = to_e4m3x4(g[0] * inv, g[1] * inv, g[2] * inv, g[3] * inv);
        if (l == 0) (kind == 0 ? a.cache.ks : a.cache.vs)[row] = __fdiv_rn(amax, kMaxCode);
      }
    }
  }
}

// Sixteen values to a multiple of 32 bytes: whole sectors per store (two stores of
// 16 bytes leave each sector to be put together: 84 K tokens x 8 KV heads x 128 in
// bf16 94 us for 86, in fp32 168 for 140).
template <typename T>
__device__ __forceinline__ void store_sectors(T* p, const float (&f)[16]) {
  constexpr int W = 4 * sizeof(T);
  uint32_t w[W];
#pragma unroll
  for (int i = 0; i < 16; ++i) reinterpret_cast<T*>(w)[i] = tb::from_f32<T>(f[i]);
#pragma unroll
  for (int i = 0; i < W; i += 8)
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(reinterpret_cast<uint32_t*>(p) + i),
                 "r"(w[i]), "r"(w[i + 1]), "r"(w[i + 2]), "r"(w[i + 3]), "r"(w[i + 4]), "r"(w[i + 5]), "r"(w[i + 6]),
                 "r"(w[i + 7])
                 : "memory");
}

// D / 16 lanes per row, sixteen codes each, four heads in flight (as fast as two or
// eight).  align: what rows start on a multiple of, 32, 16 or fewer bytes.
template <typename T, int D>
__global__ void __launch_bounds__(128) kv_quant_read_kernel(TbKvQuantReadArgs a, Split sp, int align) {
  constexpr int L = D / 16, G = 32 / L, U = 4;
  const int lane = threadIdx.x % 32, l = lane % L, Hk = a.cache.Hk;
  const long long item = blockIdx.x * (blockDim.x / 32ll) + threadIdx.x / 32, group = item / sp.parts, t = group * G + lane / L;
  if (t >= a.T) return;
  const int row0 = static_cast<int>(slot_row(a.cache, a.seq[t], a.pos[t], l == 0 ? a.err : nullptr));
  if (row0 < 0) return;
  const uint8_t* kc = static_cast<const uint8_t*>(a.cache.kc) + static_cast<long long>(row0) * D + 16 * l;
  const uint8_t* vc = static_cast<const uint8_t*>(a.cache.vc) + static_cast<long long>(row0) * D + 16 * l;
  T* kp = static_cast<T*>(a.k) + t * a.ks_t + 16 * l;
  T* vp = static_cast<T*>(a.v) + t * a.vs_t + 16 * l;
  const int part = static_cast<int>(item - group * sp.parts), hi_slot = (part + 1) * sp.slots / sp.parts;
  for (int s0 = part * sp.slots / sp.parts; s0 < hi_slot; s0 += U) {
    uint4 w[U];
    float s[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int slot = s0 + u, h = slot < Hk ? slot : slot - Hk;
      if (slot >= hi_slot) continue;
      w[u] = *reinterpret_cast<const uint4*>((slot < Hk ? kc : vc) + static_cast<long long>(h) * a.cache.bs * D);
      s[u] = ((slot < Hk ? a.cache.ks : a.cache.vs) + h * a.cache.bs)[row0];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int slot = s0 + u;
      if (slot >= hi_slot) continue;
      T* y = slot < Hk ? kp + slot * a.ks_h : vp + (slot - Hk) * a.vs_h;
      const uint32_t ww[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
      float f[16];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float q[4];
        from_e4m3x4(ww[j], q);
#pragma unroll
        for (int e = 0; e < 4; ++e) f[4 * j + e] = q[e] * s[u];
      }
      if (align == 32) {
        store_sectors<T>(y, f);
      } else if (align == 16) {
        tb::store_vec<T, 16>(y, f);
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) y[j] = tb::from_f32<T>(f[j]);
      }
    }
  }
}

// Whether every row of a [T, H, D] view starts on a multiple of `bytes`.
bool rows_aligned(const void* p, long long st, long long sh, int dtype, int bytes) {
  const int e = dtype == TB_F32 ? 4 : 2;
  return reinterpret_cast<uintptr_t>(p) % bytes == 0 && st * e % bytes == 0 && sh * e % bytes == 0;
}

// Warps that share the rounds of their tokens (few tokens: latency counts), as
// many as fill 16 warps per SM (512 tokens of 16 rows: 3.9 us so, 4.6 with 8 or 32);
// in blocks of two warps, over more SMs, where there are few, else of four (ragged
// batches: 1 us in 33 less than with eight).
constexpr int kFewWarps = 148 * 16, kSpread = 148 * 8;
int parts_of(long long groups, int rounds) {
  int n = 1;
  while (2 * n <= rounds && 2 * n * groups <= kFewWarps && 2ll * n * rounds <= 0x7fffffff) n *= 2;
  return n;
}
struct Shape {
  int grid, block;
  explicit Shape(long long warps)
      : grid(static_cast<int>(warps <= kSpread ? (warps + 1) / 2 : (warps + 3) / 4)), block(warps <= kSpread ? 64 : 128) {}
};

template <typename T, int D>
int write_as(const TbKvQuantWriteArgs& a, cudaStream_t s) {
  auto on = [&](int bytes) {
    return rows_aligned(a.k, a.ks_t, a.ks_h, a.rot.dtype, bytes) && rows_aligned(a.v, a.vs_t, a.vs_h, a.rot.dtype, bytes);
  };
  Split sp = {1, 2 * a.cache.Hk};
  if (a.rot.R == 0) {
    constexpr int kRows = 32 / (D * static_cast<int>(sizeof(T)) / 32);  // tokens per warp
    const long long groups = (a.T + kRows - 1ll) / kRows;
    sp.parts = parts_of(groups, sp.slots);
    const Shape g(groups * sp.parts);
    kv_quant_write_kernel<T, D><<<g.grid, g.block, 0, s>>>(a, sp, on(32) ? 32 : on(16) ? 16 : 0);
    return static_cast<int>(cudaGetLastError());
  }
  constexpr int G = 32 / (D / 8), v = 4 * static_cast<int>(sizeof(T));  // rows per warp and round, bytes of a vector
  bool al = on(v);
  if (a.rot.x) {
    sp.slots += a.rot.H;
    al = al && rows_aligned(a.rot.x, a.rot.xs_t, a.rot.xs_h, a.rot.dtype, v) &&
         rows_aligned(a.rot.y, a.rot.ys_t, a.rot.ys_h, a.rot.dtype, v);
  }
  const bool wide_table = reinterpret_cast<uintptr_t>(a.rot.table) % 16 == 0;
  sp.parts = parts_of(a.T, (sp.slots + G - 1) / G);
  const Shape g(static_cast<long long>(a.T) * sp.parts);
  kv_quant_write_rot_kernel<T, D><<<g.grid, g.block, 0, s>>>(a, sp, al, wide_table);
  return static_cast<int>(cudaGetLastError());
}

template <typename T, int D>
int read_as(const TbKvQuantReadArgs& a, cudaStream_t s) {
  constexpr int G = 32 / (D / 16);
  auto on = [&](int bytes) {
    return rows_aligned(a.k, a.ks_t, a.ks_h, a.dtype, bytes) && rows_aligned(a.v, a.vs_t, a.vs_h, a.dtype, bytes);
  };
  const long long groups = (a.T + G - 1ll) / G;
  Split sp = {1, 2 * a.cache.Hk};
  sp.parts = parts_of(groups, sp.slots);
  const Shape g(groups * sp.parts);
  kv_quant_read_kernel<T, D><<<g.grid, g.block, 0, s>>>(a, sp, on(32) ? 32 : on(16) ? 16 : 0);
  return static_cast<int>(cudaGetLastError());
}

bool cache_ok(const TbQuantCache& c) {
  return c.Hk > 0 && c.bs > 0 && c.num_blocks >= 0 && (c.D == 64 || c.D == 128 || c.D == 256) &&
         c.Hk <= 0x7fffffff / c.D &&
         static_cast<long long>(c.num_blocks) * c.Hk <= 0x7fffffff / c.bs;
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
