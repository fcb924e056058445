// Attention of one new token per sequence over the 8-bit paged KV cache:
//
//   a_j = scale * ks_j * (q . k_j),   out = sum_j softmax(a)_j * vs_j * v_j
//
// with k_j, v_j the e4m3 codes and ks_j, vs_j the scales of token j, for the
// G = Hq / Hk query heads that share a KV head.
//
// The pages are the traffic (2 (D + 4) bytes per token and KV head), read once:
//
//  * Work is cut into tiles of 16 tokens and dealt out evenly over the warps of
//    a resident grid, whatever the contexts' lengths: worker i of n takes its
//    share of the list (sequence, KV head, tile), read off ctx_len on the
//    device, so one captured call serves contexts that grow.  (Equal shares end
//    up to 15% apart, SMs of different GPCs reaching memory at different rates;
//    that, the 4 us until the first tile is there and the 5 us of joining are
//    what separates the kernel from its bytes: with every product and widening
//    left out lists take 98 to 99% of their time, clusters 91%, and lists with 16
//    query heads on a KV head 96%.)
//  * A warp fills a ring of tiles in its shared memory with cp.async, running
//    ahead over the borders of contexts, and waits for no other warp before
//    the end of its list.  Contexts that end inside its list it writes out; the
//    parts at the list's two ends (maximum, sum, unnormalised output) the CTA
//    merges, and what is split over CTAs a second kernel joins, all in a fixed
//    order: no atomics, the same bits every time.
//  * Few or short contexts go to clusters instead, one per (sequence, KV head),
//    joined over distributed shared memory in the one launch.
//  * Products run on mma.sync m16n8k16 in fp16 (every e4m3 value is an fp16
//    value) with the tokens, then the head's dimensions, as the 16 rows and the
//    query heads as the 8 columns: with 5 to 8 query heads per KV head hardly a
//    column is idle, and a tcgen05 tile (128 rows by 8 columns) would want the
//    codes widened through shared memory first.  S^T = K q, whose accumulator,
//    transposed in registers (movmatrix), is the operand of O^T = V^T w.
//  * The weights' reference m follows the running maximum of a_j + log2 vs_j
//    (a_j in units of log 2), 7 below it: then w_j = exp2(a_j - m) vs_j fits fp16
//    however much the scales of tokens differ (rounded to 2^-11 relative, 2^-32 of
//    the largest at the small end), while the sum l of exp2(a_j - m) stays in fp32
//    range.  m moves only once the maximum is 15 above it, so weights stay below
//    2^15 and most tiles need no reduction over the warp and no rescaling.  q is
//    brought into fp16 range by a power of two per head (exact).
//
// On one B200, D = 128, in a graph: 2 x 131,072 tokens x 8 KV heads (554 MB) 97 us,
// 5.7 TB/s; 512 ragged contexts up to 768 tokens x 2 KV heads (96 MB) 29 us; 1 x
// 1,000 tokens x 8 KV heads 6.2 us.
#include <float.h>
#include <math.h>

#include <atomic>

#include "device_common.cuh"
#include "kernels.h"
#include "pdl.cuh"
#include "vec_io.cuh"

namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr int kTile = 16;       // tokens per tile
constexpr int kMinTiles = 8;    // tiles per CTA, at least, where there are that many
constexpr int kStart = 3;       // what beginning a (sequence, group) costs a warp, in tiles
constexpr int kMostCluster = 8;   // CTAs of a cluster (the portable bound)
constexpr float kMinVsLog = -92.f;   // keeps the sum of exp2(a - m), 2^(15 + 92) per token at most, in fp32 range
constexpr float kLowest = -FLT_MAX;  // the reference before the first token: below every score, and finite
// The reference of the weights is set 2^7 below their maximum, and left until that is 2^15 above it: the weights use
// fp16's upper range, so that a token has to be 2^-32 of the largest one before its weight rounds to 0 (with the
// reference at the maximum 2^-25, and 2^18 such tokens of a context lost 2^-7 of the sum).  The slack is added rounding
// down: where neighbouring scores are 8 or 16 apart, it could round up and let weights of 2^16 through, past fp16.
constexpr float kAhead = 7.f, kSlack = 15.f;

// The four codes of a word as two fp16 pairs.
__device__ __forceinline__ void widen(uint32_t codes, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(codes));
}
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float log2_fast(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// What a sum of 0 over a context stands for, M being the reference it was taken with: no token (M = -inf: zeros), or
// scores that are all -inf (NaN, as 0 / 0).
__device__ __forceinline__ float of_nothing(float M) { return M == -INFINITY ? 0.f : NAN; }
// 2^e for e in [-126, 127]
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Shared memory.  A ring stage holds 16 K rows and 16 V rows of codes (rows
// padded by 16 bytes against bank conflicts), their scales and a mask of the
// tokens that count.  Two stages are enough at D = 128 and 256, the next tile being
// asked for before one is used (2 x 131,072 tokens x 8 KV heads x 128: 98 us, with
// three 104); small tiles and two sets of heads take three.  A part is heads x D
// outputs, then heads x (maximum, sum): a warp's first one goes to its place behind
// the rings, its last one into its own ring, drained by then.
template <int D, int NT>
struct Smem {
  static constexpr int kStages = D == 64 || NT == 2 ? 3 : 2;
  static constexpr int kRow = D + 16;
  static constexpr int kStage = 2 * kTile * kRow + 2 * kTile * 4 + 16;
  static constexpr int kHeads = 8 * NT;
  static constexpr int kPart = kHeads * (D + 2) * 4;
  static constexpr int kRing = kStages * kStage;
  static constexpr int kScan = (kThreads + kWarps + 2) * 4 + 2 * kWarps * 8;
  static constexpr int kBytes = kWarps * (kRing + kPart) + kScan;
  static_assert(kRing >= kPart && kRing % 16 == 0 && kPart % 16 == 0, "a part fits a ring");
};

// CTAs per SM: those that shared memory (228 KB, 1 KB of it per CTA the system's)
// leaves room for, up to 4.  Lists at D = 128 have three of them: with four, 2 x
// 131,072 tokens x 8 KV heads took 100 us for 98, and no mix of contexts gained over 2%.
template <int D, int NT>
constexpr int resident() {
  constexpr int kFit = 233472 / (Smem<D, NT>::kBytes + 1024);
  return kFit < 4 ? kFit : 4;
}
template <int D, int NT>
constexpr int list_ctas() {
  return D == 128 && resident<D, NT>() > 3 ? 3 : resident<D, NT>();
}

// Workspace: two parts per CTA (what its list's ends leave), then one record per
// CTA: of the context whose first part it holds (sequence x group, part, CTAs that
// share it or 0), and the first CTA of the one that came over from the CTA before
// (or -1).
template <int D, int NT>
struct Partials {
  static constexpr int kHeads = 8 * NT;
  static constexpr size_t kSlot = static_cast<size_t>(kHeads) * (D + 2);
  __device__ static float* out(float* ws, long long slot, int h) { return ws + slot * kSlot + h * D; }
  __device__ static float* stat(float* ws, long long slot, int h) {
    return ws + slot * kSlot + kHeads * D + h * 2;
  }
  __device__ static int4* record(float* ws, int grid, int c) {
    return reinterpret_cast<int4*>(ws + 2ll * grid * kSlot) + c;
  }
  static size_t bytes(int grid) { return (2 * grid * kSlot + 4 * static_cast<size_t>(grid)) * 4; }
};

struct Geometry {
  int G, NG, HG;   // query heads per KV head, groups of 8 NT of them, groups per sequence
  int cap;         // tokens that a table row can name
  int shift;       // log2 of the page size, or -1
  int tile_pages;  // pages hold whole tiles
  int cs;          // CTAs (a cluster) for each (sequence, group), or 0: work dealt out evenly
};

__device__ __forceinline__ int tokens_of(const TbDecodeAttnQuantArgs& a, const Geometry& g, int b) {
  const int n = a.ctx_len[b];
  return n < 0 ? 0 : n < g.cap ? n : g.cap;
}

__device__ __forceinline__ int tiles(int tokens) { return tokens / kTile + (tokens % kTile != 0); }

// The list is counted in units: kStart for beginning a (sequence, group), then
// its tiles.  Of n workers the first `more` take each + 1 units, the others each.
__device__ __forceinline__ int units(int tokens) { return tokens > 0 ? tiles(tokens) + kStart : 0; }
struct Shares {
  uint32_t each, more;
  __device__ __forceinline__ uint32_t start(uint32_t i) const { return i * each + min(i, more); }
  __device__ __forceinline__ uint32_t owner(uint32_t unit) const {
    const uint32_t head = more * (each + 1);
    return unit < head ? unit / (each + 1) : more + (unit - head) / each;
  }
};

// Where a warp (or its prefetch) stands in its list of tiles: in sequence b,
// group r, at tile t of the portion [.., end), with `rest` units behind it.
struct Cursor {
  int b, r, tokens, t, end, rest;
};

// Moves on to the next portion; false at the end of the list.
__device__ __forceinline__ bool next_portion(const TbDecodeAttnQuantArgs& a, const Geometry& g, Cursor& c) {
  if (c.rest <= 0) return false;
  if (++c.r == g.HG) {
    c.r = 0;
    do {
      if (++c.b >= a.B) return false;
      c.tokens = tokens_of(a, g, c.b);
    } while (c.tokens == 0);
  }
  const int n = units(c.tokens), take = n < c.rest ? n : c.rest;
  c.t = 0;
  c.end = take - kStart;
  c.rest -= take;
  return c.end > 0;  // (nothing is behind a portion without a tile)
}

template <typename T>
__device__ __forceinline__ void store_out4(T* p, bool aligned, float x, float y, float z, float w) {
  if (aligned) {
    const float f[4] = {x, y, z, w};
    tb::store_vec<T, 4>(p, f);
  } else {
    p[0] = tb::from_f32<T>(x);
    p[1] = tb::from_f32<T>(y);
    p[2] = tb::from_f32<T>(z);
    p[3] = tb::from_f32<T>(w);
  }
}

// A value in the shared memory of CTA `rank` of the cluster, at the place that p has here.
__device__ __forceinline__ uint32_t peer_address(const void* p, int rank) {
  uint32_t d;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(d) : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(p))), "r"(rank));
  return d;
}
__device__ __forceinline__ float peer_load(uint32_t at) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ float4 peer_load4(uint32_t at) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(at)
               : "memory");
  return v;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Joins the parts of a (sequence, group) that a cluster (or one CTA) shares: each
// CTA its warps', then a warp of the cluster for each query head the CTAs', over
// distributed shared memory.
template <typename T, int D>
__device__ __forceinline__ void cluster_join(const TbDecodeAttnQuantArgs& a, const Geometry& g, uint8_t* smem, int2* meta,
                                             bool out4) {
  using S = Smem<D, 1>;
  constexpr int kHeads = S::kHeads, E = D / 32, V = E < 4 ? E : 4;
  const int w = threadIdx.x / 32, lane = threadIdx.x % 32, rank = blockIdx.x % g.cs, seg = blockIdx.x / g.cs;
  const int b = seg / g.HG, r = seg - b * g.HG, kh = r / g.NG, left = g.G - (r - kh * g.NG) * kHeads;
  const int nh = min(left, kHeads), h0 = kh * g.G + g.G - left;
  float* sum = reinterpret_cast<float*>(smem);  // the CTA's part, in the ring of warp 0 (drained)
  auto write = [&](int h, const float (&o)[E], float inv) {
    T* out = static_cast<T*>(a.out) + static_cast<long long>(b) * a.os_b + static_cast<long long>(h0 + h) * a.os_h;
#pragma unroll
    for (int i = 0; i < E; i += V) {
      float z[V];
#pragma unroll
      for (int e = 0; e < V; ++e) z[e] = o[i + e] * inv;
      if (out4) {
        tb::store_vec<T, V>(out + i * 32 + lane * V, z);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) out[i * 32 + lane * V + e] = tb::from_f32<T>(z[e]);
      }
    }
  };
  __syncthreads();
  for (int h = w; h < nh; h += kWarps) {
    float m[kWarps], l[kWarps], M = -INFINITY, L = 0.f, o[E] = {};
    const float* part[kWarps];
    bool any = false;
#pragma unroll
    for (int p = 0; p < kWarps; ++p) {
      part[p] = reinterpret_cast<const float*>(smem + kWarps * S::kRing + p * S::kPart);
      const bool have = meta[2 * p].x >= 0;
      any |= have;
      m[p] = have ? part[p][kHeads * D + 2 * h] : -INFINITY;
      l[p] = have ? part[p][kHeads * D + 2 * h + 1] : 0.f;
      M = fmaxf(M, m[p]);
    }
#pragma unroll
    for (int p = 0; p < kWarps; ++p) {
      const float f = m[p] == -INFINITY ? 0.f : exp2_fast(m[p] - M);
      L += f * l[p];
      if (meta[2 * p].x < 0) continue;
#pragma unroll
      for (int i = 0; i < E; i += V) {
        float y[V];
        tb::load_vec<float, V>(part[p] + h * D + i * 32 + lane * V, y);
#pragma unroll
        for (int e = 0; e < V; ++e) o[i + e] += f * y[e];
      }
    }
    if (g.cs == 1) {
      if (any) write(h, o, L == 0.f ? of_nothing(M) : 1.f / L);  // (else one warp had the whole context, and wrote it)
      continue;
    }
#pragma unroll
    for (int i = 0; i < E; i += V) {
      float y[V];
#pragma unroll
      for (int e = 0; e < V; ++e) y[e] = o[i + e];
      tb::store_vec<float, V>(sum + h * D + i * 32 + lane * V, y);
    }
    if (lane == 0) *reinterpret_cast<float2*>(sum + kHeads * D + 2 * h) = make_float2(M, any ? L : -1.f);  // -1: no part
  }
  if (g.cs == 1) return;
  cluster_barrier();
  for (int h = rank + g.cs * w; h < nh; h += g.cs * kWarps) {
    float m = -INFINITY, l = -1.f;
    if (lane < g.cs) {
      const uint32_t at = peer_address(sum + kHeads * D + 2 * h, lane);
      m = peer_load(at);
      l = peer_load(at + 4);
    }
    if (!__any_sync(0xffffffffu, l != -1.f)) break;  // one warp had the whole context, and wrote it
    float o[kMostCluster][E];
#pragma unroll
    for (int p = 0; p < kMostCluster; ++p) {
#pragma unroll
      for (int i = 0; i < E; ++i) o[p][i] = 0.f;
      if (p >= g.cs) continue;
      const uint32_t at = peer_address(sum + h * D + lane * V, p);
#pragma unroll
      for (int i = 0; i < E; i += V) {
        if constexpr (V == 4) {
          const float4 y = peer_load4(at + i * 32 * 4);
          o[p][i] = y.x;
          o[p][i + 1] = y.y;
          o[p][i + 2] = y.z;
          o[p][i + 3] = y.w;
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) o[p][i + e] = peer_load(at + e * 4);
        }
      }
    }
    const float M = tb::warp_max(m), f = m == -INFINITY ? 0.f : exp2_fast(m - M);
    const float L = tb::warp_sum(f * l), inv = L == 0.f ? of_nothing(M) : 1.f / L;
    float y[E] = {};
#pragma unroll
    for (int p = 0; p < kMostCluster; ++p) {
      const float fp = __shfl_sync(0xffffffffu, f, p);
#pragma unroll
      for (int i = 0; i < E; ++i) y[i] += fp * o[p][i];
    }
    write(h, y, inv);
  }
  cluster_barrier();  // nobody leaves while another still reads its shared memory
}

// kClusters: a cluster (or one CTA) for each (sequence, eight query heads), else even
// lists: two kernels, since what a CTA does not need costs it instruction fetches (one
// short context: 4.2 us, from one kernel for both 5.1).  kPlain: pages of whole tiles,
// and q and out aligned for vectors, else as the flags say (with the flags: 512 ragged
// contexts up to 768 x 2 KV heads 29.5 us for 29.0, 37 up to 1,536 x 8 18.7 for 18.1).
template <typename T, int D, int NT, bool kClusters, bool kPlain>
__global__ void __launch_bounds__(kThreads, kClusters ? resident<D, NT>() : list_ctas<D, NT>())
    decode_attn_quant_kernel(TbDecodeAttnQuantArgs a, Geometry g, bool q_aligned, bool out_aligned) {
  const bool q8 = kPlain || q_aligned, out4 = kPlain || out_aligned, tile_pages = kPlain || g.tile_pages;
  using S = Smem<D, NT>;
  using P = Partials<D, NT>;
  constexpr int kStages = S::kStages, kHeads = S::kHeads, kRow = S::kRow;
  constexpr int NCH = D / 64;  // 16-byte chunks of a K row per lane
  constexpr int NW = D / 32;   // 4-byte words of a V row per lane
  extern __shared__ __align__(16) uint8_t smem[];
  const TbQuantCache& c = a.cache;
  const int w = threadIdx.x / 32, lane = threadIdx.x % 32, gq = lane / 4, tq = lane % 4;
  uint8_t* ring = smem + w * S::kRing;
  float* first_part = reinterpret_cast<float*>(smem + kWarps * S::kRing + w * S::kPart);
  uint32_t* before = reinterpret_cast<uint32_t*>(smem + kWarps * (S::kRing + S::kPart));  // [threads]
  uint32_t* sums = before + kThreads;                                                     // [warps]
  int* shared = reinterpret_cast<int*>(sums + kWarps);  // first CTA of the list's first context, last one of its last
  int2* meta = reinterpret_cast<int2*>(shared + 2);     // [2 warps] parts: (sequence x group or -1, opens | closes << 1)

  // ---- this warp's list of tiles
  Cursor cur;
  int ctas = 0;  // that have a list
  // zeros for empty contexts, and word of contexts longer than their tables, each by one of n CTAs
  auto empty_rows = [&](int n) {
    for (int b = blockIdx.x; b < a.B; b += n) {
      const int ctx = a.ctx_len[b];
      if (a.err && threadIdx.x == 0 && ctx > g.cap) atomicCAS(a.err, 0, 1);
      if (ctx > 0) continue;
      T* o = static_cast<T*>(a.out) + static_cast<long long>(b) * a.os_b;
      for (int i = threadIdx.x; i < a.Hq * (D / 4); i += kThreads)
        store_out4<T>(o + static_cast<long long>(i / (D / 4)) * a.os_h + i % (D / 4) * 4, out4, 0.f, 0.f, 0.f, 0.f);
    }
  };
  uint32_t total = 0;
  Shares sh = {};
  // the sequence b of a unit and its place in the sequence: the run of sequences that holds it (the last one that does
  // not begin behind it; a lane looks at four), then the sequence in the run
  auto find = [&](uint32_t unit, int& b, uint32_t& off) {
    const int per = (a.B + kThreads - 1) / kThreads;
    uint32_t base = 0;
    for (int i = 0; i < lane * 4 / 32; ++i) base += sums[i];
    const uint4 x = *reinterpret_cast<const uint4*>(before + lane * 4);
    const uint32_t at[4] = {(base + x.x) * g.HG, (base + x.y) * g.HG, (base + x.z) * g.HG, (base + x.w) * g.HG};
    int n = 0;
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (at[i] <= unit) {
        ++n;
        top = at[i];
      }
    const int run = __reduce_add_sync(0xffffffffu, n) - 1;
    off = unit - __reduce_max_sync(0xffffffffu, top);
    b = run * per;
    if (per == 1) return;
    for (int i = 0; i < per; i += 32) {
      const int c = b + lane;
      uint32_t inc = i + lane < per && c < a.B ? units(tokens_of(a, g, c)) * g.HG : 0;
      const uint32_t mine = inc;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += y;
      }
      const unsigned behind = __ballot_sync(0xffffffffu, off < inc);
      if (behind) {
        const int l = __ffs(behind) - 1;
        b += l;
        off -= __shfl_sync(0xffffffffu, inc - mine, l);
        return;
      }
      b += 32;
      off -= __shfl_sync(0xffffffffu, inc, 31);
    }
  };
  if constexpr (kClusters) {
    const int seg = blockIdx.x / g.cs, part = blockIdx.x % g.cs * kWarps + w, parts = g.cs * kWarps;
    cur.b = seg / g.HG;
    cur.r = seg % g.HG;
    // the table row (its first 1,024 entries) comes nearer while the context's length is read
    if (lane * 32 < c.max_blocks)
      asm volatile("prefetch.global.L1 [%0];" ::"l"(c.block_table + static_cast<long long>(cur.b) * c.max_blocks + lane * 32));
    cur.tokens = tokens_of(a, g, cur.b);
    const int n = tiles(cur.tokens);
    if (a.err && threadIdx.x == 0 && a.ctx_len[cur.b] > g.cap) atomicCAS(a.err, 0, 1);
    if (n == 0) {  // (the whole cluster)
      T* o = static_cast<T*>(a.out) + static_cast<long long>(cur.b) * a.os_b;
      const int h0 = cur.r / g.NG * g.G + cur.r % g.NG * kHeads, left = g.G - cur.r % g.NG * kHeads;
      if (part < kWarps)
        for (int i = threadIdx.x; i < (left < kHeads ? left : kHeads) * D; i += kThreads)
          o[static_cast<long long>(h0 + i / D) * a.os_h + i % D] = tb::from_f32<T>(0.f);
      return;
    }
    cur.t = static_cast<int>(static_cast<long long>(n) * part / parts);
    cur.end = static_cast<int>(static_cast<long long>(n) * (part + 1) / parts);
    cur.rest = 0;
  } else {
    // prefix sums of the sequences' units: each thread a run of sequences
    const int per = (a.B + kThreads - 1) / kThreads, b0 = threadIdx.x * per;
    const int b1 = min(b0 + per, a.B);
    uint32_t mine = 0;
#pragma unroll 4
    for (int b = b0; b < b1; ++b) mine += units(tokens_of(a, g, b));
    uint32_t inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    before[threadIdx.x] = inc - mine;  // within the warp
    if (lane == 31) sums[w] = inc;
    if (threadIdx.x == 0) *P::record(a.ws, gridDim.x, blockIdx.x) = make_int4(0, 0, 0, -1);
    __syncthreads();
    total = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) total += sums[i];
    total *= g.HG;
    // all CTAs, unless that leaves them less than kMinTiles
    uint32_t N = gridDim.x;
    if (total < N * kMinTiles) N = (total + kMinTiles - 1) / kMinTiles;
    if (N == 0) empty_rows(gridDim.x);
    if (blockIdx.x >= N) return;
    ctas = static_cast<int>(N);
    sh.each = total / (N * kWarps);
    sh.more = total - sh.each * (N * kWarps);
    const uint32_t me = blockIdx.x * kWarps + w, first = sh.start(me);
    uint32_t off;
    find(min(first, total - 1), cur.b, off);  // (a warp without units starts behind the last one)
    cur.tokens = tokens_of(a, g, cur.b);
    const int n = units(cur.tokens);
    cur.r = off / n;
    const int at = off - cur.r * n;
    cur.t = at > kStart ? at - kStart : 0;
    cur.rest = sh.start(me + 1) - first;
    const int take = min(n - at, cur.rest);
    cur.end = at + take - kStart;
    cur.rest -= take;
  }
  if (lane == 0) meta[2 * w] = meta[2 * w + 1] = make_int2(-1, 0);

  // ---- prefetch: a cursor that runs ahead, and where its next tile lies: with pages of whole tiles the tile's first row
  // and its number of tokens (32 tiles looked up at once), else (lanes 0-15) each token's row
  Cursor pre = cur;
  bool more = true;
  int row = -1, count = 0, pre_kh = cur.r / g.NG;
  int rows = -1, first = 0, last = 0;  // with pages of whole tiles: a lane for each of the tiles [first, last)
  auto row_of = [&](int tok) {
    const int pb = g.shift >= 0 ? tok >> g.shift : tok / c.bs;
    const int blk = c.block_table[static_cast<long long>(pre.b) * c.max_blocks + pb];
    if (blk >= 0 && blk < c.num_blocks) return (blk * c.Hk + pre_kh) * c.bs + (tok - pb * c.bs);
    if (a.err) atomicCAS(a.err, 0, 1);
    return -1;
  };
  auto look = [&]() {
    if (more && pre.t >= pre.end) {
      more = next_portion(a, g, pre);
      pre_kh = pre.r / g.NG;
      last = 0;
    }
    if (!more) return;
    if (tile_pages) {
      if (pre.t >= last) {
        first = pre.t;
        last = min(first + 32, pre.end);
        rows = first + lane < last ? row_of((first + lane) * kTile) : -1;
      }
      row = __shfl_sync(0xffffffffu, rows, pre.t - first);
      count = row < 0 ? 0 : min(pre.tokens - pre.t * kTile, kTile);
    } else {
      const int tok = pre.t * kTile + lane;
      row = lane < kTile && tok < pre.tokens ? row_of(tok) : -1;
    }
  };
  const uint32_t ring_s = static_cast<uint32_t>(__cvta_generic_to_shared(ring));
  constexpr int kChunks = D / 16, kRows = 32 / kChunks;  // chunks per row, rows per instruction
  const uint32_t to_lane = ring_s + lane / kChunks * kRow + lane % kChunks * 16;
  int put = 0;
  auto issue = [&]() {  // copies the tile that the cursor stands on, then moves the cursor on
    if (more) {
      const uint32_t st = ring_s + put * S::kStage, dst = to_lane + put * S::kStage;
      unsigned mask;
      if (tile_pages) {
        // rows behind the context are copied as K (their scores are masked), but not as V: a NaN there times a weight of 0
        const long long at = static_cast<long long>(count > 0 ? row : 0) * D + lane * 16;
        const uint8_t *kp = static_cast<const uint8_t*>(c.kc) + at, *vp = static_cast<const uint8_t*>(c.vc) + at;
#pragma unroll
        for (int i = 0; i < kTile / kRows; ++i) {
          cp_async16(dst + i * kRows * kRow, kp + i * 512, count > 0 ? 16 : 0);
          cp_async16(dst + (kTile + i * kRows) * kRow, vp + i * 512, i * kRows + lane / kChunks < count ? 16 : 0);
        }
        if (lane < 8)  // 16 scales of K, 16 of V
          cp_async16(st + 2 * kTile * kRow + lane * 16,
                     (lane < 4 ? c.ks : c.vs) + (count > 0 ? row : 0) + lane % 4 * 4, count > 0 ? 16 : 0);
        mask = (1u << count) - 1;
      } else {
#pragma unroll
        for (int i = 0; i < kTile / kRows; ++i) {
          const int rr = __shfl_sync(0xffffffffu, row, i * kRows + lane / kChunks);
          const long long at = static_cast<long long>(rr < 0 ? 0 : rr) * D + lane % kChunks * 16;
          cp_async16(dst + i * kRows * kRow, static_cast<const uint8_t*>(c.kc) + at, rr < 0 ? 0 : 16);
          cp_async16(dst + (kTile + i * kRows) * kRow, static_cast<const uint8_t*>(c.vc) + at, rr < 0 ? 0 : 16);
        }
        mask = __ballot_sync(0xffffffffu, row >= 0);
        if (lane < kTile) {
          const int rr = row < 0 ? 0 : row;
          cp_async4(st + 2 * kTile * kRow + lane * 4, c.ks + rr, row < 0 ? 0 : 4);
          cp_async4(st + 2 * kTile * kRow + kTile * 4 + lane * 4, c.vs + rr, row < 0 ? 0 : 4);
        }
      }
      if (lane == 0) *reinterpret_cast<unsigned*>(ring + put * S::kStage + 2 * kTile * kRow + 2 * kTile * 4) = mask;
      put = put + 1 == kStages ? 0 : put + 1;
      ++pre.t;
      look();
    }
    cp_commit();
  };
  // q of a portion as it lies in memory: asked for before what stands between the portions
  tb::Packed<T, 8> q_raw[NT][D / 32];
  auto ask_q = [&]() {
    const int h0 = cur.r / g.NG * g.G + cur.r % g.NG * kHeads, left = g.G - cur.r % g.NG * kHeads;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const T* q = static_cast<const T*>(a.q) + static_cast<long long>(cur.b) * a.qs_b +
                   static_cast<long long>(h0 + (n * 8 + gq < left ? n * 8 + gq : 0)) * a.qs_h + tq * (D / 4);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        if (q8) {
          q_raw[n][i].load(q + 8 * i);
        } else {
          const unsigned short* e = reinterpret_cast<const unsigned short*>(q + 8 * i);
          auto two = [&](int j) { return e[j] | static_cast<uint32_t>(e[j + 1]) << 16; };
          q_raw[n][i].raw = make_uint4(two(0), two(2), two(4), two(6));
        }
      }
    }
  };
  bool going = cur.t < cur.end;
  if (going) ask_q();
  look();
#pragma unroll 1
  for (int i = 0; i < kStages - 1; ++i) issue();
  if constexpr (!kClusters) {
    empty_rows(ctas);
    // which CTAs share the contexts at the two ends of this CTA's list (used by the merge, if they are split)
    if (w == 0) {
      if (lane == 0) shared[0] = sh.owner(sh.start(blockIdx.x * kWarps) - cur.t) / kWarps;
    } else if (w == kWarps - 1) {
      const uint32_t last = sh.start((blockIdx.x + 1) * kWarps) - 1;
      int b;
      uint32_t off;
      find(last, b, off);
      const uint32_t n = units(tokens_of(a, g, b));
      if (lane == 0) shared[1] = sh.owner(last + n - 1 - off % n) / kWarps;
    }
  }

  // ---- portions of this warp, one (sequence, group) each
  int get = 0;
  bool first_portion = true;
  while (going) {
    const int h0 = cur.r / g.NG * g.G + cur.r % g.NG * kHeads;  // first query head of the group
    const int left = g.G - cur.r % g.NG * kHeads, nh = left < kHeads ? left : kHeads;
    // q as B fragments: lane (head gq, tq) holds, for k step (i, j), the dimensions (tq NCH + i) 16 + 4 j .. + 3, the
    // same that it reads of a K row.  A power of two per head brings them into fp16's range.
    uint2 qf[NT * (D / 16)];
    float ch[NT][2], m[NT][2], l[NT][2], acc[2 * NW][NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float v[D / 4];
      uint32_t top = 0;
      const bool live = n * 8 + gq < nh;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        float f[8];
        q_raw[n][i].unpack(f);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[8 * i + e] = f[e];
      }
#pragma unroll
      for (int i = 0; i < D / 4; ++i) {
        if (!live) v[i] = 0.f;
        top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
      }
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int e2 = max(static_cast<int>(top >> 23) - 127, -100);
      const float f = pow2i(13 - e2);
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
        qf[i * NT + n] =
            make_uint2(pack_f16(v[4 * i] * f, v[4 * i + 1] * f), pack_f16(v[4 * i + 2] * f, v[4 * i + 3] * f));
      // 2^(e2 - 13), times the scale in units of log 2; a lane's columns are heads 2 tq and 2 tq + 1
      const float mine = a.scale * 1.4426950408889634f * pow2i(e2 - 13);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        ch[n][e] = __shfl_sync(0xffffffffu, mine, (2 * tq + e) * 4);
        m[n][e] = kLowest;
        l[n][e] = 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < 2 * NW; ++i)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][n][e] = 0.f;

    unsigned seen = 0;  // whether any token counted
    for (int t = cur.t; t < cur.end; ++t) {
      cp_wait<kStages - 2>();
      __syncwarp();
      issue();  // into the stage of the tile before
      const uint8_t* st = ring + get * S::kStage;
      const float* scales = reinterpret_cast<const float*>(st + 2 * kTile * kRow);
      const unsigned mask = *reinterpret_cast<const unsigned*>(st + 2 * kTile * kRow + 2 * kTile * 4);
      seen |= mask;
      // S^T [16 tokens, heads] = K q
      float s[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        const uint4 x = *reinterpret_cast<const uint4*>(st + gq * kRow + (tq * NCH + i) * 16);
        const uint4 y = *reinterpret_cast<const uint4*>(st + (gq + 8) * kRow + (tq * NCH + i) * 16);
        const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t a0, a1, a2, a3;
          widen(xs[j], a0, a2);
          widen(ys[j], a1, a3);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const uint2 b = qf[(i * 4 + j) * NT + n];
            mma16816(s[n], a0, a1, a2, a3, b.x, b.y);
          }
        }
      }
      // weights of tokens gq and gq + 8 for heads 2 tq and 2 tq + 1; tokens that do not count have a score of -inf
      const bool in0 = mask >> gq & 1, in1 = mask >> (gq + 8) & 1;
      const float k0 = scales[gq], k1 = scales[gq + 8];
      const float v0 = in0 ? scales[kTile + gq] : 0.f, v1 = in1 ? scales[kTile + gq + 8] : 0.f;
      const float e0 = fmaxf(log2_fast(v0), kMinVsLog), e1 = fmaxf(log2_fast(v1), kMinVsLog);
      bool grew = false;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          s[n][e] = in0 ? s[n][e] * ch[n][e] * k0 : -INFINITY;
          s[n][2 + e] = in1 ? s[n][2 + e] * ch[n][e] * k1 : -INFINITY;
          grew |= fmaxf(s[n][e] + e0, s[n][2 + e] + e1) > __fadd_rd(m[n][e], kSlack);
        }
      if (__any_sync(0xffffffffu, grew)) {  // the maximum outran the reference: move it, and what was summed with it
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float top = fmaxf(s[n][e] + e0, s[n][2 + e] + e1);
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
            top = fmaxf(top - kAhead, m[n][e]);
            const float cor = exp2_fast(m[n][e] - top);
            m[n][e] = top;
            l[n][e] *= cor;
#pragma unroll
            for (int i = 0; i < 2 * NW; ++i) {
              acc[i][n][e] *= cor;
              acc[i][n][2 + e] *= cor;
            }
          }
      }
      uint32_t wb[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float p[4];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          p[e] = exp2_fast(s[n][e] - m[n][e]);
          p[2 + e] = exp2_fast(s[n][2 + e] - m[n][e]);
          l[n][e] += p[e] + p[2 + e];
        }
        wb[n][0] = transpose8x8(pack_f16(p[0] * v0, p[1] * v0));
        wb[n][1] = transpose8x8(pack_f16(p[2] * v1, p[3] * v1));
      }
      // O^T [16 dimensions, heads] += V^T w: bytes of neighbouring tokens are paired before they are widened
      const uint8_t* vr = st + kTile * kRow + 2 * tq * kRow;
#pragma unroll
      for (int kk = 0; kk < NW; kk += (NW < 4 ? NW : 4)) {
        constexpr int U = NW < 4 ? NW : 4;  // words per load
        using V = typename tb::RawOf<U * 4>::type;
        const int at = NW < 4 ? gq * 8 : (kk / 4) * 128 + gq * 16;
        V r[4];
        r[0] = *reinterpret_cast<const V*>(vr + at);
        r[1] = *reinterpret_cast<const V*>(vr + kRow + at);
        r[2] = *reinterpret_cast<const V*>(vr + 8 * kRow + at);
        r[3] = *reinterpret_cast<const V*>(vr + 9 * kRow + at);
        const uint32_t* rw[4] = {reinterpret_cast<const uint32_t*>(&r[0]), reinterpret_cast<const uint32_t*>(&r[1]),
                                 reinterpret_cast<const uint32_t*>(&r[2]), reinterpret_cast<const uint32_t*>(&r[3])};
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const uint32_t lo0 = __byte_perm(rw[0][u], rw[1][u], 0x5140), hi0 = __byte_perm(rw[0][u], rw[1][u], 0x7362);
          const uint32_t lo1 = __byte_perm(rw[2][u], rw[3][u], 0x5140), hi1 = __byte_perm(rw[2][u], rw[3][u], 0x7362);
          uint32_t a0, a1, a2, a3, c0, c1, c2, c3;
          widen(lo0, a0, a1);
          widen(lo1, a2, a3);
          widen(hi0, c0, c1);
          widen(hi1, c2, c3);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma16816(acc[2 * (kk + u)][n], a0, a1, a2, a3, wb[n][0], wb[n][1]);
            mma16816(acc[2 * (kk + u) + 1][n], c0, c1, c2, c3, wb[n][0], wb[n][1]);
          }
        }
      }
      get = get + 1 == kStages ? 0 : get + 1;
    }

    // ---- the end of the portion: a whole context is written out, a part kept for the CTA's merge
    const bool opens = cur.t == 0;
    const bool closes = cur.end == tiles(cur.tokens);
    const int b = cur.b, r = cur.r;
    going = next_portion(a, g, cur);
    if (going) ask_q();
    const float nothing = seen ? NAN : 0.f;
    float* part = first_portion ? first_part : reinterpret_cast<float*>(ring);
    if (!first_portion && !(opens && closes)) {  // the list's last portion: the ring is done with
      cp_wait<0>();
      __syncwarp();
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int h = n * 8 + 2 * tq + e;
        float v = l[n][e];
        v += __shfl_xor_sync(0xffffffffu, v, 4);
        v += __shfl_xor_sync(0xffffffffu, v, 8);
        v += __shfl_xor_sync(0xffffffffu, v, 16);
        const float inv = v == 0.f ? nothing : 1.f / v;
        T* o = static_cast<T*>(a.out) + static_cast<long long>(b) * a.os_b + static_cast<long long>(h0 + h) * a.os_h;
#pragma unroll
        for (int k = 0; k < NW; ++k) {
          const int d = NW < 4 ? gq * 8 + 4 * k : (k / 4) * 128 + gq * 16 + 4 * (k % 4);
          const float y0 = acc[2 * k][n][e], y1 = acc[2 * k][n][2 + e], y2 = acc[2 * k + 1][n][e],
                      y3 = acc[2 * k + 1][n][2 + e];
          if (opens && closes) {
            if (h < nh) store_out4<T>(o + d, out4, y0 * inv, y1 * inv, y2 * inv, y3 * inv);
          } else {
            *reinterpret_cast<float4*>(part + h * D + d) = make_float4(y0, y1, y2, y3);
          }
        }
        if (!(opens && closes) && gq == 0)
          *reinterpret_cast<float2*>(part + kHeads * D + 2 * h) = make_float2(seen ? m[n][e] : -INFINITY, v);
      }
    if (!(opens && closes) && lane == 0)
      meta[2 * w + (first_portion ? 0 : 1)] = make_int2(b * g.HG + r, (opens ? 1 : 0) | (closes ? 2 : 0));
    first_portion = false;
  }
  cp_wait<0>();
  if constexpr (kClusters) {
    cluster_join<T, D>(a, g, smem, meta, out4);
    return;
  }
  __syncthreads();
  tb::pdl_trigger();

  // ---- merge the parts of this CTA: those of the same (sequence, group), a warp for each query head
  constexpr int E = D / 32, V = E < 4 ? E : 4;
  const int2 mt = lane < 2 * kWarps ? meta[lane] : make_int2(-1, 0);
  bool first_run = true;
  int turn = 0;  // (set of parts, head) pairs so far: they go round the warps
#pragma unroll 1
  for (unsigned parts = __ballot_sync(0xffffffffu, mt.x >= 0); parts != 0;) {
    const int seg = __shfl_sync(0xffffffffu, mt.x, __ffs(parts) - 1);
    const unsigned set = __ballot_sync(0xffffffffu, mt.x == seg);
    const bool opens = __any_sync(0xffffffffu, mt.x == seg && mt.y & 1);
    const bool whole = __any_sync(0xffffffffu, mt.x == seg && mt.y & 2) && opens;
    parts &= ~set;
    const int b = seg / g.HG, r = seg - b * g.HG, kh = r / g.NG, left = g.G - (r - kh * g.NG) * kHeads;
    const int nh = min(left, kHeads), h0 = kh * g.G + g.G - left;
    const long long slot = 2ll * blockIdx.x + (first_run ? 0 : 1);
    first_run = false;
    if (!whole && threadIdx.x == 0) {  // a part of a context that other CTAs share
      int4* rec = P::record(a.ws, gridDim.x, blockIdx.x);
      if (opens) {
        rec->x = seg;
        rec->y = static_cast<int>(slot);
        rec->z = shared[1] - static_cast<int>(blockIdx.x) + 1;
      } else {
        rec->w = shared[0];
      }
    }
    auto part_of = [&](int p) {
      return reinterpret_cast<const float*>(smem + (p % 2 ? p / 2 * S::kRing : kWarps * S::kRing + p / 2 * S::kPart));
    };
#pragma unroll 1
    for (int h = (w - turn) & (kWarps - 1); h < nh; h += kWarps) {
      float M = -INFINITY, L = 0.f, o[E] = {};
      for (unsigned r = set; r; r &= r - 1) M = fmaxf(M, part_of(__ffs(r) - 1)[kHeads * D + 2 * h]);
      for (unsigned r = set; r; r &= r - 1) {
        const float* p = part_of(__ffs(r) - 1);
        const float2 st = *reinterpret_cast<const float2*>(p + kHeads * D + 2 * h);
        const float f = st.x == -INFINITY ? 0.f : exp2_fast(st.x - M);
        L += f * st.y;
#pragma unroll
        for (int i = 0; i < E; i += V) {
          float y[V];
          tb::load_vec<float, V>(p + h * D + i * 32 + lane * V, y);
#pragma unroll
          for (int e = 0; e < V; ++e) o[i + e] += f * y[e];
        }
      }
      const float inv = !whole ? 1.f : L == 0.f ? of_nothing(M) : 1.f / L;
      T* out = static_cast<T*>(a.out) + static_cast<long long>(b) * a.os_b + static_cast<long long>(h0 + h) * a.os_h;
      float* part = P::out(a.ws, slot, h);
#pragma unroll
      for (int i = 0; i < E; i += V) {
        float y[V];
#pragma unroll
        for (int e = 0; e < V; ++e) y[e] = o[i + e] * inv;
        if (!whole) {
          tb::store_vec<float, V>(part + i * 32 + lane * V, y);
        } else if (out4) {
          tb::store_vec<T, V>(out + i * 32 + lane * V, y);
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) out[i * 32 + lane * V + e] = tb::from_f32<T>(y[e]);
        }
      }
      if (!whole && lane == 0) *reinterpret_cast<float2*>(P::stat(a.ws, slot, h)) = make_float2(M, L);
    }
    turn += nh;
  }
}

// Joins the contexts that were split over CTAs.  Up to kFewParts parts: the CTA
// of the first part joins them, a warp for each query head.  More: each of the CTAs
// that share the context joins a slice of a query head, its lanes and warps
// different parts.
constexpr int kFewParts = 16, kJoinWarps = 8;

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kJoinWarps * 32)
    decode_attn_quant_join_kernel(TbDecodeAttnQuantArgs a, Geometry g, int grid, bool out4) {
  using P = Partials<D, NT>;
  static_assert(P::kHeads <= kFewParts + 1, "a CTA for each head of a context with many parts");
  constexpr int E = D / 32, V = E < 4 ? E : 4;
  __shared__ float red[kJoinWarps], sl[kJoinWarps], so[kJoinWarps][D];
  tb::pdl_wait();
  const int4 mine = *P::record(a.ws, grid, blockIdx.x);
  const int w = threadIdx.x / 32, lane = threadIdx.x % 32;
  auto add = [&](float (&o)[E], float f, const float* v) {
#pragma unroll
    for (int i = 0; i < E; i += V) {
      float x[V];
      tb::load_vec<float, V>(v + i * 32 + lane * V, x);
#pragma unroll
      for (int e = 0; e < V; ++e) o[i + e] += f * x[e];
    }
  };
  auto write = [&](int seg, int h, float inv, const float (&o)[E]) {
    const int r = seg % g.HG, head = r / g.NG * g.G + r % g.NG * P::kHeads + h;
    T* p = static_cast<T*>(a.out) + static_cast<long long>(seg / g.HG) * a.os_b + static_cast<long long>(head) * a.os_h +
           lane * V;
#pragma unroll
    for (int i = 0; i < E; i += V) {
      float x[V];
#pragma unroll
      for (int e = 0; e < V; ++e) x[e] = o[i + e] * inv;
      if (out4) {
        tb::store_vec<T, V>(p + i * 32, x);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) p[i * 32 + e] = tb::from_f32<T>(x[e]);
      }
    }
  };
  auto heads_of = [&](int seg) {
    const int left = g.G - seg % g.HG % g.NG * P::kHeads;
    return left < P::kHeads ? left : P::kHeads;
  };
  if (mine.z > 0 && mine.z <= kFewParts) {
    const int nh = heads_of(mine.x);
    for (int h = w; h < nh; h += kJoinWarps) {
      const long long slot = lane == 0 ? mine.y : 2ll * (blockIdx.x + lane);
      const float* st = P::stat(a.ws, slot, h);
      const float m = lane < mine.z ? st[0] : -INFINITY;
      const float M = tb::warp_max(m);
      const float f = lane < mine.z ? exp2_fast(m - (M == -INFINITY ? 0.f : M)) : 0.f;
      const float L = tb::warp_sum(lane < mine.z ? f * st[1] : 0.f);
      float o[E] = {};
#pragma unroll 4
      for (int p = 0; p < mine.z; ++p)
        add(o, __shfl_sync(0xffffffffu, f, p), P::out(a.ws, p == 0 ? mine.y : 2ll * (blockIdx.x + p), h));
      write(mine.x, h, L == 0.f ? of_nothing(M) : 1.f / L, o);
    }
  }
#pragma unroll 1
  for (int role = 0; role < 2; ++role) {  // the first of a long run; one of the others
    const int lead = role == 0 ? static_cast<int>(blockIdx.x) : mine.w;
    if (lead < 0) continue;
    const int4 rec = role == 0 ? mine : *P::record(a.ws, grid, lead);
    if (rec.z <= kFewParts) continue;
    // slices of a head's dimensions, so that more of the CTAs that share the context take part
    const int nh = heads_of(rec.x), n = rec.z;
    int slices = 1;
    while (2 * slices <= D / 32 && 2 * slices * nh <= n) slices *= 2;
    const int item = blockIdx.x - lead, h = item / slices, size = D / slices;
    if (h >= nh) continue;  // the same for the whole CTA
    auto slot = [&](int p) { return p == 0 ? static_cast<long long>(rec.y) : 2ll * (lead + p); };
    float M = -INFINITY;
    for (int p = threadIdx.x; p < n; p += kJoinWarps * 32) M = fmaxf(M, P::stat(a.ws, slot(p), h)[0]);
    M = tb::warp_max(M);
    __syncthreads();
    if (lane == 0) red[w] = M;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kJoinWarps; ++i) M = fmaxf(M, red[i]);
    const float m0 = M == -INFINITY ? 0.f : M;
    // `lanes` lanes hold a part's slice, four dimensions each (at D = 256 in one slice: and the four 128 further)
    const int lanes = min(size / 4, 32), at_once = 32 / lanes, d = item % slices * size + lane % lanes * 4;
    const bool wide = D == 256 && size == 256;
    float L = 0.f, o[8] = {};
#pragma unroll 4
    for (int p = w * at_once + lane / lanes; p < n; p += kJoinWarps * at_once) {
      const float2 st = *reinterpret_cast<const float2*>(P::stat(a.ws, slot(p), h));
      const float f = exp2_fast(st.x - m0), *v = P::out(a.ws, slot(p), h) + d;
      L += f * st.y;
      float x[4];
      tb::load_vec<float, 4>(v, x);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += f * x[e];
      if (wide) {
        tb::load_vec<float, 4>(v + 128, x);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[4 + e] += f * x[e];
      }
    }
    for (int x = lanes; x < 32; x *= 2) {
      L += __shfl_xor_sync(0xffffffffu, L, x);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += __shfl_xor_sync(0xffffffffu, o[e], x);
    }
    if (lane == 0) sl[w] = L;
    if (lane < lanes) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        so[w][lane * 4 + e] = o[e];
        if (wide) so[w][128 + lane * 4 + e] = o[4 + e];
      }
    }
    __syncthreads();
    if (threadIdx.x < size) {
      float sum = 0.f, l = 0.f;
#pragma unroll
      for (int x = 0; x < kJoinWarps; ++x) {
        l += sl[x];
        sum += so[x][threadIdx.x];
      }
      const int r = rec.x % g.HG, head = r / g.NG * g.G + r % g.NG * P::kHeads + h;
      static_cast<T*>(a.out)[static_cast<long long>(rec.x / g.HG) * a.os_b + static_cast<long long>(head) * a.os_h +
                             item % slices * size + threadIdx.x] = tb::from_f32<T>(l == 0.f ? of_nothing(M) : sum / l);
    }
  }
}

int sm_count() {  // of the current device, asked for once
  constexpr int kDevices = 64;
  static std::atomic<int> known[kDevices];
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0) return 148;
  if (dev < kDevices) n = known[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
    if (dev < kDevices) known[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

// How the work of `segs` (sequence, group) pairs with contexts of up to `cap`
// tokens is dealt out: a cluster of so many CTAs for each pair, or 0, the even
// lists.  The lists pay for their start and for the joining kernel, a cluster for
// the longest context, with a warp's latency per tile, and for the memory that all
// of them share.  Measured on one B200 (D = 128): lists 10.5 us and 0.76 ns per tile, of
// which contexts of mixed lengths have half of `cap`; clusters 5.7 us, 0.85 us per
// tile of a warp and a fifth of the lists' time for the tiles.  Clusters and lists: 1 x
// 1,000 tokens x 8 KV heads 6.2 and 10.4 us, 8 x 4,096 x 8 17.9 and 22.2, 37 ragged up to
// 1,536 x 8 18.3 and 20.2, 64 x 1,000 x 8 26.9 and 33.1 (ragged 21.2 and 21.8), 16 ragged
// up to 8,000 x 8 35.1 and 32.3.  The numbers were fitted there and serve D = 64 and 256
// too, where the same contexts take 5.6 and 9.9, 13.6 and 17.4, 14.0 and 15.9, 18.6 and
// 23.8 (16.0 and 17.1), 26.1 and 23.9 us at 64; 7.9 and 11.8, 29.2 and 33.4 (lists are
// taken), 32.5 and 29.6, 55 either way (32.1 and 32.2), 70 and 52 us at 256.  Where it is
// farthest off, lists are taken for contexts of one length that just fill the machine:
// 100 x 1,600 x 4 in 38 us for 32 (D = 64: 27 for 22).
// Lists count their units in 31 bits; more take the clusters.
int cluster_of(int segs, int cap, int fit) {
  const long long tiles = cap / kTile + 1, units = (tiles + kStart) * segs;
  if (units > 0x7fffffff) return 1;
  if (segs > fit) return 0;
  int cs = 1;
  while (cs < kMostCluster && 2 * cs * segs <= fit && cs * kWarps < tiles) cs *= 2;
  const double all = segs * tiles * 0.0004;
  return 5.7 + 0.85 * ((tiles + cs * kWarps - 1) / (cs * kWarps)) + 0.2 * all < 10.5 + all ? cs : 0;
}

// CTAs of a cluster for each (sequence, eight query heads), or 0: even lists.
template <int D>
int clusters(int B, int Hq, int Hk, int cap) {
  return cluster_of(B * Hk * ((Hq / Hk + 7) / 8), cap, sm_count() * resident<D, 1>());
}

template <int D, int NT>
Geometry geometry(const TbDecodeAttnQuantArgs& a) {
  Geometry g;
  g.G = a.Hq / a.cache.Hk;
  g.NG = (g.G + 8 * NT - 1) / (8 * NT);
  g.HG = a.cache.Hk * g.NG;
  g.cap = a.cache.max_blocks * a.cache.bs;
  g.shift = -1;
  for (int i = 0; i < 31; ++i)
    if (a.cache.bs == 1 << i) g.shift = i;
  g.tile_pages = a.cache.bs % kTile == 0;
  g.cs = NT == 1 ? clusters<D>(a.B, a.Hq, a.cache.Hk, g.cap) : 0;
  return g;
}

template <typename T, int D, int NT, bool kPlain>
int launch_as(const TbDecodeAttnQuantArgs& a, const Geometry& g, bool q8, bool out4, cudaStream_t s) {
  using S = Smem<D, NT>;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = S::kBytes;
  cfg.stream = s;
  cfg.attrs = attr;
  if constexpr (NT == 1) {
    if (g.cs) {
      auto kernel = decode_attn_quant_kernel<T, D, 1, true, kPlain>;
      const cudaError_t e = tb::ensure_dyn_smem(reinterpret_cast<const void*>(kernel), S::kBytes);
      if (e != cudaSuccess) return static_cast<int>(e);
      cfg.gridDim = dim3(a.B * g.HG * g.cs);
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim = {static_cast<unsigned>(g.cs), 1, 1};
      cfg.numAttrs = 1;
      if (g.cs > 1) return static_cast<int>(cudaLaunchKernelEx(&cfg, kernel, a, g, q8, out4));
      kernel<<<cfg.gridDim, kThreads, S::kBytes, s>>>(a, g, q8, out4);
      return static_cast<int>(cudaGetLastError());
    }
  }
  auto kernel = decode_attn_quant_kernel<T, D, NT, false, kPlain>;
  const cudaError_t e = tb::ensure_dyn_smem(reinterpret_cast<const void*>(kernel), S::kBytes);
  if (e != cudaSuccess) return static_cast<int>(e);
  const int grid = sm_count() * list_ctas<D, NT>();
  if (a.ws == nullptr || a.ws_bytes < Partials<D, NT>::bytes(grid)) return static_cast<int>(cudaErrorInvalidValue);
  kernel<<<grid, kThreads, S::kBytes, s>>>(a, g, q8, out4);
  const cudaError_t e1 = cudaGetLastError();
  if (e1 != cudaSuccess) return static_cast<int>(e1);
  // programmatic launch: the joining CTAs are in place when the last list ends
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kJoinWarps * 32);
  cfg.dynamicSmemBytes = 0;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.numAttrs = 1;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, decode_attn_quant_join_kernel<T, D, NT>, a, g, grid, out4));
}

template <typename T, int D, int NT>
int launch(const TbDecodeAttnQuantArgs& a, cudaStream_t s) {
  const Geometry g = geometry<D, NT>(a);
  const bool q8 = reinterpret_cast<uintptr_t>(a.q) % 16 == 0 && a.qs_b % 8 == 0 && a.qs_h % 8 == 0;
  const bool out4 = reinterpret_cast<uintptr_t>(a.out) % 8 == 0 && a.os_b % 4 == 0 && a.os_h % 4 == 0;
  return g.tile_pages && q8 && out4 ? launch_as<T, D, NT, true>(a, g, q8, out4, s)
                                    : launch_as<T, D, NT, false>(a, g, q8, out4, s);
}

// Query heads that a warp takes, in eights: two where more than 8 share a KV head,
// which widens the pages once for both (64 x 1,000 tokens x 8 KV heads, 16 query heads
// on each: 41 us against 50 with one; D = 64: 46 against 59), but in clusters one, for the
// shorter way of a tile (1 x 2,000 tokens, 16 heads on 1: 9.2 us against 11.2), and for D =
// 256 one, whose output fills the registers (64 x 1,000 x 4 KV heads, 16 on each: 59 against
// 66, both before tiles were looked up 32 at a time; 49 now).
template <int D>
bool take_two(int B, int Hq, int Hk, int cap) {
  return D < 256 && Hq / Hk > 8 && clusters<D>(B, Hq, Hk, cap) == 0;
}

template <typename T, int D>
int launch_dim(const TbDecodeAttnQuantArgs& a, cudaStream_t s) {
  if constexpr (D < 256)
    if (take_two<D>(a.B, a.Hq, a.cache.Hk, a.cache.max_blocks * a.cache.bs)) return launch<T, D, 2>(a, s);
  return launch<T, D, 1>(a, s);
}

template <typename T>
int launch_type(const TbDecodeAttnQuantArgs& a, cudaStream_t s) {
  switch (a.cache.D) {
    case 64: return launch_dim<T, 64>(a, s);
    case 128: return launch_dim<T, 128>(a, s);
    case 256: return launch_dim<T, 256>(a, s);
  }
  return static_cast<int>(cudaErrorInvalidValue);
}

template <int D>
size_t ws_bytes(int B, int Hq, int Hk, int cap) {
  if (clusters<D>(B, Hq, Hk, cap)) return 0;
  return take_two<D>(B, Hq, Hk, cap) ? Partials<D, 2>::bytes(sm_count() * list_ctas<D, 2>())
                                     : Partials<D, 1>::bytes(sm_count() * list_ctas<D, 1>());
}

}  // namespace

extern "C" size_t tb_decode_attention_quant_ws_bytes(int B, int Hq, int Hk, int D, int max_tokens) {
  if (B <= 0 || Hk <= 0) return 0;
  switch (D) {
    case 64: return ws_bytes<64>(B, Hq, Hk, max_tokens);
    case 128: return ws_bytes<128>(B, Hq, Hk, max_tokens);
    case 256: return ws_bytes<256>(B, Hq, Hk, max_tokens);
  }
  return 0;
}

extern "C" int tb_decode_attention_quant(const TbDecodeAttnQuantArgs* args, cudaStream_t s) {
  const TbDecodeAttnQuantArgs& a = *args;
  if (a.B <= 0 || a.Hq <= 0) return 0;
  if (a.cache.Hk <= 0 || a.Hq % a.cache.Hk || a.cache.bs <= 0 || a.cache.num_seqs != a.B ||
      a.cache.max_blocks < 0 || a.cache.max_blocks > 0x7fffffff / a.cache.bs || a.cache.num_blocks < 0 ||
      static_cast<long long>(a.cache.num_blocks) * a.cache.Hk > 0x7fffffff / a.cache.bs ||
      a.B > 0x7fffffff / a.Hq || static_cast<long long>(a.Hq) * a.cache.D > 0x7fffffff)
    return static_cast<int>(cudaErrorInvalidValue);
  if (a.dtype == TB_BF16) return launch_type<__nv_bfloat16>(a, s);
  if (a.dtype == TB_F16) return launch_type<__half>(a, s);
  return static_cast<int>(cudaErrorInvalidValue);
}
