// Embedding lookup with a scale, and its gradient:
//
//   y_t = s W[id_t],      dW[v] (+)= s sum_{t: id_t = v} dy_t.
//
// Both move bytes (one product and one addition per value).  The gradient's sums are
// fp32 in a fixed order, so the same inputs give the same bits:
//
// * Few tokens: one CTA for each token and slab of columns.  The first token of an id
//   finds the others by comparing all ids and sums their rows; one launch, no workspace.
// * More: the tokens are sorted by id (stable, so by token within an id); then each CTA
//   sums a piece of 128 sorted tokens for 256 columns, a warp 16 of them.  An id whose
//   tokens lie within a warp's share is finished there, one within the piece after an
//   exchange over shared memory; what goes on into other pieces is left in a workspace, and
//   a last launch adds it up.  A token that fills a third of the batch is thus spread over
//   the machine like any other.
//
// Up to 8,192 tokens the sort counts, for each token, the ones before it (N^2 comparisons
// in one launch); above it is a radix sort in digits of up to 9 bits, one launch to count
// the first digit and one for each digit, which also counts the next one.
//
// What bounds it, measured with bf16 rows: the lookup moves its bytes (16,384 rows of 4,096:
// 32 us; 134 MB written and as much asked for, of which the repeated rows come out of the L2
// cache: 151 MB from and to DRAM, 4.7 TB/s); the sums do where rows are 16-byte vectors (the
// same batch: 48 us beside no zeros, 134 MB read and as much written), while rows of odd length
// take an element per lane (65,537 of 1,025 fp16: 59 us, 134 MB read, 40% of the copy rate) and
// small batches the chain of launches (6,144 tokens of 1,536: sort 11, sums 16, join 5 us, of
// 19 MB).  The sort waits on shared memory and on its own launches: 11 us for 6,144 tokens, 24
// for 65,537.  Narrow rows are all sort and launches: 12,000 tokens of 64 columns take 33 us and
// 65,536 43 (floors of 0.8 and 3.3), where unordered additions of fp32 rows take 14 and 41.
#include <limits.h>
#include <math.h>

#include "device_common.cuh"
#include "kernels.h"
#include "pdl.cuh"
#include "vec_io.cuh"

namespace {

__device__ __forceinline__ long long id_of(const void* ids, int ids64, long long t) {
  return ids64 ? static_cast<const long long*>(ids)[t] : static_cast<const int*>(ids)[t];
}

// A token's row in the lookup: whether it has one, and (in place of the id) where.
__device__ __forceinline__ bool row_of(const TbEmbeddingArgs& a, long long& id, bool tells) {
  if (id >= 0 && id < a.V) return true;
  if ((id >= a.V || a.first_row) && a.err && tells) *a.err = 1;
  if (!a.first_row) return false;
  id = 0;
  return true;
}

// ---- rows of any alignment: 16 bytes that begin `shift` bytes into the first of two vectors.
// (What lies beside a row within its tensor is read along and not used.)
template <typename T>
struct Two {
  static constexpr int E = 16 / sizeof(T);
  uint4 a, b;
  __device__ __forceinline__ static unsigned shift_of(const T* p) { return static_cast<unsigned>(reinterpret_cast<uintptr_t>(p) & 15); }
  // Whether the vectors that hold the elements [p, p + n) lie between first and last.
  __device__ __forceinline__ static bool inside(const T* p, int n, const T* first, const T* last) {
    return p - shift_of(p) / sizeof(T) >= first && p + (n + E - 1) / E * E + E <= last;
  }
  __device__ __forceinline__ void load(const T* p) {
    const uint4* v = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(p) & ~static_cast<uintptr_t>(15));
    a = v[0];
    b = v[1];
  }
  __device__ __forceinline__ void values(unsigned s, float (&x)[E]) const {
    uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 6; ++i) w[i] = s & 8 ? w[i + 2] : w[i];
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = s & 4 ? w[i + 1] : w[i];
    uint4 q;
    q.x = __funnelshift_r(w[0], w[1], (s & 3) * 8);
    q.y = __funnelshift_r(w[1], w[2], (s & 3) * 8);
    q.z = __funnelshift_r(w[2], w[3], (s & 3) * 8);
    q.w = __funnelshift_r(w[3], w[4], (s & 3) * 8);
    const T* e = reinterpret_cast<const T*>(&q);
#pragma unroll
    for (int j = 0; j < E; ++j) x[j] = tb::to_f32(e[j]);
  }
};

// ------------------------------------------------------------------ lookup
constexpr int kUnroll = 4;  // vectors that a lane has in flight

// A warp takes 32 x kUnroll vectors of a row (aligned rows of 32 vectors and more).
template <typename T>
__global__ void __launch_bounds__(256) lookup_wide_kernel(TbEmbeddingArgs a, int segs) {
  constexpr int E = 16 / sizeof(T);
  const int lane = threadIdx.x & 31, per = a.H / E;
  const long long tasks = static_cast<long long>(a.N) * segs;
  for (long long task = blockIdx.x * 8ll + threadIdx.x / 32; task < tasks; task += gridDim.x * 8ll) {
    const long long t = segs == 1 ? task : task / segs;
    const int first = static_cast<int>(task - t * segs) * 32 * kUnroll + lane;
    long long id = id_of(a.ids, a.ids64, t);
    const bool good = row_of(a, id, lane == 0);
    const T* src = static_cast<const T*>(a.weight) + (good ? id : 0) * a.ld_w;
    T* dst = static_cast<T*>(a.out) + t * a.ld_out;
    tb::Packed<T, E> p[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (first + u * 32 < per && good) p[u].load(src + (first + u * 32) * E);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (first + u * 32 < per) {
        float x[E];
        p[u].unpack(x);
#pragma unroll
        for (int j = 0; j < E; ++j) x[j] = good ? x[j] * a.scale : id < 0 ? 0.f : NAN;
        tb::store_vec<T, E>(dst + (first + u * 32) * E, x);
      }
  }
}

// The same for rows of any alignment, a row per warp: the output's whole vectors, then the
// elements before and behind them.
template <typename T>
__global__ void __launch_bounds__(256) lookup_shift_kernel(TbEmbeddingArgs a) {
  constexpr int E = 16 / sizeof(T);
  const int lane = threadIdx.x & 31;
  const T* table = static_cast<const T*>(a.weight);
  const T* end = table + (a.V - 1) * a.ld_w + a.H;
  for (long long t = blockIdx.x * 8ll + threadIdx.x / 32; t < a.N; t += gridDim.x * 8ll) {
    long long id = id_of(a.ids, a.ids64, t);
    const bool good = row_of(a, id, lane == 0);
    const T* src = table + (good ? id : 0) * a.ld_w;
    T* dst = static_cast<T*>(a.out) + t * a.ld_out;
    const auto one = [&](int h) { dst[h] = tb::from_f32<T>(good ? tb::to_f32(src[h]) * a.scale : id < 0 ? 0.f : NAN); };
    const int head = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(dst) & 15)) & 15) / static_cast<int>(sizeof(T));
    const int per = (a.H - head) / E;
    if (!good || !Two<T>::inside(src + head, per * E, table, end)) {
#pragma unroll 4
      for (int h = lane; h < a.H; h += 32) one(h);
      continue;
    }
    const unsigned s = Two<T>::shift_of(src + head);
    for (int v = lane; v < per; v += 32 * kUnroll) {
      Two<T> p[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (v + u * 32 < per) p[u].load(src + head + (v + u * 32) * E);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (v + u * 32 < per) {
          float x[E];
          p[u].values(s, x);
#pragma unroll
          for (int j = 0; j < E; ++j) x[j] *= a.scale;
          tb::store_vec<T, E>(dst + head + (v + u * 32) * E, x);
        }
    }
    const int tail = head + per * E;
    if (lane < head) one(lane);
    if (tail + lane < a.H) one(tail + lane);
  }
}

// A thread for every N elements (shorter rows).
template <typename T, int N>
__global__ void __launch_bounds__(256) lookup_narrow_kernel(TbEmbeddingArgs a) {
  const int per = a.H / N;
  const long long total = static_cast<long long>(a.N) * per;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    const long long t = total <= UINT_MAX ? static_cast<unsigned>(i) / static_cast<unsigned>(per) : i / per;
    const int h = static_cast<int>(i - t * per) * N;
    long long id = id_of(a.ids, a.ids64, t);
    const bool good = row_of(a, id, true);
    float x[N];
    if (good) tb::load_vec<T, N>(static_cast<const T*>(a.weight) + id * a.ld_w + h, x);
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = good ? x[j] * a.scale : id < 0 ? 0.f : NAN;
    tb::store_vec<T, N>(static_cast<T*>(a.out) + t * a.ld_out + h, x);
  }
}

// ------------------------------------------------------------------ gradient
// Adds (or writes) a finished sum of N columns of row `id`.
template <typename G, int N>
__device__ __forceinline__ void finish(const TbEmbeddingGradArgs& a, bool vec, long long id, int h, const float (&sum)[N]) {
  G* p = static_cast<G*>(a.grad) + id * a.ld_grad + h;
  float x[N];
#pragma unroll
  for (int j = 0; j < N; ++j) x[j] = sum[j] * a.scale;
  if constexpr (sizeof(G) == 4) {
    if (!a.zero) {  // each element has one addition per call: the order is fixed
      if (N % 4 == 0 && vec) {
#pragma unroll
        for (int j = 0; j < N; j += 4) atomicAdd(reinterpret_cast<float4*>(p + j), make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]));
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j) atomicAdd(p + j, x[j]);
      }
      return;
    }
  }
  if (!vec) {
#pragma unroll
    for (int j = 0; j < N; ++j) p[j] = tb::from_f32<G>(a.zero ? x[j] : tb::to_f32(p[j]) + x[j]);
    return;
  }
  if (!a.zero) {
    float old[N];
    tb::load_vec<G, N>(p, old);
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] += old[j];
  }
  tb::store_vec<G, N>(p, x);
}

// Tokens of the one-launch form (512 of 1,536 bf16 take 11.5 us with it and 15.4 sorted, 64 take
// 3.0 and 9.5).  The rule looks at the tokens alone, and so loses where hundreds of tokens have
// wide rows, whose every slab compares the ids again (512 of 4,096 columns: 25.8 and 20.4).
constexpr int kFew = 512;

template <typename T, typename G, int N>
__global__ void __launch_bounds__(256) grad_few_kernel(TbEmbeddingGradArgs a, int slabs, bool vec) {
  __shared__ unsigned hit[kFew / 32];
  __shared__ int list[kFew];
  __shared__ float part[8][32 * N];
  const int t = blockIdx.x / slabs, slab = blockIdx.x % slabs;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long id = id_of(a.ids, a.ids64, t);
  if (id < 0) return;
  if (id >= a.V) {
    if (a.err && threadIdx.x == 0) *a.err = 1;
    return;
  }
  // the tokens of this id; an earlier one among them has the sum
  int earlier = 0;
  for (int u = threadIdx.x; u < kFew; u += 256) {
    const bool same = u < a.N && id_of(a.ids, a.ids64, u) == id;
    const unsigned b = __ballot_sync(0xffffffffu, same);
    if (lane == 0) hit[u / 32] = b;
    earlier |= same && u < t;
  }
  if (__syncthreads_or(earlier)) return;
  int n = 0;
  for (int w = 0; w < kFew / 32; ++w) n += __popc(hit[w]);
  for (int u = threadIdx.x; u < kFew; u += 256) {
    const unsigned b = hit[u / 32];
    if (b >> lane & 1) {
      int at = __popc(b & ((1u << lane) - 1));
      for (int w = 0; w < u / 32; ++w) at += __popc(hit[w]);
      list[at] = u;
    }
  }
  __syncthreads();
  const int h = (slab * 32 + lane) * N;
  float sum[N];
#pragma unroll
  for (int j = 0; j < N; ++j) sum[j] = 0.f;
  const int lo = n * warp / 8, hi = n * (warp + 1) / 8;  // (one token: the last warp)
  if (h < a.H) {
    const T* dy = static_cast<const T*>(a.dy) + h;
    for (int i = lo; i < hi; i += 4) {
      tb::Packed<T, N> p[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (i + u < hi) p[u].load(dy + list[i + u] * a.ld_dy);
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (i + u < hi) {
          float x[N];
          p[u].unpack(x);
#pragma unroll
          for (int j = 0; j < N; ++j) sum[j] += x[j];
        }
    }
  }
  if (n > 1) {
#pragma unroll
    for (int j = 0; j < N; ++j) part[warp][j * 32 + lane] = sum[j];
    __syncthreads();
    if (warp != 7) return;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      sum[j] = 0.f;
      for (int w = 0; w < 8; ++w) sum[j] += part[w][j * 32 + lane];
    }
  }
  if (warp == 7 && h < a.H) finish<G, N>(a, vec, id, h, sum);
}

// ---- the sort
constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32, kMaxBins = 512, kMaxBlocks = 64, kMaxPasses = 4;
constexpr int kSms = 148;
// Tokens that are sorted by comparing them all.  The rule looks at the tokens alone.  Whole
// gradients of 1,536 bf16 columns, by comparison and by the radix sort, in us: tables of 30,000
// rows (two digits) 17.6 and 18.1 for 513 tokens, 24.8 and 20.3 for 2,048, 32.5 and 34.4 for
// 6,144, 36.1 and 34.1 for 8,192; of 262,145 (three) 15.9 and 18.3, 22.7 and 21.3, 31.3 and
// 37.7, 38.2 and 44.0.  So it loses up to 4 us from 1,000 to 3,000 tokens and 2 us at 8,192 of
// tables up to 18 bits, and gains up to 6 us elsewhere.
constexpr int kCompared = 8192;

struct Plan {
  int N, V;
  int bits, passes, blocks, share;  // radix: bits of a digit; blocks of `share` tokens
  int P, pieces;                    // sums: pieces of P tokens
  int slabs;                        // of 256 columns
  long long row;                    // floats of a row of `part`
};
struct Work {  // in the workspace; pairs are (id, token), ids without a row are V
  uint2 *a, *b;
  unsigned* counts;  // [passes][blocks][bins]
  int* owners;       // [0]: how many; then the pieces where an id begins that goes on in the next one
  float* part;       // [pieces][2][row]: the sums of the id that came in, and of the one that goes on
  unsigned* named;   // a bit for each row of grad that an id names
};

__device__ __forceinline__ unsigned key_from(const TbEmbeddingGradArgs& a, long long id) {
  if (id >= a.V && a.err) *a.err = 1;
  return id < 0 || id >= a.V ? static_cast<unsigned>(a.V) : static_cast<unsigned>(id);
}
__device__ __forceinline__ unsigned key_of(const TbEmbeddingGradArgs& a, long long t) {
  return key_from(a, id_of(a.ids, a.ids64, t));
}

// A token's place is the number of tokens with smaller ids, and of earlier ones with the
// same.  A CTA places `own` tokens (N over the SMs); its threads share each one's
// comparisons, kSortThreads / own to a token.
__global__ void __launch_bounds__(kSortThreads) compare_sort_kernel(TbEmbeddingGradArgs a, Plan plan, Work work, int own) {
  extern __shared__ unsigned keys[];  // [N], padded to a multiple of 4 with keys above all; then [own] places
  constexpr int U = 8;
  tb::pdl_trigger();
  const int tid = threadIdx.x, N = plan.N, n4 = (N + 3) / 4;
  int* place = reinterpret_cast<int*>(keys + n4 * 4);
  for (int t0 = tid; t0 < n4 * 4; t0 += U * kSortThreads) {
    long long id[U];
#pragma unroll
    for (int u = 0; u < U; ++u) id[u] = t0 + u * kSortThreads < N ? id_of(a.ids, a.ids64, t0 + u * kSortThreads) : -1;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = t0 + u * kSortThreads;
      if (t < n4 * 4) keys[t] = t < N ? key_from(a, id[u]) : 0xffffffffu;
    }
  }
  for (int i = tid; i < own; i += kSortThreads) place[i] = 0;
  if (blockIdx.x == 0 && tid == 0) work.owners[0] = 0;
  __syncthreads();
  const int slices = kSortThreads / own, slice = tid / own, i = tid - slice * own, first = blockIdx.x * own;
  const int t = first + i;
  const bool on = slice < slices && t < N;
  const unsigned key = on ? keys[t] : 0;
  if (on) {
    const uint4* all = reinterpret_cast<const uint4*>(keys);
    // four keys at a time: equal ones count before the token and not behind it
    const int lo = static_cast<int>(static_cast<long long>(n4) * slice / slices), hi = static_cast<int>(static_cast<long long>(n4) * (slice + 1) / slices);
    const int mid = min(max(t / 4, lo), hi);
    int n = 0;
#pragma unroll 4
    for (int k = lo; k < mid; ++k) {
      const uint4 x = all[k];
      n += (x.x <= key) + (x.y <= key) + (x.z <= key) + (x.w <= key);
    }
    int k = mid;
    if (k < hi && k == t / 4) {
      const uint4 x = all[k];
      const int r = t & 3;
      n += (x.x < key || (x.x == key && r > 0)) + (x.y < key || (x.y == key && r > 1)) + (x.z < key || (x.z == key && r > 2)) +
           (x.w < key);
      ++k;
    }
#pragma unroll 4
    for (; k < hi; ++k) {
      const uint4 x = all[k];
      n += (x.x < key) + (x.y < key) + (x.z < key) + (x.w < key);
    }
    atomicAdd(&place[i], n);
  }
  __syncthreads();
  if (on && slice == 0) work.a[place[i]] = make_uint2(key, t);
}

// Counts of the first digit, a block of tokens per CTA.
__global__ void __launch_bounds__(kSortThreads) count_kernel(TbEmbeddingGradArgs a, Plan plan, Work work) {
  __shared__ unsigned hist[kMaxBins];
  const int bins = 1 << plan.bits, tid = threadIdx.x;
  tb::pdl_trigger();
  if (tid < bins) {
    hist[tid] = 0;
    for (int p = 1; p < plan.passes; ++p) work.counts[(p * plan.blocks + blockIdx.x) * bins + tid] = 0;
  }
  if (blockIdx.x == 0 && tid == 0) work.owners[0] = 0;
  __syncthreads();
  const long long lo = static_cast<long long>(blockIdx.x) * plan.share;
  const long long hi = min(static_cast<long long>(plan.N), lo + plan.share);
  for (long long t = lo + tid; t < hi; t += kSortThreads) atomicAdd(&hist[key_of(a, t) & (bins - 1)], 1u);
  __syncthreads();
  if (tid < bins) work.counts[blockIdx.x * bins + tid] = hist[tid];
}

// One digit: the pairs of a block to their places (stable), and the next digit counted
// for the blocks that they come to.
__global__ void __launch_bounds__(kSortThreads, 1) scatter_kernel(TbEmbeddingGradArgs a, Plan plan, Work work, int pass) {
  extern __shared__ unsigned hist[];  // [warps][bins]: counts, then places
  __shared__ unsigned scan[kMaxBins], warp_sum[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int bins = 1 << plan.bits, shift = pass * plan.bits;
  tb::pdl_trigger();
  for (int i = tid; i < kSortWarps * bins; i += kSortThreads) hist[i] = 0;
  __syncthreads();
  tb::pdl_wait();
  const uint2* in = (plan.passes - pass) % 2 ? work.b : work.a;  // the last pass writes a
  uint2* out = (plan.passes - pass) % 2 ? work.a : work.b;
  // a warp's pairs: consecutive, a multiple of 32 of them
  const long long end = min(static_cast<long long>(plan.N), (blockIdx.x + 1ll) * plan.share);
  const int per = (plan.share + kSortThreads - 1) / kSortThreads * 32;
  const long long lo = min(end, static_cast<long long>(blockIdx.x) * plan.share + warp * static_cast<long long>(per));
  const long long hi = min(end, lo + per);
  const auto pair_at = [&](long long i) {
    if (pass) return __ldcg(in + i);
    return make_uint2(key_of(a, i), static_cast<unsigned>(i));
  };
  // lanes with the same digit (a ballot for each bit)
  const auto peers_of = [&](unsigned d, bool on) {
    unsigned peers = __ballot_sync(0xffffffffu, on);
    for (int b = 0; b < plan.bits; ++b) {
      const unsigned x = __ballot_sync(0xffffffffu, d >> b & 1);
      peers &= d >> b & 1 ? x : ~x;
    }
    return peers;
  };
  unsigned* mine = hist + warp * bins;
  uint2 p = make_uint2(0, 0);
  if (lo + lane < hi) p = pair_at(lo + lane);
  // ---- the digit's counts in all blocks, and in the ones before (asked for beside the pairs)
  unsigned all = 0, before = 0;
  if (tid < bins) {
    const unsigned* counts = work.counts + pass * plan.blocks * bins + tid;
#pragma unroll 16
    for (int b = 0; b < plan.blocks; ++b) {
      const unsigned c = __ldcg(counts + b * bins);
      if (b < static_cast<int>(blockIdx.x)) before += c;
      all += c;
    }
  }
  unsigned peers = 0;
  for (long long i = lo + lane; i - lane < hi; i += 32) {
    const bool on = i < hi;
    if (on && i >= lo + 32) p = pair_at(i);
    const unsigned d = p.x >> shift & (bins - 1);
    peers = peers_of(d, on);
    if (on && lane == __ffs(peers) - 1) mine[d] += __popc(peers);
    __syncwarp();
  }
  // ---- the digit's places over all blocks
  unsigned incl = all;  // inclusive sum over the digits (threads past the last digit hold 0)
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned x = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += x;
  }
  if (lane == 31) warp_sum[warp] = incl;
  __syncthreads();
  if (warp == 0) {
    unsigned x = warp_sum[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    warp_sum[lane] = x;
  }
  __syncthreads();
  // ---- and over the warps of this one (two halves of the warps per digit)
  const int half = tid >> plan.bits, w0 = half * (kSortWarps / 2);
  const unsigned digit = tid & (bins - 1);
  unsigned c[kSortWarps / 2], sum = 0;
  if (half < 2) {
#pragma unroll
    for (int w = 0; w < kSortWarps / 2; ++w) c[w] = hist[(w0 + w) * bins + digit];
#pragma unroll
    for (int w = 0; w < kSortWarps / 2; ++w) sum += c[w];
    if (half == 0) scan[digit] = incl - all + (warp ? warp_sum[warp - 1] : 0) + before + sum;  // where the second half begins
  }
  __syncthreads();
  if (half < 2) {
    unsigned at = scan[digit] - (half == 0 ? sum : 0);
#pragma unroll
    for (int w = 0; w < kSortWarps / 2; ++w) {
      hist[(w0 + w) * bins + digit] = at;
      at += c[w];
    }
  }
  __syncthreads();
  // ---- to their places
  const bool once = per == 32;
  for (long long i = lo + lane; i - lane < hi; i += 32) {
    const bool on = i < hi;
    if (!once && on) p = pair_at(i);
    const unsigned d = p.x >> shift & (bins - 1);
    if (!once) peers = peers_of(d, on);
    const unsigned at = on ? mine[d] + __popc(peers & ((1u << lane) - 1)) : 0;
    __syncwarp();
    if (on) {
      if (lane == __ffs(peers) - 1) mine[d] += __popc(peers);
      __stcg(out + at, p);
      if (pass + 1 < plan.passes)
        atomicAdd(&work.counts[((pass + 1) * plan.blocks + at / plan.share) * bins + (p.x >> (shift + plan.bits) & (bins - 1))], 1u);
    }
    __syncwarp();
  }
}

// ---- a dense gradient's zeros: by CTAs beside those of the sums, which write the rows that
// an id names; these write the runs of others, a warp `unit` rows at a time.  The rows' bits
// were set before the sort began, so nothing is waited for: the stores go on beside the sort,
// too.  (8,192 tokens of 151,936 rows of 1,536 bf16, 467 MB: 94 us, 5.0 TB/s, and 193 with
// zeros in all rows before the sums; 16,384 of 128,256 rows of 4,096: 205 and 252.)
__global__ void __launch_bounds__(256) mark_kernel(TbEmbeddingGradArgs a, unsigned* named) {
  const long long t = blockIdx.x * 256ll + threadIdx.x;
  if (t >= a.N) return;
  const long long id = id_of(a.ids, a.ids64, t);
  if (id < 0 || id >= a.V) return;
  const unsigned bit = 1u << (id & 31);
  if (!(__ldcg(named + (id >> 5)) & bit)) atomicOr(named + (id >> 5), bit);  // (a token may fill the batch)
}
constexpr int kFillers = 4 * 148;  // CTAs (with 3 x 148 the same tokens take 99 us, with 8 x 148 90)
// Rows of a task (a power of two): 8, so that even a small table has one for every warp (1,024
// tokens of 32,000 rows of 1,024: 24.6 us, and 36.8 with 32); short rows 32.
__device__ __forceinline__ int unit_of(long long row) { return row < 1024 ? 32 : 8; }
template <typename G>
__device__ __forceinline__ void fill_others(G* grad, int H, int V, const unsigned* named) {
  const int lane = threadIdx.x & 31, unit = unit_of(H * static_cast<long long>(sizeof(G))), tasks = (V - 1) / unit + 1;
  for (int task = blockIdx.x * 8 + threadIdx.x / 32; task < tasks; task += kFillers * 8) {
    const long long v = static_cast<long long>(task) * unit;
    const int rows = static_cast<int>(min(static_cast<long long>(unit), V - v));
    unsigned left = ~__ldcg(named + (v >> 5)) >> (v & 31);
    if (rows < 32) left &= (1u << rows) - 1;
    while (left) {
      const int first = __ffs(left) - 1, end = __ffs(~(left >> first)), n = end ? end - 1 : 32;
      G* p = grad + (v + first) * H;
      const long long count = static_cast<long long>(n) * H;
      const int head = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / static_cast<int>(sizeof(G));
      const long long vecs = count > head ? (count - head) * sizeof(G) / 16 : 0, tail = head + vecs * (16 / sizeof(G));
      if (lane < head && lane < count) p[lane] = tb::from_f32<G>(0.f);
      uint4* q = reinterpret_cast<uint4*>(p + head);
#pragma unroll 4
      for (long long i = lane; i < vecs; i += 32) __stcs(q + i, make_uint4(0, 0, 0, 0));
      if (tail + lane < count) p[tail + lane] = tb::from_f32<G>(0.f);
      left = first + n < 32 ? left >> (first + n) << (first + n) : 0u;
    }
  }
}

// ---- the sums.  A lane has eight columns of a slab, as M vectors of N.
template <typename T, typename G, int N>
struct Tile {
  static constexpr int M = 8 / N, kNext = 32 * N;  // columns between a lane's vectors
  int h;     // the lane's first column
  int n;     // its vectors
  bool all;  // every lane has M
  __device__ __forceinline__ Tile(const TbEmbeddingGradArgs& a, int slab) {
    const int lane = threadIdx.x & 31, count = min(a.H / N - slab * (256 / N), 256 / N);
    h = (slab * (256 / N) + lane) * N;
    n = min(M, max(0, count - lane + 31) / 32);
    all = count == 256 / N;
  }
  template <typename F>
  __device__ __forceinline__ void each(F f) const {  // f(vector, its first column)
    if (all) {
#pragma unroll
      for (int m = 0; m < M; ++m) f(m, h + m * kNext);
    } else {
#pragma unroll
      for (int m = 0; m < M; ++m)
        if (m < n) f(m, h + m * kNext);
    }
  }
  __device__ __forceinline__ void finish_row(const TbEmbeddingGradArgs& a, bool vec, long long id, const float (&sum)[M][N]) const {
    each([&](int m, int column) { finish<G, N>(a, vec, id, column, sum[m]); });
  }
  __device__ __forceinline__ void leave(float* row, const float (&sum)[M][N]) const {
    each([&](int m, int column) { tb::store_vec<float, N>(row + column, sum[m]); });
  }
  __device__ __forceinline__ static void zero(float (&sum)[M][N]) {
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int j = 0; j < N; ++j) sum[m][j] = 0.f;
  }
  __device__ __forceinline__ static void put(float* s, const float (&sum)[M][N]) {  // 256 floats of shared memory
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int j = 0; j < N; ++j) s[(m * N + j) * 32 + (threadIdx.x & 31)] = sum[m][j];
  }
  __device__ __forceinline__ static void add(const float* s, float (&sum)[M][N]) {
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int j = 0; j < N; ++j) sum[m][j] += s[(m * N + j) * 32 + (threadIdx.x & 31)];
  }
};

constexpr int kWarps = 8;

template <typename T, typename G, int N>
__global__ void __launch_bounds__(kWarps * 32, 3) pieces_kernel(TbEmbeddingGradArgs a, Plan plan, Work work, bool vec, int fillers) {
  using Sum = Tile<T, G, N>;
  constexpr int M = Sum::M, U = N * sizeof(T) == 16 ? 8 / M : 4;
  __shared__ float in[kWarps][256], on[kWarps][256];  // sums of the ids that came in, that go on
  __shared__ bool through[kWarps];                    // the id that came in goes on
  tb::pdl_trigger();
  if (static_cast<int>(blockIdx.x) < fillers) {
    fill_others(static_cast<G*>(a.grad), a.H, plan.V, work.named);
    return;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = (blockIdx.x - fillers) / plan.slabs, slab = (blockIdx.x - fillers) % plan.slabs;
  const Sum tile(a, slab);
  const unsigned V = plan.V;
  const T* dy = static_cast<const T*>(a.dy);
  float* part = work.part + static_cast<long long>(c) * 2 * plan.row;
  const uint2* pairs = work.a;
  const int lo = min(static_cast<long long>(plan.N), static_cast<long long>(c) * plan.P + warp * (plan.P / kWarps));
  const int hi = min(static_cast<long long>(plan.N), static_cast<long long>(c) * plan.P + (warp + 1) * (plan.P / kWarps));
  float sum[M][N];
  Sum::zero(sum);
  bool came = false, goes = false, ends = false;  // ends: what came in has its end here
  unsigned id = V;
  tb::pdl_wait();
  if (lo < hi) {
    const unsigned prev = lo > 0 ? __ldcg(pairs + lo - 1).x : V, next = hi < plan.N ? __ldcg(pairs + hi).x : V;
    uint2 mine = lo + lane < hi ? __ldcg(pairs + lo + lane) : make_uint2(V, 0);
    id = __shfl_sync(0xffffffffu, mine.x, 0);
    came = id < V && prev == id;
    bool first = came;  // the sum is of what came in
    for (int i0 = lo; i0 < hi && id < V; i0 += 32) {
      if (i0 != lo) mine = i0 + lane < hi ? __ldcg(pairs + i0 + lane) : make_uint2(V, 0);
      const int n = min(32, hi - i0);
      for (int u0 = 0; u0 < n; u0 += U) {
        unsigned key[U];
        tb::Packed<T, N> x[U][M];
#pragma unroll
        for (int u = 0; u < U; ++u) {  // (u0 + u < 32: U divides 32; lanes behind the end hold V)
          key[u] = __shfl_sync(0xffffffffu, mine.x, u0 + u);
          const T* row = dy + static_cast<long long>(__shfl_sync(0xffffffffu, mine.y, u0 + u)) * a.ld_dy;
          if (key[u] < V) tile.each([&](int m, int column) { x[u][m].load(row + column); });
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (u0 + u >= n) break;
          if (key[u] != id) {
            if (id < V) {
              if (first) {
                Sum::put(in[warp], sum);
                ends = true;
              } else {
                tile.finish_row(a, vec, id, sum);
              }
            }
            first = false;
            id = key[u];
            Sum::zero(sum);
          }
          if (id < V) {
#pragma unroll
            for (int m = 0; m < M; ++m) {
              float f[N];
              x[u][m].unpack(f);
#pragma unroll
              for (int j = 0; j < N; ++j) sum[m][j] += f[j];
            }
          }
        }
      }
    }
    goes = id < V && next == id;
    if (first) {
      Sum::put(in[warp], sum);
      ends = !goes;
    } else if (goes) {
      Sum::put(on[warp], sum);
    } else if (id < V) {
      tile.finish_row(a, vec, id, sum);
    }
  }
  if (lane == 0) through[warp] = came && !ends;
  __syncthreads();
  // ---- what goes on within the piece
  if (warp == 0 && came) {  // and what came into it
    Sum::zero(sum);
    for (int w = 0;; ++w) {
      Sum::add(in[w], sum);
      if (!through[w] || w + 1 == kWarps) break;
    }
    tile.leave(part, sum);
  }
  if (goes && !(came && !ends)) {
    Sum::zero(sum);
    Sum::add(on[warp], sum);
    for (int w = warp + 1;; ++w) {
      if (w == kWarps) {  // into the next piece
        tile.leave(part + plan.row, sum);
        if (slab == 0 && lane == 0) work.owners[1 + atomicAdd(&work.owners[0], 1)] = c;
        break;
      }
      Sum::add(in[w], sum);
      if (!through[w]) {
        tile.finish_row(a, vec, id, sum);
        break;
      }
    }
  }
}

// ---- ids over several pieces: a warp takes a slab of one; over many pieces the CTA's warps
// share them (the order of the additions follows from the number of pieces alone)
constexpr int kShared = 32;
template <typename G, int N>
__global__ void __launch_bounds__(kWarps * 32) join_kernel(TbEmbeddingGradArgs a, Plan plan, Work work, bool vec) {
  using Sum = Tile<float, G, N>;
  constexpr int M = Sum::M, U = 4;
  __shared__ float buf[kWarps][256];
  __shared__ int count[kWarps], begin[kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  tb::pdl_wait();
  const int owners = __ldcg(work.owners);
  const long long tasks = static_cast<long long>(owners) * plan.slabs;
  const auto sum_of = [&](const Sum& tile, long long first, int n, float (&sum)[M][N]) {
    for (int i = 0; i < n; i += U) {
      float x[U][M][N];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i + u < n) tile.each([&](int m, int column) { tb::load_vec<float, N>(work.part + (first + i + u) * 2 * plan.row + column, x[u][m]); });
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i + u < n) {
#pragma unroll
          for (int m = 0; m < M; ++m)
#pragma unroll
            for (int j = 0; j < N; ++j) sum[m][j] += x[u][m][j];
        }
    }
  };
  const auto first_of = [&](const Sum& tile, long long c, float (&sum)[M][N]) {
    tile.each([&](int m, int column) { tb::load_vec<float, N>(work.part + (c * 2 + 1) * plan.row + column, sum[m]); });
  };
  for (long long base = blockIdx.x * static_cast<long long>(kWarps); base < tasks; base += gridDim.x * static_cast<long long>(kWarps)) {
    const long long task = base + warp;
    if (task < tasks) {
      const int c = __ldcg(work.owners + 1 + task % owners);  // (slabs of one id in different CTAs)
      const unsigned id = __ldcg(work.a + (c + 1ll) * plan.P).x;
      int n = 0;  // pieces that the id comes into
      for (;;) {
        const long long p = c + 1ll + n + lane;
        const int k = __popc(__ballot_sync(0xffffffffu, p < plan.pieces && __ldcg(work.a + min(p, plan.pieces - 1ll) * plan.P).x == id));
        n += k;
        if (k < 32) break;
      }
      if (lane == 0) {
        count[warp] = n;
        begin[warp] = c;
      }
      if (n <= kShared) {
        const Sum tile(a, static_cast<int>(task / owners));
        float sum[M][N];
        Sum::zero(sum);
        first_of(tile, c, sum);
        sum_of(tile, c + 1ll, n, sum);
        tile.finish_row(a, vec, id, sum);
      }
    } else if (lane == 0) {
      count[warp] = 0;
    }
    __syncthreads();
    for (int w = 0; w < kWarps; ++w) {
      const int n = count[w];
      if (n <= kShared) continue;
      const Sum tile(a, static_cast<int>((base + w) / owners));
      const int c = begin[w], lo = static_cast<int>(static_cast<long long>(n) * warp / kWarps);
      const int hi = static_cast<int>(static_cast<long long>(n) * (warp + 1) / kWarps);
      float sum[M][N];
      Sum::zero(sum);
      if (warp == 0) first_of(tile, c, sum);
      sum_of(tile, c + 1ll + lo, hi - lo, sum);
      Sum::put(buf[warp], sum);
      __syncthreads();
      if (warp == 0) {
        for (int v = 1; v < kWarps; ++v) Sum::add(buf[v], sum);
        tile.finish_row(a, vec, __ldcg(work.a + (c + 1ll) * plan.P).x, sum);
      }
      __syncthreads();
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------ host
bool aligned(const void* p, long long stride_bytes, long long to) {
  return (reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>(stride_bytes)) % to == 0;
}

unsigned grid_of(long long ctas) { return static_cast<unsigned>(ctas < (1 << 24) ? ctas : 1 << 24); }

template <typename T, int N>
cudaError_t lookup_narrow(const TbEmbeddingArgs& a, cudaStream_t s) {
  lookup_narrow_kernel<T, N><<<grid_of((static_cast<long long>(a.N) * (a.H / N) + 255) / 256), 256, 0, s>>>(a);
  return cudaGetLastError();
}

template <typename T>
cudaError_t lookup_of(const TbEmbeddingArgs& a, cudaStream_t s) {
  constexpr int e = sizeof(T), E = 16 / e;
  const auto fits = [&](int b) { return a.H * e % b == 0 && aligned(a.weight, a.ld_w * e, b) && aligned(a.out, a.ld_out * e, b); };
  const bool whole = fits(16);
  if (a.H < 32 * E) {
    if (whole) return lookup_narrow<T, E>(a, s);
    if (fits(8)) return lookup_narrow<T, E / 2>(a, s);
    if constexpr (e == 2) {
      if (fits(4)) return lookup_narrow<T, 2>(a, s);
    }
    return lookup_narrow<T, 1>(a, s);
  }
  if (whole) {
    const int segs = (a.H / E + 32 * kUnroll - 1) / (32 * kUnroll);
    lookup_wide_kernel<T><<<grid_of((static_cast<long long>(a.N) * segs + 7) / 8), 256, 0, s>>>(a, segs);
  } else {
    lookup_shift_kernel<T><<<grid_of((static_cast<long long>(a.N) + 7) / 8), 256, 0, s>>>(a);
  }
  return cudaGetLastError();
}

size_t up16(size_t b) { return (b + 15) / 16 * 16; }

Plan plan_of(int N, int H, int V) {
  Plan p{};
  p.N = N;
  p.V = V;
  int bits = 1;
  while (bits < 31 && (V >> bits) != 0) ++bits;  // keys 0 .. V
  p.passes = (bits + 8) / 9;
  p.bits = (bits + p.passes - 1) / p.passes;
  // radix: a token per thread, up to the blocks whose counts a block adds up by itself
  p.blocks = (N + kSortThreads - 1) / kSortThreads;
  if (p.blocks > kMaxBlocks) p.blocks = kMaxBlocks;
  p.share = ((N + p.blocks - 1) / p.blocks + 31) / 32 * 32;
  // pieces of 128 tokens, at most 8,192 of them (and of the workspace's rows)
  p.P = 128;
  while ((N + p.P - 1) / p.P > 8192) p.P *= 2;
  p.pieces = (N + p.P - 1) / p.P;
  p.slabs = (H + 255) / 256;
  p.row = (H + 3) / 4 * 4;
  return p;
}

size_t work_of(const Plan& p, char* w, Work* out) {
  size_t at = 0;
  const auto take = [&](size_t bytes) {
    char* q = w + at;
    at += up16(bytes);
    return q;
  };
  Work k;
  k.a = reinterpret_cast<uint2*>(take(p.N * sizeof(uint2)));
  k.b = reinterpret_cast<uint2*>(take(p.N * sizeof(uint2)));
  k.counts = reinterpret_cast<unsigned*>(take(static_cast<size_t>(kMaxPasses) * kMaxBlocks * kMaxBins * sizeof(unsigned)));
  k.owners = reinterpret_cast<int*>(take((p.pieces + 1) * sizeof(int)));
  k.part = reinterpret_cast<float*>(take(static_cast<size_t>(p.pieces) * 2 * p.row * sizeof(float)));
  k.named = reinterpret_cast<unsigned*>(take((static_cast<size_t>(p.V) + 31) / 32 * sizeof(unsigned)));
  if (out) *out = k;
  return at;
}

// `after`: may start before the kernel ahead of it has ended.  The first kernel of a gradient
// (the sort's first, and the marks) is launched without it and has to stay so: the kernels here
// let the next one start before they wait themselves, and the CTAs that write zeros never wait.
// What keeps them behind the caller's earlier work (and the marks, and the workspace's last user)
// is that the first kernel does not begin before all of it has ended.
template <typename... P, typename... Args>
cudaError_t launch(void (*kernel)(P...), unsigned grid, unsigned block, size_t smem, cudaStream_t s, bool after, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = after ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Zeros in all rows of grad.
template <typename G>
cudaError_t fill(const TbEmbeddingGradArgs& a, cudaStream_t s) {
  const size_t row = a.H * sizeof(G);
  if (a.ld_grad == a.H || a.V == 1) return cudaMemsetAsync(a.grad, 0, row * a.V, s);
  return cudaMemset2DAsync(a.grad, a.ld_grad * sizeof(G), 0, row, a.V, s);
}
// Zeros beside the sums (rows without gaps): the rows' bits cost two launches, which pay from
// some 32 MB on (4,096 tokens of 33.6 MB: 25 us beside, and 32 before; 600 of 4.2 MB: 16.5 and 12).
constexpr size_t kBeside = 32 << 20;

template <typename T, typename G, int N>
cudaError_t grad(const TbEmbeddingGradArgs& a, cudaStream_t s) {
  const bool vec = aligned(a.grad, a.ld_grad * sizeof(G), N * sizeof(G) < 16 ? N * sizeof(G) : 16);
  const bool few = a.N <= kFew, beside = a.zero && !few && a.ld_grad == a.H && a.H * sizeof(G) * a.V >= kBeside;
  cudaError_t e = cudaSuccess;
  if (a.zero && !beside) e = fill<G>(a, s);
  if (e != cudaSuccess || a.N == 0) return e;
  if (few) {
    const int slabs = (a.H + 32 * N - 1) / (32 * N);
    grad_few_kernel<T, G, N><<<static_cast<unsigned>(a.N) * slabs, 256, 0, s>>>(a, slabs, vec);
    return cudaGetLastError();
  }
  const Plan plan = plan_of(a.N, a.H, a.V);
  const int fillers = beside ? kFillers : 0;
  Work work;
  work_of(plan, static_cast<char*>(a.ws), &work);
  if (beside) {
    e = cudaMemsetAsync(work.named, 0, (static_cast<size_t>(a.V) + 31) / 32 * sizeof(unsigned), s);
    if (e == cudaSuccess) e = launch(mark_kernel, (a.N + 255) / 256, 256u, 0, s, false, a, work.named);
    if (e != cudaSuccess) return e;
  }
  if (a.N <= kCompared) {
    const int own = (a.N + kSms - 1) / kSms;
    e = launch(compare_sort_kernel, (a.N + own - 1) / own, kSortThreads, (a.N + 3) / 4 * 16 + own * 4, s, false, a, plan, work, own);
  } else {
    e = tb::ensure_dyn_smem(reinterpret_cast<const void*>(&scatter_kernel), kSortWarps * kMaxBins * 4);
    if (e == cudaSuccess) e = launch(count_kernel, plan.blocks, kSortThreads, 0, s, false, a, plan, work);
    for (int p = 0; p < plan.passes && e == cudaSuccess; ++p)
      e = launch(scatter_kernel, plan.blocks, kSortThreads, (kSortWarps << plan.bits) * sizeof(unsigned), s, true, a, plan, work, p);
  }
  if (e != cudaSuccess) return e;
  e = launch(pieces_kernel<T, G, N>, static_cast<unsigned>(plan.pieces) * plan.slabs + fillers, kWarps * 32, 0, s, true, a, plan, work, vec,
             fillers);
  if (e != cudaSuccess) return e;
  const long long tasks = static_cast<long long>(plan.pieces) * plan.slabs;
  const long long ctas = (tasks + kWarps - 1) / kWarps;
  return launch(join_kernel<G, N>, static_cast<unsigned>(ctas < 592 ? ctas : 592), kWarps * 32, 0, s, true, a, plan, work, vec);
}

template <typename T, typename G>
cudaError_t grad_vec(const TbEmbeddingGradArgs& a, cudaStream_t s) {
  constexpr long long e = sizeof(T);
  const auto fits = [&](long long b) { return a.H * e % b == 0 && aligned(a.dy, a.ld_dy * e, b); };
  if (fits(16)) return grad<T, G, 16 / e>(a, s);
  if constexpr (e == 2) {
    if (fits(4)) return grad<T, G, 2>(a, s);
  }
  return grad<T, G, 1>(a, s);
}

template <typename T>
cudaError_t grad_of(const TbEmbeddingGradArgs& a, cudaStream_t s) {
  switch (a.grad_dtype) {
    case TB_BF16: return grad_vec<T, __nv_bfloat16>(a, s);
    case TB_F16: return grad_vec<T, __half>(a, s);
    case TB_F32: return grad_vec<T, float>(a, s);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace

extern "C" int tb_embedding(const TbEmbeddingArgs* args, cudaStream_t s) {
  const TbEmbeddingArgs& a = *args;
  if (a.N < 0 || a.H < 1 || a.V < 1) return static_cast<int>(cudaErrorInvalidValue);
  if (a.N == 0) return 0;
  switch (a.dtype) {
    case TB_BF16: return static_cast<int>(lookup_of<__nv_bfloat16>(a, s));
    case TB_F16: return static_cast<int>(lookup_of<__half>(a, s));
    case TB_F32: return static_cast<int>(lookup_of<float>(a, s));
    default: return static_cast<int>(cudaErrorInvalidValue);
  }
}

extern "C" size_t tb_embedding_grad_ws_bytes(int N, int H, int V) {
  if (N <= kFew) return 0;
  return work_of(plan_of(N, H, V), nullptr, nullptr);
}

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
