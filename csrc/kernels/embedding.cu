// Embedding lookup with a scale, and its gradient:
//
//   y_t = s W[id_t],      dW[v] (+)= s sum_{t: id_t = v} dy_t.
//
// Both move bytes (one product and one addition per value).  The gradient's sums are
// fp32 in a fixed order, so the same inputs give the same bits:
//
// * Few tokens: one CTA for each token and slab of columns.  The first token of an id
//   finds the others by comparing all ids and sums their rows; one launch, no workspace.
// * More: the tokens are sorted by id (stable, so by token within an id), then threads
//   sum pieces of a fixed number of sorted tokens, a vector of columns each.  An id whose
//   tokens lie within a piece is finished there; what an id has in the pieces that it
//   shares with other pieces is left in a workspace, and a last launch adds those up.  A
//   token that fills a third of the batch is thus as well spread as any other.
//
// The sort is a radix sort of one thread-block cluster (digits of up to 9 bits, counts
// per warp in shared memory, totals exchanged over distributed shared memory), because
// one launch with cluster barriers is shorter than the six launches of a sort over the
// whole machine; a dense gradient's zeros are written by the other clusters meanwhile.
#include <cooperative_groups.h>
#include <limits.h>
#include <math.h>

#include "device_common.cuh"
#include "kernels.h"
#include "pdl.cuh"
#include "vec_io.cuh"

namespace {

namespace cg = cooperative_groups;

__device__ __forceinline__ long long id_of(const void* ids, int ids64, long long t) {
  return ids64 ? static_cast<const long long*>(ids)[t] : static_cast<const int*>(ids)[t];
}

// ------------------------------------------------------------------ lookup
constexpr int kUnroll = 4;

template <typename T, int N>
__device__ __forceinline__ void scaled_row(const TbEmbeddingArgs& a, long long id, float (&x)[N]) {
  if (id >= 0 && id < a.V) {
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] *= a.scale;
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = id < 0 ? 0.f : NAN;
  }
}

// A warp takes 32 x kUnroll vectors of N elements of a row (rows of 32 vectors and more).
template <typename T, int N>
__global__ void __launch_bounds__(256) lookup_wide_kernel(TbEmbeddingArgs a, int segs) {
  const int lane = threadIdx.x & 31, per = a.H / N;
  const long long tasks = static_cast<long long>(a.N) * segs;
  for (long long task = blockIdx.x * 8ll + threadIdx.x / 32; task < tasks; task += gridDim.x * 8ll) {
    const long long t = segs == 1 ? task : task / segs;
    const int first = static_cast<int>(task - t * segs) * 32 * kUnroll + lane;
    const long long id = id_of(a.ids, a.ids64, t);
    const bool good = id >= 0 && id < a.V;
    if (id >= a.V && a.err && lane == 0) *a.err = 1;
    const T* src = static_cast<const T*>(a.weight) + (good ? id : 0) * a.ld_w;
    T* dst = static_cast<T*>(a.out) + t * a.ld_out;
    tb::Packed<T, N> p[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (first + u * 32 < per && good) p[u].load(src + (first + u * 32) * N);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (first + u * 32 < per) {
        float x[N];
        p[u].unpack(x);
        scaled_row<T, N>(a, id, x);
        tb::store_vec<T, N>(dst + (first + u * 32) * N, x);
      }
  }
}

// A thread for every vector (shorter rows).
template <typename T, int N>
__global__ void __launch_bounds__(256) lookup_narrow_kernel(TbEmbeddingArgs a) {
  const int per = a.H / N;
  const long long total = static_cast<long long>(a.N) * per;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    const long long t = total <= UINT_MAX ? static_cast<unsigned>(i) / static_cast<unsigned>(per) : i / per;
    const int h = static_cast<int>(i - t * per) * N;
    const long long id = id_of(a.ids, a.ids64, t);
    if (id >= a.V && a.err) *a.err = 1;
    float x[N];
    if (id >= 0 && id < a.V) tb::load_vec<T, N>(static_cast<const T*>(a.weight) + id * a.ld_w + h, x);
    scaled_row<T, N>(a, id, x);
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

constexpr int kFew = 512;  // tokens of the one-launch form

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
constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32, kMaxBins = 512;

struct SortPlan {
  int N, V, bits, passes, L, pieces;  // L: tokens of a piece
};
struct SortWork {  // in the workspace; pairs are (id, token)
  uint2 *a, *b;
  int* owners;  // [0]: how many; then the pieces where an id begins that goes on in the next one
  float* part;  // [pieces][2][H]: the sums of the id that came in, and of the one that goes on
};

__device__ __forceinline__ uint2 ld_pair(const uint2* p) { return __ldcg(p); }

// 16-byte stores of zeros over rows of `bytes` bytes, `stride` apart.
__device__ void fill_zero(char* base, long long rows, long long bytes, long long stride, long long thread, long long threads) {
  if (bytes == stride) {
    bytes *= rows;
    rows = 1;
  }
  if (rows == 1) {
    const long long head = min(bytes, static_cast<long long>((16 - (reinterpret_cast<uintptr_t>(base) & 15)) & 15));
    const long long body = (bytes - head) / 16;
    uint4* p = reinterpret_cast<uint4*>(base + head);
    const uint4 z = make_uint4(0, 0, 0, 0);
    long long i = thread;
    for (; i + 3 * threads < body; i += 4 * threads) {
#pragma unroll
      for (int u = 0; u < 4; ++u) p[i + u * threads] = z;
    }
    for (; i < body; i += threads) p[i] = z;
    const long long tail = bytes - head - body * 16;
    if (thread < head) base[thread] = 0;
    if (thread < tail) base[head + body * 16 + thread] = 0;
    return;
  }
  for (long long i = thread; i < rows * (bytes / 2); i += threads)  // (rows with gaps; elements of 2 or 4 bytes)
    reinterpret_cast<uint16_t*>(base + i / (bytes / 2) * stride)[i % (bytes / 2)] = 0;
}

// Cluster 0 sorts; the others (a dense gradient) write the zeros.
__global__ void __launch_bounds__(kSortThreads, 1) sort_kernel(TbEmbeddingGradArgs a, SortPlan plan, SortWork work, int elem) {
  extern __shared__ unsigned hist[];  // [warps][bins], then offsets
  __shared__ unsigned total[kMaxBins], scan[kMaxBins];
  __shared__ unsigned warp_sum[32];
  cg::cluster_group cl = cg::this_cluster();
  const int rank = cl.block_rank(), ranks = cl.num_blocks();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  tb::pdl_trigger();
  if (blockIdx.x >= static_cast<unsigned>(ranks)) {
    fill_zero(static_cast<char*>(a.grad), a.V, static_cast<long long>(a.H) * elem, a.ld_grad * elem,
              (blockIdx.x - ranks) * static_cast<long long>(kSortThreads) + tid,
              (gridDim.x - ranks) * static_cast<long long>(kSortThreads));
    return;
  }
  const int N = plan.N, bins = 1 << plan.bits;
  // a warp's tokens: consecutive, a multiple of 32 of them
  const int per = (N + ranks * kSortThreads - 1) / (ranks * kSortThreads) * 32;
  const int lo = min(N, (rank * kSortWarps + warp) * per), hi = min(N, lo + per);
  if (rank == 0 && tid == 0) work.owners[0] = 0;
  uint2* in = nullptr;
  for (int pass = 0; pass < plan.passes; ++pass) {
    uint2* out = (plan.passes - pass) % 2 ? work.a : work.b;  // the last pass writes a
    const int shift = pass * plan.bits;
    const auto pair_at = [&](int i) {
      if (pass) return ld_pair(in + i);
      const long long id = id_of(a.ids, a.ids64, i);
      if (id >= a.V && a.err) *a.err = 1;
      return make_uint2(id < 0 || id >= a.V ? plan.V : static_cast<unsigned>(id), i);
    };
    for (int i = tid; i < kSortWarps * bins; i += kSortThreads) hist[i] = 0;
    __syncthreads();
    unsigned* mine = hist + warp * bins;
    // ---- counts of each warp
    for (int i0 = lo; i0 < hi; i0 += 128) {
      unsigned key[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) key[u] = i0 + u * 32 + lane < hi ? pair_at(i0 + u * 32 + lane).x : 0;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const bool on = i0 + u * 32 + lane < hi;
        const unsigned d = on ? key[u] >> shift & (bins - 1) : 0xffffffffu;
        const unsigned peers = __match_any_sync(0xffffffffu, d);
        if (on && lane == __ffs(peers) - 1) mine[d] += __popc(peers);
        __syncwarp();
      }
    }
    __syncthreads();
    // ---- where each warp's tokens of a digit go
    if (tid < bins) {
      unsigned s = 0;
      for (int w = 0; w < kSortWarps; ++w) {
        const unsigned c = hist[w * bins + tid];
        hist[w * bins + tid] = s;
        s += c;
      }
      total[tid] = s;
    }
    cl.sync();
    unsigned all = 0, before = 0;
    if (tid < bins)
      for (int r = 0; r < ranks; ++r) {
        const unsigned c = *cl.map_shared_rank(&total[tid], r);
        if (r < rank) before += c;
        all += c;
      }
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
    if (tid < bins) scan[tid] = incl - all + (warp ? warp_sum[warp - 1] : 0) + before;
    __syncthreads();
    for (int i = tid; i < kSortWarps * bins; i += kSortThreads) hist[i] += scan[i & (bins - 1)];
    __syncthreads();
    // ---- to their places
    for (int i0 = lo; i0 < hi; i0 += 128) {
      uint2 p[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) p[u] = i0 + u * 32 + lane < hi ? pair_at(i0 + u * 32 + lane) : make_uint2(0, 0);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const bool on = i0 + u * 32 + lane < hi;
        const unsigned d = on ? p[u].x >> shift & (bins - 1) : 0xffffffffu;
        const unsigned peers = __match_any_sync(0xffffffffu, d);
        const unsigned at = on ? mine[d] + __popc(peers & ((1u << lane) - 1)) : 0;
        __syncwarp();
        if (on) {
          if (lane == __ffs(peers) - 1) mine[d] += __popc(peers);
          __stcg(out + at, p[u]);
        }
        __syncwarp();
      }
    }
    cl.sync();
    in = out;
  }
  // ---- pieces where an id begins that the next piece goes on with
  for (int c = rank * kSortThreads + tid; c + 1 < plan.pieces; c += ranks * kSortThreads) {
    const int e = (c + 1) * plan.L;
    const unsigned id = ld_pair(in + e).x;
    if (id < static_cast<unsigned>(plan.V) && ld_pair(in + e - 1).x == id &&
        (c == 0 || ld_pair(in + c * plan.L - 1).x != id))
      work.owners[1 + atomicAdd(&work.owners[0], 1)] = c;
  }
}

// ---- sums of pieces: a thread takes N columns of a piece
template <typename T, typename G, int N>
__global__ void __launch_bounds__(256) pieces_kernel(TbEmbeddingGradArgs a, SortPlan plan, SortWork work, bool vec) {
  constexpr int U = 8;
  const int per = a.H / N;
  const unsigned V = plan.V;
  tb::pdl_trigger();
  tb::pdl_wait();
  const long long i = blockIdx.x * 256ll + threadIdx.x;
  const long long c = static_cast<long long>(plan.pieces) * per <= UINT_MAX ? static_cast<unsigned>(i) / static_cast<unsigned>(per) : i / per;
  if (c >= plan.pieces) return;
  const int h = static_cast<int>(i - c * per) * N;
  const uint2* pairs = work.a;
  const int lo = static_cast<int>(c) * plan.L, hi = min(plan.N, lo + plan.L);
  unsigned id = ld_pair(pairs + lo).x;
  if (id >= V) return;
  bool came = lo > 0 && ld_pair(pairs + lo - 1).x == id;  // the id began in an earlier piece
  float* part = work.part + c * 2 * a.H + h;
  const T* dy = static_cast<const T*>(a.dy) + h;
  float sum[N];
#pragma unroll
  for (int j = 0; j < N; ++j) sum[j] = 0.f;
  const auto leave = [&](int which) {
    float* p = part + static_cast<long long>(which) * a.H;
#pragma unroll
    for (int j = 0; j < N; ++j) p[j] = sum[j];
  };
  for (int i0 = lo; i0 < hi && id < V; i0 += U) {
    uint2 p[U];
    tb::Packed<T, N> x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) p[u] = i0 + u < hi ? ld_pair(pairs + i0 + u) : make_uint2(V, 0);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (p[u].x < V) x[u].load(dy + static_cast<long long>(p[u].y) * a.ld_dy);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i0 + u >= hi) break;
      if (p[u].x != id) {
        if (id < V) {
          if (came) {
            leave(0);
          } else {
            finish<G, N>(a, vec, id, h, sum);
          }
        }
        came = false;
        id = p[u].x;
#pragma unroll
        for (int j = 0; j < N; ++j) sum[j] = 0.f;
      }
      if (id < V) {
        float f[N];
        x[u].unpack(f);
#pragma unroll
        for (int j = 0; j < N; ++j) sum[j] += f[j];
      }
    }
  }
  if (id >= V) return;
  if (came) {
    leave(0);
  } else if (hi < plan.N && ld_pair(pairs + hi).x == id) {
    leave(1);
  } else {
    finish<G, N>(a, vec, id, h, sum);
  }
}

// ---- ids over several pieces: a CTA takes 32 vectors of columns of one; its warps share
// the pieces, the first one's sum comes first
constexpr int kJoinWarps = 16;
template <typename G, int N>
__global__ void __launch_bounds__(kJoinWarps * 32) join_kernel(TbEmbeddingGradArgs a, SortPlan plan, SortWork work, int slabs, bool vec) {
  constexpr int U = 8;
  __shared__ float buf[kJoinWarps][32 * N];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  tb::pdl_wait();
  const long long tasks = static_cast<long long>(work.owners[0]) * slabs;
  for (long long task = blockIdx.x; task < tasks; task += gridDim.x) {
    const int c = work.owners[1 + task / slabs];
    const int h = static_cast<int>(task % slabs) * 32 * N + lane * N;
    const unsigned id = ld_pair(work.a + (c + 1ll) * plan.L).x;
    int n = 0;  // pieces that the id comes into
    for (;;) {
      const long long p = c + 1ll + n + threadIdx.x;
      const int on = __syncthreads_count(p < plan.pieces && ld_pair(work.a + p * plan.L).x == id);
      n += on;
      if (on < kJoinWarps * 32) break;
    }
    float sum[N];
#pragma unroll
    for (int j = 0; j < N; ++j) sum[j] = 0.f;
    if (h < a.H) {
      const int lo = static_cast<int>(static_cast<long long>(n) * warp / kJoinWarps);
      const int hi = static_cast<int>(static_cast<long long>(n) * (warp + 1) / kJoinWarps);
      const float* p = work.part + (c + 1ll) * 2 * a.H + h;
      if (warp == 0) {
#pragma unroll
        for (int j = 0; j < N; ++j) sum[j] = p[-static_cast<long long>(a.H) + j];
      }
      for (int i = lo; i < hi; i += U) {
        float x[U][N];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int j = 0; j < N; ++j) x[u][j] = i + u < hi ? p[(i + u) * 2ll * a.H + j] : 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int j = 0; j < N; ++j) sum[j] += x[u][j];
      }
    }
#pragma unroll
    for (int j = 0; j < N; ++j) buf[warp][j * 32 + lane] = sum[j];
    __syncthreads();
    if (warp == 0 && h < a.H) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        sum[j] = 0.f;
        for (int w = 0; w < kJoinWarps; ++w) sum[j] += buf[w][j * 32 + lane];
      }
      finish<G, N>(a, vec, id, h, sum);
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------ host
bool aligned(const void* p, long long stride_bytes, long long to) {
  return (reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>(stride_bytes)) % to == 0;
}

template <typename T, int N>
cudaError_t lookup(const TbEmbeddingArgs& a, cudaStream_t s) {
  const int per = a.H / N;
  if (per >= 32) {
    const int segs = (per + 32 * kUnroll - 1) / (32 * kUnroll);
    const long long ctas = (static_cast<long long>(a.N) * segs + 7) / 8;
    lookup_wide_kernel<T, N><<<static_cast<unsigned>(ctas < (1 << 24) ? ctas : 1 << 24), 256, 0, s>>>(a, segs);
  } else {
    const long long ctas = (static_cast<long long>(a.N) * per + 255) / 256;
    lookup_narrow_kernel<T, N><<<static_cast<unsigned>(ctas < (1 << 24) ? ctas : 1 << 24), 256, 0, s>>>(a);
  }
  return cudaGetLastError();
}

// Vectors of 16 bytes, of 4, or single elements, as the rows' lengths and places allow.
template <typename T>
cudaError_t lookup_of(const TbEmbeddingArgs& a, cudaStream_t s) {
  constexpr long long e = sizeof(T);
  const auto fits = [&](long long b) {
    return a.H * e % b == 0 && aligned(a.weight, a.ld_w * e, b) && aligned(a.out, a.ld_out * e, b);
  };
  if (fits(16)) return lookup<T, 16 / e>(a, s);
  if constexpr (e == 2) {
    if (fits(4)) return lookup<T, 2>(a, s);
  }
  return lookup<T, 1>(a, s);
}

SortPlan plan_of(int N, int V) {
  SortPlan p{};
  p.N = N;
  p.V = V;
  int bits = 1;
  while (bits < 31 && (V >> bits) != 0) ++bits;  // keys 0 .. V
  p.passes = (bits + 8) / 9;
  p.bits = (bits + p.passes - 1) / p.passes;
  // pieces of at least 16 tokens, at most 4,096 of them (and of the workspace's rows)
  p.L = 16;
  while ((N + p.L - 1) / p.L > 4096) p.L *= 2;
  p.pieces = (N + p.L - 1) / p.L;
  return p;
}
size_t up16(size_t b) { return (b + 15) / 16 * 16; }

template <typename K, typename... Args>
cudaError_t launch_after(K kernel, unsigned grid, unsigned block, cudaStream_t s, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <typename T, typename G, int N>
cudaError_t grad(const TbEmbeddingGradArgs& a, cudaStream_t s) {
  const bool vec = aligned(a.grad, a.ld_grad * sizeof(G), N * sizeof(G) < 16 ? N * sizeof(G) : 16);
  const int slabs = (a.H + 32 * N - 1) / (32 * N);
  if (a.N <= kFew) {
    if (a.zero) {
      const size_t row = a.H * sizeof(G);
      const cudaError_t e = a.ld_grad == a.H ? cudaMemsetAsync(a.grad, 0, row * a.V, s)
                                             : cudaMemset2DAsync(a.grad, a.ld_grad * sizeof(G), 0, row, a.V, s);
      if (e != cudaSuccess) return e;
    }
    if (a.N > 0) grad_few_kernel<T, G, N><<<static_cast<unsigned>(a.N) * slabs, 256, 0, s>>>(a, slabs, vec);
    return cudaGetLastError();
  }
  const SortPlan plan = plan_of(a.N, a.V);
  SortWork work;
  char* w = static_cast<char*>(a.ws);
  work.a = reinterpret_cast<uint2*>(w);
  work.b = reinterpret_cast<uint2*>(w += up16(a.N * sizeof(uint2)));
  work.owners = reinterpret_cast<int*>(w += up16(a.N * sizeof(uint2)));
  work.part = reinterpret_cast<float*>(w += up16((plan.pieces + 1) * sizeof(int)));
  const int ranks = a.N <= 2048 ? 1 : a.N <= 4096 ? 2 : a.N <= 8192 ? 4 : 8;
  const int smem = kSortWarps * (1 << plan.bits) * static_cast<int>(sizeof(unsigned));
  cudaError_t e = tb::ensure_dyn_smem(reinterpret_cast<const void*>(&sort_kernel), kSortWarps * kMaxBins * 4);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ranks + (a.zero ? (148 - ranks) / ranks * ranks : 0));
  cfg.blockDim = dim3(kSortThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, sort_kernel, a, plan, work, static_cast<int>(sizeof(G)));
  if (e != cudaSuccess) return e;
  const long long threads = static_cast<long long>(plan.pieces) * (a.H / N);
  e = launch_after(pieces_kernel<T, G, N>, static_cast<unsigned>((threads + 255) / 256), 256, s, a, plan, work, vec);
  if (e != cudaSuccess) return e;
  const long long tasks = static_cast<long long>(plan.pieces) * slabs;
  return launch_after(join_kernel<G, N>, static_cast<unsigned>(tasks < 296 ? tasks : 296), kJoinWarps * 32, s, a, plan, work, slabs, vec);
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
  const SortPlan p = plan_of(N, V);
  return 2 * up16(N * sizeof(uint2)) + up16((p.pieces + 1) * sizeof(int)) + static_cast<size_t>(p.pieces) * 2 * H * sizeof(float);
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
