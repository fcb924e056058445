// The k largest logits of each row as log-probabilities: for a row z of V logits
//
//   lse = log sum_j exp(z_j / T),   logp_i = z_{a_i} / T - lse,
//
// a_1 .. a_k the ids in order of (z descending, id ascending).
//
// One pass over the row forms the softmax's running maximum and sum, and the maximum of
// every group of 8 vectors (128 bytes; of every vector in short rows).  The k largest
// elements lie in the k first groups by (maximum descending, index ascending): for an element
// outside them, each of those groups holds one that comes before it.  So the selection looks at V / 64 maxima in
// shared memory and reads some k groups again, whatever the data (all equal, ascending).
// A histogram of the maxima, filled during the pass, gives a value that k groups reach and
// few more; of those groups the elements that reach it, some k, are ordered by counting.
// Where too many do (equal values, the largest side by side), the k-th place is searched by
// bisection with counts over the block, first of the value and then of the index.
//
// The floor is one read of the logits.  4,096 rows of 151,936 bf16 take 251 us (4.9 TB/s, 77%
// of the copy rate): the exponentials keep their unit 59% busy, and while one CTA selects, the
// other three of its SM load.  512 rows, one wave, take 40 us (3.8 TB/s): all CTAs select at
// the same time.
#include <type_traits>

#include "kernels.h"
#include "vocab_rows.cuh"

namespace {

namespace cg = cooperative_groups;
using tb::Row;
using tb::SoftSum;
using tb::Vec;

constexpr int kThreads = 256;
constexpr int kMaxK = 256;
constexpr int kIndexBits = 21;  // indexes below 2^20 elements (and the row's offset in its vectors)
constexpr uint32_t kIndexMask = (1u << kIndexBits) - 1;
constexpr int kRank = 512;  // elements that are ordered by counting
constexpr int kSingle = 2048;  // vectors of a part up to which each is a group of its own
constexpr int kBins = 8192;   // of the histogram, two to a word
using Key = unsigned long long;

// Groups that are looked at again: by the histogram, whose bins hold several values, and by
// the exact search.
__host__ __device__ constexpr int most_groups(int k) { return 2 * k + 32; }
__host__ __device__ constexpr int few_groups(int k) { return k + k / 4 + 16; }

// Whole numbers in the order of the values: +0 and -0 are equal, NaN is -inf, 0 is below all.
template <typename T>
struct Order;
template <>
struct Order<float> {
  using Type = uint32_t;
  __device__ __forceinline__ static uint32_t of(float x) {
    const uint32_t b = __float_as_uint(isnan(x) ? -INFINITY : x + 0.f);
    return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
  }
  __device__ __forceinline__ static float value(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o); }
};
template <uint32_t INF>
struct Order16 {  // INF: the bits of infinity
  using Type = uint16_t;
  __device__ __forceinline__ static uint32_t of_bits(uint32_t b) {
    if ((b & 0x7fffu) > INF) b = 0x8000u | INF;
    if (b == 0x8000u) b = 0;
    return b & 0x8000u ? b ^ 0xffffu : b | 0x8000u;
  }
  __device__ __forceinline__ static uint32_t bits(uint32_t o) { return o & 0x8000u ? o ^ 0x8000u : o ^ 0xffffu; }
};
template <>
struct Order<__nv_bfloat16> : Order16<0x7f80u> {
  __device__ __forceinline__ static uint32_t of(float x) { return of_bits(__float_as_uint(x) >> 16); }  // (a bf16 value)
  __device__ __forceinline__ static float value(uint32_t o) { return __uint_as_float(bits(o) << 16); }
};
template <>
struct Order<__half> : Order16<0x7c00u> {
  __device__ __forceinline__ static uint32_t of(float x) { return of_bits(__half_as_ushort(__float2half_rn(x))); }
  __device__ __forceinline__ static float value(uint32_t o) { return __half2float(__ushort_as_half(static_cast<unsigned short>(bits(o)))); }
};

// The orders of a vector's elements, 0 outside the row, and how many are at or above `floor`.
template <typename T>
__device__ __forceinline__ uint4 orders_of(const Row<T>& row, int v, const uint4& p, uint32_t floor, int& above) {
  constexpr int E = Row<T>::E;
  uint32_t o[E];
#pragma unroll
  for (int j = 0; j < E; ++j) {
    if constexpr (sizeof(T) == 4) {
      o[j] = Order<T>::of(__uint_as_float(j == 0 ? p.x : j == 1 ? p.y : j == 2 ? p.z : p.w));
    } else {
      const uint32_t w = j < 2 ? p.x : j < 4 ? p.y : j < 6 ? p.z : p.w;
      o[j] = Order<T>::of_bits(j & 1 ? w >> 16 : w & 0xffffu);
    }
  }
  if (v >= row.v1 || !row.inside(v, v + 1)) {
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const int e = v * E - row.mis + j;
      if (v >= row.v1 || e < 0 || e >= row.V) o[j] = 0;
    }
  }
#pragma unroll
  for (int j = 0; j < E; ++j) above += o[j] >= floor;
  if constexpr (sizeof(T) == 4) {
    return make_uint4(o[0], o[1], o[2], o[3]);
  } else {
    return make_uint4(o[0] | o[1] << 16, o[2] | o[3] << 16, o[4] | o[5] << 16, o[6] | o[7] << 16);
  }
}

// The histogram's bins, ascending with the order's upper 16 bits: single bf16 values from
// 2^-8 to 2^24 (8 fp16 values), 16 of them below and above and of the negative ones.
template <typename T>
struct Bin {
  static constexpr bool kHalf = std::is_same<T, __half>::value;
  static constexpr int kShift = sizeof(T) == 4 ? 16 : 0;
  __device__ __forceinline__ static int of(uint32_t order) {
    const uint32_t h = order >> kShift, p = h - 0x8000u;
    if (h < 0x8000u) return h >> 4;
    if (kHalf) return 2048 + (p >> 3);
    return p < 0x3b80u ? 2048 + (p >> 4) : p < 0x4b80u ? 3000 + (p - 0x3b80u) : 7096 + ((p - 0x4b80u) >> 4);
  }
  __device__ __forceinline__ static uint32_t lowest(int b) {
    uint32_t h;
    if (b < 2048) {
      h = b << 4;
    } else if (kHalf) {
      h = 0x8000u + ((b - 2048) << 3);
    } else {
      h = 0x8000u + (b < 3000 ? (b - 2048) << 4 : b < 7096 ? 0x3b80 + (b - 3000) : 0x4b80 + ((b - 7096) << 4));
    }
    return h << kShift;
  }
};

struct Shared {
  Key cand[kRank];
  Key sorted[kMaxK];  // this CTA's own list, read by the others of its cluster
  float part[2][kThreads / 32];
  float mine[2];
  uint32_t lo, hi;
  int count[3];
  int groups, cands, own;
  int list[most_groups(kMaxK)];
};

// Sum of `c` over the block; `turn` counts the calls.
__device__ __forceinline__ int block_count(Shared& s, int c, int& turn) {
  c = __reduce_add_sync(0xffffffffu, c);
  int* slot = &s.count[turn % 3];
  if ((threadIdx.x & 31) == 0 && c) atomicAdd(slot, c);
  __syncthreads();
  if (threadIdx.x == 0) s.count[(turn + 2) % 3] = 0;
  ++turn;
  return *slot;
}

// A place in the order (value descending, index ascending): at least k and at most `most`
// of the n orders in shared memory are at or before it.  n >= k of them are at or above lo,
// none at or above hi; `index_of` gives the index of position i, ascending or not.
struct Place {
  uint32_t order;
  int index;
  __device__ __forceinline__ bool takes(uint32_t o, int i) const { return o > order || (o == order && i <= index); }
};
template <typename O, typename IndexOf>
__device__ Place place_of(Shared& s, const O* orders, int n, int k, int most, int at_lo, uint32_t lo, Key hi, int last, int& turn,
                          IndexOf index_of) {
  int at_hi = 0;
  Place p{lo, last};
  while (at_lo > most && hi - p.order > 1) {
    const uint32_t mid = p.order + static_cast<uint32_t>((hi - p.order) / 2);
    int c = 0;
    for (int i = threadIdx.x; i < n; i += kThreads) c += orders[i] >= mid;
    c = block_count(s, c, turn);
    if (c >= k) {
      p.order = mid;
      at_lo = c;
    } else {
      hi = mid;
      at_hi = c;
    }
  }
  int low = -1;  // too many equal ones: the first of them
  while (at_lo > most && p.index - low > 1) {
    const int mid = low + (p.index - low) / 2;
    int c = 0;
    for (int i = threadIdx.x; i < n; i += kThreads) c += orders[i] == p.order && index_of(i) <= mid;
    c = block_count(s, c, turn) + at_hi;
    if (c >= k) {
      p.index = mid;
      at_lo = c;
    } else {
      low = mid;
    }
  }
  return p;
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 4) topk_kernel(TbTopkLogprobsArgs a, float k1, float inv_t) {
  using O = typename Order<T>::Type;
  constexpr int E = Row<T>::E;
  // the histogram and the groups' maxima; in their place, where too many elements are equal,
  // the chosen groups' elements; then the cluster's lists.  (Little of it: what shared memory
  // leaves of the L1 cache holds the loads in flight.)
  extern __shared__ uint4 dynamic[];
  uint32_t* hist = reinterpret_cast<uint32_t*>(dynamic);
  O* orders = reinterpret_cast<O*>(dynamic + kBins / 8);
  __shared__ Shared s;
  cg::cluster_group cl = cg::this_cluster();
  const int rank = cl.block_rank(), ranks = cl.num_blocks();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int k = a.k;
  for (int i = threadIdx.x; i < kBins / 8; i += kThreads) dynamic[i] = make_uint4(0, 0, 0, 0);
  for (long long r = blockIdx.x / ranks; r < a.R; r += gridDim.x / ranks) {
    const Row<T> row(static_cast<const T*>(a.logits) + r * a.ld, a.V, rank, ranks);
    const bool single = row.v1 - row.v0 <= kSingle;
    const int GV = single ? 1 : 8, ng = (row.v1 - row.v0 + GV - 1) / GV;  // vectors of a group, groups
    if (threadIdx.x == 0) {
      s.lo = 0xffffffffu;
      s.hi = 0;
      s.groups = s.cands = 0;
      s.count[0] = s.count[1] = s.count[2] = 0;
    }
    __syncthreads();
    int turn = 0;
    // ---- the pass
    tb::RunningSum<T> running;
    uint32_t olo = 0xffffffffu, ohi = 0;
    const auto keep = [&](int g, typename Vec<T>::Max top) {
      const uint32_t o = Order<T>::of(Vec<T>::value(top));
      orders[g] = static_cast<O>(o);
      const int bin = Bin<T>::of(o);
      atomicAdd(&hist[bin >> 1], 1u << (bin & 1) * 16);
      olo = min(olo, o);
      ohi = max(ohi, o);
    };
    for (int c = row.v0 + warp * tb::kChunk; c < row.v1; c += kThreads / 32 * tb::kChunk) {
      uint4 p[8];
      row.load_chunk(c, p);
      typename Vec<T>::Max top[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) top[i] = Vec<T>::top(p[i]);
      typename Vec<T>::Max all = top[0];
#pragma unroll
      for (int i = 1; i < 8; ++i) all = Vec<T>::max(all, top[i]);
      running.add(p, Vec<T>::value(all), k1);
      if (single) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int g = c - row.v0 + i * 32 + lane;
          if (g < ng) keep(g, top[i]);
        }
        continue;
      }
      // maxima over eight lanes of eight vectors: lane l ends with those of its vector l % 8
#pragma unroll
      for (int h = 4; h > 0; h >>= 1) {
        const bool up = lane & h;
#pragma unroll
        for (int i = 0; i < h; ++i) {
          const auto send = up ? top[i] : top[i + h], keep = up ? top[i + h] : top[i];
          top[i] = Vec<T>::max(keep, __shfl_xor_sync(0xffffffffu, send, h));
        }
      }
      const int g = (c - row.v0) / 8 + (lane & 7) * 4 + lane / 8;
      if (g < ng) keep(g, top[0]);
    }
    SoftSum sum = running.done(k1);
    sum.merge_lanes(k1);
    olo = __reduce_min_sync(0xffffffffu, olo);
    ohi = __reduce_max_sync(0xffffffffu, ohi);
    if (lane == 0) {
      s.part[0][warp] = sum.m;
      s.part[1][warp] = sum.s;
      atomicMin(&s.lo, olo);
      atomicMax(&s.hi, ohi);
    }
    __syncthreads();
    sum.m = lane < kThreads / 32 ? s.part[0][lane] : -INFINITY;
    sum.s = lane < kThreads / 32 ? s.part[1][lane] : 0.f;
    sum.merge_lanes(k1);
    // ---- the first k groups, and a few more: from the highest bin down (each warp for itself)
    uint32_t floor = 1;
    int at_floor = ng;
    const Key above_all = static_cast<Key>(s.hi) + 1;
    Place t{1, 0x7fffffff};
    if (ng > k) {
      int at = 0;  // groups in the words above
      for (int word = Bin<T>::of(s.hi) >> 1; word >= 0; word -= 32) {
        const uint32_t h = word >= lane ? hist[word - lane] : 0;
        const int c = (h >> 16) + (h & 0xffffu);
        int incl = c;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int x = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += x;
        }
        const unsigned enough = __ballot_sync(0xffffffffu, at + incl >= k);
        if (!enough) {
          at += __shfl_sync(0xffffffffu, incl, 31);
          continue;
        }
        const int l = __ffs(enough) - 1;
        const int before = at + __shfl_sync(0xffffffffu, incl - c, l);
        const uint32_t w = __shfl_sync(0xffffffffu, h, l);
        const bool upper = before + static_cast<int>(w >> 16) >= k;
        floor = Bin<T>::lowest((word - l) * 2 + (upper ? 1 : 0));
        at = before + static_cast<int>(w >> 16) + (upper ? 0 : static_cast<int>(w & 0xffffu));
        break;
      }
      t.order = floor = max(floor, s.lo);
      at_floor = at;
    }
    const auto choose = [&] {
      for (int i = threadIdx.x; i < ng; i += kThreads)
        if (t.takes(orders[i], i)) s.list[atomicAdd(&s.groups, 1)] = i;
      __syncthreads();
    };
    if (at_floor > most_groups(k) && ng > k) {
      t = place_of(s, orders, ng, k, few_groups(k), at_floor, floor, above_all, ng - 1, turn, [](int i) { return i; });
      floor = t.order;
    }
    choose();
    int groups = s.groups;
    // ---- their elements at or above it: k of them at least
    const auto vector_of = [&](int i) { return row.v0 + (single ? s.list[i] : s.list[i >> 3] * 8 + (i & 7)); };
    const auto push = [&](uint32_t o, int e) {
      const int at = atomicAdd(&s.cands, 1);
      if (at < kRank) s.cand[at] = static_cast<Key>(o) << kIndexBits | (kIndexMask - static_cast<uint32_t>(e));
    };
    for (int i0 = threadIdx.x; i0 < groups * GV; i0 += 4 * kThreads) {
      uint4 p[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) p[u] = i0 + u * kThreads < groups * GV ? row.load(vector_of(i0 + u * kThreads)) : Row<T>::lowest();
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + u * kThreads;
        if (i >= groups * GV || Order<T>::of(Vec<T>::value(Vec<T>::top(p[u]))) < floor) continue;
        const int v = vector_of(i);
        int above = 0;
        const uint4 q = orders_of(row, v, p[u], floor, above);
        if (above) {
#pragma unroll
          for (int j = 0; j < E; ++j) {
            const uint32_t word = j / (E / 4) == 0 ? q.x : j / (E / 4) == 1 ? q.y : j / (E / 4) == 2 ? q.z : q.w;
            const uint32_t o = sizeof(T) == 4 ? word : j & 1 ? word >> 16 : word & 0xffffu;
            if (o >= floor) push(o, v * E - row.mis + j);
          }
        }
      }
    }
    __syncthreads();
    int cands = s.cands;
    bool trashed = ranks > 1;  // (the lists come to lie there)
    const int own = min(k, cands);  // (fewer than k: a short part of a row)
    if (cands > kRank) {  // ---- too many: the first k groups' elements in shared memory, and the first `own` of them
      if (groups > few_groups(k) && ng > k) {
        t = place_of(s, orders, ng, k, few_groups(k), at_floor, floor, above_all, ng - 1, turn, [](int i) { return i; });
        if (threadIdx.x == 0) s.groups = 0;
        __syncthreads();
        choose();
        groups = s.groups;
      }
      floor = t.order;
      const int n = groups * GV * E;
      int above = 0;
      for (int i = threadIdx.x; i < groups * GV; i += kThreads) {
        const int v = vector_of(i);
        dynamic[i] = orders_of(row, v, row.load(v), floor, above);
      }
      cands = block_count(s, above, turn);
      orders = reinterpret_cast<O*>(dynamic);
      const auto element = [&](int i) { return vector_of(i / E) * E + i % E - row.mis; };
      const Place e = place_of(s, orders, n, own, kRank, cands, floor, above_all, a.V, turn, element);
      if (threadIdx.x == 0) s.cands = 0;
      __syncthreads();
      for (int i = threadIdx.x; i < n; i += kThreads) {
        const uint32_t o = orders[i];
        if (o >= e.order && e.takes(o, element(i))) push(o, element(i));
      }
      __syncthreads();
      cands = s.cands;
      orders = reinterpret_cast<O*>(dynamic + kBins / 8);
      trashed = true;
    } else if (!trashed) {  // the bins that were in use, for the next row
      for (int i = (Bin<T>::of(s.lo) >> 1) + threadIdx.x; i <= Bin<T>::of(s.hi) >> 1; i += kThreads) hist[i] = 0;
    }
    for (int i = threadIdx.x; i < cands; i += kThreads) {
      const Key x = s.cand[i];
      int place = 0;
#pragma unroll 8
      for (int j = 0; j < cands; ++j) place += s.cand[j] > x;
      if (place < own) s.sorted[place] = x;
    }
    if (ranks > 1) {
      if (threadIdx.x == 0) {
        s.own = own;
        s.mine[0] = sum.m;
        s.mine[1] = sum.s;
      }
      cl.sync();
      // ---- the cluster's sums, and its lists side by side
      SoftSum whole;
      for (int o = 0; o < ranks; ++o) {
        const float* m = cl.map_shared_rank(s.mine, o);
        whole.merge(m[0], m[1], k1);
      }
      sum = whole;
      Key* lists = reinterpret_cast<Key*>(dynamic);
      for (int i = threadIdx.x; i < ranks * k; i += kThreads) {
        const int o = i / k, j = i - o * k;
        lists[i] = j < *cl.map_shared_rank(&s.own, o) ? cl.map_shared_rank(s.sorted, o)[j] : 0;
      }
    }
    __syncthreads();
    // ---- a place is the sum of the places in every list
    const bool plain = !isinf(sum.m) && !isnan(sum.s);
    const float2 lns = plain ? tb::log_of(sum.s) : make_float2(0.f, 0.f);
    if (rank == 0 && threadIdx.x == 0)
      a.lse[r] = plain ? fmaf(sum.m, inv_t, lns.x + lns.y) : isnan(sum.s) ? NAN : sum.m;
    for (int i = threadIdx.x; i < own; i += kThreads) {
      const Key x = s.sorted[i];
      int place = i;
      if (ranks > 1) {
        const Key* lists = reinterpret_cast<const Key*>(dynamic);
        for (int o = 0; o < ranks; ++o) {
          if (o == rank) continue;
          int lo = 0, hi = k;
          while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (lists[o * k + mid] > x) {
              lo = mid + 1;
            } else {
              hi = mid;
            }
          }
          place += lo;
        }
        if (place >= k) continue;
      }
      const float z = Order<T>::value(static_cast<uint32_t>(x >> kIndexBits));
      float y;
      if (plain) {
        y = tb::Scaled{inv_t}(z, sum.m, lns);
      } else {
        y = isnan(sum.s) || (sum.m > 0 && z == sum.m) ? NAN : -INFINITY;
      }
      a.logp[r * k + place] = y;
      a.ids[r * k + place] = static_cast<int>(kIndexMask - (static_cast<uint32_t>(x) & kIndexMask));
    }
    if (ranks > 1) {
      cl.sync();
    } else {
      __syncthreads();
    }
    if (trashed)
      for (int i = threadIdx.x; i < kBins / 8; i += kThreads) dynamic[i] = make_uint4(0, 0, 0, 0);
  }
}

// CTAs of a cluster: as many as half the machine holds beside the other rows (clusters that
// would fill it wait for one another: 74 rows of 2,374 groups take 18.5 us with one CTA, 15.6
// with four, 25.1 with eight), 512 groups at least to each (joining the lists costs 3 us: four
// rows of 500 groups take 8.1 us with one CTA and 9.2 with two, of 1,024 groups 10.9 and 9.4,
// of 2,374 groups 18.1, and 11.5 with four); enough of them that the maxima of a part fit its
// shared memory.
int ranks_of(int R, int groups) {
  int ranks = 1;
  while (ranks < 8 && ((groups + ranks - 1) / ranks > 8192 || (R * 4ll * ranks <= 148 * 4 && groups >= 1024 * ranks))) ranks *= 2;
  return ranks;
}

template <typename T>
cudaError_t launch(const TbTopkLogprobsArgs& a, cudaStream_t stream) {
  constexpr int E = Row<T>::E;
  using O = typename Order<T>::Type;
  const int groups = (a.V + E - 2 + 8 * E) / (8 * E), ranks = ranks_of(a.R, groups), per = (groups + ranks - 1) / ranks;
  const int chosen = (per > a.k && per > few_groups(a.k) ? few_groups(a.k) : per) * 8 * E;
  const int maxima = per * 8 < kSingle ? per * 8 : per > kSingle ? per : kSingle;
  size_t smem = kBins * 2 + (sizeof(O) * maxima + 15) / 16 * 16;
  if (smem < sizeof(O) * chosen) smem = sizeof(O) * chosen;
  if (smem < ranks * a.k * sizeof(Key)) smem = ranks * a.k * sizeof(Key);
  cudaError_t e = tb::ensure_dyn_smem(reinterpret_cast<const void*>(&topk_kernel<T>), 64 * 1024);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  const int rows = a.R < (1 << 20) ? a.R : 1 << 20;
  cfg.gridDim = dim3(static_cast<unsigned>(rows) * ranks);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, topk_kernel<T>, a, static_cast<float>(tb::kLog2e / a.temperature),
                            static_cast<float>(1.0 / a.temperature));
}

}  // namespace

extern "C" int tb_topk_logprobs(const TbTopkLogprobsArgs* args, cudaStream_t s) {
  const TbTopkLogprobsArgs& a = *args;
  if (a.R < 0 || a.V < 1 || a.V > 1 << 20 || a.k < 1 || a.k > kMaxK || a.k > a.V)
    return static_cast<int>(cudaErrorInvalidValue);
  if (a.R == 0) return 0;
  switch (a.dtype) {
    case TB_BF16: return static_cast<int>(launch<__nv_bfloat16>(a, s));
    case TB_F16: return static_cast<int>(launch<__half>(a, s));
    case TB_F32: return static_cast<int>(launch<float>(a, s));
    default: return static_cast<int>(cudaErrorInvalidValue);
  }
}
