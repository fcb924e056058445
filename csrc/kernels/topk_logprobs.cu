// The k largest logits of each row as log-probabilities: for a row z of V logits
//
//   lse = log sum_j exp(z_j / T),   logp_i = z_{a_i} / T - lse,
//
// a_1 .. a_k the ids in order of (z descending, id ascending).
//
// One pass over the row forms the softmax's running maximum and sum, and the maximum of
// every group of 8 vectors (128 bytes).  The k largest elements lie in the k first groups
// by (maximum descending, index ascending): for an element outside them, each of those
// groups holds one that comes before it.  So the selection looks at V / 64 maxima in
// shared memory and reads some k groups again, whatever the data (all equal, ascending).
// Both selections search the k-th place by bisection over unique keys (value, index) with
// counts over the block, and stop at the first threshold that leaves few more than k;
// what is left is ordered by counting.
#include "kernels.h"
#include "vocab_rows.cuh"

namespace {

namespace cg = cooperative_groups;
using tb::Row;
using tb::SoftSum;

constexpr int kMaxK = 256;
constexpr int kIndexBits = 21;  // indexes below 2^20 elements (and the row's offset in its vectors)
constexpr uint32_t kIndexMask = (1u << kIndexBits) - 1;
constexpr int kRank = 512;  // elements that are ordered by counting
using Key = unsigned long long;

// Keeps the order of the values; +0 and -0 are equal, NaN is -inf.
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t b = __float_as_uint(isnan(x) ? -INFINITY : x + 0.f);
  return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}
// Larger keys come first: larger values, then lower indexes.
__device__ __forceinline__ Key key_of(uint32_t order, int index) {
  return (static_cast<Key>(order) << kIndexBits) | (kIndexMask - static_cast<uint32_t>(index));
}

struct Shared {
  Key cand[kRank];
  Key sorted[kMaxK];  // this CTA's own list, read by the others of its cluster
  float merge[64];
  float mine[2];
  uint32_t lo, hi;
  int count[3];
  int groups, cands, own;
  int list[kMaxK + kMaxK / 4 + 16];
};

__host__ __device__ constexpr int most_groups(int k) { return k + k / 4 + 16; }

// Sum of `c` over the block; `turn` counts the calls.
__device__ __forceinline__ int block_count(Shared& s, int c, int turn) {
  c = __reduce_add_sync(0xffffffffu, c);
  if ((threadIdx.x & 31) == 0 && c) atomicAdd(&s.count[turn % 3], c);
  __syncthreads();
  if (threadIdx.x == 0) s.count[(turn + 2) % 3] = 0;
  return s.count[turn % 3];
}

// A key with at least k and at most `most` of the n orders (index = position, or the
// element that `index_of` names) at or above it; n >= k.  `order` is in shared memory.
template <typename IndexOf>
__device__ Key threshold(Shared& s, const uint32_t* order, int n, int k, int most, Key lo, Key hi, int& turn,
                         IndexOf index_of) {
  int at_lo = n;
  while (at_lo > most && hi - lo > 1) {
    const Key mid = lo + (hi - lo) / 2;
    int c = 0;
    for (int i = threadIdx.x; i < n; i += blockDim.x) c += key_of(order[i], index_of(i)) >= mid;
    c = block_count(s, c, turn++);
    if (c >= k) {
      lo = mid;
      at_lo = c;
    } else {
      hi = mid;
    }
  }
  return lo;
}

template <typename T>
__global__ void __launch_bounds__(512, 2) topk_kernel(TbTopkLogprobsArgs a, float k1) {
  constexpr int E = Row<T>::E, GE = 8 * E;
  extern __shared__ uint32_t orders[];  // the groups' maxima, then the chosen groups' elements
  __shared__ Shared s;
  cg::cluster_group cl = cg::this_cluster();
  const int rank = cl.block_rank(), ranks = cl.num_blocks();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarps = blockDim.x >> 5;
  const int k = a.k;
  int turn = 0;
  for (long long r = blockIdx.x / ranks; r < a.R; r += gridDim.x / ranks) {
    const Row<T> row(static_cast<const T*>(a.logits) + r * a.ld, a.V, rank, ranks);
    const int g0 = row.v0 / 8, ng = (row.v1 - row.v0 + 7) / 8;
    if (threadIdx.x == 0) {
      s.lo = 0xffffffffu;
      s.hi = 0;
      s.groups = s.cands = 0;
      s.count[0] = s.count[1] = s.count[2] = 0;
    }
    __syncthreads();
    turn = 0;
    // ---- the pass: a warp takes 32 groups, lane l one vector of groups l / 8, 4 + l / 8, ...
    SoftSum sum;
    uint32_t olo = 0xffffffffu, ohi = 0;
    for (int c = row.v0 + warp * 256; c < row.v1; c += nwarps * 256) {
      float x[8][E], top[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int v = c + i * 32 + lane;
        if (v < row.v1) {
          row.load(v, x[i]);
        } else {
#pragma unroll
          for (int j = 0; j < E; ++j) x[i][j] = -INFINITY;
        }
      }
      float all = -INFINITY;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        top[i] = x[i][0];
#pragma unroll
        for (int j = 1; j < E; ++j) top[i] = fmaxf(top[i], x[i][j]);
        all = fmaxf(all, top[i]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) sum.add(x[i], all, k1);
      // maxima over eight lanes of eight vectors: lane l ends with those of vector l % 8
#pragma unroll
      for (int h = 4; h > 0; h >>= 1) {
        const bool up = lane & h;
#pragma unroll
        for (int i = 0; i < h; ++i) {
          const float send = up ? top[i] : top[i + h], keep = up ? top[i + h] : top[i];
          top[i] = fmaxf(keep, __shfl_xor_sync(0xffffffffu, send, h));
        }
      }
      const int g = c / 8 - g0 + (lane & 7) * 4 + lane / 8;
      if (g < ng) {
        const uint32_t o = order_of(top[0]);
        orders[g] = o;
        olo = min(olo, o);
        ohi = max(ohi, o);
      }
    }
    olo = __reduce_min_sync(0xffffffffu, olo);
    ohi = __reduce_max_sync(0xffffffffu, ohi);
    if (lane == 0) {
      atomicMin(&s.lo, olo);
      atomicMax(&s.hi, ohi);
    }
    sum = tb::block_merge(sum, k1, s.merge);  // (synchronises)
    // ---- the first k groups, and a few more
    uint32_t floor_order = 0;
    const uint32_t last = s.hi;
    if (ng > k) {
      const Key t = threshold(s, orders, ng, k, most_groups(k), static_cast<Key>(s.lo) << kIndexBits,
                              static_cast<Key>(last + 1ull) << kIndexBits, turn, [](int i) { return i; });
      floor_order = static_cast<uint32_t>(t >> kIndexBits);  // k elements are at or above it
      for (int i = threadIdx.x; i < ng; i += blockDim.x)
        if (key_of(orders[i], i) >= t) s.list[atomicAdd(&s.groups, 1)] = i;
    } else {
      for (int i = threadIdx.x; i < ng; i += blockDim.x) s.list[i] = i;
      if (threadIdx.x == 0) s.groups = ng;
    }
    __syncthreads();
    // ---- their elements
    const int groups = s.groups, n = groups * GE;
    int above = 0;
    for (int i = threadIdx.x; i < groups * 8; i += blockDim.x) {
      const int v = (g0 + s.list[i >> 3]) * 8 + (i & 7);
      float x[E];
      if (v < row.v1) {
        row.load(v, x);
      } else {
#pragma unroll
        for (int j = 0; j < E; ++j) x[j] = -INFINITY;
      }
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const int e = v * E - row.mis + j;  // outside the row: 0, below every order
        const uint32_t o = e >= 0 && e < a.V ? order_of(x[j]) : 0;
        orders[i * E + j] = o;
        above += o >= max(floor_order, 1u);
      }
    }
    const auto element = [&](int i) {
      return (g0 + s.list[i / GE]) * GE + i % GE - row.mis;
    };
    above = block_count(s, above, turn++);
    const int own = min(k, above);  // (fewer than k: a short part of a row)
    Key t = static_cast<Key>(max(floor_order, 1u)) << kIndexBits;
    if (above > kRank) {
      t = threshold(s, orders, n, own, kRank, t, static_cast<Key>(last + 1ull) << kIndexBits, turn,
                    [&](int i) { return max(element(i), 0); });
    }
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
      if (orders[i] == 0) continue;
      const Key x = key_of(orders[i], element(i));
      if (x >= t) s.cand[atomicAdd(&s.cands, 1)] = x;
    }
    __syncthreads();
    const int cands = s.cands;
    for (int i = threadIdx.x; i < cands; i += blockDim.x) {
      const Key x = s.cand[i];
      int place = 0;
      for (int j = 0; j < cands; ++j) place += s.cand[j] > x;
      if (place < own) s.sorted[place] = x;
    }
    if (threadIdx.x == 0) s.own = own;
    __syncthreads();
    // ---- the cluster's lists joined: a place is the sum of the places in every list
    sum = tb::cluster_merge(sum, k1, s.mine);
    const double inv_t = 1.0 / a.temperature, lns = log(static_cast<double>(sum.s));
    if (rank == 0 && threadIdx.x == 0)
      a.lse[r] = isinf(sum.m) && !isnan(sum.s) ? sum.m : static_cast<float>(sum.m * inv_t + lns);
    for (int i = threadIdx.x; i < own; i += blockDim.x) {
      const Key x = s.sorted[i];
      int place = i;
      for (int o = 0; o < ranks; ++o) {
        if (o == rank) continue;
        const Key* theirs = cl.map_shared_rank(s.sorted, o);
        int lo = 0, hi = *cl.map_shared_rank(&s.own, o);
        while (lo < hi) {
          const int mid = (lo + hi) / 2;
          if (theirs[mid] > x) {
            lo = mid + 1;
          } else {
            hi = mid;
          }
        }
        place += lo;
      }
      if (place >= k) continue;
      const int e = static_cast<int>(kIndexMask - (static_cast<uint32_t>(x) & kIndexMask));
      // the element's own value (the order has NaN as -inf)
      const float z = tb::to_f32(row.row[e]);
      float y;
      if (isnan(sum.s)) {
        y = NAN;
      } else if (isinf(sum.m)) {
        y = sum.m > 0 && z == sum.m ? NAN : -INFINITY;
      } else {
        y = static_cast<float>((static_cast<double>(z) - sum.m) * inv_t - lns);
      }
      a.logp[r * k + place] = y;
      a.ids[r * k + place] = e;
    }
    if (ranks > 1) {
      cl.sync();
    } else {
      __syncthreads();
    }
  }
}

template <typename T>
cudaError_t launch(const TbTopkLogprobsArgs& a, cudaStream_t stream) {
  constexpr int E = Row<T>::E;
  const int groups = (a.V + E - 2 + 8 * E) / (8 * E);
  int ranks = 1;
  while (ranks < 8 && (groups + ranks - 1) / ranks > 8192) ranks *= 2;
  const int per = (groups + ranks - 1) / ranks;
  const int chosen = (per > a.k ? (per < most_groups(a.k) ? per : most_groups(a.k)) : per) * 8 * E;
  const size_t smem = sizeof(uint32_t) * static_cast<size_t>(per > chosen ? per : chosen);
  cudaError_t e = tb::ensure_dyn_smem(reinterpret_cast<const void*>(&topk_kernel<T>), 128 * 1024);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  const int rows = a.R < (1 << 20) ? a.R : 1 << 20;
  cfg.gridDim = dim3(static_cast<unsigned>(rows) * ranks);
  cfg.blockDim = dim3(512);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, topk_kernel<T>, a, static_cast<float>(tb::kLog2e / a.temperature));
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
