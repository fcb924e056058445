// The distillation loss of rows of logits against a teacher's list, and its gradient.
//
// For a row z, its list (a_k, l_k) with the set S of its ids, t_k = exp(l_k), and
// p = softmax(z / T), the row's loss is w KL + c (-log p_y), with
//
//   forward:        KL = sum_S t (log t - log p),                 T dKL/dz_j = p_j - t_j
//                   (t divided by its sum, whatever the list's own scale)
//   forward, rest:  ... + t_R (log t_R - log p_R),                T dKL/dz_j = p_j - t_j in S,
//                                                                 (p_R - t_R) q_j outside
//                   (p times sum t + t_R where that is not 1)
//   reverse:        KL = sum_S p (log p - log t)
//                        + p_R (log p_R - log t_R),               T dKL/dz_j = p_j (f_j - KL)
//
// t_R = 1 - sum t, p_R = sum of p outside S, q = p / p_R there, f = log p - log t of the
// element's class.  Outside S every gradient is one number of the row times
// x_j = exp((z_j - m) / T), m the largest logit there.
//
// The pass over the row leaves the elements of S out (a bitmap in shared memory, a byte
// per vector), so that p_R is a sum of its own terms and not a difference from 1; the
// elements of S join afterwards.  A second pass writes the gradient, then the elements of S
// are written over.  Where both passes are one launch, the second finds most of the row in
// the L2 cache, by the policy that the first one read it with.  Masses are summed in 64 bits
// (t_R is 1 less their sum), and log S is kept as the sum of two fp32 numbers: the loss is a
// small difference of large ones.
//
// Sums over a row and the KL are in fp32 (a loss of ordinary size is off by 1e-7 to 3e-7 of its
// terms, 64-bit sums would give 3e-8): what they round is far below the logits' own type, and
// 64-bit additions for every logit would bound the kernel.
//
// The floor is one read of the live rows and one write of the gradient.  4,096 rows of 151,936
// bf16 (all live) take 517 us out of an empty L2 cache and 530 to 554 (by the machine) one call
// after another from Python, 4.5 to 4.7 TB/s; in place, as a trainer calls it, 4% more: what is
// written are the lines that the first pass asked to be kept.  A third of the rows' second reads
// misses the L2 cache (495 MB read for 360 of 1,184 rows), whose writes pass through it.  Rows
// kept in shared memory, rings of bulk loads and the next row's first loads ahead gained nothing:
// then too few loads are in flight, or the sums wait for the stores.  The loss alone, 1,184 rows:
// 76 us, 4.7 TB/s.  Short rows (777 of 32,003 fp16, odd: 37 us for a floor of 14) wait four times
// per row for all warps (list, repeats, sums, numbers), and the last wave of rows is thin (622
// live rows on 592 places).
#include "kernels.h"
#include "vocab_rows.cuh"

namespace {

namespace cg = cooperative_groups;
using tb::Row;
using tb::SoftSum;
using tb::Vec;

constexpr int kMaxList = 256;  // (a thread for each entry)
constexpr int kMaxWarps = 16;
constexpr int kLane = 8;  // vectors of a lane at a time
constexpr float kPlain = 46.f;  // log-masses up to here (1e20, and 1e-20) are summed as they are
constexpr double kRestMin = 1.0 / (1 << 20);
enum { kLoss, kBoth, kGrad };  // what a launch computes (kGrad: from the numbers that kLoss kept)

// What a row's passes share.
struct Numbers {
  float origin, factor;  // the gradient outside the list: factor x 2^((z - origin) k1)
  float top;
  float2 lns;       // log p = (z - top) / T - lns
  float kl, whole;  // whole: sum t + t_R
};

// The weights of the KL and of the target, and the target (-1: none).
struct Weights {
  float w, c;
  int y;
  bool bad;  // a target past the vocabulary
  __device__ __forceinline__ Weights(const TbDistillArgs& a, float w_, float c_, int y_) : w(w_), c(y_ < 0 ? 0.f : c_), y(y_) {
    bad = y >= a.V && live();
    if (y >= a.V) {
      y = -1;
      c = 0.f;
    }
  }
  __device__ __forceinline__ bool live() const { return w != 0.f || c != 0.f; }
};

struct Shared {
  float part[2][kMaxWarps];
  float mine[2][2];  // of rows in turn, read by the others of the cluster
  Numbers n;
  // the row's weights and list: what lives over the passes is here, not in registers
  float w, c, z_y;
  int y, y_listed, special;
  __align__(16) int id[kMaxList];  // -1: padding
  float z[kMaxList], l[kMaxList];
  double t[kMaxList];  // mass of the class (l: its logarithm), both perhaps relative to the largest without the rest;
                       // -1 where the entry is not its id's first
  // the softmax sum of the list's elements, the masses' sum, t_R, and their logarithms
  float in_m, in_s;
  float mass, log_mass, t_rest, log_t_rest;
};

// Warp 0: the list's sums.
__device__ __forceinline__ void list_sums(const TbDistillArgs& a, Shared& s, float k1) {
  const int lane = threadIdx.x & 31;
  SoftSum in;
  double mass = 0.0;
  for (int k = lane; k < a.K; k += 32) {
    if (s.id[k] < 0 || s.t[k] < 0.0) continue;
    const float x = s.z[k];
    in.merge(isnan(x) ? -INFINITY : x, isnan(x) ? NAN : 1.f, k1);
    mass += s.t[k];
  }
  in.merge_lanes(k1);
  mass = tb::warp_sum(mass);
  if (lane) return;
  s.in_m = in.m;
  s.in_s = in.s;
  s.mass = static_cast<float>(mass);
  s.log_mass = a.kind == TB_DISTILL_FORWARD && s.mass != 0.f ? logf(s.mass) : 0.f;
  const double t = fmax(1.0 - mass, a.kind == TB_DISTILL_REVERSE ? kRestMin : 0.0);
  s.t_rest = isnan(mass) ? NAN : static_cast<float>(t);
  s.log_t_rest = s.t_rest > 0.f ? logf(s.t_rest) : 0.f;
}

// Warp 0, when the row's sums are known: the loss, and what the gradient needs.
__device__ __forceinline__ void numbers_of(const TbDistillArgs& a, Shared& s, long long r, const SoftSum& sum, float k1, float inv_t,
                                           bool write) {
  const int lane = threadIdx.x & 31;
  const float w = s.w, c = s.c;
  const bool listed = w != 0.f;
  SoftSum all = sum;
  all.merge(s.in_m, s.in_s, k1);
  const bool good = !isnan(all.s) && !isinf(all.m);
  const float2 lns = good ? tb::log_of(all.s) : make_float2(0.f, 0.f);
  const tb::Scaled log_p{inv_t};
  // log p of the elements outside; none there: their terms are left out
  const bool none = sum.m == -INFINITY || !good;
  float lp_rest = 0.f, p_rest = 0.f;
  if (!none) {
    const float2 l = tb::log_of(sum.s);
    lp_rest = fmaf(sum.m - all.m, inv_t, l.x - lns.x) + (l.y - lns.y);
    p_rest = tb::ex2(lp_rest * static_cast<float>(tb::kLog2e));
  }
  float kl = 0.f, h = 0.f, whole = 1.f;  // h: factor of q_j outside the list
  if (listed) {
    for (int k = lane; k < a.K; k += 32) {
      const float t = static_cast<float>(s.t[k]);
      if (s.id[k] < 0 || t < 0.f) continue;
      const float lp = log_p(s.z[k], all.m, lns);
      const float lt = s.l[k] - s.log_mass;
      if (a.kind == TB_DISTILL_REVERSE) {
        const float p = tb::ex2(lp * static_cast<float>(tb::kLog2e));
        if (p != 0.f) kl += p * (lp - lt);
      } else if (const float u = a.kind == TB_DISTILL_FORWARD && t != 0.f ? t / s.mass : t; u != 0.f) {
        kl += u * (lt - lp);
      } else if (lp == -INFINITY && s.t[k] != 0.0) {
        kl += INFINITY;  // (a mass below 2^-149 that the student rules out)
      }
    }
    kl = tb::warp_sum(kl);
    if (a.kind == TB_DISTILL_FORWARD) {
      whole = s.mass != 0.f ? 1.f : 0.f;
      h = whole * p_rest;
    } else if (a.kind == TB_DISTILL_FORWARD_REST) {
      const float t_out = none ? 0.f : s.t_rest;
      if (t_out > 0.f) kl += t_out * (s.log_t_rest - lp_rest);
      whole = s.mass + t_out;
      h = whole * p_rest - t_out;
    } else {
      const float f_rest = none ? 0.f : lp_rest - s.log_t_rest;
      if (p_rest != 0.f) kl += p_rest * f_rest;
      if (p_rest != 0.f) h = p_rest * (f_rest - kl);
    }
  }
  if (lane) return;
  const tb::Exponent ex(sum.m, k1);
  const float f = (listed ? w * h : 0.f) + (c != 0.f ? c * p_rest : 0.f);
  const float factor = !good ? NAN : none ? 0.f : f * inv_t / sum.s * ex.fix;
  s.n = {ex.m, factor, all.m, good ? lns : make_float2(NAN, NAN), kl, whole};
  if (!write) return;
  // (in 64 bits: with masked logits the two may be near fp32's end and cancel)
  const double from_list = listed ? static_cast<double>(w) * kl : 0.0;
  const double from_target = c != 0.f ? -static_cast<double>(c) * log_p(s.z_y, all.m, lns) : 0.0;
  a.loss[r] = good ? static_cast<float>(from_list + from_target) : NAN;
  if (a.kl) a.kl[r] = good || !listed ? kl : NAN;
  if (a.stats) {
    float4* st = reinterpret_cast<float4*>(a.stats + r * TB_DISTILL_STATS);
    st[0] = make_float4(s.n.origin, s.n.factor, s.n.top, s.n.lns.x);
    st[1] = make_float4(s.n.lns.y, s.n.kl, s.n.whole, s.mass);
    st[2] = make_float4(s.special ? 1.f : 0.f, 0.f, 0.f, 0.f);
  }
}

template <typename T, int MODE, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) distill_kernel(TbDistillArgs a, float k1, float inv_t, int part) {
  constexpr int E = Row<T>::E, kWarps = kThreads / 32, kStep = kLane * 32;
  extern __shared__ uint4 dynamic[];  // [part]: a byte for each vector of this CTA's part, its elements in the list
  unsigned char* bytes = reinterpret_cast<unsigned char*>(dynamic);
  __shared__ Shared s;
  cg::cluster_group cl = cg::this_cluster();
  const int rank = cl.block_rank(), ranks = cl.num_blocks();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, K = a.K;
  int live = 0;  // live rows so far
  for (long long r = blockIdx.x / ranks; r < a.R; r += gridDim.x / ranks) {
    const Row<T> row(static_cast<const T*>(a.logits) + r * a.ld, a.V, rank, ranks);
    T* grad = MODE == kLoss ? nullptr : static_cast<T*>(a.grad) + r * a.ld_grad;
    const bool same = MODE != kLoss && ((reinterpret_cast<uintptr_t>(grad) ^ reinterpret_cast<uintptr_t>(row.row)) & 15) == 0;
    {
      // ---- the weights, and a thread for each entry of the list (all asked for at once)
      int id = -1;
      float l = 0.f;
      if (tid < K) {
        id = a.ids[r * K + tid];
        l = a.logp[r * K + tid];
      }
      const Weights q(a, a.weight ? a.weight[r] : 1.f, a.target_weight ? a.target_weight[r] : 1.f, a.target ? a.target[r] : -1);
      if (MODE != kGrad && a.err && q.bad && tid == 0) *a.err = 1;
      if (!q.live()) {
        if (MODE != kGrad && rank == 0 && tid == 0) {
          a.loss[r] = 0.f;
          if (a.kl) a.kl[r] = 0.f;
        }
        if (MODE != kLoss) {
          for (int v = row.v0 + tid; v < row.v1; v += kThreads) {
            const int e = v * E - row.mis;
            if (same && row.inside(v, v + 1)) {
              __stcs(reinterpret_cast<uint4*>(grad + e), make_uint4(0, 0, 0, 0));
            } else {
              for (int j = max(0, -e); j < min(E, a.V - e); ++j) grad[e + j] = tb::from_f32<T>(0.f);
            }
          }
        }
        continue;
      }
      if (q.w == 0.f || id < 0 || l == -INFINITY) id = -1;
      if (id >= a.V) {
        if (MODE != kGrad && a.err) *a.err = 1;
        id = -1;
      }
      if (tid < kMaxList) {
        s.id[tid] = id;
        s.l[tid] = l;
        if (id >= 0) s.z[tid] = tb::to_f32(row.row[id]);
        s.t[tid] = id >= 0 ? exp(static_cast<double>(l)) : 0.0;
      }
      if (tid == 0) {
        s.w = q.w;
        s.c = q.c;
        s.y = q.y;
        s.z_y = q.y >= 0 ? tb::to_f32(row.row[q.y]) : 0.f;
      }
      if (MODE != kGrad)
        for (int i = tid; i < part; i += kThreads) dynamic[i] = make_uint4(0, 0, 0, 0);
      const int y_listed = __syncthreads_or(id >= 0 && id == q.y);
      if (tid == 0) s.y_listed = y_listed;
      // ---- an id that occurs twice counts once, with the sum of its masses; without the rest they
      // count relative to the largest where their sum may leave fp32's range (faint lists, scores)
      int seen = 0;
      if (MODE == kGrad) {
        seen = a.stats[r * TB_DISTILL_STATS + 8] != 0.f;
      } else if (id >= 0) {
        const int4* ids = reinterpret_cast<const int4*>(s.id);
#pragma unroll 4
        for (int j = 0; j < tid / 4; ++j) {
          const int4 x = ids[j];
          seen |= x.x == id || x.y == id || x.z == id || x.w == id;
        }
        for (int j = tid & ~3; j < tid; ++j) seen |= s.id[j] == id;
        const int v = (id + row.mis) / E - row.v0, b = (id + row.mis) % E;
        if (v >= 0 && v < row.v1 - row.v0) atomicOr(reinterpret_cast<uint32_t*>(bytes) + v / 4, 1u << (v % 4 * 8 + b));
      }
      const bool odd = a.kind == TB_DISTILL_FORWARD && id >= 0 && !(fabsf(l) <= kPlain);
      const int special = __syncthreads_or(seen || odd);
      if (tid == 0) s.special = special;
      if (special) {
        float largest = 0.f;
        if (a.kind == TB_DISTILL_FORWARD) {
          largest = -INFINITY;
          for (int j = lane; j < K; j += 32)
            if (s.id[j] >= 0) largest = fmaxf(largest, s.l[j]);
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, o));
        }
        if (!__syncthreads_or(seen)) {
          if (id >= 0) s.t[tid] = exp(static_cast<double>(l) - largest);
          l -= largest;
        } else if (id >= 0) {  // (the logarithm from the largest of its entries: the mass itself may be below 2^-1074)
          bool first = true;
          float top = l;
          for (int j = 0; j < K; ++j) {
            if (s.id[j] != id) continue;
            if (j < tid) first = false;
            top = fmaxf(top, s.l[j]);
          }
          double m = 0.0;
          for (int j = 0; j < K; ++j)
            if (s.id[j] == id) m += exp(static_cast<double>(s.l[j]) - top);
          s.t[tid] = first ? m * exp(static_cast<double>(top) - largest) : -1.0;
          l = static_cast<float>(static_cast<double>(top) - largest + log(m));
        }
        __syncthreads();
        if (id >= 0) s.l[tid] = l;
        __syncthreads();
      }
    }
    Numbers n;
    if (MODE != kGrad) {
      // ---- the pass over what is outside the list
      tb::RunningSum<T> running;
      const uint64_t again = MODE == kBoth ? tb::read_again() : tb::read_once();
      for (int v = row.v0 + warp * kStep; v < row.v1; v += kWarps * kStep) {
        uint4 p[kLane];
        row.template load_some<kLane>(v, p, again);
        uint32_t in[kLane], any = 0;
#pragma unroll
        for (int j = 0; j < kLane; ++j) {
          const int u = v + j * 32 + lane;
          in[j] = u < row.v1 ? bytes[u - row.v0] : 0;
          any |= in[j];
        }
        if (any) {
#pragma unroll
          for (int j = 0; j < kLane; ++j)
            if (in[j]) p[j] = tb::without<T>(p[j], in[j]);
        }
        typename Vec<T>::Max top = Vec<T>::top(p[0]);
#pragma unroll
        for (int j = 1; j < kLane; ++j) top = Vec<T>::max(top, Vec<T>::top(p[j]));
        running.add(p, Vec<T>::value(top), k1);
      }
      SoftSum sum = running.done(k1);
      sum.merge_lanes(k1);
      if (lane == 0) {
        s.part[0][warp] = sum.m;
        s.part[1][warp] = sum.s;
      }
      if (warp == kWarps - 1) list_sums(a, s, k1);  // (the warp with the fewest vectors)
      __syncthreads();
      if (warp == 0) {
        sum = SoftSum();
        if (lane < kWarps) {
          sum.m = s.part[0][lane];
          sum.s = s.part[1][lane];
        }
        sum.merge_lanes(k1);
      }
      if (ranks > 1) {
        if (tid == 0) {
          s.mine[live & 1][0] = sum.m;
          s.mine[live & 1][1] = sum.s;
        }
        cl.sync();
        if (warp == 0) {
          sum = SoftSum();
          if (lane < ranks) {
            const float* m = cl.map_shared_rank(s.mine[live & 1], lane);
            sum.m = m[0];
            sum.s = m[1];
          }
          sum.merge_lanes(k1);
        }
      }
      if (warp == 0) numbers_of(a, s, r, sum, k1, inv_t, rank == 0);
      __syncthreads();
      n = s.n;
    } else {
      const float4* st = reinterpret_cast<const float4*>(a.stats + r * TB_DISTILL_STATS);
      const float4 x = st[0], y = st[1];
      n = {x.x, x.y * a.dloss[r], x.z, make_float2(x.w, y.x), y.y, y.z};
      if (tid == 0) s.mass = y.w;
    }
    ++live;
    if (MODE != kLoss) {
      // ---- the gradient outside the list (in place: every element is read by its writer)
      const tb::Exponent ex(n.origin, k1);
      const float2 factor = make_float2(n.factor, n.factor);
      const uint64_t once = tb::read_once();
      for (int v = row.v0 + warp * kStep; v < row.v1; v += kWarps * kStep) {
        uint4 p[kLane];
        row.template load_some<kLane>(v, p, once);
        if (same && v + kStep <= row.v1 && row.inside(v, v + kStep)) {
#pragma unroll
          for (int j = 0; j < kLane; ++j)
            __stcs(reinterpret_cast<uint4*>(grad + (v + j * 32 + lane) * E - row.mis), tb::scaled_powers<T>(p[j], ex, factor));
        } else {
#pragma unroll
          for (int j = 0; j < kLane; ++j) {
            const int u = v + j * 32 + lane, e = u * E - row.mis;
            if (u >= row.v1) continue;
            union {
              uint4 q;
              T x[E];
            } x;
            x.q = tb::scaled_powers<T>(p[j], ex, factor);
            if (same && row.inside(u, u + 1)) {
              __stcs(reinterpret_cast<uint4*>(grad + e), x.q);
            } else {
#pragma unroll
              for (int b = 0; b < E; ++b)
                if (e + b >= 0 && e + b < a.V) grad[e + b] = x.x[b];
            }
          }
        }
      }
      __syncthreads();
      // ---- the list's elements, and the target
      const float scale = inv_t * (MODE == kGrad ? a.dloss[r] : 1.f), c = s.c;
      const int y = s.y;
      const auto mine = [&](int id) {
        const int v = (id + row.mis) / E;
        return v >= row.v0 && v < row.v1;
      };
      if (tid < K) {
        const int id = s.id[tid];
        const float t = static_cast<float>(s.t[tid]);
        if (id >= 0 && t >= 0.f && mine(id)) {
          const float lp = tb::Scaled{inv_t}(s.z[tid], n.top, n.lns), p = tb::ex2(lp * static_cast<float>(tb::kLog2e));
          float d;
          if (a.kind == TB_DISTILL_REVERSE) {
            d = p == 0.f ? 0.f : p * (lp - s.l[tid] - n.kl);
          } else {
            d = p * n.whole - (a.kind == TB_DISTILL_FORWARD ? (s.mass != 0.f ? t / s.mass : 0.f) : t);
          }
          d *= s.w;
          if (c != 0.f) d += c * (id == y ? p - 1.f : p);
          grad[id] = tb::from_f32<T>(d * scale);
        }
      }
      if (tid == 0 && c != 0.f && !s.y_listed && mine(y)) grad[y] = tb::from_f32<T>(ex.power(s.z_y) * n.factor - c * scale);
    }
    __syncthreads();
  }
  if (ranks > 1) cl.sync();  // the others have read this CTA's numbers
}

constexpr int kSms = 148;
constexpr int kPart = 32 * 1024;  // vectors of a part at most (of its bitmap, bytes)

// CTAs of a cluster: as many as half the machine holds beside the other rows (clusters that
// would fill it wait for one another: loss and gradient of 36 rows of 2,374 groups take 20.9 us
// with one CTA, 14.8 with four, 21.0 with eight; 4 rows 20.4, 12.3 and 9.3), some 100 groups at
// least to each (4 rows of 250 groups take 8.7 us with one and 9.1 with two, of 500 groups 10.7,
// and 8.8 with four); and enough of them that a part's bitmap fits its shared memory.
int ranks_of(int R, int groups, int slots) {
  int ranks = 1;
  while (ranks < 8 && ((groups + ranks - 1) / ranks * 8 > kPart || (R * 4ll * ranks <= slots && groups >= 128 * (ranks + 1)))) ranks *= 2;
  return ranks;
}

template <typename T, int MODE, int kThreads>
cudaError_t launch(const TbDistillArgs& a, int groups, cudaStream_t stream) {
  const int ranks = ranks_of(a.R, groups, kSms * (1024 / kThreads));
  const int part = MODE == kGrad ? 0 : ((groups + ranks - 1) / ranks * 8 + 15) / 16;
  cudaError_t e = tb::ensure_dyn_smem(reinterpret_cast<const void*>(&distill_kernel<T, MODE, kThreads>), 2 * kPart);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  const int rows = a.R < (1 << 20) ? a.R : 1 << 20;
  cfg.gridDim = dim3(static_cast<unsigned>(rows) * ranks);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(part) * 16;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, distill_kernel<T, MODE, kThreads>, a, static_cast<float>(tb::kLog2e / a.temperature),
                            static_cast<float>(1.0 / a.temperature), part);
}

// Both passes in one launch: the rows in work, read twice, have to fit the L2 cache beside
// what is written, so long rows get two CTAs of 512 threads on an SM instead of four of 256
// (all rows live, an empty L2 cache: 1,024 rows of 1,024 groups take 79 us with 512 threads and
// 71 with 256, of 1,536 groups 99 and 99, of 2,004 groups 124 and 130; 4,096 rows of 2,374
// groups 517 and 566).
template <typename T>
cudaError_t launch_mode(const TbDistillArgs& a, cudaStream_t s) {
  constexpr int E = Row<T>::E;
  const int groups = (a.V + E - 2 + 8 * E) / (8 * E);
  if (!a.loss) return launch<T, kGrad, 256>(a, groups, s);
  if (!a.grad) return launch<T, kLoss, 256>(a, groups, s);
  return groups > 1536 ? launch<T, kBoth, 512>(a, groups, s) : launch<T, kBoth, 256>(a, groups, s);
}

}  // namespace

extern "C" int tb_distill(const TbDistillArgs* args, cudaStream_t s) {
  const TbDistillArgs& a = *args;
  if (a.R < 0 || a.V < 1 || a.V > 1 << 20 || a.K < 1 || a.K > kMaxList || (!a.loss && (!a.grad || !a.stats || !a.dloss)))
    return static_cast<int>(cudaErrorInvalidValue);
  if (a.R == 0) return 0;
  switch (a.dtype) {
    case TB_BF16: return static_cast<int>(launch_mode<__nv_bfloat16>(a, s));
    case TB_F16: return static_cast<int>(launch_mode<__half>(a, s));
    case TB_F32: return static_cast<int>(launch_mode<float>(a, s));
    default: return static_cast<int>(cudaErrorInvalidValue);
  }
}
