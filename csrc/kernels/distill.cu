// The distillation loss of rows of logits against a teacher's list, and its gradient.
//
// For a row z, its list (a_k, l_k) with the set S of its ids, t_k = exp(l_k), and
// p = softmax(z / T), the row's loss is w KL + c (-log p_y), with
//
//   forward:        KL = sum_S t (log t - log p),                 T dKL/dz_j = p_j - t_j
//                   (t divided by its sum)
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
// elements of S join afterwards, a thread to each.  A second pass writes the gradient, then
// the elements of S are written over.  Numbers of the row (logarithms, t_R, KL) are formed
// in 64 bits: the loss is a small difference of large ones.
#include "kernels.h"
#include "vocab_rows.cuh"

namespace {

namespace cg = cooperative_groups;
using tb::Row;
using tb::SoftSum;
using tb::Vec;

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMaxList = kThreads;  // a thread for each entry
constexpr int kSlots = 148 * 4;  // CTAs that the machine holds
constexpr double kRestMin = 1.0 / (1 << 20);
enum { kLoss, kBoth, kGrad };  // what a launch computes (kGrad: from the numbers that kLoss kept)

struct Shared {
  float part[4][kWarps];
  double mass[kWarps], term[kWarps];
  float mine[2];
  int twice;     // an id of this CTA's part occurs twice in the list
  int y_listed;  // the target is in the list
  int id[kMaxList];
  float l[kMaxList];
};

// What a row's passes share, the same in all threads.
struct Numbers {
  float origin, factor;  // the gradient outside the list: factor x 2^((z - origin) k1)
  float top, lns;        // log p = (z - top) / T - lns
  float kl, whole;       // whole: sum t + t_R
  float mass;            // sum t as listed
};

// The entry of a list that a thread has.
struct Entry {
  int id = -1;  // -1: padding, or not the id's first entry
  float z = 0.f, l = 0.f;
  double t = 0.0, lt = 0.0;  // mass of the class, and its logarithm
};

template <typename T, int MODE>
__global__ void __launch_bounds__(kThreads, 4) distill_kernel(TbDistillArgs a, float k1, double inv_t, int part) {
  constexpr int E = Row<T>::E;
  extern __shared__ uint4 dynamic[];  // [part]: a byte for each vector of this CTA's part, its elements in the list
  unsigned char* bytes = reinterpret_cast<unsigned char*>(dynamic);
  uint32_t* bits = reinterpret_cast<uint32_t*>(dynamic);
  __shared__ Shared s;
  cg::cluster_group cl = cg::this_cluster();
  const int rank = cl.block_rank(), ranks = cl.num_blocks();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, K = a.K;
  for (long long r = blockIdx.x / ranks; r < a.R; r += gridDim.x / ranks) {
    const Row<T> row(static_cast<const T*>(a.logits) + r * a.ld, a.V, rank, ranks);
    T* grad = MODE == kLoss ? nullptr : static_cast<T*>(a.grad) + r * a.ld_grad;
    const bool same = MODE != kLoss && ((reinterpret_cast<uintptr_t>(grad) ^ reinterpret_cast<uintptr_t>(row.row)) & 15) == 0;
    // ---- the weights, and the thread's entry of the list
    const float w = a.weight ? a.weight[r] : 1.f;
    int y = a.target ? a.target[r] : -1;
    float c = y < 0 ? 0.f : a.target_weight ? a.target_weight[r] : 1.f;
    Entry mine;
    if (tid < K) {
      mine.id = a.ids[r * K + tid];
      mine.l = a.logp[r * K + tid];
    }
    if (y >= a.V) {
      if (MODE != kGrad && a.err && tid == 0 && (c != 0.f || w != 0.f)) *a.err = 1;
      y = -1;
      c = 0.f;
    }
    const bool live = w != 0.f || c != 0.f, listed = w != 0.f;
    if (!live) {
      if (MODE != kGrad && rank == 0 && tid == 0) a.loss[r] = 0.f;
      if (MODE != kLoss) {
        for (int v = row.v0 + tid; v < row.v1; v += kThreads) {
          const int e = v * E - row.mis;
          if (same && row.inside(v, v + 1)) {
            *reinterpret_cast<uint4*>(grad + e) = make_uint4(0, 0, 0, 0);
          } else {
            for (int j = max(0, -e); j < min(E, a.V - e); ++j) grad[e + j] = tb::from_f32<T>(0.f);
          }
        }
      }
      continue;
    }
    if (!listed || mine.l == -INFINITY || mine.id < 0) mine.id = -1;
    if (mine.id >= a.V) {
      if (MODE != kGrad && a.err) *a.err = 1;
      mine.id = -1;
    }
    if (mine.id >= 0) {
      mine.z = tb::to_f32(row.row[mine.id]);
      mine.t = exp(static_cast<double>(mine.l));
      mine.lt = mine.l;
    }
    float z_y = 0.f;
    if (tid == 0 && y >= 0) z_y = tb::to_f32(row.row[y]);
    const int at = mine.id + row.mis;  // the entry's place among this CTA's vectors
    const bool here = mine.id >= 0 && at / E >= row.v0 && at / E < row.v1;
    s.id[tid] = mine.id;
    s.l[tid] = mine.l;
    if (tid == 0) s.twice = s.y_listed = 0;
    // an id that occurs twice counts once, with the sum of its masses
    const auto unite = [&] {
      if (mine.id < 0) return;
      bool first = true;
      double t = 0.0;
      for (int j = 0; j < K; ++j) {
        if (s.id[j] != mine.id) continue;
        if (j < tid) first = false;
        t += exp(static_cast<double>(s.l[j]));
      }
      mine.t = t;
      mine.lt = log(t);
      if (!first) mine.id = -1;
    };
    Numbers n;
    if (MODE != kGrad) {
      for (int i = tid; i < part; i += kThreads) dynamic[i] = make_uint4(0, 0, 0, 0);
      __syncthreads();
      const uint32_t bit = here ? 1u << ((at / E - row.v0) % 4 * 8 + at % E) : 0;
      uint32_t* word = bits + (here ? (at / E - row.v0) / 4 : 0);
      if (here && atomicOr(word, bit) & bit) s.twice = 1;
      if (mine.id >= 0 && mine.id == y) s.y_listed = 1;
      __syncthreads();
      // ---- the pass over what is outside the list
      tb::RunningSum<T> running;
      for (int v = row.v0 + warp * tb::kChunk; v < row.v1; v += kWarps * tb::kChunk) {
        uint4 p[8];
        row.load_chunk(v, p);
        uint32_t in[8], any = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int j = v + i * 32 + lane;
          in[i] = j < row.v1 ? bytes[j - row.v0] : 0;
          any |= in[i];
        }
        if (any) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (in[i]) p[i] = tb::without<T>(p[i], in[i]);
        }
        typename Vec<T>::Max top = Vec<T>::top(p[0]);
#pragma unroll
        for (int i = 1; i < 8; ++i) top = Vec<T>::max(top, Vec<T>::top(p[i]));
        running.add(p, Vec<T>::value(top), k1);
      }
      // ---- sums over the block: outside the list, the list's first entries, the masses
      SoftSum sum = running.done(k1), in;
      if (mine.id >= 0 && !s.twice) {
        in.m = mine.z;
        in.s = isnan(mine.z) ? NAN : 1.f;
        if (isnan(mine.z)) in.m = -INFINITY;
      }
      sum.merge_lanes(k1);
      in.merge_lanes(k1);
      const double mass_w = tb::warp_sum(mine.id >= 0 ? mine.t : 0.0);
      if (lane == 0) {
        s.part[0][warp] = sum.m;
        s.part[1][warp] = sum.s;
        s.part[2][warp] = in.m;
        s.part[3][warp] = in.s;
        s.mass[warp] = mass_w;
      }
      __syncthreads();
      sum = in = SoftSum();
      double mass = 0.0;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) {
        sum.merge(s.part[0][i], s.part[1][i], k1);
        in.merge(s.part[2][i], s.part[3][i], k1);
        mass += s.mass[i];
      }
      int twice = s.twice;
      if (ranks > 1) {
        if (tid == 0) {
          s.mine[0] = sum.m;
          s.mine[1] = sum.s;
        }
        cl.sync();
        sum = SoftSum();
        twice = 0;
        for (int o = 0; o < ranks; ++o) {
          const float* m = cl.map_shared_rank(s.mine, o);
          sum.merge(m[0], m[1], k1);
          twice |= *cl.map_shared_rank(&s.twice, o);
        }
      }
      if (twice) {  // (the same in the whole cluster)
        unite();
        in = SoftSum();
        if (mine.id >= 0) {
          in.m = isnan(mine.z) ? -INFINITY : mine.z;
          in.s = isnan(mine.z) ? NAN : 1.f;
        }
        in.merge_lanes(k1);
        __syncthreads();
        if (lane == 0) {
          s.part[2][warp] = in.m;
          s.part[3][warp] = in.s;
        }
        __syncthreads();
        in = SoftSum();
        for (int i = 0; i < kWarps; ++i) in.merge(s.part[2][i], s.part[3][i], k1);
      }
      if (a.kind == TB_DISTILL_FORWARD) {
        mine.t = mass != 0.0 ? mine.t / mass : 0.0;
        mine.lt -= log(mass);
      }
      // ---- the whole row
      SoftSum all = sum;
      all.merge(in.m, in.s, k1);
      const bool good = !isnan(all.s) && !isinf(all.m);
      const double lns = good ? tb::log_of(all.s) : 0.0;
      // log p of the elements outside; none there: their terms are left out
      const bool none = sum.m == -INFINITY || !good;
      const double lp_rest = none ? 0.0 : (static_cast<double>(sum.m) - all.m) * inv_t + tb::log_of(sum.s) - lns;
      const double p_rest = none ? 0.0 : tb::exp_of(lp_rest);
      const double t_rest = 1.0 - mass;
      double kl = 0.0, h = 0.0;  // h: factor of q_j outside the list
      n.whole = 1.f;
      if (listed) {
        double term = 0.0;
        if (mine.id >= 0) {
          const double lp = (static_cast<double>(mine.z) - all.m) * inv_t - lns;
          if (a.kind == TB_DISTILL_REVERSE) {
            const float p = tb::exp_of(lp);
            if (p != 0.f) term = p * (lp - mine.lt);
          } else if (mine.t != 0.0) {
            term = mine.t * (mine.lt - lp);
          }
        }
        term = tb::warp_sum(term);
        if (lane == 0) s.term[warp] = term;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kWarps; ++i) kl += s.term[i];
        if (a.kind == TB_DISTILL_FORWARD) {
          n.whole = mass != 0.0 ? 1.f : 0.f;
          h = n.whole * p_rest;
        } else if (a.kind == TB_DISTILL_FORWARD_REST) {
          const double t_out = none ? 0.0 : fmax(t_rest, 0.0);
          if (t_out > 0.0) kl += t_out * (log(t_out) - lp_rest);
          n.whole = static_cast<float>(mass + t_out);
          h = (mass + t_out) * p_rest - t_out;
        } else {
          const double f_rest = none ? 0.0 : lp_rest - log(fmax(t_rest, kRestMin));
          kl += p_rest * f_rest;
          h = p_rest * (f_rest - kl);
        }
      }
      if (rank == 0 && tid == 0) {
        const double ce = lns - (static_cast<double>(z_y) - all.m) * inv_t;
        a.loss[r] = good ? static_cast<float>((listed ? w * kl : 0.0) + (c != 0.f ? c * ce : 0.0)) : NAN;
      }
      const tb::Exponent ex(sum.m, k1);
      const double f = (listed ? w * h : 0.0) + (c != 0.f ? c * p_rest : 0.0);
      n.origin = ex.m;
      n.factor = !good ? NAN : none ? 0.f : static_cast<float>(f * inv_t / sum.s * ex.fix);
      n.top = all.m;
      n.lns = good ? static_cast<float>(lns) : NAN;
      n.kl = static_cast<float>(kl);
      n.mass = static_cast<float>(mass);
      if (MODE == kLoss && a.stats && rank == 0 && tid == 0) {
        float4* st = reinterpret_cast<float4*>(a.stats + r * TB_DISTILL_STATS);
        st[0] = make_float4(n.origin, n.factor, n.top, n.lns);
        st[1] = make_float4(n.kl, n.whole, n.mass, twice ? 1.f : 0.f);
      }
    } else {
      const float4* st = reinterpret_cast<const float4*>(a.stats + r * TB_DISTILL_STATS);
      const float4 x = st[0], z = st[1];
      const float g = a.dloss[r];
      n = {x.x, x.y * g, x.z, x.w, z.x, z.y, z.z};
      __syncthreads();
      if (mine.id >= 0 && mine.id == y) s.y_listed = 1;
      if (z.w != 0.f) unite();
      if (a.kind == TB_DISTILL_FORWARD) mine.t = n.mass != 0.f ? mine.t / n.mass : 0.0;
    }
    if (MODE != kLoss) {
      // ---- the gradient outside the list (in place: every element is read by its writer)
      const tb::Exponent ex(n.origin, k1);
      const float2 factor = make_float2(n.factor, n.factor);
      for (int v = row.v0 + warp * tb::kChunk; v < row.v1; v += kWarps * tb::kChunk) {
        uint4 p[8];
        row.load_chunk(v, p);
        if (same && v + tb::kChunk <= row.v1 && row.inside(v, v + tb::kChunk)) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            *reinterpret_cast<uint4*>(grad + (v + i * 32 + lane) * E - row.mis) = tb::scaled_powers<T>(p[i], ex, factor);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int j = v + i * 32 + lane, e = j * E - row.mis;
            if (j >= row.v1) continue;
            union {
              uint4 q;
              T x[E];
            } u;
            u.q = tb::scaled_powers<T>(p[i], ex, factor);
            if (same && row.inside(j, j + 1)) {
              *reinterpret_cast<uint4*>(grad + e) = u.q;
            } else {
#pragma unroll
              for (int q = 0; q < E; ++q)
                if (e + q >= 0 && e + q < a.V) grad[e + q] = u.x[q];
            }
          }
        }
      }
      __syncthreads();
      // ---- the list's elements, and the target
      const float scale = static_cast<float>(inv_t) * (MODE == kGrad ? a.dloss[r] : 1.f);
      if (mine.id >= 0 && here) {
        const double lp = (static_cast<double>(mine.z) - n.top) * inv_t - n.lns;
        const float p = isnan(lp) ? NAN : tb::exp_of(lp), t = static_cast<float>(mine.t);
        float d = p * n.whole - t;
        if (a.kind == TB_DISTILL_REVERSE)
          d = p == 0.f ? 0.f : p * static_cast<float>(lp - mine.lt - n.kl);
        d *= w;
        if (c != 0.f) d += c * (mine.id == y ? p - 1.f : p);
        grad[mine.id] = tb::from_f32<T>(d * scale);
      }
      const int vy = (y + row.mis) / E;
      if (tid == 0 && c != 0.f && !s.y_listed && vy >= row.v0 && vy < row.v1)
        grad[y] = tb::from_f32<T>(ex.power(z_y) * n.factor - c * scale);
    }
    if (ranks > 1) {
      cl.sync();
    } else {
      __syncthreads();
    }
  }
}

// CTAs of a cluster: as many as the machine has room for beside the other rows, a chunk at
// least to each; enough of them that a part's bitmap fits its shared memory; and, where rows
// are read twice, that the rows in work fit the L2 cache beside what is written.
int ranks_of(int R, int groups, bool twice) {
  const auto more = [&](int ranks) {
    if ((groups + ranks - 1) / ranks > 4096) return true;
    if (groups < 64 * ranks) return false;
    return R * 2ll * ranks <= kSlots || (twice && static_cast<long long>(min(R, kSlots / ranks)) * groups * 128 > (48 << 20));
  };
  int ranks = 1;
  while (ranks < 8 && more(ranks)) ranks *= 2;
  return ranks;
}

template <typename T, int MODE>
cudaError_t launch(const TbDistillArgs& a, cudaStream_t stream) {
  constexpr int E = Row<T>::E;
  const int groups = (a.V + E - 2 + 8 * E) / (8 * E);
  const int ranks = ranks_of(a.R, groups, MODE == kBoth);
  const size_t smem = MODE == kGrad ? 0 : (static_cast<size_t>((groups + ranks - 1) / ranks) * 8 + 15) / 16 * 16;
  cudaError_t e = tb::ensure_dyn_smem(reinterpret_cast<const void*>(&distill_kernel<T, MODE>), 64 * 1024);
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
  return cudaLaunchKernelEx(&cfg, distill_kernel<T, MODE>, a, static_cast<float>(tb::kLog2e / a.temperature),
                            1.0 / a.temperature, static_cast<int>(smem / 16));
}

template <typename T>
cudaError_t launch_mode(const TbDistillArgs& a, cudaStream_t s) {
  if (!a.loss) return launch<T, kGrad>(a, s);
  return a.grad ? launch<T, kBoth>(a, s) : launch<T, kLoss>(a, s);
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
