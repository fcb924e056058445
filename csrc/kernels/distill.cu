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
// elements of S join afterwards.  A second pass writes the gradient, then the elements of
// S are written over.  Numbers of the row (logarithms, t_R, KL) are formed in 64 bits:
// the loss is a small difference of large ones.
#include "kernels.h"
#include "vocab_rows.cuh"

namespace {

namespace cg = cooperative_groups;
using tb::Row;
using tb::SoftSum;

constexpr int kMaxList = 256;
constexpr int kThreads = 512;
constexpr double kRestMin = 1.0 / (1 << 20);
enum { kLoss, kBoth, kGrad };  // what a launch computes (kGrad: from the numbers that kLoss kept)

struct Shared {
  float merge[64];
  float mine[2];
  double sums[32];
  int id[kMaxList];      // -1: padding
  float z[kMaxList];     // the student's logits
  float l[kMaxList];     // the teacher's log-probabilities
  float mass[kMaxList];  // t of the class, 0 for the later ones of an id that occurs twice
  int first[kMaxList];   // whether this is the id's first entry
  // numbers of the row
  double t_total, lns;
  float m_all, z_y;
  int y_listed;
};

__device__ double block_sum_d(double v, double* buf) { return tb::block_sum(v, buf); }

template <typename T, int E>
__device__ __forceinline__ void store_row(T* p, const float (&x)[E], int first, int last, bool vec) {
  // elements first .. last - 1 of a vector whose first element is p[0]
  if (vec) {
    tb::store_vec<T, E>(p, x);
  } else {
#pragma unroll
    for (int j = 0; j < E; ++j)
      if (j >= first && j < last) p[j] = tb::from_f32<T>(x[j]);
  }
}

template <typename T, int MODE>
__global__ void __launch_bounds__(kThreads, 2) distill_kernel(TbDistillArgs a, float k1) {
  constexpr int E = Row<T>::E;
  extern __shared__ uint32_t bits[];  // a byte for each vector of this CTA's part
  __shared__ Shared s;
  cg::cluster_group cl = cg::this_cluster();
  const int rank = cl.block_rank(), ranks = cl.num_blocks();
  const int tid = threadIdx.x, K = a.K;
  const double inv_t = 1.0 / a.temperature;
  const unsigned char* bytes = reinterpret_cast<const unsigned char*>(bits);
  for (long long r = blockIdx.x / ranks; r < a.R; r += gridDim.x / ranks) {
    const Row<T> row(static_cast<const T*>(a.logits) + r * a.ld, a.V, rank, ranks);
    T* grad = MODE == kLoss ? nullptr : static_cast<T*>(a.grad) + r * a.ld_grad;
    const float w = a.weight ? a.weight[r] : 1.f;
    int y = a.target ? a.target[r] : -1;
    float c = y < 0 ? 0.f : a.target_weight ? a.target_weight[r] : 1.f;
    if (y >= a.V) {
      if (a.err && tid == 0 && (c != 0.f || w != 0.f)) *a.err = 1;
      y = -1;
      c = 0.f;
    }
    const float g = MODE == kGrad ? a.dloss[r] : 1.f;
    const bool live = w != 0.f || c != 0.f, listed = w != 0.f;
    const bool same = MODE != kLoss && ((reinterpret_cast<uintptr_t>(grad) ^ reinterpret_cast<uintptr_t>(row.row)) & 15) == 0;
    float factor = 0.f, origin = 0.f, coef[2] = {0.f, 0.f}, whole = 1.f;
    double kl = 0.0;
    if (live) {
      // ---- the list
      const int words = (row.v1 - row.v0 + 3) / 4;
      for (int i = tid; i < words; i += kThreads) bits[i] = 0;
      if (tid == 0) s.y_listed = 0;
      __syncthreads();
      double mass = 0.0;
      if (listed) {
        for (int k = tid; k < K; k += kThreads) {
          int id = a.ids[r * K + k];
          const float l = a.logp[r * K + k];
          if (id < 0 || l == -INFINITY) id = -1;
          if (id >= a.V) {
            if (a.err) *a.err = 1;
            id = -1;
          }
          s.id[k] = id;
          s.l[k] = l;
          if (id >= 0) {
            s.z[k] = tb::to_f32(row.row[id]);
            mass += exp(static_cast<double>(l));
            const int v = (id + row.mis) / E - row.v0, b = (id + row.mis) % E;
            if (v >= 0 && v < row.v1 - row.v0) atomicOr(&bits[v / 4], 1u << (v % 4 * 8 + b));
            if (id == y) s.y_listed = 1;
          }
        }
        mass = block_sum_d(mass, s.sums);  // (synchronises)
        for (int k = tid; k < K; k += kThreads) {
          // an id that occurs twice counts once, with the sum of its masses
          const int id = s.id[k];
          int first = id >= 0;
          double t = 0.0;
          for (int j = 0; j < K; ++j) {
            if (s.id[j] != id) continue;
            if (j < k) first = 0;
            t += exp(static_cast<double>(s.l[j]));
          }
          s.first[k] = first;
          if (a.kind == TB_DISTILL_FORWARD) t = mass != 0.0 ? t / mass : 0.0;
          s.mass[k] = first ? static_cast<float>(t) : 0.f;
        }
      }
      if (tid == 0) s.z_y = y >= 0 ? tb::to_f32(row.row[y]) : 0.f;
      __syncthreads();
      const double t_rest = 1.0 - mass;
      float* st = a.stats ? a.stats + r * TB_DISTILL_STATS : nullptr;
      if (MODE != kGrad) {
        // ---- the pass over what is outside the list
        SoftSum sum;
        for (int v = row.v0 + tid; v < row.v1; v += kThreads) {
          float x[E];
          row.load(v, x);
          const int b = bytes[v - row.v0];
          if (b) {
#pragma unroll
            for (int j = 0; j < E; ++j)
              if (b >> j & 1) x[j] = -INFINITY;
          }
          float top = x[0];
#pragma unroll
          for (int j = 1; j < E; ++j) top = fmaxf(top, x[j]);
          sum.add(x, top, k1);
        }
        sum = tb::block_merge(sum, k1, s.merge);
        sum = tb::cluster_merge(sum, k1, s.mine);
        // ---- the whole row
        SoftSum in;
        if (listed)
          for (int k = tid; k < K; k += kThreads)
            if (s.first[k]) {
              const float z[1] = {s.z[k]};
              in.add(z, z[0], k1);
            }
        in = tb::block_merge(in, k1, s.merge);
        SoftSum all = sum;
        all.merge(in.m, in.s, k1);
        if (tid == 0) s.lns = log(static_cast<double>(all.s));
        __syncthreads();
        const double lns = s.lns;
        // log p of the elements outside; none there: their terms are left out
        const bool none = sum.m == -INFINITY && !isnan(sum.s);
        const double lp_rest = none ? 0.0 : (static_cast<double>(sum.m) - all.m) * inv_t + log(static_cast<double>(sum.s)) - lns;
        const double p_rest = none ? 0.0 : exp(lp_rest);
        double h = 0.0, f_rest = 0.0;  // factor of q_j (forward) or of p_j (reverse) outside the list
        if (listed) {
          double term = 0.0;
          for (int k = tid; k < K; k += kThreads) {
            if (!s.first[k]) continue;
            const double lp = (static_cast<double>(s.z[k]) - all.m) * inv_t - lns, t = s.mass[k];
            if (a.kind == TB_DISTILL_REVERSE) {
              const double p = exp(lp);
              term += p == 0.0 ? 0.0 : p * (lp - log(t));
            } else if (t != 0.0) {
              term += t * (log(t) - lp);
            }
          }
          kl = block_sum_d(term, s.sums);
          if (a.kind == TB_DISTILL_FORWARD) {
            whole = mass != 0.0 ? 1.f : 0.f;
            h = whole * p_rest;
          } else if (a.kind == TB_DISTILL_FORWARD_REST) {
            if (t_rest > 0.0 && !none) kl += t_rest * (log(t_rest) - lp_rest);
            const double t_out = none ? 0.0 : fmax(t_rest, 0.0);
            whole = static_cast<float>(mass + t_out);
            h = (mass + t_out) * p_rest - t_out;
          } else {
            f_rest = none ? 0.0 : lp_rest - log(fmax(t_rest, kRestMin));
            kl += p_rest * f_rest;
            h = p_rest * (f_rest - kl);
          }
          if (isnan(all.s) || isinf(all.m)) kl = NAN;
        }
        double ce = 0.0;
        if (c != 0.f) ce = lns - (static_cast<double>(s.z_y) - all.m) * inv_t;
        if (a.loss && rank == 0 && tid == 0)
          a.loss[r] = static_cast<float>((listed ? w * kl : 0.0) + (c != 0.f ? c * ce : 0.0));
        origin = SoftSum::origin(sum.m);
        double f = (listed ? w * h : 0.0) + (c != 0.f ? c * p_rest : 0.0);
        f = none ? 0.0 : f * inv_t / sum.s;
        if (isnan(all.s) || isinf(all.m)) f = NAN;
        factor = static_cast<float>(f);
        coef[0] = all.m;
        coef[1] = static_cast<float>(lns);
        if (MODE == kLoss && st && rank == 0 && tid == 0) {
          st[0] = origin;
          st[1] = factor;
          st[2] = coef[0];
          st[3] = coef[1];
          st[4] = static_cast<float>(kl);
          st[5] = whole;
        }
      } else {
        origin = st[0];
        factor = st[1] * g;
        coef[0] = st[2];
        coef[1] = st[3];
        kl = st[4];
        whole = st[5];
      }
    } else if (MODE != kGrad && a.loss && rank == 0 && tid == 0) {
      a.loss[r] = 0.f;
    }
    if (MODE != kLoss) {
      // ---- the gradient outside the list (in place: every element is read by its writer)
      for (int v = row.v0 + tid; v < row.v1; v += kThreads) {
        float x[E];
        if (live) {
          row.load(v, x);
#pragma unroll
          for (int j = 0; j < E; ++j) x[j] = tb::ex2((x[j] - origin) * k1) * factor;
        } else {
#pragma unroll
          for (int j = 0; j < E; ++j) x[j] = 0.f;
        }
        const int e = v * E - row.mis;
        store_row<T, E>(grad + e, x, -e, a.V - e, same && row.inside(v, v + 1));
      }
      __syncthreads();
      if (live) {
        // ---- the list's elements, and the target
        const float scale = static_cast<float>(inv_t) * g;
        const auto mine = [&](int id) {
          const int v = (id + row.mis) / E;
          return v >= row.v0 && v < row.v1;
        };
        const auto p_of = [&](float z) {
          return static_cast<float>(exp((static_cast<double>(z) - coef[0]) * inv_t - coef[1]));
        };
        if (listed)
          for (int k = tid; k < K; k += kThreads) {
            if (!s.first[k] || !mine(s.id[k])) continue;
            const float p = p_of(s.z[k]), t = s.mass[k];
            float d = p * whole - t;
            if (a.kind == TB_DISTILL_REVERSE)
              d = p == 0.f ? 0.f : p * static_cast<float>((static_cast<double>(s.z[k]) - coef[0]) * inv_t - coef[1] - log(static_cast<double>(t)) - kl);
            d *= w;
            if (c != 0.f) d += c * (s.id[k] == y ? p - 1.f : p);
            grad[s.id[k]] = tb::from_f32<T>(d * scale);
          }
        if (tid == 0 && c != 0.f && !s.y_listed && mine(y))
          grad[y] = tb::from_f32<T>(tb::ex2((s.z_y - origin) * k1) * factor - c * scale);
      }
    }
    if (ranks > 1) {
      cl.sync();
    } else {
      __syncthreads();
    }
  }
}

template <typename T, int MODE>
cudaError_t launch(const TbDistillArgs& a, cudaStream_t stream) {
  constexpr int E = Row<T>::E;
  const int groups = (a.V + E - 2 + 8 * E) / (8 * E);
  int ranks = 1;
  while (ranks < 8 && (groups + ranks - 1) / ranks * 8 > 65536) ranks *= 2;
  const size_t smem = static_cast<size_t>((groups + ranks - 1) / ranks) * 8;
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
  return cudaLaunchKernelEx(&cfg, distill_kernel<T, MODE>, a, static_cast<float>(tb::kLog2e / a.temperature));
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
