// GroupNorm + activation (+ dropout) on channels-last rows, forward and backward, bf16 / f16 / f32.
//
//   m = mean x, v = mean (x - m)^2 over the hw rows and C / G channels of one (image, level, group)
//   t = (x - m) / sqrt(v + eps) * gamma_c + beta_c,   y = act(t) * keep / (1 - p)
//   d = dy * keep / (1 - p) * act'(t);  dbeta_c = sum d;  dgamma_c = sum d xhat;
//   dx = rstd (d gamma_c - mean(d gamma) - xhat mean(d gamma xhat))
//
// Everything here is bound by memory: forward reads x twice (the second time mostly out of the 256 MB memory-side cache) and writes y
// once, backward reads x and dy twice and writes dx.  A channels-last row is C * e contiguous bytes, so a block takes a tile of columns
// (8 channels = one thread's 16-byte access) and strides over rows; a group's sum is then spread over every block of its (image,
// level).  The blocks leave partial sums in the workspace and the next launch adds them in a fixed order: no atomics, so the result
// does not depend on which block came first, and there is nothing to clear between the replays of a captured graph.
//
// Maps of a few hundred rows take one launch instead (ga_small_*): a block holds all rows of its columns in registers, reads x (and dy)
// once and needs no partials -- there the launches, not the bytes, are the time.  Of many such maps a block takes several (ga_many_*).
//
// Measured (a copy of 2 GiB runs at 4.9 TB/s here):
//   89 600 x 256 bf16 rows of five levels, ReLU, p = 0.1: forward 40 us (sums 15, apply 26), backward 65 (sums 34, apply 32); without
//     dropout 38 and 56.  The rows are 46 MB, so a pass over them is 9 us; what is over that is latency at 1.4 blocks per CU (more row
//     blocks cost more in partials than they hide) and the generator (9 us of the two backward launches).
//   295 936 x 256 bf16, SiLU (151 MB, behind the memory-side cache): forward 85 us = 5.3 TB/s over its three passes, backward 158 =
//     4.8 TB/s over five: bandwidth.
//   77 x 256 f16, SiLU: one launch, 8 us, of which the loads are less than 2: the two reductions.
//
// The sums are held in f64: x and x^2 add exactly enough that E[x^2] - m^2 keeps its digits for |m| >> sqrt(v) (1e4 standard deviations
// cost 1e-8), and three f64 operations per element stay under the memory time for 16-bit rows.
#include <algorithm>

#include "common.h"
#include "elem.h"
#include "philox.h"

namespace {

constexpr int GA_THREADS = 256;     // element-wise launches
constexpr int GA_STAT = 1024;       // threads of the forward's reduction: few blocks with many waves, so that few partials are left
constexpr int GA_STAT1 = 256;       // ... where a vector spans groups (16 sums a thread)
constexpr int GA_SUM = 512;         // threads of the backward's reduction
constexpr int GA_COMBINE = 1024;    // partials that an element-wise block has to add up (16 KB out of L2), see ga_plan
constexpr int GA_TILE = 32;         // column vectors per block: 512-byte row segments for 16-bit types
constexpr int GA_TILE1 = 64;        // columns per block of the any-alignment path

struct GaArgs {
  int nlev, batch, C, G, cpg, act;
  int cols, ct, ntile;              // column vectors, per block, column tiles
  long long hw[SM_MAX_LEVELS], row0[SM_MAX_LEVELS];
  int sblk0[SM_MAX_LEVELS + 1];     // reductions: first row block of each level (per image)
  int ablk0[SM_MAX_LEVELS + 1];     // element-wise launches
  int srpb, arpb;                   // rows per block
  long long ldx, ldy, lddx;         // row strides in elements: x and dy, y, dx
  long long lddy;
  float eps;
  DropArgs drop;
};

__device__ __forceinline__ int ga_level(const int* blk0, int nlev, int b) {
  int lev = 0;
#pragma unroll
  for (int l = 1; l < SM_MAX_LEVELS; ++l)
    if (l < nlev && b >= blk0[l]) lev = l;
  return lev;
}

// sum over the block's row lanes of NV values per thread, left in sh[k][column] (fixed tree)
template <int NV, int NT, typename V>
__device__ __forceinline__ void lane_tree(V (*sh)[NT], const V* v, int lane, int ct, int lanes) {
  const int t = threadIdx.x;
#pragma unroll
  for (int k = 0; k < NV; ++k) sh[k][t] = v[k];
  __syncthreads();
  int top = 1;
  while (top < lanes) top <<= 1;
  for (int st = top >> 1; st > 0; st >>= 1) {
    if (lane < st && lane + st < lanes) {
#pragma unroll
      for (int k = 0; k < NV; ++k) sh[k][t] += sh[k][t + st * ct];
    }
    __syncthreads();
  }
}

// what a block works on: image, level and rows [rb, re) of it
struct GaBlock {
  int n, b, lev;
  long long rb, re;
};
__device__ __forceinline__ GaBlock ga_block(const GaArgs& a, const int* blk0, int rpb, int block) {
  GaBlock k;
  const int nblk = blk0[a.nlev];
  k.n = block / nblk, k.b = block - k.n * nblk;
  k.lev = ga_level(blk0, a.nlev, k.b);
  k.rb = (long long)(k.b - blk0[k.lev]) * rpb;
  k.re = min(k.rb + (long long)rpb, a.hw[k.lev]);
  return k;
}

// launch 1, forward: part[image][row block][tile][group - first group of the tile] = (sum x, sum x^2)
// WHOLE: a vector lies in one group (cpg % VEC == 0), so a thread needs two sums instead of 2 * VEC
template <int DT, int VEC, bool WHOLE>
__global__ __launch_bounds__(WHOLE ? GA_STAT : GA_STAT1) void ga_stats_kernel(const typename Elem<DT>::type* __restrict__ x, double2* __restrict__ part,
                                                              const GaArgs a, int gpt) {
  typedef RowVec<DT, VEC> RV;
  constexpr int NS = WHOLE ? 1 : VEC, NT = WHOLE ? GA_STAT : GA_STAT1;
  __shared__ double sh[2 * NS][NT];
  const GaBlock k = ga_block(a, a.sblk0, a.srpb, blockIdx.x);
  const int tile = blockIdx.y, lanes = NT / a.ct;
  const int cl = threadIdx.x % a.ct, lane = threadIdx.x / a.ct, col = tile * a.ct + cl;
  const bool live = lane < lanes && col < a.cols;
  double v[2 * NS];
#pragma unroll
  for (int k = 0; k < 2 * NS; ++k) v[k] = 0.0;
  if (live) {
    const typename Elem<DT>::type* p = x + (a.row0[k.lev] + (long long)k.n * a.hw[k.lev]) * a.ldx + (long long)col * VEC;
    auto add = [&](const typename RV::raw& q) {
      float f[VEC];
      RV::unpack(q, f);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const double d = (double)f[e];
        const int w = WHOLE ? 0 : e;
        v[w] += d;
        v[NS + w] = __builtin_fma(d, d, v[NS + w]);
      }
    };
    long long r = k.rb + lane;
    for (; r + 3 * lanes < k.re; r += 4 * lanes) {     // four loads in flight
      typename RV::raw q[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) q[u] = RV::load(p + (r + u * lanes) * a.ldx);
#pragma unroll
      for (int u = 0; u < 4; ++u) add(q[u]);
    }
    for (; r < k.re; r += lanes) add(RV::load(p + r * a.ldx));
  }
  lane_tree<2 * NS, NT>(sh, v, lane, a.ct, lanes);
  // one thread per group of the tile adds its channels
  const int c0 = tile * a.ct * VEC, c1 = min(c0 + a.ct * VEC, a.C);
  const int g0 = c0 / a.cpg, g1 = (c1 - 1) / a.cpg;
  for (int g = g0 + threadIdx.x; g <= g1; g += NT) {
    const int lo = max(g * a.cpg, c0) - c0, hi = min((g + 1) * a.cpg, c1) - c0;
    double s = 0.0, ss = 0.0;
    if constexpr (WHOLE) {
      for (int q = lo / VEC; q < hi / VEC; ++q) s += sh[0][q], ss += sh[1][q];
    } else {
      for (int c = lo; c < hi; ++c) s += sh[c % VEC][c / VEC], ss += sh[NS + c % VEC][c / VEC];
    }
    part[((long long)blockIdx.x * a.ntile + tile) * gpt + (g - g0)] = make_double2(s, ss);
  }
}

__device__ __forceinline__ double2 ga_mean_rstd(double s, double ss, double cnt, float eps) {
  const double m = s / cnt;
  double var = ss / cnt - m * m;
  var = var < 0.0 ? 0.0 : var;                   // (NaN stays NaN)
  return make_double2(m, 1.0 / sqrt(var + (double)eps));
}

// The partials of every group of this block's column tile, added into s_sum[group - first group]: every element-wise block does it for
// itself (a launch of its own for it cost 6 us, more than these few KB out of L2).  Threads share a group's entries and join in order.
__device__ __forceinline__ int ga_combine(const double2* __restrict__ part, double2* s_sum, double2* s_red, const GaArgs& a, int gpt, int tc,
                                          int n, int lev, int tile) {
  const int c0 = tile * tc, c1 = min(c0 + tc, a.C);
  const int g0 = c0 / a.cpg, ng = (c1 - 1) / a.cpg - g0 + 1;
  const int b0 = a.sblk0[lev], nb = a.sblk0[lev + 1] - b0;
  int tpg = 1;                                   // threads per group, a power of two
  while (tpg * 2 * ng <= GA_THREADS) tpg <<= 1;
  const int gi = threadIdx.x / tpg, ti = threadIdx.x - gi * tpg;
  double s = 0.0, ss = 0.0;
  if (gi < ng) {
    const int g = g0 + gi;
    for (int t = g * a.cpg / tc; t <= ((g + 1) * a.cpg - 1) / tc; ++t) {
      const double2* q = part + (((long long)n * a.sblk0[a.nlev] + b0) * a.ntile + t) * gpt + (g - t * tc / a.cpg);
      for (int i = ti; i < nb; i += tpg) {
        const double2 e = q[(long long)i * a.ntile * gpt];
        s += e.x, ss += e.y;
      }
    }
  }
  s_red[threadIdx.x] = make_double2(s, ss);
  __syncthreads();
  if (gi < ng && ti == 0) {
    for (int i = 1; i < tpg; ++i) s += s_red[threadIdx.x + i].x, ss += s_red[threadIdx.x + i].y;
    s_sum[gi] = make_double2(s, ss);
  }
  __syncthreads();
  return ng;
}

// what a thread of the forward element pass needs of its channels.  The mean is a sum of two floats: x - m keeps its digits for
// |m| >> sqrt(v)
template <int VEC, bool WHOLE>
struct GaNorm {
  static constexpr int NS = WHOLE ? 1 : VEC;
  float mh[NS], ml[NS], ga[VEC], be[VEC];
  __device__ __forceinline__ void set(int e, double2 st, float gamma, float beta) {
    if (!WHOLE || e == 0) {
      mh[WHOLE ? 0 : e] = (float)st.x;
      ml[WHOLE ? 0 : e] = (float)(st.x - (double)(float)st.x);
    }
    ga[e] = (float)(st.y * (double)gamma);
    be[e] = beta;
  }
  template <int ACT, bool DROP>
  __device__ __forceinline__ void apply(float (&f)[VEC], uint32_t keep, float scale) const {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const int k = WHOLE ? 0 : e;
      f[e] = act_fwd<ACT>(__builtin_fmaf((f[e] - mh[k]) - ml[k], ga[e], be[e]));
      if constexpr (DROP) f[e] = (keep >> e) & 1u ? f[e] * scale : 0.f;
    }
  }
};

// keep bits of the VEC channels from column vector `col` of row `row`
template <int VEC, bool DROP>
__device__ __forceinline__ uint32_t ga_keep(const GaArgs& a, unsigned long long off, long long row, int col) {
  if constexpr (!DROP) return 0xffu;
  const unsigned long long i = (unsigned long long)row * a.C + (unsigned long long)col * VEC;
  const uint32_t keep = drop_keep8(i >> 3, off, a.drop.seed, a.drop.thr);
  return VEC == 1 ? keep >> (int)(i & 7) : keep;
}

// launch 2, forward; the first row block of a level writes (mean, rstd) out for the backward pass
template <int DT, int VEC, bool WHOLE, int ACT, bool DROP>
__global__ __launch_bounds__(GA_THREADS) void ga_apply_kernel(const typename Elem<DT>::type* __restrict__ x,
                                                              typename Elem<DT>::type* __restrict__ y, const float* __restrict__ gamma,
                                                              const float* __restrict__ beta, const double2* __restrict__ part,
                                                              double2* __restrict__ stats, const GaArgs a, int gpt) {
  typedef RowVec<DT, VEC> RV;
  __shared__ double2 s_stat[GA_THREADS], s_red[GA_THREADS];
  const GaBlock k = ga_block(a, a.ablk0, a.arpb, blockIdx.x);
  const int tile = blockIdx.y, lanes = GA_THREADS / a.ct, tc = a.ct * VEC, g0 = tile * tc / a.cpg;
  const int ng = ga_combine(part, s_stat, s_red, a, gpt, tc, k.n, k.lev, tile);
  for (int g = threadIdx.x; g < ng; g += GA_THREADS) {
    const double2 st = ga_mean_rstd(s_stat[g].x, s_stat[g].y, (double)a.hw[k.lev] * (double)a.cpg, a.eps);
    s_stat[g] = st;
    // (a group is written by the tile that it starts in)
    if (stats != nullptr && k.b == a.ablk0[k.lev] && (g0 + g) * a.cpg >= tile * tc)
      stats[((long long)k.n * a.nlev + k.lev) * a.G + g0 + g] = st;
  }
  __syncthreads();
  const int cl = threadIdx.x % a.ct, lane = threadIdx.x / a.ct, col = tile * a.ct + cl;
  if (lane >= lanes || col >= a.cols) return;
  GaNorm<VEC, WHOLE> nm;
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    const int c = col * VEC + e;
    nm.set(e, s_stat[c / a.cpg - g0], gamma != nullptr ? gamma[c] : 1.f, beta != nullptr ? beta[c] : 0.f);
  }
  const unsigned long long off = DROP ? drop_offset(a.drop) : 0ull;
  const long long row_base = a.row0[k.lev] + (long long)k.n * a.hw[k.lev];
  const typename Elem<DT>::type* px = x + row_base * a.ldx + (long long)col * VEC;
  typename Elem<DT>::type* py = y + row_base * a.ldy + (long long)col * VEC;
  auto one = [&](const typename RV::raw& q, long long r) {
    float f[VEC];
    RV::unpack(q, f);
    nm.template apply<ACT, DROP>(f, ga_keep<VEC, DROP>(a, off, row_base + r, col), a.drop.scale);
    RV::store(py + r * a.ldy, f);
  };
  long long r = k.rb + lane;
  for (; r + 3 * lanes < k.re; r += 4 * lanes) {
    typename RV::raw q[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) q[u] = RV::load(px + (r + u * lanes) * a.ldx);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      one(q[u], r + u * lanes);
      __builtin_amdgcn_sched_barrier(0);         // one row at a time: interleaved, four generator blocks took 30 more registers
    }
  }
  for (; r < k.re; r += lanes) one(RV::load(px + r * a.ldx), r);
}

// what a thread of the backward launches needs of its channels
template <int VEC, bool WHOLE>
struct GaChan {
  static constexpr int NS = WHOLE ? 1 : VEC;
  float mh[NS], ml[NS], rs[NS], ga[VEC], be[VEC];
  double2 st[NS];
  __device__ __forceinline__ void fill(const GaArgs& a, const double2* __restrict__ stats, const float* __restrict__ gamma,
                                       const float* __restrict__ beta, long long sbase, int col) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const int c = col * VEC + e;
      if (!WHOLE || e == 0) {
        const int k = WHOLE ? 0 : e;
        st[k] = stats[sbase + c / a.cpg];
        mh[k] = (float)st[k].x;
        ml[k] = (float)(st[k].x - (double)mh[k]);
        rs[k] = (float)st[k].y;
      }
      ga[e] = gamma != nullptr ? gamma[c] : 1.f;
      be[e] = beta != nullptr ? beta[c] : 0.f;
    }
  }
  // xhat and d = dy * keep / (1 - p) * act'(t) of VEC elements
  template <int ACT, bool DROP>
  __device__ __forceinline__ void grad(const float (&x)[VEC], const float (&dy)[VEC], uint32_t keep, float scale, float (&xh)[VEC],
                                       float (&d)[VEC]) const {
    float t[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const int k = WHOLE ? 0 : e;
      xh[e] = ((x[e] - mh[k]) - ml[k]) * rs[k];
      if constexpr (ACT != SM_ACT_NONE) t[e] = __builtin_fmaf(xh[e], ga[e], be[e]);
      d[e] = dy[e];
      if constexpr (DROP) d[e] = (keep >> e) & 1u ? d[e] * scale : 0.f;
    }
    if constexpr (ACT == SM_ACT_RELU) {
      // the ReLU passes the whole gradient or nothing: within rounding of the border (t = xh * gamma + beta is off by at most
      // 3 * 2^-24 (|xh gamma| + |beta|), and near 0 the two are alike) t is taken in f64.  One test for the vector: its arm is entered
      // by one in 10^4 and must not cost the others a branch per element.
      float near = 1.f;
#pragma unroll
      for (int e = 0; e < VEC; ++e) near = fminf(near, __builtin_fmaf(-1e-6f, __builtin_fabsf(be[e]), __builtin_fabsf(t[e])));
      if (near <= 0.f) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const double2 s = st[WHOLE ? 0 : e];
          const double t64 = ((double)x[e] - s.x) * s.y * (double)ga[e] + (double)be[e];
          if (__builtin_fabsf(t[e]) <= 1e-6f * __builtin_fabsf(be[e])) t[e] = t64 > 0.0 ? 1.f : (t64 <= 0.0 ? -1.f : t[e]);
          __builtin_amdgcn_sched_barrier(0);     // (one at a time: this arm must not set the kernel's register count)
        }
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) d[e] = t[e] <= 0.f ? 0.f : d[e];
    } else if constexpr (ACT != SM_ACT_NONE) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) d[e] *= act_grad<ACT>(t[e]);
    }
  }
};

// launch 1, backward, over the rows of a block: chan[image][row block][channel] = (sum d, sum d xhat) and, weighted with gamma, the same
// per group of the column tile: part[image][row block][tile][group - first group of the tile]
template <int DT, int VEC, bool WHOLE, int ACT, bool DROP>
__global__ __launch_bounds__(GA_SUM, WHOLE ? 4 : 2) void ga_bwd_sum_kernel(const typename Elem<DT>::type* __restrict__ x,
                                                                const typename Elem<DT>::type* __restrict__ dy,
                                                                const float* __restrict__ gamma, const float* __restrict__ beta,
                                                                const double2* __restrict__ stats, float2* __restrict__ chan,
                                                                double2* __restrict__ part, const GaArgs a, int gpt) {
  typedef RowVec<DT, VEC> RV;
  __shared__ float sh[VEC][GA_SUM], s_chan[2][GA_THREADS];
  const GaBlock k = ga_block(a, a.sblk0, a.srpb, blockIdx.x);
  const int tile = blockIdx.y, lanes = GA_SUM / a.ct;
  const int cl = threadIdx.x % a.ct, lane = threadIdx.x / a.ct, col = tile * a.ct + cl;
  const bool live = lane < lanes && col < a.cols;
  float v[2 * VEC];
#pragma unroll
  for (int k = 0; k < 2 * VEC; ++k) v[k] = 0.f;
  if (live) {
    GaChan<VEC, WHOLE> ch;
    ch.fill(a, stats, gamma, beta, ((long long)k.n * a.nlev + k.lev) * a.G, col);
    const unsigned long long off = DROP ? drop_offset(a.drop) : 0ull;
    const long long row_base = a.row0[k.lev] + (long long)k.n * a.hw[k.lev];
    const typename Elem<DT>::type* px = x + row_base * a.ldx + (long long)col * VEC;
    const typename Elem<DT>::type* pd = dy + row_base * a.lddy + (long long)col * VEC;
    auto one = [&](const typename RV::raw& qx, const typename RV::raw& qd, long long r) {
      float fx[VEC], fd[VEC];
      RV::unpack(qx, fx);
      RV::unpack(qd, fd);
      const uint32_t keep = ga_keep<VEC, DROP>(a, off, row_base + r, col);
      float xh[VEC], d[VEC];
      ch.template grad<ACT, DROP>(fx, fd, keep, a.drop.scale, xh, d);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        v[e] += d[e];
        v[VEC + e] = __builtin_fmaf(d[e], xh[e], v[VEC + e]);
      }
    };
    long long r = k.rb + lane;
    for (; r + lanes < k.re; r += 2 * lanes) {
      typename RV::raw qx[2], qd[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) qx[u] = RV::load(px + (r + u * lanes) * a.ldx), qd[u] = RV::load(pd + (r + u * lanes) * a.lddy);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        one(qx[u], qd[u], r + u * lanes);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    for (; r < k.re; r += lanes) one(RV::load(px + r * a.ldx), RV::load(pd + r * a.lddy), r);
  }
  const int c0 = tile * a.ct * VEC, nc = min(a.ct * VEC, a.C - c0);
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    lane_tree<VEC, GA_SUM>(sh, v + q * VEC, lane, a.ct, lanes);
    for (int c = threadIdx.x; c < nc; c += GA_SUM) s_chan[q][c] = sh[c % VEC][c / VEC];
    __syncthreads();
  }
  for (int c = threadIdx.x; c < nc; c += GA_SUM)
    chan[(long long)blockIdx.x * a.C + c0 + c] = make_float2(s_chan[0][c], s_chan[1][c]);
  const int g0 = c0 / a.cpg, ng = (c0 + nc - 1) / a.cpg - g0 + 1;
  for (int g = threadIdx.x; g < ng; g += GA_SUM) {
    const int lo = max((g0 + g) * a.cpg - c0, 0), hi = min((g0 + g + 1) * a.cpg - c0, nc);
    double s = 0.0, ss = 0.0;
    for (int c = lo; c < hi; ++c) {
      const double w = gamma != nullptr ? (double)gamma[c0 + c] : 1.0;
      s += w * (double)s_chan[0][c], ss += w * (double)s_chan[1][c];
    }
    part[((long long)blockIdx.x * a.ntile + tile) * gpt + g] = make_double2(s, ss);
  }
}

// dgamma / dbeta of 32 channels: entries chan[0 .. n)[channel], 8 slices joined in order
template <typename V2>
__device__ __forceinline__ void ga_param_grads(double2 (*sh)[32], const V2* __restrict__ chan, long long n, float* __restrict__ dgamma,
                                               float* __restrict__ dbeta, const GaArgs& a, int cblock) {
  const int ci = threadIdx.x & 31, sl = threadIdx.x >> 5, c = cblock * 32 + ci;
  double s = 0.0, ss = 0.0;
  if (c < a.C) {
#pragma unroll 4
    for (long long i = sl; i < n; i += GA_THREADS / 32) {
      const V2 e = chan[i * a.C + c];
      s += (double)e.x, ss += (double)e.y;
    }
  }
  sh[sl][ci] = make_double2(s, ss);
  __syncthreads();
  if (sl == 0 && c < a.C) {
    for (int k = 1; k < GA_THREADS / 32; ++k) s += sh[k][ci].x, ss += sh[k][ci].y;
    if (dbeta != nullptr) dbeta[c] = (float)s;
    if (dgamma != nullptr) dgamma[c] = (float)ss;
  }
}
__global__ __launch_bounds__(GA_THREADS) void ga_param_grads_kernel(const double2* __restrict__ chan, long long n, float* __restrict__ dgamma,
                                                                    float* __restrict__ dbeta, const GaArgs a) {
  __shared__ double2 sh[GA_THREADS / 32][32];
  ga_param_grads(sh, chan, n, dgamma, dbeta, a, blockIdx.x);
}

// launch 2, backward: the first nparam blocks add up dgamma / dbeta (a long walk over few bytes: they start first), the others write dx
template <int DT, int VEC, bool WHOLE, int ACT, bool DROP>
__global__ __launch_bounds__(GA_THREADS) void ga_bwd_apply_kernel(const typename Elem<DT>::type* __restrict__ x,
                                                                  const typename Elem<DT>::type* __restrict__ dy,
                                                                  const float* __restrict__ gamma, const float* __restrict__ beta,
                                                                  const double2* __restrict__ stats, const float2* __restrict__ chan,
                                                                  const double2* __restrict__ part, typename Elem<DT>::type* __restrict__ dx,
                                                                  float* __restrict__ dgamma, float* __restrict__ dbeta, const GaArgs a, int gpt,
                                                                  int nparam) {
  typedef RowVec<DT, VEC> RV;
  __shared__ double2 s_sum[GA_THREADS], s_red[GA_THREADS / 32][32];
  if ((int)blockIdx.x < nparam) {
    if (blockIdx.y == 0) ga_param_grads(s_red, chan, (long long)a.batch * a.sblk0[a.nlev], dgamma, dbeta, a, blockIdx.x);
    return;
  }
  const GaBlock k = ga_block(a, a.ablk0, a.arpb, blockIdx.x - nparam);
  const int tile = blockIdx.y, lanes = GA_THREADS / a.ct, tc = a.ct * VEC, g0 = tile * tc / a.cpg;
  ga_combine(part, s_sum, &s_red[0][0], a, gpt, tc, k.n, k.lev, tile);
  const int cl = threadIdx.x % a.ct, lane = threadIdx.x / a.ct, col = tile * a.ct + cl;
  if (lane >= lanes || col >= a.cols) return;
  GaChan<VEC, WHOLE> ch;
  ch.fill(a, stats, gamma, beta, ((long long)k.n * a.nlev + k.lev) * a.G, col);
  constexpr int NS = WHOLE ? 1 : VEC;
  const double cnt = (double)a.hw[k.lev] * (double)a.cpg;
  float m1[NS], m2[NS];                          // means over the group of d gamma and d gamma xhat
#pragma unroll
  for (int e = 0; e < NS; ++e) {
    const double2 sum = s_sum[(col * VEC + e) / a.cpg - g0];
    m1[e] = (float)(sum.x / cnt), m2[e] = (float)(sum.y / cnt);
  }
  const unsigned long long off = DROP ? drop_offset(a.drop) : 0ull;
  const long long row_base = a.row0[k.lev] + (long long)k.n * a.hw[k.lev];
  const typename Elem<DT>::type* px = x + row_base * a.ldx + (long long)col * VEC;
  const typename Elem<DT>::type* pd = dy + row_base * a.lddy + (long long)col * VEC;
  typename Elem<DT>::type* po = dx + row_base * a.lddx + (long long)col * VEC;
  auto one = [&](const typename RV::raw& qx, const typename RV::raw& qd, long long r) {
    float fx[VEC], fd[VEC];
    RV::unpack(qx, fx);
    RV::unpack(qd, fd);
    const uint32_t keep = ga_keep<VEC, DROP>(a, off, row_base + r, col);
    float xh[VEC], d[VEC];
    ch.template grad<ACT, DROP>(fx, fd, keep, a.drop.scale, xh, d);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const int w = WHOLE ? 0 : e;
      fx[e] = ch.rs[w] * (__builtin_fmaf(d[e], ch.ga[e], -m1[w]) - xh[e] * m2[w]);
    }
    RV::store(po + r * a.lddx, fx);
  };
  long long r = k.rb + lane;
  for (; r + lanes < k.re; r += 2 * lanes) {
    typename RV::raw qx[2], qd[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) qx[u] = RV::load(px + (r + u * lanes) * a.ldx), qd[u] = RV::load(pd + (r + u * lanes) * a.lddy);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      one(qx[u], qd[u], r + u * lanes);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  for (; r < k.re; r += lanes) one(RV::load(px + r * a.ldx), RV::load(pd + r * a.lddy), r);
}

// ------------------------------------------------------------------------------------------------ small maps: one launch
constexpr int GA_SMALL = 1024;                   // threads
// rows per thread that are kept in registers: 16 (f32: 32) bytes each; 1024 threads have 128 registers
template <int DT>
constexpr int ga_small_rows = DT == SM_DT_F32 ? 2 : 4;

// channel sums sh[0 / 1][channel] of a block that owns whole groups -> weighted group sums
template <int VEC, typename F>
__device__ __forceinline__ void ga_small_groups(double (*sh)[GA_SMALL / 4], double2* s_grp, int c0, int nc, int cpg, const F& weight) {
  for (int g = threadIdx.x; g * cpg < nc; g += GA_SMALL) {
    double s = 0.0, ss = 0.0;
    for (int c = g * cpg; c < (g + 1) * cpg; ++c) {
      const double w = weight(c0 + c);
      s += w * sh[0][c], ss += w * sh[1][c];
    }
    s_grp[g] = make_double2(s, ss);
  }
  __syncthreads();
}

// sum over the row lanes of the block: NV values per thread of each of VEC channels -> out[k][channel of the tile].  Waves first (the
// lanes of a wave that share a column), then the waves in order.
template <int VEC, typename V>
__device__ __forceinline__ void ga_small_reduce(V (*red)[32 * VEC], double (*out)[GA_SMALL / 4], V (&a0)[VEC], V (&a1)[VEC], int ct) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    V(&v)[VEC] = q == 0 ? a0 : a1;
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      for (int d = ct; d < 64; d <<= 1) v[e] += __shfl_xor(v[e], d, 64);
    __syncthreads();                             // (the loop before this one has read red)
    if (lane < ct) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) red[wave][lane * VEC + e] = v[e];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < ct * VEC; c += GA_SMALL) {
      double t = 0.0;
#pragma unroll
      for (int w = 0; w < GA_SMALL / 64; ++w) t += (double)red[w][c];
      out[q][c] = t;
    }
  }
  __syncthreads();
}

// grid (image, level) x column tile of whole groups, groups of whole vectors; ct (columns per tile) is a power of two of at most 32
template <int DT, int ACT, bool DROP>
__global__ __launch_bounds__(GA_SMALL) void ga_small_kernel(const typename Elem<DT>::type* __restrict__ x, typename Elem<DT>::type* __restrict__ y,
                                                            const float* __restrict__ gamma, const float* __restrict__ beta,
                                                            double2* __restrict__ stats, const GaArgs a, int ct) {
  typedef RowVec<DT, 8> RV;
  constexpr int NR = ga_small_rows<DT>;
  __shared__ double2 s_red[GA_SMALL / 64][32], s_grp[32];
  const int lev = blockIdx.x % a.nlev, n = blockIdx.x / a.nlev, hw = (int)a.hw[lev];
  if (hw == 0) return;
  const int cl = threadIdx.x & (ct - 1), lane = threadIdx.x / ct, lanes = GA_SMALL / ct, col = blockIdx.y * ct + cl;
  const int c0 = blockIdx.y * ct * 8, nc = min(ct * 8, a.C - c0);
  const bool live = col < a.cols;
  const long long row_base = a.row0[lev] + (long long)n * hw;
  const typename Elem<DT>::type* px = x + row_base * a.ldx + (long long)col * 8;
  typename RV::raw q[NR];
  double s = 0.0, ss = 0.0;                      // (a vector lies in one group)
#pragma unroll
  for (int u = 0; u < NR; ++u) {
    const int r = lane + u * lanes;
    if (live && r < hw) q[u] = RV::load(px + (long long)r * a.ldx);
  }
#pragma unroll
  for (int u = 0; u < NR; ++u) {
    const int r = lane + u * lanes;
    if (live && r < hw) {
      float f[8];
      RV::unpack(q[u], f);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const double d = (double)f[e];
        s += d, ss = __builtin_fma(d, d, ss);
      }
    }
  }
  // the row lanes of a wave, then waves x columns of the group, in order
  for (int d = ct; d < 64; d <<= 1) s += __shfl_xor(s, d, 64), ss += __shfl_xor(ss, d, 64);
  if ((threadIdx.x & 63) < ct) s_red[threadIdx.x >> 6][threadIdx.x & 63] = make_double2(s, ss);
  __syncthreads();
  const int gcols = a.cpg / 8;
  for (int g = threadIdx.x; g * a.cpg < nc; g += GA_SMALL) {
    double t = 0.0, tt = 0.0;
    for (int k = g * gcols; k < (g + 1) * gcols; ++k)
#pragma unroll
      for (int w = 0; w < GA_SMALL / 64; ++w) t += s_red[w][k].x, tt += s_red[w][k].y;
    const double2 st = ga_mean_rstd(t, tt, (double)hw * (double)a.cpg, a.eps);
    s_grp[g] = st;
    if (stats != nullptr) stats[(long long)blockIdx.x * a.G + c0 / a.cpg + g] = st;
  }
  __syncthreads();
  if (!live) return;
  GaNorm<8, true> nm;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int c = col * 8 + e;
    nm.set(e, s_grp[(c - c0) / a.cpg], gamma != nullptr ? gamma[c] : 1.f, beta != nullptr ? beta[c] : 0.f);
  }
  const unsigned long long off = DROP ? drop_offset(a.drop) : 0ull;
  typename Elem<DT>::type* py = y + row_base * a.ldy + (long long)col * 8;
#pragma unroll
  for (int u = 0; u < NR; ++u) {
    const int r = lane + u * lanes;
    if (r < hw) {
      float f[8];
      RV::unpack(q[u], f);
      nm.template apply<ACT, DROP>(f, ga_keep<8, DROP>(a, off, row_base + r, col), a.drop.scale);
      RV::store(py + (long long)r * a.ldy, f);
    }
  }
}

// backward: dx (may be null) and the channel sums chan[image, level][channel] = (sum d, sum d xhat); of one (image, level) the sums are
// the parameters' gradients themselves
template <int DT, int ACT, bool DROP>
__global__ __launch_bounds__(GA_SMALL) void ga_small_bwd_kernel(const typename Elem<DT>::type* __restrict__ x,
                                                                const typename Elem<DT>::type* __restrict__ dy,
                                                                const float* __restrict__ gamma, const float* __restrict__ beta,
                                                                const double2* __restrict__ stats, typename Elem<DT>::type* __restrict__ dx,
                                                                double2* __restrict__ chan, float* __restrict__ dgamma,
                                                                float* __restrict__ dbeta, const GaArgs a, int ct) {
  typedef RowVec<DT, 8> RV;
  constexpr int NR = ga_small_rows<DT>;
  __shared__ float s_red[GA_SMALL / 64][32 * 8];
  __shared__ double s_chan[2][GA_SMALL / 4];
  __shared__ double2 s_grp[GA_SMALL / 4];
  const int lev = blockIdx.x % a.nlev, n = blockIdx.x / a.nlev, hw = (int)a.hw[lev];
  const int cl = threadIdx.x & (ct - 1), lane = threadIdx.x / ct, lanes = GA_SMALL / ct, col = blockIdx.y * ct + cl;
  const int c0 = blockIdx.y * ct * 8, nc = min(ct * 8, a.C - c0);
  if (hw == 0) {                                 // an empty level adds nothing to the parameters' gradients
    if (chan != nullptr)
      for (int c = threadIdx.x; c < nc; c += GA_SMALL) chan[(long long)blockIdx.x * a.C + c0 + c] = make_double2(0.0, 0.0);
    return;
  }
  const bool live = col < a.cols;
  const long long row_base = a.row0[lev] + (long long)n * hw;
  const typename Elem<DT>::type* px = x + row_base * a.ldx + (long long)col * 8;
  const typename Elem<DT>::type* pd = dy + row_base * a.lddy + (long long)col * 8;
  typename RV::raw qx[NR], qd[NR];
#pragma unroll
  for (int u = 0; u < NR; ++u) {
    const int r = lane + u * lanes;
    if (live && r < hw) qx[u] = RV::load(px + (long long)r * a.ldx), qd[u] = RV::load(pd + (long long)r * a.lddy);
  }
  GaChan<8, true> ch;
  if (live) ch.fill(a, stats, gamma, beta, (long long)blockIdx.x * a.G, col);
  const unsigned long long off = DROP ? drop_offset(a.drop) : 0ull;
  uint32_t keep[NR];
  float s[8], ss[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) s[e] = 0.f, ss[e] = 0.f;
#pragma unroll
  for (int u = 0; u < NR; ++u) {
    const int r = lane + u * lanes;
    keep[u] = 0xffu;
    if (live && r < hw) {
      keep[u] = ga_keep<8, DROP>(a, off, row_base + r, col);
      float fx[8], fd[8];
      RV::unpack(qx[u], fx);
      RV::unpack(qd[u], fd);
      float xh[8], d[8];
      ch.template grad<ACT, DROP>(fx, fd, keep[u], a.drop.scale, xh, d);
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] += d[e], ss[e] = __builtin_fmaf(d[e], xh[e], ss[e]);
    }
  }
  ga_small_reduce<8>(s_red, s_chan, s, ss, ct);
  for (int c = threadIdx.x; c < nc; c += GA_SMALL) {
    if (chan != nullptr) chan[(long long)blockIdx.x * a.C + c0 + c] = make_double2(s_chan[0][c], s_chan[1][c]);
    if (dbeta != nullptr) dbeta[c0 + c] = (float)s_chan[0][c];
    if (dgamma != nullptr) dgamma[c0 + c] = (float)s_chan[1][c];
  }
  if (dx == nullptr) return;
  ga_small_groups<8>(s_chan, s_grp, c0, nc, a.cpg, [&](int c) { return gamma != nullptr ? (double)gamma[c] : 1.0; });
  if (!live) return;
  const double cnt = (double)hw * (double)a.cpg;
  const double2 gs = s_grp[(col * 8 - c0) / a.cpg];
  const float m1 = (float)(gs.x / cnt), m2 = (float)(gs.y / cnt);
  typename Elem<DT>::type* po = dx + row_base * a.lddx + (long long)col * 8;
#pragma unroll
  for (int u = 0; u < NR; ++u) {
    const int r = lane + u * lanes;
    if (r < hw) {
      float fx[8], fd[8];
      RV::unpack(qx[u], fx);
      RV::unpack(qd[u], fd);
      float xh[8], d[8];
      ch.template grad<ACT, DROP>(fx, fd, keep[u], a.drop.scale, xh, d);
#pragma unroll
      for (int e = 0; e < 8; ++e) fx[e] = ch.rs[0] * (__builtin_fmaf(d[e], ch.ga[e], -m1) - xh[e] * m2);
      RV::store(po + (long long)r * a.lddx, fx);
    }
  }
}

// ------------------------------------------------------------------------------------------------ many small maps
// The same for more maps than the chip holds at once: a block has just the threads that hold a map's rows and takes every gridDim.x-th
// (image, level), so that neither the launch of a thousand idle threads per map nor, backward, a row of channel sums per map is left over.
// 67 200 maps of 1 x 256 bf16, forward / backward: 274 / 872 us, with a block of 1024 threads to each 5740 / 11 690; 1000 maps of 7 x 7 x
// 256: 18 / 50 and 95 / 178; 100 of them: 8 / 14 and 14 / 26.
constexpr int GA_MANY = 512;                     // threads at most; a power of two of at least 64

constexpr int ga_many_lds(int waves, int ct) { return (waves + 1) * ct * 16; }
constexpr int ga_many_bwd_lds(int waves, int ct) { return ct * 16 + 4 * ct * 8 * 8 + waves * ct * 8 * 4; }

template <int DT, int ACT, bool DROP>
__global__ __launch_bounds__(GA_MANY) void ga_many_kernel(const typename Elem<DT>::type* __restrict__ x, typename Elem<DT>::type* __restrict__ y,
                                                          const float* __restrict__ gamma, const float* __restrict__ beta,
                                                          double2* __restrict__ stats, const GaArgs a, int ct) {
  typedef RowVec<DT, 8> RV;
  constexpr int NR = ga_small_rows<DT>;
  extern __shared__ __attribute__((aligned(16))) double2 s_red[];     // [waves][ct], then the groups'
  const int waves = blockDim.x >> 6;
  double2* const s_grp = s_red + waves * ct;
  const int cl = threadIdx.x & (ct - 1), lane = threadIdx.x / ct, lanes = blockDim.x / ct, col = blockIdx.y * ct + cl;
  const int c0 = blockIdx.y * ct * 8, nc = min(ct * 8, a.C - c0), gcols = a.cpg / 8;
  const bool live = col < a.cols;
  const unsigned long long off = DROP ? drop_offset(a.drop) : 0ull;
  for (int item = blockIdx.x; item < a.batch * a.nlev; item += gridDim.x) {
    const int lev = item % a.nlev, n = item / a.nlev, hw = (int)a.hw[lev];
    if (hw == 0) continue;
    const long long row_base = a.row0[lev] + (long long)n * hw;
    const typename Elem<DT>::type* px = x + row_base * a.ldx + (long long)col * 8;
    typename RV::raw q[NR];
#pragma unroll
    for (int u = 0; u < NR; ++u) {
      const int r = lane + u * lanes;
      if (live && r < hw) q[u] = RV::load(px + (long long)r * a.ldx);
    }
    double s = 0.0, ss = 0.0;
#pragma unroll
    for (int u = 0; u < NR; ++u) {
      if (live && lane + u * lanes < hw) {
        float f[8];
        RV::unpack(q[u], f);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const double d = (double)f[e];
          s += d, ss = __builtin_fma(d, d, ss);
        }
      }
    }
    for (int d = ct; d < 64; d <<= 1) s += __shfl_xor(s, d, 64), ss += __shfl_xor(ss, d, 64);
    if ((threadIdx.x & 63) < ct) s_red[(threadIdx.x >> 6) * ct + (threadIdx.x & 63)] = make_double2(s, ss);
    __syncthreads();                             // (behind it nobody reads the last map's s_grp any more)
    for (int g = threadIdx.x; g * a.cpg < nc; g += blockDim.x) {
      double t = 0.0, tt = 0.0;
      for (int k = g * gcols; k < (g + 1) * gcols; ++k)
        for (int w = 0; w < waves; ++w) t += s_red[w * ct + k].x, tt += s_red[w * ct + k].y;
      const double2 st = ga_mean_rstd(t, tt, (double)hw * (double)a.cpg, a.eps);
      s_grp[g] = st;
      if (stats != nullptr) stats[(long long)item * a.G + c0 / a.cpg + g] = st;
    }
    __syncthreads();                             // (and behind this one nobody reads s_red)
    if (!live) continue;
    GaNorm<8, true> nm;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int c = col * 8 + e;
      nm.set(e, s_grp[(c - c0) / a.cpg], gamma != nullptr ? gamma[c] : 1.f, beta != nullptr ? beta[c] : 0.f);
    }
    typename Elem<DT>::type* py = y + row_base * a.ldy + (long long)col * 8;
#pragma unroll
    for (int u = 0; u < NR; ++u) {
      const int r = lane + u * lanes;
      if (r < hw) {
        float f[8];
        RV::unpack(q[u], f);
        nm.template apply<ACT, DROP>(f, ga_keep<8, DROP>(a, off, row_base + r, col), a.drop.scale);
        RV::store(py + (long long)r * a.ldy, f);
      }
    }
  }
}

// backward: dx (may be null) and the channel sums over the block's maps, chan[block][channel]
template <int DT, int ACT, bool DROP>
__global__ __launch_bounds__(GA_MANY) void ga_many_bwd_kernel(const typename Elem<DT>::type* __restrict__ x,
                                                              const typename Elem<DT>::type* __restrict__ dy, const float* __restrict__ gamma,
                                                              const float* __restrict__ beta, const double2* __restrict__ stats,
                                                              typename Elem<DT>::type* __restrict__ dx, double2* __restrict__ chan,
                                                              const GaArgs a, int ct) {
  typedef RowVec<DT, 8> RV;
  constexpr int NR = ga_small_rows<DT>;
  extern __shared__ __attribute__((aligned(16))) double2 s_grp[];     // [ct], then per channel: [2] of a map, [2] of all maps, [waves]
  const int tc = ct * 8, waves = blockDim.x >> 6;
  double *const s_chan = reinterpret_cast<double*>(s_grp + ct), *const s_acc = s_chan + 2 * tc;
  float* const s_red = reinterpret_cast<float*>(s_acc + 2 * tc);
  const int cl = threadIdx.x & (ct - 1), lane = threadIdx.x / ct, lanes = blockDim.x / ct, col = blockIdx.y * ct + cl;
  const int c0 = blockIdx.y * tc, nc = min(tc, a.C - c0);
  const bool live = col < a.cols;
  const unsigned long long off = DROP ? drop_offset(a.drop) : 0ull;
  for (int c = threadIdx.x; c < tc; c += blockDim.x) s_acc[c] = 0.0, s_acc[tc + c] = 0.0;             // (its thread's own from here on)
  for (int item = blockIdx.x; item < a.batch * a.nlev; item += gridDim.x) {
    const int lev = item % a.nlev, n = item / a.nlev, hw = (int)a.hw[lev];
    if (hw == 0) continue;
    const long long row_base = a.row0[lev] + (long long)n * hw;
    const typename Elem<DT>::type* px = x + row_base * a.ldx + (long long)col * 8;
    const typename Elem<DT>::type* pd = dy + row_base * a.lddy + (long long)col * 8;
    typename RV::raw qx[NR], qd[NR];
#pragma unroll
    for (int u = 0; u < NR; ++u) {
      const int r = lane + u * lanes;
      if (live && r < hw) qx[u] = RV::load(px + (long long)r * a.ldx), qd[u] = RV::load(pd + (long long)r * a.lddy);
    }
    GaChan<8, true> ch;
    if (live) ch.fill(a, stats, gamma, beta, (long long)item * a.G, col);
    float v[2][8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[0][e] = v[1][e] = 0.f;
#pragma unroll
    for (int u = 0; u < NR; ++u) {
      const int r = lane + u * lanes;
      if (live && r < hw) {
        float fx[8], fd[8];
        RV::unpack(qx[u], fx);
        RV::unpack(qd[u], fd);
        float xh[8], d[8];
        ch.template grad<ACT, DROP>(fx, fd, ga_keep<8, DROP>(a, off, row_base + r, col), a.drop.scale, xh, d);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[0][e] += d[e], v[1][e] = __builtin_fmaf(d[e], xh[e], v[1][e]);
      }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        for (int d = ct; d < 64; d <<= 1) v[k][e] += __shfl_xor(v[k][e], d, 64);
      __syncthreads();                           // (s_red, and the last map's s_grp, have been read)
      if ((threadIdx.x & 63) < ct) {
#pragma unroll
        for (int e = 0; e < 8; ++e) s_red[(threadIdx.x >> 6) * tc + (threadIdx.x & 63) * 8 + e] = v[k][e];
      }
      __syncthreads();
      for (int c = threadIdx.x; c < tc; c += blockDim.x) {
        double t = 0.0;
        for (int w = 0; w < waves; ++w) t += (double)s_red[w * tc + c];
        s_chan[k * tc + c] = t, s_acc[k * tc + c] += t;
      }
    }
    if (dx == nullptr) continue;
    __syncthreads();
    for (int g = threadIdx.x; g * a.cpg < nc; g += blockDim.x) {
      double s = 0.0, ss = 0.0;
      for (int c = g * a.cpg; c < (g + 1) * a.cpg; ++c) {
        const double w = gamma != nullptr ? (double)gamma[c0 + c] : 1.0;
        s += w * s_chan[c], ss += w * s_chan[tc + c];
      }
      s_grp[g] = make_double2(s, ss);
    }
    __syncthreads();
    if (!live) continue;
    const double cnt = (double)hw * (double)a.cpg;
    const double2 gs = s_grp[(col * 8 - c0) / a.cpg];
    const float m1 = (float)(gs.x / cnt), m2 = (float)(gs.y / cnt);
    typename Elem<DT>::type* po = dx + row_base * a.lddx + (long long)col * 8;
#pragma unroll
    for (int u = 0; u < NR; ++u) {
      const int r = lane + u * lanes;
      if (r < hw) {
        float fx[8], fd[8];
        RV::unpack(qx[u], fx);
        RV::unpack(qd[u], fd);
        float xh[8], d[8];
        ch.template grad<ACT, DROP>(fx, fd, ga_keep<8, DROP>(a, off, row_base + r, col), a.drop.scale, xh, d);
#pragma unroll
        for (int e = 0; e < 8; ++e) fx[e] = ch.rs[0] * (__builtin_fmaf(d[e], ch.ga[e], -m1) - xh[e] * m2);
        RV::store(po + (long long)r * a.lddx, fx);
      }
    }
  }
  if (chan == nullptr) return;
  for (int c = threadIdx.x; c < nc; c += blockDim.x) chan[(long long)blockIdx.x * a.C + c0 + c] = make_double2(s_acc[c], s_acc[tc + c]);
}

struct GaPlan {
  GaArgs a;
  bool vec, whole;
  int small_ct;                     // > 0: the one-launch kernels, that many column vectors per block
  int many, maps;                   // > 0: ga_many_*, that many threads and blocks (per column tile); else maps is their number
  int gpt;                          // groups per column tile (slots of a partial)
  long long items, ablocks;         // batch * row blocks of all levels: reductions, element-wise launches
  long long fwd_ws, bwd_ws;         // bytes
};

int ga_plan(const sm_gn_act_desc* d, bool aligned, bool backward, GaPlan* p) {
  if (d == nullptr) return SM_ERR_BAD_ARG;
  if (d->nlev < 1 || d->nlev > SM_MAX_LEVELS || d->batch < 0 || d->channels < 1 || d->groups < 1 || d->channels % d->groups != 0)
    return SM_ERR_BAD_SHAPE;
  if (d->dtype < SM_DT_BF16 || d->dtype > SM_DT_F32 || d->act < SM_ACT_NONE || d->act > SM_ACT_GELU) return SM_ERR_BAD_ARG;
  if (!(d->eps >= 0.f)) return SM_ERR_BAD_ARG;
  const long long ld_min = d->channels;
  if (d->x_stride < ld_min || d->y_stride < ld_min || d->dy_stride < ld_min || d->dx_stride < ld_min) return SM_ERR_BAD_SHAPE;
  GaArgs& a = p->a;
  a.nlev = d->nlev, a.batch = d->batch, a.C = d->channels, a.G = d->groups, a.cpg = d->channels / d->groups, a.act = d->act;
  a.eps = d->eps;
  a.ldx = d->x_stride, a.ldy = d->y_stride, a.lddy = d->dy_stride, a.lddx = d->dx_stride;
  const int st = drop_args_fill(&a.drop, d->drop_threshold, d->drop_seed, d->drop_offset, d->drop_offset_dev);
  if (st != SM_OK) return st;
  const int per16 = 16 / sm_dtype_bytes(d->dtype);
  p->vec = aligned && a.C % 8 == 0 && a.ldx % per16 == 0 && a.ldy % per16 == 0 && a.lddy % per16 == 0 && a.lddx % per16 == 0;
  const int vec = p->vec ? 8 : 1;
  p->whole = a.cpg % vec == 0;
  a.cols = a.C / vec;
  a.ct = sm_cdiv(a.cols, sm_cdiv(a.cols, p->vec ? GA_TILE : GA_TILE1));      // (tiles of one width: 320 channels are 2 x 20 vectors)
  a.ntile = sm_cdiv(a.cols, a.ct);
  if (a.ntile > 65535 || a.G > 65535 * 32) return SM_ERR_UNSUPPORTED;
  const int tc = a.ct * vec;
  // Groups in a tile, and the partials of a row block that a tile has to add up: a group may lie in several tiles, one at a tile's end in two
  int entries;
  if (tc % a.cpg == 0) p->gpt = entries = tc / a.cpg;
  else if (a.cpg % tc == 0) p->gpt = 1, entries = a.cpg / tc;
  else {
    p->gpt = std::min(std::min(a.G, (tc - 1) / a.cpg + 2), tc);
    entries = a.cpg < tc ? p->gpt + 2 : p->gpt * std::min(a.ntile, (a.cpg - 1) / tc + 2);
  }
  long long rows = 0, hw_max = 0;
  for (int l = 0; l < d->nlev; ++l) {
    if (d->hw[l] < 0 || d->row0[l] < 0) return SM_ERR_BAD_SHAPE;
    a.hw[l] = d->hw[l], a.row0[l] = d->row0[l];
    rows += d->hw[l], hw_max = std::max<long long>(hw_max, d->hw[l]);
  }
  // Element-wise: about 1024 blocks (all resident at once) of at least 4 rows per row lane.  Reductions: about 512 blocks of at least
  // 2 rows per row lane; every element-wise block adds up the partials of its (image, level), so a level has no more row blocks than
  // fit into GA_COMBINE entries: 32 for 256 channels in 32 groups (four 100 x 168 maps forward / backward: 31 / 47 us, with 64: 36 / 52),
  // twice as many where the chip would else be empty (one such map: 20 / 34 us with 64, 22 / 33 with 128).  With many groups that would
  // leave a large map to four row blocks: up to 32 there, as long as one has 1024 rows (in 256 groups, with four, doubled, and with this:
  // 280 x 320 x 256 214 / 292 and 67 / 106 us, 136 x 136 43 / 82 and 30 / 52; of smaller maps the partials cost more than the rows: 25 x 42
  // backward 23, with 16 row blocks 27).
  const long long total = rows * a.batch * a.ntile;
  long long arpb = std::max<long long>(4 * (GA_THREADS / a.ct), (total + 1023) / 1024);
  long long smin = 4;
  while (smin < 32 && smin * 2048 <= hw_max) smin *= 2;
  const long long smax = std::max<long long>(smin, std::min(256, GA_COMBINE / entries));
  const long long few = (hw_max + smax - 1) / smax, many = (hw_max + 2 * smax - 1) / (2 * smax);
  long long srpb = std::max(std::max<long long>(2 * ((backward ? GA_SUM : GA_STAT) / a.ct), (total + 511) / 512),
                            few > 0 && total / few < 256 ? many : few);
  // Two blocks fit a CU, so a few more than 512 take twice the time of 512 (18 496 rows x 1024 channels backward, 516 blocks: 78 us, 512:
  // 65): up to a quarter more rows per block where that does it
  auto blocks = [&](long long rpb) {
    long long n = 0;
    for (int l = 0; l < d->nlev; ++l) n += (d->hw[l] + rpb - 1) / rpb;
    return n * a.batch * a.ntile;
  };
  for (long long t = srpb; blocks(srpb) > 512 && t <= srpb + srpb / 4; t += std::max<long long>(1, srpb / 32))
    if (blocks(t) <= 512) srpb = t;
  // (the element-wise launches likewise: 1024 with their 128 registers, less the blocks that add up the parameters' gradients; 89 600 x
  // 256 rows of five levels 66 -> 63 us, 29 400 x 512 49 -> 46)
  const long long extra = backward ? (long long)sm_cdiv(a.C, 32) * a.ntile : 0;
  for (long long t = arpb; blocks(arpb) + extra > 1024 && t <= arpb + arpb / 4; t += std::max<long long>(1, arpb / 32))
    if (blocks(t) + extra <= 1024) arpb = t;
  if (srpb > 0x3fffffff || arpb > 0x3fffffff) return SM_ERR_UNSUPPORTED;
  a.srpb = (int)srpb, a.arpb = (int)arpb;
  long long sb = 0, ab = 0;
  for (int l = 0; l < d->nlev; ++l) {
    a.sblk0[l] = (int)sb, a.ablk0[l] = (int)ab;
    sb += (d->hw[l] + srpb - 1) / srpb;
    ab += (d->hw[l] + arpb - 1) / arpb;
    if (ab > 0x7fffffff) return SM_ERR_UNSUPPORTED;
  }
  for (int l = d->nlev; l <= SM_MAX_LEVELS; ++l) a.sblk0[l] = (int)sb, a.ablk0[l] = (int)ab;
  p->items = sb * a.batch, p->ablocks = ab * a.batch;
  const long long nl = (long long)a.batch * a.nlev;
  // (a launch dimension holds fewer than 2^32 threads)
  if (p->items > 0x3ff000 || p->ablocks + a.C / 32 > 0xfff000 || nl > 0x3ff000 || nl * a.G > 0x3fffffff) return SM_ERR_UNSUPPORTED;
  // One launch when a block can hold every row of its columns: the columns of whole groups, 8 (128 bytes of a row for 16-bit types) or
  // the next power of two that is a multiple of the group
  p->small_ct = p->many = 0, p->maps = (int)nl;
  if (p->vec && p->whole) {
    int ct = 8;
    while (ct <= 32 && (ct * 8) % a.cpg != 0 && ct * 8 < a.C) ct <<= 1;
    const int nr = d->dtype == SM_DT_F32 ? ga_small_rows<SM_DT_F32> : ga_small_rows<SM_DT_BF16>;
    if (ct <= 32 && hw_max <= (long long)nr * (GA_SMALL / ct)) p->small_ct = ct;
    // More of them than CUs: blocks of fewer threads that take several maps, as many blocks as the chip holds (with twice as many 1000
    // maps of 7 x 7 x 256 take 19 / 58 us instead of 18 / 53)
    int threads = 64;
    while ((long long)nr * (threads / ct) < hw_max && threads < GA_SMALL) threads <<= 1;
    const long long tiles = sm_cdiv(a.cols, ct);
    if (p->small_ct && nl * tiles > 256 && threads <= GA_MANY) {
      p->many = threads;
      p->maps = (int)std::min<long long>(nl, std::max<long long>(1, 256 * 1024 / threads / tiles));
    }
  }
  p->fwd_ws = p->small_ct ? 0 : p->items * a.ntile * p->gpt * 16;
  p->bwd_ws = p->small_ct ? (long long)p->maps * a.C * 16 : p->items * a.ntile * p->gpt * 16 + p->items * a.C * 8;
  return SM_OK;
}

template <int DT, int VEC, bool WHOLE, int ACT, bool DROP>
int ga_fwd_launch(const GaPlan& p, const void* x, const float* gamma, const float* beta, void* y, void* stats, void* ws, hipStream_t s) {
  typedef typename Elem<DT>::type T;
  const GaArgs& a = p.a;
  if constexpr (VEC == 8 && WHOLE) {
    if (p.small_ct > 0) {
      const dim3 grid(p.maps, sm_cdiv(a.cols, p.small_ct));
      if (p.many > 0)
        hipLaunchKernelGGL((ga_many_kernel<DT, ACT, DROP>), grid, dim3(p.many), ga_many_lds(p.many / 64, p.small_ct), s, (const T*)x, (T*)y,
                           gamma, beta, (double2*)stats, a, p.small_ct);
      else
        hipLaunchKernelGGL((ga_small_kernel<DT, ACT, DROP>), grid, dim3(GA_SMALL), 0, s, (const T*)x, (T*)y, gamma, beta, (double2*)stats, a,
                           p.small_ct);
      SM_LAUNCH_CHECK();
      return SM_OK;
    }
  }
  double2* part = (double2*)ws;
  hipLaunchKernelGGL((ga_stats_kernel<DT, VEC, WHOLE>), dim3((unsigned)p.items, a.ntile), dim3(WHOLE ? GA_STAT : GA_STAT1), 0, s,
                     (const T*)x, part, a, p.gpt);
  hipLaunchKernelGGL((ga_apply_kernel<DT, VEC, WHOLE, ACT, DROP>), dim3((unsigned)p.ablocks, a.ntile), dim3(GA_THREADS), 0, s, (const T*)x,
                     (T*)y, gamma, beta, part, (double2*)stats, a, p.gpt);
  SM_LAUNCH_CHECK();
  return SM_OK;
}

template <int DT, int VEC, bool WHOLE, int ACT, bool DROP>
int ga_bwd_launch(const GaPlan& p, const void* x, const void* dy, const float* gamma, const float* beta, const void* stats, void* dx,
                  float* dgamma, float* dbeta, void* ws, hipStream_t s) {
  typedef typename Elem<DT>::type T;
  const GaArgs& a = p.a;
  const bool params = dgamma != nullptr || dbeta != nullptr;
  if constexpr (VEC == 8 && WHOLE) {
    if (p.small_ct > 0) {
      const dim3 grid(p.maps, sm_cdiv(a.cols, p.small_ct));
      double2* chan = (p.maps > 1 || p.many > 0) && params ? (double2*)ws : nullptr;
      if (p.many > 0)
        hipLaunchKernelGGL((ga_many_bwd_kernel<DT, ACT, DROP>), grid, dim3(p.many), ga_many_bwd_lds(p.many / 64, p.small_ct), s, (const T*)x,
                           (const T*)dy, gamma, beta, (const double2*)stats, (T*)dx, chan, a, p.small_ct);
      else
        hipLaunchKernelGGL((ga_small_bwd_kernel<DT, ACT, DROP>), grid, dim3(GA_SMALL), 0, s, (const T*)x, (const T*)dy, gamma, beta,
                           (const double2*)stats, (T*)dx, chan, chan ? nullptr : dgamma, chan ? nullptr : dbeta, a, p.small_ct);
      if (chan)
        hipLaunchKernelGGL(ga_param_grads_kernel, dim3(sm_cdiv(a.C, 32)), dim3(GA_THREADS), 0, s, chan, (long long)p.maps, dgamma, dbeta, a);
      SM_LAUNCH_CHECK();
      return SM_OK;
    }
  }
  double2* part = (double2*)ws;
  float2* chan = (float2*)(part + p.items * a.ntile * p.gpt);
  hipLaunchKernelGGL((ga_bwd_sum_kernel<DT, VEC, WHOLE, ACT, DROP>), dim3((unsigned)p.items, a.ntile), dim3(GA_SUM), 0, s, (const T*)x,
                     (const T*)dy, gamma, beta, (const double2*)stats, chan, part, a, p.gpt);
  const long long rowb = dx != nullptr ? p.ablocks : 0, chb = params ? sm_cdiv(a.C, 32) : 0;
  if (rowb + chb > 0)
    hipLaunchKernelGGL((ga_bwd_apply_kernel<DT, VEC, WHOLE, ACT, DROP>), dim3((unsigned)(rowb + chb), a.ntile), dim3(GA_THREADS), 0, s,
                       (const T*)x, (const T*)dy, gamma, beta, (const double2*)stats, chan, part, (T*)dx, dgamma, dbeta, a, p.gpt, (int)chb);
  SM_LAUNCH_CHECK();
  return SM_OK;
}

// (dtype, access width, group shape, activation, dropout) -> instantiation
template <typename F, int DT, int VEC, bool WHOLE, int ACT>
int ga_pick4(const GaPlan& p, const F& f) {
  return p.a.drop.thr != 0 ? f.template run<DT, VEC, WHOLE, ACT, true>() : f.template run<DT, VEC, WHOLE, ACT, false>();
}
template <typename F, int DT, int VEC, bool WHOLE>
int ga_pick3(const GaPlan& p, const F& f) {
  switch (p.a.act) {
    case SM_ACT_RELU: return ga_pick4<F, DT, VEC, WHOLE, SM_ACT_RELU>(p, f);
    case SM_ACT_SILU: return ga_pick4<F, DT, VEC, WHOLE, SM_ACT_SILU>(p, f);
    case SM_ACT_GELU: return ga_pick4<F, DT, VEC, WHOLE, SM_ACT_GELU>(p, f);
    default: return ga_pick4<F, DT, VEC, WHOLE, SM_ACT_NONE>(p, f);
  }
}
template <typename F, int DT>
int ga_pick2(const GaPlan& p, const F& f) {
  if (!p.vec) return ga_pick3<F, DT, 1, true>(p, f);
  return p.whole ? ga_pick3<F, DT, 8, true>(p, f) : ga_pick3<F, DT, 8, false>(p, f);
}
template <typename F>
int ga_pick(const GaPlan& p, int dtype, const F& f) {
  if (dtype == SM_DT_BF16) return ga_pick2<F, SM_DT_BF16>(p, f);
  if (dtype == SM_DT_F16) return ga_pick2<F, SM_DT_F16>(p, f);
  return ga_pick2<F, SM_DT_F32>(p, f);
}

struct GaFwd {
  const GaPlan& p;
  const void* x;
  const float *gamma, *beta;
  void *y, *stats, *ws;
  hipStream_t s;
  template <int DT, int VEC, bool WHOLE, int ACT, bool DROP>
  int run() const { return ga_fwd_launch<DT, VEC, WHOLE, ACT, DROP>(p, x, gamma, beta, y, stats, ws, s); }
};
struct GaBwd {
  const GaPlan& p;
  const void *x, *dy;
  const float *gamma, *beta;
  const void* stats;
  void* dx;
  float *dgamma, *dbeta;
  void* ws;
  hipStream_t s;
  template <int DT, int VEC, bool WHOLE, int ACT, bool DROP>
  int run() const { return ga_bwd_launch<DT, VEC, WHOLE, ACT, DROP>(p, x, dy, gamma, beta, stats, dx, dgamma, dbeta, ws, s); }
};

inline bool al16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

// a workspace serves either alignment
extern "C" int64_t sm_group_norm_act_workspace(const sm_gn_act_desc* d, int backward) {
  int64_t need = 0;
  for (int al = 0; al < 2; ++al) {
    GaPlan p;
    const int st = ga_plan(d, al != 0, backward != 0, &p);
    if (st != SM_OK) return st;
    need = std::max<int64_t>(need, backward ? p.bwd_ws : p.fwd_ws);
  }
  return need;
}

extern "C" int sm_group_norm_act(const sm_gn_act_desc* d, const void* x, const float* gamma, const float* beta, void* y, double* stats,
                                 void* workspace, int64_t workspace_bytes, sm_stream_t stream) {
  GaPlan p;
  const int st = ga_plan(d, al16(x) && al16(y), false, &p);
  if (st != SM_OK) return st;
  if (p.items == 0) return SM_OK;
  if (!x || !y || (p.fwd_ws > 0 && !workspace) || !al16(workspace) || (stats != nullptr && !al16(stats))) return SM_ERR_BAD_ARG;
  if (workspace_bytes < p.fwd_ws) return SM_ERR_WORKSPACE;
  return ga_pick(p, d->dtype, GaFwd{p, x, gamma, beta, y, stats, workspace, sm_hip_stream(stream)});
}

extern "C" int sm_group_norm_act_bwd(const sm_gn_act_desc* d, const void* x, const void* dy, const float* gamma, const float* beta,
                                     const double* stats, void* dx, float* dgamma, float* dbeta, void* workspace,
                                     int64_t workspace_bytes, sm_stream_t stream) {
  GaPlan p;
  const int st = ga_plan(d, al16(x) && al16(dy) && al16(dx), true, &p);
  if (st != SM_OK) return st;
  hipStream_t s = sm_hip_stream(stream);
  if (p.items == 0) {          // no rows: the parameter gradients are sums over nothing
    if (dgamma && sm_zero_async(dgamma, sizeof(float) * d->channels, s) != hipSuccess) return SM_ERR_LAUNCH;
    if (dbeta && sm_zero_async(dbeta, sizeof(float) * d->channels, s) != hipSuccess) return SM_ERR_LAUNCH;
    return SM_OK;
  }
  if (!x || !dy || !stats || !al16(stats) || (p.bwd_ws > 0 && !workspace) || !al16(workspace)) return SM_ERR_BAD_ARG;
  if (workspace_bytes < p.bwd_ws) return SM_ERR_WORKSPACE;
  return ga_pick(p, d->dtype, GaBwd{p, x, dy, gamma, beta, stats, dx, dgamma, dbeta, workspace, s});
}
