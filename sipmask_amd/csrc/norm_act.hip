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
// The sums are held in f64: x and x^2 add exactly enough that E[x^2] - m^2 keeps its digits for |m| >> sqrt(v) (1e4 standard deviations
// cost 1e-8), and three f64 operations per element stay under the memory time for 16-bit rows.
#include <algorithm>

#include "common.h"
#include "elem.h"
#include "philox.h"

namespace {

constexpr int GA_THREADS = 256;
constexpr int GA_TILE = 32;         // column vectors per block: 512-byte row segments for 16-bit types
constexpr int GA_TILE1 = 64;        // columns per block of the any-alignment path
constexpr int GA_COMBINE = 2048;    // partial entries a block of the second launch may add up (32 KB out of L2)
constexpr int GA_GPT = 256;         // groups that a column tile can touch (32 vectors of 8 channels, one channel per group)

struct GaArgs {
  int nlev, batch, C, G, cpg, act;
  int cols, ct, lanes, ntile;       // column vectors, per block, row lanes of a block, column tiles
  long long hw[SM_MAX_LEVELS], row0[SM_MAX_LEVELS];
  int sblk0[SM_MAX_LEVELS + 1];     // first split of each level (per image); partials of a level are hw / srpb apart
  int ablk0[SM_MAX_LEVELS + 1];     // the same for the element-wise launch
  int srpb[SM_MAX_LEVELS], arpb;    // rows per block
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

// sum over the block's row lanes of NV values per thread, left on the threads of lane 0 (fixed tree)
template <int NV, typename V>
__device__ __forceinline__ void lane_tree(V (*sh)[GA_THREADS], V (&v)[NV], int lane, int ct, int lanes) {
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

// launch 1, forward: part[image][split][tile][group - first group of the tile] = (sum x, sum x^2)
// WHOLE: a vector lies in one group (cpg % VEC == 0), so a thread needs two sums instead of 2 * VEC
template <int DT, int VEC, bool WHOLE>
__global__ __launch_bounds__(GA_THREADS) void ga_stats_kernel(const typename Elem<DT>::type* __restrict__ x, double2* __restrict__ part,
                                                              const GaArgs a, int gpt) {
  typedef RowVec<DT, VEC> RV;
  constexpr int NS = WHOLE ? 1 : VEC;
  __shared__ double sh[2 * NS][GA_THREADS];
  const int nsplit = a.sblk0[a.nlev];
  const int n = blockIdx.x / nsplit, b = blockIdx.x - n * nsplit, tile = blockIdx.y;
  const int lev = ga_level(a.sblk0, a.nlev, b);
  const long long rb = (long long)(b - a.sblk0[lev]) * a.srpb[lev], re = min(rb + (long long)a.srpb[lev], a.hw[lev]);
  const int cl = threadIdx.x % a.ct, lane = threadIdx.x / a.ct, col = tile * a.ct + cl;
  const bool live = lane < a.lanes && col < a.cols;
  double v[2 * NS];
#pragma unroll
  for (int k = 0; k < 2 * NS; ++k) v[k] = 0.0;
  if (live) {
    const typename Elem<DT>::type* p = x + (a.row0[lev] + (long long)n * a.hw[lev]) * a.ldx + (long long)col * VEC;
    auto add = [&](const typename RV::raw& q) {
      float f[VEC];
      RV::unpack(q, f);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const double d = (double)f[e];
        const int k = WHOLE ? 0 : e;
        v[k] += d;
        v[NS + k] = __builtin_fma(d, d, v[NS + k]);
      }
    };
    long long r = rb + lane;
    for (; r + 3 * a.lanes < re; r += 4 * a.lanes) {     // four loads in flight
      typename RV::raw q[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) q[u] = RV::load(p + (r + u * a.lanes) * a.ldx);
#pragma unroll
      for (int u = 0; u < 4; ++u) add(q[u]);
    }
    for (; r < re; r += a.lanes) add(RV::load(p + r * a.ldx));
  }
  lane_tree<2 * NS>(sh, v, lane, a.ct, a.lanes);
  // one thread per group of the tile adds its channels
  const int c0 = tile * a.ct * VEC, c1 = min(c0 + a.ct * VEC, a.C);
  const int g0 = c0 / a.cpg, g1 = (c1 - 1) / a.cpg;
  for (int g = g0 + threadIdx.x; g <= g1; g += GA_THREADS) {
    const int lo = max(g * a.cpg, c0) - c0, hi = min((g + 1) * a.cpg, c1) - c0;
    double s = 0.0, ss = 0.0;
    if constexpr (WHOLE) {
      for (int k = lo / VEC; k < hi / VEC; ++k) s += sh[0][k], ss += sh[1][k];
    } else {
      for (int c = lo; c < hi; ++c) s += sh[c % VEC][c / VEC], ss += sh[NS + c % VEC][c / VEC];
    }
    part[((long long)blockIdx.x * a.ntile + tile) * gpt + (g - g0)] = make_double2(s, ss);
  }
}

// (mean, rstd) of every group of this block's column tile from the partials, into LDS; the block that owns a (level, first row
// block) also writes them out for the backward pass.  Threads share a group's entries and join in a fixed order.
template <int VEC>
__device__ __forceinline__ void ga_combine(const double2* __restrict__ part, double2* __restrict__ stats, double2* s_stat, double2* s_red,
                                           const GaArgs& a, int gpt, int n, int lev, int tile, bool publish) {
  const int tc = a.ct * VEC;
  const int c0 = tile * tc, c1 = min(c0 + tc, a.C);
  const int g0 = c0 / a.cpg, ng = (c1 - 1) / a.cpg - g0 + 1;
  const int nsplit = a.sblk0[a.nlev], s0 = a.sblk0[lev], ns = a.sblk0[lev + 1] - s0;
  int tpg = 1;                                   // threads per group, a power of two
  while (tpg * 2 * ng <= GA_THREADS) tpg <<= 1;
  const int gi = threadIdx.x / tpg, ti = threadIdx.x - gi * tpg;
  double s = 0.0, ss = 0.0;
  if (gi < ng) {
    const int g = g0 + gi;
    const int t0 = g * a.cpg / tc, t1 = ((g + 1) * a.cpg - 1) / tc;
    for (int t = t0; t <= t1; ++t) {
      const int slot = g - t * tc / a.cpg;
      const double2* q = part + (((long long)n * nsplit + s0) * a.ntile + t) * gpt + slot;
      for (int i = ti; i < ns; i += tpg) {
        const double2 e = q[(long long)i * a.ntile * gpt];
        s += e.x, ss += e.y;
      }
    }
  }
  s_red[threadIdx.x] = make_double2(s, ss);
  __syncthreads();
  if (gi < ng && ti == 0) {
    for (int k = 1; k < tpg; ++k) {
      const double2 e = s_red[threadIdx.x + k];
      s += e.x, ss += e.y;
    }
    const double cnt = (double)a.hw[lev] * (double)a.cpg, m = s / cnt;
    double var = ss / cnt - m * m;
    var = var < 0.0 ? 0.0 : var;                 // (NaN stays NaN)
    const double2 st = make_double2(m, 1.0 / sqrt(var + (double)a.eps));
    s_stat[gi] = st;
    const int g = g0 + gi;
    if (publish && g * a.cpg >= c0) stats[((long long)n * a.nlev + lev) * a.G + g] = st;   // (the tile that a group starts in)
  }
  __syncthreads();
}

// launch 2, forward
template <int DT, int VEC, bool WHOLE, int ACT, bool DROP>
__global__ __launch_bounds__(GA_THREADS) void ga_apply_kernel(const typename Elem<DT>::type* __restrict__ x,
                                                              typename Elem<DT>::type* __restrict__ y, const float* __restrict__ gamma,
                                                              const float* __restrict__ beta, const double2* __restrict__ part,
                                                              double2* __restrict__ stats, const GaArgs a, int gpt) {
  typedef RowVec<DT, VEC> RV;
  __shared__ double2 s_stat[GA_GPT], s_red[GA_THREADS];
  const int nblk = a.ablk0[a.nlev];
  const int n = blockIdx.x / nblk, b = blockIdx.x - n * nblk, tile = blockIdx.y;
  const int lev = ga_level(a.ablk0, a.nlev, b);
  ga_combine<VEC>(part, stats, s_stat, s_red, a, gpt, n, lev, tile, b == a.ablk0[lev] && stats != nullptr);
  const long long rb = (long long)(b - a.ablk0[lev]) * a.arpb, re = min(rb + (long long)a.arpb, a.hw[lev]);
  const int cl = threadIdx.x % a.ct, lane = threadIdx.x / a.ct, col = tile * a.ct + cl;
  if (lane >= a.lanes || col >= a.cols) return;
  const int g0 = tile * a.ct * VEC / a.cpg;
  constexpr int NS = WHOLE ? 1 : VEC;
  float mh[NS], ml[NS], ga[VEC], be[VEC];     // the mean as a sum of two floats: x - m keeps its digits for |m| >> sqrt(v)
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    const int c = col * VEC + e;
    const double2 st = s_stat[c / a.cpg - g0];
    if (!WHOLE || e == 0) {
      mh[WHOLE ? 0 : e] = (float)st.x;
      ml[WHOLE ? 0 : e] = (float)(st.x - (double)(float)st.x);
    }
    ga[e] = (float)(st.y * (gamma != nullptr ? (double)gamma[c] : 1.0));
    be[e] = beta != nullptr ? beta[c] : 0.f;
  }
  const unsigned long long off = DROP ? drop_offset(a.drop) : 0ull;
  const long long row_base = a.row0[lev] + (long long)n * a.hw[lev];
  const typename Elem<DT>::type* px = x + row_base * a.ldx + (long long)col * VEC;
  typename Elem<DT>::type* py = y + row_base * a.ldy + (long long)col * VEC;
  auto one = [&](const typename RV::raw& q, long long r) {
    float f[VEC];
    RV::unpack(q, f);
    uint32_t keep = 0xffu;
    if constexpr (DROP) {
      const unsigned long long i = (unsigned long long)(row_base + r) * a.C + (unsigned long long)col * VEC;
      keep = drop_keep8(i >> 3, off, a.drop.seed, a.drop.thr);
      if constexpr (VEC == 1) keep >>= (int)(i & 7);
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const int k = WHOLE ? 0 : e;
      f[e] = act_fwd<ACT>(__builtin_fmaf((f[e] - mh[k]) - ml[k], ga[e], be[e]));
      if constexpr (DROP) f[e] = (keep >> e) & 1u ? f[e] * a.drop.scale : 0.f;
    }
    RV::store(py + r * a.ldy, f);
  };
  long long r = rb + lane;
  for (; r + 3 * a.lanes < re; r += 4 * a.lanes) {
    typename RV::raw q[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) q[u] = RV::load(px + (r + u * a.lanes) * a.ldx);
#pragma unroll
    for (int u = 0; u < 4; ++u) one(q[u], r + u * a.lanes);
  }
  for (; r < re; r += a.lanes) one(RV::load(px + r * a.ldx), r);
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
  // xhat and d = dy * keep / (1 - p) * act'(t) of one element
  template <int ACT, bool DROP>
  __device__ __forceinline__ void grad(float x, float dy, int e, uint32_t keep, float scale, float& xh, float& d) const {
    const int k = WHOLE ? 0 : e;
    xh = ((x - mh[k]) - ml[k]) * rs[k];
    d = dy;
    if constexpr (DROP) d = (keep >> e) & 1u ? d * scale : 0.f;
    if constexpr (ACT == SM_ACT_NONE) return;
    float t = __builtin_fmaf(xh, ga[e], be[e]);
    if constexpr (ACT == SM_ACT_RELU) {
      // the ReLU passes the whole gradient or nothing: within rounding of the border (t = xh * gamma + beta is off by at most
      // 3 * 2^-24 (|xh gamma| + |beta|), and near 0 the two are alike) t is taken in f64
      if (__builtin_fabsf(t) <= 1e-6f * __builtin_fabsf(be[e])) {
        const double t64 = ((double)x - st[k].x) * st[k].y * (double)ga[e] + (double)be[e];
        t = t64 > 0.0 ? 1.f : (t64 <= 0.0 ? -1.f : t);
      }
      d = t <= 0.f ? 0.f : d;
    } else {
      d *= act_grad<ACT>(t);
    }
  }
};

// launch 1, backward: part[image][split][channel] = (sum d, sum d xhat) of the split's rows
template <int DT, int VEC, bool WHOLE, int ACT, bool DROP>
__global__ __launch_bounds__(GA_THREADS) void ga_bwd_sum_kernel(const typename Elem<DT>::type* __restrict__ x,
                                                                const typename Elem<DT>::type* __restrict__ dy,
                                                                const float* __restrict__ gamma, const float* __restrict__ beta,
                                                                const double2* __restrict__ stats, float2* __restrict__ part,
                                                                const GaArgs a) {
  typedef RowVec<DT, VEC> RV;
  __shared__ float sh[2 * VEC][GA_THREADS];
  const int nsplit = a.sblk0[a.nlev];
  const int n = blockIdx.x / nsplit, b = blockIdx.x - n * nsplit, tile = blockIdx.y;
  const int lev = ga_level(a.sblk0, a.nlev, b);
  const long long rb = (long long)(b - a.sblk0[lev]) * a.srpb[lev], re = min(rb + (long long)a.srpb[lev], a.hw[lev]);
  const int cl = threadIdx.x % a.ct, lane = threadIdx.x / a.ct, col = tile * a.ct + cl;
  const bool live = lane < a.lanes && col < a.cols;
  float v[2 * VEC];
#pragma unroll
  for (int k = 0; k < 2 * VEC; ++k) v[k] = 0.f;
  if (live) {
    GaChan<VEC, WHOLE> ch;
    ch.fill(a, stats, gamma, beta, ((long long)n * a.nlev + lev) * a.G, col);
    const unsigned long long off = DROP ? drop_offset(a.drop) : 0ull;
    const long long row_base = a.row0[lev] + (long long)n * a.hw[lev];
    const typename Elem<DT>::type* px = x + row_base * a.ldx + (long long)col * VEC;
    const typename Elem<DT>::type* pd = dy + row_base * a.lddy + (long long)col * VEC;
    auto one = [&](const typename RV::raw& qx, const typename RV::raw& qd, long long r) {
      float fx[VEC], fd[VEC];
      RV::unpack(qx, fx);
      RV::unpack(qd, fd);
      uint32_t keep = 0xffu;
      if constexpr (DROP) {
        const unsigned long long i = (unsigned long long)(row_base + r) * a.C + (unsigned long long)col * VEC;
        keep = drop_keep8(i >> 3, off, a.drop.seed, a.drop.thr);
        if constexpr (VEC == 1) keep >>= (int)(i & 7);
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        float xh, d;
        ch.template grad<ACT, DROP>(fx[e], fd[e], e, keep, a.drop.scale, xh, d);
        v[e] += d;
        v[VEC + e] = __builtin_fmaf(d, xh, v[VEC + e]);
      }
    };
    long long r = rb + lane;
    for (; r + a.lanes < re; r += 2 * a.lanes) {
      typename RV::raw qx[2], qd[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) qx[u] = RV::load(px + (r + u * a.lanes) * a.ldx), qd[u] = RV::load(pd + (r + u * a.lanes) * a.lddy);
#pragma unroll
      for (int u = 0; u < 2; ++u) one(qx[u], qd[u], r + u * a.lanes);
    }
    for (; r < re; r += a.lanes) one(RV::load(px + r * a.ldx), RV::load(pd + r * a.lddy), r);
  }
  lane_tree<2 * VEC>(sh, v, lane, a.ct, a.lanes);
  const int c0 = tile * a.ct * VEC, nc = min(a.ct * VEC, a.C - c0);
  for (int c = threadIdx.x; c < nc; c += GA_THREADS)
    part[(long long)blockIdx.x * a.C + c0 + c] = make_float2(sh[c % VEC][c / VEC], sh[VEC + c % VEC][c / VEC]);
}

// launch 2, backward: per (image, level) the channel sums chan[c] = (sum d, sum d xhat) and the group means
// gmean[g] = (mean d gamma, mean d gamma xhat).  A block takes gb whole groups, 32 channels x 8 slices of the splits at a time.
__global__ __launch_bounds__(GA_THREADS) void ga_bwd_combine_kernel(const float2* __restrict__ part, const float* __restrict__ gamma,
                                                                    double2* __restrict__ chan, double2* __restrict__ gmean, const GaArgs a,
                                                                    int gb) {
  __shared__ double2 sh[8][32];
  const int nl = blockIdx.x, n = nl / a.nlev, lev = nl - n * a.nlev;
  const int nsplit = a.sblk0[a.nlev], s0 = a.sblk0[lev], ns = a.sblk0[lev + 1] - s0;
  const int g0 = blockIdx.y * gb, g1 = min(g0 + gb, a.G);
  const int ci = threadIdx.x & 31, sl = threadIdx.x >> 5;
  const double cnt = (double)a.hw[lev] * (double)a.cpg;
  for (int c0 = g0 * a.cpg; c0 < g1 * a.cpg; c0 += 32) {
    const int c = c0 + ci;
    double s = 0.0, ss = 0.0;
    if (c < g1 * a.cpg)
      for (int i = sl; i < ns; i += 8) {
        const float2 e = part[((long long)n * nsplit + s0 + i) * a.C + c];
        s += (double)e.x, ss += (double)e.y;
      }
    __syncthreads();
    sh[sl][ci] = make_double2(s, ss);
    __syncthreads();
    if (sl == 0 && c < g1 * a.cpg) {
      for (int k = 1; k < 8; ++k) s += sh[k][ci].x, ss += sh[k][ci].y;
      chan[(long long)nl * a.C + c] = make_double2(s, ss);
    }
  }
  __syncthreads();                               // (the block's own global writes are visible to it behind the barrier)
  for (int g = g0 + threadIdx.x; g < g1; g += GA_THREADS) {
    double m1 = 0.0, m2 = 0.0;
    for (int c = g * a.cpg; c < (g + 1) * a.cpg; ++c) {
      const double2 e = chan[(long long)nl * a.C + c];
      const double w = gamma != nullptr ? (double)gamma[c] : 1.0;
      m1 += w * e.x, m2 += w * e.y;
    }
    gmean[(long long)nl * a.G + g] = make_double2(m1 / cnt, m2 / cnt);
  }
}

// launch 3, backward: dx element by element; the blocks behind the last row block add up dgamma / dbeta over images and levels
template <int DT, int VEC, bool WHOLE, int ACT, bool DROP>
__global__ __launch_bounds__(GA_THREADS) void ga_bwd_apply_kernel(const typename Elem<DT>::type* __restrict__ x,
                                                                  const typename Elem<DT>::type* __restrict__ dy,
                                                                  const float* __restrict__ gamma, const float* __restrict__ beta,
                                                                  const double2* __restrict__ stats, const double2* __restrict__ chan,
                                                                  const double2* __restrict__ gmean, typename Elem<DT>::type* __restrict__ dx,
                                                                  float* __restrict__ dgamma, float* __restrict__ dbeta, const GaArgs a,
                                                                  long long nrow_blocks) {
  typedef RowVec<DT, VEC> RV;
  __shared__ double2 sh[8][32];
  if ((long long)blockIdx.x >= nrow_blocks) {
    if (blockIdx.y != 0) return;
    const int ci = threadIdx.x & 31, sl = threadIdx.x >> 5;
    const int c = (int)(blockIdx.x - nrow_blocks) * 32 + ci;
    double s = 0.0, ss = 0.0;
    if (c < a.C)
      for (int i = sl; i < a.batch * a.nlev; i += 8) {
        const double2 e = chan[(long long)i * a.C + c];
        s += e.x, ss += e.y;
      }
    sh[sl][ci] = make_double2(s, ss);
    __syncthreads();
    if (sl == 0 && c < a.C) {
      for (int k = 1; k < 8; ++k) s += sh[k][ci].x, ss += sh[k][ci].y;
      if (dbeta != nullptr) dbeta[c] = (float)s;
      if (dgamma != nullptr) dgamma[c] = (float)ss;
    }
    return;
  }
  const int nblk = a.ablk0[a.nlev];
  const int n = blockIdx.x / nblk, b = blockIdx.x - n * nblk, tile = blockIdx.y;
  const int lev = ga_level(a.ablk0, a.nlev, b);
  const long long rb = (long long)(b - a.ablk0[lev]) * a.arpb, re = min(rb + (long long)a.arpb, a.hw[lev]);
  const int cl = threadIdx.x % a.ct, lane = threadIdx.x / a.ct, col = tile * a.ct + cl;
  if (lane >= a.lanes || col >= a.cols) return;
  GaChan<VEC, WHOLE> ch;
  const long long sbase = ((long long)n * a.nlev + lev) * a.G;
  ch.fill(a, stats, gamma, beta, sbase, col);
  constexpr int NS = WHOLE ? 1 : VEC;
  float m1[NS], m2[NS];
#pragma unroll
  for (int k = 0; k < NS; ++k) {
    const double2 e = gmean[sbase + (col * VEC + k) / a.cpg];
    m1[k] = (float)e.x, m2[k] = (float)e.y;
  }
  const unsigned long long off = DROP ? drop_offset(a.drop) : 0ull;
  const long long row_base = a.row0[lev] + (long long)n * a.hw[lev];
  const typename Elem<DT>::type* px = x + row_base * a.ldx + (long long)col * VEC;
  const typename Elem<DT>::type* pd = dy + row_base * a.lddy + (long long)col * VEC;
  typename Elem<DT>::type* po = dx + row_base * a.lddx + (long long)col * VEC;
  auto one = [&](const typename RV::raw& qx, const typename RV::raw& qd, long long r) {
    float fx[VEC], fd[VEC];
    RV::unpack(qx, fx);
    RV::unpack(qd, fd);
    uint32_t keep = 0xffu;
    if constexpr (DROP) {
      const unsigned long long i = (unsigned long long)(row_base + r) * a.C + (unsigned long long)col * VEC;
      keep = drop_keep8(i >> 3, off, a.drop.seed, a.drop.thr);
      if constexpr (VEC == 1) keep >>= (int)(i & 7);
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const int k = WHOLE ? 0 : e;
      float xh, d;
      ch.template grad<ACT, DROP>(fx[e], fd[e], e, keep, a.drop.scale, xh, d);
      fx[e] = ch.rs[k] * (__builtin_fmaf(d, ch.ga[e], -m1[k]) - xh * m2[k]);
    }
    RV::store(po + r * a.lddx, fx);
  };
  long long r = rb + lane;
  for (; r + a.lanes < re; r += 2 * a.lanes) {
    typename RV::raw qx[2], qd[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) qx[u] = RV::load(px + (r + u * a.lanes) * a.ldx), qd[u] = RV::load(pd + (r + u * a.lanes) * a.lddy);
#pragma unroll
    for (int u = 0; u < 2; ++u) one(qx[u], qd[u], r + u * a.lanes);
  }
  for (; r < re; r += a.lanes) one(RV::load(px + r * a.ldx), RV::load(pd + r * a.lddy), r);
}

struct GaPlan {
  GaArgs a;
  bool vec, whole;
  int gpt;                          // groups per column tile (slots of a partial)
  long long items;                  // batch * splits of all levels
  long long ablocks;                // row blocks of the element-wise launch
  long long fwd_ws, bwd_ws;         // bytes
};

int ga_plan(const sm_gn_act_desc* d, bool aligned, GaPlan* p) {
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
  a.ct = std::min(a.cols, p->vec ? GA_TILE : GA_TILE1);
  a.lanes = GA_THREADS / a.ct;
  a.ntile = sm_cdiv(a.cols, a.ct);
  if (a.ntile > 65535 || a.G > 65535 * 32) return SM_ERR_UNSUPPORTED;
  const int tc = a.ct * vec;
  p->gpt = std::min(a.G, (tc - 1) / a.cpg + 2);
  if (p->gpt > tc) p->gpt = tc;
  // rows per block.  The second launch adds splits x tiles-of-a-group x groups-of-a-tile partials: at most GA_COMBINE of them
  const long long tiles_per_group = (a.cpg - 1) / tc + 2;
  const long long smax = std::max<long long>(4, std::min<long long>(256, GA_COMBINE / (tiles_per_group * p->gpt)));
  long long sb = 0, ab = 0, hw_sum = 0;
  for (int l = 0; l < d->nlev; ++l) hw_sum += d->hw[l] > 0 ? d->hw[l] : 0;
  // element-wise blocks: about 2048 of them over the chip, between 8 and 32 rows per row lane
  const long long want = hw_sum * (long long)a.batch * a.ntile / 2048;
  a.arpb = (int)std::max<long long>(8 * a.lanes, std::min<long long>(32 * a.lanes, want));
  for (int l = 0; l < d->nlev; ++l) {
    if (d->hw[l] < 0 || d->row0[l] < 0) return SM_ERR_BAD_SHAPE;
    a.hw[l] = d->hw[l], a.row0[l] = d->row0[l];
    const long long rpb = std::max<long long>((d->hw[l] + smax - 1) / smax, 4 * a.lanes);
    if (rpb > 0x3fffffff) return SM_ERR_UNSUPPORTED;
    a.srpb[l] = (int)rpb;
    a.sblk0[l] = (int)sb, a.ablk0[l] = (int)ab;
    sb += (d->hw[l] + rpb - 1) / rpb;
    ab += (d->hw[l] + a.arpb - 1) / a.arpb;
    if (ab > 0x7fffffff) return SM_ERR_UNSUPPORTED;
  }
  for (int l = d->nlev; l <= SM_MAX_LEVELS; ++l) a.sblk0[l] = (int)sb, a.ablk0[l] = (int)ab;
  p->items = sb * a.batch, p->ablocks = ab * a.batch;
  // (256 threads a block: a launch dimension holds fewer than 2^32 threads)
  if (p->items > 0xfff000 || p->ablocks > 0xff0000 || (long long)a.batch * a.nlev > 0xfff000) return SM_ERR_UNSUPPORTED;
  p->fwd_ws = p->items * a.ntile * p->gpt * 16;
  const long long nl = (long long)a.batch * a.nlev;
  p->bwd_ws = (p->items * a.C * 8 + 15) / 16 * 16 + nl * a.C * 16 + nl * a.G * 16;
  return SM_OK;
}

template <int DT, int VEC, bool WHOLE, int ACT, bool DROP>
int ga_fwd_launch(const GaPlan& p, const void* x, const float* gamma, const float* beta, void* y, void* stats, void* ws, hipStream_t s) {
  typedef typename Elem<DT>::type T;
  hipLaunchKernelGGL((ga_stats_kernel<DT, VEC, WHOLE>), dim3((unsigned)p.items, p.a.ntile), dim3(GA_THREADS), 0, s, (const T*)x,
                     (double2*)ws, p.a, p.gpt);
  hipLaunchKernelGGL((ga_apply_kernel<DT, VEC, WHOLE, ACT, DROP>), dim3((unsigned)p.ablocks, p.a.ntile), dim3(GA_THREADS), 0, s,
                     (const T*)x, (T*)y, gamma, beta, (const double2*)ws, (double2*)stats, p.a, p.gpt);
  SM_LAUNCH_CHECK();
  return SM_OK;
}

template <int DT, int VEC, bool WHOLE, int ACT, bool DROP>
int ga_bwd_launch(const GaPlan& p, const void* x, const void* dy, const float* gamma, const float* beta, const void* stats, void* dx,
                  float* dgamma, float* dbeta, void* ws, hipStream_t s) {
  typedef typename Elem<DT>::type T;
  const GaArgs& a = p.a;
  const long long nl = (long long)a.batch * a.nlev;
  float2* part = (float2*)ws;
  double2* chan = (double2*)((char*)ws + (p.items * a.C * 8 + 15) / 16 * 16);
  double2* gmean = chan + nl * a.C;
  hipLaunchKernelGGL((ga_bwd_sum_kernel<DT, VEC, WHOLE, ACT, DROP>), dim3((unsigned)p.items, a.ntile), dim3(GA_THREADS), 0, s,
                     (const T*)x, (const T*)dy, gamma, beta, (const double2*)stats, part, a);
  const int gb = std::max(1, 32 / a.cpg);
  hipLaunchKernelGGL(ga_bwd_combine_kernel, dim3((unsigned)nl, sm_cdiv(a.G, gb)), dim3(GA_THREADS), 0, s, part, gamma, chan, gmean, a, gb);
  const long long rowb = dx != nullptr ? p.ablocks : 0, chb = dgamma != nullptr || dbeta != nullptr ? sm_cdiv(a.C, 32) : 0;
  if (rowb + chb > 0)
    hipLaunchKernelGGL((ga_bwd_apply_kernel<DT, VEC, WHOLE, ACT, DROP>), dim3((unsigned)(rowb + chb), a.ntile), dim3(GA_THREADS), 0, s,
                       (const T*)x, (const T*)dy, gamma, beta, (const double2*)stats, (const double2*)chan, (const double2*)gmean,
                       (T*)dx, dgamma, dbeta, a, rowb);
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
  int64_t need = 16;
  for (int al = 0; al < 2; ++al) {
    GaPlan p;
    const int st = ga_plan(d, al != 0, &p);
    if (st != SM_OK) return st;
    need = std::max<int64_t>(need, backward ? p.bwd_ws : p.fwd_ws);
  }
  return need;
}

extern "C" int sm_group_norm_act(const sm_gn_act_desc* d, const void* x, const float* gamma, const float* beta, void* y, double* stats,
                                 void* workspace, int64_t workspace_bytes, sm_stream_t stream) {
  GaPlan p;
  const int st = ga_plan(d, al16(x) && al16(y), &p);
  if (st != SM_OK) return st;
  if (p.items == 0) return SM_OK;
  if (!x || !y || !workspace || !al16(workspace) || (stats != nullptr && !al16(stats))) return SM_ERR_BAD_ARG;
  if (workspace_bytes < p.fwd_ws) return SM_ERR_WORKSPACE;
  return ga_pick(p, d->dtype, GaFwd{p, x, gamma, beta, y, stats, workspace, sm_hip_stream(stream)});
}

extern "C" int sm_group_norm_act_bwd(const sm_gn_act_desc* d, const void* x, const void* dy, const float* gamma, const float* beta,
                                     const double* stats, void* dx, float* dgamma, float* dbeta, void* workspace,
                                     int64_t workspace_bytes, sm_stream_t stream) {
  GaPlan p;
  const int st = ga_plan(d, al16(x) && al16(dy) && al16(dx), &p);
  if (st != SM_OK) return st;
  hipStream_t s = sm_hip_stream(stream);
  if (p.items == 0) {          // no rows: the parameter gradients are sums over nothing
    if (dgamma && sm_zero_async(dgamma, sizeof(float) * d->channels, s) != hipSuccess) return SM_ERR_LAUNCH;
    if (dbeta && sm_zero_async(dbeta, sizeof(float) * d->channels, s) != hipSuccess) return SM_ERR_LAUNCH;
    return SM_OK;
  }
  if (!x || !dy || !stats || !al16(stats) || !workspace || !al16(workspace)) return SM_ERR_BAD_ARG;
  if (workspace_bytes < p.bwd_ws) return SM_ERR_WORKSPACE;
  return ga_pick(p, d->dtype, GaBwd{p, x, dy, gamma, beta, stats, dx, dgamma, dbeta, workspace, s});
}
