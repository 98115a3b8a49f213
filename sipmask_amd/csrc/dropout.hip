// Dropout whose mask is a function of (seed, offset, element) -- philox.h -- optionally added to a residual:
//   y = keep * x / (1 - p) [+ residual],   dx = keep * dy / (1 - p) (the same kernel without the residual)
// Bound by memory (read x [and the residual], write y); nothing else is read or written.  A thread takes the 8 consecutive elements of
// one generator block where rows and alignment allow it.  268 800 x 256 bf16: 49 us = 5.6 TB/s (a copy of the same tensor: 47 us); the
// generator's share of the vector units is about half of that time.  Dropped elements are selected away, not multiplied by 0: Inf and
// NaN in x do not survive where keep = 0.
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "elem.h"
#include "philox.h"

namespace {

struct DoArgs {
  long long n, cols, ldx, ldr, ldy;   // n = rows * cols elements
  DropArgs drop;
};

// Any strides and alignment: a wave takes 512 consecutive elements, 64 neighbours at a time; lane l generates the bits of elements
// 8 l .. 8 l + 7 and fetches those of the others.  268 800 x 255 in rows of 512: f32 115 us, bf16 159 (2-byte stores); with a lane on
// eight neighbours 413 and 184.
template <int DT, bool RES>
__global__ __launch_bounds__(256) void dropout_any_kernel(const typename Elem<DT>::type* __restrict__ x,
                                                          const typename Elem<DT>::type* __restrict__ res,
                                                          typename Elem<DT>::type* __restrict__ y, const DoArgs a) {
  typedef Elem<DT> E;
  const unsigned long long off = drop_offset(a.drop);
  const int lane = threadIdx.x & 63;
  const long long step = (long long)gridDim.x * 2048, rows64 = 64 / a.cols, cols64 = 64 - rows64 * a.cols;
  // 64 elements on, and what is to be added where that crosses one row more
  const long long ax = rows64 * a.ldx + cols64, ar = rows64 * a.ldr + cols64, ay = rows64 * a.ldy + cols64;
  const long long wx = a.ldx - a.cols, wr = a.ldr - a.cols, wy = a.ldy - a.cols;
  for (long long i0 = ((long long)blockIdx.x * 4 + (threadIdx.x >> 6)) * 512; i0 < a.n; i0 += step) {
    const uint32_t keep = drop_keep8((unsigned long long)(i0 >> 3) + lane, off, a.drop.seed, a.drop.thr);
    const long long i = i0 + lane, r = a.n <= 0xffffffffll ? (uint32_t)i / (uint32_t)a.cols : i / a.cols;
    long long c = i - r * a.cols;
    const typename E::type* px = x + r * a.ldx + c;
    const typename E::type* pr = RES ? res + r * a.ldr + c : nullptr;
    typename E::type* py[8];
    py[0] = y + r * a.ldy + c;
    float v[8], g[8];
#pragma unroll
    for (int p = 0; p < 8; ++p) {                // all loads first: eight in flight
      v[p] = g[p] = 0.f;
      if (i + p * 64 < a.n) {
        v[p] = E::load(px);
        if constexpr (RES) g[p] = E::load(pr);
      }
      const bool wrap = (c += cols64) >= a.cols;
      if (wrap) c -= a.cols;
      px += ax + (wrap ? wx : 0);
      if constexpr (RES) pr += ar + (wrap ? wr : 0);
      if (p < 7) py[p + 1] = py[p] + ay + (wrap ? wy : 0);
    }
#pragma unroll
    for (int p = 0; p < 8; ++p) {
      const bool k = ((uint32_t)__shfl((int)keep, p * 8 + (lane >> 3), 64) >> (lane & 7)) & 1u;
      if constexpr (RES) v[p] = k ? __builtin_fmaf(v[p], a.drop.scale, g[p]) : g[p];
      else v[p] = k ? v[p] * a.drop.scale : 0.f;
      if (i + p * 64 < a.n) E::store(py[p], v[p]);
    }
  }
}

// MODE 0: dense rows, 16-byte accesses; 1: strided rows of a multiple of 8 columns, 16-byte accesses
template <int DT, int MODE, bool RES>
__global__ __launch_bounds__(256) void dropout_kernel(const typename Elem<DT>::type* __restrict__ x,
                                                      const typename Elem<DT>::type* __restrict__ res,
                                                      typename Elem<DT>::type* __restrict__ y, const DoArgs a) {
  typedef Elem<DT> E;
  const unsigned long long off = drop_offset(a.drop);
  const long long n8 = (a.n + 7) >> 3, step = (long long)gridDim.x * 256;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n8; i += step) {
    const uint32_t keep = drop_keep8((unsigned long long)i, off, a.drop.seed, a.drop.thr);
    if (8 * i + 8 <= a.n) {
      long long ox = 8 * i, orr = 8 * i, oy = 8 * i;
      if constexpr (MODE == 1) {
        const long long r = ox / a.cols, c = ox - r * a.cols;
        ox = r * a.ldx + c, orr = r * a.ldr + c, oy = r * a.ldy + c;
      }
      float f[8], g[8];
      const typename E::raw8 qx = E::load8(x + ox);
      if constexpr (RES) E::unpack(E::load8(res + orr), g);
      E::unpack(qx, f);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool k = (keep >> e) & 1u;
        if constexpr (RES) f[e] = k ? __builtin_fmaf(f[e], a.drop.scale, g[e]) : g[e];
        else f[e] = k ? f[e] * a.drop.scale : 0.f;
      }
      E::store8(y + oy, f);
    } else {                                     // the last, partial block
      long long r = 8 * i / a.cols, c = 8 * i - r * a.cols;
      for (int e = 0; e < 8 && 8 * i + e < a.n; ++e) {
        const bool k = (keep >> e) & 1u;
        float v = k ? E::load(x + r * a.ldx + c) : 0.f;
        if constexpr (RES) v = k ? __builtin_fmaf(v, a.drop.scale, E::load(res + r * a.ldr + c)) : E::load(res + r * a.ldr + c);
        else v *= a.drop.scale;
        E::store(y + r * a.ldy + c, v);
        if (++c == a.cols) c = 0, ++r;
      }
    }
  }
}

template <int DT>
int dropout_launch(const void* x, const void* res, void* y, const DoArgs& a, int mode, hipStream_t s) {
  typedef typename Elem<DT>::type T;
  const unsigned blocks = (unsigned)std::min<long long>(((a.n + 7) / 8 + 255) / 256, 256 * 64);
  auto go = [&](auto M, auto R) {
    constexpr int mode_c = decltype(M)::value;
    constexpr bool res_c = decltype(R)::value;
    if constexpr (mode_c == 2) hipLaunchKernelGGL((dropout_any_kernel<DT, res_c>), dim3(blocks), dim3(256), 0, s, (const T*)x, (const T*)res, (T*)y, a);
    else hipLaunchKernelGGL((dropout_kernel<DT, mode_c, res_c>), dim3(blocks), dim3(256), 0, s, (const T*)x, (const T*)res, (T*)y, a);
  };
  using std::integral_constant;
  auto with_res = [&](auto M) {
    if (res != nullptr) go(M, integral_constant<bool, true>{});
    else go(M, integral_constant<bool, false>{});
  };
  if (mode == 0) with_res(integral_constant<int, 0>{});
  else if (mode == 1) with_res(integral_constant<int, 1>{});
  else with_res(integral_constant<int, 2>{});
  SM_LAUNCH_CHECK();
  return SM_OK;
}

}  // namespace

extern "C" int sm_dropout(int dtype, const void* x, const void* residual, void* y, int64_t rows, int64_t cols, int64_t x_stride,
                          int64_t res_stride, int64_t y_stride, int drop_threshold, uint64_t seed, uint64_t offset,
                          const int64_t* offset_dev, sm_stream_t stream) {
  if (dtype < SM_DT_BF16 || dtype > SM_DT_F32) return SM_ERR_BAD_ARG;
  if (rows < 0 || cols < 0) return SM_ERR_BAD_SHAPE;
  DoArgs a;
  const int st = drop_args_fill(&a.drop, drop_threshold, seed, offset, offset_dev);
  if (st != SM_OK) return st;
  if (rows == 0 || cols == 0) return SM_OK;
  if (!x || !y) return SM_ERR_BAD_ARG;
  if (x_stride < cols || y_stride < cols || (residual && res_stride < cols) || cols > INT64_MAX / 8 / rows) return SM_ERR_BAD_SHAPE;
  a.n = rows * cols, a.cols = cols, a.ldx = x_stride, a.ldr = residual ? res_stride : cols, a.ldy = y_stride;
  const bool al = (((uintptr_t)x | (uintptr_t)residual | (uintptr_t)y) & 15) == 0;
  const bool dense = (a.ldx == cols && a.ldr == cols && a.ldy == cols) || rows == 1;
  const int per16 = 16 / sm_dtype_bytes(dtype);
  const int mode = al && dense ? 0 : (al && cols % 8 == 0 && a.ldx % per16 == 0 && a.ldr % per16 == 0 && a.ldy % per16 == 0 ? 1 : 2);
  hipStream_t s = sm_hip_stream(stream);
  if (dtype == SM_DT_BF16) return dropout_launch<SM_DT_BF16>(x, residual, y, a, mode, s);
  if (dtype == SM_DT_F16) return dropout_launch<SM_DT_F16>(x, residual, y, a, mode, s);
  return dropout_launch<SM_DT_F32>(x, residual, y, a, mode, s);
}
