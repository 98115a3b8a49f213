// 8-bit products with a power-of-two scale per block of 128: quantiser, product, column sums.
//
//   scale_b = smallest 2^e (e >= -127) with max |x| / 2^e <= 448 over the block (1 for a block of zeros), code = e4m3(x / 2^e)
//   y[m][n] = sum_kb 2^(ea[m][kb] + eb[n][kb]) sum_{k in kb} a[m][k] b[n][k] (+ bias_n) (+ residual) (ReLU)
//
// Why powers of two: x / 2^e is exact (the one rounding is the one to e4m3), e4m3's own exponent hides the up to one binary digit of
// range that a power of two gives away, and the scale enters the product for nothing: v_cvt_scalef32_pk_bf16_fp8 multiplies by it while
// it widens two codes.
//
// Why bf16 MFMAs and not the 8-bit ones: a code times a power of two is exact in bf16, and v_mfma_f32_32x32x16_bf16 adds the exact
// products in f32.  The 8-bit MFMAs (plain and block-scaled) align the products of an instruction to the largest one and drop what
// lies 2^-14 below it (measured with one large and one small product; sums of 64 products over 8 binades were off by 2^-12 of the
// largest): less than f32 sums.  The price is the matrix peak, 2.5 instead of 5 PFLOP/s; the widening itself hides behind the MFMAs
// (one conversion is 8 cycles; 16 of them beside 4 MFMAs measured 161 cycles against 154 for the MFMAs alone), and the bytes moved
// through HBM and LDS stay 8-bit.
//
// Layout of a quantised matrix: codes [rows][Kp] with Kp = K rounded up to 128 (the tail is zero codes), scales
// [row blocks][Kb4], Kb4 = K blocks rounded up to 4 (a K loop reads four scales of a row as one dword; padding = 127, i.e. 1).
#include <algorithm>

#include "common.h"
#include "elem.h"

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

namespace {

// ------------------------------------------------------------------------------------------------ quantiser
// biased exponent of the block's scale: 1.m * 2^(E-127) <= 1.75 * 2^(8+e)
__device__ __forceinline__ int fp8_scale_byte(float amax) {
  const uint32_t u = __float_as_uint(amax);
  if (u == 0u) return 127;
  const int e = (int)(u >> 23) - 135 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return (e < -127 ? -127 : e) + 127;
}
// 2^-e of a scale byte: 254 - byte is a normal exponent for every byte the quantiser makes (0 .. 247)
__device__ __forceinline__ float fp8_inv_scale(int byte) { return __uint_as_float((uint32_t)(254 - byte) << 23); }

// Inf and NaN have no code but NaN: they are left out of the block's maximum and stored as NaN
__device__ __forceinline__ float fp8_abs_finite(float x) {
  const float a = __builtin_fabsf(x);
  return a <= 3.402823466e38f ? a : 0.f;
}
__device__ __forceinline__ float fp8_prep(float x, float inv) {
  return __builtin_fabsf(x) <= 3.402823466e38f ? x * inv : __uint_as_float(0x7fc00000u);
}
__device__ __forceinline__ uint2 fp8_pack8(const float* f, float inv) {
  int lo = 0, hi = 0;
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(fp8_prep(f[0], inv), fp8_prep(f[1], inv), lo, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(fp8_prep(f[2], inv), fp8_prep(f[3], inv), lo, true);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(fp8_prep(f[4], inv), fp8_prep(f[5], inv), hi, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(fp8_prep(f[6], inv), fp8_prep(f[7], inv), hi, true);
  return make_uint2((uint32_t)lo, (uint32_t)hi);
}

// 8 consecutive values of a row from column c; columns >= cols read as 0
template <int DT, bool VEC>
__device__ __forceinline__ void fp8_load8(const typename Elem<DT>::type* row, long long c, long long cols, float* f) {
  if (VEC && c + 8 <= cols) {
    Elem<DT>::unpack(Elem<DT>::load8(row + c), f);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = c + e < cols ? Elem<DT>::load(row + c + e) : 0.f;
  }
}

// 1 x 128 blocks along the row: 16 threads per block of 128, 8 values each
template <int DT, bool VEC>
__global__ __launch_bounds__(256) void fp8_quant_rows_kernel(const typename Elem<DT>::type* __restrict__ x, long long rows, long long cols,
                                                             long long ldx, int kb4, long long kp, uint8_t* __restrict__ q,
                                                             uint8_t* __restrict__ scale) {
  const long long units = rows * kb4;
  for (long long u = (long long)blockIdx.x * 16 + (threadIdx.x >> 4); u < units; u += (long long)gridDim.x * 16) {
    const long long r = u / kb4;
    const int kb = (int)(u - r * kb4), l = threadIdx.x & 15;
    if ((long long)kb * 128 >= kp) {             // padding of the scale row
      if (l == 0) scale[u] = 127;
      continue;
    }
    float f[8];
    fp8_load8<DT, VEC>(x + r * ldx, (long long)kb * 128 + l * 8, cols, f);
    float m = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = fmaxf(m, fp8_abs_finite(f[e]));
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
    const int sb = fp8_scale_byte(m);
    *reinterpret_cast<uint2*>(q + r * kp + (long long)kb * 128 + l * 8) = fp8_pack8(f, fp8_inv_scale(sb));
    if (l == 0) scale[u] = (uint8_t)sb;
  }
}

// One 128 x 64 piece (rows x columns) per block, 8 columns x 4 rows per thread.
//   TRANS   codes go to q[column][row], blocks run along the rows: 1 x 128 (SQUARE false) or 128 x 128 (SQUARE true)
//   !TRANS  codes go to q[row][column], 128 x 128 blocks (SQUARE)
// A 128 x 128 block is two pieces: each reads the other half once more for its maximum (weights only: megabytes at most).
template <int DT, bool VEC, bool TRANS, bool SQUARE>
__global__ __launch_bounds__(256) void fp8_quant_tile_kernel(const typename Elem<DT>::type* __restrict__ x, long long rows, long long cols,
                                                             long long ldx, int kb4, long long kp, uint8_t* __restrict__ q,
                                                             uint8_t* __restrict__ scale) {
  __shared__ float s_max[32][64 + 1];
  __shared__ int s_byte[64];
  __shared__ __attribute__((aligned(16))) uint8_t s_q[64][128 + 16];
  const long long rb = blockIdx.x, r0 = rb * 128, c0 = (long long)blockIdx.y * 64;
  const int cv = threadIdx.x & 7, rl = threadIdx.x >> 3;
  float f[4][8], m[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) m[e] = 0.f;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const long long r = r0 + u * 32 + rl;
    if (r < rows) {
      fp8_load8<DT, VEC>(x + r * ldx, c0 + cv * 8, cols, f[u]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[u][e] = 0.f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) m[e] = fmaxf(m[e], fp8_abs_finite(f[u][e]));
  }
  if constexpr (SQUARE) {
    const long long co = c0 ^ 64;                // the block's other half
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const long long r = r0 + u * 32 + rl;
      if (r < rows) {
        float g[8];
        fp8_load8<DT, VEC>(x + r * ldx, co + cv * 8, cols, g);
#pragma unroll
        for (int e = 0; e < 8; ++e) m[e] = fmaxf(m[e], fp8_abs_finite(g[e]));
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) s_max[rl][cv * 8 + e] = m[e];
  __syncthreads();
  if (threadIdx.x < 64) {
    float t = 0.f;
    for (int k = 0; k < 32; ++k) t = fmaxf(t, s_max[k][threadIdx.x]);
    if constexpr (SQUARE) {
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) t = fmaxf(t, __shfl_xor(t, d, 64));
    }
    s_byte[threadIdx.x] = fp8_scale_byte(t);
  }
  __syncthreads();
  if constexpr (!TRANS) {
    const float inv = fp8_inv_scale(s_byte[0]);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const long long r = r0 + u * 32 + rl;
      if (r < rows && c0 + cv * 8 < kp) *reinterpret_cast<uint2*>(q + r * kp + c0 + cv * 8) = fp8_pack8(f[u], inv);
    }
    const int kb = (int)(c0 >> 7);
    if ((c0 & 64) == 0 && threadIdx.x == 0) scale[rb * kb4 + kb] = (uint8_t)s_byte[0];
    if (c0 + 128 >= kp && (c0 & 64) == 0 && threadIdx.x < 4 && kb + 1 + (int)threadIdx.x < kb4) scale[rb * kb4 + kb + 1 + threadIdx.x] = 127;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float inv = fp8_inv_scale(s_byte[cv * 8 + e]);
#pragma unroll
      for (int u = 0; u < 4; ++u)
        s_q[cv * 8 + e][u * 32 + rl] = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(fp8_prep(f[u][e], inv), 0.f, 0, false);
    }
    __syncthreads();
    const int kb = (int)rb;
    const bool last = r0 + 128 >= kp;            // the scale row's padding behind the last block
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int i = threadIdx.x + 256 * p, c = i >> 3, ch = i & 7;
      if (c0 + c < cols) *reinterpret_cast<uint4*>(q + (c0 + c) * kp + r0 + ch * 16) = *reinterpret_cast<const uint4*>(&s_q[c][ch * 16]);
    }
    if (threadIdx.x < 64 && c0 + threadIdx.x < cols) {
      const long long srow = SQUARE ? (c0 >> 7) : c0 + threadIdx.x;
      if (!SQUARE || (threadIdx.x == 0 && (c0 & 64) == 0)) {
        scale[srow * kb4 + kb] = (uint8_t)s_byte[threadIdx.x];
        if (last)
          for (int k = kb + 1; k < kb4; ++k) scale[srow * kb4 + k] = 127;
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------ column sums
// out[c] = sum over the rows, two launches, a fixed order: part[row block][c], then f64 over the row blocks
constexpr int CS_ROWS = 512;
template <int DT>
__global__ __launch_bounds__(256) void col_sum_kernel(const typename Elem<DT>::type* __restrict__ x, long long rows, int cols, long long ldx,
                                                      float* __restrict__ part) {
  __shared__ float sh[4][64];
  const int cl = threadIdx.x & 63, rl = threadIdx.x >> 6, c = blockIdx.x * 64 + cl;
  const long long r0 = (long long)blockIdx.y * CS_ROWS, r1 = r0 + CS_ROWS < rows ? r0 + CS_ROWS : rows;
  float s = 0.f;
  if (c < cols)
    for (long long r = r0 + rl; r < r1; r += 4) s += Elem<DT>::load(x + r * ldx + c);
  sh[rl][cl] = s;
  __syncthreads();
  if (rl == 0 && c < cols) part[(long long)blockIdx.y * cols + c] = (sh[0][cl] + sh[1][cl]) + (sh[2][cl] + sh[3][cl]);
}
__global__ __launch_bounds__(256) void col_sum_finish_kernel(const float* __restrict__ part, int nb, int cols, float* __restrict__ out) {
  __shared__ double sh[8][32];
  const int cl = threadIdx.x & 31, sl = threadIdx.x >> 5, c = blockIdx.x * 32 + cl;
  double s = 0.0;
  if (c < cols)
    for (int i = sl; i < nb; i += 8) s += (double)part[(long long)i * cols + c];
  sh[sl][cl] = s;
  __syncthreads();
  if (sl == 0 && c < cols) {
    for (int k = 1; k < 8; ++k) s += sh[k][cl];
    out[c] = (float)s;
  }
}

// ------------------------------------------------------------------------------------------------ product
struct MmArgs {
  const uint8_t *a, *b, *sa, *sb;    // activations [m][kp], weights [n][kp] and their scales
  const float* bias;
  const void* res;
  void* y;
  float* part;                       // [ksplit][m][n] when ksplit > 1
  long long m, ldy, ldr, kp;
  int n, nkb, kb4, sha, shb;         // sha / shb: row >> sh = row of the scale matrix
  int ksplit, relu, out, vec4;       // vec4: four consecutive n of y / residual are one aligned access
  int tm, tn;                        // tiles
};

__device__ __forceinline__ float mm_load(const void* p, int dt, long long i) {
  if (dt == SM_DT_BF16) return bf16_bits_to_f32(((const uint16_t*)p)[i]);
  if (dt == SM_DT_F16) return (float)((const _Float16*)p)[i];
  return ((const float*)p)[i];
}
__device__ __forceinline__ void mm_store(void* p, int dt, long long i, float v) {
  if (dt == SM_DT_BF16) ((uint16_t*)p)[i] = (uint16_t)f32_to_bf16_bits(v);
  else if (dt == SM_DT_F16) ((_Float16*)p)[i] = (_Float16)v;
  else ((float*)p)[i] = v;
}

// 2^(byte - 127) of the low byte (byte 0 = 2^-127 is a subnormal)
__device__ __forceinline__ float fp8_scale_float(uint32_t w) {
  const uint32_t u = (w & 0xffu) << 23;
  return __uint_as_float(u == 0u ? 0x00400000u : u);
}
// 8 codes (two dwords) times a power of two as bf16: exact
__device__ __forceinline__ bf16x8 fp8_widen8(int lo, int hi, float scale) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
  const auto ab = __builtin_shufflevector(a, b, 0, 1, 2, 3), cd = __builtin_shufflevector(c, d, 0, 1, 2, 3);
  return __builtin_shufflevector(ab, cd, 0, 1, 2, 3, 4, 5, 6, 7);
}

// bias, residual, ReLU and the store of four consecutive n (n0 a multiple of 4) of row m
__device__ __forceinline__ void mm_finish4(const MmArgs& a, long long m, int n0, float (&v)[4]) {
  if (a.vec4 && n0 + 4 <= a.n) {
    if (a.bias != nullptr) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += a.bias[n0 + e];
    }
    if (a.res != nullptr) {
      const long long o = m * a.ldr + n0;
      if (a.out == SM_DT_F32) {
        const float4 r = *reinterpret_cast<const float4*>((const float*)a.res + o);
        v[0] += r.x, v[1] += r.y, v[2] += r.z, v[3] += r.w;
      } else {
        const uint2 r = *reinterpret_cast<const uint2*>((const uint16_t*)a.res + o);
        const uint32_t w[2] = {r.x, r.y};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint16_t h = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
          v[e] += a.out == SM_DT_BF16 ? bf16_bits_to_f32(h) : (float)__builtin_bit_cast(_Float16, h);
        }
      }
    }
    if (a.relu) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = v[e] < 0.f ? 0.f : v[e];
    }
    const long long o = m * a.ldy + n0;
    if (a.out == SM_DT_F32) {
      *reinterpret_cast<float4*>((float*)a.y + o) = make_float4(v[0], v[1], v[2], v[3]);
    } else if (a.out == SM_DT_BF16) {
      *reinterpret_cast<uint2*>((uint16_t*)a.y + o) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
    } else {
      uint32_t h[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) h[e] = __builtin_bit_cast(uint16_t, (_Float16)v[e]);
      *reinterpret_cast<uint2*>((uint16_t*)a.y + o) = make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
    }
    return;
  }
  for (int e = 0; e < 4 && n0 + e < a.n; ++e) {
    float t = v[e];
    if (a.bias != nullptr) t += a.bias[n0 + e];
    if (a.res != nullptr) t += mm_load(a.res, a.out, m * a.ldr + n0 + e);
    if (a.relu) t = t < 0.f ? 0.f : t;
    mm_store(a.y, a.out, m * a.ldy + n0 + e, t);
  }
}

// Tile of BN weights x BM activations, waves of WN x WM, K steps of one block of 128 through two LDS stages filled by direct
// global -> LDS loads.  A row of a stage is the 128 codes of one K block = 8 chunks of 16 bytes; chunk c of row r lies at slot
// c ^ (r & 7), so the 32 rows that one fragment read touches spread over all banks.  The weights are the MFMA's first operand: a lane
// of the accumulator then holds four consecutive n of one m.
template <int BN, int BM, int WN, int WM>
__global__ __launch_bounds__((BN / WN) * (BM / WM) * 64) void fp8_mm_kernel(const MmArgs a) {
  constexpr int WAVES = (BN / WN) * (BM / WM), TN = WN / 32, TM = WM / 32;
  constexpr int STAGE = (BN + BM) * 128, PIECES = (BN + BM) / 8, PW = PIECES / WAVES;
  static_assert(PIECES % WAVES == 0, "whole pieces per wave");
  typedef __attribute__((address_space(3))) uint8_t lds_u8;
  typedef __attribute__((address_space(3))) void lds_void;
  typedef const __attribute__((address_space(1))) void glb_void;
  __shared__ __attribute__((aligned(16))) uint8_t smem[2 * STAGE];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const long long tile = blockIdx.x;
  const int n0 = (int)(tile % a.tn) * BN;
  const long long m0 = (tile / a.tn) * BM;
  const int ks = blockIdx.y;
  const int kb0 = (int)((long long)ks * a.nkb / a.ksplit), kb1 = (int)((long long)(ks + 1) * a.nkb / a.ksplit);

  // DMA sources: piece p = 8 rows; lane -> row p * 8 + lane / 8, the chunk that belongs into its slot.  Rows behind the end read the
  // last row (their results are not stored).
  const uint8_t* src[PW];
#pragma unroll
  for (int i = 0; i < PW; ++i) {
    const int row = (wave * PW + i) * 8 + (lane >> 3), ch = (lane & 7) ^ (row & 7);
    if (row < BN) {
      const int r = n0 + row < a.n ? n0 + row : a.n - 1;
      src[i] = a.b + (long long)r * a.kp + ch * 16;
    } else {
      const long long r = m0 + row - BN < a.m ? m0 + row - BN : a.m - 1;
      src[i] = a.a + r * a.kp + ch * 16;
    }
  }
  auto dma = [&](int kb, int buf) {
#pragma unroll
    for (int i = 0; i < PW; ++i)
      __builtin_amdgcn_global_load_lds((glb_void*)(src[i] + (long long)kb * 128),
                                       (lds_void*)((lds_u8*)smem + buf * STAGE + (wave * PW + i) * 1024), 16, 0, 0);
  };
  const int wn = (wave % (BN / WN)) * WN, wm = (wave / (BN / WN)) * WM, l31 = lane & 31, kh = lane >> 5;
  const uint8_t *ps_n[TN], *ps_m[TM];
#pragma unroll
  for (int i = 0; i < TN; ++i) {
    const int r = std::min(n0 + wn + i * 32 + l31, a.n - 1);
    ps_n[i] = a.sb + (long long)(r >> a.shb) * a.kb4;
  }
#pragma unroll
  for (int j = 0; j < TM; ++j) {
    const long long r = std::min<long long>(m0 + wm + j * 32 + l31, a.m - 1);
    ps_m[j] = a.sa + (r >> a.sha) * a.kb4;
  }
  f32x16 acc[TN][TM];
#pragma unroll
  for (int i = 0; i < TN; ++i)
#pragma unroll
    for (int j = 0; j < TM; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
  // 16 codes of a row: chunk c = 2 step + lane / 32 of the K block (the order of k inside a block is free as long as both operands
  // share it), two MFMA operands of 8 values
  auto frag = [&](int buf, int row, int step) -> i32x4 {
    return *reinterpret_cast<const i32x4*>(smem + buf * STAGE + row * 128 + (((step * 2 + kh) ^ (row & 7)) * 16));
  };
  uint32_t dn[TN], dm[TM];
  if (kb0 < kb1) dma(kb0, 0);
  __syncthreads();
  for (int kb = kb0; kb < kb1; ++kb) {
    const int buf = (kb - kb0) & 1;
    if (kb + 1 < kb1) dma(kb + 1, buf ^ 1);
    if (kb == kb0 || (kb & 3) == 0) {
#pragma unroll
      for (int i = 0; i < TN; ++i) dn[i] = *reinterpret_cast<const uint32_t*>(ps_n[i] + (kb & ~3));
#pragma unroll
      for (int j = 0; j < TM; ++j) dm[j] = *reinterpret_cast<const uint32_t*>(ps_m[j] + (kb & ~3));
    }
    const int sh = (kb & 3) * 8;
    float sn[TN], sm[TM];
#pragma unroll
    for (int i = 0; i < TN; ++i) sn[i] = fp8_scale_float(dn[i] >> sh);
#pragma unroll
    for (int j = 0; j < TM; ++j) sm[j] = fp8_scale_float(dm[j] >> sh);
#pragma unroll
    for (int step = 0; step < 4; ++step) {
      i32x4 fn[TN], fm[TM];
#pragma unroll
      for (int i = 0; i < TN; ++i) fn[i] = frag(buf, wn + i * 32 + l31, step);
#pragma unroll
      for (int j = 0; j < TM; ++j) fm[j] = frag(buf, BN + wm + j * 32 + l31, step);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        bf16x8 on[TN], om[TM];
#pragma unroll
        for (int i = 0; i < TN; ++i) on[i] = fp8_widen8(fn[i][2 * h], fn[i][2 * h + 1], sn[i]);
#pragma unroll
        for (int j = 0; j < TM; ++j) om[j] = fp8_widen8(fm[j][2 * h], fm[j][2 * h + 1], sm[j]);
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
          for (int j = 0; j < TM; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(on[i], om[j], acc[i][j], 0, 0, 0);
      }
    }
    __syncthreads();
  }
  // accumulator e of a lane: n = 8 (e / 4) + 4 (lane / 32) + e % 4, m = lane % 32
#pragma unroll
  for (int j = 0; j < TM; ++j) {
    const long long m = m0 + wm + j * 32 + l31;
    if (m >= a.m) continue;
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int n = n0 + wn + i * 32 + g * 8 + kh * 4;
        float v[4] = {acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
        if (a.ksplit > 1) {
          float* p = a.part + ((long long)ks * a.m + m) * a.n + n;
          if ((a.n & 3) == 0) {
            if (n < a.n) *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
          } else {
            for (int e = 0; e < 4 && n + e < a.n; ++e) p[e] = v[e];
          }
        } else if (n < a.n) {
          mm_finish4(a, m, n, v);
        }
      }
  }
}

// split-K: add the partials in order, then the epilogue
__global__ __launch_bounds__(256) void fp8_mm_finish_kernel(const MmArgs a) {
  const int n4 = (a.n + 3) >> 2;
  const long long total = a.m * n4;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
    const long long m = i / n4;
    const int n = (int)(i - m * n4) * 4;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    for (int k = 0; k < a.ksplit; ++k) {
      const float* p = a.part + ((long long)k * a.m + m) * a.n + n;
      if ((a.n & 3) == 0) {
        const float4 t = *reinterpret_cast<const float4*>(p);
        v[0] += t.x, v[1] += t.y, v[2] += t.z, v[3] += t.w;
      } else {
        for (int e = 0; e < 4 && n + e < a.n; ++e) v[e] += p[e];
      }
    }
    mm_finish4(a, m, n, v);
  }
}

struct MmPlan {
  int bm, bn, ksplit;
  long long tm;
  int tn;
  long long ws;
};

// 128 x 128 tiles; K is split while there are fewer than two tiles per CU and every split keeps four blocks of 128
int mm_plan(const sm_fp8_matmul_desc* d, MmPlan* p) {
  if (d == nullptr) return SM_ERR_BAD_ARG;
  if (d->m < 0 || d->n < 1 || d->k < 1) return SM_ERR_BAD_SHAPE;
  if ((d->a_block_rows != 1 && d->a_block_rows != 128) || (d->b_block_rows != 1 && d->b_block_rows != 128) ||
      d->out_dtype < SM_DT_BF16 || d->out_dtype > SM_DT_F32)
    return SM_ERR_BAD_ARG;
  if (d->y_stride < d->n || d->n > 0x7fffff00 || d->k > 0x7fffff00) return SM_ERR_BAD_SHAPE;
  p->bm = p->bn = 128;
  p->tm = (d->m + 127) / 128;
  p->tn = sm_cdiv(d->n, 128);
  const int nkb = sm_cdiv(d->k, 128);
  const long long tiles = p->tm * p->tn;
  if (tiles > 0xfff000) return SM_ERR_UNSUPPORTED;
  p->ksplit = tiles == 0 ? 1 : (int)std::max<long long>(1, std::min<long long>(512 / tiles, nkb / 4));
  p->ws = p->ksplit > 1 ? (long long)p->ksplit * d->m * d->n * 4 : 0;
  return SM_OK;
}

}  // namespace

extern "C" int64_t sm_fp8_cols_padded(int64_t cols) { return (cols + 127) / 128 * 128; }
extern "C" int64_t sm_fp8_scale_cols(int64_t cols) { return ((cols + 127) / 128 + 3) / 4 * 4; }

namespace {
template <int DT>
int fp8_quant_launch(const void* xv, long long rows, long long cols, long long ldx, int block_rows, int transpose, void* qv, void* sv,
                     hipStream_t s) {
  typedef typename Elem<DT>::type T;
  const T* x = (const T*)xv;
  uint8_t *q = (uint8_t*)qv, *sc = (uint8_t*)sv;
  const bool vec = ((uintptr_t)x & 15) == 0 && ldx % (16 / sm_dtype_bytes(DT)) == 0;
  const long long along = transpose ? rows : cols;
  const long long kp = sm_fp8_cols_padded(along);
  const int kb4 = (int)sm_fp8_scale_cols(along);
  if (!transpose && block_rows == 1) {
    const unsigned blocks = (unsigned)std::min<long long>((rows * kb4 + 15) / 16, 256 * 32);
    if (vec) hipLaunchKernelGGL((fp8_quant_rows_kernel<DT, true>), dim3(blocks), dim3(256), 0, s, x, rows, cols, ldx, kb4, kp, q, sc);
    else hipLaunchKernelGGL((fp8_quant_rows_kernel<DT, false>), dim3(blocks), dim3(256), 0, s, x, rows, cols, ldx, kb4, kp, q, sc);
    SM_LAUNCH_CHECK();
    return SM_OK;
  }
  const long long rb = (rows + 127) / 128, cb = transpose ? (cols + 63) / 64 : kp / 64;
  if (cb > 65535 || rb > 0xfff000) return SM_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)rb, (unsigned)cb);
#define SM_Q(V, T_, S_) hipLaunchKernelGGL((fp8_quant_tile_kernel<DT, V, T_, S_>), grid, dim3(256), 0, s, x, rows, cols, ldx, kb4, kp, q, sc)
  if (!transpose) {
    if (vec) SM_Q(true, false, true);
    else SM_Q(false, false, true);
  } else if (block_rows == 128) {
    if (vec) SM_Q(true, true, true);
    else SM_Q(false, true, true);
  } else {
    if (vec) SM_Q(true, true, false);
    else SM_Q(false, true, false);
  }
#undef SM_Q
  SM_LAUNCH_CHECK();
  return SM_OK;
}
}  // namespace

extern "C" int sm_fp8_quantize(int dtype, const void* x, int64_t rows, int64_t cols, int64_t x_stride, int block_rows, int transpose,
                               void* q, void* scale, sm_stream_t stream) {
  if (dtype < SM_DT_BF16 || dtype > SM_DT_F32 || (block_rows != 1 && block_rows != 128)) return SM_ERR_BAD_ARG;
  if (rows < 0 || cols < 1 || x_stride < cols || cols > 0x7fffff00 || rows > (int64_t)1 << 40) return SM_ERR_BAD_SHAPE;
  if (rows == 0) return transpose ? SM_ERR_BAD_SHAPE : SM_OK;
  if (transpose && rows > 0x7fffff00) return SM_ERR_BAD_SHAPE;
  if (!x || !q || !scale || ((uintptr_t)q & 15) != 0 || ((uintptr_t)scale & 3) != 0) return SM_ERR_BAD_ARG;
  hipStream_t s = sm_hip_stream(stream);
  if (dtype == SM_DT_BF16) return fp8_quant_launch<SM_DT_BF16>(x, rows, cols, x_stride, block_rows, transpose, q, scale, s);
  if (dtype == SM_DT_F16) return fp8_quant_launch<SM_DT_F16>(x, rows, cols, x_stride, block_rows, transpose, q, scale, s);
  return fp8_quant_launch<SM_DT_F32>(x, rows, cols, x_stride, block_rows, transpose, q, scale, s);
}

extern "C" int64_t sm_col_sum_workspace(int64_t rows, int cols) {
  if (rows < 0 || cols < 1) return SM_ERR_BAD_SHAPE;
  return std::max<int64_t>(16, (rows + CS_ROWS - 1) / CS_ROWS * cols * 4);
}

extern "C" int sm_col_sum(int dtype, const void* x, int64_t rows, int cols, int64_t x_stride, float* out, void* workspace,
                          int64_t workspace_bytes, sm_stream_t stream) {
  if (dtype < SM_DT_BF16 || dtype > SM_DT_F32) return SM_ERR_BAD_ARG;
  if (rows < 0 || cols < 1 || x_stride < cols) return SM_ERR_BAD_SHAPE;
  if (!out || !workspace || (rows > 0 && !x)) return SM_ERR_BAD_ARG;
  if (workspace_bytes < sm_col_sum_workspace(rows, cols)) return SM_ERR_WORKSPACE;
  const long long nb = (rows + CS_ROWS - 1) / CS_ROWS;
  if (nb > 65535) return SM_ERR_UNSUPPORTED;
  hipStream_t s = sm_hip_stream(stream);
  float* part = (float*)workspace;
  if (nb > 0) {
    const dim3 grid(sm_cdiv(cols, 64), (unsigned)nb);
    if (dtype == SM_DT_BF16)
      hipLaunchKernelGGL((col_sum_kernel<SM_DT_BF16>), grid, dim3(256), 0, s, (const uint16_t*)x, (long long)rows, cols, (long long)x_stride, part);
    else if (dtype == SM_DT_F16)
      hipLaunchKernelGGL((col_sum_kernel<SM_DT_F16>), grid, dim3(256), 0, s, (const _Float16*)x, (long long)rows, cols, (long long)x_stride, part);
    else
      hipLaunchKernelGGL((col_sum_kernel<SM_DT_F32>), grid, dim3(256), 0, s, (const float*)x, (long long)rows, cols, (long long)x_stride, part);
  }
  hipLaunchKernelGGL(col_sum_finish_kernel, dim3(sm_cdiv(cols, 32)), dim3(256), 0, s, part, (int)nb, cols, out);
  SM_LAUNCH_CHECK();
  return SM_OK;
}

extern "C" int64_t sm_fp8_matmul_workspace(const sm_fp8_matmul_desc* d) {
  MmPlan p;
  const int st = mm_plan(d, &p);
  if (st != SM_OK) return st;
  return std::max<int64_t>(16, p.ws);
}

extern "C" int sm_fp8_matmul(const sm_fp8_matmul_desc* d, const void* a, const void* a_scale, const void* b, const void* b_scale,
                             const float* bias, const void* residual, void* y, void* workspace, int64_t workspace_bytes,
                             sm_stream_t stream) {
  MmPlan p;
  const int st = mm_plan(d, &p);
  if (st != SM_OK) return st;
  if (d->m == 0) return SM_OK;
  if (!a || !a_scale || !b || !b_scale || !y) return SM_ERR_BAD_ARG;
  if (residual && d->res_stride < d->n) return SM_ERR_BAD_SHAPE;
  if ((((uintptr_t)a | (uintptr_t)b) & 15) != 0 || (((uintptr_t)a_scale | (uintptr_t)b_scale) & 3) != 0) return SM_ERR_BAD_ARG;
  if (p.ws > 0 && (!workspace || ((uintptr_t)workspace & 15) != 0)) return SM_ERR_BAD_ARG;
  if (workspace_bytes < p.ws) return SM_ERR_WORKSPACE;
  MmArgs k;
  k.a = (const uint8_t*)a, k.b = (const uint8_t*)b, k.sa = (const uint8_t*)a_scale, k.sb = (const uint8_t*)b_scale;
  k.bias = bias, k.res = residual, k.y = y, k.part = (float*)workspace;
  k.m = d->m, k.n = d->n, k.ldy = d->y_stride, k.ldr = residual ? d->res_stride : 0;
  k.kp = sm_fp8_cols_padded(d->k), k.nkb = sm_cdiv(d->k, 128), k.kb4 = (int)sm_fp8_scale_cols(d->k);
  k.sha = d->a_block_rows == 128 ? 7 : 0, k.shb = d->b_block_rows == 128 ? 7 : 0;
  k.ksplit = p.ksplit, k.relu = d->relu, k.out = d->out_dtype;
  const uintptr_t al = (uintptr_t)(4 * sm_dtype_bytes(d->out_dtype) - 1);
  k.vec4 = ((uintptr_t)y & al) == 0 && d->y_stride % 4 == 0 && (!residual || (((uintptr_t)residual & al) == 0 && d->res_stride % 4 == 0));
  k.tm = (int)p.tm, k.tn = p.tn;
  hipStream_t s = sm_hip_stream(stream);
  hipLaunchKernelGGL((fp8_mm_kernel<128, 128, 64, 64>), dim3((unsigned)(p.tm * p.tn), p.ksplit), dim3(256), 0, s, k);
  if (p.ksplit > 1) {
    const long long total = k.m * ((k.n + 3) / 4);
    hipLaunchKernelGGL(fp8_mm_finish_kernel, dim3((unsigned)std::min<long long>((total + 255) / 256, 256 * 16)), dim3(256), 0, s, k);
  }
  SM_LAUNCH_CHECK();
  return SM_OK;
}
