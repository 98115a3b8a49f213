// 8-bit products with a power-of-two scale per block of 128: quantiser, product, column sums.
//
//   scale_b = smallest 2^e (e >= -127) with max |x| / 2^e <= 448 over the block (1 for a block of zeros), code = e4m3(x / 2^e)
//   y[m][n] = sum_kb 2^(ea[m][kb] + eb[n][kb]) sum_{k in kb} a[m][k] b[n][k] (+ bias_n) (+ residual) (ReLU)
//
// Why powers of two: x / 2^e is exact (the one rounding is the one to e4m3), e4m3's own exponent hides the up to one binary digit of
// range that a power of two gives away, and the scale enters the product for nothing: v_cvt_scalef32_pk_bf16_fp8 multiplies by it while
// it widens two codes.
//
// Why bf16 MFMAs and not the 8-bit ones: a code times its scale is exact in bf16 (for scale bytes from 3 on; below, it is rounded to a
// multiple of 2^-133, bf16's smallest subnormal; a block maximum above 248 * 2^120 has the code 256 at 2^120, which is Inf in bf16 and in
// f32), and v_mfma_f32_32x32x16_bf16 adds the exact products in f32.  The 8-bit MFMAs (plain and block-scaled) align the products of an
// instruction to the largest one and drop what lies 2^-14 below it (measured with one large and one small product; sums of 64 products
// over 8 binades were off by 2^-12 of the largest): less than f32 sums.  The price is the matrix peak, 2.5 instead of 5 PFLOP/s; the
// widening itself hides behind the MFMAs (one conversion is 8 cycles; 16 of them beside 4 MFMAs measured 161 cycles against 154 for the
// MFMAs alone), and the bytes moved through HBM and LDS stay 8-bit.
//
// Layout of a quantised matrix: codes [K / 64][row][64] (two slabs per block of 128, zero codes behind the last column), scales
// [K block / 4][row block][4] (127, i.e. 1, behind the last block).  One K step of a tile is then one contiguous piece of memory, and
// a K loop reads four scales of a row as one dword, neighbouring rows side by side.
//
// Measured (m x n x k, bf16 in and out; the library's bf16 product reaches 1.28 PFLOP/s on 8192^3 here):
//   8192 x 4096 x 4096 product alone       215 to 260 us by run, 8192^3 855 = 1.29 PFLOP/s: as the library's, half of the bf16 peak
//   67 200 x 512 x 768 product alone       58 us = 0.91 PFLOP/s: twelve short steps between a block's first load and its last store
//   7 x 512 x 2048 with its quantiser      5 us: one launch, latency
//   quantiser, 67 200 x 768               29 us = 5.3 TB/s; with the transpose, 67 200 x 768: 44 us = 4.7 TB/s
#include <algorithm>
#include <type_traits>

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

// Inf and NaN have no code but NaN and are left out of the block's maximum.  A maximum skips NaN by itself, and the conversion makes
// NaN of NaN and of Inf; only the maximum of a block that holds an Inf is taken again, over what is finite (rare: one compare per block).
__device__ __forceinline__ float fp8_abs_finite(float x) {
  const float a = __builtin_fabsf(x);
  return a <= 3.402823466e38f ? a : 0.f;
}
template <int N>
__device__ __forceinline__ float fp8_amax(const float* f) {
  float m = 0.f;
#pragma unroll
  for (int e = 0; e < N; ++e) m = fmaxf(m, __builtin_fabsf(f[e]));
  if (m > 3.402823466e38f) {
    m = 0.f;
#pragma unroll
    for (int e = 0; e < N; ++e) m = fmaxf(m, fp8_abs_finite(f[e]));
  }
  return m;
}
// maximum over the 16 lanes of a DPP row, on every lane: quad permutes, then rotations by 4 and 8
__device__ __forceinline__ float max16(float m) {
  m = fmaxf(m, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(m), 0xB1, 0xf, 0xf, true)));    // lane ^ 1
  m = fmaxf(m, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(m), 0x4E, 0xf, 0xf, true)));    // lane ^ 2
  m = fmaxf(m, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(m), 0x124, 0xf, 0xf, true)));   // row_ror:4
  return fmaxf(m, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(m), 0x128, 0xf, 0xf, true)));   // row_ror:8
}
__device__ __forceinline__ uint2 fp8_pack8(const float* f, float inv) {
  int lo = 0, hi = 0;
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[0] * inv, f[1] * inv, lo, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[2] * inv, f[3] * inv, lo, true);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(f[4] * inv, f[5] * inv, hi, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(f[6] * inv, f[7] * inv, hi, true);
  return make_uint2((uint32_t)lo, (uint32_t)hi);
}

// 8 consecutive values of a row from column c as they came from memory (any alignment: as floats); columns >= cols are 0
template <int DT, bool VEC>
struct Raw8 {
  typename Elem<DT>::raw8 q;
  __device__ __forceinline__ void load(const typename Elem<DT>::type* row, long long c, long long cols) {
    if (c + 8 <= cols) {
      q = Elem<DT>::load8(row + c);
    } else {
      typename Elem<DT>::type t[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) t[e] = c + e < cols ? row[c + e] : typename Elem<DT>::type(0);
      q = __builtin_bit_cast(typename Elem<DT>::raw8, t);
    }
  }
  __device__ __forceinline__ void zero() { q = typename Elem<DT>::raw8{}; }
  __device__ __forceinline__ void get(float* f) const { Elem<DT>::unpack(q, f); }
};
template <int DT>
struct Raw8<DT, false> {
  float v[8];
  __device__ __forceinline__ void load(const typename Elem<DT>::type* row, long long c, long long cols) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = c + e < cols ? Elem<DT>::load(row + c + e) : 0.f;
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.f;
  }
  __device__ __forceinline__ void get(float* f) const {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = v[e];
  }
};

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

// 1 x 128 blocks along the row: 16 lanes of 8 values each.  A workgroup takes 64 blocks of x in storage order (row by row, whatever the
// row's number of blocks), four per wave at a time, four such pieces in flight; one pass and no loop, so the last workgroups are no
// longer than the others.
//   268800 x 256: 37 us; with a wave on four blocks of one row, half of them behind its end: 60; and with 2048 workgroups in a loop: 73
template <int DT, bool VEC>
__global__ __launch_bounds__(256) void fp8_quant_rows_kernel(const typename Elem<DT>::type* __restrict__ x, long long rows, long long cols,
                                                             long long ldx, int nkb, uint32_t inv_nkb, uint8_t* __restrict__ q,
                                                             uint8_t* __restrict__ scale) {
  constexpr int U = 4;
  const int l = threadIdx.x & 15, grp = threadIdx.x >> 4;
  const long long b0 = (long long)blockIdx.x * 64, r0 = b0 / nkb;
  const int k0 = (int)(b0 - r0 * nkb);
  Raw8<DT, VEC> f8[U];
  long long r[U];
  int kb[U];
#pragma unroll
  for (int p = 0; p < U; ++p) {
    const uint32_t k = (uint32_t)(k0 + p * 16 + grp);                 // (< nkb + 64)
    const uint32_t over = nkb >= 64 ? (k >= (uint32_t)nkb ? 1u : 0u) : (nkb == 1 ? k : __umulhi(k, inv_nkb));   // k / nkb
    r[p] = r0 + over;
    kb[p] = (int)(k - over * (uint32_t)nkb);
    if (r[p] < rows) f8[p].load(x + r[p] * ldx, (long long)kb[p] * 128 + l * 8, cols);
    else f8[p].zero();
  }
#pragma unroll
  for (int p = 0; p < U; ++p) {
    float f[8];
    f8[p].get(f);
    const int sb = fp8_scale_byte(max16(fp8_amax<8>(f)));
    if (r[p] < rows) {
      *reinterpret_cast<uint2*>(q + ((long long)(kb[p] * 2 + (l >> 3)) * rows + r[p]) * 64 + (l & 7) * 8) = fp8_pack8(f, fp8_inv_scale(sb));
      // (the last block of a row fills the dword up with 127)
      if (l == 0 || (kb[p] == nkb - 1 && l < 4 - (kb[p] & 3)))
        scale[((long long)(kb[p] >> 2) * rows + r[p]) * 4 + (kb[p] & 3) + l] = (uint8_t)(l == 0 ? sb : 127);
    }
  }
}

// One 128 x 128 piece of x per block, 8 columns x 8 consecutive rows per thread, read once for everything that is wanted of it:
//   q / scale    codes in rows: 1 x 128 blocks, or the whole piece as one block (SQUARE)
//   qt / scalet  codes of the transpose: blocks of 1 column x 128 rows, or the piece (SQUARE)
//   colsum       f32 [row block][cols] sums over the piece's rows
// each may be null.  gate (may be null): values whose gate is not > 0 count as 0 (the ReLU of a layer whose output is the gate).
// Blocks of a row of pieces follow each other, so that whole rows of x are open at a time (67200 x 768 bf16: 49 -> 44 us).
// Bound by memory: 2 + 1 + 1 bytes per 16-bit value, 4.7 TB/s; a training step that made the three from x one by one would read x three times.
template <int DT, bool VEC, bool SQUARE>
__global__ __launch_bounds__(256) void fp8_quant_pair_kernel(const typename Elem<DT>::type* __restrict__ x,
                                                             const typename Elem<DT>::type* __restrict__ gate, long long rows, long long cols,
                                                             long long ldx, long long ldg, int nkb, int nkbt, uint8_t* __restrict__ q,
                                                             uint8_t* __restrict__ scale, uint8_t* __restrict__ qt,
                                                             uint8_t* __restrict__ scalet, float* __restrict__ colsum) {
  __shared__ float s_red[16][128];
  __shared__ float s_wmax[4];
  __shared__ int s_byte[128];
  __shared__ __attribute__((aligned(16))) uint8_t s_q[128 * 128];
  const long long rb = blockIdx.x / nkb, r0 = rb * 128, c0 = (long long)(blockIdx.x % nkb) * 128;
  const int cv = threadIdx.x & 15, rl = threadIdx.x >> 4;
  // the values stay as they came and are widened again where needed (67200 x 768 bf16: 49 us, as floats from the start 56; 150 registers
  // for every type either way, three waves a SIMD)
  Raw8<DT, VEC> x8[8];
  uint32_t open[2] = {~0u, ~0u};                 // gate bits of rows 0 - 3 and 4 - 7, 8 columns each
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    const long long r = r0 + rl * 8 + u;
    if (r < rows) x8[u].load(x + r * ldx, c0 + cv * 8, cols);
    else x8[u].zero();
  }
  if (gate != nullptr) {
    open[0] = open[1] = 0u;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const long long r = r0 + rl * 8 + u;
      if (r >= rows) continue;
      float g[8];
      fp8_load8<DT, VEC>(gate + r * ldg, c0 + cv * 8, cols, g);
#pragma unroll
      for (int e = 0; e < 8; ++e) open[u >> 2] |= g[e] > 0.f ? 1u << ((u & 3) * 8 + e) : 0u;
    }
  }
  auto row = [&](int u, float (&f)[8]) {
    x8[u].get(f);
    if (gate != nullptr) {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = (open[u >> 2] >> ((u & 3) * 8 + e)) & 1u ? f[e] : 0.f;
    }
  };
  // byte of block kb of a scale row; the last block of a row fills the dword up with 127
  auto put_scale = [](uint8_t* base, long long r, long long nr, int kb, int nb, int byte) {
    uint8_t* p = base + ((long long)(kb >> 2) * nr + r) * 4;
    p[kb & 3] = (uint8_t)byte;
    if (kb == nb - 1)
      for (int k = (kb & 3) + 1; k < 4; ++k) p[k] = 127;
  };
  const int kb = (int)(c0 >> 7), kbt = (int)rb;
  int block_byte = 127;
  if constexpr (SQUARE) {
    float m = 0.f;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      float f[8];
      row(u, f);
      m = fmaxf(m, fp8_amax<8>(f));
    }
    m = max16(m);
    m = fmaxf(m, __shfl_xor(m, 16, 64));
    m = fmaxf(m, __shfl_xor(m, 32, 64));
    if ((threadIdx.x & 63) == 0) s_wmax[threadIdx.x >> 6] = m;
    __syncthreads();
    block_byte = fp8_scale_byte(fmaxf(fmaxf(s_wmax[0], s_wmax[1]), fmaxf(s_wmax[2], s_wmax[3])));
    if (threadIdx.x == 0) {
      if (q != nullptr) put_scale(scale, rb, (rows + 127) >> 7, kb, nkb, block_byte);
      if (qt != nullptr) put_scale(scalet, kb, (cols + 127) >> 7, kbt, nkbt, block_byte);
    }
  }
  if (q != nullptr) {
    int mine = 127;                              // lane cv of the 16 that share a row's block stores the scale of row cv of eight
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const long long r = r0 + rl * 8 + u;
      float f[8];
      row(u, f);
      int sb = block_byte;
      if constexpr (!SQUARE) {
        sb = fp8_scale_byte(max16(fp8_amax<8>(f)));
        mine = cv == u ? sb : mine;
      }
      if (r < rows)
        *reinterpret_cast<uint2*>(q + ((long long)(kb * 2 + (cv >> 3)) * rows + r) * 64 + (cv & 7) * 8) = fp8_pack8(f, fp8_inv_scale(sb));
    }
    if (!SQUARE && cv < 8 && r0 + rl * 8 + cv < rows) put_scale(scale, r0 + rl * 8 + cv, rows, kb, nkb, mine);
  }
  if (colsum != nullptr) {
    float t[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      float f[8];
      row(u, f);
#pragma unroll
      for (int e = 0; e < 8; ++e) t[e] += f[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) s_red[rl][cv * 8 + e] = t[e];
    __syncthreads();
    if (threadIdx.x < 128 && c0 + threadIdx.x < cols) {
      float t = 0.f;
#pragma unroll
      for (int k = 0; k < 16; ++k) t += s_red[k][threadIdx.x];
      colsum[rb * cols + c0 + threadIdx.x] = t;
    }
    __syncthreads();
  }
  if (qt == nullptr) return;
  if constexpr (!SQUARE) {
    float m[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    bool inf = false;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      float f[8];
      row(u, f);
#pragma unroll
      for (int e = 0; e < 8; ++e) m[e] = fmaxf(m[e], __builtin_fabsf(f[e]));
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) inf |= m[e] > 3.402823466e38f;
    if (inf) {                                   // (see fp8_amax)
#pragma unroll
      for (int e = 0; e < 8; ++e) m[e] = 0.f;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        float f[8];
        row(u, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) m[e] = fmaxf(m[e], fp8_abs_finite(f[e]));
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) s_red[rl][cv * 8 + e] = m[e];
    __syncthreads();
    if (threadIdx.x < 128) {
      float m = 0.f;
#pragma unroll
      for (int k = 0; k < 16; ++k) m = fmaxf(m, s_red[k][threadIdx.x]);
      const int sb = fp8_scale_byte(m);
      s_byte[threadIdx.x] = sb;
      if (c0 + threadIdx.x < cols) put_scale(scalet, c0 + threadIdx.x, cols, kbt, nkbt, sb);
    }
    __syncthreads();
  }
  // the transpose goes through LDS: 8 rows of a column = 8 bytes, chunk rl of column c at slot rl ^ (c / 8) (16 columns of a wave's
  // write then lie in 16 different slots)
  // (two rows at a time: v_cvt_pk_fp8_f32 takes a pair; the codes of rows 2 h, 2 h + 1 of a column are half of its dword h / 2)
  float inv[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) inv[e] = fp8_inv_scale(SQUARE ? block_byte : s_byte[cv * 8 + e]);
  int code[8][2];
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    float f[8], g[8];
    row(2 * h, f);
    row(2 * h + 1, g);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (h & 1) code[e][h >> 1] = __builtin_amdgcn_cvt_pk_fp8_f32(f[e] * inv[e], g[e] * inv[e], code[e][h >> 1], true);
      else code[e][h >> 1] = __builtin_amdgcn_cvt_pk_fp8_f32(f[e] * inv[e], g[e] * inv[e], 0, false);
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e)
    *reinterpret_cast<uint2*>(s_q + (cv * 8 + e) * 128 + ((rl ^ cv) * 8)) = make_uint2((uint32_t)code[e][0], (uint32_t)code[e][1]);
  __syncthreads();
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const int i = threadIdx.x + 256 * p, c = (i >> 2) & 127, ch = (i >> 9) * 4 + (i & 3), sw = c >> 3;   // slab, column, 16-byte chunk
    uint4 v = *reinterpret_cast<const uint4*>(s_q + c * 128 + ((ch ^ (sw >> 1)) * 16));
    if (sw & 1) v = make_uint4(v.z, v.w, v.x, v.y);
    if (c0 + c < cols) *reinterpret_cast<uint4*>(qt + ((long long)(kbt * 2 + (ch >> 2)) * cols + c0 + c) * 64 + (ch & 3) * 16) = v;
  }
}

// ------------------------------------------------------------------------------------------------ column sums
// out[c] = sum over the row blocks of part[block][c], f64, a fixed order
__global__ __launch_bounds__(1024) void col_sum_finish_kernel(const float* __restrict__ part, int nb, int cols, float* __restrict__ out) {
  __shared__ double sh[32][33];
  const int cl = threadIdx.x & 31, sl = threadIdx.x >> 5, c = blockIdx.x * 32 + cl;
  double s = 0.0;
  if (c < cols) {
    int i = sl;
    for (; i + 7 * 32 < nb; i += 8 * 32) {       // eight loads in flight
      float v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = part[(long long)(i + u * 32) * cols + c];
#pragma unroll
      for (int u = 0; u < 8; ++u) s += (double)v[u];
    }
    for (; i < nb; i += 32) s += (double)part[(long long)i * cols + c];
  }
  sh[sl][cl] = s;
  __syncthreads();
  if (sl == 0 && c < cols) {
    for (int k = 1; k < 32; ++k) s += sh[k][cl];
    out[c] = (float)s;
  }
}

// ------------------------------------------------------------------------------------------------ product
struct MmArgs {
  const uint8_t *a, *b, *sa, *sb;    // activations, weights and their scales
  const float* bias;
  const void* res;
  void* y;
  float* part;                       // [ksplit][m][n] when ksplit > 1
  long long m, ldy, ldr, nsa;        // nsa / nsb: rows of the scale matrices
  int n, nkb, nsb, sha, shb;         // sha / shb: row >> sh = row of the scale matrix
  int ksplit, relu, out, vec;        // vec: eight consecutive n of y / residual are 16-byte aligned accesses
  long long tm;                      // tiles
  int tn;
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
// 8 codes (two dwords) times a power of two as bf16: exact within the range stated at the top
__device__ __forceinline__ bf16x8 fp8_widen8(int lo, int hi, float scale) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
  const auto ab = __builtin_shufflevector(a, b, 0, 1, 2, 3), cd = __builtin_shufflevector(c, d, 0, 1, 2, 3);
  return __builtin_shufflevector(ab, cd, 0, 1, 2, 3, 4, 5, 6, 7);
}

// bias, residual, ReLU and the store of V = 4 or 8 consecutive n (n0 a multiple of V) of row m
template <int V>
__device__ __forceinline__ void mm_finish(const MmArgs& a, long long m, int n0, float (&v)[V]) {
  if (a.vec && n0 + V <= a.n) {
    if (a.bias != nullptr) {
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] += a.bias[n0 + e];
    }
    if (a.res != nullptr) {
      const long long o = m * a.ldr + n0;
      if (a.out == SM_DT_F32) {
#pragma unroll
        for (int q = 0; q < V / 4; ++q) {
          const float4 r = *reinterpret_cast<const float4*>((const float*)a.res + o + 4 * q);
          v[4 * q] += r.x, v[4 * q + 1] += r.y, v[4 * q + 2] += r.z, v[4 * q + 3] += r.w;
        }
      } else {
        uint32_t w[V / 2];
        if constexpr (V == 8) *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>((const uint16_t*)a.res + o);
        else *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>((const uint16_t*)a.res + o);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const uint16_t h = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
          v[e] += a.out == SM_DT_BF16 ? bf16_bits_to_f32(h) : (float)__builtin_bit_cast(_Float16, h);
        }
      }
    }
    if (a.relu) {
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = v[e] < 0.f ? 0.f : v[e];
    }
    const long long o = m * a.ldy + n0;
    if (a.out == SM_DT_F32) {
#pragma unroll
      for (int q = 0; q < V / 4; ++q)
        *reinterpret_cast<float4*>((float*)a.y + o + 4 * q) = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
      return;
    }
    uint32_t w[V / 2];
#pragma unroll
    for (int q = 0; q < V / 2; ++q) {
      if (a.out == SM_DT_BF16)
        w[q] = pack_bf16x2(v[2 * q], v[2 * q + 1]);
      else
        w[q] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[2 * q]) |
               ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[2 * q + 1]) << 16);
    }
    if constexpr (V == 8) *reinterpret_cast<uint4*>((uint16_t*)a.y + o) = make_uint4(w[0], w[1], w[2], w[3]);
    else *reinterpret_cast<uint2*>((uint16_t*)a.y + o) = make_uint2(w[0], w[1]);
    return;
  }
#pragma unroll
  for (int e = 0; e < V; ++e) {
    if (n0 + e >= a.n) break;
    float t = v[e];
    if (a.bias != nullptr) t += a.bias[n0 + e];
    if (a.res != nullptr) t += mm_load(a.res, a.out, m * a.ldr + n0 + e);
    if (a.relu) t = t < 0.f ? 0.f : t;
    mm_store(a.y, a.out, m * a.ldy + n0 + e, t);
  }
}

// the f32 partial of a K split instead
template <int V>
__device__ __forceinline__ void mm_partial(const MmArgs& a, int ks, long long m, int n0, const float (&v)[V]) {
  float* p = a.part + ((long long)ks * a.m + m) * a.n + n0;
  if ((a.n & 3) == 0) {
#pragma unroll
    for (int q = 0; q < V / 4; ++q)
      if (n0 + 4 * q < a.n) *reinterpret_cast<float4*>(p + 4 * q) = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (n0 + e < a.n) p[e] = v[e];
  }
}

// f(0), ..., f(N - 1) with compile-time indices
template <int N, int I = 0, typename F>
__device__ __forceinline__ void mm_for(const F& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    mm_for<N, I + 1>(f);
  }
}

// blockIdx.x -> tile.  The hardware hands consecutive blocks to the 8 XCDs in turn; tile numbers are laid out so that one XCD gets a
// run of consecutive tiles (its own L2 then holds the operand panels they share).  Tiles run n-fastest inside bands of GM rows of tiles.
__device__ __forceinline__ void mm_tile(const MmArgs& a, long long& tm, int& tn) {
  const long long nt = (long long)a.tm * a.tn, b = blockIdx.x;
  const long long q = nt >> 3, r = nt & 7, x = b & 7, i = b >> 3;
  const long long t = x * q + (x < r ? x : r) + i;
  constexpr int GM = 4;
  const long long band = (long long)GM * a.tn, bi = t / band, o = t - bi * band;
  const long long h = a.tm - bi * GM < GM ? a.tm - bi * GM : GM;
  tn = (int)(o / h);
  tm = bi * GM + (o - (long long)tn * h);
}

// s_waitcnt vmcnt(N) lgkmcnt(0) and a raw barrier: everything but this wave's N youngest loads has landed, nobody reads the stage
// before any more -- and, unlike __syncthreads(), the younger stages stay in flight
template <int N>
__device__ __forceinline__ void mm_stage_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// LDS of a block: the stages, under which the epilogue's 8 KB per wave lie, and two sets of scales
constexpr int mm_stage_lds(int bn, int bm, int waves, int nst) {
  return (bn + bm) * 64 * nst > waves * 8192 ? (bn + bm) * 64 * nst : waves * 8192;
}
constexpr int mm_lds(int bn, int bm, int waves, int nst) { return mm_stage_lds(bn, bm, waves, nst) + (bn + bm) * 8; }

// Tile of BN weights x BM activations, waves of WN x WM, K steps of 64 (half a scale block) through NST LDS stages filled by direct
// global -> LDS loads, NST - 1 of them in flight.  A row of a stage is 64 codes = 4 chunks of 16 bytes; chunk c of row r lies at slot
// c ^ (r / 2 & 3), so eight neighbouring rows of one chunk cover 128 bytes.  The weights are the MFMA's first operand: a lane of the
// accumulator then holds four consecutive n of one m.  The results leave through LDS (the stages are free by then), 64 n x 32 m at a
// time per wave, so that a store instruction writes whole 128-byte lines of a few rows instead of 16 bytes of 32 rows.
template <int BN, int BM, int WN, int WM, int NST>
__global__ __launch_bounds__((BN / WN) * (BM / WM) * 64, 4) void fp8_mm_kernel(const MmArgs a) {
  constexpr int WAVES = (BN / WN) * (BM / WM), TN = WN / 32, TM = WM / 32;
  constexpr int STAGE = (BN + BM) * 64, PIECES = (BN + BM) / 16, PW = PIECES / WAVES;
  static_assert(PIECES % WAVES == 0 && BN % 16 == 0, "whole pieces per wave, each all weights or all activations");
  static_assert(WN % 64 == 0 && BN % 64 == 0 && BM % 64 == 0 && NST >= 2, "the epilogue takes 64 n x 32 m at a time");
  typedef __attribute__((address_space(3))) uint8_t lds_u8;
  typedef __attribute__((address_space(3))) void lds_void;
  typedef const __attribute__((address_space(1))) void glb_void;
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];      // mm_lds(BN, BM, WAVES, NST)
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  long long tm;
  int tn;
  mm_tile(a, tm, tn);
  const int n0 = tn * BN;
  const long long m0 = tm * BM;
  const int ks = blockIdx.y;
  const int kb0 = (int)((long long)ks * a.nkb / a.ksplit), kb1 = (int)((long long)(ks + 1) * a.nkb / a.ksplit);
  const int nst = (kb1 - kb0) * 2;                                    // stages (>= 2: every split has a block)

  // DMA sources: piece p = 16 rows; lane -> row p * 16 + lane / 4, the chunk that belongs into its slot.  Rows behind the end read the
  // last row (their results are not stored).
  const uint8_t* src[PW];
#pragma unroll
  for (int i = 0; i < PW; ++i) {
    const int row = (wave * PW + i) * 16 + (lane >> 2), ch = (lane & 3) ^ ((row >> 1) & 3);
    if (row < BN) {
      const int r = n0 + row < a.n ? n0 + row : a.n - 1;
      src[i] = a.b + ((long long)kb0 * 2 * a.n + r) * 64 + ch * 16;
    } else {
      const long long r = m0 + row - BN < a.m ? m0 + row - BN : a.m - 1;
      src[i] = a.a + ((long long)kb0 * 2 * a.m + r) * 64 + ch * 16;
    }
  }
  const long long kn = (long long)a.n * 64, km = a.m * 64;
  auto dma = [&](int buf) {                      // the next K step
#pragma unroll
    for (int i = 0; i < PW; ++i) {
      __builtin_amdgcn_global_load_lds((glb_void*)src[i], (lds_void*)((lds_u8*)smem + buf * STAGE + (wave * PW + i) * 1024), 16, 0, 0);
      src[i] += (wave * PW + i) * 16 < BN ? kn : km;
    }
  };
  const int wn = (wave % (BN / WN)) * WN, wm = (wave / (BN / WN)) * WM, l31 = lane & 31, kh = lane >> 5;
  // scales: four K blocks of all rows at a time, also by direct loads (a dword per row; as ordinary loads the wait for them, on the same
  // in-order counter, drained the stages in flight), the next four blocks' while the present four are at work
  constexpr int SROWS = BN + BM, SOFF = mm_stage_lds(BN, BM, WAVES, NST);
  uint8_t* const s_scale = smem + SOFF;                        // [2][SROWS][4]
  const int qlast = (a.nkb - 1) >> 2;
  auto scales = [&](int quad) {
    const long long q = std::min(quad, qlast);
#pragma unroll
    for (int p = 0; p < (SROWS / 64 + WAVES - 1) / WAVES; ++p) {
      const int piece = wave + p * WAVES;
      if (piece < SROWS / 64) {                                       // (wave-uniform)
        const int row = piece * 64 + lane;
        const uint8_t* g;
        if (piece * 64 < BN) g = a.sb + (q * a.nsb + (std::min(n0 + row, a.n - 1) >> a.shb)) * 4;
        else g = a.sa + (q * a.nsa + (std::min<long long>(m0 + row - BN, a.m - 1) >> a.sha)) * 4;
        __builtin_amdgcn_global_load_lds((glb_void*)g, (lds_void*)((lds_u8*)smem + SOFF + ((quad & 1) * SROWS + piece * 64) * 4), 4, 0, 0);
      }
    }
  };
  scales(kb0 >> 2);
  scales((kb0 >> 2) + 1);
#pragma unroll
  for (int t = 0; t < NST - 1; ++t)
    if (t < nst) dma(t);
  f32x16 acc[TN][TM];
#pragma unroll
  for (int i = 0; i < TN; ++i)
#pragma unroll
    for (int j = 0; j < TM; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
  // 16 codes of a row: chunk 2 step + lane / 32 of the stage (the order of k inside a block is free as long as both operands share
  // it), two MFMA operands of 8 values
  const int rsw = (l31 >> 1) & 3;                // every fragment row is l31 plus a multiple of 32
  const uint8_t* const fbase_n = smem + (wn + l31) * 64;
  const uint8_t* const fbase_m = smem + (BN + wm + l31) * 64;
  float sn[TN], sm[TM];
  int buf = 0, fill = NST - 1;                   // the stage at hand, the one that the next loads go to
  for (int t = 0; t < nst; ++t) {
    // stage t has landed when at most the loads of the NST - 2 stages behind it are outstanding (other loads in between only make
    // the wait stricter); behind the barrier stage t - 1, which everybody has read, is filled again
    if (t + NST - 2 < nst) mm_stage_barrier<(NST - 2) * PW>();
    else mm_stage_barrier<0>();
    if (t + NST - 1 < nst) dma(fill);
    const int kb = kb0 + (t >> 1);
    if ((t & 1) == 0) {
      if ((kb & 3) == 0 && t != 0) scales((kb >> 2) + 1);             // (into the half that the four blocks before this one used)
      const uint8_t* const sc = s_scale + ((kb >> 2) & 1) * SROWS * 4 + (kb & 3);
#pragma unroll
      for (int i = 0; i < TN; ++i) sn[i] = fp8_scale_float(sc[(wn + i * 32 + l31) * 4]);
#pragma unroll
      for (int j = 0; j < TM; ++j) sm[j] = fp8_scale_float(sc[(BN + wm + j * 32 + l31) * 4]);
    }
    i32x4 fn[2][TN], fm[2][TM];
    auto read = [&](int step) {
      const int o = buf * STAGE + ((step * 2 + kh) ^ rsw) * 16;
#pragma unroll
      for (int i = 0; i < TN; ++i) fn[step][i] = *reinterpret_cast<const i32x4*>(fbase_n + o + i * 32 * 64);
#pragma unroll
      for (int j = 0; j < TM; ++j) fm[step][j] = *reinterpret_cast<const i32x4*>(fbase_m + o + j * 32 * 64);
    };
    read(0);
    read(1);
#pragma unroll
    for (int step = 0; step < 2; ++step) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        bf16x8 on[TN], om[TM];
#pragma unroll
        for (int i = 0; i < TN; ++i) on[i] = fp8_widen8(fn[step][i][2 * h], fn[step][i][2 * h + 1], sn[i]);
#pragma unroll
        for (int j = 0; j < TM; ++j) om[j] = fp8_widen8(fm[step][j][2 * h], fm[step][j][2 * h + 1], sm[j]);
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
          for (int j = 0; j < TM; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(on[i], om[j], acc[i][j], 0, 0, 0);
      }
    }
    buf = buf + 1 == NST ? 0 : buf + 1;
    fill = fill + 1 == NST ? 0 : fill + 1;
  }
  __syncthreads();                               // (no load is in flight: the last stages waited for all of them)
  // accumulator e of a lane: n = 8 (e / 4) + 4 (lane / 32) + e % 4, m = lane % 32.  32 m x 64 n floats of this wave's own LDS, the
  // 16-byte chunk n / 4 of row m at slot (n / 4) ^ (m & 15); the reads follow the writes of the same wave in order
  float* const E = reinterpret_cast<float*>(smem) + wave * 2048;
  mm_for<TN / 2 * TM>([&](auto IJ) {             // (an unrolled loop of this size leaves acc indexed at run time, in scratch)
    constexpr int ip = decltype(IJ)::value % (TN / 2), j = decltype(IJ)::value / (TN / 2);
#pragma unroll
    for (int i2 = 0; i2 < 2; ++i2)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int c = i2 * 8 + g * 2 + kh;
        const f32x16 t = acc[ip * 2 + i2][j];
        *reinterpret_cast<float4*>(E + l31 * 64 + ((c ^ (l31 & 15)) * 4)) = make_float4(t[4 * g], t[4 * g + 1], t[4 * g + 2], t[4 * g + 3]);
      }
    __builtin_amdgcn_wave_barrier();
    const int cl = (lane & 7) * 2, n = n0 + wn + ip * 64 + cl * 4;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int ml = r * 8 + (lane >> 3);
      const long long m = m0 + wm + j * 32 + ml;
      const float4 p = *reinterpret_cast<const float4*>(E + ml * 64 + ((cl ^ (ml & 15)) * 4));
      const float4 q = *reinterpret_cast<const float4*>(E + ml * 64 + (((cl + 1) ^ (ml & 15)) * 4));
      float v[8] = {p.x, p.y, p.z, p.w, q.x, q.y, q.z, q.w};
      if (m < a.m && n < a.n) {
        if (a.ksplit > 1) mm_partial(a, ks, m, n, v);
        else mm_finish(a, m, n, v);
      }
    }
    __builtin_amdgcn_wave_barrier();
  });
}

// A handful of activation rows (16 MT at most): the weights are what has to be read, and they are read once, straight into registers.
// A block takes 16 weight rows, its 16 waves every 16th K block; a lane holds 32 neighbouring codes of one row (the four MFMAs of a
// block share that order of k for both operands).  SRC: sm_dtype of x, which is then quantised on the way -- no launch and no buffer
// for it -- or 3 for codes.  The waves' sums meet in LDS in wave order.
template <int SRC, bool VEC, int MT>
__global__ __launch_bounds__(1024) void fp8_mm_few_kernel(const MmArgs a, const void* __restrict__ xv, long long ldx, long long cols) {
  constexpr int WAVES = 16;
  __shared__ __attribute__((aligned(16))) float s_acc[WAVES][MT][64][4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16;
  constexpr long long m0 = 0;
  const int n = std::min(n0 + r, a.n - 1);
  long long row[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) row[t] = std::min<long long>(m0 + t * 16 + r, a.m - 1);
  f32x4 acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[t][e] = 0.f;
  for (int kb = wave; kb < a.nkb; kb += WAVES) {
    const i32x4* pw = reinterpret_cast<const i32x4*>(a.b + ((long long)(kb * 2 + (g >> 1)) * a.n + n) * 64 + (g & 1) * 32);
    const i32x4 w0 = pw[0], w1 = pw[1];
    const float sw = fp8_scale_float(a.sb[((long long)(kb >> 2) * a.nsb + (n >> a.shb)) * 4 + (kb & 3)]);
    const bf16x8 on[4] = {fp8_widen8(w0[0], w0[1], sw), fp8_widen8(w0[2], w0[3], sw), fp8_widen8(w1[0], w1[1], sw), fp8_widen8(w1[2], w1[3], sw)};
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      bf16x8 om[4];
      if constexpr (SRC == 3) {
        const i32x4* pa = reinterpret_cast<const i32x4*>(a.a + ((long long)(kb * 2 + (g >> 1)) * a.m + row[t]) * 64 + (g & 1) * 32);
        const i32x4 a0 = pa[0], a1 = pa[1];
        const float sm = fp8_scale_float(a.sa[((long long)(kb >> 2) * a.nsa + (row[t] >> a.sha)) * 4 + (kb & 3)]);
        om[0] = fp8_widen8(a0[0], a0[1], sm), om[1] = fp8_widen8(a0[2], a0[3], sm);
        om[2] = fp8_widen8(a1[0], a1[1], sm), om[3] = fp8_widen8(a1[2], a1[3], sm);
      } else {
        typedef typename Elem<SRC>::type T;
        const T* px = (const T*)xv + row[t] * ldx;
        float f[4][8];
#pragma unroll
        for (int q = 0; q < 4; ++q) fp8_load8<SRC, VEC>(px, (long long)kb * 128 + g * 32 + q * 8, cols, f[q]);
        float m = fp8_amax<32>(&f[0][0]);
        m = fmaxf(m, __shfl_xor(m, 16, 64));
        m = fmaxf(m, __shfl_xor(m, 32, 64));
        const int sb = fp8_scale_byte(m);
        const float inv = fp8_inv_scale(sb), sm = fp8_scale_float((uint32_t)sb);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint2 c = fp8_pack8(f[q], inv);
          om[q] = fp8_widen8((int)c.x, (int)c.y, sm);
        }
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(on[q], om[q], acc[t], 0, 0, 0);
    }
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) *reinterpret_cast<f32x4*>(&s_acc[wave][t][lane][0]) = acc[t];
  __syncthreads();
  // accumulator e of a lane: n = 4 (lane / 16) + e, m = lane % 16
  if (threadIdx.x < MT * 64) {
    const int t = threadIdx.x >> 6;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < WAVES; ++w) v += *reinterpret_cast<const f32x4*>(&s_acc[w][t][lane][0]);
    float o[4] = {v[0], v[1], v[2], v[3]};
    const long long m = m0 + t * 16 + r;
    if (m < a.m && n0 + 4 * g < a.n) mm_finish(a, m, n0 + 4 * g, o);
  }
}

// split-K: add the partials in order (four loads in flight), then the epilogue.  A product that is split has at most 256 tiles, so its
// elements count in 32 bits
__global__ __launch_bounds__(256) void fp8_mm_finish_kernel(const MmArgs a) {
  const uint32_t n4 = (uint32_t)(a.n + 3) >> 2, total = (uint32_t)a.m * n4;
  const long long slab = a.m * a.n;
  for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < total; i += gridDim.x * 256) {
    const uint32_t m = i / n4;
    const int n = (int)(i - m * n4) * 4;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    const float* p = a.part + (long long)m * a.n + n;
    if ((a.n & 3) == 0) {
      int k = 0;
      for (; k + 4 <= a.ksplit; k += 4, p += 4 * slab) {
        float4 t[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) t[u] = *reinterpret_cast<const float4*>(p + u * slab);
#pragma unroll
        for (int u = 0; u < 4; ++u) v[0] += t[u].x, v[1] += t[u].y, v[2] += t[u].z, v[3] += t[u].w;
      }
      for (; k < a.ksplit; ++k, p += slab) {
        const float4 t = *reinterpret_cast<const float4*>(p);
        v[0] += t.x, v[1] += t.y, v[2] += t.z, v[3] += t.w;
      }
    } else {
      for (int k = 0; k < a.ksplit; ++k, p += slab)
        for (int e = 0; e < 4 && n + e < a.n; ++e) v[e] += p[e];
    }
    mm_finish(a, m, n, v);
  }
}

struct MmPlan {
  int few, bm, ksplit;               // few: fp8_mm_few_kernel; bm: activations per tile (of 128 weights)
  long long tm;
  int tn;
  long long ws;
};

// Which kernel (us at m x n x k; the other sides measured in the same run):
//   up to MM_FEW rows    fp8_mm_few_kernel
//   256 x 128 tiles      long K and enough of them for two blocks per CU: half the bytes per MFMA (8192 x 4096 x 4096: 217, 128 rows 230)
//   128 x 128            at least 512 of them, or a K long enough to make 512 by splitting with 16 blocks of 128 to each split (the
//                        weight gradients: 512 x 768 x 67200: 60, 64 rows 67; 67200 x 512 x 768: 58, 64 rows 62, 256 rows 59)
//   64 x 128             everything between: twice the blocks hide each other's latency, for 6 instead of 4 conversions per MFMA
//                        (16800 x 256 x 1024: 17 against 20, 4200 x 512 x 2048: 21 / 26, 977 x 333 x 1131: 15 / 19)
// K is split until there are 512 blocks, as long as every split keeps four blocks of 128.
constexpr int MM_BLOCKS = 512;
// Up to MM_FEW_QUANT rows the few-rows kernel quantises x itself, in every block again (a call with a 512 x 2048 weight: 16 rows 11 us,
// 17 rows behind a quantiser launch 15); with 64 rows that repeated work took 28 us against 10 behind a quantiser launch.
constexpr int MM_FEW = 64, MM_FEW_QUANT = 16;
int mm_plan(const sm_fp8_matmul_desc* d, MmPlan* p) {
  if (d == nullptr) return SM_ERR_BAD_ARG;
  if (d->m < 0 || d->n < 1 || d->k < 1) return SM_ERR_BAD_SHAPE;
  if ((d->a_block_rows != 1 && d->a_block_rows != 128) || (d->b_block_rows != 1 && d->b_block_rows != 128) ||
      d->out_dtype < SM_DT_BF16 || d->out_dtype > SM_DT_F32)
    return SM_ERR_BAD_ARG;
  if (d->y_stride < d->n || d->n > 0x7fffff00 || d->k > 0x7fffff00) return SM_ERR_BAD_SHAPE;
  p->few = d->m <= MM_FEW;
  if (p->few && d->n > 16LL * 0x3ff000) return SM_ERR_UNSUPPORTED;     // (blocks of 1024 threads: fewer than 2^32 in a launch)
  const long long tn = sm_cdiv(d->n, 128);
  const int nkb = sm_cdiv(d->k, 128);
  const long long t128 = (d->m + 127) / 128 * tn;
  p->bm = d->k >= 2048 && (d->m + 255) / 256 * tn >= MM_BLOCKS ? 256 : (t128 >= MM_BLOCKS || t128 * nkb >= 16 * MM_BLOCKS ? 128 : 64);
  p->tm = (d->m + p->bm - 1) / p->bm;
  p->tn = (int)tn;
  const long long tiles = p->tm * p->tn;
  if (tiles > 0xfff000) return SM_ERR_UNSUPPORTED;
  p->ksplit = tiles == 0 || p->few ? 1 : (int)std::max<long long>(1, std::min<long long>(MM_BLOCKS / tiles, nkb / 4));
  p->ws = p->ksplit > 1 ? (long long)p->ksplit * d->m * d->n * 4 : 0;
  return SM_OK;
}

}  // namespace

extern "C" int64_t sm_fp8_codes_bytes(int64_t rows, int64_t cols) {
  return rows < 0 || cols < 0 ? SM_ERR_BAD_SHAPE : (cols + 127) / 128 * rows * 128;
}
extern "C" int64_t sm_fp8_scales_bytes(int64_t rows, int64_t cols, int block_rows) {
  if (block_rows != 1 && block_rows != 128) return SM_ERR_BAD_ARG;
  return rows < 0 || cols < 0 ? SM_ERR_BAD_SHAPE : (cols + 511) / 512 * ((rows + block_rows - 1) / block_rows) * 4;
}

namespace {
struct QuantArgs {
  const void *x, *gate;
  long long rows, cols, ldx, ldg;
  int square;
  uint8_t *q, *scale, *qt, *scalet;
  float* colsum;
};
template <int DT>
int fp8_quant_launch(const QuantArgs& a, hipStream_t s) {
  typedef typename Elem<DT>::type T;
  const int per16 = 16 / sm_dtype_bytes(DT);
  const bool vec = ((uintptr_t)a.x & 15) == 0 && a.ldx % per16 == 0 && (!a.gate || (((uintptr_t)a.gate & 15) == 0 && a.ldg % per16 == 0));
  const int nkb = sm_cdiv(a.cols, 128);
  if (!a.square && !a.qt && !a.colsum && !a.gate) {    // rows alone: no tile, no LDS
    if (a.rows > 64LL * 0xfff000 / nkb) return SM_ERR_UNSUPPORTED;           // blocks of one launch
    const long long blocks = (a.rows * nkb + 63) / 64;
    const uint32_t inv = nkb > 1 && nkb < 64 ? (uint32_t)(((1ull << 32) + nkb - 1) / nkb) : 0u;   // k / nkb = the high word of k inv, k < 128
    if (vec) hipLaunchKernelGGL((fp8_quant_rows_kernel<DT, true>), dim3((unsigned)blocks), dim3(256), 0, s, (const T*)a.x, a.rows, a.cols, a.ldx, nkb, inv, a.q, a.scale);
    else hipLaunchKernelGGL((fp8_quant_rows_kernel<DT, false>), dim3((unsigned)blocks), dim3(256), 0, s, (const T*)a.x, a.rows, a.cols, a.ldx, nkb, inv, a.q, a.scale);
    SM_LAUNCH_CHECK();
    return SM_OK;
  }
  const long long rb = (a.rows + 127) / 128;
  if (rb * nkb > 0xfff000) return SM_ERR_UNSUPPORTED;   // blocks of one launch
#define SM_Q(V, S_)                                                                                                               \
  hipLaunchKernelGGL((fp8_quant_pair_kernel<DT, V, S_>), dim3((unsigned)(rb * nkb)), dim3(256), 0, s, (const T*)a.x, (const T*)a.gate, \
                     a.rows, a.cols, a.ldx, a.ldg, nkb, (int)rb, a.q, a.scale, a.qt, a.scalet, a.colsum)
  if (a.square) {
    if (vec) SM_Q(true, true);
    else SM_Q(false, true);
  } else {
    if (vec) SM_Q(true, false);
    else SM_Q(false, false);
  }
#undef SM_Q
  SM_LAUNCH_CHECK();
  return SM_OK;
}
int fp8_quant_run(int dtype, const QuantArgs& a, hipStream_t s) {
  if (dtype == SM_DT_BF16) return fp8_quant_launch<SM_DT_BF16>(a, s);
  if (dtype == SM_DT_F16) return fp8_quant_launch<SM_DT_F16>(a, s);
  return fp8_quant_launch<SM_DT_F32>(a, s);
}
bool fp8_out_ok(const void* q, const void* scale) {
  return (q == nullptr) == (scale == nullptr) && ((uintptr_t)q & 15) == 0 && ((uintptr_t)scale & 3) == 0;
}
}  // namespace

extern "C" int64_t sm_fp8_quantize_workspace(int64_t rows, int64_t cols, int col_sum) {
  if (rows < 0 || cols < 1) return SM_ERR_BAD_SHAPE;
  return col_sum ? (rows + 127) / 128 * cols * 4 : 0;
}

extern "C" int sm_fp8_quantize(int dtype, const void* x, int64_t rows, int64_t cols, int64_t x_stride, int block_rows, const void* gate,
                               int64_t gate_stride, void* q, void* scale, void* q_t, void* scale_t, float* col_sum, void* workspace,
                               int64_t workspace_bytes, sm_stream_t stream) {
  if (dtype < SM_DT_BF16 || dtype > SM_DT_F32 || (block_rows != 1 && block_rows != 128)) return SM_ERR_BAD_ARG;
  if (rows < 0 || cols < 1 || x_stride < cols || cols > 0x7fffff00 || rows > (int64_t)1 << 40) return SM_ERR_BAD_SHAPE;
  if (q_t && (rows < 1 || rows > 0x7fffff00)) return SM_ERR_BAD_SHAPE;     // (the transpose sums over the rows)
  if (gate && gate_stride < cols) return SM_ERR_BAD_SHAPE;
  if (!fp8_out_ok(q, scale) || !fp8_out_ok(q_t, scale_t) || (rows > 0 && !q && !q_t && !col_sum)) return SM_ERR_BAD_ARG;
  if (col_sum && cols > 32LL * 0x3ff000) return SM_ERR_UNSUPPORTED;         // (a launch dimension holds fewer than 2^32 threads)
  hipStream_t s = sm_hip_stream(stream);
  if (rows == 0) {
    if (col_sum && sm_zero_async(col_sum, sizeof(float) * cols, s) != hipSuccess) return SM_ERR_LAUNCH;
    return SM_OK;
  }
  if (!x) return SM_ERR_BAD_ARG;
  if (col_sum && (!workspace || ((uintptr_t)workspace & 15) != 0)) return SM_ERR_BAD_ARG;
  if (col_sum && workspace_bytes < sm_fp8_quantize_workspace(rows, cols, 1)) return SM_ERR_WORKSPACE;
  const QuantArgs a = {x, gate, rows, cols, x_stride, gate_stride, block_rows == 128, (uint8_t*)q, (uint8_t*)scale, (uint8_t*)q_t,
                       (uint8_t*)scale_t, col_sum ? (float*)workspace : nullptr};
  const int st = fp8_quant_run(dtype, a, s);
  if (st != SM_OK || !col_sum) return st;
  hipLaunchKernelGGL(col_sum_finish_kernel, dim3(sm_cdiv(cols, 32)), dim3(1024), 0, s, (const float*)workspace, sm_cdiv(rows, 128), (int)cols, col_sum);
  SM_LAUNCH_CHECK();
  return SM_OK;
}

extern "C" int64_t sm_fp8_matmul_workspace(const sm_fp8_matmul_desc* d) {
  MmPlan p;
  const int st = mm_plan(d, &p);
  if (st != SM_OK) return st;
  return p.ws;
}

namespace {
template <int SRC, bool VEC>
void mm_few_launch(const MmArgs& k, const void* x, long long ldx, long long cols, hipStream_t s) {
  hipLaunchKernelGGL((fp8_mm_few_kernel<SRC, VEC, 1>), dim3(sm_cdiv(k.n, 16)), dim3(1024), 0, s, k, x, ldx, cols);
}

// tiles of 128 weights x BM activations, waves of 64 x WM, two stages
template <int BM, int WM>
void mm_launch(const MmArgs& k, dim3 grid, hipStream_t s) {
  constexpr int waves = 2 * (BM / WM), lds = mm_lds(128, BM, waves, 2);
  if (lds > 65536) (void)sm_lds_optin((const void*)fp8_mm_kernel<128, BM, 64, WM, 2>, lds);     // (a refusal shows in the launch check)
  hipLaunchKernelGGL((fp8_mm_kernel<128, BM, 64, WM, 2>), grid, dim3(waves * 64), lds, s, k);
}

// the product behind its checks.  x != null: a is quantised from it (x_dtype, row stride ldx) -- by the few-rows kernel itself, else into
// the workspace behind the K splits' partials
int mm_run(const sm_fp8_matmul_desc* d, const MmPlan& p, const void* a, const void* a_scale, const void* b, const void* b_scale,
           const float* bias, const void* residual, void* y, void* workspace, int x_dtype, const void* x, long long ldx, hipStream_t s) {
  MmArgs k;
  k.a = (const uint8_t*)a, k.b = (const uint8_t*)b, k.sa = (const uint8_t*)a_scale, k.sb = (const uint8_t*)b_scale;
  k.bias = bias, k.res = residual, k.y = y, k.part = (float*)workspace;
  k.m = d->m, k.n = d->n, k.ldy = d->y_stride, k.ldr = residual ? d->res_stride : 0;
  k.nkb = sm_cdiv(d->k, 128);
  k.nsa = (d->m + d->a_block_rows - 1) / d->a_block_rows, k.nsb = (d->n + d->b_block_rows - 1) / d->b_block_rows;
  k.sha = d->a_block_rows == 128 ? 7 : 0, k.shb = d->b_block_rows == 128 ? 7 : 0;
  k.ksplit = p.ksplit, k.relu = d->relu, k.out = d->out_dtype;
  const int per16 = 16 / sm_dtype_bytes(d->out_dtype);
  k.vec = ((uintptr_t)y & 15) == 0 && d->y_stride % per16 == 0 && (!residual || (((uintptr_t)residual & 15) == 0 && d->res_stride % per16 == 0));
  k.tm = p.tm, k.tn = p.tn;
  const bool on_the_way = x != nullptr && d->m <= MM_FEW_QUANT;
  if (x != nullptr && !on_the_way) {
    uint8_t* q = (uint8_t*)workspace + (p.ws + 15) / 16 * 16;
    uint8_t* sc = q + sm_fp8_codes_bytes(d->m, d->k);
    const QuantArgs qa = {x, nullptr, d->m, d->k, ldx, 0, 0, q, sc, nullptr, nullptr, nullptr};
    const int st = fp8_quant_run(x_dtype, qa, s);
    if (st != SM_OK) return st;
    k.a = q, k.sa = sc;
  }
  if (p.few) {
    if (!on_the_way) {
      if (k.m <= 16) mm_few_launch<3, true>(k, nullptr, 0, 0, s);
      else hipLaunchKernelGGL((fp8_mm_few_kernel<3, true, 4>), dim3(sm_cdiv(k.n, 16)), dim3(1024), 0, s, k, nullptr, 0LL, 0LL);
    } else {
      const bool vec = ((uintptr_t)x & 15) == 0 && ldx % (16 / sm_dtype_bytes(x_dtype)) == 0;
      if (x_dtype == SM_DT_BF16) vec ? mm_few_launch<SM_DT_BF16, true>(k, x, ldx, d->k, s) : mm_few_launch<SM_DT_BF16, false>(k, x, ldx, d->k, s);
      else if (x_dtype == SM_DT_F16) vec ? mm_few_launch<SM_DT_F16, true>(k, x, ldx, d->k, s) : mm_few_launch<SM_DT_F16, false>(k, x, ldx, d->k, s);
      else vec ? mm_few_launch<SM_DT_F32, true>(k, x, ldx, d->k, s) : mm_few_launch<SM_DT_F32, false>(k, x, ldx, d->k, s);
    }
    SM_LAUNCH_CHECK();
    return SM_OK;
  }
  const dim3 grid((unsigned)(p.tm * p.tn), p.ksplit);
  if (p.bm == 256) mm_launch<256, 64>(k, grid, s);
  else if (p.bm == 128) mm_launch<128, 64>(k, grid, s);
  else mm_launch<64, 32>(k, grid, s);
  if (p.ksplit > 1) {
    const long long total = k.m * ((k.n + 3) / 4);
    hipLaunchKernelGGL(fp8_mm_finish_kernel, dim3((unsigned)std::min<long long>((total + 255) / 256, 256 * 16)), dim3(256), 0, s, k);
  }
  SM_LAUNCH_CHECK();
  return SM_OK;
}

int mm_check(const sm_fp8_matmul_desc* d, const void* b, const void* b_scale, const void* residual, const void* y, const void* workspace,
             int64_t workspace_bytes, int64_t need) {
  if (!b || !b_scale || !y || ((uintptr_t)b & 15) != 0 || ((uintptr_t)b_scale & 3) != 0) return SM_ERR_BAD_ARG;
  if (residual && d->res_stride < d->n) return SM_ERR_BAD_SHAPE;
  if (need > 0 && (!workspace || ((uintptr_t)workspace & 15) != 0)) return SM_ERR_BAD_ARG;
  return workspace_bytes < need ? SM_ERR_WORKSPACE : SM_OK;
}

int64_t linear_ws(const sm_fp8_matmul_desc* d, const MmPlan& p) {
  return d->m <= MM_FEW_QUANT ? 0 : (p.ws + 15) / 16 * 16 + sm_fp8_codes_bytes(d->m, d->k) + sm_fp8_scales_bytes(d->m, d->k, 1);
}
}  // namespace

extern "C" int sm_fp8_matmul(const sm_fp8_matmul_desc* d, const void* a, const void* a_scale, const void* b, const void* b_scale,
                             const float* bias, const void* residual, void* y, void* workspace, int64_t workspace_bytes,
                             sm_stream_t stream) {
  MmPlan p;
  int st = mm_plan(d, &p);
  if (st != SM_OK) return st;
  if (d->m == 0) return SM_OK;
  if (!a || !a_scale || ((uintptr_t)a & 15) != 0 || ((uintptr_t)a_scale & 3) != 0) return SM_ERR_BAD_ARG;
  st = mm_check(d, b, b_scale, residual, y, workspace, workspace_bytes, p.ws);
  if (st != SM_OK) return st;
  return mm_run(d, p, a, a_scale, b, b_scale, bias, residual, y, workspace, 0, nullptr, 0, sm_hip_stream(stream));
}

extern "C" int64_t sm_fp8_linear_workspace(const sm_fp8_matmul_desc* d) {
  MmPlan p;
  const int st = mm_plan(d, &p);
  if (st != SM_OK) return st;
  return linear_ws(d, p);
}

extern "C" int sm_fp8_linear(const sm_fp8_matmul_desc* d, int x_dtype, const void* x, int64_t x_stride, const void* b,
                             const void* b_scale, const float* bias, const void* residual, void* y, void* workspace,
                             int64_t workspace_bytes, sm_stream_t stream) {
  MmPlan p;
  int st = mm_plan(d, &p);
  if (st != SM_OK) return st;
  if (x_dtype < SM_DT_BF16 || x_dtype > SM_DT_F32 || d->a_block_rows != 1) return SM_ERR_BAD_ARG;
  if (x_stride < d->k) return SM_ERR_BAD_SHAPE;
  if (d->m == 0) return SM_OK;
  if (!x) return SM_ERR_BAD_ARG;
  st = mm_check(d, b, b_scale, residual, y, workspace, workspace_bytes, linear_ws(d, p));
  if (st != SM_OK) return st;
  return mm_run(d, p, nullptr, nullptr, b, b_scale, bias, residual, y, workspace, x_dtype, x, x_stride, sm_hip_stream(stream));
}

// ------------------------------------------------------------------------------------------------ a layer's step
namespace {
// sections of a buffer, 256 bytes apart
struct Carve {
  uint8_t* base;
  int64_t at = 0;
  void* take(int64_t bytes) {
    void* p = base == nullptr ? nullptr : base + at;
    at += (bytes + 255) / 256 * 256;
    return p;
  }
};
struct LinMat {                                  // a quantised matrix in such a buffer
  void *codes, *scales;
  LinMat() : codes(nullptr), scales(nullptr) {}
  LinMat(Carve& c, int64_t rows, int64_t cols, int br) : codes(c.take(sm_fp8_codes_bytes(rows, cols))), scales(c.take(sm_fp8_scales_bytes(rows, cols, br))) {}
};

struct LinPlan {
  sm_fp8_matmul_desc y, dx, dw;                  // the three products
  int64_t saved, fwd, bwd;                       // bytes
  LinMat xt, wt;                                 // kept for the backward: the transposes of x and w
  LinMat wq, xq, g, gt;                          // in the workspaces
  void *yws, *colws, *pws;
  int64_t yws_bytes, colws_bytes, pws_bytes;
};

int lin_plan(const sm_fp8_layer_desc* d, void* saved, void* fwd, void* bwd, LinPlan* p) {
  if (d == nullptr) return SM_ERR_BAD_ARG;
  if (d->m < 1 || d->n < 1 || d->k < 1 || d->m > 0x7fffff00 || d->x_stride < d->k || d->dy_stride < d->n) return SM_ERR_BAD_SHAPE;
  if (d->dtype < SM_DT_BF16 || d->dtype > SM_DT_F32 || d->w_dtype < SM_DT_BF16 || d->w_dtype > SM_DT_F32) return SM_ERR_BAD_ARG;
  const int64_t m = d->m, n = d->n, k = d->k;
  p->y = {m, d->n, d->k, 1, 128, d->dtype, d->relu, n, 0};
  p->dx = {m, d->k, d->n, 1, 128, d->dtype, 0, k, 0};
  p->dw = {n, d->k, (int32_t)m, 1, 1, SM_DT_F32, 0, k, 0};
  Carve s{(uint8_t*)saved}, f{(uint8_t*)fwd}, b{(uint8_t*)bwd};
  if (d->need_dw) p->xt = LinMat(s, k, m, 1);
  if (d->need_dx) p->wt = LinMat(s, k, n, 128);
  if (!d->have_wq) p->wq = LinMat(f, n, k, 128);
  if (d->need_dw) p->xq = LinMat(f, m, k, 1);
  p->yws_bytes = d->need_dw ? sm_fp8_matmul_workspace(&p->y) : sm_fp8_linear_workspace(&p->y);
  if (p->yws_bytes < 0) return (int)p->yws_bytes;
  p->yws = f.take(p->yws_bytes);
  if (d->need_dx) p->g = LinMat(b, m, n, 1);
  if (d->need_dw) p->gt = LinMat(b, n, m, 1);
  p->colws_bytes = d->need_db ? sm_fp8_quantize_workspace(m, n, 1) : 0;
  p->colws = b.take(p->colws_bytes);
  const int64_t w1 = d->need_dx ? sm_fp8_matmul_workspace(&p->dx) : 0, w2 = d->need_dw ? sm_fp8_matmul_workspace(&p->dw) : 0;
  if (w1 < 0 || w2 < 0) return (int)std::min(w1, w2);
  p->pws_bytes = std::max(w1, w2);
  p->pws = b.take(p->pws_bytes);
  p->saved = s.at, p->fwd = f.at, p->bwd = b.at;
  return SM_OK;
}
bool lin_buf_ok(const void* p, int64_t need) { return need == 0 || (p != nullptr && ((uintptr_t)p & 15) == 0); }
}  // namespace

extern "C" int sm_fp8_layer_bytes(const sm_fp8_layer_desc* d, int64_t* saved, int64_t* forward, int64_t* backward) {
  if (!saved || !forward || !backward) return SM_ERR_BAD_ARG;
  LinPlan p;
  const int st = lin_plan(d, nullptr, nullptr, nullptr, &p);
  if (st == SM_OK) *saved = p.saved, *forward = p.fwd, *backward = p.bwd;
  return st;
}

extern "C" int sm_fp8_layer_fwd(const sm_fp8_layer_desc* d, const void* x, const void* w, int64_t w_stride, const void* w_codes,
                                const void* w_scales, const float* bias, void* y, void* saved, void* workspace, int64_t workspace_bytes,
                                sm_stream_t stream) {
  LinPlan p;
  int st = lin_plan(d, saved, workspace, nullptr, &p);
  if (st != SM_OK) return st;
  if (!x || !y || !lin_buf_ok(saved, p.saved) || !lin_buf_ok(workspace, p.fwd) || (d->have_wq && (!w_codes || !w_scales))) return SM_ERR_BAD_ARG;
  if (workspace_bytes < p.fwd) return SM_ERR_WORKSPACE;
  if (!d->have_wq || d->need_dx) {
    if (!w || w_stride < d->k) return SM_ERR_BAD_ARG;
    st = sm_fp8_quantize(d->w_dtype, w, d->n, d->k, w_stride, 128, nullptr, 0, p.wq.codes, p.wq.scales, p.wt.codes, p.wt.scales, nullptr, nullptr,
                         0, stream);
    if (st != SM_OK) return st;
  }
  const void *wc = d->have_wq ? w_codes : p.wq.codes, *ws = d->have_wq ? w_scales : p.wq.scales;
  if (!d->need_dw)
    return sm_fp8_linear(&p.y, d->dtype, x, d->x_stride, wc, ws, bias, nullptr, y, p.yws, p.yws_bytes, stream);
  st = sm_fp8_quantize(d->dtype, x, d->m, d->k, d->x_stride, 1, nullptr, 0, p.xq.codes, p.xq.scales, p.xt.codes, p.xt.scales, nullptr, nullptr, 0,
                       stream);
  if (st != SM_OK) return st;
  return sm_fp8_matmul(&p.y, p.xq.codes, p.xq.scales, wc, ws, bias, nullptr, y, p.yws, p.yws_bytes, stream);
}

extern "C" int sm_fp8_layer_bwd(const sm_fp8_layer_desc* d, const void* dy, const void* y, const void* saved, void* dx, float* dw, float* dbias,
                                void* workspace, int64_t workspace_bytes, sm_stream_t stream) {
  LinPlan p;
  int st = lin_plan(d, const_cast<void*>(saved), nullptr, workspace, &p);
  if (st != SM_OK) return st;
  if (!dy || !lin_buf_ok(saved, p.saved) || !lin_buf_ok(workspace, p.bwd) || (d->need_dx && !dx) || (d->need_dw && !dw) || (d->need_db && !dbias) ||
      (d->relu && !y))
    return SM_ERR_BAD_ARG;
  if (workspace_bytes < p.bwd) return SM_ERR_WORKSPACE;
  if (!d->need_dx && !d->need_dw && !d->need_db) return SM_OK;
  st = sm_fp8_quantize(d->dtype, dy, d->m, d->n, d->dy_stride, 1, d->relu ? y : nullptr, d->n, p.g.codes, p.g.scales, p.gt.codes, p.gt.scales,
                       d->need_db ? dbias : nullptr, p.colws, p.colws_bytes, stream);
  if (st == SM_OK && d->need_dx)
    st = sm_fp8_matmul(&p.dx, p.g.codes, p.g.scales, p.wt.codes, p.wt.scales, nullptr, nullptr, dx, p.pws, p.pws_bytes, stream);
  if (st == SM_OK && d->need_dw)
    st = sm_fp8_matmul(&p.dw, p.gt.codes, p.gt.scales, p.xt.codes, p.xt.scales, nullptr, nullptr, dw, p.pws, p.pws_bytes, stream);
  return st;
}
