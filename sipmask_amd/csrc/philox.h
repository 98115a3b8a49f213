// Counter-based random bits of the dropout paths: Philox-4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as
// 1, 2, 3", SC 2011), written from the paper's round function.  Nothing is stored: element i of a call draws 16-bit lane i % 8 of the
// block with counter (i / 8 as 64 bits, offset as 64 bits) and key = seed, so the backward pass regenerates the forward's mask.
//
// 16 bits per element, not 32: one block then serves 8 elements.  A block is 20 32x32->64 multiplies (quarter rate) and 40 xors, about
// 500 cycles of a SIMD for 64 lanes; at 4 elements a block the generator alone would cap the chip at ~1.2e12 elements/s, which is
// what HBM delivers for 16-bit read + write, at 8 it stays under the memory time.  The price is the resolution of p: multiples of
// 2^-16, and the kept values are scaled by the reciprocal of the probability that is really used, so the mean is exact.
#pragma once
#include "common.h"

struct DropArgs {
  unsigned long long seed, offset;
  const long long* offset_dev;   // added to offset when not null (a captured graph advances it between replays)
  unsigned int thr;              // keep iff lane >= thr; 0 = keep all, 65536 = drop all
  float scale;                   // 65536 / (65536 - thr)
};

__device__ __forceinline__ unsigned long long drop_offset(const DropArgs& d) {
  return d.offset + (d.offset_dev != nullptr ? (unsigned long long)*d.offset_dev : 0ull);
}

// the four words of block `idx8`
__device__ __forceinline__ void philox10(unsigned long long idx8, unsigned long long offset, unsigned long long seed, uint32_t (&c)[4]) {
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
  c[0] = (uint32_t)idx8, c[1] = (uint32_t)(idx8 >> 32), c[2] = (uint32_t)offset, c[3] = (uint32_t)(offset >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const unsigned long long p0 = (unsigned long long)c[0] * 0xD2511F53u, p1 = (unsigned long long)c[2] * 0xCD9E8D57u;
    const uint32_t n0 = __builtin_amdgcn_bitop3_b32((uint32_t)(p1 >> 32), c[1], k0, 0x96);   // a ^ b ^ c in one instruction
    const uint32_t n2 = __builtin_amdgcn_bitop3_b32((uint32_t)(p0 >> 32), c[3], k1, 0x96);
    c[1] = (uint32_t)p1, c[3] = (uint32_t)p0, c[0] = n0, c[2] = n2;
    k0 += 0x9E3779B9u, k1 += 0xBB67AE85u;
  }
}

// keep bits of the block's 8 elements
__device__ __forceinline__ uint32_t drop_keep8(unsigned long long idx8, unsigned long long offset, unsigned long long seed, uint32_t thr) {
  uint32_t c[4], m = 0;
  philox10(idx8, offset, seed, c);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    m |= (c[j] & 0xffffu) >= thr ? 1u << (2 * j) : 0u;
    m |= (c[j] >> 16) >= thr ? 2u << (2 * j) : 0u;
  }
  return m;
}

// 0 <= thr <= 65536 -> host-side arguments; scale is finite for thr = 65536 as well (nothing is kept)
static inline int drop_args_fill(DropArgs* a, int thr, uint64_t seed, uint64_t offset, const int64_t* offset_dev) {
  if (thr < 0 || thr > 65536) return SM_ERR_BAD_ARG;
  a->seed = seed, a->offset = offset, a->offset_dev = (const long long*)offset_dev, a->thr = (unsigned int)thr;
  a->scale = thr < 65536 ? 65536.f / (float)(65536 - thr) : 0.f;
  return SM_OK;
}
