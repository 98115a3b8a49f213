// 16-byte access to rows of bf16 / f16 / f32 values and the activations of the row kernels, in f32.
#pragma once
#include "common.h"

template <int DT>
struct Elem;   // DT = sm_dtype
template <>
struct Elem<SM_DT_BF16> {
  typedef uint16_t type;
  static __device__ __forceinline__ float load(const type* p) { return bf16_bits_to_f32(*p); }
  static __device__ __forceinline__ void store(type* p, float v) { *p = (type)f32_to_bf16_bits(v); }
  typedef uint4 raw8;
  static __device__ __forceinline__ raw8 load8(const type* p) { return *reinterpret_cast<const uint4*>(p); }
  static __device__ __forceinline__ void unpack(const raw8& r, float* f) { unpack_bf16x8(r, f); }
  static __device__ __forceinline__ void store8(type* p, const float* f) { *reinterpret_cast<uint4*>(p) = pack_bf16x8(f); }
};
template <>
struct Elem<SM_DT_F16> {
  typedef _Float16 type;
  static __device__ __forceinline__ float load(const type* p) { return (float)*p; }
  static __device__ __forceinline__ void store(type* p, float v) { *p = (_Float16)v; }
  typedef uint4 raw8;
  static __device__ __forceinline__ raw8 load8(const type* p) { return *reinterpret_cast<const uint4*>(p); }
  static __device__ __forceinline__ void unpack(const raw8& r, float* f) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint16_t lo = (uint16_t)(w[j] & 0xffffu), hi = (uint16_t)(w[j] >> 16);
      f[2 * j] = (float)__builtin_bit_cast(_Float16, lo);
      f[2 * j + 1] = (float)__builtin_bit_cast(_Float16, hi);
    }
  }
  static __device__ __forceinline__ void store8(type* p, const float* f) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)      // one conversion per value, round to nearest even (the packed conversion rounds to zero)
      w[j] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)f[2 * j]) |
             ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)f[2 * j + 1]) << 16);
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <>
struct Elem<SM_DT_F32> {
  typedef float type;
  static __device__ __forceinline__ float load(const type* p) { return *p; }
  static __device__ __forceinline__ void store(type* p, float v) { *p = v; }
  struct raw8 {
    float4 a, b;
  };
  static __device__ __forceinline__ raw8 load8(const type* p) {
    return raw8{*reinterpret_cast<const float4*>(p), *reinterpret_cast<const float4*>(p + 4)};
  }
  static __device__ __forceinline__ void unpack(const raw8& r, float* f) {
    f[0] = r.a.x, f[1] = r.a.y, f[2] = r.a.z, f[3] = r.a.w, f[4] = r.b.x, f[5] = r.b.y, f[6] = r.b.z, f[7] = r.b.w;
  }
  static __device__ __forceinline__ void store8(type* p, const float* f) {
    *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(f[4], f[5], f[6], f[7]);
  }
};

static inline int sm_dtype_bytes(int dt) { return dt == SM_DT_F32 ? 4 : 2; }

// VEC = 8: 16-byte (f32: 2 x 16-byte) accesses; VEC = 1: any alignment
template <int DT, int VEC>
struct RowVec {
  typedef Elem<DT> E;
  typedef typename E::type T;
  typedef typename E::raw8 raw;
  static __device__ __forceinline__ raw load(const T* p) { return E::load8(p); }
  static __device__ __forceinline__ void unpack(const raw& r, float* f) { E::unpack(r, f); }
  static __device__ __forceinline__ void store(T* p, const float* f) { E::store8(p, f); }
};
template <int DT>
struct RowVec<DT, 1> {
  typedef Elem<DT> E;
  typedef typename E::type T;
  typedef T raw;
  static __device__ __forceinline__ raw load(const T* p) { return *p; }
  static __device__ __forceinline__ void unpack(const raw& r, float* f) { f[0] = E::load(&r); }
  static __device__ __forceinline__ void store(T* p, const float* f) { E::store(p, f[0]); }
};

// sigmoid(t) = 1 / (1 + 2^(-t log2 e)) on the hardware exp2 and reciprocal (1 ulp each).  Absolute errors: t sigmoid(t) is off by at most
// (0.7 + 6 |t sigmoid(t)|) 2^-24 (the exponent's rounding is 1.3 |t| 2^-24 of e^-t), its derivative by (5 + 2 t) 2^-24 up to t = 17 (from
// 1 - sigmoid(t)), 5 * 2^-24 for t < 0; relative to the derivative that is not small near its zero at t = -1.278.  The library expf and an
// IEEE division made SiLU 1.7 times as long as the copy it rides on.
__device__ __forceinline__ float fast_sigmoid(float t) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(t * -1.4426950408889634f));
}

// q = Phi(-|t|) and e = exp(-t^2 / 2) of a standard normal t.  erfc(z) = exp(-z^2) s P(s) with s = 1 / (1 + 0.4 z): P is a degree-8
// least-squares fit (reweighted to equal ripple) of erfcx(z) / s over 0 <= z <= 10, relative error 6.8e-8, so that the tail keeps its
// relative precision (1 + erf(u) cancels there) and the exponential is shared with the density.  The library erfcf took 2 x the time of
// the copy a GELU rides on.
__device__ __forceinline__ void normal_tail(float t, float& q, float& e) {
  const float z = __builtin_fabsf(t) * 0.70710678118654752f, s = __builtin_amdgcn_rcpf(__builtin_fmaf(z, 0.4f, 1.f));
  float p = 0.04125313088297844f;
  p = __builtin_fmaf(p, s, -0.14031966030597687f);
  p = __builtin_fmaf(p, s, 0.08398815244436264f);
  p = __builtin_fmaf(p, s, 0.08796337246894836f);
  p = __builtin_fmaf(p, s, 0.07975713908672333f);
  p = __builtin_fmaf(p, s, 0.19339294731616974f);
  p = __builtin_fmaf(p, s, 0.20188765227794647f);
  p = __builtin_fmaf(p, s, 0.2264430969953537f);
  p = __builtin_fmaf(p, s, 0.22563423216342926f);
  e = __builtin_amdgcn_exp2f(z * z * -1.4426950408889634f);
  q = 0.5f * (s * p * e);
}

// act(t).  NaN stays NaN (fmaxf() would swallow it; the 2019 maximum is one instruction as well).
template <int ACT>
__device__ __forceinline__ float act_fwd(float t) {
  if constexpr (ACT == SM_ACT_RELU) return __builtin_elementwise_maximum(t, 0.f);
  if constexpr (ACT == SM_ACT_SILU) return t * fast_sigmoid(t);
  if constexpr (ACT == SM_ACT_GELU) {
    float q, e;
    normal_tail(t, q, e);
    return t * (t < 0.f ? q : 1.f - q);
  }
  return t;
}
// d act / d t.  The ReLU's border is the caller's (it decides a whole gradient).
template <int ACT>
__device__ __forceinline__ float act_grad(float t) {
  if constexpr (ACT == SM_ACT_RELU) return t <= 0.f ? 0.f : 1.f;
  if constexpr (ACT == SM_ACT_SILU) {
    const float s = fast_sigmoid(t);
    return s * __builtin_fmaf(t, 1.f - s, 1.f);
  }
  if constexpr (ACT == SM_ACT_GELU) {
    float q, e;
    normal_tail(t, q, e);
    return __builtin_fmaf(t * 0.3989422804014327f, e, t < 0.f ? q : 1.f - q);
  }
  return 1.f;
}
