// What the losses over rows of logits share: series in 64 bits that take few
// registers, reductions over a block in one LDS read a lane, and where a row's
// float4s begin.
#pragma once

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "internal.h"
#include "rowtile.h"

namespace oxi {

// exp, log and exp(d) - 1 - d in 64 bits, from their series by Horner's rule: the
// coefficients are literals in scalar registers, so that the code takes few
// vector registers where a row is held in the others.
struct Factorials {
  double inv[16];  // 1/k!
  constexpr Factorials() : inv{} {
    double f = 1.0;
    for (int k = 0; k < 16; ++k) {
      if (k) f *= k;
      inv[k] = 1.0 / f;
    }
  }
};
// A constant in scalar registers (in a vector pair the scheduler loads it early).
__device__ __forceinline__ double scalar(double c) {
  asm("" : "+s"(c));
  return c;
}
constexpr double LN2_HI = 0x1.62e42feep-1, LN2_LO = 0x1.a39ef35793c76p-33;  // ln 2, the first part of 32 bits

// e^x = 2^n e^r, |r| <= ln(2)/2: 13 terms leave r^14/14! < 2^-57.
__device__ __forceinline__ double exp64(double x) {
  if (x < -746.0) return 0.0;
  if (x > 710.0) return (double)__builtin_huge_valf();
  const double n = rint(x * 1.4426950408889634);
  const double r = fma(-n, LN2_LO, fma(-n, LN2_HI, x));
  constexpr Factorials F;
  double p = F.inv[13];
#pragma unroll
  for (int k = 12; k >= 0; --k) p = fma(p, r, scalar(F.inv[k]));
  return __builtin_ldexp(p, (int)n);
}

// x = 2^e m, m in [sqrt(1/2), sqrt(2)): log m = 2 atanh s, s = (m - 1)/(m + 1), |s| < 0.172.
__device__ __forceinline__ double log64(double x) {
  if (x == 0.0) return (double)NEG_INF;
  if (!(x < (double)__builtin_huge_valf())) return x;
  double m = __builtin_amdgcn_frexp_mant(x);
  int e = __builtin_amdgcn_frexp_exp(x);
  if (m < 0.7071067811865476) {
    m += m;
    --e;
  }
  const double s = (m - 1.0) / (m + 1.0), z = s * s;
  double p = 1.0 / 23;
#pragma unroll
  for (int k = 21; k > 0; k -= 2) p = fma(p, z, scalar(1.0 / k));
  return fma((double)e, LN2_HI, fma((double)e, LN2_LO, 2.0 * s * p));
}

// d^2 (1/2! + d/3! + d^2/4! + ...) for small d.
__device__ __forceinline__ double exp_rest(double d) {
  if (!(fabs(d) < 0.5)) return exp64(d) - 1.0 - d;
  constexpr Factorials F;
  double p = F.inv[15];
#pragma unroll
  for (int k = 14; k >= 2; --k) p = fma(p, d, scalar(F.inv[k]));
  return d * d * p;
}

// Reductions over a wave and over the block in a fixed order, the same bits for
// every thread. A block's waves leave a value each in LDS, and every row of 16
// lanes combines all of them: one LDS read a lane. The caller's next reduction
// takes other slots (N/64 values), or a barrier comes between.
template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, 0xF, 0xF, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, 0xF, 0xF, false);
  return __builtin_bit_cast(double, (uint64_t)lo | (uint64_t)hi << 32);
}
__device__ __forceinline__ double readlane_f64(double v, int lane) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)b, lane);
  const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)lo | (uint64_t)hi << 32);
}
struct AddF64 {
  typedef double T;
  __device__ __forceinline__ static T op(T a, T b) { return a + b; }
  template <int C> __device__ __forceinline__ static T move(T v) { return dpp_f64<C>(v); }
  __device__ __forceinline__ static T lane(T v, int l) { return readlane_f64(v, l); }
};
struct AddF32 {
  typedef float T;
  __device__ __forceinline__ static T op(T a, T b) { return a + b; }
  template <int C> __device__ __forceinline__ static T move(T v) { return dpp_f32<C>(v); }
  __device__ __forceinline__ static T lane(T v, int l) { return readlane_f32(v, l); }
};
struct MaxF32 : AddF32 {
  __device__ __forceinline__ static T op(T a, T b) { return fmaxf(a, b); }
};
// The same of two values at once.
struct Two {
  float a, b;
};
template <class R>
struct Both {
  typedef Two T;
  __device__ __forceinline__ static T op(T x, T y) { return {R::op(x.a, y.a), R::op(x.b, y.b)}; }
  template <int C> __device__ __forceinline__ static T move(T v) {
    return {R::template move<C>(v.a), R::template move<C>(v.b)};
  }
  __device__ __forceinline__ static T lane(T v, int l) { return {R::lane(v.a, l), R::lane(v.b, l)}; }
};
template <int N, class R>
__device__ __forceinline__ typename R::T over_block(typename R::T v, typename R::T* slots) {
  v = R::op(v, R::template move<DPP_QUAD_XOR1>(v));
  v = R::op(v, R::template move<DPP_QUAD_XOR2>(v));
  v = R::op(v, R::template move<DPP_ROW_HALF_MIRROR>(v));
  v = R::op(v, R::template move<DPP_ROW_MIRROR>(v));
  v = R::op(R::op(R::lane(v, 0), R::lane(v, 16)), R::op(R::lane(v, 32), R::lane(v, 48)));
  constexpr int W = N / 64;
  static_assert(W == 1 || W == 4 || W == 8 || W == 16);
  if constexpr (W > 1) {
    if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = v;
    __syncthreads();
    v = slots[threadIdx.x & (W - 1)];
    v = R::op(v, R::template move<DPP_QUAD_XOR1>(v));
    v = R::op(v, R::template move<DPP_QUAD_XOR2>(v));
    if constexpr (W > 4) v = R::op(v, R::template move<DPP_ROW_HALF_MIRROR>(v));
    if constexpr (W > 8) v = R::op(v, R::template move<DPP_ROW_MIRROR>(v));
    v = R::lane(v, 0);
  }
  return v;
}
template <int N>
__device__ __forceinline__ double block_sum(double v, double* slots) {
  __syncthreads();
  return over_block<N, AddF64>(v, slots);
}

__device__ __forceinline__ f4 exp2_4(const f4& z) {
  return f4{__builtin_amdgcn_exp2f(z.x), __builtin_amdgcn_exp2f(z.y), __builtin_amdgcn_exp2f(z.z),
            __builtin_amdgcn_exp2f(z.w)};
}

// Classes of a row before its float4s: up to the first 128-byte line, so that a
// wave's accesses are whole lines ((4096, 50257) from the first 16 bytes on: 327
// us), or to the first 16 bytes in short rows.
__device__ __forceinline__ int row_head(const float* row, int C) {
  return (int)((0 - (reinterpret_cast<uintptr_t>(row) >> 2)) & (C >= 256 ? 31u : 3u));
}

// A value that all threads hold, in a scalar register.
__device__ __forceinline__ float uniform(float v) { return readlane_f32(v, 0); }

}  // namespace oxi
