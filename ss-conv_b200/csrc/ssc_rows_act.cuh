// Activations of rows of scalars and their slopes: 0 identity, 1 relu, 2 sigmoid, 3 silu, 4 gelu (erf).
//
// The special-function unit (sixteen lanes a cycle and SM) bounds sigmoids: an exponential and a reciprocal each would be 46 us for the 100 M values
// of 786432 rows of 128.  So two of them share a reciprocal: 1 / d0 = d1 / (d0 d1).  EXACT: the exponential to two steps,
// the reciprocal of the product correctly rounded; otherwise, for values that are rounded to 16 bits, the approximate ones, of which the
// exponential is off by |z| 2^-24 besides, the rounding of its exponent.  Where a product of denominators is beyond 2^124, or not a number, all N values take a
// reciprocal of their own: a sigmoid of a large negative argument has to be as small as it is, and 0 below 2^-125, since SiLU multiplies it by
// the argument.
// The kind is the same for a whole launch, so the branch on it stands outside the loop over the values: inside
// it cost five times the arithmetic.
#pragma once
#include "ssc_act.cuh"
#include "ssc_common.cuh"

namespace ssc {

// 2^v; results below 2^-126 are zero (the instruction that keeps them takes three more).
__device__ __forceinline__ float exp2_quick(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
constexpr float kNoSigmoid = -87.f;         // exp(-87) = 2^-125.5
__device__ __forceinline__ float max_or_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float min_or_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// (of at least 2^-125)
template <bool EXACT>
__device__ __forceinline__ float one_sigmoid(float z) {
  return quick_reciprocal(min_or_nan(1.0f + (EXACT ? expf(-z) : exp2_quick(-1.44269504f * z)), 0x1p125f));
}
template <bool EXACT, int N>
__device__ __forceinline__ void sigmoids(const float *z, float *s) {
  // log2 e as the float next to it and what is left
  constexpr float kHigh = (float)1.4426950408889634, kLow = (float)(1.4426950408889634 - (double)kHigh), kLn2 = 0.69314718f;
  const f32x2 one = pair_of(1.0f, 1.0f), high = pair_of(-kHigh, -kHigh);
  float most = 0.f;
#pragma unroll
  for (int i = 0; i + 1 < N; i += 2) {
    const f32x2 v = pair_of(z[i], z[i + 1]), t = mul_pair(v, high);
    const float2 x = halves(t);
    f32x2 e = pair_of(exp2_quick(x.x), exp2_quick(x.y));
    if (EXACT) {
      // what the product has lost, and its low part: 2^(t + left) = 2^t (1 + left ln 2) for a left below 2^-16
      const f32x2 left = fma_pair(v, pair_of(-kLow, -kLow), fma_pair(v, high, mul_pair(t, pair_of(-1.f, -1.f))));
      e = fma_pair(mul_pair(e, left), pair_of(kLn2, kLn2), e);
    }
    const float2 d = halves(add_pair(e, one));
    const float p = d.x * d.y;
    most = max_or_nan(most, p);
    float r;
    if (EXACT) r = quick_reciprocal(p);
    else asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(p));
    const float2 both = halves(mul_pair(pair_of(r, r), pair_of(d.y, d.x)));
    s[i] = both.x;
    s[i + 1] = both.y;
  }
  if (N > 1 && !(most < 0x1p124f)) {
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = z[i] < kNoSigmoid ? 0.f : one_sigmoid<EXACT>(z[i]);
  }
  if (N % 2 == 1) s[N - 1] = one_sigmoid<EXACT>(z[N - 1]);
}
// Values two at a time: half the instructions.  a * b, a * b + c; each argument is an array or one number for all.
__device__ __forceinline__ f32x2 pair_at(const float *a, int i) { return pair_of(a[i], a[i + 1]); }
__device__ __forceinline__ f32x2 pair_at(float a, int) { return pair_of(a, a); }
__device__ __forceinline__ float one_at(const float *a, int i) { return a[i]; }
__device__ __forceinline__ float one_at(float a, int) { return a; }
template <int N, class A, class B>
__device__ __forceinline__ void multiply(float *d, A a, B b) {
#pragma unroll
  for (int i = 0; i + 1 < N; i += 2) {
    const float2 p = halves(mul_pair(pair_at(a, i), pair_at(b, i)));
    d[i] = p.x;
    d[i + 1] = p.y;
  }
  if (N % 2 == 1) d[N - 1] = one_at(a, N - 1) * one_at(b, N - 1);
}
template <int N, class A, class B, class C>
__device__ __forceinline__ void multiply_add(float *d, A a, B b, C c) {
#pragma unroll
  for (int i = 0; i + 1 < N; i += 2) {
    const float2 p = halves(fma_pair(pair_at(a, i), pair_at(b, i), pair_at(c, i)));
    d[i] = p.x;
    d[i + 1] = p.y;
  }
  if (N % 2 == 1) d[N - 1] = fmaf(one_at(a, N - 1), one_at(b, N - 1), one_at(c, N - 1));
}
__device__ __forceinline__ float normal_share(float z) { return 0.5f * (1.0f + erff(z * 0.70710678118654752f)); }

template <bool EXACT, int N>
__device__ __forceinline__ void act_values(float *v, int kind) {
  float s[N];
  switch (kind) {
    case 1:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = v[i] < 0.f ? 0.f : v[i];
      break;
    case 2:
      sigmoids<EXACT, N>(v, s);
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = s[i];
      break;
    case 3:
      sigmoids<EXACT, N>(v, s);
      if (N % 2 == 1 && v[N - 1] < kNoSigmoid) s[N - 1] = 0.f;
      multiply<N>(v, v, s);
      break;
    case 4:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] *= normal_share(v[i]);
      break;
    default: break;
  }
}

// v: the activations in place, s: their slopes.
template <bool EXACT, int N>
__device__ __forceinline__ void act_slopes(float *v, float *s, int kind) {
  switch (kind) {
    case 1:
#pragma unroll
      for (int i = 0; i < N; ++i) {
        s[i] = v[i] > 0.f ? 1.f : 0.f;
        v[i] = v[i] < 0.f ? 0.f : v[i];
      }
      break;
    case 2:
      sigmoids<EXACT, N>(v, s);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        v[i] = s[i];
        s[i] = v[i] * (1.f - v[i]);
      }
      break;
    case 3:
      sigmoids<EXACT, N>(v, s);
      if (N % 2 == 1 && v[N - 1] < kNoSigmoid) s[N - 1] = 0.f;
      multiply<N>(v, v, s);
      {
        float rest[N];
        multiply_add<N>(rest, s, -1.f, 1.f);
        multiply_add<N>(s, v, rest, s);
      }
      break;
    // (the density (2 pi)^-1/2 exp(-z^2 / 2))
    case 4:
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float t = normal_share(v[i]);
        s[i] = fmaf(v[i] * 0.39894228040143268f, EXACT ? expf(-0.5f * v[i] * v[i]) : __expf(-0.5f * v[i] * v[i]), t);
        v[i] *= t;
      }
      break;
    default:
#pragma unroll
      for (int i = 0; i < N; ++i) s[i] = 1.f;
  }
}

}  // namespace ssc
