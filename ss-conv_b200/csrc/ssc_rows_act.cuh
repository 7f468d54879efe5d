// Activations of rows of scalars and their slopes: 0 identity, 1 relu, 2 sigmoid, 3 silu, 4 gelu (erf).
//
// The special-function unit (sixteen lanes a cycle and SM) bounds sigmoids: an exponential and a reciprocal each would be 46 us for the 100 M values
// of 786432 rows of 128.  So two of them share a reciprocal: 1 / d0 = d1 / (d0 d1).  The exponential is the approximate one, two
// steps and |z| 2^-24 relative, in what is added to one.  EXACT: the correctly rounded reciprocal of the product; otherwise, for
// values that are rounded to 16 bits, the approximate one.  Denominators end at 2^62 (the product stays finite): sigmoids below 2^-62
// become that.
// The kind is the same for a whole launch, so the branch on it stands outside the loop over the values: inside
// it cost five times the arithmetic.
#pragma once
#include "ssc_act.cuh"

namespace ssc {

template <bool EXACT, int N>
__device__ __forceinline__ void sigmoids(const float *z, float *s) {
  float d[N];
#pragma unroll
  for (int i = 0; i < N; ++i) d[i] = fminf(1.0f + __expf(-z[i]), 0x1p62f);      // (a number for NaN too: the neighbour keeps its value)
#pragma unroll
  for (int i = 0; i + 1 < N; i += 2) {
    const float p = d[i] * d[i + 1];
    float r;
    if (EXACT) r = quick_reciprocal(p);
    else asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(p));
    s[i] = r * d[i + 1];
    s[i + 1] = r * d[i];
  }
  if (N % 2 == 1) s[N - 1] = quick_reciprocal(d[N - 1]);
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
      for (int i = 0; i < N; ++i) v[i] = v[i] == v[i] ? s[i] : v[i];
      break;
    case 3:
      sigmoids<EXACT, N>(v, s);
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] *= s[i];
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
        v[i] = v[i] == v[i] ? s[i] : v[i];
        s[i] = v[i] * (1.f - v[i]);
      }
      break;
    case 3:
      sigmoids<EXACT, N>(v, s);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float a = v[i] * s[i];
        s[i] = fmaf(a, 1.f - s[i], s[i]);
        v[i] = a;
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
