// Activations of rows of scalars and their slopes: 0 identity, 1 relu, 2 sigmoid, 3 silu, 4 gelu (erf).
//
// EXACT: within a few steps of float32.  Otherwise for values that are rounded to 16 bits, by the approximate exponential (two
// steps and |z| 2^-24 relative) and quotient.  The kind is the same for a whole launch, so the branch on it stands outside the loop over the values: inside
// it cost five times the arithmetic (group norm with silu of 786432 rows of 128 in bf16: 427 us with it).
#pragma once
#include "ssc_act.cuh"

namespace ssc {

// Denominators beyond the quick reciprocal's end at its limit: results below 2^-125 become that.  (NaN stays.)
template <bool EXACT>
__device__ __forceinline__ float sigmoid(float z) {
  if (!EXACT) return __fdividef(1.0f, 1.0f + __expf(-z));
  const float d = 1.0f + expf(-z);
  return quick_reciprocal(d > 0x1p125f ? 0x1p125f : d);
}
__device__ __forceinline__ float normal_share(float z) { return 0.5f * (1.0f + erff(z * 0.70710678118654752f)); }

template <bool EXACT, int N>
__device__ __forceinline__ void act_values(float *v, int kind) {
  switch (kind) {
    case 1:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = v[i] < 0.f ? 0.f : v[i];
      break;
    case 2:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = sigmoid<EXACT>(v[i]);
      break;
    case 3:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] *= sigmoid<EXACT>(v[i]);
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
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float t = sigmoid<EXACT>(v[i]);
        s[i] = t * (1.f - t);
        v[i] = t;
      }
      break;
    case 3:
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float t = sigmoid<EXACT>(v[i]);
        s[i] = t * fmaf(v[i], 1.f - t, 1.f);
        v[i] *= t;
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
