// Activations of rows of scalars and their slopes: 0 identity, 1 relu, 2 sigmoid, 3 silu, 4 gelu (erf).
#pragma once
#include "ssc_act.cuh"

namespace ssc {

__device__ __forceinline__ float sigmoid(float z) { return __frcp_rn(1.0f + expf(-z)); }

__device__ __forceinline__ float act_value(float z, int kind) {
  switch (kind) {
    case 1: return z > 0.f ? z : (z != z ? z : 0.f);
    case 2: return sigmoid(z);
    case 3: return z * sigmoid(z);
    case 4: return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
    default: return z;
  }
}
__device__ __forceinline__ float act_slope(float z, int kind) {
  switch (kind) {
    case 1: return z > 0.f ? 1.f : 0.f;
    case 2: {
      const float s = sigmoid(z);
      return s * (1.f - s);
    }
    case 3: {
      const float s = sigmoid(z);
      return s * fmaf(z, 1.f - s, 1.f);
    }
    // (the density (2 pi)^-1/2 exp(-z^2 / 2))
    case 4: return fmaf(z * 0.39894228040143268f, expf(-0.5f * z * z), 0.5f * (1.0f + erff(z * 0.70710678118654752f)));
    default: return 1.f;
  }
}

}  // namespace ssc
