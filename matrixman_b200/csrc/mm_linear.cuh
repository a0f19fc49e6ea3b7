// Shared by the kernels of the linear operator: activations and their slopes.
#pragma once

#include <math.h>

#include "mm_common.cuh"

namespace mm {

constexpr float LIN_GELU_C = 1.5957691216057308f;   // 2 sqrt(2 / pi)
constexpr float LIN_GELU_A = 0.044715f;
constexpr float LIN_SQRT_HALF = 0.70710678118654752f;
constexpr float LIN_INV_SQRT_2PI = 0.39894228040143268f;

__device__ __forceinline__ float lin_sigmoid(float z) { return 1.f / (1.f + expf(-z)); }

// act(z).  GELU goes through erfc, which keeps its relative accuracy where
// 1 + erf cancels; the tanh form is z sigmoid(2 sqrt(2/pi) (z + 0.044715 z^3)).
__device__ __forceinline__ float lin_act(float z, int act) {
  switch (act) {
    case MM_LINEAR_RELU: return z != z ? z : fmaxf(z, 0.f);
    case MM_LINEAR_SILU: return z / (1.f + expf(-z));
    case MM_LINEAR_SIGMOID: return lin_sigmoid(z);
    case MM_LINEAR_GELU: return 0.5f * z * erfcf(-z * LIN_SQRT_HALF);
    case MM_LINEAR_GELU_TANH: return z * lin_sigmoid(LIN_GELU_C * (z + LIN_GELU_A * z * z * z));
    default: return z;
  }
}

// act'(z); ReLU's slope at 0 is 0.
__device__ __forceinline__ float lin_slope(float z, int act) {
  switch (act) {
    case MM_LINEAR_RELU: return z > 0.f ? 1.f : 0.f;
    case MM_LINEAR_SILU: {
      const float s = lin_sigmoid(z);
      return s * (1.f + z * (1.f - s));
    }
    case MM_LINEAR_SIGMOID: {
      const float s = lin_sigmoid(z);
      return s * (1.f - s);
    }
    case MM_LINEAR_GELU:
      return 0.5f * erfcf(-z * LIN_SQRT_HALF) + z * expf(-0.5f * z * z) * LIN_INV_SQRT_2PI;
    case MM_LINEAR_GELU_TANH: {
      const float s = lin_sigmoid(LIN_GELU_C * (z + LIN_GELU_A * z * z * z));
      return s + z * s * (1.f - s) * LIN_GELU_C * (1.f + 3.f * LIN_GELU_A * z * z);
    }
    default: return 1.f;
  }
}

// What follows the products of one output row and column.
struct LinEpilogue {
  const float* bias;      // [n] or null
  const float* residual;  // row stride rs, or null
  float* z;               // [m][n] values before the activation, or null
  int64_t rs;
  int act, residual_first;  // residual_first: act(z + r), z then holds the sum
};

__device__ __forceinline__ float lin_finish(const LinEpilogue& e, float v, int64_t row, int col, int n) {
  if (e.bias) v += e.bias[col];
  if (e.residual && e.residual_first) v += e.residual[row * e.rs + col];
  if (e.z) e.z[row * n + col] = v;
  v = lin_act(v, e.act);
  if (e.residual && !e.residual_first) v += e.residual[row * e.rs + col];
  return v;
}

}  // namespace mm
