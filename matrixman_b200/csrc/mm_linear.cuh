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
template <int ACT>
__device__ __forceinline__ float lin_act_t(float z) {
  if (ACT == MM_LINEAR_RELU) return z != z ? z : fmaxf(z, 0.f);
  if (ACT == MM_LINEAR_SILU) return z / (1.f + expf(-z));
  if (ACT == MM_LINEAR_SIGMOID) return lin_sigmoid(z);
  if (ACT == MM_LINEAR_GELU) return 0.5f * z * erfcf(-z * LIN_SQRT_HALF);
  if (ACT == MM_LINEAR_GELU_TANH) return z * lin_sigmoid(LIN_GELU_C * (z + LIN_GELU_A * z * z * z));
  return z;
}

// act'(z) but ReLU's, which selects (below).
template <int ACT>
__device__ __forceinline__ float lin_slope_t(float z) {
  if (ACT == MM_LINEAR_SILU) {
    const float s = lin_sigmoid(z);
    return s * (1.f + z * (1.f - s));
  }
  if (ACT == MM_LINEAR_SIGMOID) {
    const float s = lin_sigmoid(z);
    return s * (1.f - s);
  }
  if (ACT == MM_LINEAR_GELU)
    return 0.5f * erfcf(-z * LIN_SQRT_HALF) + z * expf(-0.5f * z * z) * LIN_INV_SQRT_2PI;
  if (ACT == MM_LINEAR_GELU_TANH) {
    const float s = lin_sigmoid(LIN_GELU_C * (z + LIN_GELU_A * z * z * z));
    return s + z * s * (1.f - s) * LIN_GELU_C * (1.f + 3.f * LIN_GELU_A * z * z);
  }
  return 1.f;
}

// The same for N values with one branch on the activation around all of them.
#define LIN_BY_ACT(CALL)                                                    \
  switch (act) {                                                            \
    case MM_LINEAR_RELU: { CALL(MM_LINEAR_RELU) } break;                    \
    case MM_LINEAR_SILU: { CALL(MM_LINEAR_SILU) } break;                    \
    case MM_LINEAR_SIGMOID: { CALL(MM_LINEAR_SIGMOID) } break;              \
    case MM_LINEAR_GELU: { CALL(MM_LINEAR_GELU) } break;                    \
    case MM_LINEAR_GELU_TANH: { CALL(MM_LINEAR_GELU_TANH) } break;          \
    default: break;                                                         \
  }

template <int N>
__device__ __forceinline__ void lin_act(float (&v)[N], int act) {
#define LIN_CALL(A) _Pragma("unroll") for (int e = 0; e < N; ++e) v[e] = lin_act_t<A>(v[e]);
  LIN_BY_ACT(LIN_CALL)
#undef LIN_CALL
}

// dy act'(z).  ReLU drops dy where z <= 0 whatever it is (an infinity or NaN times
// 0 would be NaN), and passes it where z is NaN, as threshold_backward does.
template <int ACT>
__device__ __forceinline__ float lin_grad_t(float dy, float z) {
  if (ACT == MM_LINEAR_RELU) return z <= 0.f ? 0.f : dy;
  return dy * lin_slope_t<ACT>(z);
}

// v = v act'(z).
template <int N>
__device__ __forceinline__ void lin_times_slope(float (&v)[N], const float (&z)[N], int act) {
#define LIN_CALL(A) _Pragma("unroll") for (int e = 0; e < N; ++e) v[e] = lin_grad_t<A>(v[e], z[e]);
  LIN_BY_ACT(LIN_CALL)
#undef LIN_CALL
}

// What follows the products of one output row and column.
struct LinEpilogue {
  const float* bias;      // [n] or null
  const float* residual;  // row stride rs, or null
  float* z;               // [m][n] values before the activation, or null
  int64_t rs;
  int act, residual_first;  // residual_first: act(z + r), z then holds the sum
  // 16-byte aligned (and the residual's rows a multiple of 16 bytes apart)
  int bias_vec, residual_vec, z_vec;
};

inline LinEpilogue lin_epilogue(const float* bias, const float* residual, int64_t rs, float* z, int act, bool first) {
  return {bias, residual, z, rs, act, first, (uintptr_t)bias % 16 == 0,
          (uintptr_t)residual % 16 == 0 && rs % 4 == 0, (uintptr_t)z % 16 == 0};
}

// N consecutive values (a multiple of four) of row p, of which `left` exist; vec:
// whole ones may move in 16-byte pieces.
template <int N>
__device__ __forceinline__ void lin_load_row(const float* p, int left, bool vec, float (&v)[N]) {
  if (vec && left >= N) {
#pragma unroll
    for (int q = 0; q < N / 4; ++q) {
      const float4 t = reinterpret_cast<const float4*>(p)[q];
      v[4 * q] = t.x; v[4 * q + 1] = t.y; v[4 * q + 2] = t.z; v[4 * q + 3] = t.w;
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] = e < left ? p[e] : 0.f;
}

template <int N>
__device__ __forceinline__ void lin_store_row(float* p, int left, bool vec, const float (&v)[N]) {
  if (vec && left >= N) {
#pragma unroll
    for (int q = 0; q < N / 4; ++q)
      reinterpret_cast<float4*>(p)[q] = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
    return;
  }
#pragma unroll
  for (int e = 0; e < N; ++e)
    if (e < left) p[e] = v[e];
}

// The epilogue of N consecutive columns of one row, stored into c [m][n].  vec:
// n is a multiple of four and c (so every row of it at col) 16-byte aligned.
template <int N>
__device__ __forceinline__ void lin_finish_row(const LinEpilogue& e, float (&v)[N], float* c, int64_t row, int col,
                                               int n, bool vec) {
  const int left = n - col;
  float t[N];
  if (e.bias) {
    lin_load_row<N>(e.bias + col, left, vec && e.bias_vec, t);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += t[i];
  }
  if (e.residual) {
    lin_load_row<N>(e.residual + row * e.rs + col, left, vec && e.residual_vec, t);
    if (e.residual_first) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += t[i];
    }
  }
  if (e.z) lin_store_row<N>(e.z + row * n + col, left, vec && e.z_vec, v);
  lin_act<N>(v, e.act);
  if (e.residual && !e.residual_first) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += t[i];
  }
  lin_store_row<N>(c + row * n + col, left, vec, v);
}

// The same of one value, returned.
__device__ __forceinline__ float lin_finish(const LinEpilogue& e, float v, int64_t row, int col, int n) {
  if (e.bias) v += e.bias[col];
  if (e.residual && e.residual_first) v += e.residual[row * e.rs + col];
  if (e.z) e.z[row * n + col] = v;
  float a[1] = {v};
  lin_act<1>(a, e.act);
  if (e.residual && !e.residual_first) a[0] += e.residual[row * e.rs + col];
  return a[0];
}

}  // namespace mm
