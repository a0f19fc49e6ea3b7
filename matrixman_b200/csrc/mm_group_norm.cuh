// Shared by the group-norm kernels: arguments, loads, the plan of the resident kernels.
#pragma once

#include "mm_linear.cuh"

namespace mm {

constexpr int GN_THREADS = 256;
constexpr int GN_WARPS = GN_THREADS / 32;

struct GnArgs {
  const float *x, *dy, *w, *b;
  float *y, *mean, *rstd;   // y is dx in the backward pass
  float *dw, *db;
  float* part;              // [2][n segs][channels]: mean and squared distances; sums of dz and dz xh
  float* sums;              // backward: [2][n][groups], means of g and g xh
  int64_t xi, xr, gi, gr;   // distances of images, and of pixels (channels last) or channels, in x and dy
  int64_t segs_n;           // segs * n
  int n, channels, groups, each, pixels;
  int segs, seg;            // segments of an image, pixels of each but the last
  int cols;                 // channels of a block's columns (channels last)
  int act;
  float eps;
  int* fault;               // the device's fault word (clusters)
  int tries, drop;          // of a wait; whether rank 0 gives nothing (see mm_debug_tc_fault)
};

template <int VEC>
__device__ __forceinline__ void gn_load(const float* p, float* v) {
  if (VEC == 4) {
    const float4 t = *reinterpret_cast<const float4*>(p);
    v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
  } else if (VEC == 2) {
    const float2 t = *reinterpret_cast<const float2*>(p);
    v[0] = t.x; v[1] = t.y;
  } else {
    v[0] = *p;
  }
}

template <int VEC>
__device__ __forceinline__ void gn_store(float* p, const float* v) {
  if (VEC == 4)
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  else if (VEC == 2)
    *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
  else
    *p = v[0];
}

// Two values at a time where there are two (packed float32 instructions; each is
// rounded as its scalar form is): d = a + b, a * b, a * b + c, where b and c repeat
// every P values.
template <int N, int P>
__device__ __forceinline__ void gn_add(float* d, const float* a, const float* b) {
#pragma unroll
  for (int i = 0; i + 1 < N; i += 2) {
    const float2 t = __fadd2_rn(make_float2(a[i], a[i + 1]), make_float2(b[i % P], b[(i + 1) % P]));
    d[i] = t.x;
    d[i + 1] = t.y;
  }
  if (N % 2) d[N - 1] = a[N - 1] + b[(N - 1) % P];
}

template <int N, int P>
__device__ __forceinline__ void gn_mul(float* d, const float* a, const float* b) {
#pragma unroll
  for (int i = 0; i + 1 < N; i += 2) {
    const float2 t = __fmul2_rn(make_float2(a[i], a[i + 1]), make_float2(b[i % P], b[(i + 1) % P]));
    d[i] = t.x;
    d[i + 1] = t.y;
  }
  if (N % 2) d[N - 1] = a[N - 1] * b[(N - 1) % P];
}

template <int N, int PB, int PC>
__device__ __forceinline__ void gn_fma(float* d, const float* a, const float* b, const float* c) {
#pragma unroll
  for (int i = 0; i + 1 < N; i += 2) {
    const float2 t = __ffma2_rn(make_float2(a[i], a[i + 1]), make_float2(b[i % PB], b[(i + 1) % PB]),
                                make_float2(c[i % PC], c[(i + 1) % PC]));
    d[i] = t.x;
    d[i + 1] = t.y;
  }
  if (N % 2) d[N - 1] = fmaf(a[N - 1], b[(N - 1) % PB], c[(N - 1) % PC]);
}

__device__ __forceinline__ float gn_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float gn_inverse(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Sigmoids of N values, as 2^-2 / (2^-2 + 2^(-z log2 e - 2)): the exponent's rounding moves
// them by (|z| + 2) 2^-24 relative, the two approximations by 2^-22 each.  With expf and a
// division in their place SiLU took half of the forward pass's instructions (64 x 80 x
// 80 x 64: 62 us).  The 2^-2 keeps the inverse a normal number wherever 2^(-z log2 e) is below
// infinity, as the approximation returns 0 for others: without it sigmoids below 2^-126, and so
// SiLU from z = -87.3 on, were 0.  Infinity and NaN go through: the exponential overflows to
// infinity, whose inverse is 0.
template <int N>
__device__ __forceinline__ void gn_sigmoid(float* s, const float* z) {
  const float scale[2] = {-1.44269504f, -1.44269504f}, less[2] = {-2.f, -2.f}, quarter[2] = {0.25f, 0.25f};
  gn_fma<N, 2, 2>(s, z, scale, less);
#pragma unroll
  for (int i = 0; i < N; ++i) s[i] = gn_exp2(s[i]);
  gn_add<N, 2>(s, s, quarter);
#pragma unroll
  for (int i = 0; i < N; ++i) s[i] = gn_inverse(s[i]);
  gn_mul<N, 2>(s, s, quarter);
}

// v = act(v).
template <int N>
__device__ __forceinline__ void gn_act(float (&v)[N], int act) {
  if (act == MM_LINEAR_SILU) {
    float s[N];
    gn_sigmoid<N>(s, v);
    gn_mul<N, N>(v, v, s);
  } else if (act == MM_LINEAR_SIGMOID) {
    gn_sigmoid<N>(v, v);
  } else if (act == MM_LINEAR_GELU_TANH) {
    float s[N];
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = LIN_GELU_C * (v[i] + LIN_GELU_A * v[i] * v[i] * v[i]);
    gn_sigmoid<N>(s, s);
    gn_mul<N, N>(v, v, s);
  } else {
    lin_act<N>(v, act);
  }
}

// dz = dz act'(z).  One branch per activation: with the slope selected value by value all
// of them were computed, and the backward pass's first kernel issued in 50 % of its cycles
// instead of 40 % (16 x 128 x 160 x 160: 188 us in place of 184).
template <int N>
__device__ __forceinline__ void gn_times_slope(float (&dz)[N], const float (&z)[N], int act) {
  const float one[2] = {1.f, 1.f};
  if (act == MM_LINEAR_SILU) {  // s + z s (1 - s)
    float s[N], t[N];
    gn_sigmoid<N>(s, z);
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] = -s[i];
    gn_add<N, 2>(t, t, one);
    gn_mul<N, N>(t, t, z);
    gn_fma<N, N, N>(t, t, s, s);
    gn_mul<N, N>(dz, dz, t);
  } else if (act == MM_LINEAR_SIGMOID) {
    float s[N];
    gn_sigmoid<N>(s, z);
#pragma unroll
    for (int i = 0; i < N; ++i) dz[i] *= s[i] * (1.f - s[i]);
  } else if (act == MM_LINEAR_GELU_TANH) {
    float s[N];
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = LIN_GELU_C * (z[i] + LIN_GELU_A * z[i] * z[i] * z[i]);
    gn_sigmoid<N>(s, s);
#pragma unroll
    for (int i = 0; i < N; ++i)
      dz[i] *= s[i] + z[i] * s[i] * (1.f - s[i]) * LIN_GELU_C * (1.f + 3.f * LIN_GELU_A * z[i] * z[i]);
  } else {
    lin_times_slope<N>(dz, z, act);
  }
}

// xh and dz of N / VEC vectors of x (in `xh` on entry) and dy (in `dz`); less is -mean.  ReLU
// takes the forward pass's own z, (x - mean) (w rstd) + b, so that its slope selects what its
// values were selected by: with xh w + b a value within a rounding of 0 could pass its gradient
// though it was off, or the other way round.
template <int VEC, int N>
__device__ __forceinline__ void gn_slopes(float (&xh)[N], float (&dz)[N], const float* less, const float* rstd,
                                          const float* w, const float* b, int act) {
  gn_add<N, VEC>(xh, xh, less);
  if (act == MM_LINEAR_RELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float z = fmaf(xh[i], w[i % VEC] * rstd[i % VEC], b[i % VEC]);
      dz[i] = lin_grad_t<MM_LINEAR_RELU>(dz[i], z);
    }
  }
  gn_mul<N, VEC>(xh, xh, rstd);
  if (act == MM_LINEAR_NONE || act == MM_LINEAR_RELU) return;
  float z[N];
  gn_fma<N, VEC, VEC>(z, xh, w, b);
  gn_times_slope<N>(dz, z, act);
}

// How the resident kernels divide a call: a unit is one image's `slab` groups (all
// pixels of their channels), held in the shared memory of a cluster of `ranks`
// blocks, or `units` (a power of two) images' units in one block.  A column is a
// vector of VEC channels (channels last) or a channel (first); a row is a pixel, or a
// vector of VEC pixels.
struct GnPlan {
  int ranks = 0;         // 0: too large for a cluster
  int threads;           // of a block: 256, 512 or 1024
  int slab, slabs;       // groups of a unit, units of an image
  int units, blocks;     // images of a block, and how many such there are
  int q, columns;        // columns of a unit and of an image
  int q_log, p_log;      // 2^q_log lanes hold a unit's, 2^p_log rows are walked at a time
  int rows, all;         // rows of a block and of an image
  int each;              // of a group: parts of columns (channels last; a vector may have several groups'), columns
  int lanes;             // of a group's columns that are neighbouring lanes, a power of two
  int entries;           // partial results of a block
  int smem;
  float inv_each, inv_slab;
};

constexpr int GN_RANKS = 16;    // blocks of a cluster, at most
constexpr int GN_GROUPS = 128;  // groups of a block, at most

// The way of a call on the current device: with clusters only where the device can place
// them.
GnPlan gn_plan(const GnArgs& a, int vec, bool last, bool backward);
// The same with clusters of at most `most` blocks (0: none is held on chip), wherever they
// can be placed.
GnPlan gn_plan_of(const GnArgs& a, int vec, bool last, bool backward, int most);
int gn_debug_ranks(int device, int most);
int64_t gn_plan_rows(int64_t n, int64_t pixels);  // partial rows that dw and db may take
// (the backward pass leaves p.blocks * p.ranks partial rows of dw and db)
cudaError_t gn_resident_forward(const GnArgs& a, const GnPlan& p, int vec, bool last, cudaStream_t s);
cudaError_t gn_resident_backward(const GnArgs& a, const GnPlan& p, int vec, bool last, cudaStream_t s);

}  // namespace mm
