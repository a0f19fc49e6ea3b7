// Layer norm over the last dimension, forward and backward.
//
//   mean = sum x / H, var = sum (x - mean)^2 / H, rstd = 1 / sqrt(var + eps)
//   xh = (x - mean) rstd,  y = xh w + b
//   g = dy w,  dx = rstd (g - mean(g) - xh mean(g xh))
//   dw = sum over rows of dy xh,  db = sum over rows of dy
//
// Both passes are bound by memory: the forward pass reads x and writes y (8
// bytes per element), the backward pass reads x and dy and writes dx (12).
// A row is held in registers by a group of 32 to 1024 threads, so it is read
// once and the variance is the sum of squared distances from the row's own
// mean (no cancellation between large sums).  All sums are float32.
//
// The columns' sums dw and db: a block walks rows blockIdx.x, + gridDim.x, ...
// with each thread keeping the sums of its own columns in registers, writes
// one partial row per block into the workspace, and a second kernel adds the
// partial rows in a fixed order (no atomics: the same inputs give the same
// bits).
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <string>

#include "mm_common.cuh"

namespace mm {

// VEC consecutive floats at p, and back.
template <int VEC>
__device__ __forceinline__ void ln_load(const float* p, float* v) {
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
__device__ __forceinline__ void ln_store(float* p, const float* v) {
  if (VEC == 4)
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  else if (VEC == 2)
    *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
  else
    *p = v[0];
}

// Sums of a and b over the G threads that share a row (G = 32: one warp; else
// the whole block of G threads).  Every thread gets the sums.
template <int G>
__device__ __forceinline__ void ln_sum2(float& a, float& b, float2* sm) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  if (G == 32) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __syncthreads();  // the last use of sm is over
  if (lane == 0) sm[warp] = make_float2(a, b);
  __syncthreads();
  const float2 t = lane < G / 32 ? sm[lane] : make_float2(0.f, 0.f);
  a = t.x;
  b = t.y;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
}

struct LnArgs {
  const float *x, *w, *b, *dy;
  float *y, *mean, *rstd;  // backward reads mean and rstd; y is dx there
  float* part;             // backward: [2][blocks][width] partial sums of dw, db
  int64_t rows, xs, dys;   // row strides of x and dy (y and dx are dense)
  int width;
  float eps;
};

constexpr int LN_WARPS = 4;  // rows (warps) per block where one warp holds a row

template <int VEC, int NV, int G>
__global__ void __launch_bounds__(G == 32 ? LN_WARPS * 32 : G) ln_forward_kernel(LnArgs a) {
  __shared__ float2 sm[32];
  const int lane = G == 32 ? threadIdx.x & 31 : threadIdx.x;
  const int64_t row = G == 32 ? (int64_t)blockIdx.x * LN_WARPS + (threadIdx.x >> 5) : blockIdx.x;
  if (row >= a.rows) return;  // whole warps only: G > 32 has one row per block
  const float* x = a.x + row * a.xs;
  float v[NV][VEC];
  float s = 0.f, unused = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * G + lane) * VEC;
    if (c < a.width) {
      ln_load<VEC>(x + c, v[i]);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[i][e] = 0.f;
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < VEC; ++e) s += v[i][e];
  ln_sum2<G>(s, unused, sm);
  const float inv = 1.f / (float)a.width;
  const float mean = s * inv;
  float q = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if ((i * G + lane) * VEC < a.width)
#pragma unroll
      for (int e = 0; e < VEC; ++e) q += (v[i][e] - mean) * (v[i][e] - mean);
  ln_sum2<G>(q, unused, sm);
  const float rstd = 1.f / sqrtf(q * inv + a.eps);
  if (lane == 0) {
    a.mean[row] = mean;
    a.rstd[row] = rstd;
  }
  float* y = a.y + row * (int64_t)a.width;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * G + lane) * VEC;
    if (c < a.width) {
      float w[VEC], b[VEC];
      if (a.w) ln_load<VEC>(a.w + c, w);
      if (a.b) ln_load<VEC>(a.b + c, b);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        float t = (v[i][e] - mean) * rstd;
        if (a.w) t *= w[e];
        if (a.b) t += b[e];
        v[i][e] = t;
      }
      ln_store<VEC>(y + c, v[i]);
    }
  }
}

// Rows too wide for registers: three walks over the row (the second and third
// read it from L2).
__global__ void __launch_bounds__(1024) ln_forward_wide_kernel(LnArgs a) {
  __shared__ float2 sm[32];
  const int64_t row = blockIdx.x;
  const float* x = a.x + row * a.xs;
  float s = 0.f, unused = 0.f;
  for (int c = threadIdx.x; c < a.width; c += 1024) s += x[c];
  ln_sum2<1024>(s, unused, sm);
  const float inv = 1.f / (float)a.width;
  const float mean = s * inv;
  float q = 0.f;
  for (int c = threadIdx.x; c < a.width; c += 1024) q += (x[c] - mean) * (x[c] - mean);
  ln_sum2<1024>(q, unused, sm);
  const float rstd = 1.f / sqrtf(q * inv + a.eps);
  if (threadIdx.x == 0) {
    a.mean[row] = mean;
    a.rstd[row] = rstd;
  }
  float* y = a.y + row * (int64_t)a.width;
  for (int c = threadIdx.x; c < a.width; c += 1024) {
    float t = (x[c] - mean) * rstd;
    if (a.w) t *= a.w[c];
    if (a.b) t += a.b[c];
    y[c] = t;
  }
}

// WARPS rows at a time where one warp holds a row (G = 32).
constexpr int LN_BWD_WARPS = 8;

template <int VEC, int NV, int G, bool COLS>
__global__ void __launch_bounds__(G == 32 ? LN_BWD_WARPS * 32 : G) ln_backward_kernel(LnArgs a) {
  constexpr int RPB = G == 32 ? LN_BWD_WARPS : 1;  // rows per block and step
  __shared__ float2 sm[32];
  const int lane = G == 32 ? threadIdx.x & 31 : threadIdx.x;
  const int sub = G == 32 ? threadIdx.x >> 5 : 0;
  const float inv = 1.f / (float)a.width;
  float w[NV][VEC], dw[NV][VEC], db[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * G + lane) * VEC;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      w[i][e] = 1.f;
      dw[i][e] = db[i][e] = 0.f;
    }
    if (a.w && c < a.width) ln_load<VEC>(a.w + c, w[i]);
  }
  for (int64_t row = (int64_t)blockIdx.x * RPB + sub; row < a.rows; row += (int64_t)gridDim.x * RPB) {
    const float* x = a.x + row * a.xs;
    const float* dy = a.dy + row * a.dys;
    const float mean = a.mean[row], rstd = a.rstd[row];
    float xh[NV][VEC], g[NV][VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G + lane) * VEC;
      if (c < a.width) {
        ln_load<VEC>(x + c, xh[i]);
        ln_load<VEC>(dy + c, g[i]);
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          xh[i][e] = mean;
          g[i][e] = 0.f;
        }
      }
    }
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        xh[i][e] = (xh[i][e] - mean) * rstd;
        if (COLS) {
          dw[i][e] += g[i][e] * xh[i][e];
          db[i][e] += g[i][e];
        }
        g[i][e] *= w[i][e];
        s1 += g[i][e];
        s2 += g[i][e] * xh[i][e];
      }
    if (a.y) {
      ln_sum2<G>(s1, s2, sm);
      s1 *= inv;
      s2 *= inv;
      float* dx = a.y + row * (int64_t)a.width;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * G + lane) * VEC;
        if (c < a.width) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) g[i][e] = rstd * (g[i][e] - s1 - xh[i][e] * s2);
          ln_store<VEC>(dx + c, g[i]);
        }
      }
    }
  }
  if (!COLS) return;
  float* pw = a.part + (int64_t)blockIdx.x * a.width;
  float* pb = pw + (int64_t)gridDim.x * a.width;
  if (G == 32) {
    // Add the warps' sums in a fixed order through shared memory.
    extern __shared__ float acc[];  // [2][LN_BWD_WARPS][NV * 32 * VEC]
    constexpr int W = NV * 32 * VEC;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const int c = (i * 32 + lane) * VEC + e;
        acc[sub * W + c] = dw[i][e];
        acc[(LN_BWD_WARPS + sub) * W + c] = db[i][e];
      }
    __syncthreads();
    for (int c = threadIdx.x; c < a.width; c += LN_BWD_WARPS * 32) {
      float tw = 0.f, tb = 0.f;
#pragma unroll
      for (int k = 0; k < LN_BWD_WARPS; ++k) {
        tw += acc[k * W + c];
        tb += acc[(LN_BWD_WARPS + k) * W + c];
      }
      pw[c] = tw;
      pb[c] = tb;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * G + lane) * VEC;
    if (c < a.width) {
      ln_store<VEC>(pw + c, dw[i]);
      ln_store<VEC>(pb + c, db[i]);
    }
  }
}

// Rows too wide for registers: dx from two walks over the row; the columns'
// sums by ln_columns_kernel.
__global__ void __launch_bounds__(1024) ln_backward_wide_kernel(LnArgs a) {
  __shared__ float2 sm[32];
  const int64_t row = blockIdx.x;
  const float* x = a.x + row * a.xs;
  const float* dy = a.dy + row * a.dys;
  const float mean = a.mean[row], rstd = a.rstd[row];
  const float inv = 1.f / (float)a.width;
  float s1 = 0.f, s2 = 0.f;
  for (int c = threadIdx.x; c < a.width; c += 1024) {
    const float g = dy[c] * (a.w ? a.w[c] : 1.f);
    s1 += g;
    s2 += g * ((x[c] - mean) * rstd);
  }
  ln_sum2<1024>(s1, s2, sm);
  s1 *= inv;
  s2 *= inv;
  float* dx = a.y + row * (int64_t)a.width;
  for (int c = threadIdx.x; c < a.width; c += 1024) {
    const float g = dy[c] * (a.w ? a.w[c] : 1.f);
    dx[c] = rstd * (g - s1 - (x[c] - mean) * rstd * s2);
  }
}

// Partial sums of dw and db over the rows blockIdx.y, + gridDim.y, ...
__global__ void __launch_bounds__(256) ln_columns_kernel(LnArgs a) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.width) return;
  float dw = 0.f, db = 0.f;
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const float g = a.dy[row * a.dys + c];
    dw += g * ((a.x[row * a.xs + c] - a.mean[row]) * a.rstd[row]);
    db += g;
  }
  a.part[(int64_t)blockIdx.y * a.width + c] = dw;
  a.part[((int64_t)gridDim.y + blockIdx.y) * a.width + c] = db;
}

// dw (blockIdx.y 0) or db (1) of 32 columns: 32 threads per column add the
// partial rows k, k + 32, ..., then their sums are added in order (latency: with
// eight threads per column and a plain launch the backward pass took 4 to 6 us
// more, 143 in place of 138 at 16384 x 4096, 29 in place of 23 at 5003 x 1250).
__global__ void __launch_bounds__(1024) ln_finish_kernel(const float* part, int blocks, int width, float* dw,
                                                         float* db) {
  __shared__ float acc[32][33];
  pdl_wait();
  float* out = blockIdx.y ? db : dw;
  if (!out) return;
  const int lane = threadIdx.x & 31, k = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  part += (int64_t)blockIdx.y * blocks * width;
  float s = 0.f;
  if (c < width)
#pragma unroll 4
    for (int r = k; r < blocks; r += 32) s += part[(int64_t)r * width + c];
  acc[k][lane] = s;
  __syncthreads();
  if (k == 0 && c < width) {
#pragma unroll
    for (int j = 1; j < 32; ++j) s += acc[j][lane];
    out[c] = s;
  }
}

// ---------------------------------------------------------------------------
// Choice of a kernel: the widest load that width, strides and pointers allow,
// then the smallest group of threads that holds a row with few enough
// elements per thread (the backward pass also holds dy, w and two sums of
// each element: 8 elements are 40 registers, and 1024 threads have 64 each).
// ---------------------------------------------------------------------------

static int ln_vec(const LnArgs& a) {
  const void* ptrs[] = {a.x, a.w, a.b, a.dy, a.y};
  uint64_t bits = (uint64_t)a.width | (uint64_t)a.xs | (uint64_t)a.dys;
  for (const void* p : ptrs) bits |= (uint64_t)(uintptr_t)p >> 2;
  return bits % 4 == 0 ? 4 : bits % 2 == 0 ? 2 : 1;
}

struct LnPlan {
  int vec, group, each;  // elements per load, threads per row (0: too wide), elements per thread
};

static LnPlan ln_plan(const LnArgs& a, bool backward) {
  struct Choice { int group, each; };
  static const Choice fwd[] = {{32, 4}, {32, 8}, {32, 16}, {32, 32}, {128, 12}, {128, 16}, {256, 12},
                               {256, 16}, {512, 12}, {512, 16}, {512, 24}, {512, 32}};
  static const Choice bwd[] = {{32, 4}, {32, 8}, {32, 16}, {128, 8}, {256, 8}, {512, 8}, {1024, 8}};
  LnPlan p = {ln_vec(a), 0, 0};
  const Choice* c = backward ? bwd : fwd;
  const int n = backward ? (int)(sizeof(bwd) / sizeof(Choice)) : (int)(sizeof(fwd) / sizeof(Choice));
  for (int i = 0; i < n; ++i) {
    if (a.width <= c[i].group * c[i].each) {
      p.group = c[i].group;
      p.each = c[i].each;
      break;
    }
  }
  return p;
}

constexpr int LN_MAX_BLOCKS_PER_SM = 8;

// Backward blocks (= partial rows): as many as an SM's registers hold at once
// (64 per thread, 80 and 128 where a warp's lanes hold 8 and 16 elements), no
// more than there are rows.  Two blocks per SM instead left too few loads in
// flight: 32768 x 2048 took 192 us (4.2 TB/s), 65536 x 1024 283 us (2.8 TB/s).
static int ln_blocks(const LnArgs& a, const LnPlan& p) {
  const int64_t steps = p.group == 32 ? (a.rows + LN_BWD_WARPS - 1) / LN_BWD_WARPS : a.rows;
  const int per_sm = p.group == 0 ? 2 : p.group > 32 ? 1024 / p.group : p.each <= 4 ? 4 : p.each <= 8 ? 3 : 2;
  const int64_t most = (int64_t)sm_count() * per_sm;
  return (int)(steps < 1 ? 1 : steps < most ? steps : most);
}

template <int VEC, int EACH, int G>
static void ln_launch_forward(const LnArgs& a, cudaStream_t s) {
  const int64_t blocks = G == 32 ? (a.rows + LN_WARPS - 1) / LN_WARPS : a.rows;
  ln_forward_kernel<VEC, EACH / VEC, G><<<(unsigned)blocks, G == 32 ? LN_WARPS * 32 : G, 0, s>>>(a);
}

template <int VEC, int EACH, int G>
static void ln_launch_backward(const LnArgs& a, int blocks, bool cols, cudaStream_t s) {
  const int threads = G == 32 ? LN_BWD_WARPS * 32 : G;
  const size_t smem = G == 32 ? (size_t)2 * LN_BWD_WARPS * EACH * 32 * sizeof(float) : 0;
  if (cols)
    ln_backward_kernel<VEC, EACH / VEC, G, true><<<blocks, threads, smem, s>>>(a);
  else
    ln_backward_kernel<VEC, EACH / VEC, G, false><<<blocks, threads, 0, s>>>(a);
}

#define LN_CASE(GR, E, CALL) \
  if (p.group == GR && p.each == E) { CALL; return; }

template <int V>
static void ln_forward_vec(const LnPlan& p, const LnArgs& a, cudaStream_t s) {
#define LN_F(GR, E) LN_CASE(GR, E, (ln_launch_forward<V, E, GR>(a, s)))
  LN_F(32, 4) LN_F(32, 8) LN_F(32, 16) LN_F(32, 32) LN_F(128, 12) LN_F(128, 16) LN_F(256, 12) LN_F(256, 16)
  LN_F(512, 12) LN_F(512, 16) LN_F(512, 24) LN_F(512, 32)
#undef LN_F
}

template <int V>
static void ln_backward_vec(const LnPlan& p, const LnArgs& a, int blocks, bool cols, cudaStream_t s) {
#define LN_B(GR, E) LN_CASE(GR, E, (ln_launch_backward<V, E, GR>(a, blocks, cols, s)))
  LN_B(32, 4) LN_B(32, 8) LN_B(32, 16) LN_B(128, 8) LN_B(256, 8) LN_B(512, 8) LN_B(1024, 8)
#undef LN_B
}
#undef LN_CASE

// Fills what both passes share; the Python layer hands over rows that are dense.
static int ln_setup(const char* who, const float* x, int64_t xs, int64_t rows, int64_t width, const float* w,
                    float* mean, float* rstd, LnArgs* a) {
  const std::string name(who);
  if (rows < 0 || width < 0 || xs < 0) return fail(MM_ERR_INVALID, name + ": negative size or stride");
  if (width > INT32_MAX / 2 || rows > INT32_MAX) return fail(MM_ERR_UNSUPPORTED, name + ": too many rows or columns");
  if (rows > 0 && width > 0 && (!x || !mean || !rstd)) return fail(MM_ERR_INVALID, name + ": null data pointer");
  *a = {};
  a->x = x;
  a->w = w;
  a->mean = mean;
  a->rstd = rstd;
  a->rows = rows;
  a->xs = xs;
  a->width = (int)width;
  return MM_OK;
}

// Partial rows a backward call of this size may need, whichever kernel it runs.
static int64_t ln_partial_rows(int64_t rows) {
  const int64_t most = (int64_t)sm_count() * LN_MAX_BLOCKS_PER_SM;
  return rows < 1 ? 1 : rows < most ? rows : most;
}

}  // namespace mm

using namespace mm;

extern "C" int mm_layer_norm(const float* x, int64_t x_stride, int64_t rows, int64_t width, const float* weight,
                             const float* bias, double eps, float* y, float* mean, float* rstd, void* stream) {
  LnArgs a;
  int rc = ln_setup("mm_layer_norm", x, x_stride, rows, width, weight, mean, rstd, &a);
  if (rc != MM_OK) return rc;
  if (rows == 0) return MM_OK;
  if (width == 0) return fail(MM_ERR_UNSUPPORTED, "mm_layer_norm: rows are empty");
  if (!y) return fail(MM_ERR_INVALID, "mm_layer_norm: null data pointer");
  a.b = bias;
  a.y = y;
  a.eps = (float)eps;
  cudaStream_t s = resolve_stream(stream);
  const LnPlan p = ln_plan(a, false);
  if (p.group == 0)
    ln_forward_wide_kernel<<<(unsigned)a.rows, 1024, 0, s>>>(a);
  else if (p.vec == 4)
    ln_forward_vec<4>(p, a, s);
  else if (p.vec == 2)
    ln_forward_vec<2>(p, a, s);
  else
    ln_forward_vec<1>(p, a, s);
  MM_LAUNCH_CHECK("mm_layer_norm launch");
  return MM_OK;
}

extern "C" int mm_layer_norm_backward_workspace_size(int64_t rows, int64_t width, size_t* bytes) {
  if (bytes == nullptr || rows < 0 || width < 0)
    return fail(MM_ERR_INVALID, "mm_layer_norm_backward_workspace_size: invalid argument");
  if (width > INT32_MAX / 2 || rows > INT32_MAX)
    return fail(MM_ERR_UNSUPPORTED, "mm_layer_norm_backward_workspace_size: too many rows or columns");
  *bytes = (size_t)(2 * ln_partial_rows(rows) * width) * sizeof(float);
  return MM_OK;
}

extern "C" int mm_layer_norm_backward(const float* dy, int64_t dy_stride, const float* x, int64_t x_stride,
                                      int64_t rows, int64_t width, const float* mean, const float* rstd,
                                      const float* weight, float* dx, float* dweight, float* dbias, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  LnArgs a;
  int rc = ln_setup("mm_layer_norm_backward", x, x_stride, rows, width, weight, const_cast<float*>(mean),
                    const_cast<float*>(rstd), &a);
  if (rc != MM_OK) return rc;
  const bool cols = dweight != nullptr || dbias != nullptr;
  if ((!dx && !cols) || width == 0) return MM_OK;
  if (rows > 0 && (!dy || dy_stride < 0)) return fail(MM_ERR_INVALID, "mm_layer_norm_backward: invalid gradient");
  if (rows == 0) {
    cudaStream_t s = resolve_stream(stream);
    for (float* t : {dweight, dbias})
      if (t) MM_CUDA(cudaMemsetAsync(t, 0, (size_t)width * sizeof(float), s), "mm_layer_norm_backward: zero");
    return MM_OK;
  }
  size_t need = 0;
  mm_layer_norm_backward_workspace_size(rows, width, &need);
  if (cols && workspace != nullptr && (workspace_bytes < need || (uintptr_t)workspace % 16 != 0))
    return fail(MM_ERR_INVALID, "mm_layer_norm_backward: the workspace is misaligned or too small");
  cudaStream_t s = resolve_stream(stream);
  Scratch scratch;
  if (cols && workspace == nullptr) {
    if ((rc = scratch.get(need, s)) != MM_OK) return rc;
    workspace = scratch.data;
  }
  a.dy = dy;
  a.dys = dy_stride;
  a.y = dx;
  a.part = (float*)workspace;
  const LnPlan p = ln_plan(a, true);
  const int blocks = ln_blocks(a, p);
  if (p.group == 0) {
    if (dx) ln_backward_wide_kernel<<<(unsigned)rows, 1024, 0, s>>>(a);
    if (cols) ln_columns_kernel<<<dim3((a.width + 255) / 256, blocks), 256, 0, s>>>(a);
  } else if (p.vec == 4) {
    ln_backward_vec<4>(p, a, blocks, cols, s);
  } else if (p.vec == 2) {
    ln_backward_vec<2>(p, a, blocks, cols, s);
  } else {
    ln_backward_vec<1>(p, a, blocks, cols, s);
  }
  MM_LAUNCH_CHECK("mm_layer_norm_backward launch");
  if (cols) {
    MM_CUDA(launch_pdl(ln_finish_kernel, dim3((a.width + 31) / 32, 2), dim3(1024), 0, s, (const float*)a.part,
                       (int)blocks, (int)a.width, dweight, dbias),
            "mm_layer_norm_backward columns launch");
  }
  return MM_OK;
}
