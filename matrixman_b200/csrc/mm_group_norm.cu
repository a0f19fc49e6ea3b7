// Group norm with an activation, forward and backward, over feature maps whose
// memory is channels last ([n, pixels, channels]) or channels first.
//
// With m = pixels * channels / groups values of one image and group:
//   mean = sum x / m, var = sum (x - mean)^2 / m, rstd = 1 / sqrt(var + eps)
//   xh = (x - mean) rstd,  z = xh w + b,  y = act(z)
//   dz = dy act'(z),  g = dz w,  dx = rstd (g - mean(g) - xh mean(g xh))
//   dw = sum over images and pixels of dz xh,  db = the same of dz
//
// Both passes are bound by memory: forward 8 bytes per element, backward 12.
//
// The walking kernels take any size.  A block walks a segment of an image's
// pixels and leaves each channel's moments (or sums) in the workspace, a second
// kernel joins them by group, a third reads the map again and writes y (or dx):
// 12 (20) bytes per element.
//
// Moments are held as a mean and a sum of squared distances from it and joined
// by d^2 n1 n2 / (n1 + n2) (Chan, Golub, LeVeque 1979), so large offsets do not
// cancel.  All sums are float32 in a fixed order, without atomics: the same
// inputs give the same bits.
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <string>

#include "mm_linear.cuh"

namespace mm {

constexpr int GN_THREADS = 256;
constexpr int GN_WARPS = GN_THREADS / 32;
constexpr int GN_ROWS = 4;  // rows (channels last) or vectors (first) loaded at a time by the walking kernels

struct GnArgs {
  const float *x, *dy, *w, *b;
  float *y, *mean, *rstd;   // y is dx in the backward pass
  float* part;              // [2][n segs][channels]: mean and squared distances; sums of dz and dz xh
  float* sums;              // backward: [2][n][groups], means of g and g xh
  int64_t xi, xr, gi, gr;   // distances of images, and of pixels (channels last) or channels, in x and dy
  int64_t segs_n;           // segs * n
  int n, channels, groups, each, pixels;
  int segs, seg;            // segments of an image, pixels of each but the last
  int cols;                 // channels of a block's columns (channels last)
  int act;
  float eps;
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

// Joins (n2, mean2, m2) into (n, mean, m).
__device__ __forceinline__ void gn_join(float& n, float& mean, float& m, float n2, float mean2, float m2) {
  const float all = n + n2;
  if (n2 == 0.f) return;
  const float d = mean2 - mean, share = n2 / all;
  mean += d * share;
  m += m2 + d * d * n * share;
  n = all;
}

// ---------------------------------------------------------------------------
// Walking kernels.  Channels last: thread (p, q) of a block has VEC channels and
// every P-th pixel of its segment.  Channels first: a warp has one channel.
// ---------------------------------------------------------------------------

// What a thread walks: `count` vectors of VEC values, `step` apart in x and y.
template <int VEC, bool LAST>
struct GnWalk {
  int image, seg, c, at, step, end;  // c < 0: nothing; pixels at, at + step, ... < end
  __device__ __forceinline__ GnWalk(const GnArgs& a) {
    int64_t id = blockIdx.x;
    if (LAST) {
      const int q_n = a.cols / VEC, p_n = GN_THREADS / q_n;
      const int q = threadIdx.x % q_n, p = threadIdx.x / q_n;
      c = blockIdx.y * a.cols + q * VEC;
      if (p >= p_n || c >= a.channels) c = -1;
      step = p_n;
      at = p;
    } else {
      id = id * GN_WARPS + (threadIdx.x >> 5);
      c = (int)(id % a.channels);
      id /= a.channels;
      if (id >= a.segs_n) c = -1;
      step = 32 * VEC;
      at = (threadIdx.x & 31) * VEC;
    }
    image = (int)(id / a.segs);
    seg = (int)(id % a.segs);
    const int first = seg * a.seg;
    end = min(first + a.seg, a.pixels);
    at += first;
  }
  __device__ __forceinline__ int64_t offset(int64_t image_step, int64_t row_step) const {
    return LAST ? image * image_step + c : image * image_step + c * row_step;
  }
  // Pixel px of an array whose pixels (channels last) are row_step apart.
  __device__ __forceinline__ int64_t pixel(int px, int64_t row_step) const { return LAST ? px * row_step : px; }
  __device__ __forceinline__ int64_t out(const GnArgs& a) const {
    return (int64_t)image * a.pixels * a.channels + (LAST ? c : (int64_t)c * a.pixels);
  }
};

// The channel's values of group statistics `v` [n][groups].
template <int VEC, bool LAST>
__device__ __forceinline__ void gn_of_groups(const GnArgs& a, const GnWalk<VEC, LAST>& k, const float* v, float* out) {
#pragma unroll
  for (int e = 0; e < VEC; ++e) out[e] = v[(int64_t)k.image * a.groups + (LAST ? k.c + e : k.c) / a.each];
}

template <int VEC, bool LAST>
__device__ __forceinline__ void gn_of_channels(const float* v, int c, float none, float* out) {
#pragma unroll
  for (int e = 0; e < VEC; ++e) out[e] = v ? v[LAST ? c + e : c] : none;
}

// Two values per channel of the block's threads, joined by `F` in a fixed order
// and left in part[0] and part[1].  n: what the thread's values count.
template <int VEC, bool LAST, class F>
__device__ __forceinline__ void gn_leave(const GnArgs& a, const GnWalk<VEC, LAST>& k, float n, const float* u,
                                         const float* v, F join) {
  float* pu = a.part;
  float* pv = pu + a.segs_n * a.channels;
  const int64_t row = ((int64_t)k.image * a.segs + k.seg) * a.channels;
  if (!LAST) {
    float tn = 0.f, tu = 0.f, tv = 0.f;
#pragma unroll
    for (int e = 0; e < VEC; ++e) join(tn, tu, tv, n, u[e], v[e]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float on = __shfl_down_sync(0xffffffffu, tn, o), ou = __shfl_down_sync(0xffffffffu, tu, o),
                  ov = __shfl_down_sync(0xffffffffu, tv, o);
      join(tn, tu, tv, on, ou, ov);
    }
    if ((threadIdx.x & 31) == 0 && k.c >= 0) {
      pu[row + k.c] = tu;
      pv[row + k.c] = tv;
    }
    return;
  }
  __shared__ float sn[GN_THREADS], su[GN_THREADS * VEC], sv[GN_THREADS * VEC];
  sn[threadIdx.x] = n;
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    su[threadIdx.x * VEC + e] = u[e];
    sv[threadIdx.x * VEC + e] = v[e];
  }
  __syncthreads();
  // `lanes` threads join the values of one channel.
  const int q_n = a.cols / VEC, p_n = GN_THREADS / q_n;
  int lanes = 1;
  while (lanes < 32 && 2 * lanes <= p_n) lanes *= 2;
  const int lane = threadIdx.x & (lanes - 1);
  for (int first = 0; first < a.cols; first += GN_THREADS / lanes) {
    const int i = first + threadIdx.x / lanes, c = blockIdx.y * a.cols + i;
    const bool on = i < a.cols && c < a.channels;
    float tn = 0.f, tu = 0.f, tv = 0.f;
    for (int p = lane; on && p < p_n; p += lanes) {
      const int t = p * q_n + i / VEC;
      join(tn, tu, tv, sn[t], su[t * VEC + i % VEC], sv[t * VEC + i % VEC]);
    }
    for (int o = lanes / 2; o > 0; o >>= 1) {
      const float on_ = __shfl_down_sync(0xffffffffu, tn, o), ou = __shfl_down_sync(0xffffffffu, tu, o),
                  ov = __shfl_down_sync(0xffffffffu, tv, o);
      join(tn, tu, tv, on_, ou, ov);
    }
    if (on && lane == 0) {
      pu[row + c] = tu;
      pv[row + c] = tv;
    }
  }
}

template <int VEC, bool LAST>
__global__ void __launch_bounds__(GN_THREADS) gn_moments_kernel(GnArgs a) {
  const GnWalk<VEC, LAST> k(a);
  const float* x = a.x + k.offset(a.xi, a.xr);
  float n = 0.f, mean[VEC], m2[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) mean[e] = m2[e] = 0.f;
  if (k.c >= 0) {
    for (int px = k.at; px < k.end; px += GN_ROWS * k.step) {
      float v[GN_ROWS][VEC];
      int rows = 0;
#pragma unroll
      for (int r = 0; r < GN_ROWS; ++r)
        if (px + r * (int64_t)k.step < k.end) {
          gn_load<VEC>(x + k.pixel(px + r * k.step, a.xr), v[r]);
          rows = r + 1;
        }
      const float nb = (float)rows, share = nb / (n + nb);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        float s = 0.f, q = 0.f;
#pragma unroll
        for (int r = 0; r < GN_ROWS; ++r)
          if (r < rows) s += v[r][e];
        s = rows == GN_ROWS ? s * (1.f / GN_ROWS) : s / nb;
#pragma unroll
        for (int r = 0; r < GN_ROWS; ++r)
          if (r < rows) q += (v[r][e] - s) * (v[r][e] - s);
        const float d = s - mean[e];
        mean[e] += d * share;
        m2[e] += q + d * d * n * share;
      }
      n += nb;
    }
  }
  gn_leave<VEC, LAST>(a, k, n, mean, m2, [](float& an, float& au, float& av, float bn, float bu, float bv) {
    gn_join(an, au, av, bn, bu, bv);
  });
}

// Sums of two values over a block of T threads; every thread gets them.
template <int T>
__device__ __forceinline__ void gn_sum2(float& u, float& v, float2* sm) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    u += __shfl_xor_sync(0xffffffffu, u, o);
    v += __shfl_xor_sync(0xffffffffu, v, o);
  }
  if (T == 32) return;
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = make_float2(u, v);
  __syncthreads();
  u = v = 0.f;
#pragma unroll
  for (int i = 0; i < T / 32; ++i) {
    u += sm[i].x;
    v += sm[i].y;
  }
}

// mean and rstd of one image and group per block of T threads, from the channels'
// segments.
template <int T>
__global__ void __launch_bounds__(T) gn_join_moments_kernel(GnArgs a) {
  __shared__ float2 sm[T / 32];
  pdl_wait();
  const int image = blockIdx.x / a.groups, group = blockIdx.x % a.groups;
  const float* pu = a.part + (int64_t)image * a.segs * a.channels + group * a.each;
  const float* pv = pu + a.segs_n * a.channels;
  const int64_t count = (int64_t)a.segs * a.each;
  const float m = (float)a.pixels * (float)a.each;
  float s = 0.f, q = 0.f;
  for (int64_t i = threadIdx.x; i < count; i += T) {
    const int seg = (int)(i / a.each);
    const float n = (float)min(a.seg, a.pixels - seg * a.seg);
    s += n * pu[(int64_t)seg * a.channels + i % a.each];
  }
  gn_sum2<T>(s, q, sm);
  const float mean = s / m;  // (divided, so that a constant's own mean is exact wherever the sum is)
  s = q = 0.f;
  for (int64_t i = threadIdx.x; i < count; i += T) {
    const int seg = (int)(i / a.each);
    const int64_t at = (int64_t)seg * a.channels + i % a.each;
    const float n = (float)min(a.seg, a.pixels - seg * a.seg), d = pu[at] - mean;
    s += pv[at] + n * d * d;
  }
  gn_sum2<T>(s, q, sm);
  if (threadIdx.x == 0) {
    a.mean[blockIdx.x] = mean;
    a.rstd[blockIdx.x] = 1.f / sqrtf(s / m + a.eps);
  }
}

template <int VEC, bool LAST>
__global__ void __launch_bounds__(GN_THREADS) gn_apply_kernel(GnArgs a) {
  const GnWalk<VEC, LAST> k(a);
  pdl_wait();
  if (k.c < 0) return;
  float mean[VEC], rstd[VEC], w[VEC], b[VEC];
  gn_of_groups<VEC, LAST>(a, k, a.mean, mean);
  gn_of_groups<VEC, LAST>(a, k, a.rstd, rstd);
  gn_of_channels<VEC, LAST>(a.w, k.c, 1.f, w);
  gn_of_channels<VEC, LAST>(a.b, k.c, 0.f, b);
  const float* x = a.x + k.offset(a.xi, a.xr);
  float* y = a.y + k.out(a);
  for (int px = k.at; px < k.end; px += GN_ROWS * k.step) {
    float v[GN_ROWS * VEC];
#pragma unroll
    for (int r = 0; r < GN_ROWS; ++r)
      if (px + r * (int64_t)k.step < k.end) gn_load<VEC>(x + k.pixel(px + r * k.step, a.xr), v + r * VEC);
#pragma unroll
    for (int i = 0; i < GN_ROWS * VEC; ++i) v[i] = (v[i] - mean[i % VEC]) * rstd[i % VEC] * w[i % VEC] + b[i % VEC];
    lin_act<GN_ROWS * VEC>(v, a.act);
#pragma unroll
    for (int r = 0; r < GN_ROWS; ++r)
      if (px + r * (int64_t)k.step < k.end) gn_store<VEC>(y + k.pixel(px + r * k.step, a.channels), v + r * VEC);
  }
}

// xh and dz of N / VEC vectors of x (in `xh` on entry) and dy (in `dz`).
template <int VEC, int N>
__device__ __forceinline__ void gn_slopes(float (&xh)[N], float (&dz)[N], const float* mean, const float* rstd,
                                          const float* w, const float* b, int act) {
  float z[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    xh[i] = (xh[i] - mean[i % VEC]) * rstd[i % VEC];
    z[i] = xh[i] * w[i % VEC] + b[i % VEC];
  }
  lin_times_slope<N>(dz, z, act);
}

// PASS 0: each channel's sums of dz and dz xh; 1: dx.
template <int VEC, bool LAST, int PASS>
__global__ void __launch_bounds__(GN_THREADS) gn_backward_kernel(GnArgs a) {
  constexpr int ROWS = 2;  // (both maps are loaded)
  const GnWalk<VEC, LAST> k(a);
  float u[VEC], v[VEC], mean[VEC], rstd[VEC], w[VEC], b[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) u[e] = v[e] = 0.f;
  if (PASS == 1) pdl_wait();
  if (k.c >= 0) {
    gn_of_groups<VEC, LAST>(a, k, a.mean, mean);
    gn_of_groups<VEC, LAST>(a, k, a.rstd, rstd);
    gn_of_channels<VEC, LAST>(a.w, k.c, 1.f, w);
    gn_of_channels<VEC, LAST>(a.b, k.c, 0.f, b);
    if (PASS == 1) {
      gn_of_groups<VEC, LAST>(a, k, a.sums, u);
      gn_of_groups<VEC, LAST>(a, k, a.sums + (int64_t)a.n * a.groups, v);
    }
    const float* x = a.x + k.offset(a.xi, a.xr);
    const float* dy = a.dy + k.offset(a.gi, a.gr);
    float* dx = PASS == 1 ? a.y + k.out(a) : nullptr;
    for (int px = k.at; px < k.end; px += ROWS * k.step) {
      float xh[ROWS * VEC], dz[ROWS * VEC];
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        if (px + r * (int64_t)k.step < k.end) {
          gn_load<VEC>(x + k.pixel(px + r * k.step, a.xr), xh + r * VEC);
          gn_load<VEC>(dy + k.pixel(px + r * k.step, a.gr), dz + r * VEC);
        } else {
#pragma unroll
          for (int e = 0; e < VEC; ++e) xh[r * VEC + e] = mean[e], dz[r * VEC + e] = 0.f;
        }
      }
      gn_slopes<VEC>(xh, dz, mean, rstd, w, b, a.act);
      if (PASS == 0) {
#pragma unroll
        for (int i = 0; i < ROWS * VEC; ++i) {
          u[i % VEC] += dz[i];
          v[i % VEC] += dz[i] * xh[i];
        }
      } else {
#pragma unroll
        for (int i = 0; i < ROWS * VEC; ++i)
          dz[i] = rstd[i % VEC] * (dz[i] * w[i % VEC] - u[i % VEC] - xh[i] * v[i % VEC]);
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
          if (px + r * (int64_t)k.step < k.end) gn_store<VEC>(dx + k.pixel(px + r * k.step, a.channels), dz + r * VEC);
      }
    }
  }
  if (PASS == 0)
    gn_leave<VEC, LAST>(a, k, 0.f, u, v, [](float&, float& au, float& av, float, float bu, float bv) {
      au += bu;
      av += bv;
    });
}

// Means of g and g xh of one image and group per block.
template <int T>
__global__ void __launch_bounds__(T) gn_join_sums_kernel(GnArgs a) {
  __shared__ float2 sm[T / 32];
  pdl_wait();
  const int image = blockIdx.x / a.groups, group = blockIdx.x % a.groups;
  const float* pu = a.part + (int64_t)image * a.segs * a.channels + group * a.each;
  const float* pv = pu + a.segs_n * a.channels;
  const int64_t count = (int64_t)a.segs * a.each;
  const float inv = 1.f / ((float)a.pixels * (float)a.each);
  float s1 = 0.f, s2 = 0.f;
  for (int64_t i = threadIdx.x; i < count; i += T) {
    const int64_t at = i / a.each * a.channels + i % a.each;
    const float w = a.w ? a.w[group * a.each + i % a.each] : 1.f;
    s1 += w * pu[at];
    s2 += w * pv[at];
  }
  gn_sum2<T>(s1, s2, sm);
  if (threadIdx.x == 0) {
    a.sums[blockIdx.x] = s1 * inv;
    a.sums[(int64_t)a.n * a.groups + blockIdx.x] = s2 * inv;
  }
}

// db (blockIdx.y 0) or dw (1) of 32 channels: 32 threads per channel add the
// partial rows k, k + 32, ..., then their sums are added in order.
__global__ void __launch_bounds__(1024) gn_columns_kernel(const float* part, int64_t rows, int channels, float* db,
                                                          float* dw) {
  __shared__ float acc[32][33];
  pdl_wait();
  float* out = blockIdx.y ? dw : db;
  if (!out) return;
  const int lane = threadIdx.x & 31, k = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  part += (int64_t)blockIdx.y * rows * channels;
  float s = 0.f;
  if (c < channels)
#pragma unroll 4
    for (int64_t r = k; r < rows; r += 32) s += part[r * channels + c];
  acc[k][lane] = s;
  __syncthreads();
  if (k == 0 && c < channels) {
#pragma unroll
    for (int j = 1; j < 32; ++j) s += acc[j][lane];
    out[c] = s;
  }
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------

// The widest load that sizes, distances and addresses allow, along channels or pixels.
static int gn_vec(const GnArgs& a, bool last) {
  uint64_t bits = (uint64_t)(last ? a.channels : a.pixels) | (uint64_t)a.xi | (uint64_t)a.xr | (uint64_t)a.gi |
                  (uint64_t)a.gr;
  for (const void* p : {(const void*)a.x, (const void*)a.dy, (const void*)a.y}) bits |= (uint64_t)(uintptr_t)p >> 2;
  return bits % 4 == 0 ? 4 : bits % 2 == 0 ? 2 : 1;
}

constexpr int64_t GN_BLOCKS = 148 * 8;  // walking blocks that a call of large maps has at least
constexpr int GN_LEAST = 64;            // pixels of a segment, at least (a multiple of what a load takes)

// Segments of an image for the walking kernels: enough blocks to fill the GPU,
// whatever the vector width is, so that the workspace's size follows from the sizes alone.
static int gn_segments(int64_t n, int64_t channels, int64_t pixels) {
  const int64_t columns = n * ((channels + 127) / 128);
  int64_t segs = (GN_BLOCKS + columns - 1) / columns;
  const int64_t most = (pixels + GN_LEAST - 1) / GN_LEAST;
  if (segs > most) segs = most;
  return (int)(segs < 1 ? 1 : segs);
}

static int gn_setup(const char* who, const float* x, int64_t xi, int64_t xr, int64_t n, int64_t channels,
                    int64_t pixels, int64_t groups, const float* w, const float* b, float* mean, float* rstd, int act,
                    GnArgs* a) {
  const std::string name(who);
  if (n < 0 || channels < 0 || pixels < 0 || xi < 0 || xr < 0)
    return fail(MM_ERR_INVALID, name + ": negative size or stride");
  if (groups < 1 || channels % groups != 0)
    return fail(MM_ERR_INVALID, name + ": the channels must divide into the groups");
  if (act < MM_LINEAR_NONE || act > MM_LINEAR_GELU_TANH) return fail(MM_ERR_INVALID, name + ": unknown activation");
  // (pixel and channel indexes are 32 bits wide, and a grid has one block per image and group at most)
  if (n > INT32_MAX / 2 || channels > 1 << 23 || pixels > INT32_MAX / 2 || (channels > 0 && n > INT32_MAX / channels))
    return fail(MM_ERR_UNSUPPORTED, name + ": too many images, channels or pixels");
  *a = {};
  a->x = x;
  a->w = w;
  a->b = b;
  a->mean = mean;
  a->rstd = rstd;
  a->xi = xi;
  a->xr = xr;
  a->n = (int)n;
  a->channels = (int)channels;
  a->groups = (int)groups;
  a->each = (int)(channels / groups);
  a->pixels = (int)pixels;
  a->act = act;
  if (n == 0 || channels == 0 || pixels == 0) return MM_OK;
  if (!x) return fail(MM_ERR_INVALID, name + ": null data pointer");
  const int segs = gn_segments(n, channels, pixels);
  a->seg = (int)(((pixels + segs - 1) / segs + GN_LEAST - 1) / GN_LEAST * GN_LEAST);
  a->segs = (int)((pixels + a->seg - 1) / a->seg);
  a->segs_n = n * a->segs;
  return MM_OK;
}

// Blocks of a walking kernel.
template <int VEC, bool LAST>
static dim3 gn_grid(GnArgs& a) {
  if (!LAST) return dim3((unsigned)((a.segs_n * a.channels + GN_WARPS - 1) / GN_WARPS));
  a.cols = a.channels < GN_THREADS * VEC ? a.channels : GN_THREADS * VEC;
  return dim3((unsigned)a.segs_n, (unsigned)((a.channels + a.cols - 1) / a.cols));
}

// A block of 32 threads per image and group where its partial values are few.
template <class K, class... Args>
static cudaError_t gn_launch_join(K small, K large, const GnArgs& a, cudaStream_t s) {
  const bool few = (int64_t)a.segs * a.each <= 128;
  return launch_pdl(few ? small : large, dim3((unsigned)((int64_t)a.n * a.groups)), dim3(few ? 32 : 256), 0, s, a);
}

template <int VEC, bool LAST>
static cudaError_t gn_walk_forward(GnArgs a, cudaStream_t s) {
  const dim3 grid = gn_grid<VEC, LAST>(a);
  gn_moments_kernel<VEC, LAST><<<grid, GN_THREADS, 0, s>>>(a);
  cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) e = gn_launch_join(gn_join_moments_kernel<32>, gn_join_moments_kernel<256>, a, s);
  return e == cudaSuccess ? launch_pdl(gn_apply_kernel<VEC, LAST>, grid, dim3(GN_THREADS), 0, s, a) : e;
}

template <int VEC, bool LAST>
static cudaError_t gn_walk_backward(GnArgs a, float* dw, float* db, cudaStream_t s) {
  const dim3 grid = gn_grid<VEC, LAST>(a);
  gn_backward_kernel<VEC, LAST, 0><<<grid, GN_THREADS, 0, s>>>(a);
  cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess && (dw || db))
    e = launch_pdl(gn_columns_kernel, dim3((a.channels + 31) / 32, 2), dim3(1024), 0, s, (const float*)a.part,
                   (int64_t)a.segs_n, (int)a.channels, db, dw);
  if (e == cudaSuccess && a.y) {
    e = gn_launch_join(gn_join_sums_kernel<32>, gn_join_sums_kernel<256>, a, s);
    if (e == cudaSuccess) e = launch_pdl(gn_backward_kernel<VEC, LAST, 1>, grid, dim3(GN_THREADS), 0, s, a);
  }
  return e;
}

// Floats of the workspace: two per channel and segment, and two per image and group.
static int64_t gn_floats(const GnArgs& a) {
  return 2 * a.segs_n * a.channels + 2 * (int64_t)a.n * a.groups;
}

static int gn_workspace(const char* who, const GnArgs& a, void** workspace, size_t bytes, Scratch* scratch,
                        cudaStream_t s) {
  const size_t need = (size_t)gn_floats(a) * sizeof(float);
  if (*workspace == nullptr) {
    const int rc = scratch->get(need, s);
    *workspace = scratch->data;
    return rc;
  }
  if (bytes < need || (uintptr_t)*workspace % 16 != 0)
    return fail(MM_ERR_INVALID, std::string(who) + ": the workspace is misaligned or too small");
  return MM_OK;
}

#define GN_BY_VEC(FN, ...)                                                         \
  (last ? vec == 4   ? FN<4, true>(__VA_ARGS__)                                    \
          : vec == 2 ? FN<2, true>(__VA_ARGS__)                                    \
                     : FN<1, true>(__VA_ARGS__)                                    \
        : vec == 4   ? FN<4, false>(__VA_ARGS__)                                   \
          : vec == 2 ? FN<2, false>(__VA_ARGS__)                                   \
                     : FN<1, false>(__VA_ARGS__))

}  // namespace mm

using namespace mm;

extern "C" int mm_group_norm_workspace_size(int64_t n, int64_t channels, int64_t pixels, int64_t groups,
                                            size_t* bytes) {
  if (bytes == nullptr) return fail(MM_ERR_INVALID, "mm_group_norm_workspace_size: invalid argument");
  GnArgs a;
  const float* some = (const float*)16;
  const int rc = gn_setup("mm_group_norm_workspace_size", some, 0, 0, n, channels, pixels, groups, nullptr, nullptr,
                          nullptr, nullptr, 0, &a);
  if (rc == MM_OK) *bytes = (size_t)gn_floats(a) * sizeof(float);
  return rc;
}

extern "C" int mm_group_norm(const float* x, int64_t x_image, int64_t x_row, int64_t n, int64_t channels,
                             int64_t pixels, int64_t groups, int channels_last, const float* weight, const float* bias,
                             double eps, int act, float* y, float* mean, float* rstd, void* workspace,
                             size_t workspace_bytes, void* stream) {
  GnArgs a;
  int rc = gn_setup("mm_group_norm", x, x_image, x_row, n, channels, pixels, groups, weight, bias, mean, rstd, act, &a);
  if (rc != MM_OK) return rc;
  if (n == 0 || channels == 0) return MM_OK;
  if (pixels == 0) return fail(MM_ERR_UNSUPPORTED, "mm_group_norm: images without pixels");
  if (!y || !mean || !rstd) return fail(MM_ERR_INVALID, "mm_group_norm: null data pointer");
  cudaStream_t s = resolve_stream(stream);
  Scratch scratch;
  if ((rc = gn_workspace("mm_group_norm", a, &workspace, workspace_bytes, &scratch, s)) != MM_OK) return rc;
  a.y = y;
  a.eps = (float)eps;
  a.part = (float*)workspace;
  const bool last = channels_last != 0;
  const int vec = gn_vec(a, last);
  MM_CUDA(GN_BY_VEC(gn_walk_forward, a, s), "mm_group_norm launch");
  return MM_OK;
}

extern "C" int mm_group_norm_backward(const float* dy, int64_t dy_image, int64_t dy_row, const float* x,
                                      int64_t x_image, int64_t x_row, int64_t n, int64_t channels, int64_t pixels,
                                      int64_t groups, int channels_last, const float* mean, const float* rstd,
                                      const float* weight, const float* bias, int act, float* dx, float* dweight,
                                      float* dbias, void* workspace, size_t workspace_bytes, void* stream) {
  GnArgs a;
  int rc = gn_setup("mm_group_norm_backward", x, x_image, x_row, n, channels, pixels, groups, weight, bias,
                    const_cast<float*>(mean), const_cast<float*>(rstd), act, &a);
  if (rc != MM_OK) return rc;
  if ((!dx && !dweight && !dbias) || channels == 0) return MM_OK;
  if (n == 0 || pixels == 0) {
    cudaStream_t s = resolve_stream(stream);
    for (float* t : {dweight, dbias})
      if (t) MM_CUDA(cudaMemsetAsync(t, 0, (size_t)channels * sizeof(float), s), "mm_group_norm_backward: zero");
    return MM_OK;
  }
  if (!dy || dy_image < 0 || dy_row < 0) return fail(MM_ERR_INVALID, "mm_group_norm_backward: invalid gradient");
  if (!mean || !rstd) return fail(MM_ERR_INVALID, "mm_group_norm_backward: null statistics");
  cudaStream_t s = resolve_stream(stream);
  Scratch scratch;
  if ((rc = gn_workspace("mm_group_norm_backward", a, &workspace, workspace_bytes, &scratch, s)) != MM_OK) return rc;
  a.dy = dy;
  a.gi = dy_image;
  a.gr = dy_row;
  a.y = dx;
  a.part = (float*)workspace;
  a.sums = a.part + 2 * a.segs_n * channels;
  const bool last = channels_last != 0;
  const int vec = gn_vec(a, last);
  MM_CUDA(GN_BY_VEC(gn_walk_backward, a, dweight, dbias, s), "mm_group_norm_backward launch");
  return MM_OK;
}
