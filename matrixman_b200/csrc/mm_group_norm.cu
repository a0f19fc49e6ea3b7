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
// Maps whose groups fit a cluster's shared memory are read once
// (mm_group_norm_resident.cu).  The walking kernels here take any size.  A block
// walks a segment of an image's pixels and leaves each channel's moments (or sums) in
// the workspace, a second kernel joins them by group, a third reads the map again and
// writes y (or dx): 12 (20) bytes per element.  2 x 128 x 512 x 512 with SiLU takes 145 us
// (5.6 TB/s) forward and 219 us (6.1 TB/s) backward.
//
// Moments are held as a mean and a sum of squared distances from it and joined
// by d^2 n1 n2 / (n1 + n2) (Chan, Golub, LeVeque 1979), so large offsets do not
// cancel; those of GN_ROWS rows are taken around the first row's values (see
// mm_group_norm_resident.cu).  A thread adds at most 128 values in float32, a block joins its
// threads in float32 (13 additions), what is added behind that takes float64 every 4 or 8
// values; all in a fixed order, without atomics: the same inputs give the same bits.
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <string>
#include <type_traits>

#include "mm_group_norm.cuh"

namespace mm {

// Rows (channels last) or vectors (first) that a thread of the walking kernels has under
// way: x for the moments, x for the result, x and dy (channels last four of these spill, 16 x
// 128 x 160 x 160 backward 182 us in place of 173; channels first three take 172, four 161).
constexpr int GN_ROWS = 8, GN_APPLY_ROWS = 4, GN_BACK_LAST = 3, GN_BACK_FIRST = 4;

// Blocks of the forward kernels that an SM holds.  Channels last three are the call's one
// wave (see GN_BLOCKS_LAST), and the registers of four would spill (2 x 128 x 512 x 512:
// 154 us in place of 145).
template <bool LAST>
constexpr int gn_held() {
  return LAST ? 3 : 4;
}

// Joins (n2, mean2, m2) into (n, mean, m).  d is all of the mean where n is 0, and its
// square may overflow: it meets n first.
__device__ __forceinline__ void gn_join(float& n, float& mean, float& m, float n2, float mean2, float m2) {
  const float all = n + n2;
  if (n2 == 0.f) return;
  const float d = mean2 - mean, share = n2 / all;
  mean += d * share;
  m += m2 + d * n * (d * share);
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
  // back: from the last segment to the first, since the end of what the kernel before
  // read is still in L2.
  __device__ __forceinline__ GnWalk(const GnArgs& a, bool back = false) {
    int64_t id = back ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
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
__global__ void __launch_bounds__(GN_THREADS, gn_held<LAST>()) gn_moments_kernel(GnArgs a) {
  const GnWalk<VEC, LAST> k(a);
  const float* x = a.x + k.offset(a.xi, a.xr);
  float n = 0.f, mean[VEC], m2[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) mean[e] = m2[e] = 0.f;
  if (k.c >= 0) {
    // GN_ROWS rows around the first one's values, joined to the rows before
    auto batch = [&](auto rows_, int px) {
      constexpr int ROWS = decltype(rows_)::value;
      float v[ROWS][VEC], sum[VEC], squares[VEC], less[VEC];
#pragma unroll
      for (int r = 0; r < ROWS; ++r) gn_load<VEC>(x + k.pixel(px + r * k.step, a.xr), v[r]);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        less[e] = -v[0][e];
        sum[e] = squares[e] = 0.f;
      }
#pragma unroll
      for (int r = 1; r < ROWS; ++r) {
        gn_add<VEC, VEC>(v[r], v[r], less);
        gn_add<VEC, VEC>(sum, sum, v[r]);
        gn_fma<VEC, VEC, VEC>(squares, v[r], v[r], squares);
      }
      constexpr float nb = (float)ROWS, inv = 1.f / nb;
      const float share = nb / (n + nb);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float d = -less[e] + sum[e] * inv - mean[e];
        mean[e] += d * share;
        m2[e] += squares[e] - sum[e] * sum[e] * inv + d * n * (d * share);  // (as gn_join)
      }
      n += nb;
    };
    int px = k.at;
    for (; px + (GN_ROWS - 1) * (int64_t)k.step < k.end; px += GN_ROWS * k.step)
      batch(std::integral_constant<int, GN_ROWS>{}, px);
    if (px + (GN_ROWS / 2 - 1) * (int64_t)k.step < k.end) {
      batch(std::integral_constant<int, GN_ROWS / 2>{}, px);
      px += GN_ROWS / 2 * k.step;
    }
    for (; px < k.end; px += k.step) batch(std::integral_constant<int, 1>{}, px);
  }
  gn_leave<VEC, LAST>(a, k, n, mean, m2, [](float& an, float& au, float& av, float bn, float bu, float bv) {
    gn_join(an, au, av, bn, bu, bv);
  });
}

// Sums of two values over a block of T threads; every thread gets them.
template <int T, class V, class V2>
__device__ __forceinline__ void gn_sum2(V& u, V& v, V2* sm) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    u += __shfl_xor_sync(0xffffffffu, u, o);
    v += __shfl_xor_sync(0xffffffffu, v, o);
  }
  if (T == 32) return;
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = {u, v};
  __syncthreads();
  u = v = 0;
#pragma unroll
  for (int i = 0; i < T / 32; ++i) {
    u += sm[i].x;
    v += sm[i].y;
  }
}

// The sums of both values of term(0 .. count - 1) over a thread's share of them, in float64
// every four.
template <int T, class F>
__device__ __forceinline__ double2 gn_share(unsigned count, F term) {
  double2 s = make_double2(0, 0);
  unsigned i = threadIdx.x;
  for (; i + 3 * T < count; i += 4 * T) {
    const float2 p = term(i), q = term(i + T), r = term(i + 2 * T), t = term(i + 3 * T);
    s.x += (double)((p.x + q.x) + (r.x + t.x));
    s.y += (double)((p.y + q.y) + (r.y + t.y));
  }
  float2 rest = make_float2(0.f, 0.f);
  for (; i < count; i += T) {
    const float2 p = term(i);
    rest.x += p.x;
    rest.y += p.y;
  }
  return make_double2(s.x + (double)rest.x, s.y + (double)rest.y);
}

// mean and rstd of one image and group per block of T threads, from the channels'
// segments.  Their means are weighted and added as distances from the first one's: a constant
// is its own mean, and the sum of all values overflows nowhere.  (The mean itself is rounded
// once, at its own scale: the first part may be far from the others.)
template <int T>
__global__ void __launch_bounds__(T) gn_join_moments_kernel(GnArgs a) {
  __shared__ double2 sm[T / 32];
  pdl_wait();
  const int image = blockIdx.x / a.groups, group = blockIdx.x % a.groups;
  const float* pu = a.part + (int64_t)image * a.segs * a.channels + group * a.each;
  const float* pv = pu + a.segs_n * a.channels;
  const unsigned count = (unsigned)a.segs * a.each, each = a.each;
  const double m = (double)a.pixels * (double)a.each;
  const float first = pu[0];
  auto walk = [&](auto f) {
    return gn_share<T>(count, [&](unsigned i) {
      const int seg = (int)(i / each);
      return make_float2(f((int64_t)seg * a.channels + (i - seg * each), (float)min(a.seg, a.pixels - seg * a.seg)), 0.f);
    });
  };
  double2 s = walk([&](int64_t at, float n) { return n * (pu[at] - first); });
  gn_sum2<T>(s.x, s.y, sm);
  const float mean = (float)((double)first + s.x / m);
  s = walk([&](int64_t at, float n) {
    const float d = pu[at] - mean;
    return pv[at] + n * d * d;
  });
  gn_sum2<T>(s.x, s.y, sm);
  if (threadIdx.x == 0) {
    a.mean[blockIdx.x] = mean;
    a.rstd[blockIdx.x] = 1.f / sqrtf((float)(s.x / m) + a.eps);
  }
}

template <int VEC, bool LAST>
__global__ void __launch_bounds__(GN_THREADS, gn_held<LAST>()) gn_apply_kernel(GnArgs a) {
  const GnWalk<VEC, LAST> k(a, true);
  pdl_wait();
  if (k.c < 0) return;
  float mean[VEC], rstd[VEC], w[VEC], b[VEC];  // mean is negated
  gn_of_groups<VEC, LAST>(a, k, a.mean, mean);
  gn_of_groups<VEC, LAST>(a, k, a.rstd, rstd);
  gn_of_channels<VEC, LAST>(a.w, k.c, 1.f, w);
  gn_of_channels<VEC, LAST>(a.b, k.c, 0.f, b);
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    mean[e] = -mean[e];
    w[e] *= rstd[e];
  }
  const float* x = a.x + k.offset(a.xi, a.xr);
  float* y = a.y + k.out(a);
  auto apply = [&](auto rows_, int px) {
    constexpr int N = decltype(rows_)::value * VEC;
    float v[N];
#pragma unroll
    for (int r = 0; r < N / VEC; ++r) gn_load<VEC>(x + k.pixel(px + r * k.step, a.xr), v + r * VEC);
    gn_add<N, VEC>(v, v, mean);
    gn_fma<N, VEC, VEC>(v, v, w, b);
    gn_act<N>(v, a.act);
#pragma unroll
    for (int r = 0; r < N / VEC; ++r) gn_store<VEC>(y + k.pixel(px + r * k.step, a.channels), v + r * VEC);
  };
  int px = k.at;
  for (; px + (GN_APPLY_ROWS - 1) * (int64_t)k.step < k.end; px += GN_APPLY_ROWS * k.step)
    apply(std::integral_constant<int, GN_APPLY_ROWS>{}, px);
  for (; px < k.end; px += k.step) apply(std::integral_constant<int, 1>{}, px);
}

// Batches of rows that a thread adds in float32; it adds the sums of more of them in float64,
// in its own place in shared memory.  (Of values of one sign every addition rounds the same
// way, and a thread may have thousands of rows; one of 16 x 128 x 160 x 160 has 120.)
constexpr int GN_FOLD = 32;

// PASS 0: each channel's sums of dz and dz xh; 1: dx.
template <int VEC, bool LAST, int PASS>
__global__ void __launch_bounds__(GN_THREADS, 3) gn_backward_kernel(GnArgs a) {
  const GnWalk<VEC, LAST> k(a, PASS == 1);
  float u[VEC], v[VEC], less[VEC], rstd[VEC], w[VEC], b[VEC];  // less: -mean
#pragma unroll
  for (int e = 0; e < VEC; ++e) u[e] = v[e] = 0.f;
  if (PASS == 1) pdl_wait();
  if (k.c >= 0) {
    gn_of_groups<VEC, LAST>(a, k, a.mean, less);
    gn_of_groups<VEC, LAST>(a, k, a.rstd, rstd);
    gn_of_channels<VEC, LAST>(a.w, k.c, 1.f, w);
    gn_of_channels<VEC, LAST>(a.b, k.c, 0.f, b);
    if (PASS == 1) {
      gn_of_groups<VEC, LAST>(a, k, a.sums, u);
      gn_of_groups<VEC, LAST>(a, k, a.sums + (int64_t)a.n * a.groups, v);
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      less[e] = -less[e];
      if (PASS == 1) {
        u[e] *= -rstd[e];
        v[e] *= -rstd[e];
      }
    }
    const float* x = a.x + k.offset(a.xi, a.xr);
    const float* dy = a.dy + k.offset(a.gi, a.gr);
    float* dx = PASS == 1 ? a.y + k.out(a) : nullptr;
    auto step = [&](auto rows_, int px) {
      constexpr int N = decltype(rows_)::value * VEC;
      float xh[N], dz[N];
#pragma unroll
      for (int r = 0; r < N / VEC; ++r) {
        gn_load<VEC>(x + k.pixel(px + r * k.step, a.xr), xh + r * VEC);
        gn_load<VEC>(dy + k.pixel(px + r * k.step, a.gr), dz + r * VEC);
      }
#pragma unroll
      for (int r = 0; r < N; r += VEC) {  // (a vector at a time, for the registers)
        float(&h)[VEC] = *reinterpret_cast<float(*)[VEC]>(xh + r);
        float(&z)[VEC] = *reinterpret_cast<float(*)[VEC]>(dz + r);
        gn_slopes<VEC>(h, z, less, rstd, w, b, a.act);
        if (PASS == 0) {
          gn_add<VEC, VEC>(u, u, z);
          gn_fma<VEC, VEC, VEC>(v, z, h, v);
        } else {  // dx = rstd w dz - (rstd s2 xh + rstd s1)
          gn_fma<VEC, VEC, VEC>(h, h, v, u);
          gn_mul<VEC, VEC>(z, z, w);
          gn_fma<VEC, VEC, VEC>(z, z, rstd, h);
          gn_store<VEC>(dx + k.pixel(px + r / VEC * k.step, a.channels), z);
        }
      }
    };
    constexpr int ROWS = LAST ? GN_BACK_LAST : GN_BACK_FIRST;
    __shared__ double sums[2][VEC][PASS == 0 ? GN_THREADS : 1];  // (a thread's own)
    int batches = 0;
    auto fold = [&] {
      const bool first = batches == GN_FOLD;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        double &su = sums[0][e][threadIdx.x], &sv = sums[1][e][threadIdx.x];
        su = (first ? 0 : su) + (double)u[e];
        sv = (first ? 0 : sv) + (double)v[e];
        u[e] = v[e] = 0.f;
      }
    };
    int px = k.at;
    for (; px + (ROWS - 1) * (int64_t)k.step < k.end; px += ROWS * k.step) {
      step(std::integral_constant<int, ROWS>{}, px);
      if (PASS == 0 && ++batches % GN_FOLD == 0) fold();
    }
    for (; px < k.end; px += k.step) step(std::integral_constant<int, 1>{}, px);
    if (PASS == 0 && batches >= GN_FOLD)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        u[e] = (float)(sums[0][e][threadIdx.x] + (double)u[e]);
        v[e] = (float)(sums[1][e][threadIdx.x] + (double)v[e]);
      }
  }
  if (PASS == 0)
    gn_leave<VEC, LAST>(a, k, 0.f, u, v, [](float&, float& au, float& av, float, float bu, float bv) {
      au += bu;
      av += bv;
    });
}

constexpr int GN_COLUMNS = 4;  // channels of a block that adds partial rows
constexpr int GN_COLUMN_THREADS = GN_THREADS / GN_COLUMNS;

// db and dw of a block's channels: 64 threads per channel add the partial rows k, k +
// 64, ... (in float64 every eight, as there may be as many rows as images), then their sums
// are added in order.
__device__ __forceinline__ void gn_add_rows(const GnArgs& a, int block, double2 (*acc)[GN_COLUMNS + 1]) {
  const int lane = threadIdx.x % GN_COLUMNS, k = threadIdx.x / GN_COLUMNS;
  const int c = block * GN_COLUMNS + lane;
  const float* pu = a.part + c;
  const float* pv = pu + a.segs_n * a.channels;
  double2 s = make_double2(0, 0);
  if (c < a.channels) {
    constexpr int EACH = 8;
    int64_t r = k;
    for (; r + (EACH - 1) * GN_COLUMN_THREADS < a.segs_n; r += EACH * GN_COLUMN_THREADS) {
      float u = 0.f, v = 0.f;
#pragma unroll
      for (int e = 0; e < EACH; ++e) {
        u += pu[(r + e * GN_COLUMN_THREADS) * a.channels];
        v += pv[(r + e * GN_COLUMN_THREADS) * a.channels];
      }
      s.x += (double)u;
      s.y += (double)v;
    }
    float u = 0.f, v = 0.f;
    for (; r < a.segs_n; r += GN_COLUMN_THREADS) {
      u += pu[r * a.channels];
      v += pv[r * a.channels];
    }
    s.x += (double)u;
    s.y += (double)v;
  }
  acc[k][lane] = s;
  __syncthreads();
  if (k == 0 && c < a.channels) {
    for (int j = 1; j < GN_COLUMN_THREADS; ++j) {
      s.x += acc[j][lane].x;
      s.y += acc[j][lane].y;
    }
    if (a.db) a.db[c] = (float)s.x;
    if (a.dw) a.dw[c] = (float)s.y;
  }
}

// Means of g and g xh of one image and group per block; the first `columns` blocks add
// the partial rows.
__global__ void __launch_bounds__(GN_THREADS) gn_join_sums_kernel(GnArgs a, int columns) {
  __shared__ double2 acc[GN_COLUMN_THREADS][GN_COLUMNS + 1];
  pdl_wait();
  if ((int)blockIdx.x < columns) {
    gn_add_rows(a, blockIdx.x, acc);
    return;
  }
  const int id = blockIdx.x - columns, image = id / a.groups, group = id % a.groups;
  const float* pu = a.part + (int64_t)image * a.segs * a.channels + group * a.each;
  const float* pv = pu + a.segs_n * a.channels;
  const unsigned count = (unsigned)a.segs * a.each, each = a.each;
  const double inv = 1 / ((double)a.pixels * (double)a.each);
  double2 s = gn_share<GN_THREADS>(count, [&](unsigned i) {
    const unsigned seg = i / each, c = i - seg * each;
    const int64_t at = (int64_t)seg * a.channels + c;
    const float w = a.w ? a.w[group * a.each + c] : 1.f;
    return make_float2(w * pu[at], w * pv[at]);
  });
  gn_sum2<GN_THREADS>(s.x, s.y, &acc[0][0]);
  if (threadIdx.x == 0) {
    a.sums[id] = (float)(s.x * inv);
    a.sums[(int64_t)a.n * a.groups + id] = (float)(s.y * inv);
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

// Into how many slabs of columns the channels are cut (channels last): the fewest, unless
// more leave a tenth less of a block's threads without a column (2 x 100 x 80 x 1280: four slabs
// of 80 vectors in place of 256 and 64, 65 us to 59).
static int gn_slabs(int channels, int vec) {
  const int vectors = (channels + vec - 1) / vec, fewest = (vectors + GN_THREADS - 1) / GN_THREADS;
  int best = fewest;
  float most = 0.f;
  for (int s = fewest; s < fewest + 8 && (s == fewest || vectors / s * vec >= 32); ++s) {
    const int width = (vectors + s - 1) / s;
    const float used = (float)(GN_THREADS / width * width) / GN_THREADS * vectors / ((float)width * s);
    if (used > most + 0.1f) {
      most = used;
      best = s;
    }
  }
  return best;
}

// Walking blocks of a call of large maps.  Channels last one wave of three per SM: with
// five times as many 64 x 64 x 80 x 80 backward took 111 us in place of 102, 33 x 96 x 80 x
// 50 64 in place of 55 (a block's first loads and its joins, and waves that end uneven).
// Channels first segments are short, and several waves even out (2 x 128 x 512 x 512
// forward: 136 us, with one wave 146 to 158).
constexpr int64_t GN_BLOCKS_LAST = 3, GN_BLOCKS_FIRST = 16;  // per SM
constexpr int GN_LEAST = 64;  // pixels of a segment, at least; of few channels as many more as
                              // a block has rows under way

// Cuts images into segments: enough blocks (channels first: warps of one channel) to
// fill the GPU, whatever the vector width is, so that the workspace's size follows from
// the sizes alone.
static void gn_cut(GnArgs* a, bool last) {
  if (a->n == 0 || a->channels == 0 || a->pixels == 0) return;
  const int64_t pixels = a->pixels, channels = a->channels;
  int64_t segs, least = GN_LEAST, step = GN_LEAST;
  if (last) {
    const int64_t walkers = (int64_t)a->n * gn_slabs(a->channels, 4);
    segs = std::max<int64_t>(sm_count() * GN_BLOCKS_LAST / walkers, 1);
    if (channels < 128) least = GN_LEAST * 128 / channels;
    step = 16;
  } else {
    const int64_t walkers = (a->n * channels + GN_WARPS - 1) / GN_WARPS;
    segs = (sm_count() * GN_BLOCKS_FIRST + walkers - 1) / walkers;
  }
  segs = std::min(segs, (pixels + least - 1) / least);
  a->seg = (int)(((pixels + segs - 1) / segs + step - 1) / step * step);
  a->segs = (int)((pixels - 1) / a->seg + 1);
  a->segs_n = (int64_t)a->n * a->segs;
}

static int gn_setup(const char* who, const float* x, int64_t xi, int64_t xr, int64_t n, int64_t channels,
                    int64_t pixels, int64_t groups, bool last, const float* w, const float* b, float* mean, float* rstd,
                    int act, GnArgs* a) {
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
  gn_cut(a, last);
  return MM_OK;
}

// Blocks of a walking kernel.
template <int VEC, bool LAST>
static dim3 gn_grid(GnArgs& a) {
  if (!LAST) return dim3((unsigned)((a.segs_n * a.channels + GN_WARPS - 1) / GN_WARPS));
  const int slabs = gn_slabs(a.channels, VEC);
  a.cols = (a.channels / VEC + slabs - 1) / slabs * VEC;
  return dim3((unsigned)a.segs_n, (unsigned)((a.channels + a.cols - 1) / a.cols));
}

template <int VEC, bool LAST>
static cudaError_t gn_walk_forward(GnArgs a, cudaStream_t s) {
  const dim3 grid = gn_grid<VEC, LAST>(a);
  gn_moments_kernel<VEC, LAST><<<grid, GN_THREADS, 0, s>>>(a);
  cudaError_t e = cudaGetLastError();
  // (few partial values per image and group: a warp each)
  const bool few = (int64_t)a.segs * a.each <= 128;
  if (e == cudaSuccess)
    e = launch_pdl(few ? gn_join_moments_kernel<32> : gn_join_moments_kernel<256>,
                   dim3((unsigned)((int64_t)a.n * a.groups)), dim3(few ? 32 : 256), 0, s, a);
  return e == cudaSuccess ? launch_pdl(gn_apply_kernel<VEC, LAST>, grid, dim3(GN_THREADS), 0, s, a) : e;
}

static int gn_column_blocks(const GnArgs& a) {
  return a.dw || a.db ? (a.channels + GN_COLUMNS - 1) / GN_COLUMNS : 0;
}

template <int VEC, bool LAST>
static cudaError_t gn_walk_backward(GnArgs a, cudaStream_t s) {
  const dim3 grid = gn_grid<VEC, LAST>(a);
  gn_backward_kernel<VEC, LAST, 0><<<grid, GN_THREADS, 0, s>>>(a);
  cudaError_t e = cudaGetLastError();
  const int columns = gn_column_blocks(a);
  const int64_t blocks = columns + (a.y ? (int64_t)a.n * a.groups : 0);
  if (e == cudaSuccess)
    e = launch_pdl(gn_join_sums_kernel, dim3((unsigned)blocks), dim3(GN_THREADS), 0, s, a, columns);
  if (e == cudaSuccess && a.y) e = launch_pdl(gn_backward_kernel<VEC, LAST, 1>, grid, dim3(GN_THREADS), 0, s, a);
  return e;
}

// Floats of the workspace, whichever kernels run: two per channel and segment, and two
// per image and group.
static int64_t gn_floats(const GnArgs& a) {
  int64_t rows = gn_plan_rows(a.n, a.pixels);
  for (const bool last : {true, false}) {
    GnArgs cut = a;
    gn_cut(&cut, last);
    rows = std::max(rows, cut.segs_n);
  }
  return 2 * rows * a.channels + 2 * (int64_t)a.n * a.groups;
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
  const int rc = gn_setup("mm_group_norm_workspace_size", some, 0, 0, n, channels, pixels, groups, true, nullptr,
                          nullptr, nullptr, nullptr, 0, &a);
  if (rc == MM_OK) *bytes = (size_t)gn_floats(a) * sizeof(float);
  return rc;
}

extern "C" int mm_debug_group_norm_ranks(int device, int most) { return gn_debug_ranks(device, most); }

extern "C" int mm_debug_group_norm_plan(int64_t n, int64_t channels, int64_t pixels, int64_t groups, int channels_last,
                                        int backward, int* ranks, int* images, int* segments) {
  GnArgs a;
  const bool last = channels_last != 0;
  const float* some = (const float*)16;
  if (!ranks || !images || !segments) return fail(MM_ERR_INVALID, "mm_debug_group_norm_plan: invalid argument");
  if (const int rc = gn_setup("mm_debug_group_norm_plan", some, 0, 0, n, channels, pixels, groups, last, nullptr,
                              nullptr, nullptr, nullptr, 0, &a))
    return rc;
  if (n == 0 || channels == 0 || pixels == 0)
    return fail(MM_ERR_INVALID, "mm_debug_group_norm_plan: maps without elements");
  const GnPlan p = gn_plan_of(a, gn_vec(a, last), last, backward != 0, GN_RANKS);
  *ranks = p.ranks;
  *images = p.ranks ? p.units : 0;
  *segments = p.ranks ? 0 : a.segs;
  return MM_OK;
}

extern "C" int mm_group_norm(const float* x, int64_t x_image, int64_t x_row, int64_t n, int64_t channels,
                             int64_t pixels, int64_t groups, int channels_last, const float* weight, const float* bias,
                             double eps, int act, float* y, float* mean, float* rstd, void* workspace,
                             size_t workspace_bytes, void* stream) {
  GnArgs a;
  int rc = gn_setup("mm_group_norm", x, x_image, x_row, n, channels, pixels, groups, channels_last != 0, weight, bias,
                    mean, rstd, act, &a);
  if (rc != MM_OK) return rc;
  if (n == 0 || channels == 0) return MM_OK;
  if (pixels == 0) return fail(MM_ERR_UNSUPPORTED, "mm_group_norm: images without pixels");
  if (!y || !mean != !rstd) return fail(MM_ERR_INVALID, "mm_group_norm: null data pointer");
  cudaStream_t s = resolve_stream(stream);
  a.y = y;
  a.eps = (float)eps;
  const bool last = channels_last != 0;
  const int vec = gn_vec(a, last);
  const GnPlan plan = gn_plan(a, vec, last, false);
  Scratch scratch;
  if (workspace != nullptr || plan.ranks == 0)
    if ((rc = gn_workspace("mm_group_norm", a, &workspace, workspace_bytes, &scratch, s)) != MM_OK) return rc;
  a.part = (float*)workspace;
  if (plan.ranks == 0 && !mean) {
    a.mean = a.part + 2 * a.segs_n * channels;
    a.rstd = a.mean + (int64_t)a.n * a.groups;
  }
  if (plan.ranks > 0) {
    MM_CUDA(gn_resident_forward(a, plan, vec, last, s), "mm_group_norm launch");
    return MM_OK;
  }
  MM_CUDA(GN_BY_VEC(gn_walk_forward, a, s), "mm_group_norm launch");
  return MM_OK;
}

extern "C" int mm_group_norm_backward(const float* dy, int64_t dy_image, int64_t dy_row, const float* x,
                                      int64_t x_image, int64_t x_row, int64_t n, int64_t channels, int64_t pixels,
                                      int64_t groups, int channels_last, const float* mean, const float* rstd,
                                      const float* weight, const float* bias, int act, float* dx, float* dweight,
                                      float* dbias, void* workspace, size_t workspace_bytes, void* stream) {
  GnArgs a;
  int rc = gn_setup("mm_group_norm_backward", x, x_image, x_row, n, channels, pixels, groups, channels_last != 0, weight, bias,
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
  a.dy = dy;
  a.gi = dy_image;
  a.gr = dy_row;
  a.y = dx;
  a.dw = dweight;
  a.db = dbias;
  const bool last = channels_last != 0, columns = dweight || dbias;
  const int vec = gn_vec(a, last);
  const GnPlan plan = gn_plan(a, vec, last, true);
  Scratch scratch;
  if (workspace != nullptr || plan.ranks == 0 || columns)
    if ((rc = gn_workspace("mm_group_norm_backward", a, &workspace, workspace_bytes, &scratch, s)) != MM_OK) return rc;
  if (plan.ranks > 0) {
    a.part = columns ? (float*)workspace : nullptr;
    a.segs_n = (int64_t)plan.blocks * plan.ranks;  // partial rows
    MM_CUDA(gn_resident_backward(a, plan, vec, last, s), "mm_group_norm_backward launch");
    if (columns)
      MM_CUDA(launch_pdl(gn_join_sums_kernel, dim3(gn_column_blocks(a)), dim3(GN_THREADS), 0, s, a, gn_column_blocks(a)),
              "mm_group_norm_backward columns launch");
    return MM_OK;
  }
  a.part = (float*)workspace;
  a.sums = a.part + 2 * a.segs_n * channels;
  MM_CUDA(GN_BY_VEC(gn_walk_backward, a, s), "mm_group_norm_backward launch");
  return MM_OK;
}
