// The norm of many tensors together, and clipping by it.
//
//   norm = (sum over all tensors and elements of |g|^p)^(1/p), p = 1, 2 or infinity
//   coef = min(1, max_norm / (norm + 1e-6)),  g = g coef
//
// The table of tensors travels as the kernel's parameter, so nothing is uploaded
// and a captured launch keeps its table.  All elements, cut into chunks, are
// divided evenly over a grid that fills the GPU; each block walks its range and
// leaves one partial result, and whoever needs the norm joins the partial results
// in a fixed order (no atomics: the same inputs give the same bits).  Sums are
// held in 64 bits, so squares of large and small gradients neither overflow nor
// vanish.
//
// Bound by memory: 4 bytes per element for the norm, 12 to clip (read, then read
// and written).  The norm of 72 tensors of 101 M elements takes 64 us (6.3 TB/s), to clip
// them 204 us (5.9 TB/s), of one tensor of 200 M 117 us (6.8 TB/s).
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <memory>
#include <new>
#include <string>

#include "mm_common.cuh"

namespace mm {

constexpr int GR_THREADS = 256;
constexpr int GR_CHUNK = 4096;      // elements
constexpr int GR_EACH = 8, GR_SCALE = 4;  // float4 loads in flight per thread: for the norm, to scale
// Tensors of a launch.  Its parameters may hold up to 32,764 bytes, and the driver copies
// them (72 tensors in a table of 1000: 2 us more per launch than in one of 128).
constexpr int GR_FEW = 16, GR_SOME = 128, GR_MANY = 1000;

struct GrTensor {
  float* p;
  int64_t n;
  uint32_t first;  // first chunk
};

template <int MOST>
struct GrTable {
  GrTensor t[MOST];
  int count;
  uint32_t chunks;
};

template <int ORDER>
__device__ __forceinline__ void gr_add(double& s, float v) {
  if (ORDER == MM_NORM_2) {
    const double d = (double)v;
    s = fma(d, d, s);
  } else if (ORDER == MM_NORM_1) {
    s += (double)fabsf(v);
  } else {
    // by the bits: those of NaN are above all others
    s = __longlong_as_double(max(__double_as_longlong(s), (long long)(__float_as_uint(v) & 0x7fffffffu)));
  }
}

template <int ORDER>
__device__ __forceinline__ double gr_join(double a, double b) {
  if (ORDER != MM_NORM_INF) return a + b;
  return __longlong_as_double(max(__double_as_longlong(a), __double_as_longlong(b)));
}

// The block's result; every thread gets it.
template <int ORDER, int T>
__device__ __forceinline__ double gr_block(double s, double* sm) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s = gr_join<ORDER>(s, __shfl_xor_sync(0xffffffffu, s, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = s;
  __syncthreads();
  s = sm[0];
#pragma unroll
  for (int i = 1; i < T / 32; ++i) s = gr_join<ORDER>(s, sm[i]);
  return s;
}

// Calls f(p, n) for each tensor's part of the block's range of chunks, the last
// part first where `back`.
template <int MOST, class F>
__device__ __forceinline__ void gr_walk(const GrTable<MOST>& tab, bool back, F f) {
  const uint32_t from = (uint32_t)((uint64_t)tab.chunks * blockIdx.x / gridDim.x);
  const uint32_t to = (uint32_t)((uint64_t)tab.chunks * (blockIdx.x + 1) / gridDim.x);
  if (from == to) return;
  const uint32_t start = back ? to - 1 : from;
  int lo = 0, hi = tab.count - 1;  // the last tensor whose first chunk is not behind `start`
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (tab.t[mid].first <= start) lo = mid;
    else hi = mid - 1;
  }
  for (int k = lo; k >= 0 && k < tab.count; k += back ? -1 : 1) {
    const GrTensor& t = tab.t[k];
    const int64_t begin = (int64_t)(max(from, t.first) - t.first) * GR_CHUNK;
    const int64_t end = min(t.n, (int64_t)(max(to, t.first) - t.first) * GR_CHUNK);
    if (begin < end) f(t.p + begin, end - begin);
    if (back ? t.first <= from : t.first >= to) break;
  }
}

// The part's elements in front of the first 16-byte boundary, and the vectors behind it.
struct GrPart {
  int64_t head, n4, tail;  // tail: where the rest begins
  __device__ __forceinline__ GrPart(const float* p, int64_t n) {
    head = min(n, (int64_t)((4 - ((uintptr_t)p >> 2 & 3)) & 3));
    n4 = (n - head) / 4;
    tail = head + 4 * n4;
  }
};

template <int ORDER, int MOST>
__global__ void __launch_bounds__(GR_THREADS) grad_norm_kernel(const __grid_constant__ GrTable<MOST> tab, double* part) {
  __shared__ double sm[GR_THREADS / 32];
  double s = 0.0;
  gr_walk(tab, false, [&](const float* p, int64_t n) {
    const GrPart at(p, n);
    const float4* p4 = reinterpret_cast<const float4*>(p + at.head);
    int64_t i = threadIdx.x;
    auto take = [&](const float4& v) {
      gr_add<ORDER>(s, v.x);
      gr_add<ORDER>(s, v.y);
      gr_add<ORDER>(s, v.z);
      gr_add<ORDER>(s, v.w);
    };
    for (; i + (GR_EACH - 1) * GR_THREADS < at.n4; i += GR_EACH * GR_THREADS) {
      float4 v[GR_EACH];
#pragma unroll
      for (int e = 0; e < GR_EACH; ++e) v[e] = p4[i + e * GR_THREADS];
#pragma unroll
      for (int e = 0; e < GR_EACH; ++e) take(v[e]);
    }
    for (; i < at.n4; i += GR_THREADS) take(p4[i]);
    if (threadIdx.x < at.head) gr_add<ORDER>(s, p[threadIdx.x]);
    if (threadIdx.x < n - at.tail) gr_add<ORDER>(s, p[at.tail + threadIdx.x]);
  });
  s = gr_block<ORDER, GR_THREADS>(s, sm);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

// The norm of `count` partial results; every thread of the block of T gets it.
template <int ORDER, int T>
__device__ __forceinline__ float gr_total(const double* part, int count, double* sm) {
  double s = 0.0;
  for (int i = threadIdx.x; i < count; i += T) s = gr_join<ORDER>(s, part[i]);
  s = gr_block<ORDER, T>(s, sm);
  if (ORDER == MM_NORM_2) return (float)sqrt(s);
  if (ORDER == MM_NORM_1) return (float)s;
  return __uint_as_float((uint32_t)__double_as_longlong(s));
}

// NaN stays NaN.
__device__ __forceinline__ float gr_coef(float norm, float max_norm) {
  const float c = __fdiv_rn(max_norm, __fadd_rn(norm, 1e-6f));
  return c >= 1.f ? 1.f : c;
}

template <int ORDER>
__global__ void __launch_bounds__(GR_THREADS) grad_total_kernel(const double* part, int count, float max_norm,
                                                                float* norm, float* coef) {
  __shared__ double sm[GR_THREADS / 32];
  pdl_wait();
  const float total = gr_total<ORDER, GR_THREADS>(part, count, sm);
  if (threadIdx.x == 0) {
    *norm = total;
    if (coef) *coef = gr_coef(total, max_norm);
  }
}

template <int ORDER, int MOST>
__global__ void __launch_bounds__(GR_THREADS) grad_scale_kernel(const __grid_constant__ GrTable<MOST> tab,
                                                                const double* part, int count, float max_norm,
                                                                float* norm) {
  __shared__ double sm[GR_THREADS / 32];
  pdl_wait();
  const float total = gr_total<ORDER, GR_THREADS>(part, count, sm), c = gr_coef(total, max_norm);
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = total;
  if (c == 1.f) return;  // every value stays what it is
  // (from the end, which the norm's pass read last: what L2 still holds of it comes from there)
  gr_walk(tab, true, [&](float* p, int64_t n) {
    const GrPart at(p, n);
    float4* p4 = reinterpret_cast<float4*>(p + at.head);
    int64_t left = at.n4;
    for (; left >= GR_SCALE * GR_THREADS; left -= GR_SCALE * GR_THREADS) {
      float4 v[GR_SCALE];
      float4* q = p4 + left - GR_SCALE * GR_THREADS + threadIdx.x;
#pragma unroll
      for (int e = 0; e < GR_SCALE; ++e) v[e] = q[e * GR_THREADS];
#pragma unroll
      for (int e = 0; e < GR_SCALE; ++e) q[e * GR_THREADS] = make_float4(v[e].x * c, v[e].y * c, v[e].z * c, v[e].w * c);
    }
    for (int64_t i = threadIdx.x; i < left; i += GR_THREADS) {
      const float4 v = p4[i];
      p4[i] = make_float4(v.x * c, v.y * c, v.z * c, v.w * c);
    }
    if (threadIdx.x < at.head) p[threadIdx.x] *= c;
    if (threadIdx.x < n - at.tail) p[at.tail + threadIdx.x] *= c;
  });
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------

constexpr int GR_BLOCKS_PER_SM = 4;

static int gr_blocks(uint32_t chunks) {
  const int64_t most = (int64_t)sm_count() * GR_BLOCKS_PER_SM;
  return (int)(chunks < 1 ? 1 : chunks < most ? chunks : most);
}

// Partial results that `count` tensors may leave.
static int64_t gr_partials(int count) {
  return (int64_t)((count + GR_MANY - 1) / GR_MANY) * sm_count() * GR_BLOCKS_PER_SM;
}

template <int MOST>
static int gr_fill(const mm_grad_t* in, int count, GrTable<MOST>* tab) {
  int64_t chunks = 0;
  for (int i = 0; i < count; ++i) {
    tab->t[i] = {in[i].data, in[i].numel, (uint32_t)chunks};
    chunks += (in[i].numel + GR_CHUNK - 1) / GR_CHUNK;
    if (chunks > INT32_MAX) return fail(MM_ERR_UNSUPPORTED, "mm_grad_norm: too many elements in one call");
  }
  tab->count = count;
  tab->chunks = (uint32_t)chunks;
  return MM_OK;
}

template <int ORDER, int MOST>
static int gr_norm_part(const mm_grad_t* in, int count, double* part, int* blocks, cudaStream_t s) {
  GrTable<MOST> tab;
  if (const int rc = gr_fill<MOST>(in, count, &tab)) return rc;
  *blocks = gr_blocks(tab.chunks);
  grad_norm_kernel<ORDER, MOST><<<*blocks, GR_THREADS, 0, s>>>(tab, part);
  MM_LAUNCH_CHECK("mm_grad_norm launch");
  return MM_OK;
}

template <int ORDER, int MOST>
static int gr_scale_part(const mm_grad_t* in, int count, const double* part, int parts, float max_norm, float* norm,
                         cudaStream_t s) {
  GrTable<MOST> tab;
  if (const int rc = gr_fill<MOST>(in, count, &tab)) return rc;
  MM_CUDA(launch_pdl(grad_scale_kernel<ORDER, MOST>, dim3(gr_blocks(tab.chunks)), dim3(GR_THREADS), 0, s, tab, part,
                     parts, max_norm, norm),
          "mm_grad_clip launch");
  return MM_OK;
}

template <int ORDER>
static int gr_norm(const mm_grad_t* in, int count, double* part, int* parts, cudaStream_t s) {
  *parts = 0;
  for (int at = 0; at < count || at == 0; at += GR_MANY) {
    const int n = count - at < GR_MANY ? count - at : GR_MANY;
    int blocks = 0;
    const auto launch = n <= GR_FEW    ? gr_norm_part<ORDER, GR_FEW>
                        : n <= GR_SOME ? gr_norm_part<ORDER, GR_SOME>
                                       : gr_norm_part<ORDER, GR_MANY>;
    if (const int rc = launch(in + at, n, part + *parts, &blocks, s)) return rc;
    *parts += blocks;
  }
  return MM_OK;
}

template <int ORDER>
static int gr_run(const mm_grad_t* in, int count, bool clip, float max_norm, float* norm, float* coef, double* part,
                  cudaStream_t s) {
  int parts = 0;
  if (const int rc = gr_norm<ORDER>(in, count, part, &parts, s)) return rc;
  if (!clip) {
    MM_CUDA(launch_pdl(grad_total_kernel<ORDER>, dim3(1), dim3(GR_THREADS), 0, s, (const double*)part, (int)parts,
                       max_norm, norm, coef),
            "mm_grad_norm launch");
    return MM_OK;
  }
  for (int at = 0; at < count || at == 0; at += GR_MANY) {
    const int n = count - at < GR_MANY ? count - at : GR_MANY;
    const auto launch = n <= GR_FEW    ? gr_scale_part<ORDER, GR_FEW>
                        : n <= GR_SOME ? gr_scale_part<ORDER, GR_SOME>
                                       : gr_scale_part<ORDER, GR_MANY>;
    if (const int rc = launch(in + at, n, part, parts, max_norm, at == 0 ? norm : nullptr, s)) return rc;
  }
  return MM_OK;
}

// Whether two of the arrays that are scaled overlap (the threads of both would race).
static int gr_check_apart(const mm_grad_t* in, int count) {
  struct Span {
    uintptr_t from, to;
  };
  std::unique_ptr<Span[]> spans(new (std::nothrow) Span[count > 0 ? count : 1]);
  if (!spans) return fail(MM_ERR_OOM, "mm_grad_clip: out of host memory");
  int n = 0;
  for (int i = 0; i < count; ++i)
    if (in[i].numel > 0) spans[n++] = {(uintptr_t)in[i].data, (uintptr_t)in[i].data + 4 * (uintptr_t)in[i].numel};
  std::sort(spans.get(), spans.get() + n, [](const Span& a, const Span& b) { return a.from < b.from; });
  for (int i = 1; i < n; ++i)
    if (spans[i].from < spans[i - 1].to)
      return fail(MM_ERR_INVALID, "mm_grad_clip: a tensor is given twice or shares memory with another");
  return MM_OK;
}

static int gr_call(const char* who, const mm_grad_t* in, int count, int order, bool clip, double max_norm, float* norm,
                   float* coef, void* workspace, size_t bytes, void* stream) {
  const std::string name(who);
  if (count < 0 || (count > 0 && in == nullptr)) return fail(MM_ERR_INVALID, name + ": invalid tensor list");
  if (order != MM_NORM_INF && order != MM_NORM_1 && order != MM_NORM_2)
    return fail(MM_ERR_UNSUPPORTED, name + ": the norm's order must be 1, 2 or infinity");
  if (!(max_norm >= 0)) return fail(MM_ERR_INVALID, name + ": max_norm must be non-negative");
  if (norm == nullptr) return fail(MM_ERR_INVALID, name + ": null result");
  for (int i = 0; i < count; ++i)
    if (in[i].numel < 0 || in[i].numel > INT64_MAX / 8 || (in[i].numel > 0 && !in[i].data) ||
        (uintptr_t)in[i].data % 4 != 0)
      return fail(MM_ERR_INVALID, name + ": invalid tensor " + std::to_string(i));
  if (clip)
    if (const int rc = gr_check_apart(in, count)) return rc;
  const size_t need = (size_t)gr_partials(count > 0 ? count : 1) * sizeof(double);
  if (workspace != nullptr && (bytes < need || (uintptr_t)workspace % 8 != 0))
    return fail(MM_ERR_INVALID, name + ": the workspace is misaligned or too small");
  cudaStream_t s = resolve_stream(stream);
  Scratch scratch;
  if (workspace == nullptr) {
    if (const int rc = scratch.get(need, s)) return rc;
    workspace = scratch.data;
  }
  const auto run = order == MM_NORM_INF ? gr_run<MM_NORM_INF> : order == MM_NORM_1 ? gr_run<MM_NORM_1> : gr_run<MM_NORM_2>;
  return run(in, count, clip, (float)max_norm, norm, coef, (double*)workspace, s);
}

}  // namespace mm

using namespace mm;

extern "C" int mm_grad_norm_workspace_size(int count, size_t* bytes) {
  if (bytes == nullptr || count < 0) return fail(MM_ERR_INVALID, "mm_grad_norm_workspace_size: invalid argument");
  *bytes = (size_t)gr_partials(count > 0 ? count : 1) * sizeof(double);
  return MM_OK;
}

extern "C" int mm_grad_norm(const mm_grad_t* grads, int count, int order, double max_norm, float* norm, float* coef,
                            void* workspace, size_t workspace_bytes, void* stream) {
  return gr_call("mm_grad_norm", grads, count, order, false, max_norm, norm, coef, workspace, workspace_bytes, stream);
}

extern "C" int mm_grad_clip(const mm_grad_t* grads, int count, int order, double max_norm, float* norm,
                            void* workspace, size_t workspace_bytes, void* stream) {
  return gr_call("mm_grad_clip", grads, count, order, true, max_norm, norm, nullptr, workspace, workspace_bytes,
                 stream);
}
