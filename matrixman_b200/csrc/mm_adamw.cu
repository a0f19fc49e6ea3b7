// AdamW (and Adam) over many tensors at once, with states in 32 or in 8 bits.
//
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// One launch walks every tensor: the table of pointers travels as the kernel's
// parameter, so nothing is uploaded and a captured launch keeps its table.  A
// block of threads looks its tensor up by binary search over the tensors'
// first chunks.  The pass is bound by memory: 28 bytes per element with 32-bit
// states (p, g, m, v in; p, m, v out), 16 with 8-bit ones.
//
// 8-bit states.  256 consecutive elements share one float32 scale, the largest
// magnitude among them.  m is a sign and a 7-bit code, sqrt(v) an 8-bit code:
// the share of the scale, rounded to the nearest of 8 (16) steps per power of
// two over 16 powers of two (so to 1/16 (1/32) relative), i.e. a float32's
// exponent and its upper 3 (4) mantissa bits counted down from 1.0.  Code 0 is
// zero.  sqrt(v) is stored instead of v because it is what the update divides
// by, and a non-zero sqrt(v) takes at least code 1: were it rounded to zero
// while m is not, the next update would divide by eps.  All arithmetic before
// the rounding is float32 with every operation rounded (no contraction), so a
// plain restatement gives the same codes.
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <memory>
#include <new>
#include <string>

#include "mm_common.cuh"

namespace mm {

constexpr int AW_BLOCK = 256;     // elements that share a scale
constexpr int AW_THREADS = 256;
// Elements per thread block.  With 32-bit states twice as many left too few
// blocks for small models (an MLP of 0.5 M parameters: 9.4 us, these 5.9).  With
// 8-bit states each warp has one block of 256 and leaves (two per warp: 227 us
// for 54 M elements, one 178).
constexpr int AW_CHUNK = 2048, AW_CHUNK8 = AW_BLOCK * AW_THREADS / 32;
constexpr int AW_ONE = 0x3F800000;  // 1.0f

struct AwTensor {
  float* p;
  const float* g;
  void *m, *v;
  float *ms, *vs;
  uint32_t first;   // first chunk; the end of the table's last tensor is AwTable::chunks
  uint32_t aligned; // p, g (and 32-bit m, v) are 16-byte aligned
  int64_t n;
};

// Kernel parameters may hold up to 32,764 bytes.
template <int MOST>
struct AwTable {
  AwTensor t[MOST];
  int count;
};

// The driver copies a launch's parameters, so few tensors have a small table and
// the first kernel one of the steps alone.
constexpr int AW_FEW = 16, AW_MANY = 400;

template <int MOST>
struct AwSteps {
  float* step[MOST];
  int count;
};

struct AwScalars {
  float b1, omb1, b2, omb2, eps, decay, l2;  // decay = 1 - lr wd (decoupled); l2 = wd (coupled) or 0
  int maximize;
};

// A step's own factors of each tensor: lr / (1 - b1^t) and 1 / sqrt(1 - b2^t).
template <int MOST>
__global__ void adamw_begin_kernel(const __grid_constant__ AwSteps<MOST> tab, float2* coef, double lr, double b1,
                                   double b2, int advance) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= tab.count) return;
  float t = *tab.step[i];
  if (advance) {
    t += 1.f;
    *tab.step[i] = t;
  }
  coef[i] = make_float2((float)(lr / (1.0 - pow(b1, (double)t))), (float)(1.0 / sqrt(1.0 - pow(b2, (double)t))));
}

// Magnitude code of q = size / scale <= 1: float32 bits above SHIFT, rounded to
// even, counted down from TOP at 1.0.  Only the lowest byte counts (q is NaN in
// a block whose scale is).
template <int SHIFT, int TOP>
__device__ __forceinline__ int aw_code(float size, float inv, int least) {
  const uint32_t bits = __float_as_uint(__fmul_rn(size, inv));
  return max((int)((bits + ((1u << (SHIFT - 1)) - 1u) + ((bits >> SHIFT) & 1u)) >> SHIFT) - ((AW_ONE >> SHIFT) - TOP),
             least);
}

template <int SHIFT, int TOP>
__device__ __forceinline__ float aw_value(uint32_t code, float scale) {
  const float q = code ? __uint_as_float((code + (uint32_t)(AW_ONE >> SHIFT) - TOP) << SHIFT) : 0.f;
  return __fmul_rn(q, scale);
}

__device__ __forceinline__ float aw_decode_m(uint32_t byte, float scale) {
  const float v = aw_value<20, 127>(byte & 127u, scale);
  return byte & 128u ? -v : v;
}

__device__ __forceinline__ float aw_decode_r(uint32_t byte, float scale) { return aw_value<19, 255>(byte, scale); }

// Scale of a warp's largest magnitudes, by their bits: those of infinities and
// NaNs are above all others, and make it NaN, so they stay visible.
__device__ __forceinline__ float aw_scale(float most) {
  const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(most) & 0x7fffffffu);
  return __uint_as_float(bits < 0x00800000u ? 0u : bits >= 0x7f800000u ? 0x7fc00000u : bits);
}

__device__ __forceinline__ float aw_max(float a, float b) {
  return __uint_as_float(max(__float_as_uint(a) & 0x7fffffffu, __float_as_uint(b) & 0x7fffffffu));
}

__device__ __forceinline__ float aw_moments(float& m, float vold, float g, const AwScalars& a) {
  m = __fadd_rn(__fmul_rn(m, a.b1), __fmul_rn(g, a.omb1));
  return __fadd_rn(__fmul_rn(vold, a.b2), __fmul_rn(__fmul_rn(g, g), a.omb2));
}

__device__ __forceinline__ float aw_update(float p, float m, float r, float2 coef, const AwScalars& a) {
  const float d = __fadd_rn(__fmul_rn(r, coef.y), a.eps);
  return __fsub_rn(__fmul_rn(p, a.decay), __fmul_rn(__fdiv_rn(m, d), coef.x));
}

// The gradients of N elements: negated to maximise, with coupled weight decay.
template <int N>
__device__ __forceinline__ void aw_grads(float* g, const float* p, const AwScalars& a) {
  if (a.maximize) {
#pragma unroll
    for (int e = 0; e < N; ++e) g[e] = -g[e];
  }
  if (a.l2 != 0.f) {
#pragma unroll
    for (int e = 0; e < N; ++e) g[e] = __fadd_rn(g[e], __fmul_rn(p[e], a.l2));
  }
}

// The tensor that chunk `chunk` belongs to.
template <int MOST>
__device__ __forceinline__ int aw_find(const AwTable<MOST>& tab, uint32_t chunk) {
  int lo = 0, hi = tab.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (tab.t[mid].first <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

template <int MOST>
__global__ void __launch_bounds__(AW_THREADS) adamw32_kernel(const __grid_constant__ AwTable<MOST> tab,
                                                             const float2* __restrict__ coefs, AwScalars a) {
  const int k = aw_find(tab, blockIdx.x);
  const AwTensor& t = tab.t[k];
  const float2 coef = coefs[k];
  const int64_t base = (int64_t)(blockIdx.x - t.first) * AW_CHUNK;
  float* p = t.p + base;
  const float* g = t.g + base;
  float* m = (float*)t.m + base;
  float* v = (float*)t.v + base;
  const int left = (int)min((int64_t)AW_CHUNK, t.n - base);
  if (t.aligned && left == AW_CHUNK) {
#pragma unroll
    for (int i = 0; i < AW_CHUNK / (4 * AW_THREADS); ++i) {
      const int c = i * AW_THREADS + threadIdx.x;
      float4 p4 = reinterpret_cast<const float4*>(p)[c], g4 = reinterpret_cast<const float4*>(g)[c];
      float4 m4 = reinterpret_cast<const float4*>(m)[c], v4 = reinterpret_cast<const float4*>(v)[c];
      float *pe = &p4.x, *ge = &g4.x, *me = &m4.x, *ve = &v4.x;
      aw_grads<4>(ge, pe, a);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        ve[e] = aw_moments(me[e], ve[e], ge[e], a);
        pe[e] = aw_update(pe[e], me[e], __fsqrt_rn(ve[e]), coef, a);
      }
      reinterpret_cast<float4*>(p)[c] = p4;
      reinterpret_cast<float4*>(m)[c] = m4;
      reinterpret_cast<float4*>(v)[c] = v4;
    }
    return;
  }
  for (int c = threadIdx.x; c < left; c += AW_THREADS) {
    float me = m[c], ge = g[c];
    const float pe = p[c];
    aw_grads<1>(&ge, &pe, a);
    const float ve = aw_moments(me, v[c], ge, a);
    p[c] = aw_update(pe, me, __fsqrt_rn(ve), coef, a);
    m[c] = me;
    v[c] = ve;
  }
}

// Eight consecutive floats at p + c, of which `left` exist from p on (zeros
// behind them).
__device__ __forceinline__ void aw_load8(const float* p, int c, int left, bool vec, float* out) {
  if (vec && c + 8 <= left) {
    const float4 a = *reinterpret_cast<const float4*>(p + c), b = *reinterpret_cast<const float4*>(p + c + 4);
    out[0] = a.x; out[1] = a.y; out[2] = a.z; out[3] = a.w;
    out[4] = b.x; out[5] = b.y; out[6] = b.z; out[7] = b.w;
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) out[e] = c + e < left ? p[c + e] : 0.f;
}

__device__ __forceinline__ void aw_store8(float* p, int c, int left, bool vec, const float* v) {
  if (vec && c + 8 <= left) {
    *reinterpret_cast<float4*>(p + c) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(p + c + 4) = make_float4(v[4], v[5], v[6], v[7]);
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (c + e < left) p[c + e] = v[e];
}

// Codes of eight consecutive elements, the lowest element in the lowest byte.
// The code arrays hold whole blocks (mm_adamw_state_bytes), so no code of a
// block's tail is out of range.
__device__ __forceinline__ void aw_unpack(uint2 c, uint32_t* out) {
#pragma unroll
  for (int e = 0; e < 8; ++e) out[e] = ((e < 4 ? c.x : c.y) >> (8 * (e & 3))) & 255u;
}

// The lowest bytes of eight words.
__device__ __forceinline__ uint2 aw_pack(const uint32_t* c) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    w[i] = __byte_perm(__byte_perm(c[4 * i], c[4 * i + 1], 0x0040), __byte_perm(c[4 * i + 2], c[4 * i + 3], 0x0040),
                       0x5410);
  return make_uint2(w[0], w[1]);
}

// Codes and scales of one block of 256 elements held by a warp, 8 per lane.
__device__ __forceinline__ void aw_encode_block(const float* m, const float* r, uint8_t* mc, uint8_t* vc, float* ms,
                                                float* vs, int64_t block, int lane) {
  float mm = 0.f, rr = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    mm = aw_max(mm, m[e]);
    rr = aw_max(rr, r[e]);
  }
  mm = aw_scale(mm);
  rr = aw_scale(rr);
  const float im = mm == 0.f ? 0.f : __frcp_rn(mm), ir = rr == 0.f ? 0.f : __frcp_rn(rr);
  uint32_t cm[8], cr[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    cm[e] = (uint32_t)aw_code<20, 127>(fabsf(m[e]), im, 0) | ((__float_as_uint(m[e]) >> 24) & 128u);
    cr[e] = (uint32_t)aw_code<19, 255>(r[e], ir, r[e] > 0.f ? 1 : 0);
  }
  reinterpret_cast<uint2*>(mc)[block * 32 + lane] = aw_pack(cm);
  reinterpret_cast<uint2*>(vc)[block * 32 + lane] = aw_pack(cr);
  if (lane == 0) {
    ms[block] = mm;
    vs[block] = rr;
  }
}

template <int MOST>
__global__ void __launch_bounds__(AW_THREADS) adamw8_kernel(const __grid_constant__ AwTable<MOST> tab,
                                                            const float2* __restrict__ coefs, AwScalars a) {
  const int k = aw_find(tab, blockIdx.x);
  const AwTensor& t = tab.t[k];
  const float2 coef = coefs[k];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool vec = t.aligned != 0;
  const int64_t base = (int64_t)(blockIdx.x - t.first) * AW_CHUNK8 + warp * AW_BLOCK;
  if (base >= t.n) return;
  const int64_t block = base / AW_BLOCK;
  const int left = (int)min((int64_t)AW_BLOCK, t.n - base);
  float p[8], g[8], m[8], r[8];
  aw_load8(t.p + base, lane * 8, left, vec, p);
  aw_load8(t.g + base, lane * 8, left, vec, g);
  uint32_t cm[8], cr[8];
  aw_unpack(reinterpret_cast<const uint2*>(t.m)[block * 32 + lane], cm);
  aw_unpack(reinterpret_cast<const uint2*>(t.v)[block * 32 + lane], cr);
  const float ms = t.ms[block], vs = t.vs[block];
  aw_grads<8>(g, p, a);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    m[e] = aw_decode_m(cm[e], ms);
    const float rold = aw_decode_r(cr[e], vs);
    r[e] = __fsqrt_rn(aw_moments(m[e], __fmul_rn(rold, rold), g[e], a));
    p[e] = aw_update(p[e], m[e], r[e], coef, a);
  }
  if (left < AW_BLOCK) {  // nothing behind the tensor's end counts for the scale
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (lane * 8 + e >= left) m[e] = r[e] = 0.f;
  }
  aw_store8(t.p + base, lane * 8, left, vec, p);
  aw_encode_block(m, r, (uint8_t*)t.m, (uint8_t*)t.v, t.ms, t.vs, block, lane);
}

// 8-bit states of given float32 moments: one warp per block of 256 elements.
__global__ void __launch_bounds__(AW_THREADS) adamw_encode_kernel(const float* m, const float* v, int64_t n,
                                                                  uint8_t* mc, float* ms, uint8_t* vc, float* vs) {
  const int lane = threadIdx.x & 31;
  const int64_t block = (int64_t)blockIdx.x * (AW_THREADS / 32) + (threadIdx.x >> 5);
  const int64_t base = block * AW_BLOCK;
  if (base >= n) return;
  const int left = (int)min((int64_t)AW_BLOCK, n - base);
  float me[8], re[8];
  aw_load8(m + base, lane * 8, left, false, me);
  aw_load8(v + base, lane * 8, left, false, re);
#pragma unroll
  for (int e = 0; e < 8; ++e) re[e] = __fsqrt_rn(re[e]);
  aw_encode_block(me, re, mc, vc, ms, vs, block, lane);
}

// The float32 values that 8-bit states stand for (v is the square of its root).
__global__ void __launch_bounds__(AW_THREADS) adamw_decode_kernel(const uint8_t* mc, const float* ms,
                                                                  const uint8_t* vc, const float* vs, int64_t n,
                                                                  float* m, float* v, int vec) {
  const int lane = threadIdx.x & 31;
  const int64_t block = (int64_t)blockIdx.x * (AW_THREADS / 32) + (threadIdx.x >> 5);
  const int64_t base = block * AW_BLOCK;
  if (base >= n) return;
  const int left = (int)min((int64_t)AW_BLOCK, n - base);
  uint32_t cm[8], cr[8];
  aw_unpack(reinterpret_cast<const uint2*>(mc)[block * 32 + lane], cm);
  aw_unpack(reinterpret_cast<const uint2*>(vc)[block * 32 + lane], cr);
  float me[8], ve[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    me[e] = aw_decode_m(cm[e], ms[block]);
    const float r = aw_decode_r(cr[e], vs[block]);
    ve[e] = __fmul_rn(r, r);
  }
  aw_store8(m + base, lane * 8, left, vec != 0, me);
  aw_store8(v + base, lane * 8, left, vec != 0, ve);
}

static bool aw_aligned(const void* p, uintptr_t to) { return (uintptr_t)p % to == 0; }

template <int MOST>
static int aw_launch(const mm_adamw_tensor_t* in, int count, int bits, double lr, double b1, double b2, int advance,
                     const AwScalars& a, float2* coef, cudaStream_t s) {
  AwTable<MOST> tab;
  AwSteps<MOST> steps;
  int64_t chunks = 0;
  for (int i = 0; i < count; ++i) {
    AwTensor& t = tab.t[i];
    t = {in[i].param, in[i].grad, in[i].exp_avg, in[i].exp_avg_sq, in[i].exp_avg_scale, in[i].exp_avg_sq_scale,
         (uint32_t)chunks, 0, in[i].numel};
    steps.step[i] = in[i].step;
    t.aligned = aw_aligned(t.p, 16) && aw_aligned(t.g, 16) &&
                (bits == 8 || (aw_aligned(t.m, 16) && aw_aligned(t.v, 16)));
    chunks += bits == 8 ? (t.n + AW_CHUNK8 - 1) / AW_CHUNK8 : (t.n + AW_CHUNK - 1) / AW_CHUNK;
  }
  if (chunks > INT32_MAX) return fail(MM_ERR_UNSUPPORTED, "mm_adamw: too many elements in one call");
  tab.count = steps.count = count;
  adamw_begin_kernel<MOST><<<(count + 127) / 128, 128, 0, s>>>(steps, coef, lr, b1, b2, advance);
  MM_LAUNCH_CHECK("mm_adamw launch");
  if (chunks == 0) return MM_OK;  // every tensor is empty: only the steps move
  if (bits == 32)
    adamw32_kernel<MOST><<<(unsigned)chunks, AW_THREADS, 0, s>>>(tab, coef, a);
  else
    adamw8_kernel<MOST><<<(unsigned)chunks, AW_THREADS, 0, s>>>(tab, coef, a);
  MM_LAUNCH_CHECK("mm_adamw launch");
  return MM_OK;
}

static int aw_check_state(const void* mc, const float* ms, const void* vc, const float* vs, const char* who) {
  if (!mc || !ms || !vc || !vs) return fail(MM_ERR_INVALID, std::string(who) + ": null state");
  if (!aw_aligned(mc, 8) || !aw_aligned(vc, 8))
    return fail(MM_ERR_INVALID, std::string(who) + ": 8-bit states must be 8-byte aligned");
  return MM_OK;
}

// Whether two of the arrays that a step writes start at one address (whole
// tensors given twice; the threads of both would race).  A set of addresses in
// a table of twice their number, 1 us for 72 tensors.
static int aw_check_distinct(const mm_adamw_tensor_t* in, int count, int bits, int advance) {
  size_t size = 16;
  while (size < (size_t)count * 12) size *= 2;
  std::unique_ptr<const void*[]> seen(new (std::nothrow) const void*[size]());
  if (!seen) return fail(MM_ERR_OOM, "mm_adamw: out of host memory");
  for (int i = 0; i < count; ++i) {
    const mm_adamw_tensor_t& t = in[i];
    const bool any = t.numel > 0;
    const void* written[] = {advance ? t.step : nullptr,
                             any ? t.param : nullptr,
                             any ? t.exp_avg : nullptr,
                             any ? t.exp_avg_sq : nullptr,
                             any && bits == 8 ? t.exp_avg_scale : nullptr,
                             any && bits == 8 ? t.exp_avg_sq_scale : nullptr};
    for (const void* p : written) {
      if (p == nullptr) continue;
      size_t at = ((uintptr_t)p >> 2) * 0x9E3779B97F4A7C15ull >> 32 & (size - 1);
      for (; seen[at] != nullptr; at = (at + 1) & (size - 1))
        if (seen[at] == p)
          return fail(MM_ERR_INVALID, "mm_adamw: tensor " + std::to_string(i) +
                                          " shares its parameter, a state or its step with another or with itself");
      seen[at] = p;
    }
  }
  return MM_OK;
}

}  // namespace mm

using namespace mm;

extern "C" int mm_adamw_workspace_size(int count, size_t* bytes) {
  if (bytes == nullptr || count < 0) return fail(MM_ERR_INVALID, "mm_adamw_workspace_size: invalid argument");
  *bytes = (size_t)count * sizeof(float2);
  return MM_OK;
}

extern "C" int mm_adamw(const mm_adamw_tensor_t* tensors, int count, int state_bits, double lr, double beta1,
                        double beta2, double eps, double weight_decay, int decoupled, int maximize, int advance,
                        void* workspace, size_t workspace_bytes, void* stream) {
  if (count < 0 || (count > 0 && tensors == nullptr)) return fail(MM_ERR_INVALID, "mm_adamw: invalid tensor list");
  if (state_bits != 32 && state_bits != 8) return fail(MM_ERR_UNSUPPORTED, "mm_adamw: states are held in 32 or 8 bits");
  if (!(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1))
    return fail(MM_ERR_INVALID, "mm_adamw: betas must lie in [0, 1)");
  for (int i = 0; i < count; ++i) {
    const mm_adamw_tensor_t& t = tensors[i];
    if (t.numel < 0 || !t.step || (t.numel > 0 && (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq)))
      return fail(MM_ERR_INVALID, "mm_adamw: invalid tensor " + std::to_string(i));
    if (state_bits == 8 && t.numel > 0) {
      int rc = aw_check_state(t.exp_avg, t.exp_avg_scale, t.exp_avg_sq, t.exp_avg_sq_scale, "mm_adamw");
      if (rc != MM_OK) return rc;
    }
  }
  if (count == 0) return MM_OK;
  if (const int rc = aw_check_distinct(tensors, count, state_bits, advance)) return rc;
  if (workspace != nullptr && (workspace_bytes < (size_t)count * sizeof(float2) || !aw_aligned(workspace, 8)))
    return fail(MM_ERR_INVALID, "mm_adamw: the workspace is misaligned or too small");
  AwScalars a;
  a.b1 = (float)beta1;
  a.omb1 = (float)(1.0 - beta1);
  a.b2 = (float)beta2;
  a.omb2 = (float)(1.0 - beta2);
  a.eps = (float)eps;
  a.decay = decoupled ? (float)(1.0 - lr * weight_decay) : 1.f;
  a.l2 = decoupled ? 0.f : (float)weight_decay;
  a.maximize = maximize != 0;
  cudaStream_t s = resolve_stream(stream);
  Scratch scratch;
  if (workspace == nullptr) {
    const int rc = scratch.get((size_t)count * sizeof(float2), s);
    if (rc != MM_OK) return rc;
    workspace = scratch.data;
  }
  float2* coef = (float2*)workspace;
  for (int at = 0; at < count; at += AW_MANY) {
    const int n = count - at < AW_MANY ? count - at : AW_MANY;
    const auto launch = n <= AW_FEW ? aw_launch<AW_FEW> : aw_launch<AW_MANY>;
    const int rc = launch(tensors + at, n, state_bits, lr, beta1, beta2, advance, a, coef + at, s);
    if (rc != MM_OK) return rc;
  }
  return MM_OK;
}

extern "C" int mm_adamw_encode(const float* exp_avg, const float* exp_avg_sq, int64_t numel, uint8_t* exp_avg_code,
                               float* exp_avg_scale, uint8_t* exp_avg_sq_code, float* exp_avg_sq_scale, void* stream) {
  if (numel < 0) return fail(MM_ERR_INVALID, "mm_adamw_encode: negative size");
  if (numel == 0) return MM_OK;
  if (!exp_avg || !exp_avg_sq) return fail(MM_ERR_INVALID, "mm_adamw_encode: null moments");
  int rc = aw_check_state(exp_avg_code, exp_avg_scale, exp_avg_sq_code, exp_avg_sq_scale, "mm_adamw_encode");
  if (rc != MM_OK) return rc;
  const int64_t grid = (numel + AW_BLOCK * 8 - 1) / (AW_BLOCK * 8);
  if (grid > INT32_MAX) return fail(MM_ERR_UNSUPPORTED, "mm_adamw_encode: too many elements in one call");
  adamw_encode_kernel<<<(unsigned)grid, AW_THREADS, 0, resolve_stream(stream)>>>(
      exp_avg, exp_avg_sq, numel, exp_avg_code, exp_avg_scale, exp_avg_sq_code, exp_avg_sq_scale);
  MM_LAUNCH_CHECK("mm_adamw_encode launch");
  return MM_OK;
}

extern "C" int mm_adamw_decode(const uint8_t* exp_avg_code, const float* exp_avg_scale,
                               const uint8_t* exp_avg_sq_code, const float* exp_avg_sq_scale, int64_t numel,
                               float* exp_avg, float* exp_avg_sq, void* stream) {
  if (numel < 0) return fail(MM_ERR_INVALID, "mm_adamw_decode: negative size");
  if (numel == 0) return MM_OK;
  if (!exp_avg || !exp_avg_sq) return fail(MM_ERR_INVALID, "mm_adamw_decode: null moments");
  int rc = aw_check_state(exp_avg_code, exp_avg_scale, exp_avg_sq_code, exp_avg_sq_scale, "mm_adamw_decode");
  if (rc != MM_OK) return rc;
  const int64_t grid = (numel + AW_BLOCK * 8 - 1) / (AW_BLOCK * 8);
  if (grid > INT32_MAX) return fail(MM_ERR_UNSUPPORTED, "mm_adamw_decode: too many elements in one call");
  adamw_decode_kernel<<<(unsigned)grid, AW_THREADS, 0, resolve_stream(stream)>>>(
      exp_avg_code, exp_avg_scale, exp_avg_sq_code, exp_avg_sq_scale, numel, exp_avg, exp_avg_sq,
      aw_aligned(exp_avg, 16) && aw_aligned(exp_avg_sq, 16));
  MM_LAUNCH_CHECK("mm_adamw_decode launch");
  return MM_OK;
}
