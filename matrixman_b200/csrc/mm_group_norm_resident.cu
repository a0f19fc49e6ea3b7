// Group norm whose maps stay in shared memory between the statistics and the
// result: each map is read once.  The formulas are in mm_group_norm.cu.
//
// A unit is all pixels of a few whole groups of one image.  A cluster of up to 16
// blocks divides its pixels, each block copies its share into shared memory
// (asynchronously, so that every byte of it is in flight at once), and the blocks'
// moments or sums are joined through distributed shared memory.  Every thread
// reads only what it copied itself: columns of VEC channels (channels last) or a
// channel's pixels (first), every P-th row.
//
// A block lives for about 10 us, of which the way from its loads to its stores keeps
// its shared memory without using the memory's rate.  So that way is short: one pass
// over the values, one exchange per level (lanes, warps, blocks), and between the
// blocks of a cluster asynchronous stores that complete on a barrier in the receiver's
// shared memory (a cluster barrier with release and acquire took 0.5 us more at each
// of its two places).
//
// 64 x 64 x 80 x 80 with SiLU takes 48 us channels last (4.4 TB/s; a bare copy in the same
// pieces of 64 bytes 36), 32 x 256 x 40 x 40 27 us and backward 49 us (3.2 TB/s).
//
// Channels last, the slab of groups is wide enough that a row's piece fills whole
// sectors.
//
// Moments.  A thread sums d = x - c and d^2 with its first value as c, and has the
// mean c + sum d / n and the squared distances sum d^2 - (sum d)^2 / n.  c is one of
// the n values, so the squared distances are at least (c - mean)^2 n / (n - 1): the
// difference is no less than 1 / n of its terms and loses n (13 to 52) roundings at
// most, whatever the offset.  Threads, warps and blocks are joined the same way, with
// the first one's mean as c and the squared distances added.  A constant keeps its
// exact mean.
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "mm_group_norm.cuh"

namespace mm {

constexpr int GN_MOST_THREADS = 1024;

template <int VEC>
__device__ __forceinline__ void gn_copy(float* to, const float* from) {
  const uint32_t dst = (uint32_t)__cvta_generic_to_shared(to);
  if (VEC == 4)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(from) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(from), "n"(VEC * 4) : "memory");
}

__device__ __forceinline__ void gn_copied() { asm volatile("cp.async.wait_all;" ::: "memory"); }

__device__ __forceinline__ uint32_t gn_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t gn_cluster() {
  uint32_t r;
  asm("mov.u32 %0, %%clusterid.x;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void gn_arrive() { asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory"); }
__device__ __forceinline__ void gn_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

// The barrier that completes once `bytes` have been given to this block (by one thread).
__device__ __forceinline__ void gn_expect(uint64_t* bar, uint32_t bytes) {
  const uint32_t at = (uint32_t)__cvta_generic_to_shared(bar);
  asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(at) : "memory");
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(at), "r"(bytes) : "memory");
}

// Writes v at the place of `p` in block `rank` of the cluster, counted by its barrier.
__device__ __forceinline__ void gn_give(float2* p, uint64_t* bar, uint32_t rank, float2 v) {
  const uint32_t at = (uint32_t)__cvta_generic_to_shared(p), b = (uint32_t)__cvta_generic_to_shared(bar);
  uint32_t to, counted;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(at), "r"(rank));
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(counted) : "r"(b), "r"(rank));
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];" ::"r"(to),
               "f"(v.x), "f"(v.y), "r"(counted)
               : "memory");
}

// One try, which may sleep 1 ms.  The acquire has the cluster's scope, as the stores come from
// its other blocks.
__device__ __forceinline__ bool gn_try(uint64_t* bar) {
  const uint32_t at = (uint32_t)__cvta_generic_to_shared(bar);
  uint32_t done;
  asm volatile(
      "{ .reg .pred p; mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], 0, 1000000; selp.u32 %0, 1, 0, p; }"
      : "=r"(done)
      : "r"(at)
      : "memory");
  return done;
}

// Waits until everything was given: GN_TRIES tries (the cluster's blocks run at the same
// time), then leaves a code in the fault word and goes on.
constexpr int GN_FAULT = 111, GN_TRIES = 2000;
__device__ __forceinline__ bool gn_given(uint64_t* bar, const GnArgs& a) {
  for (int i = 0; i < a.tries; ++i)
    if (gn_try(bar)) return true;
  if (*(volatile int*)a.fault == 0) *(volatile int*)a.fault = GN_FAULT;
  return false;
}

// The end of a cluster's block: none leaves while one may give to it.  Where it gave up its
// wait, what the others have given since then is still on its way: one more try (a store of
// theirs takes a microsecond).
__device__ __forceinline__ void gn_leave_cluster(uint64_t* bar, bool given) {
  gn_wait();
  if (!given) gn_try(bar);
}

// i / d for 0 <= i < 2^20, by the float32 inverse of d: i + 0.5 is at least 0.5 / d
// away from a multiple of d, the product is off by less than i 2^-22.
__device__ __forceinline__ int gn_div(int i, float inverse) { return (int)(((float)i + 0.5f) * inverse); }

__device__ __forceinline__ int gn_block() { return (int)(blockIdx.z * gridDim.y + blockIdx.y); }

// Where a thread stands, and what its block holds.  (Blocks live for about 10 us, so
// the way to the first load counts: no integer division on it.)
template <int VEC, int PARTS, bool LAST>
struct GnPlace {
  int u, q, p, c, rows, n, step, image;         // n vectors, `step` floats apart in shared memory
  int rank, slab, kk;                           // kk: groups that the unit has
  int lead;                                     // first lane of the thread's columns and group
  int lo, hi, glo, ghi;                         // lanes of one column, and of one group's columns
  int row, r_n, j_n;                            // row and rows of partial results, columns of each
  bool writes;
  int slot;

  __device__ __forceinline__ GnPlace(const GnArgs& a, const GnPlan& k) {
    const int q_n = 1 << k.q_log, p_n = 1 << k.p_log, tu_log = k.q_log + k.p_log;
    const int t = threadIdx.x & ((1 << tu_log) - 1), lane = threadIdx.x & 31;
    u = threadIdx.x >> tu_log;
    rank = k.ranks > 1 ? (int)gn_rank() : 0;
    slab = k.ranks > 1 ? (int)gn_cluster() : (int)blockIdx.x;
    kk = min(k.slab, a.groups - slab * k.slab);
    if (LAST) {
      q = t & (q_n - 1);
      p = t >> k.q_log;
    } else {
      p = t & (p_n - 1);
      q = t >> k.p_log;
    }
    const int column = slab * k.q + q;
    c = LAST ? column * VEC : column;
    rows = max(0, min(k.rows, k.all - rank * k.rows));
    image = gn_block() * k.units + u;
    n = image < a.n && q < k.q && column < k.columns && rows > p ? (rows - p + p_n - 1) >> k.p_log : 0;
    slot = (LAST ? (u * p_n + p) * k.q + q : (u * k.q + q) * p_n + p) * VEC;
    step = ((k.units * k.q) << k.p_log) * VEC;
    // Lanes of one column: channels last those q_n apart, first neighbouring ones.
    const int tu_n = min(1 << tu_log, 32);
    if (LAST) {
      lo = q_n;
      hi = tu_n;
      glo = 1;
      ghi = k.lanes;
      r_n = q_n >= 32 ? p_n : max(1, (1 << tu_log) >> 5);
      row = q_n >= 32 ? p : t >> 5;
      writes = (lane & (tu_n - 1)) < q_n;
      j_n = q_n * PARTS;
    } else {
      lo = 1;
      hi = min(p_n, 32);
      glo = p_n;
      ghi = p_n * k.lanes;
      r_n = max(1, p_n >> 5);
      row = p >> 5;
      writes = (lane & (hi - 1)) == 0;
      j_n = q_n;
    }
    lead = lane & ~((hi > lo ? hi - lo : 0) | (PARTS == 1 && ghi > glo ? ghi - glo : 0));
  }
  // Offset of the thread's first vector in a map, and from one to the next.
  __device__ __forceinline__ int64_t offset(const GnPlan& k, int64_t images, int64_t row_step) const {
    const int64_t at = (int64_t)rank * k.rows + p;
    return image * images + (LAST ? at * row_step + c : (int64_t)c * row_step + at * VEC);
  }
  __device__ __forceinline__ int64_t next(const GnPlan& k, int64_t row_step) const {
    return LAST ? row_step << k.p_log : (int64_t)VEC << k.p_log;
  }
  // Values of one group that `rows` rows hold.
  static __device__ __forceinline__ float count(const GnArgs& a, int rows) {
    return (float)rows * (float)(LAST ? a.each : a.each * VEC);
  }
  __device__ __forceinline__ int group(const GnPlan& k, int part) const {
    return u * k.slab + min(gn_div(LAST ? q * PARTS + part : q, k.inv_each), k.slab - 1);
  }
};

template <int M>
__device__ __forceinline__ void gn_lanes(float (&v)[M], int lo, int hi) {
  for (int o = lo; o < hi; o <<= 1) {
#pragma unroll
    for (int m = 0; m < M; ++m) v[m] += __shfl_xor_sync(0xffffffffu, v[m], o);
  }
}

// Over the first `span` lanes (a power of two; the others hold 0); all of them get it.
__device__ __forceinline__ float gn_sum(float v, int span) {
  for (int o = span >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ int gn_span(int n) { return n > 16 ? 32 : n > 8 ? 16 : n > 4 ? 8 : n > 2 ? 4 : n; }

// Calls f(group of the block, its image of the block, group of the unit) for the warp's
// share of the block's groups; all lanes of a warp together.
template <int VEC, int PARTS, bool LAST, class F>
__device__ __forceinline__ void gn_groups(const GnArgs& a, const GnPlan& k, const GnPlace<VEC, PARTS, LAST>& t, F f) {
  for (int i = threadIdx.x >> 5; i < k.units * k.slab; i += blockDim.x >> 5) {
    const int u = gn_div(i, k.inv_slab), g = i - u * k.slab;
    if (g < t.kk && gn_block() * k.units + u < a.n) f(i, u, g);
  }
}

// Calls f(index) for the lane's partial results of a group.
template <int VEC, int PARTS, bool LAST, class F>
__device__ __forceinline__ void gn_partials(const GnPlan& k, const GnPlace<VEC, PARTS, LAST>& t, int u, int g, F f) {
  const int m_n = k.each / k.lanes;
  for (int i = threadIdx.x & 31; i < t.r_n * m_n; i += 32) {
    const int row = m_n == 1 ? i : i / m_n, m = i - row * m_n;
    f((u * t.r_n + row) * t.j_n + g * k.each + m * k.lanes);
  }
}

template <int VEC, int PARTS, bool LAST>
__global__ void __launch_bounds__(GN_MOST_THREADS) gn_resident_kernel(const __grid_constant__ GnArgs a,
                                                                      const __grid_constant__ GnPlan k) {
  extern __shared__ float4 gn_smem[];
  __shared__ float2 stat[GN_GROUPS];
  __shared__ uint64_t bar;
  bool given = true;
  GnPlace<VEC, PARTS, LAST> t(a, k);
  if (k.ranks > 1) {
    if (threadIdx.x == 0) gn_expect(&bar, gn_block() < k.blocks ? k.ranks * t.kk * 8 : 0);
    gn_arrive();
  }
  constexpr int PER = VEC / PARTS;  // values of a vector's part (channels last), all of which are one group's
  const int vectors = (k.rows + (1 << k.p_log) - 1) >> k.p_log;
  float* data = reinterpret_cast<float*>(gn_smem) + t.slot;
  float2* peer = reinterpret_cast<float2*>(reinterpret_cast<float*>(gn_smem) + ((vectors * t.step + 3) & ~3));
  float2* entry = peer + (k.ranks > 1 ? k.slab * GN_RANKS : 0);  // mean and squared distances ...
  float* count = reinterpret_cast<float*>(entry + k.entries);    // ... of this many values
  pdl_wait();
  {
    const float* x = a.x + t.offset(k, a.xi, a.xr);
    const int64_t next = t.next(k, a.xr);
#pragma unroll 4
    for (int i = 0; i < t.n; ++i, x += next) gn_copy<VEC>(data + i * t.step, x);
  }
  float w[VEC], b[VEC];
  int group[PARTS];
#pragma unroll
  for (int h = 0; h < PARTS; ++h) group[h] = t.group(k, h);
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    w[e] = a.w && t.n ? a.w[t.c + (LAST ? e : 0)] : 1.f;
    b[e] = a.b && t.n ? a.b[t.c + (LAST ? e : 0)] : 0.f;
  }
  const int lane = threadIdx.x & 31, r_all = t.r_n * (k.each / k.lanes);
  const float all = (float)a.pixels * (float)a.each;
  const bool direct = k.ranks == 1 && r_all == 1;  // every lane of a group has its results
  gn_copied();
  // The thread's own moments, ...
  float less[VEC];
  float m[PARTS], q[PARTS], n = (float)(t.n * PER);
  {
    float sum[VEC], squares[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) less[e] = sum[e] = squares[e] = 0.f;
    if (t.n) {
      float v[VEC];
      gn_load<VEC>(data, v);
#pragma unroll
      for (int e = 0; e < VEC; ++e) less[e] = -v[e / PER * PER];
    }
#pragma unroll 4
    for (int i = 0; i < t.n; ++i) {
      float v[VEC];
      gn_load<VEC>(data + i * t.step, v);
      gn_add<VEC, VEC>(v, v, less);
      gn_add<VEC, VEC>(sum, sum, v);
      gn_fma<VEC, VEC, VEC>(squares, v, v, squares);
    }
    const float inv = t.n ? 1.f / n : 0.f;
#pragma unroll
    for (int h = 0; h < PARTS; ++h) {
      float s = 0.f, sq = 0.f;
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        s += sum[h * PER + e];
        sq += squares[h * PER + e];
      }
      m[h] = -less[h * PER] + s * inv;
      q[h] = sq - s * s * inv;
    }
  }
  // ... joined by lanes, ...
  {
    float v[2 * PARTS + 1], first[PARTS];
    v[2 * PARTS] = n;
#pragma unroll
    for (int h = 0; h < PARTS; ++h) {
      first[h] = __shfl_sync(0xffffffffu, m[h], t.lead);
      const float away = t.n ? m[h] - first[h] : 0.f;
      v[h] = n * away;
      v[PARTS + h] = q[h] + n * away * away;
    }
    gn_lanes<2 * PARTS + 1>(v, t.lo, t.hi);
    if (PARTS == 1) gn_lanes<2 * PARTS + 1>(v, t.glo, t.ghi);
    n = v[2 * PARTS];
    const float inv = n > 0.f ? 1.f / n : 0.f;
#pragma unroll
    for (int h = 0; h < PARTS; ++h) {
      m[h] = first[h] + v[h] * inv;
      q[h] = v[PARTS + h] - v[h] * v[h] * inv;
    }
  }
  auto rstd_of = [&](float q) { return 1.f / sqrtf((q < 0.f ? 0.f : q) / all + a.eps); };  // (NaN stays)
  auto keep = [&](int image, int g, float mean, float rstd) {
    if (t.rank == 0 && a.mean) {
      const int64_t at = (int64_t)image * a.groups + t.slab * k.slab + g;
      a.mean[at] = mean;
      a.rstd[at] = rstd;
    }
  };
  if (direct) {
#pragma unroll
    for (int h = 0; h < PARTS; ++h) {
      const float rstd = rstd_of(q[h]);
      const int g = group[h] - t.u * k.slab;
      // (the first of the group's lanes)
      if (t.n && t.p == 0 && (LAST ? t.q * PARTS + h : t.q) == g * k.each) keep(t.image, g, m[h], rstd);
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        less[h * PER + e] = -m[h];
        w[h * PER + e] *= rstd;
      }
    }
  } else {
    if (t.writes) {
#pragma unroll
      for (int h = 0; h < PARTS; ++h) {
        const int at = (t.u * t.r_n + t.row) * t.j_n + (LAST ? t.q * PARTS + h : t.q);
        entry[at] = make_float2(m[h], q[h]);
        count[at] = n;
      }
    }
    if (k.ranks > 1) gn_wait();  // every block of the cluster runs, and its barrier is set up
    __syncthreads();
    // ... by a warp for the block ...
    const int span = gn_span(max(r_all, k.ranks));  // (every lane that gives the result to a rank needs it)
    gn_groups(a, k, t, [&](int i, int u, int g) {
      const float first = entry[u * t.r_n * t.j_n + g * k.each].x;
      float v[3] = {0.f, 0.f, 0.f};
      gn_partials(k, t, u, g, [&](int at) {
        const float c = count[at], away = c > 0.f ? entry[at].x - first : 0.f;
        v[0] += c * away;
        v[1] += entry[at].y + c * away * away;
        v[2] += c;
      });
      gn_lanes<3>(v, 1, span);
      const float inv = v[2] > 0.f ? 1.f / v[2] : 0.f, mean = first + v[0] * inv, away = v[1] - v[0] * v[0] * inv;
      if (k.ranks > 1) {
        if (lane < k.ranks && (t.rank || !a.drop)) gn_give(peer + i * GN_RANKS + t.rank, &bar, lane, make_float2(mean, away));
      } else if (lane == 0) {
        const float rstd = rstd_of(away);
        stat[i] = make_float2(mean, rstd);
        keep(gn_block() * k.units + u, g, mean, rstd);
      }
    });
    // ... and for the cluster.
    if (k.ranks > 1) {
      const int ranks = gn_span(k.ranks);
      const float held = lane < k.ranks ? t.count(a, max(0, min(k.rows, k.all - lane * k.rows))) : 0.f;
      given = gn_given(&bar, a);
      gn_groups(a, k, t, [&](int i, int u, int g) {
        const float first = peer[i * GN_RANKS].x;
        const float2 one = held > 0.f ? peer[i * GN_RANKS + lane] : make_float2(first, 0.f);
        float v[2] = {held * (one.x - first), one.y + held * (one.x - first) * (one.x - first)};
        gn_lanes<2>(v, 1, ranks);
        if (lane == 0) {
          const float mean = first + v[0] / all, rstd = rstd_of(v[1] - v[0] * v[0] / all);
          stat[i] = make_float2(mean, rstd);
          keep(gn_block() * k.units + u, g, mean, rstd);
        }
      });
    }
    __syncthreads();
    if (k.ranks > 1) gn_arrive();
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float2 v = stat[group[e / PER]];
      less[e] = -v.x;
      w[e] *= v.y;
    }
  }
  {
    float* y = a.y + t.offset(k, (int64_t)a.pixels * a.channels, LAST ? a.channels : a.pixels);
    const int64_t next = t.next(k, a.channels);
    auto apply = [&](auto vectors_) {
      constexpr int N = decltype(vectors_)::value * VEC;
      float v[N];
#pragma unroll
      for (int r = 0; r < N; r += VEC) gn_load<VEC>(data + r / VEC * t.step, v + r);
      gn_add<N, VEC>(v, v, less);
      gn_fma<N, VEC, VEC>(v, v, w, b);
      gn_act<N>(v, a.act);
#pragma unroll
      for (int r = 0; r < N; r += VEC) {
        gn_store<VEC>(y, v + r);
        y += next;
      }
      data += N / VEC * t.step;
    };
    int i = 0;
    for (; i + 1 < t.n; i += 2) apply(std::integral_constant<int, 2>{});
    if (i < t.n) apply(std::integral_constant<int, 1>{});
  }
  if (k.ranks > 1) gn_leave_cluster(&bar, given);
}

template <int VEC, int PARTS, bool LAST>
__global__ void __launch_bounds__(GN_MOST_THREADS) gn_resident_backward_kernel(const __grid_constant__ GnArgs a,
                                                                              const __grid_constant__ GnPlan k) {
  extern __shared__ float4 gn_smem[];
  __shared__ float2 stat[GN_GROUPS];
  __shared__ uint64_t bar;
  constexpr int PER = VEC / PARTS, CH = LAST ? VEC : 1;  // CH: channels of a thread
  bool given = true;
  GnPlace<VEC, PARTS, LAST> t(a, k);
  if (k.ranks > 1) {
    if (threadIdx.x == 0) gn_expect(&bar, gn_block() < k.blocks ? k.ranks * t.kk * 8 : 0);
    gn_arrive();
  }
  const int vectors = (k.rows + (1 << k.p_log) - 1) >> k.p_log;
  const int held = (vectors * t.step + 3) & ~3;
  float* xs = reinterpret_cast<float*>(gn_smem) + t.slot;
  float* ds = xs + held;
  float2* peer = reinterpret_cast<float2*>(reinterpret_cast<float*>(gn_smem) + 2 * held);
  float2* entry = peer + (k.ranks > 1 ? k.slab * GN_RANKS : 0);
  pdl_wait();
  {
    const float* x = a.x + t.offset(k, a.xi, a.xr);
    const float* dy = a.dy + t.offset(k, a.gi, a.gr);
    const int64_t xn = t.next(k, a.xr), gn = t.next(k, a.gr);
#pragma unroll 2
    for (int i = 0; i < t.n; ++i, x += xn, dy += gn) {
      gn_copy<VEC>(xs + i * t.step, x);
      gn_copy<VEC>(ds + i * t.step, dy);
    }
  }
  float less[VEC], rstd[VEC], w[VEC], da[2 * CH];  // less: -mean
  int group[PARTS];
#pragma unroll
  for (int h = 0; h < PARTS; ++h) group[h] = t.group(k, h);
  {
    float b[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const int c = t.c + (LAST ? e : 0);
      const int64_t g = (int64_t)t.image * a.groups + t.slab * k.slab + group[e / PER] - t.u * k.slab;
      less[e] = t.n ? -a.mean[g] : 0.f;
      rstd[e] = t.n ? a.rstd[g] : 0.f;
      w[e] = a.w && t.n ? a.w[c] : 1.f;
      b[e] = a.b && t.n ? a.b[c] : 0.f;
    }
#pragma unroll
    for (int e = 0; e < 2 * CH; ++e) da[e] = 0.f;
    gn_copied();
    auto sums = [&](auto two, int i) {
      constexpr int N = decltype(two)::value;
      float xh[N * VEC], dz[N * VEC];
#pragma unroll
      for (int r = 0; r < N; ++r) {
        gn_load<VEC>(xs + (i + r) * t.step, xh + r * VEC);
        gn_load<VEC>(ds + (i + r) * t.step, dz + r * VEC);
      }
#pragma unroll
      for (int r = 0; r < N; ++r) {  // (a vector at a time, for the registers)
        float(&h)[VEC] = *reinterpret_cast<float(*)[VEC]>(xh + r * VEC);
        float(&z)[VEC] = *reinterpret_cast<float(*)[VEC]>(dz + r * VEC);
        gn_slopes<VEC>(h, z, less, rstd, w, b, a.act);
#pragma unroll
        for (int e = 0; e < VEC; e += CH) {
          gn_add<CH, CH>(da, da, z + e);
          gn_fma<CH, CH, CH>(da + CH, z + e, h + e, da + CH);
        }
        gn_store<VEC>(xs + (i + r) * t.step, h);
        gn_store<VEC>(ds + (i + r) * t.step, z);
      }
    };
    int i = 0;
    for (; i + 1 < t.n; i += 2) sums(std::integral_constant<int, 2>{}, i);
    if (i < t.n) sums(std::integral_constant<int, 1>{}, i);
  }
  gn_lanes<2 * CH>(da, t.lo, t.hi);
  const int lane = threadIdx.x & 31, r_all = t.r_n * (k.each / k.lanes);
  const float inv = 1.f / ((float)a.pixels * (float)a.each);
  const bool direct = k.ranks == 1 && r_all == 1;  // every lane of a group has its sums
  float s[2 * PARTS];
#pragma unroll
  for (int h = 0; h < 2 * PARTS; ++h) s[h] = 0.f;
#pragma unroll
  for (int e = 0; e < CH; ++e) {
    s[e / PER] += w[e] * da[e];
    s[PARTS + e / PER] += w[e] * da[CH + e];
  }
  if (PARTS == 1) gn_lanes<2 * PARTS>(s, t.glo, t.ghi);
  float2* column = entry + k.entries;
  if (t.writes) {
    const int row = t.u * t.r_n + t.row;
    if (!direct) {
#pragma unroll
      for (int h = 0; h < PARTS; ++h)
        entry[row * t.j_n + (LAST ? t.q * PARTS + h : t.q)] = make_float2(s[h], s[PARTS + h]);
    }
    if (a.part) {
#pragma unroll
      for (int e = 0; e < CH; ++e) column[((row << k.q_log) + t.q) * CH + e] = make_float2(da[e], da[CH + e]);
    }
  }
  if (k.ranks > 1) gn_wait();  // every block of the cluster runs, and its barrier is set up
  if (!direct || a.part) __syncthreads();
  if (!direct) {
    const int span = gn_span(max(r_all, k.ranks));  // (every lane that gives the sums to a rank needs them)
    gn_groups(a, k, t, [&](int i, int u, int g) {
      float v[2] = {0.f, 0.f};
      gn_partials(k, t, u, g, [&](int at) {
        v[0] += entry[at].x;
        v[1] += entry[at].y;
      });
      gn_lanes<2>(v, 1, span);
      if (k.ranks > 1) {
        if (lane < k.ranks && (t.rank || !a.drop)) gn_give(peer + i * GN_RANKS + t.rank, &bar, lane, make_float2(v[0], v[1]));
      } else if (lane == 0) {
        stat[i] = make_float2(v[0] * inv, v[1] * inv);
      }
    });
  }
  if (a.part) {  // the channels' sums of all images of the block
    const int first = t.slab * k.slab * a.each, n = t.kk * a.each, block = gn_block();
    const int64_t row = (int64_t)block * k.ranks + t.rank;
    for (int c = threadIdx.x; c < n && block < k.blocks; c += blockDim.x) {
      float2 v = make_float2(0.f, 0.f);
      for (int r = 0; r < k.units * t.r_n; ++r) {
        const float2 o = column[(r << k.q_log) * CH + c];
        v.x += o.x;
        v.y += o.y;
      }
      a.part[row * a.channels + first + c] = v.x;
      a.part[(a.segs_n + row) * a.channels + first + c] = v.y;
    }
  }
  if (k.ranks > 1) {
    const int ranks = gn_span(k.ranks);
    given = gn_given(&bar, a);
    gn_groups(a, k, t, [&](int i, int, int) {
      const float2 one = lane < k.ranks ? peer[i * GN_RANKS + lane] : make_float2(0.f, 0.f);
      float v[2] = {one.x, one.y};
      gn_lanes<2>(v, 1, ranks);
      if (lane == 0) stat[i] = make_float2(v[0] * inv, v[1] * inv);
    });
  }
  if (!direct) __syncthreads();
  if (k.ranks > 1) gn_arrive();
  if (a.y && t.n) {
    // dx = rstd w dz - (rstd s2 xh + rstd s1), each product rounded once
    float s1[VEC], s2[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float2 v = direct ? make_float2(s[e / PER] * inv, s[PARTS + e / PER] * inv) : stat[group[e / PER]];
      w[e] *= rstd[e];
      s1[e] = -rstd[e] * v.x;
      s2[e] = -rstd[e] * v.y;
    }
    float* dx = a.y + t.offset(k, (int64_t)a.pixels * a.channels, LAST ? a.channels : a.pixels);
    const int64_t next = t.next(k, a.channels);
#pragma unroll 2
    for (int i = 0; i < t.n; ++i, dx += next) {
      float xh[VEC], dz[VEC];
      gn_load<VEC>(xs + i * t.step, xh);
      gn_load<VEC>(ds + i * t.step, dz);
      gn_fma<VEC, VEC, VEC>(xh, xh, s2, s1);
      gn_fma<VEC, VEC, VEC>(dz, dz, w, xh);
      gn_store<VEC>(dx, dz);
    }
  }
  if (k.ranks > 1) gn_leave_cluster(&bar, given);
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------

// Set by mm_debug_tc_fault for a device's later launches (0 tries: GN_TRIES).
static std::atomic<int> g_gn_tries[64], g_gn_drop[64];

void gn_debug_fault(int device, int64_t wait_ns, int drop) {
  if (device < 0 || device >= 64) return;
  g_gn_tries[device] = wait_ns > 0 ? (int)std::min<int64_t>(std::max<int64_t>(wait_ns / 1000000, 1), GN_TRIES) : 0;
  g_gn_drop[device] = drop;
}

constexpr int GN_SMEM = 227 * 1024;      // of an SM; a block's 1 KB and its static part come off it
constexpr int GN_SMEM_FIXED = 1024 + GN_GROUPS * 8 + 16;

static int gn_log(int v) {  // the least power of two that holds v
  int l = 0;
  while ((1 << l) < v) ++l;
  return l;
}

int64_t gn_plan_rows(int64_t n, int64_t pixels) {
  const int64_t ranks = (pixels + 63) / 64;
  return n * (ranks < GN_RANKS ? ranks : GN_RANKS);
}

// Completes a plan of given threads, slab, units and ranks: false where a block's
// share does not fit `room` bytes.
static bool gn_fit(GnPlan& p, const GnArgs& a, int vec, int part, bool last, bool backward, int room) {
  const int64_t width = (int64_t)p.slab * a.each;
  p.q = (int)(last ? width / vec : width);
  p.columns = last ? a.channels / vec : a.channels;
  p.q_log = gn_log(p.q);
  p.p_log = gn_log(p.threads / p.units) - p.q_log;
  if (p.p_log < 0) return false;
  p.all = last ? a.pixels : a.pixels / vec;
  p.rows = (p.all + p.ranks - 1) / p.ranks;
  p.slabs = (a.groups + p.slab - 1) / p.slab;
  p.blocks = (a.n + p.units - 1) / p.units;
  p.each = last ? a.each / part : a.each;
  p.lanes = 1;
  const int lanes = !last ? 32 >> std::min(p.p_log, 5) : part == vec ? 32 : 1;
  while (2 * p.lanes <= lanes && p.each % (2 * p.lanes) == 0) p.lanes *= 2;
  const int unit = 1 << (p.q_log + p.p_log), q_n = 1 << p.q_log, p_n = 1 << p.p_log;
  const int rows = last ? (q_n >= 32 ? p_n : std::max(1, unit / 32)) : std::max(1, p_n / 32);
  const int parts = last ? vec / part : 1;
  p.entries = p.units * rows * q_n * parts;
  const int64_t vectors = (p.rows + p_n - 1) / p_n;
  const int64_t held = (vectors * p.units * p.q * p_n * vec + 3) & ~(int64_t)3;
  const int64_t bytes = held * (backward ? 8 : 4) + (p.ranks > 1 ? p.slab * GN_RANKS * 8 : 0) +
                        (int64_t)p.entries * (backward ? 8 : 12) +
                        (backward ? (int64_t)p.units * rows * q_n * (last ? vec : 1) * 8 : 0);
  if (bytes > room) return false;
  p.smem = (int)bytes;
  p.inv_each = 1.f / (float)p.each;
  p.inv_slab = 1.f / (float)p.slab;
  return true;
}

// The plan of least estimated time, in us; none (ranks 0) where the walking kernels
// take less.  The rates are those that maps larger than L2 were measured at, by the
// blocks that an SM holds: forward 64 x 64 x 80 x 80 4.4 TB/s with four, 3.9 with two,
// 3.5 with one (walking: 3.2), 16 x 128 x 160 x 160 3.3, 3.6, 3.2 (3.6: 32-byte rows, 64,
// 64); backward 32 x 256 x 40 x 40 3.1, 2.7, 2.1 (2.7), 16 x 128 x 160 x 160 none, 2.0, 2.1
// (3.6).
static const struct GnShape {
  int threads, blocks;
  double forward, backward;  // bytes per us
} gn_shapes[] = {{256, 4, 4.5e6, 3.4e6}, {512, 2, 4.0e6, 2.9e6}, {1024, 1, 3.5e6, 2.1e6}};

static int gn_room(const GnShape& shape) { return GN_SMEM / shape.blocks - GN_SMEM_FIXED; }

GnPlan gn_plan_of(const GnArgs& a, int vec, bool last, bool backward, int most_ranks) {
  if (most_ranks < 1) return GnPlan();
  const double bytes = (double)a.n * a.channels * a.pixels * (backward ? 12 : 8);  // in and out
  const int64_t most = std::min<int64_t>(most_ranks, (a.pixels + 63) / 64), sms = sm_count();
  // Values of one group in a vector.
  const int part = a.each % vec == 0 || !last ? vec : a.each % 2 == 0 && vec == 4 ? 2 : 1;
  GnPlan best;
  double least = backward ? 12.0 + bytes / 3.5e6 : 10.0 + bytes / 3.95e6;  // walking
  int slab = 1;  // the fewest groups that whole vectors hold, then twice as many up to rows of 256 bytes
  while (last && slab < a.groups && (int64_t)slab * a.each % vec != 0) slab *= 2;
  for (slab = std::min(slab, a.groups); slab <= GN_GROUPS; slab = std::min(2 * slab, a.groups)) {
    const int64_t width = (int64_t)slab * a.each;
    for (const GnShape& shape : gn_shapes) {
      GnPlan p;
      p.slab = slab;
      p.units = 1;
      p.threads = shape.threads;
      const int room = gn_room(shape);
      const int64_t share = width * a.pixels * (backward ? 8 : 4) / room;
      if (share > most) continue;
      bool fits = false;
      for (p.ranks = (int)std::max<int64_t>(share, 1); p.ranks <= most; ++p.ranks)
        if ((fits = gn_fit(p, a, vec, part, last, backward, room))) break;
      if (!fits) continue;
      while (p.ranks == 1 && 2 * p.units * p.slab <= GN_GROUPS && (int64_t)p.blocks * p.slabs >= 2 * sms * 4) {
        GnPlan more = p;  // several small images' units in a block, while its threads have few vectors
        more.units *= 2;
        if (!gn_fit(more, a, vec, part, last, backward, room) || ((more.rows - 1) >> more.p_log) >= 4) break;
        p = more;
      }
      // Rows narrower than a line's half waste sectors; lanes without a column copy nothing
      // (8 x 320 x 64 x 64 in 32 groups, five of eight lanes: 3.7 and 2.8 TB/s).
      const double piece = last ? (double)std::min<int64_t>(width, a.channels) * 4 : 128;
      const double lanes = last ? 0.7 + 0.3 * (1 << p.q_log) / p.q : 1.0;
      const double waste = (piece >= 64 ? 1.0 : piece >= 32 ? 1.3 : 2.2) * lanes;
      const double grid = (double)p.blocks * p.slabs * p.ranks, waves = grid / ((double)sms * shape.blocks);
      const double rate = std::min(backward ? shape.backward : shape.forward, grid * 5e4);
      const double time = 5.0 + 0.1 * p.ranks + bytes / rate * waste * (0.5 + 0.5 * std::ceil(waves) / std::max(waves, 1.0));
      if (time < least) {
        least = time;
        best = p;
      }
    }
    if (slab == a.groups || width * 4 >= 256) break;
  }
  if (best.ranks && ((int64_t)best.blocks > 65535LL * 65535 || (int64_t)best.slabs * best.ranks > INT32_MAX))
    best.ranks = 0;
  return best;
}

// What is known of a kernel on a device.  Host threads may race here, which only repeats
// the calls.
struct GnKnown {
  std::atomic<bool> ready;                           // its attributes are set
  std::atomic<int8_t> places[3][GN_RANKS + 1];       // by shape and ranks: 1 a cluster has room, 2 it has not
};

template <class K>
static cudaError_t gn_ready(K kernel, GnKnown* known, int dev) {
  if (dev >= 0 && dev < 64 && known[dev].ready.load(std::memory_order_acquire)) return cudaSuccess;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, GN_SMEM - GN_SMEM_FIXED);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e == cudaSuccess && dev >= 0 && dev < 64) known[dev].ready.store(true, std::memory_order_release);
  return e;
}

// Whether the device can place a cluster of the plan's blocks, each with all of the shared
// memory that its shape may take.
template <class K>
static bool gn_places(K kernel, GnKnown* known, const GnPlan& p, int dev) {
  int shape = 0;
  while (gn_shapes[shape].threads != p.threads) ++shape;
  std::atomic<int8_t>* at = dev >= 0 && dev < 64 ? &known[dev].places[shape][p.ranks] : nullptr;
  if (at)
    if (const int8_t v = at->load(std::memory_order_relaxed)) return v == 1;
  int clusters = 0;
  cudaError_t e = gn_ready(kernel, known, dev);
  if (e == cudaSuccess) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)p.ranks);
    cfg.blockDim = dim3(p.threads);
    cfg.dynamicSmemBytes = gn_room(gn_shapes[shape]);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)p.ranks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg);
  }
  if (e != cudaSuccess) {
    cudaGetLastError();
    return false;
  }
  if (at) at->store(clusters > 0 ? 1 : 2, std::memory_order_relaxed);
  return clusters > 0;
}

template <class K>
static cudaError_t gn_resident_launch(K kernel, GnKnown* known, const GnArgs& args, const GnPlan& p, cudaStream_t s) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = gn_ready(kernel, known, dev);
  if (e != cudaSuccess) return e;
  GnArgs a = args;
  const unsigned z = (unsigned)((p.blocks + 65534) / 65535), y = (unsigned)((p.blocks + z - 1) / z);
  const dim3 grid((unsigned)(p.slabs * p.ranks), y, z);
  if (p.ranks == 1) return launch_pdl(kernel, grid, dim3(p.threads), p.smem, s, a, p);
  a.fault = fault_word(dev, true);
  if (a.fault == nullptr) return cudaErrorMemoryAllocation;
  const int tries = g_gn_tries[dev];  // (a device with a fault word is below 64)
  a.tries = tries ? tries : GN_TRIES;
  a.drop = g_gn_drop[dev];
  return launch_pdl_cluster(kernel, grid, dim3(p.threads), p.ranks, p.smem, s, a, p);
}

template <int VEC, int PARTS, bool LAST, bool BACKWARD>
struct GnResident {
  static inline GnKnown known[64];
  static constexpr auto kernel() {
    if constexpr (BACKWARD) return gn_resident_backward_kernel<VEC, PARTS, LAST>;
    else return gn_resident_kernel<VEC, PARTS, LAST>;
  }
  static cudaError_t launch(const GnArgs& a, const GnPlan& p, cudaStream_t s) {
    return gn_resident_launch(kernel(), known, a, p, s);
  }
  static bool places(const GnPlan& p, int dev) { return gn_places(kernel(), known, p, dev); }
};

// Calls f with the kernel of a call.
template <bool BACKWARD, class F>
static auto gn_resident_of(const GnArgs& a, int vec, bool last, F f) {
  if (!last) {
    if (vec == 4) return f(GnResident<4, 1, false, BACKWARD>());
    if (vec == 2) return f(GnResident<2, 1, false, BACKWARD>());
    return f(GnResident<1, 1, false, BACKWARD>());
  }
  if (vec == 4) {
    if (a.each % 4 == 0) return f(GnResident<4, 1, true, BACKWARD>());
    if (a.each % 2 == 0) return f(GnResident<4, 2, true, BACKWARD>());
    return f(GnResident<4, 4, true, BACKWARD>());
  }
  if (vec == 2) {
    if (a.each % 2 == 0) return f(GnResident<2, 1, true, BACKWARD>());
    return f(GnResident<2, 2, true, BACKWARD>());
  }
  return f(GnResident<1, 1, true, BACKWARD>());
}

cudaError_t gn_resident_forward(const GnArgs& a, const GnPlan& p, int vec, bool last, cudaStream_t s) {
  return gn_resident_of<false>(a, vec, last, [&](auto k) { return k.launch(a, p, s); });
}

cudaError_t gn_resident_backward(const GnArgs& a, const GnPlan& p, int vec, bool last, cudaStream_t s) {
  return gn_resident_of<true>(a, vec, last, [&](auto k) { return k.launch(a, p, s); });
}

// Set by mm_debug_group_norm_ranks for a device's later calls, plus one (0: GN_RANKS).
static std::atomic<int> g_gn_most[64];

int gn_debug_ranks(int device, int most) {
  if (device < 0 || device >= 64) return fail(MM_ERR_INVALID, "mm_debug_group_norm_ranks: invalid device");
  g_gn_most[device] = most < 0 ? 0 : std::min(most, GN_RANKS) + 1;
  return MM_OK;
}

GnPlan gn_plan(const GnArgs& a, int vec, bool last, bool backward) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) cudaGetLastError();
  const int set = dev >= 0 && dev < 64 ? g_gn_most[dev].load(std::memory_order_relaxed) : 0;
  for (int most = set ? set - 1 : GN_RANKS;;) {
    const GnPlan p = gn_plan_of(a, vec, last, backward, most);
    if (p.ranks <= 1) return p;
    const auto places = [&](auto k) { return k.places(p, dev); };
    if (backward ? gn_resident_of<true>(a, vec, last, places) : gn_resident_of<false>(a, vec, last, places)) return p;
    most = p.ranks - 1;
  }
}

}  // namespace mm
