// Matrix products of the linear operator on the tensor cores, in float32
// accuracy.
//
// A float32 value is the exact sum of three bf16 values: a1 = a rounded to
// bf16, a2 = (a - a1) rounded to bf16, a3 = a - a1 - a2 (24 significant bits =
// 3 x 8, and bf16 has float32's exponents, so nothing is scaled).  That holds from
// 2^-110 (8e-34) on; bf16's smallest step is 2^-133, so a smaller value is kept to
// within 2^-133 (products with values around 1e-36: 3e-5 relative).  Of the nine products of pieces the six largest are
// formed, a1 b1, a1 b2, a2 b1, a2 b2, a1 b3, a3 b1; the other three are below
// 2^-24 of the whole.  Six bf16 products instead of one bound the rate at a
// sixth of the bf16 rate.
//
//   linear_split_kernel   float32 operands -> three bf16 planes each (6 bytes
//                         per value), with dz = dy act'(z) and the partial
//                         sums of db on the way in the backward pass
//   linear_gemm_kernel    C = A B^T (+ epilogue) over the planes
//   linear_join_kernel    sums of the tiles whose reduction was divided
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <string>

#include "mm_linear_tc.cuh"

namespace mm {

// ---------------------------------------------------------------------------
// Splitting
// ---------------------------------------------------------------------------

constexpr int SP_ROWS = 64, SP_COLS = 128;  // values per block

// Three bf16 pieces (as their float32 bits, low halves zero).  a1 is rounded to
// nearest but stays finite; infinities and NaNs keep a2 = a3 = 0.
__device__ __forceinline__ void split3(float a, uint32_t& h1, uint32_t& h2, uint32_t& h3) {
  const uint32_t u = __float_as_uint(a);
  const uint32_t mag = u & 0x7fffffffu, sign = u & 0x80000000u;
  if (mag >= 0x7f800000u) {
    h1 = mag > 0x7f800000u ? 0x7fc00000u : u;
    h2 = h3 = 0u;
    return;
  }
  h1 = sign | min((mag + 0x8000u) & 0xffff0000u, 0x7f7f0000u);
  const float r = a - __uint_as_float(h1);
  h2 = (__float_as_uint(r) + 0x8000u) & 0xffff0000u;
  h3 = __float_as_uint(r - __uint_as_float(h2)) & 0xffff0000u;
}

// Blocks of 64 x 128 values: 16 threads x 8 values across a row, 16 rows at a
// time, the next rows' values on their way meanwhile.  Bound by memory (4 bytes
// in, with z 8, and 6 out per value) but for GELU's slope.
__global__ void __launch_bounds__(256) linear_split_kernel(const __grid_constant__ LinSplits all) {
  __shared__ float sums[16][SP_COLS + 4];
  int k = 0;
  while (k + 1 < all.count && blockIdx.x >= all.s[k + 1].first) ++k;
  const LinSplit& s = all.s[k];
  const int block = (int)(blockIdx.x - s.first);
  const int bc = block % s.blocks_c, br = block / s.blocks_c;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int c0 = bc * SP_COLS + tx * 8, left = s.cols - c0;
  const int64_t end = min((int64_t)(br + 1) * SP_ROWS, s.rows);
  int64_t row = (int64_t)br * SP_ROWS + ty;
  float sum[8] = {}, next[8], znext[8] = {};
  int inf = 0;
  pdl_wait();
  pdl_trigger();
  const bool any = left > 0;
  auto fetch = [&](int64_t r) {
    const float* src = s.src + r * s.s0;
    if (s.s1 == 1) {
      lin_load_row<8>(src + c0, left, s.vec, next);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) next[e] = e < left ? src[(int64_t)(c0 + e) * s.s1] : 0.f;
    }
    if (s.z) lin_load_row<8>(s.z + r * s.cols + c0, left, s.vec, znext);
  };
  if (any && row < end) fetch(row);
#pragma unroll 1
  for (; any && row < end; row += 16) {
    float v[8], z[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = next[e];
      z[e] = znext[e];
    }
    if (row + 16 < end) fetch(row + 16);
    if (s.z) lin_times_slope<8>(v, z, s.act);
    if (s.out) lin_store_row<8>(s.out + row * s.cols + c0, left, false, v);
    uint32_t p[3][4];
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      uint32_t a1, a2, a3, b1, b2, b3;
      split3(v[e], a1, a2, a3);
      split3(v[e + 1], b1, b2, b3);
      p[0][e / 2] = a1 >> 16 | b1;
      p[1][e / 2] = a2 >> 16 | b2;
      p[2][e / 2] = a3 >> 16 | b3;
    }
#pragma unroll
    for (int q = 0; q < 3; ++q)
      *reinterpret_cast<uint4*>(s.planes + (q * s.rows + row) * s.ld + c0) = make_uint4(p[q][0], p[q][1], p[q][2], p[q][3]);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      sum[e] += v[e];
      inf |= (__float_as_uint(v[e]) & 0x7fffffffu) == 0x7f800000u;
    }
  }
  inf = __syncthreads_or(inf);
  if (threadIdx.x == 0) s.flags[block] = inf;
  if (!s.part) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) sums[ty][tx * 8 + e] = sum[e];
  __syncthreads();
  const int c = bc * SP_COLS + threadIdx.x;
  if (threadIdx.x < SP_COLS && c < s.cols) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) t += sums[i][threadIdx.x];
    s.part[(int64_t)br * s.cols + c] = t;
  }
}

// ---------------------------------------------------------------------------
// Tensor-core product
// ---------------------------------------------------------------------------

enum { LG_ERR_FULL = 101, LG_ERR_EMPTY = 102, LG_ERR_ACC = 103, LG_ERR_FREE = 104, LG_ERR_DRAIN = 105 };

constexpr int LG_BM = 128, LG_BK = 32;
constexpr int LG_ACCS = 4;  // accumulators in tensor memory (at most 512 columns)
constexpr int LG_EPI_WARPS = 8, LG_WARP_TMA = 8, LG_WARP_MMA = 9, LG_ISSUERS = 2, LG_THREADS = 352;
constexpr int64_t LG_WAIT_NS = 200ll * 1000 * 1000;
// Set by mm_debug_tc_fault for a device's later launches (0: the limit above).
static std::atomic<int64_t> g_lin_wait_ns[64];
static std::atomic<int> g_lin_drop[64];

__device__ __forceinline__ uint32_t lg_smem(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void lg_bar_init(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(lg_smem(bar)), "r"(count));
}

// CLUSTER: threads of both CTAs arrive.
template <bool CLUSTER>
__device__ __forceinline__ bool lg_try(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  if (CLUSTER)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(lg_smem(bar)), "r"(parity), "r"(1000u)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(lg_smem(bar)), "r"(parity), "r"(1000u)
        : "memory");
  return ok != 0;
}

// Bounded wait.  It gives up after 200 ms and records which one did in the
// device's fault word, which is host memory: the host sees it at its next wait
// for the stream.  Nothing else reads it, so one launch's error shortens no
// wait of another's.
template <bool CLUSTER = false>
__device__ __forceinline__ bool lg_wait(const LinGemm& a, uint64_t* bar, uint32_t parity, int code) {
  if (lg_try<CLUSTER>(bar, parity)) return true;
  uint64_t t0, t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t0));
  for (uint32_t i = 1; i < (1u << 26); ++i) {
    if (lg_try<CLUSTER>(bar, parity)) return true;
    if ((i & 63) == 0) {
      asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
      if ((int64_t)(t - t0) > a.wait_ns) break;
    }
  }
  volatile int* fault = a.fault;
  if (fault != nullptr && *fault == 0) *fault = code;  // (of several, one of them)
  return false;
}

__device__ __forceinline__ void lg_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(lg_smem(bar)) : "memory");
}

// The cluster's address of CTA 0's barrier (or another one's of this CTA).
__device__ __forceinline__ uint32_t lg_lead(uint64_t* bar) {
  uint32_t addr;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(addr) : "r"(lg_smem(bar)));
  return addr;
}

// To a barrier of the pair's CTA 0 from either CTA, so with the cluster's scope.  It
// says that tensor memory has been read: tcgen05.wait::ld has ended and
// tcgen05.fence::before_thread_sync stands before it, which order the reads
// before it, and the fence behind the wait of CTA 0's issuer orders its MMAs
// after it, whatever the arrival's semantics; no other memory has to be seen by
// the other CTA, so it is relaxed (a release to the cluster waits for the stores
// under way, 1,000 to 2,000 clocks).
__device__ __forceinline__ void lg_arrive_at(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// All threads of the CTA, of both in a pair.
template <bool PAIR>
__device__ __forceinline__ void lg_sync() {
  if (PAIR) {
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
  } else {
    __syncthreads();
  }
}

// When the MMAs issued so far are done, arrive on the barrier; in a pair on
// both CTAs'.
template <bool PAIR>
__device__ __forceinline__ void lg_commit(uint64_t* bar) {
  if (PAIR) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            lg_smem(bar)),
        "h"((uint16_t)3)
        : "memory");
    return;
  }
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(lg_smem(bar))
               : "memory");
}

template <bool PAIR>
__device__ __forceinline__ void lg_load(void* dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
  if (PAIR) {  // the barrier may be the other CTA's
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
        "%3, %4}], [%5];" ::"r"(lg_smem(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(0), "r"(bar)
        : "memory");
    return;
  }
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(lg_smem(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(0), "r"(bar)
      : "memory");
}

template <bool PAIR>
__device__ __forceinline__ void lg_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if (PAIR) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
    return;
  }
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ bool lg_elect() {
  uint32_t leader;
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b32 l;\n\t"
      "elect.sync l|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(leader));
  return leader != 0;
}

__device__ __forceinline__ void lg_tmem_load32(uint32_t addr, float* v) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// An operand tile of ROWS rows (of C's m or n) and 32 of the reduction, three
// planes.  K-major (the planes' rows are dense along the reduction): ROWS rows
// of 64 bytes per plane, 64-byte swizzle, 8-row groups 512 bytes apart.
// MN-major (dense along m or n): groups of 64 of them, 32 rows of 128 bytes per
// plane and group, 128-byte swizzle; groups 12 KB apart, 8-row groups 1 KB.
template <int ROWS, bool MN>
struct LgTile {
  static constexpr uint32_t plane = MN ? 4096u : ROWS * 64u;
  static constexpr uint32_t bytes = ROWS * 192u;
  static constexpr uint32_t hi = (MN ? (1024u >> 4) : (512u >> 4)) | 1u << 14 | (MN ? 2u : 4u) << 29;
  // Descriptor of piece p (0..2), step kk (16 of the reduction) of the tile at addr.
  static __device__ __forceinline__ uint64_t desc(uint32_t addr, int p, int kk) {
    const uint32_t at = addr + (uint32_t)p * plane + (uint32_t)kk * (MN ? 2048u : 32u);
    const uint32_t lo = ((at >> 4) & 0x3fffu) | ((MN ? 12288u >> 4 : 1u) << 16);
    return (uint64_t)hi << 32 | lo;
  }
  template <bool PAIR>
  static __device__ __forceinline__ void load(uint8_t* dst, const CUtensorMap* map, uint32_t bar, int row, int k) {
    if (MN) {
#pragma unroll
      for (int g = 0; g < ROWS / 64; ++g) lg_load<PAIR>(dst + g * 12288, map, bar, row + 64 * g, k);
    } else {
      lg_load<PAIR>(dst, map, bar, k, row);
    }
  }
};

// Stages that shared memory holds: 48 KB each, or 36.
template <int BN, bool PAIR>
constexpr int lg_stages() {
  return BN == 128 && !PAIR ? 4 : 5;
}

// One unit of work: an output tile and a range of its reduction's stages.
struct LgUnit {
  int m0, n0, begin, end;
  int part;  // index of its partial tile, or -1: the whole reduction
};

__device__ __forceinline__ LgUnit lg_unit(const LinGemm& a, int u, int bn) {
  LgUnit w;
  int tile = u, split = 0, splits = 1;
  w.part = -1;
  if (u >= a.full) {
    tile = a.full + (u - a.full) / a.splits;
    split = (u - a.full) % a.splits;
    splits = a.splits;
    if (splits > 1) w.part = u - a.full;
  }
  // Tiles in groups of eight rows of tiles, column by column, so that those
  // running together share operand tiles in L2.
  const int per = LIN_GROUP * a.tiles_n;
  const int group = tile / per, in = tile - group * per;
  const int rows = min(LIN_GROUP, a.tiles_m - group * LIN_GROUP);
  w.m0 = (group * LIN_GROUP + in % rows) * a.bm;
  w.n0 = (in / rows) * bn;
  w.begin = (int)((int64_t)a.stages * split / splits);
  w.end = (int)((int64_t)a.stages * (split + 1) / splits);
  return w;
}

// ---------------------------------------------------------------------------
// Infinities.  Their pieces are (inf, 0, 0), and inf times another operand's
// zero piece is NaN where the whole product is infinite.  linear_split_kernel
// says which of its blocks hold an infinity; a tile's rows of A and of B (rows
// and columns of C) that hold one and no NaN are computed again, from the
// pieces' sums in float32, by the block that has stored the tile.
// ---------------------------------------------------------------------------

__device__ __forceinline__ float lin_value(const LinPlanes& p, int64_t line, int64_t k) {
  const int64_t at = p.mn ? k * p.ld + line : line * p.ld + k;
  const int64_t plane = p.mn ? p.k * p.ld : p.lines * p.ld;
  float v = 0.f;
#pragma unroll
  for (int q = 2; q >= 0; --q) v += __uint_as_float((uint32_t)__ldcg(&p.planes[q * plane + at]) << 16);
  return v;
}

// Whether any flag of the blocks of lines [l0, l1) is set, for the whole thread
// block (every thread calls).
__device__ __forceinline__ bool lin_flagged(const LinPlanes& p, int l0, int l1) {
  const int per = p.mn ? SP_COLS : SP_ROWS;
  const int across = (int)((p.k + (p.mn ? SP_ROWS : SP_COLS) - 1) / (p.mn ? SP_ROWS : SP_COLS));
  const int blocks_c = (int)(((p.mn ? p.lines : p.k) + SP_COLS - 1) / SP_COLS);
  const int b0 = l0 / per, b1 = (l1 + per - 1) / per;
  int any = 0;
  for (int i = threadIdx.x; i < (b1 - b0) * across; i += blockDim.x) {
    const int block = b0 + i / across, at = i % across;
    any |= __ldcg(&p.flags[p.mn ? at * blocks_c + block : block * blocks_c + at]);
  }
  return __syncthreads_or(any) != 0;
}

template <bool B>
__device__ __noinline__ void lin_fix_lines(const LinGemm& a, int m0, int m1, int n0, int n1) {
  const LinPlanes& p = B ? a.pb : a.pa;
  const LinPlanes& other = B ? a.pa : a.pb;
  const int l0 = B ? n0 : m0, l1 = B ? n1 : m1, o0 = B ? m0 : n0, o1 = B ? m1 : n1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  for (int line = l0; line < l1; ++line) {
    int inf = 0, nan = 0;
    for (int64_t k = threadIdx.x; k < p.k; k += blockDim.x) {
      const float v = lin_value(p, line, k);
      inf |= isinf(v);
      nan |= isnan(v);
    }
    inf = __syncthreads_or(inf);
    nan = __syncthreads_or(nan);
    if (!inf || nan) continue;  // a NaN makes the whole line NaN already
    for (int o = o0 + warp; o < o1; o += warps) {
      float v = 0.f;
      for (int64_t k = lane; k < p.k; k += 32) v += lin_value(p, line, k) * lin_value(other, o, k);
#pragma unroll
      for (int s = 16; s > 0; s >>= 1) v += __shfl_xor_sync(0xffffffffu, v, s);
      const int row = B ? o : line, col = B ? line : o;
      if (lane == 0) a.c[(int64_t)row * a.n + col] = lin_finish(a.e, v, row, col, a.n);
    }
  }
}

// Every thread of the block calls, after the tile [m0, m0 + rows) x [n0, n0 +
// cols) has been stored and a __syncthreads.
__device__ __forceinline__ void lin_fix(const LinGemm& a, int m0, int rows, int n0, int cols) {
  const int m1 = min(m0 + rows, a.m), n1 = min(n0 + cols, a.n);
  if (m0 >= m1 || n0 >= n1) return;
  if (lin_flagged(a.pa, m0, m1)) lin_fix_lines<false>(a, m0, m1, n0, n1);
  if (lin_flagged(a.pb, n0, n1)) lin_fix_lines<true>(a, m0, m1, n0, n1);
}

// The epilogue of N columns from col on of one row, held by one thread, where
// all of them exist and rows are 16-byte aligned.
template <int N>
__device__ __forceinline__ void lg_finish_row(const LinGemm& a, float (&acc)[N], int64_t row, int col) {
  const LinEpilogue& e = a.e;
  if (row >= a.m) return;
  float* out = a.c + row * a.n + col;
  const float* res = e.residual ? e.residual + row * e.rs + col : nullptr;
  if (e.bias) {
#pragma unroll
    for (int j = 0; j < N / 4; ++j) {
      const float4 b = reinterpret_cast<const float4*>(e.bias + col)[j];
      acc[4 * j] += b.x; acc[4 * j + 1] += b.y; acc[4 * j + 2] += b.z; acc[4 * j + 3] += b.w;
    }
  }
  if (res && e.residual_first) {
#pragma unroll
    for (int j = 0; j < N / 4; ++j) {
      const float4 t = reinterpret_cast<const float4*>(res)[j];
      acc[4 * j] += t.x; acc[4 * j + 1] += t.y; acc[4 * j + 2] += t.z; acc[4 * j + 3] += t.w;
    }
  }
  if (e.z) {
    float4* z = reinterpret_cast<float4*>(e.z + row * a.n + col);
#pragma unroll
    for (int j = 0; j < N / 4; ++j) z[j] = make_float4(acc[4 * j], acc[4 * j + 1], acc[4 * j + 2], acc[4 * j + 3]);
  }
  // Eight columns at a time; the totals move down by eight registers per step,
  // so that the activations' code is there once.
#pragma unroll 1
  for (int j = 0; j < N / 8; ++j) {
    float v[8], t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = acc[i];
    if (res && !e.residual_first) lin_load_row<8>(res + 8 * j, 8, true, t);
    lin_act<8>(v, e.act);
    if (res && !e.residual_first) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] += t[i];
    }
    lin_store_row<8>(out + 8 * j, 8, true, v);
#pragma unroll
    for (int i = 0; i + 8 < N; ++i) acc[i] = acc[i + 8];
  }
}

// The epilogue elsewhere (a width that is no multiple of four, the last tile's
// columns): of 32 x 32 outputs that a warp has put into shared memory (row r,
// column c at 32 r + (c ^ r): no bank conflicts either way), a column per lane,
// so that every row is read and written in one piece of 128 bytes whatever its
// alignment.  1111 x 1502 x 2501: 72 us, a row per thread 83; where both apply
// (2000 x 1280 x 1000) 47, a row per thread 41.
template <int ACT>
__device__ __forceinline__ void lg_finish_rows(const LinGemm& a, const float* tile, int row0, int col, int lane) {
  const LinEpilogue& e = a.e;
  const bool valid = col < a.n;
  const int rows = min(32, a.m - row0);
  const float bias = e.bias && valid ? e.bias[col] : 0.f;
  const float* res = e.residual ? e.residual + (int64_t)row0 * e.rs + col : nullptr;
  float* z = e.z ? e.z + (int64_t)row0 * a.n + col : nullptr;
  float* out = a.c + (int64_t)row0 * a.n + col;
  constexpr int U = 8;  // rows at a time: their residuals are on their way together
  for (int r0 = 0; r0 < rows; r0 += U) {
    float t[U] = {}, v[U];
    if (res) {
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (valid && r0 + i < rows) t[i] = res[(r0 + i) * e.rs];
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int r = r0 + i;
      v[i] = tile[32 * r + (lane ^ r)] + bias;
      if (e.residual_first) v[i] += t[i];
      if (z && valid && r < rows) z[(int64_t)r * a.n] = v[i];
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      v[i] = lin_act_t<ACT>(v[i]);
      if (!e.residual_first) v[i] += t[i];
      if (valid && r0 + i < rows) out[(int64_t)(r0 + i) * a.n] = v[i];
    }
  }
}

// Persistent CTAs, one per SM.  Warps 0-7 add up and store, warp 8 loads (TMA),
// warps 9 and 10 issue the MMAs of alternate stages.  The MMAs of one stage (32
// of the reduction, twelve products of 128 x BN x 16) go into one of four
// accumulators in tensor memory, small products first; warps 0-7 add it to
// float32 totals in registers while the next stages run in the others.  The
// tensor core rounds its sums toward zero, which over a long reduction drifts
// by about K 2^-24; with one stage per accumulator only the two a1 b1 products
// of a stage are added at full size.  One issuer left the tensor core idle for
// the 300 to 400 clocks of its waits and commits in each stage (2000 x 1280 x
// 1000: 49 us, with two 44).
//
// PAIR: two CTAs on neighbouring SMs share a tile of 256 rows.  Each loads its
// 128 rows of A and half of B's, which is what bounds a stage (36 KB in place
// of 48); CTA 0 issues the MMAs of both, each CTA keeps and stores its rows.
template <int BN, bool AMN, bool BMN, bool PAIR>
__global__ void __launch_bounds__(LG_THREADS, 1) linear_gemm_kernel(const __grid_constant__ CUtensorMap ma,
                                                                    const __grid_constant__ CUtensorMap mb,
                                                                    const LinGemm a) {
  using TA = LgTile<LG_BM, AMN>;
  using TB = LgTile<PAIR ? BN / 2 : BN, BMN>;
  constexpr int S = lg_stages<BN, PAIR>();
  constexpr uint32_t stage_bytes = TA::bytes + TB::bytes;
  constexpr int ACCS = LG_ACCS;
  constexpr uint32_t cols = ACCS * BN;
  constexpr int HALF = BN / 2;  // columns per warp
  extern __shared__ uint8_t raw[];
  uint8_t* smem = raw + ((1024 - (lg_smem(raw) & 1023)) & 1023);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S * stage_bytes);
  uint64_t *empty = full + S, *acc_full = empty + S, *acc_free = acc_full + ACCS, *drain = acc_free + ACCS;
  uint32_t* slot = reinterpret_cast<uint32_t*>(drain + LG_ISSUERS);
  int* special = reinterpret_cast<int*>(slot + 1);
  float* store = reinterpret_cast<float*>(smem + S * stage_bytes + 256);  // a 32 x 32 block per adding warp
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // (a cluster is a pair, and neighbours in the grid)
  const int rank = PAIR ? blockIdx.x & 1 : 0, worker = blockIdx.x >> (PAIR ? 1 : 0);
  const int workers = gridDim.x >> (PAIR ? 1 : 0), row_in_tile = rank * LG_BM;
  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) {
      lg_bar_init(&full[i], 1);
      lg_bar_init(&empty[i], 1);
    }
    for (int i = 0; i < ACCS; ++i) {
      lg_bar_init(&acc_full[i], 1);
      lg_bar_init(&acc_free[i], PAIR ? 2 * LG_EPI_WARPS : LG_EPI_WARPS);
    }
    for (int i = 0; i < LG_ISSUERS; ++i) lg_bar_init(&drain[i], 1);
    *special = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == LG_WARP_MMA) {
    if (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(lg_smem(slot)), "r"(cols)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(lg_smem(slot)), "r"(cols)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  lg_sync<PAIR>();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *slot;
  if (!a.early) pdl_wait();
  pdl_trigger();

  // The loading and the issuing warps work with one thread each.
  if (warp == LG_WARP_TMA) {
    if (lane == 0) {
      int st = 0, filled = 0, dropped = -1;
      uint32_t par = 1;
      bool alive = true;
      for (int u = worker; u < a.units && alive; u += workers) {
        const LgUnit w = lg_unit(a, u, BN);
        for (int k = w.begin; k < w.end; ++k) {
          if (!lg_wait<PAIR>(a, &empty[st], par, LG_ERR_EMPTY)) {
            alive = false;
            break;
          }
          if (filled == 0 && a.drop && blockIdx.x == 0) {  // see mm_debug_tc_fault
            dropped = filled++;
            ++st;
            continue;
          }
          // (in a pair CTA 0's barrier counts the bytes of both)
          if (rank == 0)
            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(lg_smem(&full[st])),
                         "r"(PAIR ? 2 * stage_bytes : stage_bytes)
                         : "memory");
          uint8_t* dst = smem + (uint32_t)st * stage_bytes;
          const uint32_t bar = PAIR ? lg_lead(&full[st]) : lg_smem(&full[st]);
          TA::template load<PAIR>(dst, &ma, bar, w.m0 + row_in_tile, k * LG_BK);
          TB::template load<PAIR>(dst + TA::bytes, &mb, bar, w.n0 + rank * (BN / 2), k * LG_BK);
          ++filled;
          if (++st == S) {
            st = 0;
            par ^= 1u;
          }
        }
      }
      // Nothing may land in shared memory after the CTA has gone: wait for the
      // last fill of every stage (over already unless a wait gave up), in a
      // pair's CTA 1 for the MMAs that have read it, and there for the last
      // arrivals of CTA 0's issuers (CTA 0 waits for its own below).
      for (int i = max(0, filled - S); i < filled; ++i)
        if (i != dropped)
          lg_wait<PAIR>(a, rank == 0 ? &full[i % S] : &empty[i % S], (uint32_t)(i / S) & 1u, LG_ERR_DRAIN);
      if (rank == 1)
        for (int i = 0; i < LG_ISSUERS; ++i) lg_wait<PAIR>(a, &drain[i], 0u, LG_ERR_DRAIN);
    }
    __syncwarp();
  } else if (warp >= LG_WARP_MMA) {
    const int issuer = warp - LG_WARP_MMA;
    if (lane == 0 && rank == 0) {
      constexpr uint32_t idesc = 1u << 4 | 1u << 7 | 1u << 10 | (AMN ? 1u << 15 : 0u) | (BMN ? 1u << 16 : 0u) |
                                 (uint32_t)(BN >> 3) << 17 | (uint32_t)((PAIR ? 2 * LG_BM : LG_BM) >> 4) << 24;
      const uint32_t base = lg_smem(smem);
      int st = 0, buf = 0;
      uint32_t par = 0, bpar = 1;
      bool alive = true;
      for (int u = worker; u < a.units && alive; u += workers) {
        const LgUnit w = lg_unit(a, u, BN);
        for (int k = w.begin; k < w.end; ++k) {
          if (buf % LG_ISSUERS == issuer) {
            if (!lg_wait<PAIR>(a, &acc_free[buf], bpar, LG_ERR_FREE) || !lg_wait<PAIR>(a, &full[st], par, LG_ERR_FULL)) {
              alive = false;
              break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t at = base + (uint32_t)st * stage_bytes, bt = at + TA::bytes;
            const uint32_t d = tmem + (uint32_t)(buf * BN);
            constexpr int pa[6] = {2, 0, 1, 0, 1, 0}, pb[6] = {0, 2, 1, 1, 0, 0};
#pragma unroll
            for (int q = 0; q < 6; ++q)
#pragma unroll
              for (int kk = 0; kk < 2; ++kk)
                lg_mma<PAIR>(d, TA::desc(at, pa[q], kk), TB::desc(bt, pb[q], kk), idesc, q + kk > 0 ? 1u : 0u);
            lg_commit<PAIR>(&empty[st]);
            lg_commit<PAIR>(&acc_full[buf]);
          }
          if (++st == S) {
            st = 0;
            par ^= 1u;
          }
          if (++buf == ACCS) {
            buf = 0;
            bpar ^= 1u;
          }
        }
      }
      // No MMA may still write tensor memory when it is freed.
      lg_commit<PAIR>(&drain[issuer]);
      lg_wait(a, &drain[issuer], 0u, LG_ERR_DRAIN);
    }
    __syncwarp();
  } else {
    const int quarter = warp & 3, half = warp >> 2;
    float* stage = store + warp * 1024;
    const uint32_t base = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(half * HALF);
    int buf = 0;
    uint32_t par = 0;
    bool alive = true;
    int inf = 0;  // read while the first stages are on their way
    for (int i = threadIdx.x; i < a.flags_a; i += LG_EPI_WARPS * 32) inf |= __ldcg(&a.pa.flags[i]);
    for (int i = threadIdx.x; i < a.flags_b; i += LG_EPI_WARPS * 32) inf |= __ldcg(&a.pb.flags[i]);
    if (inf) *special = 1;
    for (int u = worker; u < a.units && alive; u += workers) {
      const LgUnit w = lg_unit(a, u, BN);
      float acc[HALF];
#pragma unroll
      for (int i = 0; i < HALF; ++i) acc[i] = 0.f;
      for (int k = w.begin; k < w.end; ++k) {
        if (!__all_sync(0xffffffffu, lg_wait<PAIR>(a, &acc_full[buf], par, LG_ERR_ACC))) {
          alive = false;
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
        for (int j = 0; j < HALF / 32; ++j) {
          float v[32];
          lg_tmem_load32(base + (uint32_t)(buf * BN + 32 * j), v);
#pragma unroll
          for (int i = 0; i < 32; ++i) acc[32 * j + i] += v[i];
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
          if (PAIR)
            lg_arrive_at(lg_lead(&acc_free[buf]));
          else
            lg_arrive(&acc_free[buf]);
        }
        if (++buf == ACCS) {
          buf = 0;
          par ^= 1u;
        }
      }
      if (!alive) break;
      const int in_tile = row_in_tile + quarter * 32;
      const int64_t row = (int64_t)w.m0 + in_tile + lane;
      const int col = w.n0 + half * HALF;
      if (w.part >= 0) {
        float4* part = reinterpret_cast<float4*>(a.part + ((int64_t)w.part * a.bm + in_tile + lane) * BN + half * HALF);
#pragma unroll
        for (int j = 0; j < HALF / 4; ++j) part[j] = make_float4(acc[4 * j], acc[4 * j + 1], acc[4 * j + 2], acc[4 * j + 3]);
        continue;
      }
      if (a.vec && col + HALF <= a.n) {
        lg_finish_row<HALF>(a, acc, row, col);
        continue;
      }
#pragma unroll
      for (int j = 0; j < HALF / 32; ++j) {
        __syncwarp();  // the last block has been read
#pragma unroll
        for (int i = 0; i < 32; ++i) stage[32 * lane + (i ^ lane)] = acc[32 * j + i];
        __syncwarp();
        const int c = col + 32 * j + lane, row0 = w.m0 + in_tile;
        switch (a.e.act) {
          case MM_LINEAR_RELU: lg_finish_rows<MM_LINEAR_RELU>(a, stage, row0, c, lane); break;
          case MM_LINEAR_SILU: lg_finish_rows<MM_LINEAR_SILU>(a, stage, row0, c, lane); break;
          case MM_LINEAR_SIGMOID: lg_finish_rows<MM_LINEAR_SIGMOID>(a, stage, row0, c, lane); break;
          case MM_LINEAR_GELU: lg_finish_rows<MM_LINEAR_GELU>(a, stage, row0, c, lane); break;
          case MM_LINEAR_GELU_TANH: lg_finish_rows<MM_LINEAR_GELU_TANH>(a, stage, row0, c, lane); break;
          default: lg_finish_rows<MM_LINEAR_NONE>(a, stage, row0, c, lane); break;
        }
      }
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  lg_sync<PAIR>();  // in a pair: both CTAs have waited for all that arrives in their shared memory
  if (warp == LG_WARP_MMA) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (PAIR)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols) : "memory");
    else
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols) : "memory");
  }
  if (*special) {
    for (int u = worker; u < a.units; u += workers) {
      const LgUnit w = lg_unit(a, u, BN);
      if (w.part < 0) lin_fix(a, w.m0 + row_in_tile, LG_BM, w.n0, BN);
    }
  }
  if (a.early) pdl_wait();
}

// Tiles whose reduction was divided: the partial tiles are added in order and
// go through the epilogue, four columns per thread.  One block per 8 rows of a
// tile.
template <int BN>
__global__ void __launch_bounds__(2 * BN) linear_join_kernel(const LinGemm a) {
  if (!a.early) pdl_wait();
  pdl_trigger();
  const int tile = blockIdx.x / (a.bm / 8), r0 = blockIdx.x % (a.bm / 8) * 8;
  const LgUnit w = lg_unit(a, a.full + tile * a.splits, BN);
  const int r = r0 + threadIdx.x / (BN / 4), c = threadIdx.x % (BN / 4) * 4;
  const float* part = a.part + ((int64_t)tile * a.splits * a.bm + r) * BN + c;
  float v[4] = {};
#pragma unroll 4
  for (int s = 0; s < a.splits; ++s) {
    const float4 t = __ldcg(reinterpret_cast<const float4*>(part + (int64_t)s * a.bm * BN));
    v[0] += t.x; v[1] += t.y; v[2] += t.z; v[3] += t.w;
  }
  if (w.m0 + r < a.m && w.n0 + c < a.n) lin_finish_row<4>(a.e, v, a.c, w.m0 + r, w.n0 + c, a.n, a.vec);
  __syncthreads();
  lin_fix(a, w.m0 + r0, 8, w.n0, BN);
  if (a.early) pdl_wait();
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

void lin_debug_fault(int device, int64_t wait_ns, int drop) {
  if (device < 0 || device >= 64) return;
  g_lin_wait_ns[device] = wait_ns > 0 ? wait_ns : 0;
  g_lin_drop[device] = drop;
}

int64_t lin_flag_words(int64_t rows, int64_t cols) {
  return ((rows + SP_ROWS - 1) / SP_ROWS) * ((cols + SP_ROWS - 1) / SP_ROWS);
}

int64_t lin_plane_bytes(int64_t rows, int64_t cols) { return 6 * ((rows + 7) / 8 * 8) * ((cols + 7) / 8 * 8); }

int64_t lin_part_rows(int64_t m) { return (m + SP_ROWS - 1) / SP_ROWS; }

void lin_add_split(LinSplits* all, const LinSplit& s) {
  LinSplit& t = all->s[all->count];
  t = s;
  t.first = (uint32_t)all->blocks;
  t.blocks_c = (s.cols + SP_COLS - 1) / SP_COLS;
  all->blocks += (int64_t)t.blocks_c * ((s.rows + SP_ROWS - 1) / SP_ROWS);
  ++all->count;
}

int lin_run_splits(const LinSplits& all, cudaStream_t s) {
  if (all.blocks > INT32_MAX) return fail(MM_ERR_UNSUPPORTED, "mm_linear: operands too large");
  cudaError_t e = launch_pdl(linear_split_kernel, dim3((unsigned)all.blocks), dim3(256), 0, s, all);
  return e == cudaSuccess ? MM_OK : cuda_fail(e, "mm_linear split launch");
}

// Tiles and division of the reduction, by an estimate in SM clocks.  What bounds
// a stage is shared memory at 128 bytes per clock: each of its twelve MMAs reads
// its operands there and TMA writes them once.  128 x 128: 12 x 8 KB + 48 KB,
// 1,125 clocks (1,150 to 1,250 measured; the MMAs alone 768); 128 x 64: 12 x 6 +
// 36, 844 (880; 384); 256 x 128 of a CTA pair, per CTA: 12 x 6 + 36, 844 (980;
// 768).  Pairs are the best where there is work for all of them (us, without and
// with): 8192 x 2048 x 4096 686 -> 607, 2048 x 2048 x 2048 110 -> 95, gradients of
// 2000 x 1280 x 1000 118 -> 104.  A tile takes about 4,000 more to fill the
// pipeline and store.  Tiles 256 wide of one CTA were slower at every size, as
// they leave only two accumulators and the MMAs wait for the additions; so was
// asking L2 for the stages ahead of their loads.
// Whole waves of tiles run undivided; the rest is divided where that ends
// sooner although its partial tiles are written and read once more.  Sharing
// the rest's stages out evenly, across the tiles' borders, is slower: CTAs that
// share operand tiles are then at different stages and find them in L2 less
// often (forward 1111 x 1502 x 2501: 72 -> 79 us, gradients 156 -> 170).
LinChoice lin_choose(int64_t m, int64_t n, int64_t k) {
  static const struct {
    int bm, bn;
    double stage;
  } kinds[] = {{256, 128, 980}, {128, 128, 1150}, {128, 64, 880}};
  LinChoice best = {};
  for (const auto& kind : kinds) {
    const int workers = kind.bm == 256 ? sm_count() / 2 : sm_count();
    const int64_t tm = (m + kind.bm - 1) / kind.bm, tn = (n + kind.bn - 1) / kind.bn, tiles = tm * tn;
    const int64_t stages = (k + LG_BK - 1) / LG_BK;
    const double tile = 4000;
    const int64_t full = tiles / workers * workers, rest = tiles - full;
    const double base = (double)(full / workers) * (stages * kind.stage + tile);
    for (int s = 1; s <= LIN_MAX_SPLITS; ++s) {
      if (s > 1 && (rest == 0 || s > stages || rest * s > 2 * workers)) break;
      double t = base;
      if (rest) {
        const int64_t waves = (rest * s + workers - 1) / workers;
        t += waves * (((stages + s - 1) / s) * kind.stage + tile);
        if (s > 1) t += 10000 + (double)rest * s * kind.bm * kind.bn * 8 / 3500;  // one more launch, 3,500 bytes per clock
      }
      if (best.bn == 0 || t < best.clocks)
        best = {kind.bm, kind.bn, (int)full, s, (int)tm, (int)tn, (int)stages, (int)(full + rest * s), t};
    }
  }
  return best;
}

int64_t lin_part_bytes(const LinChoice& c) {
  return c.splits > 1 ? (int64_t)(c.units - c.full) * c.bm * c.bn * 4 : 0;
}

// Blocks that linear_split_kernel made of an operand.
static int lin_flag_count(const LinPlanes& p) {
  const int64_t r = p.mn ? p.k : p.lines, c = p.mn ? p.lines : p.k;
  return (int)(((r + SP_ROWS - 1) / SP_ROWS) * ((c + SP_COLS - 1) / SP_COLS));
}

static int lin_map(const LinPlanes& p, int rows, CUtensorMap* out) {
  using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static const EncodeFn encode = [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    const cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q);
    return e == cudaSuccess && q == cudaDriverEntryPointSuccess ? (EncodeFn)fn : nullptr;
  }();
  if (encode == nullptr) return fail(MM_ERR_CUDA, "mm_linear: cuTensorMapEncodeTiled entry point unavailable");
  const cuuint64_t r = (cuuint64_t)(p.mn ? p.k : p.lines), c = (cuuint64_t)(p.mn ? p.lines : p.k);
  const cuuint64_t dims[3] = {c, r, 3}, strides[2] = {(cuuint64_t)p.ld * 2, r * (cuuint64_t)p.ld * 2};
  const cuuint32_t box[3] = {p.mn ? 64u : (cuuint32_t)LG_BK, p.mn ? (cuuint32_t)LG_BK : (cuuint32_t)rows, 3};
  const cuuint32_t ones[3] = {1, 1, 1};
  const CUresult e = encode(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, (void*)p.planes, dims, strides, box, ones,
                            CU_TENSOR_MAP_INTERLEAVE_NONE,
                            p.mn ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (e != CUDA_SUCCESS)
    return fail(MM_ERR_CUDA, "mm_linear: cuTensorMapEncodeTiled failed (CUresult " + std::to_string((int)e) + ")");
  return MM_OK;
}

template <int BN, bool AMN, bool BMN, bool PAIR>
static int lin_launch(const CUtensorMap& ma, const CUtensorMap& mb, const LinGemm& g, cudaStream_t s) {
  // alignment, stages, barriers, 32 x 32 blocks of the adding warps
  constexpr size_t smem =
      1024 + (size_t)lg_stages<BN, PAIR>() * (LG_BM + (PAIR ? BN / 2 : BN)) * 192 + 256 + LG_EPI_WARPS * 4096;
  static_assert(smem <= 227 * 1024, "shared memory of a block");
  auto kernel = linear_gemm_kernel<BN, AMN, BMN, PAIR>;
  MM_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem),
          "mm_linear: shared memory attribute");
  const int size = PAIR ? 2 : 1, workers = sm_count() / size;
  MM_CUDA(launch_pdl_cluster(kernel, dim3((unsigned)(size * (g.units < workers ? g.units : workers))),
                             dim3(LG_THREADS), size, smem, s, ma, mb, g),
          "mm_linear launch");
  return MM_OK;
}

template <int BN, bool PAIR>
static int lin_launch_kind(bool amn, bool bmn, const CUtensorMap& ma, const CUtensorMap& mb, const LinGemm& g,
                           cudaStream_t s) {
  if (amn)
    return bmn ? lin_launch<BN, true, true, PAIR>(ma, mb, g, s) : lin_launch<BN, true, false, PAIR>(ma, mb, g, s);
  return bmn ? lin_launch<BN, false, true, PAIR>(ma, mb, g, s) : lin_launch<BN, false, false, PAIR>(ma, mb, g, s);
}

int lin_run_gemm(const LinPlanes& pa, const LinPlanes& pb, float* c, const LinEpilogue& e, const LinChoice& ch,
                 float* part, bool early, LinGemm* out, cudaStream_t s) {
  LinGemm& g = *out;
  g.m = (int)pa.lines;
  g.n = (int)pb.lines;
  g.bm = ch.bm;
  g.stages = ch.stages;
  g.tiles_m = ch.tiles_m;
  g.tiles_n = ch.tiles_n;
  g.full = ch.full;
  g.splits = ch.splits;
  g.units = ch.units;
  // Whole rows of four columns may move in 16-byte pieces.
  g.vec = g.n % 4 == 0 && (uintptr_t)c % 16 == 0 && (!e.bias || e.bias_vec) && (!e.residual || e.residual_vec) &&
          (!e.z || e.z_vec);
  g.c = c;
  g.part = part;
  g.e = e;
  g.pa = pa;
  g.pb = pb;
  g.flags_a = lin_flag_count(pa);
  g.flags_b = lin_flag_count(pb);
  g.early = early;
  int device = 0;
  cudaGetDevice(&device);
  g.fault = fault_word(device, true);
  if (g.fault == nullptr) return fail(MM_ERR_OOM, "mm_linear: no page-locked memory for the fault word");
  const int64_t limit = device >= 0 && device < 64 ? g_lin_wait_ns[device].load() : 0;
  g.wait_ns = limit > 0 ? limit : LG_WAIT_NS;
  g.drop = device >= 0 && device < 64 ? g_lin_drop[device].load() : 0;
  CUtensorMap ma, mb;
  int rc = lin_map(pa, LG_BM, &ma);
  if (rc == MM_OK) rc = lin_map(pb, ch.bm == 256 ? ch.bn / 2 : ch.bn, &mb);
  if (rc != MM_OK) return rc;
  return ch.bm == 256   ? lin_launch_kind<128, true>(pa.mn, pb.mn, ma, mb, g, s)
         : ch.bn == 128 ? lin_launch_kind<128, false>(pa.mn, pb.mn, ma, mb, g, s)
                        : lin_launch_kind<64, false>(pa.mn, pb.mn, ma, mb, g, s);
}

int lin_run_join(const LinGemm& gemm, const LinChoice& ch, bool early, cudaStream_t s) {
  if (ch.splits == 1) return MM_OK;
  LinGemm g = gemm;
  g.early = early;
  const unsigned grid = (unsigned)((ch.units - ch.full) / ch.splits * (ch.bm / 8));
  MM_CUDA(ch.bn == 128 ? launch_pdl(linear_join_kernel<128>, dim3(grid), dim3(256), 0, s, g)
                       : launch_pdl(linear_join_kernel<64>, dim3(grid), dim3(128), 0, s, g),
          "mm_linear join launch");
  return MM_OK;
}

}  // namespace mm
