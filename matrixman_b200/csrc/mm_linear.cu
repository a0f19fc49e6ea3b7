// y = act(x w^T + b) + r (or act(x w^T + b + r)) and its gradients, float32.
//
//   z = x w^T + b [+ r],  y = act(z) [+ r]
//   dz = dy act'(z),  dx = dz w,  dw = dz^T x,  db = sum over rows of dz
//
// x [m, k], w [n, k], r and y [m, n].
#include <cuda_runtime.h>
#include <stdint.h>

#include <string>

#include "mm_linear_tc.cuh"

namespace mm {

// C[m, n] = sum over k of A[m, k] B[n, k], any strides; C dense.
struct LinProduct {
  const float *a, *b;
  float* c;
  int64_t as0, as1, bs0, bs1;
  int m, n, k;
  // A's values times act'(z), z strided like A (null: as they are)
  const float* z;
  int64_t zs0, zs1;
  int act;
};

// ---------------------------------------------------------------------------
// Small products: 32 x 32 outputs per block, the reduction in chunks of eight
// per warp (64 or 128), whose sums are added in order at the end.  A lane holds
// 4 x 8 outputs and reads its lines of A and B in 16-byte pieces along the
// reduction: 12 such reads feed 128 multiply-adds.  Used where a product is so
// small that latency bounds it: many blocks with a short walk each, one launch,
// no workspace.  Sixteen warps where a block has an SM to itself anyway.
// ---------------------------------------------------------------------------

constexpr int LS_T = 32;

template <int NW>
struct LsShape {
  static constexpr int K = 8 * NW, ROW = K + 4;  // + 4: 16-byte reads of neighbouring lines hit other banks
  static constexpr int TILE = LS_T * ROW;
  // two buffers of A's and B's tile; at the end the warps' sums [NW][32][33]
  static constexpr int FLOATS = 4 * TILE > NW * LS_T * 33 ? 4 * TILE : NW * LS_T * 33;
};

// How an operand's tile is read: 16 bytes along the reduction, along the lines,
// or value by value.
enum { LS_ALONG_K = 0, LS_ALONG_LINES = 1, LS_SINGLE = 2 };

// The eight values of a 32 x K tile that a thread brings in.
template <int NW>
__device__ __forceinline__ void ls_fetch(const float* p, int64_t s0, int64_t s1, int lines, int k, int l0, int k0,
                                         int mode, float (&v)[8]) {
  constexpr int KQ = 2 * NW;  // 16-byte pieces along the reduction
  const int t = threadIdx.x;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int line = mode == LS_ALONG_LINES ? (t & 7) * 4 : i * 16 + t / KQ;
    const int kk = mode == LS_ALONG_LINES ? i * 4 * NW + (t >> 3) : t % KQ * 4;
    const int l = l0 + line, kg = k0 + kk;
    if (mode == LS_ALONG_K && l < lines && kg + 4 <= k) {
      const float4 q = *reinterpret_cast<const float4*>(p + l * s0 + kg);
      v[4 * i] = q.x; v[4 * i + 1] = q.y; v[4 * i + 2] = q.z; v[4 * i + 3] = q.w;
    } else if (mode == LS_ALONG_LINES && l + 4 <= lines && kg < k) {
      const float4 q = *reinterpret_cast<const float4*>(p + kg * s1 + l);
      v[4 * i] = q.x; v[4 * i + 1] = q.y; v[4 * i + 2] = q.z; v[4 * i + 3] = q.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int le = mode == LS_ALONG_LINES ? l + e : l, ke = mode == LS_ALONG_LINES ? kg : kg + e;
        v[4 * i + e] = le < lines && ke < k ? p[le * s0 + ke * s1] : 0.f;
      }
    }
  }
}

template <int NW>
__device__ __forceinline__ void ls_put(float* tile, int mode, const float (&v)[8]) {
  constexpr int KQ = 2 * NW, ROW = LsShape<NW>::ROW;
  const int t = threadIdx.x;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (mode == LS_ALONG_LINES) {
#pragma unroll
      for (int e = 0; e < 4; ++e) tile[((t & 7) * 4 + e) * ROW + i * 4 * NW + (t >> 3)] = v[4 * i + e];
    } else {
      *reinterpret_cast<float4*>(tile + (i * 16 + t / KQ) * ROW + t % KQ * 4) =
          make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    }
  }
}

// How a small product reads and writes.
struct LsModes {
  int tiles_n, a, b, z, vec;
};

// One 32 x 32 tile of a product.
template <int NW, bool SLOPE>
__device__ __forceinline__ void ls_tile(const LinProduct& p, const LinEpilogue& e, const LsModes& md, int tile) {
  using S = LsShape<NW>;
  extern __shared__ float4 ls_mem[];
  float* tiles = reinterpret_cast<float*>(ls_mem);
  const int m0 = tile / md.tiles_n * LS_T, n0 = tile % md.tiles_n * LS_T;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ga = lane >> 2, gb = lane & 3;  // A lines 4 ga + i, B lines gb + 4 j
  float acc[4][8] = {};
  float av[2][8], bv[2][8], zv[2][8];  // the next two chunks, on their way
  auto fetch = [&](int i, int k0) {
    ls_fetch<NW>(p.a, p.as0, p.as1, p.m, p.k, m0, k0, md.a, av[i]);
    // (z in A's own order: the threads' values have to match)
    if (SLOPE) ls_fetch<NW>(p.z, p.zs0, p.zs1, p.m, p.k, m0, k0, md.z, zv[i]);
    ls_fetch<NW>(p.b, p.bs0, p.bs1, p.n, p.k, n0, k0, md.b, bv[i]);
  };
#pragma unroll
  for (int i = 0; i < 2; ++i) fetch(i, i * S::K);
  for (int k0 = 0; k0 < p.k; k0 += 2 * S::K) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (k0 + i * S::K >= p.k) break;
      float* ta = tiles + i * 2 * S::TILE;
      float* tb = ta + S::TILE;
      if (SLOPE) lin_times_slope<8>(av[i], zv[i], p.act);
      ls_put<NW>(ta, md.a, av[i]);
      ls_put<NW>(tb, md.b, bv[i]);
      __syncthreads();  // also: every warp has finished with this buffer's last chunk
      if (k0 + (i + 2) * S::K < p.k) fetch(i, k0 + (i + 2) * S::K);
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int kk = warp * 8 + q * 4;
        float4 a[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) a[x] = *reinterpret_cast<const float4*>(ta + (ga * 4 + x) * S::ROW + kk);
#pragma unroll
        for (int y = 0; y < 8; ++y) {
          const float4 b = *reinterpret_cast<const float4*>(tb + (gb + 4 * y) * S::ROW + kk);
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            acc[x][y] += a[x].x * b.x;
            acc[x][y] += a[x].y * b.y;
            acc[x][y] += a[x].z * b.z;
            acc[x][y] += a[x].w * b.w;
          }
        }
      }
    }
  }
  __syncthreads();
  float* red = tiles;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) red[(warp * LS_T + ga * 4 + i) * 33 + gb + 4 * j] = acc[i][j];
  __syncthreads();
  const int r = threadIdx.x >> 3, c = (threadIdx.x & 7) * 4;
  const int row = m0 + r, col = n0 + c;
  if (r >= LS_T || row >= p.m || col >= p.n) return;
  float v[4] = {};
#pragma unroll
  for (int w = 0; w < NW; ++w)
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] += red[(w * LS_T + r) * 33 + c + j];
  lin_finish_row<4>(e, v, p.c, row, col, p.n, md.vec);
}

template <int NW>
__global__ void __launch_bounds__(NW * 32) linear_small_kernel(LinProduct p, LinEpilogue e, LsModes md) {
  pdl_wait();
  ls_tile<NW, false>(p, e, md, blockIdx.x);
}

// All gradients of a small call in one launch: the tiles of dx, then those of
// dw, then the columns of db (and dz itself where it is asked for), 32 to a
// block.  Each block takes dz = dy act'(z) from dy and z as it reads them.
struct LsBackward {
  LinProduct dx, dw;
  LsModes mx, mw;
  LinEpilogue none;
  int tiles_dx, tiles_dw;
  float *db, *dz;
};

__global__ void __launch_bounds__(256) linear_small_backward_kernel(const __grid_constant__ LsBackward g) {
  pdl_wait();
  int block = blockIdx.x;
  const bool slope = g.dw.z != nullptr;
  if (block < g.tiles_dx) {
    if (slope)
      ls_tile<8, true>(g.dx, g.none, g.mx, block);
    else
      ls_tile<8, false>(g.dx, g.none, g.mx, block);
    return;
  }
  block -= g.tiles_dx;
  if (block < g.tiles_dw) {
    if (slope)
      ls_tile<8, true>(g.dw, g.none, g.mw, block);
    else
      ls_tile<8, false>(g.dw, g.none, g.mw, block);
    return;
  }
  block -= g.tiles_dw;
  // dw's A is dz transposed: its lines are dz's columns.
  extern __shared__ float4 ls_mem[];
  float* acc = reinterpret_cast<float*>(ls_mem);  // [8][33]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = block * 32 + lane, n = g.dw.m, m = g.dw.k;
  float s = 0.f;
  if (c < n) {
#pragma unroll 4
    for (int r = warp; r < m; r += 8) {
      float v[1] = {g.dw.a[c * g.dw.as0 + r * g.dw.as1]};
      if (slope) {
        const float z[1] = {g.dw.z[c * g.dw.zs0 + r * g.dw.zs1]};
        lin_times_slope<1>(v, z, g.dw.act);
      }
      if (g.dz) g.dz[(int64_t)r * n + c] = v[0];
      s += v[0];
    }
  }
  acc[warp * 33 + lane] = s;
  __syncthreads();
  if (g.db && warp == 0 && c < n) {
#pragma unroll
    for (int j = 1; j < 8; ++j) s += acc[j * 33 + lane];
    g.db[c] = s;
  }
}

template <int NW>
static cudaError_t lin_small(const LinProduct& p, const LinEpilogue& e, int64_t tiles, const LsModes& md,
                             cudaStream_t s) {
  constexpr size_t smem = LsShape<NW>::FLOATS * sizeof(float);
  if (smem > 48 * 1024) {
    const cudaError_t err =
        cudaFuncSetAttribute(linear_small_kernel<NW>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (err != cudaSuccess) return err;
  }
  return launch_pdl(linear_small_kernel<NW>, dim3((unsigned)tiles), dim3(NW * 32), smem, s, p, e, md);
}

// ---------------------------------------------------------------------------
// A few rows (tokens) times a weight with dense rows: bound by reading the
// weight once.  A group of KW warps computes up to CN columns for MT rows, each
// warp every KW-th piece of the reduction, 32 lanes x VEC values at a time.  BLOCKS
// per SM and UNROLL keep some 64 to 128 KB of the weight on their way per SM; more
// registers for more loads per warp cost blocks, and one more wave costs more (us,
// weight from HBM, 4096 x 4096: 1 row 13.9, floor 10.3; 2 rows 14.2; 4 rows 15.4; 8
// rows 19.9; 16 rows, the weight once more from L2, 31.3.  Four columns always and
// no rule for even waves: 14.9, 16.6, 20.2, 31.8, 47.8).
// ---------------------------------------------------------------------------

template <int MT, int CN, int BLOCKS, int UNROLL, int VEC>
__global__ void __launch_bounds__(256, BLOCKS) linear_tokens_kernel(LinProduct p, LinEpilogue e, int kw, int cols) {
  __shared__ float red[8][MT * CN];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int part = warp % kw;
  const int n0 = (int)(blockIdx.x * (8 / kw) + warp / kw) * cols, count = min(cols, p.n - n0);
  const int m0 = blockIdx.y * MT;
  float acc[MT][CN] = {};
  pdl_wait();
  const float* wp = p.b + (int64_t)n0 * p.bs0;
  const float* xp[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) xp[i] = p.a + (int64_t)min(m0 + i, p.m - 1) * p.as0;
  const int step = 32 * VEC * kw;
#pragma unroll UNROLL
  for (int k = (part * 32 + lane) * VEC; k < p.k; k += step) {
    float w[CN][VEC] = {}, x[MT][VEC];
    const float* at = wp + k;
#pragma unroll
    for (int j = 0; j < CN; ++j, at += p.bs0) {
      if (j >= count) {
        if (MT == 1) break;
        continue;
      }
      if (VEC == 4) {
        const float4 t = __ldcs(reinterpret_cast<const float4*>(at));
        w[j][0] = t.x; w[j][VEC > 1 ? 1 : 0] = t.y; w[j][VEC > 2 ? 2 : 0] = t.z; w[j][VEC > 3 ? 3 : 0] = t.w;
      } else {
        w[j][0] = __ldcs(at);
      }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      if (VEC == 4) {
        const float4 t = *reinterpret_cast<const float4*>(xp[i] + k);
        x[i][0] = t.x; x[i][VEC > 1 ? 1 : 0] = t.y; x[i][VEC > 2 ? 2 : 0] = t.z; x[i][VEC > 3 ? 3 : 0] = t.w;
      } else {
        x[i][0] = xp[i][k];
      }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < CN; ++j)
#pragma unroll
        for (int v = 0; v < VEC; ++v) acc[i][j] += x[i][v] * w[j][v];
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < CN; ++j) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) acc[i][j] += __shfl_xor_sync(0xffffffffu, acc[i][j], o);
      if (lane == 0) red[warp][i * CN + j] = acc[i][j];
    }
  __syncthreads();
  // One thread per output of the block: (8 / kw) groups x MT x CN.
  for (int t = threadIdx.x; t < 8 / kw * MT * CN; t += 256) {
    const int g = t / (MT * CN), o = t % (MT * CN);
    const int row = m0 + o / CN, col = (int)(blockIdx.x * (8 / kw) + g) * cols + o % CN;
    if (row >= p.m || col >= p.n || o % CN >= cols) continue;
    float v = 0.f;
    for (int q = 0; q < kw; ++q) v += red[g * kw + q][o];
    p.c[(int64_t)row * p.n + col] = lin_finish(e, v, row, col, p.n);
  }
}

// Adds the partial rows in a fixed order.
__global__ void __launch_bounds__(256) linear_columns_kernel(const float* part, int rows, int n, float* db,
                                                               int early) {
  if (!early) pdl_wait();
  __shared__ float acc[8][33];
  const int lane = threadIdx.x & 31, k = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (c < n)
    for (int r = k; r < rows; r += 8) s += __ldcg(&part[(int64_t)r * n + c]);
  acc[k][lane] = s;
  __syncthreads();
  if (k == 0 && c < n) {
#pragma unroll
    for (int j = 1; j < 8; ++j) s += acc[j][lane];
    db[c] = s;
  }
  if (early) pdl_wait();
}

// A strided matrix of the call's arguments.
struct LinMatrix {
  const float* data;
  int64_t s0, s1;
};

constexpr int LIN_TOKENS = 16;  // rows up to which a product is a walk over the weight

static bool lin_aligned(const float* p, int64_t stride) { return (uintptr_t)p % 16 == 0 && stride % 4 == 0; }

template <int MT, int CN, int BLOCKS, int UNROLL>
static void lin_tokens(const LinProduct& p, const LinEpilogue& e, cudaStream_t s) {
  // Warps per column group and columns per group: waves of blocks times a
  // block's steps (a piece of each column and, from L1, of each row of A) and its
  // start and end (about four steps).
  const bool wide = lin_aligned(p.a, p.m > 1 ? p.as0 : 0) && lin_aligned(p.b, p.n > 1 ? p.bs0 : 0) && p.k % 4 == 0;
  const int64_t rows = (p.m + MT - 1) / MT, slots = (int64_t)sm_count() * BLOCKS, piece = wide ? 128 : 32;
  int kw = 1, cols = 1;
  double best = 0;
  for (int w = 1; w <= 8 && (w == 1 || p.k > (w / 2) * piece); w *= 2)
    for (int c = 1; c <= CN; ++c) {
      const int64_t blocks = (p.n + 8 / w * c - 1) / (8 / w * c) * rows;
      const double t = (double)((blocks + slots - 1) / slots) *
                       ((double)((p.k + w * piece - 1) / (w * piece)) * (c + 0.25 * MT) + 4);
      if (best == 0 || t < best) {
        best = t;
        kw = w;
        cols = c;
      }
    }
  const int per = 8 / kw * cols;
  const dim3 grid((unsigned)((p.n + per - 1) / per), (unsigned)((p.m + MT - 1) / MT));
  if (wide)
    launch_pdl(linear_tokens_kernel<MT, CN, BLOCKS, UNROLL, 4>, grid, dim3(256), 0, s, p, e, kw, cols);
  else
    launch_pdl(linear_tokens_kernel<MT, CN, BLOCKS, UNROLL, 1>, grid, dim3(256), 0, s, p, e, kw, cols);
}

static int ls_mode(const float* p, int64_t s0, int64_t s1) {
  if (s1 == 1 && lin_aligned(p, s0)) return LS_ALONG_K;
  if (s0 == 1 && lin_aligned(p, s1)) return LS_ALONG_LINES;
  return LS_SINGLE;
}

// The modes of a small product, and its number of tiles.
static int64_t ls_modes(const LinProduct& p, LsModes* md) {
  md->tiles_n = (p.n + LS_T - 1) / LS_T;
  md->a = ls_mode(p.a, p.as0, p.as1);
  md->b = ls_mode(p.b, p.bs0, p.bs1);
  md->z = LS_SINGLE;
  if (p.z) {  // read in A's order, so in A's mode where z allows it
    md->z = ls_mode(p.z, p.zs0, p.zs1);
    if (md->z != md->a) md->a = md->z = LS_SINGLE;
  }
  md->vec = p.n % 4 == 0 && (uintptr_t)p.c % 16 == 0;
  return (int64_t)md->tiles_n * ((p.m + LS_T - 1) / LS_T);
}

// A product on the multiply-add units.
static int lin_product(const LinProduct& p, const LinEpilogue& e, cudaStream_t s) {
  if (p.m == 0 || p.n == 0) return MM_OK;
  if (p.m <= LIN_TOKENS && p.as1 == 1 && p.bs1 == 1 && p.k > 0) {
    if (p.m == 1)
      lin_tokens<1, 8, 4, 1>(p, e, s);
    else if (p.m == 2)
      lin_tokens<2, 4, 4, 1>(p, e, s);
    else if (p.m <= 4)
      lin_tokens<4, 8, 2, 1>(p, e, s);
    else
      lin_tokens<8, 4, 2, 2>(p, e, s);
  } else {
    LsModes md;
    const int64_t tiles = ls_modes(p, &md);
    if (tiles > INT32_MAX) return fail(MM_ERR_UNSUPPORTED, "mm_linear: output too large");
    MM_CUDA(tiles <= sm_count() && p.k > 256 ? lin_small<16>(p, e, tiles, md, s) : lin_small<8>(p, e, tiles, md, s),
            "mm_linear launch");
  }
  MM_LAUNCH_CHECK("mm_linear launch");
  return MM_OK;
}

// Clocks of a small product: a block per SM at a time, 64 of the reduction in
// about 1,700 (with one block per SM latency, with several the multiply-adds
// and their operands from shared memory), 3,500 to start and end, and 3,000
// once.  Measured: 128 x 1024 x 1024 18 us, 512 x 512 x 512 19 us, 64 x 4096 x
// 4096 112 us (a call that runs on the tensor cores, in 81).
static double lin_small_clocks(int64_t m, int64_t n, int64_t k) {
  const int64_t tiles = ((m + LS_T - 1) / LS_T) * ((n + LS_T - 1) / LS_T);
  const int64_t waves = (tiles + sm_count() - 1) / sm_count();
  return 3000.0 + waves * (3500.0 + 1700.0 * ((k + 63) / 64));
}

// How a call runs: on the tensor cores where the estimate of its products, with
// 10 bytes per value to split the operands (about 3,400 bytes per clock) and
// 24,000 clocks for the launches this takes (34,000 in the backward pass), is
// below the small kernels'.  Measured on both sides: 128 x 1024 x 1024 25 us
// against the small kernel's 18, 256 x 1024 x 1024 26 against 32, 8192 x 256 x
// 256 24 against 68.
// `first` is the forward product or dx, `second` dw.
struct LinRoute {
  bool tensor;
  LinChoice first, second;
};

static LinRoute lin_route(int64_t m, int64_t n, int64_t k, bool backward) {
  LinRoute r = {};
  if ((m <= LIN_TOKENS && !backward) || m <= 0 || n <= 0 || k <= 0) return r;
  double small, tensor = backward ? 34000 : 24000;
  if (backward) {
    // (each tile takes the slope of the dz it reads: some 60 operations per value)
    small = lin_small_clocks(m, k, n) + lin_small_clocks(n, k, m) + 60.0 * m * n * (k / 16 + 2) / (sm_count() * 128);
    r.first = lin_choose(m, k, n);
    r.second = lin_choose(n, k, m);
    tensor += r.first.clocks + r.second.clocks + 10.0 * (m * n + m * k + n * k) / 3400;
  } else {
    small = lin_small_clocks(m, n, k);
    r.first = lin_choose(m, n, k);
    tensor += r.first.clocks + 10.0 * (m * k + n * k) / 3400;
  }
  r.tensor = tensor < small;
  return r;
}

// Workspace pieces, 256-byte aligned.
struct LinCarve {
  char* base;
  size_t used;
  void* take(int64_t bytes) {
    void* p = base ? base + used : nullptr;
    used += ((size_t)bytes + 255) & ~(size_t)255;
    return p;
  }
};

// A matrix in planes.
struct LinStored {
  uint16_t* planes;
  int* flags;
  int64_t rows, cols, ld;
  // As a product's operand whose lines run along the stored rows, or columns.
  LinPlanes by_rows() const { return {planes, flags, rows, cols, ld, 0}; }
  LinPlanes by_cols() const { return {planes, flags, cols, rows, ld, 1}; }
};

// Adds the split of a [r, c] matrix to the list, stored along whichever
// direction is dense; *turned says that it is stored transposed.
static LinStored lin_store(LinCarve* ws, LinSplits* all, const float* src, int64_t s0, int64_t s1, int64_t r, int64_t c,
                           bool* turned) {
  *turned = s1 != 1 && c > 1 && (s0 == 1 || r == 1);
  if (*turned) {
    int64_t t = r; r = c; c = t;
    t = s0; s0 = s1; s1 = t;
  }
  LinStored st;
  st.rows = r;
  st.cols = c;
  st.ld = (c + 7) / 8 * 8;
  st.planes = (uint16_t*)ws->take(lin_plane_bytes(r, c));
  st.flags = (int*)ws->take(4 * lin_flag_words(r, c));
  if (c == 1) s1 = 1;
  LinSplit s = {src, s0, s1, nullptr, 0, 0, r, (int)c, st.ld, st.planes, st.flags, nullptr, nullptr, 0, 0};
  s.vec = s1 == 1 && s0 % 4 == 0 && (uintptr_t)src % 16 == 0;
  lin_add_split(all, s);
  return st;
}

static int lin_forward_tc(const LinRoute& r, const LinMatrix& x, const LinMatrix& w, int64_t m, int64_t n, int64_t k,
                          const LinEpilogue& e, float* y, void* workspace, cudaStream_t s) {
  LinCarve ws = {(char*)workspace, 0};
  LinSplits all;
  all.count = 0;
  all.blocks = 0;
  bool xt, wt;
  const LinStored xs = lin_store(&ws, &all, x.data, x.s0, x.s1, m, k, &xt);
  const LinStored wst = lin_store(&ws, &all, w.data, w.s0, w.s1, n, k, &wt);
  float* part = (float*)ws.take(lin_part_bytes(r.first));
  int rc = lin_run_splits(all, s);
  if (rc != MM_OK) return rc;
  LinGemm g;
  rc = lin_run_gemm(xt ? xs.by_cols() : xs.by_rows(), wt ? wst.by_cols() : wst.by_rows(), y, e, r.first, part, false,
                    &g, s);
  return rc == MM_OK ? lin_run_join(g, r.first, false, s) : rc;
}

static int lin_backward_tc(const LinRoute& r, const LinMatrix& dy, const LinMatrix& x, const LinMatrix& w, const float* z, int act,
                           int64_t m, int64_t n, int64_t k, float* dx, float* dw, float* db, float* dz,
                           void* workspace, cudaStream_t s) {
  LinCarve ws = {(char*)workspace, 0};
  LinSplits all;
  all.count = 0;
  all.blocks = 0;
  bool gt, xt = false, wt = false;
  const LinStored g = lin_store(&ws, &all, dy.data, dy.s0, 1, m, n, &gt);
  LinSplit& gs = all.s[0];
  if (act != MM_LINEAR_NONE) {
    gs.z = z;
    gs.act = act;
    gs.vec = gs.vec && n % 4 == 0 && (uintptr_t)z % 16 == 0;
  }
  gs.out = dz;
  if (db) gs.part = (float*)ws.take(4 * lin_part_rows(m) * n);
  LinStored wst = {}, xs = {};
  if (dx) wst = lin_store(&ws, &all, w.data, w.s0, w.s1, n, k, &wt);
  if (dw) xs = lin_store(&ws, &all, x.data, x.s0, x.s1, m, k, &xt);
  int rc = lin_run_splits(all, s);
  if (rc != MM_OK) return rc;
  // The kernels behind the split do not need one another's results, but for the
  // sums of divided tiles.  One that is `early` starts as the blocks of the
  // kernel before it leave, and waits for that kernel's end before its own: so a
  // kernel's end still means that all before it have ended.  What it reads is
  // there: the kernel before it let it start only when its own wait for the
  // split was over (or was itself let start by one that had waited), and is read
  // from L2.  All gradients, us, one after another and so: 2000 x 1280 x 1000 105 ->
  // 98, 1111 x 1502 x 2501 150 -> 137, 5000 x 512 x 777 101 -> 93.
  const LinEpilogue none = lin_epilogue(nullptr, nullptr, 0, nullptr, MM_LINEAR_NONE, false);
  LinGemm gx, gw;
  float* part_x = dx ? (float*)ws.take(lin_part_bytes(r.first)) : nullptr;
  float* part_w = dw ? (float*)ws.take(lin_part_bytes(r.second)) : nullptr;
  if (dx) rc = lin_run_gemm(g.by_rows(), wt ? wst.by_rows() : wst.by_cols(), dx, none, r.first, part_x, false, &gx, s);
  if (rc == MM_OK && dw)
    rc = lin_run_gemm(g.by_cols(), xt ? xs.by_rows() : xs.by_cols(), dw, none, r.second, part_w, dx != nullptr, &gw, s);
  if (rc == MM_OK && dx) rc = lin_run_join(gx, r.first, false, s);
  if (rc == MM_OK && dw) rc = lin_run_join(gw, r.second, dx && r.first.splits > 1, s);
  if (rc == MM_OK && db)
    MM_CUDA(launch_pdl(linear_columns_kernel, dim3((unsigned)((n + 31) / 32)), dim3(256), 0, s, (const float*)gs.part,
                       (int)lin_part_rows(m), (int)n, db, (int)(dx || dw)),
            "mm_linear_backward launch");
  return rc;
}

static size_t lin_workspace(const LinRoute& r, int64_t m, int64_t n, int64_t k, bool backward) {
  LinCarve ws = {nullptr, 0};
  if (r.tensor) {
    ws.take(lin_plane_bytes(m, k));
    ws.take(4 * lin_flag_words(m, k));
    ws.take(lin_plane_bytes(n, k));
    ws.take(4 * lin_flag_words(n, k));
    if (!backward) {
      ws.take(lin_part_bytes(r.first));
    } else {
      ws.take(lin_plane_bytes(m, n));
      ws.take(4 * lin_flag_words(m, n));
      ws.take(4 * lin_part_rows(m) * n);
      ws.take(lin_part_bytes(r.first));
      ws.take(lin_part_bytes(r.second));
    }
  }
  return ws.used;
}

// Before anything is computed from them.
static int lin_check_sizes(const char* who, int64_t m, int64_t n, int64_t k) {
  if (m < 0 || n < 0 || k < 0) return fail(MM_ERR_INVALID, std::string(who) + ": negative size");
  if (m > INT32_MAX / 2 || n > INT32_MAX / 2 || k > INT32_MAX / 2)
    return fail(MM_ERR_UNSUPPORTED, std::string(who) + ": dimension too large");
  return MM_OK;
}

static int lin_check(const char* who, int act, const void* workspace, size_t workspace_bytes, size_t need) {
  const std::string name(who);
  if (act < MM_LINEAR_NONE || act > MM_LINEAR_GELU_TANH) return fail(MM_ERR_INVALID, name + ": unknown activation");
  if (workspace != nullptr && (workspace_bytes < need || (uintptr_t)workspace % 256 != 0))
    return fail(MM_ERR_INVALID, name + ": the workspace is misaligned or too small");
  return MM_OK;
}

}  // namespace mm

using namespace mm;

extern "C" int mm_linear_workspace_size(int64_t m, int64_t n, int64_t k, int backward, size_t* bytes) {
  if (bytes == nullptr) return fail(MM_ERR_INVALID, "mm_linear_workspace_size: null output");
  if (const int rc = lin_check_sizes("mm_linear_workspace_size", m, n, k)) return rc;
  *bytes = lin_workspace(lin_route(m, n, k, backward != 0), m, n, k, backward != 0);
  return MM_OK;
}

extern "C" int mm_linear(const float* x, int64_t xs0, int64_t xs1, const float* w, int64_t ws0, int64_t ws1,
                         const float* bias, const float* residual, int64_t residual_stride, int64_t m, int64_t n,
                         int64_t k, int act, int residual_before_act, float* y, float* z, void* workspace,
                         size_t workspace_bytes, void* stream) {
  int rc = lin_check_sizes("mm_linear", m, n, k);
  if (rc != MM_OK) return rc;
  const LinRoute route = lin_route(m, n, k, false);
  const size_t need = lin_workspace(route, m, n, k, false);
  if ((rc = lin_check("mm_linear", act, workspace, workspace_bytes, need)) != MM_OK) return rc;
  if (xs0 < 0 || xs1 < 0 || ws0 < 0 || ws1 < 0 || residual_stride < 0)
    return fail(MM_ERR_INVALID, "mm_linear: negative stride");
  if (m == 0 || n == 0) return MM_OK;
  if (!y || (k > 0 && (!x || !w))) return fail(MM_ERR_INVALID, "mm_linear: null data pointer");
  cudaStream_t s = resolve_stream(stream);
  const LinEpilogue e = lin_epilogue(bias, residual, residual_stride, z, act, residual_before_act != 0);
  if (!route.tensor)
    return lin_product({x, w, y, xs0, xs1, ws0, ws1, (int)m, (int)n, (int)k, nullptr, 0, 0, MM_LINEAR_NONE}, e, s);
  Scratch scratch;
  if (workspace == nullptr) {
    if ((rc = scratch.get(need, s)) != MM_OK) return rc;
    workspace = scratch.data;
  }
  return lin_forward_tc(route, {x, xs0, xs1}, {w, ws0, ws1}, m, n, k, e, y, workspace, s);
}

extern "C" int mm_linear_backward(const float* dy, int64_t dy_stride, const float* x, int64_t xs0, int64_t xs1,
                                  const float* w, int64_t ws0, int64_t ws1, const float* z, int64_t m, int64_t n,
                                  int64_t k, int act, float* dx, float* dw, float* db, float* dz, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  int rc = lin_check_sizes("mm_linear_backward", m, n, k);
  if (rc != MM_OK) return rc;
  const LinRoute route = lin_route(m, n, k, true);
  const size_t need = lin_workspace(route, m, n, k, true);
  if ((rc = lin_check("mm_linear_backward", act, workspace, workspace_bytes, need)) != MM_OK) return rc;
  if (dy_stride < 0 || xs0 < 0 || xs1 < 0 || ws0 < 0 || ws1 < 0)
    return fail(MM_ERR_INVALID, "mm_linear_backward: negative stride");
  if (!dx && !dw && !db && !dz) return MM_OK;
  if (m > 0 && n > 0 && (!dy || (act != MM_LINEAR_NONE && !z) || (k > 0 && ((dx && !w) || (dw && !x)))))
    return fail(MM_ERR_INVALID, "mm_linear_backward: null data pointer");
  cudaStream_t s = resolve_stream(stream);
  if (m == 0 || n == 0) {
    if (dx && m * k > 0) MM_CUDA(cudaMemsetAsync(dx, 0, (size_t)(m * k) * 4, s), "mm_linear_backward: zero");
    if (dw && n * k > 0) MM_CUDA(cudaMemsetAsync(dw, 0, (size_t)(n * k) * 4, s), "mm_linear_backward: zero");
    if (db && n > 0) MM_CUDA(cudaMemsetAsync(db, 0, (size_t)n * 4, s), "mm_linear_backward: zero");
    return MM_OK;
  }
  Scratch scratch;
  if (workspace == nullptr && need > 0) {
    if ((rc = scratch.get(need, s)) != MM_OK) return rc;
    workspace = scratch.data;
  }
  if (route.tensor)
    return lin_backward_tc(route, {dy, dy_stride, 1}, {x, xs0, xs1}, {w, ws0, ws1}, z, act, m, n, k, dx, dw, db, dz,
                           workspace, s);
  LsBackward g = {};
  const float* zp = act == MM_LINEAR_NONE ? nullptr : z;
  g.none = lin_epilogue(nullptr, nullptr, 0, nullptr, MM_LINEAR_NONE, false);
  g.dx = {dy, w, dx, dy_stride, 1, ws1, ws0, (int)m, (int)k, (int)n, zp, n, 1, act};
  g.dw = {dy, x, dw, 1, dy_stride, xs1, xs0, (int)n, (int)k, (int)m, zp, 1, n, act};
  const int64_t tx = ls_modes(g.dx, &g.mx), tw = ls_modes(g.dw, &g.mw);
  g.tiles_dx = dx ? (int)tx : 0;
  g.tiles_dw = dw ? (int)tw : 0;
  g.db = db;
  g.dz = dz;
  const int64_t blocks = (dx ? tx : 0) + (dw ? tw : 0) + (db || dz ? (n + 31) / 32 : 0);
  if (blocks > INT32_MAX) return fail(MM_ERR_UNSUPPORTED, "mm_linear_backward: output too large");
  if (blocks == 0) return MM_OK;
  MM_CUDA(launch_pdl(linear_small_backward_kernel, dim3((unsigned)blocks), dim3(256),
                     LsShape<8>::FLOATS * sizeof(float), s, g),
          "mm_linear_backward launch");
  return MM_OK;
}
