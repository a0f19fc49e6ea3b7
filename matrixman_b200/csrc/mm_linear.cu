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
};

constexpr int LS_T = 64, LS_K = 16, LS_PAD = 4;

// 64 x 64 outputs per block, 4 x 4 per thread, 16 of k at a time through
// shared memory.
__global__ void __launch_bounds__(256) linear_simt_kernel(LinProduct p, LinEpilogue e) {
  __shared__ float as[LS_K][LS_T + LS_PAD], bs[LS_K][LS_T + LS_PAD];
  const int m0 = blockIdx.y * LS_T, n0 = blockIdx.x * LS_T;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[4][4] = {};
  // Neighbouring threads load along whichever direction is dense.
  const bool ak = p.as1 <= p.as0, bk = p.bs1 <= p.bs0;
  for (int k0 = 0; k0 < p.k; k0 += LS_K) {
#pragma unroll
    for (int i = 0; i < LS_T * LS_K / 256; ++i) {
      const int at = i * 256 + threadIdx.x;
      const int ar = ak ? at / LS_K : at % LS_T, ac = ak ? at % LS_K : at / LS_T;
      const int br = bk ? at / LS_K : at % LS_T, bc = bk ? at % LS_K : at / LS_T;
      as[ac][ar] = m0 + ar < p.m && k0 + ac < p.k ? p.a[(m0 + ar) * p.as0 + (k0 + ac) * p.as1] : 0.f;
      bs[bc][br] = n0 + br < p.n && k0 + bc < p.k ? p.b[(n0 + br) * p.bs0 + (k0 + bc) * p.bs1] : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < LS_K; ++kk) {
      float av[4], bv[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        av[i] = as[kk][ty * 4 + i];
        bv[i] = bs[kk][tx * 4 + i];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] += av[i] * bv[j];
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = m0 + ty * 4 + i, col = n0 + tx * 4 + j;
      if (row < p.m && col < p.n) p.c[(int64_t)row * p.n + col] = lin_finish(e, acc[i][j], row, col, p.n);
    }
}

// dz = dy act'(z), dense [m, n], and the partial sums of its columns over the
// rows blockIdx.y, + gridDim.y, ...
__global__ void __launch_bounds__(256) linear_dz_kernel(const float* dy, int64_t dys, const float* z, int act, int m,
                                                        int n, float* dz, float* part) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= n) return;
  float s = 0.f;
  for (int64_t row = blockIdx.y; row < m; row += gridDim.y) {
    float g = dy[row * dys + c];
    if (z) g *= lin_slope(z[row * n + c], act);
    dz[row * n + c] = g;
    s += g;
  }
  part[(int64_t)blockIdx.y * n + c] = s;
}

// Adds the partial rows in a fixed order.
__global__ void __launch_bounds__(256) linear_columns_kernel(const float* part, int rows, int n, float* db) {
  __shared__ float acc[8][33];
  const int lane = threadIdx.x & 31, k = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (c < n)
    for (int r = k; r < rows; r += 8) s += part[(int64_t)r * n + c];
  acc[k][lane] = s;
  __syncthreads();
  if (k == 0 && c < n) {
#pragma unroll
    for (int j = 1; j < 8; ++j) s += acc[j][lane];
    db[c] = s;
  }
}

// A strided matrix of the call's arguments.
struct LinMatrix {
  const float* data;
  int64_t s0, s1;
};

static int lin_product(const LinProduct& p, const LinEpilogue& e, cudaStream_t s) {
  if (p.m == 0 || p.n == 0) return MM_OK;
  const dim3 grid((p.n + LS_T - 1) / LS_T, (p.m + LS_T - 1) / LS_T);
  if (grid.y > 65535) return fail(MM_ERR_UNSUPPORTED, "mm_linear: too many rows");
  linear_simt_kernel<<<grid, 256, 0, s>>>(p, e);
  MM_LAUNCH_CHECK("mm_linear launch");
  return MM_OK;
}

constexpr int LIN_DZ_ROWS = 256;  // partial rows of the bias gradient

// Whether a product of this size runs on the tensor cores.
static bool lin_on_tensor_cores(int64_t m, int64_t n, int64_t k) { return m > 32 && k >= 32 && n >= 32; }

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

static int lin_forward_tc(const LinMatrix& x, const LinMatrix& w, int64_t m, int64_t n, int64_t k,
                          const LinEpilogue& e, float* y, void* workspace, cudaStream_t s) {
  LinCarve ws = {(char*)workspace, 0};
  LinSplits all;
  all.count = 0;
  all.blocks = 0;
  bool xt, wt;
  const LinStored xs = lin_store(&ws, &all, x.data, x.s0, x.s1, m, k, &xt);
  const LinStored wst = lin_store(&ws, &all, w.data, w.s0, w.s1, n, k, &wt);
  const LinChoice c = lin_choose(m, n, k);
  float* part = (float*)ws.take(lin_part_bytes(c));
  int rc = lin_run_splits(all, s);
  if (rc != MM_OK) return rc;
  return lin_run_gemm(xt ? xs.by_cols() : xs.by_rows(), wt ? wst.by_cols() : wst.by_rows(), y, e, c, part, s);
}

static int lin_backward_tc(const LinMatrix& dy, const LinMatrix& x, const LinMatrix& w, const float* z, int act,
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
  if (db) {
    linear_columns_kernel<<<(unsigned)((n + 31) / 32), 256, 0, s>>>(gs.part, (int)lin_part_rows(m), (int)n, db);
    MM_LAUNCH_CHECK("mm_linear_backward launch");
  }
  const LinEpilogue none = {nullptr, nullptr, nullptr, 0, MM_LINEAR_NONE, 0};
  if (dx) {
    const LinChoice c = lin_choose(m, k, n);
    float* part = (float*)ws.take(lin_part_bytes(c));
    rc = lin_run_gemm(g.by_rows(), wt ? wst.by_rows() : wst.by_cols(), dx, none, c, part, s);
    if (rc != MM_OK) return rc;
  }
  if (dw) {
    const LinChoice c = lin_choose(n, k, m);
    float* part = (float*)ws.take(lin_part_bytes(c));
    rc = lin_run_gemm(g.by_cols(), xt ? xs.by_rows() : xs.by_cols(), dw, none, c, part, s);
  }
  return rc;
}

static size_t lin_workspace(int64_t m, int64_t n, int64_t k, bool backward) {
  LinCarve ws = {nullptr, 0};
  if (lin_on_tensor_cores(m, n, k)) {
    ws.take(lin_plane_bytes(m, k));
    ws.take(4 * lin_flag_words(m, k));
    ws.take(lin_plane_bytes(n, k));
    ws.take(4 * lin_flag_words(n, k));
    if (!backward) {
      ws.take(lin_part_bytes(lin_choose(m, n, k)));
    } else {
      ws.take(lin_plane_bytes(m, n));
      ws.take(4 * lin_flag_words(m, n));
      ws.take(4 * lin_part_rows(m) * n);
      ws.take(lin_part_bytes(lin_choose(m, k, n)));
      ws.take(lin_part_bytes(lin_choose(n, k, m)));
    }
  } else if (backward) {
    ws.take(4 * m * n);
    ws.take(4 * LIN_DZ_ROWS * n);
  }
  return ws.used;
}

static int lin_check(const char* who, int64_t m, int64_t n, int64_t k, int act, const void* workspace,
                     size_t workspace_bytes, size_t need) {
  const std::string name(who);
  if (m < 0 || n < 0 || k < 0) return fail(MM_ERR_INVALID, name + ": negative size");
  if (m > INT32_MAX / 2 || n > INT32_MAX / 2 || k > INT32_MAX / 2)
    return fail(MM_ERR_UNSUPPORTED, name + ": dimension too large");
  if (act < MM_LINEAR_NONE || act > MM_LINEAR_GELU_TANH) return fail(MM_ERR_INVALID, name + ": unknown activation");
  if (workspace != nullptr && (workspace_bytes < need || (uintptr_t)workspace % 256 != 0))
    return fail(MM_ERR_INVALID, name + ": the workspace is misaligned or too small");
  return MM_OK;
}

}  // namespace mm

using namespace mm;

extern "C" int mm_linear_workspace_size(int64_t m, int64_t n, int64_t k, int backward, size_t* bytes) {
  if (bytes == nullptr || m < 0 || n < 0 || k < 0) return fail(MM_ERR_INVALID, "mm_linear_workspace_size: invalid argument");
  *bytes = lin_workspace(m, n, k, backward != 0);
  return MM_OK;
}

extern "C" int mm_linear(const float* x, int64_t xs0, int64_t xs1, const float* w, int64_t ws0, int64_t ws1,
                         const float* bias, const float* residual, int64_t residual_stride, int64_t m, int64_t n,
                         int64_t k, int act, int residual_before_act, float* y, float* z, void* workspace,
                         size_t workspace_bytes, void* stream) {
  const size_t need = m < 0 || n < 0 || k < 0 ? 0 : lin_workspace(m, n, k, false);
  int rc = lin_check("mm_linear", m, n, k, act, workspace, workspace_bytes, need);
  if (rc != MM_OK) return rc;
  if (xs0 < 0 || xs1 < 0 || ws0 < 0 || ws1 < 0 || residual_stride < 0)
    return fail(MM_ERR_INVALID, "mm_linear: negative stride");
  if (m == 0 || n == 0) return MM_OK;
  if (!y || (k > 0 && (!x || !w))) return fail(MM_ERR_INVALID, "mm_linear: null data pointer");
  cudaStream_t s = resolve_stream(stream);
  const LinEpilogue e = {bias, residual, z, residual_stride, act, residual_before_act != 0};
  if (!lin_on_tensor_cores(m, n, k))
    return lin_product({x, w, y, xs0, xs1, ws0, ws1, (int)m, (int)n, (int)k}, e, s);
  Scratch scratch;
  if (workspace == nullptr) {
    if ((rc = scratch.get(need, s)) != MM_OK) return rc;
    workspace = scratch.data;
  }
  return lin_forward_tc({x, xs0, xs1}, {w, ws0, ws1}, m, n, k, e, y, workspace, s);
}

extern "C" int mm_linear_backward(const float* dy, int64_t dy_stride, const float* x, int64_t xs0, int64_t xs1,
                                  const float* w, int64_t ws0, int64_t ws1, const float* z, int64_t m, int64_t n,
                                  int64_t k, int act, float* dx, float* dw, float* db, float* dz, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  const size_t need = m < 0 || n < 0 || k < 0 ? 0 : lin_workspace(m, n, k, true);
  int rc = lin_check("mm_linear_backward", m, n, k, act, workspace, workspace_bytes, need);
  if (rc != MM_OK) return rc;
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
  if (lin_on_tensor_cores(m, n, k))
    return lin_backward_tc({dy, dy_stride, 1}, {x, xs0, xs1}, {w, ws0, ws1}, z, act, m, n, k, dx, dw, db, dz,
                           workspace, s);
  LinCarve ws = {(char*)workspace, 0};
  float* own = (float*)ws.take(4 * m * n);
  float* part = (float*)ws.take(4 * LIN_DZ_ROWS * n);
  float* g = dz ? dz : own;
  const int rows = m < LIN_DZ_ROWS ? (int)m : LIN_DZ_ROWS;
  linear_dz_kernel<<<dim3((unsigned)((n + 255) / 256), rows), 256, 0, s>>>(
      dy, dy_stride, act == MM_LINEAR_NONE ? nullptr : z, act, (int)m, (int)n, g, part);
  MM_LAUNCH_CHECK("mm_linear_backward launch");
  if (db) {
    linear_columns_kernel<<<(unsigned)((n + 31) / 32), 256, 0, s>>>(part, rows, (int)n, db);
    MM_LAUNCH_CHECK("mm_linear_backward launch");
  }
  const LinEpilogue none = {nullptr, nullptr, nullptr, 0, MM_LINEAR_NONE, 0};
  if (dx) {
    rc = lin_product({g, w, dx, n, 1, ws1, ws0, (int)m, (int)k, (int)n}, none, s);
    if (rc != MM_OK) return rc;
  }
  return dw ? lin_product({g, x, dw, 1, n, xs1, xs0, (int)n, (int)k, (int)m}, none, s) : MM_OK;
}
