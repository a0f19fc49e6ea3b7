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

static int lin_matrix(const mm_tensor_t* t, const char* name, int64_t rows, int64_t cols, bool dense) {
  int rc = validate(t, name, MM_F32);
  if (rc != MM_OK) return rc;
  if (t->ndim != 2 || (rows >= 0 && t->size[0] != rows) || (cols >= 0 && t->size[1] != cols))
    return fail(MM_ERR_INVALID, std::string(name) + ": has the wrong shape");
  if (t->size[0] > INT32_MAX / 2 || t->size[1] > INT32_MAX / 2)
    return fail(MM_ERR_UNSUPPORTED, std::string(name) + ": dimension too large");
  if (dense && t->size[1] > 1 && t->stride[1] != 1)
    return fail(MM_ERR_UNSUPPORTED, std::string(name) + ": rows must be dense");
  return MM_OK;
}

static int lin_output(const mm_tensor_t* t, const char* name, int64_t rows, int64_t cols) {
  int rc = lin_matrix(t, name, rows, cols, true);
  if (rc == MM_OK && rows > 1 && cols > 0 && t->stride[0] != cols)
    return fail(MM_ERR_UNSUPPORTED, std::string(name) + ": must be dense");
  return rc;
}

static int lin_vector(const mm_tensor_t* t, const char* name, int64_t n) {
  int rc = validate(t, name, MM_F32);
  if (rc != MM_OK) return rc;
  if (t->ndim != 1 || t->size[0] != n) return fail(MM_ERR_INVALID, std::string(name) + ": has the wrong length");
  if (n > 1 && t->stride[0] != 1) return fail(MM_ERR_UNSUPPORTED, std::string(name) + ": must be dense");
  return MM_OK;
}

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

static int lin_forward_tc(const mm_tensor_t* x, const mm_tensor_t* w, const LinEpilogue& e, float* y, void* workspace,
                          cudaStream_t s) {
  const int64_t m = x->size[0], k = x->size[1], n = w->size[0];
  LinCarve ws = {(char*)workspace, 0};
  LinSplits all;
  all.count = 0;
  all.blocks = 0;
  bool xt, wt;
  const LinStored xs = lin_store(&ws, &all, (const float*)x->data, x->stride[0], x->stride[1], m, k, &xt);
  const LinStored wst = lin_store(&ws, &all, (const float*)w->data, w->stride[0], w->stride[1], n, k, &wt);
  const LinChoice c = lin_choose(m, n, k);
  float* part = (float*)ws.take(lin_part_bytes(c));
  int rc = lin_run_splits(all, s);
  if (rc != MM_OK) return rc;
  return lin_run_gemm(xt ? xs.by_cols() : xs.by_rows(), wt ? wst.by_cols() : wst.by_rows(), y, e, c, part, s);
}

static int lin_backward_tc(const mm_tensor_t* dy, const mm_tensor_t* x, const mm_tensor_t* w, const mm_tensor_t* z,
                           int act, const mm_tensor_t* dx, const mm_tensor_t* dw, const mm_tensor_t* db,
                           const mm_tensor_t* dz, void* workspace, cudaStream_t s) {
  const int64_t m = x->size[0], k = x->size[1], n = w->size[0];
  LinCarve ws = {(char*)workspace, 0};
  LinSplits all;
  all.count = 0;
  all.blocks = 0;
  bool gt, xt = false, wt = false;
  const LinStored g = lin_store(&ws, &all, (const float*)dy->data, n > 1 ? dy->stride[0] : 1, 1, m, n, &gt);
  LinSplit& gs = all.s[0];
  gs.s0 = dy->stride[0];
  if (act != MM_LINEAR_NONE) {
    gs.z = (const float*)z->data;
    gs.act = act;
    gs.vec = gs.vec && n % 4 == 0 && (uintptr_t)gs.z % 16 == 0;
  }
  gs.out = dz ? (float*)dz->data : nullptr;
  if (db) gs.part = (float*)ws.take(4 * lin_part_rows(m) * n);
  LinStored wst = {}, xs = {};
  if (dx) wst = lin_store(&ws, &all, (const float*)w->data, w->stride[0], w->stride[1], n, k, &wt);
  if (dw) xs = lin_store(&ws, &all, (const float*)x->data, x->stride[0], x->stride[1], m, k, &xt);
  int rc = lin_run_splits(all, s);
  if (rc != MM_OK) return rc;
  if (db) {
    linear_columns_kernel<<<(unsigned)((n + 31) / 32), 256, 0, s>>>(gs.part, (int)lin_part_rows(m), (int)n,
                                                                    (float*)db->data);
    MM_LAUNCH_CHECK("mm_linear_backward launch");
  }
  const LinEpilogue none = {nullptr, nullptr, nullptr, 0, MM_LINEAR_NONE, 0};
  if (dx) {
    const LinChoice c = lin_choose(m, k, n);
    float* part = (float*)ws.take(lin_part_bytes(c));
    rc = lin_run_gemm(g.by_rows(), wt ? wst.by_rows() : wst.by_cols(), (float*)dx->data, none, c, part, s);
    if (rc != MM_OK) return rc;
  }
  if (dw) {
    const LinChoice c = lin_choose(n, k, m);
    float* part = (float*)ws.take(lin_part_bytes(c));
    rc = lin_run_gemm(g.by_cols(), xt ? xs.by_rows() : xs.by_cols(), (float*)dw->data, none, c, part, s);
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

}  // namespace mm

using namespace mm;

extern "C" int mm_linear_workspace_size(int64_t m, int64_t n, int64_t k, int backward, size_t* bytes) {
  if (bytes == nullptr || m < 0 || n < 0 || k < 0) return fail(MM_ERR_INVALID, "mm_linear_workspace_size: invalid argument");
  *bytes = lin_workspace(m, n, k, backward != 0);
  return MM_OK;
}

extern "C" int mm_linear(const mm_tensor_t* x, const mm_tensor_t* w, const mm_tensor_t* bias,
                         const mm_tensor_t* residual, int act, int residual_before_act, const mm_tensor_t* y,
                         const mm_tensor_t* z, void* workspace, size_t workspace_bytes, void* stream) {
  int rc;
  if (act < MM_LINEAR_NONE || act > MM_LINEAR_GELU_TANH) return fail(MM_ERR_INVALID, "mm_linear: unknown activation");
  if ((rc = lin_matrix(x, "mm_linear input", -1, -1, false)) != MM_OK) return rc;
  const int64_t m = x->size[0], k = x->size[1];
  if ((rc = lin_matrix(w, "mm_linear weight", -1, k, false)) != MM_OK) return rc;
  const int64_t n = w->size[0];
  if (bias && (rc = lin_vector(bias, "mm_linear bias", n)) != MM_OK) return rc;
  if (residual && (rc = lin_matrix(residual, "mm_linear residual", m, n, true)) != MM_OK) return rc;
  if ((rc = lin_output(y, "mm_linear output", m, n)) != MM_OK) return rc;
  if (z && (rc = lin_output(z, "mm_linear pre-activation", m, n)) != MM_OK) return rc;
  size_t need = 0;
  if ((rc = mm_linear_workspace_size(m, n, k, 0, &need)) != MM_OK) return rc;
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || (uintptr_t)workspace % 256 != 0))
    return fail(MM_ERR_INVALID, "mm_linear: the workspace is missing, misaligned or too small");
  LinProduct p = {(const float*)x->data, (const float*)w->data, (float*)y->data, x->stride[0], x->stride[1],
                  w->stride[0], w->stride[1], (int)m, (int)n, (int)k};
  LinEpilogue e = {bias ? (const float*)bias->data : nullptr, residual ? (const float*)residual->data : nullptr,
                   z ? (float*)z->data : nullptr, residual ? residual->stride[0] : 0, act, residual_before_act != 0};
  if (lin_on_tensor_cores(m, n, k)) return lin_forward_tc(x, w, e, (float*)y->data, workspace, resolve_stream(stream));
  return lin_product(p, e, resolve_stream(stream));
}

extern "C" int mm_linear_backward(const mm_tensor_t* dy, const mm_tensor_t* x, const mm_tensor_t* w,
                                  const mm_tensor_t* z, int act, const mm_tensor_t* dx, const mm_tensor_t* dw,
                                  const mm_tensor_t* db, const mm_tensor_t* dz, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  int rc;
  if (act < MM_LINEAR_NONE || act > MM_LINEAR_GELU_TANH)
    return fail(MM_ERR_INVALID, "mm_linear_backward: unknown activation");
  if ((rc = lin_matrix(x, "mm_linear_backward input", -1, -1, false)) != MM_OK) return rc;
  const int64_t m = x->size[0], k = x->size[1];
  if ((rc = lin_matrix(w, "mm_linear_backward weight", -1, k, false)) != MM_OK) return rc;
  const int64_t n = w->size[0];
  if ((rc = lin_matrix(dy, "mm_linear_backward output gradient", m, n, true)) != MM_OK) return rc;
  if (act != MM_LINEAR_NONE && (rc = lin_output(z, "mm_linear_backward pre-activation", m, n)) != MM_OK) return rc;
  if (dx && (rc = lin_output(dx, "mm_linear_backward input gradient", m, k)) != MM_OK) return rc;
  if (dw && (rc = lin_output(dw, "mm_linear_backward weight gradient", n, k)) != MM_OK) return rc;
  if (db && (rc = lin_vector(db, "mm_linear_backward bias gradient", n)) != MM_OK) return rc;
  if (dz && (rc = lin_output(dz, "mm_linear_backward pre-activation gradient", m, n)) != MM_OK) return rc;
  size_t need = 0;
  if ((rc = mm_linear_workspace_size(m, n, k, 1, &need)) != MM_OK) return rc;
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || (uintptr_t)workspace % 256 != 0))
    return fail(MM_ERR_INVALID, "mm_linear_backward: the workspace is missing, misaligned or too small");
  cudaStream_t s = resolve_stream(stream);
  if (m == 0 || n == 0) {
    if (dx && m * k > 0) MM_CUDA(cudaMemsetAsync(dx->data, 0, (size_t)(m * k) * 4, s), "mm_linear_backward: zero");
    if (dw && n * k > 0) MM_CUDA(cudaMemsetAsync(dw->data, 0, (size_t)(n * k) * 4, s), "mm_linear_backward: zero");
    if (db && n > 0) MM_CUDA(cudaMemsetAsync(db->data, 0, (size_t)n * 4, s), "mm_linear_backward: zero");
    return MM_OK;
  }
  if (lin_on_tensor_cores(m, n, k)) return lin_backward_tc(dy, x, w, z, act, dx, dw, db, dz, workspace, s);
  LinCarve ws = {(char*)workspace, 0};
  float* own = (float*)ws.take(4 * m * n);
  float* part = (float*)ws.take(4 * LIN_DZ_ROWS * n);
  float* g = dz ? (float*)dz->data : own;
  const int rows = m < LIN_DZ_ROWS ? (int)m : LIN_DZ_ROWS;
  linear_dz_kernel<<<dim3((unsigned)((n + 255) / 256), rows), 256, 0, s>>>(
      (const float*)dy->data, dy->stride[0], act == MM_LINEAR_NONE ? nullptr : (const float*)z->data, act, (int)m,
      (int)n, g, part);
  MM_LAUNCH_CHECK("mm_linear_backward launch");
  if (db) {
    linear_columns_kernel<<<(unsigned)((n + 31) / 32), 256, 0, s>>>(part, rows, (int)n, (float*)db->data);
    MM_LAUNCH_CHECK("mm_linear_backward launch");
  }
  const LinEpilogue none = {nullptr, nullptr, nullptr, 0, MM_LINEAR_NONE, 0};
  if (dx) {
    LinProduct p = {g, (const float*)w->data, (float*)dx->data, n, 1, w->stride[1], w->stride[0], (int)m, (int)k, (int)n};
    if ((rc = lin_product(p, none, s)) != MM_OK) return rc;
  }
  if (dw) {
    LinProduct p = {g, (const float*)x->data, (float*)dw->data, 1, n, x->stride[1], x->stride[0], (int)n, (int)k, (int)m};
    if ((rc = lin_product(p, none, s)) != MM_OK) return rc;
  }
  return MM_OK;
}
