// Interface of the linear operator's tensor-core path (mm_linear_tc.cu).
#pragma once

#include "mm_linear.cuh"

namespace mm {

// A float32 matrix to be split: element (r, c) at src[r * s0 + c * s1].
struct LinSplit {
  const float* src;
  int64_t s0, s1;
  const float* z;    // values times act'(z) of a dense [rows][cols] z, or null
  int act;
  int vec;           // src (and z) may be read in 16-byte pieces along c
  int64_t rows;
  int cols;
  int64_t ld;        // planes [3][rows][ld], ld a multiple of 8
  uint16_t* planes;
  int* flags;        // one per block: holds an infinity
  float* part;       // partial column sums [lin_part_rows(rows)][cols], or null
  float* out;        // the values themselves, dense, or null
  uint32_t first;
  int blocks_c;
};

struct LinSplits {
  LinSplit s[3];
  int count;
  int64_t blocks;
};

// The planes of a product's operand: `lines` rows of A or B (rows or columns
// of C) and k values of the reduction.  mn: stored [k][lines], else [lines][k].
struct LinPlanes {
  const uint16_t* planes;
  const int* flags;
  int64_t lines, k, ld;
  int mn;
};

constexpr int LIN_GROUP = 8;        // rows of tiles that run together
constexpr int LIN_MAX_SPLITS = 32;

struct LinChoice {
  int bm, bn;           // rows of a tile (256: of a CTA pair's) and columns
  int full;             // tiles that run undivided
  int splits;           // parts of the reduction of each tile behind them
  int tiles_m, tiles_n, stages, units;
  double clocks;        // the estimate
};

struct LinGemm {
  int m, n, bm, stages, tiles_m, tiles_n, full, splits, units, vec;
  float* c;      // dense [m][n]
  float* part;   // partial tiles
  LinEpilogue e;
  LinPlanes pa, pb;
  int flags_a, flags_b;  // their numbers of flags
  int early;             // see lin_backward_tc
  int* fault;            // the device's fault word (host memory), or null
  int64_t wait_ns;       // limit of the kernel's waits
  int drop;              // test hook: CTA 0 leaves its first loads out
};

int64_t lin_flag_words(int64_t rows, int64_t cols);
int64_t lin_plane_bytes(int64_t rows, int64_t cols);
int64_t lin_part_rows(int64_t m);
void lin_add_split(LinSplits* all, const LinSplit& s);
int lin_run_splits(const LinSplits& all, cudaStream_t s);
LinChoice lin_choose(int64_t m, int64_t n, int64_t k);
int64_t lin_part_bytes(const LinChoice& c);
// C[m, n] = A B^T through the epilogue, up to the divided tiles' sums; the latter
// (if any; g from lin_run_gemm).
int lin_run_gemm(const LinPlanes& a, const LinPlanes& b, float* c, const LinEpilogue& e, const LinChoice& ch,
                 float* part, bool early, LinGemm* g, cudaStream_t s);
int lin_run_join(const LinGemm& g, const LinChoice& ch, bool early, cudaStream_t s);
void lin_debug_fault(int device, int64_t wait_ns, int drop);

}  // namespace mm
