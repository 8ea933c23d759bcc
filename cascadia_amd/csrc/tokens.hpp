// tokens.hpp -- tokens sorted by expert and back, and low-rank adapters over rows
// sorted by adapter: what abi.hip calls.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace cai4 {

// Value types of rows (gather: of one byte too, which is copied).
enum RowType { kRowBf16 = 0, kRowF32 = 1, kRowByte = 2 };

constexpr int kSortMaxGroups = 1024, kSortMaxTopK = 16, kSortMaxTokens = 1 << 20;
constexpr int kRowMaxCols = 1 << 20;

// Slots t * top_k + j in order of their group (stable), those left out behind.
struct SortTokens {
  const int32_t *ids;    // [n]
  const float *weights;  // [n] or null
  float threshold;
  int n, E;
  int32_t *offsets;  // [E + 1]
  int32_t *slots;    // [n]: sorted row -> slot
  int32_t *rows;     // [n]: slot -> sorted row, -1: left out
};
size_t sort_tokens_workspace(int n, int E);
hipError_t sort_tokens(const SortTokens &s, void *workspace, hipStream_t st);

// xs[rows[t, j]] = x[t] (cols values each; n = T * top_k rows of xs at most).
hipError_t gather_tokens(const void *x, RowType x_type, const int32_t *rows, int T, int top_k,
                         int cols, void *xs, RowType xs_type, hipStream_t st);

// out[t] = residual[t] + sum_j weights[t, j] * ys[rows[t, j]]
struct CombineTokens {
  const void *ys;
  const int32_t *rows;
  const float *weights;  // null: 1
  const void *residual;  // of out's type, or null
  void *out;
  int T, top_k, cols;
  int y_f32, out_f32;
};
hipError_t combine_tokens(const CombineTokens &c, hipStream_t st);

// dys[rows[t, j]] = weights[t, j] * dout[t]; dweights[t, j] = ys[rows[t, j]] . dout[t]
struct CombineGrad {
  const void *dout, *ys;
  const int32_t *rows;
  const float *weights;
  void *dys;        // of ys's type; may be ys
  float *dweights;  // [T, top_k]
  int T, top_k, cols;
  int dout_f32, y_f32;
};
hipError_t combine_tokens_grad(const CombineGrad &c, hipStream_t st);

// ys = base + scale_a B_a (A_a x) for rows sorted by adapter (SortTokens, top_k 1).
constexpr int kAdaptersMaxRank = 256;
struct Adapters {
  int K, N, R, E;            // R: rows kept of each A (a multiple of 8)
  const uint16_t *a, *b;     // [E, R, K], [E, N, R] bf16
  const int32_t *ranks;      // [E] or null: R
  const float *scales;       // [E] or null: 1
  const int32_t *offsets, *slots;
  int T;
  const void *x, *base;      // base null: zero
  void *y;
  uint32_t ldx, ldb, ldy;    // row strides in bytes
  int x_f32, base_f32, y_f32;
};
size_t adapters_workspace(int K, int R, int E, int T);
hipError_t adapters_forward(const Adapters &a, void *workspace, hipStream_t st);

}  // namespace cai4
