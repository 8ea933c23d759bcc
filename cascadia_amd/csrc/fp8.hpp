// fp8.hpp -- 8-bit floating point (OCP e4m3) with a scale per block of 128, and
// the routing of tokens to experts: what abi.hip calls.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace cai4 {

// Whether a launch takes so many workgroups along one dimension of its grid: fewer
// than 2^32 threads.
inline bool launch_fits(size_t workgroups, size_t threads) {
  return workgroups < ((size_t)1 << 32) / threads;
}

// Choice of top_k of E experts per token from router logits (route.hip).
struct RouteExperts {
  const void *logits;  // [T, E], f32 or bf16
  const float *bias;   // [E] or null: added to the scores for the choice only
  int T, E, top_k;
  int x_f32, sigmoid;                      // logits' type; scores: sigmoid, else softmax
  int n_groups, top_groups, group_best;    // groups of E / n_groups neighbours
  int normalize;
  float scale;
  int32_t *ids;    // [T, top_k]
  float *weights;  // [T, top_k]
};
constexpr int kRouteMaxExperts = 1024, kRouteMaxTopK = 16, kRouteMaxGroups = 64;
constexpr int kRouteMaxTokens = 1 << 25;  // (64 threads each)
hipError_t route_experts(const RouteExperts &r, hipStream_t st);

constexpr int kFp8Block = 128;
inline int fp8_blocks(int n) { return (n + kFp8Block - 1) / kFp8Block; }

// Scales per row inside a workspace: rows of 16 bytes' multiple.
inline int fp8_ld(int K) { return (fp8_blocks(K) + 3) & ~3; }

// x [rows, K] (bf16 or f32) -> e4m3 codes [rows, K] and scales [rows, ld], ceil(K /
// 128) of them.  K a multiple of 16; x, codes 16-byte aligned.
hipError_t fp8_quantize_rows(const void *x, bool x_f32, size_t rows, int K, uint8_t *codes,
                             float *scales, int ld, hipStream_t st);
// Scales [rows, KB] to rows of ld.
hipError_t fp8_pad_scales(const float *scales, size_t rows, int KB, float *to, int ld,
                          hipStream_t st);
// w bf16 [N, K] -> codes [N, K] and scales [ceil(N / 128), ceil(K / 128)].
hipError_t fp8_quantize_blocks(const uint16_t *w, int N, int K, uint8_t *codes, float *scales,
                               hipStream_t st);

// Rows row0 .. row0 + count of the grouped rows, of one expert; chunk first +
// [0, number) are that expert's.
struct Fp8Chunk {
  int expert, row0, count, first, number;
};

// Codes [count, N, K] -> blocks of 128 rows x 128 columns, each contiguous (16 KB, row
// by row), padded with zeros: [count, ceil(N / 128), ceil(K / 128), 128, 128].
constexpr size_t kFp8BlockBytes = 128 * 128;
inline size_t fp8_tiled_bytes(int N, int K) {
  return (size_t)fp8_blocks(N) * fp8_blocks(K) * kFp8BlockBytes;
}
hipError_t fp8_tile_weights(const uint8_t *codes, int count, int N, int K, uint8_t *tiled,
                            hipStream_t st);

// y = x w^T over e4m3 codes and their blocks' scales, for one matrix or for the
// row groups of many experts in one launch (chunks).
struct Fp8Gemm {
  const uint8_t *w;  // [N, K] codes (SwiGLU: gate [N, K], then up [N, K])
  int w_tiled;       // w in blocks (fp8_tile_weights)
  const float *ws;   // [ceil(N / 128), KB] (SwiGLU: gate's, then up's)
  const uint8_t *x;  // [rows, K] codes
  const float *xs;   // [rows, ld_xs], KB of them used (tiles: 16-byte aligned rows)
  int ld_xs;
  void *y;           // [M, N]
  int N, K, M;       // M: rows of y
  int out_f32;       // y f32, else bf16
  // experts: chunks of grouped rows (null: one matrix over M rows)
  const Fp8Chunk *chunks;
  int max_chunks, chunk_rows;
  const int32_t *n_chunks;     // how many of them there are (device)
  const int32_t *row_map;      // grouped row -> row of x (null: the same)
  int x_rows;                  // rows of x (row_map)
  size_t w_stride, ws_stride;  // between experts
  int swiglu;                  // y = silu(gate) * up: f32, or codes with ys
  int exact;                   // experts on tiles: no 8-bit sums
  float *ys;                   // SwiGLU on tiles: y's scales [rows, ld_ys]
  int ld_ys;
  float *part;                 // tiles: workspace of fp8_partial_bytes
  int kper;                    // (set by fp8_tile_gemm)
};
hipError_t fp8_gemm(const Fp8Gemm &g, hipStream_t st);
// Forms of a product of one matrix: 16 x 32 or 32 x 32 outputs per workgroup, or tiles
// of 128 x 128 (with K in slices or not), 256 x 128, 256 x 256.
enum Fp8Form {
  kFp8Rows16 = 1,
  kFp8Rows32,
  kFp8Tiles128,
  kFp8Slices128,
  kFp8Tiles256x128,
  kFp8Tiles256
};
constexpr int kFp8FewRows = 16;  // no more rows than these run on tiles
Fp8Form fp8_form(int M, int N, int K, bool out_f32);
Fp8Form fp8_tile_form(int M, int N, int K, bool out_f32);  // of one on tiles
float fp8_tile_us(int M, int N, int K, bool out_f32);      // its estimated time
// Bytes of partial sums of a product on tiles, for any number of rows up to M.
size_t fp8_partial_bytes(int M, int N, int K);
constexpr int kFp8TileRows = 128;  // rows of a chunk on the tile kernel (16 else)
hipError_t fp8_tile_gemm(const Fp8Gemm &g, hipStream_t st);

// One layer's experts in e4m3.
struct Fp8Moe {
  int H, I, E, tiled;
  const uint8_t *gate_up, *down;      // [E, 2, I, H], [E, H, I]
  const float *gate_up_s, *down_s;    // [E, 2, ib, hb], [E, hb, ib]
  int T, top_k;
  const int32_t *ids;
  const float *weights;
  float threshold;
  const void *x;
  int x_f32;
  const void *residual;  // [T, H] of out's type, or null
  void *out;
  int out_f32;
};
// One row of x (bf16 or f32), quantised in the kernel (fp8_one_row).
bool fp8_one_row(int K);
bool fp8_one_token(int H, int I, int top_k);
hipError_t fp8_gemv(const Fp8Gemm &g, const void *x, bool x_f32, hipStream_t st);
// One token (fp8_one_token): gate / up into h [top_k, I], down and the weighted sum.
hipError_t fp8_moe_one(const Fp8Moe &m, const Fp8Gemm &gate_up, const Fp8Gemm &down, float *h,
                       hipStream_t st);
size_t fp8_moe_workspace(int H, int I, int E, int top_k, int T);
bool fp8_moe_fits(int H, int I, int E, int top_k, int T);  // every launch_fits
int fp8_moe_chunk_rows(int T, int E, int top_k);  // 16, or kFp8TileRows: on tiles
hipError_t fp8_moe_forward(const Fp8Moe &m, void *workspace, hipStream_t st);

}  // namespace cai4
