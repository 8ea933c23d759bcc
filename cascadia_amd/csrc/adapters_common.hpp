// adapters_common.hpp -- device helpers: chunks of rows of one adapter.
#pragma once
#include "int4_common.hpp"
#include "tokens.hpp"

namespace cai4 {
namespace {

// Sorted rows row0 .. row0 + rows of one group (rows 0: there is no such chunk).
struct Chunk {
  int group, row0, rows;
};

// First sorted row of group e (group E: the rows without an adapter; past it T), within
// [0, T] whatever the offsets hold.
CAI4_DEV int first_row(const Adapters &a, int e) {
  const int v = a.offsets[e < a.E ? e : a.E];  // (loaded in any case: no branch)
  return e > a.E || v > a.T ? a.T : v < 0 ? 0 : v;
}
template <int ROWS>
CAI4_DEV int chunks_of(int first, int last) {
  return last > first ? (last - first + ROWS - 1) / ROWS : 0;
}

// Sum of v over the lanes up to this one.
CAI4_DEV int lanes_upto(int v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int u = __shfl_up(v, d);
    if (lane >= d) v += u;
  }
  return v;
}

// Chunk b (of ROWS rows) of all groups' in order (bare: group E among them), by each wave
// for itself: lane i holds the offsets of `per` neighbouring groups and adds up their chunks.
template <int ROWS>
CAI4_DEV Chunk find_chunk(const Adapters &a, int b, bool bare) {
  constexpr int kMostPer = (kSortMaxGroups + 1 + 63) / 64;
  const int lane = threadIdx.x & 63;
  const int groups = a.E + (bare ? 1 : 0), per = (groups + 63) / 64;
  int row[kMostPer + 1], n = 0;
#pragma unroll
  for (int i = 0; i <= kMostPer; ++i) {  // (every load before the first use)
    const int e = lane * per + i;
    if (i <= per) row[i] = first_row(a, e < groups ? e : groups);
  }
#pragma unroll
  for (int i = 0; i < kMostPer; ++i)
    if (i < per) n += chunks_of<ROWS>(row[i], row[i + 1]);
  const int upto = lanes_upto(n);
  const uint64_t hit = __ballot(upto > b);
  if (!hit) return Chunk{0, 0, 0};
  const int l = __builtin_ctzll(hit);
  int left = b - __builtin_amdgcn_readlane(upto - n, l);
  Chunk ch{0, 0, 0};
#pragma unroll
  for (int i = 0; i < kMostPer; ++i) {
    if (i < per) {
      const int first = __builtin_amdgcn_readlane(row[i], l);
      const int last = __builtin_amdgcn_readlane(row[i + 1], l), m = chunks_of<ROWS>(first, last);
      const int rows = last - first - left * ROWS;
      if (left >= 0 && left < m)
        ch = Chunk{l * per + i, first + left * ROWS, rows < ROWS ? rows : ROWS};
      left -= m;  // (negative once found)
    }
  }
  return ch;
}

// The row of x and y that is row i of the chunk; -1: none.
CAI4_DEV int row_of(const Adapters &a, const Chunk &ch, int i) {
  if (i >= ch.rows) return -1;
  const int t = a.slots[ch.row0 + i];
  return t >= 0 && t < a.T ? t : -1;
}

CAI4_DEV int rank_of(const Adapters &a, int e) {
  const int r = a.ranks ? a.ranks[e] : a.R;
  return __builtin_amdgcn_readfirstlane(r < 0 ? 0 : r > a.R ? a.R : r);
}

}  // namespace
}  // namespace cai4
