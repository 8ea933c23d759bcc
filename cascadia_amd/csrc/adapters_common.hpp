// adapters_common.hpp -- device helpers: chunks of rows of one adapter.
#pragma once
#include "int4_common.hpp"
#include "tokens.hpp"

namespace cai4 {
namespace {

constexpr int kChunkRows = 64;

// Sorted rows row0 .. row0 + rows of one group (rows 0: there is no such chunk).
struct Chunk {
  int group, row0, rows;
};

// First sorted row of group e (group E: the rows without an adapter), within [0, T]
// whatever the offsets hold.
CAI4_DEV int first_row(const Adapters &a, int e) {
  const int v = e > a.E ? a.T : a.offsets[e];
  return v < 0 ? 0 : v > a.T ? a.T : v;
}
CAI4_DEV int chunks_of(int first, int last) {
  return last > first ? (last - first + kChunkRows - 1) / kChunkRows : 0;
}

// Chunk b of all groups' in order (bare: group E among them).  By each wave for
// itself: lane i adds up the chunks of `per` neighbouring groups.
CAI4_DEV Chunk find_chunk(const Adapters &a, int b, bool bare) {
  const int lane = threadIdx.x & 63;
  const int groups = a.E + (bare ? 1 : 0), per = (groups + 63) / 64, e0 = lane * per;
  int n = 0;
  if (e0 < groups) {
    int first = first_row(a, e0);
    for (int e = e0; e < e0 + per && e < groups; ++e) {
      const int last = first_row(a, e + 1);
      n += chunks_of(first, last);
      first = last;
    }
  }
  int upto = n;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int v = __shfl_up(upto, d);
    if (lane >= d) upto += v;
  }
  const uint64_t hit = __ballot(upto > b);
  if (!hit) return Chunk{0, 0, 0};
  const int l = __builtin_ctzll(hit);
  int left = b - (__shfl(upto, l) - __shfl(n, l));
  for (int e = l * per; e < (l + 1) * per && e < groups; ++e) {
    const int first = first_row(a, e), last = first_row(a, e + 1), m = chunks_of(first, last);
    if (left < m) {
      const int row0 = first + left * kChunkRows;
      Chunk ch{e, row0, last - row0 < kChunkRows ? last - row0 : kChunkRows};
      ch.group = __builtin_amdgcn_readfirstlane(ch.group);
      ch.row0 = __builtin_amdgcn_readfirstlane(ch.row0);
      ch.rows = __builtin_amdgcn_readfirstlane(ch.rows);
      return ch;
    }
    left -= m;
  }
  return Chunk{0, 0, 0};
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
