// Rows in consecutive groups given by offsets on the device ([groups + 1], group g = rows [offsets[g], offsets[g + 1])), cut into tiles of at
// most TILE rows of one group each.  The host knows the number of rows and of groups but not the offsets, so a launch has as many
// blocks as there can be tiles (max_tiles) and each block looks its own up.
//
// The rows in front of the first group and behind the last one are tiles as well, of no group (group -1).  Offsets are held within [0, rows]
// and a group that would end in front of its beginning is empty: offsets that are not what they should be give wrong results
// in rows of the call's own tensors, not accesses outside of them.
#pragma once

#include "common.cuh"

namespace ac4k {

__host__ __device__ constexpr int64_t ragged_max_tiles(int64_t rows, int64_t groups, int tile) { return groups + 2 + rows / tile; }

struct RaggedTile {
  int group;      // -1: rows of no group, -2: no such tile
  int row0, row1; // rows [row0, row1)
};

struct RaggedScratch {
  int warp_sums[32];
  RaggedTile found;
};

// Tile number `want`, for a whole block of THREADS threads (all of them call this).
template <int THREADS>
__device__ __forceinline__ RaggedTile ragged_tile(const int32_t *__restrict__ offsets, int groups, int rows, int tile, int want, RaggedScratch *sh) {
  // entries: 0 the rows in front, 1 .. groups the groups, groups + 1 the rows behind
  const int entries = groups + 2, per = (entries + THREADS - 1) / THREADS;
  auto bound = [&](int e) {        // where entry e begins; entry `entries` begins at the end
    if (e == 0) return 0;
    if (groups == 0) return rows;  // (no offsets are read)
    return e == entries ? rows : min(max(__ldg(offsets + e - 1), 0), rows);
  };
  const int e0 = min((int)threadIdx.x * per, entries), e1 = min(e0 + per, entries);
  int count = 0;
  if (e0 < e1) {
    int lo = bound(e0);
    for (int e = e0; e < e1; ++e) {
      const int hi = bound(e + 1);
      if (hi > lo) count += (hi - lo + tile - 1) / tile;
      lo = hi;
    }
  }
  // tiles in front of this thread's entries
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int upto = count;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xFFFFFFFFu, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) sh->warp_sums[warp] = upto;
  if (threadIdx.x == 0) sh->found.group = -2;
  __syncthreads();
  int before = upto - count;
  for (int w = 0; w < warp; ++w) before += sh->warp_sums[w];
  if (want >= before && want < before + count) {
    int lo = bound(e0);
    for (int e = e0; e < e1; ++e) {
      const int hi = bound(e + 1), n = hi > lo ? (hi - lo + tile - 1) / tile : 0;
      if ((unsigned)(want - before) < (unsigned)n) {        // (within the group whatever the sums of offsets that are none have come to)
        const int r = lo + (want - before) * tile;
        sh->found = RaggedTile{e == 0 || e == entries - 1 ? -1 : e - 1, r, min(r + tile, hi)};
        break;
      }
      before += n;
      lo = hi;
    }
  }
  __syncthreads();
  return sh->found;
}

}  // namespace ac4k
