// Distances between the positions of a map, and which of them the bias gradient's rings hold at a time (attention, backward).
// Whole-number arithmetic only, and no HIP in it, so that the host can walk through the same functions.
#pragma once

#ifdef __HIPCC__
#define YAMD_BOTH __host__ __device__ __forceinline__
#else
#define YAMD_BOTH inline
#endif

namespace yamd {

constexpr int kTile = 64;                // rows of a tile that passes through LDS (keys, or queries in the dK / dV kernel)
constexpr int kBlockRows = 128;          // rows that a workgroup owns: 32 for each of its four waves

// A position t of a map of width w at (t / w, t % w) has the coordinate a(t) = (t / w)(2 w - 1) + t % w, and the distance of
// two positions the index a(query) - a(key) + a(last) among the (2 h - 1)(2 w - 1) distances of the map.
YAMD_BOTH int map_coord(int t, int w) { return t + (t / w) * (w - 1); }

// Positions of a ring of sums by distance: a power of two that holds the distances of two tiles of keys, one being added to
// while the other is written out: 2 * 127 + 1 and the 4 below that quads touch, and where a map has several rows
// 127 + 127 + 2 w more.
YAMD_BOTH int ring_len(int map_h, int map_w)
{
    const int span = 2 * kBlockRows + 8 + (map_h > 1 ? 2 * kBlockRows + 2 * map_w : 0);
    int n = 256;
    while (n < span) n *= 2;
    return n;
}

// distances of the 128 rows of a workgroup against `keys` keys, at most
YAMD_BOTH int distances_of(int keys, int map_h, int map_w)
{
    return keys + kBlockRows + (map_h > 1 ? keys + kBlockRows + 2 * map_w : 0);
}

// From this distance on all sums are final when a workgroup starts on the keys from `key` on.  The row that it counts from is
// the last of the workgroup's 128, also where the queries end before: lanes beyond them still add (zeros) at distances of
// their own, while other waves take the final sums out of the rings.
YAMD_BOTH int final_from(int tile, int key, int coord_last, int map_w)
{
    return coord_last + map_coord(tile * kBlockRows + kBlockRows - 1, map_w) - map_coord(key, map_w) + 1;
}

}  // namespace yamd
