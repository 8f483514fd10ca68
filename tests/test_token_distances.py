"""The bias gradient's rings of sums by distance, walked through on the host with the kernel's own index arithmetic
(csrc/yamd_distance.h): what one wave adds to is never what another takes out at the same time, every distance is taken out
once and complete, and nothing leaves the ring or the row of the workspace."""
import ctypes
import os
import subprocess

import pytest

from conftest import ROOT

CSRC = os.path.join(ROOT, "yolo_amd", "csrc")

# One workgroup (128 rows from `tile` on) over the key tiles [t0, t1), as the kernel of dq walks them: at step t it takes the
# distances [final_from(t), the last bound) out of the rings, and in the same step the lanes of every wave that has a row
# below q_len add at their distances to the tile's keys (quads: also 4 below; a quad starts at every fourth key).
WALK = r"""
#include <vector>
#include "yamd_distance.h"
using namespace yamd;
enum { OK, MEETS, NOT_CLEARED, TWICE, MISSING, OUTSIDE_ROW };
extern "C" int walk(int h, int w, int tile, int t0, int t1, int quads)
{
    const int n = h * w, mw = h > 1 ? w : 1, ring = ring_len(h, w), last = map_coord(n - 1, mw), size = 2 * last + 1;
    const int row0 = tile * kBlockRows, end_key = t1 * kTile < n ? t1 * kTile : n;
    const int base = last + map_coord(row0, mw) - map_coord(end_key - 1, mw);
    const int row_len = distances_of(end_key - t0 * kTile, h, w);
    const int margin = 4096 + 8 * w;                                       // lanes beyond the queries, and 4 below
    std::vector<int> added(size + 2 * margin, 0), taken(size + 2 * margin, 0), holds(ring, 1 << 30);
    std::vector<char> flushing(ring);
    auto at = [&](int d) { return d + margin; };
    int high = final_from(tile, t0 * kTile, last, mw);
    auto flush = [&](int low) {
        for (int e = low; e < high; ++e) {
            const int slot = e & (ring - 1);
            if (holds[slot] != 1 << 30 && holds[slot] != e) return (int)NOT_CLEARED;       // sums of another distance
            if (e - base < 0 || e - base >= row_len) return (int)OUTSIDE_ROW;
            if (taken[at(e)]++) return (int)TWICE;
            holds[slot] = 1 << 30;
            flushing[slot] = 1;
        }
        high = low;
        return (int)OK;
    };
    for (int t = t0; t < t1; ++t) {
        flushing.assign(ring, 0);
        if (int rc = flush(final_from(tile, t * kTile, last, mw))) return rc;
        for (int row = row0; row < row0 + kBlockRows; ++row) {
            if (row / 32 * 32 >= n) break;                                 // a wave without rows adds nothing
            const int cq = last + map_coord(row, mw);
            for (int k = 0; k < kTile; k += quads ? 4 : 1)
                for (int below = 0; below <= (quads ? 4 : 0); below += 4) {
                    const int d = cq - map_coord(t * kTile + k, mw) - below, slot = d & (ring - 1);
                    if (flushing[slot]) return MEETS;
                    // (what it holds: the zeros of places that no pair is at may share a slot with nothing that has been added)
                    if (holds[slot] != 1 << 30 && holds[slot] != d) return NOT_CLEARED;
                    holds[slot] = d;
                }
            for (int k = 0; k < kTile && row < n && t * kTile + k < n; ++k) {
                const int d = cq - map_coord(t * kTile + k, mw);
                if (taken[at(d)]) return MISSING;                          // added after it was taken out
                added[at(d)] = 1;
            }
        }
    }
    flushing.assign(ring, 0);
    if (int rc = flush(base)) return rc;
    for (int d = 0; d < size; ++d)
        if (added[at(d)] && !taken[at(d)]) return MISSING;
    return OK;
}
"""


@pytest.fixture(scope="module")
def walk(tmp_path_factory):
    d = tmp_path_factory.mktemp("walk")
    (d / "walk.cpp").write_text(WALK)
    subprocess.check_call(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-I", CSRC, str(d / "walk.cpp"), "-o", str(d / "walk.so")])
    return ctypes.CDLL(str(d / "walk.so")).walk


def _all(walk, h, w, quads):
    n = h * w
    tiles, steps = (n + 127) // 128, (n + 63) // 64
    for tile in {0, tiles // 2, tiles - 1}:
        for t0, t1 in {(0, steps), (0, (steps + 1) // 2), (steps // 2, steps), (steps - 1, steps)}:
            if t0 < t1:
                assert walk(h, w, tile, t0, t1, quads) == 0, (h, w, tile, t0, t1, quads)


@pytest.mark.parametrize("quads", [0, 1])
def test_sequences(walk, quads):
    for n in list(range(1, 300)) + [400, 800, 1000, 1447, 1999, 2000]:
        _all(walk, 1, n, quads)


@pytest.mark.parametrize("h,w", [(2, 1), (130, 1), (300, 2), (3, 7), (5, 7), (9, 12), (11, 13), (19, 19), (38, 38), (20, 20), (8, 100), (3, 100),
                                 (2, 150), (40, 12), (25, 30), (2, 420), (5, 63), (4, 64), (7, 65), (3, 126), (3, 127), (3, 128), (2, 760), (3, 759)])
def test_maps(walk, h, w):
    for quads in ([0, 1] if w % 4 == 0 else [0]):
        _all(walk, h, w, quads)
