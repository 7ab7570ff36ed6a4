// kxw4_groups.hpp — how a work-group of a launch over grouped rows finds the
// tile it works on.
//
// The rows of group e are the sorted places [offsets[e], offsets[e + 1]), cut
// into tiles of TT places that never reach over two groups. The counts are
// known on the device only, so the host launches enough work-groups for any
// counts (tiles_at_most) and each finds its tile from the offsets: every lane
// adds up the tiles of a run of groups, a scan over the lanes places them.
// That is one memory round trip and about 300 cycles at up to 64 groups.
#pragma once

#include <hip/hip_runtime.h>

namespace kxw4 {

// Tiles of TT places that N rows in `groups` groups come to at most.
inline long long tiles_at_most(long long N, int groups, int TT) {
    return N / TT + (N < groups ? N : groups);
}

// What to count of a group's rows: all its tiles, those that are full, or the
// one that is not.
enum { kTilesAll = 0, kTilesFull = 1, kTilesPart = 2 };
template <int WHICH>
__device__ __forceinline__ int tiles_of(int rows, int TT) {
    return WHICH == kTilesAll ? (rows + TT - 1) / TT : WHICH == kTilesFull ? rows / TT : (rows % TT != 0);
}

struct GroupTiles {
    int first, end, tiles_before, total;                     // this lane's run of groups, the tiles before it, all tiles
};

template <int WHICH = kTilesAll>
__device__ __forceinline__ GroupTiles scan_tiles(const int *offsets, int groups, int TT, int lane) {
    const int run = (groups + 63) / 64;
    GroupTiles s;
    s.first = min(lane * run, groups);
    s.end = min(s.first + run, groups);
    int sum = 0;
    int lo = offsets[s.first];
    for (int e = s.first; e < s.end; ++e) {
        const int hi = offsets[e + 1];
        sum += tiles_of<WHICH>(hi - lo, TT);
        lo = hi;
    }
    int inc = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int v = __shfl_up(inc, o, 64);
        if (lane >= o) inc += v;
    }
    s.tiles_before = inc - sum;
    s.total = __builtin_amdgcn_readlane(inc, 63);
    return s;
}

struct GroupTile {
    int e, index, before, count, begin, end;                 // group, tile among its `count`, tiles before them, its places
};

// Tile u < s.total.
template <int WHICH = kTilesAll>
__device__ __forceinline__ GroupTile tile_at(const GroupTiles &s, const int *offsets, int TT, int u) {
    // (the last lane whose run starts at or before u has the tile, since
    // every later one starts past it: lanes without tiles share their start)
    const int l = 63 - __builtin_clzll(__ballot(s.first < s.end && s.tiles_before <= u));
    GroupTile t;
    t.e = __builtin_amdgcn_readlane(s.first, l);
    t.before = __builtin_amdgcn_readlane(s.tiles_before, l);
    for (;;) {
        t.begin = offsets[t.e];
        t.end = offsets[t.e + 1];
        t.count = tiles_of<WHICH>(t.end - t.begin, TT);
        if (u < t.before + t.count) break;
        t.before += t.count;
        ++t.e;
    }
    t.index = u - t.before;
    return t;
}

}  // namespace kxw4
