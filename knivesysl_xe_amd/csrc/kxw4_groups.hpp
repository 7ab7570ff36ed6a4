// kxw4_groups.hpp — how a work-group of a launch over grouped rows finds the
// tile it works on.
//
// The rows of group e are the sorted places [offsets[e], offsets[e + 1]), cut
// into tiles of TT places that never reach over two groups. The counts are
// known on the device only, so the host launches enough work-groups for any
// counts (tiles_at_most) and each finds its tile from the offsets: every lane
// adds up the tiles of a run of groups, a scan over the lanes (on DPP moves, no
// LDS) places them. At up to 64 groups that is one memory round trip.
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
    int begin, begin_end;                                    // the places of its first group
};

// v plus the lane of the DPP control's, 0 where there is none (row_mask: rows
// of 16 lanes that take part).
template <int CTRL, int ROW_MASK>
__device__ __forceinline__ int dpp_add(int v) {
    return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROW_MASK, 0xF, false);
}

// Inclusive sum over the wave's lanes: row_shr 1, 2, 4, 8 within rows of 16,
// then row_bcast:15 (a row's last lane to the next row) into rows 1 and 3 and
// row_bcast:31 into rows 2 and 3.
__device__ __forceinline__ int wave_scan(int v) {
    v = dpp_add<0x111, 0xF>(v);
    v = dpp_add<0x112, 0xF>(v);
    v = dpp_add<0x114, 0xF>(v);
    v = dpp_add<0x118, 0xF>(v);
    v = dpp_add<0x142, 0xA>(v);
    return dpp_add<0x143, 0xC>(v);
}

template <int WHICH = kTilesAll>
__device__ __forceinline__ GroupTiles scan_tiles(const int *offsets, int groups, int TT, int lane) {
    const int run = (groups + 63) / 64;
    GroupTiles s;
    s.first = min(lane * run, groups);
    s.end = min(s.first + run, groups);
    int sum = 0;
    int lo = offsets[s.first];
    s.begin = lo;
    s.begin_end = lo;
    for (int e = s.first; e < s.end; ++e) {
        const int hi = offsets[e + 1];
        if (e == s.first) s.begin_end = hi;
        sum += tiles_of<WHICH>(hi - lo, TT);
        lo = hi;
    }
    const int inc = wave_scan(sum);
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
    t.begin = __builtin_amdgcn_readlane(s.begin, l);
    t.end = __builtin_amdgcn_readlane(s.begin_end, l);
    for (;;) {
        t.count = tiles_of<WHICH>(t.end - t.begin, TT);
        if (u < t.before + t.count) break;
        t.before += t.count;
        ++t.e;
        t.begin = t.end;
        t.end = offsets[t.e + 1];
    }
    t.index = u - t.before;
    return t;
}

}  // namespace kxw4
