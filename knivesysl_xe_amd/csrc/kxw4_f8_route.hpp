// kxw4_f8_route.hpp — which kernel and tile a product of the 8-bit floating tier
// takes, from its sizes alone (figures: us on the MI355X, replayed from a graph
// over copies of the weights larger than the caches).
#pragma once

#include <algorithm>

namespace kxw4 {

struct F8Sizes {
    int cus, rows, kb, count, M[4];                          // kb: column blocks
    int groups;                                              // 0: one weight for all rows; else rows: of all groups together
    bool bf16;                                               // outputs
};

inline long long f8_row_groups(const F8Sizes &s) {
    long long rgs = 0;
    for (int i = 0; i < s.count; ++i) rgs += s.M[i] / 16;
    return rgs;
}

// Tiles of `rows` rows, at most, of all groups.
inline long long f8_tiles_of(const F8Sizes &s, int rows) {
    return s.groups ? s.rows / rows + std::min(s.rows, s.groups) : (s.rows + rows - 1) / rows;
}

// Rows of a stream tile (16 or 32; kxw4_f8_stream.hip), 0 for the large tiles.
// Up to 16 rows a weight the weights' stream bounds the product and one tile
// reads it once (16 rows, 5120 x 5120: 9.8 us, large tiles 13; 128 rows over 64
// experts of 1,024 x 5120: 69, 71). Past that tiles of 32 are ahead while the
// launch is short, up to 13,000 weight tiles of 16 x 128 read (32 rows, 5120 x
// 5120, 12,800: 11.4 us for 14.1; 64 rows, 25,600: 18.7 for 15.5; 128 rows, 1456
// x 2064, 6,192: 8.6 for 9.3; 17 rows, 17408 x 5120, 43,520: 28.4 for 24.8).
inline int f8_stream_rows(const F8Sizes &s) {
    const long long groups = std::max(s.groups, 1);
    if (s.rows <= 16 * groups) return 16;
    return f8_tiles_of(s, 32) * f8_row_groups(s) * s.kb <= 13000 ? 32 : 0;
}

// Whether the stream kernel quantizes values itself: each wave does so for the
// blocks it takes, which saves the quantizer's launch (2.5 us, and 5 of the
// host's) and costs every work-group its share: up to 32 MB of weights (4096 x
// 4096, one row: 8.0 us for 8.7; 5120 x 17408, one row: 29 for 22).
inline bool f8_stream_quantizes(const F8Sizes &s) {
    const long long used = s.groups ? std::min(s.rows, s.groups) : 1;
    return used * f8_row_groups(s) * s.kb <= (32ll << 20) / 2048;
}

// The same in tiles of 32 rows, of x_bytes a value: where the four waves hold all
// blocks of FP32 rows in flight (BF16: half of them), and the work-groups' reads of
// the same rows are few. Launches of both, then of one, replayed / called in turn:
// FP32, 256 rows, 1,024 x 1,024: 8.9 / 12.0, then 9.6 / 8.1; 200, 768 -> 1,024: 8.7 /
// 12.2, 9.0 / 8.0; 150 x 3 rows over 5 experts, 208 -> 336: 8.2 / 12.2, 6.6 / 8.7;
// past it 64 rows, 2,048 x 2,048: 9.9 / 11.8, 12.8 / 11.1; 97, 1,456 -> 2,064: 11.5 /
// 11.9, 14.4 / 12.9. BF16, 97 rows, 1,456 -> 2,064: 11.4 / 11.8, 11.5 / 9.9; 64 x 4
// over 8, 1,024 x 1,024: 11.4 / 12.5, 10.9 / 9.2; past it 32 rows, 4,096 x 4,096:
// 12.8 / 11.8, 14.4 / 12.9.
inline bool f8_stream32_quantizes(const F8Sizes &s, int x_bytes) {
    return s.kb * x_bytes <= 32 && f8_tiles_of(s, 32) * f8_row_groups(s) * s.kb * x_bytes <= 17500;
}

// A stream work-group's row-groups and waves, for tiles of `rows` rows: two
// row-groups, or one where they do not fill the CUs; four waves, or eight for long
// sums of few work-groups (codes, one row: 5120 x 17408 19 us for 25, 17408 x 5120
// 33 for 35, 4096 x 4096 6.2 either way).
struct F8StreamShape {
    int row_groups, waves;
};
inline F8StreamShape f8_stream_shape(const F8Sizes &s, int rows) {
    const long long rgs = f8_tiles_of(s, rows) * f8_row_groups(s);
    if (rgs <= s.cus) return {1, 4};
    return {2, s.kb >= 64 && rgs < 4ll * s.cus ? 8 : 4};
}

// The tiles of the dense launch and what a step (128 columns) of one takes, in
// us: with up to half of the card's places taken, and with all (there the power
// limit and the L2 count too).
struct F8Config {
    int id, bt, br, per_cu;
    double alone, full;
};
constexpr F8Config kF8Fast[] = {{0, 256, 256, 1, 1.35, 1.60}, {1, 256, 128, 1, 0.75, 1.05}, {2, 128, 128, 1, 0.60, 0.75}, {3, 64, 128, 2, 0.49, 0.80}};
constexpr F8Config kF8Exact[] = {{4, 128, 128, 2, 1.18, 2.15}, {5, 64, 128, 2, 0.63, 1.02}};

struct F8Choice {
    int id, splits;                                          // tile, parts of the sum over the columns
    double us;
};

// A launch is rounds of work-groups over the card's places, each its steps and
// 5 us of start and end; parts are written and read again by a second launch.
inline F8Choice f8_choose(const F8Sizes &s) {
    const F8Config *cs = s.bf16 ? kF8Fast : kF8Exact;
    const int n = s.bf16 ? 4 : 2;
    long long outputs = 0;
    for (int i = 0; i < s.count; ++i) outputs += (long long)s.rows * s.M[i];
    F8Choice best{cs[0].id, 1, 0.0};
    for (int c = 0; c < n; ++c) {
        long long tiles = 0;
        for (int i = 0; i < s.count; ++i) tiles += (s.M[i] + cs[c].br - 1) / cs[c].br;
        tiles *= (s.rows + cs[c].bt - 1) / cs[c].bt;
        const long long places = (long long)s.cus * cs[c].per_cu;
        for (int S = 1; S <= 8; ++S) {
            // (parts of four steps at least, in one round)
            if (S > 1 && (tiles * S > places || s.kb / S < 4)) break;
            const double steps = (s.kb + S - 1) / S;
            const long long items = tiles * S, rounds = items / places, rest = items % places;
            double us = (double)rounds * (steps * cs[c].full + 5.0);
            // (two work-groups on one CU hold the round up as much as on all)
            const double busy = cs[c].per_cu > 1 ? (rest > s.cus ? 1.0 : 0.0) : std::max(0.0, 2.0 * (double)rest / (double)places - 1.0);
            if (rest) us += steps * (cs[c].alone + (cs[c].full - cs[c].alone) * busy) + 5.0;
            if (S > 1) us += 3.0 + (double)outputs * (8.0 * S + 4.0) / 4.5e6;
            if (best.us == 0.0 || us < best.us) best = F8Choice{cs[c].id, S, us};
        }
    }
    return best;
}

// Tiles of rows sorted by group: 64 rows x 128, two a CU, or with 128 rows a group
// and more 128 x 256 (BF16) and 128 x 128 (FP32). Rows x k over groups, K, M:
// 1,000 x 4 over 64, 2048, 1024: 42 us for 48 (FP32 48 for 50); 256 x 8 over 64,
// 5120, 1024: 84 for 98 (89 for 94); 2,048 x 8 over 64, 5120, 1024: 181 for 137
// (249 for 247); 4,000 x 2 over 8, 4096, 2048: 122 for 99 (170 for 158). Rows
// without a group count, since the host knows no better.
inline bool f8_long_groups(const F8Sizes &s) { return s.rows >= 128ll * s.groups; }

}  // namespace kxw4
