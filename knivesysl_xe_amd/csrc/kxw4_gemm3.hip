// kxw4_gemm3.hip — launches of the large-tile kernel (kxw4_gemm3.hpp) and the
// choice of its tile.
#include "kxw4_gemm3.hpp"

#include <algorithm>

namespace kxw4 {

constexpr int kG3GroupTT = 4;      // token tiles per raster group (option gemm3_raster)

template <int TA, int TB, int WMW, int WNW, int UNIT, int NST, int OCC = 2, int XB = 0>
static int launch_g3(GemmArgs &a, hipStream_t st) {
    using S = G3Shape<TA, TB, WMW, WNW, UNIT, XB>;
    int nt = 0;
    for (int i = 0; i < a.count; ++i) {
        a.w[i].nt_begin = nt;
        nt += (a.w[i].M / 16 + S::BNG - 1) / S::BNG;
    }
    a.n_tiles = nt;
    a.t_tiles = (a.T + S::BM - 1) / S::BM;
    a.raster_tt = options().gemm3_raster > 0 ? options().gemm3_raster : kG3GroupTT;
    const dim3 grid(a.n_tiles * a.t_tiles), block(S::NTH);
    auto k = gemm3_kernel<TA, TB, WMW, WNW, UNIT, NST, OCC, XB>;
    const size_t lds = (size_t)S::template lds_bytes<NST>();
    // the attribute is per device
    static bool attr[64] = {};
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return -6;
    if (!attr[dev]) {
        if (hipFuncSetAttribute((const void *)k, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) != hipSuccess)
            return -6;
        attr[dev] = true;
    }
    hipLaunchKernelGGL(k, grid, block, lds, st, a);
    return hipGetLastError() == hipSuccess ? 0 : -6;
}

// Tile choice. Per SIMD the kernel is bound by the FP32 chain of its
// blocks, so each candidate is scored by the rounds of work-groups it needs
// over the CUs times the 32x32 blocks per K step its busiest SIMD carries
// per round (waves on that SIMD x blocks per wave); the small tile pays ~10%
// for its larger L2 traffic per MAC (measured):
//   256 x 256, 8 waves (2 per SIMD, 8 blocks each), one work-group per CU;
//   256 x 160 (G128) / 64 x 160 (G64), 10 waves (3 on the busiest SIMD),
//     one work-group per CU: fits the grid when the 256-row tile leaves
//     CUs idle;
//   256 x 160 at G128 as 8 waves of 4 + 1 blocks (each wave's four blocks
//     of its own 32-row column and one block of the fifth column): 10 blocks
//     on every SIMD (the waves of a work-group go to the SIMDs in turn, so
//     ten one-column waves put 12 on two SIMDs and 8 on the others);
//   128 x 64, 4 waves of 2 blocks, three work-groups per CU;
//   128 x 256 (G128), 4 waves of 8 blocks, two work-groups per CU: the same
//     16 blocks per SIMD and step as 256 x 256, but a SIMD's two waves
//     belong to different work-groups and never wait for each other at the
//     step barrier (with one 8-wave work-group the older wave of each SIMD
//     finishes its step ~1,700 cycles early and idles): 8% faster on cfg4
//     (measured), so it is preferred at an equal number of rounds.
static int choose_tile(const GemmArgs &a, int *bm) {
    const bool g128 = a.group == 128;
    struct Cand { int sel, bm, bng, wgs, simd_blocks; double penalty; };
    const Cand cands[4] = {
        {0, 256, g128 ? 16 : 8, 1, g128 ? 16 : 8, 1.0},
        {g128 ? 11 : 8, g128 ? 256 : 64, 10, 1, g128 ? 10 : 3, 1.0},
        {g128 ? 3 : 4, 128, 4, 3, 6, 1.1},
        {1, 128, 16, 2, 16, 0.92},
    };
    const long long cus = device_cus();
    double best = 0.0;
    int sel = -1;
    for (const Cand &c : cands) {
        if (c.sel == 1 && !g128) continue;                   // (tile 1 is 128 x 128 at G64)
        long long nt = 0;
        for (int i = 0; i < a.count; ++i) nt += (a.w[i].M / 16 + c.bng - 1) / c.bng;
        const long long tiles = nt * ((a.T + c.bm - 1) / c.bm);
        const long long rounds = (tiles + cus * c.wgs - 1) / (cus * c.wgs);
        const double cost = (double)rounds * c.simd_blocks * c.penalty;
        if (sel < 0 || cost < best) {
            best = cost;
            sel = c.sel;
            *bm = c.bm;
        }
    }
    return sel;
}

static int launch_tile(GemmArgs &a, int sel, hipStream_t st);

int launch_gemm3(GemmArgs &a, hipStream_t st) {
    // per-token activation scale, plain FP16 weight scales, one split per token
    if (a.block != 0 || a.scale_enc != 0 || (a.group != 64 && a.group != 128)) return 1;
    if ((long long)a.T * a.K >= (1ll << 31)) return 1;          // 32-bit activation offsets
    for (int i = 0; i < a.count; ++i) {
        if ((long long)a.w[i].M * a.K / 2 >= (1ll << 31)) return 1;
        for (int s = 0; s < a.seg_count; ++s)
            if (a.w[i].seg_split[s] != 1) return 1;
    }
    // the gemm3_tile option (0..11) picks one configuration (tests, tuning)
    const int forced = options().gemm3_tile;
    if (forced >= 0) return launch_tile(a, forced, st);
    int bm = 0;
    const int sel = choose_tile(a, &bm);
    return launch_tile(a, sel, st);
}

static int launch_tile(GemmArgs &a, int sel, hipStream_t st) {
    if (a.group == 128) {
        switch (sel) {
        case 8: return launch_g3<4, 1, 2, 5, 128, 3, 3>(a, st);   // 256 x 160, 10 waves
        case 10: return launch_g3<4, 1, 2, 4, 128, 3, 2, 1>(a, st);  // 256 x 160, 8 waves of 4 + 1 blocks
        case 11: return launch_g3<4, 1, 2, 4, 128, 2, 2, 1>(a, st);  // the same, 2 stages
        case 9: return launch_g3<4, 1, 2, 5, 128, 2, 3>(a, st);   // 256 x 160, 10 waves, 2 stages
        case 5: return launch_g3<2, 2, 2, 2, 128, 3, 2>(a, st);   // 128 x 128, 4 waves
        case 6: return launch_g3<2, 2, 1, 4, 128, 3, 2>(a, st);   // 64 x 256, 4 waves
        case 7: return launch_g3<1, 2, 2, 2, 128, 3, 3>(a, st);   // 64 x 128, 4 waves, three per CU
        case 1: return launch_g3<4, 2, 1, 4, 128, 2>(a, st);      // 128 x 256, 4 waves, two per CU
        case 2: return launch_g3<4, 2, 2, 4, 128, 2>(a, st);      // 256 x 256, 8 waves, 2 stages
        case 3: return launch_g3<2, 1, 2, 2, 128, 2, 3>(a, st);   // 128 x 64, 4 waves, three per CU
        default: return launch_g3<4, 2, 2, 4, 128, 3>(a, st);     // 256 x 256, 8 waves, 3 stages
        }
    }
    // group 64: two chain updates per block and step
    switch (sel) {
    case 8: return launch_g3<1, 1, 2, 5, 64, 3, 3>(a, st);        // 64 x 160, 10 waves
    case 9: return launch_g3<2, 1, 2, 5, 64, 3, 3>(a, st);        // 128 x 160, 10 waves
    case 5: return launch_g3<2, 2, 2, 2, 64, 2, 2>(a, st);        // 128 x 128, 4 waves
    case 6: return launch_g3<2, 1, 1, 4, 64, 3, 2>(a, st);        // 64 x 128, 4 waves
    case 7: return launch_g3<1, 2, 2, 2, 64, 3, 3>(a, st);        // 64 x 128, 4 waves, three per CU
    case 1: return launch_g3<4, 1, 1, 4, 64, 2>(a, st);           // 128 x 128, 4 waves
    case 2: return launch_g3<2, 2, 2, 4, 64, 2>(a, st);           // 128 x 256, 8 waves
    case 4: return launch_g3<2, 1, 2, 2, 64, 2, 3>(a, st);        // 128 x 64, 4 waves, three per CU
    default: return launch_g3<4, 1, 2, 4, 64, 3>(a, st);          // 256 x 128, 8 waves
    }
}

}  // namespace kxw4
