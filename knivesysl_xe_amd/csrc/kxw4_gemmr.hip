// kxw4_gemmr.hip — launches of the reference-mode large-tile kernel
// (kxw4_gemmr.hpp) and the choice of its tile.
#include "kxw4_gemmr.hpp"
#include "kxw4_route.hpp"

#include <algorithm>

namespace kxw4 {

constexpr int kGrGroupTT = 4;      // token tiles per raster group

template <int NT, int WR, int WT, int GROUP, bool ZP, int NST, int OCC>
static int launch_gr(GemmArgs &a, hipStream_t st) {
    using S = GrShape<NT, WR, WT, GROUP>;
    int nt = 0;
    for (int i = 0; i < a.count; ++i) {
        a.w[i].nt_begin = nt;
        nt += (a.w[i].M / 16 + S::RGS - 1) / S::RGS;
    }
    a.n_tiles = nt;
    a.t_tiles = (a.T + S::BM - 1) / S::BM;
    a.raster_tt = kGrGroupTT;
    const dim3 grid(a.n_tiles * a.t_tiles), block(S::NTH);
    auto k = gemmr_kernel<NT, WR, WT, GROUP, ZP, NST, OCC>;
    const size_t lds = (size_t)S::template lds_bytes<NST>();
    static_assert(S::template lds_bytes<NST>() <= 160 * 1024, "LDS");
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

// Tiles (wave tile 32 rows x 32*NT tokens). The kernel is bound by each
// SIMD's VALU issue and, nearly as much, by the CU's LDS reads (a wave's
// scales and operands cost ~37 LDS cycles per 32x32 block and unit against
// ~33 of VALU per SIMD), so what decides is how evenly the blocks spread over
// the SIMDs, how many waves share a SIMD and how many token blocks share the
// scales (graph replay, bit-exact, T=2048 K=N=5120 group 32 / T=512 K=17408
// N=5120 group 64):
//   4: 128 x 64, 4 waves of 2 token blocks, four work-groups per CU:
//     191 / 264 us;
//   9: 128 x 32, 4 waves of one token block: 217 / 234 us (4 or 9, whichever
//     loads the busiest CU less: gemmr_wide in kxw4_route.hpp);
//   0: 160 x 256, 10 waves of 4 token blocks (3, 3, 2, 2 per SIMD), one
//     work-group per CU: 187 / 586 us;
//   5: 160 x 64, 10 waves of one token block: 281 / 221 us;
//   1, 2, 3, 6, 7, 8: 4- and 5-wave tiles with 4 token blocks, and lean
//     (one MFMA result live) tiles at 5 or 6 waves per SIMD: all slower.
// The scales are read as FP32, converted once per stage: a product is then a
// plain multiplication at twice the rate of v_fma_mix_f32 on FP16 pairs (rate
// probe, four waves per SIMD: 1.15 against 1.94 ns), 205 -> 194 us; the
// fourth wave per SIMD (no second set of scale registers) 194 -> 191 us.
template <int GROUP, bool ZP>
static int launch_gr_tile(GemmArgs &a, int sel, hipStream_t st) {
    switch (sel) {
    case 0: return launch_gr<4, 5, 2, GROUP, ZP, 3, 3>(a, st);    // 160 rows x 256 tokens, 10 waves
    case 1: return launch_gr<4, 4, 1, GROUP, ZP, 2, 3>(a, st);    // 128 rows x 128 tokens, 4 waves
    case 2: return launch_gr<4, 5, 1, GROUP, ZP, 2, 3>(a, st);    // 160 rows x 128 tokens, 5 waves
    case 3: return launch_gr<2, 5, 2, GROUP, ZP, 3, 3>(a, st);    // 160 rows x 128 tokens, 10 waves
    case 5: return launch_gr<1, 5, 2, GROUP, ZP, 3, 3>(a, st);    // 160 rows x 64 tokens, 10 waves
    case 6: return launch_gr<2, 5, 1, GROUP, ZP, 2, 5>(a, st);    // 160 rows x 64 tokens, 5 waves, lean
    case 7: return launch_gr<1, 4, 2, GROUP, ZP, 2, 6>(a, st);    // 128 rows x 64 tokens, 8 waves, lean
    case 8: return launch_gr<2, 4, 1, GROUP, ZP, 2, 5>(a, st);    // 128 rows x 64 tokens, 4 waves, lean
    case 9: return launch_gr<1, 4, 1, GROUP, ZP, 2, 4>(a, st);    // 128 rows x 32 tokens, 4 waves
    default: return launch_gr<2, 4, 1, GROUP, ZP, 2, 4>(a, st);   // 128 rows x 64 tokens, 4 waves (4)
    }
}

int launch_gemmr(GemmArgs &a, hipStream_t st) {
    // activation scales per (token, K32 block), one split per token, W4 codes
    if (a.block != 32 || a.w8 || (a.group != 32 && a.group != 64 && a.group != 128)) return 1;
    if (a.scale_enc == 1 && a.group == 128) return 1;
    if ((long long)a.T * a.K >= (1ll << 31)) return 1;               // 32-bit activation offsets
    for (int i = 0; i < a.count; ++i) {
        if ((long long)a.w[i].M * a.K / 2 >= (1ll << 31)) return 1;
        for (int s = 0; s < a.seg_count; ++s)
            if (a.w[i].seg_split[s] != 1) return 1;
    }
    int sel = options().gemmr_tile;
    if (sel < 0) {
        long long rows = 0;                                          // 128-row tiles
        for (int i = 0; i < a.count; ++i) rows += (a.w[i].M / 16 + 7) / 8;
        sel = gemmr_wide(device_cus(), rows, a.T) ? 4 : 9;
    }
    const bool zp = a.scale_enc == 1;
    switch (a.group) {
    case 32: return zp ? launch_gr_tile<32, true>(a, sel, st) : launch_gr_tile<32, false>(a, sel, st);
    case 64: return zp ? launch_gr_tile<64, true>(a, sel, st) : launch_gr_tile<64, false>(a, sel, st);
    default: return launch_gr_tile<128, false>(a, sel, st);
    }
}

}  // namespace kxw4
