// kxw4_experts.hip — projections whose weight depends on the row: the rows of
// a batch sorted by expert (kxw4_rows.hip), each expert's rows against its own
// slice of the stacked weights. No counterpart in the reference, whose model
// is dense. The arithmetic of a row is that of kxw4_gemm under the split count
// of expert_splits (one on the large tiles).
//
// Grouped instances of the strip kernel and of the two large-tile kernels do
// the work; a work-group finds its expert and tile from the plan's offsets
// (kxw4_groups.hpp), and the activations are read through the plan's order, so
// no copy of them is made. What bounds them: with few rows an expert, reading
// the weights (128 rows over 64 experts, 2 x 1,024 rows, K = 5120: 46.7 us for
// 300 MB, 6.4 TB/s, a pure read's rate); with many, the large tiles' FP32 chain
// beside the MFMAs, the power limit and the last round of work-groups (16,384
// rows: 227 us, 1.51 POPS; strips 402 us; with K32 blocks the chain, three VALU
// operations per output and unit, x 1,024 rows 333 us, 0.52 POPS; strips 403).
#include "kxw4_gemm3.hpp"
#include "kxw4_gemmr.hpp"
#include "kxw4_route.hpp"
#include "kxw4_strip.hpp"

#include <algorithm>

namespace kxw4 {

// Allow `k` as much dynamic LDS as it asks for, once per device.
static int ex_lds(const void *k, size_t lds, bool (&done)[64]) {
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return -6;
    if (done[dev]) return 0;
    if (hipFuncSetAttribute(k, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) != hipSuccess) return -6;
    done[dev] = true;
    return 0;
}

// Strips of TT places. One split: four row waves share a tile's activations;
// several: one row wave per split.
template <int TT, int RW, int UNIT, bool BLK, int WF>
static int ex_strips(const ExpertArgs &x, int S, hipStream_t st) {
    constexpr int U = 2;
    using SH = StShape<TT, RW, U, BLK, WF>;
    StripArgs a{};
    int blk = 0;
    for (int i = 0; i < x.count; ++i) {
        a.w[i] = x.w[i];
        a.e[i] = StripEntry{i, 0, 0, S, blk};
        blk += (x.w[i].M / 16 + RW - 1) / RW;
    }
    a.entries = x.count;
    a.row_blocks = blk;
    a.waves = S * RW;
    a.same_s = 1;
    a.q = x.q;
    a.ascale = x.ascale;
    a.K = x.K;
    a.group = x.group;
    a.block = x.block;
    a.scale_enc = x.scale_enc;
    a.y_bf16 = x.y_bf16;
    a.variant = kVarGemm;
    a.offsets = x.offsets;
    a.order = x.order;
    a.groups = x.groups;
    a.k = x.k;
    const long long grid = tiles_at_most(x.N, x.groups, TT) * blk;
    if (grid > grid_limit(64 * a.waves)) return -2;
    const size_t lds = std::max((size_t)2 * S * SH::STAGE, (size_t)std::max(2 * a.waves, RW) * SH::NT * 1024);
    if (lds > 160 * 1024 || a.waves > 8) return -2;          // (expert_splits never asks for it)
    auto k = strip_kernel<TT, RW, U, UNIT, BLK, kVarGemm, WF, true>;
    static bool done[64] = {};
    const int rc = ex_lds(reinterpret_cast<const void *>(k), 160 * 1024, done);
    if (rc) return rc;
    hipLaunchKernelGGL(k, dim3((unsigned)grid), dim3(64 * a.waves), lds, st, a);
    return hipGetLastError() == hipSuccess ? 0 : -6;
}

template <int UNIT, bool BLK, int WF>
static int ex_shape(const ExpertArgs &x, int TT, hipStream_t st) {
    long long rgs = 0;
    for (int i = 0; i < x.count; ++i) rgs += x.w[i].M / 16;
    const int S = TT == 32 ? 1 : expert_splits(tiles_at_most(x.N, x.groups, TT) * rgs, x.K / kTileK);
    switch (TT) {
    case 2: return S == 1 ? ex_strips<2, 4, UNIT, BLK, WF>(x, S, st) : ex_strips<2, 1, UNIT, BLK, WF>(x, S, st);
    case 8: return S == 1 ? ex_strips<8, 4, UNIT, BLK, WF>(x, S, st) : ex_strips<8, 1, UNIT, BLK, WF>(x, S, st);
    case 16: return S == 1 ? ex_strips<16, 4, UNIT, BLK, WF>(x, S, st) : ex_strips<16, 1, UNIT, BLK, WF>(x, S, st);
    default:
        if constexpr (BLK) return ex_strips<32, 4, UNIT, BLK, WF>(x, S, st);
        else return -2;                                      // (per token the large tiles take these)
    }
}

// The arguments of a large-tile launch whose tiles have `rgs` row-groups.
static GemmArgs ex_args(const ExpertArgs &x, int rgs) {
    GemmArgs a{};
    int nt = 0;
    for (int i = 0; i < x.count; ++i) {
        a.w[i].codes = x.w[i].codes;
        a.w[i].scales = x.w[i].scales;
        a.w[i].y = x.w[i].y;
        a.w[i].M = x.w[i].M;
        a.w[i].nt_begin = nt;
        nt += (x.w[i].M / 16 + rgs - 1) / rgs;
    }
    a.count = x.count;
    a.q = x.q;
    a.ascale = x.ascale;
    a.T = x.N;
    a.K = x.K;
    a.group = x.group;
    a.y_bf16 = x.y_bf16;
    a.n_tiles = nt;
    a.offsets = x.offsets;
    a.order = x.order;
    a.groups = x.groups;
    a.k = x.k;
    a.rows = x.rows;
    return a;
}

// Tiles of 32 TA places x 32 TB WNW rows of the large-tile kernel.
template <int TA, int TB, int WNW, int UNIT, int NST, int OCC>
static int ex_tiles(const ExpertArgs &x, hipStream_t st) {
    using S = G3Shape<TA, TB, 1, WNW, UNIT, 0>;
    const GemmArgs a = ex_args(x, S::BNG);
    const long long grid = tiles_at_most(x.N, x.groups, S::BM) * a.n_tiles;
    if (grid > grid_limit(S::NTH)) return -2;
    auto k = gemm3_group_kernel<TA, TB, WNW, UNIT, NST, OCC>;
    // (the shorter tiles' output staging may take more than their stages)
    const size_t lds = std::max({S::template lds_bytes<NST>(), G3Shape<(TA > 1 ? TA / 2 : 1), TB, 1, WNW, UNIT, 0>::template lds_bytes<NST>(),
                                 G3Shape<1, TB, 1, WNW, UNIT, 0>::template lds_bytes<NST>()});
    static bool done[64] = {};
    const int rc = ex_lds(reinterpret_cast<const void *>(k), lds, done);
    if (rc) return rc;
    hipLaunchKernelGGL(k, dim3((unsigned)grid), dim3(S::NTH), lds, st, a);
    return hipGetLastError() == hipSuccess ? 0 : -6;
}

// Tiles of 64 places x 128 rows of the reference-mode kernel.
template <int GROUP>
static int ex_blocks(const ExpertArgs &x, hipStream_t st) {
    constexpr int NST = 2;
    using S = GrShape<2, 4, 1, GROUP>;
    const GemmArgs a = ex_args(x, S::RGS);
    const long long grid = tiles_at_most(x.N, x.groups, S::BM) * a.n_tiles;
    if (grid > grid_limit(S::NTH)) return -2;
    auto k = gemmr_group_kernel<GROUP, NST, 4>;
    const size_t lds = std::max(S::template lds_bytes<NST>(), GrShape<1, 4, 1, GROUP>::template lds_bytes<NST>());
    static bool done[64] = {};
    const int rc = ex_lds(reinterpret_cast<const void *>(k), lds, done);
    if (rc) return rc;
    hipLaunchKernelGGL(k, dim3((unsigned)grid), dim3(S::NTH), lds, st, a);
    return hipGetLastError() == hipSuccess ? 0 : -6;
}

int launch_experts(const ExpertArgs &x, hipStream_t st) {
    ExpertShape s{device_cus(), x.N, x.groups, x.group, 0, 0, x.block != 0, x.scale_enc == 2};
    for (int i = 0; i < x.count; ++i) {
        s.rows128 += (x.w[i].M + 127) / 128;
        s.rows256 += (x.w[i].M + 255) / 256;
    }
    const int route = expert_route(s);
    if (s.w8) return ex_shape<32, true, kStW8>(x, route, st);
    if (route == kExpertBlock64) return x.group == 32 ? ex_blocks<32>(x, st) : ex_blocks<64>(x, st);
    if (s.blocks) return ex_shape<32, true, kStW4>(x, route, st);
    if (x.group == 128) {
        switch (route) {
        case kExpertTile32: return ex_tiles<1, 1, 4, 128, 3, 3>(x, st);
        case kExpertTile64: return ex_tiles<2, 2, 4, 128, 3, 2>(x, st);
        case kExpertTile128: return ex_tiles<4, 2, 4, 128, 2, 2>(x, st);
        default: return ex_shape<128, false, kStW4>(x, route, st);
        }
    }
    switch (route) {
    case kExpertTile32: return ex_tiles<1, 1, 4, 64, 3, 3>(x, st);
    case kExpertTile64: return ex_tiles<2, 2, 4, 64, 2, 2>(x, st);
    default: return ex_shape<64, false, kStW4>(x, route, st);
    }
}

}  // namespace kxw4
