// kxw4_experts.hip — projections whose weight depends on the row: the rows of
// a batch sorted by expert (kxw4_rows.hip), each expert's rows against its own
// slice of the stacked weights. No counterpart in the reference, whose model
// is dense. The arithmetic of a row is that of kxw4_gemm under the split count
// chosen here.
#include "kxw4_strip.hpp"

#include <algorithm>

namespace kxw4 {

template <int TT, int RW, int U, int UNIT, bool BLK, int WF>
static int ex_launch(StripArgs &a, int S, int N, hipStream_t st) {
    using SH = StShape<TT, RW, U, BLK, WF>;
    a.waves = RW > 1 ? S * RW : std::min(S, 8);
    int blk = 0;
    for (int i = 0; i < a.entries; ++i) {
        a.e[i] = StripEntry{i, 0, 0, S, blk};
        blk += (a.w[i].M / 16 + RW - 1) / RW;
    }
    a.row_blocks = blk;
    a.same_s = 1;
    const long long grid = tiles_at_most(N, a.groups, TT) * blk;
    if (grid >= (1ll << 31)) return -2;
    const size_t lds = std::max((size_t)2 * (RW == 1 ? a.waves : S) * SH::STAGE, (size_t)std::max(2 * a.waves, RW) * SH::NT * 1024);
    if (lds > 160 * 1024 || a.waves > 8) return -2;          // (the rules below never ask for it)
    auto k = strip_kernel<TT, RW, U, UNIT, BLK, kVarGemm, WF, true>;
    static bool attr[64] = {};                               // (the attribute is per device)
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return -6;
    if (!attr[dev]) {
        if (hipFuncSetAttribute(reinterpret_cast<const void *>(k), hipFuncAttributeMaxDynamicSharedMemorySize,
                                160 * 1024) != hipSuccess)
            return -6;
        attr[dev] = true;
    }
    hipLaunchKernelGGL(k, dim3((unsigned)grid), dim3(64 * a.waves), lds, st, a);
    return hipGetLastError() == hipSuccess ? 0 : -6;
}

template <int UNIT, bool BLK, int WF>
static int ex_shape(StripArgs &a, int TT, int S, int N, hipStream_t st) {
    if (S == 1) {
        switch (TT) {
        case 1: return ex_launch<1, 4, 2, UNIT, BLK, WF>(a, S, N, st);
        case 2: return ex_launch<2, 4, 2, UNIT, BLK, WF>(a, S, N, st);
        case 8: return ex_launch<8, 4, 2, UNIT, BLK, WF>(a, S, N, st);
        case 16: return ex_launch<16, 4, 2, UNIT, BLK, WF>(a, S, N, st);
        default: return ex_launch<32, 4, 2, UNIT, BLK, WF>(a, S, N, st);
        }
    }
    switch (TT) {
    case 1: return ex_launch<1, 1, 2, UNIT, BLK, WF>(a, S, N, st);
    case 2: return ex_launch<2, 1, 2, UNIT, BLK, WF>(a, S, N, st);
    case 8: return ex_launch<8, 1, 2, UNIT, BLK, WF>(a, S, N, st);
    default: return ex_launch<16, 1, 2, UNIT, BLK, WF>(a, S, N, st);
    }
}

int launch_experts(const ExpertArgs &x, hipStream_t st) {
    StripArgs a{};
    int rgs = 0;
    for (int i = 0; i < x.count; ++i) {
        a.w[i] = x.w[i];
        rgs += x.w[i].M / 16;
    }
    a.entries = x.count;
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
    const int each = x.N / std::min(x.groups, x.N);          // rows of an expert, spread evenly
    const int TT = x.N == 1 ? 1 : each <= 2 ? 2 : each <= 8 ? 8 : each <= 32 ? 16 : 32;
    const long long strips = tiles_at_most(x.N, x.groups, TT) * rgs;
    int S = 1;
    while (TT < 32 && S < 8 && strips * S < 2048 && 2 * S <= x.K / kTileK) S *= 2;
    if (x.scale_enc == 2) return ex_shape<32, true, kStW8>(a, TT, S, x.N, st);
    if (x.block == 32) return ex_shape<32, true, kStW4>(a, TT, S, x.N, st);
    if (x.group == 128) return ex_shape<128, false, kStW4>(a, TT, S, x.N, st);
    return ex_shape<64, false, kStW4>(a, TT, S, x.N, st);
}

}  // namespace kxw4
