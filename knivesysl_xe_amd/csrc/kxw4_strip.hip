// kxw4_strip.hip — launches of the strip kernel (kxw4_strip.hpp): tile
// shapes, waves and split streams by the sizes of a projection's entries.
#include "kxw4_strip.hpp"

#include <algorithm>

namespace kxw4 {

template <int TT, int RW, int U, int UNIT, bool BLK, int VAR, int WF>
static int st_launch(StripArgs &a, hipStream_t st) {
    using S = StShape<TT, RW, U, BLK, WF>;
    int smax = 1;
    for (int i = 0; i < a.entries; ++i) smax = std::max(smax, a.e[i].S);
    a.waves = RW > 1 ? smax * RW : a.same_s ? std::min(smax, 8) : smax >= 8 ? 8 : 4;
    auto blocks = [&]() {
        int blk = 0;
        for (int i = 0; i < a.entries; ++i) {
            a.e[i].blk = blk;
            const int rows = RW == 1 ? a.waves / std::min(a.e[i].S, a.waves) : RW;   // row-groups per block
            blk += ((a.e[i].t1 - a.e[i].t0 + TT - 1) / TT) * ((a.w[a.e[i].w].M / 16 + rows - 1) / rows);
        }
        return blk;
    };
    int blk = blocks();
    // Eight streams while every work-group is resident at once, else four
    // that take their splits in turn.
    if (RW == 1 && smax == 8 && blk > device_cus() * (160 * 1024 / (16 * S::STAGE))) {
        a.waves = 4;
        blk = blocks();
    }
    const size_t lds = std::max((size_t)2 * (RW == 1 ? a.waves : smax) * S::STAGE, (size_t)std::max(2 * a.waves, RW) * S::NT * 1024);
    if (lds > 160 * 1024 || a.waves > 8) return -2;          // (the rules below never ask for it)
    auto k = strip_kernel<TT, RW, U, UNIT, BLK, VAR, WF>;
    static bool attr[64] = {};                               // (the attribute is per device)
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return -6;
    if (!attr[dev]) {
        if (hipFuncSetAttribute(reinterpret_cast<const void *>(k), hipFuncAttributeMaxDynamicSharedMemorySize,
                                160 * 1024) != hipSuccess)
            return -6;
        attr[dev] = true;
    }
    hipLaunchKernelGGL(k, dim3(blk), dim3(64 * a.waves), lds, st, a);
    return hipGetLastError() == hipSuccess ? 0 : -6;
}

// Row waves per work-group and tiles per stage. S = 1: four row waves share
// the activations; with 16-token tiles and a grid of at most one and a half
// work-groups per CU, four tiles per stage, since nothing else hides a
// stage's barrier and LDS latency (per-token N = 5120, K = 17408, T = 64:
// 37.6 -> 32.6 us; with more work-groups the LDS they take costs more than
// that: block mode N = 17408, K = 5120, T = 32: 31.7 -> 37.4 us). S > 1: one
// row wave per stream (T = 16, N = 5120, K = 17408, S = 4: 14.2 against 17.5
// us per-token and 22.2 against 24.4 us in block mode for two), two for W8
// past 16 tokens, whose tiles are twice as large (T = 48: 37.0 against 46 us).
template <int TT, int UNIT, bool BLK, int VAR, int WF>
static int st_rw(StripArgs &a, int T, int smax, hipStream_t st) {
    if constexpr (TT == 32 && VAR == kVarFanout) {          // (planned with 1, 8 or 16 splits)
        return st_launch<TT, 4, 2, UNIT, BLK, VAR, WF>(a, st);
    } else if constexpr (TT == 32) {
        return smax <= 2 ? st_launch<TT, 4, 2, UNIT, BLK, VAR, WF>(a, st) : st_launch<TT, 2, 2, UNIT, BLK, VAR, WF>(a, st);
    } else {
        if (smax == 1) {
            if constexpr (TT == 16) {
                long long blks = 0;
                for (int i = 0; i < a.entries; ++i)
                    blks += (long long)((a.e[i].t1 - a.e[i].t0 + 15) / 16) * ((a.w[a.e[i].w].M / 16 + 3) / 4);
                if (2 * blks <= 3LL * device_cus()) return st_launch<TT, 4, 4, UNIT, BLK, VAR, WF>(a, st);
            }
            return st_launch<TT, 4, 2, UNIT, BLK, VAR, WF>(a, st);
        }
        if constexpr (TT == 16 && WF == kStW8 && VAR == kVarGemm) {
            if (smax <= 4 && a.same_s && T > 16) return st_launch<TT, 2, 2, UNIT, BLK, VAR, WF>(a, st);
        }
        return st_launch<TT, 1, 2, UNIT, BLK, VAR, WF>(a, st);
    }
}

// Whether the entries of split count SC fill 32-token tiles: these share a
// row-group's unpack and scales between two blocks and
// pay once the 16-token ones fill the SIMDs four times over (W8, with no
// unpack but twice the weight bytes: twice) and their padding costs less than
// that (a 32-token strip takes 1.6 times a 16-token one).
static bool st_fills_32(const StripArgs &a, int SC, int per_simd) {
    long long strips16 = 0, strips32 = 0;
    for (int i = 0; i < a.entries; ++i) {
        if (a.e[i].S != SC) continue;
        const long long t = a.e[i].t1 - a.e[i].t0, rgs = a.w[a.e[i].w].M / 16;
        strips16 += rgs * ((t + 15) / 16);
        strips32 += rgs * ((t + 31) / 32);
    }
    return strips16 * SC > per_simd && 5 * strips16 > 8 * strips32;
}

// The entries of `a` that `pick` names, taken out of it.
template <class F>
static StripArgs st_take(StripArgs &a, F pick) {
    StripArgs own = a;
    int left = 0;
    own.entries = 0;
    for (int i = 0; i < a.entries; ++i) {
        if (pick(a.e[i])) own.e[own.entries++] = a.e[i];
        else a.e[left++] = a.e[i];
    }
    a.entries = left;
    return own;
}

template <int UNIT, bool BLK, int VAR, int WF>
static int st_shape(StripArgs &a, hipStream_t st) {
    constexpr int kFill = WF == kStW8 ? 2000 : 4400;
    constexpr bool k32 = WF == kStW4 || (WF == kStW8 && VAR == kVarGemm);   // (K16 and the W8 GEMV: 16 tokens at most)
    int T = 0, smax = 1;
    a.same_s = 1;
    for (int i = 0; i < a.entries; ++i) {
        T = std::max(T, a.e[i].t1 - a.e[i].t0);
        smax = std::max(smax, a.e[i].S);
        a.same_s &= a.e[i].S == a.e[0].S;
    }
    if constexpr (k32) {
        if (a.same_s && smax <= 4 && st_fills_32(a, smax, kFill)) return st_rw<32, UNIT, BLK, VAR, WF>(a, T, smax, st);
    }
    if (!a.same_s) {
        // entries of one split count that fill the 32-token tiles by
        // themselves: a launch of their own
        for (int SC = 1; k32 && SC <= 4; SC *= 2) {
            if (!st_fills_32(a, SC, kFill)) continue;
            StripArgs rest = a;
            StripArgs own = st_take(rest, [&](const StripEntry &e) { return e.S == SC; });
            const int r = st_shape<UNIT, BLK, VAR, WF>(own, st);
            return r ? r : st_shape<UNIT, BLK, VAR, WF>(rest, st);
        }
        // few-token entries apart from the others, once the grid is several
        // rounds deep: a 16-token tile of theirs costs as much as a full one
        // (1 + 1 + 14 + 19 + 34 tokens of two weights of 3,568 rows, K = 3712,
        // beside 371 tokens in one split: 103 -> 80 us; a shallower grid only
        // pays the second launch)
        StripArgs rest = a;
        StripArgs few = st_take(rest, [](const StripEntry &e) { return e.t1 - e.t0 <= 8; });
        long long strips16 = 0;
        for (int i = 0; i < a.entries; ++i)
            strips16 += (long long)(a.w[a.e[i].w].M / 16) * ((a.e[i].t1 - a.e[i].t0 + 15) / 16);
        if (few.entries && rest.entries && strips16 > 6ll * device_cus()) {
            const int r = st_shape<UNIT, BLK, VAR, WF>(few, st);
            return r ? r : st_shape<UNIT, BLK, VAR, WF>(rest, st);
        }
    }
    if (T == 1) return st_rw<1, UNIT, BLK, VAR, WF>(a, T, smax, st);
    if (T == 2) return st_rw<2, UNIT, BLK, VAR, WF>(a, T, smax, st);
    if (T <= 8) return st_rw<8, UNIT, BLK, VAR, WF>(a, T, smax, st);
    return st_rw<16, UNIT, BLK, VAR, WF>(a, T, smax, st);
}

bool strip_takes(int group, int block, int scale_enc, long long T, int K) {
    if (T * K >= (1ll << 31)) return false;                  // 32-bit activation offsets
    return block == 32 ? scale_enc != 0 && group != 128 : scale_enc == 0 && (group == 64 || group == 128);
}

int launch_strip(StripArgs &a, hipStream_t st) {
    if (a.scale_enc == 2)
        return a.variant == kVarGemv ? st_shape<32, true, kVarGemv, kStW8>(a, st) : st_shape<32, true, kVarGemm, kStW8>(a, st);
    if (a.group == 16) return st_shape<32, true, kVarGemv, kStK16>(a, st);
    if (a.block == 32) {
        if (a.variant == kVarGemv) return st_shape<32, true, kVarGemv, kStW4>(a, st);
        if (a.variant == kVarFanout) return st_shape<32, true, kVarFanout, kStW4>(a, st);
        return st_shape<32, true, kVarGemm, kStW4>(a, st);
    }
    // (per-token: the fan-out and GEMM arithmetic are the same)
    if (a.group == 128)
        return a.variant == kVarGemv ? st_shape<128, false, kVarGemv, kStW4>(a, st) : st_shape<128, false, kVarGemm, kStW4>(a, st);
    return a.variant == kVarGemv ? st_shape<64, false, kVarGemv, kStW4>(a, st) : st_shape<64, false, kVarGemm, kStW4>(a, st);
}

}  // namespace kxw4
