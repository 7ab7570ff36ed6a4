// kxw4_f8_gemm.hpp — products of the 8-bit floating tier for many rows.
//
// A work-group owns a tile of 32 TA WT rows of x (tokens) and 32 TB WR weight
// rows; each of its WT x WR waves TA x TB blocks of 32 x 32. Per block of 128
// columns (a step) the tile's codes and scales reach LDS by buffer loads
// straight into a ring of NST stages; the block's products are summed by the
// matrix core from zero and added to the FP32 sums with one scale: y += P * (sx
// * sw). The weights are the A operand, so a lane holds 16 outputs of one token
// and its scale is one register; sw is one for a wave's rows (32 TB divides
// 128).
//
// The dense launch has as many work-groups as the card holds; each takes tile
// after tile and the ring runs on across them: the loads of the next tile's
// first steps are in flight while this one ends and its outputs are stored.
//
// Two kinds of products (EX):
//   0  the 32x32x64 f8 MFMA on the codes, for BF16 outputs. It cuts each product,
//      towards zero, to a multiple of 2^-13 of the largest power of two among those
//      of its group of eight columns before the 32-bit sum (measured: beside 2^10
//      seven products of 1.875 are whole, beside 2^11 they are 1.75, beside 2^14
//      nothing). So P is off by up to 2^-10 of the sum of its products' magnitudes;
//      on normal data by 1.5e-5 of the output's size (a BF16 rounding: up to 2^-8).
//      Where large products cancel it may be all of a small output: products of
//      448 * 448, of both signs, each beside seven of 2.1, give 0 for the sum of
//      these. The rounding of values to codes, up to 2^-4 of each, is far above the
//      cut; a caller whose codes are exact has kind 1. The rate, twice that of kind
//      1, is why it is here.
//   1  the 32x32x16 BF16 MFMA on the codes as BF16 (exact): FP32 outputs. Half
//      the rate, and the conversions.
//
// Bounds and measurements (256 CUs; a large library product of e4m3 codes with one
// scale reaches 2,770 to 3,100 TF). BF16 out, 256 x 256 tiles: the MFMAs and the
// sums' updates beside them, 2,800 cycles a step for the MFMAs' 2,048, at the
// clock that the power limit leaves, 1.8 GHz (3,965 x 5,120 -> 2 x 17,408: 646 to
// 690 us, 2.05 to 2.19 PF; 4,096 cubed: 65 us, 2.1 PF; on zeros, which draw less
// power, the same launch reaches 2.5 PF); the last round where tiles are few
// (2,048 x 5,120 -> 5,120, 160 tiles: 67 us, 1.6 PF). FP32 out: the BF16 MFMA's
// rate and the conversions (the same: 119 us, 0.9 PF). By group: part-filled tiles
// and the last round beside these (2,048 x 8 rows over 64 experts, 5,120 -> 2 x
// 1,024: 226 to 310 us by the clock, 1.1 to 1.5 PF).
#pragma once

#include "kxw4_f8.hpp"
#include "kxw4_groups.hpp"

#include <algorithm>
#include <type_traits>
#include <utility>

namespace kxw4 {

#define KXW4_F8_LDS(p) ((__attribute__((address_space(3))) void *)(p))

template <int TA, int TB, int WT, int WR>
struct F8Shape {
    static constexpr int NW = WT * WR, NTH = 64 * NW;
    static constexpr int BT = 32 * TA * WT;                  // tokens per tile
    static constexpr int BR = 32 * TB * WR;                  // weight rows per tile
    static constexpr int X_BYTES = BT * kF8Block, W_BYTES = BR * kF8Block;
    // token scales, then the weights' (one for each 128 rows), in chunks of 256
    static constexpr int T_CHUNKS = (BT * 4 + 255) / 256, S_CHUNKS = T_CHUNKS + 1;
    static constexpr int STAGE = X_BYTES + W_BYTES + S_CHUNKS * 256;
    static constexpr int X_CHUNKS = X_BYTES / 1024, W_CHUNKS = W_BYTES / 1024;
    // loads per wave and stage: the same number for every wave, so one vmcnt
    // retires a stage (where the waves do not divide the chunks some are loaded
    // twice, the same bytes to the same place)
    static constexpr int X_LOADS = (X_CHUNKS + NW - 1) / NW, W_LOADS = (W_CHUNKS + NW - 1) / NW;
    static constexpr int S_LOADS = (S_CHUNKS + NW - 1) / NW;
    static constexpr int LOADS = X_LOADS + W_LOADS + S_LOADS;
    static constexpr int SLAB = 1024;                        // output staging of a wave: 16 tokens' 64 bytes
    template <int NST>
    static constexpr int lds_bytes() { return NST * STAGE + NW * SLAB; }
};

// f(integral_constant<int, I>) for each I of the sequence, in order
template <class F, int... I>
__device__ __forceinline__ void f8_each(F &&f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}

// Tokens [t0, t_end), weight wi's rows from row-group rg0 on, of group e, column
// blocks [k0, k1), part s of the sum; the work-group's tile number n.
struct F8Tile {
    int t0, t_end, wi, rg0, e, k0, k1, s, n;
};

// One tile after another: `tile`, then those that next(tile) gives, until it
// returns false.
template <int TA, int TB, int WT, int WR, int NST, int EX, bool GRP, class Next>
__device__ __forceinline__ void f8_tiles(const F8GemmArgs &a, F8Tile tile, Next next) {
    using S = F8Shape<TA, TB, WT, WR>;
    constexpr int NW = S::NW, BT = S::BT, STAGE = S::STAGE;
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
    const int KB = a.KB, KP = KB * kF8Block;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wt = wave / WR, wr = wave % WR;

    // ---- load issue. Chunk ch of the tokens holds tile rows 8ch..8ch+7, lane
    // l fills row 8ch + 2(l/16) + (l/8)%2, 16-byte column piece (l%8) ^ ((4ch +
    // l/16) % 8): the reads below then meet every bank once. By group: a row
    // offset for each load, 32 bits, and one descriptor of all rows, tokens past
    // the tile's end repeating its last; dense: a descriptor from each load's
    // first row, so T * K may pass 32 bits, rows past the end reading as zero,
    // and one lane part, since a wave's chunks have the wave's parity ----
    static_assert(GRP || (NW % 2 == 0 && S::X_CHUNKS % 2 == 0), "chunk parity");
    const uint32_t lane16 = lane * 16;
    uint32_t x_off[GRP ? S::X_LOADS : 1], s_off[S::S_LOADS];
    if constexpr (!GRP) {
        x_off[0] = (uint32_t)(2 * (lane >> 4) + ((lane >> 3) & 1)) * (uint32_t)KP +
                   (uint32_t)(((lane & 7) ^ ((4 * (wave & 1) + (lane >> 4)) & 7)) * 16);
#pragma unroll
        for (int i = 0; i < S::S_LOADS; ++i) s_off[i] = 4 * (64 * ((wave + NW * i) % S::S_CHUNKS) + lane);
    }
    // where the next loads come from: step lkb of tile lt. Past the last tile
    // every range is 0: nothing is read and zeros are written, so each step
    // issues as many loads. The descriptors stay, the step goes in the scalar
    // offset, which the range check counts in: a load costs few scalar
    // operations (with its descriptor built at each, a wave's 250 of them a step
    // took longer than the MFMAs)
    F8Tile lt = tile;
    int lkb = tile.k0, x_range, w_range, s_range[S::S_LOADS];
    const uint8_t *xp, *wp;
    uint64_t sp[S::S_LOADS];
    int x_so[S::X_LOADS], w_so[S::W_LOADS];
#pragma unroll
    for (int i = 0; i < S::X_LOADS; ++i) x_so[i] = GRP ? 0 : (wave + NW * i) % S::X_CHUNKS * 8 * KP;
#pragma unroll
    for (int i = 0; i < S::W_LOADS; ++i) {
        const int ch = (wave + NW * i) % S::W_CHUNKS;
        w_so[i] = (ch >> 1) * KB * kF8Tile + (ch & 1) * 1024;
    }
    auto tokens = [&](int i) { return (wave + NW * i) % S::S_CHUNKS < S::T_CHUNKS; };
    auto aim = [&]() {
        const F8GemmWeight &W = a.w[lt.wi];
        const int RG = W.M / 16, MB = f8_blocks(W.M), mb = lt.rg0 / 8;
        xp = a.q + (GRP ? 0 : (size_t)lt.t0 * KP);
        x_range = GRP ? (int)((uint32_t)a.rows * (uint32_t)KP) : (lt.t_end - lt.t0) * KP;
        if constexpr (GRP) {
            auto row_of = [&](int t) -> uint32_t {
                t = min(lt.t0 + t, lt.t_end - 1);
                return a.order ? (uint32_t)a.order[t] / (uint32_t)a.k : (uint32_t)t;
            };
#pragma unroll
            for (int i = 0; i < S::X_LOADS; ++i) {
                const int ch = (wave + NW * i) % S::X_CHUNKS;
                x_off[i] = row_of(8 * ch + 2 * (lane >> 4) + ((lane >> 3) & 1)) * (uint32_t)KP +
                           (uint32_t)(((lane & 7) ^ ((4 * (ch & 1) + (lane >> 4)) & 7)) * 16);
            }
#pragma unroll
            for (int i = 0; i < S::S_LOADS; ++i) s_off[i] = 4 * row_of(min(64 * ((wave + NW * i) % S::S_CHUNKS) + lane, BT - 1));
        }
        wp = W.codes + ((size_t)lt.e * RG + lt.rg0) * KB * kF8Tile;
        w_range = min(RG - lt.rg0, S::BR / 16) * KB * kF8Tile;
#pragma unroll
        for (int i = 0; i < S::S_LOADS; ++i) {
            // (weights' scales: lane l the block of rows l past the tile's first)
            const bool tk = tokens(i);
            const uint64_t from = reinterpret_cast<uint64_t>(tk ? a.sx + (GRP ? 0 : lt.t0) + (size_t)lt.k0 * a.rows
                                                                : W.scales + ((size_t)lt.e * MB + mb) * KB + lt.k0);
            // (selected by the wave: scalars, which the compiler does not see)
            sp[i] = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)from) |
                    (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(from >> 32)) << 32;
            s_range[i] = __builtin_amdgcn_readfirstlane(tk ? (GRP ? a.rows : lt.t_end - lt.t0) * 4 : (MB - mb) * KB * 4);
            if (!tk) s_off[i] = min(lane, MB - 1 - mb) * KB * 4;
        }
        asm volatile("" : "+s"(xp), "+s"(wp));
    };
    auto advance = [&]() {
        ++lkb;
#pragma unroll
        for (int i = 0; i < S::S_LOADS; ++i) sp[i] += tokens(i) ? (uint64_t)a.rows * 4 : 4;
        if (lkb == lt.k1) {
            if (next(lt)) {
                lkb = lt.k0;
                aim();
            } else {
                lkb = lt.k0;
                x_range = 0;
                w_range = 0;
#pragma unroll
                for (int i = 0; i < S::S_LOADS; ++i) s_range[i] = 0;
            }
        }
    };
    constexpr int kWord3 = 0x00020000;                       // untyped buffer, format 32
    auto load = [&](auto index, int st) {
        constexpr int n = decltype(index)::value;
        uint8_t *base = smem + st * STAGE;
        // (computed outside the builtins' argument lists: inside them such
        // expressions can make the host pass drop the kernel without a diagnostic)
        if constexpr (n < S::X_LOADS) {
            const int at = lkb * kF8Block + x_so[n];
            const uint32_t off = x_off[GRP ? n : 0];
            // (by group: chunks past the tile's rows read nothing)
            const int range = GRP && (wave + NW * n) % S::X_CHUNKS * 8 >= lt.t_end - lt.t0 ? 0 : x_range;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(__builtin_amdgcn_make_buffer_rsrc((void *)xp, 0, range, kWord3),
                                                     KXW4_F8_LDS(base + (wave + NW * n) % S::X_CHUNKS * 1024), 16, off, at, 0, 0);
        } else if constexpr (n < S::X_LOADS + S::W_LOADS) {
            constexpr int i = n - S::X_LOADS;
            const int at = lkb * kF8Tile + w_so[i];
            __builtin_amdgcn_raw_ptr_buffer_load_lds(__builtin_amdgcn_make_buffer_rsrc((void *)wp, 0, w_range, kWord3),
                                                     KXW4_F8_LDS(base + S::X_BYTES + (wave + NW * i) % S::W_CHUNKS * 1024), 16, lane16, at, 0, 0);
        } else {
            constexpr int i = n - S::X_LOADS - S::W_LOADS;
            const void *from = reinterpret_cast<const void *>(sp[i]);
            const int range = s_range[i];
            const uint32_t off = s_off[i];
            __builtin_amdgcn_raw_ptr_buffer_load_lds(__builtin_amdgcn_make_buffer_rsrc((void *)from, 0, range, kWord3),
                                                     KXW4_F8_LDS(base + S::X_BYTES + S::W_BYTES + (wave + NW * i) % S::S_CHUNKS * 256), 4, off, 0, 0, 0);
        }
    };
    constexpr int LD = S::LOADS;
    auto issue = [&](int st) { f8_each([&](auto n) { load(n, st); }, std::make_integer_sequence<int, LD>{}); };

    // ---- per-lane read offsets in a stage (lane = token / weight row l%32,
    // column half l/32 of each 64) ----
    const int m32 = lane & 31, kg = lane >> 5;
    // (token block i of this wave is block WT * i + wt of the tile, so a tile with
    // fewer tokens leaves every wave its share)
    // 16-byte pieces 4(c / 2) + 2kg + c % 2 of a row, c = 0..3: piece c is piece
    // 0 with two bits flipped (stages are multiples of 256, so the flips go last)
    const int xoff = ((16 * wt + (m32 >> 1)) * 16 + (((m32 & 1) << 3) | ((2 * kg) ^ ((m32 >> 1) & 7)))) * 16;
    const int woff = S::X_BYTES + (wr * 2 * TB + (m32 >> 4)) * kF8Tile + (2 * kg * 16 + (m32 & 15)) * 16;
    const int soff = S::X_BYTES + S::W_BYTES + (32 * wt + m32) * 4;
    const int goff = S::X_BYTES + S::W_BYTES + S::T_CHUNKS * 256 + (wr * TB / 4) * 4;
    auto read_w = [&](int base, int j, v4u (&w)[4]) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
            w[c] = *reinterpret_cast<const v4u *>(smem + base + woff + j * 2 * kF8Tile + (c >> 1) * 1024 + (c & 1) * 256);
    };
    auto read_x = [&](int base, int i, v4u (&x)[4]) {
#pragma unroll
        for (int c = 0; c < 4; ++c) x[c] = *reinterpret_cast<const v4u *>(smem + ((base + xoff) ^ ((c & 1) * 16 + (c >> 1) * 64)) + i * WT * 4096);
    };
    auto read_s = [&](int base, int i) { return *reinterpret_cast<const float *>(smem + base + soff + i * WT * 128); };
    auto read_g = [&](int base) { return *reinterpret_cast<const float *>(smem + base + goff); };
    auto codes8 = [](const v4u (&v)[4], int c) {
        return v8i{(int)v[2 * c].x, (int)v[2 * c].y, (int)v[2 * c].z, (int)v[2 * c].w,
                   (int)v[2 * c + 1].x, (int)v[2 * c + 1].y, (int)v[2 * c + 1].z, (int)v[2 * c + 1].w};
    };

    // token blocks of a wave that a tile runs (tiles of four run them all: a loop
    // for each number of them spilled)
    auto blocks_of = [](const F8Tile &t) { return TA > 2 ? TA : (t.t_end - t.t0 + 32 * WT - 1) / (32 * WT); };
    F8Tile ahead = tile;                                     // the tile after this one
    int na = blocks_of(tile), more = next(ahead);

    v16f f[TA][TB];
    auto clear = [&]() {
#pragma unroll
        for (int i = 0; i < TA; ++i)
#pragma unroll
            for (int j = 0; j < TB; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) f[i][j][r] = 0.0f;
    };
    // ---- output: register r of a block is row 8(r/4) + 4kg + r%4 of the lane's
    // token. BF16: 16 tokens at a time pass the wave's slab in LDS (64 bytes of
    // each, its 16-byte piece c at c ^ (t / 4 % 4)) and go out 64 bytes a token,
    // so a store meets 16 of the L2's half lines, not 32 quarters (8,192 tokens,
    // 8,192 x 1,024: 98 us without the slab, 87). FP32: four rows a lane and
    // store (through the slab 22.7 us became 24.3, 256 tokens, 5,120 x 5,120) ----
    uint8_t *slab = smem + NST * STAGE + wave * S::SLAB;
    auto store = [&]() {
        const F8GemmWeight &W = a.w[tile.wi];
        // (the lane's places are computed anew for each tile: kept over the steps
        // they would spill)
        int lane = tid & 63;
        asm volatile("" : "+v"(lane));
        const int m32 = lane & 31, kg = lane >> 5, t16 = m32 & 15, swz = t16 >> 2;
        const int M = W.M, row0 = (tile.rg0 + wr * 2 * TB) * 16;
        const bool part = !GRP && a.part;                    // (part of a sum: f8_join_kernel ends it)
#pragma unroll
        for (int i = 0; i < TA; ++i) {
            const int tb = tile.t0 + 32 * (WT * i + wt), t = tb + m32;
            if (i >= na || tb >= tile.t_end) continue;       // (uniform)
#pragma unroll
            for (int j = 0; j < TB; ++j) {
                const int row = row0 + 32 * j;
                if (row >= M) continue;                      // (uniform)
                if (!GRP && a.residual && !part) {
                    // (places past the ends read the last ones, for outputs that are not stored)
                    const float *res = a.residual + (size_t)min(t, a.rows - 1) * M;
                    v4f x[4];
#pragma unroll
                    for (int q = 0; q < 4; ++q) x[q] = *reinterpret_cast<const v4f *>(res + min(row + 8 * q + 4 * kg, M - 4));
#pragma unroll
                    for (int r = 0; r < 16; ++r) f[i][j][r] += x[r / 4][r % 4];
                }
                if (EX == 0 && !part) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {            // 16 tokens
                        if ((m32 >> 4) == h) {
#pragma unroll
                            for (int q = 0; q < 4; ++q)
                                *reinterpret_cast<v2u *>(slab + t16 * 64 + ((q ^ swz) * 16) + kg * 8) =
                                    v2u{pack_bf16(f[i][j][4 * q], f[i][j][4 * q + 1]), pack_bf16(f[i][j][4 * q + 2], f[i][j][4 * q + 3])};
                        }
                        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // (other lanes' writes)
                        const int ts = tb + 16 * h + (lane >> 2), r = row + (lane & 3) * 8;
                        const v4u v = *reinterpret_cast<const v4u *>(slab + (lane >> 2) * 64 + (((lane & 3) ^ (lane >> 4)) * 16));
                        if (ts < tile.t_end && r < M) {
                            v4u *to = reinterpret_cast<v4u *>(static_cast<uint16_t *>(W.y) + (size_t)ts * M + r);
                            if (!GRP && a.stream) store_past(v, to);
                            else *to = v;
                        }
                        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // (their reads)
                    }
                } else {
                    float *to = (part ? a.part + W.part + (size_t)tile.s * a.rows * M : static_cast<float *>(W.y)) + (size_t)t * M + row + 4 * kg;
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        if (t < tile.t_end && row + 8 * q < M)
                            *reinterpret_cast<v4f *>(to + 8 * q) = v4f{f[i][j][4 * q], f[i][j][4 * q + 1], f[i][j][4 * q + 2], f[i][j][4 * q + 3]};
                }
            }
        }
    };

    static_assert(NST >= 2 && NST <= 4, "two to four stages");
    static_assert(LD * (NST - 2) <= 63, "vmcnt field");
    // the loads of this step are in LDS for every wave, and every wave is past
    // its reads of the step before; the loads of NST - 2 steps may be in flight
    // (and stores, which make the wait longer)
    auto arrive = [&]() {
        KXW4_WAIT_VMCNT(LD * (NST - 2));
        lds_sync_after_dma();
    };
    aim();
#pragma unroll
    for (int s = 0; s < NST - 1; ++s) {
        issue(s);
        advance();
    }
    clear();
    int st = 0;
    if constexpr (EX == 0) {
        // Software pipeline over the blocks of all steps (weight block fastest):
        // a block's two MFMAs run beside the sums' updates by the block before
        // it, the next tokens are read one token block ahead, and the barrier of
        // a step sits before its last block, whose operands are in registers:
        // the stage is then free for the loads of NST steps on, and the next
        // step's first operands are read while that block runs. Those loads are
        // issued a few at a time, from that block on: all at once they hold a
        // wave for as long as they take through the L1 (16 cycles each, 72 of
        // a 256 x 256 tile), and both waves of a SIMD together.
        constexpr int NB = TA * TB;
        static_assert(TB == 2, "the last block of a step leaves the first weight block free");
        // part q of a stage's loads
        constexpr int PL = (LD + NB - 2) / (NB - 1) < 2 ? 2 : (LD + NB - 2) / (NB - 1), PARTS = (LD + PL - 1) / PL;
        static_assert(PARTS <= NB, "a stage's loads within a step");
        auto issue_part = [&](auto q, int st) {
            constexpr int from = decltype(q)::value * PL, n = from >= LD ? 0 : from + PL < LD ? PL : LD - from;
            f8_each([&](auto i) { load(std::integral_constant<int, from + decltype(i)::value>{}, st); },
                    std::make_integer_sequence<int, n>{});
        };
        v4u w[2][4], xc[4], xn[4];
        float sn, gn, g_cur = 0.0f, s_cur = 0.0f, s_prev = 0.0f;
        v16f p[2];
        const v16f zero = {};
        arrive();
        issue_part(std::integral_constant<int, 0>{}, NST - 1);
        read_w(0, 0, w[0]);
        read_x(0, na - 1, xn);
        sn = read_s(0, na - 1);
        gn = read_g(0);
        // the steps of a tile of NA token blocks a wave, downwards from the last
        auto steps = [&](auto NA) {
            constexpr int N = decltype(NA)::value;
            p[1] = zero;                                     // (a tile's first block updates with a zero scale)
            s_prev = 0.0f;
            for (int kb = tile.k0; kb < tile.k1; ++kb) {
                const int stn = st == NST - 1 ? 0 : st + 1, stp = st == 0 ? NST - 1 : st - 1;
                const int base = st * STAGE, nbase = stn * STAGE;
                g_cur = gn;
                auto block = [&](auto index) {
                    constexpr int b = decltype(index)::value, i = N - 1 - b / 2, j = b & 1, slot = j;
                    constexpr bool last = b == 2 * N - 1;
                    if constexpr (last) {
                        // (what is left of the stage before, where the blocks are few)
                        f8_each([&](auto q) { issue_part(std::integral_constant<int, 2 * N + decltype(q)::value>{}, stp); },
                                std::make_integer_sequence<int, (PARTS > 2 * N ? PARTS - 2 * N : 0)>{});
                        arrive();
                        advance();
                        issue_part(std::integral_constant<int, 0>{}, st);
                        __builtin_amdgcn_sched_barrier(0);
                    } else {
                        issue_part(std::integral_constant<int, b + 1>{}, stp);
                    }
                    if constexpr (j == 0) {
#pragma unroll
                        for (int c = 0; c < 4; ++c) xc[c] = xn[c];
                        s_cur = sn * g_cur;
                    }
                    if constexpr (last) {                    // (after the last step: harmless reads of zeros)
                        const int top = kb + 1 < tile.k1 ? N - 1 : blocks_of(ahead) - 1;
                        read_w(nbase, 0, w[0]);
                        read_x(nbase, top, xn);
                        sn = read_s(nbase, top);
                        gn = read_g(nbase);
                    } else {
                        if constexpr (b == 0) read_w(base, 1, w[1]);
                        if constexpr (j == 0 && i > 0) {
                            read_x(base, i - 1, xn);
                            sn = read_s(base, i - 1);
                        }
                    }
                    p[slot] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(codes8(w[j], 0), codes8(xc, 0), zero, 0, 0, 0, 0, 0, 0);
                    p[slot] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(codes8(w[j], 1), codes8(xc, 1), p[slot], 0, 0, 0, 0, 0, 0);
                    constexpr int ui = j == 1 ? i : b == 0 ? 0 : i + 1, uj = 1 - j;
#pragma unroll
                    for (int r = 0; r < 16; ++r) f[ui][uj][r] = __builtin_fmaf(p[slot ^ 1][r], s_prev, f[ui][uj][r]);
                    // (kept in this block: without a use here the updates sink
                    // past the barrier of the last block)
#pragma unroll
                    for (int r = 0; r < 16; ++r) asm volatile("" ::"v"(f[ui][uj][r]));
                    s_prev = s_cur;
                    __builtin_amdgcn_sched_group_barrier(0x100, 10, 0);
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x002, 8, 0);
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x002, 16, 0);
                    __builtin_amdgcn_sched_barrier(0);
                };
                f8_each(block, std::make_integer_sequence<int, 2 * N>{});
                st = stn;
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) f[0][1][r] = __builtin_fmaf(p[1][r], s_prev, f[0][1][r]);
        };
        for (;;) {
            if (TA != 2 || na == 2) steps(std::integral_constant<int, TA>{});
            else steps(std::integral_constant<int, 1>{});
            store();
            if (!more) break;
            tile = ahead;
            na = blocks_of(tile);
            more = next(ahead);
            clear();
        }
    } else {
        auto steps = [&](auto NA) {
            constexpr int N = decltype(NA)::value;
            for (int kb = tile.k0; kb < tile.k1; ++kb) {
                arrive();
                issue(st == 0 ? NST - 1 : st - 1);
                advance();
                const int base = st * STAGE;
                const float g = read_g(base);
                v4u w[TB][4];
#pragma unroll
                for (int j = 0; j < TB; ++j) read_w(base, j, w[j]);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    v4u x[4];
                    read_x(base, i, x);
                    const float s = read_s(base, i) * g;
#pragma unroll
                    for (int j = 0; j < TB; ++j) {
                        v16f p = {};
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            p = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f8_to_bf16(w[j][c].x, w[j][c].y), f8_to_bf16(x[c].x, x[c].y), p, 0, 0, 0);
                            p = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f8_to_bf16(w[j][c].z, w[j][c].w), f8_to_bf16(x[c].z, x[c].w), p, 0, 0, 0);
                        }
#pragma unroll
                        for (int r = 0; r < 16; ++r) f[i][j][r] = __builtin_fmaf(p[r], s, f[i][j][r]);
                    }
                }
                st = st == NST - 1 ? 0 : st + 1;
            }
        };
        for (;;) {
            if (TA != 2 || na == 2) steps(std::integral_constant<int, TA>{});
            else steps(std::integral_constant<int, 1>{});
            store();
            if (!more) break;
            tile = ahead;
            na = blocks_of(tile);
            more = next(ahead);
            clear();
        }
    }
    KXW4_WAIT_VMCNT(0);                                      // (no load past the last step outlives the work-group's LDS)
}

// Tile L of a launch of nt token tiles and a.n_tiles weight tiles: the
// work-groups of one XCD (blockIdx % 8) take consecutive tiles, kF8Raster token
// tiles at a time, so they share codes in that XCD's L2.
constexpr int kF8Raster = 4;

template <int TA, int TB, int WT, int WR, int NST, int EX, int OCC>
__global__ __launch_bounds__(64 * WT * WR)
__attribute__((amdgpu_waves_per_eu(OCC, OCC))) void f8_gemm_kernel(const F8GemmArgs a) {
    using S = F8Shape<TA, TB, WT, WR>;
    const int ntt = (a.rows + S::BT - 1) / S::BT, nnt = a.n_tiles, tiles = ntt * nnt, total = tiles * a.splits;
    // (with more tiles than work-groups the host launches a multiple of eight)
    auto tile_of = [&](int item) {
        const int s = item / tiles, id = item - s * tiles;
        const int q8 = tiles / 8, r8 = tiles % 8, xcd = id % 8, j8 = id / 8;
        const int L = xcd < r8 ? xcd * (q8 + 1) + j8 : r8 * (q8 + 1) + (xcd - r8) * q8 + j8;
        const int group = L / (kF8Raster * nnt), first = group * kF8Raster;
        const int gsz = min(ntt - first, kF8Raster), within = L % (kF8Raster * nnt);
        const int tt = first + within % gsz, ntg = within / gsz;
        int wi = 0;
        for (int i = 1; i < a.count; ++i)
            if (ntg >= a.w[i].nt_begin) wi = i;
        const int t0 = tt * S::BT, q = a.KB / a.splits, r = a.KB % a.splits, k0 = s * q + min(s, r);
        return F8Tile{t0, min(t0 + S::BT, a.rows), wi, (ntg - a.w[wi].nt_begin) * (S::BR / 16), 0, k0, k0 + q + (s < r), s, 0};
    };
    f8_tiles<TA, TB, WT, WR, NST, EX, false>(a, tile_of(blockIdx.x), [&](F8Tile &t) {
        const int n = t.n + 1, id = blockIdx.x + n * gridDim.x;
        if (id >= total) return 0;
        t = tile_of(id);
        t.n = n;
        return 1;
    });
}

// The parts of split sums, added up in their order, plus the residual; four
// outputs a thread.
__global__ __launch_bounds__(256) void f8_join_kernel(const F8GemmArgs a) {
    long long at = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
    int wi = 0;
    for (; wi < a.count; ++wi) {
        const long long n = (long long)a.rows * a.w[wi].M;
        if (at < n) break;
        at -= n;
    }
    if (wi == a.count) return;
    const F8GemmWeight &W = a.w[wi];
    const long long n = (long long)a.rows * W.M;
    const float *part = a.part + W.part + at;
    v4f v = *reinterpret_cast<const v4f *>(part);
    for (int s = 1; s < a.splits; ++s) {
        const v4f x = *reinterpret_cast<const v4f *>(part + s * n);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] += x[j];
    }
    if (a.residual) {
        const v4f x = *reinterpret_cast<const v4f *>(a.residual + at);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] += x[j];
    }
    if (a.y_bf16) *reinterpret_cast<v2u *>(static_cast<uint16_t *>(W.y) + at) = v2u{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
    else *reinterpret_cast<v4f *>(static_cast<float *>(W.y) + at) = v;
}

// The same over rows sorted by group: tiles of 32 TA WT places of one group, its
// last one shorter (its steps run the token blocks it has).
//
// The tiles in order: groups, in each its weight tiles, of each the group's token
// tiles. An XCD (blockIdx % 8) takes an eighth of them, one after another, and its
// work-groups those in turn: at once they run the tiles of one or two groups,
// whose tokens and codes each pass that XCD's L2 once (with each group's weight
// tiles dealt over the XCDs every one of these read all the tokens: 2,048 x 8 rows
// over 64 groups, 5,120 -> 2 x 1,024: 313 us, so 298).
struct F8Scan {
    int first, end, before, total, begin, begin_end;         // a lane's run of groups, the tiles before it, all tiles; its first group's places
};

template <int BT>
__device__ __forceinline__ F8Scan f8_scan(const int *offsets, int groups, int nnt, int lane) {
    const int run = (groups + 63) / 64;
    F8Scan s;
    s.first = min(lane * run, groups);
    s.end = min(s.first + run, groups);
    int sum = 0, lo = offsets[s.first];
    s.begin = lo;
    s.begin_end = lo;
    for (int e = s.first; e < s.end; ++e) {
        const int hi = offsets[e + 1];
        if (e == s.first) s.begin_end = hi;
        sum += (hi - lo + BT - 1) / BT * nnt;
        lo = hi;
    }
    const int inc = wave_scan(sum);
    s.before = inc - sum;
    s.total = __builtin_amdgcn_readlane(inc, 63);
    return s;
}

// Tile u < s.total: its group, places and weight tile.
template <int BT>
__device__ __forceinline__ F8Tile f8_group_tile(const F8Scan &s, const F8GemmArgs &a, int brg, int u) {
    // (lanes without tiles share the start of the next that has some, so the
    // last lane that starts at or before u has the tile)
    const int l = 63 - __builtin_clzll(__ballot(s.first < s.end && s.before <= u));
    int e = __builtin_amdgcn_readlane(s.first, l), before = __builtin_amdgcn_readlane(s.before, l);
    int begin = __builtin_amdgcn_readlane(s.begin, l), end = __builtin_amdgcn_readlane(s.begin_end, l);
    int count;
    for (;;) {
        count = (end - begin + BT - 1) / BT;
        const int n = count * a.n_tiles;
        if (u < before + n) break;
        before += n;
        ++e;
        begin = end;
        end = __builtin_amdgcn_readfirstlane(a.offsets[e + 1]);
    }
    const int ntg = (u - before) / count, t0 = begin + (u - before - ntg * count) * BT;
    int wi = 0;
    for (int i = 1; i < a.count; ++i)
        if (ntg >= a.w[i].nt_begin) wi = i;
    return F8Tile{t0, min(t0 + BT, end), wi, (ntg - a.w[wi].nt_begin) * brg, e, 0, a.KB, 0, 0};
}

template <int TA, int TB, int WT, int WR, int NST, int EX, int OCC>
__global__ __launch_bounds__(64 * WT * WR)
__attribute__((amdgpu_waves_per_eu(OCC, OCC))) void f8_group_kernel(const F8GemmArgs a) {
    constexpr int BT = 32 * TA * WT, BRG = 2 * TB * WR;
    const int x = blockIdx.x % 8, first = blockIdx.x / 8, stride = gridDim.x / 8;      // (a multiple of eight)
    const F8Scan s = f8_scan<BT>(a.offsets, a.groups, a.n_tiles, threadIdx.x & 63);
    const int from = (int)((long long)s.total * x / 8), end = (int)((long long)s.total * (x + 1) / 8);
    if (from + first >= end) return;
    f8_tiles<TA, TB, WT, WR, NST, EX, true>(a, f8_group_tile<BT>(s, a, BRG, from + first), [&](F8Tile &t) {
        const int n = t.n + 1, u = from + first + n * stride;
        if (u >= end) return 0;
        t = f8_group_tile<BT>(s, a, BRG, u);
        t.n = n;
        return 1;
    });
}

}  // namespace kxw4
