// kxw4_f8_gemm.hpp — products of the 8-bit floating tier for many rows.
//
// A work-group owns a tile of 32 TA WT rows of x (tokens) and 32 TB WR weight
// rows; each of its WT x WR waves TA x TB blocks of 32 x 32. Per block of 128
// columns the tile's codes and the tokens' scales reach LDS by buffer loads
// straight into a ring of NST stages; the block's products are summed by the
// matrix core from zero and added to the FP32 sums with one scale: y += P * (sx
// * sw). The weights are the A operand, so a lane holds 16 outputs of one token
// and its scale is one register; sw is uniform over a wave's rows (32 TB divides
// 128).
//
// Two kinds of products (EX):
//   0  the 32x32x64 f8 MFMA on the codes. It cuts each product to 2^-13 of the
//      largest power of two in its group of eight columns before the 32-bit sum
//      (measured; on normal data an error of 1.5e-5 of the output's size), far
//      below the rounding of a BF16 output, whose tier this is.
//   1  the 32x32x16 BF16 MFMA on the codes as BF16 (exact): FP32 outputs. Half
//      the rate, and the conversions.
#pragma once

#include "kxw4_f8.hpp"
#include "kxw4_groups.hpp"

#include <algorithm>
#include <type_traits>

namespace kxw4 {

#define KXW4_F8_LDS(p) ((__attribute__((address_space(3))) void *)(p))

template <int TA, int TB, int WT, int WR>
struct F8Shape {
    static constexpr int NW = WT * WR, NTH = 64 * NW;
    static constexpr int BT = 32 * TA * WT;                  // tokens per tile
    static constexpr int BR = 32 * TB * WR;                  // weight rows per tile
    static constexpr int X_BYTES = BT * kF8Block, W_BYTES = BR * kF8Block, S_BYTES = BT * 4;
    static constexpr int STAGE = X_BYTES + W_BYTES + (S_BYTES + 1023) / 1024 * 1024;
    static constexpr int X_CHUNKS = X_BYTES / 1024, W_CHUNKS = W_BYTES / 1024, S_CHUNKS = (S_BYTES + 255) / 256;
    // loads per wave and stage: the same number for every wave, so one vmcnt
    // retires a stage (where the waves do not divide the chunks some are loaded
    // twice, the same bytes to the same place)
    static constexpr int X_LOADS = (X_CHUNKS + NW - 1) / NW, W_LOADS = (W_CHUNKS + NW - 1) / NW;
    static constexpr int S_LOADS = (S_CHUNKS + NW - 1) / NW;
    static constexpr int LOADS = X_LOADS + W_LOADS + S_LOADS;
    // output staging: 32 tokens x 32 TB rows a wave, FP32; a token's stride is 4
    // past a multiple of 32, so 16-byte accesses of neighbouring tokens meet
    // other banks
    static constexpr int EPS = 32 * TB + 4;
    static constexpr int SLAB = 32 * EPS * 4;
    template <int NST>
    static constexpr int lds_bytes() { return NST * STAGE > NW * SLAB ? NST * STAGE : NW * SLAB; }
    static_assert(BT >= 64 || NW >= 1, "");
};

template <int TA, int TB, int WT, int WR, int NST, int EX, bool GRP>
__device__ __forceinline__ void f8_tile(const F8GemmArgs &a, int t0, int t_end, int wi, int rg0, int e) {
    using S = F8Shape<TA, TB, WT, WR>;
    constexpr int NW = S::NW, BT = S::BT, STAGE = S::STAGE;
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
    const F8GemmWeight &W = a.w[wi];
    const int M = W.M, RG = M / 16, KB = a.KB, KP = KB * kF8Block;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wt = wave / WR, wr = wave % WR;
    auto row_of = [&](int t) -> uint32_t {
        if constexpr (GRP) return a.order ? (uint32_t)a.order[t] / (uint32_t)a.k : (uint32_t)t;
        else return (uint32_t)t;
    };

    // ---- load issue. Chunk ch of the tokens holds tile rows 8ch..8ch+7, lane
    // l fills row 8ch + 2(l/16) + (l/8)%2, 16-byte column piece (l%8) ^ ((4ch +
    // l/16) % 8): the reads below then meet every bank once. Tokens past the
    // tile's end repeat its last; weight rows past M read as zero ----
    const uint8_t *qg = a.q;
    const uint8_t *cg = W.codes + (size_t)e * RG * KB * kF8Tile;
    const float *sg = a.sx;
    // (dense: offsets from the tile's first row, so T * K may pass 32 bits)
    if constexpr (!GRP) {
        qg += (size_t)t0 * KP;
        sg += t0;
    }
    uint32_t x_off[S::X_LOADS], s_off[S::S_LOADS];
#pragma unroll
    for (int i = 0; i < S::X_LOADS; ++i) {
        const int ch = (wave + NW * i) % S::X_CHUNKS;
        const int r = min(t0 + 8 * ch + 2 * (lane >> 4) + ((lane >> 3) & 1), t_end - 1);
        x_off[i] = (GRP ? row_of(r) : (uint32_t)(r - t0)) * (uint32_t)KP + (uint32_t)(((lane & 7) ^ ((4 * (ch & 1) + (lane >> 4)) & 7)) * 16);
    }
#pragma unroll
    for (int i = 0; i < S::S_LOADS; ++i) {
        const int c = (wave + NW * i) % S::S_CHUNKS;
        const int r = min(t0 + min(64 * c + lane, BT - 1), t_end - 1);
        s_off[i] = 4 * (GRP ? row_of(r) : (uint32_t)(r - t0));
    }
    asm volatile("" : "+s"(qg), "+s"(cg), "+s"(sg));
    constexpr int kWord3 = 0x00020000;                       // untyped buffer, format 32
    const int x_range = GRP ? (int)((uint32_t)a.rows * (uint32_t)KP) : (t_end - t0) * KP;
    auto issue = [&](int kb, int st) {
        uint8_t *base = smem + st * STAGE;
#pragma unroll
        for (int i = 0; i < S::X_LOADS; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(__builtin_amdgcn_make_buffer_rsrc((void *)qg, 0, x_range, kWord3),
                                                     KXW4_F8_LDS(base + ((wave + NW * i) % S::X_CHUNKS) * 1024), 16, x_off[i],
                                                     kb * kF8Block, 0, 0);
#pragma unroll
        for (int i = 0; i < S::W_LOADS; ++i) {
            const int ch = (wave + NW * i) % S::W_CHUNKS, rg = rg0 + (ch >> 1);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                __builtin_amdgcn_make_buffer_rsrc((void *)(cg + (size_t)min(rg, RG - 1) * KB * kF8Tile), 0, rg < RG ? KB * kF8Tile : 0, kWord3),
                KXW4_F8_LDS(base + S::X_BYTES + ch * 1024), 16, (ch & 1) * 1024 + lane * 16, kb * kF8Tile, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < S::S_LOADS; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                __builtin_amdgcn_make_buffer_rsrc((void *)(sg + (size_t)kb * a.rows), 0, (GRP ? a.rows : t_end - t0) * 4, kWord3),
                KXW4_F8_LDS(base + S::X_BYTES + S::W_BYTES + ((wave + NW * i) % S::S_CHUNKS) * 256), 4, s_off[i], 0, 0, 0);
    };

    // ---- per-lane read offsets in a stage (lane = token / weight row l%32,
    // column half l/32 of each 64) ----
    const int m32 = lane & 31, kg = lane >> 5;
    const int tw = wt * 32 * TA;                             // first token of this wave in the tile
    const int hx = (m32 >> 1) & 7;
    int xoff[4];                                             // 16-byte pieces 4c + 2kg + i, at [2c + i]
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const int piece = 4 * (c >> 1) + 2 * kg + (c & 1);
        xoff[c] = (((tw >> 1) + (m32 >> 1)) * 16 + (((m32 & 1) << 3) | (piece ^ hx))) * 16;
    }
    const int woff = S::X_BYTES + (wr * 2 * TB + (m32 >> 4)) * kF8Tile + (2 * kg * 16 + (m32 & 15)) * 16;
    const int soff = S::X_BYTES + S::W_BYTES + (tw + m32) * 4;

    // block scales of this wave's rows: 64 column blocks in a register, read by lane
    const float *sw = W.scales + ((size_t)e * f8_blocks(M) + min((rg0 + wr * 2 * TB) / 8, f8_blocks(M) - 1)) * KB;
    float swv = sw[min(lane, KB - 1)];

    v16f f[TA][TB];
#pragma unroll
    for (int i = 0; i < TA; ++i)
#pragma unroll
        for (int j = 0; j < TB; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) f[i][j][r] = 0.0f;

    asm volatile("" : "+v"(swv));                            // (arrived here, ahead of the stages' loads)
    static_assert(NST >= 2 && NST <= 4, "two to four stages");
    constexpr int LD = S::LOADS;
    static_assert(LD * (NST - 2) <= 63, "vmcnt field");
    auto arrive = [&](int k) {
        const int later = min(NST - 2, KB - 1 - k);
        if (NST >= 4 && later >= 2) KXW4_WAIT_VMCNT(2 * LD);
        else if (NST >= 3 && later >= 1) KXW4_WAIT_VMCNT(LD);
        else KXW4_WAIT_VMCNT(0);
        lds_sync_after_dma();
    };
#pragma unroll
    for (int s = 0; s < NST - 1; ++s)
        if (s < KB) issue(s, s);
    int st = 0;
    for (int kb = 0; kb < KB; ++kb) {
        arrive(kb);
        // (every wave is past its reads of the stage before this one)
        if (kb + NST - 1 < KB) issue(kb + NST - 1, st == 0 ? NST - 1 : st - 1);
        if ((kb & 63) == 0 && kb) {
            swv = sw[min(kb + lane, KB - 1)];
            asm volatile("" : "+v"(swv));
        }
        const float wsc = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(swv), kb & 63));
        const uint8_t *base = smem + st * STAGE;
        v4u wq[TB][4];
#pragma unroll
        for (int j = 0; j < TB; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c)
                wq[j][c] = *reinterpret_cast<const v4u *>(base + woff + j * 2 * kF8Tile + (c >> 1) * 1024 + (c & 1) * 256);
#pragma unroll
        for (int i = 0; i < TA; ++i) {
            v4u xq[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) xq[c] = *reinterpret_cast<const v4u *>(base + xoff[c] + i * 4096);
            const float s = *reinterpret_cast<const float *>(base + soff + i * 128) * wsc;
#pragma unroll
            for (int j = 0; j < TB; ++j) {
                v16f p = {};
                if constexpr (EX == 0) {
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const v8i wa = {(int)wq[j][2 * c].x, (int)wq[j][2 * c].y, (int)wq[j][2 * c].z, (int)wq[j][2 * c].w,
                                        (int)wq[j][2 * c + 1].x, (int)wq[j][2 * c + 1].y, (int)wq[j][2 * c + 1].z, (int)wq[j][2 * c + 1].w};
                        const v8i xb = {(int)xq[2 * c].x, (int)xq[2 * c].y, (int)xq[2 * c].z, (int)xq[2 * c].w,
                                        (int)xq[2 * c + 1].x, (int)xq[2 * c + 1].y, (int)xq[2 * c + 1].z, (int)xq[2 * c + 1].w};
                        p = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wa, xb, p, 0, 0, 0, 0, 0, 0);
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        p = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f8_to_bf16(wq[j][c].x, wq[j][c].y), f8_to_bf16(xq[c].x, xq[c].y), p, 0, 0, 0);
                        p = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f8_to_bf16(wq[j][c].z, wq[j][c].w), f8_to_bf16(xq[c].z, xq[c].w), p, 0, 0, 0);
                    }
                }
#pragma unroll
                for (int r = 0; r < 16; ++r) f[i][j][r] = __builtin_fmaf(p[r], s, f[i][j][r]);
            }
        }
        st = st == NST - 1 ? 0 : st + 1;
    }

    // ---- output: each wave stages 32 tokens at a time in its own slab and
    // writes runs of 16 bytes: register r of a block is row 8(r/4) + 4kg + r%4
    // of the lane's token ----
    lds_sync();
    float *slab = reinterpret_cast<float *>(smem + wave * S::SLAB);
    auto run = [&](auto ch, int tok) {
        constexpr int CH = decltype(ch)::value, PER = 32 * TB / CH;
#pragma unroll
        for (int it = 0; it < 32 * PER / 64; ++it) {
            const int q = it * 64 + lane, tl = q / PER, rl = (q % PER) * CH;
            const int t = t0 + tok + tl, row = (rg0 + wr * 2 * TB) * 16 + rl;
            if (t >= t_end || row >= M) continue;
            const size_t at = (size_t)t * M + row;
            float v[CH];
#pragma unroll
            for (int c = 0; c < CH; c += 4) {
                const v4f x = *reinterpret_cast<const v4f *>(slab + tl * S::EPS + rl + c);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[c + j] = x[j];
            }
            if (!GRP && a.residual) {
#pragma unroll
                for (int c = 0; c < CH; c += 4) {
                    const float4 x = *reinterpret_cast<const float4 *>(a.residual + at + c);
                    v[c] += x.x;
                    v[c + 1] += x.y;
                    v[c + 2] += x.z;
                    v[c + 3] += x.w;
                }
            }
            if constexpr (CH == 8)
                *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(W.y) + at) =
                    make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
            else
                *reinterpret_cast<float4 *>(static_cast<float *>(W.y) + at) = make_float4(v[0], v[1], v[2], v[3]);
        }
    };
#pragma unroll
    for (int i = 0; i < TA; ++i) {
#pragma unroll
        for (int j = 0; j < TB; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                *reinterpret_cast<v4f *>(slab + m32 * S::EPS + 32 * j + 8 * q + 4 * kg) =
                    v4f{f[i][j][4 * q], f[i][j][4 * q + 1], f[i][j][4 * q + 2], f[i][j][4 * q + 3]};
        if constexpr (EX == 0) run(std::integral_constant<int, 8>{}, tw + 32 * i);
        else run(std::integral_constant<int, 4>{}, tw + 32 * i);
    }
}

// Tile L of a launch of nt token tiles and a.n_tiles weight tiles: the
// work-groups of one XCD (blockIdx % 8) take consecutive tiles, kF8Raster token
// tiles at a time, so they share codes in that XCD's L2.
constexpr int kF8Raster = 4;

template <int TA, int TB, int WT, int WR, int NST, int EX, int OCC>
__global__ __launch_bounds__(64 * WT * WR)
__attribute__((amdgpu_waves_per_eu(OCC, OCC))) void f8_gemm_kernel(const F8GemmArgs a) {
    using S = F8Shape<TA, TB, WT, WR>;
    const int nblk = gridDim.x, id = blockIdx.x;
    const int q8 = nblk / 8, r8 = nblk % 8, xcd = id % 8, j8 = id / 8;
    const int L = xcd < r8 ? xcd * (q8 + 1) + j8 : r8 * (q8 + 1) + (xcd - r8) * q8 + j8;
    const int ntt = (a.rows + S::BT - 1) / S::BT, nnt = a.n_tiles;
    const int group = L / (kF8Raster * nnt), first = group * kF8Raster;
    const int gsz = min(ntt - first, kF8Raster), within = L % (kF8Raster * nnt);
    const int tt = first + within % gsz, ntg = within / gsz;
    int wi = 0;
    for (int i = 1; i < a.count; ++i)
        if (ntg >= a.w[i].nt_begin) wi = i;
    const int t0 = tt * S::BT;
    f8_tile<TA, TB, WT, WR, NST, EX, false>(a, t0, min(t0 + S::BT, a.rows), wi, (ntg - a.w[wi].nt_begin) * (S::BR / 16), 0);
}

// The same over rows sorted by group (one wave of tokens): a tile of 32 TA
// places of one group, the last one of a group on the half or quarter of its
// blocks that holds its rows.
template <int TA, int TB, int WR, int NST, int EX, int OCC>
__global__ __launch_bounds__(64 * WR)
__attribute__((amdgpu_waves_per_eu(OCC, OCC))) void f8_group_kernel(const F8GemmArgs a) {
    constexpr int BT = 32 * TA, BRG = 2 * TB * WR;
    const int nnt = a.n_tiles, lane = threadIdx.x & 63;
    // the full tiles first, then the groups' last ones, whose shorter work
    // evens out the end of the launch
    const GroupTiles full = scan_tiles<kTilesFull>(a.offsets, a.groups, BT, lane);
    const GroupTiles part = scan_tiles<kTilesPart>(a.offsets, a.groups, BT, lane);
    const bool is_full = (int)blockIdx.x < full.total * nnt;
    const int nblk = (is_full ? full.total : part.total) * nnt, id = (int)blockIdx.x - (is_full ? 0 : full.total * nnt);
    if (id >= nblk) return;
    const int q8 = nblk / 8, r8 = nblk % 8, xcd = id % 8, j8 = id / 8;
    const int L = xcd < r8 ? xcd * (q8 + 1) + j8 : r8 * (q8 + 1) + (xcd - r8) * q8 + j8;
    const GroupTile tile = is_full ? tile_at<kTilesFull>(full, a.offsets, BT, L / nnt) : tile_at<kTilesPart>(part, a.offsets, BT, L / nnt);
    const int in = L - tile.before * nnt, ntg = in / tile.count;
    const int left = is_full ? BT : (tile.end - tile.begin) % BT;
    const int t0 = is_full ? tile.begin + (in - ntg * tile.count) * BT : tile.end - left;
    const int t_end = min(t0 + BT, tile.end);
    int wi = 0;
    for (int i = 1; i < a.count; ++i)
        if (ntg >= a.w[i].nt_begin) wi = i;
    const int rg0 = (ntg - a.w[wi].nt_begin) * BRG;
    if (2 * left > BT || TA == 1) {
        f8_tile<TA, TB, 1, WR, NST, EX, true>(a, t0, t_end, wi, rg0, tile.e);
    } else if constexpr (TA == 2) {
        f8_tile<1, TB, 1, WR, NST, EX, true>(a, t0, t_end, wi, rg0, tile.e);
    } else if constexpr (TA == 4) {
        if (4 * left > BT) f8_tile<2, TB, 1, WR, NST, EX, true>(a, t0, t_end, wi, rg0, tile.e);
        else f8_tile<1, TB, 1, WR, NST, EX, true>(a, t0, t_end, wi, rg0, tile.e);
    }
}

}  // namespace kxw4
