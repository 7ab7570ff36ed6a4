// kxw4_f8.hpp — the 8-bit floating tier: e4m3 codes with an FP32 scale for each
// block of 128, of rows (activations: one row by 128 columns) and of weights
// (128 x 128). No counterpart in the reference, whose tiers are integer.
//
// y[t][m] = sum over blocks j of P_j * (sx[t][j] * sw[m / 128][j]),
// P_j = sum over the block's columns of code * code.
//
// Weights: tiles of 16 rows x 128 columns, 2,048 bytes, tile (rg, kb) of a
// weight at (rg * KB + kb) * 2048. Half h of a tile (1,024 bytes) holds columns
// 64h..64h+63, lane l's 16 bytes of it row l % 16 and columns 64h + 16 (l / 16)
// and on: a wave reads a tile as two loads of 16 bytes a lane, and the reads of
// a tile in LDS touch every bank once. Columns past K are zero codes.
// Rows: [T][128 KB] codes in their order, zeros past K; scales [KB][T], so the
// scales of a tile of rows lie together.
#pragma once

#include "kxw4_device.hpp"
#include "kxw4_internal.hpp"

namespace kxw4 {

constexpr int kF8Block = 128;
constexpr int kF8Tile = 2048;                                // 16 rows x 128 columns
constexpr float kF8Max = 448.0f;                             // the largest e4m3 value
constexpr float kF8Floor = 0x1p-100f;                        // least block maximum: 448 / it stays finite

inline __host__ __device__ int f8_blocks(int n) { return (n + kF8Block - 1) / kF8Block; }

typedef float v16f __attribute__((ext_vector_type(16)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));

// Byte of a weight tile that holds (row, 16-column piece).
__device__ __forceinline__ int f8_piece(int row, int piece) {
    return 1024 * (piece >> 2) + 16 * (16 * (piece & 3) + row);
}

// Maximum over the 16 lanes of a DPP row.
template <int CTRL>
__device__ __forceinline__ float f8_dpp_max(float v) {
    return fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, false)));
}
__device__ __forceinline__ float f8_row_max(float v) {
    v = f8_dpp_max<0xB1>(v);                                 // quad_perm [1,0,3,2], [2,3,0,1], then the mirrors of 8 and 16
    v = f8_dpp_max<0x4E>(v);
    v = f8_dpp_max<0x141>(v);
    return f8_dpp_max<0x140>(v);
}

// Four values as e4m3 codes (v_cvt_pk_fp8_f32: round to nearest even, a value
// past 464 or a NaN gives the NaN code).
__device__ __forceinline__ uint32_t f8_pack(float a, float b, float c, float d) {
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
}

// Eight codes as BF16, exactly (four mantissa bits in eight).
__device__ __forceinline__ v8bf f8_to_bf16(uint32_t lo, uint32_t hi) {
    const v2bf a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false);
    const v2bf b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
    const v2bf c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false);
    const v2bf d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
    return v8bf{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

}  // namespace kxw4
