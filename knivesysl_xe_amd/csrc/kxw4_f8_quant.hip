// kxw4_f8_quant.hip — the 8-bit floating tier's quantizers and weight layouts.
//
// Rows: top = max(max |x|, 2^-100) of a block of 128 columns, scale = top / 448,
// code = e4m3(x * (448 / top)), each operation rounded once. The floor keeps
// 448 / top finite; a block below it (zeros among them) has codes of a relative
// error past e4m3's. A NaN or an infinity in a block makes a NaN code, so a
// product of that row is NaN. Bound: memory, one read and one write; with SiLU of
// BF16 rows and no values out, its arithmetic (3,965 x 17,408: 94 us, 3.7 TB/s, VALU
// 88 % of the cycles; values too 131 us, 4.7; 4,096 x 17,408 of FP32 134 us, 4.8).
#include "kxw4_f8.hpp"

namespace kxw4 {

struct F8QuantArgs {
    const void *x, *up;                                      // up: SiLU(x) * up
    float *out;                                              // the product's values, or NULL
    uint8_t *q;
    float *scale;
    int T, K, KB;
};

template <bool BF16>
__device__ __forceinline__ void f8_load8(const void *p, size_t i, float (&v)[8]) {
    if constexpr (BF16) {
        const uint4 u = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p) + i);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[2 * j] = __uint_as_float(w[j] << 16);
            v[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
        }
    } else {
        const float *f = static_cast<const float *>(p) + i;
        const float4 a = *reinterpret_cast<const float4 *>(f), b = *reinterpret_cast<const float4 *>(f + 4);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
}

// 16 lanes a block of one row, eight columns a lane; neighbouring units are the
// same block of neighbouring rows, whose scales lie side by side. One block a
// lane: two, four and eight with their loads in flight together took as long or
// longer at every size (512 x 17,408 BF16: 7.0, 7.7, 7.7, 9.1 us; 16,384 x 5,120:
// 52, 52, 56, 59, 4.8 TB/s of the 5.0 that a copy reaches).
template <bool BF16, bool SILU>
__global__ __launch_bounds__(256) void f8_quant_kernel(const F8QuantArgs a) {
    const int l16 = threadIdx.x & 15;
    const uint32_t unit = blockIdx.x * 16u + (threadIdx.x >> 4);
    const int kb = (int)(unit / (uint32_t)a.T), t = (int)(unit % (uint32_t)a.T);
    if (kb >= a.KB) return;
    const size_t row = (size_t)t * a.K;
    const int k = kb * kF8Block + 8 * l16;
    float v[8] = {};
    if (k < a.K) f8_load8<BF16>(a.x, row + k, v);            // (K is a multiple of 16)
    if constexpr (SILU) {
        float u[8] = {};
        if (k < a.K) f8_load8<BF16>(a.up, row + k, u);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (v[j] / (1.0f + expf(-v[j]))) * u[j];
        if (a.out && k < a.K) {
            *reinterpret_cast<float4 *>(a.out + row + k) = make_float4(v[0], v[1], v[2], v[3]);
            *reinterpret_cast<float4 *>(a.out + row + k + 4) = make_float4(v[4], v[5], v[6], v[7]);
        }
    }
    float top = kF8Floor;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(v[j]));
    top = f8_row_max(top);
    const float up = kF8Max / top;
    uint2 c;
    c.x = f8_pack(v[0] * up, v[1] * up, v[2] * up, v[3] * up);
    c.y = f8_pack(v[4] * up, v[5] * up, v[6] * up, v[7] * up);
    *reinterpret_cast<uint2 *>(a.q + ((size_t)t * a.KB + kb) * kF8Block + 8 * l16) = c;
    if (l16 == 0) a.scale[(size_t)kb * a.T + t] = top / kF8Max;
}

template <bool BF16, bool SILU>
static int quant_rows(const F8QuantArgs &a, hipStream_t st) {
    const long long grid = ((long long)a.T * a.KB + 15) / 16;
    if (grid > grid_limit(256)) return -2;
    hipLaunchKernelGGL((f8_quant_kernel<BF16, SILU>), dim3((unsigned)grid), dim3(256), 0, st, a);
    return hipGetLastError() == hipSuccess ? 0 : -6;
}

int launch_f8_quantize(const void *x, bool bf16, int T, int K, uint8_t *q, float *scale, hipStream_t st) {
    const F8QuantArgs a{x, nullptr, nullptr, q, scale, T, K, f8_blocks(K)};
    return bf16 ? quant_rows<true, false>(a, st) : quant_rows<false, false>(a, st);
}

int launch_f8_silu_mul(float *out, const void *gate, const void *up, bool bf16, int T, int K, uint8_t *q, float *scale,
                       hipStream_t st) {
    const F8QuantArgs a{gate, up, out, q, scale, T, K, f8_blocks(K)};
    return bf16 ? quant_rows<true, true>(a, st) : quant_rows<false, true>(a, st);
}

// ---- weights: a work-group for each 128 x 128 block --------------------------

struct F8WeightArgs {
    const void *src;                                         // values or codes [groups][M][K], or packed tiles
    uint8_t *codes;                                          // tiles, or codes [groups][M][K]
    const float *in_scales;
    float *scales;                                           // [groups][MB][KB]
    int M, K, MB, KB;
};

// Block of a work-group: x the column block, y the row block, z the group (in
// steps of the grid).
#define KXW4_F8_BLOCK_PIECES(p, row, piece)                                                          \
    for (int i_ = 0, p = threadIdx.x, row = p >> 3, piece = p & 7; i_ < 4; ++i_, p += 256, row = p >> 3)

enum { kF8Pack = 0, kF8Unpack = 1 };

// Codes between their natural order and the tiles, 16 at a time.
template <int DIR>
__global__ __launch_bounds__(256) void f8_pack_kernel(const F8WeightArgs a, int groups) {
    const int RG = a.M / 16, kb = blockIdx.x, mb = blockIdx.y;
    for (int e = blockIdx.z; e < groups; e += gridDim.z) {
        const size_t natural = (size_t)e * a.M * a.K, packed = (size_t)e * RG * a.KB * kF8Tile;
        KXW4_F8_BLOCK_PIECES(p, row, piece) {
            const int m = mb * kF8Block + row, k = kb * kF8Block + 16 * piece;
            if (m >= a.M) continue;
            const size_t at = packed + ((size_t)(m / 16) * a.KB + kb) * kF8Tile + f8_piece(m % 16, piece);
            const size_t nat = natural + (size_t)m * a.K + k;
            if constexpr (DIR == kF8Pack) {
                uint4 v = make_uint4(0, 0, 0, 0);
                if (k < a.K) v = *reinterpret_cast<const uint4 *>(static_cast<const uint8_t *>(a.src) + nat);
                *reinterpret_cast<uint4 *>(a.codes + at) = v;
            } else if (k < a.K) {
                *reinterpret_cast<uint4 *>(a.codes + nat) = *reinterpret_cast<const uint4 *>(static_cast<const uint8_t *>(a.src) + at);
            }
        }
    }
}

// Weights' values to codes: 5,120 x 5,120 of BF16 in 20 us (3.9 TB/s), 17,408 x 5,120
// in 55 (4.9); of FP32 the first in 29 (4.5).
template <bool BF16>
__global__ __launch_bounds__(256) void f8_weight_kernel(const F8WeightArgs a, int groups) {
    __shared__ float red[4];
    const int RG = a.M / 16, kb = blockIdx.x, mb = blockIdx.y;
    for (int e = blockIdx.z; e < groups; e += gridDim.z) {
        const size_t natural = (size_t)e * a.M * a.K, packed = (size_t)e * RG * a.KB * kF8Tile;
        float v[4][16];
        float top = kF8Floor;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = (threadIdx.x >> 3) + 32 * i, piece = threadIdx.x & 7;
            const int m = mb * kF8Block + row, k = kb * kF8Block + 16 * piece;
            float lo[8] = {}, hi[8] = {};
            if (m < a.M && k < a.K) {
                f8_load8<BF16>(a.src, natural + (size_t)m * a.K + k, lo);
                f8_load8<BF16>(a.src, natural + (size_t)m * a.K + k + 8, hi);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[i][j] = lo[j];
                v[i][8 + j] = hi[j];
                top = fmaxf(top, fmaxf(fabsf(lo[j]), fabsf(hi[j])));
            }
        }
        top = f8_row_max(top);
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        __syncthreads();                                     // (the last group's reads of red)
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
        __syncthreads();
        top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        const float up = kF8Max / top;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = (threadIdx.x >> 3) + 32 * i, piece = threadIdx.x & 7;
            const int m = mb * kF8Block + row;
            if (m >= a.M) continue;
            uint32_t c[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                c[j] = f8_pack(v[i][4 * j] * up, v[i][4 * j + 1] * up, v[i][4 * j + 2] * up, v[i][4 * j + 3] * up);
            *reinterpret_cast<uint4 *>(a.codes + packed + ((size_t)(m / 16) * a.KB + kb) * kF8Tile + f8_piece(m % 16, piece)) =
                make_uint4(c[0], c[1], c[2], c[3]);
        }
        if (threadIdx.x == 0) a.scales[((size_t)e * a.MB + mb) * a.KB + kb] = top / kF8Max;
    }
}

// The transposed weight: blocks and their scales change places, codes turn
// inside a block. Columns of the result past M are zero codes.
// (LDS rows of 136 bytes: the 32 lanes of a piece read 32 banks side by side, the
// other 32 the rest. Each lane turns 16 rows of four columns, as dwords, with byte
// permutes: 5,120 x 5,120 in 17 us, 3.0 TB/s, 17,408 x 5,120 in 51, 3.5; read byte
// by byte, with 34 % of the cycles in bank conflicts, the first took 21.)
__global__ __launch_bounds__(256) void f8_transpose_kernel(const F8WeightArgs a, int groups) {
    constexpr int LD = kF8Block + 8;
    __shared__ __attribute__((aligned(16))) uint8_t s[kF8Block * LD];
    const int RG = a.M / 16, kb = blockIdx.x, mb = blockIdx.y;
    const int RGt = a.K / 16;
    for (int e = blockIdx.z; e < groups; e += gridDim.z) {
        const size_t in = (size_t)e * RG * a.KB * kF8Tile, out = (size_t)e * RGt * a.MB * kF8Tile;
        __syncthreads();                                     // (the last group's reads of s)
        KXW4_F8_BLOCK_PIECES(p, row, piece) {
            const int m = mb * kF8Block + row;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (m < a.M)
                v = *reinterpret_cast<const uint4 *>(static_cast<const uint8_t *>(a.src) + in +
                                                     ((size_t)(m / 16) * a.KB + kb) * kF8Tile + f8_piece(m % 16, piece));
            uint2 *to = reinterpret_cast<uint2 *>(s + row * LD + 16 * piece);
            to[0] = make_uint2(v.x, v.y);
            to[1] = make_uint2(v.z, v.w);
        }
        __syncthreads();
        // rows 4 c4 .. 4 c4 + 3 of the result, 16 of their columns
        const int c4 = threadIdx.x & 31, piece = threadIdx.x >> 5, k = kb * kF8Block + 4 * c4;
        uint32_t c[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t d[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) d[r] = *reinterpret_cast<const uint32_t *>(s + (16 * piece + 4 * j + r) * LD + 4 * c4);
            // bytes 0 and 1, then 2 and 3, of the rows in pairs
            const uint32_t a0 = __builtin_amdgcn_perm(d[1], d[0], 0x05010400), a1 = __builtin_amdgcn_perm(d[1], d[0], 0x07030602);
            const uint32_t b0 = __builtin_amdgcn_perm(d[3], d[2], 0x05010400), b1 = __builtin_amdgcn_perm(d[3], d[2], 0x07030602);
            c[0][j] = __builtin_amdgcn_perm(b0, a0, 0x05040100);
            c[1][j] = __builtin_amdgcn_perm(b0, a0, 0x07060302);
            c[2][j] = __builtin_amdgcn_perm(b1, a1, 0x05040100);
            c[3][j] = __builtin_amdgcn_perm(b1, a1, 0x07060302);
        }
        if (k < a.K) {                                       // (K is a multiple of 16)
            uint8_t *to = a.codes + out + ((size_t)(k / 16) * a.MB + mb) * kF8Tile + f8_piece(k % 16, piece);
#pragma unroll
            for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4 *>(to + 16 * i) = make_uint4(c[i][0], c[i][1], c[i][2], c[i][3]);
        }
        if (threadIdx.x == 0)
            a.scales[((size_t)e * a.KB + kb) * a.MB + mb] = a.in_scales[((size_t)e * a.MB + mb) * a.KB + kb];
    }
}

// A work-group a block of 128 x 128, groups in turn where the blocks of all would
// take 2^32 threads and more, which the runtime cuts without an error. False:
// those of one group do.
static bool f8_weight_grid(const F8WeightArgs &a, int groups, dim3 &grid) {
    const long long most = grid_limit(256) / ((long long)a.KB * a.MB);
    grid = dim3((unsigned)a.KB, (unsigned)a.MB, (unsigned)(groups < most ? groups : most));
    return most > 0;
}

int launch_f8_pack(const uint8_t *codes, int groups, int M, int K, uint8_t *out, hipStream_t st) {
    const F8WeightArgs a{codes, out, nullptr, nullptr, M, K, f8_blocks(M), f8_blocks(K)};
    dim3 grid;
    if (!f8_weight_grid(a, groups, grid)) return -2;
    hipLaunchKernelGGL(f8_pack_kernel<kF8Pack>, grid, dim3(256), 0, st, a, groups);
    return hipGetLastError() == hipSuccess ? 0 : -6;
}

int launch_f8_unpack(const uint8_t *tiles, int groups, int M, int K, uint8_t *codes, hipStream_t st) {
    const F8WeightArgs a{tiles, codes, nullptr, nullptr, M, K, f8_blocks(M), f8_blocks(K)};
    dim3 grid;
    if (!f8_weight_grid(a, groups, grid)) return -2;
    hipLaunchKernelGGL(f8_pack_kernel<kF8Unpack>, grid, dim3(256), 0, st, a, groups);
    return hipGetLastError() == hipSuccess ? 0 : -6;
}

int launch_f8_weight(const void *w, bool bf16, int groups, int M, int K, uint8_t *codes, float *scales, hipStream_t st) {
    const F8WeightArgs a{w, codes, nullptr, scales, M, K, f8_blocks(M), f8_blocks(K)};
    dim3 grid;
    if (!f8_weight_grid(a, groups, grid)) return -2;
    if (bf16) hipLaunchKernelGGL(f8_weight_kernel<true>, grid, dim3(256), 0, st, a, groups);
    else hipLaunchKernelGGL(f8_weight_kernel<false>, grid, dim3(256), 0, st, a, groups);
    return hipGetLastError() == hipSuccess ? 0 : -6;
}

int launch_f8_transpose(const uint8_t *tiles, const float *scales, int groups, int M, int K, uint8_t *out, float *out_scales,
                        hipStream_t st) {
    const F8WeightArgs a{tiles, out, scales, out_scales, M, K, f8_blocks(M), f8_blocks(K)};
    dim3 grid;
    if (!f8_weight_grid(a, groups, grid)) return -2;
    hipLaunchKernelGGL(f8_transpose_kernel, grid, dim3(256), 0, st, a, groups);
    return hipGetLastError() == hipSuccess ? 0 : -6;
}

}  // namespace kxw4
