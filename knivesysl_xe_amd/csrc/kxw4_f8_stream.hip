// kxw4_f8_stream.hip — products of the 8-bit floating tier for few rows (a
// decode step, or a few rows of each expert): the weights are read once for
// all rows of a tile, straight into registers.
//
// A work-group owns 16 R weight rows and a tile of up to 16 TB rows of x; its
// waves take the column blocks in turn and add their sums up in LDS, in the
// order of the waves. Codes become BF16 in registers (exactly), the products
// run on the 16x16x32 BF16 MFMA (operands: weight rows x rows of x, so a lane
// holds four outputs of one row of x and one scale): its sums are FP32 without
// the cut that the f8 MFMA makes (kxw4_f8_gemm.hpp), and the rate of either is
// far above what the weights' stream needs. Rows that come as values are
// quantized by each wave for the blocks it takes, which saves a launch.
//
// Bound: HBM, where there are weights enough (8 rows, 2 x 17,408 x 5,120: 178 MB
// in 30 to 32 us, 5.6 to 5.9 TB/s; 16 x 8 rows over 64 experts, 2 x 1,024 x 5,120:
// 582 MB, of which 499 from HBM, in 73 to 79 us; a pure read reaches 6.3); below
// that a wave's round trips, one after another (one row, 4,096 x 4,096: eight
// blocks a wave, two of them in flight: 16.8 MB in 8.0 us).
#include "kxw4_f8.hpp"
#include "kxw4_f8_route.hpp"
#include "kxw4_groups.hpp"

namespace kxw4 {

enum { kF8Codes = 0, kF8Bf16 = 1, kF8F32 = 2 };              // what the rows of x come as

// The share of a column block of one row of x that a lane holds: columns
// 64h + 16 (l / 16) and on, 16 of each half.
template <int X>
struct F8Rows {
    v4u q[2];
    float scale;
};
template <>
struct F8Rows<kF8Bf16> {
    v4u x[4];
};
template <>
struct F8Rows<kF8F32> {
    v4u x[8];
};

// Loads through a buffer descriptor: what lies past its range reads as zero and
// moves nothing, so the loads ahead of a wave's last blocks need no branch.
constexpr int kF8Word3 = 0x00020000;                         // untyped buffer, format 32
constexpr uint32_t kF8Past = 0x80000000u;                    // an offset past every range (all are below 2^31)
constexpr int kF8Stream = 2;                                 // non-temporal: the weights are read once
template <int AUX>
__device__ __forceinline__ v4u f8_buffer(const void *base, uint32_t range, uint32_t lane, uint32_t at) {
    return __builtin_amdgcn_raw_buffer_load_b128(__builtin_amdgcn_make_buffer_rsrc((void *)base, 0, range, kF8Word3), lane, at, AUX);
}

// xp: the first row's address, row: this lane's from it; both within 2^31 bytes
// of the descriptor's base.
template <int X>
__device__ __forceinline__ void f8_rows_load(F8Rows<X> &f, const F8StreamArgs &a, const void *xp, uint32_t range, const float *sp,
                                             uint32_t s_range, uint32_t row, int kb, int g) {
    if constexpr (X == kF8Codes) {
        const uint32_t at = kb < a.KB ? kb * kF8Block : kF8Past, off = row * (uint32_t)(a.KB * kF8Block) + 16 * g;
        f.q[0] = f8_buffer<0>(xp, range, off, at);
        f.q[1] = f8_buffer<0>(xp, range, off + 64, at);
        const uint32_t sat = kb < a.KB ? (uint32_t)kb * (uint32_t)a.rows * 4 : kF8Past;
        f.scale = __int_as_float(__builtin_amdgcn_raw_buffer_load_b32(__builtin_amdgcn_make_buffer_rsrc((void *)sp, 0, s_range, kF8Word3),
                                                                      row * 4, sat, 0));
    } else {
        constexpr int N = X == kF8Bf16 ? 2 : 4, B = X == kF8Bf16 ? 2 : 4;
        const uint32_t at = (uint32_t)kb * (kF8Block * B);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int k = 64 * h + 16 * g;
            // (columns past K, and with them blocks past the last)
            const uint32_t off = kb * kF8Block + k < a.K ? (row * (uint32_t)a.K + k) * B : kF8Past;
#pragma unroll
            for (int i = 0; i < N; ++i) f.x[h * N + i] = f8_buffer<0>(xp, range, off + 16 * i, at);
        }
    }
}

// The codes as operands (four of eight columns) and the row's scale.
template <int X>
__device__ __forceinline__ float f8_rows_operands(const F8Rows<X> &f, v8bf (&b)[4]) {
    if constexpr (X == kF8Codes) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            b[2 * h] = f8_to_bf16(f.q[h].x, f.q[h].y);
            b[2 * h + 1] = f8_to_bf16(f.q[h].z, f.q[h].w);
        }
        return f.scale;
    } else {
        float v[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            if constexpr (X == kF8Bf16) {
                const uint32_t w = f.x[i / 8][(i / 2) % 4];
                v[i] = __uint_as_float(i & 1 ? w & 0xFFFF0000u : w << 16);
            } else {
                v[i] = __uint_as_float(f.x[i / 4][i % 4]);
            }
        }
        float top = kF8Floor;
#pragma unroll
        for (int i = 0; i < 32; ++i) top = fmaxf(top, fabsf(v[i]));
        top = fmaxf(top, __shfl_xor(top, 16, 64));           // the four lanes of a row
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const float up = kF8Max / top;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t lo = f8_pack(v[8 * j] * up, v[8 * j + 1] * up, v[8 * j + 2] * up, v[8 * j + 3] * up);
            const uint32_t hi = f8_pack(v[8 * j + 4] * up, v[8 * j + 5] * up, v[8 * j + 6] * up, v[8 * j + 7] * up);
            b[j] = f8_to_bf16(lo, hi);
        }
        return top / kF8Max;
    }
}

// D: column blocks in flight per wave
template <int R, int TB, int X, bool GRP, int D>
__global__ __launch_bounds__(512) void f8_stream_kernel(const F8StreamArgs a) {
    extern __shared__ __attribute__((aligned(16))) float red[];
    const int lane = threadIdx.x & 63, m16 = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = blockDim.x >> 6;
    // ---- the tile: rows of x [t0, t_end) of group e, row-groups from rg0 ----
    int t0, t_end, e = 0, rb;
    if constexpr (GRP) {
        const GroupTiles s = scan_tiles(a.offsets, a.groups, 16 * TB, lane);
        const int u = blockIdx.x / a.row_blocks;
        rb = blockIdx.x - u * a.row_blocks;
        if (u >= s.total) return;
        const GroupTile tile = tile_at(s, a.offsets, 16 * TB, u);
        e = tile.e;
        t0 = tile.begin + tile.index * 16 * TB;
        t_end = min(tile.end, t0 + 16 * TB);
    } else {
        const int u = blockIdx.x / a.row_blocks;
        rb = blockIdx.x - u * a.row_blocks;
        t0 = u * 16 * TB;
        t_end = min(a.rows, t0 + 16 * TB);
    }
    int wi = 0;
    for (int i = 1; i < a.count; ++i)
        if (rb >= a.w[i].blk) wi = i;
    const F8StreamWeight W = a.w[wi];
    const int RG = W.M / 16, rg0 = (rb - W.blk) * R;
    const uint8_t *codes = W.codes + ((size_t)e * RG + rg0) * a.KB * kF8Tile;
    // (R divides 8, so the row-groups share a block of 128 rows)
    const float *sw = W.scales + ((size_t)e * f8_blocks(W.M) + rg0 / 8) * a.KB;
    const uint32_t w_range = min(R, RG - rg0) * a.KB * kF8Tile, lane16 = lane * 16;
    // the lane's row of x in each block of 16 (past the tile: its last), from
    // the tile's first row (dense) or row 0
    uint32_t xrow[TB];
#pragma unroll
    for (int b = 0; b < TB; ++b) {
        const int t = min(t0 + 16 * b + m16, t_end - 1);
        if constexpr (GRP) xrow[b] = a.order ? (uint32_t)a.order[t] / (uint32_t)a.k : t;
        else xrow[b] = t - t0;
    }
    constexpr int XB = X == kF8F32 ? 4 : X == kF8Bf16 ? 2 : 1;
    const size_t x_stride = X == kF8Codes ? (size_t)a.KB * kF8Block : (size_t)a.K * XB;
    const int x_first = GRP ? 0 : t0;
    const uint8_t *xp = static_cast<const uint8_t *>(X == kF8Codes ? a.q : a.x) + x_first * x_stride;
    const uint32_t x_range = (uint32_t)((GRP ? a.rows : t_end - t0) * x_stride);
    const float *sp = a.sx + x_first;
    const uint32_t s_range = (uint32_t)(((size_t)(a.KB - 1) * a.rows + (GRP ? a.rows : t_end - t0)) * 4);

    v4u wt[D][R][2];
    F8Rows<X> xs[D][TB];
    float ws[D];
    v4f acc[R][TB];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int b = 0; b < TB; ++b) acc[r][b] = v4f{0, 0, 0, 0};
    auto load = [&](int d, int kb) {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                // (row-groups past M and blocks past the last: nothing is read)
                const uint32_t at = kb < a.KB ? (uint32_t)(r * a.KB + kb) * kF8Tile + 1024 * h : kF8Past;
                wt[d][r][h] = f8_buffer<kF8Stream>(codes, w_range, lane16, at);
            }
        ws[d] = sw[min(kb, a.KB - 1)];
#pragma unroll
        for (int b = 0; b < TB; ++b) f8_rows_load<X>(xs[d][b], a, xp, x_range, sp, s_range, xrow[b], kb, g);
    };
#pragma unroll
    for (int d = 0; d < D; ++d) load(d, wave + d * nw);
    for (int kb0 = wave; kb0 < a.KB; kb0 += D * nw) {
#pragma unroll
        for (int d = 0; d < D; ++d) {
            if (kb0 + d * nw < a.KB) {
                v8bf xb[TB][4];
                float s[TB];
#pragma unroll
                for (int b = 0; b < TB; ++b) s[b] = f8_rows_operands<X>(xs[d][b], xb[b]) * ws[d];
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    v8bf wb[4];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        wb[2 * h] = f8_to_bf16(wt[d][r][h].x, wt[d][r][h].y);
                        wb[2 * h + 1] = f8_to_bf16(wt[d][r][h].z, wt[d][r][h].w);
                    }
#pragma unroll
                    for (int b = 0; b < TB; ++b) {
                        v4f p = {0, 0, 0, 0};
#pragma unroll
                        for (int j = 0; j < 4; ++j) p = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wb[j], xb[b][j], p, 0, 0, 0);
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[r][b][i] = __builtin_fmaf(p[i], s[b], acc[r][b][i]);
                    }
                }
            }
            load(d, kb0 + (D + d) * nw);
        }
    }
    // ---- the waves' sums, in their order ----
    v4f *part = reinterpret_cast<v4f *>(red);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int b = 0; b < TB; ++b) part[(wave * R * TB + r * TB + b) * 64 + lane] = acc[r][b];
    __syncthreads();
    for (int i = threadIdx.x; i < R * TB * 64; i += blockDim.x) {
        v4f v = part[i];
        for (int w = 1; w < nw; ++w) {
            const v4f o = part[w * R * TB * 64 + i];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] += o[j];
        }
        const int l = i & 63, rbk = i >> 6, r = rbk / TB, b = rbk % TB;
        const int t = t0 + 16 * b + (l & 15), row = (rg0 + r) * 16 + 4 * (l >> 4);
        if (t >= t_end || rg0 + r >= RG) continue;
        const size_t at = (size_t)t * W.M + row;
        if (a.residual) {
            const float4 x = *reinterpret_cast<const float4 *>(a.residual + at);
            v[0] += x.x;
            v[1] += x.y;
            v[2] += x.z;
            v[3] += x.w;
        }
        if (a.y_bf16)
            *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(W.y) + at) = make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));
        else
            *reinterpret_cast<float4 *>(static_cast<float *>(W.y) + at) = make_float4(v[0], v[1], v[2], v[3]);
    }
}

template <int R, int TB, int X, bool GRP, int D>
static int f8_stream(F8StreamArgs &a, int nw, hipStream_t st) {
    int blk = 0;
    for (int i = 0; i < a.count; ++i) {
        a.w[i].blk = blk;
        blk += (a.w[i].M / 16 + R - 1) / R;
    }
    a.row_blocks = blk;
    const long long tiles = GRP ? tiles_at_most(a.N, a.groups, 16 * TB) : (a.rows + 16 * TB - 1) / (16 * TB);
    const long long grid = tiles * blk;
    if (grid > grid_limit(64 * nw)) return -2;
    const size_t lds = (size_t)nw * R * TB * 1024;
    hipLaunchKernelGGL((f8_stream_kernel<R, TB, X, GRP, D>), dim3((unsigned)grid), dim3(64 * nw), lds, st, a);
    return hipGetLastError() == hipSuccess ? 0 : -6;
}

template <int TB, int X, bool GRP>
static int f8_stream_shaped(F8StreamArgs &a, hipStream_t st) {
    F8Sizes s{device_cus(), GRP ? a.N : a.rows, a.KB, a.count, {}, a.groups, a.y_bf16 != 0};
    for (int i = 0; i < a.count; ++i) s.M[i] = a.w[i].M;
    const F8StreamShape shape = f8_stream_shape(s, 16 * TB);
    return shape.row_groups == 1 ? f8_stream<1, TB, X, GRP, 2>(a, shape.waves, st) : f8_stream<2, TB, X, GRP, 2>(a, shape.waves, st);
}

template <bool GRP>
static int f8_stream_typed(F8StreamArgs &a, int x, int rows, hipStream_t st) {
    if (x == kF8Bf16) return rows == 16 ? f8_stream_shaped<1, kF8Bf16, GRP>(a, st) : f8_stream_shaped<2, kF8Bf16, GRP>(a, st);
    if (x == kF8F32) return rows == 16 ? f8_stream_shaped<1, kF8F32, GRP>(a, st) : f8_stream_shaped<2, kF8F32, GRP>(a, st);
    return rows == 16 ? f8_stream_shaped<1, kF8Codes, GRP>(a, st) : f8_stream_shaped<2, kF8Codes, GRP>(a, st);
}

int launch_f8_stream(F8StreamArgs &a, int x, int rows, hipStream_t st) {
    return a.groups ? f8_stream_typed<true>(a, x, rows, st) : f8_stream_typed<false>(a, x, rows, st);
}

}  // namespace kxw4
