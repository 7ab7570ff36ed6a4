// kxw4_adapter.hip — low-rank adapters of many requests beside a shared
// projection: out[t] = y[t] + scale_e B_e (A_e x[t]), e the adapter of token
// t, out[t] = y[t] for a token without one. No counterpart in the reference.
//
// The tokens come sorted by adapter (RouteArgs' plan with one choice per
// token), in tiles that belong to one adapter. Two launches: `low` = A x into
// FP32 scratch, K split over waves and work-groups, then the update.
//
// Arithmetic. A and B are BF16, so a BF16 x makes exact products on the BF16
// MFMA, summed in FP32. An FP32 value is cut into three BF16 parts of eight
// mantissa bits each, which hold all 24 (split3), and each part takes an MFMA
// of its own: the products are exact again. `low` stays FP32 between the
// launches and is cut the same way. The sums run in a fixed order: within a
// wave's steps, then the waves of a work-group, then the work-groups' parts.
//
// v_mfma_f32_16x16x32_bf16: lane l supplies row (A) / column (B) l%16 and the
// eight K slots 8*(l/16)..+7; result register i of lane l is row 4*(l/16)+i,
// column l%16.
#include "kxw4_device.hpp"
#include "kxw4_groups.hpp"
#include "kxw4_internal.hpp"

#include <algorithm>
#include <type_traits>

namespace kxw4 {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));

__device__ __forceinline__ v4f mfma_bf16(v4u a, v4u b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
}

// x as the sum of three BF16 values, by cutting: each part takes the leading
// eight mantissa bits of what the one before left, and the differences are
// exact. An infinity or NaN goes into the first part whole.
__device__ __forceinline__ void split3(float x, uint32_t (&part)[3]) {
    const uint32_t b = __float_as_uint(x);
    const bool finite = (b & 0x7F800000u) != 0x7F800000u;
    part[0] = (b & 0xFFFF0000u) | (x != x ? 0x00400000u : 0u);
    const float r1 = finite ? x - __uint_as_float(part[0]) : 0.0f;
    part[1] = __float_as_uint(r1) & 0xFFFF0000u;
    const float r2 = r1 - __uint_as_float(part[1]);
    part[2] = __float_as_uint(r2) & 0xFFFF0000u;
}

// Eight values as three operands.
__device__ __forceinline__ void split8(const float (&v)[8], v4u (&op)[3]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t lo[3], hi[3];
        split3(v[2 * i], lo);
        split3(v[2 * i + 1], hi);
#pragma unroll
        for (int q = 0; q < 3; ++q) op[q][i] = lo[q] >> 16 | hi[q];
    }
}

__device__ __forceinline__ void load8(const float *p, float (&v)[8]) {
    const v4f lo = reinterpret_cast<const v4f *>(p)[0], hi = reinterpret_cast<const v4f *>(p)[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[i] = lo[i];
        v[4 + i] = hi[i];
    }
}

constexpr int kLowWaves = 4, kLowTile = 16;

// low[s][p][c] = sum over the s-th part of K of A[c][k] x[order[p]][k]: a
// work-group takes 16 places of one adapter and part s, its waves consecutive
// runs of 32-K steps, all r columns (CT tiles of 16). Operands come straight
// from memory: a step's x piece is used by every column tile, an A piece once.
template <int CT, bool XB>
__global__ __launch_bounds__(64 * kLowWaves) void adapter_low_kernel(const AdapterArgs a) {
    __shared__ float part[kLowWaves - 1][CT][256];
    const int tid = threadIdx.x, lane = tid & 63, m = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const GroupTiles tiles = scan_tiles(a.offsets, a.n, kLowTile, lane);
    if ((int)blockIdx.x >= tiles.total) return;
    const GroupTile tile = tile_at(tiles, a.offsets, kLowTile, blockIdx.x);
    const int p0 = tile.begin + tile.index * kLowTile;
    const int steps = a.K / 32, ways = a.splits * kLowWaves, way = blockIdx.y * kLowWaves + wave;
    const int k0 = (int)((long long)steps * way / ways), k1 = (int)((long long)steps * (way + 1) / ways);

    const int token = a.order[min(p0 + m, tile.end - 1)];
    const size_t xrow = (size_t)token * a.K + 8 * g;
    const uint16_t *arow[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c)
        arow[c] = a.a + ((size_t)tile.e * a.r + min(c * 16 + m, a.r - 1)) * a.K + 8 * g;
    v4f acc[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) acc[c] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    // U steps' loads are requested before the first of them is used
    auto run = [&](int k, auto uc) {
        constexpr int U = decltype(uc)::value;
        v4u w[U][CT];
        if constexpr (XB) {
            v4u x[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                x[u] = *reinterpret_cast<const v4u *>(static_cast<const uint16_t *>(a.x) + xrow + 32 * (k + u));
#pragma unroll
                for (int c = 0; c < CT; ++c) w[u][c] = *reinterpret_cast<const v4u *>(arow[c] + 32 * (k + u));
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int c = 0; c < CT; ++c) acc[c] = mfma_bf16(x[u], w[u][c], acc[c]);
        } else {
            float v[U][8];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                load8(static_cast<const float *>(a.x) + xrow + 32 * (k + u), v[u]);
#pragma unroll
                for (int c = 0; c < CT; ++c) w[u][c] = *reinterpret_cast<const v4u *>(arow[c] + 32 * (k + u));
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                v4u x[3];
                split8(v[u], x);
#pragma unroll
                for (int c = 0; c < CT; ++c)
#pragma unroll
                    for (int q = 2; q >= 0; --q) acc[c] = mfma_bf16(x[q], w[u][c], acc[c]);
            }
        }
    };
    constexpr int kSteps = CT <= 2 ? 4 : CT <= 4 ? 2 : 1;
    int k = k0;
    for (; k + kSteps <= k1; k += kSteps) run(k, std::integral_constant<int, kSteps>{});
    for (; k < k1; ++k) run(k, std::integral_constant<int, 1>{});
    if (wave > 0) {
#pragma unroll
        for (int c = 0; c < CT; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) part[wave - 1][c][i * 64 + lane] = acc[c][i];
    }
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        const int col = c * 16 + m;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float v = acc[c][i];
#pragma unroll
            for (int w = 0; w < kLowWaves - 1; ++w) v += part[w][c][i * 64 + lane];
            const int p = p0 + 4 * g + i;
            if (p < tile.end && col < a.r) a.low[((size_t)blockIdx.y * a.T + p) * a.r + col] = v;
        }
    }
}

// out = y + scale B low. A wave takes 64 rows of B x TS tiles of 16 places of
// one adapter. B is the MFMA's first operand, its rows dealt so that lane group
// g ends up with 16 consecutive outputs (m0 + 16 g ..) of one token: tile c's
// row 4 g + i is m0 + 16 g + 4 c + i. Bound by reading y and writing out.
constexpr int kUpWaves = 4, kUpRows = 64;
template <int TS, bool YB>
__global__ __launch_bounds__(64 * kUpWaves) void adapter_up_kernel(const AdapterArgs a) {
    const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const GroupTiles tiles = scan_tiles(a.offsets, a.n, 16 * TS, lane);
    const int m0 = (blockIdx.y * kUpWaves + wave) * kUpRows;
    int p0, p1, e = -1;
    if ((int)blockIdx.x < tiles.total) {
        const GroupTile tile = tile_at(tiles, a.offsets, 16 * TS, blockIdx.x);
        e = tile.e;
        p0 = tile.begin + tile.index * 16 * TS;
        p1 = tile.end;
    } else {
        // the tokens without an adapter keep y (already there when out is y)
        p0 = a.offsets[a.n] + ((int)blockIdx.x - tiles.total) * 16 * TS;
        p1 = a.T;
        if (a.out == a.y || p0 >= p1) return;
    }
    if (m0 >= a.M) return;
    const int mg = m0 + 16 * g;                              // this lane's 16 outputs
    v4f acc[TS][4];
#pragma unroll
    for (int s = 0; s < TS; ++s)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[s][c] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    if (e >= 0) {
        const float scale = a.scale[e];
        for (int k = 8 * g; k - 8 * g < a.r; k += 32) {
            const bool in = k < a.r;
            v4u b[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int row = min(m0 + 16 * (n >> 2) + 4 * c + (n & 3), a.M - 1);
                b[c] = in ? *reinterpret_cast<const v4u *>(a.b + ((size_t)e * a.M + row) * a.r + k) : v4u{0, 0, 0, 0};
            }
#pragma unroll
            for (int s = 0; s < TS; ++s) {
                float v[8] = {};
                const int p = min(p0 + 16 * s + n, p1 - 1);
                if (in) {
                    load8(a.low + (size_t)p * a.r + k, v);
                    for (int q = 1; q < a.splits; ++q) {
                        float o[8];
                        load8(a.low + ((size_t)q * a.T + p) * a.r + k, o);
#pragma unroll
                        for (int i = 0; i < 8; ++i) v[i] += o[i];
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] *= scale;
                }
                v4u x[3];
                split8(v, x);
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int q = 2; q >= 0; --q) acc[s][c] = mfma_bf16(b[c], x[q], acc[s][c]);
            }
        }
    }
    if (mg >= a.M) return;
#pragma unroll
    for (int s = 0; s < TS; ++s) {
        const int p = p0 + 16 * s + n;
        if (p >= p1) continue;
        const size_t at = (size_t)a.order[p] * a.M + mg;
        if constexpr (YB) {
            const v4u *y = reinterpret_cast<const v4u *>(static_cast<const uint16_t *>(a.y) + at);
            v4u *out = reinterpret_cast<v4u *>(static_cast<uint16_t *>(a.out) + at);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const v4u u = y[h];
                v4u o;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int c = 2 * h + (i >> 1), r = 2 * (i & 1);
                    o[i] = round_bf16(__uint_as_float(u[i] << 16) + acc[s][c][r]) |
                           round_bf16(__uint_as_float(u[i] & 0xFFFF0000u) + acc[s][c][r + 1]) << 16;
                }
                out[h] = o;
            }
        } else {
            const v4f *y = reinterpret_cast<const v4f *>(static_cast<const float *>(a.y) + at);
            v4f *out = reinterpret_cast<v4f *>(static_cast<float *>(a.out) + at);
#pragma unroll
            for (int c = 0; c < 4; ++c) out[c] = y[c] + acc[s][c];
        }
    }
}

// Work-groups per 16-token tile of the first launch: enough to give each CU
// one while a wave keeps at least four 32-K steps.
int adapter_splits(int n, int T, int K) {
    const long long tiles = std::max(1ll, tiles_at_most(T, n, kLowTile));
    const long long most = std::max(1, K / (32 * kLowWaves * 4));
    return (int)std::max(1ll, std::min({most, 256 / tiles, 32ll}));
}

template <int CT>
static void launch_low(const AdapterArgs &a, bool x_bf16, dim3 grid, hipStream_t st) {
    if (x_bf16) hipLaunchKernelGGL((adapter_low_kernel<CT, true>), grid, dim3(64 * kLowWaves), 0, st, a);
    else hipLaunchKernelGGL((adapter_low_kernel<CT, false>), grid, dim3(64 * kLowWaves), 0, st, a);
}

template <int TS>
static void launch_up(const AdapterArgs &a, bool y_bf16, hipStream_t st) {
    const dim3 grid((unsigned)(tiles_at_most(a.T, a.n, 16 * TS) + 1), (a.M + kUpWaves * kUpRows - 1) / (kUpWaves * kUpRows));
    if (y_bf16) hipLaunchKernelGGL((adapter_up_kernel<TS, true>), grid, dim3(64 * kUpWaves), 0, st, a);
    else hipLaunchKernelGGL((adapter_up_kernel<TS, false>), grid, dim3(64 * kUpWaves), 0, st, a);
}

int launch_adapter(AdapterArgs &a, bool x_bf16, bool y_bf16, hipStream_t st) {
    a.splits = adapter_splits(a.n, a.T, a.K);
    const dim3 grid((unsigned)tiles_at_most(a.T, a.n, kLowTile), a.splits);
    if (a.r <= 16) launch_low<1>(a, x_bf16, grid, st);
    else if (a.r <= 32) launch_low<2>(a, x_bf16, grid, st);
    else if (a.r <= 64) launch_low<4>(a, x_bf16, grid, st);
    else if (a.r <= 128) launch_low<8>(a, x_bf16, grid, st);
    else launch_low<16>(a, x_bf16, grid, st);
    if (a.T > 16 * a.n) launch_up<4>(a, y_bf16, st);
    else launch_up<1>(a, y_bf16, st);
    return hipGetLastError() == hipSuccess ? 0 : -6;
}

}  // namespace kxw4
