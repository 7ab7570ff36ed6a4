// kxw4_adapter.hip — low-rank adapters of many requests beside a shared
// projection: out[t] = y[t] + scale_e B_e (A_e x[t]), e the adapter of token
// t, out[t] = y[t] for a token without one. No counterpart in the reference.
//
// The tokens come sorted by adapter (RouteArgs' plan with one choice per
// token), in tiles that belong to one adapter. `low` = A x comes first, K split
// over waves and work-groups, then the update: in one launch where both are
// short, else in two with `low` in scratch between them, and for many tokens in
// two that keep B in registers.
//
// Arithmetic. A and B are BF16, so a BF16 x makes exact products on the BF16
// MFMA, summed in FP32. An FP32 value is cut into three BF16 parts of eight
// mantissa bits each, which hold all 24 (split3), and each part takes an MFMA
// of its own: the products are exact again. `low` is held in FP32 and cut the
// same way. The sums run in a fixed order: within a
// wave's steps, then the waves of a work-group, then the work-groups' parts.
// A part that is zero makes a NaN of an infinity in A or B that the whole value
// does not, so a wave whose sums are not finite works them out again, the second
// and third parts times the finite elements alone (finite8). Looking for that
// costs 0-2 %, 0.2 us of the shortest launches.
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
// exact (what lies below 2^-133, the least BF16 value, is cut off). An infinity
// or NaN goes into the first part whole.
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

// An operand's BF16 elements, zeros for those that are not finite. (The empty
// statement keeps the compiler from working this out ahead of the branch it is
// needed in, and holding it.)
__device__ __forceinline__ v4u finite8(v4u w) {
    asm volatile("" : "+v"(w));
#pragma unroll
    for (int i = 0; i < 4; ++i)
        w[i] &= ((w[i] & 0x7F80u) == 0x7F80u ? 0u : 0xFFFFu) | ((w[i] & 0x7F800000u) == 0x7F800000u ? 0u : 0xFFFF0000u);
    return w;
}

// acc + w times the three parts of a value, as mfma_bf16 of each adds them, but
// w's infinities by the first part alone. (Nothing is moved across: the branches
// that come here are not to cost the others registers.)
template <class Part>
__device__ __forceinline__ void mfma_again(v4u w, Part part, bool w_first, v4f &acc) {
    __builtin_amdgcn_sched_barrier(0);
    const v4u f = finite8(w);
#pragma unroll
    for (int q = 2; q >= 0; --q) {
        const v4u o = q > 0 ? f : w;
        acc = w_first ? mfma_bf16(o, part(q), acc) : mfma_bf16(part(q), o, acc);
    }
    __builtin_amdgcn_sched_barrier(0);
}

// Whether an infinity or NaN of the weights may have reached a wave's sums: it
// reaches those of every token. ROWS: registers of an MFMA's result that differ
// in the weights' row (1: they differ in the token alone).
template <int ROWS, int N>
__device__ __forceinline__ bool any_far(const v4f (&acc)[N]) {
    float s = 0.0f;
#pragma unroll
    for (int c = 0; c < N; ++c) {
        if constexpr (ROWS == 1) s += acc[c][0];
        else s += (acc[c][0] + acc[c][1]) + (acc[c][2] + acc[c][3]);
    }
    return __ballot(!(__builtin_fabsf(s) <= 3.40282347e38f)) != 0;
}

__device__ __forceinline__ void load8(const float *p, float (&v)[8]) {
    const v4f lo = reinterpret_cast<const v4f *>(p)[0], hi = reinterpret_cast<const v4f *>(p)[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[i] = lo[i];
        v[4 + i] = hi[i];
    }
}

// An operand's 16 rows x 64 bytes are loaded with four lanes to a row, so that
// sixteen lanes touch four rows, then go to the lanes that supply them: lane n
// + 16 g takes row n's piece g from lane 4 n + g. (With a lane for each row
// sixteen touched sixteen, and the L1 looks each up: 7.7 against 2.0 million
// lookups for 3,965 tokens, r = 32, and 24 against 20 us; 61 tokens of 24
// adapters, r = 64, K = 17408 25.9 / 24.9, r = 128 238 / 226 in all.)
__device__ __forceinline__ uint32_t to_operand(uint32_t v, int lane) {
    return (uint32_t)__builtin_amdgcn_ds_bpermute((4 * (lane & 15) + (lane >> 4)) * 4, (int)v);
}
__device__ __forceinline__ v4u to_operand(v4u v, int lane) {
    return v4u{to_operand(v.x, lane), to_operand(v.y, lane), to_operand(v.z, lane), to_operand(v.w, lane)};
}

constexpr int kLowTile = 16, kFewWaves = 4;
// 32-column chunks that r comes to, and BF16 elements of one chunk's three
// parts of a tile in the order of the MFMA's operand: [part][lane][8]
__host__ __device__ constexpr int chunks_of(int r) { return (r + 31) / 32; }
constexpr int kCutChunk = 3 * 64 * 8;

// acc[t][c] = the 32-K steps [k0, k1) of A_e's columns 16 c .. + 15 times the x
// of token tile t. Each lane loads 16-byte pieces of the row of `token[t]` (place
// lane / 4 of the tile) and of A's rows; an x piece is used by every column tile,
// an A piece by every token tile. AGAIN: where any_far says so, for an FP32 x.
template <int CT, bool XB, int TT, bool AGAIN>
__device__ __forceinline__ void low_steps_of(const AdapterArgs &a, int e, const int (&token)[TT], int k0, int k1, int lane, v4f (&acc)[TT][CT]) {
    const int lr = lane >> 2, lk = 8 * (lane & 3);           // row and columns that this lane loads
    size_t xrow[TT];
    const uint16_t *arow[CT];
#pragma unroll
    for (int t = 0; t < TT; ++t) xrow[t] = (size_t)token[t] * a.K + lk;
#pragma unroll
    for (int c = 0; c < CT; ++c)
        arow[c] = a.a + ((size_t)e * a.r + min(c * 16 + lr, a.r - 1)) * a.K + lk;
#pragma unroll
    for (int t = 0; t < TT; ++t)
#pragma unroll
        for (int c = 0; c < CT; ++c) acc[t][c] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    // U steps' loads are requested before the first of them is used
    auto run = [&](int k, auto uc) {
        constexpr int U = decltype(uc)::value;
        v4u w[U][CT];
        if constexpr (XB) {
            v4u x[U][TT];
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
                for (int t = 0; t < TT; ++t)
                    x[u][t] = *reinterpret_cast<const v4u *>(static_cast<const uint16_t *>(a.x) + xrow[t] + 32 * (k + u));
#pragma unroll
                for (int c = 0; c < CT; ++c) w[u][c] = *reinterpret_cast<const v4u *>(arow[c] + 32 * (k + u));
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
                for (int t = 0; t < TT; ++t) x[u][t] = to_operand(x[u][t], lane);
#pragma unroll
                for (int c = 0; c < CT; ++c) {
                    const v4u b = to_operand(w[u][c], lane);
#pragma unroll
                    for (int t = 0; t < TT; ++t) acc[t][c] = mfma_bf16(x[u][t], b, acc[t][c]);
                }
            }
        } else {
            float v[U][TT][8];
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
                for (int t = 0; t < TT; ++t) load8(static_cast<const float *>(a.x) + xrow[t] + 32 * (k + u), v[u][t]);
#pragma unroll
                for (int c = 0; c < CT; ++c) w[u][c] = *reinterpret_cast<const v4u *>(arow[c] + 32 * (k + u));
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                v4u x[TT][3];
#pragma unroll
                for (int t = 0; t < TT; ++t) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[u][t][i] = __uint_as_float(to_operand(__float_as_uint(v[u][t][i]), lane));
                    split8(v[u][t], x[t]);
                }
#pragma unroll
                for (int c = 0; c < CT; ++c) {
                    const v4u b = to_operand(w[u][c], lane);
#pragma unroll
                    for (int t = 0; t < TT; ++t) {
                        if constexpr (AGAIN) {
                            mfma_again(b, [&](int q) { return x[t][q]; }, false, acc[t][c]);
                        } else {
#pragma unroll
                            for (int q = 2; q >= 0; --q) acc[t][c] = mfma_bf16(x[t][q], b, acc[t][c]);
                        }
                    }
                }
            }
        }
    };
    constexpr int kSteps = AGAIN ? 1 : CT * TT <= 2 ? 4 : CT <= 4 ? 2 : 1;
    int k = k0;
    for (; k + kSteps <= k1; k += kSteps) run(k, std::integral_constant<int, kSteps>{});
    if constexpr (kSteps > 2) {
        if (k + 2 <= k1) {
            run(k, std::integral_constant<int, 2>{});
            k += 2;
        }
    }
#pragma unroll 1
    for (; k < k1; ++k) run(k, std::integral_constant<int, 1>{});
}

template <int CT, bool XB, int TT>
__device__ __forceinline__ void low_steps(const AdapterArgs &a, int e, const int (&token)[TT], int k0, int k1, int lane, v4f (&acc)[TT][CT]) {
    low_steps_of<CT, XB, TT, false>(a, e, token, k0, k1, lane, acc);
    if constexpr (!XB) {
#pragma unroll
        for (int t = 0; t < TT; ++t) {
            if (!any_far<1>(acc[t])) continue;
            const int one[1] = {token[t]};
            v4f sum[1][CT];
            low_steps_of<CT, XB, 1, true>(a, e, one, k0, k1, lane, sum);
#pragma unroll
            for (int c = 0; c < CT; ++c) acc[t][c] = sum[0][c];
        }
    }
}

// low[s][p][c] = sum over the s-th part of K of A[c][k] x[order[p]][k]: a
// work-group takes 16 TT places of one adapter and part s, its WAVES waves
// consecutive runs of 32-K steps, all r columns (CT tiles of 16). CUT: one part;
// scale * low is cut into its three BF16 parts here, in the order the second
// launch's operand takes them. The places [p, p + 16) of adapter e are cut tile p
// / 16 + e, a number of its own for each tile.
template <int CT, int WAVES, bool XB, bool CUT, int TT>
__global__ __launch_bounds__(64 * WAVES) void adapter_low_kernel(const AdapterArgs a) {
    __shared__ float part[WAVES - 1][CT][256];
    const int tid = threadIdx.x, lane = tid & 63, m = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const GroupTiles tiles = scan_tiles(a.offsets, a.n, kLowTile * TT, lane);
    const int u = a.tile0 + blockIdx.x;
    if (u >= tiles.total) return;
    const GroupTile tile = tile_at(tiles, a.offsets, kLowTile * TT, u);
    const int p0 = tile.begin + tile.index * kLowTile * TT;
    const int steps = a.K / 32, ways = a.splits * WAVES, way = blockIdx.y * WAVES + wave;
    const int k0 = (int)((long long)steps * way / ways), k1 = (int)((long long)steps * (way + 1) / ways);

    v4f acc[TT][CT];
    int token[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) token[t] = a.order[min(p0 + kLowTile * t + (lane >> 2), tile.end - 1)];
    low_steps<CT, XB, TT>(a, tile.e, token, k0, k1, lane, acc);
#pragma unroll
    for (int t = 0; t < TT; ++t) {
        const int pt = p0 + kLowTile * t;
        if (pt >= tile.end) return;
        if (t > 0) __syncthreads();
        if (wave > 0) {
#pragma unroll
            for (int c = 0; c < CT; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) part[wave - 1][c][i * 64 + lane] = acc[t][c][i];
        }
        __syncthreads();
        if constexpr (CUT) {
            // every thread adds up and cuts elements of the tile: lane l of
            // chunk h holds token l%16 and columns 32 h + 8 (l/16) .. + 7
            const float scale = a.scale[tile.e];
            if (wave == 0) {
#pragma unroll
                for (int c = 0; c < CT; ++c)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float v = acc[t][c][i];
#pragma unroll
                        for (int w = 0; w < WAVES - 1; ++w) v += part[w][c][i * 64 + lane];
                        part[0][c][i * 64 + lane] = c * 16 + m < a.r ? v * scale : 0.0f;
                    }
            }
            __syncthreads();
            uint16_t *to = reinterpret_cast<uint16_t *>(a.low) + (size_t)(pt / kLowTile + tile.e) * chunks_of(a.r) * kCutChunk;
            for (int h = wave; h < chunks_of(a.r); h += WAVES) {
                float v[8];
                v4u op[3];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    // column 32 h + 8 g + j of token m: tile c, register i = m % 4 of lane group m / 4
                    const int column = 32 * h + 8 * g + j;
                    v[j] = column < 16 * CT ? part[0][min(column >> 4, CT - 1)][(m & 3) * 64 + 16 * (m >> 2) + (column & 15)] : 0.0f;
                }
                split8(v, op);
#pragma unroll
                for (int q = 0; q < 3; ++q) *reinterpret_cast<v4u *>(to + (h * 3 + q) * 512 + lane * 8) = op[q];
            }
        } else if (wave == 0) {
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                const int col = c * 16 + m;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float v = acc[t][c][i];
#pragma unroll
                    for (int w = 0; w < WAVES - 1; ++w) v += part[w][c][i * 64 + lane];
                    const int p = pt + 4 * g + i;
                    if (p < tile.end && col < a.r) a.low[((size_t)blockIdx.y * a.T + p) * a.r + col] = v;
                }
            }
        }
    }
}

// out = y + scale B low for few tokens: a work-group takes 16 places of one
// adapter x 256 rows of B, 64 a wave. It adds up the parts of `low`, cuts scale
// * low into three BF16 parts in LDS, and each wave multiplies them by its
// rows. B is the MFMA's first operand, its rows dealt so that a lane ends up
// with 16-byte runs of one token's outputs. A chain of round trips (offsets,
// order, y and low) bounds it: all that a step needs is requested together.
constexpr int kUpWaves = 4, kUpRows = 64, kUpBlock = kUpWaves * kUpRows;
// BF16 elements of a token's row of one part: r padded to whole MFMAs, with 16
// bytes more so that neighbouring rows start in different banks
__host__ __device__ constexpr int up_pitch(int r) { return 32 * chunks_of(r) + 8; }

// out = y + acc for a lane's pieces of one token, rounded once; piece q's
// outputs are acc[2 q], acc[2 q + 1] (BF16) or acc[q]. Without `add` out = y, bit
// for bit (-0 + 0 is another zero).
template <int NY, bool YB, class Col>
__device__ __forceinline__ void store_up(const AdapterArgs &a, size_t at, Col col, const v4u (&yv)[NY], const v4f (&acc)[4], bool add) {
#pragma unroll
    for (int q = 0; q < NY; ++q) {
        if (col(q) >= a.M) continue;
        v4u o;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (YB) {
                const v4f f = acc[2 * q + (i >> 1)];
                o[i] = pack_bf16(__uint_as_float(yv[q][i] << 16) + f[2 * (i & 1)],
                                 __uint_as_float(yv[q][i] & 0xFFFF0000u) + f[2 * (i & 1) + 1]);
            } else {
                o[i] = __float_as_uint(__uint_as_float(yv[q][i]) + acc[q][i]);
            }
        }
        if (!add) o = yv[q];
        *reinterpret_cast<v4u *>(static_cast<uint8_t *>(a.out) + (at + col(q)) * (YB ? 2 : 4)) = o;
    }
}

// KC: 32-column chunks of B requested together; from two on a row of B is long
// enough for the loads of to_operand (us in all for KC = 1 / 2, 1,500 tokens of 8,
// all in use, K = 5120, M = 8192, r = 128 70.0 / 63.0, r = 64 39.8 / 36.0; r = 32
// 26.8 / 26.7, 250 tokens 9.7 / 10.1).
template <int KC, bool YB>
__global__ __launch_bounds__(64 * kUpWaves) void adapter_up_kernel(const AdapterArgs a) {
    constexpr int NY = YB ? 2 : 4;                           // 16-byte pieces of a lane's 16 outputs
    constexpr bool SPREAD = KC > 1;
    extern __shared__ __attribute__((aligned(16))) uint16_t cut[];       // [3][16][pitch]
    const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int mblocks = (a.M + kUpBlock - 1) / kUpBlock;
    const int v = blockIdx.x / mblocks, u = a.tile0 + v, m0 = (blockIdx.x - v * mblocks) * kUpBlock + wave * kUpRows;
    const GroupTiles tiles = scan_tiles(a.offsets, a.n, kLowTile, lane);
    int p0, p1, e = -1;
    if (u < tiles.total) {
        const GroupTile tile = tile_at(tiles, a.offsets, kLowTile, u);
        e = tile.e;
        p0 = tile.begin + tile.index * kLowTile;
        p1 = tile.end;
    } else {
        // the tokens without an adapter keep y (already there when out is y)
        p0 = a.offsets[a.n] + (u - tiles.total) * kLowTile;
        p1 = a.T;
        if (a.out == a.y || p0 >= p1) return;
    }
    const bool on = m0 < a.M;                                // (the others only help with `low`)
    const size_t at = (size_t)a.order[min(p0 + n, p1 - 1)] * a.M;
    // column of a lane's piece q, and the row of B that MFMA c has as its row i
    auto col = [&](int q) { return m0 + (YB ? 32 * q + 8 * g : 16 * q + 4 * g); };
    auto row = [&](int c, int i) { return m0 + (YB ? 32 * (c >> 1) + 8 * (i >> 2) + 4 * (c & 1) + (i & 3) : 16 * c + i); };
    v4u yv[NY];
#pragma unroll
    for (int q = 0; q < NY; ++q)
        yv[q] = *reinterpret_cast<const v4u *>(static_cast<const uint8_t *>(a.y) + (at + min(col(q), a.M - (YB ? 8 : 4))) * (YB ? 2 : 4));
    v4f acc[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) acc[c] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    if (e >= 0) {
        const int pitch = up_pitch(a.r), quads = (pitch - 8) / 4;
        const float scale = a.scale[e];
        const size_t part = (size_t)a.T * a.r;
        for (int i = tid; i < kLowTile * quads; i += 64 * kUpWaves) {
            const int t = i / quads, c = (i - t * quads) * 4;
            v4f v = {0.0f, 0.0f, 0.0f, 0.0f};
            if (c < a.r) {
                const float *low = a.low + (size_t)min(p0 + t, p1 - 1) * a.r + c;
                for (int q = 0; q < a.splits; q += 8) {
                    v4f o[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) o[j] = *reinterpret_cast<const v4f *>(low + (size_t)min(q + j, a.splits - 1) * part);
#pragma unroll
                    for (int j = 0; j < 8; ++j)
#pragma unroll
                        for (int x = 0; x < 4; ++x) v[x] = q + j < a.splits ? v[x] + o[j][x] : v[x];
                }
            }
            uint32_t w[4][3];
#pragma unroll
            for (int x = 0; x < 4; ++x) split3(v[x] * scale, w[x]);
#pragma unroll
            for (int q = 0; q < 3; ++q)
                *reinterpret_cast<v2u *>(cut + (q * kLowTile + t) * pitch + c) = v2u{w[0][q] >> 16 | w[1][q], w[2][q] >> 16 | w[3][q]};
        }
        __syncthreads();
        if (!on) return;
        // (MFMA c's rows of B, columns from k0 on)
        auto load_b = [&](int k0, int c) {
            const int k = k0 + 8 * (SPREAD ? lane & 3 : g);
            v4u w = *reinterpret_cast<const v4u *>(a.b + ((size_t)e * a.M + min(row(c, SPREAD ? lane >> 2 : n), a.M - 1)) * a.r + min(k, a.r - 8));
#pragma unroll
            for (int x = 0; x < 4; ++x) w[x] = k < a.r ? w[x] : 0u;
            return w;
        };
        for (int k0 = 0; k0 < a.r; k0 += 32 * KC) {
            v4u b[KC][4];
#pragma unroll
            for (int h = 0; h < KC; ++h)
#pragma unroll
                for (int c = 0; c < 4; ++c) b[h][c] = load_b(k0 + 32 * h, c);
#pragma unroll
            for (int h = 0; h < KC; ++h) {
                if (k0 + 32 * h >= a.r) break;
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if constexpr (SPREAD) b[h][c] = to_operand(b[h][c], lane);
#pragma unroll
                for (int q = 2; q >= 0; --q) {
                    const v4u x = *reinterpret_cast<const v4u *>(cut + (q * kLowTile + n) * pitch + k0 + 32 * h + 8 * g);
#pragma unroll
                    for (int c = 0; c < 4; ++c) acc[c] = mfma_bf16(b[h][c], x, acc[c]);
                }
            }
        }
        if (any_far<4>(acc)) {
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[c] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
            for (int k0 = 0; k0 < a.r; k0 += 32) {
                auto part = [&](int q) { return *reinterpret_cast<const v4u *>(cut + (q * kLowTile + n) * pitch + k0 + 8 * g); };
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const v4u b = load_b(k0, c);
                    mfma_again(SPREAD ? to_operand(b, lane) : b, part, true, acc[c]);
                }
            }
        }
    }
    if (!on || p0 + n >= p1) return;
    store_up<NY, YB>(a, at, [&](int q) { return col(q); }, yv, acc, e >= 0);
}

// Both in one launch, for few tokens and small adapters: a work-group takes 16
// places of one adapter x 1,024 rows of B, 64 a wave, and works out the whole
// `low` of its places first, its sixteen waves K split between them. The A rows
// are read again by every work-group of a tile, from the L2 (one_launch says what
// that costs and saves).
constexpr int kOneWaves = 16, kOneBlock = kOneWaves * kUpRows;
template <int CT, bool XB, bool YB>
__global__ __launch_bounds__(64 * kOneWaves) void adapter_one_kernel(const AdapterArgs a) {
    constexpr int NY = YB ? 2 : 4, PITCH = up_pitch(16 * CT);
    __shared__ float part[kOneWaves][CT][256];
    __shared__ __attribute__((aligned(16))) uint16_t cut[3 * kLowTile * PITCH];
    const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int mblocks = (a.M + kOneBlock - 1) / kOneBlock;
    const int u = blockIdx.x / mblocks, m0 = (blockIdx.x - u * mblocks) * kOneBlock + wave * kUpRows;
    const GroupTiles tiles = scan_tiles(a.offsets, a.n, kLowTile, lane);
    int p0, p1, e = -1;
    if (u < tiles.total) {
        const GroupTile tile = tile_at(tiles, a.offsets, kLowTile, u);
        e = tile.e;
        p0 = tile.begin + tile.index * kLowTile;
        p1 = tile.end;
    } else {
        // the tokens without an adapter keep y (already there when out is y)
        p0 = a.offsets[a.n] + (u - tiles.total) * kLowTile;
        p1 = a.T;
        if (a.out == a.y || p0 >= p1) return;
    }
    const bool on = m0 < a.M;                                // (the others only help with `low`)
    const int row[1] = {a.order[min(p0 + (lane >> 2), p1 - 1)]};
    const size_t at = (size_t)a.order[min(p0 + n, p1 - 1)] * a.M;
    // (columns and rows as in adapter_up_kernel)
    auto col = [&](int q) { return m0 + (YB ? 32 * q + 8 * g : 16 * q + 4 * g); };
    auto brow = [&](int c) { return m0 + (YB ? 32 * (c >> 1) + 8 * (n >> 2) + 4 * (c & 1) + (n & 3) : 16 * c + n); };
    v4u yv[NY], b[4];
#pragma unroll
    for (int q = 0; q < NY; ++q)
        yv[q] = *reinterpret_cast<const v4u *>(static_cast<const uint8_t *>(a.y) + (at + min(col(q), a.M - (YB ? 8 : 4))) * (YB ? 2 : 4));
    v4f acc[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) acc[c] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    if (e >= 0) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
            b[c] = *reinterpret_cast<const v4u *>(a.b + ((size_t)e * a.M + min(brow(c), a.M - 1)) * a.r + min(8 * g, a.r - 8));
        const int steps = a.K / 32;
        v4f low[1][CT];
        low_steps<CT, XB, 1>(a, e, row, steps * wave / kOneWaves, steps * (wave + 1) / kOneWaves, lane, low);
#pragma unroll
        for (int c = 0; c < CT; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) part[wave][c][i * 64 + lane] = low[0][c][i];
        __syncthreads();
        // element i of tile c: token 4 (i%64 / 16) + i / 64, column 16 c + i % 16
        if (tid < 512) {
            const int c = tid >> 8, i = tid & 255, t = 4 * ((i & 63) >> 4) + (i >> 6), column = 16 * c + (i & 15);
            float v = 0.0f;
            if (c < CT && column < a.r) {
#pragma unroll
                for (int w = 0; w < kOneWaves; ++w) v += part[w][min(c, CT - 1)][i];
                v *= a.scale[e];
            }
            uint32_t w[3];
            split3(v, w);
#pragma unroll
            for (int q = 0; q < 3; ++q) cut[(q * kLowTile + t) * PITCH + column] = (uint16_t)(w[q] >> 16);
        }
        __syncthreads();
        if (!on) return;
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int x = 0; x < 4; ++x) b[c][x] = 8 * g < a.r ? b[c][x] : 0u;
        v4u x[3];
#pragma unroll
        for (int q = 2; q >= 0; --q) {
            x[q] = *reinterpret_cast<const v4u *>(cut + (q * kLowTile + n) * PITCH + 8 * g);
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[c] = mfma_bf16(b[c], x[q], acc[c]);
        }
        if (any_far<4>(acc)) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                acc[c] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
                mfma_again(b[c], [&](int q) { return x[q]; }, true, acc[c]);
            }
        }
    }
    if (!on || p0 + n >= p1) return;
    store_up<NY, YB>(a, at, [&](int q) { return col(q); }, yv, acc, e >= 0);
}

// The same for many tokens. A wave takes 128 rows of B, whose operands stay in
// its registers, and walks up to a.run tiles of 16 places of one adapter. `low`
// is the MFMA's first operand (rows are tokens), in the order the first launch
// left it, so a load of it is one contiguous kilobyte; B's rows are dealt so
// that a lane ends up with 16-byte runs of outputs and sixteen lanes with 256
// consecutive bytes of one token (the other way round sixteen lanes touched
// sixteen rows, 42 lookups of the L1 an access against 16). The next tile's y
// and low are requested before this one's products. Bound by reading y and
// writing out: 3,965 tokens, M = 17408, BF16, r = 32 60 us for 276 MB (4.6 TB/s).
constexpr int kManyWaves = 4, kManyRows = 128, kManyBlock = kManyWaves * kManyRows;
template <int KC, bool YB>
__global__ __launch_bounds__(64 * kManyWaves) void adapter_many_kernel(const AdapterArgs a) {
    constexpr int NQ = YB ? 1 : 2, RUN = YB ? 8 : 4;         // 16-byte pieces of a lane and token, outputs of a piece
    const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int mblocks = (a.M + kManyBlock - 1) / kManyBlock;
    const int v = blockIdx.x / mblocks, u = a.tile0 + v, m0 = (blockIdx.x - v * mblocks) * kManyBlock + wave * kManyRows;
    // a run: a.run tiles of one adapter; `first`: the cut tile of its first
    const GroupTiles runs = scan_tiles(a.offsets, a.n, kLowTile * a.run, lane);
    int p0, p1, e = -1;
    size_t first = 0;
    if (u < runs.total) {
        const GroupTile run = tile_at(runs, a.offsets, kLowTile * a.run, u);
        e = run.e;
        p0 = run.begin + run.index * kLowTile * a.run;
        p1 = min(run.end, p0 + kLowTile * a.run);
        first = p0 / kLowTile + e;
    } else {
        // the tokens without an adapter keep y (already there when out is y)
        p0 = a.offsets[a.n] + (u - runs.total) * kLowTile * a.run;
        p1 = min(a.T, p0 + kLowTile * a.run);
        if (a.out == a.y || p0 >= p1) return;
    }
    if (m0 >= a.M) return;
    // column of output j of MFMA c = (piece, run element): a lane's own, and of
    // the row of B that it supplies
    auto col = [&](int q) { return m0 + 16 * RUN * q + RUN * n; };
    v4u b[KC][8];
    if (e >= 0) {
#pragma unroll
        for (int h = 0; h < KC; ++h)
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                const int k = 32 * h + 8 * g, row = min(col(c / RUN) + c % RUN, a.M - 1);
                const v4u w = *reinterpret_cast<const v4u *>(a.b + ((size_t)e * a.M + row) * a.r + min(k, a.r - 8));
#pragma unroll
                for (int x = 0; x < 4; ++x) b[h][c][x] = k < a.r ? w[x] : 0u;
            }
    }
    auto tokens = [&](int p, size_t (&at)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) at[i] = (size_t)a.order[min(p + 4 * g + i, p1 - 1)] * a.M;
    };
    auto load_y = [&](const size_t (&at)[4], v4u (&yv)[4][NQ]) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int q = 0; q < NQ; ++q)
                yv[i][q] = *reinterpret_cast<const v4u *>(static_cast<const uint8_t *>(a.y) + (at[i] + min(col(q), a.M - RUN)) * (YB ? 2 : 4));
    };
    const uint16_t *cut = reinterpret_cast<const uint16_t *>(a.low) + first * chunks_of(a.r) * kCutChunk + lane * 8;
    auto load_low = [&](int tile, v4u (&x)[KC][3]) {
#pragma unroll
        for (int h = 0; h < KC; ++h)
#pragma unroll
            for (int q = 0; q < 3; ++q)
                x[h][q] = *reinterpret_cast<const v4u *>(cut + ((size_t)tile * chunks_of(a.r) + min(h, chunks_of(a.r) - 1)) * kCutChunk + q * 512);
    };
    const int tiles = (p1 - p0 + kLowTile - 1) / kLowTile;
    size_t at[4], atnext[4];
    v4u yv[4][NQ], ynext[4][NQ], x[KC][3], xnext[KC][3];
    tokens(p0, atnext);
    load_y(atnext, ynext);
    if (e >= 0) load_low(0, xnext);
    for (int tile = 0; tile < tiles; ++tile) {
        const int p = p0 + kLowTile * tile;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            at[i] = atnext[i];
#pragma unroll
            for (int q = 0; q < NQ; ++q) yv[i][q] = ynext[i][q];
        }
        v4f acc[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) acc[c] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        const bool more = tile + 1 < tiles;
        if (e >= 0) {
#pragma unroll
            for (int h = 0; h < KC; ++h)
#pragma unroll
                for (int q = 0; q < 3; ++q) x[h][q] = xnext[h][q];
        }
        if (more) {
            tokens(p + kLowTile, atnext);
            if (e >= 0) load_low(tile + 1, xnext);
            load_y(atnext, ynext);
        }
        if (e >= 0) {
#pragma unroll
            for (int h = 0; h < KC; ++h)
#pragma unroll
                for (int q = 2; q >= 0; --q)
#pragma unroll
                    for (int c = 0; c < 8; ++c) acc[c] = mfma_bf16(x[h][q], b[h][c], acc[c]);
            if (any_far<1>(acc)) {
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    acc[c] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int h = 0; h < KC; ++h) mfma_again(b[h][c], [&](int q) { return x[h][q]; }, false, acc[c]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (p + 4 * g + i >= p1) continue;
#pragma unroll
            for (int q = 0; q < NQ; ++q) {
                if (col(q) >= a.M) continue;
                v4u o;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if constexpr (YB)
                        o[j] = pack_bf16(__uint_as_float(yv[i][q][j] << 16) + acc[2 * j][i],
                                         __uint_as_float(yv[i][q][j] & 0xFFFF0000u) + acc[2 * j + 1][i]);
                    else
                        o[j] = __float_as_uint(__uint_as_float(yv[i][q][j]) + acc[4 * q + j][i]);
                }
                if (e < 0) o = yv[i][q];
                *reinterpret_cast<v4u *>(static_cast<uint8_t *>(a.out) + (at[i] + col(q)) * (YB ? 2 : 4)) = o;
            }
        }
    }
}

// Many tokens, while B's rows fit the registers: from 20 million outputs on, where
// what the first launch loses (no split of K) is less than what the second gains.
// Swept over 144 shapes of 1,100-6,000 tokens, 2-24 adapters, r 16-128, K 512-
// 12,288, M 1,024-17,408: 0.5 % behind the better of the two on average (us few /
// many: 3,965 tokens of 6, K = 5120, M = 17408, r = 32 101 / 74, r = 128 196 / 144;
// M = 4096, r = 32 32.3 / 32.2; 1,536 of 8, K = 512, M = 16384, r = 64 40.0 / 36.5;
// K = 12288, M = 1024 26.3 / 35.0; 2,048 of 8, K = 5120, M = 4096 29.6 / 34.7).
static bool many_tokens(int n, int T, int r, int M) { return (long long)T * M >= 20000000 && T >= 1024 && T >= 64ll * n && r <= 128; }

// Work-groups per 16-token tile of the first launch for few tokens: enough to
// give each CU four while a wave keeps at least four 32-K steps, and as many
// as the second launch adds up in one round (us for 4 / 8 / 16: 8 tokens of 8,
// K = 5120 8.3 / 7.7 / 8.2; 61 of 24, K = 17408, r = 64 30.0 / 21.7 / 22.3).
static int adapter_splits(int n, int T, int K) {
    const long long tiles = std::max(1ll, tiles_at_most(T, n, kLowTile));
    const long long most = std::max(1, K / (32 * kFewWaves * 4));
    return (int)std::max(1ll, std::min({most, 1024 / tiles, 8ll}));
}

// One launch, while a work-group's waves have at most ten 32-K steps of one
// column tile each and every CU at most one work-group: the host's second launch
// costs more than what the GPU loses. Both sides, us two launches / one, 8 tokens
// of 8, r = 16, M = 5120 (1 token, 32 of 16, and M = 1024 within 0.8 of these):
//   K                       1,024      2,560      4,096      5,120      6,144      8,192
//   BF16 called in turn   13.2/9.3   13.2/9.2   13.1/9.3   13.2/9.1   13.0/9.2   13.1/9.7
//   BF16 from a graph      6.9/5.0    6.8/6.0    6.8/7.0    7.0/7.7    7.0/8.4    7.2/9.6
//   FP32 called in turn   13.2/9.3   13.2/9.1   13.2/10.6  13.2/11.9  13.2/13.5  13.2/16.2
//   FP32 from a graph      7.8/6.1    7.8/8.4    7.8/10.6   8.2/12.0   8.5/13.6   9.2/16.3
// So the line is where FP32 calls stop gaining; a graph's replays would have it at
// 2,000 to 4,000. At r = 32 half the K: BF16 2,560 13.2/9.2 and 7.2/7.1, 4,096
// 13.2/9.2 and 7.2/8.8, FP32 2,560 13.2/10.1 and 8.5/10.1. 200 tokens of 100, r =
// 32 21.4/39.1 in turn.
static bool one_launch(int n, int T, int r, int K, int M) {
    const long long groups = (tiles_at_most(T, n, kLowTile) + 1) * ((M + kOneBlock - 1) / kOneBlock);
    return (long long)(r + 15) / 16 * K <= 5120 && r <= 32 && groups <= device_cus();
}

size_t adapter_scratch(int n, int T, int r, int K, int M) {
    if (many_tokens(n, T, r, M)) return (size_t)tiles_at_most(T, n, kLowTile) * chunks_of(r) * kCutChunk * 2;
    return one_launch(n, T, r, K, M) ? 0 : (size_t)adapter_splits(n, T, K) * T * r * sizeof(float);
}

// One launch for as many tiles as its grid holds (grid_limit), each of `blocks`
// work-groups. (134 million tokens of one adapter at 1,024 threads a tile of 32.)
typedef void (*AdapterKernel)(const AdapterArgs);
static int launch_tiles(AdapterKernel k, AdapterArgs &a, long long tiles, int blocks, int parts, int threads, size_t lds, hipStream_t st) {
    const long long most = grid_limit(threads) / blocks;
    for (long long t0 = 0; t0 < tiles; t0 += most) {
        a.tile0 = (int)t0;
        hipLaunchKernelGGL(k, dim3((unsigned)(std::min(most, tiles - t0) * blocks), parts), dim3(threads), lds, st, a);
        if (hipGetLastError() != hipSuccess) return -6;
    }
    return 0;
}

template <int CT>
static int launch_one(const AdapterArgs &a, bool x_bf16, bool y_bf16, hipStream_t st) {
    const long long grid = (tiles_at_most(a.T, a.n, kLowTile) + 1) * ((a.M + kOneBlock - 1) / kOneBlock);      // (at most the CUs: one_launch)
    auto k = x_bf16 ? (y_bf16 ? adapter_one_kernel<CT, true, true> : adapter_one_kernel<CT, true, false>)
                    : (y_bf16 ? adapter_one_kernel<CT, false, true> : adapter_one_kernel<CT, false, false>);
    hipLaunchKernelGGL(k, dim3((unsigned)grid), dim3(64 * kOneWaves), 0, st, a);
    return hipGetLastError() == hipSuccess ? 0 : -6;
}

// (WF: waves for an FP32 x)
template <int CT, int WAVES, bool CUT, int TT, int WF = WAVES>
static int launch_low(AdapterArgs &a, bool x_bf16, hipStream_t st) {
    return launch_tiles(x_bf16 ? adapter_low_kernel<CT, WAVES, true, CUT, TT> : adapter_low_kernel<CT, WF, false, CUT, TT>, a,
                        tiles_at_most(a.T, a.n, kLowTile * TT), 1, a.splits, 64 * (x_bf16 ? WAVES : WF), 0, st);
}

// The first launch for many tokens. One work-group of either takes about as long
// as it has bytes to fetch through its CU's L1 (24 a clock): x of its tokens and
// all of A, so two tiles, which share A, pay once there are more tiles than CUs
// (us in all for one / two, all adapters in use: 8,000 tokens of 12, K = 5120, M =
// 4096, r = 32 51.8 / 47.9, but r = 128 121 / 128; 21,000 of 12, K = 12288, M =
// 1024, r = 64 261 / 205; 3,965 of 6, K = 5120, M = 17408, r = 32 77 / 83). Two tiles of FP32 x at r = 32 take eight waves, whose
// registers hold more loads (sixteen / eight: 9,000 tokens of 40, K = 5120, M =
// 2560 112 / 105, 6,000 of 12, K = 2048, M = 4096 54.2 / 50.5, 12,000 of 6, K = M =
// 5120 132 / 125).
template <int TT>
static int launch_cut(AdapterArgs &a, bool x_bf16, hipStream_t st) {
    if (a.r <= 16) return launch_low<1, 16, true, TT>(a, x_bf16, st);
    if (a.r <= 32) return launch_low<2, 16, true, TT, TT == 2 ? 8 : 16>(a, x_bf16, st);
    if (a.r <= 64) return launch_low<4, 8, true, TT>(a, x_bf16, st);
    return launch_low<8, 8, true, TT>(a, x_bf16, st);
}

template <int KC>
static int launch_up(AdapterArgs &a, bool y_bf16, hipStream_t st) {
    const size_t lds = (size_t)3 * kLowTile * up_pitch(a.r) * 2;          // (at most 25.3 KB: r = 256)
    return launch_tiles(y_bf16 ? adapter_up_kernel<KC, true> : adapter_up_kernel<KC, false>, a,
                        tiles_at_most(a.T, a.n, kLowTile) + 1, (a.M + kUpBlock - 1) / kUpBlock, 1, 64 * kUpWaves, lds, st);
}

// Tiles per run: up to twelve, so that B is read seldom, while six (three,
// where its rows take most of the registers) work-groups a CU are left (r =
// 32: runs of 4 / 6 / 12 78.5 / 77.9 / 82.1 us; r = 128 169 / 153 / 144).
template <int KC>
static int launch_many(AdapterArgs &a, bool y_bf16, hipStream_t st) {
    const int mblocks = (a.M + kManyBlock - 1) / kManyBlock;
    const long long work = tiles_at_most(a.T, a.n, kLowTile) * mblocks, groups = (KC <= 2 ? 6ll : 3ll) * device_cus();
    a.run = (int)std::max(1ll, std::min(12ll, (work + groups / 2) / groups));
    return launch_tiles(y_bf16 ? adapter_many_kernel<KC, true> : adapter_many_kernel<KC, false>, a,
                        tiles_at_most(a.T, a.n, kLowTile * a.run) + 1, mblocks, 1, 64 * kManyWaves, 0, st);
}

int launch_adapter(AdapterArgs &a, bool x_bf16, bool y_bf16, hipStream_t st) {
    if (many_tokens(a.n, a.T, a.r, a.M)) {
        a.splits = 1;
        const int rc = tiles_at_most(a.T, a.n, kLowTile) <= device_cus() ? launch_cut<1>(a, x_bf16, st) : launch_cut<2>(a, x_bf16, st);
        if (rc) return rc;
        return a.r <= 32 ? launch_many<1>(a, y_bf16, st) : a.r <= 64 ? launch_many<2>(a, y_bf16, st) : launch_many<4>(a, y_bf16, st);
    }
    if (one_launch(a.n, a.T, a.r, a.K, a.M)) return a.r <= 16 ? launch_one<1>(a, x_bf16, y_bf16, st) : launch_one<2>(a, x_bf16, y_bf16, st);
    a.splits = adapter_splits(a.n, a.T, a.K);
    // Two token tiles share A where many tiles read a long one (us in all for
    // one / two, all adapters in use: 2,520 tokens of 24, M = 1024, K = 12288, r =
    // 128 171 / 96, r = 64 67.1 / 47.5; 1,536 of 8, r = 128 83.0 / 62.0, M = 4096, K
    // = 5120 52.6 / 48.4; K = 2048 32.2 / 33.4; 1,100 of 2, K = 5120 33.3 / 34.6;
    // r = 16 alike. Below 1,536 tokens M decides too: 1,500 of 8, K = 5120, M =
    // 8192, r = 128 63.0 / 56.0).
    const bool two = a.T >= 1536 && a.K >= 4096;
    int rc;
    if (a.r <= 16) rc = launch_low<1, kFewWaves, false, 1>(a, x_bf16, st);
    else if (a.r <= 32) rc = two ? launch_low<2, kFewWaves, false, 2>(a, x_bf16, st) : launch_low<2, kFewWaves, false, 1>(a, x_bf16, st);
    else if (a.r <= 64) rc = two ? launch_low<4, kFewWaves, false, 2>(a, x_bf16, st) : launch_low<4, kFewWaves, false, 1>(a, x_bf16, st);
    else if (a.r <= 128) rc = two ? launch_low<8, kFewWaves, false, 2>(a, x_bf16, st) : launch_low<8, kFewWaves, false, 1>(a, x_bf16, st);
    else rc = launch_low<16, kFewWaves, false, 1>(a, x_bf16, st);
    if (rc) return rc;
    return a.r <= 32 ? launch_up<1>(a, y_bf16, st) : launch_up<2>(a, y_bf16, st);
}

}  // namespace kxw4
