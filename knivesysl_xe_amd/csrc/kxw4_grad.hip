// kxw4_grad.hip — the gradient of a projection's weight, for one weight or by
// group: dw_g[m][k] = sum over the rows p of group g of dy[p][m] * x[p][k]. No
// counterpart in the reference, which trains nothing.
//
// BF16 rows, exact products, FP32 sums (the 32x32x16 BF16 MFMA). The sum runs
// over rows, which lie apart in memory, so both operands are read transposed: a
// step's rows reach LDS as they lie, by buffer loads straight into a ring of
// NST stages, and ds_read_b64_tr_b16 gives a lane four rows of its column. A
// work-group takes tiles of 32 AM WM x 32 AK WK outputs of one group in turn, its
// ring running on from one to the next; the rows past a group's end read as zero
// through the buffer's range. Where there are few tiles the rows are split over
// work-groups and their FP32 parts added in order by a second launch.
//
// Bounds and measurements (256 CUs; a large BF16 library product reaches 1,176 to
// 1,265 TF): the matrix units, at the clock that the power limit leaves them, for
// many rows of a group (4,096 rows, 5,120 x 5,120, FP32 out: 218 to 224 us, 957 TF
// and more; 2,048 rows, 17,408 x 5,120, BF16 out: 320 to 345 us, 1,058 TF and more);
// the last round of tiles where these are few (2,048 rows, 5,120 x 5,120, FP32 out:
// 400 tiles on 256 CUs, 122 to 143 us, 749 TF and more; with `add` 147 for 122); the
// stores where a group has few rows (64 groups of 256 rows, 1,024 x 2,048, BF16 out:
// 134 us, 512 TF). A first version with a tile per work-group and 32-byte stores took
// 177 us for the 2,048 rows and 290 for 8 groups of 1,000 rows, 2,048 x 4,096 (now
// 168: 800 TF).
#include "kxw4_device.hpp"
#include "kxw4_internal.hpp"

#include <algorithm>
#include <type_traits>
#include <utility>

namespace kxw4 {

typedef float v16f __attribute__((ext_vector_type(16)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef short v8s __attribute__((ext_vector_type(8)));

#define KXW4_GRAD_LDS(p) ((__attribute__((address_space(3))) void *)(p))

constexpr int kGradRows = 32;                                // rows of a step
constexpr int kGradRaster = 4;                               // m-tiles side by side

// The transposing LDS read. (Through a restricted pointer, whose scope the read
// keeps when inlined: without alias information the compiler assumes that it
// depends on the loads into LDS still in flight and waits for all of them.)
typedef __attribute__((address_space(3))) v4s lds_v4s;
__device__ __forceinline__ v4s read_tr16(lds_v4s *__restrict__ p) { return __builtin_amdgcn_ds_read_tr16_b64_v4i16(p); }

template <int AM, int AK, int WM, int WK>
struct GradShape {
    static constexpr int NW = WM * WK, NTH = 64 * NW;
    static constexpr int BM = 32 * AM * WM, BK = 32 * AK * WK;
    static constexpr int M_BYTES = kGradRows * BM * 2, K_BYTES = kGradRows * BK * 2, STAGE = M_BYTES + K_BYTES;
    static constexpr int M_LOADS = M_BYTES / 1024 / NW, K_LOADS = K_BYTES / 1024 / NW, LOADS = M_LOADS + K_LOADS;
    static_assert(M_BYTES % (1024 * NW) == 0 && K_BYTES % (1024 * NW) == 0, "every wave loads whole chunks of 1 KB");
    static constexpr int SLAB = 4096;                        // output staging: 32 rows of 128 bytes a wave
    static_assert(BM >= 64 && BK >= 64 && BM <= 512 && BK <= 512, "");
    template <int NST>
    static constexpr int lds_bytes() { return NST * STAGE + NW * SLAB; }
};

// Place of 16-column unit u of row r in a row of B columns: the four rows by two
// units that 32 lanes of a transposing read take together lie on other banks
// (eight places of 32 bytes).
template <int B>
__device__ __forceinline__ int grad_unit(int r, int u) {
    return u ^ (B >= 128 ? 2 * (r & 3) : r & 2);
}

// f(integral_constant<int, I>) for each I of the sequence, in order
template <class F, int... I>
__device__ __forceinline__ void grad_each(F &&f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}

// Outputs [m0, m0 + BM) x [k0, k0 + BK) of group grp, rows [p0, p1) of the sum,
// its part `part`; the work-group's tile number n.
struct GradTile {
    int m0, k0, grp, p0, p1, part, n;
};

template <int AM, int AK, int WM, int WK, int NST, int OCC>
__global__ __launch_bounds__(64 * WM * WK)
__attribute__((amdgpu_waves_per_eu(OCC, OCC))) void grad_kernel(const GradArgs a) {
    using S = GradShape<AM, AK, WM, WK>;
    constexpr int NW = S::NW, STAGE = S::STAGE;
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave / WK, wk = wave % WK;
    const int M = a.M, K = a.K;
    // an XCD (blockIdx % 8) takes neighbouring tiles of a group, kGradRaster
    // m-tiles side by side, which share columns in its L2, and of every group as
    // many as the others: groups differ in their rows
    const int tiles = a.m_tiles * a.k_tiles, sums = a.groups * a.splits;
    const int x = blockIdx.x % 8, first = blockIdx.x / 8, stride = gridDim.x / 8;      // (a multiple of eight)
    auto chunk = [&](int c) { return (int)((long long)c * tiles / 8); };
    // item u of XCD x: groups (and the parts of their sums) in turn, of each an
    // eighth of the tiles, another one for each
    auto tile_of = [&](int u) {
        int gp = u / tiles * 8, L = u % tiles, c;
        for (;; ++gp) {
            c = (x + gp) & 7;
            const int n = chunk(c + 1) - chunk(c);
            if (L < n) break;
            L -= n;
        }
        L += chunk(c);
        GradTile t;
        t.part = gp / a.groups;
        t.grp = gp - t.part * a.groups;
        const int from = L / (kGradRaster * a.k_tiles) * kGradRaster, size = min(a.m_tiles - from, kGradRaster);
        L -= from * a.k_tiles;
        t.m0 = (from + L % size) * S::BM;
        t.k0 = L / size * S::BK;
        int p0 = 0, p1 = a.N;
        if (a.offsets) {
            // (scalar loads: a vector load would wait for all loads and stores in flight)
            const auto *offsets = (const __attribute__((address_space(4))) int *)(uintptr_t)a.offsets;
            p0 = offsets[t.grp];
            p1 = offsets[t.grp + 1];
        }
        const int steps = (p1 - p0 + kGradRows - 1) / kGradRows, q = steps / a.splits, r = steps % a.splits;
        t.p0 = min(p0 + (t.part * q + min(t.part, r)) * kGradRows, p1);
        t.p1 = min(t.p0 + (q + (t.part < r)) * kGradRows, p1);
        t.n = 0;
        return t;
    };
    int mine = sums / 8 * tiles;                             // the XCD's items
    for (int gp = sums / 8 * 8; gp < sums; ++gp) mine += chunk(((x + gp) & 7) + 1) - chunk((x + gp) & 7);
    if (first >= mine) return;
    auto next = [&](GradTile &t) {
        const int n = t.n + 1, u = first + n * stride;
        if (u >= mine) return 0;
        t = tile_of(u);
        t.n = n;
        return 1;
    };
    // (a group or part without rows takes one step of zeros)
    auto steps_of = [](const GradTile &t) { return max((t.p1 - t.p0 + kGradRows - 1) / kGradRows, 1); };

    // ---- load issue: a chunk of 1 KB holds 512 columns' worth of rows; lane l's
    // 16 bytes of it ----
    auto lane_off = [&](auto b, int ch, int cols) -> uint32_t {
        constexpr int B = decltype(b)::value, PER = B / 8;   // 16-byte pieces of a row
        const int piece = ch * 64 + lane, r = piece / PER, c = piece % PER;
        return ((uint32_t)r * cols + (uint32_t)(2 * grad_unit<B>(r, c >> 1) + (c & 1)) * 8) * 2;
    };
    uint32_t m_off[S::M_LOADS], k_off[S::K_LOADS];
#pragma unroll
    for (int i = 0; i < S::M_LOADS; ++i) m_off[i] = lane_off(std::integral_constant<int, S::BM>{}, wave + NW * i, M);
#pragma unroll
    for (int i = 0; i < S::K_LOADS; ++i) k_off[i] = lane_off(std::integral_constant<int, S::BK>{}, wave + NW * i, K);
    // where the next loads come from: the rows from `left` before the end of tile
    // lt. Columns past M and K hold the next row's, whose outputs are not stored;
    // rows past the end read as zero. Past the last tile nothing is read and zeros
    // are written, so each step issues as many loads
    GradTile tile = tile_of(first), lt = tile;
    const uint16_t *dyg, *xg;
    int left, lsteps;
    auto aim = [&]() {
        dyg = a.dy + (size_t)lt.p0 * M + lt.m0;
        xg = a.x + (size_t)lt.p0 * K + lt.k0;
        left = lt.p1 - lt.p0;
        lsteps = steps_of(lt);
        asm volatile("" : "+s"(dyg), "+s"(xg));
    };
    constexpr int kWord3 = 0x00020000;                       // untyped buffer, format 32
    auto load = [&](auto index, int st) {
        constexpr int n = decltype(index)::value;
        uint8_t *base = smem + st * STAGE;
        // (computed outside the builtins' argument lists: inside them such
        // expressions make the host pass drop the kernel without a diagnostic)
        if constexpr (n < S::M_LOADS) {
            const int range = max(min(left, kGradRows) * M - lt.m0, 0) * 2;
            const uint32_t off = m_off[n];
            __builtin_amdgcn_raw_ptr_buffer_load_lds(__builtin_amdgcn_make_buffer_rsrc((void *)dyg, 0, range, kWord3),
                                                     KXW4_GRAD_LDS(base + (wave + NW * n) * 1024), 16, off, 0, 0, 0);
        } else {
            constexpr int i = n - S::M_LOADS;
            const int range = max(min(left, kGradRows) * K - lt.k0, 0) * 2;
            const uint32_t off = k_off[i];
            __builtin_amdgcn_raw_ptr_buffer_load_lds(__builtin_amdgcn_make_buffer_rsrc((void *)xg, 0, range, kWord3),
                                                     KXW4_GRAD_LDS(base + S::M_BYTES + (wave + NW * i) * 1024), 16, off, 0, 0, 0);
        }
    };
    auto advance = [&]() {
        left -= kGradRows;
        dyg += (size_t)kGradRows * M;
        xg += (size_t)kGradRows * K;
        if (--lsteps == 0) {
            if (next(lt)) {
                aim();
            } else {
                left = 0;
                lsteps = 1 << 30;
            }
        }
    };
    auto issue = [&](int st) {
        grad_each([&](auto n) { load(n, st); }, std::make_integer_sequence<int, S::LOADS>{});
    };
    // transposing reads: the 16 lanes of a group supply four rows of 16 columns
    // (lane 4r + q row r, columns 4q..4q+3) and lane i receives column i; group
    // a takes columns 16 (a % 2) and on and rows 4 (a / 2) and on, of eight
    const int i16 = lane & 15, r7 = 4 * (lane >> 5) + (i16 >> 2), half = (lane >> 4) & 1;
    int m_at[AM], k_at[AK];
#pragma unroll
    for (int i = 0; i < AM; ++i) m_at[i] = r7 * S::BM * 2 + grad_unit<S::BM>(r7, 2 * (wm * AM + i) + half) * 32 + (i16 & 3) * 8;
#pragma unroll
    for (int j = 0; j < AK; ++j)
        k_at[j] = S::M_BYTES + r7 * S::BK * 2 + grad_unit<S::BK>(r7, 2 * (wk * AK + j) + half) * 32 + (i16 & 3) * 8;
    auto read = [&](int off, int step8) -> v8bf {            // rows 0..15 of a half step, eight apart
        const v4s lo = read_tr16((lds_v4s *)(smem + off));
        const v4s hi = read_tr16((lds_v4s *)(smem + off + step8));
        return __builtin_bit_cast(v8bf, (v8s){lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w});
    };

    v16f f[AM][AK];
    auto clear = [&]() {
#pragma unroll
        for (int i = 0; i < AM; ++i)
#pragma unroll
            for (int j = 0; j < AK; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) f[i][j][r] = 0.0f;
    };
    // ---- output: x is the A operand, so register r of a block is column 8(r/4) +
    // 4 (l/32) + r%4 of the lane's row. 32 rows at a time pass the wave's own slab
    // in LDS (rows of 128 bytes, 16-byte chunk c of row m at c ^ (m % 8)) and go
    // out as whole lines: stores of 32 bytes a row reached 2.1 TB/s of BF16, these
    // 8 times 128 bytes a store. Non-temporal, which leaves the L2s to dy and x (64
    // groups of 256 rows, 1,024 x 2,048, BF16: 136 us for 153; 2,048 rows, 5,120 x
    // 5,120: 136 for 141), but for parts of a sum, which are read again at once
    // (8,192 rows, 512 x 512: 22.4 us for 21.0) ----
    const int m32 = lane & 31, kg = lane >> 5;
    const size_t outputs = (size_t)a.groups * M * K;
    uint8_t *slab = smem + NST * STAGE + wave * S::SLAB;
    auto store = [&]() {
        const size_t base = (size_t)tile.grp * M * K;
        auto lines = [&](auto bytes, void *out, int m, int k) {          // the slab's rows to `out`
            constexpr int B = decltype(bytes)::value;        // of an output
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");               // (other lanes' writes)
#pragma unroll
            for (int it = 0; it < 4; ++it) {
                const int r = it * 8 + (lane >> 3), c = lane & 7;
                const v4u v = *reinterpret_cast<const v4u *>(slab + r * 128 + ((c ^ (r & 7)) * 16));
                const int col = k + c * (16 / B);
                if (m + r < M && col < K) {
                    v4u *to = reinterpret_cast<v4u *>(static_cast<uint8_t *>(out) + (base + (size_t)(m + r) * K + col) * B);
                    if (a.splits > 1) *to = v;
                    else store_past(v, to);
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");               // (their reads)
        };
#pragma unroll
        for (int i = 0; i < AM; ++i) {
            const int mrow = tile.m0 + 32 * (wm * AM + i), m = mrow + m32, kcol = tile.k0 + 32 * wk * AK;
            if (a.splits == 1 && a.add && m < M) {
#pragma unroll
                for (int j = 0; j < AK; ++j)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int k = kcol + 32 * j + 8 * q + 4 * kg;
                        if (k >= K) continue;
                        const size_t at = base + (size_t)m * K + k;
                        float x[4];
                        if (a.dw_bf16) {
                            const v2u u = *reinterpret_cast<const v2u *>(static_cast<const uint16_t *>(a.add) + at);
#pragma unroll
                            for (int r = 0; r < 4; ++r) x[r] = __uint_as_float(r & 1 ? u[r / 2] & 0xFFFF0000u : u[r / 2] << 16);
                        } else {
                            const v4f u = *reinterpret_cast<const v4f *>(static_cast<const float *>(a.add) + at);
#pragma unroll
                            for (int r = 0; r < 4; ++r) x[r] = u[r];
                        }
#pragma unroll
                        for (int r = 0; r < 4; ++r) f[i][j][4 * q + r] += x[r];
                    }
            }
            if (a.splits == 1 && a.dw_bf16) {
                static_assert(AK == 2, "64 columns a row of the slab");
#pragma unroll
                for (int j = 0; j < AK; ++j)
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        *reinterpret_cast<v2u *>(slab + m32 * 128 + (((4 * j + q) ^ (m32 & 7)) * 16) + kg * 8) =
                            v2u{pack_bf16(f[i][j][4 * q], f[i][j][4 * q + 1]), pack_bf16(f[i][j][4 * q + 2], f[i][j][4 * q + 3])};
                lines(std::integral_constant<int, 2>{}, a.dw, mrow, kcol);
            } else {
                // (parts of a sum: grad_join_kernel ends it)
                void *out = a.splits > 1 ? static_cast<void *>(a.part + (size_t)tile.part * outputs) : a.dw;
#pragma unroll
                for (int j = 0; j < AK; ++j) {
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        *reinterpret_cast<v4f *>(slab + m32 * 128 + (((2 * q + kg) ^ (m32 & 7)) * 16)) =
                            v4f{f[i][j][4 * q], f[i][j][4 * q + 1], f[i][j][4 * q + 2], f[i][j][4 * q + 3]};
                    lines(std::integral_constant<int, 4>{}, out, mrow, kcol + 32 * j);
                }
            }
        }
    };

    // The two halves of a step (16 rows each) take operands in turn: each half's
    // MFMAs run while the next half's are read. A step's barrier sits between its
    // halves, when all of its operands are in registers: its stage is then free
    // for the loads of NST steps on, which go out between the MFMAs. The ring runs
    // on from tile to tile: the next one's first steps are in flight while this
    // one's outputs are stored.
    constexpr int LD = S::LOADS;
    static_assert(NST >= 2 && NST <= 4 && LD * (NST - 2) <= 63, "two to four stages; vmcnt field");
    static_assert(kGradRows == 32, "two halves");
    // the loads of a step have arrived; those of the NST - 2 after it may be in
    // flight, and for the NST - 1 steps after a whole tile's stores these too,
    // which went out after the loads that are waited for
    constexpr int NS = AM * 4;                               // stores of BF16 rows (FP32: AK = 2 times as many)
    static_assert(LD * (NST - 2) + 2 * NS <= 63, "vmcnt field");
    int stored = 0;
    const bool wide = a.splits > 1 || !a.dw_bf16;
    auto arrive = [&]() {
        if (stored == 0) KXW4_WAIT_VMCNT(LD * (NST - 2));
        else if (wide) KXW4_WAIT_VMCNT(LD * (NST - 2) + 2 * NS);
        else KXW4_WAIT_VMCNT(LD * (NST - 2) + NS);
        stored = max(stored - 1, 0);
        lds_sync_after_dma();
    };
    v8bf mb[2][AM], kb[2][AK];
    auto operands = [&](int h, int base) {
#pragma unroll
        for (int j = 0; j < AK; ++j) kb[h][j] = read(base + k_at[j] + h * 16 * S::BK * 2, 8 * S::BK * 2);
#pragma unroll
        for (int i = 0; i < AM; ++i) mb[h][i] = read(base + m_at[i] + h * 16 * S::BM * 2, 8 * S::BM * 2);
    };
    auto products = [&](int h) {
#pragma unroll
        for (int i = 0; i < AM; ++i)
#pragma unroll
            for (int j = 0; j < AK; ++j) f[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kb[h][j], mb[h][i], f[i][j], 0, 0, 0);
    };
    aim();
#pragma unroll
    for (int s = 0; s < NST; ++s) {
        if (s == NST - 1) arrive();
        issue(s);
        advance();
    }
    operands(0, 0);
    clear();
    int st = 0;
    for (;;) {
        const int NT = steps_of(tile);
        for (int s = 0; s < NT; ++s) {
            const int stn = st == NST - 1 ? 0 : st + 1;
            operands(1, st * STAGE);
            products(0);
            __builtin_amdgcn_sched_barrier(0);
            arrive();
            operands(0, stn * STAGE);                        // (after the last step: harmless reads of zeros)
            issue(st);
            products(1);
            __builtin_amdgcn_sched_group_barrier(0x100, 2 * (AM + AK), 0);
#pragma unroll
            for (int n = 0; n < LD; ++n) {
                __builtin_amdgcn_sched_group_barrier(0x008, AM * AK / LD > 0 ? AM * AK / LD : 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x010, 1, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
            advance();
            st = stn;
        }
        store();
        // (every lane of a whole tile stores; one with `add` has waited for loads)
        stored = tile.m0 + S::BM <= M && tile.k0 + S::BK <= K && !a.add ? NST - 1 : 0;
        if (!next(tile)) break;
        clear();
    }
    KXW4_WAIT_VMCNT(0);                                      // (no load past the last step outlives the work-group's LDS)
}

// The parts of a split sum, in order, and `add` last; four outputs a thread.
__global__ __launch_bounds__(256) void grad_join_kernel(const GradArgs a) {
    const size_t n = (size_t)a.groups * a.M * a.K;
    const size_t at = ((size_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (at >= n) return;
    float4 v = *reinterpret_cast<const float4 *>(a.part + at);
    for (int s = 1; s < a.splits; ++s) {
        const float4 u = *reinterpret_cast<const float4 *>(a.part + s * n + at);
        v.x += u.x;
        v.y += u.y;
        v.z += u.z;
        v.w += u.w;
    }
    if (a.dw_bf16) {
        if (a.add) {
            const uint2 u = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(a.add) + at);
            v.x += __uint_as_float(u.x << 16);
            v.y += __uint_as_float(u.x & 0xFFFF0000u);
            v.z += __uint_as_float(u.y << 16);
            v.w += __uint_as_float(u.y & 0xFFFF0000u);
        }
        *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(a.dw) + at) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
    } else {
        if (a.add) {
            const float4 u = *reinterpret_cast<const float4 *>(static_cast<const float *>(a.add) + at);
            v.x += u.x;
            v.y += u.y;
            v.z += u.z;
            v.w += u.w;
        }
        *reinterpret_cast<float4 *>(static_cast<float *>(a.dw) + at) = v;
    }
}

// Parts of the rows: as many as fill the card where the tiles do not, each of
// eight steps at least.
static int grad_splits(int N, int groups, int M, int K) {
    const long long tiles = (long long)groups * ((M + 127) / 128) * ((K + 127) / 128);
    const long long most = std::max<long long>(1, N / groups / (8 * kGradRows));
    return (int)std::max<long long>(1, std::min({most, device_cus() / std::max<long long>(tiles, 1), 32ll}));
}

size_t grad_scratch(int N, int groups, int M, int K) {
    const int s = grad_splits(N, groups, M, K);
    return s > 1 ? (size_t)s * groups * M * K * sizeof(float) : 0;
}

template <int AM, int AK, int WM, int WK, int NST, int OCC>
static int grad_launch(GradArgs &a, hipStream_t st) {
    using S = GradShape<AM, AK, WM, WK>;
    a.m_tiles = (a.M + S::BM - 1) / S::BM;
    a.k_tiles = (a.K + S::BK - 1) / S::BK;
    const long long items = (long long)a.groups * a.m_tiles * a.k_tiles * a.splits;
    if (items >= (1ll << 31) - (1 << 16)) return -2;         // (32-bit tile numbers)
    constexpr size_t lds = S::template lds_bytes<NST>();
    static_assert(lds <= 160 * 1024, "LDS");
    constexpr int per_cu = std::min(4 * OCC / S::NW, (int)(160 * 1024 / lds));
    const long long grid = std::min<long long>((items + 63) / 8 * 8, (long long)std::max(8, device_cus() / 8 * 8) * per_cu);
    auto k = grad_kernel<AM, AK, WM, WK, NST, OCC>;
    static bool done[64] = {};
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return -6;
    if (!done[dev]) {
        if (hipFuncSetAttribute(reinterpret_cast<const void *>(k), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) != hipSuccess) return -6;
        done[dev] = true;
    }
    hipLaunchKernelGGL(k, dim3((unsigned)grid), dim3(S::NTH), lds, st, a);
    return hipGetLastError() == hipSuccess ? 0 : -6;
}

int launch_grad(GradArgs &a, hipStream_t st) {
    a.splits = grad_splits(a.N, a.groups, a.M, a.K);
    // 256 x 256 outputs a work-group read half the bytes of 128 x 128 from LDS and
    // the caches; they need a tile for each CU. Measured on 256 CUs (this, then
    // 128 x 128, us): 4,096 rows 5,120 x 5,120 224 / 241; 2,048 rows 17,408 x 5,120
    // 345 / 388; 64 groups of 256 rows 1,024 x 2,048 150 / 167 (134 now); 16 groups of 512
    // rows 63 / 62.
    const long long big = (long long)a.groups * ((a.M + 255) / 256) * ((a.K + 255) / 256);
    const int rc = a.splits == 1 && big >= device_cus() ? grad_launch<4, 2, 2, 4, 4, 2>(a, st)
                                                        : grad_launch<2, 2, 2, 2, 4, 2>(a, st);
    if (rc || a.splits == 1) return rc;
    const long long grid = ((long long)a.groups * a.M * a.K / 4 + 255) / 256;
    if (grid > grid_limit(256)) return -2;
    hipLaunchKernelGGL(grad_join_kernel, dim3((unsigned)grid), dim3(256), 0, st, a);
    return hipGetLastError() == hipSuccess ? 0 : -6;
}

}  // namespace kxw4
