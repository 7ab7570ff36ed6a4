// kxw4_grad.hip — the gradient of a projection's weight, for one weight or by
// group: dw_g[m][k] = sum over the rows p of group g of dy[p][m] * x[p][k]. No
// counterpart in the reference, which trains nothing.
//
// BF16 rows, exact products, FP32 sums (the 32x32x16 BF16 MFMA). The sum runs
// over rows, which lie apart in memory, so both operands are read transposed: a
// step's rows reach LDS as they lie, by buffer loads straight into a ring of
// NST stages, and ds_read_b64_tr_b16 gives a lane four rows of its column. A
// work-group owns 32 AM WM x 32 AK WK outputs of one group; the rows past the
// group's end read as zero through the buffer's range. Where there are few
// tiles the rows are split over work-groups and their FP32 parts added in order
// by a second launch.
#include "kxw4_device.hpp"
#include "kxw4_internal.hpp"

#include <algorithm>
#include <type_traits>

namespace kxw4 {

typedef float v16f __attribute__((ext_vector_type(16)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef short v8s __attribute__((ext_vector_type(8)));

#define KXW4_GRAD_LDS(p) ((__attribute__((address_space(3))) void *)(p))

constexpr int kGradRows = 32;                                // rows of a step

template <int AM, int AK, int WM, int WK>
struct GradShape {
    static constexpr int NW = WM * WK, NTH = 64 * NW;
    static constexpr int BM = 32 * AM * WM, BK = 32 * AK * WK;
    static constexpr int M_BYTES = kGradRows * BM * 2, K_BYTES = kGradRows * BK * 2, STAGE = M_BYTES + K_BYTES;
    static constexpr int M_LOADS = M_BYTES / 1024 / NW, K_LOADS = K_BYTES / 1024 / NW, LOADS = M_LOADS + K_LOADS;
    static_assert(M_BYTES % (1024 * NW) == 0 && K_BYTES % (1024 * NW) == 0, "every wave loads whole chunks of 1 KB");
    static_assert(BM >= 64 && BK >= 64 && BM <= 512 && BK <= 512, "");
    static constexpr int EPS = 32 * AK + 4, SLAB = 32 * EPS * 4;
    template <int NST>
    static constexpr int lds_bytes() { return NST * STAGE > NW * SLAB ? NST * STAGE : NW * SLAB; }
};

// Place of 16-column unit u of row r in a row of B columns: the four rows that
// a transposing read takes together, and the four beside them, meet other banks.
template <int B>
__device__ __forceinline__ int grad_unit(int r, int u) {
    return B >= 128 ? u ^ (r & 7) : u ^ ((r >> 1) & 3);
}

template <int AM, int AK, int WM, int WK, int NST, int OCC, bool SPLIT>
__global__ __launch_bounds__(64 * WM * WK)
__attribute__((amdgpu_waves_per_eu(OCC, OCC))) void grad_kernel(const GradArgs a) {
    using S = GradShape<AM, AK, WM, WK>;
    constexpr int NW = S::NW, STAGE = S::STAGE;
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave / WK, wk = wave % WK;
    // neighbouring tiles of a group to one XCD
    const int nblk = gridDim.x, id = blockIdx.x;
    const int q8 = nblk / 8, r8 = nblk % 8, xcd = id % 8, j8 = id / 8;
    int L = xcd < r8 ? xcd * (q8 + 1) + j8 : r8 * (q8 + 1) + (xcd - r8) * q8 + j8;
    const int kt = L % a.k_tiles;
    L /= a.k_tiles;
    const int mt = L % a.m_tiles;
    L /= a.m_tiles;
    const int grp = L % a.groups, split = L / a.groups;
    const int M = a.M, K = a.K;
    int p0 = a.offsets ? a.offsets[grp] : 0, p1 = a.offsets ? a.offsets[grp + 1] : a.N;
    if constexpr (SPLIT) {
        const int steps = (p1 - p0 + kGradRows - 1) / kGradRows, per = (steps + a.splits - 1) / a.splits;
        p0 = min(p0 + split * per * kGradRows, p1);
        p1 = min(p0 + per * kGradRows, p1);
    }
    const int m0 = mt * S::BM, k0 = kt * S::BK, NT = (p1 - p0 + kGradRows - 1) / kGradRows;

    // a chunk of 1 KB: 512 columns' worth of rows; lane l's 16 bytes
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
    const uint16_t *dyg = a.dy + m0, *xg = a.x + k0;
    asm volatile("" : "+s"(dyg), "+s"(xg));
    constexpr int kWord3 = 0x00020000;
    auto issue = [&](int s, int st) {
        const int p = p0 + s * kGradRows, rows = min(p1 - p, kGradRows);
        uint8_t *base = smem + st * STAGE;
        // (computed outside the builtins' argument lists: inside them such
        // expressions make the host pass drop the kernel without a diagnostic)
        const uint16_t *dyp = dyg + (size_t)p * M, *xp = xg + (size_t)p * K;
        const int dy_range = (rows * M - m0) * 2, x_range = (rows * K - k0) * 2;
#pragma unroll
        for (int i = 0; i < S::M_LOADS; ++i) {
            const uint32_t off = m_off[i];
            __builtin_amdgcn_raw_ptr_buffer_load_lds(__builtin_amdgcn_make_buffer_rsrc((void *)dyp, 0, dy_range, kWord3),
                                                     KXW4_GRAD_LDS(base + (wave + NW * i) * 1024), 16, off, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < S::K_LOADS; ++i) {
            const uint32_t off = k_off[i];
            __builtin_amdgcn_raw_ptr_buffer_load_lds(__builtin_amdgcn_make_buffer_rsrc((void *)xp, 0, x_range, kWord3),
                                                     KXW4_GRAD_LDS(base + S::M_BYTES + (wave + NW * i) * 1024), 16, off, 0, 0, 0);
        }
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
    auto read = [&](int off, int step8) -> v8bf {            // rows 0..15 of a K16 step, eight apart
        const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s *)(smem + off));
        const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s *)(smem + off + step8));
        return __builtin_bit_cast(v8bf, (v8s){lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w});
    };

    v16f f[AM][AK];
#pragma unroll
    for (int i = 0; i < AM; ++i)
#pragma unroll
        for (int j = 0; j < AK; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) f[i][j][r] = 0.0f;

    constexpr int LD = S::LOADS;
    static_assert(NST >= 2 && NST <= 4 && LD * (NST - 2) <= 63, "two to four stages; vmcnt field");
    auto arrive = [&](int k) {
        const int later = min(NST - 2, NT - 1 - k);
        if (NST >= 4 && later >= 2) KXW4_WAIT_VMCNT(2 * LD);
        else if (NST >= 3 && later >= 1) KXW4_WAIT_VMCNT(LD);
        else KXW4_WAIT_VMCNT(0);
        lds_sync_after_dma();
    };
#pragma unroll
    for (int s = 0; s < NST - 1; ++s)
        if (s < NT) issue(s, s);
    int st = 0;
    for (int s = 0; s < NT; ++s) {
        arrive(s);
        if (s + NST - 1 < NT) issue(s + NST - 1, st == 0 ? NST - 1 : st - 1);
        const int base = st * STAGE;
#pragma unroll
        for (int h = 0; h < kGradRows / 16; ++h) {
            v8bf kb[AK];
#pragma unroll
            for (int j = 0; j < AK; ++j) kb[j] = read(base + k_at[j] + h * 16 * S::BK * 2, 8 * S::BK * 2);
#pragma unroll
            for (int i = 0; i < AM; ++i) {
                const v8bf mb = read(base + m_at[i] + h * 16 * S::BM * 2, 8 * S::BM * 2);
#pragma unroll
                for (int j = 0; j < AK; ++j) f[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(mb, kb[j], f[i][j], 0, 0, 0);
            }
        }
        st = st == NST - 1 ? 0 : st + 1;
    }
    // ---- output: register r of a block is row 8(r/4) + 4 (l/32) + r%4, column
    // l % 32; 32 rows at a time through the wave's own slab ----
    lds_sync();
    float *slab = reinterpret_cast<float *>(smem + wave * S::SLAB);
    const size_t out0 = (size_t)grp * M * K;
    float *part = SPLIT ? a.part + (size_t)split * a.groups * M * K : nullptr;
    auto run = [&](auto ch, int mrow) {
        constexpr int CH = decltype(ch)::value, PER = 32 * AK / CH;
#pragma unroll
        for (int it = 0; it < 32 * PER / 64; ++it) {
            const int q = it * 64 + lane, ml = q / PER, kl = (q % PER) * CH;
            const int m = m0 + mrow + ml, k = k0 + wk * 32 * AK + kl;
            if (m >= M || k >= K) continue;
            const size_t at = out0 + (size_t)m * K + k;
            float v[CH];
#pragma unroll
            for (int c = 0; c < CH; c += 4) {
                const v4f x = *reinterpret_cast<const v4f *>(slab + ml * S::EPS + kl + c);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[c + j] = x[j];
            }
            if constexpr (SPLIT) {
                *reinterpret_cast<float4 *>(part + at) = make_float4(v[0], v[1], v[2], v[3]);
            } else if constexpr (CH == 8) {
                if (a.add) {
                    const uint4 u = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(a.add) + at);
                    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        v[2 * j] += __uint_as_float(w[j] << 16);
                        v[2 * j + 1] += __uint_as_float(w[j] & 0xFFFF0000u);
                    }
                }
                *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(a.dw) + at) =
                    make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
            } else {
                if (a.add) {
                    const float4 u = *reinterpret_cast<const float4 *>(static_cast<const float *>(a.add) + at);
                    v[0] += u.x;
                    v[1] += u.y;
                    v[2] += u.z;
                    v[3] += u.w;
                }
                *reinterpret_cast<float4 *>(static_cast<float *>(a.dw) + at) = make_float4(v[0], v[1], v[2], v[3]);
            }
        }
    };
#pragma unroll
    for (int i = 0; i < AM; ++i) {
#pragma unroll
        for (int j = 0; j < AK; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) slab[(8 * (r >> 2) + 4 * (lane >> 5) + (r & 3)) * S::EPS + 32 * j + (lane & 31)] = f[i][j][r];
        const int mrow = (wm * AM + i) * 32;
        if (!SPLIT && a.dw_bf16) run(std::integral_constant<int, 8>{}, mrow);
        else run(std::integral_constant<int, 4>{}, mrow);
    }
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

template <int AM, int AK, int WM, int WK, int NST, int OCC, bool SPLIT>
static int grad_launch(GradArgs &a, hipStream_t st) {
    using S = GradShape<AM, AK, WM, WK>;
    a.m_tiles = (a.M + S::BM - 1) / S::BM;
    a.k_tiles = (a.K + S::BK - 1) / S::BK;
    const long long grid = (long long)a.groups * a.m_tiles * a.k_tiles * a.splits;
    if (grid > grid_limit(S::NTH)) return -2;
    auto k = grad_kernel<AM, AK, WM, WK, NST, OCC, SPLIT>;
    constexpr size_t lds = S::template lds_bytes<NST>();
    static_assert(lds <= 160 * 1024, "LDS");
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
    if (a.splits > 1) {
        const int rc = grad_launch<2, 2, 2, 2, 3, 2, true>(a, st);
        if (rc) return rc;
        const long long grid = ((long long)a.groups * a.M * a.K / 4 + 255) / 256;
        if (grid > grid_limit(256)) return -2;
        hipLaunchKernelGGL(grad_join_kernel, dim3((unsigned)grid), dim3(256), 0, st, a);
        return hipGetLastError() == hipSuccess ? 0 : -6;
    }
    const long long big = (long long)a.groups * ((a.M + 255) / 256) * ((a.K + 255) / 256);
    if (big >= device_cus()) return grad_launch<4, 2, 2, 4, 3, 2, false>(a, st);
    return grad_launch<2, 2, 2, 2, 3, 2, false>(a, st);
}

}  // namespace kxw4
