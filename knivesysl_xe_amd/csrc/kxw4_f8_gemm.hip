// kxw4_f8_gemm.hip — launches of the 8-bit floating tier's large tiles
// (kxw4_f8_gemm.hpp).
#include "kxw4_f8_gemm.hpp"

namespace kxw4 {

// Allow `k` as much dynamic LDS as it asks for, once per device.
static int f8_lds(const void *k, size_t lds, bool (&done)[64]) {
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return -6;
    if (done[dev]) return 0;
    if (hipFuncSetAttribute(k, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) != hipSuccess) return -6;
    done[dev] = true;
    return 0;
}

static int f8_plan(F8GemmArgs &a, int rgs) {
    int nt = 0;
    for (int i = 0; i < a.count; ++i) {
        a.w[i].nt_begin = nt;
        nt += (a.w[i].M / 16 + rgs - 1) / rgs;
    }
    a.n_tiles = nt;
    return nt;
}

template <int TA, int TB, int WT, int WR, int NST, int EX, int OCC>
static int f8_dense(F8GemmArgs &a, hipStream_t st) {
    using S = F8Shape<TA, TB, WT, WR>;
    const long long grid = (long long)f8_plan(a, S::BR / 16) * ((a.rows + S::BT - 1) / S::BT);
    if (grid > grid_limit(S::NTH)) return -2;
    auto k = f8_gemm_kernel<TA, TB, WT, WR, NST, EX, OCC>;
    constexpr size_t lds = S::template lds_bytes<NST>();
    static_assert(lds <= 160 * 1024, "LDS");
    static bool done[64] = {};
    const int rc = f8_lds(reinterpret_cast<const void *>(k), lds, done);
    if (rc) return rc;
    hipLaunchKernelGGL(k, dim3((unsigned)grid), dim3(S::NTH), lds, st, a);
    return hipGetLastError() == hipSuccess ? 0 : -6;
}

template <int TA, int TB, int WR, int NST, int EX, int OCC>
static int f8_grouped(F8GemmArgs &a, hipStream_t st) {
    using S = F8Shape<TA, TB, 1, WR>;
    const long long grid = tiles_at_most(a.N, a.groups, S::BT) * f8_plan(a, S::BR / 16);
    if (grid > grid_limit(S::NTH)) return -2;
    auto k = f8_group_kernel<TA, TB, WR, NST, EX, OCC>;
    constexpr size_t lds = std::max({S::template lds_bytes<NST>(), F8Shape<(TA > 1 ? TA / 2 : 1), TB, 1, WR>::template lds_bytes<NST>(),
                                     F8Shape<1, TB, 1, WR>::template lds_bytes<NST>()});
    static_assert(lds <= 160 * 1024, "LDS");
    static bool done[64] = {};
    const int rc = f8_lds(reinterpret_cast<const void *>(k), lds, done);
    if (rc) return rc;
    hipLaunchKernelGGL(k, dim3((unsigned)grid), dim3(S::NTH), lds, st, a);
    return hipGetLastError() == hipSuccess ? 0 : -6;
}

int launch_f8_gemm(F8GemmArgs &a, hipStream_t st) {
    if (a.groups) return a.y_bf16 ? f8_grouped<2, 2, 2, 2, 0, 2>(a, st) : f8_grouped<2, 2, 2, 2, 1, 2>(a, st);
    if (a.y_bf16) return f8_dense<4, 2, 2, 4, 2, 0, 2>(a, st);
    return f8_dense<2, 2, 2, 2, 2, 1, 2>(a, st);
}

}  // namespace kxw4
