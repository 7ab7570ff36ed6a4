// kxw4_f8_gemm.hip — launches of the 8-bit floating tier's large tiles
// (kxw4_f8_gemm.hpp).
#include "kxw4_f8_gemm.hpp"
#include "kxw4_f8_route.hpp"

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

// Work-groups that the card holds at once, a multiple of eight.
template <class S, int NST, int OCC>
static long long f8_slots() {
    constexpr int per_cu = std::min(4 * OCC / S::NW, 160 * 1024 / S::template lds_bytes<NST>());
    static_assert(per_cu >= 1, "");
    return (long long)std::max(8, device_cus() / 8 * 8) * per_cu;
}

template <int TA, int TB, int WT, int WR, int NST, int EX, int OCC>
static int f8_dense(F8GemmArgs &a, hipStream_t st) {
    using S = F8Shape<TA, TB, WT, WR>;
    const long long tiles = (long long)f8_plan(a, S::BR / 16) * ((a.rows + S::BT - 1) / S::BT) * a.splits;
    if (tiles >= (1ll << 31) - (1 << 16)) return -2;         // (32-bit tile numbers)
    const long long grid = std::min<long long>(tiles, f8_slots<S, NST, OCC>());
    auto k = f8_gemm_kernel<TA, TB, WT, WR, NST, EX, OCC>;
    constexpr size_t lds = S::template lds_bytes<NST>();
    static_assert(lds <= 160 * 1024, "LDS");
    static bool done[64] = {};
    const int rc = f8_lds(reinterpret_cast<const void *>(k), lds, done);
    if (rc) return rc;
    hipLaunchKernelGGL(k, dim3((unsigned)grid), dim3(S::NTH), lds, st, a);
    return hipGetLastError() == hipSuccess ? 0 : -6;
}

template <int TA, int TB, int WT, int WR, int NST, int EX, int OCC>
static int f8_grouped(F8GemmArgs &a, hipStream_t st) {
    using S = F8Shape<TA, TB, WT, WR>;
    const long long tiles = tiles_at_most(a.N, a.groups, S::BT) * f8_plan(a, S::BR / 16);
    if (tiles >= (1ll << 31) - (1 << 20)) return -2;         // (32-bit tile numbers)
    const long long grid = std::min<long long>((tiles + 7) / 8 * 8, f8_slots<S, NST, OCC>());
    auto k = f8_group_kernel<TA, TB, WT, WR, NST, EX, OCC>;
    constexpr size_t lds = S::template lds_bytes<NST>();
    static_assert(lds <= 160 * 1024, "LDS");
    static bool done[64] = {};
    const int rc = f8_lds(reinterpret_cast<const void *>(k), lds, done);
    if (rc) return rc;
    hipLaunchKernelGGL(k, dim3((unsigned)grid), dim3(S::NTH), lds, st, a);
    return hipGetLastError() == hipSuccess ? 0 : -6;
}

static F8Sizes f8_sizes(const F8GemmArgs &a) {
    F8Sizes s{device_cus(), a.groups ? a.N : a.rows, a.KB, a.count, {}, a.groups, a.y_bf16 != 0};
    for (int i = 0; i < a.count; ++i) s.M[i] = a.w[i].M;
    return s;
}

size_t f8_gemm_scratch(const F8GemmArgs &a) {
    if (a.groups) return 0;
    const F8Choice c = f8_choose(f8_sizes(a));
    size_t outputs = 0;
    for (int i = 0; i < a.count; ++i) outputs += (size_t)a.rows * a.w[i].M;
    return c.splits > 1 ? outputs * c.splits * sizeof(float) : 0;
}

static int f8_config(F8GemmArgs &a, int id, hipStream_t st) {
    switch (id) {
    case 0: return f8_dense<4, 2, 2, 4, 2, 0, 2>(a, st);
    case 1: return f8_dense<2, 2, 4, 2, 3, 0, 2>(a, st);
    case 2: return f8_dense<2, 2, 2, 2, 4, 0, 2>(a, st);
    case 3: return f8_dense<1, 2, 2, 2, 3, 0, 2>(a, st);
    case 4: return f8_dense<2, 2, 2, 2, 2, 1, 2>(a, st);
    default: return f8_dense<1, 2, 2, 2, 3, 1, 2>(a, st);
    }
}

int launch_f8_gemm(F8GemmArgs &a, hipStream_t st) {
    if (!a.groups) {
        const F8Choice c = f8_choose(f8_sizes(a));
        a.splits = c.splits;
        long long outputs = 0;
        for (int i = 0; i < a.count; ++i) {
            a.w[i].part = outputs * a.splits;
            outputs += (long long)a.rows * a.w[i].M;
        }
        if (a.splits == 1) a.part = nullptr;
        // Outputs of twice the L2s (4 MB an XCD) and more go past them, which leaves
        // them to the codes: 8,192 rows, 1,024 -> 16,384 (268 MB): 168 us, else 221;
        // 4,096 -> 16,384: 487, 504; 2 x 17,408 of 3,965 rows: 685, 697; 33 MB: as
        // long. (By group 1,024 -> 5,120 took 313 us so, else 291.)
        a.stream = outputs * 2 >= 64ll << 20;
        const int rc = f8_config(a, c.id, st);
        if (rc || a.splits == 1) return rc;
        const long long grid = (outputs / 4 + 255) / 256;
        if (grid > grid_limit(256)) return -2;
        hipLaunchKernelGGL(f8_join_kernel, dim3((unsigned)grid), dim3(256), 0, st, a);
        return hipGetLastError() == hipSuccess ? 0 : -6;
    }
    a.splits = 1;
    a.part = nullptr;
    const bool long_runs = f8_long_groups(f8_sizes(a));
    if (a.y_bf16) return long_runs ? f8_grouped<2, 2, 2, 4, 3, 0, 2>(a, st) : f8_grouped<1, 2, 2, 2, 3, 0, 2>(a, st);
    return long_runs ? f8_grouped<2, 2, 2, 2, 2, 1, 2>(a, st) : f8_grouped<1, 2, 2, 2, 3, 1, 2>(a, st);
}

}  // namespace kxw4
