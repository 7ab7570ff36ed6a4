// kxw4_rows.hip — rows sorted by the group (expert, adapter) that each of
// their slots names, and back: the plan, the dispatch, the weighted
// combination and its gradient. No counterpart in the reference, whose model
// is dense.
//
// A slot is one (token t, choice j) pair, numbered t*k + j; N = T*k. The plan
// is a stable counting sort of the slots by group, those that name no group
// last:
//   offsets[e]  slots with a group below e (offsets[groups] slots have one)
//   order[p]    the slot at sorted place p, all N of them
//   position[s] the place of slot s, -1 when it names no group
// Integers only, so the plan is the same every time. Every sum below runs in
// FP32 in a fixed order (choices in turn; the dot products over 256-thread
// strides, then lanes, then waves) and is rounded once, to the output's type.
#include "kxw4_device.hpp"
#include "kxw4_internal.hpp"

#include <algorithm>

namespace kxw4 {

// ---- the plan --------------------------------------------------------------

constexpr int kPlanWaves = 8, kPlanThreads = 64 * kPlanWaves;

// Group of slot s, `groups` for none. (64-bit ids are compared before they
// are narrowed.)
__device__ __forceinline__ int slot_key(const RouteArgs &a, int s) {
    if (a.ids64) {
        const long long v = static_cast<const long long *>(a.ids)[s];
        return v < 0 || v >= a.groups ? a.groups : (int)v;
    }
    const int v = static_cast<const int *>(a.ids)[s];
    return v < 0 || v >= a.groups ? a.groups : v;
}

// Counts of the keys in [b0, b1), by wave: wave w takes the w-th of kPlanWaves
// consecutive runs of `per` slots. cnt: [waves][groups + 1], cleared here.
__device__ __forceinline__ void plan_count(const RouteArgs &a, int b0, int b1, int per, int *cnt) {
    const int G1 = a.groups + 1, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int i = tid; i < kPlanWaves * G1; i += kPlanThreads) cnt[i] = 0;
    __syncthreads();
    const int w1 = min(b1, b0 + (wave + 1) * per);
    for (int s = b0 + wave * per + lane; s < w1; s += 64) atomicAdd(&cnt[wave * G1 + slot_key(a, s)], 1);
    __syncthreads();
}

// Large plans, first launch: hist[block][key].
__global__ __launch_bounds__(kPlanThreads) void plan_hist_kernel(const RouteArgs a) {
    extern __shared__ int cnt[];
    const int G1 = a.groups + 1, b0 = blockIdx.x * a.per_block, b1 = min(a.N, b0 + a.per_block);
    plan_count(a, b0, b1, a.per_block / kPlanWaves, cnt);
    for (int g = threadIdx.x; g < G1; g += kPlanThreads) {
        int sum = 0;
        for (int w = 0; w < kPlanWaves; ++w) sum += cnt[w * G1 + g];
        a.hist[(size_t)blockIdx.x * G1 + g] = sum;
    }
}

// The plan (one block), or the last launch of a large one: each block counts
// its own run of slots again, adds up the blocks before it, and places its
// slots. Within a wave the slots of one key find their rank by comparing keys
// bit by bit over the lanes, so the sort is stable and no order of atomics
// shows. A plan of 64 to 16,384 slots is a chain of a few memory and LDS
// round trips.
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(const RouteArgs a) {
    extern __shared__ int cnt[];                             // [waves][groups + 1], then [groups + 1] totals
    const int G = a.groups, G1 = G + 1, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int *tot = cnt + kPlanWaves * G1;
    const int b0 = blockIdx.x * a.per_block, b1 = min(a.N, b0 + a.per_block), per = a.per_block / kPlanWaves;
    plan_count(a, b0, b1, per, cnt);
    // cnt becomes each wave's first place within its key's slots, tot the
    // key's slots over all blocks
    for (int g = tid; g < G1; g += kPlanThreads) {
        int before = 0, all = 0;
        for (int b = 0; b < (int)gridDim.x && gridDim.x > 1; ++b) {
            const int h = a.hist[(size_t)b * G1 + g];
            before += b < (int)blockIdx.x ? h : 0;
            all += h;
        }
        for (int w = 0; w < kPlanWaves; ++w) {
            const int c = cnt[w * G1 + g];
            cnt[w * G1 + g] = before;
            before += c;
        }
        tot[g] = gridDim.x > 1 ? all : before;
    }
    __syncthreads();
    // exclusive scan of the totals: lane l takes a run of keys
    if (wave == 0) {
        const int run = (G1 + 63) / 64, g0 = min(lane * run, G1), g1 = min(g0 + run, G1);
        int sum = 0;
        for (int g = g0; g < g1; ++g) sum += tot[g];
        int inc = sum;
        for (int o = 1; o < 64; o <<= 1) {
            const int v = __shfl_up(inc, o, 64);
            if (lane >= o) inc += v;
        }
        int at = inc - sum;
        for (int g = g0; g < g1; ++g) {
            const int c = tot[g];
            tot[g] = at;
            if (blockIdx.x == 0) a.offsets[g] = at;          // (offsets[groups]: where those without a group begin)
            at += c;
        }
    }
    __syncthreads();
    int bits = 32 - __builtin_clz(G);                        // (keys run to G itself)
    volatile int *mine = cnt + wave * G1;
    const int w1 = min(b1, b0 + (wave + 1) * per);
    for (int s0 = b0 + wave * per; s0 < w1; s0 += 64) {
        const int s = s0 + lane;
        const bool on = s < w1;
        const int key = on ? slot_key(a, s) : 0;
        unsigned long long same = __ballot(on);
        for (int b = 0; b < bits; ++b) {
            const unsigned long long one = __ballot(key >> b & 1);
            same &= (key >> b & 1) ? one : ~one;
        }
        const unsigned long long below = same & ((1ull << lane) - 1);
        if (on) {
            const int first = mine[key], place = tot[key] + first + __popcll(below);
            a.order[place] = s;
            a.position[s] = key < G ? place : -1;
        }
        // (the wave's reads above come before this write: LDS accesses of one
        // wave complete in order)
        __builtin_amdgcn_wave_barrier();
        if (on && below == 0) mine[key] = mine[key] + __popcll(same);
        __builtin_amdgcn_wave_barrier();
    }
}

// Slots per block: one block up to 16,384, else at most 256 blocks of a
// multiple of 512.
int route_blocks_of(int N, int *per_block) {
    constexpr int kOne = 16384, kLeast = 2048;
    auto round = [](long long v) { return (int)((v + kPlanThreads - 1) / kPlanThreads * kPlanThreads); };
    if (N <= kOne) {
        *per_block = std::max(kPlanThreads, round(N));
        return 1;
    }
    *per_block = std::max(kLeast, round((N + 255) / 256));
    return (N + *per_block - 1) / *per_block;
}

int launch_route(RouteArgs &a, hipStream_t st) {
    const int nb = route_blocks_of(a.N, &a.per_block), G1 = a.groups + 1;
    const size_t lds = (size_t)(kPlanWaves + 1) * G1 * sizeof(int);       // (at most 36.9 KB: 1,024 groups)
    if (nb > 1) {
        if (!a.hist) return -1;
        hipLaunchKernelGGL(plan_hist_kernel, dim3(nb), dim3(kPlanThreads), lds, st, a);
    }
    hipLaunchKernelGGL(plan_kernel, dim3(nb), dim3(kPlanThreads), lds, st, a);
    return hipGetLastError() == hipSuccess ? 0 : -6;
}

// ---- rows ------------------------------------------------------------------

constexpr int kRowThreads = 256;

template <int V>
struct Raw;                                                  // V bytes moved as one
template <> struct Raw<16> { typedef v4u type; };
template <> struct Raw<8> { typedef v2u type; };
template <> struct Raw<4> { typedef uint32_t type; };
template <> struct Raw<2> { typedef uint16_t type; };

// rows[position[t, j]] = x[t]: a thread reads one piece of a token's row and
// writes it to each of the token's places, so x is read once. Bound by the
// writes.
template <int V>
__global__ __launch_bounds__(kRowThreads) void dispatch_kernel(const RowArgs a) {
    typedef typename Raw<V>::type P;
    const int pieces = a.pieces, bpr = (pieces + kRowThreads - 1) / kRowThreads;
    const int t = blockIdx.x / bpr, c = (blockIdx.x - t * bpr) * kRowThreads + threadIdx.x;
    if (c >= pieces) return;
    const P v = static_cast<const P *>(a.x)[(size_t)t * pieces + c];
    const int *pos = a.position + (size_t)t * a.k;
    for (int j = 0; j < a.k; ++j) {
        const int p = pos[j];
        if (p >= 0) static_cast<P *>(a.rows)[(size_t)p * pieces + c] = v;
    }
}

// V consecutive elements of a row as FP32, and back with one rounding.
template <int V, bool BF>
__device__ __forceinline__ void load_row(const void *base, size_t at, float (&v)[V]) {
    if constexpr (BF && V == 8) {
        const v4u u = *reinterpret_cast<const v4u *>(static_cast<const uint16_t *>(base) + at);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(u[i] << 16);
            v[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
        }
    } else if constexpr (!BF && V == 8) {
        const v4f *p = reinterpret_cast<const v4f *>(static_cast<const float *>(base) + at);
        const v4f lo = p[0], hi = p[1];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = lo[i];
            v[4 + i] = hi[i];
        }
    } else {
        static_assert(V == 1, "one or eight elements");
        v[0] = BF ? bf16_to_float(static_cast<const uint16_t *>(base)[at]) : static_cast<const float *>(base)[at];
    }
}

template <int V, bool BF>
__device__ __forceinline__ void store_row(void *base, size_t at, const float (&v)[V]) {
    if constexpr (BF && V == 8) {
        v4u u;
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = round_bf16(v[2 * i]) | round_bf16(v[2 * i + 1]) << 16;
        *reinterpret_cast<v4u *>(static_cast<uint16_t *>(base) + at) = u;
    } else if constexpr (!BF && V == 8) {
        v4f *p = reinterpret_cast<v4f *>(static_cast<float *>(base) + at);
        p[0] = v4f{v[0], v[1], v[2], v[3]};
        p[1] = v4f{v[4], v[5], v[6], v[7]};
    } else if constexpr (BF) {
        static_cast<uint16_t *>(base)[at] = (uint16_t)round_bf16(v[0]);
    } else {
        static_cast<float *>(base)[at] = v[0];
    }
}

// y[t] = sum_j w[t, j] rows[position[t, j]] (w 1 where none is given): a
// thread owns V elements of a token's row; up to kAhead choices' pieces are
// requested before the first is added. Bound by the reads.
constexpr int kAhead = 4;
template <int V, bool RB, bool YB>
__global__ __launch_bounds__(kRowThreads) void combine_kernel(const RowArgs a) {
    const int pieces = a.pieces, bpr = (pieces + kRowThreads - 1) / kRowThreads;
    const int t = blockIdx.x / bpr, c = (blockIdx.x - t * bpr) * kRowThreads + threadIdx.x;
    if (c >= pieces) return;
    const int *pos = a.position + (size_t)t * a.k;
    const float *w = a.weights ? a.weights + (size_t)t * a.k : nullptr;
    float acc[V] = {};
    for (int j0 = 0; j0 < a.k; j0 += kAhead) {
        float v[kAhead][V], wj[kAhead];
        int p[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            p[i] = j0 + i < a.k ? pos[j0 + i] : -1;
            wj[i] = w && j0 + i < a.k ? w[j0 + i] : 1.0f;
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            if (p[i] >= 0) load_row<V, RB>(a.rows, (size_t)p[i] * a.H + (size_t)c * V, v[i]);
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            if (p[i] >= 0)
#pragma unroll
                for (int e = 0; e < V; ++e) acc[e] = __builtin_fmaf(wj[i], v[i][e], acc[e]);
    }
    store_row<V, YB>(a.y, (size_t)t * a.H + (size_t)c * V, acc);
}

// drows[position[t, j]] = w[t, j] dy[t], dw[t, j] = <dy[t], rows[position[t,
// j]]>: one block per token and run of kDots choices, which reads dy once for
// all of them. Bound by the rows read and written.
constexpr int kDots = 4;
template <int V, bool DB, bool RB>
__global__ __launch_bounds__(kRowThreads) void combine_backward_kernel(const RowArgs a) {
    __shared__ float part[kRowThreads / 64][kDots];
    const int runs = (a.k + kDots - 1) / kDots;
    const int t = blockIdx.x / runs, j0 = (blockIdx.x - t * runs) * kDots;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int p[kDots];
    float w[kDots], dot[kDots] = {};
#pragma unroll
    for (int i = 0; i < kDots; ++i) {
        p[i] = j0 + i < a.k ? a.position[(size_t)t * a.k + j0 + i] : -1;
        w[i] = j0 + i < a.k ? a.weights[(size_t)t * a.k + j0 + i] : 0.0f;
    }
    for (int c = tid; c < a.pieces; c += kRowThreads) {
        float dy[V], v[kDots][V];
        load_row<V, DB>(a.x, (size_t)t * a.H + (size_t)c * V, dy);
#pragma unroll
        for (int i = 0; i < kDots; ++i)
            if (p[i] >= 0) load_row<V, RB>(a.rows, (size_t)p[i] * a.H + (size_t)c * V, v[i]);
#pragma unroll
        for (int i = 0; i < kDots; ++i) {
            if (p[i] < 0) continue;
            float d[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                dot[i] = __builtin_fmaf(dy[e], v[i][e], dot[i]);
                d[e] = w[i] * dy[e];
            }
            store_row<V, RB>(a.y, (size_t)p[i] * a.H + (size_t)c * V, d);
        }
    }
#pragma unroll
    for (int i = 0; i < kDots; ++i) {
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) dot[i] += __shfl_xor(dot[i], o, 64);
        if (lane == 0) part[wave][i] = dot[i];
    }
    __syncthreads();
    if (tid < kDots && j0 + tid < a.k) {
        float sum = 0.0f;
        for (int q = 0; q < kRowThreads / 64; ++q) sum += part[q][tid];
        a.dweights[(size_t)t * a.k + j0 + tid] = sum;        // (0 where the slot names no group)
    }
}

// Whether 16-byte pieces fit every row: aligned bases, eight elements or whole
// 16 bytes at a time.
static bool rows_aligned(const void *p) { return ((uintptr_t)p & 15) == 0; }

template <class K>
static int launch_rows(K kernel, const RowArgs &a, long long blocks, hipStream_t st) {
    if (blocks >= (1ll << 31)) return -2;
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kRowThreads), 0, st, a);
    return hipGetLastError() == hipSuccess ? 0 : -6;
}

int launch_dispatch(RowArgs &a, int elem_bytes, hipStream_t st) {
    const long long bytes = (long long)a.H * elem_bytes;
    const uintptr_t at = (uintptr_t)a.x | (uintptr_t)a.rows | (uintptr_t)bytes;
    const int V = at % 16 == 0 ? 16 : at % 8 == 0 ? 8 : at % 4 == 0 ? 4 : 2;
    a.pieces = (int)(bytes / V);
    const long long blocks = (long long)a.T * ((a.pieces + kRowThreads - 1) / kRowThreads);
    switch (V) {
    case 16: return launch_rows(dispatch_kernel<16>, a, blocks, st);
    case 8: return launch_rows(dispatch_kernel<8>, a, blocks, st);
    case 4: return launch_rows(dispatch_kernel<4>, a, blocks, st);
    default: return launch_rows(dispatch_kernel<2>, a, blocks, st);
    }
}

template <int V>
static int combine_typed(const RowArgs &a, bool rb, bool yb, hipStream_t st) {
    const long long blocks = (long long)a.T * ((a.pieces + kRowThreads - 1) / kRowThreads);
    if (rb) return yb ? launch_rows(combine_kernel<V, true, true>, a, blocks, st) : launch_rows(combine_kernel<V, true, false>, a, blocks, st);
    return yb ? launch_rows(combine_kernel<V, false, true>, a, blocks, st) : launch_rows(combine_kernel<V, false, false>, a, blocks, st);
}

int launch_combine(RowArgs &a, bool rows_bf16, bool y_bf16, hipStream_t st) {
    const bool wide = a.H % 8 == 0 && rows_aligned(a.rows) && rows_aligned(a.y);
    a.pieces = wide ? a.H / 8 : a.H;
    return wide ? combine_typed<8>(a, rows_bf16, y_bf16, st) : combine_typed<1>(a, rows_bf16, y_bf16, st);
}

template <int V>
static int backward_typed(const RowArgs &a, bool db, bool rb, hipStream_t st) {
    const long long blocks = (long long)a.T * ((a.k + kDots - 1) / kDots);
    if (db) return rb ? launch_rows(combine_backward_kernel<V, true, true>, a, blocks, st) : launch_rows(combine_backward_kernel<V, true, false>, a, blocks, st);
    return rb ? launch_rows(combine_backward_kernel<V, false, true>, a, blocks, st) : launch_rows(combine_backward_kernel<V, false, false>, a, blocks, st);
}

int launch_combine_backward(RowArgs &a, bool dy_bf16, bool rows_bf16, hipStream_t st) {
    const bool wide = a.H % 8 == 0 && rows_aligned(a.x) && rows_aligned(a.rows) && rows_aligned(a.y);
    a.pieces = wide ? a.H / 8 : a.H;
    return wide ? backward_typed<8>(a, dy_bf16, rows_bf16, st) : backward_typed<1>(a, dy_bf16, rows_bf16, st);
}

}  // namespace kxw4
