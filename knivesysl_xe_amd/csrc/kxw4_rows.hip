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
#include "kxw4_groups.hpp"
#include "kxw4_internal.hpp"

#include <algorithm>

namespace kxw4 {

// ---- the plan --------------------------------------------------------------

constexpr int kPlanWaves = 16, kPlanThreads = 64 * kPlanWaves;       // at most
constexpr int kPlanAhead = 8;                                // keys of a lane requested together (one in plans of up to 1,024)
constexpr int kPlanOne = kPlanThreads * kPlanAhead;          // slots of a plan in one block

// The keys of the AH 64-slot pieces from slot s0 < end on: a slot's
// group, `groups` for none, -1 past the end. (64-bit ids are compared before
// they are narrowed.)
template <class Id, int AH>
__device__ __forceinline__ void plan_keys_of(const Id *ids, int groups, int s0, int end, int lane, int (&key)[AH]) {
    Id v[AH];
#pragma unroll
    for (int i = 0; i < AH; ++i) v[i] = ids[min(s0 + 64 * i + lane, end - 1)];
#pragma unroll
    for (int i = 0; i < AH; ++i)
        key[i] = s0 + 64 * i + lane >= end ? -1 : v[i] < 0 || v[i] >= groups ? groups : (int)v[i];
}

template <int AH>
__device__ __forceinline__ void plan_keys(const RouteArgs &a, int s0, int end, int lane, int (&key)[AH]) {
    if (s0 >= end) {
#pragma unroll
        for (int i = 0; i < AH; ++i) key[i] = -1;
    } else if (a.ids64) {
        plan_keys_of(static_cast<const long long *>(a.ids), a.groups, s0, end, lane, key);
    } else {
        plan_keys_of(static_cast<const int *>(a.ids), a.groups, s0, end, lane, key);
    }
}

// Counts of the keys in [b0, b1), by wave: wave w takes the w-th of the block's
// consecutive runs of `per` slots. cnt: [waves][groups + 1], cleared here; key:
// the wave's last piece of its run.
template <int AH>
__device__ __forceinline__ void plan_count(const RouteArgs &a, int b0, int b1, int per, int *cnt, int (&key)[AH]) {
    const int G1 = a.groups + 1, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int w0 = b0 + wave * per, w1 = min(b1, w0 + per);
    plan_keys(a, w0, w1, lane, key);
    for (int i = tid; i < (int)(blockDim.x / 64) * G1; i += blockDim.x) cnt[i] = 0;
    __syncthreads();
    for (int s0 = w0;;) {
#pragma unroll
        for (int i = 0; i < AH; ++i) {
            if (s0 + 64 * i >= w1) break;
            if (key[i] >= 0) atomicAdd(&cnt[wave * G1 + key[i]], 1);
        }
        s0 += 64 * AH;
        if (s0 >= w1) break;
        plan_keys(a, s0, w1, lane, key);
    }
    __syncthreads();
}

// Large plans, first launch: hist[block][key].
__global__ __launch_bounds__(kPlanThreads) void plan_hist_kernel(const RouteArgs a) {
    extern __shared__ int cnt[];
    const int G1 = a.groups + 1, b0 = blockIdx.x * a.per_block, b1 = min(a.N, b0 + a.per_block);
    int key[kPlanAhead];
    plan_count(a, b0, b1, a.per_block / kPlanWaves, cnt, key);
    for (int g = threadIdx.x; g < G1; g += kPlanThreads) {
        int sum = 0;
#pragma unroll
        for (int w = 0; w < kPlanWaves; ++w) sum += cnt[w * G1 + g];     // (kPlanWaves in a block of these)
        a.hist[(size_t)blockIdx.x * G1 + g] = sum;
    }
}

// The plan (one block), or the last launch of a large one: each block counts
// its own run of slots again, adds up the blocks before it, and places its
// slots. Within a wave the slots of one key find their rank by comparing keys
// bit by bit over the lanes, so the sort is stable and no order of atomics
// shows. What bounds it is the chain of round trips to memory and LDS (a lane's
// keys and a key's block counts are requested eight at a time) and, in one block
// of many slots, the ranks' VALU work on one CU (graph replays, 64 groups: 64
// slots 3.7 us, 1,024 4.4, 8,192 9.8, 32,768 in two launches 9.5; `order` staged in
// LDS and ranks kept from the count gained nothing).
template <int AH>
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(const RouteArgs a) {
    extern __shared__ int cnt[];                             // [waves][groups + 1], then [groups + 1] totals
    const int G = a.groups, G1 = G + 1, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int waves = blockDim.x / 64;
    int *tot = cnt + waves * G1;
    const int b0 = blockIdx.x * a.per_block, b1 = min(a.N, b0 + a.per_block), per = a.per_block / waves;
    int key[AH];
    plan_count(a, b0, b1, per, cnt, key);
    // cnt becomes each wave's first place within its key's slots, tot the
    // key's slots over all blocks
    const int nb = gridDim.x;
    for (int g = tid; g < G1; g += blockDim.x) {
        int before = 0, all = 0;
        for (int q = 0; q < nb && nb > 1; q += 8) {
            int h[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] = q + i < nb ? a.hist[(size_t)(q + i) * G1 + g] : 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                before += q + i < (int)blockIdx.x ? h[i] : 0;
                all += h[i];
            }
        }
        int c[kPlanWaves];
#pragma unroll
        for (int w = 0; w < kPlanWaves; ++w) c[w] = w < waves ? cnt[w * G1 + g] : 0;
#pragma unroll
        for (int w = 0; w < kPlanWaves; ++w) {
            if (w < waves) cnt[w * G1 + g] = before;
            before += c[w];
        }
        tot[g] = nb > 1 ? all : before;
    }
    __syncthreads();
    // exclusive scan of the totals: lane l takes a run of keys
    if (wave == 0) {
        const int run = (G1 + 63) / 64, g0 = min(lane * run, G1), g1 = min(g0 + run, G1);
        int sum = 0;
        for (int g = g0; g < g1; ++g) sum += tot[g];
        const int inc = wave_scan(sum);
        int at = inc - sum;
        for (int g = g0; g < g1; ++g) {
            const int c = tot[g];
            tot[g] = at;
            if (blockIdx.x == 0) a.offsets[g] = at;          // (offsets[groups]: where those without a group begin)
            at += c;
        }
    }
    __syncthreads();
    const int bits = 32 - __builtin_clz(G);                  // (keys run to G itself)
    volatile int *mine = cnt + wave * G1;
    const int w0 = b0 + wave * per, w1 = min(b1, w0 + per);
    for (int s0 = w0; s0 < w1; s0 += 64 * AH) {
        if (per > 64 * AH) plan_keys(a, s0, w1, lane, key);      // (a run of one piece still holds its keys)
#pragma unroll
        for (int i = 0; i < AH; ++i) {
            if (s0 + 64 * i >= w1) break;
            const int s = s0 + 64 * i + lane, kk = key[i];
            const bool on = kk >= 0;
            // (lanes with this lane's key: for each bit those that agree with
            // it, the bit spread over a word)
            const unsigned long long all = __ballot(on);
            uint32_t lo = (uint32_t)all, hi = (uint32_t)(all >> 32);
            for (int b = 0; b < bits; ++b) {
                const uint32_t bit = (uint32_t)((int32_t)((uint32_t)kk << (31 - b)) >> 31);
                const unsigned long long one = __ballot(bit);
                lo &= ~((uint32_t)one ^ bit);
                hi &= ~((uint32_t)(one >> 32) ^ bit);
            }
            const int below = __builtin_amdgcn_mbcnt_hi(hi, __builtin_amdgcn_mbcnt_lo(lo, 0));
            if (on) {
                const int place = tot[kk] + mine[kk] + below;
                a.order[place] = s;
                a.position[s] = kk < G ? place : -1;
            }
            // (the wave's reads above come before this write: LDS accesses of
            // one wave complete in order)
            __builtin_amdgcn_wave_barrier();
            if (on && below == 0) mine[kk] = mine[kk] + __popc(lo) + __popc(hi);
            __builtin_amdgcn_wave_barrier();
        }
    }
}

// Slots per block: one block up to kPlanOne, past which the scattered writes
// of `order` by one CU cost more than a second launch; else blocks of 2,048 up
// to 256 of them, then larger ones. A small plan's block has a wave for each
// 64 slots, and for each 64 groups (64 slots of 1,024 groups: one wave 13.3 us,
// sixteen 6.4; of 256 6.0 / 4.3).
static int plan_round(long long v, int to) { return (int)((v + to - 1) / to * to); }
int route_blocks_of(int N, int *per_block) {
    if (N <= kPlanOne) {
        *per_block = std::max(64, plan_round(N, N < kPlanThreads ? 64 : kPlanThreads));
        return 1;
    }
    *per_block = std::max(2 * kPlanThreads, plan_round((N + 255) / 256, kPlanThreads));
    return (N + *per_block - 1) / *per_block;
}

int launch_route(RouteArgs &a, hipStream_t st) {
    const int nb = route_blocks_of(a.N, &a.per_block), G1 = a.groups + 1;
    const int waves = std::min(std::max(a.per_block, plan_round(G1, 64)) / 64, kPlanWaves);
    if (a.per_block < 64 * waves) a.per_block = 64 * waves;  // (one block: the later waves' runs are empty)
    const size_t lds = (size_t)(waves + 1) * G1 * sizeof(int);            // (at most 69.7 KB: 1,024 groups)
    static bool attr[64] = {};                               // (the attribute is per device)
    int dev = 0;
    if (lds > 64 * 1024 && (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64)) return -6;
    if (lds > 64 * 1024 && !attr[dev]) {
        for (const void *k : {reinterpret_cast<const void *>(plan_hist_kernel), reinterpret_cast<const void *>(plan_kernel<1>),
                              reinterpret_cast<const void *>(plan_kernel<kPlanAhead>)})
            if (hipFuncSetAttribute(k, hipFuncAttributeMaxDynamicSharedMemorySize, 80 * 1024) != hipSuccess) return -6;
        attr[dev] = true;
    }
    if (nb > 1) {
        if (!a.hist) return -1;
        hipLaunchKernelGGL(plan_hist_kernel, dim3(nb), dim3(kPlanThreads), lds, st, a);
    }
    hipLaunchKernelGGL(a.N <= kPlanThreads ? plan_kernel<1> : plan_kernel<kPlanAhead>, dim3(nb), dim3(64 * waves), lds, st, a);
    return hipGetLastError() == hipSuccess ? 0 : -6;
}

// ---- rows ------------------------------------------------------------------
//
// A thread owns a piece of a row: the 16 bytes that V elements of the rows'
// type take. Rows of any length and alignment take the same instructions: the
// hardware reads and writes 16 bytes at any address of whole elements, and the
// last piece of a row ends at its end, over the piece before it (two threads
// write the same values there). Only rows shorter than a piece go element by
// element. H = 2049, float32, 8,000 rows: dispatch 27 -> 19 us, combine 27 ->
// 19 (4 bytes a thread before).

constexpr int kRowThreads = 256;

// V elements at `at`; SHORT: of a row that may have only n of them.
template <int V, bool BF, bool SHORT>
struct Piece {
    static constexpr int BYTES = V * (BF ? 2 : 4);
    static constexpr int WORDS = BYTES / 4;
    typedef uint32_t Words __attribute__((ext_vector_type(WORDS), aligned(BF ? 2 : 4)));
    Words w;

    __device__ __forceinline__ void load(const void *base, size_t at, int n) {
        const uint8_t *p = static_cast<const uint8_t *>(base) + at * (BF ? 2 : 4);
        if (!SHORT || n >= V) {
            w = __builtin_nontemporal_load(reinterpret_cast<const Words *>(p));
        } else {
#pragma unroll
            for (int i = 0; i < WORDS; ++i) w[i] = 0;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                if (i >= n) continue;
                if constexpr (BF) w[i / 2] |= (uint32_t) reinterpret_cast<const uint16_t *>(p)[i] << 16 * (i & 1);
                else w[i] = reinterpret_cast<const uint32_t *>(p)[i];
            }
        }
    }
    __device__ __forceinline__ void store(void *base, size_t at, int n, int past) const {
        uint8_t *p = static_cast<uint8_t *>(base) + at * (BF ? 2 : 4);
        if (!SHORT || n >= V) {
            if (past) {
                // (the empty statements keep the compiler from making one
                // plain store of the two)
                asm volatile("");
                __builtin_nontemporal_store(w, reinterpret_cast<Words *>(p));
                asm volatile("");
            } else {
                *reinterpret_cast<Words *>(p) = w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                if (i >= n) continue;
                if constexpr (BF) reinterpret_cast<uint16_t *>(p)[i] = (uint16_t)(w[i / 2] >> 16 * (i & 1));
                else reinterpret_cast<uint32_t *>(p)[i] = w[i];
            }
        }
    }
    __device__ __forceinline__ float get(int i) const {
        if constexpr (BF) return __uint_as_float(i & 1 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
        else return __uint_as_float(w[i]);
    }
    __device__ __forceinline__ void set(const float (&v)[V]) {       // one rounding each
#pragma unroll
        for (int i = 0; i < WORDS; ++i) {
            if constexpr (BF) w[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
            else w[i] = __float_as_uint(v[i]);
        }
    }
};

// The thread's token and piece. WIDE: a row takes `a.chunks` blocks, so the
// token is the block's and its plan entries come through scalar loads; else a
// block takes `a.per` tokens of `a.lanes` threads each.
struct RowAt {
    int t, c;
};
template <bool WIDE>
__device__ __forceinline__ RowAt row_at(const RowArgs &a) {
    const int block = blockIdx.x;
    if constexpr (WIDE) {
        const int t = block / a.chunks;
        return {a.t0 + t, (block - t * a.chunks) * a.lanes + (int)threadIdx.x};
    } else {
        const int sub = threadIdx.x / a.lanes;
        return {a.t0 + block * a.per + sub, (int)threadIdx.x - sub * a.lanes};
    }
}
template <int V, bool SHORT>
__device__ __forceinline__ int piece_at(int H, int c) { return SHORT && H < V ? 0 : min(c * V, H - V); }

// rows[position[t, j]] = x[t]: a thread reads one piece of a token's row and
// writes it to each of the token's places, so x is read once. Bound by the
// writes.
template <bool BF, bool WIDE>
__global__ __launch_bounds__(512) void dispatch_kernel(const RowArgs a) {
    constexpr int V = BF ? 8 : 4;
    const RowAt r = row_at<WIDE>(a);
    if (r.t >= a.T || r.c >= a.pieces) return;
    const int n = min(a.H, V), at = piece_at<V, !WIDE>(a.H, r.c);
    Piece<V, BF, !WIDE> v;
    v.load(a.x, (size_t)r.t * a.H + at, n);
    const int *pos = a.position + (size_t)r.t * a.k;
    for (int j0 = 0; j0 < a.k; j0 += 4) {
        int p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = j0 + i < a.k ? pos[j0 + i] : -1;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (p[i] >= 0) v.store(a.rows, (size_t)p[i] * a.H + at, n, a.past);
    }
}

// y[t] = sum_j w[t, j] rows[position[t, j]] (w 1 where none is given): AH
// choices' pieces are requested before the first is added, those of slots
// without a group from row 0 (a load under a branch waits for the one before
// it). Bound by the reads.
template <bool RB, bool YB, bool WIDE, int AH>
__global__ __launch_bounds__(512) void combine_kernel(const RowArgs a) {
    constexpr int V = RB ? 8 : 4;
    const RowAt r = row_at<WIDE>(a);
    if (r.t >= a.T || r.c >= a.pieces) return;
    const int n = min(a.H, V), at = piece_at<V, !WIDE>(a.H, r.c);
    const int *pos = a.position + (size_t)r.t * a.k;
    const float *w = a.weights ? a.weights + (size_t)r.t * a.k : nullptr;
    float acc[V] = {};
    for (int j0 = 0; j0 < a.k; j0 += AH) {
        Piece<V, RB, !WIDE> v[AH];
        float wj[AH];
        int p[AH];
#pragma unroll
        for (int i = 0; i < AH; ++i) p[i] = j0 + i < a.k ? pos[j0 + i] : -1;
#pragma unroll
        for (int i = 0; i < AH; ++i) wj[i] = w && j0 + i < a.k ? w[j0 + i] : 1.0f;
#pragma unroll
        for (int i = 0; i < AH; ++i)
            v[i].load(a.rows, (size_t)max(p[i], 0) * a.H + at, n);
#pragma unroll
        for (int i = 0; i < AH; ++i)
            if (p[i] >= 0)
#pragma unroll
                for (int e = 0; e < V; ++e) acc[e] = __builtin_fmaf(wj[i], v[i].get(e), acc[e]);
    }
    Piece<V, YB, !WIDE> y;
    y.set(acc);
    y.store(a.y, (size_t)r.t * a.H + at, n, a.past);
}

// drows[position[t, j]] = w[t, j] dy[t], dw[t, j] = <dy[t], rows[position[t,
// j]]>: one block per token and run of kDots choices, which reads dy once for
// all of them. Bound by the rows read and written.
constexpr int kDots = 4;
template <bool DB, bool RB, bool SHORT>
__global__ __launch_bounds__(kRowThreads) void combine_backward_kernel(const RowArgs a) {
    constexpr int V = RB ? 8 : 4;
    __shared__ float part[kRowThreads / 64][kDots];
    const int runs = (a.k + kDots - 1) / kDots;
    const int run = blockIdx.x / runs, t = a.t0 + run, j0 = (blockIdx.x - run * runs) * kDots;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int p[kDots];
    float w[kDots], dot[kDots] = {};
#pragma unroll
    for (int i = 0; i < kDots; ++i) {
        p[i] = j0 + i < a.k ? a.position[(size_t)t * a.k + j0 + i] : -1;
        w[i] = j0 + i < a.k ? a.weights[(size_t)t * a.k + j0 + i] : 0.0f;
    }
    for (int c = tid; c < a.pieces; c += kRowThreads) {
        const int n = min(a.H, V), at = piece_at<V, SHORT>(a.H, c), seen = c * V - at;
        Piece<V, DB, SHORT> dy;
        Piece<V, RB, SHORT> v[kDots];
        dy.load(a.x, (size_t)t * a.H + at, n);
#pragma unroll
        for (int i = 0; i < kDots; ++i)
            v[i].load(a.rows, (size_t)max(p[i], 0) * a.H + at, n);
#pragma unroll
        for (int i = 0; i < kDots; ++i) {
            if (p[i] < 0) continue;
            float d[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float sum = __builtin_fmaf(dy.get(e), v[i].get(e), dot[i]);
                dot[i] = e >= seen ? sum : dot[i];
                d[e] = w[i] * dy.get(e);
            }
            Piece<V, RB, SHORT> o;
            o.set(d);
            o.store(a.y, (size_t)p[i] * a.H + at, n, a.past);
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

// One launch for as many tokens as its grid holds (grid_limit); a block takes
// `tokens` of them, or a token `blocks` blocks. (16.8 million tokens at 256
// threads each.)
typedef void (*RowKernel)(const RowArgs);
static int launch_tokens(RowKernel k, RowArgs &a, int tokens, int blocks, int threads, hipStream_t st) {
    const long long most = grid_limit(threads) / blocks * tokens;
    if (most == 0) return -2;
    for (long long t0 = 0; t0 < a.T; t0 += most) {
        a.t0 = (int)t0;
        const long long grid = (std::min(most, a.T - t0) + tokens - 1) / tokens * blocks;
        hipLaunchKernelGGL(k, dim3((unsigned)grid), dim3(threads), 0, st, a);
        if (hipGetLastError() != hipSuccess) return -6;
    }
    return 0;
}

// Threads and blocks of a row kernel: rows of up to 32 pieces share a
// 256-thread block, longer ones take a block each, or several of up to 512
// threads.
static int launch_rows(RowKernel wide, RowKernel narrow, RowArgs &a, hipStream_t st) {
    if (a.pieces <= 32) {
        a.lanes = 1;
        while (a.lanes < a.pieces) a.lanes *= 2;
        a.per = kRowThreads / a.lanes;
        a.chunks = 1;
        return launch_tokens(narrow, a, a.per, 1, kRowThreads, st);
    }
    a.per = 1;
    a.chunks = (a.pieces + 511) / 512;
    a.lanes = ((a.pieces + a.chunks - 1) / a.chunks + 63) / 64 * 64;
    return launch_tokens(wide, a, 1, a.chunks, a.lanes, st);
}

// Every row is read once, so the loads are marked as not to be kept. The
// stores are where they write more than 64 MiB, a quarter of the last-level
// cache, which would push out more than the next kernel finds there (us with /
// without: a dispatch and a combine of 32,768 rows of 10 KB 148 / 157, the
// gradients of 8,186 such rows 66.2 / 67.9, of 8,192 rows of 8 KB 40.7 / 37.5).
static int past_cache(long long bytes) { return bytes > (64ll << 20); }

static int pieces_of(int H, bool bf16) { return bf16 ? (H + 7) / 8 : (H + 3) / 4; }

int launch_dispatch(RowArgs &a, bool bf16, hipStream_t st) {
    a.pieces = pieces_of(a.H, bf16);
    a.past = past_cache((long long)a.T * a.k * a.H * (bf16 ? 2 : 4));
    return bf16 ? launch_rows(dispatch_kernel<true, true>, dispatch_kernel<true, false>, a, st)
                : launch_rows(dispatch_kernel<false, true>, dispatch_kernel<false, false>, a, st);
}

template <bool RB, bool YB>
static int combine_typed(RowArgs &a, hipStream_t st) {
    const RowKernel narrow = combine_kernel<RB, YB, false, 2>;
    if (a.k == 1) return launch_rows(combine_kernel<RB, YB, true, 1>, narrow, a, st);
    if (a.k == 2) return launch_rows(combine_kernel<RB, YB, true, 2>, narrow, a, st);
    if (a.k <= 4) return launch_rows(combine_kernel<RB, YB, true, 4>, narrow, a, st);
    return launch_rows(combine_kernel<RB, YB, true, 8>, narrow, a, st);
}

int launch_combine(RowArgs &a, bool rows_bf16, bool y_bf16, hipStream_t st) {
    a.pieces = pieces_of(a.H, rows_bf16);
    a.past = past_cache((long long)a.T * a.H * (y_bf16 ? 2 : 4));
    if (rows_bf16) return y_bf16 ? combine_typed<true, true>(a, st) : combine_typed<true, false>(a, st);
    return y_bf16 ? combine_typed<false, true>(a, st) : combine_typed<false, false>(a, st);
}

template <bool SHORT>
static RowKernel backward_of(bool dy_bf16, bool rows_bf16) {
    if (dy_bf16) return rows_bf16 ? combine_backward_kernel<true, true, SHORT> : combine_backward_kernel<true, false, SHORT>;
    return rows_bf16 ? combine_backward_kernel<false, true, SHORT> : combine_backward_kernel<false, false, SHORT>;
}

int launch_combine_backward(RowArgs &a, bool dy_bf16, bool rows_bf16, hipStream_t st) {
    a.pieces = pieces_of(a.H, rows_bf16);
    a.past = past_cache((long long)a.T * a.k * a.H * (rows_bf16 ? 2 : 4));
    const RowKernel k = a.pieces == 1 ? backward_of<true>(dy_bf16, rows_bf16) : backward_of<false>(dy_bf16, rows_bf16);
    return launch_tokens(k, a, 1, (a.k + kDots - 1) / kDots, kRowThreads, st);
}

}  // namespace kxw4
