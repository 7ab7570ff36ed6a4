// kxw4_f8_abi.hip — entry points of the 8-bit floating tier and of the weights'
// gradient (include/kxw4.h): argument checks and the choice of kernel.
#include "kxw4_checks.hpp"
#include "kxw4_f8.hpp"
#include "kxw4_f8_route.hpp"

using namespace kxw4;

namespace {

constexpr int kMaxDim = 1 << 22;

bool valid_f8(int groups, int M, int K) {
    return groups > 0 && groups <= kMaxGroups && M > 0 && K > 0 && M % 16 == 0 && K % 16 == 0 && M <= kMaxDim && K <= kMaxDim;
}

int check_weight_f8(const kxw4_weight_f8_t *w) {
    if (!w || !w->codes || !w->scales) return KXW4_EARG;
    if (!valid_f8(w->groups, w->M, w->K)) return KXW4_ESHAPE;
    if (!aligned(w->codes, 16) || !aligned(w->scales, 4)) return KXW4_EARG;
    return KXW4_OK;
}

// What both products ask of their weights, outputs and activation; *rows: the
// activation's.
int check_product(const kxw4_weight_f8_t *const *ws, void *const *ys, int count, const kxw4_act_f8_t *a, int groups,
                  long long rows, int y_dtype) {
    if (!ws || !ys || count <= 0 || count > kMaxWeights || !a) return KXW4_EARG;
    for (int i = 0; i < count; ++i) {
        const int rc = check_weight_f8(ws[i]);
        if (rc) return rc;
        if (ws[i]->groups != groups || ws[i]->K != ws[0]->K) return KXW4_ESHAPE;
    }
    if (!valid_dtype(y_dtype) || a->T != rows || rows < 0 || rows > kMaxSlots || a->K != ws[0]->K) return KXW4_ESHAPE;
    if (!a->q && !valid_dtype(a->x_dtype)) return KXW4_ESHAPE;
    if (rows == 0) return KXW4_OK;
    if (a->q ? !a->scale : !a->x) return KXW4_EPREP;
    if (!aligned(a->q, 16) || !aligned(a->scale, 4) || !aligned(a->x, 16)) return KXW4_EARG;
    for (int i = 0; i < count; ++i) {
        if (!ys[i] || !aligned(ys[i], 16) || ys[i] == a->x || ys[i] == a->q) return KXW4_EARG;
        for (int j = 0; j < i; ++j)
            if (ys[i] == ys[j]) return KXW4_EARG;
    }
    return KXW4_OK;
}

size_t codes_bytes(long long rows, int K) { return (size_t)rows * f8_blocks(K) * kF8Block; }
// (multiples of 16 bytes)
size_t act_bytes(long long rows, int K) {
    return codes_bytes(rows, K) + ((size_t)rows * f8_blocks(K) * sizeof(float) + 15) / 16 * 16;
}

struct Rows {                                                // the rows sorted by group, or groups 0
    const int *offsets, *order;
    int N, groups, k;
};

F8GemmArgs gemm_args(const kxw4_weight_f8_t *const *ws, void *const *ys, int count, const kxw4_act_f8_t *a, int y_dtype,
                     const Rows &r) {
    F8GemmArgs x{};
    for (int i = 0; i < count; ++i) x.w[i] = F8GemmWeight{ws[i]->codes, ws[i]->scales, ys ? ys[i] : nullptr, ws[i]->M, 0, 0};
    x.count = count;
    x.q = a->q;
    x.sx = a->scale;
    x.rows = a->T;
    x.K = a->K;
    x.KB = f8_blocks(a->K);
    x.y_bf16 = y_dtype == KXW4_BF16 ? 1 : 0;
    x.offsets = r.offsets;
    x.order = r.order;
    x.N = r.N;
    x.groups = r.groups;
    x.k = r.k;
    return x;
}

// The kernel of a product: rows of a stream tile or 0, and whether values are
// quantized by a launch of their own.
struct Way {
    int rows;
    bool quantizes;
};

Way way_of(const F8GemmArgs &x, const kxw4_act_f8_t *a) {
    F8Sizes s{device_cus(), x.groups ? x.N : x.rows, x.KB, x.count, {}, x.groups, x.y_bf16 != 0};
    for (int i = 0; i < x.count; ++i) s.M[i] = x.w[i].M;
    Way w{f8_stream_rows(s), false};
    // (the stream kernel takes values with 32-bit offsets)
    if (!a->q)
        w.quantizes = !(w.rows && (w.rows == 16 ? f8_stream_quantizes(s) : f8_stream32_quantizes(s, elem_bytes(a->x_dtype))) &&
                        (long long)a->T * a->K * elem_bytes(a->x_dtype) < (1ll << 31));
    return w;
}

// Scratch of a product: the codes and scales of values, then the parts of
// split sums.
size_t workspace_of(const kxw4_weight_f8_t *const *ws, int count, const kxw4_act_f8_t *a, int y_dtype, const Rows &r) {
    if (!ws || count <= 0 || count > kMaxWeights || !a || a->T <= 0 || !valid_f8(1, 16, a->K) || !valid_dtype(y_dtype)) return 0;
    for (int i = 0; i < count; ++i)
        if (!ws[i] || !valid_f8(1, ws[i]->M, a->K)) return 0;
    const F8GemmArgs x = gemm_args(ws, nullptr, count, a, y_dtype, r);
    const Way way = way_of(x, a);
    return (way.quantizes ? act_bytes(a->T, a->K) : 0) + (way.rows ? 0 : f8_gemm_scratch(x));
}

int product(const kxw4_weight_f8_t *const *ws, void *const *ys, int count, const kxw4_act_f8_t *a, int y_dtype,
            const float *residual, const Rows &r, void *workspace, hipStream_t st) {
    F8GemmArgs x = gemm_args(ws, ys, count, a, y_dtype, r);
    const Way way = way_of(x, a);
    const uint8_t *q = a->q;
    const float *sx = a->scale;
    uint8_t *scratch = static_cast<uint8_t *>(workspace);
    if (way.quantizes) {
        float *scales = reinterpret_cast<float *>(scratch + codes_bytes(a->T, a->K));
        const int rc = launch_f8_quantize(a->x, a->x_dtype == KXW4_BF16, a->T, a->K, scratch, scales, st);
        if (rc) return rc;
        q = scratch;
        sx = scales;
        scratch += act_bytes(a->T, a->K);
    }
    if (way.rows) {
        F8StreamArgs s{};
        for (int i = 0; i < count; ++i) s.w[i] = F8StreamWeight{ws[i]->codes, ws[i]->scales, ys[i], ws[i]->M, 0};
        s.count = count;
        s.q = q;
        s.sx = sx;
        s.x = a->x;
        s.residual = residual;
        s.rows = x.rows;
        s.K = x.K;
        s.KB = x.KB;
        s.y_bf16 = x.y_bf16;
        s.offsets = r.offsets;
        s.order = r.order;
        s.N = r.N;
        s.groups = r.groups;
        s.k = r.k;
        return launch_f8_stream(s, q ? 0 : a->x_dtype == KXW4_BF16 ? 1 : 2, way.rows, st);
    }
    x.q = q;
    x.sx = sx;
    x.residual = residual;
    x.part = reinterpret_cast<float *>(scratch);
    return launch_f8_gemm(x, st);
}

}  // namespace

extern "C" {

size_t kxw4_f8_code_bytes(int groups, int M, int K) {
    return valid_f8(groups, M, K) ? (size_t)groups * M * f8_blocks(K) * kF8Block : 0;
}

int kxw4_pack_weight_f8(const uint8_t *codes, int groups, int M, int K, uint8_t *out_codes, void *stream) {
    if (!codes || !out_codes || codes == out_codes || !aligned(codes, 16) || !aligned(out_codes, 16)) return KXW4_EARG;
    if (!valid_f8(groups, M, K)) return KXW4_ESHAPE;
    return launch_f8_pack(codes, groups, M, K, out_codes, as_stream(stream));
}

int kxw4_unpack_weight_f8(const kxw4_weight_f8_t *w, uint8_t *codes, void *stream) {
    const int rc = check_weight_f8(w);
    if (rc) return rc;
    if (!codes || codes == w->codes || !aligned(codes, 16)) return KXW4_EARG;
    return launch_f8_unpack(w->codes, w->groups, w->M, w->K, codes, as_stream(stream));
}

int kxw4_quantize_weight_f8(const void *w, int dtype, int groups, int M, int K, uint8_t *out_codes, float *out_scales,
                            void *stream) {
    if (!w || !out_codes || !out_scales || !aligned(w, 16) || !aligned(out_codes, 16) || !aligned(out_scales, 4))
        return KXW4_EARG;
    if (!valid_f8(groups, M, K) || !valid_dtype(dtype)) return KXW4_ESHAPE;
    return launch_f8_weight(w, dtype == KXW4_BF16, groups, M, K, out_codes, out_scales, as_stream(stream));
}

int kxw4_transpose_weight_f8(const kxw4_weight_f8_t *w, uint8_t *out_codes, float *out_scales, void *stream) {
    const int rc = check_weight_f8(w);
    if (rc) return rc;
    if (!out_codes || !out_scales || out_codes == w->codes || out_scales == w->scales || !aligned(out_codes, 16) ||
        !aligned(out_scales, 4))
        return KXW4_EARG;
    return launch_f8_transpose(w->codes, w->scales, w->groups, w->M, w->K, out_codes, out_scales, as_stream(stream));
}

int kxw4_quantize_act_f8(const void *x, int x_dtype, int T, int K, uint8_t *q, float *scale, void *stream) {
    if (T < 0 || T > kMaxSlots || !valid_f8(1, 16, K) || !valid_dtype(x_dtype)) return KXW4_ESHAPE;
    if (T == 0) return KXW4_OK;
    if (!x || !q || !scale || x == q || !aligned(x, 16) || !aligned(q, 16) || !aligned(scale, 4)) return KXW4_EARG;
    return launch_f8_quantize(x, x_dtype == KXW4_BF16, T, K, q, scale, as_stream(stream));
}

int kxw4_silu_mul_quant_f8(float *out, const void *gate, const void *up, int dtype, int T, int K, uint8_t *q, float *scale,
                           void *stream) {
    if (T < 0 || T > kMaxSlots || !valid_f8(1, 16, K) || !valid_dtype(dtype)) return KXW4_ESHAPE;
    if (T == 0) return KXW4_OK;
    if (!gate || !up || !q || !scale || gate == q || up == q || !aligned(gate, 16) || !aligned(up, 16) || !aligned(q, 16) ||
        !aligned(scale, 4) || !aligned(out, 16) || (out && (out == gate || out == up)))
        return KXW4_EARG;
    return launch_f8_silu_mul(out, gate, up, dtype == KXW4_BF16, T, K, q, scale, as_stream(stream));
}

size_t kxw4_gemm_f8_workspace(const kxw4_weight_f8_t *const *ws, int count, const kxw4_act_f8_t *a, int y_dtype) {
    return workspace_of(ws, count, a, y_dtype, Rows{});
}

int kxw4_gemm_f8(const kxw4_weight_f8_t *const *ws, void *const *ys, int count, const kxw4_act_f8_t *a, int y_dtype,
                 const float *residual, void *workspace, void *stream) {
    const int rc = check_product(ws, ys, count, a, 1, a ? a->T : 0, y_dtype);
    if (rc) return rc;
    // (an FP32 output may be the residual itself; a BF16 one would overwrite parts of it that are still to be read)
    if (residual && (count != 1 || !aligned(residual, 16) || (y_dtype == KXW4_BF16 && ys[0] == residual))) return KXW4_EARG;
    if (a->T == 0) return KXW4_OK;
    if (!aligned(workspace, 16) || (!workspace && kxw4_gemm_f8_workspace(ws, count, a, y_dtype))) return KXW4_EARG;
    return product(ws, ys, count, a, y_dtype, residual, Rows{}, workspace, as_stream(stream));
}

size_t kxw4_expert_gemm_f8_workspace(const kxw4_weight_f8_t *const *ws, int count, const kxw4_act_f8_t *a,
                                     const kxw4_route_t *route, int sorted_rows, int y_dtype) {
    if (!route || !valid_plan(route->T, route->k, route->groups)) return 0;
    return workspace_of(ws, count, a, y_dtype, Rows{nullptr, nullptr, route->T * route->k, route->groups, route->k});
}

int kxw4_expert_gemm_f8(const kxw4_weight_f8_t *const *ws, void *const *ys, int count, const kxw4_act_f8_t *a,
                        const kxw4_route_t *route, int sorted_rows, int y_dtype, void *workspace, void *stream) {
    int rc = check_route(route);
    if (rc) return rc;
    const long long N = (long long)route->T * route->k, rows = sorted_rows ? N : route->T;
    rc = check_product(ws, ys, count, a, route->groups, rows, y_dtype);
    if (rc) return rc;
    // (32-bit offsets of the rows' codes)
    if (rows * f8_blocks(a->K) * kF8Block >= (1ll << 31)) return KXW4_ESHAPE;
    if (rows == 0) return KXW4_OK;
    if (!aligned(workspace, 16) || (!workspace && kxw4_expert_gemm_f8_workspace(ws, count, a, route, sorted_rows, y_dtype)))
        return KXW4_EARG;
    return product(ws, ys, count, a, y_dtype, nullptr,
                   Rows{route->offsets, sorted_rows ? nullptr : route->order, (int)N, route->groups, route->k}, workspace,
                   as_stream(stream));
}

size_t kxw4_grad_weight_workspace(int N, int groups, int M, int K) {
    return N <= 0 || N > kMaxSlots || !valid_f8(groups, M, K) ? 0 : grad_scratch(N, groups, M, K);
}

int kxw4_grad_weight(const uint16_t *dy, const uint16_t *x, int N, int M, int K, const kxw4_route_t *route, const void *add,
                     void *dw, int dw_dtype, void *workspace, void *stream) {
    if (route) {
        const int rc = check_route(route);
        if (rc) return rc;
        if ((long long)route->T * route->k != N) return KXW4_ESHAPE;
    }
    const int groups = route ? route->groups : 1;
    if (N < 0 || N > kMaxSlots || !valid_f8(groups, M, K) || !valid_dtype(dw_dtype)) return KXW4_ESHAPE;
    if (!dw || !aligned(dw, 16) || !aligned(add, 16)) return KXW4_EARG;
    if (N > 0 && (!dy || !x || !aligned(dy, 16) || !aligned(x, 16) || dw == dy || dw == x)) return KXW4_EARG;
    if (!aligned(workspace, 16) || (!workspace && kxw4_grad_weight_workspace(N, groups, M, K))) return KXW4_EARG;
    GradArgs a{};
    a.dy = dy;
    a.x = x;
    a.add = add;
    a.dw = dw;
    a.part = static_cast<float *>(workspace);
    a.offsets = route && N > 0 ? route->offsets : nullptr;
    a.N = N;
    a.groups = groups;
    a.M = M;
    a.K = K;
    a.dw_bf16 = dw_dtype == KXW4_BF16 ? 1 : 0;
    return launch_grad(a, as_stream(stream));
}

}  // extern "C"
