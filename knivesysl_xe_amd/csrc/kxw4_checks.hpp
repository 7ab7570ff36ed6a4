// kxw4_checks.hpp — argument checks that the entry points share.
#pragma once

#include "../../include/kxw4.h"

#include <hip/hip_runtime.h>

namespace kxw4 {

inline hipStream_t as_stream(void *s) { return reinterpret_cast<hipStream_t>(s); }

inline bool valid_dtype(int d) { return d == KXW4_F32 || d == KXW4_BF16; }
inline int elem_bytes(int dtype) { return dtype == KXW4_BF16 ? 2 : 4; }
inline bool aligned(const void *p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

constexpr int kMaxGroups = 1024;
constexpr long long kMaxSlots = 1ll << 30;

inline bool valid_plan(int T, int k, int groups) {
    return T >= 0 && k > 0 && groups > 0 && groups <= kMaxGroups && (long long)T * k <= kMaxSlots;
}

// A plan that kxw4_route_rows filled. (With T = 0 only its sizes count.)
inline int check_route(const kxw4_route_t *r) {
    if (!r) return KXW4_EARG;
    if (!valid_plan(r->T, r->k, r->groups)) return KXW4_ESHAPE;
    if (r->T > 0 && (!r->offsets || !r->order || !r->position)) return KXW4_EPREP;
    return KXW4_OK;
}

}  // namespace kxw4
