// The cache in 4 bits (include/orth_hip.h, orth_hip_int4_cache_t): its layout
// as the kernels see it, and their launchers, whose arguments
// orth_serve4.hip has validated.
#pragma once

#include <type_traits>

#include "orth_serve.h"

namespace orth {

hipError_t launch_cache_append4(const orth_hip_int4_cache_t &c, const orth_hip_append_t &a, int32_t dtype, int cus,
                                hipStream_t stream);
hipError_t launch_cache_read4(const orth_hip_int4_cache_t &c, const orth_hip_read_t &r, int32_t dtype, int cus,
                              hipStream_t stream);

// (`groups`: the counters that a call takes)
int64_t attention4_workspace_bytes(const orth_hip_int4_cache_t &c, const orth_hip_attend_t &a, int cus, int64_t *groups);
hipError_t launch_paged_attention4(const orth_hip_int4_cache_t &c, const orth_hip_attend_t &a, int32_t dtype, int cus,
                                   void *work, uint32_t *counters, hipStream_t stream);

// f(unit, steps) with a cache's W bytes of a unit and its groups of 32 GS
// elements (GS = W: the whole vector) as integral constants.
template <int N>
using Int = std::integral_constant<int, N>;
template <class F>
hipError_t by_int4_layout(const orth_hip_int4_cache_t &c, F &&f) {
    const int D = c.head_dim, gs = c.group_size / 32;
    const bool whole = c.group_size == D;
    if (D <= 64) return whole ? f(Int<2>(), Int<2>()) : f(Int<2>(), Int<1>());
    if (D <= 96) return whole ? f(Int<3>(), Int<3>()) : f(Int<3>(), Int<1>());
    if (D <= 128) return whole ? f(Int<4>(), Int<4>()) : gs == 2 ? f(Int<4>(), Int<2>()) : f(Int<4>(), Int<1>());
    return whole ? f(Int<8>(), Int<8>()) : gs == 4 ? f(Int<8>(), Int<4>()) : gs == 2 ? f(Int<8>(), Int<2>()) : f(Int<8>(), Int<1>());
}

}  // namespace orth
