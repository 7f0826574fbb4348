// Host-only stand-ins for the launchers over a cache in 4 bits, so that their
// C entry points (orth_serve4.hip) can be built under AddressSanitizer and
// UBSan on a machine without a GPU (tests/test_int4_sanitizers.py).
#include "orth_serve4.h"

namespace orth {
hipError_t launch_cache_append4(const orth_hip_int4_cache_t &, const orth_hip_append_t &, int32_t, int, hipStream_t) {
    return hipErrorInvalidValue;
}
hipError_t launch_cache_read4(const orth_hip_int4_cache_t &, const orth_hip_read_t &, int32_t, int, hipStream_t) {
    return hipErrorInvalidValue;
}
int64_t attention4_workspace_bytes(const orth_hip_int4_cache_t &, const orth_hip_attend_t &, int, int64_t *groups) {
    *groups = 1;
    return 64;
}
hipError_t launch_paged_attention4(const orth_hip_int4_cache_t &, const orth_hip_attend_t &, int32_t, int, void *, uint32_t *,
                                   hipStream_t) {
    return hipErrorInvalidValue;
}
}  // namespace orth
