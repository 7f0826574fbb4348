// Host-only stand-ins for the serving operators' launchers, so that their C
// entry points (orth_serve.hip) can be built under AddressSanitizer and UBSan
// on a machine without a GPU (tests/test_serve_sanitizers.py).
#include "orth_serve.h"

namespace orth {
hipError_t launch_page_step(const orth_hip_step_t &, hipStream_t) { return hipErrorInvalidValue; }
hipError_t launch_cache_append(const orth_hip_cache_t &, const orth_hip_append_t &, int, hipStream_t) { return hipErrorInvalidValue; }
int64_t attention_workspace_bytes(const orth_hip_cache_t &, const orth_hip_attend_t &, int, int64_t *groups) {
    *groups = 1;
    return 64;
}
hipError_t launch_paged_attention(const orth_hip_cache_t &, const orth_hip_attend_t &, int, void *, uint32_t *, hipStream_t) {
    return hipErrorInvalidValue;
}
int64_t adapter_workspace_bytes(const orth_hip_adapter_t &, int) { return 64; }
hipError_t launch_adapter_add(const orth_hip_adapter_t &, int, void *, hipStream_t) { return hipErrorInvalidValue; }
}  // namespace orth
