// The recording launchers over a cache in 4 bits, beside those of
// threads_stubs.hip.
#include "orth_serve4.h"
#include "threads.h"

namespace threads {
void launch(hipStream_t stream, void *work);
}

namespace orth {
hipError_t launch_cache_append4(const orth_hip_int4_cache_t &, const orth_hip_append_t &, int32_t, int, hipStream_t) { return hipSuccess; }
hipError_t launch_cache_read4(const orth_hip_int4_cache_t &, const orth_hip_read_t &, int32_t, int, hipStream_t) { return hipSuccess; }
int64_t attention4_workspace_bytes(const orth_hip_int4_cache_t &, const orth_hip_attend_t &, int, int64_t *groups) {
    *groups = 5;
    return 4096;
}
hipError_t launch_paged_attention4(const orth_hip_int4_cache_t &, const orth_hip_attend_t &, int32_t, int, void *work, uint32_t *,
                                   hipStream_t stream) {
    threads::launch(stream, work);
    return hipSuccess;
}
}  // namespace orth
