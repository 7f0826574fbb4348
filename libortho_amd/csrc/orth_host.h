// Host-side services of orth_capi.hip for the entry points in other files:
// the per-thread error message, the device check and the per-stream
// workspace (under capture: the memory of captured calls).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <mutex>

namespace orth {

int host_fail(int status, const char *message);
int host_fail_hip(hipError_t e, const char *what);
void host_begin();  // clears the thread's error message
int host_device(int *dev, int *cus);
// Both take the stream's workspace into `held`, which the caller keeps until
// the call's last launch: other threads' calls on the stream wait there.
int host_workspace(int dev, hipStream_t stream, int64_t bytes, void **p, std::unique_lock<std::mutex> *held);
// Counters that are zero when the call's kernels begin: the stream's own,
// which each kernel that counts in them leaves at zero, or, under capture,
// those of all captured calls, cleared by a launch in front (a graph's replays
// find whatever other graphs left there).
int host_counters(int dev, hipStream_t stream, int64_t count, uint32_t **p, std::unique_lock<std::mutex> *held);

}  // namespace orth
