// Host-only stand-ins for the GPU, for tests/test_serve_threads.py: the HIP
// calls that the C ABI's host side makes (a gfx950 that is not there, memory
// from malloc, a stream that is under capture) and launchers that record
// which of their calls were inside at the same time, and with what memory.
#include <unistd.h>

#include <cstdlib>
#include <cstring>
#include <new>

#include "orth_common.h"
#include "orth_serve.h"
#include "threads.h"

namespace threads {
std::atomic<int> inside[kStreams], overlaps{0}, together{0}, all{0}, kernels{0};
std::atomic<bool> throws{false};
std::mutex mu;
std::map<void *, std::set<void *>> works;  // of each thread's tag

void launch(hipStream_t stream, void *work) {
    if (throws) throw std::bad_alloc();
    const int i = (int)((uintptr_t)stream % kStreams);
    if (inside[i]++ != 0) overlaps++;
    if (all++ != 0) together++;
    {
        std::lock_guard<std::mutex> lk(mu);
        works[tag()].insert(work);
    }
    usleep(1500);  // (between a call's two launches)
    all--;
    inside[i]--;
}

void *tag() {
    thread_local char t;
    return &t;
}
}  // namespace threads

extern "C" {
hipError_t hipGetDevice(int *d) {
    *d = 0;
    return hipSuccess;
}
hipError_t hipGetDeviceProperties(hipDeviceProp_t *p, int) {
    std::memset(p, 0, sizeof(*p));
    std::strcpy(p->gcnArchName, "gfx950");
    p->multiProcessorCount = 256;
    return hipSuccess;
}
hipError_t hipGetSymbolAddress(void **p, const void *) {
    static char memory[64 << 10] __attribute__((aligned(256)));
    *p = memory;
    return hipSuccess;
}
hipError_t hipEventCreateWithFlags(hipEvent_t *e, unsigned) {
    *e = nullptr;
    return hipSuccess;
}
hipError_t hipStreamIsCapturing(hipStream_t s, hipStreamCaptureStatus *c) {
    *c = s == threads::kCapturing ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone;
    return hipSuccess;
}
hipError_t hipMalloc(void **p, size_t n) {
    *p = std::malloc(n);
    return *p ? hipSuccess : hipErrorOutOfMemory;
}
hipError_t hipFree(void *p) {
    std::free(p);
    return hipSuccess;
}
hipError_t hipLaunchKernel(const void *, dim3, dim3, void **, size_t, hipStream_t) {
    threads::kernels++;
    return hipSuccess;
}
hipError_t __hipPushCallConfiguration(dim3, dim3, size_t, hipStream_t) { return hipSuccess; }
hipError_t __hipPopCallConfiguration(dim3 *, dim3 *, size_t *, hipStream_t *) { return hipSuccess; }
hipError_t hipGetLastError() { return hipSuccess; }
hipError_t hipMemsetAsync(void *p, int v, size_t n, hipStream_t) {
    std::memset(p, v, n);
    return hipSuccess;
}
}

namespace orth {
hipError_t launch_page_step(const orth_hip_step_t &, hipStream_t) { return hipSuccess; }
hipError_t launch_cache_append(const orth_hip_cache_t &, const orth_hip_append_t &, int, hipStream_t) { return hipSuccess; }
int64_t attention_workspace_bytes(const orth_hip_cache_t &, const orth_hip_attend_t &, int, int64_t *groups) {
    *groups = 5;
    return 4096;
}
hipError_t launch_paged_attention(const orth_hip_cache_t &, const orth_hip_attend_t &, int, void *work, uint32_t *,
                                  hipStream_t stream) {
    threads::launch(stream, work);
    return hipSuccess;
}
int64_t adapter_workspace_bytes(const orth_hip_adapter_t &, int) { return 4096; }
hipError_t launch_adapter_add(const orth_hip_adapter_t &, int, void *work, hipStream_t stream) {
    threads::launch(stream, work);
    return hipSuccess;
}

// the split-K forward (the other launchers: capi_stubs.hip)
bool skinny_supported(const ForwardArgs &) { return true; }
int64_t skinny_workspace_bytes(const ForwardArgs &, int) { return 4096; }
hipError_t launch_skinny(const ForwardArgs &, const void *, int, float *part, hipStream_t stream) {
    threads::launch(stream, part);
    return hipSuccess;
}
}  // namespace orth
