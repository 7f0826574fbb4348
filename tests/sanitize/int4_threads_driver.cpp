// Host threads that call paged_attention over a cache in 4 bits at the same
// time, beside the operators that use the same workspaces, over the stand-ins
// of threads_stubs.hip and int4_threads_stubs.hip.
#include <cstdio>
#include <functional>
#include <set>
#include <thread>
#include <vector>

#include "orth_hip.h"
#include "threads.h"

namespace {

int failures = 0;
void expect(bool ok, const char *what) {
    if (ok) return;
    std::printf("failed: %s (%s)\n", what, orth_hip_last_error());
    failures++;
}

// a pointer that nothing follows
struct Any {
    uintptr_t n;
    template <class T>
    operator T *() const { return reinterpret_cast<T *>(n); }
};
Any P(uintptr_t n) { return {n}; }

const orth_hip_attend_t kAttend = {P(16), P(32), {256, 64}, {256, 64}, P(48), P(64), nullptr, 8, 8, 8, 5, 4, 0, 0.125f, 0};

int attend4(hipStream_t s) {
    const orth_hip_int4_cache_t c = {P(0x10000), P(0x20000), P(0x30000), P(0x40000), 16, 2, 64, 32, 8,
                                     {1024, 64, 32}, {1024, 64, 32}, {128, 8, 4}, {128, 8, 4}};
    return orth_paged_attention_int4_hip(&c, &kAttend, ORTH_DT_F16, s);
}
int attend(hipStream_t s) {
    const orth_hip_cache_t c = {P(0x10000), P(0x20000), ORTH_DT_F16, 16, 2, 64, 8, {2048, 128, 64}, {2048, 128, 64}};
    return orth_paged_attention_hip(&c, &kAttend, s);
}

// every call of a list by a thread of its own, 12 times
void run(const std::vector<std::function<int()>> &calls, const char *what) {
    threads::overlaps = 0;
    threads::together = 0;
    threads::works.clear();
    std::atomic<int> ready{0}, errors{0};
    std::vector<std::thread> ts;
    for (const auto &f : calls)
        ts.emplace_back([&] {
            ready++;
            while (ready < (int)calls.size()) std::this_thread::yield();
            for (int i = 0; i < 12; i++) errors += f() != ORTH_OK;
        });
    for (auto &t : ts) t.join();
    expect(errors == 0, what);
}

}  // namespace

int main() {
    const hipStream_t one = reinterpret_cast<hipStream_t>(0x1000), two = reinterpret_cast<hipStream_t>(0x2001);
    expect(attend4(one) == ORTH_OK, "one thread");

    // A call's launches share one workspace: no other call's come between them
    run({[&] { return attend4(one); }, [&] { return attend4(one); }, [&] { return attend(one); }}, "attention");
    expect(threads::overlaps == 0, "attention over both caches on one stream");
    run({[&] { return attend4(threads::kCapturing); }, [&] { return attend(threads::kCapturing); }}, "captured");
    expect(threads::overlaps == 0, "two threads' calls on one captured stream");
    run({[&] { return attend4(one); }, [&] { return attend4(two); }}, "two streams");
    expect(threads::together > 0, "two streams at once");
    run({[&] { return attend4(hipStreamPerThread); }, [&] { return attend4(hipStreamPerThread); }}, "streams per thread");
    expect(threads::works.size() == 2, "two threads");
    {
        const std::set<void *> &a = threads::works.begin()->second, &b = threads::works.rbegin()->second;
        for (void *p : a) expect(b.count(p) == 0, "the workspaces of two threads' own streams");
    }

    // captured attention records the clearing of its counters, eager attention none
    threads::kernels = 0;
    expect(attend4(one) == ORTH_OK && threads::kernels == 0, "eager counters");
    expect(attend4(threads::kCapturing) == ORTH_OK && threads::kernels == 1, "captured counters start from zero");

    // an exception ends as a status with a message, and the workspace is free again
    threads::throws = true;
    expect(attend4(one) == ORTH_ERR_HIP && orth_hip_last_error()[0] != 0, "an exception");
    threads::throws = false;
    run({[&] { return attend4(one); }}, "after an exception");

    if (failures) return 1;
    std::printf("threads ok\n");
    return 0;
}
