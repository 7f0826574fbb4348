// Host threads that call the entry points of include/orth_hip.h at the same
// time, over the stand-ins of threads_stubs.hip.
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

int adapter(hipStream_t s) {
    const orth_hip_adapter_t a = {P(16), P(32), P(48), P(64), P(80), P(96), nullptr, 64, 32, 32, 5, 64, 32, 3, 8, ORTH_DT_F16};
    return orth_adapter_add_hip(&a, s);
}
int attend(hipStream_t s) {
    const orth_hip_cache_t c = {P(0x10000), P(0x20000), ORTH_DT_F16, 16, 2, 64, 8, {2048, 128, 64}, {2048, 128, 64}};
    const orth_hip_attend_t a = {P(16), P(32), {256, 64}, {256, 64}, P(48), P(64), nullptr, 8, 8, 8, 5, 4, 0, 0.125f, 0};
    return orth_paged_attention_hip(&c, &a, s);
}
int forward(hipStream_t s, bool noalloc = false) {
    const orth_hip_layer_t l = {{P(0x30000), P(0x40000), 4, ORTH_DT_F16, 2, 256, 256}, {nullptr, nullptr, nullptr, ORTH_DT_F16, 0, 0}, 0.f};
    return noalloc ? orth_layer_forward_hip_noalloc(&l, nullptr, 0, nullptr, ORTH_DT_F32, P(0x50000), P(0x60000), 8, ORTH_DT_F16, s)
                   : orth_layer_forward_hip(&l, P(0x50000), P(0x60000), 8, ORTH_DT_F16, s);
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
    expect(adapter(one) == ORTH_OK && attend(one) == ORTH_OK && forward(one) == ORTH_OK, "one thread");

    // A call's launches share one workspace: no other call's come between them
    run({[&] { return adapter(one); }, [&] { return adapter(one); }}, "adapters");
    expect(threads::overlaps == 0, "two threads' adapters on one stream");
    run({[&] { return attend(nullptr); }, [&] { return attend(nullptr); }}, "attention");
    expect(threads::overlaps == 0, "two threads' attention on the null stream");
    run({[&] { return attend(one); }, [&] { return adapter(one); }, [&] { return forward(one); }}, "mixed");
    expect(threads::overlaps == 0, "attention, adapters and split-K on one stream");
    run({[&] { return forward(one); }, [&] { return forward(one); }}, "split-K");
    expect(threads::overlaps == 0, "two threads' split-K on one stream");
    run({[&] { return adapter(threads::kCapturing); }, [&] { return attend(threads::kCapturing); }}, "captured");
    expect(threads::overlaps == 0, "two threads' calls on one captured stream");
    run({[&] { return forward(threads::kCapturing, true); }, [&] { return attend(threads::kCapturing); }}, "captured, no allocation");
    expect(threads::overlaps == 0, "no-allocation and other calls on one captured stream");
    // streams of their own do not wait for each other
    run({[&] { return adapter(one); }, [&] { return adapter(two); }}, "two streams");
    expect(threads::together > 0, "two streams at once");

    // hipStreamPerThread is one handle and a stream of each thread: no memory in common
    run({[&] { return adapter(hipStreamPerThread); }, [&] { return attend(hipStreamPerThread); }}, "streams per thread");
    expect(threads::works.size() == 2, "two threads");
    {
        const std::set<void *> &a = threads::works.begin()->second, &b = threads::works.rbegin()->second;
        for (void *p : a) expect(b.count(p) == 0, "the workspaces of two threads' own streams");
    }

    // captured attention records the clearing of its counters, eager attention none
    threads::kernels = 0;
    expect(attend(one) == ORTH_OK && threads::kernels == 0, "eager counters");
    expect(attend(threads::kCapturing) == ORTH_OK && threads::kernels == 1, "captured counters start from zero");

    // an exception ends as a status with a message, and the workspace is free again
    threads::throws = true;
    expect(adapter(one) == ORTH_ERR_HIP && orth_hip_last_error()[0] != 0, "an exception under adapter_add");
    expect(attend(one) == ORTH_ERR_HIP && orth_hip_last_error()[0] != 0, "an exception under paged_attention");
    threads::throws = false;
    run({[&] { return adapter(one); }}, "after an exception");

    if (failures) return 1;
    std::printf("threads ok\n");
    return 0;
}
