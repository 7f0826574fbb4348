// What threads_stubs.hip records for threads_driver.cpp.
#pragma once

#include <hip/hip_runtime_api.h>

#include <atomic>
#include <map>
#include <mutex>
#include <set>

namespace threads {
constexpr int kStreams = 31;
const hipStream_t kCapturing = reinterpret_cast<hipStream_t>(0x4000);
// launches inside on each stream; how often one came in while another of its
// stream, or of any stream, was inside
extern std::atomic<int> inside[kStreams], overlaps, together, all;
extern std::atomic<int> kernels;  // launched by the host side itself
extern std::atomic<bool> throws;      // launchers throw, as an allocation does
extern std::mutex mu;
extern std::map<void *, std::set<void *>> works;
void launch(hipStream_t stream, void *work);
void *tag();  // of the calling thread
}  // namespace threads
