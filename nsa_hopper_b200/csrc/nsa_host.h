// Host helpers that the library's translation units share: the per-thread error text and the checked
// current device.  Not part of the ABI.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace nsa {
namespace host {

constexpr int kMaxDevices = 64;

// Sets the calling thread's error text and returns `code`; an empty text clears it.
__attribute__((visibility("hidden"))) int fail(int code, const char* fmt, ...);
// "what: name (text)" of a CUDA error, returns NSA_ERR_CUDA.
__attribute__((visibility("hidden"))) int cuda_fail(cudaError_t e, const char* what);
// SM count and ordinal of the current device; an error for anything but sm_100.
__attribute__((visibility("hidden"))) int current_sm_count(int* sm_count, int* device);

}  // namespace host
}  // namespace nsa
