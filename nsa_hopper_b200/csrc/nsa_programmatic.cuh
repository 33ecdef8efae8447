// Kernels that are launched programmatically (while the stream's kernel before them still runs, if that one allows it).
#pragma once

namespace nsa {

// Lets the next kernel be launched.
__device__ __forceinline__ void allow_next() { asm volatile("griddepcontrol.launch_dependents;"); }
// Until all earlier kernels have ended.
__device__ __forceinline__ void wait_for_earlier() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// Lets the next kernel be launched, and touches no memory before all earlier ones have ended.
__device__ __forceinline__ void start_in_order() {
  allow_next();
  wait_for_earlier();
}

}  // namespace nsa
