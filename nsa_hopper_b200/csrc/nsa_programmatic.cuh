// Kernels that are launched programmatically (while the stream's kernel before them still runs, if that one allows it).
#pragma once

namespace nsa {

// Lets the next kernel be launched, and touches no memory before all earlier ones have ended.
__device__ __forceinline__ void start_in_order() {
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

}  // namespace nsa
