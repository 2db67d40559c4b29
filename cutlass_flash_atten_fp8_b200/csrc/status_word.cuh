// What kernels leave in the status words (a device word, and a mapped one of the host) and what they make of what is there.
#pragma once
#include "fa8_kernel.h"

namespace fa8 {

// A bounded wait ran out.  That takes the place of an index out of range that an earlier launch reported: the answers of this launch
// are lost, of that one only what the index was of.
__device__ __forceinline__ void report_expired_wait(int* status, volatile int* host_status, int code) {
  if (status != nullptr && atomicCAS(status, 0, code) == kBadIndex) atomicCAS(status, kBadIndex, code);
  if (host_status != nullptr) {
    *host_status = code;
    __threadfence_system();
  }
}

// A wait of an earlier CTA or launch ran out and nobody has cleared the word: there is nothing to be computed.  An index out of
// range concerns the launch that reported it alone.
__device__ __forceinline__ bool wait_has_expired(const int* status) {
  if (status == nullptr) return false;
  const int code = *reinterpret_cast<const volatile int*>(status);
  return code != 0 && code != kBadIndex;
}

}  // namespace fa8
