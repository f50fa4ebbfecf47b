// What kernels of the scoring operators tell of (include/raven_gpu.h, RAVEN_S_*).
#pragma once

#include <cuda_runtime.h>

namespace raven_score {

enum : int { kStatusOffsets = 1, kStatusCapacity = 2, kStatusWait = 4, kStatusIds = 8 };

// The status of calls that are given no word for it, per device and translation
// unit, until it is taken (raven_scoring_status_device).
static __device__ int g_status;
__device__ inline void tell(int* status, int bits) { atomicOr(status ? status : &g_status, bits); }

}  // namespace raven_score
