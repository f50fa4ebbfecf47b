// Shared by the library's translation units; not part of the C ABI.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <string>

namespace raven_internal {

// Sets the calling thread's raven_last_error() message and returns `code`.
int fail(int code, const std::string& msg);

// cuTensorMapEncodeTiled (null without a driver).
PFN_cuTensorMapEncodeTiled_v12000 encode_tiled();

// FP8 codes of f32 rows held in the index's lane-major order (pitch dim).
int fp8_encode_lane_major(const float* d_rows, uint64_t n, uint32_t dim, uint8_t* d_codes, uint64_t ld_codes,
                          uint8_t* d_exps, uint64_t ld_exps, cudaStream_t st);

}  // namespace raven_internal

#ifdef __CUDACC__
namespace raven_score {
// Start of a kernel's memory accesses: the kernel before it in the stream is
// done and its writes are seen; the kernel after it may be set up. A kernel that
// begins before its inputs are written reads them by ordinary loads, never as
// data that is constant while it runs (__ldg, const __restrict__).
__device__ inline void after_previous() {
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
}
}  // namespace raven_score
#endif
