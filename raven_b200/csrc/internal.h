// Shared by the library's translation units; not part of the C ABI.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <string>

#include "../../include/raven_gpu.h"

namespace raven_internal {

// Sets the calling thread's raven_last_error() message and returns `code`.
int fail(int code, const std::string& msg);

// cuTensorMapEncodeTiled (null without a driver).
PFN_cuTensorMapEncodeTiled_v12000 encode_tiled();

// FP8 codes of f32 rows held in the index's lane-major order (pitch dim).
int fp8_encode_lane_major(const float* d_rows, uint64_t n, uint32_t dim, uint8_t* d_codes, uint64_t ld_codes,
                          uint8_t* d_exps, uint64_t ld_exps, cudaStream_t st);

// Values under one scale word of 4-bit rows of a type, 0 for other types.
uint32_t int4_group(int32_t type);
// raven_scores_device with 4-bit vectors.
int int4_scores(const raven_rows* q, const raven_rows* v, uint32_t dim, float alpha, const float* d_bias, void* d_out,
                int32_t out_type, uint64_t ld, int32_t* d_status, void* stream);
// Takes the status of the operators of rows4.cu (raven_scoring_status_device).
int rows4_status(int* d_status, cudaStream_t st);
// 4-bit rows of f32 rows held in the index's lane-major order.
int int4_write_lane_major(const float* d_rows, uint64_t n, uint32_t dim, const raven_rows* out, cudaStream_t st);

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
