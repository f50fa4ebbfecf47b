// Host side that the library's operators share: launches, sizes, checks.
#pragma once

#include <cuda_runtime.h>
#include <nvtx3/nvToolsExt.h>

#include <atomic>
#include <cstdint>
#include <mutex>
#include <string>

#include "../../include/raven_gpu.h"
#include "internal.h"

namespace raven_launch {

using raven_internal::fail;

struct NvtxRange {
  explicit NvtxRange(const char* name) { nvtxRangePushA(name); }
  ~NvtxRange() { nvtxRangePop(); }
  NvtxRange(const NvtxRange&) = delete;
  NvtxRange& operator=(const NvtxRange&) = delete;
};

#define CU(call)                                                                        \
  do {                                                                                  \
    cudaError_t e_ = (call);                                                            \
    if (e_ != cudaSuccess) return fail(RAVEN_ECUDA, std::string(#call ": ") + cudaGetErrorString(e_)); \
  } while (0)

constexpr uint64_t kMaxRows = 0x7fffffffull;  // rows are TMA coordinates (int32)
constexpr uint32_t kMaxDim = 65536;
constexpr uint32_t kBlock = 128;              // values under one scale

inline uint64_t type_size(int32_t t) {
  return t == RAVEN_TYPE_F32 ? 4 : t == RAVEN_TYPE_F16 || t == RAVEN_TYPE_BF16 ? 2 : t == RAVEN_TYPE_FP8 ? 1 : 0;
}
inline bool aligned(const void* p, uint64_t a) { return (uintptr_t)p % a == 0; }

// What a device's first call sets up is no part of a stream's work: this thread
// does it although one of its streams is being captured, which otherwise ends
// the capture.
struct Apart {
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  Apart() { cudaThreadExchangeStreamCaptureMode(&mode); }
  ~Apart() { cudaThreadExchangeStreamCaptureMode(&mode); }
};

// SMs of the current device. On a device's first call its default memory pool
// is told to keep freed scratch (as raven_index_upload does): a pool that gives
// it back at every synchronisation makes the next call wait for an allocation.
inline int sm_count(int* out) {
  static std::mutex mu;
  static int count[256] = {};
  int dev = 0;
  CU(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 256) return fail(RAVEN_EINVAL, "device ordinal out of range");
  std::lock_guard<std::mutex> lk(mu);
  if (!count[dev]) {
    CU(cudaDeviceGetAttribute(&count[dev], cudaDevAttrMultiProcessorCount, dev));
    Apart apart;
    cudaMemPool_t pool;
    uint64_t keep = ~0ull;
    if (cudaDeviceGetDefaultMemPool(&pool, dev) == cudaSuccess)
      cudaMemPoolSetAttribute(pool, cudaMemPoolAttrReleaseThreshold, &keep);
  }
  *out = count[dev];
  return RAVEN_OK;
}

// Launches `kern` so that it may start while the kernel before it in the stream
// ends. Every kernel here waits for that one (after_previous) before it touches
// memory, and lets its own successor start at once. `allowed`: devices (bits)
// on which the kernel may already use `smem` bytes; the attribute is set again
// when a launch is refused (a context replaced since).
struct Allowed {
  std::atomic<uint64_t> mask{0};
  const uint32_t most;  // of a kernel whose launches differ in size: the largest
  explicit Allowed(uint32_t m = 0) : most(m) {}
};
template <typename... K, typename... A>
cudaError_t launch(void (*kern)(K...), uint64_t grid, int threads, uint32_t smem, Allowed& allowed, cudaStream_t st,
                   A&&... args) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = 1ull << (dev & 63);
  cudaLaunchConfig_t c{};
  c.gridDim = dim3((unsigned)grid);
  c.blockDim = dim3((unsigned)threads);
  c.dynamicSmemBytes = smem;
  c.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  c.attrs = &at;
  c.numAttrs = 1;
  for (int turn = 0;; ++turn) {
    if (smem > 48 * 1024 && (turn || dev >= 64 || !(allowed.mask.load(std::memory_order_relaxed) & bit))) {
      Apart apart;
      e = cudaFuncSetAttribute((const void*)kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               (int)(smem > allowed.most ? smem : allowed.most));
      if (e != cudaSuccess) return e;
      allowed.mask.fetch_or(bit, std::memory_order_relaxed);
    }
    e = cudaLaunchKernelEx(&c, kern, args...);
    if (e != cudaErrorInvalidValue || turn || smem <= 48 * 1024) return e;
    (void)cudaGetLastError();
  }
}

inline bool float_type(int32_t t) { return t == RAVEN_TYPE_F32 || t == RAVEN_TYPE_F16 || t == RAVEN_TYPE_BF16; }
inline int check_dim(uint32_t dim) {
  if (dim == 0 || dim > kMaxDim) return fail(RAVEN_ELIMIT, "dim must be in 1..65536");
  return RAVEN_OK;
}

}  // namespace raven_launch
