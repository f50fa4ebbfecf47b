// Scores put right before the best are taken (include/raven_gpu.h,
// raven_adjust_scores_device): less for rows that a query has seen, a bias per
// row, and rows that it may not see.
//
// Each operation is one f32 operation, rounded (no fused multiply-add), and the
// result is rounded to the scores' type: the same bits whatever the tiles are.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>

#include "fp8.cuh"
#include "internal.h"
#include "status.cuh"

namespace raven_adjust {

using raven_score::after_previous;

using raven_score::kStatusIds;
using raven_score::kStatusOffsets;

struct Params {
  const void* x;
  void* out;
  uint64_t nq, n, ld, ld_out;
  const float* bias;
  uint64_t ld_bias;
  const uint32_t* allow;
  uint64_t allow_count, ld_allow;
  const int32_t* allow_rows;
  const int32_t* seen;
  uint64_t seen_total;
  const int64_t* starts;
  const float *repetition, *presence, *frequency;
  float repetition_all, presence_all, frequency_all;
  uint32_t tile;    // columns of a CTA
  uint64_t tiles;   // of a row
  int* status;
};

// A CTA takes a tile of a row. How often each of its columns was seen is counted
// in shared memory: the history's ids within the tile get a count of 0, then are
// counted; a bit per column says which counts are there, so that no table is
// cleared and columns that were not seen cost a bit.
template <typename T, bool LARGEST>
__global__ void __launch_bounds__(256) adjust_kernel(const Params p) {
  extern __shared__ uint32_t shared[];
  uint32_t* count = shared;
  uint32_t* mark = shared + p.tile;
  after_previous();
  const uint64_t row = blockIdx.x / p.tiles, c0 = (blockIdx.x - row * p.tiles) * p.tile;
  const uint32_t cols = (uint32_t)min((uint64_t)p.tile, p.n - c0);
  if (p.seen) {
    for (uint32_t i = threadIdx.x; i < (cols + 31) / 32; i += 256) mark[i] = 0;
    int64_t a = p.starts[row], b = p.starts[row + 1];
    if (a < 0 || b < a || (uint64_t)b > p.seen_total) {
      if (threadIdx.x == 0) raven_score::tell(p.status, kStatusOffsets);
      a = b = 0;
    }
    bool some = false;
    for (int64_t i = a + threadIdx.x; i < b; i += 256) {
      const int64_t id = p.seen[i], at = id - (int64_t)c0;
      if (id >= (int64_t)p.n) raven_score::tell(p.status, kStatusIds);
      if (id >= 0 && at >= 0 && at < cols) {
        count[at] = 0;
        some = true;
      }
    }
    if (__syncthreads_or(some)) {
      for (int64_t i = a + threadIdx.x; i < b; i += 256) {
        const int64_t id = p.seen[i], at = id - (int64_t)c0;
        if (id >= 0 && at >= 0 && at < cols) {
          atomicAdd(&count[at], 1u);
          atomicOr(&mark[at / 32], 1u << (at % 32));
        }
      }
      __syncthreads();
    }
  }
  const float rep = p.repetition ? p.repetition[row] : p.repetition_all;
  const float pre = p.presence ? p.presence[row] : p.presence_all;
  const float freq = p.frequency ? p.frequency[row] : p.frequency_all;
  const uint32_t* allow = nullptr;
  bool none = false;
  if (p.allow) {
    const int64_t f = p.allow_rows ? (int64_t)p.allow_rows[row] : p.allow_count == 1 ? 0 : (int64_t)row;
    none = f >= (int64_t)p.allow_count;
    if (none && threadIdx.x == 0) raven_score::tell(p.status, kStatusIds);
    if (f >= 0 && !none) allow = p.allow + f * p.ld_allow;
  }
  const T* x = (const T*)p.x + row * p.ld + c0;
  T* out = (T*)p.out + row * p.ld_out + c0;
  for (uint32_t i = threadIdx.x; i < cols; i += 256) {
    float v;
    if constexpr (sizeof(T) == 4)
      v = x[i];
    else
      v = raven_fp8::load_value(x + i);
    if (p.seen && (mark[i / 32] >> (i % 32) & 1u)) {
      const float by = __fadd_rn(pre, __fmul_rn(freq, (float)count[i]));
      v = (v > 0.f) == LARGEST ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
      v = LARGEST ? __fsub_rn(v, by) : __fadd_rn(v, by);
    }
    if (p.bias) v = __fadd_rn(v, p.bias[row * p.ld_bias + c0 + i]);
    const uint64_t c = c0 + i;
    if (none || (allow && !(allow[c / 32] >> (c % 32) & 1u))) v = LARGEST ? -INFINITY : INFINITY;
    if constexpr (sizeof(T) == 4)
      out[i] = v;
    else if constexpr (std::is_same<T, __half>::value)
      out[i] = __float2half_rn(v);
    else
      out[i] = __float2bfloat16_rn(v);
  }
}

}  // namespace raven_adjust
