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

constexpr uint32_t kHits = 2048;  // seen ids of a tile that are kept between the scan and the counts
constexpr int kBatch = 4;         // vectors of a thread that are read together

// Shared memory of a tile: a count per column, a bit per column that says whether
// its count is there, the ids found.
__host__ __device__ inline uint32_t shared_bytes(uint32_t tile) { return tile * 4 + tile / 8 + kHits * 2; }

template <typename T, int V>
__device__ inline void put(T* to, const float (&v)[V]) {
  __align__(16) T o[V];
#pragma unroll
  for (int k = 0; k < V; ++k) {
    if constexpr (sizeof(T) == 4)
      o[k] = v[k];
    else if constexpr (std::is_same<T, __half>::value)
      o[k] = __float2half_rn(v[k]);
    else
      o[k] = __float2bfloat16_rn(v[k]);
  }
  *(uint4*)to = *(const uint4*)o;
}
template <typename T>
__device__ inline T one(float v) {
  if constexpr (sizeof(T) == 4)
    return v;
  else if constexpr (std::is_same<T, __half>::value)
    return __float2half_rn(v);
  else
    return __float2bfloat16_rn(v);
}

// A CTA takes a tile of a row, 16 bytes a thread at a time. Rows may start
// anywhere: columns are counted from the last 16-byte boundary before the row
// (`shift` columns before its first), so that vectors are whole but for the row's
// ends. What it has beside the scores (bias, filter) is read at any alignment.
//
// How often each column was seen is counted in shared memory: one scan over the
// history keeps the ids within the tile (16 bits each), their counts are set to 0,
// then counted; a bit per column says which counts are there, so that no table is
// cleared and columns that were not seen cost a bit of a word.
template <typename T, bool LARGEST>
__global__ void __launch_bounds__(256) adjust_kernel(const Params p) {
  constexpr int V = 16 / sizeof(T);
  extern __shared__ uint32_t shared[];
  __shared__ uint32_t found;
  uint32_t* count = shared;
  uint32_t* mark = shared + p.tile;
  uint16_t* hits = (uint16_t*)(mark + p.tile / 32);
  after_previous();
  const uint64_t row = blockIdx.x / p.tiles;
  const T* x = (const T*)p.x + row * p.ld;
  T* out = (T*)p.out + row * p.ld_out;
  const uint32_t shift = (uint32_t)((uintptr_t)x % 16 / sizeof(T));
  // columns [c0, c0 + tile) of the row, c0 <= 0 in the first tile
  const int64_t c0 = (int64_t)(blockIdx.x - row * p.tiles) * p.tile - shift;
  if (c0 >= (int64_t)p.n) return;  // a row that needs no last tile
  bool some = false;
  if (p.seen) {
    for (uint32_t i = threadIdx.x; i < p.tile / 32; i += 256) mark[i] = 0;
    if (threadIdx.x == 0) found = 0;
    int64_t a = p.starts[row], b = p.starts[row + 1];
    if (a < 0 || b < a || (uint64_t)b > p.seen_total) {
      if (threadIdx.x == 0) raven_score::tell(p.status, kStatusOffsets);
      a = b = 0;
    }
    // an id's place in the tile is below `cols` where the tile has it, at least `from` where the row has it
    const uint32_t cols = (uint32_t)min((int64_t)p.tile, (int64_t)p.n - c0), from = c0 < 0 ? shift : 0;
    const bool first = c0 <= 0 && p.tile + c0 > 0;
    auto place = [&](int32_t id) { return (uint32_t)((int64_t)id - c0); };
    __syncthreads();
#pragma unroll 4
    for (int64_t i = a + threadIdx.x; i < b; i += 256) {
      const int32_t id = p.seen[i];
      const uint32_t at = place(id);
      if (first && id >= 0 && (uint32_t)id >= p.n) raven_score::tell(p.status, kStatusIds);
      if (id >= 0 && at < cols && at >= from) {
        const uint32_t k = atomicAdd(&found, 1u);
        if (k < kHits) hits[k] = (uint16_t)at;
        count[at] = 0;
      }
    }
    __syncthreads();
    const uint32_t n = found;
    some = n > 0;
    auto add = [&](uint32_t at) {
      atomicAdd(&count[at], 1u);
      atomicOr(&mark[at / 32], 1u << (at % 32));
    };
    if (n <= kHits) {
      for (uint32_t i = threadIdx.x; i < n; i += 256) add(hits[i]);
    } else {
      for (int64_t i = a + threadIdx.x; i < b; i += 256) {
        const int32_t id = p.seen[i];
        const uint32_t at = place(id);
        if (id >= 0 && at < cols && at >= from) add(at);
      }
    }
    if (some) __syncthreads();
  }
  const float rep = p.repetition ? p.repetition[row] : p.repetition_all;
  const float pre = p.presence ? p.presence[row] : p.presence_all;
  const float freq = p.frequency ? p.frequency[row] : p.frequency_all;
  const float* bias = p.bias ? p.bias + row * p.ld_bias : nullptr;
  const uint32_t* allow = nullptr;
  bool none = false;
  if (p.allow) {
    const int64_t f = p.allow_rows ? (int64_t)p.allow_rows[row] : p.allow_count == 1 ? 0 : (int64_t)row;
    none = f >= (int64_t)p.allow_count;
    if (none && threadIdx.x == 0) raven_score::tell(p.status, kStatusIds);
    if (f >= 0 && !none) allow = p.allow + f * p.ld_allow;
  }
  constexpr float kHidden = LARGEST ? -INFINITY : INFINITY;
  auto seen_before = [&](float v, uint32_t at) {
    const float by = __fadd_rn(pre, __fmul_rn(freq, (float)count[at]));
    v = (v > 0.f) == LARGEST ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
    return LARGEST ? __fsub_rn(v, by) : __fadd_rn(v, by);
  };
  const bool same = (uintptr_t)x % 16 == (uintptr_t)out % 16;
  const uint32_t skew = bias ? (uint32_t)(((uintptr_t)bias / 4 + 4 - shift % 4) % 4) : 0;  // of the bias of a vector's first column
  for (uint32_t l0 = threadIdx.x * V; l0 < p.tile; l0 += 256 * V * kBatch) {
    uint4 raw[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const uint32_t l = l0 + i * 256 * V;
      const int64_t c = c0 + l;
      if (l < p.tile && c >= 0 && c + V <= (int64_t)p.n) raw[i] = *(const uint4*)(x + c);
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const uint32_t l = l0 + i * 256 * V;
      const int64_t c = c0 + l;
      if (l >= p.tile || c >= (int64_t)p.n || c + V <= 0) continue;
      const uint32_t marks = some ? mark[l / 32] >> (l % 32) & ((1u << V) - 1) : 0;
      if (c >= 0 && c + V <= (int64_t)p.n) {
        float v[V];
        const T* r = (const T*)&raw[i];
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = raven_fp8::load_value(r + k);
        if (marks) {
#pragma unroll
          for (int k = 0; k < V; ++k)
            if (marks >> k & 1u) v[k] = seen_before(v[k], l + k);
        }
        if (bias) {
          // from the 16 bytes that hold the first one on; at the ends one by one
          if (c >= 4 && c + V + 4 <= (int64_t)p.n) {
            float b[V + 4];
            const float4* from = (const float4*)(bias + c - skew);
#pragma unroll
            for (int k = 0; k < V / 4; ++k) ((float4*)b)[k] = from[k];
            if (skew) ((float4*)b)[V / 4] = from[V / 4];
            auto shifted = [&](auto s) {
#pragma unroll
              for (int k = 0; k < V; ++k) v[k] = __fadd_rn(v[k], b[k + decltype(s)::value]);
            };
            if (skew == 0)
              shifted(std::integral_constant<int, 0>());
            else if (skew == 1)
              shifted(std::integral_constant<int, 1>());
            else if (skew == 2)
              shifted(std::integral_constant<int, 2>());
            else
              shifted(std::integral_constant<int, 3>());
          } else {
#pragma unroll
            for (int k = 0; k < V; ++k) v[k] = __fadd_rn(v[k], bias[c + k]);
          }
        }
        if (allow) {
          const uint64_t w = (uint64_t)c / 32, w1 = ((uint64_t)c + V - 1) / 32;
          const uint32_t lo = allow[w], bits = __funnelshift_r(lo, w1 != w ? allow[w1] : lo, (uint32_t)c % 32);
#pragma unroll
          for (int k = 0; k < V; ++k)
            if (!(bits >> k & 1u)) v[k] = kHidden;
        }
        if (none) {
#pragma unroll
          for (int k = 0; k < V; ++k) v[k] = kHidden;
        }
        if (same) {
          put<T, V>(out + c, v);
        } else {
#pragma unroll
          for (int k = 0; k < V; ++k) out[c + k] = one<T>(v[k]);
        }
      } else {
        for (int k = 0; k < V; ++k) {
          const int64_t e = c + k;
          if (e < 0 || e >= (int64_t)p.n) continue;
          float v = raven_fp8::load_value(x + e);
          if (marks >> k & 1u) v = seen_before(v, l + k);
          if (bias) v = __fadd_rn(v, bias[e]);
          if (none || (allow && !(allow[e / 32] >> (e % 32) & 1u))) v = kHidden;
          out[e] = one<T>(v);
        }
      }
    }
  }
}

}  // namespace raven_adjust
