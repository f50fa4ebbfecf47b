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
  uint32_t tiles;   // of a row
  int* status;
};

constexpr uint32_t kThreads = 256;
constexpr uint32_t kMostPlaces = 8192;  // of a tile
constexpr uint32_t kHits = 2048;        // seen ids of a tile that are kept between the scan and the counts
constexpr uint32_t kBatch = 4;          // vectors of a thread that are read together

// Shared memory of a tile: a word per place (how often it was seen, then its
// finished score), per 32 places which were seen and which are hidden, the ids found.
__host__ __device__ inline uint32_t shared_bytes(uint32_t tile, bool seen) {
  return tile / 4 + (seen ? tile * 4 + kHits * 2 : 0);
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
// A score as its bits, in the low half of a word where it has 16.
template <typename T>
__device__ inline uint32_t bits_of(T v) {
  if constexpr (sizeof(T) == 4)
    return __float_as_uint(v);
  else
    return *(const uint16_t*)&v;
}

// 16 bytes of scores as four words: what is done to them.
template <typename T>
struct Vector {
  static constexpr uint32_t V = 16 / sizeof(T);
  uint32_t w[4];

  // V values from b[S] on; each sum is rounded to f32 and to the type.
  template <int S>
  __device__ void add(const float* from) {
    const float* b = from + S;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (sizeof(T) == 4) {
        w[j] = __float_as_uint(__fadd_rn(__uint_as_float(w[j]), b[j]));
      } else if constexpr (std::is_same<T, __half>::value) {
        const float2 v = __half22float2(*(const __half2*)&w[j]);
        const __half2 r = __floats2half2_rn(__fadd_rn(v.x, b[2 * j]), __fadd_rn(v.y, b[2 * j + 1]));
        w[j] = *(const uint32_t*)&r;
      } else {
        const float x = __uint_as_float(w[j] << 16), y = __uint_as_float(w[j] & 0xffff0000u);
        const __nv_bfloat162 r = __floats2bfloat162_rn(__fadd_rn(x, b[2 * j]), __fadd_rn(y, b[2 * j + 1]));
        w[j] = *(const uint32_t*)&r;
      }
    }
  }
  __device__ void set(uint32_t k, uint32_t bits) {  // k: known when compiled
    if constexpr (sizeof(T) == 4)
      w[k] = bits;
    else
      w[k / 2] = __byte_perm(w[k / 2], bits, k & 1 ? 0x5410 : 0x3254);
  }
  // Places whose bit is set become `bits` (two of them a word where they have 16).
  __device__ void hide(uint32_t hidden, uint32_t bits) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (sizeof(T) == 4) {
        if (hidden >> j & 1u) w[j] = bits;
      } else {
        // the two bits at the tops of two bytes, each copied over half a word
        uint32_t m;
        asm("prmt.b32 %0, %1, 0, 0x9988;" : "=r"(m) : "r"((hidden >> (2 * j) & 3u) * 0x4080u));
        w[j] = (w[j] & ~m) | (bits & m);
      }
    }
  }
};

// A CTA takes a tile of a row, 16 bytes a thread at a time. Rows may start
// anywhere: places are counted from the last 16-byte boundary before the row (its
// first column is place `shift`), so that vectors are whole but for the row's ends.
// What it has beside the scores (bias, filter) is read at any alignment.
//
// What a query has seen is worked out before: one scan over the history keeps the
// ids within the tile (16 bits each), their counts are set to 0, then counted; a
// bit per place says which counts are there, so that no table is cleared. Then each
// id's score takes the place of its count. Scores that were not seen cost a bit of a
// word, and the division is done for seen ones alone (where each thread did it for
// its own vectors, a warp took the branch for nearly every one: 256 x 250007 bf16
// 216 us, 142 now). The first vectors are on their way meanwhile.
//
// What bounds it: memory where histories are short (64 x 1000000 f32 94 us, 5.5 TB/s;
// with 16-bit scores instructions about as much), the scans where they are long, since
// each tile of a row scans it: tiles are as large as counts in shared memory and four
// CTAs an SM allow.
template <typename T, bool LARGEST>
__global__ void __launch_bounds__(kThreads, 4) adjust_kernel(const Params p) {
  constexpr uint32_t V = 16 / sizeof(T);
  extern __shared__ uint2 shared[];
  __shared__ uint32_t found;
  uint2* bits = shared;  // x: seen, y: hidden
  uint32_t* count = (uint32_t*)(bits + p.tile / 32);  // then the bits of a score
  uint16_t* hits = (uint16_t*)(count + p.tile);
  after_previous();
  const uint32_t row = blockIdx.x / p.tiles;  // 32-bit: the 64-bit division took as long as a vector
  const T* x = (const T*)p.x + row * p.ld;
  T* out = (T*)p.out + row * p.ld_out;
  const uint32_t shift = (uint32_t)((uintptr_t)x % 16 / sizeof(T));
  x -= shift;
  out -= shift;
  // places [first, last) of the row, of which the tile has those from t0 on
  const uint32_t first = shift, last = (uint32_t)p.n + shift, t0 = (blockIdx.x - row * p.tiles) * p.tile;
  if (t0 >= last) return;  // a row that needs no last tile
  const uint32_t worst = bits_of(one<T>(LARGEST ? -INFINITY : INFINITY)) * (V == 8 ? 0x10001u : 1u);
  const bool inner = t0 >= first + 4 && t0 + p.tile + 4 <= last;  // the row's ends, and what is beside them, are elsewhere
  int64_t a = 0, b = 0;
  if (p.starts) {
    a = p.starts[row];
    b = p.starts[row + 1];
  }
  const float* bias = p.bias ? p.bias + row * p.ld_bias - shift : nullptr;  // of place 0
  const uint32_t skew = (uint32_t)((uintptr_t)bias / 4 % 4);                // of a vector's first bias from 16 bytes
  // The scores of the thread's first vectors are on their way from here on.
  uint4 raw[kBatch];
  auto read = [&](auto in, uint32_t l0) {
#pragma unroll
    for (uint32_t i = 0; i < kBatch; ++i) {
      const uint32_t l = l0 + i * kThreads * V, c = t0 + l;
      if (l < p.tile && (decltype(in)::value || (c >= first && c + V <= last))) raw[i] = *(const uint4*)(x + c);
    }
  };
  if (inner)
    read(std::true_type(), threadIdx.x * V);
  else
    read(std::false_type(), threadIdx.x * V);
  const uint32_t* allow = nullptr;
  bool none = false;
  if (p.allow) {
    const int64_t f = p.allow_rows ? (int64_t)p.allow_rows[row] : p.allow_count == 1 ? 0 : (int64_t)row;
    none = f >= (int64_t)p.allow_count;
    if (none && threadIdx.x == 0) raven_score::tell(p.status, kStatusIds);
    if (f >= 0 && !none) allow = p.allow + f * p.ld_allow;
  }
  for (uint32_t i = threadIdx.x; i < p.tile / 32; i += kThreads) {
    uint32_t hidden = none ? ~0u : 0u;
    if (allow) {
      // places from t0 + 32 i on are columns from c on: the bits of two words
      const int64_t c = (int64_t)t0 + 32 * i - shift;
      const int64_t w = c >> 5, words = ((int64_t)p.n + 31) / 32;
      const uint32_t a = w >= 0 && w < words ? allow[w] : 0, b = (c & 31) && w + 1 < words ? allow[w + 1] : 0;
      hidden = ~__funnelshift_r(a, b, (uint32_t)c & 31);
    }
    bits[i] = make_uint2(0, hidden);
  }
  if (threadIdx.x == 0) found = 0;
  __syncthreads();
  if (p.starts) {
    if (a < 0 || b < a || (uint64_t)b > p.seen_total || (uint64_t)(b - a) >> 32) {  // ids are counted in 32 bits
      if (threadIdx.x == 0) raven_score::tell(p.status, kStatusOffsets);
      a = b = 0;
    }
    const uint32_t ends = min(p.tile, last - t0);
    // false for what is no column of the tile; `at`: its place there
    auto within = [&](int32_t id, uint32_t& at) {
      at = (uint32_t)id + shift - t0;
      return id >= 0 && (uint32_t)id < (uint32_t)p.n && at < ends;
    };
    constexpr int kIds = 8;  // of a thread at once
    for (int64_t i0 = a + threadIdx.x; i0 < b; i0 += kIds * kThreads) {
      int32_t id[kIds];
#pragma unroll
      for (int k = 0; k < kIds; ++k) id[k] = i0 + k * kThreads < b ? p.seen[i0 + k * kThreads] : -1;
#pragma unroll
      for (int k = 0; k < kIds; ++k) {
        uint32_t at;
        if (within(id[k], at)) {
          const uint32_t h = atomicAdd(&found, 1u);
          if (h < kHits) hits[h] = (uint16_t)at;
          count[at] = 0;
        } else if (t0 == 0 && id[k] >= 0 && (uint32_t)id[k] >= (uint32_t)p.n) {
          raven_score::tell(p.status, kStatusIds);
        }
      }
    }
    __syncthreads();
    const uint32_t n = found;
    if (n) {
      auto add = [&](uint32_t at) {
        atomicAdd(&count[at], 1u);
        atomicOr(&bits[at / 32].x, 1u << (at % 32));
      };
      if (n <= kHits) {
        for (uint32_t i = threadIdx.x; i < n; i += kThreads) add(hits[i]);
      } else {
        for (int64_t i = a + threadIdx.x; i < b; i += kThreads) {
          uint32_t at;
          if (within(p.seen[i], at)) add(at);
        }
      }
      __syncthreads();
      const float rep = p.repetition ? p.repetition[row] : p.repetition_all;
      const float pre = p.presence ? p.presence[row] : p.presence_all;
      const float freq = p.frequency ? p.frequency[row] : p.frequency_all;
      auto worse = [&](uint32_t at) {
        const float v = raven_fp8::load_value(x + t0 + at);
        const float by = __fadd_rn(pre, __fmul_rn(freq, (float)count[at]));
        float y = (v > 0.f) == LARGEST ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
        y = LARGEST ? __fsub_rn(y, by) : __fadd_rn(y, by);
        return bits_of(one<T>(bias ? __fadd_rn(y, bias[t0 + at]) : y));
      };
      if (n <= kHits) {
        uint32_t y[kHits / kThreads];  // an id that is there twice: both read its count before either writes
#pragma unroll
        for (uint32_t i = 0; i < kHits / kThreads; ++i)
          if (threadIdx.x + kThreads * i < n) y[i] = worse(hits[threadIdx.x + kThreads * i]);
        __syncthreads();
#pragma unroll
        for (uint32_t i = 0; i < kHits / kThreads; ++i)
          if (threadIdx.x + kThreads * i < n) count[hits[threadIdx.x + kThreads * i]] = y[i];
      } else {
#pragma unroll 8
        for (uint32_t at = threadIdx.x; at < p.tile; at += kThreads)
          if (bits[at / 32].x >> (at % 32) & 1u) count[at] = worse(at);
      }
      __syncthreads();
    }
  }
  const bool same = (uintptr_t)x % 16 == (uintptr_t)out % 16;
  // IN: all the tile's places are the row's, and so are four more on either side.
  auto finish = [&](auto in) {
    constexpr bool IN = decltype(in)::value;
    for (uint32_t l0 = threadIdx.x * V; l0 < p.tile; l0 += kBatch * kThreads * V) {
      if (l0 >= kBatch * kThreads * V) read(in, l0);
      // Biases of two vectors are read before either is written: the compiler cannot know that they lie apart.
#pragma unroll
      for (uint32_t i0 = 0; i0 < kBatch; i0 += 2) {
        float b[2][V + 4];
        if (bias) {
#pragma unroll
          for (uint32_t h = 0; h < 2; ++h) {
            const uint32_t l = l0 + (i0 + h) * kThreads * V, c = t0 + l;
            if (l >= p.tile || (!IN && (c < first || c + V > last))) continue;
            if (IN || (c >= first + 4 && c + V + 4 <= last)) {
              // the 16 bytes that hold the first one, and those after them
              const float4* from = (const float4*)(bias + c - skew);
#pragma unroll
              for (uint32_t k = 0; k < V / 4; ++k) ((float4*)b[h])[k] = from[k];
              if (skew) ((float4*)b[h])[V / 4] = from[V / 4];
            } else {
#pragma unroll
              for (uint32_t k = 0; k < V + 4; ++k) b[h][k] = k >= skew && k < skew + V ? bias[c + k - skew] : 0.f;
            }
          }
        }
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h) {
          const uint32_t l = l0 + (i0 + h) * kThreads * V, c = t0 + l;
          if (l >= p.tile || (!IN && c >= last)) continue;
          const uint2 m = bits[l / 32];
          const uint32_t seen = m.x >> (l % 32) & ((1u << V) - 1), hidden = m.y >> (l % 32);
          if (IN || (c >= first && c + V <= last)) {
            Vector<T> v{{raw[i0 + h].x, raw[i0 + h].y, raw[i0 + h].z, raw[i0 + h].w}};
            if (bias) {
              if (skew == 0)
                v.template add<0>(b[h]);
              else if (skew == 1)
                v.template add<1>(b[h]);
              else if (skew == 2)
                v.template add<2>(b[h]);
              else
                v.template add<3>(b[h]);
            }
            if (seen) {
#pragma unroll
              for (uint32_t k = 0; k < V; ++k)
                if (seen >> k & 1u) v.set(k, count[l + k]);
            }
            if (p.allow) v.hide(hidden, worst);
            if (same) {
              *(uint4*)(out + c) = make_uint4(v.w[0], v.w[1], v.w[2], v.w[3]);
            } else {
#pragma unroll
              for (uint32_t k = 0; k < V; ++k) out[c + k] = ((const T*)v.w)[k];
            }
          } else {
            for (uint32_t k = 0; k < V; ++k)
              if (c + k >= first && c + k < last) {
                const float f = raven_fp8::load_value(x + c + k);
                T o = one<T>(bias ? __fadd_rn(f, bias[c + k]) : f);
                if (seen >> k & 1u) o = *(const T*)&count[l + k];
                out[c + k] = hidden >> k & 1u ? *(const T*)&worst : o;
              }
          }
        }
      }
    }
  };
  if (inner)
    finish(std::true_type());
  else
    finish(std::false_type());
}

}  // namespace raven_adjust
