// Scores of queries against 4-bit rows (int4.cuh has their layout):
//
//   S[i, j] = alpha * sum_g step_jg (z_jg sum_k q_ik + sum_k code_jk q_ik) + bias[j]
//
// The inner sums run on the tensor cores (mma m16n8k16, f16 operands, f32 sums)
// with rows as the M side and queries as the N side. A code is not converted: 4
// bits at the bottom of a 16-bit lane are the f16 subnormal code * 2^-24, at bits
// 4-7 code * 2^-20, so one AND makes two operands (five instructions per eight
// codes). What a fragment's lane holds of K is free as long as both sides agree:
// lane t of a row's four takes the eight values 8t.. of each unit of 32 (one
// word), as pairs (0, 4), (1, 5), (2, 6), (3, 7).
//
// Queries are brought to a largest magnitude in [2^14, 2^15) by a power of two
// each, so that f16 holds what f32, f16 and bf16 values may be: 11 bits of a value
// in one part, 22 in two (f32), nothing below 2^-35 of the largest (values paired
// with codes at bits 4-7 are kept as sixteenths). The sum of a group starts at
// z * sum(q), and its step is applied in f32 when the group ends: the scale is
// never rounded into an operand.
//
// What bounds it: reading the codes. Each warp has its own ring of copies to shared
// memory (cp.async) for tiles of 32 rows x 128 values (2 KB); a lane reads back
// what it copied, so only the scale words, which the lanes of a row share, need
// the warp to meet. Few rows of many values are split over K between the warps of
// a CTA, which add up in a fixed order.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>

#include "fp8.cuh"
#include "int4.cuh"
#include "internal.h"

namespace raven_score4 {

using raven_int4::kBlock;
using raven_int4::kUnit;
using raven_score::after_previous;

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMT = 2;                  // M tiles of a warp
constexpr uint32_t kRows = 16 * kMT;    // rows of a warp's tile
constexpr int kDepth = 4;               // tiles under way per warp

struct Params {
  const void* q;      // queries that each CTA lays out for itself, or null: `laid` holds them
  const uint8_t* laid;
  int q_type;         // 0 f32, 1 f16, 2 bf16
  uint64_t nq, ld_q;
  const uint8_t* codes;
  const uint32_t* words;
  uint64_t n, ld_codes, ld_words;
  uint32_t dim, units, blocks, groups;  // of a row
  uint32_t split;     // warps of a CTA that share a row's blocks
  uint32_t chunks;    // of NT * 8 queries
  uint64_t tiles;     // of a CTA's rows
  float alpha;
  const float* bias;
  void* out;
  int out_type;
  uint64_t ld;
  bool whole;         // four scores of a query can be written at once
};

// A chunk of queries as the kernel takes it: fragments (for each unit, N tile and
// part 16 bytes a lane), then per group the sums of the queries' values, then per
// query two powers of two whose product brings sums back.
template <int NT, int PARTS>
struct Laid {
  static constexpr uint32_t kUnitBytes = NT * PARTS * 512;
  __host__ __device__ static uint64_t frags(uint32_t units) { return (uint64_t)units * kUnitBytes; }
  __host__ __device__ static uint64_t sums(uint32_t groups) { return (uint64_t)groups * NT * 8 * 4; }
  __host__ __device__ static uint64_t bytes(uint32_t units, uint32_t groups) {
    return frags(units) + sums(groups) + NT * 8 * 8;
  }
};

__device__ inline float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // -126 <= e <= 127

// Column `col` of a chunk from query `x` (null: none, zeros), by one warp.
template <int NT, int PARTS, int G, typename T>
__device__ inline void lay_out(const T* x, uint32_t dim, uint32_t units, uint32_t groups, uint32_t col, uint8_t* to) {
  const uint32_t lane = threadIdx.x & 31;
  float* sums = (float*)(to + Laid<NT, PARTS>::frags(units));
  float* back = sums + groups * NT * 8;
  uint32_t top = 0;
  if (x)
    for (uint32_t d = lane; d < dim; d += 32) top = max(top, __float_as_uint(raven_fp8::load_value(x + d)) & 0x7fffffffu);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  const bool bad = top >= 0x7f800000u;
  const int e = top == 0 || bad ? 14 : 14 - (ilogbf(__uint_as_float(top)));  // -113 .. 163
  const float m0 = pow2(e / 2), m1 = pow2(e - e / 2);
  const bool none = x == nullptr || bad;
  constexpr uint32_t L = G / 8;
  const uint32_t n8 = (units * 4 + L - 1) / L * L;  // eights, up to whole groups
  for (uint32_t i0 = 0; i0 < n8; i0 += 32) {
    const uint32_t i = i0 + lane;
    float v[8], sum = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t d = 8 * i + k;
      v[k] = !none && d < dim ? raven_fp8::load_value(x + d) * m0 * m1 : 0.f;
      sum += v[k];
    }
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (i % L == 0 && i / L < groups) sums[i / L * (NT * 8) + col] = sum * 0x1p-24f;
    if (i < units * 4) {
      const uint32_t unit = i >> 2, at = (unit * NT + col / 8) * PARTS * 512 + ((col & 7) * 4 + (i & 3)) * 16;
      __align__(16) __half part[PARTS][8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float w = k & 1 ? v[k] * 0.0625f : v[k];
        const int s = (k & 3) * 2 + (k >> 2);
        part[0][s] = __float2half_rn(w);
        if constexpr (PARTS == 2) part[1][s] = __float2half_rn(w - __half2float(part[0][s]));
      }
#pragma unroll
      for (int p = 0; p < PARTS; ++p) *(uint4*)(to + at + p * 512) = *(const uint4*)part[p];
    }
  }
  if (lane == 0) {
    const int b = 24 - e;  // -139 .. 137
    back[2 * col] = bad ? __uint_as_float(0x7fc00000u) : pow2(b / 2);
    back[2 * col + 1] = pow2(b - b / 2);
  }
}

template <int NT, int PARTS, int G>
__device__ inline void lay_out_any(const Params& p, uint64_t query, uint32_t col, uint8_t* to) {
  const bool there = query < p.nq;
  const uint64_t at = query * p.ld_q;
  if (p.q_type == 0)
    lay_out<NT, PARTS, G>(there ? (const float*)p.q + at : nullptr, p.dim, p.units, p.groups, col, to);
  else if (p.q_type == 1)
    lay_out<NT, PARTS, G>(there ? (const __half*)p.q + at : nullptr, p.dim, p.units, p.groups, col, to);
  else
    lay_out<NT, PARTS, G>(there ? (const __nv_bfloat16*)p.q + at : nullptr, p.dim, p.units, p.groups, col, to);
}

// All chunks, a warp per column.
template <int NT, int PARTS, int G>
__global__ void __launch_bounds__(kThreads) lay_out_kernel(const Params p, uint8_t* to) {
  after_previous();
  const uint64_t w = (uint64_t)blockIdx.x * kWarps + threadIdx.x / 32;
  const uint64_t chunk = w / (NT * 8);
  if (chunk >= p.chunks) return;
  const uint32_t col = (uint32_t)(w - chunk * (NT * 8));
  lay_out_any<NT, PARTS, G>(p, w, col, to + chunk * Laid<NT, PARTS>::bytes(p.units, p.groups));
}

template <int B>
__device__ inline void copy_async(uint32_t to, const void* from) {
  if constexpr (B == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(to), "l"(from) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;\n" ::"r"(to), "l"(from), "n"(B) : "memory");
}
__device__ inline void copies_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N>
__device__ inline void copies_wait() {
  asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory");
}

__device__ inline void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <int NT, int PARTS, int G, bool HELD>
struct Smem {
  static constexpr uint32_t kWords = kBlock / G;                          // scale words of a row's block
  static constexpr uint32_t kStage = kMT * 2 * 512 + kRows * kWords * 4;  // codes, 16 bytes a lane and row; words by row
  static constexpr uint32_t kRing = kWarps * kDepth * kStage;
  static constexpr uint32_t kPart = 32 * 4 * kMT * NT * 4;                // a warp's sums
  __host__ __device__ static uint64_t bytes(uint32_t units, uint32_t groups, uint32_t split) {
    return kRing + (split > 1 ? kWarps * kPart : kWarps * 32 * 9 * 4) + (HELD ? Laid<NT, PARTS>::bytes(units, groups) : 0);
  }
};

template <typename T>
__device__ inline T rounded(float v) {
  if constexpr (std::is_same<T, float>::value)
    return v;
  else if constexpr (std::is_same<T, __half>::value)
    return __float2half_rn(v);
  else
    return __float2bfloat16_rn(v);
}

// HELD: the chunk's queries are in shared memory; else read through L1.
template <int NT, int PARTS, int G, bool HELD, typename O>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 2 : 1) score4_kernel(const Params p) {
  using S = Smem<NT, PARTS, G, HELD>;
  using Q = Laid<NT, PARTS>;
  extern __shared__ __align__(16) uint8_t smem[];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x / 32, g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem + warp * kDepth * S::kStage;
  float* scratch = (float*)(smem + S::kRing);
  const uint32_t scratch_bytes = p.split > 1 ? kWarps * S::kPart : kWarps * 32 * 9 * 4;
  uint8_t* held = smem + S::kRing + scratch_bytes;
  const uint32_t kw = warp % p.split, wr = warp / p.split, across = kWarps / p.split;
  const uint64_t chunk = blockIdx.x % p.chunks, step = gridDim.x / p.chunks;
  const uint64_t first = blockIdx.x / p.chunks;
  after_previous();

  // the ring: what is copied next
  uint64_t ahead = first;
  uint32_t ahead_b = kw, slot = 0;
  const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
  auto copy_next = [&]() {
    if (ahead < p.tiles) {
      const uint64_t row0 = (ahead * across + wr) * kRows;
      const uint32_t at = ring_at + slot * S::kStage;
      const uint32_t u = min(4u, p.units - 4 * ahead_b);
#pragma unroll
      for (int r = 0; r < 2 * kMT; ++r) {
        const uint64_t row = min(row0 + g * (2 * kMT) + r, p.n - 1);
        const uint8_t* from = p.codes + row * p.ld_codes + 64 * ahead_b + 4 * u * t;
        const uint32_t to = at + r * 512 + lane * 16;
        if (u == 4)
          copy_async<16>(to, from);
        else
          for (uint32_t w = 0; w < u; ++w) copy_async<4>(to + 4 * w, from + 4 * w);
        if (t == (uint32_t)r % 4)
          copy_async<4 * S::kWords>(at + kMT * 1024 + (g * 2 * kMT + r) * S::kWords * 4,
                                    p.words + row * p.ld_words + ahead_b * S::kWords);
      }
      ahead_b += p.split;
      if (ahead_b >= p.blocks) {
        ahead_b = kw;
        ahead += step;
      }
    }
    copies_commit();
    slot = slot + 1 == kDepth ? 0 : slot + 1;
  };
#pragma unroll
  for (int i = 0; i < kDepth - 1; ++i) copy_next();

  const uint8_t* laid = held;
  if constexpr (HELD) {
    if (p.q) {
      for (uint32_t col = warp; col < NT * 8; col += kWarps) lay_out_any<NT, PARTS, G>(p, chunk * NT * 8 + col, col, held);
    } else {
      const uint64_t bytes = Q::bytes(p.units, p.groups);
      const uint8_t* from = p.laid + chunk * bytes;
      for (uint64_t i = threadIdx.x * 16; i < bytes; i += kThreads * 16) *(uint4*)(held + i) = *(const uint4*)(from + i);
    }
    __syncthreads();
  } else {
    laid = p.laid + chunk * Q::bytes(p.units, p.groups);
  }
  const float* sums = (const float*)(laid + Q::frags(p.units));
  const float* back = sums + p.groups * NT * 8;

  uint32_t now = 0;  // the stage that is taken next
  for (uint64_t tile = first; tile < p.tiles; tile += step) {
    float total[kMT][NT][4] = {};
    for (uint32_t b = kw; b < p.blocks; b += p.split) {
      copies_wait<kDepth - 2>();
      __syncwarp();
      copy_next();  // into the stage that every lane is done with
      const uint8_t* stage = ring + now * S::kStage;
      now = now + 1 == kDepth ? 0 : now + 1;
      uint4 code[kMT][2];
#pragma unroll
      for (int r = 0; r < 2 * kMT; ++r) code[r / 2][r % 2] = *(const uint4*)(stage + r * 512 + lane * 16);
      const uint32_t* words = (const uint32_t*)(stage + kMT * 1024) + g * 2 * kMT * S::kWords;
      const uint32_t u = min(4u, p.units - 4 * b);
#pragma unroll
      for (uint32_t gi = 0; gi < S::kWords; ++gi) {
        constexpr uint32_t U = G / kUnit;
        if (gi * U < u) {
          float sc[kMT][2], acc[kMT][NT][4];
          const float* gs = sums + (b * S::kWords + gi) * (NT * 8) + 2 * t;
#pragma unroll
          for (int m = 0; m < kMT; ++m) {
            float z[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t w = words[(2 * m + h) * S::kWords + gi];
              sc[m][h] = raven_int4::step_of(w);
              z[h] = raven_int4::zero_of(w);
            }
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              const float2 x = *(const float2*)(gs + 8 * j);
              acc[m][j][0] = z[0] * x.x;
              acc[m][j][1] = z[0] * x.y;
              acc[m][j][2] = z[1] * x.x;
              acc[m][j][3] = z[1] * x.y;
            }
          }
#pragma unroll
          for (uint32_t uu = 0; uu < U; ++uu) {
            const uint32_t unit = gi * U + uu;
            if (unit < u) {
              uint32_t a[kMT][2][4];
#pragma unroll
              for (int m = 0; m < kMT; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  const uint32_t w = unit == 0   ? code[m][h].x
                                     : unit == 1 ? code[m][h].y
                                     : unit == 2 ? code[m][h].z
                                                 : code[m][h].w;
                  a[m][h][0] = w & 0x000f000fu;
                  a[m][h][1] = w & 0x00f000f0u;
                  a[m][h][2] = (w >> 8) & 0x000f000fu;
                  a[m][h][3] = (w >> 8) & 0x00f000f0u;
                }
              const uint8_t* f = laid + (uint64_t)(4 * b + unit) * Q::kUnitBytes + lane * 16;
#pragma unroll
              for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int q = PARTS - 1; q >= 0; --q) {
                  const uint4 x = *(const uint4*)(f + (j * PARTS + q) * 512);
#pragma unroll
                  for (int m = 0; m < kMT; ++m) {
                    mma(acc[m][j], a[m][0][0], a[m][1][0], a[m][0][1], a[m][1][1], x.x, x.y);
                    mma(acc[m][j], a[m][0][2], a[m][1][2], a[m][0][3], a[m][1][3], x.z, x.w);
                  }
                }
            }
          }
#pragma unroll
          for (int m = 0; m < kMT; ++m)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
              for (int i = 0; i < 4; ++i) total[m][j][i] = fmaf(sc[m][i / 2], acc[m][j][i], total[m][j][i]);
        }
      }
    }
    // the warps that shared the rows add up, the first one's sums last
    if (p.split > 1) {
      float* mine = scratch + warp * (S::kPart / 4) + lane;
      if (kw > 0) {
#pragma unroll
        for (int i = 0; i < kMT * NT * 4; ++i) mine[32 * i] = ((const float*)total)[i];
      }
      __syncthreads();
      if (kw == 0) {
        for (uint32_t k = 1; k < p.split; ++k)
#pragma unroll
          for (int i = 0; i < kMT * NT * 4; ++i) ((float*)total)[i] += mine[k * (S::kPart / 4) + 32 * i];
      }
      __syncthreads();
      if (kw > 0) continue;
    }
    // row m * 16 + g (+ 8) of the fragments is row g * 4 + 2 m (+ 1) of the tile: a lane holds four rows side by side
    const uint64_t row = (tile * across + wr) * kRows + g * (2 * kMT);
    float bias[2 * kMT];
#pragma unroll
    for (int r = 0; r < 2 * kMT; ++r) bias[r] = p.bias && row + r < p.n ? p.bias[row + r] : 0.f;
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const uint32_t col = 8 * j + 2 * t + c;
        const uint64_t query = chunk * NT * 8 + col;
        if (query >= p.nq) continue;
        const float b0 = back[2 * col], b1 = back[2 * col + 1];
        __align__(16) O v[2 * kMT];
#pragma unroll
        for (int r = 0; r < 2 * kMT; ++r) v[r] = rounded<O>(fmaf(p.alpha, total[r / 2][j][2 * (r % 2) + c] * b0 * b1, bias[r]));
        O* to = (O*)p.out + query * p.ld + row;
        if (p.whole && row + 2 * kMT <= p.n) {
          if constexpr (sizeof(O) == 4)
            *(uint4*)to = *(const uint4*)v;
          else
            *(uint2*)to = *(const uint2*)v;
        } else {
#pragma unroll
          for (int r = 0; r < 2 * kMT; ++r)
            if (row + r < p.n) to[r] = v[r];
        }
      }
  }
  copies_wait<0>();
}

}  // namespace raven_score4
