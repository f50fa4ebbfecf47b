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
// Two parts of an f32 query are two columns of the N side, added up at the end.
//
// What bounds it: reading the codes. Each warp has its own ring of tiles of 32 rows
// x 128 values in shared memory: one TMA copy of 2 KB, and a copy of 4 to 16 bytes
// a lane for the scale words. Where a CTA's tiles are few or large, warps share a
// tile's rows and take its blocks of 128 values in turn; their sums meet in shared
// memory and are added up in a fixed order.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>

#include "fp8.cuh"
#include "int4.cuh"
#include "internal.h"
#include "knn_tc.cuh"
#include "status.cuh"

namespace raven_score4 {

using raven_int4::kBlock;
using raven_int4::kUnit;
using raven_score::after_previous;
using raven_tc::mbar_expect_tx;
using raven_tc::mbar_init;
using raven_tc::smem_u32;
using raven_tc::tma_load_2d;

constexpr int kMT = 2;                // M tiles of a warp
constexpr uint32_t kRows = 16 * kMT;  // rows of a warp's tile
constexpr uint32_t kMaxDepth = 6;     // tiles under way per warp, at most

struct Params {
  const void* q;      // queries that each CTA lays out for itself, or null: `laid` holds them
  const uint8_t* laid;
  int q_type;         // 0 f32, 1 f16, 2 bf16
  uint64_t nq, ld_q;
  bool whole_q;       // 16 bytes of a query can be read at once
  const uint32_t* words;
  uint64_t n, ld_words;
  uint32_t dim, units, blocks, groups;  // of a row
  uint32_t split;     // warps that share a row's blocks
  uint32_t depth;     // of the rings
  uint32_t chunks;    // of the queries
  uint64_t tiles;     // of a CTA's rows
  float alpha;
  const float* bias;
  void* out;
  uint64_t ld;
  bool whole;         // four scores of a query can be written at once
  int* status;
};

// A chunk of queries as the kernel takes it, NT * 8 columns: fragments (for each
// unit and N tile 16 bytes a lane), then per group the columns' sums, then per
// column two powers of two whose product brings sums back. f32 queries have two
// columns side by side, the second for what the first leaves and without sums.
template <int NT>
struct Laid {
  static constexpr uint32_t kUnitBytes = NT * 512;
  __host__ __device__ static uint64_t frags(uint32_t units) { return (uint64_t)units * kUnitBytes; }
  __host__ __device__ static uint64_t sums(uint32_t groups) { return (uint64_t)groups * NT * 8 * 4; }
  __host__ __device__ static uint64_t bytes(uint32_t units, uint32_t groups) {
    return frags(units) + sums(groups) + NT * 8 * 8;
  }
};

__device__ inline float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // -126 <= e <= 127

template <typename T>
__device__ inline void eight(const T* x, uint32_t d, uint32_t dim, bool whole, float (&v)[8]) {
  if (whole && d + 8 <= dim) {
    __align__(16) T raw[8];
    ((uint4*)raw)[0] = *(const uint4*)(x + d);
    if constexpr (sizeof(T) == 4) ((uint4*)raw)[1] = *(const uint4*)(x + d + 4);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = raven_fp8::load_value(raw + k);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = d + k < dim ? raven_fp8::load_value(x + d + k) : 0.f;
  }
}

// Queries [first, first + count) as columns from `col` on, by all of a CTA's
// threads. top: `count` words of shared memory.
template <int NT, int G, typename T>
__device__ inline void lay_out(const Params& p, uint64_t first, uint32_t count, uint32_t col, uint8_t* to, uint32_t* top) {
  constexpr bool F32 = std::is_same<T, float>::value;
  constexpr uint32_t L = G / 8;
  float* sums = (float*)(to + Laid<NT>::frags(p.units));
  float* back = sums + p.groups * NT * 8;
  const uint32_t n8 = (p.units * 4 + L - 1) / L * L;  // eights, up to whole groups
  const uint32_t items = count * n8;
  auto load = [&](uint32_t q, uint32_t i, float(&v)[8]) {
    if (first + q < p.nq) {
      eight((const T*)p.q + (first + q) * p.ld_q, 8 * i, p.dim, p.whole_q, v);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = 0.f;
    }
  };
  for (uint32_t i = threadIdx.x; i < count; i += blockDim.x) top[i] = 0;
  __syncthreads();
  for (uint32_t u = threadIdx.x; u < items; u += blockDim.x) {
    const uint32_t q = u / n8;
    float v[8];
    load(q, u - q * n8, v);
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) m = max(m, __float_as_uint(v[k]) & 0x7fffffffu);
    atomicMax(&top[q], m);
  }
  __syncthreads();
  for (uint32_t u0 = 0; u0 < items; u0 += blockDim.x) {
    const uint32_t u = u0 + threadIdx.x, q = min(u / n8, count - 1), i = u - q * n8;  // past the last item: past the last unit
    const bool bad = top[q] >= 0x7f800000u;
    const int e = top[q] == 0 || bad ? 14 : 14 - ilogbf(__uint_as_float(top[q]));  // -113 .. 163
    const float m0 = pow2(e / 2), m1 = pow2(e - e / 2);
    float v[8], sum = 0.f;
    load(q, i, v);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      v[k] = bad ? 0.f : v[k] * m0 * m1;
      sum += v[k];
    }
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const uint32_t c = col + (F32 ? 2 * q : q);
    if (i % L == 0 && i / L < p.groups) {
      sums[i / L * (NT * 8) + c] = sum * 0x1p-24f;
      if (F32) sums[i / L * (NT * 8) + c + 1] = 0.f;
    }
    if (i < p.units * 4) {
      __align__(16) __half part[F32 ? 2 : 1][8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float w = k & 1 ? v[k] * 0.0625f : v[k];
        const int s = (k & 3) * 2 + (k >> 2);
        part[0][s] = __float2half_rn(w);
        if constexpr (F32) part[1][s] = __float2half_rn(w - __half2float(part[0][s]));
      }
#pragma unroll
      for (int h = 0; h < (F32 ? 2 : 1); ++h)
        *(uint4*)(to + ((i >> 2) * NT + (c + h) / 8) * 512 + (((c + h) & 7) * 4 + (i & 3)) * 16) = *(const uint4*)part[h];
    }
    if (i == 0) {
      const int b = 24 - e;  // -139 .. 137
#pragma unroll
      for (int h = 0; h < (F32 ? 2 : 1); ++h) {
        back[2 * (c + h)] = bad ? __uint_as_float(0x7fc00000u) : pow2(b / 2);
        back[2 * (c + h) + 1] = pow2(b - b / 2);
      }
    }
  }
}

template <int NT, int G, bool F32>
__device__ inline void lay_out_any(const Params& p, uint64_t first, uint32_t count, uint32_t col, uint8_t* to, uint32_t* top) {
  if constexpr (F32)
    lay_out<NT, G, float>(p, first, count, col, to, top);
  else if (p.q_type == 1)
    lay_out<NT, G, __half>(p, first, count, col, to, top);
  else
    lay_out<NT, G, __nv_bfloat16>(p, first, count, col, to, top);
}

// All chunks, a CTA per query.
template <int NT, int G, bool F32>
__global__ void __launch_bounds__(256) lay_out_kernel(const Params p, uint8_t* to) {
  constexpr uint32_t Q = F32 ? NT * 4 : NT * 8;
  __shared__ uint32_t top[1];
  after_previous();
  const uint32_t chunk = blockIdx.x / Q, q = blockIdx.x - chunk * Q;
  lay_out_any<NT, G, F32>(p, blockIdx.x, 1, F32 ? 2 * q : q, to + chunk * Laid<NT>::bytes(p.units, p.groups), top);
}

template <int B>
__device__ inline void copy_async(uint32_t to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;\n" ::"r"(to), "l"(from), "n"(B) : "memory");
}
// Arrives at the barrier when this thread's copies have landed.
__device__ inline void copies_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];\n" ::"r"(bar) : "memory");
}
// Waits for a phase of the barrier; false after about two seconds.
__device__ inline bool wait(uint32_t bar, uint32_t parity) {
  auto done = [&]() {
    uint32_t d;
    asm volatile(
        "{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(d)
        : "r"(bar), "r"(parity)
        : "memory");
    return d != 0;
  };
  if (done()) return true;
  const long long t0 = clock64();
  while (clock64() - t0 < raven_tc::kWaitCycles)
    if (done()) return true;
  return false;
}
__device__ inline void meet(uint32_t id, uint32_t threads) {
  asm volatile("bar.sync %0, %1;\n" ::"r"(id), "r"(threads) : "memory");
}

__device__ inline void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <int NT, int G>
struct Layout {
  static constexpr uint32_t kWarps = NT <= 2 ? 16 : 8;    // as many as their registers allow
  static constexpr uint32_t kThreads = kWarps * 32;
  static constexpr uint32_t kWords = kBlock / G;          // scale words of a row's block
  static constexpr uint32_t kCodeBytes = kRows * 64, kWordBytes = kRows * kWords * 4;
  static constexpr uint32_t kPart = 32 * 4 * kMT * NT * 4;  // a warp's sums
  static constexpr uint32_t kBars = kWarps * kMaxDepth * 8;  // in front of the rings
  static constexpr uint32_t kTops = NT * 8 * 4;
  __host__ __device__ static uint64_t ring(uint32_t depth) { return (uint64_t)kWarps * depth * (kCodeBytes + kWordBytes); }
  __host__ __device__ static uint64_t shared(uint32_t split) { return split > 1 ? kWarps * kPart : 0; }
  __host__ __device__ static uint64_t bytes(uint32_t units, uint32_t groups, uint32_t split, uint32_t depth, bool held) {
    return kBars + ring(depth) + kTops + shared(split) + (held ? Laid<NT>::bytes(units, groups) : 0);
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
template <int NT, int G, bool F32, bool HELD, typename O>
__global__ void __launch_bounds__(Layout<NT, G>::kThreads, 1) score4_kernel(const __grid_constant__ CUtensorMap map,
                                                                            const Params p) {
  using S = Layout<NT, G>;
  using Q = Laid<NT>;
  constexpr uint32_t kQueries = F32 ? NT * 4 : NT * 8;
  extern __shared__ __align__(128) uint8_t smem[];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x / 32, g = lane >> 2, t = lane & 3, odd = g & 1;
  const uint32_t bars = smem_u32(smem) + warp * kMaxDepth * 8;
  uint8_t* codes = smem + S::kBars + warp * p.depth * S::kCodeBytes;
  uint8_t* words = smem + S::kBars + S::kWarps * p.depth * S::kCodeBytes + warp * p.depth * S::kWordBytes;
  uint8_t* after = smem + S::kBars + S::ring(p.depth);
  uint32_t* tops = (uint32_t*)after;
  float* shared = (float*)(after + S::kTops);
  uint8_t* held = after + S::kTops + S::shared(p.split);
  const uint32_t kw = warp % p.split, wr = warp / p.split, across = S::kWarps / p.split;
  const uint64_t chunk = blockIdx.x % p.chunks, step = gridDim.x / p.chunks, first = blockIdx.x / p.chunks;
  const uint32_t pitch = min(64u, 16 * p.units);  // of a tile's rows of codes
  if (lane < p.depth) mbar_init(bars + 8 * lane, 33);
  asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  __syncwarp();
  after_previous();

  // the ring: what is copied next
  uint64_t ahead = first;
  uint32_t ahead_b = kw, slot = 0, pending = 0;
  const uint32_t codes_at = smem_u32(codes), words_at = smem_u32(words);
  auto copy_next = [&]() {
    if (ahead < p.tiles) {
      const uint64_t row0 = (ahead * across + wr) * kRows;
      const uint32_t bar = bars + 8 * slot;
      copy_async<4 * S::kWords>(words_at + slot * S::kWordBytes + lane * (4 * S::kWords),
                                p.words + min(row0 + lane, p.n - 1) * p.ld_words + ahead_b * S::kWords);
      copies_arrive(bar);
      if (lane == 0) {
        mbar_expect_tx(bar, kRows * pitch);
        tma_load_2d(codes_at + slot * S::kCodeBytes, &map, (int)(64 * ahead_b), (int)min(row0, p.n), bar);
      }
      pending |= 1u << slot;
      slot = slot + 1 == p.depth ? 0 : slot + 1;
      ahead_b += p.split;
      if (ahead_b >= p.blocks) {
        ahead_b = kw;
        ahead += step;
      }
    }
  };
  for (uint32_t i = 0; i + 1 < p.depth; ++i) copy_next();

  const uint8_t* laid = held;
  if constexpr (HELD) {
    if (p.q) {
      lay_out_any<NT, G, F32>(p, chunk * kQueries, kQueries, 0, held, tops);
    } else {
      const uint32_t bytes = (uint32_t)Q::bytes(p.units, p.groups);
      const uint8_t* from = p.laid + chunk * bytes;
      for (uint32_t i = threadIdx.x * 16; i < bytes; i += S::kThreads * 16) *(uint4*)(held + i) = *(const uint4*)(from + i);
    }
    __syncthreads();
  } else {
    laid = p.laid + chunk * Q::bytes(p.units, p.groups);
  }
  const float* sums = (const float*)(laid + Q::frags(p.units));
  const float* back = sums + p.groups * NT * 8;

  bool ok = true;  // no wait has run out
  uint32_t now = 0, phases = 0;  // the stage that is taken next; parities of the stages
  // row m * 16 + g (+ 8) of the fragments is row 8 (g / 2) + g % 2 + 4 m (+ 2) of the tile: two lanes next to one
  // another in g read 128 bytes side by side
  const uint32_t my_row = 8 * (g >> 1) + odd;
  for (uint64_t tile = first; tile < p.tiles; tile += step) {
    float total[kMT][NT][4] = {};
    for (uint32_t b = kw; b < p.blocks; b += p.split) {
      if (ok && !__all_sync(0xffffffffu, wait(bars + 8 * now, phases >> now & 1u))) {
        ok = false;
        if (lane == 0) raven_score::tell(p.status, raven_score::kStatusWait);
      }
      if (!ok) continue;  // but meets the warps it shares rows with
      __syncwarp();
      const uint8_t* stage = codes + now * S::kCodeBytes;
      const uint32_t* word = (const uint32_t*)(words + now * S::kWordBytes) + my_row * S::kWords;
      phases ^= 1u << now;
      pending &= ~(1u << now);
      now = now + 1 == p.depth ? 0 : now + 1;
      copy_next();  // into the stage that every lane is done with
      const uint32_t u = min(4u, p.units - 4 * b);
      uint4 code[kMT][2];
      if (u == 4) {
#pragma unroll
        for (int r = 0; r < 2 * kMT; ++r) code[r / 2][r % 2] = *(const uint4*)(stage + (my_row + 2 * r) * 64 + 16 * t);
      } else {
#pragma unroll
        for (int r = 0; r < 2 * kMT; ++r) {
          const uint32_t* c = (const uint32_t*)(stage + (my_row + 2 * r) * pitch + 4 * u * t);
          code[r / 2][r % 2] = make_uint4(c[0], u > 1 ? c[1] : 0, u > 2 ? c[2] : 0, 0);
        }
      }
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
              const uint32_t w = word[(4 * m + 2 * h) * S::kWords + gi];
              sc[m][h] = raven_int4::step_of(w);
              z[h] = raven_int4::zero_of(w);
            }
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              const float2 x = *(const float2*)(gs + 8 * j);
              acc[m][j][0] = z[0] * x.x;
              acc[m][j][2] = z[1] * x.x;
              acc[m][j][1] = F32 ? 0.f : z[0] * x.y;
              acc[m][j][3] = F32 ? 0.f : z[1] * x.y;
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
              const uint8_t* f = laid + (4 * b + unit) * Q::kUnitBytes + lane * 16;
#pragma unroll
              for (int j = 0; j < NT; ++j) {
                const uint4 x = *(const uint4*)(f + j * 512);
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
    // The sums of a column (of two, F32) for this lane's four rows, from one warp after the other where several
    // shared them; lanes next to one another in g swap two, so that each has four rows side by side.
    const uint64_t row = (tile * across + wr) * kRows + 4 * g;
    float* mine = shared + warp * (S::kPart / 4) + lane;
    if (p.split > 1) {
#pragma unroll
      for (int i = 0; i < kMT * NT * 4; ++i) mine[32 * i] = total[i / (4 * NT)][i / 4 % NT][i % 4];
      meet(1 + wr, 32 * p.split);
    }
    const float* theirs = shared + wr * p.split * (S::kPart / 4) + lane;
    float bias[2 * kMT];
#pragma unroll
    for (int r = 0; r < 2 * kMT; ++r) bias[r] = p.bias && row + r < p.n ? p.bias[row + r] : 0.f;
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int c = 0; c < (F32 ? 1 : 2); ++c) {
        float v[2 * kMT];
        if (p.split > 1) {
          if ((j * (F32 ? 1 : 2) + c) % p.split != kw) continue;
#pragma unroll
          for (int r = 0; r < 2 * kMT; ++r) v[r] = 0.f;
          for (uint32_t k = 0; k < p.split; ++k) {
            const float* from = theirs + k * (S::kPart / 4);
#pragma unroll
            for (int r = 0; r < 2 * kMT; ++r) {
              const float* x = from + 32 * (((r / 2) * NT + j) * 4 + 2 * (r % 2) + c);
              v[r] += F32 ? x[0] + x[32] : x[0];
            }
          }
        } else {
#pragma unroll
          for (int r = 0; r < 2 * kMT; ++r)
            v[r] = F32 ? total[r / 2][j][2 * (r % 2)] + total[r / 2][j][2 * (r % 2) + 1] : total[r / 2][j][2 * (r % 2) + c];
        }
        const float s0 = __shfl_xor_sync(0xffffffffu, odd ? v[0] : v[2], 4), s1 = __shfl_xor_sync(0xffffffffu, odd ? v[1] : v[3], 4);
        const float y[4] = {odd ? s0 : v[0], odd ? v[2] : s0, odd ? s1 : v[1], odd ? v[3] : s1};
        const uint32_t col = 8 * j + 2 * t + c;
        const uint64_t query = chunk * kQueries + (F32 ? col / 2 : col);
        if (query < p.nq) {
          const float b0 = back[2 * col], b1 = back[2 * col + 1];
          __align__(16) O o[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) o[r] = rounded<O>(fmaf(p.alpha, y[r] * b0 * b1, bias[r]));
          O* to = (O*)p.out + query * p.ld + row;
          if (p.whole && row + 4 <= p.n) {
            if constexpr (sizeof(O) == 4)
              *(uint4*)to = *(const uint4*)o;
            else
              *(uint2*)to = *(const uint2*)o;
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (row + r < p.n) to[r] = o[r];
          }
        }
      }
    if (p.split > 1) meet(1 + wr, 32 * p.split);
  }
  // a wait ran out: no copy is under way any more when the CTA ends
  if (!ok)
    for (uint32_t i = 0; i < p.depth; ++i)
      if (pending >> i & 1u) wait(bars + 8 * i, phases >> i & 1u);
}

}  // namespace raven_score4
