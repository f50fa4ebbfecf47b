// Scores of queries against 4-bit rows (int4.cuh has their layout):
//
//   S[i, j] = alpha * sum_g step_jg ((z_jg + 8) sum_k q_ik + sum_k (code_jk - 8) q_ik) + bias[j]
//
// The inner sums run on the tensor cores (here mma m16n8k16, f16 operands, f32 sums)
// with rows as the M side and queries as the N side. 4 bits at the bottom of the f16
// 1024 (times 2^-12, see below) are 1024 + code, at bits 4-7 1024 + 16 code: one LOP3 and one
// f16 addition (or multiply-add) make code - 8 of two codes, nine instructions per eight. Without the
// additions the 4 bits alone are an f16 too, a subnormal, but the tensor cores line
// products up by their exponent fields and drop what is below the sum's bits, and
// subnormals lose as many of them as they have leading zeros: scores were off by 1e-6
// to 2.3e-6 of their size. What a fragment's lane holds of K is free as long as both
// sides agree: lane t of a row's four takes the eight values 8t.. of each unit of 32
// (one word), as pairs (0, 4), (1, 5), (2, 6), (3, 7).
//
// Queries are brought to a largest magnitude in [2^14, 2^15) (less for rows of more
// than 4096 values) by a power of two each, so that f16 holds what f32, f16 and bf16
// values may be: 11 bits of a value in one part, 22 in two (f32), nothing below 2^-39
// of the largest (2^-35 in the longest rows). The sum of a
// group starts at (z + 8) * sum(q), and its step is applied in f32 when the group
// ends: the scale is never rounded into an operand. Two parts of an f32 query are two
// columns of the N side, added up at the end.
//
// What bounds it: no unit by itself. The 16 warps that an SM's registers hold issue in
// 54 to 59 % of the slots, half of that to turn codes into operands, and wait for one
// another's results in the others (1 x 1000000 x 128 24 us, 3.0 TB/s; 8 x 65536 x 1024
// 15 us, 2.5 TB/s), so what is around the operands is kept small. Each warp has its own ring of tiles of 32 or 64
// rows x 128 values in shared memory: one TMA copy of 2 or 4 KB, and a copy of 4 to
// 16 bytes a row for the scale words. Where a CTA's tiles are few or large, warps
// share a tile's rows and take its blocks of 128 values in turn; their sums meet in
// shared memory and are added up in a fixed order. A CTA holds its queries in shared
// memory; where rows are too long for that, CTAs take slices of them, and a second
// kernel adds up their sums.
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

// A row's sum is kept times 2^-28, and a query is brought to a largest magnitude in [2^14, 2^15), in rows of more than
// 4096 values to one lower by what they have more (2^10 for 65536): of dim products with values below 2^128 (a little
// above where a group goes from f32's lowest to its largest) it is at most 2^127 then, whatever the values are and
// however they cancel. It is brought to the score's size at the very end. Of the 2^-28 the operands take 2^-12 (code - 8
// and code + z are whole numbers of 8 bits: f16 holds them as well times that), which costs nothing, and the steps
// 2^-16, so that a step, of 16 significant bits, is exact down to 2^-118. A group's addition to a sum loses what is
// below 2^-136 of a query's largest value (2^-132 in the longest rows).
constexpr int kCodeShift = 12, kStepShift = 16;
constexpr float kCodeScale = 1.f / (1 << kCodeShift);
constexpr uint32_t kCodeBase = 0x34003400u;  // the f16 1024 * 2^-12, twice: 4 bits at its bottom are a code * 2^-12 more
constexpr uint32_t kMaxDepth = 6;  // tiles under way per warp, at most

struct Params {
  const void* q;      // queries that each CTA lays out for itself, or null: `laid` holds them
  const uint8_t* laid;
  int q_type;         // 0 f32, 1 f16, 2 bf16
  uint64_t nq, ld_q;
  bool whole_q;       // 16 bytes of a query can be read at once
  const uint32_t* words;
  uint64_t n, ld_words;
  uint32_t dim, units, blocks, groups;  // of a row
  uint32_t slices;    // of a row's blocks, `slice` blocks each but the last
  uint32_t slice;
  uint32_t split;     // warps that share a row's blocks
  uint32_t depth;     // of the rings
  uint32_t chunks;    // of the queries
  uint32_t tiles;     // of a CTA's rows
  float alpha;        // times 2^alpha_exp; 1 to 2 in size, or 0 or not finite
  int alpha_exp;
  int top;            // queries are brought to a largest magnitude in [2^top, 2^(top + 1))
  const float* bias;
  void* out;          // of slice s at out + s * ld_slice: sums as they are kept
  uint64_t ld, ld_slice;
  float4* backs;      // of slices: what brings each query's sums back, or null
  bool whole;         // four scores of a query can be written at once
  int* status;
};

// A chunk of queries as the kernel takes it, NT * 8 columns: fragments (for each
// unit and N tile 16 bytes a lane), then per group the columns' sums, then per
// query what brings its sums back, alpha times a power of two: as one factor, or
// where that is near the ends of f32's range as three. f32 queries have two
// columns side by side, the second for what the first leaves and without sums.
template <int NT>
struct Laid {
  static constexpr uint32_t kColumns = NT * 8;
  static constexpr uint32_t kUnitBytes = NT * 512;
  __host__ __device__ static uint64_t frags(uint32_t units) { return (uint64_t)units * kUnitBytes; }
  __host__ __device__ static uint64_t sums(uint32_t groups) { return (uint64_t)groups * NT * 8 * 4; }
  __host__ __device__ static uint64_t bytes(uint32_t units, uint32_t groups) {
    return frags(units) + sums(groups) + NT * 8 * 16;
  }
  // Where a quarter of a unit of a column is; a group's sum, where `to` are the sums.
  __device__ static uint32_t frag_at(uint32_t unit, uint32_t quarter, uint32_t col) {
    return (unit * NT + col / 8) * 512 + ((col & 7) * 4 + quarter) * 16;
  }
  __device__ static void put_sum(uint8_t* to, uint32_t group, uint32_t col, float sum) {
    ((float*)to)[group * (NT * 8) + col] = sum;
  }
  // What brings query q's sums back: three factors, whether the last two are not 1.
  __device__ static void put_back(float* back, uint32_t q, float f, float k0, float k1, float flag) {
    *(float4*)(back + 4 * q) = make_float4(f, k0, k1, flag);
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
// threads: of their values a slice of whole blocks, `units` from unit `unit0` on
// with so many groups. top: `count` words of shared memory.
template <class Q, int G, typename T>
__device__ inline void lay_out(const Params& p, uint64_t first, uint32_t count, uint32_t col, uint32_t unit0, uint32_t units,
                               uint32_t groups, uint8_t* to, uint32_t* top) {
  constexpr bool F32 = std::is_same<T, float>::value;
  constexpr uint32_t L = G / 8;
  uint8_t* sums = to + Q::frags(units);
  float* back = (float*)(sums + Q::sums(groups));
  const uint32_t all = (p.dim + 7) / 8, n8 = (units * 4 + L - 1) / L * L;  // eights: of a query, of the slice up to whole groups
  const uint32_t there = (uint32_t)min((uint64_t)count, p.nq > first ? p.nq - first : 0);
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
  for (uint32_t u0 = 0; u0 < there * all; u0 += blockDim.x) {
    const uint32_t u = u0 + threadIdx.x, q = min(u / all, there - 1);
    uint32_t m = 0;
    if (u < there * all) {
      float v[8];
      load(q, u - q * all, v);
#pragma unroll
      for (int k = 0; k < 8; ++k) m = max(m, __float_as_uint(v[k]) & 0x7fffffffu);
    }
    // one of a warp's lanes where they have one query
    if (__all_sync(0xffffffffu, q == __shfl_sync(0xffffffffu, q, 0))) {
      m = __reduce_max_sync(0xffffffffu, m);
      if ((threadIdx.x & 31) == 0) atomicMax(&top[q], m);
    } else {
      atomicMax(&top[q], m);
    }
  }
  __syncthreads();
  for (uint32_t u0 = 0; u0 < count * n8; u0 += blockDim.x) {
    const uint32_t u = u0 + threadIdx.x, q = min(u / n8, count - 1), i = u - q * n8;  // past the last item: past the last unit
    const bool bad = top[q] >= 0x7f800000u;
    const int e = top[q] == 0 || bad ? p.top : p.top - ilogbf(__uint_as_float(top[q]));  // -117 .. 163
    const float m0 = pow2(e / 2), m1 = pow2(e - e / 2);
    float v[8], sum = 0.f;
    load(q, 4 * unit0 + i, v);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      v[k] = bad ? 0.f : v[k] * m0 * m1;
      sum += v[k];
    }
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const uint32_t c = col + (F32 ? 2 * q : q);
    if (i % L == 0 && i / L < groups) {
      Q::put_sum(sums, i / L, c, sum * kCodeScale);
      if (F32) Q::put_sum(sums, i / L, c + 1, 0.f);
    }
    if (i < units * 4) {
      __align__(16) __half part[F32 ? 2 : 1][8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float w = v[k];
        const int s = (k & 3) * 2 + (k >> 2);
        part[0][s] = __float2half_rn(w);
        if constexpr (F32) part[1][s] = __float2half_rn(w - __half2float(part[0][s]));
      }
#pragma unroll
      for (int h = 0; h < (F32 ? 2 : 1); ++h)
        *(uint4*)(to + Q::frag_at(i >> 2, i & 3, c + h)) = *(const uint4*)part[h];
    }
    if (i == 0) {
      // Three factors of one third of the exponent each, so all on one side of 1: a product in between is
      // subnormal only where the score is nearer to 0 still, and infinite only where the score is. With alpha last a
      // sum of 1e-43 would have lost its bits.
      const int by = p.alpha_exp + kCodeShift + kStepShift - e;  // -284 .. 272
      const bool plain = bad || (by >= -120 && by <= 120);
      const int third = plain ? 0 : by / 3;
      const float k = pow2(third), f = bad ? __uint_as_float(0x7fc00000u) : p.alpha * pow2(by - 2 * third);
      if (p.backs) {  // the join brings sums back; CTAs that have this query write the same
        p.backs[first + q] = make_float4(f, k, k, plain ? 0.f : 1.f);
        Q::put_back(back, F32 ? c / 2 : c, 1.f, 1.f, 1.f, 0.f);
      } else {
        Q::put_back(back, F32 ? c / 2 : c, f, k, k, plain ? 0.f : 1.f);
      }
    }
  }
}

template <class Q, int G, bool F32>
__device__ inline void lay_out_any(const Params& p, uint64_t first, uint32_t count, uint32_t col, uint32_t unit0, uint32_t units,
                                   uint32_t groups, uint8_t* to, uint32_t* top) {
  if constexpr (F32)
    lay_out<Q, G, float>(p, first, count, col, unit0, units, groups, to, top);
  else if (p.q_type == 1)
    lay_out<Q, G, __half>(p, first, count, col, unit0, units, groups, to, top);
  else
    lay_out<Q, G, __nv_bfloat16>(p, first, count, col, unit0, units, groups, to, top);
}

// All chunks, a CTA per query.
template <class Q, int G, bool F32>
__global__ void __launch_bounds__(256) lay_out_kernel(const Params p, uint8_t* to) {
  constexpr uint32_t kQueries = F32 ? Q::kColumns / 2 : Q::kColumns;
  __shared__ uint32_t top[1];
  after_previous();
  const uint32_t chunk = blockIdx.x / kQueries, q = blockIdx.x - chunk * kQueries;
  lay_out_any<Q, G, F32>(p, blockIdx.x, 1, F32 ? 2 * q : q, 0, p.units, p.groups, to + chunk * Q::bytes(p.units, p.groups), top);
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

// Eight codes less 8, times 2^-12, as four operands of two.
__device__ inline void operands(uint32_t w, uint32_t& a0, uint32_t& a1, uint32_t& a2, uint32_t& a3) {
  auto low = [](uint32_t code) {
    const __half2 r = __hadd2(*(const __half2*)&code, __float2half2_rn(-1032.f * kCodeScale));
    return *(const uint32_t*)&r;
  };
  auto high = [](uint32_t code) {
    const __half2 r = __hfma2(*(const __half2*)&code, __float2half2_rn(0.0625f), __float2half2_rn(-72.f * kCodeScale));
    return *(const uint32_t*)&r;
  };
  const uint32_t v = w >> 8;
  a0 = low((w & 0x000f000fu) | kCodeBase);
  a1 = high((w & 0x00f000f0u) | kCodeBase);
  a2 = low((v & 0x000f000fu) | kCodeBase);
  a3 = high((v & 0x00f000f0u) | kCodeBase);
}

__device__ inline void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <int NT, int MT, int G>  // MT: M tiles of a warp, as many as its registers allow
struct Layout {
  static constexpr int kAtOnce = NT == 1 ? 1 : MT;       // M tiles that go through a block together
  static constexpr uint32_t kRows = 16 * MT;             // rows of its tile
  static constexpr uint32_t kWarps = 16;
  static constexpr uint32_t kThreads = kWarps * 32;
  static constexpr uint32_t kWords = kBlock / G;          // scale words of a row's block
  static constexpr uint32_t kCodeBytes = kRows * 64, kWordBytes = kRows * kWords * 4;
  static constexpr uint32_t kPart = 32 * 4 * MT * NT * 4;  // a warp's sums
  static constexpr uint32_t kBars = kWarps * kMaxDepth * 8;  // in front of the rings
  static constexpr uint32_t kTops = NT * 8 * 4;
  static_assert(kBars % 128 == 0 && kCodeBytes % 128 == 0, "a TMA copy's place in shared memory");
  static constexpr uint32_t kLeast = MT == 4 ? 2 : 3;      // stages of a ring
  // what every call needs: rings, a block of queries, sums that meet
  static_assert(kBars + kLeast * (uint64_t)kWarps * (kCodeBytes + kWordBytes) + kTops + kWarps * kPart + 4 * Laid<NT>::kUnitBytes +
                kWords * NT * 32 + NT * 64 <= 227 * 1024, "shared memory of a CTA");
  __host__ __device__ static uint64_t ring(uint32_t depth) { return (uint64_t)kWarps * depth * (kCodeBytes + kWordBytes); }
  __host__ __device__ static uint64_t shared(uint32_t split) { return split > 1 ? kWarps * kPart : 0; }
  __host__ __device__ static uint64_t bytes(uint32_t units, uint32_t groups, uint32_t split, uint32_t depth) {
    return kBars + ring(depth) + kTops + shared(split) + Laid<NT>::bytes(units, groups);
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

template <int NT, int MT, int G, bool F32, typename O>
__global__ void __launch_bounds__(Layout<NT, MT, G>::kThreads, 1) score4_kernel(const __grid_constant__ CUtensorMap map,
                                                                            const Params p) {
  using S = Layout<NT, MT, G>;
  using Q = Laid<NT>;
  constexpr int R = 2 * MT;  // rows of a lane
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
  // this CTA's queries, slice of the blocks, tiles
  const uint32_t shares = p.chunks * p.slices, share = blockIdx.x % shares;
  const uint32_t step = gridDim.x / shares, first = blockIdx.x / shares;
  const uint32_t slice = share % p.slices;
  const uint64_t chunk = share / p.slices;
  const uint32_t b0 = slice * p.slice, blocks = min(p.slice, p.blocks - b0);
  const uint32_t pitch = min(64u, 16 * p.units);  // of a tile's rows of codes
  if (lane < p.depth) mbar_init(bars + 8 * lane, 33);
  asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  __syncwarp();
  after_previous();

  // the ring: what is copied next
  uint32_t ahead = first, ahead_b = kw, slot = 0, pending = 0;
  const uint32_t codes_at = smem_u32(codes), words_at = smem_u32(words) + lane * (4 * S::kWords);
  int ahead_y = 0;
  const uint32_t* ahead_words[S::kRows / 32];
  auto aim = [&]() {
    const uint64_t row0 = ((uint64_t)ahead * across + wr) * S::kRows;
    ahead_y = (int)min(row0, p.n);
#pragma unroll
    for (uint32_t i = 0; i < S::kRows / 32; ++i)
      ahead_words[i] = p.words + min(row0 + lane + 32 * i, p.n - 1) * p.ld_words + b0 * S::kWords;
  };
  auto copy_next = [&]() {
    if (ahead < p.tiles) {
      const uint32_t bar = bars + 8 * slot;
#pragma unroll
      for (uint32_t i = 0; i < S::kRows / 32; ++i)
        copy_async<4 * S::kWords>(words_at + slot * S::kWordBytes + i * (128 * S::kWords), ahead_words[i] + ahead_b * S::kWords);
      copies_arrive(bar);
      if (lane == 0) {
        mbar_expect_tx(bar, S::kRows * pitch);
        tma_load_2d(codes_at + slot * S::kCodeBytes, &map, (int)(64 * (b0 + ahead_b)), ahead_y, bar);
      }
      pending |= 1u << slot;
      slot = slot + 1 == p.depth ? 0 : slot + 1;
      ahead_b += p.split;
      if (ahead_b >= blocks) {
        ahead_b = kw;
        ahead += step;
        aim();
      }
    }
  };
  if (kw >= blocks) ahead = p.tiles;  // a last slice of fewer blocks than warps
  aim();
  for (uint32_t i = 0; i + 1 < p.depth; ++i) copy_next();

  const uint32_t units = min(4 * p.slice, p.units - 4 * b0), groups = min(p.slice * S::kWords, p.groups - b0 * S::kWords);
  float* sums = (float*)(held + Q::frags(units));
  float* back = sums + groups * NT * 8;
  if (p.q) {
    lay_out_any<Q, G, F32>(p, chunk * kQueries, kQueries, 0, 4 * b0, units, groups, held, tops);
  } else {
    const uint8_t* from = p.laid + chunk * Q::bytes(p.units, p.groups);
    auto bring = [&](void* to, const uint8_t* what, uint32_t bytes) {
      for (uint32_t i = threadIdx.x * 16; i < bytes; i += S::kThreads * 16)
        *(uint4*)((uint8_t*)to + i) = *(const uint4*)(what + i);
    };
    bring(held, from + Q::frags(4 * b0), (uint32_t)Q::frags(units));
    from += Q::frags(p.units);
    bring(sums, from + Q::sums(b0 * S::kWords), (uint32_t)Q::sums(groups));
    bring(back, from + Q::sums(p.groups), NT * 8 * 16);
  }
  __syncthreads();
  bool plain = true;  // every column has one factor
  for (uint32_t q = 0; q < kQueries; ++q) plain &= back[4 * q + 3] == 0.f;

  bool ok = true;  // no wait has run out
  uint32_t now = 0, phases = 0;  // the stage that is taken next; parities of the stages
  // Row 16 m + g (+ 8) of the fragments is row R (g / 2) * 2 + g % 2 + 4 m (+ 2) of the tile: two lanes next to one
  // another in g read 128 bytes side by side.
  const uint32_t my_row = 2 * R * (g >> 1) + odd;
  for (uint32_t tile = first; tile < p.tiles; tile += step) {
    float total[MT][NT][4] = {};
    auto block = [&](auto full, const uint8_t* stage, const uint32_t* word, uint32_t b, uint32_t u) {
      constexpr bool FULL = decltype(full)::value;
      constexpr int MG = S::kAtOnce;  // M tiles at once
      uint4 x[4][NT];                 // the queries' fragments
      auto fetch = [&](uint32_t unit) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
          if (FULL || unit < u) x[unit][j] = *(const uint4*)(held + (4 * b + unit) * Q::kUnitBytes + lane * 16 + j * 512);
      };
      if constexpr (MG < MT) {
#pragma unroll
        for (uint32_t unit = 0; unit < 4; ++unit) fetch(unit);
      }
#pragma unroll
      for (int m0 = 0; m0 < MT; m0 += MG) {
        uint4 code[MG][2];
#pragma unroll
        for (int m = 0; m < MG; ++m)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t r = my_row + 4 * (m0 + m) + 2 * h;
            if constexpr (FULL) {
              code[m][h] = *(const uint4*)(stage + r * 64 + 16 * t);
            } else {
              const uint32_t* c = (const uint32_t*)(stage + r * pitch + 4 * u * t);
              code[m][h] = make_uint4(c[0], u > 1 ? c[1] : 0, u > 2 ? c[2] : 0, 0);
            }
          }
#pragma unroll
        for (uint32_t gi = 0; gi < S::kWords; ++gi) {
          constexpr uint32_t U = G / kUnit;
          if (!FULL && gi * U >= u) break;
          float sc[MG][2], acc[MG][NT][4];
          const float* gs = sums + (b * S::kWords + gi) * (NT * 8) + 2 * t;
#pragma unroll
          for (int m = 0; m < MG; ++m) {
            float z[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t w = word[(4 * (m0 + m) + 2 * h) * S::kWords + gi];
              sc[m][h] = raven_int4::step_of(w) * (1.f / (1 << kStepShift));
              z[h] = raven_int4::zero_of(w) + 8.f;
            }
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              const float2 q = *(const float2*)(gs + 8 * j);
              acc[m][j][0] = z[0] * q.x;
              acc[m][j][2] = z[1] * q.x;
              acc[m][j][1] = F32 ? 0.f : z[0] * q.y;
              acc[m][j][3] = F32 ? 0.f : z[1] * q.y;
            }
          }
#pragma unroll
          for (uint32_t uu = 0; uu < U; ++uu) {
            const uint32_t unit = gi * U + uu;
            if (!FULL && unit >= u) break;
            if constexpr (MG == MT) fetch(unit);
#pragma unroll
            for (int m = 0; m < MG; ++m) {
              uint32_t a[2][4];
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const uint4 c = code[m][h];
                const uint32_t w = unit == 0 ? c.x : unit == 1 ? c.y : unit == 2 ? c.z : c.w;
                operands(w, a[h][0], a[h][1], a[h][2], a[h][3]);
              }
#pragma unroll
              for (int j = 0; j < NT; ++j) mma(acc[m][j], a[0][0], a[1][0], a[0][1], a[1][1], x[unit][j].x, x[unit][j].y);
#pragma unroll
              for (int j = 0; j < NT; ++j) mma(acc[m][j], a[0][2], a[1][2], a[0][3], a[1][3], x[unit][j].z, x[unit][j].w);
            }
          }
#pragma unroll
          for (int m = 0; m < MG; ++m)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
              for (int i = 0; i < 4; ++i) total[m0 + m][j][i] = fmaf(sc[m][i / 2], acc[m][j][i], total[m0 + m][j][i]);
        }
      }
    };
    for (uint32_t b = kw; b < blocks; b += p.split) {
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
      const uint32_t u = units - 4 * b;
      if (u >= 4)
        block(std::true_type(), stage, word, b, 4);
      else
        block(std::false_type(), stage, word, b, u);
    }
    // The sums of a column (of two, F32) for this lane's rows, from one warp after the other where several shared
    // them; lanes next to one another in g swap half of theirs, so that each has rows side by side.
    const uint64_t row = ((uint64_t)tile * across + wr) * S::kRows + R * g;
    if (p.split > 1) {
      float* mine = shared + warp * (S::kPart / 4) + lane;
#pragma unroll
      for (int i = 0; i < MT * NT * 4; ++i) mine[32 * i] = total[i / (4 * NT)][i / 4 % NT][i % 4];
      meet(1 + wr, 32 * p.split);
    }
    const float* theirs = shared + wr * p.split * (S::kPart / 4) + lane;
    float bias[R];
#pragma unroll
    for (int r = 0; r < R; ++r) bias[r] = 0.f;
    if (p.bias) {
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (row + r < p.n) bias[r] = p.bias[row + r];
    }
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int c = 0; c < (F32 ? 1 : 2); ++c) {
        if (chunk * kQueries + (F32 ? 4 * j : 8 * j + c) >= p.nq) continue;  // no lane has a query
        float v[R];
        if (p.split > 1) {
          if ((j * (F32 ? 1 : 2) + c) % p.split != kw) continue;
#pragma unroll
          for (int r = 0; r < R; ++r) v[r] = 0.f;
          for (uint32_t k = 0; k < p.split; ++k) {
            const float* from = theirs + k * (S::kPart / 4);
#pragma unroll
            for (int r = 0; r < R; ++r) {
              const float* x = from + 32 * (((r / 2) * NT + j) * 4 + 2 * (r % 2) + c);
              v[r] += F32 ? x[0] + x[32] : x[0];
            }
          }
        } else {
#pragma unroll
          for (int r = 0; r < R; ++r)
            v[r] = F32 ? total[r / 2][j][2 * (r % 2)] + total[r / 2][j][2 * (r % 2) + 1] : total[r / 2][j][2 * (r % 2) + c];
        }
        float y[R];
#pragma unroll
        for (int i = 0; i < R / 2; ++i) {
          const float s = __shfl_xor_sync(0xffffffffu, odd ? v[i] : v[R / 2 + i], 4);
          y[2 * i] = odd ? s : v[i];
          y[2 * i + 1] = odd ? v[R / 2 + i] : s;
        }
        const uint32_t col = 8 * j + 2 * t + c;
        const uint64_t query = chunk * kQueries + (F32 ? col / 2 : col);
        if (query < p.nq) {
          __align__(16) O o[R];
          if (plain) {
            const float f = back[4 * (F32 ? col / 2 : col)];
#pragma unroll
            for (int r = 0; r < R; ++r) o[r] = rounded<O>(fmaf(f, y[r], bias[r]));
          } else {
            const float4 f = *(const float4*)(back + 4 * (F32 ? col / 2 : col));
#pragma unroll
            for (int r = 0; r < R; ++r) o[r] = rounded<O>(fmaf(y[r] * f.x * f.y, f.z, bias[r]));
          }
          O* to = (O*)p.out + slice * p.ld_slice + query * p.ld + row;
          if (p.whole && row + R <= p.n) {
            constexpr int B = R * sizeof(O) >= 16 ? 16 : R * sizeof(O);
#pragma unroll
            for (int i = 0; i < (int)(R * sizeof(O)) / B; ++i) {
              if constexpr (B == 16)
                ((uint4*)to)[i] = ((const uint4*)o)[i];
              else if constexpr (B == 8)
                ((uint2*)to)[i] = ((const uint2*)o)[i];
              else
                ((uint32_t*)to)[i] = ((const uint32_t*)o)[i];
            }
          } else {
#pragma unroll
            for (int r = 0; r < R; ++r)
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

// Scores from the slices' sums, in order: four at a time, pitch ld_slice / nq a multiple of 4.
struct Join {
  const float* part;
  uint64_t ld, ld_slice;  // of the sums
  uint32_t slices;
  uint64_t nq, n;
  const float4* backs;
  const float* bias;
  void* out;
  uint64_t ld_out;
};
template <typename O>
__global__ void __launch_bounds__(256) join_kernel(const Join p) {
  after_previous();
  const uint64_t per = (p.n + 3) / 4, total = p.nq * per;
  for (uint64_t u = (uint64_t)blockIdx.x * 256 + threadIdx.x; u < total; u += (uint64_t)gridDim.x * 256) {
    const uint64_t q = u / per, j = 4 * (u - q * per);
    const float* from = p.part + q * p.ld + j;
    float4 v = *(const float4*)from;
    for (uint32_t s = 1; s < p.slices; ++s) {
      const float4 x = *(const float4*)(from + s * p.ld_slice);
      v.x += x.x;
      v.y += x.y;
      v.z += x.z;
      v.w += x.w;
    }
    const float y[4] = {v.x, v.y, v.z, v.w};
    const float4 f = p.backs[q];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if (j + r >= p.n) continue;
      const float bias = p.bias ? p.bias[j + r] : 0.f;
      ((O*)p.out)[q * p.ld_out + j + r] = rounded<O>(f.w == 0.f ? fmaf(f.x, y[r], bias) : fmaf(y[r] * f.x * f.y, f.z, bias));
    }
  }
}

}  // namespace raven_score4
