// Rows of 4-bit codes with a scale word per group of 32, 64 or 128 values
// (include/raven_gpu.h): written from values, whole or into slots, and read back,
// whole or by id.
//
// A group's word is the f32 bits of its step, of which the low 8 hold a signed
// number z instead: value = (code + z) * step. The step has 16 significant bits,
// so with |code + z| <= 127 every value, and every border between two codes
// (half a step further), is an f32: rounding to a code is decided exactly.
//
//   need = max((hi - lo) / 15, max|x| / 127)   over the group, in 64 bits
//   step = need, rounded up to 16 significant bits
//   z    = rint(lo / step)                     nearest even, as all below
//   code = min(rint(x / step) - z, 15)
//
// Layout of a row: 32 values are a unit of 16 bytes, a block of 128 values holds
// four units, the last block what is left. Eight values (a quarter of a unit) are
// one 32-bit word, the first lowest; in a block the words of one quarter of its
// units stand side by side, so that the four lanes of a tensor-core fragment's row
// each read 16 bytes that hold their quarter of every unit.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>

#include "fp8.cuh"
#include "internal.h"
#include "status.cuh"

namespace raven_int4 {

using raven_score::after_previous;

constexpr uint32_t kBlock = 128, kUnit = 32;
constexpr uint32_t kNaN = 0x7fc00000u;  // the word of a group that held an infinity or a NaN
using raven_score::kStatusIds;

// Where the eight values 8i .. 8i + 7 of a row of `units` units are: which word.
__device__ inline uint32_t word_at(uint32_t i, uint32_t units) {
  const uint32_t block = i >> 4, unit = (i >> 2) & 3, quarter = i & 3;
  return 16 * block + min(4u, units - 4 * block) * quarter + unit;
}

__device__ inline float step_of(uint32_t word) { return __uint_as_float(word & 0xffffff00u); }
// z: as the low bits of an f32 of 2^23, offset by 128
__device__ inline float zero_of(uint32_t word) { return __uint_as_float((word & 0xffu) ^ 0x4b000080u) - 8388736.f; }

// ---------------------------------------------------------------------------
// Slots named more than once: the last of their rows is the one that is held.
// Which one that is, is settled before anything is written, since two rows
// written at once would mix. Few rows: every CTA looks through the slots behind
// its own. Many: a table of slots (open addressing, at most half full).
// ---------------------------------------------------------------------------
struct Claim {
  uint32_t slot;  // ~0: free
  int32_t row;    // the last row so far, -1
};
__device__ inline uint32_t claim_hash(uint32_t slot) { return slot * 0x9e3779b1u; }

__global__ void __launch_bounds__(256) claim_kernel(const int32_t* slots, uint32_t m, uint64_t n, Claim* table,
                                                    uint32_t bits) {
  after_previous();
  const uint32_t i = blockIdx.x * 256u + threadIdx.x;
  if (i >= m) return;
  const int32_t s = slots[i];
  if (s < 0 || (uint64_t)s >= n) return;
  uint32_t h = claim_hash((uint32_t)s) >> (32 - bits);
  for (uint32_t tries = 0; tries >> bits == 0; ++tries) {
    const uint32_t was = atomicCAS(&table[h].slot, ~0u, (uint32_t)s);
    if (was == ~0u || was == (uint32_t)s) {
      atomicMax(&table[h].row, (int32_t)i);
      return;
    }
    h = (h + 1) & ((1u << bits) - 1);
  }
}

struct Write {
  const void* x;
  uint64_t m, ld;          // rows and their pitch in values
  uint32_t dim, group, units;
  uint8_t* codes;
  uint32_t* words;
  uint64_t n, ld_codes, ld_words;  // rows held, pitches in bytes and words
  const int32_t* slots;    // null: row i is held as row i
  const Claim* table;      // null: few rows
  uint32_t bits;
  uint32_t run;            // rows of a CTA at once
  uint32_t per, magic;     // eights of a row, and what divides by them
  int* status;
};

constexpr uint32_t kRun = 64;  // most rows of a run
constexpr int kItems = 4;      // eights of a lane at once

// u / per for u * per < 2^32; magic: 2^32 / per rounded up, 0 for 1.
__device__ inline uint32_t divided(uint32_t u, uint32_t magic) { return magic ? __umulhi(u, magic) : u; }

// The step of a group of values from lo to hi, as bits: the least with 16
// significant bits for which hi - lo <= 15 * step and the largest magnitude <=
// 127 * step. That is (hi - lo) / 15 and m / 127 in 64 bits, rounded up: 15 * step
// is exact there, and a difference above it by a unit in its last place has a
// quotient above the step by more than half of one. 127 * step is exact in f32. From an
// estimate a little below, at most three units of 16 bits too low.
__device__ inline uint32_t step_bits(float lo, float hi) {
  const float m = fmaxf(hi, -lo);
  if (m == 0.f) return 0;
  const double range = (double)hi - (double)lo;
  const float near = fmaxf(__double2float_rn(range * (1.0 / 15.0)), m * (1.f / 127.f));
  uint32_t bits = __float_as_uint(near * (1.f - 0x1p-20f)) & ~255u;
  for (int i = 0; i < 4; ++i) {
    const float s = __uint_as_float(bits);
    if (range <= 15.0 * (double)s && m <= 127.f * s) break;
    bits += 256;
  }
  return bits;
}
__device__ inline float reciprocal(float x) {
  float r;
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// A lane takes eight values (two 16-byte loads of f32, one of 16-bit types), the
// L = group / 8 lanes of a group share its range by shuffles, and of four such
// pieces at once every group's word is worked out by a lane of its own (64-bit
// arithmetic that 16 lanes did alike took as long as the reading).
// VEC: pitch and address let 16 bytes be read at once. LANE: lane-major rows
// (element e of the first 16C at (e % 16) * C + e / 16).
template <typename T, uint32_t L, bool VEC, bool LANE>
__global__ void __launch_bounds__(256, 3) write_kernel(const Write p) {
  __shared__ int32_t dest[kRun];
  __shared__ uint32_t later[kRun];
  after_previous();
  constexpr uint32_t G = 8 * L, kGroups = 32 / L;  // groups of a warp's piece
  const uint32_t ng = (p.dim + G - 1) / G, lane = threadIdx.x & 31;
  const uint32_t wide = (p.dim + kBlock - 1) / kBlock * (kBlock / G);  // words of a row as it is held
  for (uint64_t r0 = (uint64_t)blockIdx.x * p.run; r0 < p.m; r0 += (uint64_t)gridDim.x * p.run) {
    const uint32_t rows = (uint32_t)min((uint64_t)p.run, p.m - r0);
    if (threadIdx.x < rows) {
      int64_t s = p.slots ? (int64_t)p.slots[r0 + threadIdx.x] : (int64_t)(r0 + threadIdx.x);
      if (s >= (int64_t)p.n) {
        raven_score::tell(p.status, kStatusIds);
        s = -1;
      }
      if (s >= 0 && p.table) {
        uint32_t h = claim_hash((uint32_t)s) >> (32 - p.bits);
        for (uint32_t tries = 0; tries >> p.bits == 0 && p.table[h].slot != (uint32_t)s; ++tries)
          h = (h + 1) & ((1u << p.bits) - 1);
        if (p.table[h].row != (int32_t)(r0 + threadIdx.x)) s = -1;
      }
      dest[threadIdx.x] = s < 0 ? -1 : (int32_t)s;
      later[threadIdx.x] = 0;
    }
    __syncthreads();
    if (p.slots && !p.table) {
      for (uint64_t j = r0 + 1 + threadIdx.x; j < p.m; j += 256) {
        const int32_t s = p.slots[j];
        for (uint32_t k = 0; k < rows && r0 + k < j; ++k)
          if (dest[k] == s) later[k] = 1;
      }
      __syncthreads();
    }
    const uint32_t items = rows * p.per;
    for (uint32_t u0 = 0; u0 < items; u0 += 256 * kItems) {
      float x[kItems][8], lo[kItems], hi[kItems];
      int32_t to[kItems];
      uint32_t at[kItems];
      bool odd[kItems];
#pragma unroll
      for (int n = 0; n < kItems; ++n) {
        const uint32_t u = u0 + n * 256 + threadIdx.x, r = divided(u, p.magic), i = u - r * p.per, d = 8 * i;
        to[n] = u < items && !later[r] ? dest[r] : -1;
        at[n] = i;
        if (to[n] >= 0) {
          const T* row = (const T*)p.x + (r0 + r) * p.ld;
          if (VEC && d + 8 <= p.dim) {
            __align__(16) T raw[8];
            ((uint4*)raw)[0] = *(const uint4*)(row + d);
            if constexpr (sizeof(T) == 4) ((uint4*)raw)[1] = *(const uint4*)(row + d + 4);
#pragma unroll
            for (int k = 0; k < 8; ++k) x[n][k] = raven_fp8::load_value(raw + k);
          } else {
            const uint32_t C = p.dim / 16;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              // past the row its last value again, which changes no range
              const uint32_t e = min(d + k, p.dim - 1);
              x[n][k] = raven_fp8::load_value(row + (LANE && e < 16 * C ? (e % 16) * C + e / 16 : e));
            }
          }
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k) x[n][k] = 0.f;
        }
      }
#pragma unroll
      for (int n = 0; n < kItems; ++n) {
        uint32_t top = 0;
        lo[n] = hi[n] = x[n][0];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          top = max(top, __float_as_uint(x[n][k]) & 0x7fffffffu);
          lo[n] = fminf(lo[n], x[n][k]);
          hi[n] = fmaxf(hi[n], x[n][k]);
        }
        const uint32_t votes = __ballot_sync(0xffffffffu, top >= 0x7f800000u);
        odd[n] = votes >> (lane & ~(L - 1)) & ((1u << L) - 1);
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) {
          lo[n] = fminf(lo[n], __shfl_xor_sync(0xffffffffu, lo[n], o));
          hi[n] = fmaxf(hi[n], __shfl_xor_sync(0xffffffffu, hi[n], o));
        }
      }
      // lane n * kGroups + g: group g of piece n
      float glo = 0.f, ghi = 0.f;
#pragma unroll
      for (int n = 0; n < kItems; ++n) {
        const float a = __shfl_sync(0xffffffffu, lo[n], lane % kGroups * L), b = __shfl_sync(0xffffffffu, hi[n], lane % kGroups * L);
        if (lane / kGroups == n) {
          glo = a;
          ghi = b;
        }
      }
      const uint32_t bits = step_bits(glo, ghi);
      const uint32_t scale = bits ? bits | ((uint32_t)(int)rintf(__fdiv_rn(glo, __uint_as_float(bits))) & 255u) : 0u;
#pragma unroll
      for (int n = 0; n < kItems; ++n) {
        uint32_t w = __shfl_sync(0xffffffffu, scale, n * kGroups + lane / L);
        if (to[n] < 0) continue;
        const uint32_t i = at[n], d = 8 * i;
        uint32_t word = 0;
        if (odd[n]) {
          w = kNaN;
        } else if (w & ~255u) {
          const float step = step_of(w), inv = reciprocal(step);
          const int z = (int)(int8_t)(w & 0xffu);
          uint32_t near = 0;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            // x * inv is off by less than 2^-15 here (infinite or NaN for the smallest steps): next to a border the
            // quotient itself decides. It is an f32 rounded once, and a value and a border that differ do so by more
            // than its rounding.
            // Rounding by adding 1.5 * 2^23, whose low bits are then the whole number.
            const float q = x[n][k] * inv, t = q + 12582912.f;
            near |= !(fabsf(q - (t - 12582912.f)) < 0.5f - 0x1p-12f) ? 1u << k : 0u;
            const int c = min(max(__float_as_int(t) - 0x4b400000 - z, 0), 15);
            word |= d + k < p.dim ? (uint32_t)c << (4 * k) : 0u;
          }
          if (near) {
#pragma unroll
            for (int k = 0; k < 8; ++k)
              if ((near >> k & 1u) && d + k < p.dim)
                word = (word & ~(15u << (4 * k))) | (uint32_t)min((int)rintf(__fdiv_rn(x[n][k], step)) - z, 15) << (4 * k);
          }
        }
        if (i < 4 * p.units) *(uint32_t*)(p.codes + to[n] * p.ld_codes + 4 * word_at(i, p.units)) = word;
        uint32_t* words = p.words + to[n] * p.ld_words;
        if (i % L == 0) words[i / L] = w;
        if (i == 0)
          for (uint32_t g = ng; g < wide; ++g) words[g] = 0;
      }
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// Reading: a lane writes 16 bytes of the output, half a word of f32 or a whole one
// of 16-bit values, four such pieces at once. Rows of no id are 0.
// ---------------------------------------------------------------------------
struct Read {
  const uint8_t* codes;
  const uint32_t* words;
  uint64_t n, ld_codes, ld_words;
  uint32_t dim, group, units;
  const int32_t* ids;   // null: row i
  uint64_t m;
  uint32_t run;         // rows of a CTA at once
  uint32_t per, magic;  // pieces of a row
  void* out;
  uint64_t ld;
  int* status;
};

template <typename T, bool VEC>
__global__ void __launch_bounds__(256) read_kernel(const Read p) {
  constexpr uint32_t V = 16 / sizeof(T);
  after_previous();
  const uint32_t shift = 31 - __clz(p.group);
  for (uint64_t r0 = (uint64_t)blockIdx.x * p.run; r0 < p.m; r0 += (uint64_t)gridDim.x * p.run) {
    const uint32_t rows = (uint32_t)min((uint64_t)p.run, p.m - r0), items = rows * p.per;
    for (uint32_t u0 = 0; u0 < items; u0 += 256 * kItems) {
      uint32_t word[kItems], scale[kItems];
#pragma unroll
      for (int n = 0; n < kItems; ++n) {
        const uint32_t u = u0 + n * 256 + threadIdx.x, r = divided(u, p.magic), d = (u - r * p.per) * V;
        word[n] = scale[n] = 0;
        if (u < items) {
          const int64_t from = p.ids ? (int64_t)p.ids[r0 + r] : (int64_t)(r0 + r);
          if (from >= 0 && from < (int64_t)p.n) {
            scale[n] = p.words[from * p.ld_words + (d >> shift)];
            word[n] = *(const uint32_t*)(p.codes + from * p.ld_codes + 4 * word_at(d / 8, p.units)) >> (4 * (d % 8));
          } else if (from >= 0 && d == 0) {
            raven_score::tell(p.status, kStatusIds);
          }
        }
      }
#pragma unroll
      for (int n = 0; n < kItems; ++n) {
        const uint32_t u = u0 + n * 256 + threadIdx.x, r = divided(u, p.magic), d = (u - r * p.per) * V;
        if (u >= items) continue;
        // code + z: the code as the low bits of 2^23, all exact
        const float step = step_of(scale[n]), z = zero_of(scale[n]) - 8388608.f;
        __align__(16) T v[V];
#pragma unroll
        for (uint32_t k = 0; k < V; ++k) {
          const float f = (__uint_as_float((word[n] >> (4 * k) & 15u) | 0x4b000000u) + z) * step;
          if constexpr (sizeof(T) == 4)
            v[k] = f;
          else if constexpr (std::is_same<T, __half>::value)
            v[k] = __float2half_rn(f);
          else
            v[k] = __float2bfloat16_rn(f);
        }
        T* to = (T*)p.out + (r0 + r) * p.ld + d;
        if (VEC && d + V <= p.dim) {
          *(uint4*)to = *(const uint4*)v;
        } else {
#pragma unroll
          for (uint32_t k = 0; k < V; ++k)
            if (d + k < p.dim) to[k] = v[k];
        }
      }
    }
  }
}

}  // namespace raven_int4
