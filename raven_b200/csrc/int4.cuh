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

// Row `row` at a pitch: one multiply-add.
template <typename T>
__device__ inline T* row_at(T* base, uint32_t row, uint32_t pitch) {
  return base + (uint64_t)row * pitch;
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
  uint32_t m, ld;          // rows and their pitch in values
  uint32_t dim, group, units;
  uint8_t* codes;
  uint32_t* words;
  uint32_t n, ld_codes, ld_words;  // rows held, pitches in bytes and words
  const int32_t* slots;    // null: row i is held as row i
  const Claim* table;      // null: few rows
  uint32_t bits;
  uint32_t run;            // rows of a CTA at once
  uint32_t per, magic;     // eights of a row, and what divides by them
  int* status;
};

constexpr uint32_t kRun = 64;  // most rows of a run
constexpr int kEights = 2;     // of a lane at once, written (four, with three CTAs an SM, 30000 x 768 f16 took 51 us, two 44)
constexpr int kItems = 4;      // pieces of a lane at once, read

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

// The codes of eight values: rint(x / step) - z, at most 15, the first lowest.
// The quotient has to be x / step rounded to f32: of values that differ from a
// border between two codes (a multiple of step / 2 of up to 24 bits, so an f32) it
// lies on the right side of it then, and on it for those that do not, which go to
// the even code. q = x * inv is off by a unit or two in its last place; its
// remainder is exact (18 bits), and what that adds is off by 2^-22 of such a unit,
// where a value next to a border is at least 2^-17 of one further from it than half
// a unit. Rounding is adding 1.5 * 2^23, whose low bits are then the whole number;
// sums of them, 4 bits apart, are a word of codes (mod 2^32). Steps are whole
// numbers of up to 16 bits times a power of two.
__device__ inline uint32_t codes_of(float (&x)[8], float step, int z) {
  if (step < 0x1p-80f) {  // remainders and reciprocals stay within f32's range; all values are below 2^-73
    step *= 0x1p64f;
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] *= 0x1p64f;
  }
  constexpr float kRound = 12582912.f;
  const float inv = reciprocal(step), most = kRound + (float)(z + 15);
  uint32_t word = 0u - (0x4b400000u + (uint32_t)z) * 0x11111111u;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float q = x[k] * inv, t = fmaf(fmaf(-q, step, x[k]), inv, q) + kRound;
    word += __float_as_uint(fminf(t, most)) << (4 * k);
  }
  return word;
}

// A lane takes eight values (two 16-byte loads of f32, one of 16-bit types), the
// L = group / 8 lanes of a group share its range by shuffles, and of two such
// pieces at once every group's word is worked out by a lane of its own (64-bit
// arithmetic that 16 lanes did alike took as long as the reading). What bounds it:
// the barrier before a run's slots are known (the largest stall) and issue slots (67 %);
// memory is at 3.4 TB/s (1000000 x 128 f32 into slots in random order 200 us, 680 MB:
// words and codes fill sectors in part, which are read first).
// VEC: pitch and address let 16 bytes be read at once. LANE: lane-major rows
// (element e of the first 16C at (e % 16) * C + e / 16).
template <typename T, uint32_t L, bool VEC, bool LANE>
__global__ void __launch_bounds__(256, 5) write_kernel(const Write p) {
  __shared__ int32_t dest[2][kRun];  // where the rows of a run, and of the next one, are held; -1: nowhere
  __shared__ uint32_t later[kRun];
  after_previous();
  // With a table the next run's rows are settled while this one's are worked on: two reads far apart, one after the other.
  // A CTA has a next run where there are more than 64 an SM (1000000 x 128: 3.3 runs a CTA; 30000 x 768 has none).
  auto settle = [&](uint64_t r0, int32_t* to) {
    if (r0 + threadIdx.x >= p.m || threadIdx.x >= p.run) return;
    int64_t s = (int64_t)p.slots[r0 + threadIdx.x];
    if (s >= (int64_t)p.n) {
      raven_score::tell(p.status, kStatusIds);
      s = -1;
    }
    if (s >= 0 && p.table) {
      uint32_t h = claim_hash((uint32_t)s) >> (32 - p.bits);
      for (uint32_t tries = 0; tries >> p.bits == 0; ++tries) {
        const Claim c = p.table[h];
        if (c.slot == (uint32_t)s) {
          if (c.row != (int32_t)(r0 + threadIdx.x)) s = -1;
          break;
        }
        h = (h + 1) & ((1u << p.bits) - 1);
      }
    }
    to[threadIdx.x] = s < 0 ? -1 : (int32_t)s;
    if (!p.table) later[threadIdx.x] = 0;
  };
  const uint64_t stride = (uint64_t)gridDim.x * p.run;
  uint32_t cur = 0;
  if (p.slots) settle((uint64_t)blockIdx.x * p.run, dest[0]);
  constexpr uint32_t G = 8 * L, kGroups = 32 / L;  // groups of a warp's piece
  const uint32_t ng = (p.dim + G - 1) / G, lane = threadIdx.x & 31;
  const uint32_t wide = (p.dim + kBlock - 1) / kBlock * (kBlock / G);  // words of a row as it is held
  for (uint64_t r0 = (uint64_t)blockIdx.x * p.run; r0 < p.m; r0 += stride) {
    const uint32_t rows = (uint32_t)min((uint64_t)p.run, p.m - r0), items = rows * p.per;
    float x[kEights][8];
    uint32_t from[kEights], at[kEights];  // a piece's row of the run, which of its eights
    auto load = [&](uint32_t u0) {
#pragma unroll
      for (int n = 0; n < kEights; ++n) {
        const uint32_t u = u0 + n * 256 + threadIdx.x;
        from[n] = divided(u, p.magic);
        at[n] = u - from[n] * p.per;
        const uint32_t d = 8 * at[n];
        if (u < items) {
          const T* row = row_at((const T*)p.x, (uint32_t)r0 + from[n], p.ld);
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
    };
    load(0);  // on the way while the slots are settled
    if (p.slots) {
      __syncthreads();
      if (p.table) {
        settle(r0 + stride, dest[cur ^ 1]);
      } else {
        for (uint64_t j = r0 + 1 + threadIdx.x; j < p.m; j += 256) {
          const int32_t s = p.slots[j];
          for (uint32_t k = 0; k < rows && r0 + k < j; ++k)
            if (dest[cur][k] == s) later[k] = 1;
        }
        __syncthreads();
      }
    }
    for (uint32_t u0 = 0; u0 < items; u0 += 256 * kEights) {
      if (u0) load(u0);
      float lo[kEights], hi[kEights];
      bool odd[kEights];
#pragma unroll
      for (int n = 0; n < kEights; ++n) {
        float not_finite = 0.f;  // NaN after an infinity or a NaN
        lo[n] = hi[n] = x[n][0];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          not_finite = fmaf(x[n][k], 0.f, not_finite);
          lo[n] = fminf(lo[n], x[n][k]);
          hi[n] = fmaxf(hi[n], x[n][k]);
        }
        const uint32_t votes = __ballot_sync(0xffffffffu, not_finite != 0.f);
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
      for (int n = 0; n < kEights; ++n) {
        const float a = __shfl_sync(0xffffffffu, lo[n], lane % kGroups * L), b = __shfl_sync(0xffffffffu, hi[n], lane % kGroups * L);
        if (lane / kGroups == n) {
          glo = a;
          ghi = b;
        }
      }
      const uint32_t bits = step_bits(glo, ghi);
      const uint32_t scale = bits ? bits | ((uint32_t)(int)rintf(__fdiv_rn(glo, __uint_as_float(bits))) & 255u) : 0u;
#pragma unroll
      for (int n = 0; n < kEights; ++n) {
        uint32_t w = __shfl_sync(0xffffffffu, scale, n * kGroups + lane / L);
        const uint32_t i = at[n], d = 8 * i;
        int32_t to = -1;
        if (u0 + n * 256 + threadIdx.x < items)
          to = !p.slots ? (int32_t)(r0 + from[n]) : !p.table && later[from[n]] ? -1 : dest[cur][from[n]];
        if (to < 0) continue;
        uint32_t word = 0;
        if (odd[n]) {
          w = kNaN;
        } else if (w & ~255u) {
          word = codes_of(x[n], step_of(w), (int)(int8_t)(w & 0xffu));
          if (d + 8 > p.dim) word &= d < p.dim ? (1u << (4 * (p.dim - d))) - 1 : 0u;
        }
        if (i < 4 * p.units) *(uint32_t*)(row_at(p.codes, to, p.ld_codes) + 4 * word_at(i, p.units)) = word;
        uint32_t* words = row_at(p.words, to, p.ld_words);
        if (i % L == 0) words[i / L] = w;
        if (i == 0)
          for (uint32_t g = ng; g < wide; ++g) words[g] = 0;
      }
    }
    if (p.slots && !p.table) {
      __syncthreads();
      settle(r0 + stride, dest[cur ^ 1]);
    }
    cur ^= 1;
  }
}

// ---------------------------------------------------------------------------
// Reading: a lane writes 16 bytes of the output, half a word of f32 or a whole one
// of 16-bit values, four such pieces at once. Rows of no id are 0. 1000000 random rows x
// 128 as bf16 71 us, 360 MB at 5.1 TB/s: memory and issue slots about even.
// ---------------------------------------------------------------------------
struct Read {
  const uint8_t* codes;
  const uint32_t* words;
  uint32_t n, ld_codes, ld_words;
  uint32_t dim, group, units;
  const int32_t* ids;   // null: row i
  uint32_t m;
  uint32_t run;         // rows of a CTA at once
  uint32_t per, magic;  // pieces of a row
  void* out;
  uint32_t ld;
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
      uint32_t word[kItems], scale[kItems], at[kItems], to_row[kItems];
      int32_t from[kItems];
#pragma unroll
      for (int n = 0; n < kItems; ++n) {
        const uint32_t u = u0 + n * 256 + threadIdx.x, r = divided(u, p.magic);
        at[n] = (u - r * p.per) * V;
        to_row[n] = (uint32_t)r0 + r;
        from[n] = -1;
        if (u < items) from[n] = p.ids ? p.ids[to_row[n]] : (int32_t)to_row[n];
      }
#pragma unroll
      for (int n = 0; n < kItems; ++n) {
        const uint32_t d = at[n];
        word[n] = scale[n] = 0;
        if ((uint32_t)from[n] < p.n) {
          scale[n] = row_at(p.words, from[n], p.ld_words)[d >> shift];
          word[n] = *(const uint32_t*)(row_at(p.codes, from[n], p.ld_codes) + 4 * word_at(d / 8, p.units)) >> (4 * (d % 8));
        } else if (from[n] >= 0 && d == 0) {
          raven_score::tell(p.status, kStatusIds);
        }
      }
#pragma unroll
      for (int n = 0; n < kItems; ++n) {
        if (u0 + n * 256 + threadIdx.x >= items) continue;
        const uint32_t d = at[n];
        // code + z, exactly: four bits at place 4 k of an f32's significand are a code on top of 2^(23 - 4 k)
        const float step = step_of(scale[n]), z = zero_of(scale[n]);
        __align__(16) T v[V];
#pragma unroll
        for (uint32_t k = 0; k < V; ++k) {
          const uint32_t at = 4 * (k % 4), w = k < 4 ? word[n] : word[n] >> 16;
          const float f = (__uint_as_float((w & (15u << at)) | (150u - at) << 23) + (z - (float)(8388608u >> at))) * step;
          if constexpr (sizeof(T) == 4)
            v[k] = f;
          else if constexpr (std::is_same<T, __half>::value)
            v[k] = __float2half_rn(f);
          else
            v[k] = __float2bfloat16_rn(f);
        }
        T* to = row_at((T*)p.out, to_row[n], p.ld) + d;
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
