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
__device__ inline float zero_of(uint32_t word) { return (float)(int8_t)(word & 0xffu); }

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
  int* status;
};

constexpr uint32_t kRun = 64;  // most rows of a run

// A lane takes eight values (two 16-byte loads of f32, one of 16-bit types), the
// group / 8 lanes of a group share its range by shuffles.
// VEC: pitch and address let 16 bytes be read at once. LANE: lane-major rows
// (element e of the first 16C at (e % 16) * C + e / 16).
template <typename T, bool VEC, bool LANE>
__global__ void __launch_bounds__(256) write_kernel(const Write p) {
  __shared__ int32_t dest[kRun];
  __shared__ uint32_t later[kRun];
  after_previous();
  const uint32_t lanes = p.group / 8, ng = (p.dim + p.group - 1) / p.group, per = ng * lanes;
  const uint32_t wide = (p.dim + kBlock - 1) / kBlock * (kBlock / p.group);  // words of a row as it is held
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
    const uint32_t items = rows * per;
    for (uint32_t u0 = 0; u0 < items; u0 += 256) {
      const uint32_t u = u0 + threadIdx.x, r = u / per, i = u - r * per, d = 8 * i;
      const int64_t to = u < items && !later[r] ? dest[r] : -1;
      float x[8];
      uint32_t top = 0;
      float lo = INFINITY, hi = -INFINITY;
      if (to >= 0) {
        const T* row = (const T*)p.x + (r0 + r) * p.ld;
        if (VEC && d + 8 <= p.dim) {
          __align__(16) T raw[8];
          ((uint4*)raw)[0] = *(const uint4*)(row + d);
          if constexpr (sizeof(T) == 4) ((uint4*)raw)[1] = *(const uint4*)(row + d + 4);
#pragma unroll
          for (int k = 0; k < 8; ++k) x[k] = raven_fp8::load_value(raw + k);
        } else {
          const uint32_t C = p.dim / 16;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const uint32_t e = d + k;
            x[k] = e < p.dim ? raven_fp8::load_value(row + (LANE && e < 16 * C ? (e % 16) * C + e / 16 : e)) : 0.f;
          }
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (d + k < p.dim) {
            top = max(top, __float_as_uint(x[k]) & 0x7fffffffu);
            lo = fminf(lo, x[k]);
            hi = fmaxf(hi, x[k]);
          }
      }
      for (uint32_t o = lanes / 2; o > 0; o >>= 1) {
        top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
      }
      if (to < 0) continue;
      uint32_t word = 0, scale = kNaN;
      if (top < 0x7f800000u) {
        const double need = fmax(((double)hi - (double)lo) / 15.0, (double)fmaxf(hi, -lo) / 127.0);
        const uint32_t bits = (__float_as_uint(__double2float_ru(need)) + 255u) & ~255u;
        const float step = __uint_as_float(bits), inv = 1.f / step;
        scale = bits;
        if (bits) {
          const int z = (int)rintf(__fdiv_rn(lo, step));
          scale = bits | ((uint32_t)z & 255u);
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            // x * inv is off by less than 2^-15 here: near a border the quotient itself decides. It is an
            // f32 rounded once, and between a value and a border that differ at least half a unit of it lies.
            const float q = x[k] * inv;
            float t = rintf(q);
            if (!(fabsf(q - t) < 0.5f - 0x1p-12f)) t = rintf(__fdiv_rn(x[k], step));
            const int c = min(max((int)t - z, 0), 15);
            word |= (d + k < p.dim ? (uint32_t)c : 0u) << (4 * k);
          }
        }
      }
      if (i < 4 * p.units) *(uint32_t*)(p.codes + to * p.ld_codes + 4 * word_at(i, p.units)) = word;
      uint32_t* words = p.words + to * p.ld_words;
      if (i % lanes == 0) words[i / lanes] = scale;
      if (i == 0)
        for (uint32_t g = ng; g < wide; ++g) words[g] = 0;
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// Reading: a lane writes 16 bytes of the output, half a word of f32 or a whole one
// of 16-bit values. Rows of no id are 0.
// ---------------------------------------------------------------------------
struct Read {
  const uint8_t* codes;
  const uint32_t* words;
  uint64_t n, ld_codes, ld_words;
  uint32_t dim, group, units;
  const int32_t* ids;  // null: row i
  uint64_t m;
  void* out;
  uint64_t ld;
  int* status;
};

template <typename T, bool VEC>
__global__ void __launch_bounds__(256) read_kernel(const Read p) {
  constexpr uint32_t V = 16 / sizeof(T);
  after_previous();
  const uint32_t per = (p.dim + V - 1) / V;
  const uint64_t total = p.m * per;
  for (uint64_t u = (uint64_t)blockIdx.x * 256 + threadIdx.x; u < total; u += (uint64_t)gridDim.x * 256) {
    const uint64_t r = u / per;
    const uint32_t d = (uint32_t)(u - r * per) * V;
    const int64_t from = p.ids ? (int64_t)p.ids[r] : (int64_t)r;
    const bool there = from >= 0 && from < (int64_t)p.n;
    if (from >= (int64_t)p.n && d == 0) raven_score::tell(p.status, kStatusIds);
    float step = 0.f, z = 0.f;
    uint32_t word = 0;
    if (there) {
      const uint32_t w = p.words[from * p.ld_words + d / p.group];
      step = step_of(w);
      z = zero_of(w);
      word = *(const uint32_t*)(p.codes + from * p.ld_codes + 4 * word_at(d / 8, p.units)) >> (4 * (d % 8));
    }
    __align__(16) T v[V];
#pragma unroll
    for (uint32_t k = 0; k < V; ++k) {
      const float f = there ? ((float)((word >> (4 * k)) & 15u) + z) * step : 0.f;
      if constexpr (sizeof(T) == 4)
        v[k] = f;
      else if constexpr (std::is_same<T, __half>::value)
        v[k] = __float2half_rn(f);
      else
        v[k] = __float2bfloat16_rn(f);
    }
    T* to = (T*)p.out + r * p.ld + d;
    if (VEC && d + V <= p.dim) {
      *(uint4*)to = *(const uint4*)v;
    } else {
#pragma unroll
      for (uint32_t k = 0; k < V; ++k)
        if (d + k < p.dim) to[k] = v[k];
    }
  }
}

}  // namespace raven_int4
