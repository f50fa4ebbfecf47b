// The best k of each row of scores: values, indexes and counts, best first,
// equal scores by the lower index, NaN after every number.
//
// A score becomes a 32-bit key whose unsigned order is the wanted one (largest
// or smallest first); with the complement of its index below it, 64 bits order
// the row totally, so the answer does not depend on how the row is split. A
// team of threads (a warp for short rows, a CTA for long ones) streams its
// part of a row once, a tile at a time in registers, and keeps the elements
// above a threshold in shared memory:
//   * first tile: the k-th best of the threads' own maxima is a bound that at
//     least k elements reach, so about k elements are kept instead of all;
//   * then: the k-th best kept so far; a later element must beat it, since an
//     equal one has a higher index.
// The kept ones are ranked when the tile that set them is done, when they fill
// the buffer, and at the end. A tile whose survivors do not fit (rising data,
// equal scores) is taken again slice by slice, ranked in between: slower, with
// the same result. Few long rows are split into parts over the GPU; the parts'
// lists are joined by the same code.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace raven_topk {

constexpr uint32_t kMaxK = 256;
constexpr int kCtaThreads = 256;

struct Params {
  const void* x;              // scores, or lists of 64-bit entries
  uint64_t nq;
  uint64_t n;                 // dense: row length; lists: entries per row
  uint64_t ld;                // dense: row pitch
  const int64_t* starts;      // ragged: [nq + 1], or null
  uint64_t total;             // ragged: scores in x
  uint32_t k;
  uint32_t parts;             // teams per row
  int largest;
  int type;                   // of the values written (lists need it too)
  uint64_t* lists;            // parts > 1: [nq][parts][k] entries, zero where there is none
  void* vals;
  uint32_t* ids;
  uint32_t* counts;           // or null
};

// NaN is 1, below every number; 0 is no element.
__device__ inline uint32_t key_of(float x, int largest) {
  const uint32_t b = __float_as_uint(x + 0.0f);  // -0 counts as 0
  const uint32_t up = (b & 0x80000000u) ? ~b : b | 0x80000000u;
  return x != x ? 1u : largest ? up : ~up;
}
__device__ inline float value_of(uint32_t key, int largest) {
  const uint32_t up = largest ? key : ~key;
  return key == 1u ? __int_as_float(0x7fc00000) : __uint_as_float((up & 0x80000000u) ? up & 0x7fffffffu : ~up);
}

template <int TEAM>
struct Team {
  static constexpr int kBuf = TEAM == 32 ? 1024 : 2048;
  static constexpr int kTeams = kCtaThreads / TEAM;
  __device__ static void sync() {
    if constexpr (TEAM == 32)
      __syncwarp();
    else
      __syncthreads();
  }
};
template <int TEAM>
struct Shared {
  uint64_t buf[Team<TEAM>::kBuf];
  uint32_t max[TEAM];
  uint32_t count;
  uint32_t bound;
};

// Elements a thread holds of a tile, as pieces of 16 bytes.
template <typename T>
struct Loader {
  static constexpr int kPer = 16 / (int)sizeof(T);
  static constexpr int kPieces = 16 / kPer;
  static constexpr int kE = 16;
  __device__ static float get(const uint4& w, int c) {
    const uint32_t* u = &w.x;
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(u[c]);
    } else {
      const uint16_t h = (uint16_t)(u[c >> 1] >> (16 * (c & 1)));
      return (float)*(const T*)&h;
    }
  }
};

template <int TEAM>
struct Keeper {
  using TM = Team<TEAM>;
  static constexpr uint32_t kRank = TEAM == 32 ? 128 : 384;  // up to here ranks are counted, above sorted
  Shared<TEAM>& s;
  uint32_t tid, k;
  uint32_t above = 0;   // only keys over it can matter
  uint32_t held = 0;    // entries in the buffer (= s.count between calls)
  bool ranked = true;   // they are the best so far in order, at most k
  bool few;             // no more elements than are ranked by counting: no bound is needed

  __device__ Keeper(Shared<TEAM>& s_, uint32_t tid_, uint32_t k_, uint64_t n) : s(s_), tid(tid_), k(k_), few(n <= kRank) {
    if (tid == 0) s.count = 0;
    TM::sync();
  }

  // The buffer's best k, in order, at its front. Entry and exit are synchronised.
  __device__ void rank() {
    const uint32_t c = held;
    if (c <= kRank) {
      constexpr int kOwn = (kRank + TEAM - 1) / TEAM;
      uint64_t own[kOwn];
      uint32_t at[kOwn];
#pragma unroll
      for (int i = 0; i < kOwn; ++i) {
        const uint32_t e = tid + i * TEAM;
        own[i] = e < c ? s.buf[e] : 0;
        at[i] = 0;
      }
      for (uint32_t j = 0; j < c; ++j) {
        const uint64_t o = s.buf[j];
#pragma unroll
        for (int i = 0; i < kOwn; ++i) at[i] += o > own[i];
      }
      TM::sync();
#pragma unroll
      for (int i = 0; i < kOwn; ++i)
        if (tid + i * TEAM < c && at[i] < k) s.buf[at[i]] = own[i];
    } else {
      uint32_t p2 = 2 * TEAM;
      while (p2 < c) p2 <<= 1;
      for (uint32_t i = c + tid; i < p2; i += TEAM) s.buf[i] = 0;
      TM::sync();
      for (uint32_t w = 2; w <= p2; w <<= 1)
        for (uint32_t h = w >> 1; h > 0; h >>= 1) {
          for (uint32_t i = tid; i < p2 / 2; i += TEAM) {
            const uint32_t a = 2 * i - (i & (h - 1)), b = a + h;
            const uint64_t x = s.buf[a], y = s.buf[b];
            if ((x < y) == ((a & w) == 0)) {
              s.buf[a] = y;
              s.buf[b] = x;
            }
          }
          TM::sync();
        }
    }
    held = min(c, k);
    ranked = true;
    if (tid == 0) s.count = held;
    TM::sync();
    if (c >= k) above = max(above, (uint32_t)(s.buf[k - 1] >> 32));
  }

  // Takes a tile: key[e] (0: none) with index idx(e). Indexes of a later tile
  // are higher than those of an earlier one. `more`: this is not the last.
  template <int E, typename Idx>
  __device__ void take(const uint32_t (&key)[E], bool more, Idx idx) {
    const uint32_t old = held;
    if (above == 0 && !few) bound(key);
    if (!push(key, idx)) {
      undo(old);
      bound(key);  // now from this tile
      if (!push(key, idx)) {
        undo(old);
        rank();
        slices(key, idx);
        return;
      }
    }
    // when the first tile's survivors are ranked, the k-th is the threshold
    if (more && held >= k && (old < k || held > (uint32_t)TM::kBuf / 2)) rank();
  }

  // Appends the keys over `above`; false if they do not fit. Exit is synchronised.
  template <int E, typename Idx>
  __device__ bool push(const uint32_t (&key)[E], Idx idx) {
    uint32_t mine = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) mine += key[e] > above;
    if (mine) {
      uint32_t p = atomicAdd(&s.count, mine);
      if (p + mine <= (uint32_t)TM::kBuf) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (key[e] > above) s.buf[p++] = ((uint64_t)key[e] << 32) | (uint32_t)~idx(e);
      }
    }
    TM::sync();
    const uint32_t c = s.count;
    TM::sync();  // read by all before the next append
    ranked &= c == held;
    held = c;
    return c <= (uint32_t)TM::kBuf;
  }
  __device__ void undo(uint32_t old) {
    held = old;
    if (tid == 0) s.count = old;
    TM::sync();
  }

  // The tile one element a thread at a time, ranked in between. Slices are not
  // in the order of their indexes, so an equal of the k-th is kept until the end.
  template <int E, typename Idx>
  __device__ void slices(const uint32_t (&key)[E], Idx idx) {
    const uint32_t was = above;
    uint32_t lower = was;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (held + TEAM > (uint32_t)TM::kBuf) {
        rank();
        lower = max(was, above - 1);
      }
      if (key[e] > lower) {
        const uint32_t p = atomicAdd(&s.count, 1u);
        s.buf[p] = ((uint64_t)key[e] << 32) | (uint32_t)~idx(e);
      }
      TM::sync();
      held = s.count;
      TM::sync();
    }
    rank();
  }

  // A bound from the tile's own maxima: the k-th best of G of them is reached
  // by at least k elements, so lower keys are out.
  template <int E>
  __device__ void bound(const uint32_t (&key)[E]) {
    uint32_t g = 32;  // maxima: twice k, as far as there are threads
    while (g < 2 * k && g < (uint32_t)TEAM) g <<= 1;
    if (g < k) return;
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) m = max(m, key[e]);
    for (uint32_t o = 1; o < (uint32_t)TEAM / g; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    const uint32_t per = (uint32_t)TEAM / g;  // threads per maximum (at most 8: one warp's lanes)
    if (tid % per == 0) s.max[tid / per] = m;
    TM::sync();
    if (tid < g) {
      const uint32_t mine = s.max[tid];
      uint32_t at = 0;
      for (uint32_t j = 0; j < g; ++j) {
        const uint32_t o = s.max[j];
        at += o > mine || (o == mine && j < tid);
      }
      if (at == k - 1) s.bound = mine;
    }
    TM::sync();
    const uint32_t b = s.bound;
    if (b > 1) above = max(above, b - 1);
    TM::sync();
  }
};

template <int TEAM>
__device__ inline void write_out(const Params& p, Keeper<TEAM>& kp, uint64_t row, uint32_t part, uint32_t parts) {
  if (!kp.ranked) kp.rank();
  const uint32_t c = kp.held;
  if (parts > 1) {
    uint64_t* o = p.lists + (row * parts + part) * p.k;
    for (uint32_t i = kp.tid; i < p.k; i += TEAM) o[i] = i < c ? kp.s.buf[i] : 0;
    return;
  }
  for (uint32_t i = kp.tid; i < p.k; i += TEAM) {
    const uint64_t e = i < c ? kp.s.buf[i] : 0;
    const float v = i < c ? value_of((uint32_t)(e >> 32), p.largest) : 0.0f;
    const uint64_t at = row * p.k + i;
    if (p.type == 0)
      ((float*)p.vals)[at] = v;
    else if (p.type == 1)
      ((__half*)p.vals)[at] = __float2half_rn(v);  // exact: the value came from this type
    else
      ((__nv_bfloat16*)p.vals)[at] = __float2bfloat16_rn(v);
    p.ids[at] = i < c ? ~(uint32_t)e : 0u;
  }
  if (p.counts && kp.tid == 0) p.counts[row] = c;
}

template <typename T, int TEAM>
__global__ void __launch_bounds__(kCtaThreads) topk_kernel(const Params p) {
  extern __shared__ __align__(16) uint8_t raw[];
  Shared<TEAM>* sh = (Shared<TEAM>*)raw + threadIdx.x / TEAM;
  const uint32_t tid = threadIdx.x % TEAM;
  const uint64_t unit = (uint64_t)blockIdx.x * Team<TEAM>::kTeams + threadIdx.x / TEAM;
  const uint64_t row = unit / p.parts;
  if (row >= p.nq) return;  // a whole team
  const uint32_t part = (uint32_t)(unit - row * p.parts);
  uint64_t lo = row * p.ld, len = p.n;
  if (p.starts) {
    const int64_t a = p.starts[row], b = p.starts[row + 1];
    lo = a < 0 || (uint64_t)a > p.total ? p.total : (uint64_t)a;
    const uint64_t hi = b < 0 ? 0 : min((uint64_t)b, p.total);
    len = hi > lo ? min(hi - lo, (uint64_t)0xffffffffu) : 0;
  }
  // this part's elements: [from, to) of the row
  const uint64_t each = (len + p.parts - 1) / p.parts;
  const uint64_t from = min(len, each * part), to = min(len, from + each);
  Keeper<TEAM> kp(*sh, tid, p.k, to - from);
  using L = Loader<T>;
  // pieces of 16 bytes from the boundary at or before the first element: the
  // bytes around a row are in the same 16 as some of its own
  const uint8_t* base = (const uint8_t*)p.x + (lo + from) * sizeof(T);
  const uint32_t skip = (uint32_t)(((uintptr_t)base & 15) / sizeof(T));
  const uint4* w = (const uint4*)((uintptr_t)base & ~(uintptr_t)15);
  const uint64_t end = skip + (to - from);  // in elements from w
  constexpr uint64_t kTile = (uint64_t)TEAM * L::kE;
  for (uint64_t t = 0; to > from && t < end; t += kTile) {
    uint4 v[L::kPieces];
#pragma unroll
    for (int i = 0; i < L::kPieces; ++i) {
      const uint64_t e = t + (uint64_t)(i * TEAM + tid) * L::kPer;
      v[i] = e < end ? __ldg(w + e / L::kPer) : make_uint4(0, 0, 0, 0);
    }
    uint32_t key[L::kE];
#pragma unroll
    for (int i = 0; i < L::kPieces; ++i)
#pragma unroll
      for (int c = 0; c < L::kPer; ++c) {
        const uint64_t e = t + (uint64_t)(i * TEAM + tid) * L::kPer + c;
        key[i * L::kPer + c] = e >= skip && e < end ? key_of(L::get(v[i], c), p.largest) : 0u;
      }
    const uint32_t i0 = (uint32_t)(from - skip + t) + tid * L::kPer;  // wraps where the element does not exist
    kp.take(key, t + kTile < end,
            [&](int e) { return i0 + (uint32_t)((e / L::kPer) * TEAM * L::kPer + e % L::kPer); });
  }
  write_out<TEAM>(p, kp, row, part, p.parts);
}

// Joins a row's lists (p.x: [nq][n] entries, n = lists x k).
__global__ void __launch_bounds__(kCtaThreads) topk_join_kernel(const Params p) {
  constexpr int TEAM = kCtaThreads, E = 8;
  extern __shared__ __align__(16) uint8_t raw[];
  const uint64_t row = blockIdx.x;
  Keeper<TEAM> kp(*(Shared<TEAM>*)raw, threadIdx.x, p.k, p.n);
  const uint64_t* x = (const uint64_t*)p.x + row * p.n;
  for (uint64_t t = 0; t < p.n; t += (uint64_t)TEAM * E) {
    uint32_t key[E], id[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint64_t at = t + (uint64_t)e * TEAM + threadIdx.x;
      const uint64_t v = at < p.n ? x[at] : 0;
      key[e] = (uint32_t)(v >> 32);
      id[e] = ~(uint32_t)v;
    }
    kp.take(key, t + (uint64_t)TEAM * E < p.n, [&](int e) { return id[e]; });
  }
  write_out<TEAM>(p, kp, row, 0, 1);
}

}  // namespace raven_topk
