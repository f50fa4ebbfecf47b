// The best k of each row of scores: values, indexes and counts, best first,
// equal scores by the lower index, NaN after every number.
//
// A score becomes a 32-bit key whose unsigned order is the wanted one (largest
// or smallest first); with the complement of its index below it, 64 bits order
// the row totally, so the answer does not depend on how the row is split. A
// team of threads (a warp for short rows, a CTA for long ones) streams its
// part of a row once, a tile of 16 elements per thread at a time in registers,
// and keeps the elements above a bound in shared memory:
//   * first tile: the k-th best of the threads' own maxima is reached by at
//     least k elements, so little more than k of the tile are kept;
//   * when many are kept, the k-th best of them is the new bound. A later
//     element must beat it, since an equal one has a higher index.
// Once there is a bound, a tile costs one minimum or maximum per score (one for two
// 16-bit ones) and one comparison per thread: keys are made only for what passes.
// Both k-th bests are found by one warp with the values in registers, a bit of
// the key at a time from the highest one in which they differ. At the end one
// warp orders the few left over in registers. A tile whose survivors do not fit
// (rising data, equal scores) is taken again slice by slice, pruned in between:
// slower, with the same result. Few long rows are split into parts over the
// GPU; the parts' lists are joined by the same code.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "internal.h"

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
  uint32_t mul, add;          // of the keys: 1, 0x7fffff, or for the smallest first -1, 0x7ffffe
  int type;                   // of the values written (lists need it too)
  uint64_t* lists;            // parts > 1: [nq][parts][k] entries, zero where there is none
  void* vals;
  uint32_t* ids;
  uint32_t* counts;           // or null
};

// Keys: 0xffffffff for the best infinity down to kWorst for the worst one; NaN
// (canonical after the addition) below it, and 0 for no element. With `up` the
// usual order-preserving image of the bits, the key is up + 0x7fffff, or
// ~up + 0x7fffff for the smallest first: one multiply-add.
constexpr uint32_t kWorst = 0x00fffffeu;
__device__ inline uint32_t key_of(float x, uint32_t mul, uint32_t add) {
  const uint32_t b = __float_as_uint(x + 0.0f);  // -0 counts as 0
  const uint32_t up = b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
  return up * mul + add;
}
__device__ inline float value_of(uint32_t key, uint32_t mul, uint32_t add) {
  const uint32_t up = (key - add) * mul;  // mul is 1 or -1: its own inverse
  return key < kWorst ? __int_as_float(0x7fc00000) : __uint_as_float((up & 0x80000000u) ? up & 0x7fffffffu : ~up);
}

// A team of 32 is a warp, a larger one a CTA.
// BIG: k above half of a CTA's threads, whose least maximum bounds nothing; the
// bound is then found among their quarters' maxima. A kernel of its own: the
// registers that takes cost the others a fifth.
template <int TEAM, bool BIG>
struct Team {
  static constexpr int kBuf = TEAM == 32 ? 1024 : 2048;
  static constexpr int kThreads = TEAM == 32 ? kCtaThreads : TEAM;  // of a CTA
  static constexpr int kTeams = kThreads / TEAM;
  __device__ static void sync() {
    if constexpr (TEAM == 32)
      __syncwarp();
    else
      __syncthreads();
  }
};
template <int TEAM, bool BIG>
struct Shared {
  uint64_t buf[Team<TEAM, BIG>::kBuf];
  uint32_t top[TEAM == 32 ? 1 : BIG ? 4 * TEAM : TEAM];
  uint32_t count;
  uint32_t bound;
};

// Elements a thread holds of a tile, as pieces of 16 bytes.
template <typename T>
struct Loader {
  static constexpr int kPer = 16 / (int)sizeof(T);
  static constexpr int kPieces = 16 / kPer;
  static constexpr int kE = 16;
  // Low bits of a key that tell no values of the type apart: zeros of the f32
  // image, ones of a negative's, and a sum with them.
  static constexpr int kLow = sizeof(T) == 4 ? 0 : std::is_same<T, __half>::value ? 13 : 16;
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

// The best score of a thread's pieces, NaN ignored (all NaN: the worst infinity).
__device__ inline float best_of(const uint4 (&v)[4], bool largest, const float*) {
  const uint32_t* u = (const uint32_t*)v;
  float m = largest ? -__int_as_float(0x7f800000) : __int_as_float(0x7f800000);
  if (largest) {
#pragma unroll
    for (int e = 0; e < 16; ++e) m = fmaxf(m, __uint_as_float(u[e]));
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e) m = fminf(m, __uint_as_float(u[e]));
  }
  return m;
}
template <typename H2, typename H>
__device__ inline float best_of_pairs(const uint4 (&v)[2], bool largest, uint32_t worst) {
  const uint32_t* u = (const uint32_t*)v;
  H2 m = *(const H2*)&worst;
  if (largest) {
#pragma unroll
    for (int e = 0; e < 8; ++e) m = __hmax2(m, *(const H2*)&u[e]);
    m.x = __hmax(m.x, m.y);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) m = __hmin2(m, *(const H2*)&u[e]);
    m.x = __hmin(m.x, m.y);
  }
  return (float)m.x;
}
__device__ inline float best_of(const uint4 (&v)[2], bool largest, const __half*) {
  return best_of_pairs<__half2, __half>(v, largest, largest ? 0xfc00fc00u : 0x7c007c00u);
}
__device__ inline float best_of(const uint4 (&v)[2], bool largest, const __nv_bfloat16*) {
  return best_of_pairs<__nv_bfloat162, __nv_bfloat16>(v, largest, largest ? 0xff80ff80u : 0x7f807f80u);
}

// By one warp, N values per lane (0: none): the largest T that at least k of
// them reach, 0 if fewer than k are there. Bits below LOW tell no values apart
// and are not tried (4096 rows of 6667 f16, k = 100: 67 to 63 us). `slack`: a T
// that is reached by up to k + slack will do.
template <int LOW, int N>
__device__ inline uint32_t kth_of_warp(const uint32_t (&v)[N], uint32_t k, uint32_t slack) {
  uint32_t hi = 0, lo = 0xffffffffu;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    hi = max(hi, v[i]);
    lo = min(lo, v[i]);
  }
  hi = __reduce_max_sync(0xffffffffu, hi);
  lo = __reduce_min_sync(0xffffffffu, lo);
  if (hi == lo) return hi;
  int bit = 31 - __clz(hi ^ lo);
  uint32_t t = bit < 31 ? hi & ~((2u << bit) - 1u) : 0u;
  for (; bit >= LOW; --bit) {
    const uint32_t next = t | (1u << bit);
    uint32_t c = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) c += v[i] >= next;
    c = __reduce_add_sync(0xffffffffu, c);
    if (c >= k) {
      t = next;
      if (c <= k + slack) break;
    }
  }
  if (LOW && t) {  // a value there
    uint32_t least = 0xffffffffu;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (v[i] >= t) least = min(least, v[i]);
    t = __reduce_min_sync(0xffffffffu, least);
  }
  return t;
}

// By one warp: v (element 32 i + lane in v[i]) in descending order. A bitonic sort
// of 32 N entries with 5 exchanges between lanes for each power of two above 32
// and none through memory: 100 entries cost 600 instructions of one warp, where
// counting each one's place among the others cost 1800.
template <int N>
__device__ inline void sort_of_warp(uint64_t (&v)[N], uint32_t lane) {
#pragma unroll
  for (uint32_t w = 2; w <= 32 * N; w <<= 1)
#pragma unroll
    for (uint32_t h = w >> 1; h > 0; h >>= 1) {
      if (h >= 32) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int j = i ^ (int)(h / 32);
          if (j > i) {
            const bool down = (((uint32_t)i * 32) & w) == 0;  // w > 32 here
            const uint64_t a = v[i], b = v[j];
            const bool swap = (a < b) == down;
            v[i] = swap ? b : a;
            v[j] = swap ? a : b;
          }
        }
      } else {
        const bool low = (lane & h) == 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const bool down = (((uint32_t)i * 32 + lane) & w) == 0;
          const uint64_t a = v[i], b = __shfl_xor_sync(0xffffffffu, a, h);
          v[i] = (a < b) == (low == down) ? b : a;
        }
      }
    }
}

template <int TEAM, bool BIG, int LOW>
struct Keeper {
  using TM = Team<TEAM, BIG>;
  static constexpr uint32_t kPrune = 1024;  // entries that one warp prunes
  static constexpr uint32_t kFew = 128;     // rows up to here need no bound
  static_assert(kPrune <= (uint32_t)TM::kBuf && kMaxK <= 256, "sizes");
  Shared<TEAM, BIG>& s;
  uint32_t tid, k;
  uint32_t above = 0;   // only keys over it can matter
  uint32_t held = 0;    // entries in the buffer (= s.count between calls)
  bool few;

  __device__ Keeper(Shared<TEAM, BIG>& s_, uint32_t tid_, uint32_t k_, uint64_t n) : s(s_), tid(tid_), k(k_), few(n <= kFew) {
    if (tid == 0) s.count = 0;
    TM::sync();
  }

  // Drops entries below the k-th key. Entry and exit are synchronised.
  __device__ void prune() {
    if (held > kPrune) {
      sort();
      return;
    }
    if (tid < 32) {
      uint32_t t;
      if (held <= 64)
        t = kth_of_held<2>();
      else if (held <= kPrune / 4)
        t = kth_of_held<kPrune / 128>();
      else if (held <= kPrune / 2)
        t = kth_of_held<kPrune / 64>();
      else
        t = kth_of_held<kPrune / 32>();
      // in place, 64 entries at a time, read before any of them is written over;
      // the whole team did it slower (20000 rows of 500 f32, k = 30: 57, 53 us)
      constexpr uint32_t U = 2;
      uint32_t c = 0;
      for (uint32_t i = tid; i < held + tid; i += 32 * U) {
        uint64_t e[U];
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) e[u] = i + 32 * u < held ? s.buf[i + 32 * u] : 0;
        __syncwarp();
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
          const bool keep = e[u] && (uint32_t)(e[u] >> 32) >= t;
          const uint32_t all = __ballot_sync(0xffffffffu, keep);
          if (keep) s.buf[c + __popc(all & ((1u << tid) - 1u))] = e[u];
          c += __popc(all);
        }
        __syncwarp();
      }
      if (tid == 0) {
        s.bound = t;
        s.count = c;
      }
    }
    TM::sync();
    const uint32_t t = s.bound;
    held = s.count;
    TM::sync();  // read by all before the next append
    if (held >= k) above = max(above, t);
    if (held > kPrune / 2) sort();  // many equals
  }
  template <int N>
  __device__ uint32_t kth_of_held() const {
    uint32_t v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = tid + 32 * i < held ? (uint32_t)(s.buf[tid + 32 * i] >> 32) : 0u;
    return kth_of_warp<LOW>(v, k, 0);
  }

  // The best k in order at the front, by sorting all.
  __device__ void sort() {
    const uint32_t c = held;
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
    held = min(c, k);
    if (tid == 0) s.count = held;
    TM::sync();
    if (c >= k) above = max(above, (uint32_t)(s.buf[k - 1] >> 32));
  }

  // The best k in order, at the front of the buffer.
  __device__ void finish() {
    if (held > 256 || (held > 128 && k <= 128)) prune();  // half the entries cost less than half to order
    if (held > 256) sort();  // many equals
    if (tid < 32) {
      if (held <= 32)
        order<1>();
      else if (held <= 64)
        order<2>();
      else if (held <= 128)
        order<4>();
      else
        order<8>();
    }
    held = min(held, k);
    TM::sync();
  }
  template <int N>
  __device__ void order() {
    uint64_t v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = tid + 32 * i < held ? s.buf[tid + 32 * i] : 0;
    sort_of_warp(v, tid);
#pragma unroll
    for (int i = 0; i < N; ++i) s.buf[tid + 32 * i] = v[i];  // the warp has read what it writes over
  }

  // Takes a tile as it was loaded, elements that do not exist being the worst
  // infinity. key(e): the key of an element in registers, 0 if it does not exist.
  template <typename T, int P, typename Key, typename Idx, typename Again>
  __device__ void take_raw(const uint4 (&v)[P], bool more, uint32_t mul, uint32_t add, Key key, Idx idx, Again again) {
    constexpr int E = Loader<T>::kE;
    const bool largest = mul == 1u;
    const float best = best_of(v, largest, (const T*)0);
    if constexpr (!BIG)
      if (above == 0 && !few && (TEAM > 32 || k <= 32)) bound_of(key_of(best, mul, add));
    // a bound over the worst infinity excludes NaN, as comparisons do
    if (above >= kWorst) {
      // the least value over the bound; no value is over the best infinity
      const float least = above == 0xffffffffu ? __int_as_float(0x7fc00000) : value_of(above + 1, mul, add);
      const uint32_t old = held;
      if (largest ? best >= least : best <= least) {
        uint32_t mine = 0;
        if (largest) {
#pragma unroll
          for (int e = 0; e < E; ++e) mine |= Loader<T>::get(v[e / Loader<T>::kPer], e % Loader<T>::kPer) >= least ? 1u << e : 0u;
        } else {
#pragma unroll
          for (int e = 0; e < E; ++e) mine |= Loader<T>::get(v[e / Loader<T>::kPer], e % Loader<T>::kPer) <= least ? 1u << e : 0u;
        }
        append(mine, idx, again);
      }
      if (appended()) {
        if (more && held > (TEAM == 32 ? 2 * k + 16 : kPrune / 2)) prune();  // the k-th best so far bounds the next tiles
        return;
      }
      undo(old);
    }
    uint32_t keys[E];
#pragma unroll
    for (int e = 0; e < E; ++e) keys[e] = key(e);
    take(keys, more, idx, again);
  }
  // Appends the marked elements of a thread, if they fit.
  template <typename Idx, typename Again>
  __device__ void append(uint32_t mine, Idx idx, Again again) {
    uint32_t at = atomicAdd(&s.count, (uint32_t)__popc(mine));
    if (at + __popc(mine) <= (uint32_t)TM::kBuf)
      for (; mine; mine &= mine - 1) {
        const int e = __ffs(mine) - 1;
        s.buf[at++] = ((uint64_t)again(e) << 32) | (uint32_t)~idx(e);
      }
  }
  // Synchronises, and whether all fitted.
  __device__ bool appended() {
    TM::sync();
    held = s.count;
    TM::sync();  // read by all before the next append
    return held <= (uint32_t)TM::kBuf;
  }

  // Takes a tile: key[e] (0: none) with index idx(e), and again(e) the key from
  // where it came. Indexes of a later tile are higher than those of an earlier
  // one. `more`: this is not the last.
  template <int E, typename Idx, typename Again>
  __device__ void take(const uint32_t (&key)[E], bool more, Idx idx, Again again) {
    static_assert(E % 4 == 0 && E <= 32, "quarters, bits");
    const uint32_t old = held;
    uint32_t top[4];  // best of each quarter
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      top[g] = key[g * (E / 4)];
#pragma unroll
      for (int e = 1; e < E / 4; ++e) top[g] = max(top[g], key[g * (E / 4) + e]);
    }
    if (above == 0 && !few) bound(key, top);
    if (!push(key, top, idx, again)) {
      undo(old);
      bound(key, top);  // now from this tile
      if (!push(key, top, idx, again)) {
        undo(old);
        slices(key, idx);
        return;
      }
    }
    if (more && held > (TEAM == 32 ? 2 * k + 16 : kPrune / 2)) prune();  // the k-th best so far bounds the next tiles
  }

  // Appends the keys over `above`; false if they do not fit. Exit is synchronised.
  template <int E, typename Idx, typename Again>
  __device__ bool push(const uint32_t (&key)[E], const uint32_t (&top)[4], Idx idx, Again again) {
    if (max(max(top[0], top[1]), max(top[2], top[3])) > above) {
      uint32_t mine = 0;
#pragma unroll
      for (int e = 0; e < E; ++e) mine |= key[e] > above ? 1u << e : 0u;
      append(mine, idx, again);
    }
    return appended();
  }
  __device__ void undo(uint32_t old) {
    held = old;
    if (tid == 0) s.count = old;
    TM::sync();
  }

  // The tile one element a thread at a time, pruned in between. Slices are not
  // in the order of their indexes, so an equal of the k-th is kept until the end.
  template <int E, typename Idx>
  __device__ void slices(const uint32_t (&key)[E], Idx idx) {
    const uint32_t was = above;
    uint32_t lower = was;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (held + TEAM > (uint32_t)TM::kBuf) {
        sort();
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
    if (held > k) sort();
  }

  // A bound from a tile: the k-th best of its threads' maxima, which k of them
  // and so k elements reach; where k is above a warp's threads, of its elements.
  template <int E>
  __device__ void bound(const uint32_t (&key)[E], const uint32_t (&top)[4]) {
    if constexpr (BIG) {  // k <= kMaxK <= 4 * TEAM
#pragma unroll
      for (int i = 0; i < 4; ++i) s.top[tid + i * TEAM] = top[i];
      TM::sync();
      bound_of_tops<4>();
    } else if (TEAM == 32 && k > 32) {
      const uint32_t t = kth_of_warp<LOW>(key, k, k / 8);
      if (t > 1) above = max(above, t - 1);
    } else {
      bound_of(max(max(top[0], top[1]), max(top[2], top[3])));
    }
  }
  // The same from each thread's best key.
  __device__ void bound_of(uint32_t top) {
    if constexpr (TEAM == 32) {
      const uint32_t v[1] = {top};
      const uint32_t t = kth_of_warp<LOW>(v, k, k / 4);
      if (t > kWorst) above = max(above, t - 1);
    } else {
      if (k > (uint32_t)TEAM) return;
      s.top[tid] = top;
      TM::sync();
      bound_of_tops<1>();
    }
  }
  template <int PER>
  __device__ void bound_of_tops() {
    if (tid < 32) {
      uint32_t v[PER * TEAM / 32];
#pragma unroll
      for (int i = 0; i < PER * TEAM / 32; ++i) v[i] = s.top[tid + 32 * i];
      const uint32_t t = kth_of_warp<LOW>(v, k, k / 4);
      if (tid == 0) s.bound = t;
    }
    TM::sync();
    const uint32_t t = s.bound;
    TM::sync();
    // not among NaN or the worst infinity: a thread without a number counts as that
    if (t > kWorst) above = max(above, t - 1);
  }
};

template <int TEAM, bool BIG, int LOW>
__device__ inline void write_out(const Params& p, Keeper<TEAM, BIG, LOW>& kp, uint64_t row, uint32_t part, uint32_t parts) {
  kp.finish();
  const uint64_t* best = kp.s.buf;
  const uint32_t c = kp.held;
  if (parts > 1) {
    uint64_t* o = p.lists + (row * parts + part) * p.k;
    for (uint32_t i = kp.tid; i < p.k; i += TEAM) o[i] = i < c ? best[i] : 0;
    return;
  }
  for (uint32_t i = kp.tid; i < p.k; i += TEAM) {
    const uint64_t e = i < c ? best[i] : 0;
    const float v = i < c ? value_of((uint32_t)(e >> 32), p.mul, p.add) : 0.0f;
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

template <typename T, int TEAM, bool BIG>
__global__ void __launch_bounds__((Team<TEAM, BIG>::kThreads), TEAM == 32 ? 3 : 1024 / TEAM) topk_kernel(const Params p) {
  extern __shared__ __align__(16) uint8_t raw[];
  raven_score::after_previous();
  Shared<TEAM, BIG>* sh = (Shared<TEAM, BIG>*)raw + threadIdx.x / TEAM;
  const uint32_t tid = threadIdx.x % TEAM;
  const uint64_t unit = (uint64_t)blockIdx.x * Team<TEAM, BIG>::kTeams + threadIdx.x / TEAM;
  const uint64_t row = p.parts == 1 ? unit : unit / p.parts;
  if (row >= p.nq) return;  // a whole team
  const uint32_t part = (uint32_t)(unit - row * p.parts);
  uint64_t lo = row * p.ld, len = p.n;
  if (p.starts) {
    const int64_t a = p.starts[row], b = p.starts[row + 1];
    lo = a < 0 || (uint64_t)a > p.total ? p.total : (uint64_t)a;
    const uint64_t hi = b < 0 ? 0 : min((uint64_t)b, p.total);
    len = hi > lo ? min(hi - lo, (uint64_t)0xffffffffu) : 0;
  }
  // this part's elements: [from, to) of the row. Parts are whole tiles less 16
  // bytes, for a row that starts between 16-byte boundaries
  using L = Loader<T>;
  constexpr uint32_t kTile = TEAM * L::kE;
  uint64_t each = len;
  if (p.parts > 1) each = ((len + p.parts - 1) / p.parts + kTile + L::kPer - 1) / kTile * kTile - L::kPer;
  const uint64_t from = min(len, each * part), to = min(len, from + each);
  Keeper<TEAM, BIG, Loader<T>::kLow> kp(*sh, tid, p.k, to - from);
  // pieces of 16 bytes from the boundary at or before the first element: the
  // bytes around a row are in the same 16 as some of its own
  const uint8_t* base = (const uint8_t*)p.x + (lo + from) * sizeof(T);
  const uint32_t skip = (uint32_t)(((uintptr_t)base & 15) / sizeof(T));
  const uint4* w = (const uint4*)((uintptr_t)base & ~(uintptr_t)15) + tid;
  const uint64_t end = to > from ? skip + (to - from) : 0;  // in elements from the boundary
  // the worst infinity, for what does not exist
  const uint32_t inf = sizeof(T) == 4                            ? 0x7f800000u
                       : std::is_same<T, __half>::value ? 0x7c007c00u
                                                        : 0x7f807f80u;
  const uint32_t none = p.mul == 1u ? inf | (sizeof(T) == 4 ? 0x80000000u : 0x80008000u) : inf;
  uint4 v[L::kPieces], ahead[L::kPieces];
  auto load = [&](uint64_t t) {  // pieces of the tile at t that hold an element
    if (t + kTile <= end) {
#pragma unroll
      for (int i = 0; i < L::kPieces; ++i) ahead[i] = w[i * TEAM];
    } else {
      const uint32_t left = t < end ? (uint32_t)(end - t) : 0;
#pragma unroll
      for (int i = 0; i < L::kPieces; ++i)
        ahead[i] = (i * TEAM + tid) * L::kPer < left ? w[i * TEAM] : make_uint4(none, none, none, none);
    }
    w += TEAM * L::kPieces;
  };
  load(0);
  for (uint64_t t = 0; t < end; t += kTile) {
    const uint32_t lo_ = t ? 0 : skip, hi_ = (uint32_t)min(end - t, (uint64_t)kTile);  // elements of the tile that exist
#pragma unroll
    for (int i = 0; i < L::kPieces; ++i) v[i] = ahead[i];
    if (lo_ || hi_ < kTile) {  // pieces at the row's edges
#pragma unroll
      for (int i = 0; i < L::kPieces; ++i) {
        const uint32_t e0 = (i * TEAM + tid) * L::kPer;
        if (e0 < lo_ || (e0 < hi_ && e0 + L::kPer > hi_)) {
          T* x = (T*)&v[i];
#pragma unroll
          for (int c = 0; c < L::kPer; ++c)
            if (e0 + c < lo_ || e0 + c >= hi_) x[c] = *(const T*)&none;
        }
      }
    }
    load(t + kTile);  // on its way while this tile is taken
    const uint32_t i0 = (uint32_t)(from - skip + t) + tid * L::kPer;  // wraps where the element does not exist
    const T* x0 = (const T*)((uintptr_t)base & ~(uintptr_t)15) + t + tid * L::kPer;
    auto place = [&](int e) { return (uint32_t)((e / L::kPer) * TEAM * L::kPer + e % L::kPer); };
    kp.template take_raw<T>(
        v, t + kTile < end, p.mul, p.add,
        [&](int e) {
          const uint32_t at = tid * L::kPer + place(e);
          return at >= lo_ && at < hi_ ? key_of(L::get(v[e / L::kPer], e % L::kPer), p.mul, p.add) : 0u;
        },
        [&](int e) { return i0 + place(e); },
        [&](int e) { return key_of((float)x0[place(e)], p.mul, p.add); });
  }
  write_out(p, kp, row, part, p.parts);
}

// Joins a row's lists (p.x: [nq][n] entries, n = lists x k).
template <bool BIG>
__global__ void __launch_bounds__(kCtaThreads) topk_join_kernel(const Params p) {
  constexpr int TEAM = kCtaThreads, E = 8;
  extern __shared__ __align__(16) uint8_t raw[];
  raven_score::after_previous();
  const uint64_t row = blockIdx.x;
  Keeper<TEAM, BIG, 0> kp(*(Shared<TEAM, BIG>*)raw, threadIdx.x, p.k, p.n);
  const uint64_t* x = (const uint64_t*)p.x + row * p.n;
  for (uint64_t t = 0; t < p.n; t += (uint64_t)TEAM * E) {
    uint32_t key[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint64_t at = t + (uint64_t)e * TEAM + threadIdx.x;
      const uint64_t v = at < p.n ? x[at] : 0;
      key[e] = (uint32_t)(v >> 32);
    }
    auto again = [&](int e) { return x[t + (uint64_t)e * TEAM + threadIdx.x]; };
    kp.take(
        key, t + (uint64_t)TEAM * E < p.n, [&](int e) { return ~(uint32_t)again(e); },
        [&](int e) { return (uint32_t)(again(e) >> 32); });
  }
  write_out(p, kp, row, 0, 1);
}

}  // namespace raven_topk
