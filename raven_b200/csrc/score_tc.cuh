// Scores of queries against rows on the 5th-generation tensor cores: dense
// (every query against every row) or grouped (the queries of group g against
// the rows of group g, both of any size), over 16-bit values or FP8 codes.
//
//   S[i, j] = alpha * sum_t q[i, t] v[j, t] + bias[j]
//
// FP8 rows are e4m3 codes with one exponent byte per block of 128 values
// (value = code * 2^(byte - 127)). The block's exponents go to the tensor core
// beside the codes (kind::mxf8f6f4 with block scaling): a power of two scales a
// product exactly, so all blocks of a row sum in one f32 accumulator and
// nothing is rescaled in registers. The instruction takes an exponent for each
// 32 values and selects it as one byte of a 32-bit column in tensor memory:
// the four instructions of a block name the same byte, and a column's four
// bytes serve four blocks.
//
// Roles. 128 rows of v are the M side of an instruction (tensor-memory lanes),
// up to BN queries the N side (columns): a lane then owns one row, and the 32
// lanes of a warp store 32 consecutive scores of one query without a detour
// through shared memory. One 128-byte swizzled row of shared memory is a block
// of 128 codes or 64 16-bit values, so both types share one pipeline.
//   warp 0      TMA: per K block 128 rows of v and the tile's queries
//   warp 1      issues the MMAs
//   warp 2      owns the tensor memory; finds the CTA's tiles
//   warps 4-7   epilogue: one accumulator is stored while the next is filled
//   warps 8-11  (FP8) bring the tile's exponents to tensor memory, each warp
//               its 32 lanes (every lane quadrant holds a copy)
// A tile's size is known on the device only (group sizes are device data): the
// N of its instructions and the queries it loads follow the group.
//
// Rows of another group, which a tile at a group's end also loads, only reach
// lanes and columns that are not stored. Offsets are clamped to the arrays, and
// nothing is written past the output's capacity. Every wait is bounded; one
// that runs out sets a status bit, and copies and MMAs in flight end before the
// tensor memory is freed.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "knn_tc.cuh"

namespace raven_score {

using raven_tc::mbar_arrive;
using raven_tc::mbar_expect_tx;
using raven_tc::mbar_init;
using raven_tc::mbar_wait;
using raven_tc::mma_commit;
using raven_tc::smem_u32;
using raven_tc::sw128_desc;
using raven_tc::tc_fence_after;
using raven_tc::tc_fence_before;
using raven_tc::tma_load_2d;
using raven_tc::tmem_ld32;

constexpr int kBM = 128;               // rows of v per tile
constexpr int kQBox = 32;              // queries per TMA box
constexpr uint32_t kABytes = kBM * 128;
constexpr uint32_t kQBoxBytes = kQBox * 128;
constexpr int kInfo = 4;               // tiles found ahead
constexpr int kSf = 4;                 // exponent buffers in tensor memory
constexpr int kSfCols = 16;            // columns of one: 4 for the rows, 8 for the queries
constexpr uint64_t kBand = 8;          // query tiles walked together (they share a tile of v in L2)

enum : int { kOutF32 = 0, kOutF16 = 1, kOutBf16 = 2 };
enum : int { kStatusOffsets = 1, kStatusCapacity = 2, kStatusWait = 4 };

struct Params {
  uint64_t nq, n;             // rows of q and v
  uint32_t nkb;               // 128-byte K blocks
  uint32_t last_k;            // instructions (32 bytes of K) in the last block
  uint32_t groups;            // 1 with null offsets: dense
  const int64_t* qo;          // [groups + 1] or null
  const int64_t* vo;
  const uint8_t* qe;          // exponents (FP8)
  const uint8_t* ve;
  uint64_t ld_qe, ld_ve;
  uint32_t idesc;             // without N, and without exponent selectors
  float alpha;
  const float* bias;          // per row of v, or null
  void* out;
  int out_type;
  uint64_t ld;                // dense: output pitch; grouped: the pitch is the group's rows
  uint64_t capacity;          // grouped: output elements
  int* status;                // or null
};

struct Tile {
  int64_t out;                // element of (first query, first row)
  int64_t ld;
  uint32_t vrow, qrow;        // first row and query
  uint32_t vcnt, qcnt;        // how many; qcnt 0: no more tiles
};

template <bool FP8, int BN>
struct Layout {
  static constexpr uint32_t kStage = kABytes + BN * 128;
  static constexpr int kStages = (int)((204u * 1024) / kStage) < 10 ? (int)((204u * 1024) / kStage) : 10;
  static constexpr int kThreads = FP8 ? 384 : 256;
  static constexpr int kConsumers = FP8 ? 10 : 6;  // arrivals that free a tile slot
  static constexpr uint32_t kBars = kStages * kStage;
  // full[S], empty[S], acc_full[2], acc_empty[2], info_full[I], info_empty[I], sf_full[F], sf_empty[F], drain
  static constexpr uint32_t kNumBars = 2 * kStages + 4 + 2 * kInfo + 2 * kSf + 1;
  static constexpr uint32_t kTiles = (kBars + kNumBars * 8 + 15) / 16 * 16;
  static constexpr uint32_t kSlot = kTiles + kInfo * (uint32_t)sizeof(Tile);
  static constexpr uint32_t kBytes = kSlot + 16 + 1024;
  static constexpr uint32_t kAcc = 2 * BN;  // accumulator columns
  static constexpr uint32_t kUsed = kAcc + (FP8 ? kSf * kSfCols : 0);
  static constexpr uint32_t kTmem = kUsed <= 64 ? 64 : kUsed <= 128 ? 128 : kUsed <= 256 ? 256 : 512;
  static_assert(kUsed <= 512, "tensor memory has 512 columns");
};

__device__ inline void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %6, %7, %8}, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(0u), "r"(0u), "r"(0u), "r"(0u)
      : "memory");
}
__device__ inline void mma_mxf8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                uint32_t acc) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %6, 0;\n"
      "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n}\n" ::"r"(
          d),
      "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(acc)
      : "memory");
}

// Finds the tiles of one CTA, in order, by one warp: groups are read 32 at a
// time (one per lane) and their tiles counted by a warp scan; a CTA's tiles
// rise, so the groups are walked once.
template <int BN>
struct TileFinder {
  const Params& p;
  int lane;
  uint64_t first = 0;       // first tile of the chunk
  int64_t out0 = 0;         // output elements before the chunk
  uint32_t g0 = 0;          // its first group
  uint64_t incl = 0;        // this lane's group: tiles up to and with it, in the chunk
  uint64_t tiles = 0;
  int64_t before = 0;       // output elements before it, in the chunk
  uint64_t chunk_tiles = 0;
  int64_t chunk_out = 0;
  uint64_t qa = 0, va = 0, m = 0, nn = 0;
  bool bad = false;

  __device__ TileFinder(const Params& p_, int lane_) : p(p_), lane(lane_) { load(); }

  __device__ void load() {
    const uint32_t g = g0 + (uint32_t)lane;
    qa = va = m = nn = 0;
    if (g < p.groups) {
      if (p.qo) {
        const int64_t q0 = p.qo[g], q1 = p.qo[g + 1], v0 = p.vo[g], v1 = p.vo[g + 1];
        if (q0 < 0 || q1 < q0 || (uint64_t)q1 > p.nq || v0 < 0 || v1 < v0 || (uint64_t)v1 > p.n) {
          bad = true;  // the group counts as empty
        } else {
          qa = (uint64_t)q0;
          va = (uint64_t)v0;
          m = (uint64_t)(q1 - q0);
          nn = (uint64_t)(v1 - v0);
        }
      } else {
        m = p.nq;
        nn = p.n;
      }
    }
    tiles = ((m + BN - 1) / BN) * ((nn + kBM - 1) / kBM);
    incl = tiles;
    int64_t e = (int64_t)(m * nn);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t t = __shfl_up_sync(0xffffffffu, incl, o);
      const int64_t x = __shfl_up_sync(0xffffffffu, e, o);
      if (lane >= o) {
        incl += t;
        e += x;
      }
    }
    before = e - (int64_t)(m * nn);
    chunk_tiles = __shfl_sync(0xffffffffu, incl, 31);
    chunk_out = __shfl_sync(0xffffffffu, e, 31);
  }

  // Tile t (rising between calls); qcnt 0 when there is none.
  __device__ Tile find(uint64_t t) {
    Tile r;
    r.qcnt = 0;
    while (t >= first + chunk_tiles) {
      first += chunk_tiles;
      out0 += chunk_out;
      if (g0 + 32 >= p.groups || g0 + 32 < g0) {
        g0 = p.groups;
        chunk_tiles = 0;
        return r;
      }
      g0 += 32;
      load();
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, t - first < incl);
    const int s = __ffs(hit) - 1;
    const uint64_t in = t - first - (__shfl_sync(0xffffffffu, incl, s) - __shfl_sync(0xffffffffu, tiles, s));
    const uint64_t gm = __shfl_sync(0xffffffffu, m, s), gn = __shfl_sync(0xffffffffu, nn, s);
    const uint64_t gq = __shfl_sync(0xffffffffu, qa, s), gv = __shfl_sync(0xffffffffu, va, s);
    const int64_t go = out0 + __shfl_sync(0xffffffffu, before, s);
    // bands of kBand query tiles; in a band, all its query tiles of one row tile before the next
    const uint64_t mt = (gm + BN - 1) / BN, nt = (gn + kBM - 1) / kBM;
    const uint64_t band = in / (kBand * nt), rest = in - band * kBand * nt;
    const uint64_t wide = min(kBand, mt - band * kBand);
    const uint64_t ti = rest / wide, qi = band * kBand + rest - ti * wide;
    r.ld = p.qo ? (int64_t)gn : (int64_t)p.ld;
    r.out = go + (int64_t)(qi * BN) * r.ld + (int64_t)(ti * kBM);
    r.vrow = (uint32_t)(gv + ti * kBM);
    r.qrow = (uint32_t)(gq + qi * BN);
    r.vcnt = (uint32_t)min((uint64_t)kBM, gn - ti * kBM);
    r.qcnt = (uint32_t)min((uint64_t)BN, gm - qi * BN);
    return r;
  }
};

// A reader's place in the ring of tiles.
struct TileReader {
  uint32_t slot = 0, phase = 0;
  __device__ void next() {
    if (++slot == kInfo) {
      slot = 0;
      phase ^= 1u;
    }
  }
};

__device__ inline void store_score(void* out, int type, int64_t at, float v) {
  if (type == kOutF32)
    ((float*)out)[at] = v;
  else if (type == kOutF16)
    ((__half*)out)[at] = __float2half_rn(v);
  else
    ((__nv_bfloat16*)out)[at] = __float2bfloat16_rn(v);
}

template <bool FP8, int BN>
__global__ void __launch_bounds__((Layout<FP8, BN>::kThreads), 1)
    score_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_v, const Params p) {
  using L = Layout<FP8, BN>;
  constexpr int S = L::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const uint32_t sbase = smem_u32(smem);
  const uint32_t bar0 = sbase + L::kBars;
  auto full = [&](uint32_t s) { return bar0 + 8u * s; };
  auto empty = [&](uint32_t s) { return bar0 + 8u * (S + s); };
  auto acc_full = [&](uint32_t b) { return bar0 + 8u * (2 * S + b); };
  auto acc_empty = [&](uint32_t b) { return bar0 + 8u * (2 * S + 2 + b); };
  auto info_full = [&](uint32_t i) { return bar0 + 8u * (2 * S + 4 + i); };
  auto info_empty = [&](uint32_t i) { return bar0 + 8u * (2 * S + 4 + kInfo + i); };
  auto sf_full = [&](uint32_t i) { return bar0 + 8u * (2 * S + 4 + 2 * kInfo + i); };
  auto sf_empty = [&](uint32_t i) { return bar0 + 8u * (2 * S + 4 + 2 * kInfo + kSf + i); };
  const uint32_t drain = bar0 + 8u * (2 * S + 4 + 2 * kInfo + 2 * kSf);
  Tile* tiles = (Tile*)(smem + L::kTiles);
  uint32_t* tmem_slot = (uint32_t*)(smem + L::kSlot);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(acc_full(b), 1);
      mbar_init(acc_empty(b), 4);
    }
    for (int i = 0; i < kInfo; ++i) {
      mbar_init(info_full(i), 1);
      mbar_init(info_empty(i), L::kConsumers);
    }
    for (int i = 0; i < kSf; ++i) {
      mbar_init(sf_full(i), 4);
      mbar_init(sf_empty(i), 1);
    }
    mbar_init(drain, 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(tmem_slot)),
                 "r"(L::kTmem)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  bool ok = true;

  if (warp == 0) {
    if (lane == 0) {  // TMA
      TileReader rd;
      uint32_t s = 0, ph = 0, used = 0, last_ph = 0;
      while (ok) {
        if (!mbar_wait(info_full(rd.slot), rd.phase)) {
          ok = false;
          break;
        }
        const Tile t = tiles[rd.slot];
        mbar_arrive(info_empty(rd.slot));
        rd.next();
        if (t.qcnt == 0) break;
        const uint32_t boxes = (t.qcnt + kQBox - 1) / kQBox;
        for (uint32_t kb = 0; kb < p.nkb; ++kb) {
          if (!mbar_wait(empty(s), ph ^ 1u)) {
            ok = false;
            break;
          }
          mbar_expect_tx(full(s), kABytes + boxes * kQBoxBytes);
          const uint32_t a = sbase + s * L::kStage;
          const int x = (int)(kb * (FP8 ? 128u : 64u));
          tma_load_2d(a, &tm_v, x, (int)t.vrow, full(s));
          for (uint32_t b = 0; b < boxes; ++b)
            tma_load_2d(a + kABytes + b * kQBoxBytes, &tm_q, x, (int)(t.qrow + b * kQBox), full(s));
          used |= 1u << s;
          last_ph = (last_ph & ~(1u << s)) | (ph << s);
          if (++s == S) {
            s = 0;
            ph ^= 1u;
          }
        }
      }
      // every load issued has landed (immediate unless a wait ran out)
      for (uint32_t st = 0; st < S; ++st)
        if ((used >> st) & 1u) ok &= mbar_wait(full(st), (last_ph >> st) & 1u);
    }
  } else if (warp == 1) {
    if (lane == 0) {  // MMA
      TileReader rd;
      uint32_t s = 0, ph = 0, b = 0, bph = 0, f = 0, fph = 0;
      while (ok) {
        if (!mbar_wait(info_full(rd.slot), rd.phase)) {
          ok = false;
          break;
        }
        const uint32_t qcnt = tiles[rd.slot].qcnt;
        mbar_arrive(info_empty(rd.slot));
        rd.next();
        if (qcnt == 0) break;
        const uint32_t idesc = p.idesc | (((qcnt + 15u) / 16u * 2u) << 17);  // N, a multiple of 16, in eights
        if (!mbar_wait(acc_empty(b), bph ^ 1u)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem + b * BN;
        for (uint32_t kb = 0; kb < p.nkb; ++kb) {
          if (FP8 && (kb & 3u) == 0 && !mbar_wait(sf_full(f), fph)) {
            ok = false;
            break;
          }
          if (!mbar_wait(full(s), ph)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a = sbase + s * L::kStage;
          const uint64_t da = sw128_desc(a), db = sw128_desc(a + kABytes);
          const uint32_t steps = kb + 1 == p.nkb ? p.last_k : 4u;
          for (uint32_t k = 0; k < steps; ++k) {  // 32 bytes along the swizzled row
            if constexpr (FP8) {
              const uint32_t sel = kb & 3u;
              mma_mxf8(d, da + 2 * k, db + 2 * k, idesc | (sel << 4) | (sel << 29), tmem + L::kAcc + f * kSfCols,
                       tmem + L::kAcc + f * kSfCols + 4, (kb | k) != 0u);
            } else {
              mma_f16(d, da + 2 * k, db + 2 * k, idesc, (kb | k) != 0u);
            }
          }
          mma_commit(empty(s));
          if (++s == S) {
            s = 0;
            ph ^= 1u;
          }
          if (FP8 && ((kb & 3u) == 3u || kb + 1 == p.nkb)) {
            mma_commit(sf_empty(f));
            if (++f == kSf) {
              f = 0;
              fph ^= 1u;
            }
          }
        }
        if (!ok) break;
        mma_commit(acc_full(b));
        b ^= 1u;
        bph ^= b == 0u;
      }
      mma_commit(drain);  // every MMA issued has completed
      ok &= mbar_wait(drain, 0);
    }
  } else if (warp == 2) {  // tiles
    TileFinder<BN> find(p, lane);
    TileReader wr;
    for (uint64_t t = blockIdx.x;; t += gridDim.x) {
      const Tile r = find.find(t);
      const bool got = mbar_wait(info_empty(wr.slot), wr.phase ^ 1u);
      if (!__all_sync(0xffffffffu, got)) {
        ok = false;
        break;
      }
      if (lane == 0) {
        tiles[wr.slot] = r;
        mbar_arrive(info_full(wr.slot));
      }
      __syncwarp();
      wr.next();
      if (r.qcnt == 0) break;
    }
    if (__any_sync(0xffffffffu, find.bad) && lane == 0 && p.status) atomicOr(p.status, kStatusOffsets);
  } else if (warp >= 4 && warp < 8) {  // epilogue
    const int quad = warp & 3;
    const uint32_t r = (uint32_t)(quad * 32 + lane);
    const uint32_t lane_base = (uint32_t)(quad * 32) << 16;
    TileReader rd;
    uint32_t b = 0, bph = 0;
    while (true) {
      bool got = mbar_wait(info_full(rd.slot), rd.phase);
      if (!__all_sync(0xffffffffu, got)) {
        ok = false;
        break;
      }
      const Tile t = tiles[rd.slot];
      __syncwarp();
      if (lane == 0) mbar_arrive(info_empty(rd.slot));
      rd.next();
      if (t.qcnt == 0) break;
      const float bias = p.bias && r < t.vcnt ? p.bias[t.vrow + r] : 0.0f;
      got = mbar_wait(acc_full(b), bph);
      if (!__all_sync(0xffffffffu, got)) {
        ok = false;
        break;
      }
      tc_fence_after();
      // queries whose scores of this tile lie within the output
      uint32_t qcnt = t.qcnt;
      if (p.qo) {
        const int64_t room = (int64_t)p.capacity - t.out - (int64_t)t.vcnt;
        const int64_t fit = room < 0 || t.out < 0 ? 0 : room / t.ld + 1;  // a sum of wild offsets may have wrapped
        if (fit < (int64_t)qcnt) {
          qcnt = (uint32_t)fit;
          if (lane == 0 && p.status) atomicOr(p.status, kStatusCapacity);
        }
      }
      for (uint32_t c = 0; c < qcnt; c += 32) {
        uint32_t v[32];
        tmem_ld32(tmem + lane_base + b * BN + c, v);
        if (r < t.vcnt) {
          const int64_t at = t.out + (int64_t)c * t.ld + r;
          const uint32_t m = min(32u, qcnt - c);
#pragma unroll
          for (uint32_t j = 0; j < 32; ++j)
            if (j < m) store_score(p.out, p.out_type, at + (int64_t)j * t.ld, fmaf(p.alpha, __uint_as_float(v[j]), bias));
        }
        __syncwarp();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(acc_empty(b));
      b ^= 1u;
      bph ^= b == 0u;
    }
  } else if (FP8 && warp >= 8) {  // exponents
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    TileReader rd;
    uint32_t f = 0, fph = 0;
    while (ok) {
      bool got = mbar_wait(info_full(rd.slot), rd.phase);
      if (!__all_sync(0xffffffffu, got)) {
        ok = false;
        break;
      }
      const Tile t = tiles[rd.slot];
      __syncwarp();
      if (lane == 0) mbar_arrive(info_empty(rd.slot));
      rd.next();
      if (t.qcnt == 0) break;
      for (uint32_t kb = 0; kb < p.nkb; kb += 4) {
        // column j, lane i: the word of row 32 j + i (rows past the arrays' ends repeat the last one)
        uint32_t w[12];
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
          const uint64_t row = min((uint64_t)t.vrow + 32 * j + lane, p.n - 1);
          w[j] = *(const uint32_t*)(p.ve + row * p.ld_ve + kb);
        }
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) {
          const uint64_t row = min((uint64_t)t.qrow + 32 * j + lane, p.nq - 1);
          w[4 + j] = 32 * j < t.qcnt ? *(const uint32_t*)(p.qe + row * p.ld_qe + kb) : 0u;
        }
        got = mbar_wait(sf_empty(f), fph ^ 1u);
        if (!__all_sync(0xffffffffu, got)) {
          ok = false;
          break;
        }
        const uint32_t at = tmem + lane_base + L::kAcc + f * kSfCols;
        tc_fence_after();
        asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(at), "r"(w[0]), "r"(w[1]),
                     "r"(w[2]), "r"(w[3])
                     : "memory");
        asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"r"(at + 4),
                     "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]), "r"(w[8]), "r"(w[9]), "r"(w[10]), "r"(w[11])
                     : "memory");
        asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(sf_full(f));
        if (++f == kSf) {
          f = 0;
          fph ^= 1u;
        }
      }
    }
  }
  if (!ok && lane == 0 && p.status) atomicOr(p.status, kStatusWait);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 2) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(L::kTmem) : "memory");
  }
}

}  // namespace raven_score
