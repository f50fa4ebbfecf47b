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
//   warps 4-11  epilogue: one accumulator is stored while the next is filled
//   warps 12-15 (FP8) gather the tile's exponents, which start at any row of
//               a group, into the order that tensor memory takes; the MMA warp
//               copies them there in line with its instructions
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

#include "internal.h"
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

constexpr int kBM = 128;               // rows of v per tile
constexpr int kQBox = 32;              // queries per TMA box
constexpr uint32_t kABytes = kBM * 128;
constexpr uint32_t kQBoxBytes = kQBox * 128;
constexpr int kInfo = 4;               // tiles found ahead
constexpr int kSf = 4;                 // exponent buffers, in shared and in tensor memory
constexpr int kSfCols = 16;            // columns of one: 4 for the rows, 8 for the queries
constexpr uint32_t kSfBytes = 512;     // 128 rows: 32 lanes x 4 columns
constexpr uint32_t kBand = 8;          // query tiles walked together (they share a tile of v in L2)

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
  static constexpr int kThreads = FP8 ? 512 : 384;
  static constexpr int kConsumers = FP8 ? 14 : 10;  // arrivals that free a tile slot
  static constexpr uint32_t kBars = kStages * kStage;
  // full[S], empty[S], acc_full[2], acc_empty[2], info_full[I], info_empty[I], sf_full[F], sf_empty[F], drain
  static constexpr uint32_t kNumBars = 2 * kStages + 4 + 2 * kInfo + 2 * kSf + 1;
  static constexpr uint32_t kExps = (kBars + kNumBars * 8 + 127) / 128 * 128;
  static constexpr uint32_t kExpBuf = (1 + (BN + 127) / 128) * kSfBytes;
  static constexpr uint32_t kTiles = kExps + (FP8 ? kSf * kExpBuf : 0);
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
// 512 bytes of exponents (32 lanes x 16 bytes) to four columns, the same in each
// lane quadrant. Plain layout: groups of 8 lanes 128 bytes apart.
__device__ inline void copy_exps(uint32_t taddr, uint32_t smem) {
  const uint64_t desc = (uint64_t)((smem >> 4) & 0x3FFFu) | ((uint64_t)8 << 16) | ((uint64_t)8 << 32) | ((uint64_t)1 << 46);
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;\n" ::"r"(taddr), "l"(desc) : "memory");
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
// rise, so the groups are walked once. The lane that holds a tile's group works
// out the tile. Its divisions are 32-bit ones unless the group has 2^32 tiles.
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
  uint32_t qa = 0, va = 0, m = 0, nn = 0;  // its first query and row, how many
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
          qa = (uint32_t)q0;
          va = (uint32_t)v0;
          m = (uint32_t)(q1 - q0);
          nn = (uint32_t)(v1 - v0);
        }
      } else {
        m = (uint32_t)p.nq;
        nn = (uint32_t)p.n;
      }
    }
    tiles = (uint64_t)((m + BN - 1) / BN) * ((nn + kBM - 1) / kBM);
    incl = tiles;
    int64_t e = (int64_t)m * nn;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t t = __shfl_up_sync(0xffffffffu, incl, o);
      const int64_t x = __shfl_up_sync(0xffffffffu, e, o);
      if (lane >= o) {
        incl += t;
        e += x;
      }
    }
    before = e - (int64_t)m * nn;
    chunk_tiles = __shfl_sync(0xffffffffu, incl, 31);
    chunk_out = __shfl_sync(0xffffffffu, e, 31);
  }

  // The lane whose group holds tile t (rising between calls); -1 when there is none.
  __device__ int find(uint64_t t) {
    while (t >= first + chunk_tiles) {
      if (g0 + 32 >= p.groups || g0 + 32 < g0) return -1;
      first += chunk_tiles;
      out0 += chunk_out;
      g0 += 32;
      load();
    }
    return __ffs(__ballot_sync(0xffffffffu, t - first < incl)) - 1;
  }
  // Tile t of this lane's group.
  __device__ Tile tile(uint64_t t) const {
    const uint64_t in = t - first - (incl - tiles);
    // bands of kBand query tiles; in a band, all its query tiles of one row tile before the next
    const uint32_t mt = (m + BN - 1) / BN, nt = (nn + kBM - 1) / kBM;
    uint32_t band, rest;
    if (in >> 32) {
      band = (uint32_t)(in / (kBand * nt));
      rest = (uint32_t)(in - (uint64_t)band * kBand * nt);
    } else {
      band = mt <= kBand ? 0u : (uint32_t)in / (kBand * nt);
      rest = (uint32_t)in - band * kBand * nt;
    }
    const uint32_t wide = min(kBand, mt - band * kBand);
    const uint32_t ti = rest / wide, qi = band * kBand + rest - ti * wide;
    // even query tiles (at most BN, so mt - 1 of them are less than m): with a
    // short last one, the CTAs that always got that one had less to do
    const uint32_t step = mt == 1 ? BN : ((m + mt - 1) / mt + 15) / 16 * 16;
    Tile r;
    r.ld = p.qo ? (int64_t)nn : (int64_t)p.ld;
    r.out = out0 + before + (int64_t)(qi * step) * r.ld + (int64_t)(ti * kBM);
    r.vrow = va + ti * kBM;
    r.qrow = qa + qi * step;
    r.vcnt = min((uint32_t)kBM, nn - ti * kBM);
    r.qcnt = min(step, m - qi * step);
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

// 16 consecutive accumulator columns of this thread's lane, without waiting.
__device__ inline void tmem_ld16(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];\n"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr));
}
__device__ inline void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory"); }

__device__ inline bool elect_one() {
  uint32_t is;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(is)::"memory");
  return is != 0;
}
// The whole warp waits; one answer for all lanes. The clock is read only when
// the first look does not find the phase complete.
__device__ inline bool warp_wait(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  if (__all_sync(0xffffffffu, done != 0)) return true;
  return __all_sync(0xffffffffu, mbar_wait(bar, parity));
}

__device__ inline void put(float* p, float v) { *p = v; }
__device__ inline void put(__half* p, float v) { *p = __float2half_rn(v); }
__device__ inline void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// One epilogue warp's share of a tile: columns first, first + 32, ... in pieces
// of 16. `at`: this lane's score of query 0.
template <typename T>
__device__ inline void store_tile(T* at, int64_t ld, uint32_t acc, uint32_t first, uint32_t qcnt, bool row, float alpha,
                                  float bias) {
  for (uint32_t c = first; c < qcnt; c += 32) {
    uint32_t v[16];
    tmem_ld16(acc + c, v);
    tmem_wait_ld();
    if (row) {
      T* o = at + (int64_t)c * ld;
      if (c + 16 <= qcnt) {
#pragma unroll
        for (int j = 0; j < 16; ++j, o += ld) put(o, fmaf(alpha, __uint_as_float(v[j]), bias));
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j, o += ld)
          if (c + j < qcnt) put(o, fmaf(alpha, __uint_as_float(v[j]), bias));
      }
    }
    __syncwarp();
  }
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
      mbar_init(acc_empty(b), 8);
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
  after_previous();

  // Warps 0 and 1 run their loops as whole warps and elect a lane only where
  // they issue: loop state then lives in uniform registers, which is what the
  // copies and MMAs take their operands from. One lane looping alone moved
  // every operand over at each use, about 500 cycles per K block.
  if (warp == 0) {  // TMA
    TileReader rd;
    uint32_t s = 0, ph = 0, used = 0, last_ph = 0;
    while (ok) {
      if (!warp_wait(info_full(rd.slot), rd.phase)) {
        ok = false;
        break;
      }
      const uint32_t qcnt = tiles[rd.slot].qcnt, vrow = tiles[rd.slot].vrow, qrow = tiles[rd.slot].qrow;
      __syncwarp();
      if (lane == 0) mbar_arrive(info_empty(rd.slot));
      rd.next();
      if (qcnt == 0) break;
      const uint32_t boxes = (qcnt + kQBox - 1) / kQBox;
      for (uint32_t kb = 0; kb < p.nkb; ++kb) {
        if (!warp_wait(empty(s), ph ^ 1u)) {
          ok = false;
          break;
        }
        if (elect_one()) {
          mbar_expect_tx(full(s), kABytes + boxes * kQBoxBytes);
          const uint32_t a = sbase + s * L::kStage;
          const int x = (int)(kb * (FP8 ? 128u : 64u));
          tma_load_2d(a, &tm_v, x, (int)vrow, full(s));
          for (uint32_t b = 0; b < boxes; ++b)
            tma_load_2d(a + kABytes + b * kQBoxBytes, &tm_q, x, (int)(qrow + b * kQBox), full(s));
        }
        __syncwarp();
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
      if ((used >> st) & 1u) ok &= warp_wait(full(st), (last_ph >> st) & 1u);
  } else if (warp == 1) {  // MMA
    TileReader rd;
    uint32_t s = 0, ph = 0, b = 0, bph = 0, f = 0, fph = 0;
    while (ok) {
      if (!warp_wait(info_full(rd.slot), rd.phase)) {
        ok = false;
        break;
      }
      const uint32_t qcnt = __shfl_sync(0xffffffffu, tiles[rd.slot].qcnt, 0);
      if (lane == 0) mbar_arrive(info_empty(rd.slot));
      rd.next();
      if (qcnt == 0) break;
      const uint32_t idesc = p.idesc | (((qcnt + 15u) / 16u * 2u) << 17);  // N, a multiple of 16, in eights
      if (!warp_wait(acc_empty(b), bph ^ 1u)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint32_t d = tmem + b * BN;
      for (uint32_t kb = 0; kb < p.nkb; ++kb) {
        if (FP8 && (kb & 3u) == 0 && !warp_wait(sf_full(f), fph)) {
          ok = false;
          break;
        }
        if (!warp_wait(full(s), ph)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t a = sbase + s * L::kStage;
        const uint64_t da = sw128_desc(a), db = sw128_desc(a + kABytes);
        const bool last = kb + 1 == p.nkb;
        const bool sf_done = FP8 && ((kb & 3u) == 3u || last);
        const uint32_t steps = last ? p.last_k : 4u;
        const uint32_t sel = kb & 3u;
        const uint32_t sf = tmem + L::kAcc + f * kSfCols;
        if (elect_one()) {
          if (FP8 && sel == 0) {  // in order before the MMAs that read them
            const uint32_t e = sbase + L::kExps + f * L::kExpBuf;
#pragma unroll
            for (int j = 0; j < 1 + (BN + 127) / 128; ++j) copy_exps(sf + 4 * j, e + j * kSfBytes);
          }
#pragma unroll
          for (uint32_t k = 0; k < 4; ++k) {  // 32 bytes along the swizzled row
            if (k >= steps) break;
            if constexpr (FP8)
              mma_mxf8(d, da + 2 * k, db + 2 * k, idesc | (sel << 4) | (sel << 29), sf, sf + 4, (kb | k) != 0u);
            else
              mma_f16(d, da + 2 * k, db + 2 * k, idesc, (kb | k) != 0u);
          }
          mma_commit(empty(s));
          if (sf_done) mma_commit(sf_empty(f));
          if (last) mma_commit(acc_full(b));
        }
        __syncwarp();
        if (++s == S) {
          s = 0;
          ph ^= 1u;
        }
        if (sf_done && ++f == kSf) {
          f = 0;
          fph ^= 1u;
        }
      }
      if (!ok) break;
      b ^= 1u;
      bph ^= b == 0u;
    }
    if (elect_one()) mma_commit(drain);  // every MMA issued has completed
    __syncwarp();
    ok &= warp_wait(drain, 0);
  } else if (warp == 2) {  // tiles
    TileFinder<BN> finder(p, lane);
    TileReader wr;
    for (uint64_t t = blockIdx.x;; t += gridDim.x) {
      const int at = finder.find(t);
      if (!warp_wait(info_empty(wr.slot), wr.phase ^ 1u)) {
        ok = false;
        break;
      }
      if (lane == max(at, 0)) {
        if (at < 0)
          tiles[wr.slot].qcnt = 0;
        else
          tiles[wr.slot] = finder.tile(t);
        mbar_arrive(info_full(wr.slot));
      }
      __syncwarp();
      wr.next();
      if (at < 0) break;
    }
    if (__any_sync(0xffffffffu, finder.bad) && lane == 0 && p.status) atomicOr(p.status, kStatusOffsets);
  } else if (warp >= 4 && warp < 12) {  // epilogue: two warps per lane quadrant, 16 columns in turn
    const int quad = warp & 3;
    const uint32_t first = warp < 8 ? 0u : 16u;
    const uint32_t r = (uint32_t)(quad * 32 + lane);
    const uint32_t lane_base = (uint32_t)(quad * 32) << 16;
    TileReader rd;
    uint32_t b = 0, bph = 0;
    while (true) {
      if (!warp_wait(info_full(rd.slot), rd.phase)) {
        ok = false;
        break;
      }
      const Tile t = tiles[rd.slot];
      __syncwarp();
      if (lane == 0) mbar_arrive(info_empty(rd.slot));
      rd.next();
      if (t.qcnt == 0) break;
      const float bias = p.bias && r < t.vcnt ? p.bias[t.vrow + r] : 0.0f;
      if (!warp_wait(acc_full(b), bph)) {
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
      const uint32_t acc = tmem + lane_base + b * BN;
      const int64_t at = t.out + r;
      const bool row = r < t.vcnt;
      if (p.out_type == kOutF32)
        store_tile((float*)p.out + at, t.ld, acc, first, qcnt, row, p.alpha, bias);
      else if (p.out_type == kOutF16)
        store_tile((__half*)p.out + at, t.ld, acc, first, qcnt, row, p.alpha, bias);
      else
        store_tile((__nv_bfloat16*)p.out + at, t.ld, acc, first, qcnt, row, p.alpha, bias);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(acc_empty(b));
      b ^= 1u;
      bph ^= b == 0u;
    }
  } else if (FP8 && warp >= 12) {  // exponents
    // Thread r takes row r of the tile and queries r and r + 128: the word of
    // row 32 j + i goes to lane i, column j. The next words are on their way
    // while these are stored.
    constexpr int kParts = 1 + (BN + 127) / 128;
    const uint32_t r = threadIdx.x - 384;
    TileReader rd;
    uint32_t kb = p.nkb;
    const uint8_t* src[kParts];
    auto load = [&](uint32_t (&w)[kParts]) {  // false: no more, or a wait ran out
      kb += 4;
      if (kb >= p.nkb) {
        if (!warp_wait(info_full(rd.slot), rd.phase)) {
          ok = false;
          return false;
        }
        const uint32_t vrow = tiles[rd.slot].vrow, qrow = tiles[rd.slot].qrow, qcnt = tiles[rd.slot].qcnt;
        __syncwarp();
        if (lane == 0) mbar_arrive(info_empty(rd.slot));
        rd.next();
        if (qcnt == 0) return false;
        kb = 0;
        // rows past the arrays' ends repeat the last one
        src[0] = p.ve + min((uint64_t)vrow + r, p.n - 1) * p.ld_ve;
#pragma unroll
        for (int j = 1; j < kParts; ++j)
          src[j] = p.qe + min((uint64_t)qrow + min(r + 128u * (j - 1), qcnt - 1), p.nq - 1) * p.ld_qe;
      }
#pragma unroll
      for (int j = 0; j < kParts; ++j) w[j] = __ldg((const uint32_t*)(src[j] + kb));
      return true;
    };
    uint32_t f = 0, fph = 0, w[kParts], next[kParts];
    bool more = load(w);
    while (more) {
      more = load(next);
      if (!ok) break;
      if (!warp_wait(sf_empty(f), fph ^ 1u)) {
        ok = false;
        break;
      }
      uint8_t* to = smem + L::kExps + f * L::kExpBuf + (r % 32) * 16 + (r / 32) * 4;
#pragma unroll
      for (int j = 0; j < kParts; ++j) {
        *(uint32_t*)(to + j * kSfBytes) = w[j];
        w[j] = next[j];
      }
      asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(sf_full(f));
      if (++f == kSf) {
        f = 0;
        fph ^= 1u;
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
