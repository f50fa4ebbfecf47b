// Scores of queries against rows on the 5th-generation tensor cores: dense
// (every query against every row) or grouped (the queries of group g against
// the rows of group g, both of any size), over 16-bit values or FP8 codes.
//
//   S[i, j] = alpha * sum_t q[i, t] v[j, t] + bias[j]
//
// FP8 rows are e4m3 codes with one exponent byte per block of 128 values
// (value = code * 2^(byte - 127), byte 255 NaN). The block's exponents go to the tensor core
// beside the codes (kind::mxf8f6f4 with block scaling): a power of two scales a
// product exactly, so all blocks of a row sum in one f32 accumulator and
// nothing is rescaled in registers. The instruction takes an exponent for each
// 32 values and selects it as one byte of a 32-bit column in tensor memory:
// the four instructions of a block name the same byte, and a column's four
// bytes serve four blocks.
//
// Two layouts. The M side of an instruction is 128 rows (tensor-memory lanes), the
// N side up to BN rows (columns).
//   rows    M = rows of v, N = queries: few queries cost the tensor cores and the
//           shared memory little, and the 32 lanes of a warp write 32 consecutive
//           scores of a query. For few queries, and for f32 scores that start on
//           sectors.
//   pairs   M = queries, N = rows of v: a lane owns a query and reads its scores in
//           order, so it packs them into whole 32-byte sectors of the output,
//           wherever a query's scores start.
// One 128-byte swizzled row of shared memory is a block of 128 codes or 64
// 16-bit values, so both types share one pipeline. Warp roles:
//   warp 0      TMA: per K block the tile's rows and queries
//   warp 1      issues the MMAs
//   warp 2      owns the tensor memory; finds the CTA's tiles
//   next 8 (16) epilogue: one tile is stored while the next is computed
//   last 4 (FP8) gather the tile's exponents, which start at any row of
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

#include <type_traits>

#include "fp8.cuh"
#include "internal.h"
#include "knn_tc.cuh"

namespace raven_score {

using raven_tc::mbar_arrive;
using raven_tc::mbar_expect_tx;
using raven_tc::mbar_init;
using raven_tc::mma_commit;
using raven_tc::smem_u32;
using raven_tc::sw128_desc;
using raven_tc::tc_fence_after;
using raven_tc::tc_fence_before;
using raven_tc::tma_load_2d;

constexpr int kBM = 128;               // rows of the M side
constexpr int kQBox = 32;              // queries per TMA box where they are the N side
constexpr uint32_t kABytes = kBM * 128;
constexpr uint32_t kSleepNs = 1000000;  // how long a wait may sleep before it looks at the clock
constexpr int kInfo = 4;               // tiles found ahead
constexpr int kSf = 4;                 // exponent buffers, in shared and in tensor memory
constexpr int kSfCols = 16;            // columns of one: 4 for the M side, 8 for the N side
constexpr uint32_t kSfBytes = 512;     // 128 rows: 32 lanes x 4 columns
constexpr uint32_t kBand = 8;          // query tiles walked together (they share a tile of v in L2)

constexpr uint32_t kHeldBlocks = 8;    // (HELD) K blocks of queries that a CTA holds
constexpr uint32_t kHeldUnits = 32;    // and query blocks that it encodes
enum : int { kOutF32 = 0, kOutF16 = 1, kOutBf16 = 2 };
enum : int { kStatusOffsets = 1, kStatusCapacity = 2, kStatusWait = 4 };

// The status of calls that are given no word for it, per device, until it is taken
// (raven_scoring_status_device).
__device__ int g_status;
__device__ inline void tell(int* status, int bits) { atomicOr(status ? status : &g_status, bits); }

// Sums over the groups before a chunk of 32 groups: their tiles, their scores.
struct alignas(16) Chunk {
  int64_t tiles, out;
};
constexpr uint32_t kChunk = 32;

// Group g's first query and row, how many of each; false, and an empty group,
// where its offsets are not within the arrays or fall.
__device__ inline bool group_of(const int64_t* qo, const int64_t* vo, uint32_t g, uint64_t nq, uint64_t n, int64_t& q0,
                                int64_t& v0, int64_t& m, int64_t& nn) {
  const int64_t a = qo[g], q1 = qo[g + 1], b = vo[g], v1 = vo[g + 1];
  const bool ok = a >= 0 && q1 >= a && (uint64_t)q1 <= nq && b >= 0 && v1 >= b && (uint64_t)v1 <= n;
  q0 = ok ? a : 0;
  v0 = ok ? b : 0;
  m = ok ? q1 - a : 0;
  nn = ok ? v1 - b : 0;
  return ok;
}

struct Params {
  uint64_t nq, n;             // rows of q and v
  uint32_t nkb;               // 128-byte K blocks
  uint32_t last_k;            // instructions (32 bytes of K) in the last block
  uint32_t subs;              // (rows) accumulators per tile: a tile has up to 128 * subs rows of v
  uint32_t halo;              // (pairs) scores that a tile computes past its own, 0 where every query starts on a sector
  uint32_t groups;            // 1 with null offsets: dense
  uint32_t nchunks;           // many groups: chunks[nchunks + 1], else null
  const Chunk* chunks;
  const int64_t* qo;          // [groups + 1] or null
  const int64_t* vo;
  const uint8_t* qe;          // exponents (FP8)
  const uint8_t* ve;
  uint64_t ld_qe, ld_ve;
  const void* qx;             // (HELD) the queries, of type kOut..., dim values at pitch ld_qx
  int q_type;
  uint32_t dim;
  uint64_t ld_qx;
  uint32_t idesc;             // without N, and without exponent selectors
  float alpha;
  const float* bias;          // per row of v, or null
  void* out;
  int out_type;
  uint64_t ld;                // dense: output pitch; grouped: the pitch is the group's rows
  uint64_t capacity;          // grouped: output elements
  int* status;                // null: g_status
};

struct Tile {
  int64_t out;                // element of (first query, first row)
  int64_t ld;
  uint32_t vrow, qrow;        // first row and query
  uint32_t vcnt, qcnt;        // how many; qcnt 0: no more tiles
  uint32_t vext;              // (pairs) rows computed: vcnt and up to a sector of the next tile's scores
  uint32_t first;             // whether the tile starts its queries' scores
};

// BN: most rows of the N side. ROWS: the layout with rows of v as the M side.
// HELD: a handful of queries, not encoded yet: every CTA encodes them into its
// shared memory and keeps them there. Saves the launch and the scratch of an
// encoding before (1 x 100000 x 128: 10.5 to 8.0 us).
template <bool FP8, int BN, bool ROWS, bool HELD>
struct Layout {
  static_assert(!HELD || (FP8 && ROWS && BN == 32), "one box of queries");
  static constexpr uint32_t kHeld = HELD ? kHeldBlocks * BN * 128 : 0;
  // K blocks per stage: with few queries a block is so little work that handing
  // it over took longer (256 groups of FP8, 32 x 1024 x 512 on average: 37.6 us with
  // one block, 34.5 with two)
  static constexpr uint32_t kPer = ROWS && BN <= 64 ? 2 : 1;
  static constexpr uint32_t kBlockBytes = kABytes + (HELD ? 0 : BN * 128);
  static constexpr uint32_t kStage = kPer * kBlockBytes;
  static constexpr int kStages = (int)((200u * 1024 - kHeld) / kStage);
  static constexpr int kEpiWarps = ROWS ? 8 : 16;
  static constexpr int kThreads = 32 * (4 + kEpiWarps + (FP8 ? 4 : 0));
  static constexpr int kConsumers = 2 + kEpiWarps + (FP8 ? 4 : 0);  // arrivals that free a tile slot
  static constexpr int kSubs = ROWS && BN < 128 ? 128 / BN : 1;              // most accumulators per tile
  static constexpr uint32_t kTileQ = ROWS ? BN : kBM;                // queries per tile
  static constexpr uint32_t kTileV = ROWS ? kBM : BN;                // rows of v per accumulator
  static constexpr uint32_t kBars = kStages * kStage + kHeld;
  // full[S], empty[S], acc_full[2], acc_empty[2], info_full[I], info_empty[I], sf_full[F], sf_empty[F], drain, held
  static constexpr uint32_t kNumBars = 2 * kStages + 4 + 2 * kInfo + 2 * kSf + 2;
  static constexpr uint32_t kExps = (kBars + kNumBars * 8 + 127) / 128 * 128;
  static constexpr uint32_t kExpBuf = (1 + (BN + 127) / 128) * kSfBytes;
  static constexpr uint32_t kHeldExps = kExps + (FP8 ? kSf * kExpBuf : 0);
  static constexpr uint32_t kTiles = kHeldExps + (HELD ? BN * kHeldBlocks : 0);
  static constexpr uint32_t kSlot = kTiles + kInfo * (uint32_t)sizeof(Tile);
  static constexpr uint32_t kBytes = kSlot + 16 + 1024;
  static constexpr uint32_t kAccBuf = kSubs * BN;
  static constexpr uint32_t kAcc = 2 * kAccBuf;  // accumulator columns
  static constexpr uint32_t kUsed = kAcc + (FP8 ? kSf * kSfCols : 0);
  static constexpr uint32_t kTmem = kUsed <= 64 ? 64 : kUsed <= 128 ? 128 : kUsed <= 256 ? 256 : 512;
  static_assert(kUsed <= 512, "tensor memory has 512 columns");
  static_assert(kBytes <= 227 * 1024, "shared memory of a CTA");
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

// The last chunk with at most t tiles before it (t is less than all their tiles),
// 32 guesses at a time.
__device__ __noinline__ uint32_t chunk_of_tile(const Chunk* chunks, uint32_t count, uint64_t t) {
  uint32_t lo = 0;
  while (count > 1) {
    const uint32_t step = (count + 31) / 32, c = (threadIdx.x & 31) * step;
    const uint32_t at = 31 - __clz(__ballot_sync(0xffffffffu, c < count && (uint64_t)chunks[lo + c].tiles <= t));
    lo += at * step;
    count = min(step, count - at * step);
  }
  return lo;
}

// Finds the tiles of one CTA, in order, by one warp: groups are read 32 at a
// time (one per lane) and their tiles counted by a warp scan; a CTA's tiles
// rise, so the groups are walked once. MANY groups, whose walk would take longer
// than the tiles: the sums before each chunk of 32 groups are there, a tile's
// chunk is searched for, and a CTA takes runs of up to 32 consecutive tiles,
// which mostly share a chunk (65536 groups of 1 x 8 scores 1400 to 313 us).
// The lane that holds a tile's group works out the tile. Its divisions are 32-bit
// ones unless the group has 2^32 tiles.
// A group whose scores start past the output's capacity ends the CTA's tiles:
// what they hold cannot be stored, and offsets that fall again and again could
// ask for any amount of it. It also keeps the place of a tile's scores below
// 2^62 plus a group's, so sums with it do not wrap.
template <typename L, bool MANY>
struct TileFinder {
  static constexpr uint32_t TQ = L::kTileQ;
  const Params& p;
  int lane;
  uint64_t first = 0;       // first tile of the chunk
  int64_t out0 = 0;         // output elements before the chunk
  uint32_t g0 = 0u - kChunk;  // its first group
  uint64_t incl = 0;        // this lane's group: tiles up to and with it, in the chunk
  uint64_t tiles = 0;
  int64_t before = 0;       // output elements before it, in the chunk
  uint64_t chunk_tiles = 0;
  int64_t chunk_out = 0;
  uint32_t qa = 0, va = 0, m = 0, nn = 0;  // its first query and row, how many
  uint32_t rows;            // of v per tile
  uint64_t t;               // the CTA's next tile
  uint64_t skip;            // from the last tile of a run to the next run
  uint32_t run = 1, left;   // consecutive tiles that the CTA takes, how many are left
  uint32_t open = 0;        // lanes whose group's scores start within the output
  bool bad = false, past = false;

  __device__ TileFinder(const Params& p_, int lane_) : p(p_), lane(lane_), rows(L::kTileV * p_.subs - p_.halo) {
    if constexpr (MANY) {
      const uint64_t total = (uint64_t)p.chunks[p.nchunks].tiles;
      run = (uint32_t)max((uint64_t)1, min((uint64_t)kChunk, total / (8 * (uint64_t)gridDim.x)));
    }
    left = run;
    t = (uint64_t)blockIdx.x * run;
    skip = (uint64_t)(gridDim.x - 1) * run + 1;
  }
  __device__ void next() {
    if (MANY && --left) {
      ++t;
    } else {
      t += skip;
      left = run;
    }
  }

  __device__ void load() {
    const uint32_t g = g0 + (uint32_t)lane;
    qa = va = m = nn = 0;
    if (g < p.groups) {
      if (p.qo) {
        int64_t q0, v0, mq, mv;
        bad |= !group_of(p.qo, p.vo, g, p.nq, p.n, q0, v0, mq, mv);
        qa = (uint32_t)q0;
        va = (uint32_t)v0;
        m = (uint32_t)mq;
        nn = (uint32_t)mv;
      } else {
        m = (uint32_t)p.nq;
        nn = (uint32_t)p.n;
      }
    }
    tiles = (uint64_t)((m + TQ - 1) / TQ) * ((nn + rows - 1) / rows);
    incl = tiles;
    int64_t e = (int64_t)m * nn;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t y = __shfl_up_sync(0xffffffffu, incl, o);
      const int64_t x = __shfl_up_sync(0xffffffffu, e, o);
      if (lane >= o) {
        incl += y;
        e += x;
      }
    }
    before = e - (int64_t)m * nn;
    // (unsigned: a sum of wild offsets that has wrapped is past it too)
    open = __ballot_sync(0xffffffffu, !p.qo || (uint64_t)out0 + (uint64_t)before < p.capacity);
    chunk_tiles = __shfl_sync(0xffffffffu, incl, 31);
    chunk_out = __shfl_sync(0xffffffffu, e, 31);
  }

  // The lane whose group holds tile t; -1 when there is none.
  __device__ int find() {
    while (t >= first + chunk_tiles) {
      uint32_t g = g0 + kChunk;
      first += chunk_tiles;
      out0 += chunk_out;
      if constexpr (MANY) {
        if (t >= (uint64_t)p.chunks[p.nchunks].tiles) return -1;
        const uint32_t c = chunk_of_tile(p.chunks, p.nchunks, t);
        g = c * kChunk;
        first = (uint64_t)p.chunks[c].tiles;
        out0 = p.chunks[c].out;
      }
      if (g >= p.groups) return -1;
      g0 = g;
      load();
      if (MANY) break;  // it is this one
    }
    const int at = __ffs(__ballot_sync(0xffffffffu, t - first < incl)) - 1;
    if (at < 0 || (open >> at & 1u)) return at;
    past = true;
    if (!MANY)  // the offsets behind it are looked at all the same
      for (uint32_t g = g0 + kChunk; g < p.groups; g += kChunk) {
        g0 = g;
        load();
      }
    return -1;
  }
  // Tile t of this lane's group.
  __device__ Tile tile() const {
    const uint64_t in = t - first - (incl - tiles);
    // bands of kBand query tiles; in a band, all its query tiles of one row tile before the next
    const uint32_t mt = (m + TQ - 1) / TQ, nt = (nn + rows - 1) / rows;
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
    // even query tiles (at most TQ, so mt - 1 of them are less than m): with a
    // short last one, the CTAs that always got that one had less to do
    const uint32_t step = mt == 1 ? TQ : ((m + mt - 1) / mt + 15) / 16 * 16;
    Tile r;
    r.ld = p.qo ? (int64_t)nn : (int64_t)p.ld;
    r.out = out0 + before + (int64_t)(qi * step) * r.ld + (int64_t)ti * rows;
    r.vrow = va + ti * rows;
    r.qrow = qa + qi * step;
    r.vcnt = min(rows, nn - ti * rows);
    r.qcnt = min(step, m - qi * step);
    r.vext = min(rows + p.halo, nn - ti * rows);
    r.first = ti == 0;
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

// 8 or 16 consecutive accumulator columns of this thread's lane, without waiting.
__device__ inline void tmem_ld(uint32_t taddr, uint32_t (&v)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
               : "r"(taddr));
}
__device__ inline void tmem_ld(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];\n"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr));
}
// Waits for the loads; ties the registers to the wait.
template <int N>
__device__ inline void tmem_wait_ld(uint32_t (&v)[N]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(v[i]));
}

__device__ inline bool elect_one() {
  uint32_t is;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(is)::"memory");
  return is != 0;
}
// The whole warp waits; one answer for all lanes. The clock is read only when
// the phase is not complete at the first look.
__device__ inline bool warp_wait(uint32_t bar, uint32_t parity) {
  long long t0 = 0;
  while (true) {
    uint32_t done;
    asm volatile(
        "{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\nselp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(done)
        : "r"(bar), "r"(parity), "r"(kSleepNs)
        : "memory");
    if (__all_sync(0xffffffffu, done != 0)) return true;
    const long long t = clock64();
    if (t0 == 0) t0 = t;
    if (__any_sync(0xffffffffu, t - t0 > raven_tc::kWaitCycles)) return false;
  }
}

// The accumulators of a tile are read: the MMA warp may fill them again.
__device__ inline void free_acc(uint32_t bar, uint32_t lane) {
  tc_fence_before();
  __syncwarp();
  if (lane == 0) mbar_arrive(bar);
}
__device__ inline void put(float* p, float v) { *p = v; }
__device__ inline void put(__half* p, float v) { *p = __float2half_rn(v); }
__device__ inline void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// Layout by rows: a lane holds one row of v. Two warps per lane quadrant take 16
// queries in turn.
template <int BN, typename T>
__device__ inline void store_rows(T* out, const Tile& t, uint32_t qcnt, uint32_t acc, uint32_t warp, uint32_t lane,
                                 float alpha, const float* bias, uint32_t acc_empty) {
  const uint32_t r = (warp & 3) * 32 + lane, first = 16 * (warp >> 2);
  const uint32_t subs = (t.vcnt + kBM - 1) / kBM;
  for (uint32_t sub = 0; sub < subs && first < qcnt; ++sub) {
    const bool row = r + sub * kBM < t.vcnt;
    const float add = bias && row ? bias[sub * kBM + r] : 0.0f;
    T* o = out + t.out + sub * kBM + r + (int64_t)first * t.ld;
    for (uint32_t c = first; c < qcnt; c += 32, o += 32 * t.ld) {
      uint32_t v[16];
      tmem_ld(acc + sub * BN + c, v);
      tmem_wait_ld(v);
      if (row) {
        T* q = o;
        if (c + 16 <= qcnt) {
#pragma unroll
          for (int j = 0; j < 16; ++j, q += t.ld) put(q, fmaf(alpha, __uint_as_float(v[j]), add));
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j, q += t.ld)
            if (c + j < qcnt) put(q, fmaf(alpha, __uint_as_float(v[j]), add));
        }
      }
      __syncwarp();
    }
  }
  free_acc(acc_empty, lane);
}

__device__ inline uint32_t word_of(const uint32_t (&v)[8], int i, const float*) { return v[i]; }
__device__ inline uint32_t word_of(const uint32_t (&v)[16], int i, const __half*) {
  const __half2 h = __floats2half2_rn(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
  return *(const uint32_t*)&h;
}
__device__ inline uint32_t word_of(const uint32_t (&v)[16], int i, const __nv_bfloat16*) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
  return *(const uint32_t*)&h;
}

// Layout by pairs: a lane holds one query; four warps per lane quadrant share the
// columns. A step makes one 32-byte sector (8 words, SC scores) of each query.
// Where a query's scores start inside a sector (after `lead` others), the sector
// is put together from the words of this step and the last: selects move the
// pair of them by 8, 4, 2 and 1 words, a funnel shift by half a word. A warp
// writes the sectors that start among its own scores, and takes what the last
// one needs from the columns after them (a tile computes that much of the next
// one), so that only a query's first and last sectors are written in part:
// 999 x 250007 bf16 scores took 460 us when every warp wrote its ends in part, and
// 999 x 250000, where every sector is whole, 124. Halves of sectors are as bad
// (2.1 TB/s for 16-byte stores alone, 4.9 for 32-byte ones).
template <int BN, typename T>
__device__ inline void store_pairs(T* out, const Tile& t, uint32_t qcnt, uint32_t acc, uint32_t warp, uint32_t lane,
                                   float alpha, const float* bias, uint32_t acc_empty) {
  constexpr uint32_t SC = 32 / sizeof(T);
  const uint32_t per = (t.vcnt + 63) / 64 * 16;  // columns per warp
  const uint32_t first = (warp >> 2) * per, q = (warp & 3) * 32 + lane;
  if ((warp & 3) * 32 >= qcnt || first >= t.vcnt) {
    free_acc(acc_empty, lane);
    return;
  }
  const uint32_t cols = min(per, t.vcnt - first), avail = t.vext - first;
  const uint64_t start = (uint64_t)(uintptr_t)(out + t.out + (int64_t)q * t.ld + first);
  const uint32_t lead = (uint32_t)(start & 31u) / sizeof(T);
  const uint32_t shift = SC - lead;  // scores from the last step's first to the sector's
  const bool straight = !__any_sync(0xffffffffu, lead != 0);
  const uint32_t steps = (cols + SC - 1) / SC + (straight ? 0 : 1);
  const uint32_t own = q < qcnt ? lead + cols : 0;                   // sectors from here on are another's
  const uint32_t from = t.first && first == 0 ? 0 : lead;            // and before here
  uint64_t sector = start & ~(uint64_t)31;
  uint32_t v[SC], x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  tmem_ld(acc + first, v);
  for (uint32_t k = 0; k < steps; ++k, sector += 32) {
    tmem_wait_ld(v);
    uint32_t w[8];
    if (alpha != 1.0f || bias) {
#pragma unroll
      for (uint32_t i = 0; i < SC; ++i) {
        const uint32_t c = SC * k + i;
        v[i] = __float_as_uint(fmaf(alpha, __uint_as_float(v[i]), bias && c < avail ? bias[first + c] : 0.0f));
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = word_of(v, i, (const T*)0);
    if (k + 1 < steps)
      tmem_ld(acc + min(first + SC * (k + 1), (uint32_t)BN - SC), v);  // the last may have no columns left, nor use for them
    if (!straight) {
      uint32_t y[17];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        y[i] = x[i];
        y[8 + i] = x[i] = w[i];
      }
      y[16] = 0;
      const uint32_t by = shift * sizeof(T) / 4;  // words, 0..8: 8 takes this step's words as they are
#pragma unroll
      for (int i = 0; i < 9; ++i) y[i] = by & 8 ? y[i + 8] : y[i];
#pragma unroll
      for (int i = 0; i < 13; ++i) y[i] = by & 4 ? y[i + 4] : y[i];
#pragma unroll
      for (int i = 0; i < 11; ++i) y[i] = by & 2 ? y[i + 2] : y[i];
#pragma unroll
      for (int i = 0; i < 9; ++i) y[i] = by & 1 ? y[i + 1] : y[i];
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = sizeof(T) == 2 ? __funnelshift_r(y[i], y[i + 1], (shift & 1) * 16) : y[i];
    }
    const uint32_t at = SC * k;  // scores from the first sector's start
    if (at >= lead && at < own && at + SC <= lead + avail) {
      asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"l"(sector), "r"(w[0]), "r"(w[1]),
                   "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                   : "memory");
    } else if (at >= from && at < own) {  // a query's first or last sector
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i) {
        if constexpr (sizeof(T) == 4) {
          if (at + i >= lead && at + i < lead + avail) *(uint32_t*)(sector + 4 * i) = w[i];
        } else {
          const uint32_t h = at + 2 * i;
          if (h >= lead && h < lead + avail) *(uint16_t*)(sector + 4 * i) = (uint16_t)w[i];
          if (h + 1 >= lead && h + 1 < lead + avail) *(uint16_t*)(sector + 4 * i + 2) = (uint16_t)(w[i] >> 16);
        }
      }
    }
  }
  free_acc(acc_empty, lane);
}

// (HELD) Encodes the queries into shared memory as the copies would leave them
// (128-byte rows, 16-byte pieces swizzled by row), by the epilogue warps.
template <typename T>
__device__ inline void hold_queries(const Params& p, uint8_t* held, uint8_t* exps, uint32_t warp, uint32_t lane) {
  constexpr uint32_t W = 8, U = kHeldUnits / W;
  const uint32_t units = (uint32_t)p.nq * p.nkb;
  float x[U][4];
#pragma unroll
  for (uint32_t k = 0; k < U; ++k) {  // all reads under way at once
    const uint32_t u = warp + W * k, row = u / p.nkb, d = (u - row * p.nkb) * 128 + 4 * lane;
    const T* r = (const T*)p.qx + row * p.ld_qx;
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) x[k][i] = u < units && d + i < p.dim ? raven_fp8::load_value(r + d + i) : 0.0f;
  }
#pragma unroll
  for (uint32_t k = 0; k < U; ++k) {
    const uint32_t u = warp + W * k, row = u / p.nkb, b = u - row * p.nkb;
    if (u >= units) break;
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t a = __float_as_uint(x[k][i]) & 0x7fffffffu;
      if (a < 0x7f800000u) top = max(top, a);
    }
    const int e = raven_fp8::exponent_of(__reduce_max_sync(0xffffffffu, top));
    const uint32_t word = raven_fp8::with_nan(raven_fp8::codes_of(x[k], raven_fp8::inverse_of(e)), x[k]);
    *(uint32_t*)(held + b * (32 * 128) + row * 128 + ((lane / 4) ^ (row & 7)) * 16 + (lane % 4) * 4) = word;
    if (lane == 0) exps[row * kHeldBlocks + b] = (uint8_t)(e + 127);
  }
}

template <bool FP8, int BN, bool ROWS, bool HELD>
__global__ void __launch_bounds__((Layout<FP8, BN, ROWS, HELD>::kThreads), 1)
    score_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_v, const Params p) {
  using L = Layout<FP8, BN, ROWS, HELD>;
  constexpr int S = L::kStages, kEpiWarps = L::kEpiWarps;
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
  const uint32_t held = drain + 8;  // (HELD) the queries are in place
  const uint32_t held_at = sbase + (uint32_t)S * L::kStage;
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
      mbar_init(acc_empty(b), kEpiWarps);
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
    mbar_init(held, kEpiWarps);
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
      const uint32_t qcnt = tiles[rd.slot].qcnt, vcnt = tiles[rd.slot].vcnt, qrow = tiles[rd.slot].qrow;
      const uint32_t vrow = tiles[rd.slot].vrow;
      __syncwarp();
      if (lane == 0) mbar_arrive(info_empty(rd.slot));
      rd.next();
      if (qcnt == 0) break;
      const uint32_t boxes = (qcnt + kQBox - 1) / kQBox;  // (rows)
      for (uint32_t sub = 0; sub * L::kTileV < vcnt && ok; ++sub)
        for (uint32_t kb = 0; kb < p.nkb; kb += L::kPer) {
          if (!warp_wait(empty(s), ph ^ 1u)) {
            ok = false;
            break;
          }
          if (elect_one()) {
            const uint32_t bar = full(s), blocks = min(L::kPer, p.nkb - kb);
            if constexpr (ROWS)
              mbar_expect_tx(bar, blocks * (kABytes + (HELD ? 0 : boxes * (kQBox * 128))));
            else
              mbar_expect_tx(bar, blocks * L::kBlockBytes);
#pragma unroll
            for (uint32_t j = 0; j < L::kPer; ++j) {
              if (j >= blocks) break;
              const uint32_t a = sbase + s * L::kStage + j * L::kBlockBytes;
              const int x = (int)((kb + j) * (FP8 ? 128u : 64u));
              if constexpr (ROWS) {
                tma_load_2d(a, &tm_v, x, (int)(vrow + sub * kBM), bar);
                if constexpr (!HELD)
                  for (uint32_t b = 0; b < boxes; ++b)
                    tma_load_2d(a + kABytes + b * (kQBox * 128), &tm_q, x, (int)(qrow + b * kQBox), bar);
              } else {
                tma_load_2d(a, &tm_q, x, (int)qrow, bar);
                tma_load_2d(a + kABytes, &tm_v, x, (int)vrow, bar);
              }
            }
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
    if (HELD) ok = warp_wait(held, 0);
    while (ok) {
      if (!warp_wait(info_full(rd.slot), rd.phase)) {
        ok = false;
        break;
      }
      const uint32_t qcnt = __shfl_sync(0xffffffffu, tiles[rd.slot].qcnt, 0);
      const uint32_t vcnt = __shfl_sync(0xffffffffu, ROWS ? tiles[rd.slot].vcnt : tiles[rd.slot].vext, 0);
      if (lane == 0) mbar_arrive(info_empty(rd.slot));
      rd.next();
      if (qcnt == 0) break;
      const uint32_t idesc = p.idesc | ((((ROWS ? qcnt : vcnt) + 15u) / 16u * 2u) << 17);  // N, a multiple of 16, in eights
      if (!warp_wait(acc_empty(b), bph ^ 1u)) {
        ok = false;
        break;
      }
      tc_fence_after();
      for (uint32_t sub = 0; sub * L::kTileV < vcnt && ok; ++sub) {
        const uint32_t d = tmem + b * L::kAccBuf + sub * BN;
        const bool last_sub = (sub + 1) * L::kTileV >= vcnt;
        for (uint32_t kb = 0; kb < p.nkb; kb += L::kPer) {
          if (FP8 && (kb & 3u) == 0 && !warp_wait(sf_full(f), fph)) {
            ok = false;
            break;
          }
          if (!warp_wait(full(s), ph)) {
            ok = false;
            break;
          }
          const uint32_t a0 = sbase + s * L::kStage, done = empty(s);
          const bool last = kb + L::kPer >= p.nkb;
          const bool sf_done = FP8 && ((kb & 3u) == 4u - L::kPer || last);
          const uint32_t sf = tmem + L::kAcc + f * kSfCols;
          if (++s == S) {
            s = 0;
            ph ^= 1u;
          }
          if (elect_one()) {
            if (FP8 && (kb & 3u) == 0) {  // in order before the MMAs that read them
              const uint32_t e = sbase + L::kExps + f * L::kExpBuf;
#pragma unroll
              for (int j = 0; j < 1 + (BN + 127) / 128; ++j) copy_exps(sf + 4 * j, e + j * kSfBytes);
            }
#pragma unroll
            for (uint32_t j = 0; j < L::kPer; ++j) {
              if (kb + j >= p.nkb) break;
              const uint32_t a = a0 + j * L::kBlockBytes;
              const uint64_t da = sw128_desc(a), db = sw128_desc(HELD ? held_at + (kb + j) * (BN * 128) : a + kABytes);
              const uint32_t steps = kb + j + 1 == p.nkb ? p.last_k : 4u, sel = (kb + j) & 3u;
#pragma unroll
              for (uint32_t k = 0; k < 4; ++k) {  // 32 bytes along the swizzled row
                if (k >= steps) break;
                if constexpr (FP8)
                  mma_mxf8(d, da + 2 * k, db + 2 * k, idesc | (sel << 4) | (sel << 29), sf, sf + 4, (kb | j | k) != 0u);
                else
                  mma_f16(d, da + 2 * k, db + 2 * k, idesc, (kb | j | k) != 0u);
              }
            }
            mma_commit(done);
            if (sf_done) mma_commit(sf_empty(f));
            if (last && last_sub) mma_commit(acc_full(b));
          }
          __syncwarp();
          if (sf_done && ++f == kSf) {
            f = 0;
            fph ^= 1u;
          }
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
    auto find_tiles = [&](auto finder) {
      TileReader wr;
      for (;; finder.next()) {
        const int at = finder.find();
        if (!warp_wait(info_empty(wr.slot), wr.phase ^ 1u)) {
          ok = false;
          break;
        }
        if (lane == max(at, 0)) {
          if (at < 0)
            tiles[wr.slot].qcnt = 0;
          else
            tiles[wr.slot] = finder.tile();
          mbar_arrive(info_full(wr.slot));
        }
        __syncwarp();
        wr.next();
        if (at < 0) break;
      }
      const int bits = (__any_sync(0xffffffffu, finder.bad) ? kStatusOffsets : 0) | (finder.past ? kStatusCapacity : 0);
      if (bits && lane == 0) tell(p.status, bits);
    };
    if (p.chunks)
      find_tiles(TileFinder<L, true>(p, lane));
    else
      find_tiles(TileFinder<L, false>(p, lane));
  } else if (warp >= 4 && warp < 4 + kEpiWarps) {  // epilogue
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    if constexpr (HELD) {
      uint8_t *to = smem + S * L::kStage, *ex = smem + L::kHeldExps;
      if (p.q_type == kOutF32)
        hold_queries<float>(p, to, ex, (uint32_t)(warp - 4), (uint32_t)lane);
      else if (p.q_type == kOutF16)
        hold_queries<__half>(p, to, ex, (uint32_t)(warp - 4), (uint32_t)lane);
      else
        hold_queries<__nv_bfloat16>(p, to, ex, (uint32_t)(warp - 4), (uint32_t)lane);
      asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(held);
    }
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
      // queries whose scores of this tile lie within the output
      uint32_t qcnt = t.qcnt;
      if (p.qo && t.out + (int64_t)(qcnt - 1) * t.ld + t.vext > (int64_t)p.capacity) {
        const int64_t room = (int64_t)p.capacity - t.out - (int64_t)t.vext;
        qcnt = room < 0 ? 0u : (uint32_t)min(room / t.ld + 1, (int64_t)qcnt);
        if (lane == 0 && qcnt < t.qcnt) tell(p.status, kStatusCapacity);
      }
      if (!warp_wait(acc_full(b), bph)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint32_t acc = tmem + lane_base + b * L::kAccBuf, w = (uint32_t)(warp - 4);
      const float* bias = p.bias ? p.bias + t.vrow : nullptr;
      if constexpr (ROWS) {
        if (p.out_type == kOutF32)
          store_rows<BN>((float*)p.out, t, qcnt, acc, w, lane, p.alpha, bias, acc_empty(b));
        else if (p.out_type == kOutF16)
          store_rows<BN>((__half*)p.out, t, qcnt, acc, w, lane, p.alpha, bias, acc_empty(b));
        else
          store_rows<BN>((__nv_bfloat16*)p.out, t, qcnt, acc, w, lane, p.alpha, bias, acc_empty(b));
      } else {
        if (p.out_type == kOutF32)
          store_pairs<BN>((float*)p.out, t, qcnt, acc, w, lane, p.alpha, bias, acc_empty(b));
        else if (p.out_type == kOutF16)
          store_pairs<BN>((__half*)p.out, t, qcnt, acc, w, lane, p.alpha, bias, acc_empty(b));
        else
          store_pairs<BN>((__nv_bfloat16*)p.out, t, qcnt, acc, w, lane, p.alpha, bias, acc_empty(b));
      }
      b ^= 1u;
      bph ^= b == 0u;
    }
  } else if (FP8 && warp >= 4 + kEpiWarps) {  // exponents
    // Thread r takes row r of the M side and rows r and r + 128 of the N side:
    // the word of row 32 j + i goes to lane i, column j. The next words are on
    // their way while these are stored.
    constexpr int kParts = 1 + (BN + 127) / 128;
    const uint32_t r = threadIdx.x - 32 * (4 + kEpiWarps);
    TileReader rd;
    uint32_t kb = p.nkb, sub = 0, vrow = 0, vcnt = 0;
    const uint8_t* src[kParts];
    auto load = [&](uint32_t (&w)[kParts]) {  // false: no more, or a wait ran out
      kb += 4;
      if (kb >= p.nkb) {
        kb = 0;
        if (++sub * L::kTileV >= vcnt) {
          if (!warp_wait(info_full(rd.slot), rd.phase)) {
            ok = false;
            return false;
          }
          const uint32_t qrow = tiles[rd.slot].qrow, qcnt = tiles[rd.slot].qcnt;
          vrow = tiles[rd.slot].vrow;
          vcnt = ROWS ? tiles[rd.slot].vcnt : tiles[rd.slot].vext;
          __syncwarp();
          if (lane == 0) mbar_arrive(info_empty(rd.slot));
          rd.next();
          if (qcnt == 0) return false;
          sub = 0;
          // rows past what the tile or the array has repeat the last one
          if constexpr (HELD) {
            src[1] = smem + L::kHeldExps + min(r, qcnt - 1) * kHeldBlocks;
          } else if constexpr (ROWS) {
#pragma unroll
            for (int j = 1; j < kParts; ++j)
              src[j] = p.qe + ((uint64_t)qrow + min(r + 128u * (j - 1), qcnt - 1)) * p.ld_qe;
          } else {
            src[0] = p.qe + ((uint64_t)qrow + min(r, qcnt - 1)) * p.ld_qe;
#pragma unroll
            for (int j = 1; j < kParts; ++j)
              src[j] = p.ve + ((uint64_t)vrow + min(r + 128u * (j - 1), vcnt - 1)) * p.ld_ve;
          }
        }
        if constexpr (ROWS) src[0] = p.ve + min((uint64_t)vrow + sub * kBM + r, p.n - 1) * p.ld_ve;
      }
#pragma unroll
      for (int j = 0; j < kParts; ++j)
        w[j] = *(const uint32_t*)(src[j] + kb);
      return true;
    };
    uint32_t f = 0, fph = 0, w[kParts], next[kParts];
    if (HELD) ok = warp_wait(held, 0);
    bool more = ok && load(w);
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
  if (!ok && lane == 0) tell(p.status, kStatusWait);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 2) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(L::kTmem) : "memory");
  }
}

}  // namespace raven_score
