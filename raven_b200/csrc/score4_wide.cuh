// Scores of more than a few queries against 4-bit rows: as score4.cuh, with the sums
// by tcgen05.mma. 32, 64 or 96 columns (queries; two for one of f32) are the N side, 128
// rows the M side. What a warp of mma.sync instructions does per query (fragments
// from shared memory, sums in registers) took more instructions than the codes
// themselves from 16 columns on.
//
// A group of four warps takes a tile of 128 rows, a row a thread. Codes come by TMA;
// a thread turns its row's 128 codes of a block into f16 operands code + z (as many
// instructions as code - 8 in score4.cuh; z is its own row's) and writes them to
// tensor memory, which the instruction reads its M side from: shared memory holds
// queries only, and its bandwidth goes to them. A scale group is a chain of
// instructions of its own; the thread then reads its row's sums of the group and adds
// them, times the group's step, to its own in registers. Three or four such groups of
// warps per SM (teams) work on tiles of their own, so that one's instructions and waits
// are hidden by the others'. A thread has all scores of its row, and a warp writes 32
// scores of a query side by side, wherever the query's scores start.
//
// What bounds it: a team's chain on a block (operands, instructions, sums). Chains of 32
// and of 64 columns took the same time, as if an instruction of 16 values took about 64
// cycles, three teams' waiting for one another. 64 x 1000000 x 128 70 us, 4.7 TB/s;
// 32 x 65536 x 1024 23.5 us, 1.9 TB/s.
#pragma once

#include "score4.cuh"
#include "waits.h"

namespace raven_score4 {

// A chunk of queries: K blocks of 64 values (two units), for each column 128 bytes
// in the 128-byte swizzle; then what brings sums back.
template <int NC>
struct WideLaid {
  static constexpr uint32_t kColumns = NC;
  static constexpr uint32_t kBlockBytes = NC * 128;
  __host__ __device__ static uint64_t frags(uint32_t units) { return (uint64_t)((units + 1) / 2) * kBlockBytes; }
  __host__ __device__ static uint64_t sums(uint32_t) { return 0; }  // z is added to the codes
  __host__ __device__ static uint64_t bytes(uint32_t units, uint32_t) { return frags(units) + NC * 16; }
  __device__ static uint32_t frag_at(uint32_t unit, uint32_t quarter, uint32_t col) {
    return unit / 2 * kBlockBytes + col * 128 + ((((unit & 1) * 4 + quarter) ^ (col & 7)) * 16);
  }
  __device__ static void put_sum(uint8_t*, uint32_t, uint32_t, float) {}
  // What brings query q's sums back: three factors, whether the last two are not 1.
  __device__ static void put_back(float* back, uint32_t q, float f, float k0, float k1, float flag) {
    back[q] = f;
    back[NC + 2 * q] = k0;
    back[NC + 2 * q + 1] = k1;
    back[3 * NC + q] = flag;
  }
};

constexpr uint32_t kWideRows = 128;  // of a tile
constexpr uint32_t kWideDepth = 4;   // tiles under way per team, at most
constexpr uint32_t kWideStage = kWideRows * 64;

template <int NC>
struct Wide {
  // tensor memory of a team: operands of a block, a group's sums
  static constexpr uint32_t kAcc = 64, kTeam = kAcc + NC;
  static constexpr uint32_t kTeams = NC == 32 ? 4 : 3, kThreads = kTeams * 128;
  static_assert(kTeams * kTeam <= 512, "tensor memory has 512 columns");
  static constexpr uint32_t kHead = 1024;  // barriers, the place of the tensor memory; TMA's places start on 1024 bytes
  static constexpr uint32_t kTops = NC * 4;
  __host__ __device__ static uint64_t bytes(uint32_t units, uint32_t depth) {
    return 1024 + kHead + (uint64_t)kTeams * depth * kWideStage + WideLaid<NC>::bytes(units, 0) + kTops;
  }
};

// What is added to a row's codes of a group, in units of 2^-12 (kCodeShift): z - 1024 to 1024 + code, z - 64 to a
// sixteenth of 1024 + 16 code. All are whole numbers below 2048, which f16 holds. z + 128 at the bottom of 1024
// is 1152 + z.
struct Offsets {
  __half2 low, high;
  __device__ explicit Offsets(uint32_t word) {
    const uint32_t b = __byte_perm(word, kCodeBase >> 24, 0x4040) ^ 0x00800080u;
    const __half2 z = __hsub2(*(const __half2*)&b, __float2half2_rn(1152.f * kCodeScale));
    low = __hadd2(z, __float2half2_rn(-1024.f * kCodeScale));
    high = __hadd2(z, __float2half2_rn(-64.f * kCodeScale));
  }
};
// Eight codes, with z, as four operands of two.
__device__ inline void operands(uint32_t w, const Offsets& z, uint32_t& a0, uint32_t& a1, uint32_t& a2, uint32_t& a3) {
  auto low = [&](uint32_t code) {
    const __half2 r = __hadd2(*(const __half2*)&code, z.low);
    return *(const uint32_t*)&r;
  };
  auto high = [&](uint32_t code) {
    const __half2 r = __hfma2(*(const __half2*)&code, __float2half2_rn(0.0625f), z.high);
    return *(const uint32_t*)&r;
  };
  const uint32_t v = w >> 8;
  a0 = low((w & 0x000f000fu) | kCodeBase);
  a1 = high((w & 0x00f000f0u) | kCodeBase);
  a2 = low((v & 0x000f000fu) | kCodeBase);
  a3 = high((v & 0x00f000f0u) | kCodeBase);
}

__device__ inline void tmem_st16(uint32_t at, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};\n" ::"r"(at),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ inline void tmem_ld16(uint32_t at, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];\n"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(at));
}
// Waits for the loads; ties the registers to the wait.
template <int N>
__device__ inline void tmem_wait_ld(uint32_t (&v)[N][16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
  for (int j = 0; j < N; ++j)
#pragma unroll
    for (int i = 0; i < 16; ++i) asm volatile("" : "+r"(v[j][i]));
}
// M side in tensor memory, N side in shared memory.
__device__ inline void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t add) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(add)
      : "memory");
}
// All lanes of a warp wait; one answer.
__device__ inline bool warp_waits(uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)); }

template <int NC, int G, bool F32, typename O>
__global__ void __launch_bounds__(Wide<NC>::kThreads, 1) wide_kernel(const __grid_constant__ CUtensorMap map, const Params p) {
  using Q = WideLaid<NC>;
  using S = Wide<NC>;
  constexpr uint32_t kQueries = F32 ? NC / 2 : NC, W = kBlock / G, U = G / kUnit;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t tid = threadIdx.x, warp = tid / 32, lane = tid & 31, team = warp / 4, row_of = tid & 127;
  const uint32_t bars = smem_u32(smem) + team * 64;  // full[depth], done
  const uint32_t done = bars + 8 * kWideDepth;
  volatile uint32_t* slot_of_tmem = (volatile uint32_t*)(smem + 512);
  uint8_t* ring = smem + S::kHead + team * p.depth * kWideStage;
  uint8_t* held = smem + S::kHead + S::kTeams * p.depth * kWideStage;
  const uint32_t shares = p.chunks * p.slices, share = blockIdx.x % shares;
  const uint32_t step = gridDim.x / shares * S::kTeams, first = blockIdx.x / shares * S::kTeams + team;
  const uint32_t slice = share % p.slices;
  const uint64_t chunk = share / p.slices;
  const uint32_t b0 = slice * p.slice, blocks = min(p.slice, p.blocks - b0);
  const uint32_t units = min(4 * p.slice, p.units - 4 * b0);
  if (row_of == 0) {
    for (uint32_t i = 0; i < kWideDepth + 1; ++i) mbar_init(bars + 8 * i, 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32((void*)slot_of_tmem)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  raven_tc::tc_fence_before();
  __syncthreads();
  raven_tc::tc_fence_after();
  const uint32_t tmem = *slot_of_tmem + team * S::kTeam;
  const uint32_t mine = tmem + ((warp & 3) << 21);  // this warp's 32 lanes
  after_previous();

  // copies: by the team's first thread
  Ring stages;
  uint32_t ahead = first, ahead_b = 0;
  auto copy_next = [&]() {
    if (ahead < p.tiles) {
      const uint32_t bar = bars + 8 * stages.slot;
      mbar_expect_tx(bar, kWideStage);
      tma_load_2d(smem_u32(ring) + stages.slot * kWideStage, &map, (int)(64 * (b0 + ahead_b)),
                  (int)min((uint64_t)ahead * kWideRows, p.n), bar);
      stages.begun(p.depth);
      if (++ahead_b == blocks) {
        ahead_b = 0;
        ahead += step;
      }
    }
  };
  if (row_of == 0)
    for (uint32_t i = 0; i < p.depth; ++i) copy_next();

  float* back = (float*)(held + Q::frags(units));
  if (p.q) {
    lay_out_any<Q, G, F32>(p, chunk * kQueries, kQueries, 0, 4 * b0, units, 0, held, (uint32_t*)(back + 4 * NC));
  } else {
    const uint8_t* from = p.laid + chunk * Q::bytes(p.units, 0);
    auto bring = [&](void* to, const uint8_t* what, uint32_t bytes) {
      for (uint32_t i = tid * 16; i < bytes; i += S::kThreads * 16) *(uint4*)((uint8_t*)to + i) = *(const uint4*)(what + i);
    };
    bring(held, from + Q::frags(4 * b0), (uint32_t)Q::frags(units));
    bring(back, from + Q::frags(p.units), NC * 16);
  }
  asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");  // the queries, to the instructions
  __syncthreads();
  bool plain = true;  // every column has one factor
  for (uint32_t q = 0; q < kQueries; ++q) plain &= back[3 * NC + q] == 0.f;
  const uint64_t b_desc = raven_tc::sw128_desc(smem_u32(held));
  constexpr uint32_t idesc = (1u << 4) | ((uint32_t)(NC >> 3) << 17) | (8u << 24);  // f32 sums, f16 operands

  bool ok = true;
  Chain chain;
  // the words of the thread's row, one block ahead
  uint32_t next[W];
  auto fetch = [&](uint32_t tile, uint32_t b) {
    const uint32_t* from = p.words + min((uint64_t)tile * kWideRows + row_of, p.n - 1) * p.ld_words + (b0 + b) * W;
    if constexpr (W == 4) {
      const uint4 v = *(const uint4*)from;
      next[0] = v.x, next[1] = v.y, next[2] = v.z, next[3] = v.w;
    } else if constexpr (W == 2) {
      const uint2 v = *(const uint2*)from;
      next[0] = v.x, next[1] = v.y;
    } else {
      next[0] = *from;
    }
  };
  if (first < p.tiles) fetch(first, 0);
  for (uint32_t tile = first; tile < p.tiles; tile += step) {
    float total[NC] = {};
    for (uint32_t b = 0; b < blocks; ++b) {
      const uint32_t u = min(4u, units - 4 * b);
      uint32_t word[W];
#pragma unroll
      for (uint32_t g = 0; g < W; ++g) word[g] = next[g];
      if (b + 1 < blocks)
        fetch(tile, b + 1);
      else if (tile + step < p.tiles)
        fetch(tile + step, 0);
      if (ok && !warp_waits(bars + 8 * stages.now, stages.parity())) ok = false;
      if (ok) {
        // 64 bytes of the row, 16 at a time in the 64-byte swizzle
        const uint8_t* stage = ring + stages.now * kWideStage + row_of * 64;
        uint32_t c[16];
#pragma unroll
        for (int i = 0; i < 4; ++i) *(uint4*)&c[4 * i] = *(const uint4*)(stage + ((i ^ ((row_of >> 1) & 3)) * 16));
        // word u * quarter + unit of a block of u units
        auto put_unit = [&](uint32_t unit, uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3) {
          const uint32_t w[4] = {c0, c1, c2, c3};
          const Offsets z(word[unit / U]);
          uint32_t a[16];
#pragma unroll
          for (int i = 0; i < 4; ++i) operands(w[i], z, a[4 * i], a[4 * i + 1], a[4 * i + 2], a[4 * i + 3]);
          tmem_st16(mine + 16 * unit, a);
        };
        if (u == 4) {
          put_unit(0, c[0], c[4], c[8], c[12]);
          put_unit(1, c[1], c[5], c[9], c[13]);
          put_unit(2, c[2], c[6], c[10], c[14]);
          put_unit(3, c[3], c[7], c[11], c[15]);
        } else if (u == 3) {
          put_unit(0, c[0], c[3], c[6], c[9]);
          put_unit(1, c[1], c[4], c[7], c[10]);
          put_unit(2, c[2], c[5], c[8], c[11]);
        } else if (u == 2) {
          put_unit(0, c[0], c[2], c[4], c[6]);
          put_unit(1, c[1], c[3], c[5], c[7]);
        } else {
          put_unit(0, c[0], c[1], c[2], c[3]);
        }
        asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
        stages.taken(p.depth);
      }
#pragma unroll
      for (uint32_t g = 0; g < W; ++g) {
        if (g * U >= u) break;
        raven_tc::tc_fence_before();
        meet(1 + team, 128);  // operands are written, the sums before them read
        if (row_of == 0 && ok) {
          if (g == 0) copy_next();  // into the stage that every thread has read
          raven_tc::tc_fence_after();
          uint32_t add = 0;
#pragma unroll
          for (uint32_t uu = 0; uu < U; ++uu) {
            const uint32_t unit = g * U + uu;
            if (unit >= u) break;
            const uint64_t at = b_desc + ((4 * b + unit) / 2 * Q::kBlockBytes >> 4) + (unit & 1) * 4;
            mma_ts(tmem + S::kAcc, tmem + 16 * unit, at, idesc, add);
            mma_ts(tmem + S::kAcc, tmem + 16 * unit + 8, at + 2, idesc, 1);
            add = 1;
          }
          raven_tc::mma_commit(done);
        }
        if (ok && !warp_waits(done, chain.phase)) ok = false;
        if (ok) chain.over();
        raven_tc::tc_fence_after();
        const float sc = raven_int4::step_of(word[g]) * (1.f / (1 << kStepShift));
        constexpr int P = 2;  // pieces of 16 columns at once
#pragma unroll
        for (int j = 0; j < NC / (16 * P); ++j) {
          uint32_t v[P][16];
#pragma unroll
          for (int k = 0; k < P; ++k) tmem_ld16(mine + S::kAcc + 16 * (P * j + k), v[k]);
          tmem_wait_ld(v);
#pragma unroll
          for (int i = 0; i < 16 * P; ++i)
            total[16 * P * j + i] = fmaf(sc, __uint_as_float(v[i / 16][i % 16]), total[16 * P * j + i]);
        }
      }
    }
    const uint64_t row = (uint64_t)tile * kWideRows + row_of;
    if (row < p.n) {
      const float bias = p.bias ? p.bias[row] : 0.f;
      O* to = (O*)p.out + slice * p.ld_slice + chunk * kQueries * p.ld + row;
      const uint32_t here = (uint32_t)min((uint64_t)kQueries, p.nq - chunk * kQueries);
      if (plain && here == kQueries) {  // four at a time, without a branch between them
#pragma unroll
        for (uint32_t q = 0; q < kQueries; q += 4) {
          const float4 f = *(const float4*)(back + q);
          const float by[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
          for (uint32_t k = 0; k < 4; ++k) {
            const float y = F32 ? total[2 * (q + k)] + total[2 * (q + k) + 1] : total[q + k];
            *to = rounded<O>(fmaf(by[k], y, bias));
            to += p.ld;
          }
        }
      } else {
#pragma unroll
        for (uint32_t q = 0; q < kQueries; ++q) {
          if (q < here) {
            const float y = F32 ? total[2 * q] + total[2 * q + 1] : total[q];
            *to = rounded<O>(plain ? fmaf(back[q], y, bias)
                                   : fmaf(y * back[q] * back[NC + 2 * q], back[NC + 2 * q + 1], bias));
            to += p.ld;
          }
        }
      }
    }
  }
  if (!ok && lane == 0) raven_score::tell(p.status, raven_score::kStatusWait);
  // a wait ran out: neither a copy nor an instruction of this team is under way any more
  if (!ok && row_of == 0) {
    stages.rest(p.depth, [&](uint32_t stage, uint32_t parity) { wait(bars + 8 * stage, parity); });
    chain.rest([&](uint32_t parity) { wait(done, parity); });
  }
  raven_tc::tc_fence_before();
  __syncthreads();
  raven_tc::tc_fence_after();
  if (warp == 0)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(*slot_of_tmem), "r"(512) : "memory");
}

}  // namespace raven_score4
