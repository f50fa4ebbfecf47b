// Scoring operators of the C ABI (include/raven_gpu.h): FP8 rows with a scale
// for each block of 128 values, scores of queries against rows (dense and
// grouped, score_tc.cuh) and the best k of each row of scores (topk.cuh).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "../../include/raven_gpu.h"
#include "fp8.cuh"
#include "internal.h"
#include "launch.h"
#include "score_tc.cuh"
#include "topk.cuh"

using raven_internal::encode_tiled;

using raven_score::after_previous;

using namespace raven_launch;

namespace {

// ---------------------------------------------------------------------------
// FP8 rows. Block b of a row: e = the least exponent with max|x| <= 448 * 2^e
// over its finite values (0 when they are all zero, at least -127), code =
// e4m3(x * 2^-e) to nearest even, exponent byte = e + 127. A power of two
// scales exactly, so the only rounding is e4m3's own (half a step, 2^-4 of the
// value; 2^-10 * 2^e below the type's normal range).
// A block is read by 32 lanes (f32) or 16 (16-bit), 16 bytes each, and a warp has
// two such reads under way (30000 x 768 f16 17 us, 4.0 TB/s, 1000000 x 128 f32 139 us,
// 4.6; four, with half the warps, were
// slower, and 8 bytes a lane, one read at a time, took half as long again).
// ---------------------------------------------------------------------------
using raven_fp8::load_value;

// A CTA takes a run of rows and gathers their exponents in shared memory: single
// bytes of a 32-byte sector written at different times cost a read each.
// VEC: pitch and address let 16 bytes be read at once. LANE: lane-major rows
// (element e of the first 16C at (e % 16) * C + e / 16).
constexpr uint32_t kExpBytes = 4096;  // of a run: rows x blocks padded to 4

template <typename T, bool VEC, bool LANE>
__global__ void __launch_bounds__(256, 8) fp8_encode_kernel(const T* in, uint64_t n, uint32_t dim, uint64_t ld,
                                                         uint8_t* codes, uint64_t ld_codes, uint8_t* exps,
                                                         uint64_t ld_exps, uint32_t run) {
  constexpr int E = 16 / sizeof(T), G = (int)kBlock / E, U = 2;  // values per lane, lanes per block, blocks under way
  __shared__ __align__(16) uint8_t se[kExpBytes];
  after_previous();
  const uint32_t sub = threadIdx.x % G, group = threadIdx.x / G;
  const uint32_t nb = (dim + kBlock - 1) / kBlock, nb4 = (nb + 3) / 4 * 4, dim16 = (dim + 15) / 16 * 16;
  for (uint64_t r0 = (uint64_t)blockIdx.x * run; r0 < n; r0 += (uint64_t)gridDim.x * run) {
    const uint32_t rows = (uint32_t)min((uint64_t)run, n - r0), units = rows * nb;
    if (nb4 != nb)
      for (uint32_t i = threadIdx.x; i < rows * nb4 / 4; i += 256) ((uint32_t*)se)[i] = 0x7f7f7f7fu;
    __syncthreads();
    for (uint32_t u0 = 0; u0 < units; u0 += U * (256 / G)) {
      uint32_t row[U], blk[U];
      uint4 raw[U];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const uint32_t u = u0 + k * (256 / G) + group;
        row[k] = u / nb;
        blk[k] = u - row[k] * nb;
        const uint32_t d = blk[k] * kBlock + E * sub;
        raw[k] = make_uint4(0, 0, 0, 0);
        if (u < units) {
          const T* r = in + (r0 + row[k]) * ld;
          if (VEC && d + E <= dim) {
            raw[k] = *(const uint4*)(r + d);
          } else {
            const uint32_t C = dim / 16;
            T* x = (T*)&raw[k];
#pragma unroll
            for (int i = 0; i < E; ++i) {
              const uint32_t e = d + i;
              if (e < dim) x[i] = r[LANE && e < 16 * C ? (e % 16) * C + e / 16 : e];
            }
          }
        }
      }
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const uint32_t u = u0 + k * (256 / G) + group;
        float x[E];
        uint32_t top = 0;  // largest magnitude, as bits
#pragma unroll
        for (int i = 0; i < E; ++i) {
          x[i] = load_value((const T*)&raw[k] + i);
          top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
        }
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        const bool odd = __any_sync(0xffffffffu, top >= 0x7f800000u);  // infinities or NaN: the largest finite one, then
        if (odd) {
          top = 0;
#pragma unroll
          for (int i = 0; i < E; ++i) {
            const uint32_t a = __float_as_uint(x[i]) & 0x7fffffffu;
            if (a < 0x7f800000u) top = max(top, a);
          }
#pragma unroll
          for (int o = G / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        }
        const int e = raven_fp8::exponent_of(top);
        const float inv = raven_fp8::inverse_of(e);
        uint32_t word[E / 4];
#pragma unroll
        for (int i = 0; i < E; i += 4) {
          word[i / 4] = raven_fp8::codes_of(x + i, inv);
          if (odd) word[i / 4] = raven_fp8::with_nan(word[i / 4], x + i);
        }
        if (u < units) {
          const uint32_t d = blk[k] * kBlock + E * sub;
          if (d < dim16) {
            uint8_t* c = codes + (r0 + row[k]) * ld_codes + d;
            if constexpr (E == 4)
              *(uint32_t*)c = word[0];
            else
              *(uint2*)c = make_uint2(word[0], word[1]);
          }
          if (sub == 0) se[row[k] * nb4 + blk[k]] = (uint8_t)(e + 127);
        }
      }
    }
    __syncthreads();
    const uint32_t per = nb4 / 4;
    for (uint32_t i = threadIdx.x; i < rows * per; i += 256) {
      const uint32_t r = i / per;
      *(uint32_t*)(exps + (r0 + r) * ld_exps + 4 * (i - r * per)) = ((const uint32_t*)se)[i];
    }
    __syncthreads();
  }
}

__global__ void __launch_bounds__(256) fp8_decode_kernel(const uint8_t* codes, uint64_t ld_codes, const uint8_t* exps,
                                                         uint64_t ld_exps, uint64_t n, uint32_t dim, float* out,
                                                         uint64_t ld) {
  after_previous();
  const uint64_t total = n * dim;
  for (uint64_t t = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; t < total; t += (uint64_t)gridDim.x * blockDim.x) {
    const uint64_t row = t / dim;
    const uint32_t d = (uint32_t)(t - row * dim);
    const __half_raw h = __nv_cvt_fp8_to_halfraw(codes[row * ld_codes + d], __NV_E4M3);
    // the scale as f32 bits: 0 is 2^-127, below the normal range, and 255 the scales'
    // NaN, as the tensor cores take it; the product with a power of two is rounded as
    // ldexpf would (infinite from 2^128)
    const uint32_t e = exps[row * ld_exps + d / kBlock];
    const float scale = __uint_as_float(e == 0 ? 0x400000u : e == 255 ? 0x7fc00000u : e << 23);
    out[row * ld + d] = __half2float(*(const __half*)&h) * scale;
  }
}

template <typename T, bool LANE>
cudaError_t launch_encode(const void* x, uint64_t n, uint32_t dim, uint64_t ld, uint8_t* codes, uint64_t ld_codes,
                          uint8_t* exps, uint64_t ld_exps, int sms, cudaStream_t st) {
  // rows of a run: a multiple of 8 (their exponents fill whole sectors), one read
  // of the CTA's threads and more, up to four while SMs keep several runs
  const uint32_t nb = (dim + kBlock - 1) / kBlock, nb4 = (nb + 3) / 4 * 4;
  const uint32_t once = 256 * 16 / (kBlock * (uint32_t)sizeof(T));  // blocks the threads read at once
  uint32_t run = std::max(1u, once / nb);
  if (run > 8 || n >= 8ull * sms) run = (run + 7) / 8 * 8;
  while (run * nb < 4 * once && n / run > 8ull * sms) run *= 2;
  run = std::min(run, kExpBytes / nb4);
  const uint64_t grid = std::min<uint64_t>((n + run - 1) / run, (uint64_t)sms * 64);
  const bool vec = !LANE && ld * sizeof(T) % 16 == 0 && aligned(x, 16);
  static Allowed none;
  return launch(vec ? fp8_encode_kernel<T, true, LANE> : fp8_encode_kernel<T, false, LANE>, grid, 256, 0, none, st,
                (const T*)x, n, dim, ld, codes, ld_codes, exps, ld_exps, run);
}

int encode_rows(const void* x, int32_t type, uint64_t n, uint32_t dim, uint64_t ld, uint8_t* codes, uint64_t ld_codes,
                uint8_t* exps, uint64_t ld_exps, cudaStream_t st) {
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  if (type == RAVEN_TYPE_F32)
    CU((launch_encode<float, false>(x, n, dim, ld, codes, ld_codes, exps, ld_exps, sms, st)));
  else if (type == RAVEN_TYPE_F16)
    CU((launch_encode<__half, false>(x, n, dim, ld, codes, ld_codes, exps, ld_exps, sms, st)));
  else
    CU((launch_encode<__nv_bfloat16, false>(x, n, dim, ld, codes, ld_codes, exps, ld_exps, sms, st)));
  return RAVEN_OK;
}

uint64_t exps_pitch(uint32_t dim) { return ((dim + kBlock - 1) / kBlock + 3) / 4 * 4; }
uint64_t codes_pitch(uint32_t dim) { return (dim + 15) / 16 * 16; }

int check_fp8(const uint8_t* codes, uint64_t ld_codes, const uint8_t* exps, uint64_t ld_exps, uint32_t dim) {
  if (!codes || !exps) return fail(RAVEN_EINVAL, "FP8 rows need codes and exponents");
  if (!aligned(codes, 16) || ld_codes % 16 || ld_codes < codes_pitch(dim))
    return fail(RAVEN_EINVAL, "FP8 codes must start on 16 bytes, their pitch a multiple of 16 of at least dim");
  if (!aligned(exps, 4) || ld_exps % 4 || ld_exps < exps_pitch(dim))
    return fail(RAVEN_EINVAL, "FP8 exponents must start on 4 bytes, their pitch a multiple of 4 of at least dim / 128");
  return RAVEN_OK;
}

// ---------------------------------------------------------------------------
// Scores.
// ---------------------------------------------------------------------------
// K-major rows as boxes of 128 bytes x `box` rows with the 128-byte swizzle;
// elements past dim, and rows past the last, read 0.
bool rows_map(CUtensorMap* m, const void* base, int32_t type, uint32_t dim, uint64_t rows, uint64_t ld, uint32_t box) {
  PFN_cuTensorMapEncodeTiled_v12000 f = encode_tiled();
  if (!f) return false;
  const uint64_t size = type_size(type);
  cuuint64_t gdim[2] = {dim, rows};
  cuuint64_t gstride[1] = {ld * size};
  cuuint32_t b[2] = {(cuuint32_t)(128 / size), box};
  cuuint32_t es[2] = {1, 1};
  return f(m, size == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, (void*)base, gdim, gstride,
           b, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// ---------------------------------------------------------------------------
// Many groups: sums over the groups before each chunk of 32, so that neither a
// tile's group nor a query's place is found by walking them all.
// ---------------------------------------------------------------------------
using raven_score::Chunk;
using raven_score::kChunk;
// From how many groups on: the sums' two launches take 4 us and more, and a walk
// is partly hidden by the tiles (1000 groups of 1 x 8 scores 22 us walked, 18 with
// sums, but 1000 of 10 x 1000 44 and 49; 2000 of 20 x 300 59 and 45). The blocks of
// group_rows, which sum what is before them by themselves, reach that later (16384
// groups 10.8 us a call, 14.6 with sums; 32768: 21.3, 14; 65536: 39.9, 14).
constexpr uint32_t kManyGroups = 1536, kManyGroupRows = 16384;

// Per chunk, the tiles (of tq queries and `rows` rows of v) and scores of its groups.
__global__ void __launch_bounds__(256) group_chunks_kernel(const int64_t* qo, const int64_t* vo, uint32_t groups,
                                                           uint64_t nq, uint64_t n, uint32_t tq, uint32_t rows,
                                                           Chunk* chunks, int* status) {
  after_previous();
  const uint32_t g = blockIdx.x * 256u + threadIdx.x, lane = threadIdx.x & 31;
  int64_t a, b, m = 0, nn = 0;
  const bool bad = g < groups && !raven_score::group_of(qo, vo, g, nq, n, a, b, m, nn);
  int64_t tiles = (m + tq - 1) / tq * ((nn + rows - 1) / rows), out = m * nn;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    tiles += __shfl_xor_sync(0xffffffffu, tiles, o);
    out += __shfl_xor_sync(0xffffffffu, out, o);
  }
  if (lane == 0 && g < groups) chunks[g / kChunk] = Chunk{tiles, out};
  if (__any_sync(0xffffffffu, bad) && lane == 0) raven_score::tell(status, raven_score::kStatusOffsets);
}

// Chunks' sums to sums over the chunks before; chunks[count]: over all. One CTA.
__global__ void __launch_bounds__(1024) group_scan_kernel(Chunk* chunks, uint32_t count) {
  constexpr uint32_t N = 4;  // chunks of a thread at once
  __shared__ Chunk part[32];
  after_previous();
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  Chunk before{0, 0};
  for (uint32_t base = 0; base < count; base += 1024 * N) {
    Chunk x[N], sum{0, 0};
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) {
      const uint32_t c = base + tid * N + i;
      x[i] = c < count ? chunks[c] : Chunk{0, 0};
      sum.tiles += x[i].tiles;
      sum.out += x[i].out;
    }
    Chunk up = sum;
    auto scan = [&](Chunk& s) {
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t t = __shfl_up_sync(0xffffffffu, s.tiles, o), u = __shfl_up_sync(0xffffffffu, s.out, o);
        if ((int)lane >= o) {
          s.tiles += t;
          s.out += u;
        }
      }
    };
    scan(up);
    if (lane == 31) part[warp] = up;
    __syncthreads();
    if (warp == 0) {
      Chunk s = part[lane];
      scan(s);
      part[lane] = s;
    }
    __syncthreads();
    Chunk at{before.tiles + up.tiles - sum.tiles, before.out + up.out - sum.out};
    if (warp) {
      at.tiles += part[warp - 1].tiles;
      at.out += part[warp - 1].out;
    }
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) {
      const uint32_t c = base + tid * N + i;
      if (c < count) chunks[c] = at;
      at.tiles += x[i].tiles;
      at.out += x[i].out;
    }
    before.tiles += part[31].tiles;
    before.out += part[31].out;
    __syncthreads();
  }
  if (tid == 0) chunks[count] = before;
}

uint32_t chunks_of(uint32_t groups) { return (groups + kChunk - 1) / kChunk; }

cudaError_t launch_chunks(const int64_t* qo, const int64_t* vo, uint32_t groups, uint64_t nq, uint64_t n, uint32_t tq,
                          uint32_t rows, Chunk* chunks, int* status, cudaStream_t st) {
  static Allowed none, none_scan;
  const cudaError_t e = launch(group_chunks_kernel, (groups + 255) / 256, 256, 0, none, st, qo, vo, groups, nq, n, tq,
                               rows, chunks, status);
  return e != cudaSuccess ? e : launch(group_scan_kernel, 1, 1024, 0, none_scan, st, chunks, chunks_of(groups));
}

constexpr uint32_t kHalo = 16;  // scores that a tile by pairs computes past its own: a sector of 16-bit ones

struct Operands {
  const raven_rows* q;
  const raven_rows* v;
  uint32_t dim;
};

template <bool FP8, int BN, bool ROWS, bool HELD = false>
cudaError_t launch_score(const Operands& o, raven_score::Params p, bool whole, int sms, cudaStream_t st) {
  using L = raven_score::Layout<FP8, BN, ROWS, HELD>;
  CUtensorMap mq{}, mv;
  if ((!HELD &&
       !rows_map(&mq, o.q->data, o.q->type, o.dim, o.q->rows, o.q->ld, ROWS ? raven_score::kQBox : raven_score::kBM)) ||
      !rows_map(&mv, o.v->data, o.v->type, o.dim, o.v->rows, o.v->ld, ROWS ? raven_score::kBM : BN))
    return cudaErrorInvalidValue;
  // Rows per tile, where M is the rows. A tile of few queries has little to do
  // when K is short, and what it costs to find it, to hand it over and to start
  // its epilogue shows: it takes several accumulators at once, as long as every
  // SM keeps a few tiles (grouped: and a tile does not outgrow a mean group).
  const uint64_t per = p.qo ? std::max<uint64_t>(p.n / p.groups, 1) : p.n;
  uint64_t subs = p.nkb <= 4 ? L::kSubs : 1;
  p.halo = ROWS || whole ? 0 : kHalo;
  auto tiles = [&](uint64_t s) {
    const uint64_t rows = s * L::kTileV - p.halo;
    return (p.qo ? p.groups : 1) * ((per + rows - 1) / rows) *
           (p.qo ? 1 : (p.nq + L::kTileQ - 1) / L::kTileQ);
  };
  while (subs > 1 && (tiles(subs) < 4ull * sms || (p.qo && subs * L::kTileV > 2 * per))) subs /= 2;
  p.subs = (uint32_t)subs;
  const uint64_t grid = p.qo ? (uint64_t)sms : std::min<uint64_t>(tiles(subs), (uint64_t)sms);
  Chunk* chunks = nullptr;
  cudaError_t e = cudaSuccess;
  if (p.groups > kManyGroups) {
    p.nchunks = chunks_of(p.groups);
    if ((e = cudaMallocAsync((void**)&chunks, (p.nchunks + 1ull) * sizeof(Chunk), st)) != cudaSuccess) return e;
    p.chunks = chunks;
    e = launch_chunks(p.qo, p.vo, p.groups, p.nq, p.n, L::kTileQ, L::kTileV * p.subs - p.halo, chunks, p.status, st);
  }
  static Allowed allowed;
  if (e == cudaSuccess)
    e = launch(raven_score::score_kernel<FP8, BN, ROWS, HELD>, grid, L::kThreads, L::kBytes, allowed, st, mq, mv, p);
  if (chunks) cudaFreeAsync(chunks, st);
  return e;
}

// `want`: queries of a group, twice the mean where groups differ. Up to 64: the
// layout by rows of v. More: by pairs, whose sectors are whole wherever a query's
// scores start (785 x 132491 f32 99 us, by rows 167; 999 x 250007 bf16 152, 271),
// except
//   f32 scores that all start on sectors: by rows, a warp writes whole lines;
//   queries 1.5 MB apart and more: a lane of the layout by pairs comes back to
//   its query's page for every sector, and the pages of 128 queries are too many
//   (100 x 1000003 f32 323 us, by rows 131).
// The N side is as wide as the queries need and no wider than leaves SMs a tile.
constexpr uint64_t kFar = 3 << 19;

template <bool FP8>
cudaError_t dispatch_score(const Operands& o, const raven_score::Params& p, int sms, cudaStream_t st) {
  const uint64_t want = p.qo ? 2 * ((p.nq + p.groups - 1) / p.groups) : p.nq;
  const uint64_t size = p.out_type == raven_score::kOutF32 ? 4 : 2;
  const bool whole = !p.qo && (uintptr_t)p.out % 32 == 0 && p.ld * size % 32 == 0;  // every query starts on a sector
  const bool far = !p.qo && p.ld * size >= kFar;
  if (want > 64 && !(whole && size == 4) && !far) {
    const uint64_t rows = 224 - (whole ? 0 : kHalo);
    if (!p.qo && (p.nq + 127) / 128 * ((p.n + rows - 1) / rows) < (uint64_t)sms)
      return launch_score<FP8, 96, false>(o, p, whole, sms, st);
    return launch_score<FP8, 224, false>(o, p, whole, sms, st);
  }
  if constexpr (FP8)
    if (p.qx) return launch_score<FP8, 32, true, true>(o, p, whole, sms, st);
  const uint64_t vt = (p.n + raven_score::kBM - 1) / raven_score::kBM;
  auto fills = [&](uint64_t bn) { return p.qo || vt * ((p.nq + bn - 1) / bn) >= (uint64_t)sms; };
  if (want > 64 && fills(192)) return launch_score<FP8, 192, true>(o, p, whole, sms, st);
  if (want > 32 && fills(64)) return launch_score<FP8, 64, true>(o, p, whole, sms, st);
  return launch_score<FP8, 32, true>(o, p, whole, sms, st);
}

int check_rows(const raven_rows* r, uint32_t dim, const char* what) {
  const std::string w(what);
  if (!r) return fail(RAVEN_EINVAL, w + ": null");
  const uint64_t size = type_size(r->type);
  if (!size) return fail(RAVEN_EINVAL, w + ": unknown type");
  if (r->rows > kMaxRows) return fail(RAVEN_ELIMIT, w + ": more than 2^31 - 1 rows");
  if (r->rows == 0) return RAVEN_OK;
  if (!r->data) return fail(RAVEN_EINVAL, w + ": null data");
  if (r->ld < dim) return fail(RAVEN_EINVAL, w + ": pitch below dim");
  if (!aligned(r->data, size)) return fail(RAVEN_EINVAL, w + ": data is not aligned to its type");
  if (r->type == RAVEN_TYPE_FP8)
    return check_fp8((const uint8_t*)r->data, r->ld, r->exps, r->ld_exps, dim);
  return RAVEN_OK;
}

// Dense (qo null) and grouped scores.
int run_scores(const raven_rows* q, const int64_t* qo, const raven_rows* v, const int64_t* vo, uint32_t groups,
               uint32_t dim, float alpha, const float* bias, void* out, int32_t out_type, uint64_t ld, uint64_t capacity,
               int32_t* status, void* stream) {
  if (int rc = check_dim(dim)) return rc;
  if (int rc = check_rows(q, dim, "queries")) return rc;
  if (int rc = check_rows(v, dim, "vectors")) return rc;
  if (v->type == RAVEN_TYPE_F32) return fail(RAVEN_EINVAL, "vectors: type must be f16, bf16 or FP8");
  const bool fp8 = v->type == RAVEN_TYPE_FP8;
  if (!fp8 && q->type != v->type) return fail(RAVEN_EINVAL, "queries must have the vectors' type");
  if (out_type != RAVEN_TYPE_F32 && out_type != RAVEN_TYPE_F16 && out_type != RAVEN_TYPE_BF16)
    return fail(RAVEN_EINVAL, "scores: type must be f32, f16 or bf16");
  if (!aligned(bias, 4) || !aligned(status, 4)) return fail(RAVEN_EINVAL, "scores: bias and status must start on 4 bytes");
  if (q->rows == 0 || v->rows == 0 || groups == 0) return RAVEN_OK;
  if (!out && !(qo && capacity == 0)) return fail(RAVEN_EINVAL, "scores: null output");
  if (!aligned(out, type_size(out_type))) return fail(RAVEN_EINVAL, "scores: output is not aligned to its type");
  if (!qo && ld < v->rows) return fail(RAVEN_EINVAL, "scores: output pitch below the number of vectors");
  const bool encode = fp8 && q->type != RAVEN_TYPE_FP8;
  if (!fp8)
    for (const raven_rows* r : {q, v})
      if (!aligned(r->data, 16) || r->ld % 8)
        return fail(RAVEN_EINVAL, "16-bit rows must start on 16 bytes, their pitch a multiple of 8 values");
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  cudaStream_t st = (cudaStream_t)stream;  // NULL: the CUDA default stream

  raven_score::Params p{};
  p.nq = q->rows;
  p.n = v->rows;
  const uint64_t bytes = (uint64_t)dim * type_size(v->type);
  p.nkb = (uint32_t)((bytes + 127) / 128);
  p.last_k = (uint32_t)((bytes - (p.nkb - 1) * 128ull + 31) / 32);
  p.groups = groups;
  p.qo = qo;
  p.vo = vo;
  p.alpha = alpha;
  p.bias = bias;
  p.out = out;
  p.out_type = out_type == RAVEN_TYPE_F32 ? raven_score::kOutF32
               : out_type == RAVEN_TYPE_F16 ? raven_score::kOutF16 : raven_score::kOutBf16;
  p.ld = ld;
  p.capacity = std::min<uint64_t>(capacity, 1ull << 62);  // signed on the device; no output is larger
  p.status = status;
  // instruction descriptor, M = 128. FP8: types e4m3 (0), exponent scales (bit 23);
  // 16-bit: f32 accumulator (bit 4), types f16 (0) or bf16 (1)
  const uint32_t ty = v->type == RAVEN_TYPE_BF16 ? 1u : 0u;
  p.idesc = fp8 ? (1u << 23) | (1u << 27) : (1u << 4) | (ty << 7) | (ty << 10) | (8u << 24);

  raven_rows qq = *q;
  uint8_t* tmp = nullptr;
  if (encode && !qo && q->rows <= 32 && p.nkb <= raven_score::kHeldBlocks && q->rows * p.nkb <= raven_score::kHeldUnits) {
    p.qx = q->data;  // every CTA encodes them for itself
    p.q_type = q->type == RAVEN_TYPE_F32 ? raven_score::kOutF32
               : q->type == RAVEN_TYPE_F16 ? raven_score::kOutF16 : raven_score::kOutBf16;
    p.dim = dim;
    p.ld_qx = q->ld;
  } else if (encode) {  // the queries' codes live until the product is done, in stream order
    qq.type = RAVEN_TYPE_FP8;
    qq.ld = codes_pitch(dim);
    qq.ld_exps = exps_pitch(dim);
    const uint64_t cb = (qq.rows * qq.ld + 255) / 256 * 256;
    CU(cudaMallocAsync((void**)&tmp, cb + qq.rows * qq.ld_exps, st));
    qq.data = tmp;
    qq.exps = tmp + cb;
    const int rc = encode_rows(q->data, q->type, q->rows, dim, q->ld, tmp, qq.ld, tmp + cb, qq.ld_exps, st);
    if (rc) {
      cudaFreeAsync(tmp, st);
      return rc;
    }
  }
  p.qe = qq.exps;
  p.ve = v->exps;
  p.ld_qe = qq.ld_exps;
  p.ld_ve = v->ld_exps;

  const Operands o{&qq, v, dim};
  const cudaError_t e = fp8 ? dispatch_score<true>(o, p, sms, st) : dispatch_score<false>(o, p, sms, st);
  if (tmp) cudaFreeAsync(tmp, st);
  if (e != cudaSuccess) return fail(RAVEN_ECUDA, std::string("scores: ") + cudaGetErrorString(e));
  return RAVEN_OK;
}

// A query's group is where a bisection of the offsets for it ends: by the first
// offset (queries before it have no group), then bit by bit from the highest one
// of the group's number, right of offset s where qo[s] <= i. So every query has
// one place, a group with qo[g] <= i < qo[g + 1] or, as number `groups`, what is
// behind the last, where offsets fall too (several groups cover a query there),
// and places rise with their queries. Which offsets lead to place x does not
// depend on the query; they bound its queries [lo, hi). By one warp, a bit of x
// from `low` on per lane (one lane after the other took 2 to 3 us of a call more).
__device__ inline void queries_of(const int64_t* qo, uint32_t groups, int64_t nq, uint32_t x, uint32_t low, int64_t& lo,
                                  int64_t& hi) {
  const uint32_t bit = threadIdx.x & 31, s = (x >> bit | 1u) << bit;
  lo = max((int64_t)0, qo[0]);
  hi = nq;
  if (bit >= low && s <= groups) {
    if (x >> bit & 1u)
      lo = max(lo, qo[s]);
    else
      hi = min(hi, qo[s]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    lo = max(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = min(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  lo = min(lo, nq);
  hi = max(hi, lo);
}

// Where each query's scores start in grouped scores: starts[i] for query i of
// group g is sum over earlier groups of m h_n plus its place times n_g; a group
// that counts as empty gives its queries the sum alone. Blocks take runs of 256
// groups; each sums the groups before its run by itself, unless the sums are
// given (many groups).
__global__ void __launch_bounds__(256) group_rows_kernel(const int64_t* qo, const int64_t* vo, uint32_t groups,
                                                         uint64_t nq, uint64_t n, const Chunk* chunks, int64_t* starts,
                                                         int* status) {
  after_previous();
  __shared__ int64_t part[256];
  __shared__ int64_t from[256], size[256], start[256], per[256];  // groups of many queries
  __shared__ uint32_t large, huge;
  __shared__ int64_t edge[256], ends[2][2];  // the run's offsets; its queries by the bits above it, those behind the last group
  const uint32_t g0 = blockIdx.x * 256u, tid = threadIdx.x;
  bool bad = false;
  auto read = [&](uint32_t g, int64_t& a, int64_t& m, int64_t& c) {
    int64_t v0;
    bad |= !raven_score::group_of(qo, vo, g, nq, n, a, v0, m, c);
  };
  const bool last = g0 + 256 >= groups;
  if (tid < 32 || (last && tid < 64)) {
    int64_t lo, hi;
    queries_of(qo, groups, (int64_t)nq, tid < 32 ? g0 : groups, tid < 32 ? 8 : 0, lo, hi);
    if ((tid & 31) == 0) {
      ends[tid >> 5][0] = lo;
      ends[tid >> 5][1] = hi;
    }
  }
  if (tid == 0) large = huge = 0;
  edge[tid] = g0 + tid <= groups ? qo[g0 + tid] : INT64_MAX;
  int64_t sum = 0, a, m, c;
  for (uint32_t g = tid; g < g0 && !chunks; g += 256) {
    read(g, a, m, c);
    sum += m * c;
  }
  part[tid] = sum;
  __syncthreads();
  for (int o = 128; o > 0; o >>= 1) {
    if ((int)tid < o) part[tid] += part[tid + o];
    __syncthreads();
  }
  const int64_t before = chunks ? chunks[g0 / kChunk].out : part[0];
  __syncthreads();
  int64_t lo = 0, hi = 0;
  a = m = c = 0;
  if (g0 + tid < groups) {
    read(g0 + tid, a, m, c);
    lo = ends[0][0];
    hi = ends[0][1];
#pragma unroll
    for (uint32_t bit = 0; bit < 8; ++bit) {
      const int64_t x = edge[(tid >> bit | 1u) << bit];
      if (tid >> bit & 1u)
        lo = max(lo, x);
      else
        hi = min(hi, x);
    }
    lo = min(lo, (int64_t)nq);
    hi = max(hi, lo);  // [lo, hi) within the queries whatever the offsets are: sums with them do not wrap
  }
  part[tid] = m * c;
  __syncthreads();
  for (int o = 1; o < 256; o <<= 1) {
    const int64_t x = (int)tid >= o ? part[tid - o] : 0;
    __syncthreads();
    part[tid] += x;
    __syncthreads();
  }
  // a group of up to 64 queries is written by 8 lanes, of up to 4096 by a warp, a larger one by all
  const uint32_t lane = tid & 31;
  const int64_t count = hi - lo, base = before + part[tid] - m * c + (lo - a) * c;  // of the first query that is its own
  auto write = [&](int64_t first, int64_t n, int64_t at, int64_t width, uint32_t i, uint32_t step) {
    int64_t* to = starts + first;
    at += i * width;
    width *= step;
#pragma unroll 4
    for (; i < n; i += step, at += width) to[i] = at;
  };
#pragma unroll 2
  for (int r = 0; r < 8; ++r) {
    const int64_t first = __shfl_sync(0xffffffffu, lo, r, 8), at = __shfl_sync(0xffffffffu, base, r, 8);
    const int64_t width = __shfl_sync(0xffffffffu, c, r, 8);
    write(first, __shfl_sync(0xffffffffu, count <= 64 ? (int)count : 0, r, 8), at, width, lane & 7, 8);
  }
  if (count > 64) {  // in any order: each is written by itself
    const uint32_t k = count <= 4096 ? atomicAdd(&large, 1u) : 255u - atomicAdd(&huge, 1u);
    from[k] = lo;
    size[k] = count;
    start[k] = base;
    per[k] = c;
  }
  __syncthreads();
  for (uint32_t k = tid / 32; k < large; k += 8) write(from[k], size[k], start[k], per[k], lane, 32);
  for (uint32_t k = 256 - huge; k < 256; ++k) write(from[k], size[k], start[k], per[k], tid, 256);
  // queries before the first group start at 0, those behind the last one at the end
  if (last) {
    const int64_t total = before + part[255];
    for (int64_t i = ends[1][0] + tid; i < ends[1][1]; i += 256) starts[i] = total;
    if (tid == 0) starts[nq] = total;
  }
  if (blockIdx.x == 0)
    for (int64_t i = tid; i < min(qo[0], (int64_t)nq); i += 256) starts[i] = 0;
  if (bad) raven_score::tell(status, raven_score::kStatusOffsets);
}

__global__ void status_kernel(int* status) {
  after_previous();
  atomicOr(status, atomicExch(&raven_score::g_status, 0));
}

// ---------------------------------------------------------------------------
// Top-k of rows.
// ---------------------------------------------------------------------------
template <typename T, int TEAM, bool BIG>
cudaError_t launch_topk(const raven_topk::Params& p, cudaStream_t st) {
  using TM = raven_topk::Team<TEAM, BIG>;
  const uint32_t smem = TM::kTeams * (uint32_t)sizeof(raven_topk::Shared<TEAM, BIG>);
  const uint64_t units = p.nq * p.parts;
  static Allowed allowed;
  return launch(raven_topk::topk_kernel<T, TEAM, BIG>, (units + TM::kTeams - 1) / TM::kTeams, TM::kThreads, smem, allowed,
                st, p);
}
template <int TEAM, bool BIG>
cudaError_t dispatch_topk(int32_t type, const raven_topk::Params& p, cudaStream_t st) {
  return type == RAVEN_TYPE_F32   ? launch_topk<float, TEAM, BIG>(p, st)
         : type == RAVEN_TYPE_F16 ? launch_topk<__half, TEAM, BIG>(p, st)
                                  : launch_topk<__nv_bfloat16, TEAM, BIG>(p, st);
}
template <bool BIG>
cudaError_t launch_join(const raven_topk::Params& p, cudaStream_t st) {
  static Allowed none;
  return launch(raven_topk::topk_join_kernel<BIG>, p.nq, raven_topk::kCtaThreads,
                (uint32_t)sizeof(raven_topk::Shared<raven_topk::kCtaThreads, BIG>), none, st, p);
}

}  // namespace

namespace raven_internal {

int fp8_encode_lane_major(const float* d_rows, uint64_t n, uint32_t dim, uint8_t* d_codes, uint64_t ld_codes,
                          uint8_t* d_exps, uint64_t ld_exps, cudaStream_t st) {
  if (int rc = check_fp8(d_codes, ld_codes, d_exps, ld_exps, dim)) return rc;
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  CU((launch_encode<float, true>(d_rows, n, dim, dim, d_codes, ld_codes, d_exps, ld_exps, sms, st)));
  return RAVEN_OK;
}

}  // namespace raven_internal

extern "C" {

int raven_fp8_encode_device(const void* d_rows, int32_t type, uint64_t n, uint32_t dim, uint64_t ld, uint8_t* d_codes,
                            uint64_t ld_codes, uint8_t* d_exps, uint64_t ld_exps, void* stream) {
  NvtxRange nvtx_range("raven.fp8_encode");
  if (int rc = check_dim(dim)) return rc;
  if (type != RAVEN_TYPE_F32 && type != RAVEN_TYPE_F16 && type != RAVEN_TYPE_BF16)
    return fail(RAVEN_EINVAL, "rows: type must be f32, f16 or bf16");
  if (n == 0) return RAVEN_OK;
  if (n > kMaxRows) return fail(RAVEN_ELIMIT, "rows: more than 2^31 - 1");
  if (!d_rows) return fail(RAVEN_EINVAL, "rows: null");
  if (ld < dim) return fail(RAVEN_EINVAL, "rows: pitch below dim");
  if (!aligned(d_rows, type_size(type))) return fail(RAVEN_EINVAL, "rows: not aligned to their type");
  if (int rc = check_fp8(d_codes, ld_codes, d_exps, ld_exps, dim)) return rc;
  return encode_rows(d_rows, type, n, dim, ld, d_codes, ld_codes, d_exps, ld_exps, (cudaStream_t)stream);
}

int raven_fp8_decode_device(const uint8_t* d_codes, uint64_t ld_codes, const uint8_t* d_exps, uint64_t ld_exps,
                            uint64_t n, uint32_t dim, float* d_out, uint64_t ld, void* stream) {
  NvtxRange nvtx_range("raven.fp8_decode");
  if (int rc = check_dim(dim)) return rc;
  if (n == 0) return RAVEN_OK;
  if (n > kMaxRows) return fail(RAVEN_ELIMIT, "rows: more than 2^31 - 1");
  if (int rc = check_fp8(d_codes, ld_codes, d_exps, ld_exps, dim)) return rc;
  if (!d_out || !aligned(d_out, 4)) return fail(RAVEN_EINVAL, "output: null or not aligned to f32");
  if (ld < dim) return fail(RAVEN_EINVAL, "output: pitch below dim");
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  const unsigned grid = (unsigned)std::min<uint64_t>((n * dim + 255) / 256, (uint64_t)sms * 16);
  static Allowed none;
  CU(launch(fp8_decode_kernel, grid, 256, 0, none, (cudaStream_t)stream, d_codes, ld_codes, d_exps, ld_exps, n, dim,
            d_out, ld));
  return RAVEN_OK;
}

int raven_scores_device(const raven_rows* q, const raven_rows* v, uint32_t dim, float alpha, const float* d_bias,
                        void* d_out, int32_t out_type, uint64_t ld_out, int32_t* d_status, void* stream) {
  NvtxRange nvtx_range("raven.scores");
  if (v && raven_internal::int4_group(v->type))
    return raven_internal::int4_scores(q, v, dim, alpha, d_bias, d_out, out_type, ld_out, d_status, stream);
  return run_scores(q, nullptr, v, nullptr, 1, dim, alpha, d_bias, d_out, out_type, ld_out, 0, d_status, stream);
}

int raven_group_scores_device(const raven_rows* q, const int64_t* d_q_offsets, const raven_rows* v,
                              const int64_t* d_v_offsets, uint32_t groups, uint32_t dim, float alpha,
                              const float* d_bias, void* d_out, int32_t out_type, uint64_t capacity, int32_t* d_status,
                              void* stream) {
  NvtxRange nvtx_range("raven.group_scores");
  if (v && raven_internal::int4_group(v->type)) return fail(RAVEN_EINVAL, "vectors: grouped scores take f16, bf16 or FP8 rows");
  if (groups && (!d_q_offsets || !d_v_offsets)) return fail(RAVEN_EINVAL, "offsets: null");
  if (groups && (!aligned(d_q_offsets, 8) || !aligned(d_v_offsets, 8)))
    return fail(RAVEN_EINVAL, "offsets: not aligned to 64 bits");
  if (groups > kMaxRows) return fail(RAVEN_ELIMIT, "more than 2^31 - 1 groups");
  if (capacity == 0 && !d_status) groups = 0;  // a call for nothing
  return run_scores(q, d_q_offsets, v, d_v_offsets, groups, dim, alpha, d_bias, d_out, out_type, 0, capacity, d_status,
                    stream);
}

int raven_group_rows_device(const int64_t* d_q_offsets, const int64_t* d_v_offsets, uint32_t groups, uint64_t nq,
                            uint64_t n, int64_t* d_row_starts, int32_t* d_status, void* stream) {
  NvtxRange nvtx_range("raven.group_rows");
  if (groups == 0) return fail(RAVEN_EINVAL, "groups must be >= 1");
  if (nq > kMaxRows || n > kMaxRows) return fail(RAVEN_ELIMIT, "more than 2^31 - 1 queries or vectors");
  if (!d_q_offsets || !d_v_offsets || !d_row_starts) return fail(RAVEN_EINVAL, "null argument");
  if (!aligned(d_q_offsets, 8) || !aligned(d_v_offsets, 8) || !aligned(d_row_starts, 8))
    return fail(RAVEN_EINVAL, "offsets and row starts: not aligned to 64 bits");
  if (!aligned(d_status, 4)) return fail(RAVEN_EINVAL, "status must start on 4 bytes");
  if (groups > kMaxRows) return fail(RAVEN_ELIMIT, "more than 2^31 - 1 groups");
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  Chunk* chunks = nullptr;
  cudaError_t e = cudaSuccess;
  if (groups > kManyGroupRows) {
    CU(cudaMallocAsync((void**)&chunks, (chunks_of(groups) + 1ull) * sizeof(Chunk), st));
    e = launch_chunks(d_q_offsets, d_v_offsets, groups, nq, n, 1, 1, chunks, d_status, st);
  }
  static Allowed none;
  if (e == cudaSuccess)
    e = launch(group_rows_kernel, (groups + 255) / 256, 256, 0, none, st, d_q_offsets, d_v_offsets, groups, nq, n, chunks,
               d_row_starts, d_status);
  if (chunks) cudaFreeAsync(chunks, st);
  CU(e);
  return RAVEN_OK;
}

int raven_scoring_status_device(int32_t* d_status, void* stream) {
  NvtxRange nvtx_range("raven.scoring_status");
  if (!d_status) return fail(RAVEN_EINVAL, "null status");
  if (!aligned(d_status, 4)) return fail(RAVEN_EINVAL, "status must start on 4 bytes");
  static Allowed none;
  CU(launch(status_kernel, 1, 1, 0, none, (cudaStream_t)stream, d_status));
  return raven_internal::rows4_status(d_status, (cudaStream_t)stream);
}

int raven_topk_rows_device(const void* d_scores, int32_t type, uint64_t nq, uint64_t n, uint64_t ld,
                           const int64_t* d_row_starts, uint32_t k, int32_t largest, void* d_vals, uint32_t* d_ids,
                           uint32_t* d_counts, void* stream) {
  NvtxRange nvtx_range("raven.topk_rows");
  if (type != RAVEN_TYPE_F32 && type != RAVEN_TYPE_F16 && type != RAVEN_TYPE_BF16)
    return fail(RAVEN_EINVAL, "scores: type must be f32, f16 or bf16");
  if (k == 0 || k > raven_topk::kMaxK) return fail(RAVEN_ELIMIT, "k must be in 1..256");
  if (nq > kMaxRows) return fail(RAVEN_ELIMIT, "more than 2^31 - 1 rows");
  if (!d_row_starts && n > kMaxRows) return fail(RAVEN_ELIMIT, "rows of more than 2^31 - 1 scores");
  if (nq == 0) return RAVEN_OK;
  if (!d_vals || !d_ids) return fail(RAVEN_EINVAL, "null output");
  if (!d_scores && n) return fail(RAVEN_EINVAL, "scores: null");
  if (!d_row_starts && ld < n) return fail(RAVEN_EINVAL, "scores: pitch below the row length");
  const uint64_t size = type_size(type);
  if (!aligned(d_scores, size) || !aligned(d_vals, size) || !aligned(d_ids, 4) || !aligned(d_counts, 4) ||
      !aligned(d_row_starts, 8))
    return fail(RAVEN_EINVAL, "an argument is not aligned to its type");
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  raven_topk::Params p{};
  p.x = d_scores;
  p.nq = nq;
  p.n = n;
  p.ld = ld;
  p.starts = d_row_starts;
  p.total = n;
  p.k = k;
  p.mul = largest ? 1u : ~0u;
  p.add = largest ? 0x7fffffu : 0x7ffffeu;
  p.type = type == RAVEN_TYPE_F32 ? 0 : type == RAVEN_TYPE_F16 ? 1 : 2;
  p.vals = d_vals;
  p.ids = d_ids;
  p.counts = d_counts;
  // A warp takes a row when rows are short, or so many that warps fill the GPU
  // and k is small (no barriers, and every warp's loads overlap the others' work:
  // 10000 x 10007, k = 10, took 94 us by warps and 120 by CTAs, 4096 x 6667, k = 100,
  // 88 and 77, since a warp's 32 maxima bound k = 100 loosely; those taken are at 82 and 61 by now); else
  // a CTA does. Where rows are too few to fill the GPU, each is split into parts of
  // at least a tile. Ragged rows go by their mean.
  const uint64_t len = d_row_starts ? (n + nq - 1) / nq : n;
  const bool warp = len <= 1024 || (nq >= 16ull * sms && k <= 32);
  const uint64_t tile = raven_topk::kCtaThreads * 16ull;
  uint64_t parts = 1;
  if (!warp && nq < 4ull * sms) parts = std::max<uint64_t>(1, std::min<uint64_t>((4ull * sms + nq - 1) / nq, len / tile));
  p.parts = (uint32_t)parts;
  uint64_t* tmp = nullptr;
  if (parts > 1) {
    CU(cudaMallocAsync((void**)&tmp, nq * parts * k * 8, st));
    p.lists = tmp;
  }
  constexpr int kCta = raven_topk::kCtaThreads;
  const bool big = 2 * k > (uint32_t)kCta;
  // With k above a warp's threads, selecting and ordering k is a chain of one warp
  // while its CTA waits: with rows enough, CTAs of half the threads keep twice as
  // many such chains going (10000 x 10007 f32, k = 100, 220 to 179 us).
  const bool half = parts == 1 && k > 32 && nq >= 8ull * sms;
  cudaError_t e = warp                  ? dispatch_topk<32, false>(type, p, st)
                  : half && 2 * k > 128 ? dispatch_topk<128, true>(type, p, st)
                  : half                ? dispatch_topk<128, false>(type, p, st)
                  : big                 ? dispatch_topk<kCta, true>(type, p, st)
                                        : dispatch_topk<kCta, false>(type, p, st);
  if (e == cudaSuccess && parts > 1) {
    raven_topk::Params j = p;
    j.x = tmp;
    j.n = parts * k;
    j.parts = 1;
    e = big ? launch_join<true>(j, st) : launch_join<false>(j, st);
  }
  if (tmp) cudaFreeAsync(tmp, st);
  if (e != cudaSuccess) return fail(RAVEN_ECUDA, std::string("topk: ") + cudaGetErrorString(e));
  return RAVEN_OK;
}

}  // extern "C"
