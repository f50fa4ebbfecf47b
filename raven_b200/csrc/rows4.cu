// Operators of the C ABI (include/raven_gpu.h) on 4-bit rows: written, read back
// and scored against (int4.cuh); and scores put right for what a query has seen, a
// bias and filters (adjust.cuh).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>

#include "../../include/raven_gpu.h"
#include "internal.h"
#include "launch.h"
#include "status.cuh"
#include "adjust.cuh"
#include "int4.cuh"
#include "score4.cuh"
#include "score4_wide.cuh"

using namespace raven_launch;

namespace {

// Rows of memory, in bytes; wide enough for any pitch.
struct Rows {
  using U = unsigned __int128;
  U at, rows, pitch, width;
  Rows(const void* p, U n, U apart, U wide) : at((uintptr_t)p), rows(p && wide ? n : 0), pitch(n > 1 ? apart : wide), width(wide) {}
  U end() const { return at + (rows - 1) * pitch + width; }
};
// Whether rows of a and of b share memory; of different pitches, whether they may.
bool overlap(Rows a, Rows b) {
  if (a.rows == 0 || b.rows == 0 || a.at >= b.end() || b.at >= a.end()) return false;
  if (a.rows == 1) a.pitch = b.pitch;
  if (b.rows == 1) b.pitch = a.pitch;
  if (a.pitch != b.pitch || a.width > a.pitch || b.width > a.pitch) return true;
  // how far behind a row of a the next one of b starts: within it, or so far that the one before reaches into it
  const Rows::U p = a.pitch, d = (b.at + p * (a.at / p + 1) - a.at) % p;
  return d < a.width || p - d < b.width;
}

// ---------------------------------------------------------------------------
// 4-bit rows.
// ---------------------------------------------------------------------------
using raven_internal::int4_group;
using raven_int4::kBlock;

int kind_of(int32_t t) { return t == RAVEN_TYPE_F32 ? 0 : t == RAVEN_TYPE_F16 ? 1 : 2; }

constexpr uint64_t kMaxPitch = 0xffffffffull;  // pitches are 32-bit factors

int check_int4(const raven_rows* r, uint32_t dim, const char* what) {
  const std::string w(what);
  if (!r) return fail(RAVEN_EINVAL, w + ": null");
  const uint64_t group = int4_group(r->type);
  if (!group) return fail(RAVEN_EINVAL, w + ": type must be 4 bits");
  if (r->rows > kMaxRows) return fail(RAVEN_ELIMIT, w + ": more than 2^31 - 1 rows");
  if (r->rows == 0) return RAVEN_OK;
  if (!r->data || !r->exps) return fail(RAVEN_EINVAL, w + ": 4-bit rows need codes and scale words");
  if (!aligned(r->data, 16) || r->ld % 16 || r->ld < (dim + 31ull) / 32 * 16)
    return fail(RAVEN_EINVAL, w + ": 4-bit codes must start on 16 bytes, their pitch a multiple of 16 of at least dim / 2");
  if (r->ld > kMaxPitch || r->ld_exps > kMaxPitch) return fail(RAVEN_ELIMIT, w + ": pitch of 2^32 and more");
  const uint64_t per = kBlock / group;
  if (!aligned(r->exps, 4 * per) || r->ld_exps % per || r->ld_exps < (dim + kBlock - 1ull) / kBlock * per)
    return fail(RAVEN_EINVAL, w + ": scale words must start on those of 128 values, their pitch a multiple of them");
  return RAVEN_OK;
}

// The memory of the first n of 4-bit rows that are as they should be: their codes, their words.
Rows codes_of(const raven_rows* r, uint64_t n, uint32_t dim) { return Rows(r->data, n, r->ld, (dim + 31ull) / 32 * 16); }
Rows words_of(const raven_rows* r, uint64_t n, uint32_t dim) {
  return Rows(r->exps, n, r->ld_exps * 4, (dim + kBlock - 1ull) / kBlock * (kBlock / int4_group(r->type)) * 4);
}

// Rows of a CTA at once: `items` pieces a thread, as long as every SM gets rows. Sets what divides by `per`.
uint32_t rows_at_once(uint64_t m, uint32_t per, uint32_t items, int sms, uint32_t most, uint32_t* magic) {
  *magic = per > 1 ? (uint32_t)((0x100000000ull + per - 1) / per) : 0;
  const uint64_t fair = (m + 2ull * sms - 1) / (2ull * sms);
  return (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>({256 * items / per, most, fair}));
}

template <typename T, uint32_t L, bool LANE>
cudaError_t launch_write(raven_int4::Write p, int sms, cudaStream_t st) {
  const bool vec = p.ld * sizeof(T) % 16 == 0 && aligned(p.x, 16);
  p.per = (p.dim + 8 * L - 1) / (8 * L) * L;
  p.run = rows_at_once(p.m, p.per, raven_int4::kEights, sms, raven_int4::kRun, &p.magic);
  const uint64_t grid = std::min<uint64_t>((p.m + p.run - 1) / p.run, (uint64_t)sms * 64);
  static Allowed none;
  if constexpr (!LANE)
    if (vec) return launch(raven_int4::write_kernel<T, L, true, false>, grid, 256, 0, none, st, p);
  return launch(raven_int4::write_kernel<T, L, false, LANE>, grid, 256, 0, none, st, p);
}
template <typename T, bool LANE>
cudaError_t group_write(const raven_int4::Write& p, int sms, cudaStream_t st) {
  return p.group == 32   ? launch_write<T, 4, LANE>(p, sms, st)
         : p.group == 64 ? launch_write<T, 8, LANE>(p, sms, st)
                         : launch_write<T, 16, LANE>(p, sms, st);
}

// Up to here every CTA looks for its slots among the later ones, without the table's two launches: 1024 rows x 128 f16
// take 4.5 us (12.0 with a table), 4096 x 768 15.0 (20.4); 4096 x 128 are just past it (18.6, 15.3), 8192 x 768 well (32.2, 26.5).
constexpr uint64_t kFewSlots = 4096;
constexpr uint64_t kMaxSlots = 1ull << 30;

int write_rows(const void* x, int32_t type, uint64_t m, uint32_t dim, uint64_t ld, bool lane, const int32_t* slots,
               const raven_rows* out, int32_t* status, cudaStream_t st) {
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  raven_int4::Write p{};
  p.x = x;
  p.m = (uint32_t)m;
  p.ld = (uint32_t)ld;
  p.dim = dim;
  p.group = int4_group(out->type);
  p.units = (dim + 31) / 32;
  p.codes = (uint8_t*)out->data;
  p.words = (uint32_t*)out->exps;
  p.n = (uint32_t)out->rows;
  p.ld_codes = (uint32_t)out->ld;
  p.ld_words = (uint32_t)out->ld_exps;
  p.slots = slots;
  p.status = status;
  raven_int4::Claim* table = nullptr;
  cudaError_t e = cudaSuccess;
  if (slots && m > kFewSlots) {
    while ((1ull << p.bits) < 2 * m) ++p.bits;
    CU(cudaMallocAsync((void**)&table, sizeof(raven_int4::Claim) << p.bits, st));
    p.table = table;
    static Allowed none;
    e = cudaMemsetAsync(table, 0xff, sizeof(raven_int4::Claim) << p.bits, st);
    if (e == cudaSuccess)
      e = launch(raven_int4::claim_kernel, (m + 255) / 256, 256, 0, none, st, slots, (uint32_t)m, p.n, table, p.bits);
  }
  if (e == cudaSuccess)
    e = type == RAVEN_TYPE_F32   ? (lane ? group_write<float, true>(p, sms, st) : group_write<float, false>(p, sms, st))
        : type == RAVEN_TYPE_F16 ? group_write<__half, false>(p, sms, st)
                                 : group_write<__nv_bfloat16, false>(p, sms, st);
  if (table) cudaFreeAsync(table, st);
  if (e != cudaSuccess) return fail(RAVEN_ECUDA, std::string("4-bit rows: ") + cudaGetErrorString(e));
  return RAVEN_OK;
}

template <typename T>
cudaError_t launch_read(raven_int4::Read p, int sms, cudaStream_t st) {
  const bool vec = p.ld * sizeof(T) % 16 == 0 && aligned(p.out, 16);
  constexpr uint32_t V = 16 / sizeof(T);
  p.per = (p.dim + V - 1) / V;
  p.run = rows_at_once(p.m, p.per, raven_int4::kItems, sms, 256 * raven_int4::kItems, &p.magic);
  const uint64_t grid = std::min<uint64_t>((p.m + p.run - 1) / p.run, (uint64_t)sms * 64);
  static Allowed none;
  return launch(vec ? raven_int4::read_kernel<T, true> : raven_int4::read_kernel<T, false>, grid, 256, 0, none, st, p);
}

// ---------------------------------------------------------------------------
// Scores.
// ---------------------------------------------------------------------------
constexpr uint32_t kMostShared = 227 * 1024;
// Values of a chunk's queries that each CTA lays out for itself; more are laid out once, by a launch before. On either
// side of it: 8 x 65536 x 1024 16.7 us (laid out before 17.2), 1 x 100000 x 1024 21.9 (23.2); 4 x 32768 x 4096 33.8 (32.2),
// 8 x 32768 x 4096 37.1 (32.1), 64 x 65536 x 512 36.4 (27.1).
constexpr uint64_t kOwnLayout = 16384;

// Codes as boxes of `wide` bytes (64: a block) x `rows` rows; what is past a row's end or the last row reads 0.
bool codes_map(CUtensorMap* m, const raven_rows* v, uint32_t units, uint32_t wide, uint32_t rows, CUtensorMapSwizzle swizzle) {
  PFN_cuTensorMapEncodeTiled_v12000 f = raven_internal::encode_tiled();
  if (!f) return false;
  cuuint64_t gdim[2] = {16ull * units, v->rows};
  cuuint64_t gstride[1] = {v->ld};
  cuuint32_t box[2] = {wide, rows};
  cuuint32_t es[2] = {1, 1};
  return f(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, (void*)v->data, gdim, gstride, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
           swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int NT, int MT, int G, bool F32, typename O>
cudaError_t launch_score4(const CUtensorMap& map, const raven_score4::Params& p, uint64_t ctas, uint64_t smem, cudaStream_t st) {
  using namespace raven_score4;
  static Allowed allowed(kMostShared);
  return launch(score4_kernel<NT, MT, G, F32, O>, ctas, Layout<NT, MT, G>::kThreads, (uint32_t)smem, allowed, st, map, p);
}

// Scratch of a call: queries laid out (as large as they are) and sums of slices (slices times what the scores take).
// Above this the queries are taken in halves of whole chunks, of which a kernel's CTAs read every code anyway, so that
// nothing is laid out twice; the sums of a single chunk in halves of the rows.
constexpr uint64_t kMostScratch = 1ull << 30;

bool too_much(uint64_t scratch, const raven_score4::Params& p, uint32_t chunk) {
  return scratch > kMostScratch && (p.nq > chunk || p.n >= 512);
}

template <typename F>
cudaError_t in_halves(const raven_rows* v, const raven_score4::Params& p, int out_type, uint32_t chunk, F&& run) {
  raven_rows a = *v, b = *v;
  raven_score4::Params pa = p, pb = p;
  const uint64_t size = out_type == 0 ? 4 : 2;
  if (p.nq > chunk) {
    const uint64_t half = (p.nq / 2 + chunk - 1) / chunk * chunk;
    pa.nq = half;
    pb.nq = p.nq - half;
    pb.q = (const uint8_t*)p.q + half * p.ld_q * (p.q_type == 0 ? 4 : 2);
    pb.out = (uint8_t*)p.out + half * p.ld * size;
  } else {
    const uint64_t half = (p.n / 2 + 127) / 128 * 128;
    a.rows = pa.n = half;
    b.rows = pb.n = p.n - half;
    b.data = (const uint8_t*)v->data + half * v->ld;
    b.exps = (const uint8_t*)((const uint32_t*)v->exps + half * v->ld_exps);
    pb.words = (const uint32_t*)b.exps;
    pb.out = (uint8_t*)p.out + half * size;
    if (p.bias) pb.bias = p.bias + half;
  }
  const cudaError_t e = run(&a, pa);
  return e == cudaSuccess ? run(&b, pb) : e;
}

cudaError_t launch_join(const raven_score4::Join& j, int out_type, int sms, cudaStream_t st) {
  using namespace raven_score4;
  static Allowed none;
  const uint64_t grid = std::min<uint64_t>((j.nq * (j.ld / 4) + 255) / 256, (uint64_t)sms * 32);
  return launch(out_type == 0 ? join_kernel<float> : out_type == 1 ? join_kernel<__half> : join_kernel<__nv_bfloat16>, grid, 256,
                0, none, st, j);
}

template <int NT, int MT, int G, bool F32>
cudaError_t run_score4(const raven_rows* v, raven_score4::Params p, int out_type, int sms, cudaStream_t st) {
  using namespace raven_score4;
  using L = Layout<NT, MT, G>;
  using Q = Laid<NT>;
  constexpr uint32_t kQueries = F32 ? NT * 4 : NT * 8;
  const Params whole = p;
  p.chunks = (uint32_t)((p.nq + kQueries - 1) / kQueries);
  // slices of a row: as few as let a CTA hold its queries beside its rings
  p.slices = 1;
  p.slice = p.blocks;
  while (L::bytes(std::min(4 * p.slice, p.units), std::min(p.slice * L::kWords, p.groups), std::min(L::kWarps, p.slice),
                  L::kLeast) >
         kMostShared) {
    ++p.slices;
    p.slice = (p.blocks + p.slices - 1) / p.slices;
  }
  p.slices = (p.blocks + p.slice - 1) / p.slice;
  const uint32_t shares = p.chunks * p.slices;
  const uint64_t columns = std::max<uint64_t>(1, (uint64_t)sms / shares);  // CTAs of a share
  // Warps that share a row: those that leave the busiest SM least, in blocks of a warp's tile, with half a block of
  // each warp for a tile's end and sums that meet.
  uint64_t best = ~0ull;
  for (uint32_t split = 1; split <= p.slice && L::kWarps % split == 0; split *= 2) {
    const uint64_t rows = L::kRows * (L::kWarps / split), tiles = (p.n + rows - 1) / rows;
    const uint64_t time = (tiles + columns - 1) / columns * (2 * ((p.slice + split - 1) / split) + 1);
    if (time < best) {
      best = time;
      p.split = split;
      p.tiles = (uint32_t)tiles;
    }
  }
  const uint32_t units = std::min(4 * p.slice, p.units), groups = std::min(p.slice * L::kWords, p.groups);
  p.depth = kMaxDepth;
  while (L::bytes(units, groups, p.split, p.depth) > kMostShared) --p.depth;
  uint8_t* tmp = nullptr;
  cudaError_t e = cudaSuccess;
  const bool lay = std::min<uint64_t>(p.nq, kQueries) * p.dim > kOwnLayout;
  const uint64_t laid = lay ? (p.chunks * Q::bytes(p.units, p.groups) + 255) / 256 * 256 : 0;
  const uint64_t wide = (p.n + 3) / 4 * 4, sums = p.slices > 1 ? p.slices * p.nq * wide * 4 : 0;
  const uint64_t backs = p.slices > 1 ? (uint64_t)p.chunks * kQueries * 16 : 0;
  if (too_much(laid + sums + backs, p, kQueries))
    return in_halves(v, whole, out_type, kQueries, [&](const raven_rows* r, const Params& q) {
      return run_score4<NT, MT, G, F32>(r, q, out_type, sms, st);
    });
  if (laid + sums + backs && (e = cudaMallocAsync((void**)&tmp, laid + sums + backs, st)) != cudaSuccess) return e;
  if (backs) p.backs = (float4*)(tmp + laid + sums);
  const Join j{(const float*)(tmp + laid), wide, p.nq * wide, p.slices, p.nq, p.n, p.backs, p.bias, p.out, p.ld};
  if (p.slices > 1) {
    p.out = tmp + laid;
    p.ld = wide;
    p.ld_slice = p.nq * wide;
    p.bias = nullptr;
  }
  if (lay) {
    static Allowed none;
    e = launch(lay_out_kernel<Q, G, F32>, (uint64_t)p.chunks * kQueries, 256, 0, none, st, p, tmp);
    p.q = nullptr;
    p.laid = tmp;
  }
  p.whole = aligned(p.out, 16) && (p.nq == 1 || p.ld % (16 / (p.slices > 1 || out_type == 0 ? 4 : 2)) == 0);
  CUtensorMap map;
  if (e == cudaSuccess && !codes_map(&map, v, p.units, std::min(64u, 16 * p.units), L::kRows, CU_TENSOR_MAP_SWIZZLE_NONE)) e = cudaErrorInvalidValue;
  const uint64_t ctas = std::min<uint64_t>(columns, p.tiles) * shares, smem = L::bytes(units, groups, p.split, p.depth);
  if (e == cudaSuccess)
    e = p.slices > 1 || out_type == 0 ? launch_score4<NT, MT, G, F32, float>(map, p, ctas, smem, st)
        : out_type == 1               ? launch_score4<NT, MT, G, F32, __half>(map, p, ctas, smem, st)
                                      : launch_score4<NT, MT, G, F32, __nv_bfloat16>(map, p, ctas, smem, st);
  if (p.slices > 1 && e == cudaSuccess) e = launch_join(j, out_type, sms, st);
  if (tmp) cudaFreeAsync(tmp, st);
  return e;
}

template <int NC, int G, bool F32, typename O>
cudaError_t launch_wide(const CUtensorMap& map, const raven_score4::Params& p, uint64_t ctas, uint64_t smem, cudaStream_t st) {
  static Allowed allowed(kMostShared);
  return launch(raven_score4::wide_kernel<NC, G, F32, O>, ctas, raven_score4::Wide<NC>::kThreads, (uint32_t)smem, allowed, st, map, p);
}

template <int NC, int G, bool F32>
cudaError_t run_wide(const raven_rows* v, raven_score4::Params p, int out_type, int sms, cudaStream_t st) {
  using namespace raven_score4;
  using L = Wide<NC>;
  using Q = WideLaid<NC>;
  constexpr uint32_t kQueries = F32 ? NC / 2 : NC;
  const Params whole = p;
  p.chunks = (uint32_t)((p.nq + kQueries - 1) / kQueries);
  p.tiles = (uint32_t)((p.n + kWideRows - 1) / kWideRows);
  // Slices of a row: those that take least time, in microseconds. A block of a team takes 0.6 and 0.55 for each scale
  // group's chain, a tile's end 0.7, a block of queries NC / 128, the join 3 and its bytes (40 x 5000 x 1000, groups of
  // 32: 30 us in one slice, 13.9 in those that this gives).
  auto bytes = [&](uint32_t slice, uint32_t depth) {
    return L::bytes(std::min(4 * slice, p.units), depth);
  };
  double best = 0;
  uint64_t columns = 1;
  for (uint32_t n = 1; n <= p.blocks; ++n) {
    const uint32_t slice = (p.blocks + n - 1) / n, slices = (p.blocks + slice - 1) / slice;
    if (slices != n || bytes(slice, 2) > kMostShared) continue;
    const uint64_t shares = (uint64_t)p.chunks * slices, c = std::max<uint64_t>(1, (uint64_t)sms / shares);
    const uint64_t rounds = (p.tiles + L::kTeams * c - 1) / (L::kTeams * c) * ((shares + sms - 1) / sms);
    const double block = 0.6 + 0.55 * (kBlock / G);
    const double time = rounds * (slice * block + 0.7) + slice * NC / 128.0 + (slices > 1 ? 3 + 1.6e-6 * p.nq * p.n * slices : 0);
    if (best == 0 || time < best) {
      best = time;
      columns = c;
      p.slice = slice;
      p.slices = slices;
    }
    if (n >= 64 && best > 0) break;
  }
  const uint32_t shares = p.chunks * p.slices;
  p.depth = kWideDepth;
  while (bytes(p.slice, p.depth) > kMostShared) --p.depth;
  uint8_t* tmp = nullptr;
  cudaError_t e = cudaSuccess;
  const bool lay = std::min<uint64_t>(p.nq, kQueries) * p.dim > kOwnLayout;
  const uint64_t laid = lay ? (p.chunks * Q::bytes(p.units, 0) + 255) / 256 * 256 : 0;
  const uint64_t wide = (p.n + 3) / 4 * 4, sums = p.slices > 1 ? p.slices * p.nq * wide * 4 : 0;
  const uint64_t backs = p.slices > 1 ? (uint64_t)p.chunks * kQueries * 16 : 0;
  if (too_much(laid + sums + backs, p, kQueries))
    return in_halves(v, whole, out_type, kQueries,
                     [&](const raven_rows* r, const Params& q) { return run_wide<NC, G, F32>(r, q, out_type, sms, st); });
  if (laid + sums + backs && (e = cudaMallocAsync((void**)&tmp, laid + sums + backs, st)) != cudaSuccess) return e;
  if (backs) p.backs = (float4*)(tmp + laid + sums);
  const Join j{(const float*)(tmp + laid), wide, p.nq * wide, p.slices, p.nq, p.n, p.backs, p.bias, p.out, p.ld};
  if (p.slices > 1) {
    p.out = tmp + laid;
    p.ld = wide;
    p.ld_slice = p.nq * wide;
    p.bias = nullptr;
  }
  if (lay) {
    static Allowed none;
    e = launch(lay_out_kernel<Q, G, F32>, (uint64_t)p.chunks * kQueries, 256, 0, none, st, p, tmp);
    p.q = nullptr;
    p.laid = tmp;
  }
  CUtensorMap map;
  if (e == cudaSuccess && !codes_map(&map, v, p.units, 64, kWideRows, CU_TENSOR_MAP_SWIZZLE_64B)) e = cudaErrorInvalidValue;
  const uint64_t ctas = std::min<uint64_t>(columns, (p.tiles + L::kTeams - 1) / L::kTeams) * shares;
  if (e == cudaSuccess)
    e = p.slices > 1 || out_type == 0 ? launch_wide<NC, G, F32, float>(map, p, ctas, bytes(p.slice, p.depth), st)
        : out_type == 1               ? launch_wide<NC, G, F32, __half>(map, p, ctas, bytes(p.slice, p.depth), st)
                                      : launch_wide<NC, G, F32, __nv_bfloat16>(map, p, ctas, bytes(p.slice, p.depth), st);
  if (p.slices > 1 && e == cudaSuccess) e = launch_join(j, out_type, sms, st);
  if (tmp) cudaFreeAsync(tmp, st);
  return e;
}

// Columns are queries, two for one of f32. An instruction of 96 columns takes no longer than one of 64, but each
// column has its additions, and its scores: as few chunks as there can be, the narrower ones where they do.
template <int G, bool F32>
cudaError_t group_score4(const raven_rows* v, const raven_score4::Params& p, int out_type, int sms, cudaStream_t st) {
  const uint64_t columns = F32 ? 2 * p.nq : p.nq;
  if (columns <= 8) {  // four M tiles a warp, but where rows are so long that a CTA could not hold its queries beside them
    using namespace raven_score4;
    using L = Layout<1, 4, G>;
    const bool fits = L::bytes(p.units, p.groups, std::min(L::kWarps, p.blocks), L::kLeast) <= kMostShared;
    return fits ? run_score4<1, 4, G, F32>(v, p, out_type, sms, st) : run_score4<1, 2, G, F32>(v, p, out_type, sms, st);
  }
  return columns <= 16 ? run_score4<2, 2, G, F32>(v, p, out_type, sms, st)
         : columns <= 32 ? run_wide<32, G, F32>(v, p, out_type, sms, st)
         : (columns + 63) / 64 > (columns + 95) / 96 ? run_wide<96, G, F32>(v, p, out_type, sms, st)
                                                     : run_wide<64, G, F32>(v, p, out_type, sms, st);
}

template <bool F32>
cudaError_t dispatch_score4(const raven_rows* v, const raven_score4::Params& p, uint32_t group, int out_type, int sms,
                            cudaStream_t st) {
  return group == 32   ? group_score4<32, F32>(v, p, out_type, sms, st)
         : group == 64 ? group_score4<64, F32>(v, p, out_type, sms, st)
                       : group_score4<128, F32>(v, p, out_type, sms, st);
}

// ---------------------------------------------------------------------------
// Adjusted scores.
// ---------------------------------------------------------------------------
template <typename T>
cudaError_t launch_adjust(const raven_adjust::Params& p, bool largest, cudaStream_t st) {
  static Allowed none;
  const uint32_t smem = raven_adjust::shared_bytes(p.tile, p.starts != nullptr);
  return launch(largest ? raven_adjust::adjust_kernel<T, true> : raven_adjust::adjust_kernel<T, false>, p.nq * p.tiles,
                raven_adjust::kThreads, smem, none, st, p);
}

__global__ void status_kernel(int* status) {
  raven_score::after_previous();
  atomicOr(status, atomicExch(&raven_score::g_status, 0));
}

}  // namespace

namespace raven_internal {

uint32_t int4_group(int32_t t) {
  return t == RAVEN_TYPE_INT4_32 ? 32 : t == RAVEN_TYPE_INT4_64 ? 64 : t == RAVEN_TYPE_INT4_128 ? 128 : 0;
}

int rows4_status(int* d_status, cudaStream_t st) {
  static Allowed none;
  CU(launch(status_kernel, 1, 1, 0, none, st, d_status));
  return RAVEN_OK;
}

int int4_scores(const raven_rows* q, const raven_rows* v, uint32_t dim, float alpha, const float* bias, void* out,
                int32_t out_type, uint64_t ld, int32_t* status, void* stream) {
  if (int rc = check_dim(dim)) return rc;
  if (int rc = check_int4(v, dim, "vectors")) return rc;
  if (!q || !float_type(q->type)) return fail(RAVEN_EINVAL, "queries: type must be f32, f16 or bf16 with 4-bit vectors");
  if (q->rows > kMaxRows) return fail(RAVEN_ELIMIT, "queries: more than 2^31 - 1 rows");
  if (q->rows && (!q->data || !aligned(q->data, type_size(q->type))))
    return fail(RAVEN_EINVAL, "queries: null or not aligned to their type");
  if (q->rows && q->ld < dim) return fail(RAVEN_EINVAL, "queries: pitch below dim");
  if (!float_type(out_type)) return fail(RAVEN_EINVAL, "scores: type must be f32, f16 or bf16");
  if (!aligned(bias, 4) || !aligned(status, 4)) return fail(RAVEN_EINVAL, "scores: bias and status must start on 4 bytes");
  if (q->rows == 0 || v->rows == 0) return RAVEN_OK;
  if (!out) return fail(RAVEN_EINVAL, "scores: null output");
  if (!aligned(out, type_size(out_type))) return fail(RAVEN_EINVAL, "scores: output is not aligned to its type");
  if (ld < v->rows) return fail(RAVEN_EINVAL, "scores: output pitch below the number of vectors");
  const uint64_t in = type_size(q->type), size = type_size(out_type);
  const Rows scores(out, q->rows, ld * Rows::U(size), v->rows * size);
  if (overlap(scores, Rows(q->data, q->rows, q->ld * Rows::U(in), dim * in)) || overlap(scores, codes_of(v, v->rows, dim)) ||
      overlap(scores, words_of(v, v->rows, dim)) || overlap(scores, Rows(bias, 1, 0, v->rows * 4)))
    return fail(RAVEN_EINVAL, "scores: the output overlaps queries, vectors or bias");
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  raven_score4::Params p{};
  p.q = q->data;
  p.q_type = kind_of(q->type);
  p.nq = q->rows;
  p.ld_q = q->ld;
  p.whole_q = aligned(q->data, 16) && (q->ld * type_size(q->type) % 16 == 0 || p.nq == 1);
  p.words = (const uint32_t*)v->exps;
  p.n = v->rows;
  p.ld_words = v->ld_exps;
  p.dim = dim;
  p.units = (dim + 31) / 32;
  p.blocks = (dim + raven_int4::kBlock - 1) / raven_int4::kBlock;
  const uint32_t group = int4_group(v->type);
  p.groups = (dim + group - 1) / group;
  p.alpha_exp = alpha != 0.f && std::isfinite(alpha) ? std::ilogb(alpha) : 0;
  p.alpha = std::scalbn(alpha, -p.alpha_exp);
  p.top = 14;
  while (p.top > 10 && dim > 4096u << (14 - p.top)) --p.top;
  p.bias = bias;
  p.out = out;
  p.ld = ld;
  p.status = status;
  CU(q->type == RAVEN_TYPE_F32 ? dispatch_score4<true>(v, p, group, kind_of(out_type), sms, st)
                               : dispatch_score4<false>(v, p, group, kind_of(out_type), sms, st));
  return RAVEN_OK;
}

int int4_write_lane_major(const float* d_rows, uint64_t n, uint32_t dim, const raven_rows* out, cudaStream_t st) {
  if (int rc = check_int4(out, dim, "out")) return rc;
  if (out->rows < n) return fail(RAVEN_EINVAL, "out: fewer rows than the index");
  return write_rows(d_rows, RAVEN_TYPE_F32, n, dim, dim, true, nullptr, out, nullptr, st);
}

}  // namespace raven_internal

extern "C" {

int raven_int4_write_device(const void* d_rows, int32_t type, uint64_t m, uint32_t dim, uint64_t ld,
                            const int32_t* d_slots, const raven_rows* out, int32_t* d_status, void* stream) {
  NvtxRange nvtx_range("raven.int4_write");
  if (int rc = check_dim(dim)) return rc;
  if (!float_type(type)) return fail(RAVEN_EINVAL, "rows: type must be f32, f16 or bf16");
  if (int rc = check_int4(out, dim, "out")) return rc;
  if (!aligned(d_slots, 4) || !aligned(d_status, 4)) return fail(RAVEN_EINVAL, "slots and status must start on 4 bytes");
  if (m == 0) return RAVEN_OK;
  if (m > (d_slots ? kMaxSlots : kMaxRows)) return fail(RAVEN_ELIMIT, "rows: more than 2^31 - 1, or 2^30 with slots");
  if (!d_rows) return fail(RAVEN_EINVAL, "rows: null");
  if (ld < dim) return fail(RAVEN_EINVAL, "rows: pitch below dim");
  if (ld > kMaxPitch) return fail(RAVEN_ELIMIT, "rows: pitch of 2^32 and more");
  if (!aligned(d_rows, type_size(type))) return fail(RAVEN_EINVAL, "rows: not aligned to their type");
  if (!d_slots && m > out->rows) return fail(RAVEN_EINVAL, "out: fewer rows than are written");
  const uint64_t n = d_slots ? out->rows : m;
  const Rows codes = codes_of(out, n, dim), words = words_of(out, n, dim), slots(d_slots, 1, 0, m * 4);
  const Rows in(d_rows, m, ld * type_size(type), dim * type_size(type));
  if (overlap(codes, in) || overlap(words, in) || overlap(codes, slots) || overlap(words, slots))
    return fail(RAVEN_EINVAL, "out: overlaps the rows that are written, or their slots");
  return write_rows(d_rows, type, m, dim, ld, false, d_slots, out, d_status, (cudaStream_t)stream);
}

int raven_int4_read_device(const raven_rows* rows, uint32_t dim, const int32_t* d_ids, uint64_t m, void* d_out,
                           int32_t out_type, uint64_t ld, int32_t* d_status, void* stream) {
  NvtxRange nvtx_range("raven.int4_read");
  if (int rc = check_dim(dim)) return rc;
  if (int rc = check_int4(rows, dim, "rows")) return rc;
  if (!float_type(out_type)) return fail(RAVEN_EINVAL, "output: type must be f32, f16 or bf16");
  if (!aligned(d_ids, 4) || !aligned(d_status, 4)) return fail(RAVEN_EINVAL, "ids and status must start on 4 bytes");
  if (m == 0) return RAVEN_OK;
  if (m > kMaxRows) return fail(RAVEN_ELIMIT, "output: more than 2^31 - 1 rows");
  if (!d_out || !aligned(d_out, type_size(out_type))) return fail(RAVEN_EINVAL, "output: null or not aligned to its type");
  if (ld < dim) return fail(RAVEN_EINVAL, "output: pitch below dim");
  if (ld > kMaxPitch) return fail(RAVEN_ELIMIT, "output: pitch of 2^32 and more");
  if (!d_ids && m > rows->rows) return fail(RAVEN_EINVAL, "rows: fewer than are read");
  const Rows out(d_out, m, ld * type_size(out_type), dim * type_size(out_type));
  const uint64_t n = d_ids ? rows->rows : m;
  if (overlap(out, codes_of(rows, n, dim)) || overlap(out, words_of(rows, n, dim)) || overlap(out, Rows(d_ids, 1, 0, m * 4)))
    return fail(RAVEN_EINVAL, "output: overlaps the rows that are read, or their ids");
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  raven_int4::Read p{};
  p.codes = (const uint8_t*)rows->data;
  p.words = (const uint32_t*)rows->exps;
  p.n = (uint32_t)rows->rows;
  p.ld_codes = (uint32_t)rows->ld;
  p.ld_words = (uint32_t)rows->ld_exps;
  p.dim = dim;
  p.group = raven_internal::int4_group(rows->type);
  p.units = (dim + 31) / 32;
  p.ids = d_ids;
  p.m = (uint32_t)m;
  p.out = d_out;
  p.ld = (uint32_t)ld;
  p.status = d_status;
  cudaStream_t st = (cudaStream_t)stream;
  CU(out_type == RAVEN_TYPE_F32   ? launch_read<float>(p, sms, st)
     : out_type == RAVEN_TYPE_F16 ? launch_read<__half>(p, sms, st)
                                  : launch_read<__nv_bfloat16>(p, sms, st));
  return RAVEN_OK;
}

int raven_adjust_scores_device(const void* d_scores, int32_t type, uint64_t nq, uint64_t n, uint64_t ld,
                               const raven_adjustments* by, int32_t largest, void* d_out, uint64_t ld_out,
                               int32_t* d_status, void* stream) {
  NvtxRange nvtx_range("raven.adjust_scores");
  if (!by) return fail(RAVEN_EINVAL, "null adjustments");
  if (!float_type(type)) return fail(RAVEN_EINVAL, "scores: type must be f32, f16 or bf16");
  if (nq > kMaxRows || n > kMaxRows) return fail(RAVEN_ELIMIT, "more than 2^31 - 1 queries or vectors");
  if (nq == 0 || n == 0) return RAVEN_OK;
  const uint64_t size = type_size(type);
  if (!d_scores || !d_out) return fail(RAVEN_EINVAL, "scores: null");
  if (!aligned(d_scores, size) || !aligned(d_out, size)) return fail(RAVEN_EINVAL, "scores: not aligned to their type");
  if (nq == 1) ld = ld_out = n;
  if (ld < n || ld_out < n) return fail(RAVEN_EINVAL, "scores: pitch below the row length");
  if (ld > 1ull << 40 || ld_out > 1ull << 40) return fail(RAVEN_ELIMIT, "scores: pitch above 2^40");
  const Rows out(d_out, nq, ld_out * Rows::U(size), n * size);
  if (!(d_scores == d_out && ld == ld_out) && overlap(out, Rows(d_scores, nq, ld * Rows::U(size), n * size)))
    return fail(RAVEN_EINVAL, "scores: the output overlaps them, but is not the same");
  if (!aligned(by->bias, 4) || !aligned(by->allow, 4) || !aligned(by->allow_rows, 4) || !aligned(by->seen, 4) ||
      !aligned(by->seen_starts, 8) || !aligned(by->repetition, 4) || !aligned(by->presence, 4) ||
      !aligned(by->frequency, 4) || !aligned(d_status, 4))
    return fail(RAVEN_EINVAL, "an argument is not aligned to its type");
  if (by->bias && by->ld_bias && by->ld_bias < n) return fail(RAVEN_EINVAL, "bias: pitch below the row length");
  if (by->allow) {
    if (by->allow_count == 0 || by->allow_count > kMaxRows) return fail(RAVEN_EINVAL, "filters: 1 to 2^31 - 1 of them");
    if (by->ld_allow < (n + 31) / 32 && by->allow_count > 1) return fail(RAVEN_EINVAL, "filters: pitch below n / 32 words");
    if (!by->allow_rows && by->allow_count != 1 && by->allow_count != nq)
      return fail(RAVEN_EINVAL, "filters: one, or one for each query, without allow_rows");
  }
  if (by->seen_starts && !by->seen && by->seen_total) return fail(RAVEN_EINVAL, "seen: null");
  if (by->seen && !by->seen_starts) return fail(RAVEN_EINVAL, "seen: needs its starts");
  const Rows others[] = {Rows(by->bias, by->ld_bias ? nq : 1, by->ld_bias * Rows::U(4), n * 4),
                         Rows(by->allow, by->allow_count, by->ld_allow * Rows::U(4), (n + 31) / 32 * 4),
                         Rows(by->allow_rows, 1, 0, nq * 4),
                         Rows(by->seen, 1, 0, by->seen_total * Rows::U(4)),
                         Rows(by->seen_starts, 1, 0, (nq + 1) * 8),
                         Rows(by->repetition, 1, 0, nq * 4),
                         Rows(by->presence, 1, 0, nq * 4),
                         Rows(by->frequency, 1, 0, nq * 4),
                         Rows(d_status, 1, 0, 4)};
  for (const Rows& r : others)
    if (overlap(out, r)) return fail(RAVEN_EINVAL, "scores: the output overlaps what they are adjusted by");
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  raven_adjust::Params p{};
  p.x = d_scores;
  p.out = d_out;
  p.nq = nq;
  p.n = n;
  p.ld = ld;
  p.ld_out = ld_out;
  p.bias = by->bias;
  p.ld_bias = by->ld_bias;
  p.allow = by->allow;
  p.allow_count = by->allow_count;
  p.ld_allow = by->ld_allow;
  p.allow_rows = by->allow_rows;
  p.seen = by->seen;
  p.seen_total = by->seen_total;
  p.starts = by->seen_starts;
  p.repetition = by->repetition;
  p.presence = by->presence;
  p.frequency = by->frequency;
  p.repetition_all = by->repetition_all;
  p.presence_all = by->presence_all;
  p.frequency_all = by->frequency_all;
  p.status = d_status;
  // the largest tiles, since each scans its row's history, that leave every SM four; 1024 places at least (1 x 100000 4.4 us,
  // 4.7 with 256 as with 2048; 4 x 100000 bf16 5.9, 8.3 with 256)
  const uint64_t most = 16 / size - 1;  // columns before a row's first
  p.tile = raven_adjust::kMostPlaces;
  while (p.tile > 1024 && nq * ((n + most + p.tile - 1) / p.tile) < 4ull * sms) p.tile /= 2;
  p.tiles = (uint32_t)((n + most + p.tile - 1) / p.tile);
  if (nq * p.tiles > kMaxRows) return fail(RAVEN_ELIMIT, "scores: more tiles than a launch holds");
  cudaStream_t st = (cudaStream_t)stream;
  CU(type == RAVEN_TYPE_F32   ? launch_adjust<float>(p, largest != 0, st)
     : type == RAVEN_TYPE_F16 ? launch_adjust<__half>(p, largest != 0, st)
                              : launch_adjust<__nv_bfloat16>(p, largest != 0, st));
  return RAVEN_OK;
}

}  // extern "C"
