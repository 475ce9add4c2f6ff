// The C entry points of the products with 4-bit weights: argument checks, and which kernel a call takes.
#include <algorithm>

#include "fp4.h"

namespace {

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
constexpr int64_t kMax31 = 2147483647;

int64_t row_tiles(const lse_fp4_gemm_args& p) { return (p.glu ? 2 : 1) * lse::ceil_div(p.N, 16); }

// Microseconds that a call takes apart from the weight's way from HBM, for the tile kernels by stages (128 k of one
// tile on each CU), for the streaming kernel by what a CU reads through its L1. Fitted to 84 sizes of both kinds of rows
// and both epilogues (M 9 to 4096, N 1024 to 28672, K 1536 to 14336), each timed with the plans below that suit it: the
// one chosen here is 0.6 % slower than the fastest in the mean, 11 % at most.
struct Tile {
  int bm, bn;
  int slots;        // workgroups that run at once on 256 CUs
  double one, all;  // of a stage: one workgroup a CU, and all slots taken
};
constexpr Tile kTiles[2][3] = {
    {{32, 128, 256, 0.29, 0.29}, {64, 128, 256, 0.46, 0.46}, {64, 256, 512, 0.82, 1.50}},   // bf16 rows
    {{32, 128, 512, 0.26, 0.45}, {64, 128, 512, 0.37, 0.64}, {128, 256, 512, 0.85, 1.62}}};  // 8-bit rows
constexpr double kLaunchUs = 2.5, kStreamBytesPerUs = 4.3e6, kTileBytesPerUs = 5e6, kL1BytesPerUs = 65e3;
constexpr double kSecondPassUs = 3.0, kPartBytesPerUs = 4e6;
constexpr int64_t kMaxPartBytes = 64 << 20;

// Which kernel a call takes, from its sizes alone: the one whose time is estimated the shortest.
lse::Fp4Plan plan_of(const lse_fp4_gemm_args& p) {
  const bool rows8 = p.x_scales != nullptr;
  const int64_t nrb = row_tiles(p), chunks = lse::ceil_div(p.K, lse::kFp4Chunk);
  const int narrow = p.glu ? 2 : 1;
  // Few rows: the narrowest panels, since x costs next to nothing.
  lse::Fp4Plan best{0, 16 * narrow, 1, (int)chunks};
  if (p.M <= (rows8 ? 8 : 4)) return best;
  const int64_t stages = lse::ceil_div(p.K, lse::kFp4Step);
  const double weight = 16.0 * nrb * stages * 68;
  double least = 1e30;
  auto take = [&](double us, int bm, int bn, int64_t splits, int64_t per) {
    if (us < least) least = us, best = {bm, bn, (int)splits, (int)per};
  };
  const int64_t groups = lse::ceil_div(p.M, 16);
  for (int rt = 4; rt >= narrow; rt /= 2) {
    const int64_t rounds = lse::ceil_div(lse::ceil_div(nrb, rt) * groups, 256);
    const double rows = p.M < 16 ? p.M : 16;
    const double bytes = stages * (rows * (rows8 ? 132.0 : 256.0) + rt * 16 * 68.0);
    const double us = kLaunchUs + std::max(weight / kStreamBytesPerUs, rounds * bytes / kL1BytesPerUs);
    take(us, 0, 16 * rt, 1, chunks);
  }
  for (const Tile& t : kTiles[rows8]) {
    if (p.M <= 16 && (t.bm > 32 || !rows8)) continue;
    const int64_t tiles = lse::ceil_div(p.M, t.bm) * lse::ceil_div(nrb, t.bn / 16);
    for (int64_t splits = 1; splits <= 8; splits *= 2) {
      const int64_t per = lse::ceil_div(chunks, splits), ranges = lse::ceil_div(chunks, per);
      if (splits > 1 && (ranges != splits || per < 2)) break;
      const double part = 64.0 * nrb * p.M * splits;
      if (splits > 1 && part > kMaxPartBytes) break;
      const int64_t blocks = tiles * splits, full = blocks / t.slots, rest = blocks % t.slots;
      const double last = rest == 0 ? 0.0 : rest <= 256 ? t.one : t.all;
      double us = std::min<double>(stages, 4 * per) * (full * t.all + last);
      us = kLaunchUs + std::max(weight / kTileBytesPerUs, us);
      if (splits > 1) us += kSecondPassUs + 2 * part / kPartBytesPerUs;
      take(us, t.bm, t.bn, splits, per);
    }
  }
  return best;
}

// LSE_OK if the sizes are a product's (K may be 0).
int check_sizes(const lse_fp4_gemm_args& p) {
  if (p.M < 0 || p.N < 0 || p.K < 0 || p.M > kMax31 || p.N > kMax31 - 64 || (p.glu != 0 && p.glu != 1))
    return LSE_E_SHAPE;
  if (p.K % lse::kFp4Group) return LSE_E_ALIGN;
  return p.K > LSE_FP4_MAX_K ? LSE_E_RANGE : LSE_OK;
}

}  // namespace

extern "C" {

int64_t lse_fp4_gemm_workspace_bytes(const struct lse_fp4_gemm_args* args) {
  if (!args || check_sizes(*args)) return -1;
  if (args->M == 0 || args->N == 0 || args->K == 0) return 0;
  const int64_t nrb = row_tiles(*args);
  const lse::Fp4Plan plan = plan_of(*args);
  return plan.splits > 1 ? plan.splits * args->M * 16 * nrb * 4 : 0;
}

int lse_fp4_gemm_choice(const struct lse_fp4_gemm_args* args, int64_t* tile_rows, int64_t* tile_columns,
                        int64_t* splits) {
  if (!args || !tile_rows || !tile_columns || !splits) return LSE_E_NULL;
  if (const int st = check_sizes(*args)) return st;
  lse::Fp4Plan plan{};
  if (args->M && args->N && args->K) plan = plan_of(*args);
  *tile_rows = plan.bm, *tile_columns = plan.bn, *splits = plan.splits;
  return LSE_OK;
}

int lse_fp4_gemm(const struct lse_fp4_gemm_args* args, void* workspace, int64_t workspace_bytes, void* stream) {
  if (!args) return LSE_E_NULL;
  const lse_fp4_gemm_args& p = *args;
  if (const int st = check_sizes(p)) return st;
  if (p.K == 0) return LSE_E_RANGE;
  if (p.M == 0 || p.N == 0) return LSE_OK;
  const bool rows8 = p.x_scales != nullptr;
  if (!p.x || !p.codes || !p.scales || !p.y) return LSE_E_NULL;
  if (p.x_stride < p.K || p.y_stride < p.N || (rows8 && p.x_scales_stride < p.K / lse::kFp4Group)) return LSE_E_SHAPE;
  if (p.x_stride % (rows8 ? 16 : 8) || !aligned16(p.x) || !aligned16(p.codes) || !aligned16(p.scales) ||
      ((uintptr_t)p.y & 1) || (rows8 && (p.x_scales_stride % 4 || ((uintptr_t)p.x_scales & 3))))
    return LSE_E_ALIGN;
  // A workgroup's rows are addressed by 32-bit offsets from its first.
  if (p.x_stride > LSE_FP4_MAX_K || (rows8 && p.x_scales_stride > LSE_FP4_MAX_K)) return LSE_E_RANGE;
  lse::Fp4Args a{};
  a.x = p.x, a.ldx = p.x_stride;
  a.xs = (const uint8_t*)p.x_scales, a.lds = rows8 ? p.x_scales_stride : 0;
  a.codes = (const uint8_t*)p.codes, a.scales = (const uint8_t*)p.scales;
  a.y = (uint16_t*)p.y, a.ldy = p.y_stride;
  a.M = (int)p.M, a.N = (int)p.N, a.K = (int)p.K;
  a.nsteps = (int)lse::ceil_div(p.K, lse::kFp4Step), a.nchunks = (int)lse::ceil_div(p.K, lse::kFp4Chunk);
  a.nrb = (int)row_tiles(p);
  const lse::Fp4Plan plan = plan_of(p);
  if (plan.bm == 0) return lse::launch_fp4_stream(a, plan.bn / 16, rows8, p.glu != 0, (hipStream_t)stream);
  if (plan.splits > 1 && (!workspace || workspace_bytes < lse_fp4_gemm_workspace_bytes(args) || !aligned16(workspace)))
    return LSE_E_WORKSPACE;
  return lse::launch_fp4_tile(a, plan, rows8, p.glu != 0, (float*)workspace, (hipStream_t)stream);
}

}  // extern "C"
