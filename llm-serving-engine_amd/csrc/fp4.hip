// The C entry points of the products with 4-bit weights: argument checks, and which kernel a call takes.
#include "fp4.h"

namespace {

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
constexpr int64_t kMax31 = 2147483647;

int64_t row_tiles(const lse_fp4_gemm_args& p) { return (p.glu ? 2 : 1) * lse::ceil_div(p.N, 16); }

// Which kernel a call takes, from its sizes alone.
lse::Fp4Plan plan_of(const lse_fp4_gemm_args& p) {
  const int64_t nrb = row_tiles(p), chunks = lse::ceil_div(p.K, lse::kFp4Chunk);
  lse::Fp4Plan plan{0, 0, 1, (int)chunks};
  if (p.M <= 64) return plan;
  auto blocks = [&](int bm, int bn) { return lse::ceil_div(p.M, bm) * lse::ceil_div(nrb, bn / 16); };
  if (blocks(256, 256) >= 192) {
    plan.bm = plan.bn = 256;
  } else if (blocks(256, 256) >= 96 && chunks >= 16) {
    plan.bm = plan.bn = 256, plan.chunks = (int)lse::ceil_div(chunks, 2), plan.splits = 2;
  } else {
    plan.bm = 64, plan.bn = 128;
  }
  return plan;
}

}  // namespace

extern "C" {

int64_t lse_fp4_gemm_workspace_bytes(const struct lse_fp4_gemm_args* args) {
  if (!args || args->M < 0 || args->N < 0 || args->K < 0 || args->M > kMax31 || args->N > kMax31 - 64 ||
      args->K > LSE_FP4_MAX_K || args->K % lse::kFp4Group)
    return -1;
  if (args->M == 0 || args->N == 0 || args->K == 0) return 0;
  const int64_t nrb = row_tiles(*args);
  const lse::Fp4Plan plan = plan_of(*args);
  return plan.splits > 1 ? plan.splits * args->M * 16 * nrb * 4 : 0;
}

int lse_fp4_gemm(const struct lse_fp4_gemm_args* args, void* workspace, int64_t workspace_bytes, void* stream) {
  if (!args) return LSE_E_NULL;
  const lse_fp4_gemm_args& p = *args;
  if (p.M < 0 || p.N < 0 || p.K < 0 || p.M > kMax31 || p.N > kMax31 - 64 || (p.glu != 0 && p.glu != 1))
    return LSE_E_SHAPE;
  if (p.K % lse::kFp4Group) return LSE_E_ALIGN;
  if (p.K == 0 || p.K > LSE_FP4_MAX_K) return LSE_E_RANGE;
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
  if (plan.bm == 0) return lse::launch_fp4_stream(a, rows8, p.glu != 0, (hipStream_t)stream);
  if (plan.splits > 1 && (!workspace || workspace_bytes < lse_fp4_gemm_workspace_bytes(args) || !aligned16(workspace)))
    return LSE_E_WORKSPACE;
  return lse::launch_fp4_tile(a, plan, rows8, p.glu != 0, (float*)workspace, (hipStream_t)stream);
}

}  // extern "C"
