// The C entry points of the products with 4-bit weights: argument checks, and which kernel a call takes.
#include "fp4.h"

namespace {

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
constexpr int64_t kMax31 = 2147483647;

}  // namespace

extern "C" {

int64_t lse_fp4_gemm_workspace_bytes(const struct lse_fp4_gemm_args* args) {
  if (!args || args->M < 0 || args->N < 0 || args->K < 0 || args->M > kMax31 || args->N > kMax31 - 64 ||
      args->K > LSE_FP4_MAX_K || args->K % lse::kFp4Group)
    return -1;
  return 0;
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
      ((uintptr_t)p.y & 1))
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
  a.nrb = (int)(p.glu ? 2 * lse::ceil_div(p.N, 16) : lse::ceil_div(p.N, 16));
  a.xs_dwords = rows8 && p.K % lse::kFp4Step == 0 && a.lds % 4 == 0 && ((uintptr_t)a.xs & 3) == 0;
  return lse::launch_fp4_stream(a, rows8, p.glu != 0, (hipStream_t)stream);
}

}  // extern "C"
