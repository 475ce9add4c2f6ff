// What makes the operands of the products with 4-bit weights (layouts and formats: fp4.h):
//  * fp4_quantize_kernel, fp4_pack_kernel: a weight's codes and scales row by row, and their tiles (load time);
//  * fp8_rows_kernel: bf16 rows to 8 bits, scales of 32 values;
//  * add_rmsnorm_fp8_kernel: the residual's addition, the RMSNorm after it and its output in 8 bits, one launch.
#include <algorithm>

#include "fp4.h"
#include "fp8_kv.h"

namespace lse {

// ---- weights (load time) -----------------------------------------------------------------------------------------

// One e2m1 code of v = weight / scale: the nearest value, ties to the even code; past 6 (which only a scale clamped
// from above could give) 6; NaN 0. The thresholds between neighbours are exact in fp32.
__device__ __forceinline__ uint32_t fp4_code(float v) {
  const float a = fabsf(v);
  const uint32_t c = (a > 0.25f) + (a >= 0.75f) + (a > 1.25f) + (a >= 1.75f) + (a > 2.5f) + (a >= 3.5f) + (a > 5.0f);
  return c && v < 0.0f ? c | 8 : c;
}

// 2^126, the largest scale of finite values: its codes 6 and 7 stand for 2^128 and more.
constexpr int kFp4ScaleTop = 253;

// One thread a group of 32 of one row: w fp32, stride ldw. A group with a value that is not finite gets the scale
// 255 (NaN): e2m1 has no code for it. Finite weights stay finite. 14336 x 4096: 52 us a call, 5.1 TB/s.
__global__ void __launch_bounds__(256)
fp4_quantize_kernel(const float* w, int64_t ldw, uint8_t* codes, uint8_t* scales, int64_t groups, int per_row) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= groups) return;
  const int64_t n = at / per_row;
  const float4* src = reinterpret_cast<const float4*>(w + n * ldw + (at - n * per_row) * kFp4Group);
  float v[kFp4Group];
  float amax = 0.0f;
  bool finite = true;
#pragma unroll
  for (int i = 0; i < kFp4Group / 4; ++i) {
    const float4 q = src[i];
    v[4 * i] = q.x, v[4 * i + 1] = q.y, v[4 * i + 2] = q.z, v[4 * i + 3] = q.w;
  }
#pragma unroll
  for (int i = 0; i < kFp4Group; ++i) {
    amax = fmaxf(amax, fabsf(v[i]));
    finite &= (__builtin_bit_cast(uint32_t, v[i]) & 0x7fffffffu) < 0x7f800000u;
  }
  const int byte = finite ? fp4_scale_byte(amax) : 255;
  const float inv = finite ? e8m0_inverse(byte) : 0.0f;
  uint32_t out[4] = {0, 0, 0, 0};
  if (finite) {
#pragma unroll
    for (int i = 0; i < kFp4Group; ++i) {
      uint32_t c = fp4_code(v[i] * inv);
      if (byte == kFp4ScaleTop && (c & 7) > 5) c = (c & 8) | 5;
      out[i / 8] |= c << (4 * (i % 8));
    }
  }
  *reinterpret_cast<uint4*>(codes + at * (kFp4Group / 2)) = make_uint4(out[0], out[1], out[2], out[3]);
  scales[at] = (uint8_t)byte;
}

// One thread 16 bytes of a code tile (a group) and one scale byte of a scale tile; threads past the code tiles' K fill
// the scale tiles up. codes (rows, K / 2), scales (rows, K / 32); glu: rows = 2 I. 14336 x 4096: 14 us a call.
__global__ void __launch_bounds__(256)
fp4_pack_kernel(const uint8_t* codes, const uint8_t* scales, uint8_t* out_codes, uint8_t* out_scales, int64_t total,
                int rows, int K, int nsteps, int nchunks, int glu) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;  // (rb, step of the chunks, lane)
  if (at >= total) return;
  const int lane = at & 63, j = (int)((at >> 6) % (4 * nchunks)), rb = (int)((at >> 6) / (4 * nchunks));
  const int half = rows / 2;
  const int in = 16 * (glu ? rb >> 1 : rb) + (lane & 15);  // row within its weight
  const bool there = in < (glu ? half : rows);
  const int64_t row = glu ? (int64_t)(rb & 1) * half + in : in;
  const int group = 4 * j + (lane >> 4), per = K / kFp4Group;
  const bool ok = there && group < per;
  if (j < nsteps) {
    uint4 v = make_uint4(0, 0, 0, 0);
    if (ok) v = *reinterpret_cast<const uint4*>(codes + (row * per + group) * 16);
    *reinterpret_cast<uint4*>(out_codes + ((int64_t)rb * nsteps + j) * kFp4TileBytes + 16 * lane) = v;
  }
  out_scales[((int64_t)rb * nchunks + (j >> 2)) * kFp4ScaleBytes + 4 * lane + (j & 3)] =
      ok ? scales[row * per + group] : 127;
}

// ---- rows in 8 bits ----------------------------------------------------------------------------------------------

// Eight values of a group, whose other three parts the lanes l ^ 1, l ^ 2, l ^ 3 hold: their codes, and the group's
// scale byte. Not finite: NaN; the scale goes by the finite ones.
__device__ __forceinline__ uint2 fp8_encode8(const float (&v)[8], int& byte) {
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = fmaxf(amax, finite_abs(v[i]));
  amax = fmaxf(amax, __shfl_xor(amax, 1, 64));
  amax = fmaxf(amax, __shfl_xor(amax, 2, 64));
  byte = fp8_scale_byte(amax);
  const float inv = e8m0_inverse(byte);
  uint2 c = make_uint2(kv_encode4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv),
                       kv_encode4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv));
  if (byte >= kKvScaleTop) c.x = kv_keep_finite4(c.x, byte), c.y = kv_keep_finite4(c.y, byte);
  return c;
}

__device__ __forceinline__ void bf16x8_to_f32(uint4 q, float (&v)[8]) {
  const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __builtin_bit_cast(float, u[i] << 16);
    v[2 * i + 1] = __builtin_bit_cast(float, u[i] & 0xffff0000u);
  }
}

// One thread eight values of a row, four threads a group, whose largest value they share by shuffles. Bound by HBM, 3
// bytes a value: 2048 rows of 14336 15.7 us, 5.6 TB/s (some of it from the cache behind L2); 64 of 4096 2.7, a launch.
// codes (M, K) contiguous, scales (M, K / 32) of row stride lds.
__global__ void __launch_bounds__(256)
fp8_rows_kernel(const uint16_t* x, int64_t ldx, uint8_t* codes, uint8_t* scales, int64_t lds, int64_t total,
                int per_row) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= total) return;  // whole groups: total and 256 are multiples of 4
  const int64_t m = at / per_row;
  float v[8];
  bf16x8_to_f32(*reinterpret_cast<const uint4*>(x + m * ldx + 8 * (at - m * per_row)), v);
  int byte;
  *reinterpret_cast<uint2*>(codes + 8 * at) = fp8_encode8(v, byte);
  if ((at & 3) == 0) scales[m * lds + ((at - m * per_row) >> 2)] = (uint8_t)byte;
}

constexpr int kNormFp8Threads = 512;

typedef unsigned u32x2_t __attribute__((ext_vector_type(2)));

// 16-byte loads, and 16- or 8-byte stores, of what a call reads and writes once.
template <bool STREAM>
__device__ __forceinline__ uint4 load16_once(const void* p) {
  return STREAM ? load16_stream(p) : *static_cast<const uint4*>(p);
}
template <bool STREAM, typename V>
__device__ __forceinline__ void store_once(void* p, V v) {
  if constexpr (STREAM)
    __builtin_nontemporal_store(v, static_cast<V*>(p));
  else
    *static_cast<V*>(p) = v;
}

// One workgroup per row, of as many waves as its first 4096 values keep busy, thread t holding elements 8 t + 4096 i
// (i < NV): s = bf16(x + res) (or x), n = bf16(w * bf16(fp32(s * r))), r = 1 / sqrt(mean(s^2) + eps), the roundings of
// LlamaRMSNorm (modeling_llama.py:62-67), then n's codes and scales. A code has two or three bits after its first, so one
// bf16 step too far, which an r of 24 bits gives now and then, can become a quarter or an eighth of the value: the sum of
// squares (of exact squares, each thread's in order, then a fixed tree) and r are held in 64 bits and s r is the nearest
// fp32, for 5 % of the time. `sum` may be x or res: a thread reads all of its elements before it writes any.
// Bound by HBM, 7 bytes a value: 4160 rows of 4096 25.5 us, 4.7 TB/s, a copy's rate; 2048 of 14336 42.8; 33 of 4096 4.8, a
// launch. Waves that would hold no element are not started (4160 of 1024: 16.9 -> 9.7 us). STREAM, for calls that move a
// good part of the 256 MB behind L2, keeps from there what is not read again (with r in 32 bits: 2048 of 14336 46.0 ->
// 42.0, 4160 of 4096 29.9 -> 24.3 after other work and 24.1 by itself either way); smaller calls are better off without
// (3200 of 4096 17.5 against 19.4, 2560 14.9 against 16.6).
template <int NV, bool STREAM>
__global__ void __launch_bounds__(kNormFp8Threads)
add_rmsnorm_fp8_kernel(const uint16_t* x, int64_t ldx, const uint16_t* res, int64_t ldr, const uint16_t* w, double eps,
                       uint16_t* sum, uint8_t* codes, uint8_t* scales, int64_t lds, int K, double inv_k) {
  __shared__ double red[kNormFp8Threads / 64];
  const int64_t m = blockIdx.x;
  float s[NV][8], g[NV][8];
  double ss = 0.0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int k = 8 * (threadIdx.x + kNormFp8Threads * i);
    const uint4 zero = make_uint4(0, 0, 0, 0);
    bf16x8_to_f32(k < K ? load16_once<STREAM>(x + m * ldx + k) : zero, s[i]);
    bf16x8_to_f32(k < K ? *reinterpret_cast<const uint4*>(w + k) : zero, g[i]);
    if (res) {
      float r[8];
      bf16x8_to_f32(k < K ? load16_once<STREAM>(res + m * ldr + k) : zero, r);
#pragma unroll
      for (int j = 0; j < 8; ++j) s[i][j] = bf16_to_f32(f32_to_bf16(s[i][j] + r[j]));
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = __builtin_fma((double)s[i][j], (double)s[i][j], ss);
  }
  if (sum) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int k = 8 * (threadIdx.x + kNormFp8Threads * i);
      if (k < K)
        store_once<STREAM>(sum + m * K + k, u32x4{pack_bf16x2(s[i][0], s[i][1]), pack_bf16x2(s[i][2], s[i][3]),
                                                  pack_bf16x2(s[i][4], s[i][5]), pack_bf16x2(s[i][6], s[i][7])});
    }
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) ss += __shfl_xor(ss, off, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = ss;
  __syncthreads();
  double total = red[0];
#pragma unroll
  for (int i = 1; i < kNormFp8Threads / 64; ++i)
    if (64 * i < blockDim.x) total += red[i];
  const double t = total * inv_k + eps;
  double r;
  const bool narrow = t > 0x1p-100 && t < 0x1p100;
  if (narrow) {  // one step of Newton's in 64 bits from 32 gives 40
    const double y = __builtin_amdgcn_rsqf((float)t);
    r = __builtin_fma(y * 0.5, __builtin_fma(-t * y, y, 1.0), y);
  } else {
    r = 1.0 / __builtin_sqrt(t);
  }
  // r = rh + rl with 16 bits in rh: s rh is exact, and s r to the nearest fp32 by one fma. Where fp32 holds r badly or not
  // at all (rows below 2^-126, or of the largest values), in 64 bits.
  const float rh = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, (float)r) & 0xffffff00u);
  const float rl = (float)(r - rh);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int k = 8 * (threadIdx.x + kNormFp8Threads * i);
    float n[8];
    if (narrow) {
#pragma unroll
      for (int j = 0; j < 8; ++j) n[j] = __builtin_fmaf(s[i][j], rl, s[i][j] * rh);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float v = s[i][j];
        asm volatile("" : "+v"(v));  // or the compiler keeps every s in 64 bits from the sum of squares to here
        n[j] = (float)(v * r);
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) n[j] = bf16_to_f32(f32_to_bf16(g[i][j] * bf16_to_f32(f32_to_bf16(n[j]))));
    int byte;
    const uint2 c = fp8_encode8(n, byte);  // every lane: K is a multiple of 32, so groups are whole
    if (k < K) {
      store_once<STREAM>(codes + m * K + k, u32x2_t{c.x, c.y});
      if ((threadIdx.x & 3) == 0) scales[m * lds + k / kFp4Group] = (uint8_t)byte;
    }
  }
}

}  // namespace lse

namespace {

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
constexpr int64_t kMax31 = 2147483647;

}  // namespace

extern "C" {

int64_t lse_fp4_codes_bytes(int64_t N, int64_t K, int64_t glu) {
  if (N < 0 || K < 0 || (glu != 0 && glu != 1) || (glu && N % 2) || K % lse::kFp4Group || N > kMax31 - 64 ||
      K > LSE_FP4_MAX_K)
    return -1;
  const int64_t tiles = glu ? 2 * lse::ceil_div(N / 2, 16) : lse::ceil_div(N, 16);
  return tiles * lse::ceil_div(K, lse::kFp4Step) * lse::kFp4TileBytes;
}

int64_t lse_fp4_scales_bytes(int64_t N, int64_t K, int64_t glu) {
  if (lse_fp4_codes_bytes(N, K, glu) < 0) return -1;
  const int64_t tiles = glu ? 2 * lse::ceil_div(N / 2, 16) : lse::ceil_div(N, 16);
  return tiles * lse::ceil_div(K, lse::kFp4Chunk) * lse::kFp4ScaleBytes;
}

int lse_quantize_weight_fp4(const float* w, int64_t ldw, void* codes, void* scales, int64_t N, int64_t K,
                            void* stream) {
  if (N < 0 || K < 0 || ldw < K || N > kMax31) return LSE_E_SHAPE;
  if (K % lse::kFp4Group || ldw % 4) return LSE_E_ALIGN;
  if (K > LSE_FP4_MAX_K) return LSE_E_RANGE;
  if (N == 0 || K == 0) return LSE_OK;
  if (!w || !codes || !scales) return LSE_E_NULL;
  if (!aligned16(w) || !aligned16(codes)) return LSE_E_ALIGN;
  const int64_t groups = N * (K / lse::kFp4Group), blocks = lse::ceil_div(groups, 256);
  if (blocks > kMax31) return LSE_E_RANGE;
  hipLaunchKernelGGL(lse::fp4_quantize_kernel, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, w, ldw,
                     (uint8_t*)codes, (uint8_t*)scales, groups, (int)(K / lse::kFp4Group));
  return lse::launch_status();
}

int lse_pack_fp4(const void* codes, const void* scales, void* out_codes, void* out_scales, int64_t N, int64_t K,
                 int64_t glu, void* stream) {
  if (N < 0 || K < 0 || (glu != 0 && glu != 1) || (glu && N % 2) || N > kMax31 - 64) return LSE_E_SHAPE;
  if (K % lse::kFp4Group) return LSE_E_ALIGN;
  if (K > LSE_FP4_MAX_K) return LSE_E_RANGE;
  if (N == 0 || K == 0) return LSE_OK;
  if (!codes || !scales || !out_codes || !out_scales) return LSE_E_NULL;
  if (!aligned16(codes) || !aligned16(out_codes)) return LSE_E_ALIGN;
  const int64_t tiles = glu ? 2 * lse::ceil_div(N / 2, 16) : lse::ceil_div(N, 16);
  const int64_t nchunks = lse::ceil_div(K, lse::kFp4Chunk), total = tiles * 4 * nchunks * 64;
  const int64_t blocks = lse::ceil_div(total, 256);
  if (blocks > kMax31) return LSE_E_RANGE;
  hipLaunchKernelGGL(lse::fp4_pack_kernel, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream,
                     (const uint8_t*)codes, (const uint8_t*)scales, (uint8_t*)out_codes, (uint8_t*)out_scales, total,
                     (int)N, (int)K, (int)lse::ceil_div(K, lse::kFp4Step), (int)nchunks, (int)glu);
  return lse::launch_status();
}

int lse_quantize_rows_fp8(const void* x, int64_t ldx, void* codes, void* scales, int64_t scales_stride, int64_t M,
                          int64_t K, void* stream) {
  if (M < 0 || K < 0 || ldx < K || M > kMax31 || scales_stride < K / lse::kFp4Group) return LSE_E_SHAPE;
  if (K % lse::kFp4Group || ldx % 8) return LSE_E_ALIGN;
  if (K > LSE_FP4_MAX_K) return LSE_E_RANGE;
  if (M == 0 || K == 0) return LSE_OK;
  if (!x || !codes || !scales) return LSE_E_NULL;
  if (!aligned16(x) || !aligned16(codes)) return LSE_E_ALIGN;
  const int64_t total = M * (K / 8), blocks = lse::ceil_div(total, 256);
  if (blocks > kMax31) return LSE_E_RANGE;
  hipLaunchKernelGGL(lse::fp8_rows_kernel, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream,
                     (const uint16_t*)x, ldx, (uint8_t*)codes, (uint8_t*)scales, scales_stride, total, (int)(K / 8));
  return lse::launch_status();
}

int lse_add_rmsnorm_fp8(const struct lse_add_rmsnorm_fp8_args* args, void* stream) {
  if (!args) return LSE_E_NULL;
  const lse_add_rmsnorm_fp8_args& x = *args;
  if (x.M < 0 || x.K < 0 || x.M > kMax31) return LSE_E_SHAPE;
  if (x.K % lse::kFp4Group) return LSE_E_ALIGN;
  if (x.K > LSE_NORM_MAX_K) return LSE_E_RANGE;
  if (x.M == 0 || x.K == 0) return LSE_OK;
  if (!x.x || !x.weight || !x.codes || !x.scales) return LSE_E_NULL;
  if (x.x_stride < x.K || (x.residual && x.residual_stride < x.K) ||
      x.scales_stride < x.K / lse::kFp4Group || !(x.eps >= 0.0))
    return LSE_E_SHAPE;
  if (x.x_stride % 8 || (x.residual && x.residual_stride % 8) || !aligned16(x.x) || !aligned16(x.residual) ||
      !aligned16(x.weight) || !aligned16(x.sum) || !aligned16(x.codes))
    return LSE_E_ALIGN;
  const int64_t waves = std::min<int64_t>(lse::ceil_div(x.K, 512), lse::kNormFp8Threads / 64);
  const dim3 grid((unsigned)x.M), wg((unsigned)(64 * waves));
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, wg, 0, (hipStream_t)stream, (const uint16_t*)x.x, x.x_stride,
                       (const uint16_t*)x.residual, x.residual_stride, (const uint16_t*)x.weight, x.eps,
                       (uint16_t*)x.sum, (uint8_t*)x.codes, (uint8_t*)x.scales, x.scales_stride, (int)x.K,
                       1.0 / (double)x.K);
  };
  auto width = [&](auto nv) {
    constexpr int NV = decltype(nv)::value;
    if (x.M * x.K * 7 > (96 << 20))
      go(lse::add_rmsnorm_fp8_kernel<NV, true>);
    else
      go(lse::add_rmsnorm_fp8_kernel<NV, false>);
  };
  if (x.K <= 8 * lse::kNormFp8Threads)
    width(std::integral_constant<int, 1>{});
  else if (x.K <= 16 * lse::kNormFp8Threads)
    width(std::integral_constant<int, 2>{});
  else
    width(std::integral_constant<int, 4>{});
  return lse::launch_status();
}

}  // extern "C"
