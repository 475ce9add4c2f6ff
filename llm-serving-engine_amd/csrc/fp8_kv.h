// The 8-bit paged K/V cache: its layout, and the device code that its writer (fp8_kv.hip) and its readers
// (attn_fp8.hip) share.
//
// Codes are float8 e4m3 (largest value 448, steps of 1/8 of a power of two, down to 2^-9), and every group of
// 16 positions of a K/V head has one scale for k and one for v, powers of two held as e8m0 bytes (2^(b - 127),
// 255 = NaN). With a floating code a power of two loses nothing against any other scale, since the codes'
// relative precision is the same everywhere in their range, and it makes everything but the one rounding
// exact: code x scale is a bf16 value (the hardware's scaled conversion gives it in half an instruction a
// value; at the three scales below 2^-124 the smallest codes are rounded to bf16's subnormals, steps of 2^-133),
// and a group whose scale grows keeps its codes but for those that fall below the smallest normal.
//
// k and v: (blocks, H_KV, S, 16 D) bytes, S = block_size / 16 groups in a block; scales: (blocks, H_KV, S, 2).
// A group's bytes lie in the order in which the matrix cores take them as 16 contiguous bytes of a lane:
//  * k: element (slot, d) at ((slot / 4 * D / 64 + d / 64) * 4 + slot % 4) * 64 + d % 64: 16 dims of a key;
//  * v: element (slot, d) at 16 d + slot: one dim of all 16 keys, so no kernel has to transpose v.
#pragma once

#include "lse_common.h"

namespace lse {

constexpr int kKvGroup = 16;      // positions that share a scale
constexpr int kKvScaleNan = 255;  // e8m0
constexpr int kKvScaleTop = 247;  // 2^120: the largest scale of finite values, and the first that some codes make infinite

struct Fp8Pool {
  uint8_t *k, *v, *scales;
  int64_t sb, ss;  // bytes from a block to the next in k and v, and in scales
  int blocks, per;  // blocks of the pool, groups of a block
};

// The e8m0 byte of the smallest power of two s >= 2^-126 with amax <= 448 s (amax finite): 448 = 1.75 x 2^8,
// so one more than amax's exponent - 8 where its mantissa is above 1.75.
__device__ __forceinline__ int kv_scale_byte(float amax) {
  return max((int)((__builtin_bit_cast(uint32_t, amax) + 0x1fffffu) >> 23) - 8, 1);
}

// 2^(byte - 127) and its inverse, bytes 1 .. 254.
__device__ __forceinline__ float kv_scale(int byte) {
  return __builtin_bit_cast(float, (uint32_t)byte << 23);
}
__device__ __forceinline__ float kv_scale_inverse(int byte) {
  return __builtin_bit_cast(float, byte < 254 ? (uint32_t)(254 - byte) << 23 : 0x00400000u);
}

// Eight codes to bf16, times a power of two; exact but for bf16's subnormals (v_cvt_scalef32_pk_bf16_fp8: of `scale`
// it takes the exponent field as an e8m0 byte, so kv_scale of bytes 0 and 255, 2^-127 and NaN, serves too).
__device__ __forceinline__ bf16x8 kv_decode8(uint32_t lo, uint32_t hi, float scale) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Four fp32 values to codes, round to nearest even; infinity and NaN become NaN.
__device__ __forceinline__ uint32_t kv_encode4(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

// Four codes of values below 2^128 at a scale from kKvScaleTop on: those rounded up to 2^128, infinity in bf16, become
// the largest code below it, less than 2^-4 of the value away (240 for 255.99 at 2^120). NaN stays.
__device__ __forceinline__ uint32_t kv_keep_finite4(uint32_t w, int byte) {
  const uint32_t most = 8 * (262 - byte) - 1;  // 2^(255 - byte) is code 8 (262 - byte)
  uint32_t out = 0;
#pragma unroll
  for (int i = 0; i < 32; i += 8) {
    const uint32_t c = w >> i & 0x7f;
    out |= (c == 0x7f ? c : min(c, most)) << i;
  }
  return out | (w & 0x80808080u);
}

// Four codes times `ratio` (a power of two up to 1), as codes.
__device__ __forceinline__ uint32_t kv_requantize4(uint32_t w, float ratio) {
  return kv_encode4(__builtin_amdgcn_cvt_f32_fp8((int)w, 0) * ratio,
                    __builtin_amdgcn_cvt_f32_fp8((int)w, 1) * ratio,
                    __builtin_amdgcn_cvt_f32_fp8((int)w, 2) * ratio,
                    __builtin_amdgcn_cvt_f32_fp8((int)w, 3) * ratio);
}

// Sum over the lanes up to and including each.
__device__ __forceinline__ int kv_wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast 15, 31
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
  return v;
}

}  // namespace lse
