// 4-bit weights (float4 e2m1 codes, a power of two for every 32 k of a row) and rows held in 8 bits (float8 e4m3
// codes, likewise): their layouts, and the device code that their makers (fp4_quant.hip) and the products over them
// (fp4_stream.hip, fp4_tile.hip) share.
//
// e2m1: a sign and the magnitudes 0, 0.5, 1, 1.5, 2, 3, 4, 6. Scales are e8m0 bytes, 2^(b - 127), 255 = NaN. With a
// power of two a weight code x scale is a bf16 value, which the scaled conversion gives in half an instruction a
// weight, and the scaled 8-bit matrix instruction takes codes of both operands with their scale bytes as they are:
// no product needs a scale of its own.
//
// A weight (N, K) lies in tiles of 16 rows x 128 k, 1 KB each, tile (rb, j) at ((rb * nsteps) + j) * 1024 with
// nsteps = ceil(K / 128): byte 16 l + i holds row 16 rb + l % 16 at k = 128 j + 32 (l / 16) + 2 i in its low half
// and the k after it in its high half, zeros past N and K. Lane l's 16 bytes are its operand of the 16x16x128
// matrix instruction, and four operands (a dword each) of the 16x16x32 one. The scales lie in tiles of 16 rows x
// 512 k, 256 bytes each, tile (rb, c) at ((rb * nchunks) + c) * 256: byte 4 l + t belongs to row 16 rb + l % 16 and
// the 32 k from 512 c + 128 t + 32 (l / 16) on, so that lane l's dword has its scales of four steps, by the byte
// that the matrix instruction's operand selector names; 127 (1) past N and K.
// Two stacked weights (2 I, K), an MLP's gate and up, take turns by row tiles: tile 2 t holds gate rows 16 t .. and
// tile 2 t + 1 the same rows of up, so a kernel that holds an even pair of row tiles holds matching rows.
#pragma once

#include "lse_common.h"

namespace lse {

constexpr int kFp4Group = 32;       // weights of a row, or values of a row in 8 bits, that share a scale
constexpr int kFp4Step = 128;       // k of a code tile
constexpr int kFp4Chunk = 512;      // k of a scale tile: four steps
constexpr int kFp4TileBytes = 1024;
constexpr int kFp4ScaleBytes = 256;

typedef int i32x8 __attribute__((ext_vector_type(8)));

// f(0), f(1), ... f(N - 1), each index a constant.
template <typename F, int... I>
__device__ __forceinline__ void unroll_seq(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void unroll(F&& f) {
  unroll_seq(f, std::make_integer_sequence<int, N>{});
}

// Eight weights of a dword times 2^(scale's exponent field - 127), in k order: exact from bf16's subnormals up, infinite
// from 2^128 on, and NaN, codes of zero too, where the field is 255 (v_cvt_scalef32_pk_bf16_fp4;
// tests/test_gpu_fp4_codes.py takes every code and scale through the products).
__device__ __forceinline__ bf16x8 fp4_decode8(uint32_t w, float scale) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Byte t of a scale dword as a float of that exponent field. The conversion reads the field alone and as an e8m0 byte: 0
// is 2^-127, where the float is zero, and 255 NaN, where it is infinity.
__device__ __forceinline__ float fp4_scale(uint32_t dword, int t) {
  return __builtin_bit_cast(float, (dword >> (8 * t) & 0xff) << 23);
}

// D(16x16 fp32) += A(16 rows x 128 4-bit weights) . B(128 x 16 8-bit row values), both scaled by a byte per 32 k.
// Lane l supplies weight row l % 16 at k = 32 (l / 16) .. + 31 and row l % 16 of the other operand at k =
// 16 (l / 16) .. + 15 (lo) and 64 + 16 (l / 16) .. + 15 (hi); byte T of ws and byte 0 of xs scale the 32 k from
// 32 (l / 16) on. D as the 16x16x32 instruction's. The instruction cuts the products of eight consecutive k off 13
// bits below the largest of them (toward zero; measured) and adds the rest in fp32: 2^-14 of the result in the mean
// of random ones, far below the steps of 2^-4 that the 8-bit operand was rounded to. One bf16 output in a hundred goes to
// its neighbour by it (64 x 4096 x 4096: 1.6493e-3 off the 64-bit product in the norm, its nearest bf16 values 1.6492e-3).
template <int T>
__device__ __forceinline__ f32x4 mfma_fp4_fp8(uint4 w, uint32_t ws, uint4 lo, uint4 hi, uint32_t xs, f32x4 c) {
  const i32x8 a = {(int)w.x, (int)w.y, (int)w.z, (int)w.w, 0, 0, 0, 0};
  const i32x8 b = {(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4, 0, T, (int)ws, 0, (int)xs);
}

// One dword a lane to LDS byte address base + IMM (+ 4 l for lane l), as dma16_lds.
template <int IMM>
__device__ __forceinline__ void dma4_lds(u32x4 r, uint32_t base, uint32_t offset) {
  asm volatile(
      "s_add_u32 m0, %0, %3\n\t"
      "s_nop 0\n\t"
      "buffer_load_dword %1, %2, 0 offen lds"
      :
      : "s"(base), "v"(offset), "s"(r), "i"(IMM)
      : "memory", "scc", "m0");
}

// Rows of one step in LDS: 256 (bf16) or 128 (codes) bytes, their 16-byte chunk c at c ^ fp4_swz(row), rows in 16s. A
// wave reads a chunk of 16 rows, lane l of row l % 16 chunk 4 (l / 16) + i (bf16) or 4 i + l / 16 (codes), and the LDS
// serves a 16-byte read as four groups of 16 lanes: 0-3, 12-15 and 20-27, 4-11, 16-19 and 28-31, and the same 32 lanes
// on. So rows {0-3, 12-15} of one l / 16 meet rows {4-11} of its neighbour, and either set has to fill whole pairs of
// the places that the neighbour's chunk changes (by 4, or 1). With row & 15, or the other kernels' spread of 128-byte
// rows, a read cost 4 conflict cycles more (SQ_LDS_BANK_CONFLICT).
template <bool A8>
__host__ __device__ constexpr int fp4_swz(int row) {
  if (!A8) return (row & 15) ^ ((row & 4) << 1);
  const int q = row >> 1 & 7;
  return ((q >> 2 ^ q >> 1) & 1) << 2 | (q >> 2) << 1 | (q & 1);
}

// The e8m0 byte of the smallest power of two s >= 2^-126 with amax <= most * s (amax finite), most = 448 or 6:
// (1 + m) 2^p, one more than amax's exponent - p where its mantissa is above m.
__device__ __forceinline__ int fp8_scale_byte(float amax) {  // 1.75 x 2^8
  return max((int)((__builtin_bit_cast(uint32_t, amax) + 0x1fffffu) >> 23) - 8, 1);
}
__device__ __forceinline__ int fp4_scale_byte(float amax) {  // 1.5 x 2^2
  return max((int)((__builtin_bit_cast(uint32_t, amax) + 0x3fffffu) >> 23) - 2, 1);
}
// 2^(127 - byte), bytes 1 .. 254.
__device__ __forceinline__ float e8m0_inverse(int byte) {
  return __builtin_bit_cast(float, byte < 254 ? (uint32_t)(254 - byte) << 23 : 0x00400000u);
}

// |v| where it is finite, 0 where it is not: what a group's scale goes by.
__device__ __forceinline__ float finite_abs(float v) {
  const uint32_t b = __builtin_bit_cast(uint32_t, v) & 0x7fffffffu;
  return b < 0x7f800000u ? __builtin_bit_cast(float, b) : 0.0f;
}

// One product's arguments, as the launchers take them.
struct Fp4Args {
  const void* x;         // bf16 rows, or e4m3 codes; stride ldx elements
  int64_t ldx;
  const uint8_t* xs;     // e8m0 (M, K / 32) of 8-bit rows, stride lds bytes
  int64_t lds;
  const uint8_t *codes, *scales;
  uint16_t* y;
  int64_t ldy;
  int M, N, K;           // N output columns (gate/up: I)
  int nsteps, nchunks;   // ceil(K / 128), ceil(K / 512)
  int nrb;               // row tiles of the weight
};

// How a call runs: bm 0: the streaming kernel, bn / 16 row tiles a workgroup; otherwise tiles of bm x bn, K in `splits`
// ranges of `chunks` chunks.
struct Fp4Plan {
  int bm, bn, splits, chunks;
};

struct Fp4Split {
  int mblocks, nblocks, splits, chunks;
  float* part;  // splits > 1: [splits][M][16 nrb] sums
};

int launch_fp4_stream(const Fp4Args& a, int rt, bool rows8, bool glu, hipStream_t stream);
int launch_fp4_tile(const Fp4Args& a, const Fp4Plan& plan, bool rows8, bool glu, float* part, hipStream_t stream);

}  // namespace lse
