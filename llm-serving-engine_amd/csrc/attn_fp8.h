// Arguments and helpers shared by the two attention kernels over the 8-bit paged K/V cache (attn_fp8_stream.h: decode
// rows and short chunks, attn_fp8_tile.h: prompts and longer chunks; attn_fp8.hip launches them).
#pragma once

#include "attention.h"
#include "fp8_kv.h"

namespace lse {

struct Fp8AttnArgs {
  const uint16_t* q;  // bf16, element (h, t, d) at h * sq_h + t * sq_t + d
  int64_t sq_h, sq_t;
  Fp8Pool pool;
  const int32_t* block_table;  // (entries, max_blocks), row stride sbt
  int64_t sbt;
  const int32_t *context_len, *query_offset, *q_start, *q_len;
  uint16_t* o;  // bf16, same indexing as q with strides so_h, so_t
  int64_t so_h, so_t;
  int entries, HKV, G, tokens;
  int max_ctx;       // positions that the table has room for
  int max_q_len;
  int tiled;         // the row-tiled kernel takes the long entries
  int tq;            // query tokens per tile: floor(16 / G)
  int slots;         // units of a split launch (f8_unit); 0: keys are not split
  int sorted;        // entries are taken in descending order of context length...
  int first_round;   // ...and, where > 0, those from this rank on in ascending order
  float scale_log2;  // softmax scale x log2(e)
  float* ws_o;       // split launch: the units' O [slots][HKV][16 rows][D], fp32
  float* ws_ml;      // split launch: their max and sum [slots][HKV][16 rows][2]
  int tile_blocks;   // workgroups of the row-tiled kernel, which come first
  int tile_parts;    // parts its items may be cut into
  float* ws_tile_o;  // their O [items][parts][HKV][128 rows][D], fp32
  float* ws_tile_ml;  // their max and sum [items][parts][HKV][128 rows][2]
};

// In a call that is tiled (fp8_attn_tiled, attn_fp8.hip) the row-tiled kernel takes the entries of 128 query rows per
// K/V head or more, the key-streaming kernel the others; otherwise the latter takes all.
constexpr int kF8LongRows = 128;
__host__ __device__ inline bool f8_is_long(int64_t q_len, int G) { return q_len * G >= kF8LongRows; }

__device__ __forceinline__ int f8_wave_total(int v) { return __builtin_amdgcn_readlane(kv_wave_scan(v), 63); }

// The keys [0, end) that an entry's first `tokens` rows may see.
__device__ __forceinline__ int f8_end(const Fp8AttnArgs& a, int qo, int ctx, int tokens) {
  return max(min((int)min((int64_t)qo + tokens, (int64_t)ctx), a.max_ctx), 0);
}

constexpr float kNegInf = -__builtin_huge_valf();

}  // namespace lse
