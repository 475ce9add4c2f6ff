// Paged attention over the 8-bit K/V cache: launches, and what adds up the states of split keys. The kernels' bodies
// are in attn_fp8_stream.h and attn_fp8_tile.h; a call that may hold long entries runs both in one launch, so
// that the decode rows of a mixed batch, bound by HBM, stream beside its prompt chunks, bound by the matrix cores.
#include <algorithm>

#include "attn_fp8_stream.h"
#include "attn_fp8_tile.h"

namespace lse {

template <int D, bool NT, bool COUNT>
__global__ void __launch_bounds__(64 * kF8Waves, 2) attn_fp8_stream_kernel(Fp8AttnArgs a) {
  __shared__ __attribute__((aligned(16))) unsigned char lds[f8_stream_lds(D)];
  f8_stream<D, NT, COUNT>(a, blockIdx.x, lds);
}

template <int D>
__global__ void __launch_bounds__(64 * kF8Waves, 2) attn_fp8_mixed_kernel(Fp8AttnArgs a) {
  static_assert(kF8Waves == kF8TileWaves, "one workgroup size");
  __shared__ __attribute__((aligned(16))) unsigned char lds[std::max(f8_stream_lds(D), f8_tile_lds(D))];
  if ((int)blockIdx.x < a.tile_blocks)
    f8_tile<D>(a, blockIdx.x, lds);
  else
    f8_stream<D, false, true>(a, blockIdx.x - a.tile_blocks, lds);
}

// Adds the state (max m, sum l, unnormalised o) of further keys to (M, L, O), if `real`.
__device__ __forceinline__ void f8_add_state(float& M, float& L, float (&O)[4], float2 ml, float4 o, bool real) {
  const float m = real ? ml.x : kNegInf, mn = fmaxf(M, m), ref = mn == kNegInf ? 0.0f : mn;
  const float fa = exp2_fast(M - ref), fb = exp2_fast(m - ref);
  L = __builtin_fmaf(real ? ml.y : 0.0f, fb, L * fa);
  O[0] = __builtin_fmaf(real ? o.x : 0.0f, fb, O[0] * fa);
  O[1] = __builtin_fmaf(real ? o.y : 0.0f, fb, O[1] * fa);
  O[2] = __builtin_fmaf(real ? o.z : 0.0f, fb, O[2] * fa);
  O[3] = __builtin_fmaf(real ? o.w : 0.0f, fb, O[3] * fa);
  M = mn;
}

struct Fp8MergeGrid {
  int stream;    // workgroups of f8_merge_stream, which come first
  int pieces;    // workgroups of one query tile
  int by_entry;  // they go by entries, of one query tile each; otherwise by units, the first of each tile's
};

// The second kernel of calls whose keys are split. Bound by latency: a thread's loads, eight states at a time, do not
// wait for each other.
//
// f8_stream's ranges, a workgroup per query tile, K/V head and 64 (row, 4 dims) pieces: wave w adds up the states
// of ranges w, w + 4, ..., then the four are merged.
template <int D>
__device__ __forceinline__ void f8_merge_stream(const Fp8AttnArgs& a, const Fp8MergeGrid& g, int block) {
  __shared__ float obuf[kF8Waves][64][5];
  __shared__ float mbuf[kF8Waves][64], lbuf[kF8Waves][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int kvh = block % a.HKV, item = block / a.HKV / g.pieces;
  const F8Unit u = f8_unit(a, item, g.by_entry);
  if (u.e < 0 || u.parts <= 1 || u.part > 0) return;
  const int qt = u.qt;
  const int qlen = u.qlen, G = a.G;
  const int piece = block / a.HKV % g.pieces * 64 + lane, orow = piece / (D / 4), c4 = 4 * (piece % (D / 4));
  const int otok = orow / G, om = qt * a.tq + otok;
  const int64_t row = (int64_t)u.qs + om;
  const bool ok = orow < a.tq * G && om < qlen && row >= 0 && row < a.tokens;
  const int end_n = f8_end(a, u.qo, u.ctx, min(qlen, (qt + 1) * a.tq));
  const int n = max((int)((end_n + u.range - 1) / u.range), 1);  // ranges with keys of this tile
  float M = kNegInf, L = 0.0f, O[4] = {0, 0, 0, 0};
  if (ok) {
    for (int p0 = wave; p0 < n; p0 += 8 * kF8Waves) {
      float2 ml[8];
      float4 v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {  // past the last range the first one again, without weight
        const int p = p0 + kF8Waves * i < n ? p0 + kF8Waves * i : p0;
        const int64_t at = ((int64_t)(u.first + p * u.tiles + qt) * a.HKV + kvh) * 16 + orow;
        ml[i] = *reinterpret_cast<const float2*>(a.ws_ml + 2 * at);
        v[i] = *reinterpret_cast<const float4*>(a.ws_o + at * D + c4);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < 8; ++i) f8_add_state(M, L, O, ml[i], v[i], p0 + kF8Waves * i < n);
    }
  }
  mbuf[wave][lane] = M, lbuf[wave][lane] = L;
#pragma unroll
  for (int i = 0; i < 4; ++i) obuf[wave][lane][i] = O[i];
  __syncthreads();
  if (wave != 0 || !ok) return;
  float m[kF8Waves], l[kF8Waves], o[4] = {0, 0, 0, 0};
#pragma unroll
  for (int w = 0; w < kF8Waves; ++w) m[w] = mbuf[w][lane], l[w] = lbuf[w][lane];
  const WaveFactors f = f8_merge_factors(m, l);
  const float inv = f8_inverse(f.sum);
#pragma unroll
  for (int w = 0; w < kF8Waves; ++w)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = __builtin_fmaf(obuf[w][lane][i], f.f[w], o[i]);
  *reinterpret_cast<uint2*>(a.o + (int64_t)(kvh * G + orow - otok * G) * a.so_h + row * a.so_t + c4) =
      make_uint2(pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv));
}

// f8_tile's parts, a workgroup per item, K/V head and eighth of its (row, 4 dims) pieces (16 workgroups of half the
// work each: two us more for 288 parts). Two parts, the most common number, are loaded without the repeats that fill up
// eight: 15 -> 10 us.
constexpr int kF8TileMerges = 8;
template <int D>
__device__ __forceinline__ void f8_merge_tile(const Fp8AttnArgs& a, int block) {
  constexpr int kPieces = kF8TileRows * (D / 4) / kF8TileMerges;
  const int kvh = block % a.HKV, rank = block / a.HKV / kF8TileMerges;
  const F8Item item = f8_tile_item(a, rank);
  if (item.e < 0) return;
  const int G = a.G, qlen = item.qlen;
  const int end_n = f8_tile_end(a, item.qo, item.ctx, qlen, item.qt);
  const int parts = f8_tile_parts(a, (end_n + 63) / 64);
  if (parts <= 1) return;
#pragma unroll
  for (int i0 = threadIdx.x; i0 < kPieces; i0 += 256) {
    const int piece = block / a.HKV % kF8TileMerges * kPieces + i0;
    const int irow = piece / (D / 4), c4 = 4 * (piece % (D / 4));
    const int r = item.qt * kF8TileRows + irow, tok = r / G;
    const int64_t row = (int64_t)item.qs + tok;
    if (r >= (int64_t)qlen * G || row < 0 || row >= a.tokens) continue;
    float M = kNegInf, L = 0.0f, O[4] = {0, 0, 0, 0};
    auto add = [&](auto BATCH) {
      constexpr int B = BATCH.value;
      for (int p0 = 0; p0 < parts; p0 += B) {
        float2 ml[B];
        float4 v[B];
#pragma unroll
        for (int i = 0; i < B; ++i) {  // past the last part the first one again, without weight
          const int p = p0 + i < parts ? p0 + i : p0;
          const int64_t at = (((int64_t)rank * a.tile_parts + p) * a.HKV + kvh) * kF8TileRows + irow;
          ml[i] = *reinterpret_cast<const float2*>(a.ws_tile_ml + 2 * at);
          v[i] = *reinterpret_cast<const float4*>(a.ws_tile_o + at * D + c4);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < B; ++i) f8_add_state(M, L, O, ml[i], v[i], p0 + i < parts);
      }
    };
    if (parts <= 2)
      add(std::integral_constant<int, 2>{});
    else
      add(std::integral_constant<int, 8>{});
    const float inv = f8_inverse(L);
    *reinterpret_cast<uint2*>(a.o + (int64_t)(kvh * G + r - tok * G) * a.so_h + row * a.so_t + c4) =
        make_uint2(pack_bf16x2(O[0] * inv, O[1] * inv), pack_bf16x2(O[2] * inv, O[3] * inv));
  }
}

template <int D>
__global__ void __launch_bounds__(256) attn_fp8_merge_kernel(Fp8AttnArgs a, Fp8MergeGrid g) {
  if ((int)blockIdx.x < g.stream)
    f8_merge_stream<D>(a, g, blockIdx.x);
  else
    f8_merge_tile<D>(a, blockIdx.x - g.stream);
}

// ---- host side -----------------------------------------------------------------------------

struct Fp8AttnPlan {
  int tq;
  bool tiled;       // the row-tiled kernel takes long entries
  int64_t short_q;  // the most tokens of an entry that is not its
  int64_t tiles;    // query tiles of the others, at most
  int slots;        // units of a split launch, 0: keys are not split
  int64_t tile_items;  // row tiles of the long entries, at most
  int tile_parts;      // parts they may be cut into
  int64_t ws_o_bytes, ws_stream_bytes, ws_tile_o_bytes, ws_bytes;
};

static int fp8_attn_cus() {
  int dev = 0, cus = 0;
  if (hipGetDevice(&dev) != hipSuccess ||
      hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess) {
    (void)hipGetLastError();
    return 256;
  }
  return cus;
}

// Whether a call's long entries go to the row-tiled kernel: where it has, as far as its sizes tell, so many items of
// them (128 rows of a K/V head) or so many (query row, key) pairs that this is faster. Measured on MI355X, us,
// row-tiled / key-streaming, 32 heads over 8 unless said:
//  * fresh prompts, items: 4 x 64 tokens (64) 8.9 / 8.0, 5 x 64 (80) 9.2 / 11.8, 4 x 128, 24 heads (96) 10.5 / 13.1,
//    8 over 8, 6 x 128 (48) 10.0 / 8.4; 1 x 384 (96) 15.0 / 15.3, 1 x 512 (128) 17.6 / 17.4; heads of 64, for which the
//    rule is the same, 3 x 128 (96) 7.6 / 6.9, 1 x 512 (128) 12.6 / 11.6, 1 x 1024 (256) 19.7 / 20.8;
//    1 x 1024, 24 heads (192) 26.6 / 29.6, 1 x 1024 (256) 28 / 35, 8 x 512 (1024) 36 / 95; 8 over 8, 1 x 2048 (128)
//    36 / 27;
//  * behind 300 positions: 2 x 192 (96) 17.6 / 15.3, 4 x 128 (128) 16.8 / 18.5; behind 500: 512 tokens (128)
//    27 / 22, 768 (192) 38 / 33, 1024 (256) 37 / 45;
//  * behind 2000, pairs: 512 tokens (37 million) 45 / 41, 768 (59) 56 / 60, 1024 (82) 65 / 80; 8 over 8, 1024 (21)
//    35 / 25, 2048 (50) 54 / 51; behind 16000, where the query tiles read more than the L2s hold and pairs count
//    twice: 128 (66) 59 / 76; 8 over 8, 128 (16) 37 / 33, 256 (33) 40 / 51;
//  * one chunk beside 40 decoding sequences, which the two kernels share the card for, behind 1000: 128 tokens (6)
//    30 / 30, 256 (11) 33 / 35, 512 (22) 41 / 47.
// Over 153 shapes, those above among them, the rule's kernel takes 0.5 % more than the better of the two in the mean, 13 %
// at most (256 tokens behind 2000 positions, 24 heads over 8: 26.5 / 29.9).
// Contexts are taken to be as long as the table, rows to be the entries' (a call with others may take the slower one:
// 128 fresh tokens take 6.7 us under a table of 128 positions and 11.3 under one of 8192).
// Left to the kernel, which knows the lengths, the choice costs every such call more than a wrong one: a launch for
// either outcome is 1.1 to 1.6 times as long as the right one.
static bool fp8_attn_tiled(int64_t entries, int64_t tokens, int64_t G, int64_t HKV, int64_t max_q_len,
                           int64_t max_ctx) {
  // Items that suffice for contexts of up to 256, of up to 512 and of more positions: where the tiles of the
  // key-streaming kernel no longer fit the card at once, short items hardly last longer than its.
  constexpr int64_t kItems256 = 72, kItems512 = 128, kItems = 200, kFar = 6000, kMixed = 128;
  constexpr double kPairs = 40e6, kPairsMixed = 12e6;
  if (!f8_is_long(max_q_len, (int)G)) return false;
  // The longest entry's items, and those of all rows where the mean entry is long, else of those that short ones
  // cannot have.
  const int64_t q = std::min(max_q_len, tokens), rows = tokens * G;
  const int64_t left = rows >= entries * kF8LongRows ? rows : rows - entries * (kF8LongRows - 1);
  const int64_t enough = max_ctx <= 256 ? kItems256 : max_ctx <= 512 ? kItems512 : kItems;
  if (std::max(ceil_div(q * G, (int64_t)kF8TileRows), left / kF8TileRows) * HKV >= enough) return true;
  const int64_t keys = std::max<int64_t>(max_ctx - q / 2, 0);
  const double pairs = (double)rows * HKV * keys * (keys < kFar ? 1 : 2);
  return pairs >= ((entries - 1) * HKV >= kMixed ? kPairsMixed : kPairs);
}

// One workgroup per (entry, K/V head, query tile) once those fill the card; otherwise, where contexts may be long
// enough, the keys are split as well. A lone entry of a call made for long ones is taken to be long.
static Fp8AttnPlan fp8_attn_plan(int64_t entries, int64_t tokens, int64_t H, int64_t HKV, int64_t D,
                                 int64_t max_q_len, int64_t max_ctx) {
  Fp8AttnPlan pl{};
  const int64_t G = H / HKV;
  pl.tq = (int)(16 / G);
  pl.tiled = fp8_attn_tiled(entries, tokens, G, HKV, max_q_len, max_ctx);
  pl.short_q = pl.tiled ? (kF8LongRows - 1) / G : max_q_len;
  pl.tiles = std::min(entries * ceil_div(pl.short_q, (int64_t)pl.tq), tokens / pl.tq + entries);
  const int64_t slots = kF8Groups / HKV;
  if (pl.tiles < slots && max_ctx > kF8MinSplit && !(pl.tiled && entries == 1)) {
    pl.slots = (int)slots;
    pl.ws_o_bytes = slots * HKV * 16 * D * 4;
    pl.ws_stream_bytes = pl.ws_o_bytes + slots * HKV * 16 * 2 * 4;
  }
  pl.tile_parts = 1;
  if (pl.tiled) {
    // Every long entry's rows round up to a tile; it has at least kF8LongRows rows.
    const int64_t rows = tokens * G;
    pl.tile_items = rows / kF8TileRows + std::min(entries, rows / kF8LongRows);
    // Parts so that all run at once, if one entry is long and the others decode (which are done in a quarter of a
    // part's time): 1, 2 and 3 parts of 144 items beside 320 decoding ones 64, 57 and 73 us.
    const int64_t likely = (std::max<int64_t>(tokens - entries + 1, 1) * G / kF8TileRows + 1) * HKV;
    const int64_t parts = kF8Groups / (likely + (entries - 1) * HKV / 4);
    const int64_t most = max_ctx / (64 * kF8PartTiles);
    pl.tile_parts = (int)std::max<int64_t>(std::min({parts, most, (int64_t)16}), 1);
    if (pl.tile_parts > 1) {
      const int64_t slots = pl.tile_items * pl.tile_parts * HKV * kF8TileRows;
      pl.ws_tile_o_bytes = slots * D * 4;
      pl.ws_bytes = pl.ws_tile_o_bytes + slots * 2 * 4;
    }
  }
  pl.ws_bytes += pl.ws_stream_bytes;
  return pl;
}

template <int D>
static int launch_fp8_attention(const Fp8AttnArgs& a, const Fp8AttnPlan& pl, hipStream_t stream) {
  const dim3 wg(64 * kF8Waves);
  const bool one = pl.short_q <= pl.tq;
  const int64_t units = (pl.slots ? pl.slots : one && !a.tiled ? a.entries : pl.tiles) * (int64_t)a.HKV;
  const dim3 grid((unsigned)(units + a.tile_blocks));
  if (a.tiled)
    hipLaunchKernelGGL(attn_fp8_mixed_kernel<D>, grid, wg, 0, stream, a);
  else if (!one)
    hipLaunchKernelGGL((attn_fp8_stream_kernel<D, false, true>), grid, wg, 0, stream, a);
  else if (pl.slots)
    hipLaunchKernelGGL((attn_fp8_stream_kernel<D, true, true>), grid, wg, 0, stream, a);
  else
    hipLaunchKernelGGL((attn_fp8_stream_kernel<D, true, false>), grid, wg, 0, stream, a);
  if (int st = launch_status()) return st;
  if (pl.slots || pl.tile_parts > 1) {
    Fp8MergeGrid g{};
    if (pl.slots) {
      const int64_t rows = std::min<int64_t>(pl.short_q, pl.tq) * a.G;
      g.pieces = (int)ceil_div(rows * (D / 4), 64);
      g.by_entry = one;
      g.stream = (int)((one ? a.entries : pl.slots) * (int64_t)a.HKV * g.pieces);
    }
    const int64_t tile = pl.tile_parts > 1 ? pl.tile_items * a.HKV * kF8TileMerges : 0;
    hipLaunchKernelGGL(attn_fp8_merge_kernel<D>, dim3((unsigned)(g.stream + tile)), dim3(256), 0, stream, a, g);
  }
  return launch_status();
}

}  // namespace lse

namespace {

constexpr int64_t kMax31 = 2147483647;
bool aligned(const void* p, uintptr_t bytes) { return ((uintptr_t)p % bytes) == 0; }

typedef lse_paged_attention_fp8_args Args;

int check_sizes(const Args& x) {
  if (x.entries < 0 || x.entries > kMax31 || x.tokens < 0 || x.tokens > kMax31 || x.H < 1 || x.H > 65536 ||
      x.H_KV < 1 || x.H % x.H_KV || x.H / x.H_KV > 16 || (x.D != 64 && x.D != 128) || x.max_q_len < 0 ||
      x.max_q_len > kMax31 || x.max_blocks < 0 || x.block_size < 16 || x.block_size % 16)
    return LSE_E_SHAPE;
  // Contexts of up to 2^30 positions: the kernels round their ends up to whole tiles in 32 bits.
  return x.block_size > kMax31 || x.max_blocks > ((int64_t)1 << 30) / x.block_size ? LSE_E_RANGE : LSE_OK;
}

lse::Fp8AttnPlan plan_of(const Args& x) {
  return lse::fp8_attn_plan(x.entries, x.tokens, x.H, x.H_KV, x.D, x.max_q_len, x.max_blocks * x.block_size);
}

}  // namespace

extern "C" {

int64_t lse_paged_attention_fp8_workspace_bytes(const struct lse_paged_attention_fp8_args* args) {
  if (!args || check_sizes(*args)) return -1;
  if (args->entries == 0 || args->tokens == 0 || args->max_q_len == 0) return 0;
  return plan_of(*args).ws_bytes;
}

int lse_paged_attention_fp8_choice(const struct lse_paged_attention_fp8_args* args, int64_t* row_tiled,
                                   int64_t* parts, int64_t* units) {
  if (!args || !row_tiled || !parts || !units) return LSE_E_NULL;
  if (int st = check_sizes(*args)) return st;
  const bool empty = args->entries == 0 || args->tokens == 0 || args->max_q_len == 0;
  const lse::Fp8AttnPlan pl = empty ? lse::Fp8AttnPlan{} : plan_of(*args);
  *row_tiled = pl.tiled, *parts = pl.tiled ? pl.tile_parts : 0, *units = pl.slots;
  return LSE_OK;
}

int lse_paged_attention_fp8(const struct lse_paged_attention_fp8_args* args, void* workspace,
                            int64_t workspace_bytes, void* stream) {
  if (!args) return LSE_E_NULL;
  const Args& x = *args;
  if (int st = check_sizes(x)) return st;
  if (x.num_blocks < 0 || x.num_blocks > kMax31 || x.block_table_stride < x.max_blocks) return LSE_E_SHAPE;
  const int64_t per = x.block_size / 16;
  if (x.pool_stride_block < x.H_KV * per * 16 * x.D || x.scales_stride_block < 2 * x.H_KV * per)
    return LSE_E_SHAPE;
  if (x.entries == 0 || x.tokens == 0 || x.max_q_len == 0) return LSE_OK;
  if (x.num_blocks < 1) return LSE_E_SHAPE;
  if (!x.q || !x.k_pool || !x.v_pool || !x.scales || !x.block_table || !x.context_len || !x.query_offset ||
      !x.q_start || !x.q_len || !x.o)
    return LSE_E_NULL;
  // Groups are addressed in 16-byte units by 32 bits.
  if (x.num_blocks > (((int64_t)1 << 36) - 1) / x.pool_stride_block) return LSE_E_RANGE;
  const int64_t strides[] = {x.q_stride_h, x.q_stride_t, x.o_stride_h, x.o_stride_t};
  for (int64_t s : strides)
    if (s < 0) return LSE_E_SHAPE;
  for (int64_t s : strides)
    if (s % 8) return LSE_E_ALIGN;
  if (x.pool_stride_block % 16 || x.scales_stride_block % 2 || !aligned(x.q, 16) || !aligned(x.o, 16) ||
      !aligned(x.k_pool, 16) || !aligned(x.v_pool, 16) || !aligned(x.scales, 2) ||
      !aligned(x.block_table, 4) || !aligned(x.context_len, 4) || !aligned(x.query_offset, 4) ||
      !aligned(x.q_start, 4) || !aligned(x.q_len, 4))
    return LSE_E_ALIGN;
  if (workspace_bytes < 0 || (workspace && !aligned(workspace, 16))) return LSE_E_WORKSPACE;
  const int cus = lse::fp8_attn_cus();
  const lse::Fp8AttnPlan pl = plan_of(x);
  if (pl.ws_bytes > 0 && (workspace_bytes < pl.ws_bytes || !workspace)) return LSE_E_WORKSPACE;
  if ((std::max(x.entries, pl.tiles) + pl.tile_items * pl.tile_parts) * x.H_KV > kMax31 ||
      pl.tile_items * x.H_KV * 16 > kMax31) return LSE_E_RANGE;
  lse::Fp8AttnArgs a{};
  a.q = (const uint16_t*)x.q, a.sq_h = x.q_stride_h, a.sq_t = x.q_stride_t;
  a.pool = {(uint8_t*)x.k_pool, (uint8_t*)x.v_pool, (uint8_t*)x.scales, x.pool_stride_block,
            x.scales_stride_block, (int)x.num_blocks, (int)per};
  a.block_table = x.block_table, a.sbt = x.block_table_stride;
  a.context_len = x.context_len, a.query_offset = x.query_offset, a.q_start = x.q_start, a.q_len = x.q_len;
  a.o = (uint16_t*)x.o, a.so_h = x.o_stride_h, a.so_t = x.o_stride_t;
  a.entries = (int)x.entries, a.HKV = (int)x.H_KV, a.G = (int)(x.H / x.H_KV);
  a.tokens = (int)x.tokens;
  a.max_ctx = (int)(x.max_blocks * x.block_size);
  a.max_q_len = (int)x.max_q_len, a.tiled = pl.tiled, a.tq = pl.tq, a.slots = pl.slots;
  a.scale_log2 = (float)x.softmax_scale * 1.4426950408889634f;
  a.ws_o = pl.slots ? (float*)workspace : nullptr;
  a.ws_ml = pl.slots ? (float*)((char*)workspace + pl.ws_o_bytes) : nullptr;
  a.tile_parts = pl.tile_parts;
  a.tile_blocks = (int)(pl.tile_items * pl.tile_parts * x.H_KV);
  a.ws_tile_o = pl.tile_parts > 1 ? (float*)((char*)workspace + pl.ws_stream_bytes) : nullptr;
  a.ws_tile_ml =
      pl.tile_parts > 1 ? (float*)((char*)workspace + pl.ws_stream_bytes + pl.ws_tile_o_bytes) : nullptr;
  const int64_t items = x.entries * x.H_KV;
  a.sorted = x.entries <= 64 && items > cus && a.max_ctx > 256;
  a.first_round = items > cus && items <= 2 * (int64_t)cus && cus % a.HKV == 0 ? cus / a.HKV : 0;
  return x.D == 64 ? lse::launch_fp8_attention<64>(a, pl, (hipStream_t)stream)
                   : lse::launch_fp8_attention<128>(a, pl, (hipStream_t)stream);
}

}  // extern "C"
