// Paged attention over the 8-bit K/V cache (fp8_kv.h) of prompts and prompt chunks: the row-tiled kernel beside
// attn_fp8_stream.h's key-streaming one, with the same semantics. It takes the entries that f8_is_long of calls
// that are tiled (fp8_attn_tiled, attn_fp8.hip).
//
// A workgroup of four waves owns 128 rows (tokens x the G query heads of one K/V head, token-major, so no G
// leaves rows idle), each wave 32 of them on v_mfma_f32_32x32x16_bf16, over tiles of 64 keys:
//  * S^T = K Q^T: K rows from LDS are the A operand, Q stays in registers; lane (i, h) then holds row i's scores with
//    keys 16 b + 8 h + r: the rows of K are put into LDS so that this is the order V has its keys in.
//  * O^T += V^T P^T: the scores, rounded to bf16, are the B operand; V's dims are the A operand's rows. O^T's columns
//    are the lane's row again, so the softmax's factors are per-lane scalars.
//
// The matrix cores, the VALU (exponentials above all) and LDS (a fragment of 1 KB per MFMA: of the 128 bytes a clock
// it delivers, with two workgroups a CU, all) each have about as much to do, so a wave keeps them busy at the same
// time: one sequence of MFMAs over K of tile j + 1 and V of tile j, whose fragments are read four MFMAs ahead, across
// the tiles; between those of K the probabilities of tile j, between those of V the maximum of tile j + 1 and
// the staging of K of tile j + 2 and V of tile j + 1 from registers, where they arrived as codes, to LDS as bf16
// values times their scale (each code converted once a workgroup). One barrier a tile, in the middle of V's MFMAs:
// with three V tiles and two K tiles in LDS nobody waits there for more than the staging.
//
// A row's reference m (probabilities are exp2(s - m)) is a maximum that may lag by up to 8: O is rescaled only
// when a tile's maximum lies further above it. Sums are taken over the probabilities as rounded to bf16, so
// that a rounding enters numerator and denominator alike.
//
// LDS: K tiles [16-dim step][32-key block][8-dim half][row], V tiles [group][8-key half][dim], 16 bytes each: 32 lanes
// of a fragment read 512 contiguous bytes (with the halves of a row side by side, half of all LDS cycles were
// bank conflicts). K's row r of step k is at r ^ 4 (k % 4), so that the staging's writes, four steps of four
// rows per 16 lanes, fall on distinct banks too.
//
// Where a call has too few items to fill the card, each is cut into parts by its key tiles, and a second kernel
// adds the parts' states up.
//
// On MI355X a tile of 64 keys takes 1.3 us in a workgroup alone on its CU, 1.7 beside another, which is the rate of a
// large bf16 product (1260 TFLOP/s); what precedes and follows an item's tiles (finding it, three loads that
// depend on each other, the first scores, the stores) 6 us. Three fresh prompts of 1285 to 1321 tokens, 32 heads
// over 8: 56 to 57 us, by the card, 720 to 750 TFLOP/s of the causal half; 1813 tokens behind 6266 positions: 207 to
// 222 us, 960 to 1030 TFLOP/s. In the latter 56 of 256 CUs have one item instead of two, but every item cut into 4, 9 or
// 10 parts took 267, 328 and 340 us, partial states and all, where whole ones took 223.
#pragma once

#include <type_traits>

#include "attn_fp8.h"

namespace lse {

constexpr int kF8TileRows = 128;  // query rows of a workgroup
constexpr int kF8TileWaves = 4;
constexpr int kF8PartTiles = 6;    // fewest key tiles of a part
constexpr float kF8Lag = 8.0f;     // log2 of how far probabilities may exceed 1
constexpr float kF8Far = 16384.0f;  // |m| from which scaled scores are rounded before m is subtracted
constexpr int f8_tile_lds(int D) { return 5 * 128 * D; }

__device__ __forceinline__ f32x16 f8_mfma32(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// Every LDS access of this wave is done, then the workgroup's barrier; global loads stay in flight.
__device__ __forceinline__ void f8_barrier() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// A lane's value and that of lane l ^ 32, in either order (see attn_tile.hip's both_halves).
struct F8Halves {
  float a, b;
};
__device__ __forceinline__ F8Halves f8_halves(float v) {
  F8Halves h{v, v};
  asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(h.a), "+v"(h.b));
  return h;
}

// The item of rank p among the row tiles of all long entries, furthest tiles (virtual tile index: the entry's
// offset in tiles + its tile) first. Entries are looked at 64 at a time, one per lane.
struct F8Item {
  int e, qt;  // e < 0: no such item
  int qlen, ctx, qo, qs;
};
__device__ __forceinline__ F8Item f8_tile_item(const Fp8AttnArgs& a, int p) {
  const int lane = threadIdx.x & 63;
  struct Entry {
    int qlen, ctx, qo, qs;
  };
  auto entry = [&](int i, int& base, int& tiles) {
    base = tiles = 0;
    Entry x{0, 0, 0, 0};
    if (i >= a.entries) return x;
    x = Entry{min(a.q_len[i], a.max_q_len), a.context_len[i], a.query_offset[i], a.q_start[i]};
    if (!f8_is_long(x.qlen, a.G)) return x;
    tiles = (int)(((int64_t)x.qlen * a.G + kF8TileRows - 1) / kF8TileRows);
    base = (int)((int64_t)min(max(x.qo, 0), a.max_ctx) * a.G / kF8TileRows);
    return x;
  };
  int base0, tiles0;
  const Entry entry0 = entry(lane, base0, tiles0);
  // Tiles at level L or above it, over all entries.
  auto above = [&](int L) {
    int n = min(max(base0 + tiles0 - L, 0), tiles0);
    for (int e0 = 64; e0 < a.entries; e0 += 64) {
      int b, t;
      entry(e0 + lane, b, t);
      n += min(max(b + t - L, 0), t);
    }
    return f8_wave_total(n);
  };
  if (above(0) <= p) return {-1, 0, 0, 0, 0, 0};
  int top = base0 + tiles0;
  for (int e0 = 64; e0 < a.entries; e0 += 64) {
    int b, t;
    entry(e0 + lane, b, t);
    top = max(top, b + t);
  }
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) top = max(top, __shfl_xor(top, off));
  int lo = 0, hi = __builtin_amdgcn_readfirstlane(top);  // above(lo) > p >= above(hi)
  while (hi - lo > 1) {
    const int mid = lo + (hi - lo) / 2;
    if (above(mid) > p) lo = mid; else hi = mid;
  }
  p -= above(lo + 1);  // among the entries that have a tile at level lo
  for (int e0 = 0; e0 < a.entries; e0 += 64) {
    int b = base0, t = tiles0;
    const Entry x = e0 ? entry(e0 + lane, b, t) : entry0;
    const int mine = t > 0 && b <= lo && lo < b + t;
    const int before = kv_wave_scan(mine) - mine;
    const unsigned long long hit = __ballot(mine && before == p);
    if (hit) {
      const int at = __ffsll(hit) - 1;
      return {e0 + at,
              lo - __builtin_amdgcn_readlane(b, at),
              __builtin_amdgcn_readlane(x.qlen, at),
              __builtin_amdgcn_readlane(x.ctx, at),
              __builtin_amdgcn_readlane(x.qo, at),
              __builtin_amdgcn_readlane(x.qs, at)};
    }
    p -= __builtin_amdgcn_readlane(before + mine, 63);
  }
  return {-1, 0, 0, 0, 0, 0};
}

// Key tiles of an item, and the parts they are cut into.
__device__ __forceinline__ int f8_tile_end(const Fp8AttnArgs& a, int qo, int ctx, int qlen, int qt) {
  return f8_end(a, qo, ctx, min(qlen - 1, (qt * kF8TileRows + kF8TileRows - 1) / a.G) + 1);
}
__device__ __forceinline__ int f8_tile_parts(const Fp8AttnArgs& a, int tiles) {
  return min(a.tile_parts, max(tiles / kF8PartTiles, 1));
}

// `lds`: f8_tile_lds(D) bytes.
template <int D>
__device__ __forceinline__ void f8_tile(const Fp8AttnArgs& a, int block, unsigned char* lds) {
  constexpr int J = D / 64, KK = D / 16, DB = D / 32;
  constexpr int kSlot = 64 * D * 2;  // bytes of a K or V tile: two of K, then three of V
  constexpr int P = D / 64;          // 16-byte pieces of a group a lane stages, of K and of V
  constexpr int N = 2 * KK;          // MFMAs of K, and of V, per tile
  static_assert(N == 4 * DB, "as many of V as of K");

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n32 = lane & 31, half = lane >> 5;
  const int G = a.G, kvh = block % a.HKV;
  const int part = block / a.HKV % a.tile_parts, rank = block / a.HKV / a.tile_parts;
  const F8Item item = f8_tile_item(a, rank);
  if (item.e < 0) return;
  const int e = item.e;
  const int qlen = item.qlen, ctx = item.ctx, qo = item.qo, qs = item.qs;
  const int row0 = item.qt * kF8TileRows;
  const int end_n = f8_tile_end(a, qo, ctx, qlen, item.qt);
  const int all_tiles = (end_n + 63) / 64, parts = f8_tile_parts(a, all_tiles);
  if (part >= parts) return;
  const int tile0 = (int)((int64_t)all_tiles * part / parts);
  const int tiles = (int)((int64_t)all_tiles * (part + 1) / parts) - tile0;

  // The wave stages group `wave` of every tile. Lane i of 64 holds place (16-byte units) and scales of that
  // group in tile tile0 + 64 w + i, for the window w of the tile to load and the one behind it.
  const int32_t* bt = a.block_table + (int64_t)e * a.sbt;
  const int per = a.pool.per, last_group = max(end_n - 1, 0) / kKvGroup;
  auto table_at = [&](int w, int& sub) {
    const int64_t first = 4 * ((int64_t)tile0 + 64 * w + lane) + wave;
    const int grp = (int)min(first, (int64_t)last_group);
    const int bi = per == 1 ? grp : grp / per;
    sub = grp - bi * per;
    return bt[bi];
  };
  int blk0 = 0, blk1 = 0, blk2 = 0, sub0 = 0, sub1 = 0, sub2 = 0;
  if (tiles > 0) blk0 = table_at(0, sub0), blk1 = table_at(1, sub1), blk2 = table_at(2, sub2);

  // The lane's row and the last position it sees.
  const int r = row0 + 32 * wave + n32, tok = r / G, gq = r - tok * G;
  const int64_t row = (int64_t)qs + tok;
  const bool row_ok = r < (int64_t)qlen * G && row >= 0 && row < a.tokens;
  const int lim = (int)min((int64_t)qo + tok, (int64_t)end_n - 1);
  // Keys up to here are seen by every row of the wave.
  const int all_see = (int)min((int64_t)qo + (row0 + 32 * wave) / G, (int64_t)end_n - 1);

  // A negative softmax scale moves into Q, a zero one makes Q zero (exactly), so that a maximum can be
  // taken before the scaling.
  const float sc = a.scale_log2 == 0.0f ? 1.0f : __builtin_fabsf(a.scale_log2);
  const bool keep = row_ok && a.scale_log2 != 0.0f;
  uint4 qw[KK];
  {
    const uint16_t* qp =
        a.q + (int64_t)(kvh * G + (row_ok ? gq : 0)) * a.sq_h + (row_ok ? row : 0) * a.sq_t + 8 * half;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) qw[kk] = *reinterpret_cast<const uint4*>(qp + 16 * kk);
  }

  auto place = [&](int blk, int sub, uint32_t& off) {
    const bool bad = blk < 0 || blk >= a.pool.blocks;
    blk = bad ? 0 : blk;
    const int inner = kvh * per + sub;
    off = (uint32_t)(((int64_t)blk * a.pool.sb + (int64_t)inner * (16 * D)) >> 4);
    const int s = *reinterpret_cast<const uint16_t*>(a.pool.scales + (int64_t)blk * a.pool.ss + 2 * inner);
    return bad ? 0xffff : s;
  };
  uint32_t off0 = 0, off1 = 0;
  int sc0 = 0, sc1 = 0;
  // The codes on their way to LDS, and the scales of these groups.
  uint4 kc[P], vc[P];
  uint32_t at_k = 0, at_v = 0;
  int scale_k = 0, scale_v = 0, scale_v_next = 0;
  auto load = [&](const uint8_t* pool, uint32_t at, uint4 (&c)[P]) {
    const uint8_t* p = pool + ((uint64_t)at << 4);
#pragma unroll
    for (int i = 0; i < P; ++i) c[i] = *reinterpret_cast<const uint4*>(p + 16 * lane + 1024 * i);
  };
  // K of tile t (counted from tile0), and V of the tile whose K the call before loaded.
  auto load_v = [&] {
    scale_v = scale_v_next;
    load(a.pool.v, at_v, vc);
  };
  auto load_k = [&](int t) {
    at_k = __builtin_amdgcn_readlane(off0, t & 63);
    scale_k = __builtin_amdgcn_readlane(sc0, t & 63);
    at_v = at_k, scale_v_next = scale_k;
    load(a.pool.k, at_k, kc);
    if ((t & 63) == 63) {
      off0 = off1, sc0 = sc1;
      sc1 = place(blk2, sub2, off1);
      blk2 = table_at((t >> 6) + 3, sub2);
    }
  };
  // Piece p = 64 i + lane of K: key 4 (p / (16 J)) + p / 4 % 4 of the group, dims 64 (p / 16 % J) + 16 (p % 4); its
  // place in a K tile, the key's row being its number with bits 2 and 3 exchanged.
  uint32_t kdst[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int p = 64 * i + lane, sq = p / (16 * J), sr = p / 4 % 4, kk = 4 * (p / 16 % J) + p % 4;
    const int to = 16 * (wave & 1) + 8 * (sq & 1) + 4 * (sq >> 1) + sr;
    kdst[i] = (kk * 2 + (wave >> 1)) * 1024 + (to ^ (4 * (kk & 3))) * 16;
  }
  const uint32_t vdst = 2 * kSlot + wave * D * 32 + lane * 16;
  // Half h of piece i, eight codes, as bf16 into the tile at `slot`.
  auto stage_k = [&](int i, int h, int slot) {
    const uint4 c = kc[i];
    const bf16x8 v = kv_decode8(h ? c.z : c.x, h ? c.w : c.y, kv_scale(scale_k & 255));
    *reinterpret_cast<uint4*>(lds + slot + kdst[i] + 512 * h) = __builtin_bit_cast(uint4, v);
  };
  auto stage_v = [&](int i, int h, int slot) {
    const uint4 c = vc[i];
    const bf16x8 v = kv_decode8(h ? c.z : c.x, h ? c.w : c.y, kv_scale(scale_v >> 8 & 255));
    *reinterpret_cast<uint4*>(lds + slot + vdst + 1024 * i + 16 * D * h) = __builtin_bit_cast(uint4, v);
  };
  // Slots of tile t past the last key hold anything: their codes become zeros, which 0 probabilities need.
  auto mask_v = [&](int t) {
    const int left = end_n - 64 * (tile0 + t) - 16 * wave;
    if (64 * (tile0 + t) + 64 <= end_n) return;
    auto mask = [&](int w) {
      const int nb = min(max(left - 4 * w, 0), 4);
      return nb == 4 ? 0xffffffffu : (1u << (8 * nb)) - 1u;
    };
    const uint32_t m0 = mask(0), m1 = mask(1), m2 = mask(2), m3 = mask(3);
#pragma unroll
    for (int i = 0; i < P; ++i) vc[i].x &= m0, vc[i].y &= m1, vc[i].z &= m2, vc[i].w &= m3;
  };

  // Fragment f of the tile at `slot`: K's step f / 2 of block f % 2, V's group f / DB of dims 32 (f % DB).
  const unsigned char* kread[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) kread[i] = lds + (n32 ^ (4 * i)) * 16 + 512 * half;
  const unsigned char* vread = lds + 2 * kSlot + n32 * 16 + 16 * D * half;
  auto read_k = [&](int f, int slot) {
    return as_bf16x8(*reinterpret_cast<const uint4*>(kread[(f >> 1) & 3] + slot + f * 1024));
  };
  auto read_v = [&](int f, int slot) {
    return as_bf16x8(*reinterpret_cast<const uint4*>(vread + slot + f / DB * (32 * D) + f % DB * 512));
  };

  bf16x8 qf[KK];
  f32x16 oacc[DB], sa[2], sb[2], zero;  // scores: of 32-key block b, keys 16 (i / 8) + 8 half + i % 8
#pragma unroll
  for (int i = 0; i < 16; ++i) zero[i] = 0.0f;
#pragma unroll
  for (int d = 0; d < DB; ++d) oacc[d] = zero;
  bf16x8 pa[4];
  constexpr float kNone = -__builtin_huge_valf();
  float m = kNone, l = 0.0f, mul = sc, shift = 0.0f, mx = kNone;  // p = exp2(s mul - shift)

  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  // Probabilities of scores 2 pair and 2 pair + 1, rounded in eights, and their sum. Here and below an empty
  // statement keeps the compiler from moving work to where its result is used, behind the MFMAs it is to run beside.
  auto exps = [&](f32x16 (&cur)[2], int pair) {
    const int i = 2 * pair;
#pragma unroll
    for (int x = i; x < i + 2; ++x)
      cur[x >> 4][x & 15] = exp2_fast(__builtin_fmaf(cur[x >> 4][x & 15], mul, -shift));
    asm volatile("" : "+v"(cur[i >> 4][i & 15]), "+v"(cur[i >> 4][(i & 15) + 1]));
    if ((i & 7) == 6) {
      f32x8 v;
#pragma unroll
      for (int x = 0; x < 8; ++x) v[x] = cur[i >> 4][(i & 8) + x];
      bf16x8 p = __builtin_convertvector(v, bf16x8);
#pragma unroll
      for (int x = 0; x < 8; x += 2)
        l = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{p[x], p[x + 1]}, bf16x2{(__bf16)1.0f, (__bf16)1.0f}, l, false);
      asm volatile("" : "+v"(p), "+v"(l));
      pa[i >> 3] = p;
    }
  };
  // The reference m from the tile's maximum, O and sum rescaled where it moves.
  auto reference = [&](f32x16 (&cur)[2]) {
#pragma clang fp contract(off)  // the maximum is a rounded product wherever it is used
    const F8Halves h = f8_halves(mx);
    const float top = fmaxf(h.a, h.b) * sc;
    const bool moves = top > m + kF8Lag;  // from -inf with the first key seen
    if (__ballot(moves)) {
      const float to = moves ? top : m;
      const float alpha = moves ? exp2_fast(m - to) : 1.0f;
      m = to;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < DB; ++d) oacc[d] *= alpha;
    }
    mul = sc, shift = m == kNone ? 0.0f : m;  // a row with no key yet keeps p = 0
    if (__ballot(__builtin_fabsf(shift) > kF8Far)) {
#pragma unroll
      for (int i = 0; i < 32; ++i) cur[i >> 4][i & 15] = cur[i >> 4][i & 15] * sc - shift;
      mul = 1.0f, shift = 0.0f;
    }
  };
  // Hides the scores of tile t that a row does not see.
  auto hide = [&](f32x16 (&cur)[2], int t) {
    if (64 * (tile0 + t) + 63 <= all_see) return;
    const int rel = lim - 64 * (tile0 + t) - 8 * half;
    mx = kNone;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      cur[i >> 4][i & 15] = 16 * (i >> 3) + (i & 7) <= rel ? cur[i >> 4][i & 15] : kNone;
      mx = fmaxf(mx, cur[i >> 4][i & 15]);
    }
  };
  constexpr int kAhead = 4, kLate = N / 4, E = 16 / N;
  bf16x8 fr[kAhead];
  // One tile: P V of tile j, whose scores are in cur, and (MORE) K Q^T of tile j + 1 into next. In LDS K of j + 1 and
  // V of j, in registers the codes of K of j + 2 and V of j + 1, in fr the first fragments of K (MORE) or V.
  auto step = [&](auto MORE, f32x16 (&cur)[2], f32x16 (&next)[2], int j, int k_slot, int v_slot, int v_next) {
    if constexpr (!MORE.value) {
      reference(cur);
#pragma unroll
      for (int p = 0; p < 12; ++p) exps(cur, p);
    } else {
#pragma unroll
      for (int f = 0; f < N; ++f) {
        // Ahead of the other workgroup's wave on the SIMD: 4 % less time (61.3 against 64.1 us, three prompts).
        if (f == 0) __builtin_amdgcn_s_setprio(1);
        if (f == kLate) reference(cur);
        next[f & 1] = f8_mfma32(fr[f % kAhead], qf[f >> 1], f < 2 ? zero : next[f & 1]);
        if (f >= kLate) {
#pragma unroll
          for (int x = 0; x < E; ++x) exps(cur, E * (f - kLate) + x);
        }
        fr[f % kAhead] = f + kAhead < N ? read_k(f + kAhead, k_slot) : read_v(f + kAhead - N, v_slot);
        __builtin_amdgcn_sched_barrier(0);
      }
      __builtin_amdgcn_s_setprio(0);
      mask_v(j + 1);
      mx = kNone;
    }
#pragma unroll
    for (int f = 0; f < N; ++f) {
      oacc[f % DB] = f8_mfma32(fr[f % kAhead], pa[f / DB], oacc[f % DB]);
      if (f < kLate) {
#pragma unroll
        for (int x = 0; x < E; ++x) exps(cur, 12 + E * f + x);
      }
      if constexpr (MORE.value) {
        if (f >= kLate && f < kLate + N / 2) {  // 32 scores over N / 2 MFMAs
          constexpr int S = 64 / N;
#pragma unroll
          for (int x = S * (f - kLate); x < S * (f - kLate + 1); x += 2) {
            mx = fmaxf(fmaxf(mx, next[x >> 4][x & 15]), next[x >> 4][(x & 15) + 1]);
            asm volatile("" : "+v"(mx));
          }
        }
        if (f >= kLate && f < N - kAhead) {  // 4 P half pieces over N - kAhead - kLate MFMAs
          constexpr int H = 4 * P / (N - kAhead - kLate);
          static_assert(H * (N - kAhead - kLate) == 4 * P, "whole half pieces per MFMA");
#pragma unroll
          for (int x = H * (f - kLate); x < H * (f - kLate + 1); ++x) {
            if (x < 2 * P) stage_v(x >> 1, x & 1, v_next);
            else stage_k((x - 2 * P) >> 1, x & 1, kSlot - k_slot);
          }
        }
        if (f == N - kAhead - 1) {
          f8_barrier();
          load_v();
          load_k(j + 3);
        }
      }
      if (f + kAhead < N) fr[f % kAhead] = read_v(f + kAhead, v_slot);
      else if constexpr (MORE.value) fr[f % kAhead] = read_k(f + kAhead - N, kSlot - k_slot);
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (MORE.value) hide(next, j + 1);
  };

  if (tiles > 0) {
    // The first codes are on their way before the first scales are waited for; K of tile 1 goes to LDS behind the first
    // scores.
    uint4 k1[P];
    sc0 = place(blk0, sub0, off0);
    at_k = __builtin_amdgcn_readfirstlane(off0);
    load(a.pool.k, at_k, kc);
    load(a.pool.v, at_k, vc);
    at_v = __builtin_amdgcn_readlane(off0, 1);
    load(a.pool.k, at_v, k1);
    __builtin_amdgcn_sched_barrier(0);
    sc1 = place(blk1, sub1, off1);
    scale_k = scale_v = __builtin_amdgcn_readfirstlane(sc0);
    scale_v_next = __builtin_amdgcn_readlane(sc0, 1);
#pragma unroll
    for (int x = 0; x < 2 * P; ++x) stage_k(x >> 1, x & 1, 0);
    mask_v(0);
#pragma unroll
    for (int x = 0; x < 2 * P; ++x) stage_v(x >> 1, x & 1, 0);
    load_v();
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      const uint32_t flip = a.scale_log2 < 0.0f ? 0x80008000u : 0u;
      const uint4 v = qw[kk];
      qf[kk] = as_bf16x8(keep ? make_uint4(v.x ^ flip, v.y ^ flip, v.z ^ flip, v.w ^ flip)
                              : make_uint4(0, 0, 0, 0));
    }
    f8_barrier();
#pragma unroll
    for (int f = 0; f < N; ++f) {
      sa[f & 1] = f8_mfma32(read_k(f, 0), qf[f >> 1], f < 2 ? zero : sa[f & 1]);
    }
    scale_k = scale_v;
#pragma unroll
    for (int i = 0; i < P; ++i) kc[i] = k1[i];
#pragma unroll
    for (int x = 0; x < 2 * P; ++x) stage_k(x >> 1, x & 1, kSlot);
    load_k(2);
#pragma unroll
    for (int i = 0; i < 32; ++i) mx = fmaxf(mx, sa[i >> 4][i & 15]);
    hide(sa, 0);
    f8_barrier();  // before K of tile 2 takes the place of tile 0's

    int k_slot = kSlot, v0 = 0, v1 = kSlot, v2 = 2 * kSlot;
    if (tiles > 1) {
#pragma unroll
      for (int f = 0; f < kAhead; ++f) fr[f] = read_k(f, k_slot);
    } else {
#pragma unroll
      for (int f = 0; f < kAhead; ++f) fr[f] = read_v(f, v0);
    }
    int j = 0;
    auto turn = [&] {
      k_slot = kSlot - k_slot;
      const int v = v0;
      v0 = v1, v1 = v2, v2 = v;
    };
    // Two tiles a round, so that the scores change places without a copy: 219 -> 211 us, a far chunk.
    for (; j + 2 < tiles; j += 2) {
      step(std::true_type{}, sa, sb, j, k_slot, v0, v1);
      turn();
      step(std::true_type{}, sb, sa, j + 1, k_slot, v0, v1);
      turn();
    }
    if (j + 1 < tiles) {
      step(std::true_type{}, sa, sb, j, k_slot, v0, v1);
      turn();
      sa[0] = sb[0], sa[1] = sb[1];
      ++j;
    }
    if (tiles > 1) {
#pragma unroll
      for (int f = 0; f < kAhead; ++f) fr[f] = read_v(f, v0);
    }
    step(std::false_type{}, sa, sb, j, 0, v0, 0);
  }

  const F8Halves h = f8_halves(l);
  const float sum = h.a + h.b;
  if (parts > 1) {
    if (!row_ok) return;
    const int64_t at = (((int64_t)rank * a.tile_parts + part) * a.HKV + kvh) * kF8TileRows + 32 * wave + n32;
    float* to = a.ws_tile_o + at * D + 4 * half;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int b = 0; b < 4; ++b)
        *reinterpret_cast<float4*>(to + 32 * d + 8 * b) =
            make_float4(oacc[d][4 * b], oacc[d][4 * b + 1], oacc[d][4 * b + 2], oacc[d][4 * b + 3]);
    if (half == 0) *reinterpret_cast<float2*>(a.ws_tile_ml + 2 * at) = make_float2(m, sum);
    return;
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;  // no key: zeros
  // Of each 16 dims a lane has two fours, lane l ^ 32 the others: an exchange gives each eight in a row.
  uint16_t* out = a.o + (int64_t)(kvh * G + gq) * a.so_h + row * a.so_t + 8 * half;
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int b = 0; b < 4; b += 2) {
      uint32_t w[2][2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int x = 4 * (b + i);
        w[i][0] = pack_bf16x2(oacc[d][x] * inv, oacc[d][x + 1] * inv);
        w[i][1] = pack_bf16x2(oacc[d][x + 2] * inv, oacc[d][x + 3] * inv);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
        asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(w[0][i]), "+v"(w[1][i]));
      if (row_ok)
        *reinterpret_cast<uint4*>(out + 32 * d + 8 * b) = make_uint4(w[0][0], w[0][1], w[1][0], w[1][1]);
    }
}

}  // namespace lse
