// Paged attention over the 8-bit K/V cache (fp8_kv.h) of prompts and prompt chunks: the row-tiled kernel beside
// attn_fp8.hip's key-streaming one, with the same semantics. It takes every entry that f8_is_long.
//
// A workgroup of four waves owns 256 rows (tokens x the G query heads of one K/V head, token-major, so no G
// leaves rows idle), each wave 64 of them as two blocks of 32 on v_mfma_f32_32x32x16_bf16, over tiles of 64 keys:
//  * S^T = K Q^T: K rows from LDS are the A operand, Q stays in registers; lane (i, h) of a block holds row i's
//    scores with keys 16 b + 8 h + r, the order V has them in, as the rows of K are put into LDS in that order.
//  * O^T += V^T P^T: the scores, rounded to bf16, are the B operand; V's dims are rows of the A operand in LDS.
//    O^T's columns are the lane's rows again: the softmax's factors are per-lane scalars.
//
// What bounds it is the matrix cores, so everything else is put beside them. Fragments are read once for both
// of a wave's row blocks: with 32 rows a wave LDS would have to deliver 128 bytes a clock, all it can, for
// the MFMAs to run without a pause; with 64 it is half of that. One wave per SIMD (the two blocks take 512
// registers) has no other wave to fill the matrix cores while it computes a softmax, so the wave does so itself:
// between the MFMAs of K Q^T of tile j + 1 stand the exponentials of tile j, between those of P V of tile j the
// maximum of tile j + 1 and the staging: K of tile j + 2 and V of tile j + 1 from registers, where they
// arrived as codes, to LDS as bf16 values times their scale (each code converted once a workgroup).
//
// A row's reference m (probabilities are exp2(s - m)) is a maximum that may lag by up to 8: O is rescaled only
// when a tile's maximum lies further above it. Sums are taken over the probabilities as rounded to bf16, so
// that a rounding enters numerator and denominator alike.
//
// LDS: K tiles [16-dim step][32-key block][8-dim half][row], V tiles [group][8-key half][dim], 16 bytes each: 32 lanes
// of a fragment read 512 contiguous bytes (with the halves of a row side by side, half of all LDS cycles were
// bank conflicts). K's row r of step k is at r ^ 4 (k % 4), so that the staging's writes, four steps of four
// rows per 16 lanes, fall on distinct banks too.
#include <algorithm>
#include <type_traits>

#include "attn_fp8.h"

namespace lse {

constexpr int kF8TileWaves = 4;
constexpr int RB = 1;
constexpr int kF8TileRows = 32 * RB * kF8TileWaves;   // query rows of a workgroup
constexpr float kF8Lag = 8.0f;     // log2 of how far probabilities may exceed 1
constexpr float kF8Far = 16384.0f;  // |m| from which scaled scores are rounded before m is subtracted

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

__device__ __forceinline__ int f8_wave_sum(int v) {
  return __builtin_amdgcn_readlane(kv_wave_scan(v), 63);
}

// The item of rank p among the row tiles of all long entries, furthest tiles (virtual tile index: the entry's
// offset in tiles + its tile) first. Entries are looked at 64 at a time, one per lane.
struct F8Item {
  int e, qt;
};
__device__ __forceinline__ F8Item f8_tile_item(const Fp8AttnArgs& a, int p) {
  const int lane = threadIdx.x & 63;
  auto entry = [&](int i, int& base, int& tiles) {
    base = tiles = 0;
    if (i >= a.entries) return;
    const int qlen = min(a.q_len[i], a.max_q_len);
    if (!f8_is_long(qlen, a.G)) return;
    tiles = (int)(((int64_t)qlen * a.G + kF8TileRows - 1) / kF8TileRows);
    base = (int)((int64_t)min(max(a.query_offset[i], 0), a.max_ctx) * a.G / kF8TileRows);
  };
  int base0, tiles0;
  entry(lane, base0, tiles0);
  // Tiles at level L or above it, over all entries.
  auto above = [&](int L) {
    int n = min(max(base0 + tiles0 - L, 0), tiles0);
    for (int e0 = 64; e0 < a.entries; e0 += 64) {
      int b, t;
      entry(e0 + lane, b, t);
      n += min(max(b + t - L, 0), t);
    }
    return f8_wave_sum(n);
  };
  if (above(0) <= p) return {-1, 0};
  int lo = 0, hi = 0x7ffffffe;  // above(lo) > p >= above(hi)
  {
    int top = base0 + tiles0;
    for (int e0 = 64; e0 < a.entries; e0 += 64) {
      int b, t;
      entry(e0 + lane, b, t);
      top = max(top, b + t);
    }
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) top = max(top, __shfl_xor(top, off));
    hi = __builtin_amdgcn_readfirstlane(top);
  }
  while (hi - lo > 1) {
    const int mid = lo + (hi - lo) / 2;
    if (above(mid) > p) lo = mid; else hi = mid;
  }
  p -= above(lo + 1);  // among the entries that have a tile at level lo
  for (int e0 = 0; e0 < a.entries; e0 += 64) {
    int b = base0, t = tiles0;
    if (e0) entry(e0 + lane, b, t);
    const int mine = t > 0 && b <= lo && lo < b + t;
    const int before = kv_wave_scan(mine) - mine;
    const unsigned long long hit = __ballot(mine && before == p);
    if (hit) {
      const int at = __ffsll(hit) - 1;
      return {e0 + at, lo - __builtin_amdgcn_readlane(b, at)};
    }
    p -= __builtin_amdgcn_readlane(before + mine, 63);
  }
  return {-1, 0};
}

template <int D>
__global__ void __launch_bounds__(64 * kF8TileWaves, 3 - RB) attn_fp8_tile_kernel(Fp8AttnArgs a) {
  constexpr int J = D / 64, KK = D / 16, DB = D / 32;
  constexpr int kSlot = 64 * D * 2;  // bytes of a K or V tile
  constexpr int P = D / 64;          // 16-byte pieces of a group a lane stages, of K and of V
  __shared__ __attribute__((aligned(16))) unsigned char lds[4 * kSlot];  // K, K, V, V

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n32 = lane & 31, half = lane >> 5;
  const int G = a.G, kvh = blockIdx.x % a.HKV;
  const F8Item item = f8_tile_item(a, blockIdx.x / a.HKV);
  if (item.e < 0) return;
  const int e = item.e;
  const int qlen = min(a.q_len[e], a.max_q_len), ctx = a.context_len[e];
  const int qo = a.query_offset[e], qs = a.q_start[e];
  const int rows = qlen * G, row0 = item.qt * kF8TileRows;
  const int last_tok = min(qlen - 1, (row0 + kF8TileRows - 1) / G);
  const int end_n = f8_end(a, qo, ctx, last_tok + 1);
  const int tiles = (end_n + 63) / 64;

  // The lane's rows and the last position each sees.
  int tok[RB], gq[RB], lim[RB];
  bool row_ok[RB];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const int r = row0 + 32 * RB * wave + 32 * rb + n32;
    tok[rb] = r / G;
    gq[rb] = r - tok[rb] * G;
    const int64_t row = (int64_t)qs + tok[rb];
    row_ok[rb] = r < rows && row >= 0 && row < a.tokens;
    lim[rb] = (int)min((int64_t)qo + tok[rb], (int64_t)end_n - 1);
  }
  // Keys up to here are seen by every row of the wave.
  const int all_see = (int)min((int64_t)qo + (row0 + 32 * RB * wave) / G, (int64_t)end_n - 1);

  // A negative softmax scale moves into Q, a zero one makes Q zero (exactly), so that a maximum can be
  // taken before the scaling.
  const float sc = a.scale_log2 == 0.0f ? 1.0f : __builtin_fabsf(a.scale_log2);
  bf16x8 qf[RB][KK];
  {
    const uint32_t flip = a.scale_log2 < 0.0f ? 0x80008000u : 0u;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const bool keep = row_ok[rb] && a.scale_log2 != 0.0f;
      const uint16_t* qp = a.q + (int64_t)(kvh * G + (row_ok[rb] ? gq[rb] : 0)) * a.sq_h +
                           (row_ok[rb] ? (int64_t)qs + tok[rb] : 0) * a.sq_t + 8 * half;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        const uint4 v = *reinterpret_cast<const uint4*>(qp + 16 * kk);
        qf[rb][kk] = as_bf16x8(keep ? make_uint4(v.x ^ flip, v.y ^ flip, v.z ^ flip, v.w ^ flip)
                                    : make_uint4(0, 0, 0, 0));
      }
    }
  }

  // The wave stages group `wave` of every tile. Lane i of 64 holds place (16-byte units) and scales of that
  // group in tile 64 w + i, for the window w of the tile to load and the one behind it.
  const int32_t* bt = a.block_table + (int64_t)e * a.sbt;
  const int per = a.pool.per, last_group = max(end_n - 1, 0) / kKvGroup;
  auto table_at = [&](int w, int& sub) {
    const int64_t first = 4 * ((int64_t)64 * w + lane) + wave;
    const int grp = (int)min(first, (int64_t)last_group);
    const int bi = per == 1 ? grp : grp / per;
    sub = grp - bi * per;
    return bt[bi];
  };
  auto place = [&](int blk, int sub, uint32_t& off) {
    const bool bad = blk < 0 || blk >= a.pool.blocks;
    blk = bad ? 0 : blk;
    const int inner = kvh * per + sub;
    off = (uint32_t)(((int64_t)blk * a.pool.sb + (int64_t)inner * (16 * D)) >> 4);
    const int s = *reinterpret_cast<const uint16_t*>(a.pool.scales + (int64_t)blk * a.pool.ss + 2 * inner);
    return bad ? 0xffff : s;
  };
  uint32_t off0 = 0, off1 = 0;
  int sc0 = 0, sc1 = 0, blk2 = 0, sub2 = 0;
  // The codes on their way to LDS, and their places and scales.
  uint4 kc[P], vc[P];
  uint32_t at_k = 0;
  int scale_k = 0, scale_v = 0, next_scale_v = 0;
  auto load_k = [&](int t) {
    at_k = __builtin_amdgcn_readlane(off0, t & 63);
    scale_k = __builtin_amdgcn_readlane(sc0, t & 63);
    const uint8_t* p = a.pool.k + ((uint64_t)at_k << 4);
#pragma unroll
    for (int i = 0; i < P; ++i) kc[i] = *reinterpret_cast<const uint4*>(p + 16 * lane + 1024 * i);
    if ((t & 63) == 63) {
      off0 = off1, sc0 = sc1;
      sc1 = place(blk2, sub2, off1);
      blk2 = table_at((t >> 6) + 3, sub2);
    }
  };
  // V of the tile whose K was loaded one call before.
  auto load_v = [&](uint32_t at, int s) {
    scale_v = s;
    const uint8_t* p = a.pool.v + ((uint64_t)at << 4);
#pragma unroll
    for (int i = 0; i < P; ++i) vc[i] = *reinterpret_cast<const uint4*>(p + 16 * lane + 1024 * i);
  };
  // Piece 64 i + lane of K: key 4 (p / (16 J)) + p / 4 % 4 of the group, dims 64 (p / 16 % J) + 16 (p % 4); its
  // place in a K tile, the key's row being its number with bits 2 and 3 exchanged.
  uint32_t kdst[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int p = 64 * i + lane, sq = p / (16 * J), sr = p / 4 % 4, kk = 4 * (p / 16 % J) + p % 4;
    const int r = 16 * (wave & 1) + 8 * (sq & 1) + 4 * (sq >> 1) + sr;
    kdst[i] = (kk * 2 + (wave >> 1)) * 1024 + (r ^ (4 * (kk & 3))) * 16;
  }
  const uint32_t vdst = 2 * kSlot + wave * D * 32 + lane * 16;
  // Half `h` of piece i: eight codes, as bf16.
  auto stage_k = [&](int i, int h, int slot) {
    const uint4 c = kc[i];
    const bf16x8 v = kv_decode8(h ? c.z : c.x, h ? c.w : c.y, kv_scale(scale_k & 255));
    *reinterpret_cast<uint4*>(lds + slot * kSlot + kdst[i] + 512 * h) = __builtin_bit_cast(uint4, v);
  };
  auto stage_v = [&](int i, int h, int slot) {
    const uint4 c = vc[i];
    const bf16x8 v = kv_decode8(h ? c.z : c.x, h ? c.w : c.y, kv_scale(scale_v >> 8 & 255));
    *reinterpret_cast<uint4*>(lds + slot * kSlot + vdst + 1024 * i + 16 * D * h) = __builtin_bit_cast(uint4, v);
  };
  // Slots of tile t past the last key hold anything: their codes become zeros, which 0 probabilities need.
  auto mask_v = [&](int t) {
    if (64 * t + 64 <= end_n) return;
    const int left = end_n - 64 * t - 16 * wave;
    auto mask = [&](int w) {
      const int nb = min(max(left - 4 * w, 0), 4);
      return nb == 4 ? 0xffffffffu : (1u << (8 * nb)) - 1u;
    };
    const uint32_t m0 = mask(0), m1 = mask(1), m2 = mask(2), m3 = mask(3);
#pragma unroll
    for (int i = 0; i < P; ++i) vc[i].x &= m0, vc[i].y &= m1, vc[i].z &= m2, vc[i].w &= m3;
  };

  // Fragment reads, relative to a slot.
  const unsigned char* kread[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) kread[i] = lds + (n32 ^ (4 * i)) * 16 + 512 * half;
  const unsigned char* vread = lds + 2 * kSlot + n32 * 16 + 16 * D * half;

  f32x16 oacc[RB][DB];
  f32x16 zero;
#pragma unroll
  for (int i = 0; i < 16; ++i) zero[i] = 0.0f;
#pragma unroll
  for (int rb = 0; rb < RB; ++rb)
#pragma unroll
    for (int d = 0; d < DB; ++d) oacc[rb][d] = zero;
  bf16x8 pa[RB][4];
  float m[RB], l[RB], mul = sc, sub[RB];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) m[rb] = -__builtin_huge_valf(), l[rb] = sub[rb] = 0.0f;

  typedef f32x16 Scores[RB][2];  // [row block][32-key block]
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  Scores cur, next;
  // Probabilities of scores i .. i + 1 of row block rb, rounded in eights, and their sum.
  auto exps = [&](int rb, int i) {
#pragma unroll
    for (int x = i; x < i + 2; ++x)
      cur[rb][x >> 4][x & 15] = exp2_fast(__builtin_fmaf(cur[rb][x >> 4][x & 15], mul, -sub[rb]));
    if ((i & 7) == 6) {
      f32x8 v;
#pragma unroll
      for (int x = 0; x < 8; ++x) v[x] = cur[rb][i >> 4][(i & 8) + x];
      bf16x8 p = __builtin_convertvector(v, bf16x8);
#pragma unroll
      for (int x = 0; x < 8; x += 2)
        l[rb] = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{p[x], p[x + 1]}, bf16x2{(__bf16)1.0f, (__bf16)1.0f},
                                                l[rb], false);
      // Here and below an empty statement keeps the compiler from moving work to where its result is used,
      // which is behind the MFMAs that it is to run beside.
      asm volatile("" : "+v"(p), "+v"(l[rb]));
      pa[rb][i >> 3] = p;
    }
  };
  constexpr int kAhead = 4;
  // K Q^T of the tile in `slot` into `next` (QK), between its MFMAs the probabilities of `cur` (EXP).
  auto scores = [&](auto QK, auto EXP, int slot) {
    constexpr int N = 2 * KK, E = 16 / N;  // fragments; pairs of exponentials beside an MFMA
    bf16x8 fr[kAhead];
    auto read = [&](int f) {
      return as_bf16x8(*reinterpret_cast<const uint4*>(kread[(f >> 1) & 3] + slot * kSlot + f * 1024));
    };
    if constexpr (QK.value) {
#pragma unroll
      for (int f = 0; f < kAhead; ++f) fr[f] = read(f);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int f = 0; f < N; ++f) {
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        if constexpr (QK.value)
          next[rb][f & 1] = f8_mfma32(fr[f % kAhead], qf[rb][f >> 1], f < 2 ? zero : next[rb][f & 1]);
        if constexpr (EXP.value) {
#pragma unroll
          for (int x = 0; x < E; ++x) {
            const int pair = (RB * f + rb) * E + x;
            exps(pair >> 4, 2 * (pair & 15));
          }
        }
        if (rb == RB - 1 && QK.value && f + kAhead < N) fr[f % kAhead] = read(f + kAhead);
        if constexpr (QK.value) __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  // P V of the tile in V slot `slot`, between its MFMAs `next` becomes `cur` with its maximum, and the staging
  // (MAX).
  float mx[RB];
  auto values = [&](auto MAX, int slot) {
    constexpr int N = 4 * DB;  // fragments
    constexpr int S = 32 / N;                   // scores whose maximum is taken beside an MFMA
    constexpr int kEvery = RB == 1 ? (N - 4) / (4 * P) : (2 * N - 8) / (4 * P), kFrom = 4 * RB;     // 4 P half pieces beside the MFMAs behind the first eight
    bf16x8 fr[kAhead];
    auto read = [&](int f) {
      return as_bf16x8(*reinterpret_cast<const uint4*>(vread + slot * kSlot + f / DB * (32 * D) + f % DB * 512));
    };
    for (int rb = 0; rb < RB; ++rb) mx[rb] = -__builtin_huge_valf();
#pragma unroll
    for (int f = 0; f < kAhead; ++f) fr[f] = read(f);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int f = 0; f < N; ++f) {
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        oacc[rb][f % DB] = f8_mfma32(fr[f % kAhead], pa[rb][f / DB], oacc[rb][f % DB]);
        const int u = RB * f + rb;
        if constexpr (MAX.value) {
#pragma unroll
          for (int x = 0; x < S; x += 2) {
            const int at = u * S + x, b = at >> 5, i = at & 31;
            cur[b][i >> 4][i & 15] = next[b][i >> 4][i & 15];
            cur[b][i >> 4][(i & 15) + 1] = next[b][i >> 4][(i & 15) + 1];
            mx[b] = fmaxf(fmaxf(mx[b], cur[b][i >> 4][i & 15]), cur[b][i >> 4][(i & 15) + 1]);
            asm volatile("" : "+v"(cur[b][i >> 4][i & 15]), "+v"(cur[b][i >> 4][(i & 15) + 1]), "+v"(mx[b]));
          }
          if (u >= kFrom && (u - kFrom) % kEvery == 0 && (u - kFrom) / kEvery < 4 * P) {
            const int hp = (u - kFrom) / kEvery;
            if (hp < 2 * P) stage_v(hp >> 1, hp & 1, slot ^ 1);
            else stage_k((hp - 2 * P) >> 1, hp & 1, slot);
          }
        }
        if (rb == RB - 1 && f + kAhead < N) fr[f % kAhead] = read(f + kAhead);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  auto maxima = [&] {
    for (int rb = 0; rb < RB; ++rb) mx[rb] = -__builtin_huge_valf();
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
#pragma unroll
      for (int i = 0; i < 32; ++i) mx[rb] = fmaxf(mx[rb], cur[rb][i >> 4][i & 15]);
  };
  // Hides the scores of tile t that a row does not see.
  auto hide = [&](int t) {
    if (64 * t + 63 <= all_see) return;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const int rel = lim[rb] - 64 * t - 8 * half;
#pragma unroll
      for (int i = 0; i < 32; ++i)
        cur[rb][i >> 4][i & 15] =
            16 * (i >> 3) + (i & 7) <= rel ? cur[rb][i >> 4][i & 15] : -__builtin_huge_valf();
    }
    maxima();
  };
  // The references m from the tile's maxima, O and sums rescaled where one moves.
  auto reference = [&] {
#pragma clang fp contract(off)  // the maximum is a rounded product wherever it is used
    bool far = false;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const F8Halves h = f8_halves(mx[rb]);
      const float top = fmaxf(h.a, h.b) * sc;
      const bool moves = top > m[rb] + kF8Lag;  // from -inf with the first key seen
      if (__ballot(moves)) {
        const float to = moves ? top : m[rb];
        const float alpha = moves ? exp2_fast(m[rb] - to) : 1.0f;
        m[rb] = to;
        l[rb] *= alpha;
#pragma unroll
        for (int d = 0; d < DB; ++d) oacc[rb][d] *= alpha;
      }
      sub[rb] = m[rb] == -__builtin_huge_valf() ? 0.0f : m[rb];  // a row with no key yet keeps p = 0
      far |= __builtin_fabsf(sub[rb]) > kF8Far;
    }
    mul = sc;
    if (__ballot(far)) {
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int i = 0; i < 32; ++i) cur[rb][i >> 4][i & 15] = cur[rb][i >> 4][i & 15] * sc - sub[rb];
      mul = 1.0f;
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) sub[rb] = 0.0f;
    }
  };
  const std::true_type on{};
  const std::false_type no{};

  if (tiles > 0) {
    {
      int sub0, sub1;
      const int blk0 = table_at(0, sub0), blk1 = table_at(1, sub1);
      blk2 = table_at(2, sub2);
      sc0 = place(blk0, sub0, off0);
      sc1 = place(blk1, sub1, off1);
    }
    load_k(0);
    load_v(at_k, scale_k);
#pragma unroll
    for (int i = 0; i < 2 * P; ++i) stage_k(i >> 1, i & 1, 0);
    load_k(1);
    uint32_t next_at_v = at_k;
    next_scale_v = scale_k;
    mask_v(0);
#pragma unroll
    for (int i = 0; i < 2 * P; ++i) stage_v(i >> 1, i & 1, 0);
    load_v(next_at_v, next_scale_v);
#pragma unroll
    for (int i = 0; i < 2 * P; ++i) stage_k(i >> 1, i & 1, 1);
    load_k(2);
    next_at_v = at_k, next_scale_v = scale_k;
    f8_barrier();
    scores(on, no, 0);
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) cur[rb][0] = next[rb][0], cur[rb][1] = next[rb][1];
    maxima();
    hide(0);
    reference();
    f8_barrier();

    // Tile j, its scores in cur with their reference; in LDS K of j + 1 and V of j, in registers the codes of K of
    // j + 2 and V of j + 1.
    int j = 0;
    for (; j + 1 < tiles; ++j) {
      scores(on, on, (j + 1) & 1);
      mask_v(j + 1);
      values(on, j & 1);
      load_v(next_at_v, next_scale_v);
      load_k(j + 3);
      next_at_v = at_k, next_scale_v = scale_k;
      hide(j + 1);
      reference();
      f8_barrier();
    }
    scores(no, on, 0);
    values(no, j & 1);
  }

#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const F8Halves h = f8_halves(l[rb]);
    const float sum = h.a + h.b, inv = sum == 0.0f ? 0.0f : 1.0f / sum;  // no key: zeros
    if (!row_ok[rb]) continue;
    uint16_t* out = a.o + (int64_t)(kvh * G + gq[rb]) * a.so_h + ((int64_t)qs + tok[rb]) * a.so_t + 4 * half;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int b = 0; b < 4; ++b)
        *reinterpret_cast<uint2*>(out + 32 * d + 8 * b) =
            make_uint2(pack_bf16x2(oacc[rb][d][4 * b] * inv, oacc[rb][d][4 * b + 1] * inv),
                       pack_bf16x2(oacc[rb][d][4 * b + 2] * inv, oacc[rb][d][4 * b + 3] * inv));
  }
}

int launch_fp8_attn_tile(const Fp8AttnArgs& a, int64_t D, hipStream_t stream) {
  // Every long entry's rows round up to a tile; a long entry has at least kF8LongRows rows.
  const int64_t rows = (int64_t)a.tokens * a.G;
  const int64_t entries = std::min<int64_t>(a.entries, rows / kF8LongRows);
  const int64_t blocks = (rows / kF8TileRows + entries) * a.HKV;
  if (blocks <= 0) return LSE_OK;
  if (blocks > 0x7fffffff) return LSE_E_RANGE;
  const dim3 grid((unsigned)blocks), wg(64 * kF8TileWaves);
  if (D == 64)
    hipLaunchKernelGGL(attn_fp8_tile_kernel<64>, grid, wg, 0, stream, a);
  else
    hipLaunchKernelGGL(attn_fp8_tile_kernel<128>, grid, wg, 0, stream, a);
  return launch_status();
}

}  // namespace lse
