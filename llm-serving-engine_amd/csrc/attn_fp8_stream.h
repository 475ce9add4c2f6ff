// Paged attention over the 8-bit K/V cache (fp8_kv.h), of decode rows and short prompt chunks: the key-
// streaming kernel. The semantics are attention.hip's, with k and v the values that codes and scales stand for:
//   o[h][q_start + m] = sum_n softmax_n(scale * q . k_n) v_n  over n < context_len, n <= query_offset + m.
// Softmax in fp32, online; probabilities rounded to bf16 before the product with V, as they are there (the
// matrix cores' operand type), sums of them before the rounding; fp32 accumulation, output rounded once.
//
// What bounds it is the cache's bytes, half of bf16's. The layout lets both operands of the matrix cores come
// from memory as they are: per 64 keys, which are four groups of 16, a wave loads
//  * K: 16 keys x 64 contiguous dims an instruction, lane (i, g) bytes 16 g.. of key (group i / 4, slot 4 b + i %
//    4): rows i of the A operand of S^T = K Q^T, so that lane (i, g) of the result holds the scores of row i of
//    Q with all 16 keys of group g;
//  * V: one dim of the 16 keys of group g a lane, which is the A operand of O^T += V^T P^T for exactly these
//    keys, P^T coming out of the scores in the lane that holds them.
// Neither K, V nor P passes through LDS, and waves do not wait for each other before the end. O^T's column is
// the lane's row of Q again, so the softmax's factors are per-lane scalars. Codes become bf16 in registers,
// times their scale, at two values an instruction.
//
// Wave w of the four takes the tiles of 64 keys w, w + 4, w + 8, ... with an online-softmax state of its own; the four
// are merged in wave order at the end. Where a call has fewer (entry, K/V head, query tile) items than the card
// takes workgroups, the keys are split too (f8_unit): into ranges of one length for all entries, chosen so
// that all ranges run at once, each leaving its state to a second kernel. With ranges of a fixed 1024 or 2048
// keys, four sequences behind 7500 to 60000 positions took 44 + 7 us.
//
// On MI355X, bytes of the cache over the kernel's time: 64 sequences behind 256 to 2048 positions, 8 K/V heads of 128,
// 25.4 us, 5.2 TB/s; heads of 64 behind 2048 to 16384, 95 us, 6.0 TB/s; four behind 15000 to 32000, 35.3 us, 5.9 TB/s,
// and 4.6 us to add the ranges up; one behind 467 positions 6.1 us, all latency.
#pragma once

#include "attn_fp8.h"

namespace lse {

constexpr int kF8Waves = 4;
constexpr int kF8Keys = 64;      // keys of a wave's tile: one group per 16 lanes
constexpr int kF8Round = kF8Keys * kF8Waves;
constexpr int kF8Window = 4 * kF8Round;  // keys of four tiles of every wave, whose blocks and scales it holds
// Workgroups of a split launch, two per CU: for heads of 128 all there is room for (204 registers; with 168, three, the
// kernel spills: four sequences behind 7500 to 60000 positions 42 -> 54 us), and with twice as many, half of them wait
// (48 us). Heads of 64 have room for twice as many, which gains 3 to 10 % where ranges are short (16 sequences behind
// 2000 to 8192 positions 21.0 -> 20.4 us, 32 37.7 -> 35.1) and loses 10 to 15 % where they are long (4 behind 24000 to 60000
// 34.0 -> 39.1, 16 behind 4000 to 32768 56 -> 62), so it is the same for both.
constexpr int kF8Groups = 512;
// Fewest keys of a range, and contexts up to which nothing is split: a wave takes 0.5 us a tile, the second
// kernel 4 us and more.
constexpr int kF8MinRange = 1024, kF8MinSplit = 2048;

// The four waves' states of a row merged in wave order.
struct WaveFactors {
  float f[kF8Waves], m, sum;
};
__device__ __forceinline__ WaveFactors f8_merge_factors(const float (&m)[kF8Waves],
                                                        const float (&l)[kF8Waves]) {
  WaveFactors r;
  r.m = kNegInf, r.sum = 0.0f;
#pragma unroll
  for (int w = 0; w < kF8Waves; ++w) r.m = fmaxf(r.m, m[w]);
  const float ref = r.m == kNegInf ? 0.0f : r.m;
#pragma unroll
  for (int w = 0; w < kF8Waves; ++w) {
    r.f[w] = exp2_fast(m[w] - ref);
    r.sum = __builtin_fmaf(l[w], r.f[w], r.sum);
  }
  return r;
}
__device__ __forceinline__ float f8_inverse(float sum) {
  return sum == 0.0f ? 0.0f : 1.0f / sum;  // a row that saw no key gives zeros
}

// The entry of rank `slot` by context length, longest first (attention.hip's attn_sorted_entry has the
// reasons); at most 64 entries, one per lane.
__device__ __forceinline__ int f8_sorted_entry(const Fp8AttnArgs& a, int slot) {
  const int lane = threadIdx.x & 63;
  int key = -1;
  if (lane < a.entries)
    key = ((a.q_len[lane] <= 0 ? 0 : 1 + min(max(a.context_len[lane], 0), (1 << 24) - 1)) << 6) + 63 - lane;
  int rank = 0;
#pragma unroll
  for (int j = 0; j < 64; ++j) rank += __builtin_amdgcn_readlane(key, j) > key;
  if (a.first_round > 0 && slot >= a.first_round) slot = a.first_round + a.entries - 1 - slot;
  return __ffsll(__ballot(rank == slot && lane < a.entries)) - 1;
}

// The units of a launch that counts them: entry by entry, its query tiles times its key ranges (the tiles that
// read a range together).
struct F8Unit {
  int e, qt, part, parts, tiles, first;  // first: number of the entry's first unit; e < 0: no such unit
  int qlen, ctx, qo, qs;
  int64_t range;                         // keys of a range
};
struct F8Work {
  int tiles, end, qlen, ctx, qo, qs;
};
__device__ __forceinline__ F8Work f8_entry_work(const Fp8AttnArgs& a, int i) {
  F8Work w{0, 0, 0, 0, 0, 0};
  if (i >= a.entries) return w;
  w.qlen = min(a.q_len[i], a.max_q_len), w.ctx = a.context_len[i];
  w.qo = a.query_offset[i], w.qs = a.q_start[i];
  if (w.qlen <= 0 || (a.tiled && f8_is_long(w.qlen, a.G))) return w;
  w.tiles = (w.qlen + a.tq - 1) / a.tq;
  w.end = f8_end(a, w.qo, w.ctx, w.qlen);
  return w;
}

// Unit b, or (of_entry) the first of entry b's. Every wave counts for itself, 64 entries at a time.
__device__ __forceinline__ F8Unit f8_unit(const Fp8AttnArgs& a, int b, bool of_entry) {
  const int lane = threadIdx.x & 63;
  const F8Work w0 = f8_entry_work(a, lane);
  int64_t range = (int64_t)1 << 40;
  if (a.slots > 0) {
    // With ranges of W / (slots - T) keys, T tiles of W keys in all (each counted as often as it has tiles) make up
    // at most slots units.
    int T = 0, W = 0;
    for (int e0 = 0; e0 < a.entries; e0 += 64) {
      const F8Work w = e0 ? f8_entry_work(a, e0 + lane) : w0;
      T += f8_wave_total(min(w.tiles, kF8Groups));
      W += f8_wave_total(min(w.tiles, kF8Groups) * min((w.end + kF8Round - 1) / kF8Round, 1 << 15));
      if (T >= a.slots) break;
    }
    if (T < a.slots)
      range = max((int64_t)kF8Round * ((W + a.slots - T - 1) / (a.slots - T)), (int64_t)kF8MinRange);
    // So long a context that its length above was cut, or so many units: no more ranges than slots.
    while (T < a.slots) {
      int n = 0;
      for (int e0 = 0; e0 < a.entries; e0 += 64) {
        const F8Work w = e0 ? f8_entry_work(a, e0 + lane) : w0;
        n += f8_wave_total(w.tiles * max((int)min((w.end + range - 1) / range, (int64_t)kF8Groups), 1));
      }
      if (n <= a.slots) break;
      range *= 2;
    }
  }
  int before0 = 0;
  for (int e0 = 0; e0 < a.entries; e0 += 64) {
    const F8Work w = e0 ? f8_entry_work(a, e0 + lane) : w0;
    const int parts = max((int)((w.end + range - 1) / range), 1);
    const int units = w.tiles * parts, before = before0 + kv_wave_scan(units) - units;
    const unsigned long long hit = __ballot(of_entry ? e0 + lane == b && units > 0
                                                     : (unsigned)(b - before) < (unsigned)units);
    if (hit) {
      const int at = __ffsll(hit) - 1;
      F8Unit u;
      u.e = e0 + at;
      u.first = __builtin_amdgcn_readlane(before, at);
      u.tiles = __builtin_amdgcn_readlane(w.tiles, at);
      u.parts = __builtin_amdgcn_readlane(parts, at);
      u.range = range;
      u.qlen = __builtin_amdgcn_readlane(w.qlen, at);
      u.ctx = __builtin_amdgcn_readlane(w.ctx, at);
      u.qo = __builtin_amdgcn_readlane(w.qo, at);
      u.qs = __builtin_amdgcn_readlane(w.qs, at);
      const int i = of_entry ? 0 : b - u.first;
      u.qt = i % u.tiles;
      u.part = i / u.tiles;
      return u;
    }
    before0 = __builtin_amdgcn_readlane(before + units, 63);
  }
  return {-1, 0, 0, 1, 0, 0, 0, 0, 0, 0, range};
}

// NT: K and V stream with the nt cache policy, where each is read by one workgroup only (one query tile: decode).
// COUNT: workgroups find their unit (f8_unit); otherwise the grid is K/V heads, then entries of one tile.
// `lds`: f8_stream_lds(D) bytes.
constexpr int f8_stream_lds(int D) { return kF8Waves * 16 * (D + 4 + 2) * 4; }
template <int D, bool NT, bool COUNT>
__device__ __forceinline__ void f8_stream(const Fp8AttnArgs& a, int block, unsigned char* lds) {
  constexpr int J = D / 64, DT = D / 16;  // 64-dim runs of a key; 16-dim tiles of O
  constexpr int OROW = D + 4;             // floats of a row of O in LDS: rows start on other banks
  float(*obuf)[16 * OROW] = reinterpret_cast<float(*)[16 * OROW]>(lds);
  float(*mbuf)[16] = reinterpret_cast<float(*)[16]>(lds + kF8Waves * 16 * OROW * 4);
  float(*lbuf)[16] = mbuf + kF8Waves;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n16 = lane & 15, g = lane >> 4;

  const int kvh = block % a.HKV, slot = block / a.HKV;
  int e, qt = 0, parts = 1, qlen, ctx, qo, qs;
  int64_t first_key = 0, end_key = (int64_t)1 << 40;
  if constexpr (COUNT) {
    const F8Unit u = f8_unit(a, slot, false);
    if (u.e < 0) return;
    e = u.e, qt = u.qt, parts = u.parts, qlen = u.qlen, ctx = u.ctx, qo = u.qo, qs = u.qs;
    first_key = u.part * u.range, end_key = first_key + u.range;
  } else {
    e = a.sorted ? f8_sorted_entry(a, slot) : slot;
    qlen = min(a.q_len[e], a.max_q_len), ctx = a.context_len[e], qo = a.query_offset[e], qs = a.q_start[e];
  }
  if (qt * a.tq >= qlen) return;
  int end_n = f8_end(a, qo, ctx, min(qlen, (qt + 1) * a.tq));
  if (first_key > 0 && first_key >= end_n) return;  // the tile has no keys in this range
  end_n = (int)min((int64_t)end_n, end_key);
  // The wave's windows: tile t of the j-th has keys 1024 j + 256 t + 64 wave on, from the range's first.
  auto win = [&](int j) -> int64_t { return first_key + (int64_t)j * kF8Window + kF8Keys * wave; };

  // This lane's row: token tq, head gq of the group; rows from tq G on are idle (G not dividing 16).
  const int G = a.G;
  const int tok = n16 / G, m_row = qt * a.tq + tok, head = kvh * G + n16 - tok * G;
  const int64_t row = (int64_t)qs + m_row;
  const bool row_ok = n16 < a.tq * G && m_row < qlen && row >= 0 && row < a.tokens;
  const int lim = min((int)min((int64_t)qo + m_row, (int64_t)0x7ffffffe), end_n - 1);
  // Keys up to here are seen by every row of the tile.
  const int all_see = min((int)min((int64_t)qo + qt * a.tq, (int64_t)0x7ffffffe), end_n - 1);

  bf16x8 qf[J][2];
  {
    const uint16_t* qp = a.q + (int64_t)(row_ok ? head : 0) * a.sq_h + (row_ok ? row : 0) * a.sq_t + 16 * g;
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4 v = *reinterpret_cast<const uint4*>(qp + 64 * j + 8 * h);
        qf[j][h] = as_bf16x8(row_ok ? v : make_uint4(0, 0, 0, 0));
      }
  }

  // Blocks and scales of the wave's windows: lane i of 16 holds those of group i % 4 of its tile i / 4. `off` is the
  // group's place in the pool in 16-byte units; a block that is not the pool's reads block 0 with NaN for a scale.
  const int32_t* bt = a.block_table + (int64_t)e * a.sbt;
  const int last_group = (end_n - 1) / kKvGroup;
  const int per = a.pool.per;
  auto table_at = [&](int j, int& sub) {
    const int64_t first = (win(j) + kF8Round * (n16 >> 2)) / kKvGroup + (n16 & 3);
    const int grp = (int)min(first, (int64_t)last_group);
    const int bi = per == 1 ? grp : grp / per;
    sub = grp - bi * per;
    return bt[bi];
  };
  auto place = [&](int blk, int sub, uint32_t& off, int& bad) {
    bad = blk < 0 || blk >= a.pool.blocks;
    blk = bad ? 0 : blk;
    const int inner = kvh * per + sub;
    off = (uint32_t)(((int64_t)blk * a.pool.sb + (int64_t)inner * (16 * D)) >> 4);
    return (int)*reinterpret_cast<const uint16_t*>(a.pool.scales + (int64_t)blk * a.pool.ss + 2 * inner);
  };

  uint4 kr[4][J], vr[DT];
  auto load_k = [&](uint32_t off, int t) {
    const uint32_t at = __shfl(off, 4 * t + (n16 >> 2));
    const uint8_t* p = a.pool.k + ((uint64_t)at << 4) + (n16 & 3) * 64 + 16 * g;
#pragma unroll
    for (int bk = 0; bk < 4; ++bk)
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const uint8_t* src = p + (bk * J + j) * 256;
        kr[bk][j] = NT ? load16_stream(src) : *reinterpret_cast<const uint4*>(src);
      }
  };
  auto load_v = [&](uint32_t off, int t) {
    const uint32_t at = __shfl(off, 4 * t + g);
    const uint8_t* p = a.pool.v + ((uint64_t)at << 4) + 16 * n16;
#pragma unroll
    for (int i = 0; i < DT; ++i) {
      const uint8_t* src = p + i * 256;
      vr[i] = NT ? load16_stream(src) : *reinterpret_cast<const uint4*>(src);
    }
  };

  float m_run = kNegInf, l_run = 0.0f;
  f32x4 oacc[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) oacc[t] = f32x4{0, 0, 0, 0};

  if (win(0) < end_n) {
    // Window j's off and scales, window j + 1's off (and its scales on their way), window j + 2's block.
    int sub0, sub1, sub2, bad0, bad1;
    uint32_t off0, off1;
    const int blk0 = table_at(0, sub0), blk1 = table_at(1, sub1);
    int blk2 = table_at(2, sub2);
    int sc0 = place(blk0, sub0, off0, bad0);
    load_k(off0, 0);
    load_v(off0, 0);
    int sc1 = place(blk1, sub1, off1, bad1);
    if (bad0) sc0 = 0xffff;

    for (int j = 0;;) {
      const int64_t start = win(j);
      const int tiles = (int)min((int64_t)4, (end_n - start + kF8Round - 1) / kF8Round);
      const bool more = win(j + 1) < end_n;
      for (int t = 0; t < tiles; ++t) {
        const int n0 = (int)start + kF8Round * t;
        const bool last = t + 1 == tiles;
        // The scores of key n0 + 16 g + 4 bk + r and row n16.
        const float ks = kv_scale(__shfl(sc0, 4 * t + (n16 >> 2)) & 255);
        const float vs = kv_scale(__shfl(sc0, 4 * t + g) >> 8 & 255);
        f32x4 st[4];
#pragma unroll
        for (int bk = 0; bk < 4; ++bk) {
          st[bk] = f32x4{0, 0, 0, 0};
#pragma unroll
          for (int c = 0; c < J; ++c) {
            st[bk] = mfma16x16x32(kv_decode8(kr[bk][c].x, kr[bk][c].y, ks), qf[c][0], st[bk]);
            st[bk] = mfma16x16x32(kv_decode8(kr[bk][c].z, kr[bk][c].w, ks), qf[c][1], st[bk]);
          }
        }
        // The next tile's K travels during the softmax and P V, its V from P V on; behind the last tile
        // this one is read again, which keeps the loads unconditional and their waits exact.
        const uint32_t next_off = last && more ? off1 : off0;
        const int next_t = last ? (more ? 0 : t) : t + 1;
        load_k(next_off, next_t);
        float s[16], tmax = kNegInf;
        if (n0 + kF8Keys - 1 > all_see) {
          const int rel = lim - n0 - 16 * g;
#pragma unroll
          for (int i = 0; i < 16; ++i) s[i] = i <= rel ? st[i >> 2][i & 3] * a.scale_log2 : kNegInf;
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) s[i] = st[i >> 2][i & 3] * a.scale_log2;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) tmax = fmaxf(tmax, s[i]);
        tmax = fmaxf(tmax, __shfl_xor(tmax, 16));
        tmax = fmaxf(tmax, __shfl_xor(tmax, 32));
        const float m_new = fmaxf(m_run, tmax);
        const float ref = m_new == kNegInf ? 0.0f : m_new;  // a row with no key yet keeps p = 0
        const float alpha = exp2_fast(m_run - ref);
        float sum = 0.0f;
        f32x8 p0, p1;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float p = exp2_fast(s[i] - ref);
          sum += p;
          if (i < 8) p0[i] = p; else p1[i - 8] = p;
        }
        l_run = __builtin_fmaf(l_run, alpha, sum);  // this lane's keys; its row's others' at the end
        if (__ballot(m_new != m_run)) {
#pragma unroll
          for (int d = 0; d < DT; ++d) oacc[d] *= alpha;
        }
        m_run = m_new;
        const bf16x8 pa = __builtin_convertvector(p0, bf16x8), pb = __builtin_convertvector(p1, bf16x8);
        // Slots past the last key hold anything: their codes become zeros, which 0 probabilities need.
        if (n0 + kF8Keys > end_n) {
          const int left = end_n - n0 - 16 * g;
          auto mask = [&](int w) {
            const int nb = min(max(left - 4 * w, 0), 4);
            return nb == 4 ? 0xffffffffu : (1u << (8 * nb)) - 1u;
          };
          const uint32_t m0 = mask(0), m1 = mask(1), m2 = mask(2), m3 = mask(3);
#pragma unroll
          for (int d = 0; d < DT; ++d)
            vr[d].x &= m0, vr[d].y &= m1, vr[d].z &= m2, vr[d].w &= m3;
        }
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          oacc[d] = mfma16x16x32(kv_decode8(vr[d].x, vr[d].y, vs), pa, oacc[d]);
          oacc[d] = mfma16x16x32(kv_decode8(vr[d].z, vr[d].w, vs), pb, oacc[d]);
        }
        load_v(next_off, next_t);
      }
      if (!more) break;
      ++j;
      off0 = off1, sc0 = bad1 ? 0xffff : sc1;
      sc1 = place(blk2, sub2, off1, bad1);
      blk2 = table_at(j + 2, sub2);
    }
  }

  // Lane (n16, g) holds row n16's dims 16 t + 4 g + r.
  l_run += __shfl_xor(l_run, 16);
  l_run += __shfl_xor(l_run, 32);
  if (g == 0) mbuf[wave][n16] = m_run, lbuf[wave][n16] = l_run;
#pragma unroll
  for (int t = 0; t < DT; ++t)
    *reinterpret_cast<float4*>(&obuf[wave][n16 * OROW + 16 * t + 4 * g]) =
        make_float4(oacc[t][0], oacc[t][1], oacc[t][2], oacc[t][3]);
  __syncthreads();
  if (threadIdx.x >= 16 * (D / 8)) return;
  const int orow = threadIdx.x / (D / 8), c8 = 8 * (threadIdx.x % (D / 8));
  const int otok = orow / G, om = qt * a.tq + otok;
  const int64_t out_row = (int64_t)qs + om;
  if (orow >= a.tq * G || om >= qlen || out_row < 0 || out_row >= a.tokens) return;
  float m[kF8Waves], l[kF8Waves], o[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
  for (int w = 0; w < kF8Waves; ++w) m[w] = mbuf[w][orow], l[w] = lbuf[w][orow];
  const WaveFactors f = f8_merge_factors(m, l);
#pragma unroll
  for (int w = 0; w < kF8Waves; ++w)
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = __builtin_fmaf(obuf[w][orow * OROW + c8 + i], f.f[w], o[i]);
  if (COUNT && parts > 1) {
    const int64_t at = ((int64_t)slot * a.HKV + kvh) * 16 + orow;
    *reinterpret_cast<float4*>(a.ws_o + at * D + c8) = make_float4(o[0], o[1], o[2], o[3]);
    *reinterpret_cast<float4*>(a.ws_o + at * D + c8 + 4) = make_float4(o[4], o[5], o[6], o[7]);
    if (c8 == 0) *reinterpret_cast<float2*>(a.ws_ml + 2 * at) = make_float2(f.m, f.sum);
    return;
  }
  const float inv = f8_inverse(f.sum);
  *reinterpret_cast<uint4*>(a.o + (int64_t)(kvh * G + orow - otok * G) * a.so_h + out_row * a.so_t + c8) =
      make_uint4(pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv),
                 pack_bf16x2(o[4] * inv, o[5] * inv), pack_bf16x2(o[6] * inv, o[7] * inv));
}

}  // namespace lse
