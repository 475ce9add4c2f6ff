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
// takes workgroups, the keys are split too (f8_units): into ranges of one length for all entries, chosen so
// that all ranges run at once, each leaving its state to a second kernel. With ranges of a fixed 1024 or 2048
// keys, four sequences behind 7500 to 60000 positions took 44 + 7 us.
#include <algorithm>

#include "attn_fp8.h"

namespace lse {

constexpr int kF8Waves = 4;
constexpr int kF8Keys = 64;      // keys of a wave's tile: one group per 16 lanes
constexpr int kF8Round = kF8Keys * kF8Waves;
constexpr int kF8Window = 4 * kF8Round;  // keys of four tiles of every wave, whose blocks and scales it holds
constexpr int kF8Groups = 512;   // workgroups of a split launch: two per CU
// Fewest keys of a range, and contexts up to which nothing is split: a wave takes 0.5 us a tile, the second
// kernel 4 us and more.
constexpr int kF8MinRange = 1024, kF8MinSplit = 2048;
constexpr float kNegInf = -__builtin_huge_valf();

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
  int64_t range;                         // keys of a range
};
struct F8Work {
  int tiles, end;
};
__device__ __forceinline__ F8Work f8_entry_work(const Fp8AttnArgs& a, int i) {
  if (i >= a.entries) return {0, 0};
  const int qlen = min(a.q_len[i], a.max_q_len);
  if (qlen <= 0 || (a.tiled && f8_is_long(qlen, a.G))) return {0, 0};
  return {(qlen + a.tq - 1) / a.tq, f8_end(a, a.query_offset[i], a.context_len[i], qlen)};
}
__device__ __forceinline__ int f8_wave_total(int v) { return __builtin_amdgcn_readlane(kv_wave_scan(v), 63); }

// Unit b, or (of_entry) the units of entry b. Every wave counts for itself, 64 entries at a time.
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
      const int i = of_entry ? 0 : b - u.first;
      u.qt = i % u.tiles;
      u.part = i / u.tiles;
      return u;
    }
    before0 = __builtin_amdgcn_readlane(before + units, 63);
  }
  return {-1, 0, 0, 1, 0, 0, range};
}

// NT: K and V stream with the nt cache policy, where each is read by one workgroup only (one query tile: decode).
// COUNT: workgroups find their unit (f8_unit); otherwise the grid is K/V heads, then entries of one tile.
template <int D, bool NT, bool COUNT>
__global__ void __launch_bounds__(64 * kF8Waves, 2) attn_fp8_kernel(Fp8AttnArgs a) {
  constexpr int J = D / 64, DT = D / 16;  // 64-dim runs of a key; 16-dim tiles of O
  constexpr int OROW = D + 4;             // floats of a row of O in LDS: rows start on other banks
  __shared__ __attribute__((aligned(16))) float obuf[kF8Waves][16 * OROW];
  __shared__ float mbuf[kF8Waves][16], lbuf[kF8Waves][16];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n16 = lane & 15, g = lane >> 4;

  const int kvh = blockIdx.x % a.HKV, slot = blockIdx.x / a.HKV;
  int e, qt = 0, parts = 1;
  int64_t first_key = 0, end_key = (int64_t)1 << 40;
  if constexpr (COUNT) {
    const F8Unit u = f8_unit(a, slot, false);
    if (u.e < 0) return;
    e = u.e, qt = u.qt, parts = u.parts;
    first_key = u.part * u.range, end_key = first_key + u.range;
  } else {
    e = a.sorted ? f8_sorted_entry(a, slot) : slot;
  }
  const int qlen = min(a.q_len[e], a.max_q_len);
  if (qt * a.tq >= qlen) return;
  const int ctx = a.context_len[e], qo = a.query_offset[e], qs = a.q_start[e];
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

// Second pass of a split launch, a workgroup per query tile, K/V head and 64 (row, 4 dims) pieces: wave w adds up the
// states of ranges w, w + 4, ..., then the four are merged. Bound by latency: a thread's loads, eight ranges at
// a time, do not wait for each other.
template <int D>
__global__ void __launch_bounds__(64 * kF8Waves) attn_fp8_merge(Fp8AttnArgs a) {
  __shared__ float obuf[kF8Waves][64][5];
  __shared__ float mbuf[kF8Waves][64], lbuf[kF8Waves][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int kvh = blockIdx.x % a.HKV;
  int e = blockIdx.x / a.HKV;
  const int qt = blockIdx.z;
  const F8Unit u = f8_unit(a, e, true);
  if (u.e < 0 || u.parts <= 1 || qt >= u.tiles) return;
  const int qlen = min(a.q_len[e], a.max_q_len), G = a.G;
  const int piece = blockIdx.y * 64 + lane, orow = piece / (D / 4), c4 = 4 * (piece % (D / 4));
  const int otok = orow / G, om = qt * a.tq + otok;
  const int64_t row = (int64_t)a.q_start[e] + om;
  const bool ok = orow < a.tq * G && om < qlen && row >= 0 && row < a.tokens;
  const int end_n = f8_end(a, a.query_offset[e], a.context_len[e], min(qlen, (qt + 1) * a.tq));
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
      for (int i = 0; i < 8; ++i) {
        const bool real = p0 + kF8Waves * i < n;
        const float m = real ? ml[i].x : kNegInf, mn = fmaxf(M, m), ref = mn == kNegInf ? 0.0f : mn;
        const float fa = exp2_fast(M - ref), fb = exp2_fast(m - ref);
        L = __builtin_fmaf(real ? ml[i].y : 0.0f, fb, L * fa);
        O[0] = __builtin_fmaf(real ? v[i].x : 0.0f, fb, O[0] * fa);
        O[1] = __builtin_fmaf(real ? v[i].y : 0.0f, fb, O[1] * fa);
        O[2] = __builtin_fmaf(real ? v[i].z : 0.0f, fb, O[2] * fa);
        O[3] = __builtin_fmaf(real ? v[i].w : 0.0f, fb, O[3] * fa);
        M = mn;
      }
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

// ---- host side -----------------------------------------------------------------------------

struct Fp8AttnPlan {
  int tq;
  bool tiled;       // some entry may be the row-tiled kernel's
  int64_t short_q;  // the most tokens of an entry that is not
  int64_t tiles;    // query tiles of all entries, at most
  int slots;        // units of a split launch, 0: keys are not split
  int64_t ws_o_bytes, ws_bytes;
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

// One workgroup per (entry, K/V head, query tile) once those fill the card; otherwise, where contexts may be long
// enough, the keys are split as well.
static Fp8AttnPlan fp8_attn_plan(int64_t entries, int64_t tokens, int64_t H, int64_t HKV, int64_t D,
                                 int64_t max_q_len, int64_t max_ctx) {
  Fp8AttnPlan pl{};
  const int64_t G = H / HKV;
  pl.tq = (int)(16 / G);
  pl.tiled = f8_is_long(max_q_len, (int)G);
  pl.short_q = pl.tiled ? (kF8LongRows - 1) / G : max_q_len;
  pl.tiles = std::min(entries * ceil_div(pl.short_q, (int64_t)pl.tq), tokens / pl.tq + entries);
  const int64_t slots = kF8Groups / HKV;
  if (pl.tiles < slots && max_ctx > kF8MinSplit) {
    pl.slots = (int)slots;
    pl.ws_o_bytes = slots * HKV * 16 * D * 4;
    pl.ws_bytes = pl.ws_o_bytes + slots * HKV * 16 * 2 * 4;
  }
  return pl;
}

template <int D>
static int launch_fp8_attention(const Fp8AttnArgs& a, const Fp8AttnPlan& pl, hipStream_t stream) {
  const dim3 wg(64 * kF8Waves);
  if (a.tiled)
    if (int st = launch_fp8_attn_tile(a, D, stream)) return st;
  const bool one = pl.short_q <= pl.tq;
  const dim3 grid((unsigned)((pl.slots ? pl.slots : one ? a.entries : pl.tiles) * a.HKV));
  if (!one)
    hipLaunchKernelGGL((attn_fp8_kernel<D, false, true>), grid, wg, 0, stream, a);
  else if (pl.slots)
    hipLaunchKernelGGL((attn_fp8_kernel<D, true, true>), grid, wg, 0, stream, a);
  else
    hipLaunchKernelGGL((attn_fp8_kernel<D, true, false>), grid, wg, 0, stream, a);
  if (int st = launch_status()) return st;
  if (pl.slots) {
    const int64_t rows = std::min<int64_t>(pl.short_q, pl.tq) * a.G;
    const dim3 pieces((unsigned)(a.entries * a.HKV), (unsigned)ceil_div(rows * (D / 4), 64),
                      (unsigned)ceil_div(pl.short_q, (int64_t)pl.tq));
    hipLaunchKernelGGL(attn_fp8_merge<D>, pieces, wg, 0, stream, a);
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
  return x.block_size > kMax31 || x.max_blocks > kMax31 / x.block_size ? LSE_E_RANGE : LSE_OK;
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
  lse::Fp8AttnArgs a{};
  a.q = (const uint16_t*)x.q, a.sq_h = x.q_stride_h, a.sq_t = x.q_stride_t;
  a.pool = {(uint8_t*)x.k_pool, (uint8_t*)x.v_pool, (uint8_t*)x.scales, x.pool_stride_block,
            x.scales_stride_block, (int)x.num_blocks, (int)per};
  a.block_table = x.block_table, a.sbt = x.block_table_stride;
  a.context_len = x.context_len, a.query_offset = x.query_offset, a.q_start = x.q_start, a.q_len = x.q_len;
  a.o = (uint16_t*)x.o, a.so_h = x.o_stride_h, a.so_t = x.o_stride_t;
  a.entries = (int)x.entries, a.H = (int)x.H, a.HKV = (int)x.H_KV, a.G = (int)(x.H / x.H_KV);
  a.tokens = (int)x.tokens;
  a.max_ctx = (int)(x.max_blocks * x.block_size);
  a.max_q_len = (int)x.max_q_len, a.tiled = pl.tiled, a.tq = pl.tq, a.slots = pl.slots;
  a.scale_log2 = (float)x.softmax_scale * 1.4426950408889634f;
  a.ws_o = pl.slots ? (float*)workspace : nullptr;
  a.ws_ml = pl.slots ? (float*)((char*)workspace + pl.ws_o_bytes) : nullptr;
  const int64_t items = x.entries * x.H_KV;
  a.sorted = x.entries <= 64 && items > cus && a.max_ctx > 256;
  a.first_round = items > cus && items <= 2 * (int64_t)cus && cus % a.HKV == 0 ? cus / a.HKV : 0;
  if (std::max(x.entries, pl.tiles) * x.H_KV > kMax31) return LSE_E_RANGE;
  return x.D == 64 ? lse::launch_fp8_attention<64>(a, pl, (hipStream_t)stream)
                   : lse::launch_fp8_attention<128>(a, pl, (hipStream_t)stream);
}

}  // extern "C"
