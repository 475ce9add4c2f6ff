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
// Order of summation. Wave w of the four takes chunks w, w + 4, ... of L keys, each with an online-softmax state
// of its own, folded into the wave's in chunk order; the four waves' are merged in wave order at the end. L is
// 256, twice that for every doubling of the entry's context past 32768 (so at most 32 chunks a wave). In a split
// launch every workgroup takes one chunk per wave and a second kernel does the same folds in the same order,
// so a row's bits depend on its own entry only, not on the batch, the table's width or the launch.
#include <algorithm>

#include "attn_fp8.h"

namespace lse {

constexpr int kF8Waves = 4;
constexpr int kF8Keys = 64;      // keys of a wave's tile: one group per 16 lanes
constexpr int kF8Window = 256;   // keys whose blocks and scales a wave holds: one group per lane of 16
constexpr int kF8MaxParts = 32;  // chunks of a wave
constexpr float kNegInf = -__builtin_huge_valf();

// log2 of a chunk's windows, for an entry of `ctx` positions.
__host__ __device__ inline int f8_chunk_shift(int ctx) {
  int k = 0;
  while (((int64_t)kF8Window * kF8Waves * kF8MaxParts << k) < ctx) ++k;
  return k;
}

// Folds the next chunk's state (max m in the base-2 domain, sum l, unnormalised O) into the state before it;
// from (-inf, 0, 0) the first fold gives the chunk's state exactly.
struct FoldFactors {
  float a, b;
};
__device__ __forceinline__ FoldFactors f8_fold_ml(float& M, float& L, float m, float l) {
  const float mn = fmaxf(M, m), ref = mn == kNegInf ? 0.0f : mn;
  const FoldFactors f{exp2_fast(M - ref), exp2_fast(m - ref)};
  L = __builtin_fmaf(l, f.b, L * f.a);
  M = mn;
  return f;
}
__device__ __forceinline__ float f8_fold(float O, float o, FoldFactors f) {
  return __builtin_fmaf(o, f.b, O * f.a);
}

// The four waves' states of a row merged in wave order.
struct WaveFactors {
  float f[kF8Waves], inv;
};
__device__ __forceinline__ WaveFactors f8_merge_factors(const float (&m)[kF8Waves],
                                                        const float (&l)[kF8Waves]) {
  float top = kNegInf, sum = 0.0f;
#pragma unroll
  for (int w = 0; w < kF8Waves; ++w) top = fmaxf(top, m[w]);
  const float ref = top == kNegInf ? 0.0f : top;
  WaveFactors r;
#pragma unroll
  for (int w = 0; w < kF8Waves; ++w) {
    r.f[w] = exp2_fast(m[w] - ref);
    sum = __builtin_fmaf(l[w], r.f[w], sum);
  }
  r.inv = sum == 0.0f ? 0.0f : 1.0f / sum;  // a row that saw no key gives zeros
  return r;
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

// ONE: every entry has at most one tile (decode); the grid is K/V heads, entries, parts. Otherwise items are
// counted entry by entry over their tiles and parts, without empty slots.
template <int D, bool ONE>
__global__ void __launch_bounds__(64 * kF8Waves, 2) attn_fp8_kernel(Fp8AttnArgs a) {
  constexpr int J = D / 64, DT = D / 16;  // 64-dim runs of a key; 16-dim tiles of O
  constexpr int OROW = D + 4;             // floats of a row of O in LDS: rows start on other banks
  __shared__ __attribute__((aligned(16))) float obuf[kF8Waves][16 * OROW];
  __shared__ float mbuf[kF8Waves][16], lbuf[kF8Waves][16];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n16 = lane & 15, g = lane >> 4;

  int b = blockIdx.x, e, qt = 0, part = 0;
  const int kvh = b % a.HKV;
  b /= a.HKV;
  if constexpr (ONE) {
    e = b % a.entries;
    part = b / a.entries;
    if (a.sorted) e = f8_sorted_entry(a, e);
  } else {
    e = -1;
    int chunk_parts = 1;
    for (int e0 = 0; e0 < a.entries; e0 += 64) {
      const int i = e0 + lane;
      int tiles = 0, parts = 1;
      if (i < a.entries) {
        const int qlen = min(a.q_len[i], a.max_q_len);
        tiles = qlen > 0 && !(a.tiled && f8_is_long(qlen, a.G)) ? (qlen + a.tq - 1) / a.tq : 0;
        if (a.parts > 1) {
          const int ctx = a.context_len[i];
          const int64_t span = (int64_t)(kF8Window * kF8Waves) << f8_chunk_shift(ctx);
          const int end = f8_end(a, a.query_offset[i], ctx, qlen);
          parts = min(max((int)((end + span - 1) / span), 1), a.parts);
        }
      }
      const int items = tiles * parts, before = kv_wave_scan(items) - items;
      const unsigned long long hit = __ballot((unsigned)(b - before) < (unsigned)items);
      if (hit) {
        const int at = __ffsll(hit) - 1;
        e = e0 + at;
        b -= __builtin_amdgcn_readlane(before, at);
        chunk_parts = __builtin_amdgcn_readlane(tiles, at);
        break;
      }
      b -= __builtin_amdgcn_readlane(before + items, 63);
    }
    if (e < 0) return;
    qt = b % chunk_parts;  // the tiles that read a chunk together
    part = b / chunk_parts;
  }
  const int qlen = min(a.q_len[e], a.max_q_len);
  if (qt * a.tq >= qlen) return;
  const int ctx = a.context_len[e], qo = a.query_offset[e], qs = a.q_start[e];
  const int end_n = f8_end(a, qo, ctx, min(qlen, (qt + 1) * a.tq));
  const int shift = f8_chunk_shift(ctx);
  // The wave's windows: j-th has keys [win(j), win(j) + 256); from j0 on, one chunk's in a split launch.
  auto win = [&](int j) -> int64_t {
    return ((((int64_t)(j >> shift) * kF8Waves + wave) << shift) + (j & ((1 << shift) - 1))) * kF8Window;
  };
  const int j0 = a.parts > 1 ? part << shift : 0;
  const int j_end = a.parts > 1 ? (part + 1) << shift : 0x7fffffff;
  if (a.parts > 1 && part > 0 && ((int64_t)part * kF8Waves << shift) * kF8Window >= end_n) return;

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

  // Blocks and scales of the wave's windows: lane i of 16 holds those of group i. `off` is the group's place
  // in the pool in 16-byte units; a block that is not the pool's reads block 0 with NaN for a scale.
  const int32_t* bt = a.block_table + (int64_t)e * a.sbt;
  const int last_group = (end_n - 1) / kKvGroup;
  const int per = a.pool.per;
  auto table_at = [&](int j, int& sub) {
    const int64_t first = win(j) / kKvGroup + n16;
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
        kr[bk][j] = ONE ? load16_stream(src) : *reinterpret_cast<const uint4*>(src);
      }
  };
  auto load_v = [&](uint32_t off, int t) {
    const uint32_t at = __shfl(off, 4 * t + g);
    const uint8_t* p = a.pool.v + ((uint64_t)at << 4) + 16 * n16;
#pragma unroll
    for (int i = 0; i < DT; ++i) {
      const uint8_t* src = p + i * 256;
      vr[i] = ONE ? load16_stream(src) : *reinterpret_cast<const uint4*>(src);
    }
  };

  float M = kNegInf, L = 0.0f, m_run = kNegInf, l_run = 0.0f;
  f32x4 oacc[DT], ofold[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) oacc[t] = ofold[t] = f32x4{0, 0, 0, 0};

  if (win(j0) < end_n) {
    // Window j's off and scales, window j + 1's off (and its scales on their way), window j + 2's block.
    int sub0, sub1, sub2, bad0, bad1;
    uint32_t off0, off1;
    const int blk0 = table_at(j0, sub0), blk1 = table_at(j0 + 1, sub1);
    int blk2 = table_at(j0 + 2, sub2);
    int sc0 = place(blk0, sub0, off0, bad0);
    load_k(off0, 0);
    load_v(off0, 0);
    int sc1 = place(blk1, sub1, off1, bad1);
    if (bad0) sc0 = 0xffff;

    for (int j = j0;; ) {
      const int64_t start = win(j);
      const int tiles = (int)min((int64_t)4, (end_n - start + kF8Keys - 1) / kF8Keys);
      const bool more = j + 1 < j_end && win(j + 1) < end_n;
      for (int t = 0; t < tiles; ++t) {
        const int n0 = (int)start + kF8Keys * t;
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
        l_run = __builtin_fmaf(l_run, alpha, sum);  // this lane's keys; its row's others' at the chunk's end
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
      // The end of a chunk: its state into the wave's.
      if (!more || ((j + 1) >> shift) != (j >> shift)) {
        l_run += __shfl_xor(l_run, 16);
        l_run += __shfl_xor(l_run, 32);
        const FoldFactors f = f8_fold_ml(M, L, m_run, l_run);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
#pragma unroll
          for (int r = 0; r < 4; ++r) ofold[d][r] = f8_fold(ofold[d][r], oacc[d][r], f);
          oacc[d] = f32x4{0, 0, 0, 0};
        }
        m_run = kNegInf, l_run = 0.0f;
      }
      if (!more) break;
      ++j;
      off0 = off1, sc0 = bad1 ? 0xffff : sc1;
      sc1 = place(blk2, sub2, off1, bad1);
      blk2 = table_at(j + 2, sub2);
    }
  }

  // Lane (n16, g) holds row n16's dims 16 t + 4 g + r.
  if (a.parts > 1) {
    if (row_ok && (((int64_t)part * kF8Waves + wave) << shift) * kF8Window < end_n) {
      const int64_t slot =
          (((int64_t)(part * kF8Waves + wave) * a.entries + e) * a.H + head) * a.ws_q + m_row;
      float* dst = a.ws_o + slot * D + 4 * g;
#pragma unroll
      for (int t = 0; t < DT; ++t)
        *reinterpret_cast<float4*>(dst + 16 * t) =
            make_float4(ofold[t][0], ofold[t][1], ofold[t][2], ofold[t][3]);
      if (g == 0) *reinterpret_cast<float2*>(a.ws_ml + 2 * slot) = make_float2(M, L);
    }
    return;
  }
  if (g == 0) mbuf[wave][n16] = M, lbuf[wave][n16] = L;
#pragma unroll
  for (int t = 0; t < DT; ++t)
    *reinterpret_cast<float4*>(&obuf[wave][n16 * OROW + 16 * t + 4 * g]) =
        make_float4(ofold[t][0], ofold[t][1], ofold[t][2], ofold[t][3]);
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
  *reinterpret_cast<uint4*>(a.o + (int64_t)(kvh * G + orow - otok * G) * a.so_h + out_row * a.so_t + c8) =
      make_uint4(pack_bf16x2(o[0] * f.inv, o[1] * f.inv), pack_bf16x2(o[2] * f.inv, o[3] * f.inv),
                 pack_bf16x2(o[4] * f.inv, o[5] * f.inv), pack_bf16x2(o[6] * f.inv, o[7] * f.inv));
}

// Second pass of a split launch: a workgroup takes 64 (entry, head, query row, 8 dims) pieces; wave w folds the
// chunk states of the first pass's waves w in order, then the four are merged as in the single pass.
template <int D>
__global__ void __launch_bounds__(64 * kF8Waves) attn_fp8_merge(Fp8AttnArgs a) {
  constexpr int C = D / 8;
  __shared__ float obuf[kF8Waves][64][9];
  __shared__ float mbuf[kF8Waves][64], lbuf[kF8Waves][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t t = (int64_t)blockIdx.x * 64 + lane;
  const int64_t rows = (int64_t)a.entries * a.H * a.ws_q;
  const int c8 = 8 * (int)(t % C);
  const int64_t r = t / C;
  const int m_row = (int)(r % a.ws_q), h = (int)(r / a.ws_q % a.H);
  const int e = (int)min(r / a.ws_q / a.H, (int64_t)a.entries - 1);
  const int qlen = min(a.q_len[e], a.max_q_len);
  const int64_t row = (int64_t)a.q_start[e] + m_row;
  const bool ok = r < rows && m_row < qlen && !(a.tiled && f8_is_long(qlen, a.G)) && row >= 0 && row < a.tokens;
  float M = kNegInf, L = 0.0f, O[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  if (ok) {
    const int ctx = a.context_len[e];
    const int end_n = f8_end(a, a.query_offset[e], ctx, min(qlen, (m_row / a.tq + 1) * a.tq));
    const int64_t chunk = (int64_t)kF8Window << f8_chunk_shift(ctx);
    const int chunks = (int)((end_n + chunk - 1) / chunk);
    const int mine = chunks > wave ? (chunks - wave + kF8Waves - 1) / kF8Waves : 0;
#pragma unroll 4
    for (int p = 0; p < mine; ++p) {
      const int64_t slot = (int64_t)(p * kF8Waves + wave) * rows + r;
      const float2 ml = *reinterpret_cast<const float2*>(a.ws_ml + 2 * slot);
      const float4 x = *reinterpret_cast<const float4*>(a.ws_o + slot * D + c8);
      const float4 y = *reinterpret_cast<const float4*>(a.ws_o + slot * D + c8 + 4);
      const FoldFactors f = f8_fold_ml(M, L, ml.x, ml.y);
      const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) O[i] = f8_fold(O[i], v[i], f);
    }
  }
  mbuf[wave][lane] = M, lbuf[wave][lane] = L;
#pragma unroll
  for (int i = 0; i < 8; ++i) obuf[wave][lane][i] = O[i];
  __syncthreads();
  if (wave != 0 || !ok) return;
  float m[kF8Waves], l[kF8Waves], o[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
  for (int w = 0; w < kF8Waves; ++w) m[w] = mbuf[w][lane], l[w] = lbuf[w][lane];
  const WaveFactors f = f8_merge_factors(m, l);
#pragma unroll
  for (int w = 0; w < kF8Waves; ++w)
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = __builtin_fmaf(obuf[w][lane][i], f.f[w], o[i]);
  *reinterpret_cast<uint4*>(a.o + (int64_t)h * a.so_h + row * a.so_t + c8) =
      make_uint4(pack_bf16x2(o[0] * f.inv, o[1] * f.inv), pack_bf16x2(o[2] * f.inv, o[3] * f.inv),
                 pack_bf16x2(o[4] * f.inv, o[5] * f.inv), pack_bf16x2(o[6] * f.inv, o[7] * f.inv));
}

// ---- host side -----------------------------------------------------------------------------

struct Fp8AttnPlan {
  int tq, parts;
  bool tiled;       // some entry may be the row-tiled kernel's
  int64_t short_q;  // the most tokens of an entry that is not
  int64_t tiles;  // at most, over all entries
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

// One workgroup per (entry, K/V head, query tile) once those fill the CUs twice over; otherwise, where the
// table has room for more than one round of chunks, one per round, and a second pass. The choice changes no
// result.
static Fp8AttnPlan fp8_attn_plan(int64_t entries, int64_t tokens, int64_t H, int64_t HKV, int64_t D,
                                 int64_t max_q_len, int64_t max_ctx, int cus) {
  Fp8AttnPlan pl{};
  pl.tq = (int)(16 / (H / HKV));
  const int64_t G = H / HKV;
  pl.tiled = f8_is_long(max_q_len, (int)G);
  pl.short_q = pl.tiled ? (kF8LongRows - 1) / G : max_q_len;
  pl.tiles = std::min(entries * ceil_div(pl.short_q, (int64_t)pl.tq), tokens / pl.tq + entries);
  const int64_t rounds = std::min<int64_t>(ceil_div(max_ctx, (int64_t)kF8Window * kF8Waves), kF8MaxParts);
  pl.parts = pl.tiles * HKV < 2 * (int64_t)cus && rounds > 1 ? (int)rounds : 1;
  if (pl.parts > 1) {
    const int64_t slots = (int64_t)pl.parts * kF8Waves * entries * H * pl.short_q;
    pl.ws_o_bytes = slots * D * 4;
    pl.ws_bytes = pl.ws_o_bytes + slots * 2 * 4;
  }
  return pl;
}

template <int D>
static int launch_fp8_attention(const Fp8AttnArgs& a, int64_t blocks, hipStream_t stream) {
  const dim3 wg(64 * kF8Waves);
  if (a.tiled)
    if (int st = launch_fp8_attn_tile(a, D, stream)) return st;
  if (a.ws_q <= a.tq)
    hipLaunchKernelGGL((attn_fp8_kernel<D, true>), dim3((unsigned)blocks), wg, 0, stream, a);
  else
    hipLaunchKernelGGL((attn_fp8_kernel<D, false>), dim3((unsigned)blocks), wg, 0, stream, a);
  if (int st = launch_status()) return st;
  if (a.parts > 1) {
    const int64_t pieces = (int64_t)a.entries * a.H * a.ws_q * (D / 8);
    hipLaunchKernelGGL(attn_fp8_merge<D>, dim3((unsigned)ceil_div(pieces, 64)), wg, 0, stream, a);
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

lse::Fp8AttnPlan plan_of(const Args& x, int cus) {
  return lse::fp8_attn_plan(x.entries, x.tokens, x.H, x.H_KV, x.D, x.max_q_len, x.max_blocks * x.block_size,
                            cus);
}

}  // namespace

extern "C" {

int64_t lse_paged_attention_fp8_workspace_bytes(const struct lse_paged_attention_fp8_args* args) {
  if (!args || check_sizes(*args)) return -1;
  if (args->entries == 0 || args->tokens == 0 || args->max_q_len == 0) return 0;
  return plan_of(*args, lse::fp8_attn_cus()).ws_bytes;
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
  const lse::Fp8AttnPlan pl = plan_of(x, cus);
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
  a.max_q_len = (int)x.max_q_len, a.ws_q = (int)pl.short_q, a.tiled = pl.tiled;
  a.tq = pl.tq, a.parts = pl.parts;
  a.scale_log2 = (float)x.softmax_scale * 1.4426950408889634f;
  a.ws_o = pl.parts > 1 ? (float*)workspace : nullptr;
  a.ws_ml = pl.parts > 1 ? (float*)((char*)workspace + pl.ws_o_bytes) : nullptr;
  const int64_t items = x.entries * x.H_KV;
  a.sorted = a.parts == 1 && x.entries <= 64 && items > cus && a.max_ctx > 256;
  a.first_round = items > cus && items <= 2 * (int64_t)cus && cus % a.HKV == 0 ? cus / a.HKV : 0;
  const int64_t blocks = (pl.short_q <= pl.tq ? x.entries : pl.tiles) * x.H_KV * pl.parts;
  if (blocks > kMax31 || x.entries * x.H * pl.short_q * (x.D / 8) / 64 > kMax31) return LSE_E_RANGE;
  return x.D == 64 ? lse::launch_fp8_attention<64>(a, blocks, (hipStream_t)stream)
                   : lse::launch_fp8_attention<128>(a, blocks, (hipStream_t)stream);
}

}  // extern "C"
