// Products of many rows with a 4-bit weight (layouts and formats: fp4.h; the arithmetic as in fp4_stream.hip), bound by
// the matrix cores.
//
// A workgroup of WGM x WGN waves computes BM token rows x BN weight rows over K, in stages of 256 bytes of a token row
// (128 k of bf16, 256 k of 8-bit codes). Token rows go to LDS by direct loads (whole 256-byte row pieces, 16-byte
// chunks swizzled by row), NST - 1 stages ahead; the weight, a quarter or a half of their bytes, goes straight to the
// registers of the wave that multiplies it, as far ahead: each wave needs BN / WGN rows of it and no other wave of its
// row of waves does. One barrier a stage. bf16 rows: a wave decodes its weight tiles (half an instruction a weight,
// shared by its WM token rows) and runs 16x16x32 bf16 instructions. 8-bit rows: codes and scale bytes of both operands
// go to the scaled 16x16x128 instruction as they are.
//
// Tile order: blocks are dealt to the 8 XCDs in turn; each XCD gets a contiguous range of tiles, in groups of kGroupM
// token blocks x consecutive weight panels, so that what it runs at once shares token rows and weights in its L2.
// K may be split over `splits` workgroups, whose fp32 sums a second kernel adds in order.
// A result depends on K and the split alone, never on other rows.
#include <algorithm>

#include "fp4.h"

namespace lse {

constexpr int kFp4GroupM = 4;

template <bool A8, int BM, int BN, int WGM, int WGN, int NST, bool GLU>
__global__ void __launch_bounds__(64 * WGM * WGN)
fp4_tile_kernel(Fp4Args a, Fp4Split p) {
  constexpr int W = WGM * WGN, WM = BM / WGM, WN = BN / WGN, TM = WM / 16, TN = WN / 16;
  static_assert(WM % 16 == 0 && WN % 16 == 0 && (!GLU || TN % 2 == 0), "whole tiles, and pairs of row tiles");
  static_assert(NST == 2 || NST == 4, "stage slots");
  constexpr int ESZ = A8 ? 1 : 2;
  constexpr int SUB = A8 ? 2 : 1;            // 128-k steps of a stage
  constexpr int CS = 4 / SUB;                // stages of a 512-k chunk
  constexpr int U = CS > NST ? CS : NST;     // stages of the unrolled loop body: whole chunks, whole rings
  constexpr int XI = BM / (4 * W);           // 1 KB loads (4 rows) of a wave and stage
  constexpr int XSI = A8 ? (BM + 32 * W - 1) / (32 * W) : 0;  // scale loads (32 rows) of a wave and stage
  static_assert(BM % (4 * W) == 0, "whole 1 KB loads per wave");
  constexpr int SLOT = BM * 16;              // uint4 of a stage's rows
  constexpr int XS = A8 ? 64 * W * XSI : 1;  // dwords of a stage's scales: two a row
  __shared__ uint4 x0[SLOT], x1[SLOT], x2[NST > 2 ? SLOT : 1], x3[NST > 2 ? SLOT : 1];
  __shared__ uint32_t s0[XS], s1[XS], s2[NST > 2 ? XS : 1], s3[NST > 2 ? XS : 1];
  auto slot = [&](int i) -> uint4* { return i == 0 ? x0 : i == 1 ? x1 : i == 2 ? x2 : x3; };
  auto sslot = [&](int i) -> uint32_t* { return i == 0 ? s0 : i == 1 ? s1 : i == 2 ? s2 : s3; };

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WGN, wn = wave % WGN;
  const int r16 = lane & 15, g = lane >> 4;

  const int sp = blockIdx.x % p.splits;
  const int T = p.mblocks * p.nblocks, b = blockIdx.x / p.splits;
  const int xcd = b & 7, q8 = T >> 3, rem = T & 7;
  const int t = xcd * q8 + min(xcd, rem) + (b >> 3);
  const int group = t / (kFp4GroupM * p.nblocks), first = group * kFp4GroupM;
  const int gm = min(p.mblocks - first, kFp4GroupM), tg = t - group * kFp4GroupM * p.nblocks;
  const int m0 = (first + tg % gm) * BM, rb0 = tg / gm * (BN / 16);
  const int rows = min(BM, a.M - m0);
  // Chunks [c0, c1) of K, and its stages counted from c0.
  const int c0 = sp * p.chunks, c1 = min(c0 + p.chunks, a.nchunks);
  const int nsteps = min(4 * c1, a.nsteps) - 4 * c0, stages = (nsteps + SUB - 1) / SUB;

  const BufferRsrc xres = make_rsrc(static_cast<const char*>(a.x) + (int64_t)m0 * a.ldx * ESZ,
                                    (uint32_t)(((int64_t)(rows - 1) * a.ldx + a.K) * ESZ));
  const int per4 = (a.K / kFp4Group + 3) & ~3;  // scale bytes of a row in whole dwords
  const BufferRsrc sres = A8 ? make_rsrc(a.xs + (int64_t)m0 * a.lds, (uint32_t)((int64_t)(rows - 1) * a.lds + per4))
                             : make_rsrc(a.x, 0);
  // This wave's row tiles; those past the weight repeat its last one, and are not stored.
  const uint8_t *wp[TN], *wsp[TN];
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    const int rb = min(rb0 + wn * TN + j, a.nrb - 1);
    wp[j] = a.codes + ((int64_t)rb * a.nsteps + 4 * c0) * kFp4TileBytes + 16 * lane;
    wsp[j] = a.scales + ((int64_t)rb * a.nchunks + c0) * kFp4ScaleBytes + 4 * lane;
  }

  // Load i of a wave: rows 4 (wave + W i) .. + 3, lane l its physical chunk l % 16 of row l / 16. W is even, so a lane's
  // logical chunk depends on i where 4 W i is no multiple of 16.
  auto load_x = [&](int s, int sl) {
#pragma unroll
    for (int i = 0; i < XI; ++i) {
      const int r = 4 * (wave + W * i) + (lane >> 4), kb = (4 * c0 * kFp4Step * ESZ) + 256 * s + 16 * (r16 ^ (r & 15));
      const bool ok = s < stages && r < rows && kb < a.K * ESZ;
      buffer_load16_lds(xres, slot(sl) + 64 * (wave + W * i), ok ? (uint32_t)(r * a.ldx * ESZ + kb) : kOutOfRange);
    }
#pragma unroll
    for (int i = 0; i < XSI; ++i) {
      const int at = 64 * (wave + W * i) + lane, r = at >> 1, b0 = 16 * c0 + 8 * s + 4 * (at & 1);
      const bool ok = s < stages && r < rows && b0 < per4;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(sres, (LdsPtr)(sslot(sl) + 64 * (wave + W * i)), 4,
                                               ok ? (uint32_t)(r * a.lds + b0) : kOutOfRange, 0, 0, 0);
    }
  };
  struct Weights {
    uint4 w[SUB][TN];
  };
  auto load_w = [&](int s, Weights& st) {
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
      const int j = min(SUB * s + u, nsteps - 1);
#pragma unroll
      for (int n = 0; n < TN; ++n) st.w[u][n] = *reinterpret_cast<const uint4*>(wp[n] + (int64_t)j * kFp4TileBytes);
    }
  };
  struct Scales {
    uint32_t w[TN];
  };
  auto load_s = [&](int c, Scales& sc) {  // chunk c0 + c
#pragma unroll
    for (int n = 0; n < TN; ++n)
      sc.w[n] = *reinterpret_cast<const uint32_t*>(wsp[n] + (int64_t)min(c, c1 - c0 - 1) * kFp4ScaleBytes);
  };

  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0, 0, 0, 0};

  // Scale bytes past K in the last step's dword, which may be anything, become 0.
  const uint32_t tail = a.K % kFp4Step ? (1u << (8 * (a.K % kFp4Step / kFp4Group))) - 1 : ~0u;
  auto compute = [&](int s, auto sl, auto phase, const Weights& st, const Scales& sc) {
    const uint4* xs = slot(sl) + (wm * WM + r16) * 16;
    if constexpr (A8) {
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const uint2 sd = *reinterpret_cast<const uint2*>(sslot(sl) + 2 * (wm * WM + 16 * i + r16));
        auto step = [&](auto u, uint32_t d) {
          if (SUB * s + u >= nsteps) return;
          if (4 * c0 + SUB * s + u == a.nsteps - 1) d &= tail;
          const uint4 lo = xs[256 * i + ((8 * u + g) ^ r16)], hi = xs[256 * i + ((8 * u + 4 + g) ^ r16)];
#pragma unroll
          for (int j = 0; j < TN; ++j)
            acc[i][j] = mfma_fp4_fp8<(SUB * phase + u) % 4>(st.w[u][j], sc.w[j], lo, hi, d >> (8 * g), acc[i][j]);
        };
        step(std::integral_constant<int, 0>{}, sd.x);
        step(std::integral_constant<int, 1>{}, sd.y);
      }
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        bf16x8 w[TN];
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          const uint32_t w4[4] = {st.w[0][j].x, st.w[0][j].y, st.w[0][j].z, st.w[0][j].w};
          w[j] = fp4_decode8(w4[q], fp4_scale(sc.w[j], phase % 4));
        }
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          const bf16x8 xv = as_bf16x8(xs[256 * i + ((4 * g + q) ^ r16)]);
#pragma unroll
          for (int j = 0; j < TN; ++j) acc[i][j] = mfma16x16x32(w[j], xv, acc[i][j]);
        }
      }
    }
  };

  constexpr int LOADS = XI + XSI + SUB * TN;
  Weights st[NST];
  Scales sc[U / CS], next[U / CS];
#pragma unroll
  for (int c = 0; c < U / CS; ++c) load_s(c, sc[c]);
#pragma unroll
  for (int i = 0; i < NST - 1; ++i) {
    load_x(i, i);
    load_w(i, st[i]);
  }
  for (int base = 0; base < stages; base += U) {
    auto stage = [&](auto u) {
      constexpr int sl = u % NST, ahead = (u + NST - 1) % NST;
      const int s = base + u;
      if (s >= stages) return;
      // This wave's rows of stage s have landed and its reads of the slot that the loads below go to are done; after
      // the barrier every wave's are.
      __builtin_amdgcn_s_waitcnt(vmcnt_lgkm0_imm((NST - 2) * LOADS));
      __builtin_amdgcn_s_barrier();
      load_x(s + NST - 1, ahead);
      load_w(s + NST - 1, st[ahead]);
      if constexpr (u == 0) {
#pragma unroll
        for (int c = 0; c < U / CS; ++c) load_s((base + U) / CS + c, next[c]);
      }
      compute(s, std::integral_constant<int, sl>{}, u, st[sl], sc[u / CS]);
    };
    [&]<int... I>(std::integer_sequence<int, I...>) {
      (stage(std::integral_constant<int, I>{}), ...);
    }(std::make_integer_sequence<int, U>{});
#pragma unroll
    for (int c = 0; c < U / CS; ++c) sc[c] = next[c];
  }
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));

  // D tile (i, j): lane holds weight rows 4 g + r (r = 0..3) of token row r16.
  const bool yvec = (a.ldy & 3) == 0 && ((uintptr_t)a.y & 7) == 0;
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int m = m0 + wm * WM + 16 * i + r16;
    if (m >= a.M) continue;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int rb = rb0 + wn * TN + j;
      if (p.splits > 1) {
        if (rb < a.nrb)
          *reinterpret_cast<f32x4*>(p.part + ((int64_t)sp * a.M + m) * (16 * a.nrb) + 16 * rb + 4 * g) = acc[i][j];
        continue;
      }
      if constexpr (GLU) {
        if (j % 2) continue;
        const int n = 16 * (rb >> 1) + 4 * g;
        if (n >= a.N) continue;
        float o[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) o[r] = silu(acc[i][j][r]) * acc[i][j + 1][r];
        store_bf16x4(a.y, a.ldy, m, n, min(4, a.N - n), o, yvec);
      } else {
        const int n = 16 * rb + 4 * g;
        if (n >= a.N) continue;
        const float o[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
        store_bf16x4(a.y, a.ldy, m, n, min(4, a.N - n), o, yvec);
      }
    }
  }
}

// Adds the splits' sums of four neighbouring columns in order, and rounds them (gate/up: silu and product first).
template <bool GLU>
__global__ void __launch_bounds__(256) fp4_reduce_kernel(Fp4Args a, Fp4Split p) {
  const int quads = (a.N + 3) / 4;
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= (int64_t)a.M * quads) return;
  const int m = (int)(at / quads), n = 4 * (int)(at % quads);
  const int64_t row = 16 * (int64_t)a.nrb;
  auto total = [&](int col) {
    const float* src = p.part + (int64_t)m * row + col;
    f32x4 s = *reinterpret_cast<const f32x4*>(src);
    for (int i = 1; i < p.splits; ++i) s += *reinterpret_cast<const f32x4*>(src + i * a.M * row);
    return s;
  };
  float o[4];
  if constexpr (GLU) {
    const int col = 32 * (n >> 4) + (n & 15);
    const f32x4 gate = total(col), up = total(col + 16);
#pragma unroll
    for (int r = 0; r < 4; ++r) o[r] = silu(gate[r]) * up[r];
  } else {
    const f32x4 s = total(n);
#pragma unroll
    for (int r = 0; r < 4; ++r) o[r] = s[r];
  }
  store_bf16x4(a.y, a.ldy, m, n, min(4, a.N - n), o, (a.ldy & 3) == 0 && ((uintptr_t)a.y & 7) == 0);
}

template <bool A8, bool GLU>
static int launch(const Fp4Args& a, const Fp4Plan& plan, float* part, hipStream_t stream) {
  Fp4Split p{};
  p.splits = plan.splits, p.chunks = plan.chunks, p.part = part;
  p.mblocks = (int)ceil_div(a.M, plan.bm), p.nblocks = (int)ceil_div(a.nrb, plan.bn / 16);
  const int64_t blocks = (int64_t)p.mblocks * p.nblocks * p.splits;
  if (blocks > 2147483647) return LSE_E_RANGE;
  auto go = [&](auto kernel, int threads) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(threads), 0, stream, a, p);
  };
  if (plan.bm == 256)
    go(fp4_tile_kernel<A8, 256, 256, 2, 4, 2, GLU>, 512);
  else if (plan.bm == 128)
    go(fp4_tile_kernel<A8, 128, 128, 2, 2, 2, GLU>, 256);
  else
    go(fp4_tile_kernel<A8, 64, 128, 1, 4, 4, GLU>, 256);
  if (p.splits > 1) {
    if (int st = launch_status()) return st;
    const int64_t quads = (int64_t)a.M * ceil_div(a.N, 4);
    hipLaunchKernelGGL(fp4_reduce_kernel<GLU>, dim3((unsigned)ceil_div(quads, 256)), dim3(256), 0, stream, a, p);
  }
  return launch_status();
}

int launch_fp4_tile(const Fp4Args& a, const Fp4Plan& plan, bool rows8, bool glu, float* part, hipStream_t stream) {
  if (rows8) return glu ? launch<true, true>(a, plan, part, stream) : launch<true, false>(a, plan, part, stream);
  return glu ? launch<false, true>(a, plan, part, stream) : launch<false, false>(a, plan, part, stream);
}

}  // namespace lse
