// Products of few rows with a 4-bit weight (layouts and formats: fp4.h), both kinds of rows:
//   bf16 rows:   y[m,n] = bf16(sum_k x[m,k] w[n,k]), w = code x scale, a bf16 value; fp32 sums
//   8-bit rows:  the same with x = code x scale; codes and scale bytes go to the scaled matrix instruction as they are
//   gate/up:     h[m,n] = bf16(silu(g) u) of the fp32 sums g and u of two stacked weights
//
// The kernel is a weight stream: 17 bytes for 32 weights, read once by each group of token rows. A workgroup takes RT
// row tiles (16 RT weight rows) and up to 16 token rows over the whole of K; its W waves take the 512-wide chunks
// of K in turns and add their sums through LDS in wave order at the end, so a result depends on K alone, never on the
// other rows of the call. A wave keeps four steps of 128 k in flight: weight tiles in registers, token rows in a slab
// of LDS of its own (direct-to-LDS loads of whole 256 or 128 byte row pieces, 16-byte chunks swizzled by row so that
// the fragment reads of 16 rows meet no bank twice); no wave waits for another before the end. Loads are
// range-checked: what lies past K, the rows or the weight reads zeros without a memory request.
// The workgroups of a panel's token groups follow each other on one XCD, whose L2 then holds the panel's weights.
//
// Bound by HBM where the weight is large, else by a CU's way from L2 (65 bytes a ns: slabs and weight tiles), for one
// small weight by the launch and a chain of two loads. GPU times, weights rotated: one row by 4096 x 4096 4.0 us, 13 by
// 6144 x 4096 6.4, 5 by two of 14336 x 4096 14.2 (4.4 TB/s, a copy's 4.7; called again on weights that the cache behind
// L2 holds 12.3, 5.1 TB/s); 8-bit rows: 64 by 4096 x 4096 6.7.
#include <algorithm>

#include "fp4.h"

namespace lse {

// XR: rows of a slab (16, or fewer where the call has fewer). RT: row tiles of a workgroup.
template <bool A8, int XR, int RT, int W, bool GLU>
__global__ void __launch_bounds__(64 * W)
fp4_stream_kernel(Fp4Args a, int panels, int groups) {
  static_assert(!GLU || RT % 2 == 0, "gate/up panels hold whole pairs of row tiles");
  constexpr int ESZ = A8 ? 1 : 2;
  constexpr int ROWB = kFp4Step * ESZ;       // bytes of a slab row
  constexpr int CH = ROWB / 16;              // its 16-byte chunks
  constexpr int XI = XR * ROWB / 1024;       // 1 KB loads of a step's slab
  static_assert(XR * ROWB % 1024 == 0, "whole 1 KB loads");
  constexpr int WAVE = XR * ROWB / 16;       // uint4 of a wave's slab
  __shared__ uint4 x0[W * WAVE], x1[W * WAVE], x2[W * WAVE], x3[W * WAVE];
  __shared__ f32x4 red[W][RT][64];
  auto slab = [&](int t) -> uint4* { return t == 0 ? x0 : t == 1 ? x1 : t == 2 ? x2 : x3; };
  constexpr auto swz = fp4_swz<A8>;

  // Workgroup (panel, token group): panel = 8 q + xcd, the groups of a panel 8 apart.
  const int xcd = blockIdx.x & 7, rest = blockIdx.x >> 3;
  const int panel = (rest / groups) * 8 + xcd, m0 = (rest % groups) * 16;
  if (panel >= panels) return;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, g = lane >> 4;
  const int rb0 = panel * RT, rows = min(16, a.M - m0), tiles = min(RT, a.nrb - rb0);

  const BufferRsrc wres = make_rsrc(a.codes + (int64_t)rb0 * a.nsteps * kFp4TileBytes,
                                    (uint32_t)tiles * (uint32_t)a.nsteps * kFp4TileBytes);
  const BufferRsrc sres = make_rsrc(a.scales + (int64_t)rb0 * a.nchunks * kFp4ScaleBytes,
                                    (uint32_t)tiles * (uint32_t)a.nchunks * kFp4ScaleBytes);
  const BufferRsrc xres = make_rsrc(static_cast<const char*>(a.x) + (int64_t)m0 * a.ldx * ESZ,
                                    (uint32_t)(((int64_t)(rows - 1) * a.ldx + a.K) * ESZ));
  const int per4 = (a.K / kFp4Group + 3) & ~3;  // scale bytes of a row in whole dwords
  const BufferRsrc xsres = A8 ? make_rsrc(a.xs + (int64_t)m0 * a.lds, (uint32_t)((int64_t)(rows - 1) * a.lds + per4))
                              : make_rsrc(a.x, 0);
  // Scale bytes past K in the last step's dword, which may be anything, become 0.
  const uint32_t tail = a.K % kFp4Step ? (1u << (8 * (a.K % kFp4Step / kFp4Group))) - 1 : ~0u;

  struct Step {
    uint4 w[RT];
  };
  struct Scales {
    uint32_t w[RT];
    uint32_t x[4];  // 8-bit rows: the scale bytes of row r16, a dword a step
  };
  auto load_step = [&](int c, auto t, Step& st) {
    const int j = 4 * c + t;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const uint32_t off = ((uint32_t)rt * (uint32_t)a.nsteps + (uint32_t)j) * kFp4TileBytes + 16u * lane;
      st.w[rt] = buffer_load16(wres, j < a.nsteps && rt < tiles ? off : kOutOfRange);
    }
#pragma unroll
    for (int i = 0; i < XI; ++i) {
      const int r = (64 * i + lane) / CH, kb = ROWB * j + 16 * (((64 * i + lane) % CH) ^ swz(r));
      const bool ok = r < rows && kb < a.K * ESZ;
      buffer_load16_lds(xres, slab(t) + wave * WAVE + 64 * i, ok ? (uint32_t)(r * a.ldx * ESZ + kb) : kOutOfRange);
    }
  };
  auto load_scales = [&](int c, Scales& s) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const uint32_t off = ((uint32_t)rt * (uint32_t)a.nchunks + (uint32_t)c) * kFp4ScaleBytes + 4u * lane;
      s.w[rt] =
          __builtin_amdgcn_raw_buffer_load_b32(sres, (int)(c < a.nchunks && rt < tiles ? off : kOutOfRange), 0, 0);
    }
    if constexpr (A8) {
      const uint32_t base = (uint32_t)(r16 * a.lds);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int b0 = 4 * (4 * c + t);  // the step's first byte of the row
        s.x[t] = __builtin_amdgcn_raw_buffer_load_b32(
            xsres, (int)(r16 < rows && b0 < per4 ? base + b0 : kOutOfRange), 0, 0);
        if (4 * c + t == a.nsteps - 1) s.x[t] &= tail;
      }
    }
  };

  // Where this lane's operands lie in a slab. The compiler is kept from taking the sums apart: it follows an LDS access
  // to its array, and so tells the slab that a load fills from those that are read, through a few additions only.
  int at[A8 ? 2 : 4];
#pragma unroll
  for (int i = 0; i < (A8 ? 2 : 4); ++i) {
    const int row = r16 & (XR - 1);
    at[i] = wave * WAVE + row * CH + ((A8 ? 4 * i + g : 4 * g + i) ^ swz(row));
    asm volatile("" : "+v"(at[i]));
  }

  f32x4 acc[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) acc[rt] = f32x4{0, 0, 0, 0};
  auto compute = [&](auto t, const Step& st, const Scales& s) {
    if constexpr (A8) {
      const uint4 lo = slab(t)[at[0]], hi = slab(t)[at[1]];
      const uint32_t xs = s.x[t] >> (8 * g);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) acc[rt] = mfma_fp4_fp8<t>(st.w[rt], s.w[rt], lo, hi, xs, acc[rt]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bf16x8 xv = as_bf16x8(slab(t)[at[i]]);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          const uint32_t w4[4] = {st.w[rt].x, st.w[rt].y, st.w[rt].z, st.w[rt].w};
          acc[rt] = mfma16x16x32(fp4_decode8(w4[i], fp4_scale(s.w[rt], t)), xv, acc[rt]);
        }
      }
    }
  };

  constexpr int LOADS = RT + XI;  // of a step
  const int iters = (a.nchunks + W - 1) / W;
  Step st[4];
  Scales cur, next;
  load_scales(wave, cur);
  unroll<4>([&](auto t) {
    load_step(wave, t, st[t]);
    __builtin_amdgcn_sched_barrier(0);
  });
  for (int it = 1; it < iters; ++it) {
    const int c = wave + W * it;
    unroll<4>([&](auto t) {
      // All but the three later steps' loads have landed, the slab among them.
      __builtin_amdgcn_s_waitcnt(vmcnt_imm(3 * LOADS));
      compute(t, st[t], cur);
      // The slab has been read before the next chunk's rows are let into it.
      __builtin_amdgcn_s_waitcnt(vmcnt_lgkm0_imm(63));
      if constexpr (t == 0) load_scales(c, next);
      load_step(c, t, st[t]);
      __builtin_amdgcn_sched_barrier(0);  // the loads stay in this order, by which they are counted
    });
    cur = next;
  }
  unroll<4>([&](auto t) {
    __builtin_amdgcn_s_waitcnt(vmcnt_imm((3 - t) * LOADS));
    compute(t, st[t], cur);
  });

  // The waves' sums, added in wave order: wave i adds tile i (gate/up: pair i).
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) red[wave][rt][lane] = acc[rt];
  __syncthreads();
  constexpr int OUT = GLU ? RT / 2 : RT;
  if (wave >= OUT) return;
  auto total = [&](int rt) {
    f32x4 s = red[0][rt][lane];
#pragma unroll
    for (int w = 1; w < W; ++w) s += red[w][rt][lane];
    return s;
  };
  const int m = m0 + r16;
  const bool yvec = (a.ldy & 3) == 0 && ((uintptr_t)a.y & 7) == 0;
  float o[4];
  int n;
  if constexpr (GLU) {
    n = 16 * ((rb0 >> 1) + wave) + 4 * g;
    const f32x4 gate = total(2 * wave), up = total(2 * wave + 1);
#pragma unroll
    for (int r = 0; r < 4; ++r) o[r] = silu(gate[r]) * up[r];
  } else {
    n = 16 * (rb0 + wave) + 4 * g;
    const f32x4 s = total(wave);
#pragma unroll
    for (int r = 0; r < 4; ++r) o[r] = s[r];
  }
  if (m < a.M && n < a.N) store_bf16x4(a.y, a.ldy, m, n, min(4, a.N - n), o, yvec);
}

template <bool A8, bool GLU>
static int launch(const Fp4Args& a, int rt, hipStream_t stream) {
  const int groups = (int)ceil_div(a.M, 16), panels = (int)ceil_div(a.nrb, rt);
  const int64_t blocks = ceil_div(panels, 8) * 8 * groups;
  if (blocks > 2147483647) return LSE_E_RANGE;
  auto go = [&](auto kernel, int waves) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(64 * waves), 0, stream, a, panels, groups);
    return launch_status();
  };
  constexpr int FEW = A8 ? 8 : 4, NARROW = GLU ? 2 : 1;
  if (a.M <= FEW) return go(fp4_stream_kernel<A8, FEW, NARROW, 8, GLU>, 8);
  // Four waves hold half the LDS, so that two workgroups share a CU; where there is one for each CU at most, 8-bit rows
  // are better off with eight (64 rows through 4096 x 4096 6.5 against 7.3 us; bf16 rows 7.4 either way).
  const bool four = !A8 || panels * groups > 256;
  auto width = [&](auto RT) {
    if constexpr (A8)
      if (!four) return go(fp4_stream_kernel<A8, 16, RT, 8, GLU>, 8);
    return go(fp4_stream_kernel<A8, 16, RT, 4, GLU>, 4);
  };
  if (rt == 4) return width(std::integral_constant<int, 4>{});
  if constexpr (!GLU)
    if (rt == 1) return width(std::integral_constant<int, 1>{});
  return width(std::integral_constant<int, 2>{});
}

int launch_fp4_stream(const Fp4Args& a, int rt, bool rows8, bool glu, hipStream_t stream) {
  if (rows8) return glu ? launch<true, true>(a, rt, stream) : launch<true, false>(a, rt, stream);
  return glu ? launch<false, true>(a, rt, stream) : launch<false, false>(a, rt, stream);
}

}  // namespace lse
