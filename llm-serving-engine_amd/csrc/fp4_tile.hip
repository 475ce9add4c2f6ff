// Products of many rows with a 4-bit weight (layouts and formats: fp4.h; the arithmetic as in fp4_stream.hip), bound by
// the matrix cores.
//
// A workgroup of four waves (KG groups of four) computes BM token rows x BN weight rows over K, in stages of 128 k a
// group, which take them in turn. Token rows go to LDS by direct loads (whole 256 or 128 byte row pieces, 16-byte chunks
// swizzled by row), NST - 1 stages ahead; the weight, a quarter or a half of their bytes, goes straight to the registers
// of the wave that multiplies it, as far ahead: each wave needs BN / 4 rows of it and no other wave of its group does.
// One barrier a stage. bf16 rows: a wave decodes its weight tiles (half an instruction a weight, shared by the BM token
// rows) and runs 16x16x32 bf16 instructions. 8-bit rows: codes and scale bytes of both operands go to the scaled
// 16x16x128 instruction as they are.
//
// Tile order: blocks are dealt to the 8 XCDs in turn; each XCD gets a contiguous range of tiles, in groups of
// kFp4GroupM token blocks x consecutive weight panels, so that what it runs at once shares token rows and weights in
// its L2.
// K may be split over `splits` workgroups, whose fp32 sums a second kernel adds in order. They are neighbours in the grid,
// so an XCD then has one range of K, of tiles out of two, four or all of the eight ranges of tiles.
// A result depends on K, the groups and the split alone, never on other rows.
//
// What it measured: bf16 rows, 64 x 256 tiles, 2048 by two of 14336 x 4096 343 us, 1400 TFLOP/s, by 4096 x 14336 166,
// 1450 (a large library product 1330 to 1380); 8-bit rows, 128 x 256 tiles, 2048 by two of 14336 x 4096 184 us, 2610
// TFLOP/s, by 4096 x 14336 92, 2610 (a library's fp8 2590 to 2930). The matrix cores bound these, but for the time around
// the barriers: two workgroups of four waves share a CU, so that one runs while the other waits. One of eight waves, of
// twice the tile, gave 205 us with 8-bit rows (256 x 256) and 345 with bf16 ones (128 x 256). Deeper rings (3, 4, 6 slots)
// gain nothing, a second barrier in mid-stage spills.
//
// A small tile's workgroup is often alone on its CU, a wave a SIMD, whose decoding, LDS reads and matrix instructions
// then wait for each other: with bf16 rows they take two groups (256 rows by 4096 x 4096: 14.1 -> 11.1 us; 777 by
// 2330 x 4128: 22.3 -> 20.1). By their times 17 or 25 KB a stage then come from L2 at 50 to 60 bytes a ns.
// 8-bit rows, half the bytes and no decoding, ran slower with two (12.5 -> 12.9) and keep one, with four slots.
//
// The compiler counts the weights' loads and waits for them in order, so it has to count the direct loads too, without
// taking them for writes of the slot that is being read: one array a slot, indexes that it does not take apart (at[]).
// With two slots it still waited for all of them in every stage; there they are issued by inline assembly (dma16_lds),
// and the only wait on them is the one written here, with nothing later in flight but weights.
#include <algorithm>

#include "fp4.h"

namespace lse {

constexpr int kFp4GroupM = 4;

template <bool A8, int BM, int BN, int KG, int NST, bool GLU>
__global__ void __launch_bounds__(256 * KG, 2)
fp4_tile_kernel(Fp4Args a, Fp4Split p) {
  static_assert(KG == 1 || KG == 2, "whole chunks");
  constexpr int W = 4, TM = BM / 16, TN = BN / W / 16;  // waves of a group, their tiles
  static_assert(BM % 16 == 0 && BN % (16 * W) == 0 && (!GLU || TN % 2 == 0), "whole tiles, and pairs of row tiles");
  constexpr int ESZ = A8 ? 1 : 2;
  constexpr int ROWB = kFp4Step * ESZ, CH = ROWB / 16;  // bytes of a token row and stage, its 16-byte chunks
  constexpr int RPL = 1024 / ROWB;                      // rows of a 1 KB load
  constexpr int XI = BM / (RPL * W);                    // such loads of a wave and stage
  constexpr int XSI = A8 ? (BM + 64 * W - 1) / (64 * W) : 0;  // loads of 64 rows' scale dwords, likewise
  static_assert(BM % (RPL * W) == 0 && RPL * W % 16 == 0, "whole loads per wave, whose lanes' chunks do not differ");
  constexpr int SLOT = BM * CH;                         // uint4 of a stage's rows
  constexpr int XS = A8 ? 64 * W * XSI : 1;             // dwords of a stage's scales
  // One array a slot, so that the compiler tells the slot a load fills from the one that is read.
  __shared__ uint4 x0[KG * SLOT], x1[KG * SLOT], x2[NST > 2 ? KG * SLOT : 1], x3[NST > 2 ? KG * SLOT : 1];
  __shared__ uint32_t s0[KG * XS], s1[KG * XS], s2[NST > 2 ? KG * XS : 1], s3[NST > 2 ? KG * XS : 1];
  auto slot_x = [&](auto i) -> uint4* { return i == 0 ? x0 : i == 1 ? x1 : i == 2 ? x2 : x3; };
  auto slot_s = [&](auto i) -> uint32_t* { return i == 0 ? s0 : i == 1 ? s1 : i == 2 ? s2 : s3; };
  constexpr auto swz = fp4_swz<A8>;

  const int lane = threadIdx.x & 63;
  const int all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kg = KG == 1 ? 0 : all / W, wave = KG == 1 ? all : all % W;  // the wave's group, and its place there
  const int r16 = lane & 15, g = lane >> 4;

  const int sp = blockIdx.x % p.splits;
  const int T = p.mblocks * p.nblocks, b = blockIdx.x / p.splits;
  const int xcd = b & 7, q8 = T >> 3, rem = T & 7;
  const int t = xcd * q8 + min(xcd, rem) + (b >> 3);
  const int group = t / (kFp4GroupM * p.nblocks), first = group * kFp4GroupM;
  const int gm = min(p.mblocks - first, kFp4GroupM), tg = t - group * kFp4GroupM * p.nblocks;
  const int m0 = (first + tg % gm) * BM, rb0 = tg / gm * (BN / 16);
  const int rows = min(BM, a.M - m0);
  // Chunks [c0, c1) of K, and its steps (stages) counted from c0.
  const int c0 = sp * p.chunks, c1 = min(c0 + p.chunks, a.nchunks);
  const int steps = min(4 * c1, a.nsteps) - 4 * c0;

  const void* xbase = static_cast<const char*>(a.x) + (int64_t)m0 * a.ldx * ESZ;
  const uint32_t xbytes = (uint32_t)(((int64_t)(rows - 1) * a.ldx + a.K) * ESZ);
  const int per4 = (a.K / kFp4Group + 3) & ~3;  // scale bytes of a row in whole dwords
  const void* sbase = A8 ? a.xs + (int64_t)m0 * a.lds : a.x;
  const uint32_t sbytes = A8 ? (uint32_t)((int64_t)(rows - 1) * a.lds + per4) : 0;
  const BufferRsrc xres = make_rsrc(xbase, xbytes), sres = make_rsrc(sbase, sbytes);
  const u32x4 xres4 = make_rsrc4(xbase, xbytes), sres4 = make_rsrc4(sbase, sbytes);
  // This wave's row tiles; those past the weight repeat its last one, and are not stored. A tile's step is a scalar
  // offset from the panel's first tile, so its loads need no address arithmetic of their own.
  const int tiles = min(BN / 16, a.nrb - rb0);
  const BufferRsrc wres = make_rsrc(a.codes + (int64_t)rb0 * a.nsteps * kFp4TileBytes,
                                    (uint32_t)tiles * (uint32_t)a.nsteps * kFp4TileBytes);
  const BufferRsrc wsres = make_rsrc(a.scales + (int64_t)rb0 * a.nchunks * kFp4ScaleBytes,
                                     (uint32_t)tiles * (uint32_t)a.nchunks * kFp4ScaleBytes);
  uint32_t wp[TN], wsp[TN];
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    const uint32_t tile = min(wave * TN + j, tiles - 1);
    wp[j] = (tile * a.nsteps + 4 * c0) * kFp4TileBytes;
    wsp[j] = (tile * a.nchunks + c0) * kFp4ScaleBytes;
  }

  // Load i of a wave: rows RPL (wave + W i) .. , lane l physical chunk l % CH of row l / CH, whose logical chunk is the
  // same for every i. Rows past the call's lie past the resource, and read zeros; so does, by its offset, what is past K.
  const int xr = RPL * wave + lane / CH, xkb = 16 * ((lane % CH) ^ swz(xr));
  const int kbytes = (a.K - 4 * c0 * kFp4Step) * ESZ;  // of a row from c0 on
  const uint32_t xoff = (uint32_t)(xr * a.ldx * ESZ + 4 * c0 * kFp4Step * ESZ + xkb);
  const uint32_t xstep = (uint32_t)(RPL * W * a.ldx * ESZ);
  const uint32_t soff = (uint32_t)((64 * wave + lane) * a.lds + 16 * c0), sstep = (uint32_t)(64 * W * a.lds);
  auto load_x = [&](int s, auto slot) {
    s = KG * s + kg;
    const uint32_t off = ROWB * s + xkb < kbytes ? xoff + ROWB * s : kOutOfRange;
    if constexpr (NST == 2) {
      const uint32_t to = lds_addr(slot_x(slot) + kg * SLOT + 64 * wave);
      unroll<XI>([&](auto i) { dma16_lds<1024 * W * i>(xres4, to, off + i * xstep); });
    } else {
#pragma unroll
      for (int i = 0; i < XI; ++i)
        buffer_load16_lds(xres, slot_x(slot) + kg * SLOT + 64 * (wave + W * i), off + i * xstep);
    }
    if constexpr (A8) {
      const uint32_t so = 4 * (4 * c0 + s) < per4 ? soff + 4 * s : kOutOfRange;
      if constexpr (NST == 2) {
        const uint32_t to4 = lds_addr(slot_s(slot) + kg * XS + 64 * wave);
        unroll<XSI>([&](auto i) { dma4_lds<256 * W * i>(sres4, to4, so + i * sstep); });
      } else {
#pragma unroll
        for (int i = 0; i < XSI; ++i)
          __builtin_amdgcn_raw_ptr_buffer_load_lds(sres, (LdsPtr)(slot_s(slot) + kg * XS + 64 * (wave + W * i)), 4,
                                                   so + i * sstep, 0, 0, 0);
      }
    }
  };
  struct Weights {
    u32x4 w[TN];
  };
  auto load_w = [&](int s, Weights& st) {  // stage s; past the range its last step, which is not used then
    const uint32_t at = min(KG * s + kg, steps - 1) * kFp4TileBytes;
#pragma unroll
    for (int n = 0; n < TN; ++n)
      st.w[n] = __builtin_amdgcn_raw_buffer_load_b128(wres, 16 * lane, (int)(wp[n] + at), 0);
  };
  struct Scales {
    uint32_t w[TN];
  };
  auto load_s = [&](int c, Scales& sc) {  // chunk c0 + c
    const uint32_t at = min(c, c1 - c0 - 1) * kFp4ScaleBytes;
#pragma unroll
    for (int n = 0; n < TN; ++n)
      sc.w[n] = __builtin_amdgcn_raw_buffer_load_b32(wsres, 4 * lane, (int)(wsp[n] + at), 0);
  };

  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0, 0, 0, 0};

  // Scale bytes past K in the last step's dword, which may be anything, become 0.
  const uint32_t tail = a.K % kFp4Step ? (1u << (8 * (a.K % kFp4Step / kFp4Group))) - 1 : ~0u;
  // Where this lane's operands of the wave's first token tile lie in a slot. The compiler is kept from taking the sums
  // apart: it follows an LDS access to its array through a few additions only.
  int at[A8 ? 2 : 4], sat = kg * XS + r16;
#pragma unroll
  for (int i = 0; i < (A8 ? 2 : 4); ++i) {
    at[i] = kg * SLOT + r16 * CH + ((A8 ? 4 * i + g : 4 * g + i) ^ swz(r16));
    asm volatile("" : "+v"(at[i]));
  }
  asm volatile("" : "+v"(sat));
  // Stage j from slot, whose step is the chunk's t + kg.
  auto compute = [&](int j, auto slot, auto t, const Weights& st, const Scales& chunk) {
    Scales sc = chunk;
    if constexpr (KG > 1) {
#pragma unroll
      for (int n = 0; n < TN; ++n) sc.w[n] >>= 8 * kg;
    }
    if constexpr (A8) {
      const uint32_t mask = 4 * c0 + KG * j + kg == a.nsteps - 1 ? tail : ~0u;
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const uint32_t d = (slot_s(slot)[sat + 16 * i] & mask) >> (8 * g);
        const uint4 lo = slot_x(slot)[at[0] + 16 * CH * i], hi = slot_x(slot)[at[1] + 16 * CH * i];
#pragma unroll
        for (int n = 0; n < TN; ++n)
          acc[i][n] = mfma_fp4_fp8<t>(__builtin_bit_cast(uint4, st.w[n]), sc.w[n], lo, hi, d, acc[i][n]);
      }
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        bf16x8 w[TN];
#pragma unroll
        for (int n = 0; n < TN; ++n) w[n] = fp4_decode8(st.w[n][q], fp4_scale(sc.w[n], t));
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          const bf16x8 xv = as_bf16x8(slot_x(slot)[at[q] + 16 * CH * i]);
#pragma unroll
          for (int n = 0; n < TN; ++n) acc[i][n] = mfma16x16x32(w[n], xv, acc[i][n]);
        }
      }
    }
  };

  // NST register sets of weights, each refilled when its step is done. Issued after a stage's rows when that stage
  // begins: the rows of the NST - 2 later stages, and the weights of the NST - 1. The compiler drops weight loads that
  // no later stage of the last, partial group uses, so there only the rows count.
  constexpr int XLOADS = XI + XSI, ROWS_LATER = (NST - 2) * XLOADS, LATER = (NST - 1) * TN + ROWS_LATER;
  static_assert(LATER < 64, "vmcnt holds at most 63");
  constexpr int U = 4, SC = 4 / KG;  // stages of the loop body: whole chunks, of SC stages, and whole rings
  const int stages = (steps + KG - 1 - kg) / KG, most = (steps + KG - 1) / KG, least = steps / KG;
  static_assert(NST == 2 || NST == 4, "whole rings");
  Weights st[NST];
  Scales sc, next;
  load_s(0, sc);
  unroll<NST - 1>([&](auto i) { load_x(i, i); });
  if constexpr (NST > 2) __builtin_amdgcn_sched_barrier(0);  // rows before weights, as LATER has it
#pragma unroll
  for (int i = 0; i < NST; ++i) load_w(i, st[i]);
  auto body = [&](int base, auto whole) {
    unroll<U>([&](auto u) {
      constexpr int slot = u % NST, ahead = (u + NST - 1) % NST;
      const int s = base + u;
      if (!whole && s >= most) return;
      asm volatile("" ::: "memory");  // the reads of the stage before stay before the barrier
      // This wave's rows of stage s have landed and its reads of the slot that the loads below go to are done; after
      // the barrier every wave's are.
      __builtin_amdgcn_s_waitcnt(vmcnt_lgkm0_imm(whole ? LATER : ROWS_LATER));
      __builtin_amdgcn_s_barrier();
      if constexpr (u % SC == 0) load_s(s / SC + 1, next);
      load_x(s + NST - 1, std::integral_constant<int, ahead>{});
      if (whole || KG == 1 || s < stages)
        compute(s, std::integral_constant<int, slot>{}, std::integral_constant<int, KG * (u % SC)>{}, st[slot], sc);
      // The order of the stage's LDS reads (0x100) and matrix instructions (0x008) of the wide tiles, where a wave has so
      // many of both that the compiler reads a tile and waits for it at once: bf16 rows 2 tiles ahead of their
      // instructions (2048 rows by two 14336 x 4096 weights, tiles of eight waves: 349 -> 340 us), 8-bit rows (two
      // chunks and a scale a tile) likewise (202 -> 198 us).
      if constexpr (TN == 4) {
        constexpr int READS = A8 ? 3 : 1, TILES = A8 ? TM : 4 * TM;
        __builtin_amdgcn_sched_group_barrier(0x100, 2 * READS, 0);
        unroll<TILES - 2>([&](auto) {
          __builtin_amdgcn_sched_group_barrier(0x008, TN, 0);
          __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
        });
        __builtin_amdgcn_sched_group_barrier(0x008, 2 * TN, 0);
      }
      // The stage's rows are issued before its weights, as LATER has it; two slots' assembly keeps its place by itself.
      if constexpr (NST > 2) __builtin_amdgcn_sched_barrier(0);
      load_w(s + NST, st[slot]);
      if constexpr (u % SC == SC - 1) sc = next;
    });
  };
  // Whole groups without tests between their stages, which would make the compiler wait for every load; then the rest.
  int base = 0;
  for (; base + U <= least; base += U) body(base, std::true_type{});
  if (base < most) body(base, std::false_type{});
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
  if constexpr (KG == 2) {
    // The second group's sums go through the slots to the first, which adds them to its own.
    constexpr int PER = 64 * W * TN;
    static_assert(PER * ((TM + NST - 1) / NST) <= KG * SLOT, "the sums fit the slots");
    auto sums = [&](auto i) {
      return reinterpret_cast<f32x4*>(slot_x(std::integral_constant<int, i % NST>{})) + i / NST * PER + 64 * wave * TN +
             lane;
    };
    __syncthreads();
    if (kg) {
      unroll<TM>([&](auto i) {
#pragma unroll
        for (int j = 0; j < TN; ++j) sums(i)[64 * j] = acc[i][j];
      });
    }
    __syncthreads();
    if (kg) return;
    unroll<TM>([&](auto i) {
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] += sums(i)[64 * j];
    });
  }

  // D tile (i, j): lane holds weight rows 4 g + r (r = 0..3) of token row r16.
  const bool yvec = (a.ldy & 3) == 0 && ((uintptr_t)a.y & 7) == 0;
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int m = m0 + 16 * i + r16;
    if (m >= a.M) continue;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int rb = rb0 + wave * TN + j;
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

// Adds the splits' sums of four neighbouring columns in order, and rounds them (gate/up: silu and product first). A launch
// and the sums' way through L2: 64 x 4096 of 4 splits 2.4 us.
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
  if constexpr (A8) {
    if (plan.bm == 128) go(fp4_tile_kernel<true, 128, 256, 1, 2, GLU>, 256);
    if (plan.bm == 64) go(fp4_tile_kernel<true, 64, 128, 1, 4, GLU>, 256);
    if (plan.bm == 32) go(fp4_tile_kernel<true, 32, 128, 1, 4, GLU>, 256);
  } else {
    if (plan.bn == 256) go(fp4_tile_kernel<false, 64, 256, 1, 2, GLU>, 256);
    if (plan.bn == 128 && plan.bm == 64) go(fp4_tile_kernel<false, 64, 128, 2, 2, GLU>, 512);
    if (plan.bn == 128 && plan.bm == 32) go(fp4_tile_kernel<false, 32, 128, 2, 2, GLU>, 512);
  }
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
