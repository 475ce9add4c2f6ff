// Rotary positions from fp32 tables, by themselves (rope_kernel) and on the way into the 8-bit paged K/V cache
// (append_kv_kernel).
//
// The rotation of a pair (a, b) by the angle whose cosine and sine the tables hold is (a c - b s, b c + a s),
// every product and sum rounded in fp32 (no fused forms, so that a value and its code depend on the formula
// alone), the result rounded once: to bf16, or to its code. Pair i of the first `rotary` dims is (i, i +
// rotary / 2), or (2 i, 2 i + 1) interleaved; the dims behind are passed on.
//
// A thread's unit is 16 dims of a token's head: eight pairs, or 16 dims to pass on.
//
// On MI355X: a batch of three prompts (about 4000 tokens, 32 heads over 8 of 128) is rotated in 18.1 us (4.5 TB/s of
// values and tables in and out) and appended in 21.9 us (4.6 TB/s); one decode row, and 64, take 2.7 and 7.1 us on the
// GPU, less than their launches.
#include <algorithm>

#include "fp8_kv.h"

namespace lse {

// Rows (token, head) of bf16 values: element (t, h, d) at t * st + h * sh + d.
struct RowsIn {
  const uint16_t* p;
  int64_t st, sh;
};

struct RopeTables {
  const float *cos, *sin;  // (rows, half) each
  int64_t rows;
  int half;  // rotary / 2
  int interleaved;
};

// Offsets of a unit's two runs of eight dims.
struct UnitDims {
  int a, b;
  bool turned;
};
__device__ __forceinline__ UnitDims unit_dims(const RopeTables& r, int unit) {
  UnitDims u{16 * unit, 16 * unit + 8, 16 * unit < 2 * r.half};
  if (u.turned && !r.interleaved) u.a = 8 * unit, u.b = r.half + 8 * unit;
  return u;
}

__device__ __forceinline__ void unpack8(uint4 w, float (&x)[8]) {
  const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __builtin_bit_cast(float, v[i] << 16);
    x[2 * i + 1] = __builtin_bit_cast(float, v[i] & 0xffff0000u);
  }
}

// The cosines and sines of a unit's eight pairs at `pos`; of a position outside the tables NaN.
struct Turn {
  float c[8], s[8];
};
__device__ __forceinline__ Turn turn_at(const RopeTables& r, int unit, int pos) {
  Turn t;
  const bool known = pos >= 0 && pos < r.rows;
  const int64_t at = (int64_t)(known ? pos : 0) * r.half + 8 * unit;
#pragma unroll
  for (int i = 0; i < 8; i += 4) {
    *reinterpret_cast<float4*>(t.c + i) = *reinterpret_cast<const float4*>(r.cos + at + i);
    *reinterpret_cast<float4*>(t.s + i) = *reinterpret_cast<const float4*>(r.sin + at + i);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    t.c[i] = known ? t.c[i] : __builtin_nanf("");
    t.s[i] = known ? t.s[i] : __builtin_nanf("");
  }
  return t;
}

// Turns the 16 dims of a unit, two runs of eight.
__device__ __forceinline__ void turn_unit(const Turn& t, bool interleaved, float (&x)[8], float (&y)[8]) {
#pragma clang fp contract(off)
  auto turn = [&](float& a, float& b, float c, float s) {
    const float p = a * c - b * s, q = b * c + a * s;
    a = p, b = q;
  };
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (interleaved) {
      float(&v)[8] = i < 4 ? x : y;
      turn(v[2 * (i & 3)], v[2 * (i & 3) + 1], t.c[i], t.s[i]);
    } else {
      turn(x[i], y[i], t.c[i], t.s[i]);
    }
  }
}

__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  return make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]),
                    pack_bf16x2(x[6], x[7]));
}

struct RopeFp32Args {
  RowsIn q, k;
  RopeTables r;
  const int32_t* positions;
  uint16_t *q_out, *k_out;  // (tokens, heads, D)
  int H, HKV, D, units;     // units: of one token
};

// One thread per unit, in the rows' order, so that a token's heads share its cosines and sines in the caches; bound by
// HBM (each value in and out once), at decode sizes by the launch.
__global__ void __launch_bounds__(256) rope_kernel(RopeFp32Args a, int64_t total) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= total) return;
  const int64_t t = i / a.units;
  const int u = (int)(i - t * a.units), per = a.D / 16;
  const int head = u / per, unit = u - head * per;
  const bool is_q = head < a.H;
  const RowsIn& in = is_q ? a.q : a.k;
  const int h = is_q ? head : head - a.H;
  const UnitDims d = unit_dims(a.r, unit);
  const uint16_t* row = in.p + t * in.st + h * in.sh;
  const uint4 lo = *reinterpret_cast<const uint4*>(row + d.a), hi = *reinterpret_cast<const uint4*>(row + d.b);
  float x[8], y[8];
  unpack8(lo, x), unpack8(hi, y);
  if (d.turned) turn_unit(turn_at(a.r, unit, a.positions[t]), a.r.interleaved, x, y);
  uint16_t* out = (is_q ? a.q_out + (t * a.H + h) * a.D : a.k_out + (t * a.HKV + h) * a.D);
  *reinterpret_cast<uint4*>(out + d.a) = pack8(x);
  *reinterpret_cast<uint4*>(out + d.b) = pack8(y);
}

struct AppendArgs {
  RowsIn q, k, v;  // q.p may be null
  RopeTables r;    // half 0: no rotation
  uint16_t* q_out;  // (tokens, H, D)
  Fp8Pool pool;
  const int32_t* block_table;  // (entries, max_blocks), row stride sbt
  int64_t sbt;
  const int32_t *query_offset, *q_start, *q_len;
  int entries, H, HKV, G, max_groups;  // max_groups: groups that the table has room for
  int64_t tokens;
  int one;  // every entry has at most one new token
};

// An entry's new tokens whose rows are the call's, [m0, m1), and the groups of 16 positions that they touch: where the
// offset is negative, those before position 0 too, whose q rows are the call's as well. Groups are counted from the
// one of the offset, in which that is slot `lead`.
struct NewTokens {
  int offset, start, m0, m1;
  __device__ __forceinline__ int offset_group() const { return offset >> 4; }
  __device__ __forceinline__ int lead() const { return offset & 15; }
  __device__ __forceinline__ int first() const { return (int)(((unsigned)lead() + (unsigned)m0) >> 4); }
  __device__ __forceinline__ int groups() const {
    return m0 >= m1 ? 0 : (int)(((unsigned)lead() + (unsigned)m1 - 1) >> 4) - first() + 1;
  }
};
static_assert(kKvGroup == 16, "groups by shifts");
__device__ __forceinline__ NewTokens new_tokens(const AppendArgs& a, int e) {
  const int start = a.q_start[e];
  return {a.query_offset[e], start, (int)min(max(-(int64_t)start, (int64_t)0), (int64_t)0x7fffffff),
          (int)min((int64_t)a.q_len[e], a.tokens - start)};
}

// A workgroup takes one group of one K/V head: its up to 16 new tokens' k and v rows, and their rows of the G
// query heads. A thread has one (token, unit): of k in the first T threads, of v in the next T, and of every (256 /
// T)th query head, whose cosines and sines are loaded once. The group's image (codes in pool order) is built in
// LDS: what it held of earlier positions, requantised where the scale grew; the new codes; zeros behind them;
// then it is written whole. At decode sizes this is bound by its chain of dependent loads (lengths, table, scale and
// codes), which are issued as soon as their addresses are known, at prompt sizes by HBM. Three prompts, us: with a
// thread's q units taken one by one behind k and v, cosines and sines loaded for each 24.7; two heads' q at a time
// 21.9, one 22.9; at six waves a SIMD instead of five, which spills, 33.3.
template <int D>
__global__ void __launch_bounds__(256) append_kv_kernel(AppendArgs a) {
  constexpr int U = D / 16;      // units of a row
  constexpr int T = 16 * U;      // threads of k, and of v
  static_assert(2 * T <= 256, "k's and v's threads in one workgroup");
  __shared__ __attribute__((aligned(16))) uint8_t image[2][16 * D];
  __shared__ float wave_max[4];

  // A group's K/V heads go to one XCD (workgroups are dealt to the eight in turn), which then reads the rows of cos and
  // sin once: three prompts 26.3 -> 24.7 us.
  int kvh = blockIdx.x % a.HKV, slot_id = blockIdx.x / a.HKV, e = -1, first = 0;
  if (!a.one) {
    kvh = blockIdx.x / 8 % a.HKV;
    slot_id = blockIdx.x / 8 / a.HKV * 8 + blockIdx.x % 8;
  }
  if (a.one) {
    e = slot_id;
  } else {
    // The entry of this unit, and the unit's place in it: a sum over the entries' groups, 64 at a time.
    const int lane = threadIdx.x & 63;
    for (int e0 = 0; e0 < a.entries; e0 += 64) {
      const int i = e0 + lane;
      const int mine = i < a.entries ? new_tokens(a, i).groups() : 0;
      const int before = kv_wave_scan(mine) - mine;
      const unsigned long long hit = __ballot((unsigned)(slot_id - before) < (unsigned)mine);
      if (hit) {
        const int at = __ffsll(hit) - 1;
        e = e0 + at;
        first = slot_id - __builtin_amdgcn_readlane(before, at);
        break;
      }
      slot_id -= __builtin_amdgcn_readlane(before + mine, 63);
    }
    if (e < 0) return;
  }
  const NewTokens entry = new_tokens(a, e);
  const int offset = entry.offset, n = entry.m1, start = entry.start;
  if (entry.groups() == 0) return;
  const int run = entry.first() + first, group = entry.offset_group() + run;
  // New tokens' slots of the group: [lo, hi), slot s being token s + base of the entry.
  const int base = run * kKvGroup - entry.lead();
  const int lo = max(0, -base), hi = (int)min((int64_t)kKvGroup, (int64_t)n - base);

  // The group's place, and what it held, if it holds earlier positions.
  const int what = threadIdx.x / T, unit = threadIdx.x % U, slot = threadIdx.x % T / U;
  const int block =
      offset >= 0 && group < a.max_groups ? a.block_table[(int64_t)e * a.sbt + group / a.pool.per] : -1;
  const bool held = block >= 0 && block < a.pool.blocks;  // dropped otherwise
  const int64_t inner = (int64_t)kvh * a.pool.per + group % a.pool.per;

  // The new rows; tokens of rows outside the call's are dropped.
  const int64_t row = (int64_t)start + base + slot;
  const bool in = slot >= lo && slot < hi && row >= 0 && row < a.tokens, mine = in && what < 2;
  const RowsIn& from = what == 0 ? a.k : a.v;
  const UnitDims turned = unit_dims(a.r, unit);
  const UnitDims dims = what == 0 ? turned : UnitDims{16 * unit, 16 * unit + 8, false};
  uint4 xa = make_uint4(0, 0, 0, 0), xb = xa;
  if (mine) {
    const uint16_t* p = from.p + row * from.st + (int64_t)kvh * from.sh;
    xa = *reinterpret_cast<const uint4*>(p + dims.a);
    xb = *reinterpret_cast<const uint4*>(p + dims.b);
  }
  Turn turn{};
  if (in && turned.turned && (a.q.p || what == 0)) turn = turn_at(a.r, unit, (int)((unsigned)group * kKvGroup + slot));
  uint8_t* scale_at = a.pool.scales + (int64_t)(held ? block : 0) * a.pool.ss + 2 * inner;
  const int64_t bytes = (int64_t)(held ? block : 0) * a.pool.sb + inner * (16 * D) + 16 * (threadIdx.x % T);
  uint8_t* at = (what == 0 ? a.pool.k : a.pool.v) + bytes;
  // A thread's 16 bytes: k, of slot 4 i + j; v, all 16 slots of a dim.
  const int in_slot = threadIdx.x % T / (D / 64 * 16) * 4 + threadIdx.x % T / 4 % 4;
  uint4 kept = make_uint4(0, 0, 0, 0);
  int old = 0;
  if (held && what < 2 && lo > 0) {
    old = scale_at[what];
    if (what == 1 || in_slot < lo) kept = *reinterpret_cast<const uint4*>(at);
  }
  if (a.q.p && in) {
    constexpr int P = 256 / T, B = 2;
    for (int g0 = what; g0 < a.G; g0 += B * P) {
      uint4 qa[B], qb[B];
#pragma unroll
      for (int i = 0; i < B; ++i) {
        const int g = min(g0 + i * P, a.G - 1);
        const uint16_t* p = a.q.p + row * a.q.st + (int64_t)(kvh * a.G + g) * a.q.sh;
        qa[i] = *reinterpret_cast<const uint4*>(p + turned.a);
        qb[i] = *reinterpret_cast<const uint4*>(p + turned.b);
      }
#pragma unroll
      for (int i = 0; i < B; ++i) {
        const int g = g0 + i * P;
        if (g >= a.G) break;
        float qx[8], qy[8];
        unpack8(qa[i], qx), unpack8(qb[i], qy);
        if (turned.turned) turn_unit(turn, a.r.interleaved, qx, qy);
        uint16_t* out = a.q_out + (row * a.H + kvh * a.G + g) * D;
        *reinterpret_cast<uint4*>(out + turned.a) = pack8(qx);
        *reinterpret_cast<uint4*>(out + turned.b) = pack8(qy);
      }
    }
  }
  if (!held) return;
  float x[8], y[8];
  unpack8(xa, x), unpack8(xb, y);
  if (dims.turned) turn_unit(turn, a.r.interleaved, x, y);

  // k's and v's largest finite magnitudes.
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float ax = __builtin_fabsf(x[i]), ay = __builtin_fabsf(y[i]);
    top = fmaxf(top, ax < __builtin_huge_valf() ? ax : 0.0f);
    top = fmaxf(top, ay < __builtin_huge_valf() ? ay : 0.0f);
  }
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
  if ((threadIdx.x & 63) == 0) wave_max[threadIdx.x >> 6] = top;
  __syncthreads();
  if (what < 2) {
    constexpr int W = T / 64;  // waves of k, and of v
    top = wave_max[what * W];
#pragma unroll
    for (int i = 1; i < W; ++i) top = fmaxf(top, wave_max[what * W + i]);
  }
  const int byte = max(kv_scale_byte(top), old == kKvScaleNan ? 0 : old);
  uint4* img = reinterpret_cast<uint4*>(image[what & 1] + 16 * (threadIdx.x % T));
  if (what < 2) {
    if (lo > 0 && (what == 1 || in_slot < lo)) {
      if (byte != old) {
        const float ratio = old == kKvScaleNan ? __builtin_nanf("")
                            : byte - old > 126 ? 0.0f
                                               : kv_scale(127 + old - byte);
        kept = make_uint4(kv_requantize4(kept.x, ratio), kv_requantize4(kept.y, ratio),
                          kv_requantize4(kept.z, ratio), kv_requantize4(kept.w, ratio));
      }
      if (what == 1) {
        auto mask = [&](int w) {
          const int nb = min(max(lo - 4 * w, 0), 4);
          return nb == 4 ? 0xffffffffu : (1u << (8 * nb)) - 1u;
        };
        kept.x &= mask(0), kept.y &= mask(1), kept.z &= mask(2), kept.w &= mask(3);
      }
    }
    *img = kept;
  }
  __syncthreads();
  if (mine) {
    const float inv = kv_scale_inverse(byte);
    uint32_t c[4] = {kv_encode4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv),
                     kv_encode4(x[4] * inv, x[5] * inv, x[6] * inv, x[7] * inv),
                     kv_encode4(y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv),
                     kv_encode4(y[4] * inv, y[5] * inv, y[6] * inv, y[7] * inv)};
    if (__builtin_expect(byte >= kKvScaleTop, 0)) {
#pragma unroll
      for (int i = 0; i < 4; ++i) c[i] = kv_keep_finite4(c[i], byte);
    }
    if (what == 0) {
      auto put = [&](int d, uint32_t w0, uint32_t w1) {
        uint8_t* to = image[0] + ((slot / 4 * (D / 64) + d / 64) * 4 + slot % 4) * 64 + d % 64;
        *reinterpret_cast<uint2*>(to) = make_uint2(w0, w1);
      };
      put(dims.a, c[0], c[1]);
      put(dims.b, c[2], c[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        image[1][16 * ((i < 8 ? dims.a : dims.b) + i % 8) + slot] = (uint8_t)(c[i / 4] >> (8 * (i % 4)));
    }
  }
  __syncthreads();
  if (what < 2) {
    *reinterpret_cast<uint4*>(at) = *img;
    if (threadIdx.x % T == 0) scale_at[what] = (uint8_t)byte;
  }
}

}  // namespace lse

namespace {

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
constexpr int64_t kMax31 = 2147483647;

int check_rows(const void* p, int64_t st, int64_t sh) {
  if (st < 0 || sh < 0) return LSE_E_SHAPE;
  return st % 8 || sh % 8 || !aligned16(p) ? LSE_E_ALIGN : LSE_OK;
}

}  // namespace

extern "C" {

int lse_rope(const struct lse_rope_args* args, void* stream) {
  if (!args) return LSE_E_NULL;
  const lse_rope_args& x = *args;
  if (x.tokens < 0 || x.tokens > kMax31 || x.H < 1 || x.H > 65536 || x.H_KV < 0 || x.H_KV > 65536 ||
      x.D < 16 || x.D > 1024 || x.D % 16 || x.rotary < 16 || x.rotary > x.D || x.rotary % 16 ||
      x.table_rows < 1 || (x.interleaved != 0 && x.interleaved != 1))
    return LSE_E_SHAPE;
  if (x.tokens == 0) return LSE_OK;
  if (!x.q || !x.q_out || !x.cos || !x.sin || !x.positions || (x.H_KV > 0 && (!x.k || !x.k_out)))
    return LSE_E_NULL;
  if (int st = check_rows(x.q, x.q_stride_t, x.q_stride_h)) return st;
  if (x.H_KV > 0)
    if (int st = check_rows(x.k, x.k_stride_t, x.k_stride_h)) return st;
  if (!aligned16(x.cos) || !aligned16(x.sin) || !aligned16(x.q_out) || !aligned16(x.k_out) ||
      ((uintptr_t)x.positions & 3))
    return LSE_E_ALIGN;
  lse::RopeFp32Args a{};
  a.q = {(const uint16_t*)x.q, x.q_stride_t, x.q_stride_h};
  a.k = {(const uint16_t*)x.k, x.k_stride_t, x.k_stride_h};
  a.r = {x.cos, x.sin, x.table_rows, (int)(x.rotary / 2), (int)x.interleaved};
  a.positions = x.positions;
  a.q_out = (uint16_t*)x.q_out, a.k_out = (uint16_t*)x.k_out;
  a.H = (int)x.H, a.HKV = (int)x.H_KV, a.D = (int)x.D;
  a.units = (int)((x.H + x.H_KV) * (x.D / 16));
  const int64_t total = x.tokens * a.units, blocks = lse::ceil_div(total, 256);
  if (blocks > kMax31) return LSE_E_RANGE;
  hipLaunchKernelGGL(lse::rope_kernel, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, a, total);
  return lse::launch_status();
}

int lse_append_kv_fp8(const struct lse_append_kv_fp8_args* args, void* stream) {
  if (!args) return LSE_E_NULL;
  const lse_append_kv_fp8_args& x = *args;
  if (x.entries < 0 || x.entries > kMax31 || x.tokens < 0 || x.tokens > kMax31 || x.max_q_len < 0 ||
      x.max_q_len > kMax31 || x.H < 1 || x.H > 65536 || x.H_KV < 1 || x.H % x.H_KV ||
      (x.D != 64 && x.D != 128) || x.rotary < 0 || x.rotary > x.D || x.rotary % 16 ||
      (x.interleaved != 0 && x.interleaved != 1) || x.num_blocks < 0 || x.num_blocks > kMax31 ||
      x.block_size < 16 || x.block_size % 16 || x.max_blocks < 0 || x.block_table_stride < x.max_blocks)
    return LSE_E_SHAPE;
  if (x.block_size > kMax31 || x.max_blocks > kMax31 / x.block_size) return LSE_E_RANGE;
  const int64_t per = x.block_size / 16;
  if (x.pool_stride_block < x.H_KV * per * 16 * x.D || x.scales_stride_block < 2 * x.H_KV * per)
    return LSE_E_SHAPE;
  if (x.entries == 0 || x.tokens == 0 || x.max_q_len == 0) return LSE_OK;
  if (!x.k || !x.v || !x.k_pool || !x.v_pool || !x.scales || !x.block_table || !x.query_offset ||
      !x.q_start || !x.q_len || (x.q && !x.q_out) || (x.rotary > 0 && (!x.cos || !x.sin)))
    return LSE_E_NULL;
  if (x.rotary > 0 && x.table_rows < 1) return LSE_E_SHAPE;
  if (x.q)
    if (int st = check_rows(x.q, x.q_stride_t, x.q_stride_h)) return st;
  if (int st = check_rows(x.k, x.k_stride_t, x.k_stride_h)) return st;
  if (int st = check_rows(x.v, x.v_stride_t, x.v_stride_h)) return st;
  if (x.pool_stride_block % 16 || !aligned16(x.cos) || !aligned16(x.sin) || !aligned16(x.q_out) ||
      !aligned16(x.k_pool) || !aligned16(x.v_pool))
    return LSE_E_ALIGN;
  lse::AppendArgs a{};
  a.q = {(const uint16_t*)x.q, x.q_stride_t, x.q_stride_h};
  a.k = {(const uint16_t*)x.k, x.k_stride_t, x.k_stride_h};
  a.v = {(const uint16_t*)x.v, x.v_stride_t, x.v_stride_h};
  a.r = {x.cos, x.sin, x.table_rows, (int)(x.rotary / 2), (int)x.interleaved};
  a.q_out = (uint16_t*)x.q_out;
  a.pool = {(uint8_t*)x.k_pool, (uint8_t*)x.v_pool, (uint8_t*)x.scales, x.pool_stride_block,
            x.scales_stride_block, (int)x.num_blocks, (int)per};
  a.block_table = x.block_table, a.sbt = x.block_table_stride;
  a.query_offset = x.query_offset, a.q_start = x.q_start, a.q_len = x.q_len;
  a.entries = (int)x.entries, a.H = (int)x.H, a.HKV = (int)x.H_KV, a.G = (int)(x.H / x.H_KV);
  a.max_groups = (int)(x.max_blocks * per);
  a.tokens = x.tokens;
  a.one = x.max_q_len == 1;
  // An entry of n tokens touches at most (n + 30) / 16 groups; the entries' rows are distinct.
  const int64_t most = std::min(x.entries * ((x.max_q_len + 30) / 16), x.tokens / 16 + 2 * x.entries);
  const int64_t blocks = (a.one ? x.entries : lse::ceil_div(most, 8) * 8) * x.H_KV;
  if (blocks > kMax31) return LSE_E_RANGE;
  const dim3 grid((unsigned)blocks), wg(256);
  if (x.D == 64)
    hipLaunchKernelGGL(lse::append_kv_kernel<64>, grid, wg, 0, (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL(lse::append_kv_kernel<128>, grid, wg, 0, (hipStream_t)stream, a);
  return lse::launch_status();
}

}  // extern "C"
