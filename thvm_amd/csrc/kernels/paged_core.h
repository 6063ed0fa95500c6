// paged_core.h -- what the paged-cache kernels share beside their indexes
// (../paged_index.h): the 16-bit types, the sequence of a row, the 4-bit codec.
#pragma once
#include "mfma_ops.h"
#include "launch.h"
#include "../paged_index.h"

// the 16-bit type of q, k, v and out
template <int XT> struct PgT;
template <> struct PgT<GX_BF16> {
  static __device__ __forceinline__ float lo(uint32_t w) { return __uint_as_float(w << 16); }
  static __device__ __forceinline__ float hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
  static __device__ __forceinline__ uint32_t pk(float a, float b) { return pk_bf16(a, b); }
  // c + both values of w, in f32
  static __device__ __forceinline__ float sum2(uint32_t w, float c) {
    typedef __bf16 b2_t __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2_t, w), __builtin_bit_cast(b2_t, 0x3f803f80u), c, false);
  }
};
template <> struct PgT<GX_F16> {
  static __device__ __forceinline__ float lo(uint32_t w) { return h2f((f16_t)(w & 0xffffu)); }
  static __device__ __forceinline__ float hi(uint32_t w) { return h2f((f16_t)(w >> 16)); }
  static __device__ __forceinline__ uint32_t pk(float a, float b) { return pk_f16(a, b); }
  static __device__ __forceinline__ float sum2(uint32_t w, float c) {
    typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2_t, w), __builtin_bit_cast(h2_t, 0x3c003c00u), c, false);
  }
};

// the sequence of row r, wave-uniform r: the one whose rows end first behind r
// (a ballot over 64 ends, beyond 64 sequences over every 64th before), or b or more
// for a row of none
__device__ __forceinline__ uint32_t pg_seq_of(const ThvmPagedArgs &a, uint32_t r) {
  if (!a.rows) return r / (a.n / a.b);
  uint32_t s0 = 0;
  if (a.b > 64) {
    const uint64_t behind = __builtin_amdgcn_ballot_w64(a.rows[min(64u * (uint32_t)lane_id() + 64u, a.b)] > (int32_t)r);
    if (!behind) return a.b;
    s0 = 64 * (uint32_t)__builtin_ctzll(behind);
  }
  const uint32_t s = s0 + lane_id();
  const uint64_t behind = __builtin_amdgcn_ballot_w64(s < a.b && a.rows[min(s, a.b - 1) + 1] > (int32_t)r);
  return behind ? s0 + (uint32_t)__builtin_ctzll(behind) : a.b;
}

// ---- 4 bits -----------------------------------------------------------------
// 32 values share a power of two 2^e, the smallest that keeps the largest within
// the codes' 6: with amax = m 2^k (1 <= m < 2) that is e = k - 2 for m <= 1.5 and
// k - 1 above, one add on the bits.  e stays where every code's value is a number
// of the 16-bit type (bf16: 2^-126..2^125, fp16: 2^-23..2^13; larger values
// saturate at 6 2^e).  A group with a value that is not finite has the scale byte
// 255, which makes all its values NaN.  Codes and back by gfx950's own
// converters: nearest, ties to even, saturating; exact on the way back.
template <int XT>
__device__ __forceinline__ uint32_t fp4_scale_byte(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return 255u;
  const int32_t e = (int32_t)((amax_bits + 0x3fffffu) >> 23) - 2;     // + 127
  return (uint32_t)min(max(e, XT == GX_BF16 ? 1 : 104), XT == GX_BF16 ? 252 : 140);
}
__device__ __forceinline__ uint32_t fp4x8(const float v[8], float scale) {
  uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, v[0], v[1], scale, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], scale, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], scale, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], scale, 3);
}
// byte SEL of w -> two 16-bit values
template <int XT, int SEL>
__device__ __forceinline__ uint32_t fp4x2(uint32_t w, float scale) {
  if (XT == GX_BF16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, SEL));
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, SEL));
}
__device__ __forceinline__ float e8m0_f(uint32_t byte) { return __uint_as_float(byte << 23); }

template <bool V> struct pg_const { static constexpr bool value = V; };

// ---- units of work -----------------------------------------------------------
// A kernel takes the sequences whose columns (rows x the G query heads of a kv
// head) number more than lo and at most hi, ct columns a tile, and splits each
// tile's cache rows into chunks of c steps of 64 rows.  Lengths are known on the
// device only and differ, so c is chosen there, by every wave for itself (beyond 64
// sequences by k_paged_plan, once) and from
// the same numbers: the smallest of a few tries between all steps / units and all
// steps / (units - tiles) with which the chunks number at most `units`.  The last
// try always does (a tile adds one chunk at most to its share); the host launches
// units >= 2 x tiles, so c never passes the mean length of the tiles: long
// sequences are split, short ones are not, and the blocks are of one size but for
// the last chunk of each tile.  Those come after the whole ones.  Where that fills
// less than `even` of units x c (short tiles, lengths that c divides badly), `slots` is
// twice `units` and c at least cbig, it is done again with twice the units: a second
// round of blocks costs some 7 us and evens out.  `fuse`: the last block of a tile
// adds its chunks.
struct PgPlan { uint32_t lo, hi, ct, units, cmin, fuse, slots, cbig; float even; const uint32_t *pre; };
struct PgUnit { PgSeq q; uint32_t s, tile, chunk, nchunk, c, first, u; };

__device__ __forceinline__ float wave_scan(float v) {           // inclusive, lane order
  v += dpp_f<0x111>(v);
  v += dpp_f<0x112>(v);
  v += dpp_f<0x114>(v);
  v += dpp_f<0x118>(v);
  v += dpp_f<0x142, 0xa>(v);
  v += dpp_f<0x143, 0xc>(v);
  return v;
}

// a sequence's tiles and steps
__device__ __forceinline__ void pg_count(const ThvmPagedArgs &a, const PgPlan &p, uint32_t s, PgSeq &q, float &tiles, float &steps) {
  const uint32_t G = a.H / a.Hkv;
  q = pg_seq(&a, s);
  const uint32_t rows = (uint32_t)(q.r1 - q.r0), cols = rows * G;
  tiles = rows <= a.t && cols > p.lo && cols <= p.hi ? (float)((cols + p.ct - 1) / p.ct) : 0.0f;
  steps = (float)max((min(q.len, (int32_t)(a.maxpages * a.page)) + 63) / 64, 1);
}
// steps in whole chunks of c, and the number with a shorter last one (steps < 2^24)
__device__ __forceinline__ void pg_chunks(float steps, uint32_t c, float &full, float &per) {
  uint32_t q = (uint32_t)(steps * __builtin_amdgcn_rcpf((float)c));
  int32_t r = (int32_t)((uint32_t)steps - q * c);          // q is off by one at most
  if (r < 0) { q--; r += (int32_t)c; }
  if (r >= (int32_t)c) { q++; r -= (int32_t)c; }
  full = (float)q;
  per = (float)(q + (r != 0));
}
// c of a plan, and its chunks, all and whole; sum(c, n, whole) adds up both over the
// sequences.  Counts stay below 2^24 (2^25 heads / ct), exact in f32; the steps' sum
// need not be.
template <typename F>
__device__ __forceinline__ uint32_t pg_choose(const PgPlan &p, float total, float tiles, F sum, float &n, float &whole) {
  uint32_t c;
  for (float units = (float)p.units;; units *= 2.0f) {
    const uint32_t c1 = max(p.cmin, (uint32_t)(total / units)), c2 = max(c1, (uint32_t)(total * 1.0001f / (units - tiles)) + 1);
    c = c1;
    for (int k = 1;; k++) {
      sum(c, n, whole);
      if (n <= units || k > 4) break;
      c = k == 4 ? c2 : c1 + (c2 - c1) * k / 4;
    }
    if (units >= (float)p.slots || c < p.cbig || total >= p.even * units * (float)c) break;
  }
  if (n > (float)p.slots) n = 0.0f;                        // row offsets that overlap: nothing is done
  return c;
}

// What k_paged_plan leaves for a batch of more than 64 sequences: c, chunks, whole
// chunks and tiles in all, then how many tiles, chunks and whole chunks the sequences
// before each have.
#define PG_PRE_WORDS(b) (4 + 3 * (((b) + 3) & ~3u))

// unit u's tile and chunk, or (tiles_only) tile u's first unit; false: none
__device__ __forceinline__ bool pg_unit(const ThvmPagedArgs &a, const PgPlan &p, uint32_t u, bool tiles_only, PgUnit &o) {
  const uint32_t lane = lane_id(), bb = (a.b + 3) & ~3u;
  float t = 0.0f, l = 1.0f, n, whole, tiles;
  PgSeq q = {0, 0, 0};
  if (p.pre) {
    const uint4 h = *(const uint4 *)p.pre;
    o.c = h.x;
    n = (float)h.y;
    whole = (float)h.z;
    tiles = (float)h.w;
  } else {
    if (lane < a.b) pg_count(a, p, lane, q, t, l);
    tiles = wave_sum(t);
    if (tiles == 0.0f) return false;
    o.c = pg_choose(p, wave_sum(t * l), tiles, [&](uint32_t c, float &sn, float &sw) {
      float full, per;
      pg_chunks(l, c, full, per);
      sn = wave_sum(t * per);
      sw = wave_sum(t * full);
    }, n, whole);
  }
  // the order of the blocks: whole chunks first, then the tiles' shorter last ones (all
  // of a tile where none is split: backwards, as a prompt's last tiles see most)
  if (n == 0.0f || (float)u >= (tiles_only ? tiles : n)) return false;
  const bool rest = !tiles_only && (float)u >= whole;
  const uint32_t at = tiles_only ? u : whole == 0.0f ? (uint32_t)n - 1 - u : rest ? u - (uint32_t)whole : u;
  float full, per;
  uint32_t i, first;                                       // among the sequence's, and its first unit
  if (p.pre) {
    const uint32_t *const tb = p.pre + 4, *const nb = tb + bb, *const wb = nb + bb;
    auto key = [&](uint32_t s) { return tiles_only ? tb[s] : rest ? nb[s] - wb[s] : wb[s]; };
    // the last sequence with no more before it than at: every 64th, then those between
    auto last = [&](uint32_t s, uint32_t most) {
      const uint64_t m = __builtin_amdgcn_ballot_w64(s < most && key(min(s, a.b - 1)) <= at);
      return 63u - (uint32_t)__builtin_clzll(m | 1);
    };
    o.s = 64 * last(64 * lane, a.b);
    o.s += last(o.s + lane, a.b);
    pg_count(a, p, o.s, o.q, t, l);
    pg_chunks(l, o.c, full, per);
    i = at - key(o.s);
    first = nb[o.s];
  } else {
    pg_chunks(l, o.c, full, per);
    const float k = tiles_only ? t : t * (rest ? per - full : full), cn = t * per;
    const float kc = wave_scan(k), nc = wave_scan(cn);
    const int w = __builtin_ctzll(__builtin_amdgcn_ballot_w64(kc > (float)at) | 1ull << 63);
    auto get = [&](float v) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), w)); };
    o.s = w;
    o.q.r0 = __builtin_amdgcn_readlane(q.r0, w);
    o.q.r1 = __builtin_amdgcn_readlane(q.r1, w);
    o.q.len = __builtin_amdgcn_readlane(q.len, w);
    i = at - (uint32_t)get(kc - k);
    first = (uint32_t)get(nc - cn);
    full = get(full);
    per = get(per);
  }
  const uint32_t f = (uint32_t)full;
  o.nchunk = (uint32_t)per;
  o.tile = tiles_only || rest ? i : i / f;
  o.chunk = tiles_only ? 0 : rest ? f : i % f;
  o.first = first + o.tile * o.nchunk;
  o.u = o.first + o.chunk;
  return true;
}

typedef void (*paged_fn)(ThvmPagedArgs, PgPlan);
// the kernel of many columns (paged_prompt.hip), PP_COLS a block
#define PP_WAVES 4
#define PP_THREADS (PP_WAVES * 64)
#define PP_COLS (PP_WAVES * 32)
paged_fn pp_tile_pick(const ThvmPagedArgs *a);
