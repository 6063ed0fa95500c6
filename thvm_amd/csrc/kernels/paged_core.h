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
// (a ballot over 64 ends at a time), or b for a row of none
__device__ __forceinline__ uint32_t pg_seq_of(const ThvmPagedArgs &a, uint32_t r) {
  if (!a.rows) return r / (a.n / a.b);
  for (uint32_t s0 = 0; s0 < a.b; s0 += 64) {
    const uint32_t s = s0 + lane_id();
    const uint64_t behind = __builtin_amdgcn_ballot_w64(s < a.b && a.rows[min(s, a.b - 1) + 1] > (int32_t)r);
    if (behind) return s0 + (uint32_t)__builtin_ctzll(behind);
  }
  return a.b;
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
// device only and differ, so c is chosen there, by every wave for itself and from
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
struct PgPlan { uint32_t lo, hi, ct, units, cmin, fuse, slots, cbig; float even; };
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

// unit u's tile and chunk, or (tiles_only) tile u's first unit; false: none.
// Counts stay below 2^24 (2^25 heads / ct), exact in f32; the steps' sum need not
// be.
__device__ __forceinline__ bool pg_unit(const ThvmPagedArgs &a, const PgPlan &p, uint32_t u, bool tiles_only, PgUnit &o) {
  const uint32_t lane = lane_id(), G = a.H / a.Hkv;
  const int32_t cap = (int32_t)(a.maxpages * a.page);
  // a lane's sequence of each 64: its tiles and steps (the first 64 kept)
  auto load = [&](uint32_t s0, PgSeq &q, float &tiles, float &steps) {
    const uint32_t s = s0 + lane;
    tiles = steps = 0.0f;
    if (s < a.b) {
      q = pg_seq(&a, s);
      const uint32_t rows = (uint32_t)(q.r1 - q.r0), cols = rows * G;
      if (rows <= a.t && cols > p.lo && cols <= p.hi) tiles = (float)((cols + p.ct - 1) / p.ct);
      steps = (float)max((min(q.len, cap) + 63) / 64, 1);
    }
  };
  PgSeq q0 = {0, 0, 0}, q;
  float t0, l0, tl, st;
  load(0, q0, t0, l0);
  auto each = [&](auto f) {
    f(0u, q0, t0, l0);
    for (uint32_t s0 = 64; s0 < a.b; s0 += 64) {
      load(s0, q, tl, st);
      f(s0, q, tl, st);
    }
  };
  float total = 0.0f, tiles = 0.0f;
  each([&](uint32_t, const PgSeq &, float t, float l) { total += wave_sum(t * l); tiles += wave_sum(t); });
  if (tiles == 0.0f) return false;
  // steps in whole chunks of c, and the number with a shorter last one (l < 2^24)
  auto chunks = [](float l, uint32_t c, float rc, float &full, float &per) {
    uint32_t q = (uint32_t)(l * rc);
    int32_t r = (int32_t)((uint32_t)l - q * c);            // q is off by one at most
    if (r < 0) { q--; r += (int32_t)c; }
    if (r >= (int32_t)c) { q++; r -= (int32_t)c; }
    full = (float)q;
    per = (float)(q + (r != 0));
  };
  uint32_t c;
  float n, whole;
  for (float units = (float)p.units;; units *= 2.0f) {
    const uint32_t c1 = max(p.cmin, (uint32_t)(total / units)), c2 = max(c1, (uint32_t)(total * 1.0001f / (units - tiles)) + 1);
    c = c1;
    for (int k = 1;; k++) {
      n = whole = 0.0f;
      const float rc = __builtin_amdgcn_rcpf((float)c);
      each([&](uint32_t, const PgSeq &, float t, float l) {
        float full, per;
        chunks(l, c, rc, full, per);
        n += wave_sum(t * per);
        whole += wave_sum(t * full);
      });
      if (n <= units || k > 4) break;
      c = k == 4 ? c2 : c1 + (c2 - c1) * k / 4;
    }
    if (units >= (float)p.slots || c < p.cbig || total >= p.even * units * (float)c) break;
  }
  if (n > (float)p.slots) return false;                    // row offsets that overlap: nothing is done
  o.c = c;
  // the order of the blocks: whole chunks first, then the tiles' shorter last ones (all
  // of a tile where none is split: backwards, as a prompt's last tiles see most)
  uint32_t at = u;
  bool rest = false;
  if (!tiles_only) {
    if ((float)u >= n) return false;
    rest = (float)u >= whole;
    at = rest ? u - (uint32_t)whole : u;
    if (whole == 0.0f) at = (uint32_t)n - 1 - u;
  }
  const float rc = __builtin_amdgcn_rcpf((float)c);
  float before = 0.0f, kbefore = 0.0f;
  bool found = false;
  each([&](uint32_t s0, const PgSeq &q, float t, float l) {
    if (found) return;
    float full, per;
    chunks(l, c, rc, full, per);
    const float n = t * per;
    const float key = tiles_only ? t : t * (rest ? per - full : full);
    const float sc = wave_scan(n), kc = wave_scan(key);
    const uint64_t hit = __builtin_amdgcn_ballot_w64(kbefore + kc > (float)at);
    if (hit) {
      const int w = __builtin_ctzll(hit);
      auto get = [&](float v) { return (uint32_t)__int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), w)); };
      found = true;
      o.s = s0 + w;
      o.q.r0 = __builtin_amdgcn_readlane(q.r0, w);
      o.q.r1 = __builtin_amdgcn_readlane(q.r1, w);
      o.q.len = __builtin_amdgcn_readlane(q.len, w);
      o.nchunk = get(per);
      const uint32_t i = at - get(kbefore + kc - key), f = get(full);
      o.tile = tiles_only || rest ? i : i / f;
      o.chunk = tiles_only ? 0 : rest ? f : i % f;
      o.first = get(before + sc - n) + o.tile * o.nchunk;
      o.u = o.first + o.chunk;
    }
    before += wave_sum(n);
    kbefore += wave_sum(key);
  });
  return found;
}

typedef void (*paged_fn)(ThvmPagedArgs, PgPlan);
// the kernel of many columns (paged_prompt.hip), PP_COLS a block
#define PP_WAVES 4
#define PP_THREADS (PP_WAVES * 64)
#define PP_COLS (PP_WAVES * 32)
paged_fn pp_tile_pick(const ThvmPagedArgs *a);
