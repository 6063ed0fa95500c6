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
};
template <> struct PgT<GX_F16> {
  static __device__ __forceinline__ float lo(uint32_t w) { return h2f((f16_t)(w & 0xffffu)); }
  static __device__ __forceinline__ float hi(uint32_t w) { return h2f((f16_t)(w >> 16)); }
  static __device__ __forceinline__ uint32_t pk(float a, float b) { return pk_f16(a, b); }
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
