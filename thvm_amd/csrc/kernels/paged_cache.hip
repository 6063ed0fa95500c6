// paged_cache.hip -- filling a paged cache and reading it back.
//
// k_kv_append: one pass over the projection's rows [n][q heads, k heads, v
// heads]: the RMS norm of each q and k head (y = (x inv) g, inv = 1 / sqrt(mean
// x^2 + eps)), the rotation at the row's position, q out and k, v into their
// pages.  The arithmetic is f32 with one rounding at the end; the sum of squares
// and inv are f64 (16-bit squares are exact in f32, and 64 bits keep their sum
// the same in any order), and products and sums of the rotation round one by one
// (no contraction): next to a border between two 4-bit codes every order of
// evaluation then picks the same code.
//   * a lane owns 8 consecutive values (one 16-byte load), 16 or 8 lanes a head,
//     a wave 4 or 8 heads of ONE row, so its sequence, position and page are
//     wave-uniform and found once;
//   * the partner of a half rotation and the 32 values of a 4-bit group lie in
//     the head's own lanes: no LDS.
// Bound by its bytes: each value read once, written once (2 or 17/32 bytes).
// k_kv_read is the way back: the same rows' k and v as 16-bit values.
#include "paged_core.h"

#define PC_THREADS 256

template <int CTRL>
__device__ __forceinline__ double dpp_d(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (uint32_t)u, CTRL, 0xf, 0xf, true);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (uint32_t)(u >> 32), CTRL, 0xf, 0xf, true);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u(uint32_t v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xf, 0xf, true);
}

template <int HD, int XT, int BITS>
__global__ __launch_bounds__(PC_THREADS) void k_kv_append(ThvmPagedArgs a) {
#pragma clang fp contract(off)
  typedef PgT<XT> P;
  constexpr int LPV = HD / 8, VPW = 64 / LPV;          // lanes a head, heads a wave
  const uint32_t heads = a.H + 2 * a.Hkv, grps = (heads + VPW - 1) / VPW;
  const uint32_t wid = __builtin_amdgcn_readfirstlane(blockIdx.x * (PC_THREADS / 64) + (threadIdx.x >> 6));
  const uint32_t row = wid / grps, lane = lane_id();
  if (row >= a.n) return;
  const uint32_t s = pg_seq_of(a, row);
  if (s >= a.b) return;
  const PgSeq sq = pg_seq(&a, s);
  if ((int32_t)row < sq.r0 || (int32_t)row >= sq.r1) return;
  const int32_t pos = sq.len - (sq.r1 - (int32_t)row);
  const uint32_t hv = (wid % grps) * VPW + lane / LPV, d0 = lane % LPV * 8;
  const bool live = hv < heads, isq = hv < a.H, isv = hv >= a.H + a.Hkv;
  const bool placed = pos >= 0 && (uint32_t)pos < a.maxpages * a.page;
  float v[8];
  {
    const uint4 w = live ? ld_stream16((const uint16_t *)a.x + (uint64_t)row * a.ldx + hv * HD + d0) : make_uint4(0, 0, 0, 0);
    const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; i++) { v[2 * i] = P::lo(ww[i]); v[2 * i + 1] = P::hi(ww[i]); }
  }
  if (a.norm) {                                         // (every lane: the sums are cross-lane)
    double ss = 0.0;
#pragma unroll
    for (int i = 0; i < 8; i++) ss += (double)(v[i] * v[i]);
    ss += dpp_d<0xB1>(ss);
    ss += dpp_d<0x4E>(ss);
    ss += dpp_d<0x141>(ss);
    if (LPV == 16) ss += dpp_d<0x140>(ss);
    const float inv = (float)(1.0 / sqrt(ss / (double)HD + (double)a.eps));
    if (!isv) {
      const float *g = (isq ? a.gq : a.gk) + d0;
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] = (v[i] * inv) * g[i];
    }
  }
  if (a.rope && placed) {
    const uint64_t tb = (uint64_t)pos * (HD / 2);
    if (a.rope == 1) {
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float c = isv ? 1.0f : a.cos_t[tb + d0 / 2 + j], sn = isv ? 0.0f : a.sin_t[tb + d0 / 2 + j];
        const float x0 = v[2 * j], x1 = v[2 * j + 1];
        if (!isv) { v[2 * j] = x0 * c - x1 * sn; v[2 * j + 1] = x1 * c + x0 * sn; }
      }
    } else {
      const uint32_t j0 = d0 % (HD / 2);
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const float o = __shfl_xor(v[j], LPV / 2);
        const float c = a.cos_t[tb + j0 + j], sn = a.sin_t[tb + j0 + j];
        if (!isv) v[j] = d0 < HD / 2 ? v[j] * c - o * sn : v[j] * c + o * sn;
      }
    }
  }
  uint4 w;
  w.x = P::pk(v[0], v[1]); w.y = P::pk(v[2], v[3]); w.z = P::pk(v[4], v[5]); w.w = P::pk(v[6], v[7]);
  if (live && isq) {
    *(uint4 *)((uint16_t *)a.q + ((uint64_t)row * a.H + hv) * HD + d0) = placed ? w : make_uint4(0, 0, 0, 0);
  }
  const int32_t id = pg_page(&a, s, pos);
  const uint32_t kvh = isv ? hv - a.H - a.Hkv : hv - a.H, slot = (uint32_t)pos & (a.page - 1);
  char *const blk = (char *)(isv ? a.vpages : a.kpages) + (id >= 0 && live && !isq ? pg_block(&a, id, kvh) : 0);
  if (BITS == 16) {
    if (live && !isq && id >= 0) *(uint4 *)(blk + (slot * HD + d0) * 2) = w;
  } else {
    uint32_t am = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) am = max(am, __float_as_uint(v[i]) & 0x7fffffffu);
    am = max(am, dpp_u<0xB1>(am));                      // the 4 lanes of the 32 values
    am = max(am, dpp_u<0x4E>(am));
    const uint32_t sb = fp4_scale_byte<XT>(am);
    const uint32_t codes = sb == 255u ? 0u : fp4x8(v, e8m0_f(sb));
    if (live && !isq && id >= 0) {
      *(uint32_t *)(blk + slot * (HD / 2) + d0 / 2) = codes;
      if ((lane & 3) == 0) blk[a.page * (HD / 2) + slot * (HD / 32) + d0 / 32] = (char)sb;
    }
  }
}

template <int HD, int XT, int BITS>
__global__ __launch_bounds__(PC_THREADS) void k_kv_read(ThvmPagedArgs a) {
  constexpr int LPV = HD / 8, VPW = 64 / LPV;
  const uint32_t heads = 2 * a.Hkv, grps = (heads + VPW - 1) / VPW;
  const uint32_t wid = __builtin_amdgcn_readfirstlane(blockIdx.x * (PC_THREADS / 64) + (threadIdx.x >> 6));
  const uint32_t row = wid / grps, lane = lane_id();
  if (row >= a.n) return;
  const uint32_t s = pg_seq_of(a, row);
  if (s >= a.b) return;
  const PgSeq sq = pg_seq(&a, s);
  if ((int32_t)row < sq.r0 || (int32_t)row >= sq.r1) return;
  const int32_t pos = sq.len - (sq.r1 - (int32_t)row), id = pg_page(&a, s, pos);
  const uint32_t hv = (wid % grps) * VPW + lane / LPV, d0 = lane % LPV * 8;
  if (hv >= heads) return;
  const uint32_t kvh = hv < a.Hkv ? hv : hv - a.Hkv, slot = (uint32_t)pos & (a.page - 1);
  uint4 w = make_uint4(0, 0, 0, 0);
  if (id >= 0) {
    const char *blk = (const char *)(hv < a.Hkv ? a.kpages : a.vpages) + pg_block(&a, id, kvh);
    if (BITS == 16) {
      w = ld_stream16(blk + (slot * HD + d0) * 2);
    } else {
      const uint32_t c = *(const uint32_t *)(blk + slot * (HD / 2) + d0 / 2);
      const float sc = e8m0_f((uint8_t)blk[a.page * (HD / 2) + slot * (HD / 32) + d0 / 32]);
      w = make_uint4(fp4x2<XT, 0>(c, sc), fp4x2<XT, 1>(c, sc), fp4x2<XT, 2>(c, sc), fp4x2<XT, 3>(c, sc));
    }
  }
  *(uint4 *)((uint16_t *)(hv < a.Hkv ? a.k : a.v) + ((uint64_t)row * a.Hkv + kvh) * HD + d0) = w;
}

typedef void (*pc_fn)(ThvmPagedArgs);
#define PC_PICK(K) (a->hd == 128 ? (bf ? (a->bits == 16 ? K<128, GX_BF16, 16> : K<128, GX_BF16, 4>)          \
                                       : (a->bits == 16 ? K<128, GX_F16, 16> : K<128, GX_F16, 4>))          \
                                 : (bf ? (a->bits == 16 ? K<64, GX_BF16, 16> : K<64, GX_BF16, 4>)            \
                                       : (a->bits == 16 ? K<64, GX_F16, 16> : K<64, GX_F16, 4>)))

static int pc_launch(pc_fn f, const ThvmPagedArgs *a, uint32_t heads, const char *who, hipStream_t s, char *err,
                     int errlen) {
  const uint32_t vpw = 64 / (a->hd / 8);
  const uint64_t waves = (uint64_t)a->n * ((heads + vpw - 1) / vpw);
  thvm_launch(true, true, f, dim3((uint32_t)((waves + 3) / 4)), dim3(PC_THREADS), 0, s, *a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) { snprintf(err, errlen, "%s launch: %s", who, hipGetErrorString(e)); return -1; }
  return 0;
}

extern "C" int thvm_k_kv_append(const ThvmPagedArgs *a, hipStream_t s, char *err, int errlen) {
  if (pg_check(a, PG_APPEND, err, errlen)) return -1;
  const int bf = a->dt == THVM_DT_BF16;
  return pc_launch(PC_PICK(k_kv_append), a, a->H + 2 * a->Hkv, "kv_append", s, err, errlen);
}

extern "C" int thvm_k_kv_read(const ThvmPagedArgs *a, hipStream_t s, char *err, int errlen) {
  if (pg_check(a, PG_READ, err, errlen)) return -1;
  const int bf = a->dt == THVM_DT_BF16;
  return pc_launch(PC_PICK(k_kv_read), a, 2 * a->Hkv, "kv_read", s, err, errlen);
}
