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
//   * a lane owns 8 consecutive values (one 16-byte load), 16 or 8 lanes a head;
//     a wave takes 1 or 4 groups of 4 or 8 heads of ONE row, so its sequence, position,
//     page and rotation are found once, with all its x already on its way;
//   * the partner of a half rotation and the 32 values of a 4-bit group lie in
//     the head's own lanes: no LDS.
// Bound by its bytes: each value read once, written once (2 or 17/32 bytes).  Six
// ragged prompts of up to 3000 rows (32 + 8 + 8 heads of 128, 300 MB) take 58 us, 5.1
// TB/s; with norms and into 4 bits, 6247 rows in 34 us (133 MB), a third of which is
// arithmetic.  Few rows: a launch and three dependent loads, 3 us.
// k_kv_read is the way back: the same rows' k and v as 16-bit values (6247 rows in 8 us).
#include "paged_core.h"

#define PC_THREADS 256
#define PC_FILL 2048                                    // waves of four groups that fill the card

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

// What a wave works on: U groups of heads of one row, the row's sequence and
// position.
struct PcRow { uint32_t row, g0; int32_t pos, id; bool ok; };
__device__ __forceinline__ uint32_t pc_wave() {
  return __builtin_amdgcn_readfirstlane(blockIdx.x * (PC_THREADS / 64) + (threadIdx.x >> 6));
}
__device__ __forceinline__ PcRow pc_place(const ThvmPagedArgs &a, uint32_t row, uint32_t g0) {
  PcRow r = {row, g0, 0, -1, false};
  const uint32_t s = pg_seq_of(a, row);
  if (s >= a.b) return r;
  const PgSeq sq = pg_seq(&a, s);
  if ((int32_t)row < sq.r0 || (int32_t)row >= sq.r1) return r;
  r.ok = true;
  r.pos = sq.len - (sq.r1 - (int32_t)row);
  r.id = pg_page(&a, s, r.pos);
  return r;
}

template <int HD, int XT, int BITS, int U>
__global__ __launch_bounds__(PC_THREADS) void k_kv_append(ThvmPagedArgs a) {
#pragma clang fp contract(off)
  typedef PgT<XT> P;
  constexpr int LPV = HD / 8, VPW = 64 / LPV;          // lanes a head, heads a group
  const uint32_t heads = a.H + 2 * a.Hkv, grps = (heads + VPW - 1) / VPW, wpr = (grps + U - 1) / U;
  const uint32_t wid = pc_wave(), row = wid / wpr, g0 = wid % wpr * U, lane = lane_id();
  if (row >= a.n) return;
  // x on its way while the row is placed
  const uint32_t d0 = lane % LPV * 8, h0 = g0 * VPW + lane / LPV;
  uint4 x[U];
#pragma unroll
  for (int u = 0; u < U; u++) {
    const uint32_t hv = h0 + u * VPW;
    x[u] = hv < heads ? ld_stream16((const uint16_t *)a.x + (uint64_t)row * a.ldx + hv * HD + d0) : make_uint4(0, 0, 0, 0);
  }
  const PcRow r = pc_place(a, row, g0);
  if (!r.ok) return;
  const bool placed = r.pos >= 0 && (uint32_t)r.pos < a.maxpages * a.page;
  // the rotation's tables: the same for every head of the row
  float c[8], sn[8];
  if (a.rope && placed) {
    const uint64_t tb = (uint64_t)r.pos * (HD / 2);
    const uint32_t j0 = a.rope == 1 ? d0 / 2 : d0 % (HD / 2);
#pragma unroll
    for (int k = 0; k < 8; k += 4) {
      if (k && a.rope == 1) break;
      const float4 cc = *(const float4 *)(a.cos_t + tb + j0 + k), ss = *(const float4 *)(a.sin_t + tb + j0 + k);
      c[k] = cc.x; c[k + 1] = cc.y; c[k + 2] = cc.z; c[k + 3] = cc.w;
      sn[k] = ss.x; sn[k + 1] = ss.y; sn[k + 2] = ss.z; sn[k + 3] = ss.w;
    }
    if (a.rope == 2 && d0 < HD / 2) {                  // x c - o s there, x c + o s in the upper half
#pragma unroll
      for (int k = 0; k < 8; k++) sn[k] = -sn[k];
    }
  }
  // (wave-uniform: a group of v heads alone is copied)
  bool turned[U];
#pragma unroll
  for (int u = 0; u < U; u++) turned[u] = (g0 + u) * VPW < a.H + a.Hkv;
  float inv[U];
  if (a.norm) {
    // each lane has its head's sums of all groups: it takes one of them through the
    // root (v_rsq_f64 and two steps of Newton's iteration), and a quad shares out four
    double one = 0.0;
#pragma unroll
    for (int u = 0; u < U; u++) {
      if (!turned[u]) break;
      const uint32_t w[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
      double ss = 0.0;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const double lo = P::lo(w[i]), hi = P::hi(w[i]);
        ss = __builtin_fma(lo, lo, ss);
        ss = __builtin_fma(hi, hi, ss);
      }
      ss += dpp_d<0xB1>(ss);
      ss += dpp_d<0x4E>(ss);
      ss += dpp_d<0x141>(ss);
      if (LPV == 16) ss += dpp_d<0x140>(ss);
      if (U == 1 || (lane & 3) == u) one = ss;
    }
    one = one * (1.0 / HD) + (double)a.eps;
    double y = __builtin_amdgcn_rsq(one);
    y = __builtin_fma(y, __builtin_fma(-0.5 * one * y, y, 0.5), y);
    y = __builtin_fma(y, __builtin_fma(-0.5 * one * y, y, 0.5), y);
    const float f = one == 0.0 ? INFINITY : one == __builtin_inf() ? 0.0f : (float)y;
    if (U == 1) {
      inv[0] = f;
    } else {
      inv[0] = dpp_f<0x00>(f);
      inv[1 % U] = dpp_f<0x55>(f);
      inv[2 % U] = dpp_f<0xAA>(f);
      inv[3 % U] = dpp_f<0xFF>(f);
    }
  }
  const uint32_t slot = (uint32_t)r.pos & (a.page - 1);
#pragma unroll
  for (int u = 0; u < U; u++) {
    const uint32_t hv = h0 + u * VPW;
    const bool live = hv < heads, isq = hv < a.H, isv = hv >= a.H + a.Hkv;
    const uint32_t xw[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; i++) { v[2 * i] = P::lo(xw[i]); v[2 * i + 1] = P::hi(xw[i]); }
    if (a.norm && turned[u] && !isv) {
      const float *g = (isq ? a.gq : a.gk) + d0;
      const float4 ga = *(const float4 *)g, gb = *(const float4 *)(g + 4);
      const float gg[8] = {ga.x, ga.y, ga.z, ga.w, gb.x, gb.y, gb.z, gb.w};
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] = (v[i] * inv[u]) * gg[i];
    }
    if (a.rope && placed && turned[u]) {
      if (a.rope == 1) {
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const float x0 = v[2 * k], x1 = v[2 * k + 1], y0 = x0 * c[k] - x1 * sn[k], y1 = x1 * c[k] + x0 * sn[k];
          v[2 * k] = isv ? x0 : y0;
          v[2 * k + 1] = isv ? x1 : y1;
        }
      } else {
#pragma unroll
        for (int k = 0; k < 8; k++) {                  // the partner is half a head away
          const float o = LPV == 16 ? dpp_f<0x128>(v[k]) : __shfl_xor(v[k], 4);
          const float y = v[k] * c[k] + o * sn[k];
          v[k] = isv ? v[k] : y;
        }
      }
    }
    uint4 w;
    w.x = P::pk(v[0], v[1]); w.y = P::pk(v[2], v[3]); w.z = P::pk(v[4], v[5]); w.w = P::pk(v[6], v[7]);
    if (live && isq) *(uint4 *)((uint16_t *)a.q + ((uint64_t)row * a.H + hv) * HD + d0) = placed ? w : make_uint4(0, 0, 0, 0);
    const bool put = live && !isq && r.id >= 0;
    const uint32_t kvh = isv ? hv - a.H - a.Hkv : hv - a.H;
    char *const blk = (char *)(isv ? a.vpages : a.kpages) + (put ? pg_block(&a, r.id, kvh) : 0);
    if (BITS == 16) {
      if (put) *(uint4 *)(blk + (slot * HD + d0) * 2) = w;
    } else if (__builtin_amdgcn_ballot_w64(put)) {     // (wave-uniform: groups of q heads have no codes)
      uint32_t am = 0;
#pragma unroll
      for (int i = 0; i < 8; i++) am = max(am, __float_as_uint(v[i]) & 0x7fffffffu);
      am = max(am, dpp_u<0xB1>(am));                   // the 4 lanes of the 32 values
      am = max(am, dpp_u<0x4E>(am));
      const uint32_t sb = fp4_scale_byte<XT>(am), codes = sb == 255u ? 0u : fp4x8(v, e8m0_f(sb));
      // a head's scale bytes together: lane 0 of its lanes has them all
      uint32_t sbs = sb | dpp_u<0x104>(sb) << 8;       // row_shl:4
      if (LPV == 16) sbs |= dpp_u<0x108>(sbs) << 16;   // row_shl:8
      if (put) {
        *(uint32_t *)(blk + slot * (HD / 2) + d0 / 2) = codes;
        char *const sp = blk + a.page * (HD / 2) + slot * (HD / 32);
        if (lane % LPV == 0) {
          if (HD == 128) *(uint32_t *)sp = sbs;
          else *(uint16_t *)sp = (uint16_t)sbs;
        }
      }
    }
  }
}

template <int HD, int XT, int BITS, int U>
__global__ __launch_bounds__(PC_THREADS) void k_kv_read(ThvmPagedArgs a) {
  constexpr int LPV = HD / 8, VPW = 64 / LPV;
  const uint32_t heads = 2 * a.Hkv, grps = (heads + VPW - 1) / VPW, wpr = (grps + U - 1) / U;
  const uint32_t wid = pc_wave(), row = wid / wpr, lane = lane_id();
  if (row >= a.n) return;
  const PcRow r = pc_place(a, row, wid % wpr * U);
  if (!r.ok) return;
  const uint32_t d0 = lane % LPV * 8, h0 = r.g0 * VPW + lane / LPV, slot = (uint32_t)r.pos & (a.page - 1);
  uint4 w[U];
  uint32_t sc[U];
#pragma unroll
  for (int u = 0; u < U; u++) {
    const uint32_t hv = h0 + u * VPW, kvh = hv < a.Hkv ? hv : hv - a.Hkv;
    w[u] = make_uint4(0, 0, 0, 0);
    sc[u] = 0;
    if (hv < heads && r.id >= 0) {
      const char *blk = (const char *)(hv < a.Hkv ? a.kpages : a.vpages) + pg_block(&a, r.id, kvh);
      if (BITS == 16) {
        w[u] = ld_stream16(blk + (slot * HD + d0) * 2);
      } else {
        w[u].x = *(const uint32_t *)(blk + slot * (HD / 2) + d0 / 2);
        sc[u] = (uint8_t)blk[a.page * (HD / 2) + slot * (HD / 32) + d0 / 32];
      }
    }
  }
#pragma unroll
  for (int u = 0; u < U; u++) {
    const uint32_t hv = h0 + u * VPW, kvh = hv < a.Hkv ? hv : hv - a.Hkv;
    if (hv >= heads) continue;
    if (BITS == 4) {
      const uint32_t cd = w[u].x;
      const float f = e8m0_f(sc[u]);
      w[u] = make_uint4(fp4x2<XT, 0>(cd, f), fp4x2<XT, 1>(cd, f), fp4x2<XT, 2>(cd, f), fp4x2<XT, 3>(cd, f));
    }
    *(uint4 *)((uint16_t *)(hv < a.Hkv ? a.k : a.v) + ((uint64_t)row * a.Hkv + kvh) * HD + d0) = w[u];
  }
}

typedef void (*pc_fn)(ThvmPagedArgs);
#define PC_PICK_U(K, U) (a->hd == 128 ? (bf ? (a->bits == 16 ? K<128, GX_BF16, 16, U> : K<128, GX_BF16, 4, U>)   \
                                            : (a->bits == 16 ? K<128, GX_F16, 16, U> : K<128, GX_F16, 4, U>))   \
                                      : (bf ? (a->bits == 16 ? K<64, GX_BF16, 16, U> : K<64, GX_BF16, 4, U>)     \
                                            : (a->bits == 16 ? K<64, GX_F16, 16, U> : K<64, GX_F16, 4, U>)))
#define PC_PICK(K) (u == 4 ? PC_PICK_U(K, 4) : PC_PICK_U(K, 1))

// Groups a wave: four, which find the row's place once, where that leaves the card
// full of waves; else one, whose way is shorter.  kv_append's 12 groups a row of 48
// heads of 128, one | four of them a wave, us: 1 row 2.8 | 4.0, 96 rows 3.7 | 5.0,
// 384 rows 5.2 | 6.1, 768 rows (9216 groups) 8.0 | 8.0, 1536 rows 12.9 | 11.6.
static uint32_t pc_groups(const ThvmPagedArgs *a, uint32_t heads) {
  const uint32_t vpw = 64 / (a->hd / 8);
  return (uint64_t)a->n * ((heads + vpw - 1) / vpw) >= 4 * PC_FILL ? 4 : 1;
}

static int pc_launch(pc_fn f, uint32_t u, const ThvmPagedArgs *a, uint32_t heads, const char *who, hipStream_t s, char *err,
                     int errlen) {
  const uint32_t vpw = 64 / (a->hd / 8);
  const uint64_t waves = (uint64_t)a->n * (((heads + vpw - 1) / vpw + u - 1) / u);
  thvm_launch(true, true, f, dim3((uint32_t)((waves + 3) / 4)), dim3(PC_THREADS), 0, s, *a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) { snprintf(err, errlen, "%s launch: %s", who, hipGetErrorString(e)); return -1; }
  return 0;
}

extern "C" int thvm_k_kv_append(const ThvmPagedArgs *a, hipStream_t s, char *err, int errlen) {
  if (pg_check(a, PG_APPEND, err, errlen)) return -1;
  const int bf = a->dt == THVM_DT_BF16;
  const uint32_t u = pc_groups(a, a->H + 2 * a->Hkv);
  return pc_launch(PC_PICK(k_kv_append), u, a, a->H + 2 * a->Hkv, "kv_append", s, err, errlen);
}

extern "C" int thvm_k_kv_read(const ThvmPagedArgs *a, hipStream_t s, char *err, int errlen) {
  if (pg_check(a, PG_READ, err, errlen)) return -1;
  const int bf = a->dt == THVM_DT_BF16;
  const uint32_t u = pc_groups(a, 2 * a->Hkv);
  return pc_launch(PC_PICK(k_kv_read), u, a, 2 * a->Hkv, "kv_read", s, err, errlen);
}
