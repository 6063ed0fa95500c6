// paged_attn.hip -- attention of a ragged batch over a paged cache.
//
// out = sum_j softmax_j(scale q.k_j) v_j over the cache rows j <= p that have a
// page, for every row (position p of its sequence) and head; no such row: zeros.
// The rows and the query heads of a kv head are the columns of its products.
// Sequences of few columns (single tokens, speculative rows) go to k_paged_split
// here, the others to k_paged_tile (paged_prompt.hip); either splits long contexts
// into chunks whose partial sums k_paged_merge adds.  Softmax statistics and sums
// are f32.
#include "paged_core.h"

#define LOG2E 1.4426950408889634f

// ---- a few columns: the split -------------------------------------------------
// k_paged_split: a unit is one tile of at most 16 columns (rows x query heads of
// one kv head) over one chunk of its cache rows; 4 waves.
//   scores  S[row][column] = K q^T by 16x16x32 MFMAs over 16-row tiles.  Heads of
//           a token fill only CG of the 16 columns, so the columns repeat them 16 /
//           CG times and a lane keeps the scores of one tile in 16 / CG: a step of
//           four tiles then costs softmax work for CG values a lane, not 16.
//   mix     O^T[d][column] += V^T P^T by 16x16x32 MFMAs over pairs of tiles (32
//           rows); the P operand is the score layout itself, zero in the columns
//           that kept another tile.  A lane loads 4 rows of HD / 16 columns of V per
//           tile and pairs them up with v_perm.
//   A wave's four tiles are 64 rows apart (wave w has rows 16 w .. of each 64), so a
//   chunk of 64 rows still feeds all four waves, and every tile lies inside a page.
// Over 4 bits a lane's K bytes are 32 (hd 64: 16) consecutive values, one scale;
// the q operand is ordered to match.  p enters the product as a pair of 16-bit terms
// (hi and what it leaves: 16 bits of p in bf16, 22 in fp16), which costs nothing where
// the cache's bytes are the bound; its sum, like all else, is f32.
// Bound by the cache's bytes.
#define PS_WAVES 4
#define PS_THREADS (PS_WAVES * 64)

// cached bytes in registers on their way to MFMA operands
template <int HD, int BITS> struct PsRegs;
template <> struct PsRegs<128, 16> { uint4 k[4][4]; uint4 v[4][4]; };
template <> struct PsRegs<64, 16> { uint4 k[4][2]; uint2 v[4][4]; };
template <> struct PsRegs<128, 4> { uint4 k[4]; uint32_t ks[4]; uint32_t v[4][4]; uint4 vs[4]; };
template <> struct PsRegs<64, 4> { uint2 k[4]; uint32_t ks[4]; uint32_t v[4][4]; uint2 vs[4]; };

template <int HD, int XT, int BITS, int CG>
__global__ __launch_bounds__(PS_THREADS, 2) void k_paged_split(ThvmPagedArgs a, PgPlan pl) {
  typedef PgT<XT> P;
  constexpr int EC = HD / 16, KS = HD / 32, NG = 16 / CG, NS = 4 / NG, RB = BITS == 16 ? HD * 2 : HD / 2;
  constexpr uint32_t EXP = XT == GX_BF16 ? 0x7f80u : 0x7c00u;
  constexpr float PSH = XT == GX_BF16 ? 0.0f : 14.0f;      // keeps small p off fp16's subnormals; cancels in acc / l
  __shared__ __align__(16) float wacc[PS_WAVES][16][HD + 4];
  __shared__ float wm[PS_WAVES][16], wl[PS_WAVES][16];
  const uint32_t kvh = blockIdx.x % a.Hkv, un = blockIdx.x / a.Hkv, G = a.H / a.Hkv;
  PgUnit u;
  if (!pg_unit(a, pl, un, false, u)) return;
  const int tid = threadIdx.x, wv = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, lc = lane & 15, lg = lane >> 4;
  const int32_t nrow = u.q.r1 - u.q.r0, cap = (int32_t)(a.maxpages * a.page), L = min(u.q.len, cap);
  // the unit's cache rows, and the rows that this lane's column sees
  const int32_t r0 = (int32_t)(u.chunk * u.c * 64), r1 = u.chunk + 1 == u.nchunk ? L : min(L, (int32_t)((u.chunk + 1) * u.c * 64));
  const uint32_t col = u.tile * 16 + (uint32_t)(lc % CG), ri = col / G, hg = col % G;
  const bool live = (int32_t)ri < nrow;
  const int32_t lim = live ? min(u.q.len - nrow + (int32_t)ri + 1, r1) : 0;
  const int32_t first = u.q.len - nrow + 1;                // rows below it are seen by every column
  uint4 qb[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ks++) {
    const uint32_t d = BITS == 16 ? 8 * lg + 32 * ks : (HD / 4) * lg + 8 * ks;
    qb[ks] = live ? ld16((const uint16_t *)a.q + ((uint64_t)(u.q.r0 + ri) * a.H + kvh * G + hg) * HD + d) : make_uint4(0, 0, 0, 0);
  }
  const buf_t tb = buf_rsrc(a.table + (uint64_t)u.s * a.maxpages, a.maxpages * 4);
  const uint32_t lgp = __builtin_ctz(a.page), pm = a.page - 1, bb = pg_block_bytes(&a);
  auto row_of = [&](int it, int t) { return r0 + 256 * it + 64 * t + 16 * wv; };
  // page ids of the four tiles, in lanes 0..3
  auto ids = [&](int it) {
    const int32_t r = row_of(it, lane & 3);
    return (int32_t)buf_ld4(tb, r < r1 ? ((uint32_t)r >> lgp) * 4 : BUF_OOB);
  };
  PsRegs<HD, BITS> R;
  uint64_t off[4];                                         // a tile's block in the pools, and its bytes (0: no page)
  uint32_t rng[4];
  auto place = [&](int32_t id, int it) {
#pragma unroll
    for (int t = 0; t < 4; t++) {
      const uint32_t i = (uint32_t)__builtin_amdgcn_readlane(id, t);
      const bool ok = i < a.npages && row_of(it, t) < r1;
      rng[t] = ok ? bb : 0u;
      off[t] = ok ? pg_block(&a, (int32_t)i, kvh) : 0;
    }
  };
  auto issue_k = [&](int it) {
#pragma unroll
    for (int t = 0; t < 4; t++) {
      const buf_t rs = buf_rsrc((const char *)a.kpages + off[t], rng[t]);
      const int32_t r = row_of(it, t) + lc;
      const uint32_t slot = ((uint32_t)row_of(it, t) & pm) + lc;
      if constexpr (BITS == 16) {
#pragma unroll
        for (int ks = 0; ks < KS; ks++)
          R.k[t][ks] = buf_ld_stream16(rs, r < r1 ? slot * RB + 16 * lg + 64 * ks : BUF_OOB);
      } else {
        if constexpr (HD == 128) R.k[t] = buf_ld_stream16(rs, r < r1 ? slot * RB + 16 * lg : BUF_OOB);
        else R.k[t] = buf_ld8(rs, r < r1 ? slot * RB + 8 * lg : BUF_OOB);
        R.ks[t] = __builtin_amdgcn_raw_buffer_load_b8(rs, r < r1 ? a.page * RB + slot * (HD / 32) + lg * HD / 128 : BUF_OOB, 0, 0);
      }
    }
  };
  auto issue_v = [&](int it) {
#pragma unroll
    for (int t = 0; t < 4; t++) {
      const buf_t rs = buf_rsrc((const char *)a.vpages + off[t], rng[t]);
      const int32_t r = row_of(it, t) + 4 * lg;
      const uint32_t slot = ((uint32_t)row_of(it, t) & pm) + 4 * lg;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        if constexpr (BITS == 16) {
          const uint32_t o = r + j < r1 ? (slot + j) * RB + EC * 2 * lc : BUF_OOB;
          if constexpr (HD == 128) R.v[t][j] = buf_ld_stream16(rs, o);
          else R.v[t][j] = buf_ld8(rs, o);
        } else {
          const uint32_t o = r + j < r1 ? (slot + j) * RB + EC / 2 * lc : BUF_OOB;
          R.v[t][j] = HD == 128 ? buf_ld4(rs, o) : buf_ld2(rs, o);
        }
      }
      if constexpr (BITS == 4) {
        const uint32_t o = r < r1 ? a.page * RB + slot * (HD / 32) : BUF_OOB;
        if constexpr (HD == 128) R.vs[t] = buf_ld16(rs, o);
        else R.vs[t] = buf_ld8(rs, o);
      }
    }
  };
  const float qs = a.scale * LOG2E;
  float m = -INFINITY, l = 0.0f;
  f32x4_t acc[EC];
#pragma unroll
  for (int e = 0; e < EC; e++) acc[e] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const int nt = r1 > r0 ? (r1 - r0 + 255) / 256 : 0;
  int32_t idn = -1;
  if (nt) {
    const int32_t id = ids(0);
    idn = ids(1);
    place(id, 0);
    issue_k(0);
    issue_v(0);
  }
  for (int it = 0; it < nt; it++) {
    f32x4_t sc[4];
#pragma unroll
    for (int t = 0; t < 4; t++) {
      sc[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ks++) {
        if constexpr (BITS == 16) {
          sc[t] = mfma16<XT>(R.k[t][ks], qb[ks], sc[t]);
        } else {
          const float f = e8m0_f(R.ks[t]);
          uint32_t w;
          if constexpr (HD == 128) w = ks == 0 ? R.k[t].x : ks == 1 ? R.k[t].y : ks == 2 ? R.k[t].z : R.k[t].w;
          else w = ks == 0 ? R.k[t].x : R.k[t].y;
          sc[t] = mfma16<XT>(make_uint4(fp4x2<XT, 0>(w, f), fp4x2<XT, 1>(w, f), fp4x2<XT, 2>(w, f), fp4x2<XT, 3>(w, f)),
                             qb[ks], sc[t]);
        }
      }
    }
    bool has[4];                                           // tiles with a page
#pragma unroll
    for (int t = 0; t < 4; t++) has[t] = rng[t] != 0;
    uint64_t voff[4];
#pragma unroll
    for (int t = 0; t < 4; t++) voff[t] = off[t];
    // this lane's scores: tile s NG + lc / CG of set s
    float p[NS][4];
    float mx = -INFINITY;
#pragma unroll
    for (int s = 0; s < NS; s++) {
      f32x4_t v = sc[s * NG];
      bool ok = has[s * NG];
#pragma unroll
      for (int j = 1; j < NG; j++) {
        if (lc / CG == j) { v = sc[s * NG + j]; ok = has[s * NG + j]; }
      }
      const int32_t rb = row_of(it, s * NG + lc / CG) + 4 * lg;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        p[s][i] = ok && rb + i < lim ? v[i] * qs : -INFINITY;
        mx = fmaxf(mx, p[s][i]);
      }
    }
    mx = fmaxf(mx, xor16_f(mx));
    mx = fmaxf(mx, xor32_f(mx));
    const float mn = fmaxf(m, mx), f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
    float ls = 0.0f;
    uint32_t pk[NS][2], pl2[NS][2];
#pragma unroll
    for (int s = 0; s < NS; s++) {
#pragma unroll
      for (int i = 0; i < 4; i++) p[s][i] = p[s][i] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(p[s][i] - (mn - PSH));
      ls += (p[s][0] + p[s][1]) + (p[s][2] + p[s][3]);
#pragma unroll
      for (int i = 0; i < 2; i++) {                        // hi + lo, the differences exact
        pk[s][i] = P::pk(p[s][2 * i], p[s][2 * i + 1]);
        pl2[s][i] = P::pk(p[s][2 * i] - P::lo(pk[s][i]), p[s][2 * i + 1] - P::hi(pk[s][i]));
      }
    }
    l = l * f + ls;
    m = mn;
    if (__builtin_amdgcn_ballot_w64(f != 1.0f)) {
#pragma unroll
      for (int e = 0; e < EC; e++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[e][i] *= f;
    }
    // the next step's K while this one's V is used
    const bool more = it + 1 < nt;
    place(more ? idn : -1, it + 1);
    idn = ids(it + 2);
    issue_k(it + 1);
    // V: 16-bit values of rows 4 lg + j, columns EC lc ..
    uint32_t w[4][4][EC / 2];
    bool odd = false;                                      // a value that is not finite
#pragma unroll
    for (int t = 0; t < 4; t++) {
      const int32_t rt = row_of(it, t);
#pragma unroll
      for (int j = 0; j < 4; j++) {
        if constexpr (BITS == 16) {
          const uint32_t *x = (const uint32_t *)&R.v[t][j];
#pragma unroll
          for (int e = 0; e < EC / 2; e++) w[t][j][e] = x[e];
        } else {
          uint32_t sb;
          if constexpr (HD == 128) sb = ((const uint32_t *)&R.vs[t])[j] >> (8 * (lc / 4)) & 0xffu;
          else sb = ((const uint32_t *)&R.vs[t])[j / 2] >> (16 * (j & 1) + 8 * (lc / 8)) & 0xffu;
          if (rt + 16 > first) {                           // wave-uniform: rows that some column does not see, or none
            if (rt + 4 * lg + j >= r1) sb = 0;
            if (sb == 255u) { odd = true; sb = 0; R.v[t][j] = 0; }
          }
          const float f = e8m0_f(sb);
          w[t][j][0] = fp4x2<XT, 0>(R.v[t][j], f);
          w[t][j][1] = fp4x2<XT, 1>(R.v[t][j], f);
          if constexpr (HD == 128) {
            w[t][j][2] = fp4x2<XT, 2>(R.v[t][j], f);
            w[t][j][3] = fp4x2<XT, 3>(R.v[t][j], f);
          }
        }
      }
    }
    if constexpr (BITS == 16) {
      typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
      u16x2 big = {0, 0};
#pragma unroll
      for (int t = 0; t < 4; t++)
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
          for (int e = 0; e < EC / 2; e++)
            big = __builtin_elementwise_max(big, __builtin_bit_cast(u16x2, w[t][j][e] & (EXP | EXP << 16)));
      odd = big[0] == EXP || big[1] == EXP;
    }
    // A zero p times a V that is not finite is NaN: such values (a stored overflow;
    // a 4-bit group that held one) leave the products, and the columns that see
    // their rows add them one by one.
    const bool fix = __builtin_amdgcn_ballot_w64(odd) != 0;
    if (fix && BITS == 16) {
#pragma unroll
      for (int t = 0; t < 4; t++)
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
          for (int e = 0; e < EC / 2; e++) {
            if ((w[t][j][e] & EXP) == EXP) w[t][j][e] &= 0xffff0000u;
            if ((w[t][j][e] >> 16 & EXP) == EXP) w[t][j][e] &= 0xffffu;
          }
    }
#pragma unroll
    for (int h = 0; h < 2; h++) {                          // tiles 2h and 2h + 1
      const int s0 = (2 * h) / NG, g0 = (2 * h) % NG, s1 = (2 * h + 1) / NG, g1 = (2 * h + 1) % NG;
      const bool in0 = NG == 1 || lc / CG == g0, in1 = NG == 1 || lc / CG == g1;
      const uint4 B = make_uint4(in0 ? pk[s0][0] : 0u, in0 ? pk[s0][1] : 0u, in1 ? pk[s1][0] : 0u, in1 ? pk[s1][1] : 0u);
      const uint4 B2 = make_uint4(in0 ? pl2[s0][0] : 0u, in0 ? pl2[s0][1] : 0u, in1 ? pl2[s1][0] : 0u, in1 ? pl2[s1][1] : 0u);
#pragma unroll
      for (int e = 0; e < EC; e++) {
        const uint32_t sel = (e & 1) ? 0x07060302u : 0x05040100u;
        uint4 A;
        A.x = __builtin_amdgcn_perm(w[2 * h][1][e >> 1], w[2 * h][0][e >> 1], sel);
        A.y = __builtin_amdgcn_perm(w[2 * h][3][e >> 1], w[2 * h][2][e >> 1], sel);
        A.z = __builtin_amdgcn_perm(w[2 * h + 1][1][e >> 1], w[2 * h + 1][0][e >> 1], sel);
        A.w = __builtin_amdgcn_perm(w[2 * h + 1][3][e >> 1], w[2 * h + 1][2][e >> 1], sel);
        acc[e] = mfma16<XT>(A, B, acc[e]);
        acc[e] = mfma16<XT>(A, B2, acc[e]);
      }
    }
    if (fix) {                                             // wave-uniform
#pragma unroll
      for (int s = 0; s < NS; s++) {
        uint64_t vo = voff[s * NG];
        bool ok = has[s * NG];
#pragma unroll
        for (int j = 1; j < NG; j++)
          if (lc / CG == j) { vo = voff[s * NG + j]; ok = has[s * NG + j]; }
        const int32_t rt = row_of(it, s * NG + lc / CG);
        const char *vb = (const char *)a.vpages + vo;
#pragma unroll 1
        for (int jj = 0; jj < 4; jj++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const float pr = __shfl(p[s][i], lc + 16 * jj);
            const int32_t r = rt + 4 * jj + i;
            if (!ok || r >= lim) continue;
            const uint32_t slot = (uint32_t)r & pm;
#pragma unroll
            for (int q = 0; q < 4; q++)                    // this lane's d = EC (4 lg + q) + e
#pragma unroll
              for (int e = 0; e < EC; e++) {
                const uint32_t d = EC * (4 * lg + q) + e;
                float x;
                if constexpr (BITS == 16) {
                  const uint32_t h = ((const uint16_t *)vb)[slot * HD + d];
                  if ((h & EXP) != EXP) continue;
                  x = P::lo(h);
                } else {
                  if ((uint8_t)vb[a.page * RB + slot * (HD / 32) + d / 32] != 255u) continue;
                  x = __builtin_nanf("");
                }
                acc[e][q] += pr * x;
              }
          }
      }
    }
    issue_v(it + 1);
  }
  // the waves (and the column groups) meet in LDS
  l += xor16_f(l);
  l += xor32_f(l);
  if (lg == 0) { wm[wv][lc] = m; wl[wv][lc] = l; }
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int e = 0; e < EC; e += 4)
      *(float4 *)&wacc[wv][lc][EC * (4 * lg + i) + e] = make_float4(acc[e][i], acc[e + 1][i], acc[e + 2][i], acc[e + 3][i]);
  __syncthreads();
  for (int o = tid; o < CG * HD / 2; o += PS_THREADS) {
    const int c = o / (HD / 2), d = 2 * (o % (HD / 2));
    const uint32_t cc = u.tile * 16 + c;
    if ((int32_t)(cc / G) >= nrow) continue;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < PS_WAVES * NG; w++) M = fmaxf(M, wm[w / NG][w % NG * CG + c]);
    float s0 = 0.0f, s1 = 0.0f, lt = 0.0f;
#pragma unroll
    for (int w = 0; w < PS_WAVES * NG; w++) {
      const float mw = wm[w / NG][w % NG * CG + c], f = mw == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mw - M);
      const float2 v = *(const float2 *)&wacc[w / NG][w % NG * CG + c][d];
      s0 += v.x * f;
      s1 += v.y * f;
      lt += wl[w / NG][w % NG * CG + c] * f;
    }
    if (u.nchunk == 1) {
      const float inv = lt != 0.0f ? 1.0f / lt : 0.0f;
      *(uint32_t *)((uint16_t *)a.out + ((uint64_t)(u.q.r0 + cc / G) * a.H + kvh * G + cc % G) * HD + d) = P::pk(s0 * inv, s1 * inv);
    } else {
      float *pp = a.ws + (((uint64_t)kvh * pl.units + un) * CG + c) * (HD + 4);
      *(float2 *)(pp + d) = make_float2(s0, s1);
      if (d == 0) *(float2 *)(pp + HD) = make_float2(M, lt);
    }
  }
}

// k_paged_merge: the chunks of a column, their partials (sum, m, l) in a fixed
// order.  HD / 4 lanes take a chunk; NP such groups take every NP-th chunk of one
// column and meet in LDS, the block's other groups have other columns.
template <int HD, int XT, int CT, int NP>
__global__ __launch_bounds__(256) void k_paged_merge(ThvmPagedArgs a, PgPlan pl) {
  typedef PgT<XT> P;
  constexpr int LN = HD / 4, NG = 256 / LN, CB = NG / NP;  // lanes a chunk, groups, columns a block
  __shared__ float4 ls[NG][LN];
  __shared__ float lm[NG], ll[NG];
  const uint32_t g = threadIdx.x / LN, x = threadIdx.x % LN, part = g % NP;
  const uint32_t c = blockIdx.x % (CT / CB) * CB + g / NP, kvh = blockIdx.x / (CT / CB) % a.Hkv, G = a.H / a.Hkv;
  PgUnit u;
  if (!pg_unit(a, pl, blockIdx.x / (CT / CB) / a.Hkv, true, u) || u.nchunk == 1) return;
  const uint32_t cc = u.tile * pl.ct + c;
  const bool live = (int32_t)(cc / G) < u.q.r1 - u.q.r0;
  const float *pp = a.ws + (((uint64_t)kvh * pl.units + u.first) * CT + c) * (HD + 4);
  const uint64_t st = (uint64_t)CT * (HD + 4);
  float m = -INFINITY, l = 0.0f;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  for (uint32_t k = part; live && k < u.nchunk; k += NP) {
    const float4 w = *(const float4 *)(pp + k * st + 4 * x);
    const float2 ml = *(const float2 *)(pp + k * st + HD);
    const float mn = fmaxf(m, ml.x), f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn),
                e = ml.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml.x - mn);
    v.x = v.x * f + w.x * e;
    v.y = v.y * f + w.y * e;
    v.z = v.z * f + w.z * e;
    v.w = v.w * f + w.w * e;
    l = l * f + ml.y * e;
    m = mn;
  }
  if (NP > 1) {
    ls[g][x] = v;
    if (x == 0) { lm[g] = m; ll[g] = l; }
    __syncthreads();
    if (part) return;
    float M = -INFINITY;
#pragma unroll
    for (int k = 0; k < NP; k++) M = fmaxf(M, lm[g + k]);
    l = 0.0f;
    v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < NP; k++) {
      const float f = lm[g + k] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(lm[g + k] - M);
      v.x += ls[g + k][x].x * f;
      v.y += ls[g + k][x].y * f;
      v.z += ls[g + k][x].z * f;
      v.w += ls[g + k][x].w * f;
      l += ll[g + k] * f;
    }
  }
  if (!live) return;
  const float inv = l != 0.0f ? 1.0f / l : 0.0f;
  *(uint2 *)((uint16_t *)a.out + ((uint64_t)(u.q.r0 + cc / G) * a.H + kvh * G + cc % G) * HD + 4 * x) =
      make_uint2(P::pk(v.x * inv, v.y * inv), P::pk(v.z * inv, v.w * inv));
}

// ---- which kernels a call takes ------------------------------------------------
// few: sequences of up to few.hi columns, cg of the MFMA's 16 columns used; many:
// the others, chunks of them (split) where their tiles do not fill the chip.
struct PaRule { bool few, many, split; uint32_t cg, few_tiles, many_tiles; PgPlan fpl, mpl; };
static PaRule pa_rule(const ThvmPagedArgs *a) {
  PaRule r;
  const uint32_t G = a->H / a->Hkv, t = a->t < a->n ? a->t : a->n, fill = (512 + a->Hkv - 1) / a->Hkv;
  const uint64_t most = (uint64_t)t * G;                   // columns of the longest sequence
  const uint32_t cols = most <= 16 ? (uint32_t)most : G;
  r.cg = cols <= 4 ? 4 : cols <= 8 ? 8 : 16;
  const uint32_t hi = most <= 16 || r.cg > G ? r.cg : G;
  r.many = most > hi;
  r.few = !r.many || a->ragged;
  r.few_tiles = a->b * ((hi + 15) / 16);
  r.fpl = PgPlan{0, hi, 16, fill > 2 * r.few_tiles ? fill : 2 * r.few_tiles, 1, 0};
  const uint32_t whole = (uint32_t)((uint64_t)a->n * G / PP_COLS);
  r.many_tiles = whole + a->b;
  r.split = (uint64_t)whole * a->Hkv < 512;
  r.mpl = PgPlan{r.few ? hi : 0, 0xffffffffu, PP_COLS, r.many_tiles + 1, 1u << 25, 1};
  if (r.split) {
    r.mpl.units = fill > 2 * r.many_tiles ? fill : 2 * r.many_tiles;
    r.mpl.cmin = 4;
  }
  return r;
}

extern "C" uint64_t thvm_k_attn_paged_ws(const ThvmPagedArgs *a) {
  const PaRule r = pa_rule(a);
  const uint64_t rec = (uint64_t)a->Hkv * (a->hd + 4) * 4, f = r.few ? rec * r.fpl.units * r.cg : 0,
                 m = r.many && r.split ? rec * r.mpl.units * PP_COLS : 0;
  return f > m ? f : m > 16 ? m : 16;
}

template <int HD, int XT, int BITS>
static paged_fn pa_split(uint32_t cg) {
  return cg == 4 ? k_paged_split<HD, XT, BITS, 4> : cg == 8 ? k_paged_split<HD, XT, BITS, 8> : k_paged_split<HD, XT, BITS, 16>;
}
struct PaKernels { paged_fn split, merge, tmerge; };
template <int HD, int XT>
static PaKernels pa_pick(const ThvmPagedArgs *a, uint32_t cg) {
  constexpr int NG = 1024 / HD;                            // one column a block
  return PaKernels{a->bits == 16 ? pa_split<HD, XT, 16>(cg) : pa_split<HD, XT, 4>(cg),
                   cg == 4 ? k_paged_merge<HD, XT, 4, NG> : cg == 8 ? k_paged_merge<HD, XT, 8, NG> : k_paged_merge<HD, XT, 16, NG>,
                   k_paged_merge<HD, XT, PP_COLS, 2>};
}

extern "C" int thvm_k_attn_paged(const ThvmPagedArgs *a, hipStream_t s, char *err, int errlen) {
  if (pg_check(a, PG_ATTN, err, errlen)) return -1;
  const PaRule r = pa_rule(a);
  const int bf = a->dt == THVM_DT_BF16;
  const PaKernels k = a->hd == 128 ? (bf ? pa_pick<128, GX_BF16>(a, r.cg) : pa_pick<128, GX_F16>(a, r.cg))
                                   : (bf ? pa_pick<64, GX_BF16>(a, r.cg) : pa_pick<64, GX_F16>(a, r.cg));
  if (r.few) {
    thvm_launch(true, false, k.split, dim3(a->Hkv * r.fpl.units), dim3(PS_THREADS), 0, s, *a, r.fpl);
    thvm_launch(false, !r.many, k.merge, dim3(a->Hkv * r.cg * r.few_tiles), dim3(256), 0, s, *a, r.fpl);
  }
  if (r.many) {
    thvm_launch(!r.few, !r.split, pp_tile_pick(a), dim3(a->Hkv * r.mpl.units), dim3(PP_THREADS), 0, s, *a, r.mpl);
    if (r.split) {
      const uint32_t cb = 256 / (a->hd / 4) / 2;           // columns a block
      thvm_launch(false, true, k.tmerge, dim3(a->Hkv * (PP_COLS / cb) * r.many_tiles), dim3(256), 0, s, *a, r.mpl);
    }
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) { snprintf(err, errlen, "attn_paged launch: %s", hipGetErrorString(e)); return -1; }
  return 0;
}
