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
#include "coh.h"

#define LOG2E 1.4426950408889634f

// Columns of a tile from their chunks' partials (sum, m, l), in a fixed order.  HD /
// 4 lanes take a chunk; NP such groups of a block take every NP-th chunk of one
// column and meet in LDS, its other groups have other columns; columns c0 to c1, in
// rounds.  COH: partials of blocks of this launch, read past the caches.
template <int HD, int XT, int CT, int NP, bool COH>
__device__ __forceinline__ void pa_fold(const ThvmPagedArgs &a, const PgPlan &pl, const PgUnit &u, uint32_t kvh,
                                        float4 (*ls)[HD / 4], float *lm, float *ll, uint32_t c0, uint32_t c1) {
  typedef PgT<XT> P;
  constexpr int LN = HD / 4, NG = 256 / LN, CB = NG / NP, BT = 8;   // lanes a chunk, groups, columns at once, loads ahead
  const uint32_t g = threadIdx.x / LN, x = threadIdx.x % LN, part = g % NP, G = a.H / a.Hkv;
  const uint64_t st = (uint64_t)CT * (HD + 4);
  const float *const base = a.ws + ((uint64_t)kvh * pl.slots + u.first) * st;
  for (uint32_t c = c0 + g / NP; c < c1; c += CB) {        // (as many rounds for every thread)
    const uint32_t cc = u.tile * pl.ct + c;
    const bool live = (int32_t)(cc / G) < u.q.r1 - u.q.r0;
    const float *pp = base + (uint64_t)c * (HD + 4);
    float m = -INFINITY, l = 0.0f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    for (uint32_t k0 = part; live && k0 < u.nchunk; k0 += NP * BT) {
      float4 w[BT];
      float2 ml[BT];
#pragma unroll
      for (int t = 0; t < BT; t++) {
        const uint32_t k = min(k0 + t * NP, u.nchunk - 1); // (past the last: read again, not added)
        if (COH) {                                         // (a wave-uniform base: the launcher keeps offsets below 2 GiB)
          const uint32_t o = (k * CT + c) * (HD + 4) * 4;
          const uint4 q = coh_ld16(base, o + x * 16);
          const uint2 e = coh_ld8(base, o + HD * 4);
          w[t] = make_float4(__uint_as_float(q.x), __uint_as_float(q.y), __uint_as_float(q.z), __uint_as_float(q.w));
          ml[t] = make_float2(__uint_as_float(e.x), __uint_as_float(e.y));
        } else {
          w[t] = *(const float4 *)(pp + k * st + 4 * x);
          ml[t] = *(const float2 *)(pp + k * st + HD);
        }
      }
#pragma unroll
      for (int t = 0; t < BT; t++) {
        if (k0 + t * NP >= u.nchunk) break;
        const float mn = fmaxf(m, ml[t].x), f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn),
                    e = ml[t].x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml[t].x - mn);
        v.x = v.x * f + w[t].x * e;
        v.y = v.y * f + w[t].y * e;
        v.z = v.z * f + w[t].z * e;
        v.w = v.w * f + w[t].w * e;
        l = l * f + ml[t].y * e;
        m = mn;
      }
    }
    if (NP > 1) {
      ls[g][x] = v;
      if (x == 0) { lm[g] = m; ll[g] = l; }
      __syncthreads();
      if (part == 0) {
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
      __syncthreads();
    }
    if (!live || part) continue;
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
    *(uint2 *)((uint16_t *)a.out + ((uint64_t)(u.q.r0 + cc / G) * a.H + kvh * G + cc % G) * HD + 4 * x) =
        make_uint2(P::pk(v.x * inv, v.y * inv), P::pk(v.z * inv, v.w * inv));
  }
}

// arrivals at a tile's hand-off: zero before the first launch, left zero by each
#define PA_COUNTERS ((1u << 20) + 2048)
static __device__ uint32_t pa_arrived[PA_COUNTERS];

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
// Bound by the cache's bytes: over 16 bits 16 requests of 30000 rows (8 kv heads of
// 128, 4 query heads each) run at 6.4 TB/s, 32 ragged ones of up to 16000 rows at 5.5;
// over 4 bits 16 of 100000 rows at 5.5 TB/s, where the codec's instructions and the
// loads share a SIMD's two waves.  Short contexts: some 7 us of dependent steps (plan,
// page ids, rows, hand-off), 11 us for one request of 2049 rows.
#define PS_WAVES 4
#define PS_THREADS (PS_WAVES * 64)

// cached bytes in registers on their way to MFMA operands
template <int HD, int BITS> struct PsRegs;
template <> struct PsRegs<128, 16> { uint4 k[4][4]; uint4 v[4][4]; };
template <> struct PsRegs<64, 16> { uint4 k[4][2]; uint2 v[4][4]; };
template <> struct PsRegs<128, 4> { uint4 k[4]; uint32_t ks[4]; uint32_t v[4][4]; uint4 vs[4]; };
template <> struct PsRegs<64, 4> { uint2 k[4]; uint32_t ks[4]; uint32_t v[4][4]; uint2 vs[4]; };

template <int HD, int XT, int BITS, int CG>
__global__ __launch_bounds__(PS_THREADS, HD == 64 && BITS == 4 ? (CG == 8 ? 3 : 4) : 2) void k_paged_split(ThvmPagedArgs a, PgPlan pl) {
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
  const uint64_t head = (uint64_t)kvh * bb;
  const uint32_t pstride = a.Hkv * bb;                     // (below 2^28)
  auto row_of = [&](int it, int t) { return r0 + 256 * it + 64 * t + 16 * wv; };
  // page ids of a step's four tiles, in lanes 0..3; -1: none, or past the chunk's rows
  auto ids = [&](int it) {
    const int32_t r = row_of(it, lane & 3);
    const uint32_t id = buf_ld4(tb, r < r1 ? ((uint32_t)r >> lgp) * 4 : BUF_OOB);
    return ((r < r1) & (id < a.npages)) ? (int32_t)id : -1;
  };
  PsRegs<HD, BITS> R;
  // A tile's place in the pools: its page and first slot, and how many rows it has (0:
  // no page).  16 bits: its resources begin at its first row and end at its last, so
  // what lies past them reads as zeros.  4 bits: they are the page's block (or empty);
  // rows past the last have a p of zero, and their scales are taken as zero below.
  struct Tile { uint64_t page; uint32_t slot, rows; } T[4];
  auto place = [&](int32_t id, int it) {
#pragma unroll
    for (int t = 0; t < 4; t++) {
      const int32_t x = __builtin_amdgcn_readlane(id, t), have = ~(x >> 31), r = row_of(it, t);
      T[t].page = (uint64_t)(uint32_t)(x & have) * pstride + head;
      T[t].slot = (uint32_t)r & pm;
      T[t].rows = (uint32_t)(min(r1 - r, 16) & have);
    }
  };
  auto res = [&](const void *pool, int t) {
    if (BITS == 16) return buf_rsrc((const char *)pool + T[t].page + T[t].slot * RB, T[t].rows * RB);
    return buf_rsrc((const char *)pool + T[t].page, T[t].rows ? bb : 0u);
  };
  const uint32_t ko = lc * RB + (BITS == 16 ? 16 : RB / 4) * lg, vo = 4 * lg * RB + RB / 16 * lc;
  const uint32_t kso = lc * (HD / 32) + lg * HD / 128, vso = 4 * lg * (HD / 32), sbase = a.page * RB;
  auto issue_k = [&]() {
#pragma unroll
    for (int t = 0; t < 4; t++) {
      const buf_t rs = res(a.kpages, t);
      if constexpr (BITS == 16) {
#pragma unroll
        for (int ks = 0; ks < KS; ks++) R.k[t][ks] = buf_ld_stream16(rs, ko + 64 * ks);
      } else {
        const uint32_t so = T[t].slot * RB, ss = sbase + T[t].slot * (HD / 32);
        if constexpr (HD == 128) R.k[t] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rs, ko, so, 2));
        else R.k[t] = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(rs, ko, so, 0));
        R.ks[t] = __builtin_amdgcn_raw_buffer_load_b8(rs, kso, ss, 0);
      }
    }
  };
  auto issue_v = [&]() {
#pragma unroll
    for (int t = 0; t < 4; t++) {
      const buf_t rs = res(a.vpages, t);
      const uint32_t so = T[t].slot * RB, ss = sbase + T[t].slot * (HD / 32);
#pragma unroll
      for (int j = 0; j < 4; j++) {
        if constexpr (BITS == 16) {
          if constexpr (HD == 128) R.v[t][j] = buf_ld_stream16(rs, vo + j * RB);
          else R.v[t][j] = buf_ld8(rs, vo + j * RB);
        } else {
          R.v[t][j] = HD == 128 ? __builtin_amdgcn_raw_buffer_load_b32(rs, vo + j * RB, so, 0)
                                : (uint32_t)__builtin_amdgcn_raw_buffer_load_b16(rs, vo + j * RB, so, 0);
        }
      }
      if constexpr (BITS == 4) {
        if constexpr (HD == 128) R.vs[t] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rs, vso, ss, 0));
        else R.vs[t] = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(rs, vso, ss, 0));
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
    issue_k();
    issue_v();
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
    uint32_t has = 0;                                      // tiles with a page
#pragma unroll
    for (int t = 0; t < 4; t++) has |= T[t].rows ? 1u << t : 0u;
    // this lane's scores: tile s NG + lc / CG of set s
    float p[NS][4];
    float mx = -INFINITY;
#pragma unroll
    for (int s = 0; s < NS; s++) {
      f32x4_t v = sc[s * NG];
#pragma unroll
      for (int j = 1; j < NG; j++)
        if (lc / CG == j) v = sc[s * NG + j];
      const bool ok = has >> (s * NG + lc / CG) & 1;
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
    place(idn, it + 1);
    idn = ids(it + 2);
    issue_k();
    // Over 4 bits the SIMD's instructions bound it: the wave at its V goes first, so the
    // two drift apart and one's scores overlap the other's products (16 requests of
    // 100000 rows 324 -> 314 us, two 51 -> 49; over 16 bits no change)
    if constexpr (BITS == 4) __builtin_amdgcn_s_setprio(1);
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
            odd |= sb == 255u;
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
    // tiles 2h and 2h + 1: the P operand from its terms, V^T's for column EC lc + e
    auto pair = [&](int h, const uint32_t (*x)[2]) {
      const int s0 = (2 * h) / NG, g0 = (2 * h) % NG, s1 = (2 * h + 1) / NG, g1 = (2 * h + 1) % NG;
      const bool in0 = NG == 1 || lc / CG == g0, in1 = NG == 1 || lc / CG == g1;
      return make_uint4(in0 ? x[s0][0] : 0u, in0 ? x[s0][1] : 0u, in1 ? x[s1][0] : 0u, in1 ? x[s1][1] : 0u);
    };
    auto vt = [&](int h, int e) {
      const uint32_t sel = (e & 1) ? 0x07060302u : 0x05040100u;
      return make_uint4(__builtin_amdgcn_perm(w[2 * h][1][e >> 1], w[2 * h][0][e >> 1], sel),
                        __builtin_amdgcn_perm(w[2 * h][3][e >> 1], w[2 * h][2][e >> 1], sel),
                        __builtin_amdgcn_perm(w[2 * h + 1][1][e >> 1], w[2 * h + 1][0][e >> 1], sel),
                        __builtin_amdgcn_perm(w[2 * h + 1][3][e >> 1], w[2 * h + 1][2][e >> 1], sel));
    };
    // A zero p times a V that is not finite is NaN: such values (a stored overflow; a
    // 4-bit group that held one) leave the products, and the columns that see their
    // rows add them one by one, over the sums in LDS.
    if (__builtin_amdgcn_ballot_w64(odd)) {                // wave-uniform
#pragma unroll
      for (int t = 0; t < 4; t++)
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
          for (int e = 0; e < EC / 2; e++) {
            if ((w[t][j][e] & EXP) == EXP) w[t][j][e] &= 0xffff0000u;
            if ((w[t][j][e] >> 16 & EXP) == EXP) w[t][j][e] &= 0xffffu;
          }
      float *const mine = &wacc[wv][lc][4 * EC * lg];      // d = EC (4 lg + i) + e
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int e = 0; e < EC; e++) mine[EC * i + e] = acc[e][i];
#pragma unroll
      for (int s = 0; s < NS; s++) {
        const int32_t rt = row_of(it, s * NG + lc / CG);
#pragma unroll 1
        for (int jj = 0; jj < 4; jj++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const float pr = __shfl(p[s][i], lc + 16 * jj);
            const int32_t r = rt + 4 * jj + i, id = r < lim ? pg_page(&a, u.s, r) : -1;
            if (id < 0) continue;
            const char *vb = (const char *)a.vpages + pg_block(&a, id, kvh);
            const uint32_t slot = (uint32_t)r & pm;
#pragma unroll 1
            for (int k = 0; k < 4 * EC; k++) {
              const uint32_t d = 4 * EC * lg + k;
              float x = __builtin_nanf("");
              if (BITS == 16) {
                const uint32_t h = ((const uint16_t *)vb)[slot * HD + d];
                if ((h & EXP) != EXP) continue;
                x = P::lo(h);
              } else if ((uint8_t)vb[a.page * RB + slot * (HD / 32) + d / 32] != 255u) {
                continue;
              }
              mine[k] += pr * x;
            }
          }
      }
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int e = 0; e < EC; e++) acc[e][i] = mine[EC * i + e];
    }
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const uint4 B = pair(h, pk), B2 = pair(h, pl2);
#pragma unroll
      for (int e = 0; e < EC; e++) {
        const uint4 A = vt(h, e);
        acc[e] = mfma16<XT>(A, B, acc[e]);
        acc[e] = mfma16<XT>(A, B2, acc[e]);
      }
    }
    issue_v();
    if constexpr (BITS == 4) __builtin_amdgcn_s_setprio(0);
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
      float *const rec = a.ws + ((uint64_t)kvh * pl.slots + u.u) * CG * (HD + 4), *pp = rec + c * (HD + 4);
      if (pl.fuse) {
        coh_st8(rec, (c * (HD + 4) + d) * 4, make_uint2(__float_as_uint(s0), __float_as_uint(s1)));
        if (d == 0) coh_st8(rec, (c * (HD + 4) + HD) * 4, make_uint2(__float_as_uint(M), __float_as_uint(lt)));
      } else {
        *(float2 *)(pp + d) = make_float2(s0, s1);
        if (d == 0) *(float2 *)(pp + HD) = make_float2(M, lt);
      }
    }
  }
  if (u.nchunk == 1 || !pl.fuse) return;
  // the tile's last block adds the chunks up, in chunk order
  __shared__ uint32_t lastf;
  vm_drain();
  __syncthreads();
  if (tid == 0) {
    uint32_t *ctr = pa_arrived + (uint64_t)kvh * pl.slots + u.first;
    const uint32_t old = __hip_atomic_fetch_add(ctr, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    lastf = old == u.nchunk - 1 ? 1u : 0u;
    if (lastf) __hip_atomic_exchange(ctr, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!lastf) return;                                      // block-uniform
  pa_fold<HD, XT, CG, (1024 / HD) / CG ? (1024 / HD) / CG : 1, true>(
      a, pl, u, kvh, (float4(*)[HD / 4])&wacc[0][0][0], &wm[0][0], &wl[0][0], 0, CG);
}

#define PA_MERGE 32                                        // columns a block of a prompt tile's merge

// k_paged_merge: the chunks of the tiles that have several, in a launch of its own, CB
// columns a block.
template <int HD, int XT, int CT, int NP, int CB>
__global__ __launch_bounds__(256) void k_paged_merge(ThvmPagedArgs a, PgPlan pl) {
  __shared__ float4 ls[1024 / HD][HD / 4];
  __shared__ float lm[1024 / HD], ll[1024 / HD];
  PgUnit u;
  if (!pg_unit(a, pl, blockIdx.x / (CT / CB) / a.Hkv, true, u) || u.nchunk == 1) return;
  const uint32_t c0 = blockIdx.x % (CT / CB) * CB;
  pa_fold<HD, XT, CT, NP, false>(a, pl, u, blockIdx.x / (CT / CB) % a.Hkv, ls, lm, ll, c0, c0 + CB);
}

// k_paged_plan: the plans of a batch of more than 64 sequences, one block each; a
// thread has up to four sequences in a row.  With it 1024 requests of 100 rows take 149
// us, 512 of 1000 rows 403; with the plan in every wave, 64 sequences at a time, 518
// and 496 (65 requests of 100 rows: 17 us there, a launch more here).
#define PL_THREADS 1024
__global__ __launch_bounds__(PL_THREADS) void k_paged_plan(ThvmPagedArgs a, PgPlan p0, PgPlan p1) {
  const PgPlan p = blockIdx.x ? p1 : p0;
  __shared__ float part[PL_THREADS / 64][2];
  const uint32_t tid = threadIdx.x, wv = tid >> 6, s0 = 4 * tid, bb = (a.b + 3) & ~3u;
  uint32_t *const pre = (uint32_t *)p.pre;
  // (sums of two values over the block, and with scan what the threads before have)
  auto sum2 = [&](float &x, float &y, bool scan) {
    const float xs = wave_scan(x), ys = wave_scan(y);
    __syncthreads();
    if ((tid & 63) == 63) { part[wv][0] = xs; part[wv][1] = ys; }
    __syncthreads();
    float X = 0.0f, Y = 0.0f;
    for (uint32_t w = 0; w < (scan ? wv : blockDim.x / 64); w++) { X += part[w][0]; Y += part[w][1]; }
    x = scan ? X + xs - x : X;
    y = scan ? Y + ys - y : Y;
  };
  float t[4], l[4], total = 0.0f, tiles = 0.0f, n, whole;
#pragma unroll
  for (int k = 0; k < 4; k++) {
    PgSeq q;
    t[k] = 0.0f;
    l[k] = 1.0f;
    if (s0 + k < a.b) pg_count(a, p, s0 + k, q, t[k], l[k]);
    total += t[k] * l[k];
    tiles += t[k];
  }
  sum2(total, tiles, false);
  float full, per, tb = 0.0f, z = 0.0f, nb = 0.0f, wb = 0.0f;
  const uint32_t c = pg_choose(p, total, tiles, [&](uint32_t c, float &sn, float &sw) {
    sn = sw = 0.0f;
#pragma unroll
    for (int k = 0; k < 4; k++) {
      pg_chunks(l[k], c, full, per);
      sn += t[k] * per;
      sw += t[k] * full;
    }
    sum2(sn, sw, false);
  }, n, whole);
#pragma unroll
  for (int k = 0; k < 4; k++) {
    pg_chunks(l[k], c, full, per);
    tb += t[k];
    nb += t[k] * per;
    wb += t[k] * full;
  }
  sum2(tb, z, true);
  sum2(nb, wb, true);
  if (tid == 0) *(uint4 *)pre = make_uint4(c, (uint32_t)n, (uint32_t)whole, (uint32_t)tiles);
#pragma unroll
  for (int k = 0; k < 4; k++)
    if (s0 + k < a.b) {
      pre[4 + s0 + k] = (uint32_t)tb;
      pre[4 + bb + s0 + k] = (uint32_t)nb;
      pre[4 + 2 * bb + s0 + k] = (uint32_t)wb;
      pg_chunks(l[k], c, full, per);
      tb += t[k];
      nb += t[k] * per;
      wb += t[k] * full;
    }
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
  r.few_tiles = (a->b < a->n ? a->b : a->n) * ((hi + 15) / 16);   // (of sequences with a row)
  r.fpl = PgPlan{0, hi, 16, fill > 2 * r.few_tiles ? fill : 2 * r.few_tiles, 4, 0, 0, 0, 0.8f, nullptr};
  // twice the units (see PgPlan) from 1.5 MB of cache a unit on: 32 ragged requests of
  // up to 16000 rows 119 -> 108 us, 24 of 16000 each 280 -> 246; with a fifth of that
  // twice the blocks lose (eight ragged requests of up to 8000 rows 29 -> 34 us)
  const uint32_t step = 64 * 2 * (a->bits == 16 ? a->hd * 2 : a->hd / 2 + a->hd / 32);
  r.fpl.cbig = (3u << 19) / step;
  // heads of 64 in 4 bits: registers for four blocks a CU, so twice the units from 40
  // steps on (16 requests of 16000 rows 48.5 -> 42.9 us, 25 heads x 4 of 100000 191 ->
  // 166; below, four of 16000 lose: 19.5 -> 20.9)
  if (a->hd == 64 && a->bits == 4) { r.fpl.cbig = 40; r.fpl.even = 2.0f; }
  r.fpl.slots = r.fpl.units << ((uint64_t)r.few_tiles * a->maxpages * a->page / 64 >= (uint64_t)r.fpl.units * r.fpl.cbig);
  // about as many chunks as a tile can have, twice the mean where the units are shared
  const uint64_t cap = ((uint64_t)a->maxpages * a->page + 64 * r.fpl.cmin - 1) / (64 * r.fpl.cmin), mean = 2 * r.fpl.slots / r.few_tiles + 1;
  const uint64_t chunks = cap < mean ? cap : mean < r.fpl.slots ? mean : r.fpl.slots;
  r.fpl.fuse = chunks * r.cg <= 96 && (uint64_t)a->Hkv * r.fpl.slots <= PA_COUNTERS &&
               (uint64_t)r.fpl.slots * r.cg * (a->hd + 4) * 4 < (1ull << 31);
  const uint32_t whole = (uint32_t)((uint64_t)a->n * G / PP_COLS);
  r.many_tiles = whole + (a->b < a->n ? a->b : a->n);
  r.split = (uint64_t)whole * a->Hkv < 512;
  r.mpl = PgPlan{r.few ? hi : 0, 0xffffffffu, PP_COLS, r.many_tiles + 1, 1u << 25, 0, 0, 0, 0.0f, nullptr};
  if (r.split) {
    r.mpl.units = fill > 2 * r.many_tiles ? fill : 2 * r.many_tiles;
    r.mpl.cmin = 4;
  }
  r.mpl.slots = r.mpl.units;
  return r;
}

// words of the plans at the workspace's start: one for each half of the rule
static uint64_t pa_pre_words(const ThvmPagedArgs *a) { return a->b > 64 ? 2 * PG_PRE_WORDS((uint64_t)a->b) : 0; }

extern "C" uint64_t thvm_k_attn_paged_ws(const ThvmPagedArgs *a) {
  const PaRule r = pa_rule(a);
  const uint64_t rec = (uint64_t)a->Hkv * (a->hd + 4) * 4, f = r.few ? rec * r.fpl.slots * r.cg : 0,
                 m = r.many && r.split ? rec * r.mpl.slots * PP_COLS : 0;
  return (f > m ? f : m > 16 ? m : 16) + pa_pre_words(a) * 4;
}

template <int HD, int XT, int BITS>
static paged_fn pa_split(uint32_t cg) {
  return cg == 4 ? k_paged_split<HD, XT, BITS, 4> : cg == 8 ? k_paged_split<HD, XT, BITS, 8> : k_paged_split<HD, XT, BITS, 16>;
}
struct PaKernels { paged_fn split, merge, tmerge; };
template <int HD, int XT>
static PaKernels pa_pick(const ThvmPagedArgs *a, uint32_t cg, uint32_t cb) {
  constexpr int NG = 1024 / HD;                            // (one column a block: all groups)
  return PaKernels{a->bits == 16 ? pa_split<HD, XT, 16>(cg) : pa_split<HD, XT, 4>(cg),
                   cg == 4 ? k_paged_merge<HD, XT, 4, NG, 1> : cg == 8 ? k_paged_merge<HD, XT, 8, NG, 1>
                   : cb == 1 ? k_paged_merge<HD, XT, 16, NG, 1> : k_paged_merge<HD, XT, 16, 2, 4>,
                   k_paged_merge<HD, XT, PP_COLS, 1, PA_MERGE>};
}

extern "C" int thvm_k_attn_paged(const ThvmPagedArgs *call, hipStream_t s, char *err, int errlen) {
  if (pg_check(call, PG_ATTN, err, errlen)) return -1;
  ThvmPagedArgs args = *call, *const a = &args;
  PaRule r = pa_rule(a);
  const int bf = a->dt == THVM_DT_BF16;
  // Columns a block of the merge: one, with all its groups on the chunks; of 16 columns
  // four from 64 tiles on, which have few chunks and would be blocks that plan more than
  // they add (1 | 4 columns, us: 16 x 8 tiles 27.3 | 25.3, 8 x 8 20.2 | 20.0, one of 4000
  // rows 14.5 | 16.6)
  const uint32_t cb = r.cg == 16 && (uint64_t)a->Hkv * r.few_tiles >= 64 ? 4 : 1;
  const PaKernels k = a->hd == 128 ? (bf ? pa_pick<128, GX_BF16>(a, r.cg, cb) : pa_pick<128, GX_F16>(a, r.cg, cb))
                                   : (bf ? pa_pick<64, GX_BF16>(a, r.cg, cb) : pa_pick<64, GX_F16>(a, r.cg, cb));
  const bool plan = a->b > 64;
  if (plan) {
    r.fpl.pre = (const uint32_t *)a->ws;
    r.mpl.pre = r.fpl.pre + PG_PRE_WORDS(a->b);
    a->ws += pa_pre_words(a);
    thvm_launch(true, false, k_paged_plan, dim3(r.few && r.many ? 2 : 1), dim3((a->b + 255) / 256 * 64), 0, s, *a,
                r.few ? r.fpl : r.mpl, r.mpl);
  }
  if (r.few) {
    const bool last = !r.many;
    thvm_launch(!plan, last && r.fpl.fuse, k.split, dim3(a->Hkv * r.fpl.slots), dim3(PS_THREADS), 0, s, *a, r.fpl);
    if (!r.fpl.fuse)
      thvm_launch(false, last, k.merge, dim3(a->Hkv * (r.cg / cb) * r.few_tiles), dim3(256), 0, s, *a, r.fpl);
  }
  if (r.many) {
    thvm_launch(!plan && !r.few, !r.split, pp_tile_pick(a), dim3(a->Hkv * r.mpl.slots), dim3(PP_THREADS), 0, s, *a, r.mpl);
    if (r.split)
      thvm_launch(false, true, k.tmerge, dim3(a->Hkv * (PP_COLS / PA_MERGE) * r.many_tiles), dim3(256), 0, s, *a, r.mpl);
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) { snprintf(err, errlen, "attn_paged launch: %s", hipGetErrorString(e)); return -1; }
  return 0;
}
