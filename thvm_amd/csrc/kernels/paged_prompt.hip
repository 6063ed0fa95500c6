// paged_prompt.hip -- attention over a paged cache for sequences with many
// columns (rows x query heads of a kv head): prompts, and chunks of them over
// long caches.
//
// A block takes a tile of 128 columns of one kv head, 32 a wave, and streams the
// cache rows in steps of 64 through LDS, so a cache row is fetched once for 128
// columns and all query heads of its group.
//   scores  S[row][column] = K q^T, 32x32x16 MFMAs, q in registers; a lane holds
//           32 rows' scores of one column (two lanes a column), so the maximum and
//           the sum are its own but for one exchange;
//   mix     O^T[d][column] += V^T P^T: the P operand is the score layout itself
//           (rows in the order the lanes hold them), and V^T in that order comes
//           out of LDS by transposing reads (4 rows of one column a lane).
//   LDS     rows of hd 16-bit values in 16-byte pieces whose order is XORed with
//           the row, so that neither the operand reads (16 rows at one piece), nor
//           the transposing ones (4 rows at 64 bytes), nor the stores meet in a
//           bank; two buffers, the next step's bytes in registers meanwhile.  A
//           4-bit cache is expanded on its way into LDS: its codec work is shared
//           by the tile's columns too.
// The running maximum moves only when a score passes it by 2^6 (the sums are f32
// and p has room: up to 2^6 in bf16, 2^14 of fp16's 2^16 with p scaled by 2^8,
// which keeps small p off fp16's subnormals); p is rounded once, to the 16-bit type
// of the values it multiplies, and its sum, in f32, is that of the rounded ones.
// Bound by the matrix and exponential units.
#include "paged_core.h"

#define PP_STEP 64
#define LOG2E 1.4426950408889634f

typedef float f32x16_t __attribute__((ext_vector_type(16)));
template <int XT>
__device__ __forceinline__ f32x16_t mfma32(const uint4 &A, const uint4 &B, f32x16_t c) {
  if (XT == GX_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, A), __builtin_bit_cast(bf16x8_t, B), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, A), __builtin_bit_cast(f16x8_t, B), c, 0, 0, 0);
}
typedef short s16x4v_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4v_t lds_s16x4_t;

template <bool V> struct pp_const { static constexpr bool value = V; };

// byte of 16-byte piece c of row r in a step's K or V
template <int HD> __device__ __forceinline__ uint32_t k_at(uint32_t r, uint32_t c) {
  return r * (HD * 2) + ((c ^ (HD == 128 ? r & 15u : r >> 1 & 7u)) << 4);
}
template <int HD> __device__ __forceinline__ uint32_t v_at(uint32_t r, uint32_t c) {
  return r * (HD * 2) + ((c ^ (HD == 128 ? (r & 3u) * 5u : (r >> 1 & 1u) * 5u)) << 4);
}

template <int HD, int XT, int BITS>
__global__ __launch_bounds__(PP_THREADS, 2) void k_paged_tile(ThvmPagedArgs a, PgPlan pl) {
  typedef PgT<XT> P;
  constexpr int KS = HD / 16, DB = HD / 32, RB = BITS == 16 ? HD * 2 : HD / 2;
  constexpr int NL = BITS == 16 ? HD / 32 : 1;             // 16-byte (4 bits, hd 64: 8-byte) loads of K a thread
  constexpr float PSH = XT == GX_BF16 ? 0.0f : 8.0f;
  constexpr uint32_t EXP = XT == GX_BF16 ? 0x7f80u : 0x7c00u;
  __shared__ __align__(16) char lk[2][PP_STEP * HD * 2], lv[2][PP_STEP * HD * 2];
  const uint32_t kvh = blockIdx.x % a.Hkv, un = blockIdx.x / a.Hkv, G = a.H / a.Hkv;
  PgUnit u;
  if (!pg_unit(a, pl, un, false, u)) return;
  const int tid = threadIdx.x, wv = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, n = lane & 31, h = lane >> 5;
  const int32_t nrow = u.q.r1 - u.q.r0, cap = (int32_t)(a.maxpages * a.page), p0 = u.q.len - nrow;
  const uint32_t ncol = (uint32_t)nrow * G, col = u.tile * PP_COLS + 32 * wv + n;
  const bool live = col < ncol;
  const uint32_t ri = col / G, hg = col % G;
  // cache rows: the chunk's, as far as the tile's last column sees
  const int32_t last = (int32_t)((min(ncol, (u.tile + 1) * PP_COLS) - 1) / G);
  const int32_t see = min(p0 + last + 1, cap);
  const int32_t r0 = (int32_t)(u.chunk * u.c * PP_STEP);
  const int32_t r1 = u.chunk + 1 == u.nchunk ? see : min(see, (int32_t)((u.chunk + 1) * u.c * PP_STEP));
  const int32_t lim = live ? min(p0 + (int32_t)ri + 1, r1) : 0;
  // from row whi on none of the wave's columns sees a row
  const uint32_t c0 = u.tile * PP_COLS + 32 * wv;
  const int32_t whi = c0 < ncol ? min(p0 + (int32_t)((min(ncol, c0 + 32) - 1) / G) + 1, r1) : 0;
  uint4 qb[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ks++)
    qb[ks] = live ? ld16((const uint16_t *)a.q + ((uint64_t)(u.q.r0 + ri) * a.H + kvh * G + hg) * HD + 16 * ks + 8 * h)
                  : make_uint4(0, 0, 0, 0);
  // scores are scaled inside the exponent, by a positive number: a negative scale's
  // sign goes to q, and with a scale of zero (or too near for f32) q is zero
  const bool none = fabsf(a.scale) < 1e-37f;
  const float qs = none ? 1.0f : fabsf(a.scale) * LOG2E;
  if (none || a.scale < 0.0f)
#pragma unroll
    for (int ks = 0; ks < KS; ks++)
      qb[ks] = none ? make_uint4(0, 0, 0, 0)
                    : make_uint4(qb[ks].x ^ 0x80008000u, qb[ks].y ^ 0x80008000u, qb[ks].z ^ 0x80008000u, qb[ks].w ^ 0x80008000u);
  const buf_t tb = buf_rsrc(a.table + (uint64_t)u.s * a.maxpages, a.maxpages * 4);
  const uint32_t lgp = __builtin_ctz(a.page), pm = a.page - 1, bb = pg_block_bytes(&a);
  const int nt = r1 > r0 ? (r1 - r0 + PP_STEP - 1) / PP_STEP : 0;
  // page ids of a step's four 16-row groups, in lanes 0..3
  auto ids = [&](int j) {
    const int32_t r = r0 + PP_STEP * j + 16 * (lane & 3);
    return (int32_t)buf_ld4(tb, r < r1 ? ((uint32_t)r >> lgp) * 4 : BUF_OOB);
  };
  auto group_ok = [&](int32_t id, int j, int g) {
    return (uint32_t)__builtin_amdgcn_readlane(id, g) < a.npages && r0 + PP_STEP * j + 16 * g < r1;
  };
  // what a thread stages of a step: pieces of rows tid / PR + i * rows-per-pass
  uint4 sk[NL], sv[NL];
  uint32_t ssc;                                            // 4 bits: K's scale byte, V's in the next
  auto load = [&](int32_t id, int j) {
#pragma unroll
    for (int i = 0; i < NL; i++) {
      // the 16-row group of this wave's rows in pass i
      const int g = BITS == 4 ? wv : HD == 128 ? i : 2 * i + (wv >> 1);
      const bool ok = group_ok(id, j, g);
      const uint64_t off = ok ? pg_block(&a, __builtin_amdgcn_readlane(id, g), kvh) : 0;
      const buf_t kr = buf_rsrc((const char *)a.kpages + off, ok ? bb : 0u), vr = buf_rsrc((const char *)a.vpages + off, ok ? bb : 0u);
      if constexpr (BITS == 16) {
        constexpr int PR = HD / 8;                         // pieces a row
        const int32_t r = r0 + PP_STEP * j + tid / PR + i * (PP_THREADS / PR);
        const uint32_t o = r < r1 ? ((uint32_t)r & pm) * RB + (tid % PR) * 16 : BUF_OOB;
        sk[i] = buf_ld16(kr, o);
        sv[i] = buf_ld16(vr, o);
      } else {
        const int32_t r = r0 + PP_STEP * j + tid / 4;
        const uint32_t slot = (uint32_t)r & pm, pc = tid & 3;
        const uint32_t o = r < r1 ? slot * RB + pc * (RB / 4) : BUF_OOB;
        const uint32_t so = r < r1 ? a.page * RB + slot * (HD / 32) + pc * HD / 128 : BUF_OOB;
        if constexpr (HD == 128) {
          sk[i] = buf_ld16(kr, o);
          sv[i] = buf_ld16(vr, o);
        } else {
          const uint2 x = buf_ld8(kr, o), y = buf_ld8(vr, o);
          sk[i] = make_uint4(x.x, x.y, 0, 0);
          sv[i] = make_uint4(y.x, y.y, 0, 0);
        }
        ssc = (uint32_t)__builtin_amdgcn_raw_buffer_load_b8(kr, so, 0, 0) |
              (uint32_t)__builtin_amdgcn_raw_buffer_load_b8(vr, so, 0, 0) << 8;
      }
    }
  };
  auto store = [&](int b) {
    if constexpr (BITS == 16) {
      constexpr int PR = HD / 8;
#pragma unroll
      for (int i = 0; i < NL; i++) {
        const uint32_t r = tid / PR + i * (PP_THREADS / PR), c = tid % PR;
        *(uint4 *)&lk[b][k_at<HD>(r, c)] = sk[i];
        *(uint4 *)&lv[b][v_at<HD>(r, c)] = sv[i];
      }
    } else {
      const uint32_t r = tid / 4, pc = tid & 3;
      const float fk = e8m0_f(ssc & 0xffu), fv = e8m0_f(ssc >> 8);
      const uint32_t wk[4] = {sk[0].x, sk[0].y, sk[0].z, sk[0].w}, wvv[4] = {sv[0].x, sv[0].y, sv[0].z, sv[0].w};
#pragma unroll
      for (int c = 0; c < HD / 32; c++) {                  // 8 values a dword of codes
        *(uint4 *)&lk[b][k_at<HD>(r, pc * (HD / 32) + c)] =
            make_uint4(fp4x2<XT, 0>(wk[c], fk), fp4x2<XT, 1>(wk[c], fk), fp4x2<XT, 2>(wk[c], fk), fp4x2<XT, 3>(wk[c], fk));
        *(uint4 *)&lv[b][v_at<HD>(r, pc * (HD / 32) + c)] =
            make_uint4(fp4x2<XT, 0>(wvv[c], fv), fp4x2<XT, 1>(wvv[c], fv), fp4x2<XT, 2>(wvv[c], fv), fp4x2<XT, 3>(wvv[c], fv));
      }
    }
  };
  // operand addresses: a piece's XOR depends on the lane alone, rows add constants
  uint32_t ka[KS], va[DB];
#pragma unroll
  for (int ks = 0; ks < KS; ks++) ka[ks] = k_at<HD>(n, 2 * ks + h);
#pragma unroll
  for (int d = 0; d < DB; d++) {
    // row 4 h + (lane % 16) / 4, 8 bytes at column 32 d + 16 (lane / 16 % 2) + 4 (lane % 4)
    const uint32_t cb = 64 * d + 32 * (lane >> 4 & 1) + 8 * (lane & 3);
    va[d] = v_at<HD>(4 * h + (lane & 15) / 4, cb >> 4) + (cb & 15);
  }
  float m = -INFINITY, l = 0.0f;
  f32x16_t acc[DB];
#pragma unroll
  for (int d = 0; d < DB; d++)
#pragma unroll
    for (int i = 0; i < 16; i++) acc[d][i] = 0.0f;
  auto step = [&](auto masked, int b, int j, uint32_t holes) {
    constexpr bool MASK = decltype(masked)::value;
    f32x16_t sc[2];
#pragma unroll
    for (int rb = 0; rb < 2; rb++) {
#pragma unroll
      for (int i = 0; i < 16; i++) sc[rb][i] = 0.0f;
#pragma unroll
      for (int ks = 0; ks < KS; ks++)
        sc[rb] = mfma32<XT>(*(const uint4 *)&lk[b][ka[ks] + 32 * rb * (HD * 2)], qb[ks], sc[rb]);
    }
    const int32_t rr = r0 + PP_STEP * j;
    float mx = -INFINITY;
#pragma unroll
    for (int rb = 0; rb < 2; rb++)
#pragma unroll
      for (int i = 0; i < 16; i++) {
        float x = sc[rb][i];                               // (scaled in the exponent)
        if (MASK) {
          const int r = 32 * rb + 8 * (i / 4) + 4 * h + i % 4;
          if (rr + r >= lim || (holes >> (r / 16) & 1)) x = -INFINITY;
        }
        sc[rb][i] = x;
        mx = fmaxf(mx, x);
      }
    mx = fmaxf(mx, xor32_f(mx)) * qs;
    if (__builtin_amdgcn_ballot_w64(mx > m + 6.0f)) {      // (m = -inf: any score)
      const float mn = fmaxf(m, mx), f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
      l *= f;
#pragma unroll
      for (int d = 0; d < DB; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) acc[d][i] *= f;
      m = mn;
    }
    const float mb = (m == -INFINITY ? 0.0f : m) - PSH;
    float ls[4] = {0.f, 0.f, 0.f, 0.f};
    uint32_t pk[2][8];
#pragma unroll
    for (int rb = 0; rb < 2; rb++)
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        pk[rb][i / 2] = P::pk(__builtin_amdgcn_exp2f(fmaf(sc[rb][i], qs, -mb)), __builtin_amdgcn_exp2f(fmaf(sc[rb][i + 1], qs, -mb)));
        ls[(i / 2) & 3] = P::sum2(pk[rb][i / 2], ls[(i / 2) & 3]);
      }
    l += (ls[0] + ls[1]) + (ls[2] + ls[3]);
#pragma unroll
    for (int s = 0; s < 4; s++) {                          // 16 rows each
      const uint4 B = make_uint4(pk[s / 2][4 * (s & 1)], pk[s / 2][4 * (s & 1) + 1], pk[s / 2][4 * (s & 1) + 2],
                                 pk[s / 2][4 * (s & 1) + 3]);
#pragma unroll
      for (int d = 0; d < DB; d++) {
        uint4 A;
        {
          // rows 16 s + 4 h .. + 3 and those 8 further on, in the order of P's
          typedef uint32_t u2_t __attribute__((ext_vector_type(2)));
          const u2_t x = __builtin_bit_cast(u2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                      (lds_s16x4_t *)&lv[b][va[d] + 16 * s * (HD * 2)]));
          const u2_t y = __builtin_bit_cast(u2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                      (lds_s16x4_t *)&lv[b][va[d] + (16 * s + 8) * (HD * 2)]));
          A = make_uint4(x[0], x[1], y[0], y[1]);
        }
        if (MASK) {
          // A zero p times a V that is not finite is NaN: where a step has masked
          // rows, such values leave the product and come back as +inf, -inf or (both)
          // NaN in the columns where one has a p above zero.
          uint32_t w[4] = {A.x, A.y, A.z, A.w}, odd = 0;
#pragma unroll
          for (int i = 0; i < 4; i++) odd |= (w[i] & EXP) == EXP || (w[i] >> 16 & EXP) == EXP;
          if (__builtin_amdgcn_ballot_w64(odd)) {          // wave-uniform
#pragma unroll 1
            for (int sign = 0; sign < 2; sign++) {
              const uint32_t one = XT == GX_BF16 ? 0x3f80u : 0x3c00u, other = sign ? EXP : EXP | 0x8000u;
              uint32_t t[4];
#pragma unroll
              for (int i = 0; i < 4; i++) {
                const uint32_t x = w[i] & 0xffffu, y = w[i] >> 16;
                t[i] = ((x & EXP) == EXP && x != other ? one : 0u) | ((y & EXP) == EXP && y != other ? one << 16 : 0u);
              }
              f32x16_t z;
#pragma unroll
              for (int i = 0; i < 16; i++) z[i] = 0.0f;
              z = mfma32<XT>(make_uint4(t[0], t[1], t[2], t[3]), B, z);
#pragma unroll
              for (int i = 0; i < 16; i++) acc[d][i] += z[i] > 0.0f ? (sign ? -INFINITY : INFINITY) : 0.0f;
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
              if ((w[i] & EXP) == EXP) w[i] &= 0xffff0000u;
              if ((w[i] >> 16 & EXP) == EXP) w[i] &= 0xffffu;
            }
            A = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        acc[d] = mfma32<XT>(A, B, acc[d]);
      }
    }
  };
  int32_t id = ids(0), idn = ids(1);
  if (nt) {
    load(id, 0);
    store(0);
  }
  __syncthreads();
  // steps that every column of the block sees whole, then (from the first page that
  // is none, or the first position of the tile) the others
  const int32_t all = p0 + (int32_t)(u.tile * PP_COLS / G) + 1;
  int j = 0;
  auto holes_of = [&](int32_t i) {
    uint32_t o = 0;
#pragma unroll
    for (int g = 0; g < 4; g++) o |= group_ok(i, j, g) ? 0u : 1u << g;
    return o;
  };
  auto next = [&](auto run) {                              // the next step's bytes on their way meanwhile
    id = idn;
    idn = ids(j + 2);
    const bool more = j + 1 < nt;
    if (more) load(id, j + 1);
    run();
    if (more) store((j + 1) & 1);
    __syncthreads();
    j++;
  };
  while (j < nt && r0 + PP_STEP * (j + 1) <= min(all, r1) && holes_of(id) == 0)
    next([&] { step(pp_const<false>{}, j & 1, j, 0); });
  while (j < nt) {
    const uint32_t holes = holes_of(id);
    next([&] { if (r0 + PP_STEP * j < whi) step(pp_const<true>{}, j & 1, j, holes); });   // wave-uniform
  }
  if (!live) return;
  l += xor32_f(l);
  if (u.nchunk == 1) {
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
    uint16_t *o = (uint16_t *)a.out + ((uint64_t)(u.q.r0 + ri) * a.H + kvh * G + hg) * HD + 4 * h;
#pragma unroll
    for (int d = 0; d < DB; d++)
#pragma unroll
      for (int q = 0; q < 4; q++)
        *(uint2 *)(o + 32 * d + 8 * q) = make_uint2(P::pk(acc[d][4 * q] * inv, acc[d][4 * q + 1] * inv),
                                                    P::pk(acc[d][4 * q + 2] * inv, acc[d][4 * q + 3] * inv));
  } else {
    float *pp = a.ws + (((uint64_t)kvh * pl.units + u.u) * PP_COLS + 32 * wv + n) * (HD + 4);
#pragma unroll
    for (int d = 0; d < DB; d++)
#pragma unroll
      for (int q = 0; q < 4; q++)
        *(float4 *)(pp + 32 * d + 8 * q + 4 * h) = make_float4(acc[d][4 * q], acc[d][4 * q + 1], acc[d][4 * q + 2], acc[d][4 * q + 3]);
    if (h == 0) *(float2 *)(pp + HD) = make_float2(m, l);
  }
}

paged_fn pp_tile_pick(const ThvmPagedArgs *a) {
  const int bf = a->dt == THVM_DT_BF16;
#define PP_PICK(HD) (bf ? (a->bits == 16 ? k_paged_tile<HD, GX_BF16, 16> : k_paged_tile<HD, GX_BF16, 4>)             \
                        : (a->bits == 16 ? k_paged_tile<HD, GX_F16, 16> : k_paged_tile<HD, GX_F16, 4>))
  return a->hd == 128 ? PP_PICK(128) : PP_PICK(64);
}
