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
// Bound by the matrix and exponential units: five ragged prompts of up to 3001 rows (8
// kv heads of 128, 4 query heads each) in 250 us, 820 TFLOP/s.  The products alone take
// 183 us of it (1136 TFLOP/s), loads and exponents what does not overlap.  Blocks of 8
// waves lose (266 us), so do deeper prefetch and wave priorities (no change).
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
// 16 bytes a lane from memory into LDS, the wave's lanes in consecutive places from dst
// on (wave-uniform); offsets past the resource write zeros
__device__ __forceinline__ void buf_lds16(buf_t r, char *dst, uint32_t off) {
#ifdef __HIP_DEVICE_COMPILE__                              // (the host pass does not know the builtin's size)
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)dst, 16, off, 0, 0, 0);
#endif
}

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
  constexpr int NL = HD / 32;                              // passes of the block over a step's K or V
  constexpr float PSH = XT == GX_BF16 ? 0.0f : 8.0f;
  constexpr uint32_t EXP = XT == GX_BF16 ? 0x7f80u : 0x7c00u;
  // (arrays apart: reads of one then need not wait for what is on its way into another)
  __shared__ __align__(16) char lk0[PP_STEP * HD * 2], lk1[PP_STEP * HD * 2], lv0[PP_STEP * HD * 2], lv1[PP_STEP * HD * 2];
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
  // rows below `all` every column of the block sees
  const int32_t all = p0 + (int32_t)(u.tile * PP_COLS / G) + 1;
  const int nt = r1 > r0 ? (r1 - r0 + PP_STEP - 1) / PP_STEP : 0;
  // page ids of a step's four 16-row groups, in lanes 0..3; -1: none, or past the rows
  auto ids = [&](int j) {
    const int32_t r = r0 + PP_STEP * j + 16 * (lane & 3);
    const uint32_t id = buf_ld4(tb, r < r1 ? ((uint32_t)r >> lgp) * 4 : BUF_OOB);
    return ((r < r1) & (id < a.npages)) ? (int32_t)id : -1;
  };
  // The way of a step's K or V into LDS.  16 bits: straight from memory, 16 bytes a
  // lane into consecutive places, so the XOR of the pieces is in what a lane asks for;
  // a group's resource begins at its first row and ends at its last (rows past it and
  // pages that are none read as zeros), which leaves a lane's offset constant.  4 bits:
  // through registers and the codec, 32 (hd 64: 16) values a thread.
  const uint64_t pstride = a.Hkv * bb, head = (uint64_t)kvh * bb;
  const uint32_t ps32 = (uint32_t)pstride;
  auto group = [&](const void *pool, int32_t id, int j, int g, uint32_t at, uint32_t rb, int32_t most = 16) {
    const int32_t x = __builtin_amdgcn_readlane(id, g), have = ~(x >> 31), gr = r0 + PP_STEP * j + 16 * g;
    return buf_rsrc((const char *)pool + head + (uint64_t)(uint32_t)(x & have) * ps32 + at + ((uint32_t)gr & pm) * rb,
                    (uint32_t)(min(r1 - gr, most) & have) * rb);
  };
  constexpr int PR = HD / 8;                               // 16-byte pieces of a row in LDS
  const uint32_t r16 = (tid / PR) & 15, pc = tid % PR;
  const uint32_t ko = r16 * RB + (k_at<HD>(r16, pc) - r16 * (HD * 2)), vo = r16 * RB + (v_at<HD>(r16, pc) - r16 * (HD * 2));
  struct Reg { uint4 c; uint32_t s; } rk, rv;
  auto load = [&](const void *pool, int32_t id, int j, char *dst, uint32_t off, Reg &x) {
    if constexpr (BITS == 16) {
      if (a.page >= PP_STEP) {                             // the whole step in one page
        const buf_t rs = group(pool, id, j, 0, 0, RB, PP_STEP);
#pragma unroll
        for (int i = 0; i < NL; i++)
          buf_lds16(rs, &dst[(i * PP_THREADS + wv * 64) * 16], off + (wv * 64 / PR / 16 * 16 + i * (PP_THREADS / PR)) * RB);
      } else
#pragma unroll
      for (int i = 0; i < NL; i++)                         // the 16-row group of this wave's rows in pass i
        buf_lds16(group(pool, id, j, HD == 128 ? i : 2 * i + (wv >> 1), 0, RB), &dst[(i * PP_THREADS + wv * 64) * 16], off);
    } else {
      const uint32_t r = (tid >> 2) & 15, p4 = tid & 3;
      const buf_t rs = group(pool, id, j, wv, 0, RB);
      if constexpr (HD == 128) {
        x.c = buf_ld16(rs, r * RB + p4 * (RB / 4));
      } else {
        const uint2 y = buf_ld8(rs, r * RB + p4 * (RB / 4));
        x.c = make_uint4(y.x, y.y, 0, 0);
      }
      x.s = (uint32_t)__builtin_amdgcn_raw_buffer_load_b8(group(pool, id, j, wv, a.page * RB, HD / 32), r * (HD / 32) + p4 * HD / 128, 0, 0);
    }
  };
  auto store = [&](char *dst, auto at, const Reg &x) {
    if constexpr (BITS == 4) {
      const uint32_t r = tid / 4, p4 = tid & 3, w[4] = {x.c.x, x.c.y, x.c.z, x.c.w};
      const float f = e8m0_f(x.s);
#pragma unroll
      for (int c = 0; c < HD / 32; c++)                    // 8 values a dword of codes
        *(uint4 *)&dst[at(r, p4 * (HD / 32) + c)] =
            make_uint4(fp4x2<XT, 0>(w[c], f), fp4x2<XT, 1>(w[c], f), fp4x2<XT, 2>(w[c], f), fp4x2<XT, 3>(w[c], f));
    }
  };
  auto load_k = [&](int32_t id, int j, char *dst) { load(a.kpages, id, j, dst, ko, rk); };
  auto load_v = [&](int32_t id, int j, char *dst) { load(a.vpages, id, j, dst, vo, rv); };
  auto store_k = [&](char *dst) { store(dst, [](uint32_t r, uint32_t c) { return k_at<HD>(r, c); }, rk); };
  auto store_v = [&](char *dst) { store(dst, [](uint32_t r, uint32_t c) { return v_at<HD>(r, c); }, rv); };
  // the block's own LDS loads done, then the other waves'
  auto arrive = [] {
    __builtin_amdgcn_s_waitcnt(0x0f70);                    // vmcnt(0)
    __syncthreads();
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
  struct Sc { f32x16_t v[2]; };
  auto scores = [&](const char *lk, Sc &S) {
#pragma unroll
    for (int rb = 0; rb < 2; rb++)
#pragma unroll
      for (int i = 0; i < 16; i++) S.v[rb][i] = 0.0f;
#pragma unroll
    for (int ks = 0; ks < KS; ks++) {
#pragma unroll
      for (int rb = 0; rb < 2; rb++)
        S.v[rb] = mfma32<XT>(*(const uint4 *)&lk[ka[ks] + 32 * rb * (HD * 2)], qb[ks], S.v[rb]);
    }
  };
  // the scores that a column does not see to -inf, and the largest
  auto top = [&](auto masked, int j, uint32_t holes, Sc &S) {
    constexpr bool MASK = decltype(masked)::value;
    float mx = -INFINITY;
    if (MASK) {
      const int32_t left = lim - (r0 + PP_STEP * j) - 4 * h;
      int32_t lg[4];
#pragma unroll
      for (int g = 0; g < 4; g++) lg[g] = holes >> g & 1 ? 0 : left;
#pragma unroll
      for (int rb = 0; rb < 2; rb++)
#pragma unroll
        for (int i = 0; i < 16; i++) {
          const int r = 32 * rb + 8 * (i / 4) + i % 4;     // (4 h is in left)
          S.v[rb][i] = r < lg[r / 16] ? S.v[rb][i] : -INFINITY;
        }
    }
#pragma unroll
    for (int rb = 0; rb < 2; rb++)
#pragma unroll
      for (int i = 0; i < 16; i++) mx = fmaxf(mx, S.v[rb][i]);
    return mx;
  };
  auto move = [&](float mx) {
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
  };
  auto expo = [&](const Sc &S, uint32_t pk[2][8]) {
    const float mb = (m == -INFINITY ? 0.0f : m) - PSH;
    float ls[2] = {0.f, 0.f};
#pragma unroll
    for (int rb = 0; rb < 2; rb++)
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        pk[rb][i / 2] = P::pk(__builtin_amdgcn_exp2f(fmaf(S.v[rb][i], qs, -mb)), __builtin_amdgcn_exp2f(fmaf(S.v[rb][i + 1], qs, -mb)));
        ls[i / 2 & 1] = P::sum2(pk[rb][i / 2], ls[i / 2 & 1]);
      }
    l += ls[0] + ls[1];
  };
  auto mix = [&](auto masked, const char *lv, const uint32_t pk[2][8]) {
    constexpr bool MASK = decltype(masked)::value;
#pragma unroll
    for (int s = 0; s < 4; s++) {                          // 16 rows each
      const uint4 B = make_uint4(pk[s / 2][4 * (s & 1)], pk[s / 2][4 * (s & 1) + 1], pk[s / 2][4 * (s & 1) + 2],
                                 pk[s / 2][4 * (s & 1) + 3]);
#pragma unroll
      for (int d = 0; d < DB; d++) {
        // rows 16 s + 4 h .. + 3 and those 8 further on, in the order of P's
        typedef uint32_t u2_t __attribute__((ext_vector_type(2)));
        const u2_t x = __builtin_bit_cast(u2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                    (lds_s16x4_t *)&lv[va[d] + 16 * s * (HD * 2)]));
        const u2_t y = __builtin_bit_cast(u2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                    (lds_s16x4_t *)&lv[va[d] + (16 * s + 8) * (HD * 2)]));
        uint4 A = make_uint4(x[0], x[1], y[0], y[1]);
        uint32_t big = 0;                                  // the largest exponents of its halves
        if (MASK) {
          typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
          const uint32_t ee = EXP | EXP << 16;
          big = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(
              __builtin_elementwise_max(__builtin_bit_cast(u16x2, A.x & ee), __builtin_bit_cast(u16x2, A.y & ee)),
              __builtin_elementwise_max(__builtin_bit_cast(u16x2, A.z & ee), __builtin_bit_cast(u16x2, A.w & ee))));
        }
        if (MASK && __builtin_amdgcn_ballot_w64((big & 0xffffu) == EXP || big >> 16 == EXP)) {   // wave-uniform
          // A zero p times a V that is not finite is NaN: such values leave the product
          // and come back as +inf, -inf or (both) NaN in the columns where one has a p
          // above zero.
          uint32_t w[4] = {A.x, A.y, A.z, A.w};
#pragma unroll 1
          for (int sign = 0; sign < 2; sign++) {
            const uint32_t one = XT == GX_BF16 ? 0x3f80u : 0x3c00u, other = sign ? EXP : EXP | 0x8000u;
            uint32_t t[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
              const uint32_t e = w[i] & 0xffffu, o = w[i] >> 16;
              t[i] = ((e & EXP) == EXP && e != other ? one : 0u) | ((o & EXP) == EXP && o != other ? one << 16 : 0u);
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
        acc[d] = mfma32<XT>(A, B, acc[d]);
      }
    }
  };
  // Steps overlap: while a step's scores go through the exponent the next one's are
  // multiplied (K runs a step ahead of V), and while its values are multiplied the
  // next one's scores are searched for their maximum.  First the steps that every
  // column of the block sees whole, two at a time, then (from the first page that is
  // none, or the first position of the tile) the others.
  int32_t i0 = ids(0), i1 = ids(1), i2 = ids(2);           // page ids of steps j, j + 1, j + 2
  Sc S0, S1;
  if (nt) {
    load_k(i0, 0, lk0);
    store_k(lk0);
    load_v(i0, 0, lv0);
    store_v(lv0);
    load_k(i1, 1, lk1);
    store_k(lk1);
  }
  arrive();
  int j = 0;
  auto holes_of = [&](int32_t id) {
    uint32_t o = 0;
#pragma unroll
    for (int g = 0; g < 4; g++) o |= (uint32_t)__builtin_amdgcn_readlane(id, g) >> 31 << g;
    return o;
  };
  auto full = [&](int32_t id, int j) { return r0 + PP_STEP * (j + 1) <= min(all, r1) && holes_of(id) == 0; };
  auto step = [&](auto masked, Sc &S, Sc &N, char *k0, char *k1, char *v0, char *v1) {
    constexpr bool MASK = decltype(masked)::value;
    const int32_t rr = r0 + PP_STEP * j;
    const bool seen = !MASK || rr < whi, seen1 = !MASK || rr + PP_STEP < whi;   // wave-uniform
    uint32_t pk[2][8];
    load_k(i2, j + 2, k0);
    load_v(i1, j + 1, v1);
    const int32_t i3 = ids(j + 3);
    __builtin_amdgcn_sched_barrier(0);
    if (seen1) scores(k1, N);
    if (seen) expo(S, pk);
    if (!MASK) {                                           // pieces of K three ahead of their products, exponents between
      __builtin_amdgcn_sched_group_barrier(0x100, 3, 0);
#pragma unroll
      for (int q = 0; q < 2 * KS; q++) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, 32 / KS, 0);
        __builtin_amdgcn_sched_group_barrier(0x400, 16 / KS, 0);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    store_k(k0);
    __builtin_amdgcn_sched_barrier(0);
    float mx = -INFINITY;
    if (seen) mix(masked, v0, pk);
    if (seen1) mx = top(masked, j + 1, MASK ? holes_of(i1) : 0, N);
    if (!MASK) {
      __builtin_amdgcn_sched_group_barrier(0x100, 6, 0);
#pragma unroll
      for (int q = 0; q < 4 * DB; q++) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    store_v(v1);
    if (seen1) move(mx);
    arrive();
    i0 = i1;
    i1 = i2;
    i2 = i3;
    j++;
  };
  if (nt) {
    scores(lk0, S0);
    move(top(pg_const<true>{}, 0, holes_of(i0), S0));
  }
  while (j + 2 < nt && full(i0, j) && full(i1, j + 1) && full(i2, j + 2)) {
    step(pg_const<false>{}, S0, S1, lk0, lk1, lv0, lv1);
    step(pg_const<false>{}, S1, S0, lk1, lk0, lv1, lv0);
  }
  while (j < nt) {
    step(pg_const<true>{}, S0, S1, lk0, lk1, lv0, lv1);
    if (j < nt) step(pg_const<true>{}, S1, S0, lk1, lk0, lv1, lv0);
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
    float *pp = a.ws + (((uint64_t)kvh * pl.slots + u.u) * PP_COLS + 32 * wv + n) * (HD + 4);
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
