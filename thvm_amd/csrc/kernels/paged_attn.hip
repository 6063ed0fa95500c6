// paged_attn.hip -- attention of a ragged batch over a paged cache.
//
// out = sum_j softmax_j(scale q.k_j) v_j over the cache rows j <= p that have a
// page, for every row (position p of its sequence) and head; no such row: zeros.
// A wave takes one (row, head): 64 cache rows at a time, a lane's own row for the
// scores, a lane's own columns for the weighted sum.  Softmax statistics and sums
// are f32.
#include "paged_core.h"

#define PA_WAVES 4
#define LOG2E 1.4426950408889634f

template <int HD, int XT, int BITS>
__global__ __launch_bounds__(PA_WAVES * 64) void k_paged_rows(ThvmPagedArgs a) {
  typedef PgT<XT> P;
  constexpr int NC = HD / 64;                             // columns of a lane
  __shared__ float qs[PA_WAVES][HD];
  const uint32_t wv = threadIdx.x >> 6, lane = lane_id();
  const uint32_t unit = __builtin_amdgcn_readfirstlane(blockIdx.x * PA_WAVES + wv), row = unit / a.H, h = unit % a.H;
  if (row >= a.n) return;
  const uint32_t s = pg_seq_of(a, row);
  if (s >= a.b) return;
  const PgSeq sq = pg_seq(&a, s);
  if ((int32_t)row < sq.r0 || (int32_t)row >= sq.r1 || (uint32_t)(sq.r1 - sq.r0) > a.t) return;
  const int32_t pos = sq.len - (sq.r1 - (int32_t)row);
  const int32_t lim = min(pos + 1, (int32_t)(a.maxpages * a.page));
  const uint32_t kvh = h / (a.H / a.Hkv);
  const uint16_t *q = (const uint16_t *)a.q + ((uint64_t)row * a.H + h) * HD;
  for (uint32_t d = lane; d < HD; d += 64) qs[wv][d] = P::lo(q[d]) * a.scale * LOG2E;
  __builtin_amdgcn_wave_barrier();                        // a wave's own LDS accesses stay in order
  float m = -INFINITY, l = 0.0f, acc[NC] = {};
  for (int32_t j0 = 0; j0 < lim; j0 += 64) {
    const int32_t j = j0 + (int32_t)lane;
    const int32_t id = j < lim ? pg_page(&a, s, j) : -1;
    const uint64_t blk = id >= 0 ? pg_block(&a, id, kvh) : 0;
    const uint32_t slot = (uint32_t)j & (a.page - 1);
    float sc = -INFINITY;
    if (id >= 0) {
      sc = 0.0f;
      const char *kb = (const char *)a.kpages + blk;
      for (int d = 0; d < HD; d += 8) {
        uint4 w;
        if (BITS == 16) {
          w = ld16(kb + (slot * HD + d) * 2);
        } else {
          const uint32_t c = *(const uint32_t *)(kb + slot * (HD / 2) + d / 2);
          const float f = e8m0_f((uint8_t)kb[a.page * (HD / 2) + slot * (HD / 32) + d / 32]);
          w = make_uint4(fp4x2<XT, 0>(c, f), fp4x2<XT, 1>(c, f), fp4x2<XT, 2>(c, f), fp4x2<XT, 3>(c, f));
        }
        const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; i++) sc += P::lo(ww[i]) * qs[wv][d + 2 * i] + P::hi(ww[i]) * qs[wv][d + 2 * i + 1];
      }
    }
    const float mn = fmaxf(m, wave_max(sc));
    const float f = m == -INFINITY ? 0.0f : exp2f(m - mn), p = id < 0 ? 0.0f : exp2f(sc - mn);
    l = l * f + wave_sum(p);
    m = mn;
#pragma unroll
    for (int c = 0; c < NC; c++) acc[c] *= f;
    for (int r = 0; r < 64; r++) {
      const int32_t rid = __builtin_amdgcn_readlane(id, r);
      if (rid < 0) continue;
      const float pr = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(p), r));
      const char *vb = (const char *)a.vpages + pg_block(&a, rid, kvh);
      const uint32_t rs = (uint32_t)(j0 + r) & (a.page - 1);
#pragma unroll
      for (int c = 0; c < NC; c++) {
        const uint32_t d = lane + 64 * c;
        float x;
        if (BITS == 16) {
          x = P::lo(((const uint16_t *)vb)[rs * HD + d]);
        } else {
          const uint32_t two = fp4x2<XT, 0>((uint8_t)vb[rs * (HD / 2) + d / 2],
                                            e8m0_f((uint8_t)vb[a.page * (HD / 2) + rs * (HD / 32) + d / 32]));
          x = d & 1 ? P::hi(two) : P::lo(two);
        }
        acc[c] += pr * x;
      }
    }
  }
  uint16_t *o = (uint16_t *)a.out + ((uint64_t)row * a.H + h) * HD;
#pragma unroll
  for (int c = 0; c < NC; c++) o[lane + 64 * c] = (uint16_t)P::pk(l != 0.0f ? acc[c] / l : 0.0f, 0.0f);
}

extern "C" uint64_t thvm_k_attn_paged_ws(const ThvmPagedArgs *a) {
  (void)a;
  return 16;
}

typedef void (*paged_fn)(ThvmPagedArgs);
extern "C" int thvm_k_attn_paged(const ThvmPagedArgs *a, hipStream_t s, char *err, int errlen) {
  if (pg_check(a, PG_ATTN, err, errlen)) return -1;
  const int bf = a->dt == THVM_DT_BF16, b16 = a->bits == 16;
  paged_fn f = a->hd == 128 ? (bf ? (b16 ? k_paged_rows<128, GX_BF16, 16> : k_paged_rows<128, GX_BF16, 4>)
                                  : (b16 ? k_paged_rows<128, GX_F16, 16> : k_paged_rows<128, GX_F16, 4>))
                            : (bf ? (b16 ? k_paged_rows<64, GX_BF16, 16> : k_paged_rows<64, GX_BF16, 4>)
                                  : (b16 ? k_paged_rows<64, GX_F16, 16> : k_paged_rows<64, GX_F16, 4>));
  const uint64_t units = (uint64_t)a->n * a->H;
  thvm_launch(true, true, f, dim3((uint32_t)((units + PA_WAVES - 1) / PA_WAVES)), dim3(PA_WAVES * 64), 0, s, *a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) { snprintf(err, errlen, "attn_paged launch: %s", hipGetErrorString(e)); return -1; }
  return 0;
}
