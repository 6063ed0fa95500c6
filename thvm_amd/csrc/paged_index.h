/* paged_index.h -- which rows a sequence has and where a position lies, for the
 * device and, compiled as C, for a host that checks it.
 *
 * rows, len and table are device data that no host check has seen, so every
 * value is brought into its range before it is used: row offsets into [0, n],
 * lengths into [0, 2^30], page ids are followed only inside [0, npages). */
#ifndef THVM_PAGED_INDEX_H
#define THVM_PAGED_INDEX_H

#include "paged_check.h"

#ifdef __HIPCC__
#define PG_FN static __host__ __device__ __forceinline__
#else
#define PG_FN static inline
#endif

PG_FN int32_t pg_clamp(int32_t v, int32_t lo, int32_t hi) { return v < lo ? lo : v > hi ? hi : v; }

/* the rows [r0, r1) of sequence s and its length */
typedef struct PgSeq { int32_t r0, r1, len; } PgSeq;
PG_FN PgSeq pg_seq(const ThvmPagedArgs *a, uint32_t s) {
  PgSeq q;
  const int32_t n = (int32_t)a->n;
  if (a->rows) {
    q.r0 = pg_clamp(a->rows[s], 0, n);
    q.r1 = pg_clamp(a->rows[s + 1], q.r0, n);
  } else {
    q.r0 = (int32_t)(s * (a->n / a->b));
    q.r1 = q.r0 + (int32_t)(a->n / a->b);
  }
  q.len = pg_clamp(a->len[s], 0, (int32_t)PG_MAX_POS);
  return q;
}

/* page id of a position of sequence s, -1: none */
PG_FN int32_t pg_page(const ThvmPagedArgs *a, uint32_t s, int32_t pos) {
  const uint32_t lg = (uint32_t)__builtin_ctz(a->page);
  if (pos < 0 || (uint32_t)pos >> lg >= a->maxpages) return -1;
  const int32_t id = a->table[(uint64_t)s * a->maxpages + ((uint32_t)pos >> lg)];
  return (uint32_t)id < a->npages ? id : -1;
}

/* bytes of one head's block of a page, and where page id's block of a head begins */
PG_FN uint32_t pg_block_bytes(const ThvmPagedArgs *a) {
  return a->page * (a->bits == 4 ? a->hd / 2 + a->hd / 32 : a->hd * 2);
}
PG_FN uint64_t pg_block(const ThvmPagedArgs *a, int32_t id, uint32_t kvh) {
  return ((uint64_t)id * a->Hkv + kvh) * pg_block_bytes(a);
}

#endif
