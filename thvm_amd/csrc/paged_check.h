/* paged_check.h -- what the paged-cache builtins accept (kv_append, kv_read,
 * attn_paged), in C without a device: the shapes and sizes a launch may rely
 * on.  Everything a kernel indexes by is bounded here or, where it comes from
 * device memory (rows, len, table), by the kernel itself. */
#ifndef THVM_PAGED_CHECK_H
#define THVM_PAGED_CHECK_H

#include <stdio.h>
#include "kern_api.h"

enum { PG_APPEND = 0, PG_READ = 1, PG_ATTN = 2 };
#define PG_MAX_SEQS 4096u
#define PG_MAX_ROWS (1u << 22)
#define PG_MAX_POS  (1u << 30)

/* bytes of a cache row of one head, and of one head's rows of a page */
static inline uint32_t pg_row_bytes(uint32_t hd, uint32_t bits) { return bits == 4 ? hd / 2 + hd / 32 : hd * 2; }
static inline uint64_t pg_pool_bytes(const ThvmPagedArgs *a) {
  return (uint64_t)a->npages * a->Hkv * a->page * pg_row_bytes(a->hd, a->bits);
}

static inline int pg_check(const ThvmPagedArgs *a, int op, char *err, int errlen) {
#define PG_REFUSE(...) do { snprintf(err, errlen, __VA_ARGS__); return -1; } while (0)
  if (a->dt != THVM_DT_BF16 && a->dt != THVM_DT_FP16) PG_REFUSE("dt must be bf16 or fp16 (dt=%u)", a->dt);
  if (a->bits != 16 && a->bits != 4) PG_REFUSE("bits must be 16 or 4 (bits=%u)", a->bits);
  if (a->hd != 64 && a->hd != 128) PG_REFUSE("hd must be 64 or 128 (hd=%u)", a->hd);
  if (a->page < 16 || a->page > 1024 || (a->page & (a->page - 1)))
    PG_REFUSE("page must be a power of two from 16 to 1024 (page=%u)", a->page);
  if (a->b == 0 || a->b > PG_MAX_SEQS || a->n == 0 || a->n > PG_MAX_ROWS)
    PG_REFUSE("b from 1 to %u sequences, n from 1 to %u rows (b=%u n=%u)", PG_MAX_SEQS, PG_MAX_ROWS, a->b, a->n);
  if (a->ragged > 1) PG_REFUSE("ragged must be 0 or 1 (ragged=%u)", a->ragged);
  if (!a->ragged && a->n % a->b) PG_REFUSE("without ragged=1 b must divide n (b=%u n=%u)", a->b, a->n);
  if (a->maxpages == 0 || (uint64_t)a->maxpages * a->page > PG_MAX_POS || a->npages == 0 || a->npages > 0x7fffffffu)
    PG_REFUSE("maxpages x page from 1 to 2^30 positions, npages below 2^31 (maxpages=%u page=%u npages=%u)", a->maxpages,
              a->page, a->npages);
  if (a->Hkv == 0 || a->Hkv > 1024) PG_REFUSE("hkv from 1 to 1024 (hkv=%u)", a->Hkv);
  if (op != PG_READ && (a->H == 0 || a->H > 1024 || a->H % a->Hkv))
    PG_REFUSE("h from 1 to 1024, a multiple of hkv (h=%u hkv=%u)", a->H, a->Hkv);
  /* (grids stay below 2^32 threads) */
  if ((uint64_t)a->b * a->Hkv > (1u << 19)) PG_REFUSE("b x hkv of more than 2^19 (b=%u hkv=%u)", a->b, a->Hkv);
  if ((uint64_t)a->n * (op == PG_READ ? 2 * a->Hkv : a->H + 2 * a->Hkv) > (1u << 25))
    PG_REFUSE("more than 2^25 heads in all rows (n=%u)", a->n);
  if (op == PG_APPEND) {
    if (a->rope > 2 || a->norm > 1) PG_REFUSE("rope must be 0, 1 or 2 and norm 0 or 1 (rope=%u norm=%u)", a->rope, a->norm);
    if (a->norm && !(a->eps >= 0.0f && a->eps < 1e30f)) PG_REFUSE("eps must be a finite number >= 0");
    if (a->ldx < (a->H + 2 * a->Hkv) * a->hd || a->ldx % 8)
      PG_REFUSE("ldx must hold (h + 2 hkv) hd values and be a multiple of 8 (ldx=%u)", a->ldx);
  }
  if (op == PG_ATTN) {
    if (!(a->scale > -1e30f && a->scale < 1e30f)) PG_REFUSE("scale must be finite");
    if (a->t == 0 || (!a->ragged && a->t < a->n / a->b)) PG_REFUSE("t=%u rows a sequence do not hold n / b", a->t);
  }
  return 0;
#undef PG_REFUSE
}

#endif
