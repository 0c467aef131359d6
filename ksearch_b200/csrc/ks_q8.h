// Shared by the translation units of the paged 8-bit cache (ks_pages.cu, ks_kv_q8.cu, ks_sdpa_q8.cu): plan layout and argument checks.
#pragma once
#include "ks_internal.h"

// Where the parts of a plan start, in words.
struct ks_plan_layout {
  unsigned row_start, row_seq, row_pos, row_slot, jobs, n_jobs;
};
static inline ks_plan_layout ks_plan_parts(size_t n_seqs, size_t max_rows, size_t page) {
  const size_t starts = (n_seqs + 1 + 3) & ~size_t(3), rows = (max_rows + 3) & ~size_t(3);
  ks_plan_layout l;
  l.row_start = KS_PAGES_PLAN_HEADER;
  l.row_seq = (unsigned)(l.row_start + starts);
  l.row_pos = (unsigned)(l.row_seq + rows);
  l.row_slot = (unsigned)(l.row_pos + rows);
  l.jobs = (unsigned)(l.row_slot + rows);
  l.n_jobs = (unsigned)(max_rows / page + 2 * n_seqs);  // a sequence of r rows touches r / page + 2 pages at most
  return l;
}
static inline bool ks_page_ok(size_t page) { return page == 16 || page == 32 || page == 64 || page == 128; }
static inline bool ks_aligned(const ks_buf* b, size_t to) { return ((uintptr_t)b->dptr & (to - 1)) == 0; }

// Behind the last check of an entry point: is there a device to launch on?
#define KS_REQUIRE_DEVICE(ctx, who) \
  do {                              \
    if ((ctx)->device < 0) return ks_fail((ctx), KS_ERR_UNSUPPORTED, "%s: no device", (who)); \
  } while (0)

int ks_check_tables(ks_ctx* ctx, const char* who, const ks_page_tables* t);                        // sizes and buffers
int ks_check_cache(ks_ctx* ctx, const char* who, const ks_q8_cache* c, const ks_page_tables* t);   // the same; t (may be null) has the same pool
