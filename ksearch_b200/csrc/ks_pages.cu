// Pages of a paged cache handed out on the GPU: tables, lengths, the stack of free pages and the plan of a step's rows.
//
// A step is integer arithmetic on three exclusive sums over the sequences (rows, new pages, touched pages) and one record per row, so it
// is bound by latency: one trip for lengths and counts, the sums, one trip for a row's page, the stores.  Every block makes the sums
// for itself and takes rows; nothing that a block reads is written by another, except lengths and the stack's count, which the block that
// arrived last at a counter writes in the end (every block arrives when it has read them; nobody waits for what the counter says).  256 sequences and some 16000 rows: 5 us, with a trim in
// front 9.4; an arrival in front of the rows, or a cluster's barrier in its place, 11.
#include "ks_q8.h"

namespace {

struct TablesArgs {
  unsigned n_seqs, max_blocks, n_pages, page_log, max_rows;
  int *lens, *tables, *free_pages, *plan;
  ks_plan_layout at;
  unsigned *bad, *arrived;
};

// Exclusive sums of three counts over the block's threads (a multiple of 32, up to 1024); totals in tot.
__device__ __forceinline__ void scan3(unsigned (&v)[3], unsigned (&tot)[3], unsigned (*red)[3]) {
  const unsigned lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, nwarp = blockDim.x >> 5;
  unsigned inc[3];
#pragma unroll
  for (int k = 0; k < 3; k++) {
    inc[k] = v[k];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned up = __shfl_up_sync(0xffffffffu, inc[k], o);
      if (lane >= (unsigned)o) inc[k] += up;
    }
    if (lane == 31u) red[warp][k] = inc[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 3; k++) {  // every warp adds up the warps' totals
    unsigned all = lane < nwarp ? red[lane][k] : 0u, before = lane < warp ? all : 0u;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      all += __shfl_xor_sync(0xffffffffu, all, o);
      before += __shfl_xor_sync(0xffffffffu, before, o);
    }
    v[k] = before + inc[k] - v[k];
    tot[k] = all;
  }
}

// A thread takes four neighbouring rows: one search for the sequence of the first, 16-byte stores.
__global__ void __launch_bounds__(1024) pages_step_kernel(const TablesArgs a, const int* n_new) {
  __shared__ unsigned red[32][3];
  __shared__ unsigned first_row[KS_PAGES_MAX_SEQS + 1], first_page[KS_PAGES_MAX_SEQS], first_job[KS_PAGES_MAX_SEQS];
  __shared__ int len_of[KS_PAGES_MAX_SEQS], worst_s;
  __shared__ bool last;
  const unsigned tid = threadIdx.x, page = 1u << a.page_log, cap = a.max_blocks << a.page_log;
  if (tid == 0) worst_s = 0;
  ks_pdl_entry();
  const int count = a.free_pages[0];
  int len = 0, add = 0;
  if (tid < a.n_seqs) {
    len = a.lens[tid];
    add = n_new[tid];
  }
  // the highest status that holds; counts out of range are nothing in the sums
  int status = 0;
  if (len < 0 || (unsigned)len > cap || add < 0) status = KS_PLAN_BAD_LENGTH;
  else if ((unsigned)add > a.max_rows) status = KS_PLAN_TOO_MANY_ROWS;
  else if ((unsigned)add > cap - (unsigned)len) status = KS_PLAN_TABLE_FULL;
  if (status >= KS_PLAN_TOO_MANY_ROWS) add = 0;  // (a sequence that would outgrow its table still counts its rows)
  if (status == KS_PLAN_BAD_LENGTH) len = 0;
  const unsigned after = (unsigned)len + (unsigned)add, held = ((unsigned)len + page - 1u) >> a.page_log;
  unsigned v[3] = {(unsigned)add, ((after + page - 1u) >> a.page_log) - held, add ? ((after - 1u) >> a.page_log) - ((unsigned)len >> a.page_log) + 1u : 0u}, tot[3];
  __syncthreads();
  if (status) atomicMax(&worst_s, status);
  scan3(v, tot, red);  // (a barrier inside: worst_s is complete behind it)
  int worst = worst_s;
  if (worst < KS_PLAN_TOO_MANY_ROWS && tot[0] > a.max_rows) worst = KS_PLAN_TOO_MANY_ROWS;
  if (worst == 0 && (count < 0 || (unsigned)count > a.n_pages || tot[1] > (unsigned)count)) worst = KS_PLAN_NO_PAGES;
  const unsigned rows = worst ? 0u : tot[0], jobs = worst ? 0u : tot[2];
  if (tid < a.n_seqs) {
    first_row[tid] = v[0];
    first_page[tid] = v[1];
    first_job[tid] = v[2];
    len_of[tid] = len;
  }
  if (tid == 0) first_row[a.n_seqs] = rows;
  __syncthreads();
  unsigned before_me = 0;  // thread 0: blocks that have arrived, once all of this one have read lengths and count
  if (tid == 0 && gridDim.x > 1u) {
    __threadfence();
    before_me = atomicAdd(a.arrived, 1u);
  }
  const unsigned step = gridDim.x * blockDim.x, quads = (a.max_rows + 3u) >> 2, me = blockIdx.x * blockDim.x + tid;
  int4 *seqs = reinterpret_cast<int4*>(a.plan + a.at.row_seq), *poss = reinterpret_cast<int4*>(a.plan + a.at.row_pos), *slots = reinterpret_cast<int4*>(a.plan + a.at.row_slot);
  for (unsigned q = me; q < quads; q += step) {
    int seq[4], pos[4], slot[4];
    unsigned lo = 0;
    if (4u * q < rows) {
      unsigned hi = a.n_seqs;  // the last sequence that starts at row 4 q or before
      while (hi - lo > 1u) {
        const unsigned mid = (lo + hi) >> 1;
        if (first_row[mid] <= 4u * q) lo = mid;
        else hi = mid;
      }
    }
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const unsigned r = 4u * q + k;
      seq[k] = pos[k] = slot[k] = -1;
      if (r >= rows) continue;
      while (first_row[lo + 1u] <= r) lo++;
      const unsigned l0 = (unsigned)len_of[lo], p = l0 + (r - first_row[lo]), b = p >> a.page_log, had = (l0 + page - 1u) >> a.page_log, off = p & (page - 1u);
      int id;
      if (b >= had) {
        id = a.free_pages[(unsigned)count - first_page[lo] - (b - had)];
        if (off == 0u) a.tables[(size_t)lo * a.max_blocks + b] = id;
      } else {
        id = a.tables[(size_t)lo * a.max_blocks + b];
      }
      seq[k] = (int)lo;
      pos[k] = (int)p;
      if (id >= 0 && (unsigned)id < a.n_pages) slot[k] = (int)(((unsigned)id << a.page_log) + off);
      else atomicOr(a.bad, KS_BAD_PAGE);
      if (r == first_row[lo] || off == 0u)
        reinterpret_cast<int4*>(a.plan + a.at.jobs)[first_job[lo] + (b - (l0 >> a.page_log))] = make_int4((int)r, (int)min(page - off, first_row[lo + 1u] - r), slot[k], (int)p);
    }
    seqs[q] = make_int4(seq[0], seq[1], seq[2], seq[3]);
    poss[q] = make_int4(pos[0], pos[1], pos[2], pos[3]);
    slots[q] = make_int4(slot[0], slot[1], slot[2], slot[3]);
  }
  for (unsigned j = jobs + me; j < a.at.n_jobs; j += step) reinterpret_cast<int4*>(a.plan + a.at.jobs)[j] = make_int4(-1, -1, -1, -1);
  if (blockIdx.x == 0) {
    if (tid < a.n_seqs) a.plan[a.at.row_start + tid] = worst ? 0 : (int)v[0];
    if (tid < KS_PAGES_PLAN_HEADER) {
      const int head[4] = {worst, (int)rows, (int)jobs, worst ? count : count - (int)tot[1]};
      a.plan[tid] = tid < 4u ? head[tid] : 0;
    }
    if (tid == 0) a.plan[a.at.row_start + a.n_seqs] = (int)rows;
  }
  if (tid == 0) last = before_me == gridDim.x - 1u;
  __syncthreads();
  if (last) {
    if (tid < a.n_seqs && !worst) a.lens[tid] = (int)after;
    if (tid == 0) {
      if (!worst) a.free_pages[0] = count - (int)tot[1];
      if (gridDim.x > 1u) *a.arrived = 0u;
    }
  }
}

// One block: the sum over the sequences, then one page per thread and step.  Ids that no page has stay out of the stack.
__global__ void __launch_bounds__(1024) pages_trim_kernel(const TablesArgs a, const int* keep) {
  __shared__ unsigned red[32][3];
  __shared__ unsigned first[KS_PAGES_MAX_SEQS], from[KS_PAGES_MAX_SEQS];
  ks_pdl_entry();
  const unsigned tid = threadIdx.x, page = 1u << a.page_log, cap = a.max_blocks << a.page_log;
  const int count = a.free_pages[0];
  int len = 0, to = -1;
  if (tid < a.n_seqs) {
    len = a.lens[tid];
    to = keep[tid];
  }
  const bool fine = len >= 0 && (unsigned)len <= cap, cut = fine && to >= 0 && to < len;
  if (!fine) atomicOr(a.bad, KS_BAD_ROWS);
  const unsigned old = fine ? ((unsigned)len + page - 1u) >> a.page_log : 0u, kept = cut ? ((unsigned)to + page - 1u) >> a.page_log : old;
  unsigned v[3] = {old - kept, 0u, 0u}, tot[3];
  scan3(v, tot, red);
  if (tid < a.n_seqs) {
    first[tid] = v[0];
    from[tid] = kept;
  }
  __syncthreads();
  if (count < 0 || (unsigned)count > a.n_pages || tot[0] > a.n_pages - (unsigned)count) {  // more pages than there are: nothing moves
    if (tid == 0) atomicOr(a.bad, KS_BAD_STACK);
    return;
  }
  if (cut) a.lens[tid] = to;
  bool bad = false;
  for (unsigned k = tid; k < tot[0]; k += blockDim.x) {
    unsigned lo = 0, hi = a.n_seqs;
    while (hi - lo > 1u) {
      const unsigned mid = (lo + hi) >> 1;
      if (first[mid] <= k) lo = mid;
      else hi = mid;
    }
    int* entry = a.tables + (size_t)lo * a.max_blocks + from[lo] + (k - first[lo]);
    const int id = *entry;
    bad |= (unsigned)id >= a.n_pages;
    a.free_pages[(unsigned)count + tot[0] - k] = id;
    *entry = -1;
  }
  unsigned back = tot[0];
  if (__syncthreads_or(bad)) {  // ids that no page has leave the stack again: the others move down, in their order
    if (tid == 0) atomicOr(a.bad, KS_BAD_PAGE);
    back = 0;
    for (unsigned k0 = 0; k0 < tot[0]; k0 += blockDim.x) {
      const int id = k0 + tid < tot[0] ? a.free_pages[(unsigned)count + 1u + k0 + tid] : -1;
      const bool good = (unsigned)id < a.n_pages;
      unsigned w[3] = {good, 0u, 0u}, n[3];
      scan3(w, n, red);  // (a barrier inside: this round's ids have been read, and no later one lies where they go)
      if (good) a.free_pages[(unsigned)count + 1u + back + w[0]] = id;
      back += n[0];
      __syncthreads();
    }
  }
  if (tid == 0) a.free_pages[0] = count + (int)back;
}

__global__ void __launch_bounds__(256) pages_reset_kernel(const TablesArgs a, size_t n_plan) {
  ks_pdl_entry();
  const size_t step = (size_t)gridDim.x * blockDim.x, i0 = (size_t)blockIdx.x * blockDim.x + threadIdx.x;
  for (size_t i = i0; i < a.n_seqs; i += step) a.lens[i] = 0;
  for (size_t i = i0; i < (size_t)a.n_seqs * a.max_blocks; i += step) a.tables[i] = -1;
  for (size_t i = i0; i <= a.n_pages; i += step) a.free_pages[i] = i ? (int)(a.n_pages - i) : (int)a.n_pages;
  for (size_t i = i0; i < n_plan; i += step) a.plan[i] = i >= a.at.row_seq ? -1 : i == 3 ? (int)a.n_pages : 0;
}

TablesArgs args_of(ks_ctx* ctx, const ks_page_tables* t) {
  TablesArgs a;
  a.n_seqs = (unsigned)t->n_seqs;
  a.max_blocks = (unsigned)t->max_blocks;
  a.n_pages = (unsigned)t->n_pages;
  a.page_log = (unsigned)__builtin_ctzll(t->page);
  a.max_rows = (unsigned)t->max_rows;
  a.lens = (int*)t->lens->dptr;
  a.tables = (int*)t->tables->dptr;
  a.free_pages = (int*)t->free_pages->dptr;
  a.plan = (int*)t->plan->dptr;
  a.at = ks_plan_parts(t->n_seqs, t->max_rows, t->page);
  a.bad = (unsigned*)ctx->ws + KS_WS_INDEX_WORD;
  a.arrived = (unsigned*)ctx->ws + KS_WS_STEP_WORD;
  return a;
}
unsigned round32(size_t n) { return (unsigned)((n + 31) & ~size_t(31)); }

bool sizes_ok(size_t n_seqs, size_t max_rows, size_t page) {
  return n_seqs >= 1 && n_seqs <= KS_PAGES_MAX_SEQS && max_rows >= 1 && max_rows <= (1u << 20) && ks_page_ok(page);
}

}  // namespace

int ks_check_tables(ks_ctx* ctx, const char* who, const ks_page_tables* t) {
  KS_REQUIRE(ctx, t, "%s: null page tables", who);
  KS_REQUIRE(ctx, ks_page_ok(t->page), "%s: pages of %zu positions not supported (16, 32, 64, 128)", who, t->page);
  KS_REQUIRE(ctx, t->n_seqs >= 1 && t->n_seqs <= KS_PAGES_MAX_SEQS, "%s: n_seqs=%zu outside 1..%d", who, t->n_seqs, KS_PAGES_MAX_SEQS);
  KS_REQUIRE(ctx, t->max_rows >= 1 && t->max_rows <= (1u << 20), "%s: max_rows=%zu outside 1..2^20", who, t->max_rows);
  const size_t most = 0x7FFFFFFFu / t->page;
  KS_REQUIRE(ctx, t->n_pages >= 1 && t->n_pages <= most && t->max_blocks >= 1 && t->max_blocks <= most / 2, "%s: %zu pages, %zu to a sequence: at least one, below 2^31 positions and 2^30", who,
             t->n_pages, t->max_blocks);
  KS_REQUIRE(ctx, t->n_seqs * t->max_blocks < (size_t(1) << 31), "%s: tables of %zu x %zu entries: below 2^31", who, t->n_seqs, t->max_blocks);  // (counts of pages are 32 bits)
  KS_REQUIRE(ctx, ks_fits(t->lens, 0, t->n_seqs * 4) && ks_fits(t->tables, 0, t->n_seqs * t->max_blocks * 4), "%s: lens or tables buffer too small", who);
  KS_REQUIRE(ctx, ks_fits(t->free_pages, 0, (1 + t->n_pages) * 4), "%s: free_pages buffer too small (1 + n_pages words)", who);
  KS_REQUIRE(ctx, ks_fits(t->plan, 0, ks_pages_plan_ints(t->n_seqs, t->max_rows, t->page) * 4), "%s: plan buffer too small", who);
  KS_REQUIRE(ctx, ks_aligned(t->lens, 4) && ks_aligned(t->tables, 4) && ks_aligned(t->free_pages, 4) && ks_aligned(t->plan, 16), "%s: tables must start on 4 bytes, the plan on 16", who);
  return KS_OK;
}

extern "C" {

size_t ks_pages_plan_offset(size_t n_seqs, size_t max_rows, size_t page, int part) {
  if (!sizes_ok(n_seqs, max_rows, page)) return 0;
  const ks_plan_layout l = ks_plan_parts(n_seqs, max_rows, page);
  const size_t at[6] = {l.row_start, l.row_seq, l.row_pos, l.row_slot, l.jobs, (size_t)l.jobs + 4 * l.n_jobs};
  return part >= KS_PLAN_ROW_START && part <= KS_PLAN_END ? at[part] : 0;
}
size_t ks_pages_plan_ints(size_t n_seqs, size_t max_rows, size_t page) { return ks_pages_plan_offset(n_seqs, max_rows, page, KS_PLAN_END); }

int ks_pages_reset(ks_ctx* ctx, const ks_page_tables* t) {
  if (!ctx) return KS_ERR_INVALID;
  int rc = ks_check_tables(ctx, "pages_reset", t);
  if (rc) return rc;
  KS_REQUIRE_DEVICE(ctx, "pages_reset");
  ks_on_device on(ctx);
  KS_LAUNCH(ctx, pages_reset_kernel, (unsigned)ctx->sm_count, 256, 0, args_of(ctx, t), ks_pages_plan_ints(t->n_seqs, t->max_rows, t->page));
  return ks_after_launch(ctx, "pages_reset");
}

int ks_pages_step(ks_ctx* ctx, const ks_page_tables* t, const ks_buf* n_new) {
  if (!ctx) return KS_ERR_INVALID;
  int rc = ks_check_tables(ctx, "pages_step", t);
  if (rc) return rc;
  KS_REQUIRE(ctx, ks_fits(n_new, 0, t->n_seqs * 4) && ks_aligned(n_new, 4), "pages_step: n_new buffer too small or not on 4 bytes");
  KS_REQUIRE_DEVICE(ctx, "pages_step");
  ks_on_device on(ctx);
  // A thread per sequence, and small blocks only where one of them holds all rows.  128 / 256 threads, with a trim in front: 8 rows of 8 sequences 4.37 / 4.45 us,
  // 512 of 8 4.73 / 4.83, 513 of 8 (two blocks of 128) 5.46 / 4.83, 128 or 512 of 128 4.87 / 4.87 and 4.59 / 4.59, 16000 of 128 8.61 / 8.52.
  const unsigned threads = round32(t->n_seqs) < 256u ? (t->max_rows <= 512 && t->n_seqs <= 128 ? 128 : 256) : round32(t->n_seqs);
  const size_t blocks = (t->max_rows + 4 * threads - 1) / (4 * threads), most = 64;
  KS_LAUNCH(ctx, pages_step_kernel, (unsigned)(blocks < most ? blocks : most), threads, 0, args_of(ctx, t), (const int*)n_new->dptr);
  return ks_after_launch(ctx, "pages_step");
}

int ks_pages_trim(ks_ctx* ctx, const ks_page_tables* t, const ks_buf* keep) {
  if (!ctx) return KS_ERR_INVALID;
  int rc = ks_check_tables(ctx, "pages_trim", t);
  if (rc) return rc;
  KS_REQUIRE(ctx, ks_fits(keep, 0, t->n_seqs * 4) && ks_aligned(keep, 4), "pages_trim: keep buffer too small or not on 4 bytes");
  KS_REQUIRE_DEVICE(ctx, "pages_trim");
  ks_on_device on(ctx);
  KS_LAUNCH(ctx, pages_trim_kernel, 1, round32(t->n_seqs) < 128u ? 128u : round32(t->n_seqs), 0, args_of(ctx, t), (const int*)keep->dptr);
  return ks_after_launch(ctx, "pages_trim");
}

}  // extern "C"
