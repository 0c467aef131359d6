// Attention of ragged rows (single tokens, drafts, prompt pieces) over a paged 8-bit cache.
//
// Row r of a sequence of `len` positions and `rows` rows sits at p = len - rows + r and sees positions max(0, p - window + 1) .. p:
//   s_j = scale q . k_j,   out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),   m = max_j s_j.
#include "ks_q8.h"
#include "ks_q8.cuh"

namespace {

struct SdpaArgs {
  const uint8_t *kc, *vc;
  const float *ks, *vs;
  const int *lens, *tables, *row_start;
  const void* q;
  void* out;
  float* tmp;
  unsigned *bad, *arrived;
  unsigned n_seqs, max_blocks, n_pages, page_log, max_rows, rows_most, n_q, n_kv, G, window;
  float scale;
};

// One warp per row and query head: 32 positions at a time, a lane a position for the scores and HD / 32 dims for the values.
template <int HD, typename T, bool FP8>
__global__ void __launch_bounds__(32) sdpa_q8_row_kernel(const SdpaArgs a) {
  constexpr int D = HD / 32;
  __shared__ float qs[HD];
  ks_pdl_entry();
  const unsigned lane = threadIdx.x, row = blockIdx.x, head = blockIdx.y, kvh = head / a.G, page = 1u << a.page_log;
  if (row >= (unsigned)max(a.row_start[a.n_seqs], 0)) return;
  unsigned lo = 0, hi = a.n_seqs;
  while (hi - lo > 1u) {
    const unsigned mid = (lo + hi) >> 1;
    if ((unsigned)a.row_start[mid] <= row) lo = mid;
    else hi = mid;
  }
  const int r0 = a.row_start[lo], rows = a.row_start[lo + 1] - r0, r = (int)row - r0;
  if (r < 0 || r >= rows || rows > (int)a.rows_most) {
    if (lane == 0) atomicOr(a.bad, KS_BAD_ROWS);
    return;
  }
  const int len = min(max(a.lens[lo], 0), (int)(a.max_blocks << a.page_log));
  const int end = len - rows + r + 1, begin = a.window && end > (int)a.window ? end - (int)a.window : 0;
  const T* q = (const T*)a.q + ((size_t)row * a.n_q + head) * HD;
  for (unsigned i = lane; i < HD; i += 32u) qs[i] = (float)q[i] * a.scale;
  __syncwarp();
  float m = -INFINITY, l = 0.0f, o[D];
#pragma unroll
  for (int d = 0; d < D; d++) o[d] = 0.0f;
  for (int base = begin; base < end; base += 32) {
    const int pos = base + (int)lane;
    float s = -INFINITY;
    size_t at = 0;
    float vs = 0.0f;
    if (pos < end) {
      const int id = a.tables[(size_t)lo * a.max_blocks + ((unsigned)pos >> a.page_log)];
      if (id < 0 || (unsigned)id >= a.n_pages) {
        atomicOr(a.bad, KS_BAD_PAGE);
      } else {
        const size_t block = (size_t)id * a.n_kv + kvh;
        at = ((block << a.page_log) + ((unsigned)pos & (page - 1u))) * HD;
        vs = q8_scale(a.vs[block]);
        float dot = 0.0f;
        for (int c = 0; c < HD; c += 4) {
          const uint32_t w = *reinterpret_cast<const uint32_t*>(a.kc + at + c);
          const float2 x = q8_decode2f<FP8>(w), y = q8_decode2f<FP8>(w >> 16);
          dot = fmaf(qs[c], x.x, fmaf(qs[c + 1], x.y, fmaf(qs[c + 2], y.x, fmaf(qs[c + 3], y.y, dot))));
        }
        s = dot * q8_scale(a.ks[block]);
      }
    }
    float mx = s;
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, k));
    mx = fmaxf(mx, m);
    if (mx == -INFINITY) continue;
    const float alpha = __expf(m - mx), p = __expf(s - mx);
    m = mx;
    l = l * alpha + q8_warp_sum(p);
#pragma unroll
    for (int d = 0; d < D; d++) o[d] *= alpha;
    for (int jj = 0; jj < 32; jj++) {
      const float w = __shfl_sync(0xffffffffu, p * vs, jj);
      const size_t from = __shfl_sync(0xffffffffu, at, jj);
      if (__shfl_sync(0xffffffffu, s, jj) == -INFINITY) continue;
#pragma unroll
      for (int d = 0; d < D; d++) o[d] = fmaf(w, q8_decode2f<FP8>(a.vc[from + lane * D + d]).x, o[d]);
    }
  }
  T* out = (T*)a.out + ((size_t)row * a.n_q + head) * HD + lane * D;
#pragma unroll
  for (int d = 0; d < D; d++) out[d] = (T)(l > 0.0f ? o[d] / l : 0.0f);
}

}  // namespace

extern "C" {

size_t ks_sdpa_paged_tmp_floats(const ks_ctx* ctx, const ks_q8_cache* c, const ks_page_tables* t, size_t n_q, size_t rows_most) {
  if (!ctx || !c || !t || !c->n_kv) return 0;
  (void)n_q;
  (void)rows_most;
  return 4;
}

int ks_sdpa_paged_q8(ks_ctx* ctx, const ks_q8_cache* c, const ks_page_tables* t, size_t n_q, size_t rows_most, size_t ctx_most, size_t window, float scale, ks_dtype act,
                     const ks_buf* q, ks_buf* tmp, ks_buf* out) {
  if (!ctx) return KS_ERR_INVALID;
  static const char who[] = "sdpa_paged_q8";
  int rc = ks_check_tables(ctx, who, t);
  if (!rc) rc = ks_check_cache(ctx, who, c, t);
  if (rc) return rc;
  KS_REQUIRE(ctx, ks_is_act(act), "%s: activation dtype must be F32 or F16", who);
  KS_REQUIRE(ctx, n_q >= 1 && n_q <= 65535 && n_q % c->n_kv == 0, "%s: n_q=%zu is not a multiple of n_kv=%zu, or above 65535", who, n_q, c->n_kv);
  const size_t G = n_q / c->n_kv;
  if (G > 64) return ks_fail(ctx, KS_ERR_UNSUPPORTED, "%s: n_q/n_kv = %zu not supported (1..64)", who, G);
  KS_REQUIRE(ctx, rows_most <= t->max_rows, "%s: rows_most=%zu above max_rows=%zu", who, rows_most, t->max_rows);
  KS_REQUIRE(ctx, window < (1u << 31), "%s: window=%zu out of range", who, window);
  KS_REQUIRE(ctx, scale - scale == 0.0f, "%s: scale is not finite", who);
  const size_t bytes = t->max_rows * n_q * c->hd * ks_act_bytes(act);
  KS_REQUIRE(ctx, ks_fits(q, 0, bytes) && ks_fits(out, 0, bytes), "%s: q/out buffer too small for %zu rows", who, t->max_rows);
  KS_REQUIRE(ctx, ks_aligned(q, 16) && ks_aligned(out, 16), "%s: q and out must start on 16 bytes", who);
  const uint8_t *qa = (const uint8_t*)q->dptr, *oa = (const uint8_t*)out->dptr;
  KS_REQUIRE(ctx, qa + bytes <= oa || oa + bytes <= qa, "%s: q and out overlap", who);
  KS_REQUIRE(ctx, ks_fits(tmp, 0, ks_sdpa_paged_tmp_floats(ctx, c, t, n_q, rows_most) * 4) && ks_aligned(tmp, 16), "%s: tmp buffer too small, or not on 16 bytes", who);
  if (rows_most == 0) return KS_OK;
  (void)ctx_most;
  KS_REQUIRE_DEVICE(ctx, who);
  ks_on_device on(ctx);
  SdpaArgs a{};
  a.kc = (const uint8_t*)c->k->dptr;
  a.vc = (const uint8_t*)c->v->dptr;
  a.ks = (const float*)c->k_scale->dptr;
  a.vs = (const float*)c->v_scale->dptr;
  a.lens = (const int*)t->lens->dptr;
  a.tables = (const int*)t->tables->dptr;
  a.row_start = (const int*)t->plan->dptr + ks_plan_parts(t->n_seqs, t->max_rows, t->page).row_start;
  a.q = q->dptr;
  a.out = out->dptr;
  a.tmp = (float*)tmp->dptr;
  a.bad = (unsigned*)ctx->ws + KS_WS_INDEX_WORD;
  a.arrived = (unsigned*)ctx->ws + KS_WS_COUNT_WORD;
  a.n_seqs = (unsigned)t->n_seqs;
  a.max_blocks = (unsigned)t->max_blocks;
  a.n_pages = (unsigned)t->n_pages;
  a.page_log = (unsigned)__builtin_ctzll(t->page);
  a.max_rows = (unsigned)t->max_rows;
  a.rows_most = (unsigned)rows_most;
  a.n_q = (unsigned)n_q;
  a.n_kv = (unsigned)c->n_kv;
  a.G = (unsigned)G;
  a.window = (unsigned)window;
  a.scale = scale;
  const dim3 grid(a.max_rows, a.n_q);
#define KS_AT(HD_, T_, F_) KS_LAUNCH(ctx, (sdpa_q8_row_kernel<HD_, T_, F_>), grid, 32, 0, a)
#define KS_AT_T(HD_, F_) do { if (act == KS_F32) KS_AT(HD_, float, F_); else KS_AT(HD_, __half, F_); } while (0)
#define KS_AT_F(HD_) do { if (c->dtype == KS_E4M3) KS_AT_T(HD_, true); else KS_AT_T(HD_, false); } while (0)
  if (c->hd == 256) KS_AT_F(256);
  else if (c->hd == 128) KS_AT_F(128);
  else KS_AT_F(64);
#undef KS_AT_F
#undef KS_AT_T
#undef KS_AT
  return ks_after_launch(ctx, who);
}

}  // extern "C"
