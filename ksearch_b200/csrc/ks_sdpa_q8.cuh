// Shared by the two attention kernels over a paged 8-bit cache (ks_sdpa_q8.cu: few rows, ks_sdpa_q8_wide.cu: many).
#pragma once
#include "ks_q8.h"
#include "ks_q8.cuh"

struct ks_sdpa_q8_args {
  const uint8_t *kc, *vc;
  const float *ks, *vs;
  const int *lens, *tables, *row_start;
  const void* q;
  void* out;
  float* part;               // records of split pieces
  int4* merges;              // [blocks][2]: first block, records, which of the first block's, first (row, head); row, KV head, (row, head)s of the sequence
  unsigned* bad;
  unsigned n_seqs, max_blocks, n_pages, page_log, max_rows, rows_most, n_q, n_kv, G, window;
  unsigned few;              // sequences of up to so many rows (times G) take the split kernel
  float scale;
};

// Rows times query heads of a group up to which a sequence takes the kernel of few rows, whatever else there is (more: ks_sdpa_q8.cu).
constexpr unsigned KS_Q8_FEW = 32;
// Sequences of more rows; tmp: ks_sdpa_q8_wide_floats.
size_t ks_sdpa_q8_wide_floats(const ks_ctx* ctx, size_t n_seqs, size_t max_rows, size_t n_kv, size_t G, size_t hd);
int ks_launch_sdpa_q8_wide(ks_ctx* ctx, const ks_sdpa_q8_args& a, size_t hd, ks_dtype act, bool fp8, float* tmp, size_t ctx_most, bool beside);
int ks_launch_sdpa_q8_wide_merge(ks_ctx* ctx, const ks_sdpa_q8_args& a, size_t hd, ks_dtype act, float* tmp, size_t ctx_most, bool beside);

namespace {

// Up to four kernels follow one another in a call: few rows, many rows, the merges of either.  Those of few and of many rows do not depend on each other,
// nor do the merges, so the second of a pair lets the first run on: a kernel starts its successor only when everything before the pair is
// done (start_next behind wait_before), the second kernel of a pair (`beside`) waits for the first one only before it ends, so that what
// follows it follows both.
__device__ __forceinline__ void wait_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void start_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// ---- what a sequence has to do ------------------------------------------------------------------------------
struct Seq {
  int row0, rows, len, begin;  // first row of the call, rows, positions, first position that some row sees
};
__device__ __forceinline__ bool seq_of(const ks_sdpa_q8_args& a, unsigned i, Seq& s) {  // false: nothing to do
  const int r0 = a.row_start[i], r1 = a.row_start[i + 1u], len = a.lens[i];
  s.row0 = r0;
  s.rows = r1 - r0;
  s.len = min(max(len, 0), (int)(a.max_blocks << a.page_log));
  const int p0 = s.len - s.rows;
  s.begin = a.window && p0 >= (int)a.window ? p0 - (int)a.window + 1 : 0;
  if (s.rows <= 0) return false;
  if (r0 < 0 || r1 > (int)a.max_rows || s.rows > (int)a.rows_most) {
    if (blockIdx.x == 0) atomicOr(a.bad, KS_BAD_ROWS);
    return false;
  }
  return true;
}

constexpr float kNone = -1.0e30f;       // the maximum of nothing
constexpr float kProbs = 1024.0f, kProbsLog2 = 10.0f;       // probabilities carry 2^10, are 2^5 at most, and 2^-35 of the largest is the least that counts
constexpr float kSlack = 4.0f;          // log2 of how far a score may exceed what probabilities refer to

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The four codes of a word as f16: 0, 1 and 2, 3.
template <bool FP8>
__device__ __forceinline__ void widen4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (FP8) {
    lo = q8_u32(q8_decode2h<true>(w));
    hi = q8_u32(q8_decode2h<true>(w >> 16));
  } else {
    w ^= 0x80808080u;
    lo = q8_u32(__hsub2(q8_h2(__byte_perm(w, 0x64646464u, 0x4140)), __float2half2_rn(1152.0f)));
    hi = q8_u32(__hsub2(q8_h2(__byte_perm(w, 0x64646464u, 0x4342)), __float2half2_rn(1152.0f)));
  }
}
// Codes j = 0..3 of two rows' words as pairs (row a, row b).
template <bool FP8>
__device__ __forceinline__ void widen_pairs(uint32_t a, uint32_t b, uint32_t (&p)[4]) {
  const uint32_t x = __byte_perm(a, b, 0x5140), y = __byte_perm(a, b, 0x7362);
  widen4<FP8>(x, p[0], p[1]);
  widen4<FP8>(y, p[2], p[3]);
}
// What a row's values are multiplied by in the end; a row that saw nothing is zero, NaN stays.
__device__ __forceinline__ float over(float l) { return l > 0.0f ? (1.0f / kProbs) / l : l == 0.0f ? 0.0f : l; }
__device__ __forceinline__ void put_dims(float* to, const float* v, int n) {
  if (n == 4) *reinterpret_cast<float4*>(to) = make_float4(v[0], v[1], v[2], v[3]);
  else *reinterpret_cast<float2*>(to) = make_float2(v[0], v[1]);
}
__device__ __forceinline__ void put_dims(__half* to, const float* v, int n) {
  const uint32_t x = q8_u32(__floats2half2_rn(v[0], v[1]));
  if (n == 4) *reinterpret_cast<uint2*>(to) = make_uint2(x, q8_u32(__floats2half2_rn(v[2], v[3])));
  else *reinterpret_cast<uint32_t*>(to) = x;
}
// A positive scale (inside q8_scale's range) as 2^e and a factor of 1 to 2, or below 1 where e is kLeastV: the least one, so that a page of zeros (2^-100)
// beside values of 2^50 still leaves its probabilities in the sum, which carries 2^(t - M) 2^-e with t - M down to -126.
constexpr int kLeastV = -60;
__device__ __forceinline__ void split_scale(float s, float& e, float& factor, float& down) {
  const int x = max((int)(__float_as_uint(s) >> 23) - 127, kLeastV);
  e = (float)x;
  down = __uint_as_float((uint32_t)(127 - x) << 23);
  factor = s * down;
}

}  // namespace
