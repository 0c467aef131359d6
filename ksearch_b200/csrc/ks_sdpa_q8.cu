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
  float* part;               // records of split pieces
  unsigned long long* first; // [n_seqs + 1]: units in front of each sequence
  unsigned* bad;
  unsigned n_seqs, max_blocks, n_pages, page_log, max_rows, rows_most, n_q, n_kv, G, window;
  unsigned few;              // sequences of up to so many rows (times G) take the split kernel
  unsigned least;            // units a block takes at least
  float scale;
};

// ---- what a sequence has to do ------------------------------------------------------------------------------
struct Seq {
  int row0, rows, len, begin;  // first row of the call, rows, positions, first position that some row sees
};
__device__ __forceinline__ bool seq_of(const SdpaArgs& a, unsigned i, Seq& s) {  // false: nothing to do
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

// ---- few rows: the context is what counts -------------------------------------------------------------------
// A piece is 16 rows (row and query head of the group, counted together) of a sequence against one KV head; its units are tiles of
// TILE positions.  All units of the launch lie in one line and every block takes a run of them of the same length, so that a block's
// share does not depend on how lengths differ; pieces that lie in several blocks leave a record (m, l, O) per block for the merge.
template <int HD_, typename T_>
struct Split {
  static constexpr int HD = HD_, TERMS = sizeof(T_) == 4 ? 2 : 1;
  static constexpr int TILE = HD == 256 ? 64 : 128, STAGES = 3, WARPS = 8, THREADS = WARPS * 32;
  static constexpr int KH = HD == 256 ? 2 : 1, KR = HD / KH;   // warps share out positions, and the halves of a head of 256: KR dims each
  static constexpr int DG = HD / 32, PG = WARPS / DG;          // of the values: 32 dims each, and 1, 2 or 4 shares of the positions
  static constexpr int CH = HD / 16, ROWS = THREADS / CH, PASSES = TILE / ROWS;  // a thread copies 16 bytes of PASSES rows
  static constexpr int SP = TILE + 8, COLS = TILE / 16, GROUPS = TILE / 16;
  static constexpr unsigned stage_bytes = 2 * TILE * HD, scales = STAGES * stage_bytes, scores = scales + STAGES * GROUPS * 8, probs = scores + KH * 16 * SP * 4,
                            alpha = probs + TERMS * 16 * SP * 2, sums = alpha + 64, red = alpha + 128, total = red + (PG - 1) * 16 * HD * 4;
  static constexpr unsigned record = 16 * (HD + 2);            // floats: m[16], l[16], O[16][HD]
  static_assert(WARPS / KH * 16 == TILE, "a warp makes the scores of 16 positions");
};
constexpr float kNone = -1.0e30f;       // the maximum of nothing
constexpr float kProbs = 16384.0f;      // probabilities carry 2^14: the second f16 term of one of 2^-16 is no denormal

__device__ __forceinline__ uint32_t smem_at(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(there ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copies_sent() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
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
__device__ __forceinline__ void put8(float* to, const float (&v)[8], float f) {
  *reinterpret_cast<float4*>(to) = make_float4(v[0] * f, v[1] * f, v[2] * f, v[3] * f);
  *reinterpret_cast<float4*>(to + 4) = make_float4(v[4] * f, v[5] * f, v[6] * f, v[7] * f);
}
__device__ __forceinline__ void put8(__half* to, const float (&v)[8], float f) {
  uint4 w;
  w.x = q8_u32(__floats2half2_rn(v[0] * f, v[1] * f));
  w.y = q8_u32(__floats2half2_rn(v[2] * f, v[3] * f));
  w.z = q8_u32(__floats2half2_rn(v[4] * f, v[5] * f));
  w.w = q8_u32(__floats2half2_rn(v[6] * f, v[7] * f));
  *reinterpret_cast<uint4*>(to) = w;
}
// A positive scale (inside q8_scale's range) as 2^e and a factor of 1 to 2.
__device__ __forceinline__ void split_scale(float s, float& e, float& factor, float& down) {
  const uint32_t b = __float_as_uint(s);
  const int x = (int)(b >> 23) - 127;
  e = (float)x;
  factor = __uint_as_float((b & 0x7FFFFFu) | 0x3F800000u);
  down = __uint_as_float((uint32_t)(127 - x) << 23);
}

template <int HD, typename T, bool FP8>
__global__ void __launch_bounds__(256, 2) sdpa_q8_split_kernel(const SdpaArgs a) {
  using S = Split<HD, T>;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ unsigned long long scan[S::WARPS], seq_first;
  __shared__ unsigned seq_at;
  ks_pdl_entry();
  const unsigned tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, g = lane >> 2, c = lane & 3u;
  const uint32_t sb = smem_at(smem);

  // ---- the line of units: a thread counts for up to four neighbouring sequences
  auto units_of = [&](const Seq& s) -> unsigned long long {
    const unsigned m = (unsigned)s.rows * a.G;
    if (m > a.few) return 0ull;
    const int t0 = s.begin / S::TILE, t1 = (s.len + S::TILE - 1) / S::TILE;
    return (unsigned long long)((m + 15u) / 16u) * a.n_kv * (unsigned)max(t1 - t0, 1);  // (a row that sees nothing still gets its zeros)
  };
  const unsigned per = (a.n_seqs + S::THREADS - 1u) / S::THREADS;
  unsigned long long mine[KS_PAGES_MAX_SEQS / 256], sum = 0;
#pragma unroll
  for (unsigned k = 0; k < KS_PAGES_MAX_SEQS / 256; k++) {
    const unsigned i = tid * per + k;
    Seq s;
    mine[k] = k < per && i < a.n_seqs && seq_of(a, i, s) ? units_of(s) : 0ull;
    sum += mine[k];
  }
  unsigned long long before = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long up = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= (unsigned)o) before += up;
  }
  if (lane == 31u) scan[warp] = before;
  __syncthreads();
  unsigned long long total = 0;
  before -= sum;
  for (unsigned w = 0; w < S::WARPS; w++) {
    before += w < warp ? scan[w] : 0ull;
    total += scan[w];
  }
  if (total == 0ull) {
    if (blockIdx.x == 0 && tid == 0) a.first[a.n_seqs] = 0ull;
    return;
  }
  const unsigned long long blocks = min((unsigned long long)gridDim.x, (total + a.least - 1u) / a.least);
  if (blockIdx.x >= blocks) return;
  const unsigned long long u_begin = blockIdx.x * total / blocks, u_end = (blockIdx.x + 1u) * total / blocks;
#pragma unroll
  for (unsigned k = 0; k < KS_PAGES_MAX_SEQS / 256; k++) {
    const unsigned i = tid * per + k;
    if (k < per && i < a.n_seqs) {
      if (blockIdx.x == 0) a.first[i] = before;
      if (u_begin >= before && u_begin - before < mine[k]) {
        seq_at = i;
        seq_first = before;
      }
      before += mine[k];
    }
  }
  if (blockIdx.x == 0 && tid == 0) a.first[a.n_seqs] = total;
  __syncthreads();

  // ---- piece after piece
  unsigned seq = seq_at, in_block = 0;
  unsigned long long u = u_begin, at = seq_first;
  Seq s;
  bool have = seq_of(a, seq, s);
  while (u < u_end) {
    while (u - at >= (have ? units_of(s) : 0ull)) {
      at += have ? units_of(s) : 0ull;
      have = seq_of(a, ++seq, s);
    }
    const int tile0 = s.begin / S::TILE, n_tiles = max((s.len + S::TILE - 1) / S::TILE - tile0, 1);
    const unsigned m_rows = (unsigned)s.rows * a.G, m_tiles = (m_rows + 15u) / 16u;
    const unsigned piece = (unsigned)((u - at) / (unsigned)n_tiles), t_first = (unsigned)((u - at) % (unsigned)n_tiles);
    const unsigned kvh = piece / m_tiles, m0 = piece % m_tiles * 16u;
    const unsigned n = (unsigned)min((unsigned long long)((unsigned)n_tiles - t_first), u_end - u);  // tiles of this piece that are ours
    const int t0 = tile0 + (int)t_first;

    // copies of tile t of the piece into stage st: 16 bytes a thread and row, chunks swapped about so that the reads below meet no bank twice
    auto send = [&](int t, unsigned st) {
      const uint32_t to = sb + st * S::stage_bytes;
      const unsigned ch = tid % S::CH;
#pragma unroll
      for (int i = 0; i < S::PASSES; i++) {
        const unsigned r = tid / S::CH + (unsigned)i * S::ROWS;
        const int pos = t * S::TILE + (int)r;
        bool there = pos >= s.begin && pos < s.len;
        size_t from = 0;
        if (there) {
          const int id = a.tables[(size_t)seq * a.max_blocks + ((unsigned)pos >> a.page_log)];
          there = id >= 0 && (unsigned)id < a.n_pages;
          if (there) from = (((((size_t)id * a.n_kv + kvh) << a.page_log) + ((unsigned)pos & ((1u << a.page_log) - 1u))) * HD) + ch * 16u;
          else if (ch == 0) atomicOr(a.bad, KS_BAD_PAGE);
        }
        const unsigned kch = HD >= 128 ? ch ^ ((r & 1u) << 2) : ch, vch = HD >= 128 ? ch ^ ((r >> 1 & 3u) << 1) : ch ^ ((r >> 1 & 1u) << 1);
        copy16(to + r * HD + kch * 16u, a.kc + from, there);
        copy16(to + S::TILE * HD + r * HD + vch * 16u, a.vc + from, there);
      }
      if (tid < 2 * S::GROUPS) {  // a scale for each 16 positions (a page has no fewer)
        const unsigned gr = tid % S::GROUPS;
        const int pos = t * S::TILE + 16 * (int)gr;
        bool there = pos + 15 >= s.begin && pos < s.len;
        size_t from = 0;
        if (there) {
          const int id = a.tables[(size_t)seq * a.max_blocks + ((unsigned)pos >> a.page_log)];
          there = id >= 0 && (unsigned)id < a.n_pages;
          if (there) from = (size_t)id * a.n_kv + kvh;
        }
        copy4(sb + S::scales + (st * 2 * S::GROUPS + tid) * 4u, (tid < S::GROUPS ? a.ks : a.vs) + from, there);
      }
    };
#pragma unroll
    for (int i = 0; i < S::STAGES - 1; i++) {
      if ((unsigned)i < n) send(t0 + i, (unsigned)i);
      copies_sent();
    }

    // ---- q: rows g and g + 8, dims 16 c .. 16 c + 15 of every 64: what the codes of a 16-byte read meet.  f32 rows are brought to 2^14 by a
    // power of two (per half of a head) and split into two f16 terms
    const unsigned kh = S::KH == 2 ? warp >> 2 : 0u, pw = S::KH == 2 ? warp & 3u : warp;
    uint32_t qa[S::TERMS][S::KR / 64][4][4];
    float up[2] = {1.0f, 1.0f};
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const unsigned m = m0 + g + 8u * h;
      const bool in = m < m_rows;
      const T* src = (const T*)a.q + ((size_t)(s.row0 + (int)(m / a.G)) * a.n_q + kvh * a.G + m % a.G) * HD + kh * S::KR + 16u * c;
      if constexpr (S::TERMS == 1) {
#pragma unroll
        for (int kk = 0; kk < S::KR / 64; kk++) {
          const uint4 x = in ? *reinterpret_cast<const uint4*>(src + 64 * kk) : make_uint4(0, 0, 0, 0), y = in ? *reinterpret_cast<const uint4*>(src + 64 * kk + 8) : make_uint4(0, 0, 0, 0);
          const uint32_t w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
          for (int k = 0; k < 4; k++) {
            qa[0][kk][k][h] = w[2 * k];
            qa[0][kk][k][h + 2] = w[2 * k + 1];
          }
        }
      } else {
        float x[S::KR / 64][16], big = 0.0f;
#pragma unroll
        for (int kk = 0; kk < S::KR / 64; kk++)
#pragma unroll
          for (int e = 0; e < 16; e += 4) {
            const float4 v = in ? *reinterpret_cast<const float4*>((const float*)src + 64 * kk + e) : make_float4(0.f, 0.f, 0.f, 0.f);
            x[kk][e] = v.x; x[kk][e + 1] = v.y; x[kk][e + 2] = v.z; x[kk][e + 3] = v.w;
            big = fmaxf(fmaxf(big, fmaxf(fabsf(v.x), fabsf(v.y))), fmaxf(fabsf(v.z), fabsf(v.w)));
          }
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
        const int ex = big > 0.0f && big < 3.0e38f ? max((int)(__float_as_uint(big) >> 23) - 127 - 14, -100) : 0;
        up[h] = __uint_as_float((uint32_t)(127 + ex) << 23);
        const float down = __uint_as_float((uint32_t)(127 - ex) << 23);
#pragma unroll
        for (int kk = 0; kk < S::KR / 64; kk++)
#pragma unroll
          for (int e = 0; e < 16; e += 2) {
            const float x0 = x[kk][e] * down, x1 = x[kk][e + 1] * down;
            const __half2 hi = __floats2half2_rn(x0, x1);
            const float2 f = __half22float2(hi);
            const int k = e / 4, r = h + (e & 2);
            qa[0][kk][k][r] = q8_u32(hi);
            qa[S::TERMS - 1][kk][k][r] = q8_u32(__floats2half2_rn(x0 - f.x, x1 - f.y));
          }
      }
    }
    // ---- a row of scores: 16 threads, COLS neighbouring positions each
    const unsigned row = tid >> 4, col = (tid & 15u) * S::COLS;
    int lo = 0, hi = -1;  // positions lo .. hi are seen
    if (m0 + row < m_rows) {
      hi = s.len - s.rows + (int)((m0 + row) / a.G);
      lo = a.window && hi >= (int)a.window ? hi - (int)a.window + 1 : 0;
    }
    float m = kNone, l = 0.0f, acc[4][4];
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
      for (int e = 0; e < 4; e++) acc[j][e] = 0.0f;
    const float to_log2 = a.scale * 1.44269504088896340736f;
    const unsigned dg = warp % S::DG, pg = warp / S::DG;

    for (unsigned i = 0; i < n; i++) {
      const unsigned st = i % S::STAGES;
      copies_wait<S::STAGES - 2>();
      __syncthreads();
      if (i + S::STAGES - 1 < n) send(t0 + (int)(i + S::STAGES - 1), (i + S::STAGES - 1) % S::STAGES);
      copies_sent();
      // scores of 16 positions
      {
        float d[2][4];
#pragma unroll
        for (int nt = 0; nt < 2; nt++)
#pragma unroll
          for (int e = 0; e < 4; e++) d[nt][e] = 0.0f;
#pragma unroll
        for (int nt = 0; nt < 2; nt++) {
          const unsigned p = pw * 16u + nt * 8u + g;
#pragma unroll
          for (int kk = 0; kk < S::KR / 64; kk++) {
            const unsigned ch = kh * (S::KR / 16) + 4u * kk + c, kch = HD >= 128 ? ch ^ ((p & 1u) << 2) : ch;
            const uint4 w = *reinterpret_cast<const uint4*>(smem + st * S::stage_bytes + p * HD + kch * 16u);
            const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int k = 0; k < 4; k++) {
              uint32_t b0, b1;
              widen4<FP8>(ww[k], b0, b1);
              if constexpr (S::TERMS == 2) mma16816(d[nt], qa[S::TERMS - 1][kk][k], b0, b1);
              mma16816(d[nt], qa[0][kk][k], b0, b1);
            }
          }
        }
        float* to = reinterpret_cast<float*>(smem + S::scores) + (size_t)kh * 16 * S::SP + pw * 16u + 2u * c;
#pragma unroll
        for (int nt = 0; nt < 2; nt++) {
          *reinterpret_cast<float2*>(to + g * S::SP + nt * 8) = make_float2(d[nt][0] * up[0], d[nt][1] * up[0]);
          *reinterpret_cast<float2*>(to + (g + 8u) * S::SP + nt * 8) = make_float2(d[nt][2] * up[1], d[nt][3] * up[1]);
        }
      }
      __syncthreads();
      {
        const float* scales = reinterpret_cast<const float*>(smem + S::scales) + st * 2 * S::GROUPS + col / 16u;
        const float ks = q8_scale(scales[0]) * to_log2;
        float ve, vf, vd;
        split_scale(q8_scale(scales[S::GROUPS]), ve, vf, vd);
        const float* from = reinterpret_cast<const float*>(smem + S::scores) + row * S::SP + col;
        float x[S::COLS], mx = m;
        const int p0 = (t0 + (int)i) * S::TILE + (int)col;
#pragma unroll
        for (int k = 0; k < S::COLS; k += 4) {
          float4 v = *reinterpret_cast<const float4*>(from + k);
          if constexpr (S::KH == 2) {
            const float4 w = *reinterpret_cast<const float4*>(from + 16 * S::SP + k);
            v = make_float4(v.x + w.x, v.y + w.y, v.z + w.z, v.w + w.w);
          }
          x[k] = v.x; x[k + 1] = v.y; x[k + 2] = v.z; x[k + 3] = v.w;
        }
#pragma unroll
        for (int k = 0; k < S::COLS; k++) {
          x[k] = p0 + k >= lo && p0 + k <= hi ? fmaf(x[k], ks, ve) : -INFINITY;
          mx = fmaxf(mx, x[k]);
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float turn = exp2_fast(m - mx);
        m = mx;
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < S::COLS; k++) {
          x[k] = exp2_fast(x[k] - mx);
          sum += x[k];
          x[k] *= vf * kProbs;
        }
        l = fmaf(l, turn, sum * vd);
        __half* to = reinterpret_cast<__half*>(smem + S::probs) + row * S::SP + col;
#pragma unroll
        for (int k = 0; k < S::COLS; k += 2) {
          const __half2 h = __floats2half2_rn(x[k], x[k + 1]);
          *reinterpret_cast<__half2*>(to + k) = h;
          if constexpr (S::TERMS == 2) {
            const float2 f = __half22float2(h);
            *reinterpret_cast<__half2*>(to + 16 * S::SP + k) = __floats2half2_rn(x[k] - f.x, x[k + 1] - f.y);
          }
        }
        if ((tid & 15u) == 0) reinterpret_cast<float*>(smem + S::alpha)[row] = turn;
      }
      __syncthreads();
      // values: 32 dims of the positions of this warp's share
      {
        float d[4][4];
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
          for (int e = 0; e < 4; e++) d[j][e] = 0.0f;
        constexpr int KS = S::TILE / S::PG / 16;
#pragma unroll
        for (int k = 0; k < KS; k++) {
          const unsigned base = pg * (S::TILE / S::PG) + 16u * k;
          uint32_t p[S::TERMS][4];
#pragma unroll
          for (int t = 0; t < S::TERMS; t++) {
            const uint32_t from = sb + S::probs + (t * 16 * S::SP + ((lane & 7u) + (lane >> 3 & 1u) * 8u) * S::SP + base + (lane >> 4) * 8u) * 2u;
            asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(p[t][0]), "=r"(p[t][1]), "=r"(p[t][2]), "=r"(p[t][3]) : "r"(from) : "memory");
          }
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const unsigned r = base + 2u * c + (e & 1) + (e >> 1) * 8u, byte = dg * 32u + 4u * g, ch = byte >> 4;
            const unsigned vch = HD >= 128 ? ch ^ ((r >> 1 & 3u) << 1) : ch ^ ((r >> 1 & 1u) << 1);
            w[e] = *reinterpret_cast<const uint32_t*>(smem + st * S::stage_bytes + S::TILE * HD + r * HD + vch * 16u + (byte & 15u));
          }
          uint32_t b0[4], b1[4];
          widen_pairs<FP8>(w[0], w[1], b0);
          widen_pairs<FP8>(w[2], w[3], b1);
#pragma unroll
          for (int j = 0; j < 4; j++) {
            if constexpr (S::TERMS == 2) mma16816(d[j], p[S::TERMS - 1], b0[j], b1[j]);
            mma16816(d[j], p[0], b0[j], b1[j]);
          }
        }
        const float t0f = reinterpret_cast<const float*>(smem + S::alpha)[g], t1f = reinterpret_cast<const float*>(smem + S::alpha)[g + 8u];
#pragma unroll
        for (int j = 0; j < 4; j++) {
          acc[j][0] = fmaf(acc[j][0], t0f, d[j][0]);
          acc[j][1] = fmaf(acc[j][1], t0f, d[j][1]);
          acc[j][2] = fmaf(acc[j][2], t1f, d[j][2]);
          acc[j][3] = fmaf(acc[j][3], t1f, d[j][3]);
        }
      }
    }
    // ---- the piece's result: to `out`, or a record if other blocks have a part of it
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    const bool whole = n == (unsigned)n_tiles;
    float* rec = a.part + ((size_t)blockIdx.x * 2u + (in_block ? 1u : 0u)) * S::record;
    if ((tid & 15u) == 0) {
      if (whole) {
        reinterpret_cast<float*>(smem + S::sums)[row] = l > 0.0f ? (1.0f / kProbs) / l : l == 0.0f ? 0.0f : l;  // (NaN stays)
      } else {
        rec[row] = m;
        rec[16 + row] = l;
      }
    }
    if constexpr (S::PG > 1) {
      float* red = reinterpret_cast<float*>(smem + S::red);
      if (pg > 0) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
          float* to = red + (size_t)(pg - 1u) * 16 * HD + (g + 8u * h) * HD + dg * 32u + 8u * c;
          *reinterpret_cast<float4*>(to) = make_float4(acc[0][2 * h], acc[1][2 * h], acc[2][2 * h], acc[3][2 * h]);
          *reinterpret_cast<float4*>(to + 4) = make_float4(acc[0][2 * h + 1], acc[1][2 * h + 1], acc[2][2 * h + 1], acc[3][2 * h + 1]);
        }
      }
    }
    __syncthreads();
    if (pg == 0) {
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const unsigned r = g + 8u * h, mm = m0 + r;
        float v[8];
#pragma unroll
        for (int j = 0; j < 4; j++) {
          v[j] = acc[j][2 * h];
          v[j + 4] = acc[j][2 * h + 1];
        }
        if constexpr (S::PG > 1)
#pragma unroll
          for (int k = 0; k < S::PG - 1; k++)
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] += reinterpret_cast<const float*>(smem + S::red)[(size_t)k * 16 * HD + r * HD + dg * 32u + 8u * c + e];
        if (mm >= m_rows) continue;
        if (whole) {
          const float f = reinterpret_cast<const float*>(smem + S::sums)[r];
          T* to = (T*)a.out + ((size_t)(s.row0 + (int)(mm / a.G)) * a.n_q + kvh * a.G + mm % a.G) * HD + dg * 32u + 8u * c;
          put8(to, v, f);
        } else {
          float* to = rec + 32 + r * HD + dg * 32u + 8u * c;
          *reinterpret_cast<float4*>(to) = make_float4(v[0], v[1], v[2], v[3]);
          *reinterpret_cast<float4*>(to + 4) = make_float4(v[4], v[5], v[6], v[7]);
        }
      }
    }
    u += n;
    in_block++;
    __syncthreads();  // everything in shared memory is free again
  }
}

// ---- the records of pieces that lie in several blocks ----------------------------------------------------------
// out = sum_b e_b O_b / sum_b e_b l_b, e_b = exp2(m_b - max m), in the order of the blocks.  Grid: (pieces, or block borders where there are more
// pieces than borders; rows; 64 dims).  Of a block's 256 threads 16 share 64 dims, and there are 16 shares of the records.
constexpr unsigned kMergeMost = 1024;  // blocks of the split kernel
template <int HD, typename T>
__global__ void __launch_bounds__(256) sdpa_q8_merge_kernel(const SdpaArgs a, unsigned split_blocks, bool by_border) {
  using S = Split<HD, T>;
  __shared__ float fac[kMergeMost], red[16][64 + 4], mx_s[8], l_s[8];
  __shared__ unsigned found;
  ks_pdl_entry();
  const unsigned tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
  const unsigned long long total = a.first[a.n_seqs];
  if (total == 0ull) return;
  const unsigned long long blocks = min((unsigned long long)split_blocks, (total + a.least - 1u) / a.least);
  unsigned seq, piece;
  unsigned long long at, border = 0;
  if (by_border) {
    if (blockIdx.x + 1u >= blocks) return;
    border = (blockIdx.x + 1u) * total / blocks;  // first unit of block blockIdx.x + 1
    for (unsigned i = tid; i < a.n_seqs; i += 256u)
      if (a.first[i] <= border && border < a.first[i + 1u]) found = i;
    __syncthreads();
    seq = found;
    piece = 0;
  } else {
    const unsigned per = a.n_kv * ((a.few + 15u) / 16u);
    seq = blockIdx.x / per;
    piece = blockIdx.x % per;
  }
  at = a.first[seq];
  const unsigned long long units = a.first[seq + 1u] - at;
  Seq s;
  if (units == 0ull || !seq_of(a, seq, s)) return;
  const unsigned m_rows = (unsigned)s.rows * a.G, m_tiles = (m_rows + 15u) / 16u;
  const unsigned long long n_tiles = units / (m_tiles * a.n_kv);
  if (by_border) piece = (unsigned)((border - at) / n_tiles);
  else if (piece >= m_tiles * a.n_kv) return;
  const unsigned long long u0 = at + piece * n_tiles, u1 = u0 + n_tiles;
  const unsigned b0 = (unsigned)(((u0 + 1u) * blocks - 1u) / total), b1 = (unsigned)((u1 * blocks - 1u) / total);  // the blocks of its first and last unit
  if (b0 == b1 || (by_border && b0 != blockIdx.x)) return;  // whole; or another border's
  const unsigned n = b1 - b0 + 1u, kvh = piece / m_tiles, m0 = piece % m_tiles * 16u;
  const unsigned slot0 = b0 * total / blocks >= u0 ? 0u : 1u;  // the first block's record is its second unless the piece starts with the block
  auto record = [&](unsigned k) { return a.part + ((size_t)(b0 + k) * 2u + (k ? 0u : slot0)) * S::record; };
  for (unsigned r = blockIdx.y; r < 16u && m0 + r < m_rows; r += gridDim.y) {
    float mx = kNone;
    for (unsigned k = tid; k < n; k += 256u) mx = fmaxf(mx, record(k)[r]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if (lane == 0) mx_s[warp] = mx;
    __syncthreads();
    for (int w = 0; w < 8; w++) mx = fmaxf(mx, mx_s[w]);
    float l = 0.0f;
    for (unsigned k = tid; k < n; k += 256u) {
      const float e = exp2_fast(record(k)[r] - mx);
      fac[k] = e;
      l = fmaf(e, record(k)[16 + r], l);
    }
    l = q8_warp_sum(l);
    if (lane == 0) l_s[warp] = l;
    __syncthreads();
    l = 0.0f;
    for (int w = 0; w < 8; w++) l += l_s[w];
    const float f = l > 0.0f ? (1.0f / kProbs) / l : l == 0.0f ? 0.0f : l;
    for (unsigned d0 = blockIdx.z * 64u; d0 < HD; d0 += gridDim.z * 64u) {
      const unsigned share = tid >> 4, d = (tid & 15u) * 4u;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (unsigned k = share; k < n; k += 16u) {
        const float4 o = *reinterpret_cast<const float4*>(record(k) + 32 + r * HD + d0 + d);
        const float e = fac[k];
        v.x = fmaf(o.x, e, v.x);
        v.y = fmaf(o.y, e, v.y);
        v.z = fmaf(o.z, e, v.z);
        v.w = fmaf(o.w, e, v.w);
      }
      *reinterpret_cast<float4*>(&red[share][d]) = v;
      __syncthreads();
      if (tid < 64u) {
        float x = 0.0f;
#pragma unroll
        for (int k = 0; k < 16; k++) x += red[k][tid];
        ((T*)a.out)[((size_t)(s.row0 + (int)((m0 + r) / a.G)) * a.n_q + kvh * a.G + (m0 + r) % a.G) * HD + d0 + tid] = (T)(x * f);
      }
      __syncthreads();
    }
  }
}

constexpr unsigned kSplitPerSm = 2;  // blocks of the split kernel an SM holds (shared memory)
unsigned split_blocks(const ks_ctx* ctx) { return (unsigned)ctx->sm_count * kSplitPerSm; }
size_t first_floats(const ks_page_tables* t) { return (2 * (t->n_seqs + 1) + 3) & ~size_t(3); }

template <int HD, typename T, bool FP8>
int launch_split(ks_ctx* ctx, const SdpaArgs& a, unsigned blocks) {
  using S = Split<HD, T>;
  static bool set[16] = {false};
  if (!set[ctx->device & 15]) {
    cudaError_t e = cudaFuncSetAttribute(sdpa_q8_split_kernel<HD, T, FP8>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::total);
    if (e != cudaSuccess) return ks_fail(ctx, KS_ERR_CUDA, "sdpa_paged_q8: cannot set %u B shared memory: %s", S::total, cudaGetErrorString(e));
    set[ctx->device & 15] = true;
  }
  KS_LAUNCH(ctx, (sdpa_q8_split_kernel<HD, T, FP8>), blocks, S::THREADS, S::total, a);
  int rc = ks_after_launch(ctx, "sdpa_paged_q8");
  if (rc || blocks == 1) return rc;
  const size_t pieces = (size_t)a.n_seqs * a.n_kv * ((a.few + 15u) / 16u);
  const bool by_border = pieces >= blocks;
  const unsigned rows = a.few < 16u ? a.few : 16u;
  KS_LAUNCH(ctx, (sdpa_q8_merge_kernel<HD, T>), dim3(by_border ? blocks - 1u : (unsigned)pieces, by_border ? 1u : rows, by_border ? 1u : HD / 64u), 256, 0, a, blocks, by_border);
  return ks_after_launch(ctx, "sdpa_paged_q8 merge");
}

}  // namespace

extern "C" {

size_t ks_sdpa_paged_tmp_floats(const ks_ctx* ctx, const ks_q8_cache* c, const ks_page_tables* t, size_t n_q, size_t rows_most) {
  if (!ctx || !c || !t || !c->n_kv || !rows_most || n_q < c->n_kv) return 0;
  return first_floats(t) + (size_t)split_blocks(ctx) * 2 * 16 * (c->hd + 2);
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
  a.first = (unsigned long long*)tmp->dptr;
  a.part = (float*)tmp->dptr + first_floats(t);
  a.few = (unsigned)(rows_most * G);
  a.least = 1;
  a.bad = (unsigned*)ctx->ws + KS_WS_INDEX_WORD;
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
  const unsigned blocks = split_blocks(ctx);
#define KS_AT(HD_, T_, F_) launch_split<HD_, T_, F_>(ctx, a, blocks)
#define KS_AT_T(HD_, F_) (act == KS_F32 ? KS_AT(HD_, float, F_) : KS_AT(HD_, __half, F_))
#define KS_AT_F(HD_) (c->dtype == KS_E4M3 ? KS_AT_T(HD_, true) : KS_AT_T(HD_, false))
  return c->hd == 256 ? KS_AT_F(256) : c->hd == 128 ? KS_AT_F(128) : KS_AT_F(64);
#undef KS_AT_F
#undef KS_AT_T
#undef KS_AT
}

}  // extern "C"
