// Attention of ragged rows (single tokens, drafts, prompt pieces) over a paged 8-bit cache.
//
// Row r of a sequence of `len` positions and `rows` rows sits at p = len - rows + r and sees positions max(0, p - window + 1) .. p:
//   s_j = scale q . k_j,   out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),   m = max_j s_j.
// With v_j = vs_j c_j, vs_j = 2^e f (1 <= f < 2) the scale of its page, everything runs on t_j = s_j log2(e) + e and the codes c_j:
//   w_j = 2^(t_j - M) f,   out = sum w_j c_j / sum 2^(t_j - M) 2^-e,   M = max_j t_j:
// weights are below 2^5 whatever the scales (they are rounded to f16 with 2^10 in front), and a sequence whose pages differ by powers of ten
// keeps what carries the sum.  e is -60 at least (f takes the rest): the sum's terms would be lost below 2^-126 of the largest t.
//
// This file: sequences of up to few_of() rows times query heads of a group, and the merge; ks_sdpa_q8_wide.cu: the others.
#include "ks_sdpa_q8.cuh"

namespace {

// ---- few rows: the context is what counts -------------------------------------------------------------------
// A piece is 8 rows (row and query head of the group, counted together) of a sequence against one KV head; its units are tiles of TILE
// positions, SUB for each warp of a block.  All units of the launch lie in one line and every block takes a run of them of the same length, so
// that a block's share does not depend on how lengths differ; pieces that lie in several blocks leave a record (m, l, O) per block for
// the merge.
//
// Inside a block the warps have nothing to do with one another until the piece ends: each brings its SUB positions into a ring of its own
// and keeps its own maximum, sum and values.  Both products are transposed, so that the 16 rows of mma.sync m16n8k16 are positions (dims)
// and its 8 columns the query rows:
//   S^T = K q^T:  a lane reads 16 bytes of two positions' codes, which are the A operand of four steps over 64 dims if q has its dims in that order;
//   O^T = V^T P^T:  the probabilities, out of S^T's accumulators, become B operands by movmatrix; a lane reads 16 dims of four positions, pairs
//   the codes of neighbouring positions by byte permutes, and has its 16 dims of two query rows in the accumulators.
// Codes become f16 exactly.  f32 queries and probabilities are two f16 terms each (the small one first), and the values of every SUB positions are added
// to registers: a chain of accumulating MMAs loses low bits at every step.  f16: queries as they are, probabilities rounded to f16 (2^-12 of
// each, as much again as rounding the result: 2.9e-4 against 2.1e-4 of a plain f32 form, both off 64 bits), values accumulate in the MMAs.
// The maximum that probabilities refer to moves only when a score exceeds it by 2^4.
//
// Bound by: many long contexts by memory (48 sequences of about 6800 positions, f16, 32 heads on 8 of 128: 664 MB in 110 us, 93 % of the measured copy
// rate, and in 124 over seconds at the power limit, 1.66 GHz; with 16 x 64 score tiles on the untransposed products and three block barriers a tile it was 314).  Turning codes into f16 is
// most of what is issued: 5 instructions per 4 codes of K, 7 of V, half the issue slots.  A lone short context by its chain: 700 positions
// (f32, 8 heads on 1 of 256) 10 us with the merge: lengths and counts 1.0, page, q and first codes 1.4, 16 positions 1.3, the warps' results 1.3,
// merge and launches the rest.  Four slots of 1024 to 16384 positions (f32, 2 KV heads): 38.8 MB in 19.1 us, four steps of 1.4 us in the middle.
// The longest context lies in no more blocks than this: each leaves a record that the merge has to read (16384 positions of one KV head: 27 us in 128
// blocks, 14 in 64).
constexpr unsigned kMostParts = 64;
// x / d: one multiplication where the numbers are small enough for it to be off by less than one.
__device__ __forceinline__ unsigned quotient(unsigned x, unsigned d) {
  if ((x | d) >> 20) return x / d;
  unsigned q = (unsigned)__fdividef((float)x, (float)d);
  const int r = (int)(x - q * d);
  if (r < 0) q--;
  else if (r >= (int)d) q++;
  return q;
}
template <int HD_, typename T_>
struct Split {
  static constexpr int HD = HD_, TERMS = sizeof(T_) == 4 ? 2 : 1;
  static constexpr int NP = HD == 64 ? 2 : 1, SUB = 16 * NP, STAGES = 3, WARPS = 8, THREADS = WARPS * 32, TILE = WARPS * SUB;
  static constexpr int PER_SM = HD == 256 ? 1 : 2;
  static constexpr int KK = HD / 64;                    // runs of 64 dims
  static constexpr int W = HD == 64 ? 64 : 128, WN = HD / W, WW = W / 32;  // windows of dims a lane's read of the values lies in, words of such a read
  static constexpr int CH = HD / 16, LR = 32 / CH, COPIES = SUB / LR;      // chunks of a row, rows a warp copies at once, such copies
  static constexpr unsigned stage_bytes = 2 * SUB * HD, ring = STAGES * stage_bytes, scales = WARPS * ring, q = scales + WARPS * STAGES * NP * 8,
                            total = q + TERMS * KK * 1024;
  static_assert(WARPS == 8, "a warp prepares a row of q");
  static constexpr unsigned OP = HD + 4;                // the warps' results on their way together: [warp][8][OP] in the rings' place
  static constexpr unsigned record = 8 * (HD + 2);      // floats: m[8], l[8], O[8][HD]
  static_assert(WARPS * 8 * OP * 4 <= WARPS * ring, "the results fit the rings");
};
__device__ __forceinline__ uint32_t smem_at(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }
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
// An 8 x 8 matrix of f16, a row's pair of columns per lane, transposed.
__device__ __forceinline__ uint32_t turn8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// 2, 4 or 8 neighbouring dims.
template <int D>
__device__ __forceinline__ void load_dims(const float* p, float (&x)[D]) {
  if constexpr (D == 2) {
    const float2 v = *reinterpret_cast<const float2*>(p);
    x[0] = v.x; x[1] = v.y;
  } else {
#pragma unroll
    for (int e = 0; e < D; e += 4) {
      const float4 v = *reinterpret_cast<const float4*>(p + e);
      x[e] = v.x; x[e + 1] = v.y; x[e + 2] = v.z; x[e + 3] = v.w;
    }
  }
}
template <int D>
__device__ __forceinline__ void load_dims(const __half* p, float (&x)[D]) {
  uint32_t w[D / 2];
  if constexpr (D == 2) w[0] = *reinterpret_cast<const uint32_t*>(p);
  else if constexpr (D == 4) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x; w[1] = v.y;
  } else {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  }
#pragma unroll
  for (int e = 0; e < D; e += 2) {
    const float2 f = __half22float2(q8_h2(w[e / 2]));
    x[e] = f.x; x[e + 1] = f.y;
  }
}

template <int HD, typename T, bool FP8>
__global__ void __launch_bounds__(Split<HD, T>::THREADS, Split<HD, T>::PER_SM) sdpa_q8_split_kernel(const ks_sdpa_q8_args a) {
  using S = Split<HD, T>;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ unsigned scan[S::WARPS], longest[S::WARPS], seq_first, line[2], seq_at;
  __shared__ float row_m[S::WARPS][8], row_l[S::WARPS][8], row_up[8];
  wait_before();
  start_next();
  const unsigned tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, g = lane >> 2, c = lane & 3u;

  // ---- the line of units: a thread counts for up to four neighbouring sequences
  auto tiles_of = [&](const Seq& s) -> unsigned { return (unsigned)max((s.len + S::TILE - 1) / S::TILE - s.begin / S::TILE, 1); };  // (a row that sees nothing still gets its zeros)
  auto units_of = [&](const Seq& s) -> unsigned {
    const unsigned m = (unsigned)s.rows * a.G;
    return m > a.few ? 0u : (m + 7u) / 8u * a.n_kv * tiles_of(s);
  };
  const unsigned per = (a.n_seqs + S::THREADS - 1u) / S::THREADS;
  unsigned mine[KS_PAGES_MAX_SEQS / 256], sum = 0, most = 0;
#pragma unroll
  for (unsigned k = 0; k < KS_PAGES_MAX_SEQS / 256; k++) {
    const unsigned i = tid * per + k;
    Seq s;
    mine[k] = k < per && i < a.n_seqs && seq_of(a, i, s) ? units_of(s) : 0u;
    sum += mine[k];
    if (mine[k]) most = max(most, tiles_of(s));
  }
  unsigned before = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned up = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= (unsigned)o) before += up;
  }
  most = __reduce_max_sync(0xffffffffu, most);
  if (lane == 31u) {
    scan[warp] = before;
    longest[warp] = most;
  }
  __syncthreads();
  unsigned total = 0;
  before -= sum;
#pragma unroll
  for (unsigned w = 0; w < S::WARPS; w++) {
    const unsigned x = scan[w];
    before += w < warp ? x : 0u;
    total += x;
    most = max(most, longest[w]);
  }
  const unsigned least = max((most + kMostParts - 1u) / kMostParts, 1u), blocks = min(gridDim.x, quotient(total + least - 1u, least));
  if (blockIdx.x >= blocks) {
    if (tid == 0) a.merges[2u * blockIdx.x] = make_int4(0, 0, 0, 0);
    return;
  }
  // the first `more` blocks take `each` + 1 units, the others `each`
  const unsigned each = quotient(total, blocks), more = total - each * blocks;
  const unsigned u_begin = blockIdx.x * each + min(blockIdx.x, more), u_end = u_begin + each + (blockIdx.x < more ? 1u : 0u);
  if (tid == 0) {
    line[0] = each;
    line[1] = more;
  }
#pragma unroll
  for (unsigned k = 0; k < KS_PAGES_MAX_SEQS / 256; k++) {
    const unsigned i = tid * per + k;
    if (k < per && i < a.n_seqs) {
      if (u_begin >= before && u_begin - before < mine[k]) {
        seq_at = i;
        seq_first = before;
      }
      before += mine[k];
    }
  }
  __syncthreads();

  unsigned char* ring = smem + warp * S::ring;
  const uint32_t ring_at = smem_at(ring), scales_at = smem_at(smem) + S::scales + warp * (S::STAGES * S::NP * 8);
  const float* scales = reinterpret_cast<const float*>(smem + S::scales) + warp * (S::STAGES * S::NP * 2);
  const float to_log2 = a.scale * 1.44269504088896340736f;

  // ---- piece after piece
  unsigned seq = seq_at, in_block = 0, u = u_begin, at = seq_first;
  Seq s;
  unsigned units = seq_of(a, seq, s) ? units_of(s) : 0u;
  while (u < u_end) {
    while (u - at >= units) {
      at += units;
      units = seq_of(a, ++seq, s) ? units_of(s) : 0u;
    }
    const int tile0 = s.begin / S::TILE, n_tiles = (int)tiles_of(s);
    const unsigned m_rows = (unsigned)s.rows * a.G, m_tiles = (m_rows + 7u) / 8u;
    const unsigned piece = quotient(u - at, (unsigned)n_tiles), t_first = u - at - piece * (unsigned)n_tiles;
    const unsigned kvh = m_tiles == 1u ? piece : quotient(piece, m_tiles), m0 = (piece - kvh * m_tiles) * 8u;
    const unsigned n = min((unsigned)n_tiles - t_first, u_end - u);  // tiles of this piece that are ours
    const int p_first = (tile0 + (int)t_first) * S::TILE + (int)warp * S::SUB;                       // this warp's positions of the first
    const int* table = a.tables + (size_t)seq * a.max_blocks;

    // q: a warp a row, its values in the order in which the codes of a 16-byte read meet them (16 c .. 16 c + 15 of every 64 dims).  f32 rows are
    // brought to 2^14 by a power of two and split into two f16 terms.  (Every warp for itself took 2500 clocks of a one-step call.)
    constexpr int QD = HD / 32;
    float qx[QD];
    {
      const unsigned m = min(m0 + warp, m_rows - 1u);  // (columns behind the last row repeat it)
      load_dims<QD>((const T*)a.q + ((size_t)(s.row0 + (int)(m / a.G)) * a.n_q + kvh * a.G + m % a.G) * HD + QD * lane, qx);
    }
    // the page of 16 positions (a page has no fewer) as the table has it: read a step before it is looked at
    auto page_of = [&](int p) -> int { return p + 15 < s.begin || p >= s.len ? -1 : table[(unsigned)p >> a.page_log]; };
    // copies of SUB positions into stage st: 16 bytes a lane, chunks swapped about so that the reads below meet no bank twice; positions that
    // nobody sees become zeros
    auto send = [&](int p0, const int (&id)[S::NP], unsigned st) {
      const unsigned ch = lane % S::CH, r0 = lane / S::CH;
#pragma unroll
      for (int b = 0; b < S::NP; b++) {
        const int p = p0 + 16 * b;
        const bool page = (unsigned)id[b] < a.n_pages;
        if (!page && p + 15 >= s.begin && p < s.len && lane == 0) atomicOr(a.bad, KS_BAD_PAGE);
        const size_t block = (size_t)(page ? id[b] : 0) * a.n_kv + kvh;
        const size_t from = (((block << a.page_log) + ((unsigned)p & ((1u << a.page_log) - 1u)) + r0) * HD) + ch * 16u;
        const uint32_t to = ring_at + st * S::stage_bytes + (unsigned)b * 16u * HD;
        if (page && p >= s.begin && p + 16 <= s.len) {  // (the usual case: 16 rows follow one another in memory)
          const uint8_t *from_k = a.kc + from, *from_v = a.vc + from;
#pragma unroll
          for (int i = 0; i < S::COPIES / S::NP; i++) {
            const unsigned r = r0 + (unsigned)(i * S::LR);
            const unsigned kch = HD >= 128 ? ch ^ ((r & 1u) << 2) : ch, vch = HD >= 128 ? ch ^ ((r >> 1 & 3u) << 1) : ch ^ ((r >> 1 & 1u) << 1);
            copy16(to + r * HD + kch * 16u, from_k + i * S::LR * HD);
            copy16(to + S::SUB * HD + r * HD + vch * 16u, from_v + i * S::LR * HD);
          }
        } else
#pragma unroll
        for (int i = 0; i < S::COPIES / S::NP; i++) {
          const unsigned r = r0 + (unsigned)(i * S::LR);
          const bool there = page && p + (int)r >= s.begin && p + (int)r < s.len;
          const unsigned kch = HD >= 128 ? ch ^ ((r & 1u) << 2) : ch, vch = HD >= 128 ? ch ^ ((r >> 1 & 3u) << 1) : ch ^ ((r >> 1 & 1u) << 1);
          copy16(to + r * HD + kch * 16u, a.kc + from + (size_t)(i * S::LR) * HD, there);
          copy16(to + S::SUB * HD + r * HD + vch * 16u, a.vc + from + (size_t)(i * S::LR) * HD, there);
        }
        if (lane < 2u) copy4(scales_at + ((st * S::NP + b) * 2u + lane) * 4u, (lane ? a.vs : a.ks) + block, page);
      }
    };
    auto pages = [&](unsigned i, int (&id)[S::NP]) {
#pragma unroll
      for (int b = 0; b < S::NP; b++) id[b] = i < n ? page_of(p_first + (int)i * S::TILE + 16 * b) : -1;
    };
    int ids[S::STAGES][S::NP], id[S::NP];
#pragma unroll
    for (int i = 0; i < S::STAGES; i++) pages((unsigned)i, ids[i]);
#pragma unroll
    for (int i = 0; i < S::STAGES - 1; i++) {
      if ((unsigned)i < n) send(p_first + i * S::TILE, ids[i], (unsigned)i);
      copies_sent();
    }
#pragma unroll
    for (int b = 0; b < S::NP; b++) id[b] = ids[S::STAGES - 1][b];

    // ---- q's terms through shared memory
    uint32_t qb[S::TERMS][S::KK][4][2];
    float up[2] = {1.0f, 1.0f};
    {
      uint32_t* qs = reinterpret_cast<uint32_t*>(smem + S::q);
      float down = 1.0f;
      if constexpr (S::TERMS == 2) {
        float big = 0.0f;
#pragma unroll
        for (int e = 0; e < QD; e++) big = fmaxf(big, fabsf(qx[e]));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
        const int ex = big > 0.0f && big < 3.0e38f ? max((int)(__float_as_uint(big) >> 23) - 127 - 14, -100) : 0;
        down = __uint_as_float((uint32_t)(127 - ex) << 23);
        if (lane == 0) row_up[warp] = __uint_as_float((uint32_t)(127 + ex) << 23);
      }
#pragma unroll
      for (int e = 0; e < QD; e += 2) {
        const unsigned dim = QD * lane + e, kk = dim >> 6, cc = dim >> 4 & 3u, k = dim >> 2 & 3u, h = dim >> 1 & 1u;
        uint32_t* to = qs + ((kk * 2u + (k >> 1)) * 32u + 4u * warp + cc) * 4u + (k & 1u) * 2u + h;
        const float x0 = qx[e] * down, x1 = qx[e + 1] * down;
        const __half2 big = __floats2half2_rn(x0, x1);
        *to = q8_u32(big);
        if constexpr (S::TERMS == 2) {
          const float2 f = __half22float2(big);
          to[S::KK * 256] = q8_u32(__floats2half2_rn(x0 - f.x, x1 - f.y));
        }
      }
      __syncthreads();
#pragma unroll
      for (int t = 0; t < S::TERMS; t++)
#pragma unroll
        for (int kk = 0; kk < S::KK; kk++)
#pragma unroll
          for (int k = 0; k < 4; k += 2) {
            const uint4 w = *reinterpret_cast<const uint4*>(qs + t * S::KK * 256 + ((kk * 2 + k / 2) * 32 + lane) * 4);
            qb[t][kk][k][0] = w.x;
            qb[t][kk][k][1] = w.y;
            qb[t][kk][k + 1][0] = w.z;
            qb[t][kk][k + 1][1] = w.w;
          }
      if constexpr (S::TERMS == 2) {
        up[0] = row_up[2u * c];
        up[1] = row_up[2u * c + 1u];
      }
    }
    // ---- this lane's scores: positions g (+ 8) of query rows 2 c and 2 c + 1, which see positions lo .. hi
    int lo[2], hi[2], lo_all, hi_all;
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const unsigned m = min(m0 + 2u * c + h, m_rows - 1u);  // (columns behind the last row repeat it)
      hi[h] = s.len - s.rows + (int)(m / a.G);
      lo[h] = a.window && hi[h] >= (int)a.window ? hi[h] - (int)a.window + 1 : 0;
    }
    hi_all = s.len - s.rows + (int)(m0 / a.G);
    {
      const int last = s.len - s.rows + (int)(min(m0 + 7u, m_rows - 1u) / a.G);
      lo_all = a.window && last >= (int)a.window ? last - (int)a.window + 1 : 0;
    }
    float m[2] = {kNone, kNone}, l[2] = {0.0f, 0.0f}, acc[S::WN][S::WW][2][4];
#pragma unroll
    for (int w = 0; w < S::WN; w++)
#pragma unroll
      for (int k = 0; k < S::WW; k++)
#pragma unroll
        for (int e = 0; e < 8; e++) acc[w][k][e / 4][e % 4] = 0.0f;

    unsigned st = 0;
    for (unsigned i = 0; i < n; i++) {
      copies_wait<S::STAGES - 2>();
      __syncwarp();
      const int p0 = p_first + (int)i * S::TILE;
      {
        const unsigned to = st == 0 ? S::STAGES - 1 : st - 1u;
        if (i + S::STAGES - 1 < n) send(p0 + (S::STAGES - 1) * S::TILE, id, to);
        copies_sent();
        pages(i + S::STAGES, id);
      }
      const unsigned char* at_k = ring + st * S::stage_bytes;
      const unsigned char* at_v = at_k + S::SUB * HD;
      // scores
      float x[S::NP][4];
#pragma unroll
      for (int b = 0; b < S::NP; b++) {
        float d[2 * S::TERMS][4];
#pragma unroll
        for (int k = 0; k < 2 * S::TERMS; k++)
#pragma unroll
          for (int e = 0; e < 4; e++) d[k][e] = 0.0f;
#pragma unroll
        for (int kk = 0; kk < S::KK; kk++) {
          const unsigned ch = 4u * kk + c, r = 16u * b + g, kch = HD >= 128 ? ch ^ ((g & 1u) << 2) : ch;
          const uint4 u0 = *reinterpret_cast<const uint4*>(at_k + r * HD + kch * 16u), u1 = *reinterpret_cast<const uint4*>(at_k + (r + 8u) * HD + kch * 16u);
          const uint32_t w0[4] = {u0.x, u0.y, u0.z, u0.w}, w1[4] = {u1.x, u1.y, u1.z, u1.w};
#pragma unroll
          for (int k = 0; k < 4; k++) {
            uint32_t af[4];
            widen4<FP8>(w0[k], af[0], af[2]);
            widen4<FP8>(w1[k], af[1], af[3]);
            if constexpr (S::TERMS == 2) mma16816(d[2 + (k & 1)], af, qb[S::TERMS - 1][kk][k][0], qb[S::TERMS - 1][kk][k][1]);
            mma16816(d[k & 1], af, qb[0][kk][k][0], qb[0][kk][k][1]);
          }
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
          x[b][e] = d[0][e] + d[1][e];
          if constexpr (S::TERMS == 2) x[b][e] += d[2][e] + d[2 * S::TERMS - 1][e];
        }
      }
      // probabilities
      float vf[S::NP], vd[S::NP], top[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int b = 0; b < S::NP; b++) {
        const float2 sc = *reinterpret_cast<const float2*>(scales + (st * S::NP + b) * 2);
        const float ks = q8_scale(sc.x) * to_log2;
        float ve;
        split_scale(q8_scale(sc.y), ve, vf[b], vd[b]);
#pragma unroll
        for (int e = 0; e < 4; e++) x[b][e] = fmaf(x[b][e], S::TERMS == 2 ? ks * up[e & 1] : ks, ve);
      }
      if (p0 < lo_all || p0 + S::SUB - 1 > hi_all) {
#pragma unroll
        for (int b = 0; b < S::NP; b++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const int p = p0 + 16 * b + (int)g + (e >> 1) * 8;
            if (p < lo[e & 1] || p > hi[e & 1]) x[b][e] = -INFINITY;
          }
      }
#pragma unroll
      for (int b = 0; b < S::NP; b++)
#pragma unroll
        for (int e = 0; e < 4; e++) top[e & 1] = fmaxf(top[e & 1], x[b][e]);
      if (__any_sync(0xffffffffu, top[0] > m[0] + kSlack || top[1] > m[1] + kSlack)) {
        float turn[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], o));
          top[h] = fmaxf(top[h], m[h]);
          turn[h] = exp2_fast(m[h] - top[h]);
          m[h] = top[h];
          l[h] *= turn[h];
        }
#pragma unroll
        for (int w = 0; w < S::WN; w++)
#pragma unroll
          for (int k = 0; k < S::WW; k++)
#pragma unroll
            for (int e = 0; e < 8; e++) acc[w][k][e / 4][e % 4] *= turn[e & 1];
      }
      uint32_t pb[S::NP][S::TERMS][2];
#pragma unroll
      for (int b = 0; b < S::NP; b++) {
        const float f = vf[b] * kProbs;
        float sum[2];
#pragma unroll
        for (int e = 0; e < 4; e++) x[b][e] = exp2_fast(x[b][e] - m[e & 1]);
        sum[0] = x[b][0] + x[b][2];
        sum[1] = x[b][1] + x[b][3];
        l[0] = fmaf(sum[0], vd[b], l[0]);
        l[1] = fmaf(sum[1], vd[b], l[1]);
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const float y0 = x[b][2 * h] * f, y1 = x[b][2 * h + 1] * f;
          const __half2 big = __floats2half2_rn(y0, y1);
          pb[b][0][h] = turn8x8(q8_u32(big));
          if constexpr (S::TERMS == 2) {
            const float2 t = __half22float2(big);
            pb[b][S::TERMS - 1][h] = turn8x8(q8_u32(__floats2half2_rn(y0 - t.x, y1 - t.y)));
          }
        }
      }
      // values
#pragma unroll
      for (int w = 0; w < S::WN; w++) {
        uint32_t v[S::NP][4][S::WW];
#pragma unroll
        for (int b = 0; b < S::NP; b++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const unsigned r = 16u * b + 2u * c + (e & 1) + (e >> 1) * 8u, byte = w * S::W + g * (S::W / 8), ch = byte >> 4;
            const unsigned vch = HD >= 128 ? ch ^ ((r >> 1 & 3u) << 1) : ch ^ ((r >> 1 & 1u) << 1);
            const unsigned char* from = at_v + r * HD + vch * 16u + (byte & 15u);
            if constexpr (S::WW == 4) {
              const uint4 y = *reinterpret_cast<const uint4*>(from);
              v[b][e][0] = y.x; v[b][e][1] = y.y; v[b][e][2] = y.z; v[b][e][3] = y.w;
            } else {
              const uint2 y = *reinterpret_cast<const uint2*>(from);
              v[b][e][0] = y.x; v[b][e][1] = y.y;
            }
          }
#pragma unroll
        for (int k = 0; k < S::WW; k++) {
          float d[2][4];
#pragma unroll
          for (int b = 0; b < S::NP; b++) {
            uint32_t p01[4], p89[4];
            widen_pairs<FP8>(v[b][0][k], v[b][1][k], p01);
            widen_pairs<FP8>(v[b][2][k], v[b][3][k], p89);
#pragma unroll
            for (int t = 0; t < 2; t++) {
              const uint32_t af[4] = {p01[2 * t], p01[2 * t + 1], p89[2 * t], p89[2 * t + 1]};
              if constexpr (S::TERMS == 2) {
                if (b == 0)
#pragma unroll
                  for (int e = 0; e < 4; e++) d[t][e] = 0.0f;
                mma16816(d[t], af, pb[b][S::TERMS - 1][0], pb[b][S::TERMS - 1][1]);
                mma16816(d[t], af, pb[b][0][0], pb[b][0][1]);
              } else {
                mma16816(acc[w][k][t], af, pb[b][0][0], pb[b][0][1]);
              }
            }
          }
          if constexpr (S::TERMS == 2)
#pragma unroll
            for (int e = 0; e < 8; e++) acc[w][k][e / 4][e % 4] += d[e / 4][e % 4];
        }
      }
      st = st + 1u == S::STAGES ? 0u : st + 1u;
      __syncwarp();  // the stage has been read
    }
    // ---- the warps' results together: to `out`, or a record if other blocks have a part of the piece
    copies_wait<0>();
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], o);
    if (g == 0) {
#pragma unroll
      for (int h = 0; h < 2; h++) {
        row_m[warp][2u * c + h] = m[h];
        row_l[warp][2u * c + h] = l[h];
      }
    }
    __syncthreads();  // every ring is free
    float* mid = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int w = 0; w < S::WN; w++)
#pragma unroll
      for (int k = 0; k < S::WW; k++)
#pragma unroll
        for (int h = 0; h < 2; h++)
          *reinterpret_cast<float4*>(mid + (size_t)(warp * 8u + 2u * c + h) * S::OP + w * S::W + g * (S::W / 8) + 4 * k) =
              make_float4(acc[w][k][0][h], acc[w][k][0][h + 2], acc[w][k][1][h], acc[w][k][1][h + 2]);
    __syncthreads();
    {
      // a warp a row: the lanes share its dims
      const unsigned r = warp, mm = m0 + r;
      float top = kNone, sum = 0.0f, e[S::WARPS];
#pragma unroll
      for (int w = 0; w < S::WARPS; w++) top = fmaxf(top, row_m[w][r]);
#pragma unroll
      for (int w = 0; w < S::WARPS; w++) {
        e[w] = exp2_fast(row_m[w][r] - top);
        sum = fmaf(e[w], row_l[w][r], sum);
      }
      const bool whole = n == (unsigned)n_tiles;
      float* rec = a.part + ((size_t)blockIdx.x * 2u + (in_block ? 1u : 0u)) * S::record;
      if (!whole && lane == 0) {
        rec[r] = top;
        rec[8 + r] = sum;
      }
      const float f = whole ? over(sum) : 1.0f;
      if (mm < m_rows) {
        constexpr int D = HD / 32;
        float v[D];
#pragma unroll
        for (int d = 0; d < D; d++) v[d] = 0.0f;
#pragma unroll
        for (int w = 0; w < S::WARPS; w++) {
          const float* from = mid + (size_t)(w * 8u + r) * S::OP;
          if constexpr (D == 2) {
            const float2 y = *reinterpret_cast<const float2*>(from + 2u * lane);
            v[0] = fmaf(y.x, e[w], v[0]);
            v[1] = fmaf(y.y, e[w], v[1]);
          } else {
#pragma unroll
            for (int d = 0; d < D; d += 4) {
              const float4 y = *reinterpret_cast<const float4*>(from + 4u * lane + 32 * d);
              v[d] = fmaf(y.x, e[w], v[d]);
              v[d + 1] = fmaf(y.y, e[w], v[d + 1]);
              v[d + 2] = fmaf(y.z, e[w], v[d + 2]);
              v[d + 3] = fmaf(y.w, e[w], v[d + 3]);
            }
          }
        }
        T* to = (T*)a.out + ((size_t)(s.row0 + (int)(mm / a.G)) * a.n_q + kvh * a.G + mm % a.G) * HD;
#pragma unroll
        for (int d = 0; d < D; d += D == 2 ? 2 : 4) {
          const unsigned dim = (D == 2 ? 2u : 4u) * lane + 32u * d;
          if (whole) {
#pragma unroll
            for (int k = 0; k < (D == 2 ? 2 : 4); k++) v[d + k] *= f;
            put_dims(to + dim, v + d, D == 2 ? 2 : 4);
          } else {
            put_dims(rec + 16 + r * HD + dim, v + d, D == 2 ? 2 : 4);
          }
        }
      }
    }
    // what the merge has to do for this block: the piece that began in an earlier one and ends here, if there is one
    if (in_block == 0 && tid == 0) {
      const bool ends = t_first > 0 && t_first + n == (unsigned)n_tiles;
      const unsigned u0 = u - t_first, each = line[0], more = line[1], big = more * (each + 1u);
      const unsigned b0 = u0 < big ? quotient(u0, each + 1u) : more + quotient(u0 - big, each), b0_begin = b0 * each + min(b0, more);
      a.merges[2u * blockIdx.x] = make_int4((int)b0, ends ? (int)(blockIdx.x - b0 + 1u) : 0, b0_begin == u0 ? 0 : 1, (int)m0);
      a.merges[2u * blockIdx.x + 1u] = make_int4(s.row0, (int)kvh, (int)m_rows, 0);
    }
    u += n;
    in_block++;
    __syncthreads();  // everything in shared memory is free again
  }
}

// ---- the records of pieces that lie in several blocks ----------------------------------------------------------
// out = sum_b e_b O_b / sum_b e_b l_b, e_b = exp2(m_b - max m), in the order of the blocks.  A block for each of the split kernel's and 64 dims, for the
// piece that ends there; its threads are 8 rows x (up to 8) shares of the records x 16 times 4 dims.
template <int HD, typename T>
__global__ void __launch_bounds__(1024) sdpa_q8_merge_kernel(const ks_sdpa_q8_args a) {
  using S = Split<HD, T>;
  __shared__ float4 red[8][8][16];
  __shared__ float tops[8][8], sums[8][8];
  wait_before();
  start_next();
  const unsigned d = threadIdx.x & 15u, r = threadIdx.x >> 4 & 7u, share = threadIdx.x >> 7, shares = blockDim.x >> 7, dim = blockIdx.y * 64u + 4u * d;
  const int4 job = a.merges[2u * blockIdx.x], where = a.merges[2u * blockIdx.x + 1u];
  const unsigned n = (unsigned)job.y, m = (unsigned)job.w + r;
  if (n == 0u) return;
  const float* rec = a.part + (size_t)job.x * 2u * S::record;
  auto record = [&](unsigned k) { return rec + (k ? k * 2u : (unsigned)job.z) * (size_t)S::record; };  // (the first block's record is its second one unless the piece starts with the block)
  // a share's records four at a time: maxima, sums and values on one trip, then together as a running softmax
  float top = kNone, l = 0.0f;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  const bool live = m < (unsigned)where.z;
  if (live) {
    constexpr unsigned FLY = 4;
    for (unsigned k0 = share; k0 < n; k0 += shares * FLY) {
      float mk[FLY], lk[FLY];
      float4 o[FLY];
#pragma unroll
      for (unsigned f = 0; f < FLY; f++) {
        const bool there = k0 + shares * f < n;
        const float* x = record(there ? k0 + shares * f : k0);
        mk[f] = there ? x[r] : kNone;
        lk[f] = there ? x[8 + r] : 0.0f;
        o[f] = there ? *reinterpret_cast<const float4*>(x + 16 + r * HD + dim) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
      float most = top;
#pragma unroll
      for (unsigned f = 0; f < FLY; f++) most = fmaxf(most, mk[f]);
      const float turn = exp2_fast(top - most);
      top = most;
      l *= turn;
      v.x *= turn; v.y *= turn; v.z *= turn; v.w *= turn;
#pragma unroll
      for (unsigned f = 0; f < FLY; f++) {
        const float e = exp2_fast(mk[f] - top);
        l = fmaf(lk[f], e, l);
        v.x = fmaf(o[f].x, e, v.x);
        v.y = fmaf(o[f].y, e, v.y);
        v.z = fmaf(o[f].z, e, v.z);
        v.w = fmaf(o[f].w, e, v.w);
      }
    }
  }
  if (d == 0) {
    tops[share][r] = top;
    sums[share][r] = l;
  }
  red[share][r][d] = v;
  __syncthreads();
  if (!live || share > 0) return;
  float most = kNone;
  for (unsigned k = 0; k < shares; k++) most = fmaxf(most, tops[k][r]);
  float y[4] = {0.f, 0.f, 0.f, 0.f};
  l = 0.0f;
  for (unsigned k = 0; k < shares; k++) {
    const float e = exp2_fast(tops[k][r] - most);
    const float4 o = red[k][r][d];
    l = fmaf(sums[k][r], e, l);
    y[0] = fmaf(o.x, e, y[0]);
    y[1] = fmaf(o.y, e, y[1]);
    y[2] = fmaf(o.z, e, y[2]);
    y[3] = fmaf(o.w, e, y[3]);
  }
  const float f = over(l);
#pragma unroll
  for (int k = 0; k < 4; k++) y[k] *= f;
  put_dims((T*)a.out + ((size_t)(where.x + (int)(m / a.G)) * a.n_q + (unsigned)where.y * a.G + m % a.G) * HD + dim, y, 4);
}

unsigned split_blocks(const ks_ctx* ctx, size_t hd) { return (unsigned)ctx->sm_count * (hd == 256 ? Split<256, float>::PER_SM : Split<128, float>::PER_SM); }  // as many as run at once

template <int HD, typename T, bool FP8>
int launch_split(ks_ctx* ctx, const ks_sdpa_q8_args& a, unsigned blocks) {
  using S = Split<HD, T>;
  static bool set[16] = {false};
  if (!set[ctx->device & 15]) {
    cudaError_t e = cudaFuncSetAttribute(sdpa_q8_split_kernel<HD, T, FP8>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::total);
    if (e != cudaSuccess) return ks_fail(ctx, KS_ERR_CUDA, "sdpa_paged_q8: cannot set %u B shared memory: %s", S::total, cudaGetErrorString(e));
    set[ctx->device & 15] = true;
  }
  KS_LAUNCH(ctx, (sdpa_q8_split_kernel<HD, T, FP8>), blocks, S::THREADS, S::total, a);
  return ks_after_launch(ctx, "sdpa_paged_q8");
}
template <int HD, typename T>
int launch_split_merge(ks_ctx* ctx, const ks_sdpa_q8_args& a, unsigned blocks) {
  // Many pieces lie in two or three blocks each: small blocks, so that all are there at once; few pieces may lie in up to 64 blocks each.  Calls of single rows
  // with 256 / 1024 threads: 32 sequences of 2000 positions (f16, 8 KV heads of 128) 29.3 / 34.7 us, 48 of about 6800 108 to 110 / 115, one of 16384 (f16, one KV
  // head of 128: one piece in 64 blocks) 13.2 / 12.0, four of up to 16384 (f32, two of 256) 19.0 / 19.2.  Where few pieces lie in few blocks each the line
  // stands too high: one of 700 (f32, one of 256) 9.1 / 10.6, 16 of 600 (f16, four of 128) 10.7 / 13.3, 16 of 4000 20.0 / 22.4.
  const size_t pieces = (size_t)a.n_seqs * a.n_kv * ((a.few + 7u) / 8u);
  KS_LAUNCH(ctx, (sdpa_q8_merge_kernel<HD, T>), dim3(blocks, HD / 64), pieces >= blocks / 4 ? 256 : 1024, 0, a);
  return ks_after_launch(ctx, "sdpa_paged_q8 merge");
}

size_t split_floats(const ks_ctx* ctx, const ks_q8_cache* c) { return (size_t)split_blocks(ctx, c->hd) * (8 + 2 * 8 * (c->hd + 2)); }

// Rows times heads up to which a sequence takes the split kernel: up to 32 always, and up to 512 as long as its blocks have no more than a dozen units
// each.  Above that the wide kernel, which reads codes once for 128 rows instead of 8, is ahead of it: calls of 16, 32, 64, 128 (row, head)s a
// sequence took, split / wide, 12 / 28, 13 / 30, 14 / 31, 19 / 34 us for one sequence of 4000 positions (f32, one KV head of 256; 0.2 to 3.5 units), 19 / 45, 25 / 32,
// 34 / 35, 54 / 39 for four with two KV heads (3.5 to 28), 14 / 29, 16 / 30, 25 / 31, 41 / 26 for sixteen of 600 (f16, four of 128; 2 to 17), 31 / 73, 48 / 77, 86 / 79,
// 160 / 57 for sixteen of 4000 (14 to 110), and 37 / 77, 57 / 54, 101 / 56, 188 / 70 for sixteen of 4000 in f32 with two of 256 (14 to 110).
unsigned few_of(const ks_ctx* ctx, const ks_q8_cache* c, const ks_page_tables* t, size_t ctx_most, size_t window) {
  if (ctx_most > (1u << 30)) ctx_most = 1u << 30;
  const size_t tile = c->hd == 64 ? 256 : 128, seen = window && window < ctx_most ? window : ctx_most, heads = t->n_seqs * c->n_kv;
  const size_t most = 12 * (size_t)split_blocks(ctx, c->hd) / (heads * ((seen + tile - 1) / tile + 1)) * 8, few = most < KS_Q8_FEW ? KS_Q8_FEW : most > 512 ? 512 : most;
  // (units are counted in 32 bits, and contexts may be longer than announced)
  return heads * (few / 8) * ((t->max_blocks * t->page + 127) / 128) < (size_t(1) << 31) ? (unsigned)few : KS_Q8_FEW;
}

}  // namespace

extern "C" {

size_t ks_sdpa_paged_tmp_floats(const ks_ctx* ctx, const ks_q8_cache* c, const ks_page_tables* t, size_t n_q, size_t rows_most) {
  if (!ctx || !c || !t || !c->n_kv || !rows_most || n_q < c->n_kv) return 0;
  const size_t G = n_q / c->n_kv;
  return split_floats(ctx, c) + (rows_most * G > KS_Q8_FEW ? ks_sdpa_q8_wide_floats(ctx, t->n_seqs, t->max_rows, c->n_kv, G, c->hd) : 0);
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
  // units of the split kernel's line are counted in 32 bits
  const size_t tiles_most = (t->max_blocks * t->page + 127) / 128, m_most = (KS_Q8_FEW + 7) / 8;
  if (t->n_seqs * tiles_most >= (size_t(1) << 31) / (m_most * c->n_kv)) return ks_fail(ctx, KS_ERR_UNSUPPORTED, "%s: %zu sequences of up to %zu positions and %zu KV heads are too much for one call", who, t->n_seqs, t->max_blocks * t->page, c->n_kv);
  KS_REQUIRE_DEVICE(ctx, who);
  ks_on_device on(ctx);
  ks_sdpa_q8_args a{};
  a.kc = (const uint8_t*)c->k->dptr;
  a.vc = (const uint8_t*)c->v->dptr;
  a.ks = (const float*)c->k_scale->dptr;
  a.vs = (const float*)c->v_scale->dptr;
  a.lens = (const int*)t->lens->dptr;
  a.tables = (const int*)t->tables->dptr;
  a.row_start = (const int*)t->plan->dptr + ks_plan_parts(t->n_seqs, t->max_rows, t->page).row_start;
  a.q = q->dptr;
  a.out = out->dptr;
  a.merges = (int4*)tmp->dptr;
  a.part = (float*)tmp->dptr + 8 * (size_t)split_blocks(ctx, c->hd);
  // (a lone sequence that may have many rows needs one kernel only, whatever it has)
  const unsigned few = few_of(ctx, c, t, ctx_most, window);
  const bool wide = rows_most * G > few, split = !wide || t->n_seqs > 1;
  a.few = !split ? 0u : wide ? few : (unsigned)(rows_most * G);
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
  const unsigned blocks = split_blocks(ctx, c->hd);
#define KS_AT(HD_, T_, F_) launch_split<HD_, T_, F_>(ctx, a, blocks)
#define KS_AT_T(HD_, F_) (act == KS_F32 ? KS_AT(HD_, float, F_) : KS_AT(HD_, __half, F_))
#define KS_AT_F(HD_) (c->dtype == KS_E4M3 ? KS_AT_T(HD_, true) : KS_AT_T(HD_, false))
  if (split) rc = c->hd == 256 ? KS_AT_F(256) : c->hd == 128 ? KS_AT_F(128) : KS_AT_F(64);
#undef KS_AT_F
#undef KS_AT_T
#undef KS_AT
  float* wide_tmp = (float*)tmp->dptr + split_floats(ctx, c);
  if (!rc && wide) rc = ks_launch_sdpa_q8_wide(ctx, a, c->hd, act, c->dtype == KS_E4M3, wide_tmp, ctx_most, split);
#define KS_AT(HD_) (act == KS_F32 ? launch_split_merge<HD_, float>(ctx, a, blocks) : launch_split_merge<HD_, __half>(ctx, a, blocks))
  if (!rc && split) rc = c->hd == 256 ? KS_AT(256) : c->hd == 128 ? KS_AT(128) : KS_AT(64);
#undef KS_AT
  if (!rc && wide) rc = ks_launch_sdpa_q8_wide_merge(ctx, a, c->hd, act, wide_tmp, ctx_most, split);
  return rc;
}

}  // extern "C"
