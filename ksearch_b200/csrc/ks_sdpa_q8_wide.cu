// Attention of many rows (prompt pieces, long drafts) over a paged 8-bit cache, on tcgen05 (formulas: ks_sdpa_q8.cu).
//
// A block takes 128 query rows (row and query head of the group, counted together), or twice 128 (f16, heads up to 128), of a sequence against one KV
// head and walks over the tiles of TILE positions that they see.  Five kinds of warps hand tiles on through mbarriers:
//   loaders     codes of a tile, page by page, by bulk copies into rings, K by one warp and V by another; what scores and probabilities are
//               scaled by per 16 positions;
//   converters  codes -> f16 (exact) core matrices: K as positions x dims, V transposed as dims x positions, by warps of their own;
//   products    S = q K^T into tensor memory and O (+)= P V with P out of tensor memory;
//   softmax     eight warps: S -> mask, maximum, probabilities -> P.
// The maximum that probabilities refer to moves only when a score exceeds it by 2^4; it is one of scores and V's scales alone, the probabilities' 2^10 comes
// behind it (in the exponent, f16, or as a factor, f32).
//   f16   q as it is, P rounded to f16 (2^-11 of each, as much as the result's rounding), O stays in tensor memory and is rescaled there when the
//         maximum moves.  Its accumulator rounds toward zero: sums of one sign came out smaller by 2^-17 to 2^-16 after 8192 positions, by 2^-11.5 after 65536.
//         Two row tiles share the converted codes (a conversion is worth half the softmax); a thread has a row.  They fill tensor memory: P lies in
//         the place of its scores, half a tile (64 positions) at a time.  While the softmax has one half, the other's values and the next scores in its
//         place are made, for each row tile by a warp of its own.
//   f32   q (first term in tensor memory, second in shared memory) and P are two f16 terms each, small terms first, and O leaves tensor memory
//         after every tile for f32 registers, because its accumulator drops the low bits of what is added.  Two threads share a row and agree by
//         one vote a tile.  (f16 heads of 256 run this way too, with one term and O left where it is.)
//
// Bound by the softmax warps, two a scheduler (f16).  4096 rows behind 4096 (f16, 16 heads on 4 of 128; 206 GFLOP): 236 us, 52 % of the measured peak, 8 % of
// it because blocks see 32 to 64 tiles.  64 positions of both row tiles take some 2050 clocks: 1250 for their exponentials (1024 at the unit's rate; the two
// warps come to them together), 800 until the scores are out of tensor memory, their maximum is known and the probabilities are handed on; products
// 1100 beside them.  Making the warps take turns at the unit: 245 us (their own chain of latencies is as long); every fourth exponential by a polynomial 231,
// every third 244, left out.  Sixteen softmax warps instead of eight were 7 % slower.  Single steps on the way there: products issued
// behind a branch 381 (90 to 130 clocks each, now 32 and up), rings for K and V together 286, 64 positions a tile 284, whole tiles handed on 251.  2047 rows (f32,
// 8 heads on 1 of 256, two splits): 71 us (75 before V's one buffer was handed on by halves), a tile of 128 x 64 2.5 us, 1.1 of them products.
#include "ks_sdpa_q8.cuh"
#include "ks_gemm_common.cuh"

namespace {

constexpr int kRows = 128;
constexpr unsigned kWait = 1u << 20;
constexpr int kWork = 8;  // softmax warps

// Barriers: codes of a ring's stage there (copies) and converted, K and V; scales of a tile there; K, V converted and multiplied; scores there and read;
// probabilities there; values done; all products done.
enum { B_RAW_FULL = 0, B_RAW_FREE = 8, B_SCALE = 16, B_K_FULL = 24, B_K_FREE = 26, B_V_FULL = 28, B_V_FREE = 30, B_S_FULL = 32, B_S_FREE = 36, B_P_FULL = 38, B_PV_DONE = 42, B_DONE = 46, B_COUNT = 48 };

template <int HD_, typename T_>
struct Wide {
  static constexpr int HD = HD_, TERMS = sizeof(T_) == 4 ? 2 : 1;
  static constexpr int QT = TERMS == 1 && HD <= 128 ? 2 : 1, ROWS = QT * kRows;  // tiles of query rows a block takes
  static constexpr int TILE = HD == 256 ? 64 : 128, GROUPS = TILE / 16, COLS = TILE / 2;  // (a softmax thread has COLS positions in registers at a time)
  static constexpr int NK = 2, NV = HD == 256 || QT == 2 ? 1 : 2;                            // buffers of converted K and V
  static constexpr unsigned PIECES = NV == 1 ? 2 : 1;  // a lone buffer of V is handed on, and back, by halves: one is converted while the other is multiplied
  static constexpr int RING = HD == 64 ? 4 : 2;     // tiles of codes
  // The loader of K is RING tiles ahead of its converters at most, those NK ahead of the products and the softmax warps one behind those: a tile's scales are
  // read before their place comes again
  static constexpr int SCALES = RING == 2 ? 6 : 8;
  static_assert(SCALES >= RING + NK + 2 && SCALES <= 8, "scales");
  static constexpr int CONV_K = TERMS == 1 ? 4 : 2, CONV_V = CONV_K, WARPS = kWork + CONV_K + CONV_V + 4, THREADS = WARPS * 32;
  static constexpr int R_WORK = TERMS == 1 ? 136 : 208, R_CONV = TERMS == 1 ? 72 : 64, R_REST = TERMS == 1 ? 56 : 32;
  static_assert(kWork * 32 * R_WORK + (CONV_K + CONV_V) * 32 * R_CONV + 128 * R_REST <= THREADS * (65536 / THREADS / 8 * 8), "registers: the shares fit the launch");
  // shared memory: barriers, the tensor-memory address and the failure flag; per row: scale, maxima of its two threads; per 16 positions: the score's
  // factor, what is added to it, the probability's factor, the sum's
  static constexpr unsigned slot = 384, row = 400, best = row + (TERMS == 2 ? kRows * 4 : 0), scale = best + 2 * kRows * 4, q = (scale + SCALES * GROUPS * 16 + 127) / 128 * 128;
  static_assert(8 * B_COUNT <= slot && slot + 16 <= row, "the words fit in front of the operands");
  static constexpr unsigned q_bytes = kRows * HD * 2, kv_bytes = TILE * HD * 2, k = q + QT * q_bytes, v = k + NK * kv_bytes, raw = v + NV * kv_bytes, raw_bytes = 2 * TILE * HD,
                            total = raw + RING * raw_bytes;
  static_assert(q % 128 == 0 && (TERMS == 1 || q_bytes <= (NK + NV) * kv_bytes), "q's first term passes through K's and V's place");
  static constexpr unsigned OP = HD + 2;
  static_assert(ROWS * OP * 4 <= total - q && total <= 232448, "the result fits the operands, and all of it a block");
  // tensor memory: scores, probabilities (two terms), O, of each row tile; q's first term.  Two row tiles fill it (HD = 128) with the probabilities
  // in the place of the scores' second half
  static constexpr unsigned t_s = 0, t_p = QT == 2 ? t_s : t_s + TILE, t_o = QT == 2 ? t_s + TILE : t_p + TERMS * TILE / 2, t_tile = t_o + HD, t_q = QT * t_tile;
  static_assert(t_q + (TERMS == 2 ? HD / 2 : 0) <= 512, "tensor memory");
  static constexpr unsigned record = ROWS * (HD + 2);  // floats: m[ROWS], l[ROWS], O[ROWS][HD]
};

__device__ __forceinline__ bool mb_test(uint32_t bar, unsigned parity) {  // has the phase ended?
  unsigned ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}
__device__ __forceinline__ void arrive1(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
// `threads` threads (whole warps) meet at barrier `id`: does any, do all of them say so?
__device__ __forceinline__ bool meet_any(unsigned id, unsigned threads, bool x) {
  unsigned r;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, %2, %3, p;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(r) : "r"((unsigned)x), "r"(id), "r"(threads) : "memory");
  return r != 0;
}
__device__ __forceinline__ bool meet_all(unsigned id, unsigned threads, bool x) { return !meet_any(id, threads, !x); }
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ float max3(float x, float y, float z) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
  return r;
}
// Two f32 at once.
__device__ __forceinline__ uint64_t pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 apart(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t x, uint64_t y, uint64_t z) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t x, uint64_t y) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t x, uint64_t y) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
  return r;
}

// Products issued by the elected lane of a warp that runs the code as one: predicates instead of a branch keep addresses and descriptors in
// uniform registers.  A descriptor's low word is its address in 16 bytes
// and the stride between chunks, its high word is the same for all: 128 bytes between groups of 8 rows.
constexpr uint32_t kDescHigh = (128u >> 4) | 1u << 14;
__device__ __forceinline__ uint32_t desc_low(uint32_t smem_addr, unsigned chunk) { return (smem_addr >> 4 & 0x3FFFu) | (chunk >> 4 & 0x3FFFu) << 16; }
__device__ __forceinline__ void issue_ss(unsigned leader, uint32_t d, uint32_t a_low, uint32_t b_low, uint32_t idesc, unsigned add) {
  asm volatile("{\n\t.reg .pred p, q;\n\t.reg .b64 a, b;\n\tsetp.ne.u32 p, %4, 0;\n\tsetp.ne.u32 q, %5, 0;\n\tmov.b64 a, {%1, %6};\n\tmov.b64 b, {%2, %6};\n\t"
               "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d), "r"(a_low), "r"(b_low), "r"(idesc), "r"(add), "r"(leader), "r"(kDescHigh)
               : "memory");
}
__device__ __forceinline__ void issue_ts(unsigned leader, uint32_t d, uint32_t a_tmem, uint32_t b_low, uint32_t idesc, unsigned add) {
  asm volatile("{\n\t.reg .pred p, q;\n\t.reg .b64 b;\n\tsetp.ne.u32 p, %4, 0;\n\tsetp.ne.u32 q, %5, 0;\n\tmov.b64 b, {%2, %6};\n\t"
               "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d), "r"(a_tmem), "r"(b_low), "r"(idesc), "r"(add), "r"(leader), "r"(kDescHigh)
               : "memory");
}
__device__ __forceinline__ void commit_if(unsigned leader, uint32_t bar) {
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %1, 0;\n\t@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar), "r"(leader) : "memory");
}

struct ks_wide_args {
  ks_sdpa_q8_args a;
  unsigned n_splits, share;  // splits of the launch, tiles that one of them takes
  bool beside;
  int4* meta;   // per block of split 0: first row of the sequence, first (row, head) of the tile, how many the sequence has, KV head + 2^16 splits
  float* part;
  unsigned* err;
};

template <int HD, typename T, bool FP8>
__global__ void __launch_bounds__(Wide<HD, T>::THREADS, 1) sdpa_q8_wide_kernel(const __grid_constant__ ks_wide_args wa) {
  using W = Wide<HD, T>;
  constexpr unsigned MMA_WARP = kWork + W::CONV_K + W::CONV_V;
  const ks_sdpa_q8_args& a = wa.a;
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned *scan = reinterpret_cast<unsigned*>(smem + W::best), *mine = reinterpret_cast<unsigned*>(smem + W::slot);  // (before those are what they are called)
  if (!wa.beside) wait_before();
  start_next();
  const unsigned tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
  const unsigned kvh = blockIdx.x % a.n_kv, index = blockIdx.x / a.n_kv, split = blockIdx.y;

  // ---- which tile of which sequence: a thread counts for a few sequences
  {
    constexpr unsigned MOST = (KS_PAGES_MAX_SEQS + W::THREADS - 1) / W::THREADS;
    const unsigned per = (a.n_seqs + W::THREADS - 1u) / W::THREADS;
    unsigned count[MOST], sum = 0;
#pragma unroll
    for (unsigned k = 0; k < MOST; k++) {
      const unsigned i = tid * per + k;
      Seq s;
      count[k] = 0;
      if (k < per && i < a.n_seqs && seq_of(a, i, s) && (unsigned)s.rows * a.G > a.few) count[k] = ((unsigned)s.rows * a.G + W::ROWS - 1u) / W::ROWS;
      sum += count[k];
    }
    unsigned before = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned up = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= (unsigned)o) before += up;
    }
    if (lane == 31u) scan[warp] = before;
    __syncthreads();
    unsigned total = 0;
    before -= sum;
    for (unsigned w = 0; w < W::WARPS; w++) {
      before += w < warp ? scan[w] : 0u;
      total += scan[w];
    }
    if (index >= total) {
      if (split == 0 && tid == 0) wa.meta[blockIdx.x] = make_int4(0, 0, 0, 0);
      wait_before();
      return;
    }
#pragma unroll
    for (unsigned k = 0; k < MOST; k++) {
      if (index >= before && index - before < count[k]) {
        mine[0] = tid * per + k;
        mine[1] = count[k] - 1u - (index - before);  // the last rows see the most: they start first
      }
      before += count[k];
    }
    __syncthreads();
  }
  Seq s;
  const unsigned seq = mine[0];
  seq_of(a, seq, s);
  const unsigned m_rows = (unsigned)s.rows * a.G, m0 = mine[1] * W::ROWS;
  const int* table = a.tables + (size_t)seq * a.max_blocks;
  __syncthreads();

  const uint32_t sb = sm32(smem);
  auto bar = [&](unsigned i) { return sb + 8u * i; };
  uint32_t* tslot = reinterpret_cast<uint32_t*>(smem + W::slot);
  volatile unsigned* fail = reinterpret_cast<volatile unsigned*>(smem + W::slot + 8);
  float* row_scale = reinterpret_cast<float*>(smem + W::row);
  float* best = reinterpret_cast<float*>(smem + W::best);

  // ---- the positions that the rows see, and this split's tiles of them
  const int tok_a = (int)(m0 / a.G), tok_b = (int)(min(m0 + W::ROWS - 1u, m_rows - 1u) / a.G), p_row0 = s.len - s.rows;
  const int seen_from = a.window && p_row0 + tok_a >= (int)a.window ? p_row0 + tok_a - (int)a.window + 1 : 0, seen_to = p_row0 + tok_b + 1;  // (may be below 1: nothing)
  const int first = seen_from & ~(W::TILE - 1), span = seen_to > first ? (seen_to - first + W::TILE - 1) / W::TILE : 0;
  const int n_splits = min(max((span + (int)wa.share - 1) / (int)wa.share, 1), (int)wa.n_splits), share = (span + n_splits - 1) / n_splits;
  if (split == 0 && tid == 0) wa.meta[blockIdx.x] = make_int4(s.row0, (int)m0, (int)m_rows, (int)(kvh | (unsigned)n_splits << 16));
  if ((int)split >= n_splits) {
    wait_before();
    return;
  }
  const int t_begin = first + (int)split * share * W::TILE;
  const unsigned n_tiles = (unsigned)max(min(share, span - (int)split * share), 0);
  const bool whole = n_splits == 1;
  float* rec = wa.part + ((size_t)blockIdx.x * wa.n_splits + split) * W::record;
  auto out_row = [&](unsigned m) { return (T*)a.out + ((size_t)(s.row0 + (int)(m / a.G)) * a.n_q + kvh * a.G + m % a.G) * HD; };
  if (n_tiles == 0u) {  // an empty record, or rows of zeros
    if (!whole) {
      for (unsigned i = tid; i < W::ROWS; i += W::THREADS) {
        rec[i] = kNone;
        rec[W::ROWS + i] = 0.0f;
      }
    } else {
      for (unsigned i = tid; i < W::ROWS * HD; i += W::THREADS)
        if (m0 + i / HD < m_rows) out_row(m0 + i / HD)[i % HD] = (T)0.0f;
    }
    wait_before();
    return;
  }
  const unsigned q_tiles = W::QT == 2 && m0 + kRows < m_rows ? 2u : 1u;  // a second tile of rows only where there are any

  if (tid == 0) {
    for (unsigned i = 0; i < W::RING; i++) {
      mb_init(bar(B_RAW_FULL + i), 1);
      mb_init(bar(B_RAW_FULL + 4u + i), 1);
      mb_init(bar(B_RAW_FREE + i), W::CONV_K);
      mb_init(bar(B_RAW_FREE + 4u + i), W::CONV_V);
    }
    for (unsigned i = 0; i < W::SCALES; i++) mb_init(bar(B_SCALE + i), 1);
    for (unsigned i = 0; i < 2u; i++) {
      mb_init(bar(B_K_FULL + i), W::CONV_K);
      mb_init(bar(B_V_FULL + i), W::CONV_V);
      mb_init(bar(B_K_FREE + i), q_tiles);
      mb_init(bar(B_V_FREE + i), q_tiles);
      mb_init(bar(B_S_FREE + i), kWork);
      mb_init(bar(B_DONE + i), 1);
    }
    for (unsigned i = 0; i < 4u; i++) {
      mb_init(bar(B_S_FULL + i), 1);
      mb_init(bar(B_P_FULL + i), W::QT == 2 ? 4 : kWork);
      mb_init(bar(B_PV_DONE + i), 1);
    }
    *fail = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    proxy_fence();
  }
  if (warp == MMA_WARP) tc_alloc(sm32(tslot), 512);

  // ---- q: a softmax warp takes eight rows at a time, lane = row lane % 8, 8 dims lane / 8 (+ 4 a step): core matrices of 8 rows x 16 bytes.  A
  // negative scale turns q's signs, so that scores are multiplied by something positive
  if (warp < kWork) {
    constexpr int STEPS = HD / 32, GR = W::ROWS / 8 / kWork;
    const uint32_t sign = a.scale < 0.0f ? 0x80008000u : 0u;
#pragma unroll 2
    for (int p = 0; p < GR; p++) {
      const unsigned r = (warp * GR + p) * 8u + (lane & 7u), m = m0 + r;
      const bool in = m < m_rows;
      const T* src = (const T*)a.q + ((size_t)(s.row0 + (int)((in ? m : m0) / a.G)) * a.n_q + kvh * a.G + (in ? m : m0) % a.G) * HD + 8u * (lane >> 3);
      if constexpr (W::TERMS == 1) {
        uint4 v[STEPS];
#pragma unroll
        for (int k = 0; k < STEPS; k++) v[k] = in ? *reinterpret_cast<const uint4*>(src + 32 * k) : make_uint4(0, 0, 0, 0);
        unsigned char* to = smem + W::q + r / kRows * W::q_bytes + r % kRows * 16u;
#pragma unroll
        for (int k = 0; k < STEPS; k++) *reinterpret_cast<uint4*>(to + (4u * k + (lane >> 3)) * kRows * 16u) = make_uint4(v[k].x ^ sign, v[k].y ^ sign, v[k].z ^ sign, v[k].w ^ sign);
      } else {
        float v[STEPS][8], big = 0.0f;
#pragma unroll
        for (int k = 0; k < STEPS; k++) {
          const float4 x = in ? *reinterpret_cast<const float4*>((const float*)src + 32 * k) : make_float4(0.f, 0.f, 0.f, 0.f);
          const float4 y = in ? *reinterpret_cast<const float4*>((const float*)src + 32 * k + 4) : make_float4(0.f, 0.f, 0.f, 0.f);
          v[k][0] = x.x; v[k][1] = x.y; v[k][2] = x.z; v[k][3] = x.w;
          v[k][4] = y.x; v[k][5] = y.y; v[k][6] = y.z; v[k][7] = y.w;
          big = fmaxf(big, absmax8(v[k]));
        }
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 8));
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 16));
        float up;
        const float down = row_scale_down(big, &up);
        if (lane < 8u) row_scale[r] = up;
#pragma unroll
        for (int k = 0; k < STEPS; k++) {
#pragma unroll
          for (int e = 0; e < 8; e++) v[k][e] *= sign ? -down : down;
          uint4 hi, lo;
          split8(v[k], hi, lo);
          const unsigned at = ((4u * k + (lane >> 3)) * kRows + r) * 16u;
          *reinterpret_cast<uint4*>(smem + W::k + at) = hi;
          *reinterpret_cast<uint4*>(smem + W::q + at) = lo;
        }
      }
    }
  }
  proxy_fence();
  __syncthreads();
  if (*tslot != 0u && tid == 0) *fail = 1;  // all 512 columns were asked for: they start at 0
  // softmax warps: a row a thread (two row tiles), or half the columns of a row
  const unsigned quad = warp & 3u, part = warp >> 2 & 1u, qt = W::QT == 2 ? part : 0u, half = W::QT == 2 ? 0u : part, row = quad * 32u + lane, r_all = qt * kRows + row;
  const uint32_t tlane = (quad << 21) + qt * W::t_tile;  // 32 rows a warp, in the address bits of the lane
  if constexpr (W::TERMS == 2) {
    if (warp < kWork) {
#pragma unroll
      for (unsigned k = 0; k < HD / 16u; k += 2u) {
        const unsigned c = half * (HD / 16u) + k;
        const uint4 x = *reinterpret_cast<const uint4*>(smem + W::k + (c * kRows + row) * 16u), y = *reinterpret_cast<const uint4*>(smem + W::k + ((c + 1u) * kRows + row) * 16u);
        const uint32_t w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
        tc_st8(tlane + W::t_q + c * 4u, w);
      }
      tc_wait_st();
    }
    tc_fence_before();
    __syncthreads();  // K's and V's place has been read
    tc_fence_after();
  }

  if (warp < kWork) {
    // ---- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(W::R_WORK));
    constexpr int COLS = W::COLS, HALF = HD / (W::QT == 2 ? 1 : 2);
    const float up = W::TERMS == 2 ? row_scale[row] : 1.0f;
    // this row sees positions lo .. hi (nothing behind the last row)
    const int hi = m0 + r_all < m_rows ? p_row0 + (int)((m0 + r_all) / a.G) : -1, lo = a.window && hi >= (int)a.window ? hi - (int)a.window + 1 : 0;
    auto factor = [&](float f) { return W::TERMS == 2 ? fmaxf(f * up, 1.0e-37f) : f; };  // (a masked score is -infinity: never 0)
    float ref = kNone, l = 0.0f;
    float acc[W::TERMS == 2 ? HALF : 1];
    if constexpr (W::TERMS == 2)
#pragma unroll
      for (int c = 0; c < HALF; c++) acc[c] = 0.0f;
    auto fold = [&] {  // f32: a tile's values into registers
      tc_fence_after();
      if constexpr (W::TERMS == 2) {
#pragma unroll
        for (int c = 0; c < HALF; c += 16) {
          uint32_t o[16];
          tc_ld16(tlane + W::t_o + half * HALF + c, o);
          tc_wait_ld16(o);
#pragma unroll
          for (int e = 0; e < 16; e++) acc[c + e] += __uint_as_float(o[e]);
        }
      }
    };
    bool ok = true;
    const unsigned my_tiles = qt < q_tiles ? n_tiles : 0u;
    const int all_lo = __reduce_max_sync(0xffffffffu, lo), all_hi = __reduce_min_sync(0xffffffffu, hi);  // every row of the warp sees these
    // COLS scores of positions p and up, masked
    auto fetch = [&](uint32_t (&r)[COLS / 16][16], uint32_t from, int p) {
#pragma unroll
      for (int c = 0; c < COLS / 16; c++) tc_ld16(from + 16u * c, r[c]);
#pragma unroll
      for (int c = 0; c < COLS / 16; c++) tc_wait_ld16(r[c]);
      if (p < all_lo || p + COLS - 1 > all_hi) {
#pragma unroll
        for (int c = 0; c < COLS; c++)
          if (p + c < lo || p + c > hi) r[c / 16][c % 16] = 0xFF800000u;  // -infinity
      }
    };
    auto largest = [&](const uint32_t (&r)[COLS / 16][16], const float4* scale) {
      float top = kNone;
#pragma unroll
      for (int c = 0; c < COLS / 16; c++) {
        float g = max3(__uint_as_float(r[c][0]), __uint_as_float(r[c][1]), __uint_as_float(r[c][2])), g2 = max3(__uint_as_float(r[c][3]), __uint_as_float(r[c][4]), __uint_as_float(r[c][5]));
#pragma unroll
        for (int e = 6; e < 14; e += 4) {
          g = max3(g, __uint_as_float(r[c][e]), __uint_as_float(r[c][e + 1]));
          g2 = max3(g2, __uint_as_float(r[c][e + 2]), __uint_as_float(r[c][e + 3]));
        }
        g = max3(fmaxf(g, g2), __uint_as_float(r[c][14]), __uint_as_float(r[c][15]));
        top = fmaxf(top, fmaf(g, factor(scale[c].x), scale[c].y));
      }
      return top;
    };
    if constexpr (W::QT == 2) {
      // What a half needs is asked for while the half before is stored: whether its scores are there, and its scales
      float4 sc[COLS / 16];
      auto scales_at = [&](unsigned i, unsigned h) { return reinterpret_cast<const float4*>(smem + W::scale) + i % W::SCALES * W::GROUPS + h * (W::GROUPS / 2); };
      auto scales_there = [&](unsigned i) { return __all_sync(0xffffffffu, mb_wait(bar(B_SCALE + i % W::SCALES), i / W::SCALES & 1u, kWait)); };
      bool early = false, early_scales = false;  // they are
      ok = my_tiles == 0u || scales_there(0);
      if (ok)
#pragma unroll
        for (int c = 0; c < COLS / 16; c++) sc[c] = scales_at(0, 0)[c];
      for (unsigned i = 0; ok && i < my_tiles; i++) {
#pragma unroll 1
        for (unsigned h = 0; h < 2u; h++) {
          ok = __all_sync(0xffffffffu, early) || __all_sync(0xffffffffu, mb_wait(bar(B_S_FULL + 2u * qt + h), i & 1u, kWait));
          if (!ok) break;
          const uint32_t at = tlane + W::t_s + h * COLS;
          uint32_t r[COLS / 16][16];
          tc_fence_after();
          fetch(r, at, t_begin + (int)(i * W::TILE + h * COLS));
          const float top = largest(r, sc);
          if (__any_sync(0xffffffffu, top > ref + kSlack)) {
            const float turn = exp2_fast(ref - fmaxf(top, ref));
            ref = fmaxf(top, ref);
            l *= turn;
            if (i + h > 0u) {  // O may be touched once the half before's values are done; the next ones wait for these probabilities
              ok = __all_sync(0xffffffffu, mb_wait(bar(B_PV_DONE + 2u * qt + (h ^ 1u)), (h ? i : i - 1u) & 1u, kWait));
              if (!ok) break;
              tc_fence_after();
#pragma unroll 1
              for (unsigned c = 0; c < HALF; c += 8u) {
                uint32_t o[8];
                tc_ld8(tlane + W::t_o + c, o);
#pragma unroll
                for (int e = 0; e < 8; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * turn);
                tc_st8(tlane + W::t_o + c, o);
              }
            }
          }
          // 16 columns' exponentials run while the 16 before are summed, packed and stored (in the scores' place)
          auto powers = [&](int c) {
            const float d = sc[c].y + (kProbsLog2 - ref);
            const uint64_t ff = pair(sc[c].x, sc[c].x), dd = pair(d, d);
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
              const float2 y = apart(fma2(pair(__uint_as_float(r[c][e]), __uint_as_float(r[c][e + 1])), ff, dd));
              r[c][e] = __float_as_uint(exp2_fast(y.x));
              r[c][e + 1] = __float_as_uint(exp2_fast(y.y));
            }
          };
          powers(0);
#pragma unroll
          for (int c = 0; c < COLS / 16; c++) {
            if (c + 1 < COLS / 16) powers(c + 1);
            if (c == 1) {
              early = mb_test(bar(B_S_FULL + 2u * qt + (h ^ 1u)), (i + h) & 1u);
              early_scales = mb_test(bar(B_SCALE + (i + 1u) % W::SCALES), (i + 1u) / W::SCALES & 1u);
            }
            uint64_t sum = 0, sum2 = 0;
            uint32_t w[8];
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
              const float y0 = __uint_as_float(r[c][e]), y1 = __uint_as_float(r[c][e + 1]);
              if (e & 2) sum2 = add2(sum2, pair(y0, y1));
              else sum = add2(sum, pair(y0, y1));
              w[e / 2] = q8_u32(__floats2half2_rn(y0, y1));  // (V's scale is in the exponent)
            }
            const float2 t = apart(add2(sum, sum2));
            l = fmaf(t.x + t.y, sc[c].w, l);
            tc_st8(at + 8u * c, w);
          }
          tc_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive1(bar(B_P_FULL + 2u * qt + h));
          if (h == 1u && i + 1u == my_tiles) break;
          if (h == 1u && !__all_sync(0xffffffffu, early_scales)) {
            ok = scales_there(i + 1u);
            if (!ok) break;
          }
#pragma unroll
          for (int c = 0; c < COLS / 16; c++) sc[c] = scales_at(i + h, h ^ 1u)[c];
        }
      }
    } else {
      for (unsigned i = 0; i < my_tiles; i++) {
        ok = __all_sync(0xffffffffu, mb_wait(bar(B_SCALE + i % W::SCALES), i / W::SCALES & 1u, kWait)) && __all_sync(0xffffffffu, mb_wait(bar(B_S_FULL), i & 1u, kWait));
        uint32_t r[COLS / 16][16];
        float top = kNone;
        const float4* scale = reinterpret_cast<const float4*>(smem + W::scale) + i % W::SCALES * W::GROUPS + half * (W::GROUPS / 2);
        const int p0 = t_begin + (int)i * W::TILE + (int)half * COLS;
        if (ok) {
          tc_fence_after();
          fetch(r, tlane + W::t_s + half * COLS, p0);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive1(bar(B_S_FREE));
          top = largest(r, scale);
        }
        float turn = 1.0f;
        bool turned = false;
        if (meet_any(1u + quad, 64u, !ok || top > ref + kSlack)) {  // the two warps that share 32 rows
          best[half * kRows + row] = top;
          if (!meet_all(1u + quad, 64u, ok)) {
            ok = false;
            break;
          }
          top = fmaxf(fmaxf(top, best[(half ^ 1u) * kRows + row]), ref);
          turn = exp2_fast(ref - top);
          ref = top;
          l *= turn;
          turned = true;
        }
        uint32_t pl[W::TERMS == 2 ? COLS / 2 : 1];
#pragma unroll
        for (int c = 0; c < COLS / 16; c++) {
          const float4 sc = scale[c];
          const float f = factor(sc.x), d = sc.y + (W::TERMS == 1 ? kProbsLog2 - ref : -ref);
          const uint64_t ff = pair(f, f), dd = pair(d, d);
          uint64_t sum = 0;
#pragma unroll
          for (int e = 0; e < 16; e += 2) {
            const float2 y = apart(fma2(pair(__uint_as_float(r[c][e]), __uint_as_float(r[c][e + 1])), ff, dd));
            const float y0 = exp2_fast(y.x), y1 = exp2_fast(y.y);
            const uint64_t yy = pair(y0, y1);
            sum = add2(sum, yy);
            if constexpr (W::TERMS == 1) {
              r[c][e / 2] = q8_u32(__floats2half2_rn(y0, y1));  // (V's scale is in the exponent)
            } else {
              const float2 z = apart(mul2(yy, pair(sc.z, sc.z)));
              const __half2 h = __floats2half2_rn(z.x, z.y);
              const float2 b = __half22float2(h);
              r[c][e / 2] = q8_u32(h);
              pl[c * 8 + e / 2] = q8_u32(__floats2half2_rn(z.x - b.x, z.y - b.y));
            }
          }
          const float2 t = apart(sum);
          l = fmaf(t.x + t.y, sc.w, l);
        }
        // the tile before's values are done: P's place is free, O may be touched
        if (i > 0) ok = __all_sync(0xffffffffu, mb_wait(bar(B_PV_DONE), (i - 1u) & 1u, kWait));
        if (ok && i > 0) {
          if constexpr (W::TERMS == 2) {
            fold();
            if (turned)
#pragma unroll
              for (int c = 0; c < HALF; c++) acc[c] *= turn;
          } else if (turned) {
            tc_fence_after();
#pragma unroll 1
            for (unsigned c = 0; c < HALF; c += 8u) {
              uint32_t o[8];
              tc_ld8(tlane + W::t_o + half * HALF + c, o);
#pragma unroll
              for (int e = 0; e < 8; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * turn);
              tc_st8(tlane + W::t_o + half * HALF + c, o);
            }
          }
        }
        if (ok) {
#pragma unroll
          for (int c = 0; c < COLS / 16; c++) {
            const uint32_t w[8] = {r[c][0], r[c][1], r[c][2], r[c][3], r[c][4], r[c][5], r[c][6], r[c][7]};
            tc_st8(tlane + W::t_p + half * (COLS / 2) + 8 * c, w);
            if constexpr (W::TERMS == 2) {
              const uint32_t z[8] = {pl[8 * c], pl[8 * c + 1], pl[8 * c + 2], pl[8 * c + 3], pl[8 * c + 4], pl[8 * c + 5], pl[8 * c + 6], pl[8 * c + 7]};
              tc_st8(tlane + W::t_p + W::TILE / 2 + half * (COLS / 2) + 8 * c, z);
            }
          }
          tc_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive1(bar(B_P_FULL));
        }
      }
    }
    if (my_tiles) ok = ok && __all_sync(0xffffffffu, mb_wait(bar(B_PV_DONE + (W::QT == 2 ? 2u * qt + 1u : 0u)), (n_tiles - 1u) & 1u, kWait));
    if (!ok && lane == 0) *fail = 1;
    // ---- the rows through shared memory, so that they leave in whole lines; every product that read it is done.  Column n of O is dim
    // 4 (n mod HD / 4) + n / (HD / 4)
    if constexpr (W::QT == 1) best[half * kRows + row] = l;
    if (meet_all(5u, kWork * 32u, ok)) {
      if constexpr (W::QT == 1) l = best[row] + best[kRows + row];
      if (my_tiles) {
        const float f = whole ? over(l) : 1.0f;
        float* to = reinterpret_cast<float*>(smem + W::q) + (size_t)r_all * W::OP + 2u * half;
        if constexpr (W::TERMS == 2) {
          fold();
#pragma unroll
          for (int c = 0; c < HD / 4; c++) *reinterpret_cast<float2*>(to + 4 * c) = make_float2(acc[c] * f, acc[c + HD / 4] * f);
        } else {
          tc_fence_after();
#pragma unroll 1
          for (unsigned h = 0; h < (W::QT == 2 ? 2u : 1u); h++)
#pragma unroll 1
            for (unsigned c = 0; c < HD / 4u; c += 8u) {
              uint32_t o0[8], o1[8];
              tc_ld8(tlane + W::t_o + (half + h) * (HD / 2) + c, o0);
              tc_ld8(tlane + W::t_o + (half + h) * (HD / 2) + HD / 4u + c, o1);
#pragma unroll
              for (int e = 0; e < 8; e++) *reinterpret_cast<float2*>(to + 2u * h + 4u * (c + e)) = make_float2(__uint_as_float(o0[e]) * f, __uint_as_float(o1[e]) * f);
            }
        }
        if (!whole && half == 0) {
          rec[r_all] = ref;
          rec[W::ROWS + r_all] = l;
        }
      }
      meet_all(5u, kWork * 32u, true);
      const float* from = reinterpret_cast<const float*>(smem + W::q);
      const unsigned end = min((unsigned)W::ROWS, m_rows - m0);
#pragma unroll 2
      for (unsigned r = warp; r < end; r += kWork) {
        float2 v[HD / 64];
#pragma unroll
        for (int k = 0; k < HD / 64; k++) v[k] = *reinterpret_cast<const float2*>(from + (size_t)r * W::OP + 2u * lane + 64 * k);
        T* o = out_row(m0 + r);
        float* rr = rec + 2 * W::ROWS + (size_t)r * HD;
#pragma unroll
        for (int k = 0; k < HD / 64; k++) {
          const float y[2] = {v[k].x, v[k].y};
          if (whole) put_dims(o + 2u * lane + 64 * k, y, 2);
          else put_dims(rr + 2u * lane + 64 * k, y, 2);
        }
      }
    }
  } else if (warp < MMA_WARP) {
    // ---- codes -> f16 core matrices, K and V by warps of their own
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(W::R_CONV));
    const bool keys = warp < kWork + W::CONV_K;
    const unsigned cw = warp - kWork - (keys ? 0u : W::CONV_K), kv4 = keys ? 0u : 4u;
    unsigned done = 0;
    for (unsigned i = 0; i < n_tiles; i++) {
      const unsigned char* raw = smem + W::raw + i % W::RING * W::raw_bytes;
      if (!__all_sync(0xffffffffu, mb_wait(bar(B_RAW_FULL + kv4 + i % W::RING), i / W::RING & 1u, kWait))) break;
      if (keys) {
        const unsigned b = i % W::NK;
        if (i >= W::NK && !__all_sync(0xffffffffu, mb_wait(bar(B_K_FREE + b), (i / W::NK - 1u) & 1u, kWait))) break;
        unsigned char* to = smem + W::k + b * W::kv_bytes;
        // 32 rows and one 16-byte chunk of each, a different one for neighbouring lanes: neither the read nor the writes meet a bank twice
        constexpr unsigned CH = HD / 16, STEPS = W::TILE / 32 * CH, PER = STEPS / W::CONV_K, RUN = HD == 64 ? 4 : 8;
        static_assert(STEPS % W::CONV_K == 0 && (PER % CH == 0 || CH % PER == 0), "steps of a warp");
        const unsigned n0 = cw * PER, r0 = n0 / CH * 32u + lane, k0 = n0 % CH, turn = HD == 64 ? lane >> 1 : lane;
#pragma unroll 4
        for (unsigned j = 0; j < PER; j++) {
          const unsigned r = r0 + j / CH * 32u, k = k0 + j % CH, ch = k / RUN * RUN + (turn + k) % RUN;
          const uint4 w = *reinterpret_cast<const uint4*>(raw + r * HD + ch * 16u);
          uint4 x, y;
          widen4<FP8>(w.x, x.x, x.y);
          widen4<FP8>(w.y, x.z, x.w);
          widen4<FP8>(w.z, y.x, y.y);
          widen4<FP8>(w.w, y.z, y.w);
          *reinterpret_cast<uint4*>(to + (2u * ch * W::TILE + r) * 16u) = x;
          *reinterpret_cast<uint4*>(to + ((2u * ch + 1u) * W::TILE + r) * 16u) = y;
        }
      } else {
        raw += W::TILE * HD;
        // eight positions and four dims a lane; dim 4 w + j becomes column j HD / 4 + w of O, so that neighbouring lanes write neighbouring chunks.  A lone
        // buffer's halves are handed on one by one
        constexpr unsigned PIECES = W::PIECES, WORDS = HD / 4, PARTS = WORDS >= 32 ? WORDS / 32 : 1, PG = WORDS >= 32 ? 1 : 2, STEPS = W::TILE / PIECES / 8 * WORDS / 32, PER = STEPS / W::CONV_V;
        static_assert(STEPS % W::CONV_V == 0, "steps of a warp");
        bool there = true;
#pragma unroll
        for (unsigned h = 0; h < PIECES; h++) {
          const unsigned b = PIECES == 2 ? h : i % W::NV, turn = PIECES == 2 ? i : i / W::NV;  // the buffer, and which time it is used
          if (turn > 0u && !__all_sync(0xffffffffu, mb_wait(bar(B_V_FREE + b), (turn - 1u) & 1u, kWait))) {
            there = false;
            break;
          }
          unsigned char* to = smem + W::v + b * (W::kv_bytes / PIECES);
          const unsigned char* half_at = raw + h * (W::TILE / PIECES) * HD;
#pragma unroll 2
          for (unsigned j = 0; j < PER; j++) {
            const unsigned n = cw * PER + j, w = PG == 2 ? lane & 15u : n % PARTS * 32u + lane, pg = PG == 2 ? 2u * n + (lane >> 4) : n / PARTS;
            uint32_t v[8], p[4][4];
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = *reinterpret_cast<const uint32_t*>(half_at + (8u * pg + e) * HD + 4u * w);
#pragma unroll
            for (int e = 0; e < 4; e++) widen_pairs<FP8>(v[2 * e], v[2 * e + 1], p[e]);
#pragma unroll
            for (int j = 0; j < 4; j++) *reinterpret_cast<uint4*>(to + (pg * HD + j * WORDS + w) * 16u) = make_uint4(p[0][j], p[1][j], p[2][j], p[3][j]);
          }
          proxy_fence();
          __syncwarp();
          if (lane == 0) arrive1(bar(B_V_FULL + b));
        }
        if (!there) break;
      }
      if (keys) {
        proxy_fence();
        __syncwarp();
        if (lane == 0) arrive1(bar(B_K_FULL + i % W::NK));
      }
      if (lane == 0) arrive1(bar(B_RAW_FREE + kv4 + i % W::RING));
      done++;
    }
    if (done < n_tiles && lane == 0) *fail = 1;
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(W::R_REST));
    if (warp == MMA_WARP || (W::QT == 2 && warp == MMA_WARP + 3u && q_tiles == 2u)) {
      // ---- products, of each row tile by a warp
      const unsigned leader = elect_one(), tiles = __reduce_max_sync(0xffffffffu, n_tiles), t = __reduce_max_sync(0xffffffffu, warp == MMA_WARP ? 0u : 1u);
      constexpr unsigned COLS_S = W::TILE / W::QT;  // positions of the scores that are made at a time
      constexpr uint32_t idesc_s = (1u << 4) | ((COLS_S >> 3) << 17) | ((kRows >> 4) << 24), idesc_o = (1u << 4) | ((HD >> 3) << 17) | ((kRows >> 4) << 24);
      auto wait = [&](unsigned b, unsigned parity) { return __all_sync(0xffffffffu, mb_wait(bar(b), parity & 1u, kWait)); };
      const uint32_t base = __reduce_max_sync(0xffffffffu, sb);
      const uint32_t d_q = desc_low(base + W::q + t * W::q_bytes, kRows * 16u), d_k = desc_low(base + W::k, W::TILE * 16u), d_v = desc_low(base + W::v, HD * 16u);
      auto scores = [&](unsigned i, unsigned h) {  // of a tile, or of half of one
        const uint32_t k = d_k + i % W::NK * (W::kv_bytes / 16u) + h * COLS_S, to = t * W::t_tile + W::t_s + h * COLS_S;
#pragma unroll
        for (unsigned ks = 0; ks < HD / 16u; ks++) issue_ss(leader, to, d_q + 2u * ks * kRows, k + 2u * ks * W::TILE, idesc_s, ks ? 1u : 0u);
        if constexpr (W::TERMS == 2)
#pragma unroll
          for (unsigned ks = 0; ks < HD / 16u; ks++) issue_ts(leader, to, W::t_q + 8u * ks, k + 2u * ks * W::TILE, idesc_s, 1u);
        commit_if(leader, base + 8u * (B_S_FULL + 2u * t + h));
        if (h + 1u == W::QT) commit_if(leader, base + 8u * (B_K_FREE + i % W::NK));
      };
      bool ok = wait(B_K_FULL, 0u);
      if (ok) {
        tc_fence_after();
#pragma unroll
        for (unsigned h = 0; h < W::QT; h++) scores(0, h);
      }
      for (unsigned i = 0; ok && i < tiles; i++) {
        if constexpr (W::QT == 2) {
          // half by half: while the softmax has one, the values of the other and, in their probabilities' place, its next scores are made
#pragma unroll
          for (unsigned h = 0; h < 2u; h++) {
            ok = ok && wait(B_V_FULL + h, i) && wait(B_P_FULL + 2u * t + h, i);
            if (!ok) continue;
            tc_fence_after();
#pragma unroll
            for (unsigned ks = 0; ks < COLS_S / 16u; ks++)
              issue_ts(leader, t * W::t_tile + W::t_o, t * W::t_tile + W::t_p + h * COLS_S + 8u * ks, d_v + h * (W::kv_bytes / 32u) + 2u * ks * HD, idesc_o, ks | h ? 1u : i);
            commit_if(leader, base + 8u * (B_PV_DONE + 2u * t + h));
            commit_if(leader, base + 8u * (B_V_FREE + h));
            if (i + 1u < tiles) {
              ok = (h || wait(B_K_FULL + (i + 1u) % W::NK, (i + 1u) / W::NK)) && wait(B_PV_DONE + 2u * t + h, i);
              if (!ok) continue;
              tc_fence_after();
              scores(i + 1u, h);
            }
          }
        } else {
          if (i + 1u < tiles) {  // the next scores in front of these values
            ok = wait(B_K_FULL + (i + 1u) % W::NK, (i + 1u) / W::NK) && wait(B_S_FREE, i);
            if (!ok) continue;
            tc_fence_after();
            scores(i + 1u, 0);
          }
          ok = wait(B_P_FULL, i);
          if (!ok) continue;
#pragma unroll
          for (unsigned h = 0; h < W::PIECES; h++) {
            const unsigned b = W::PIECES == 2 ? h : i % W::NV;
            ok = ok && wait(B_V_FULL + b, W::PIECES == 2 ? i : i / W::NV);
            if (!ok) continue;
            tc_fence_after();
            const uint32_t v = d_v + b * (W::kv_bytes / W::PIECES / 16u);
            constexpr unsigned STEPS = W::TILE / 16 / W::PIECES;
            if constexpr (W::TERMS == 2)
#pragma unroll
              for (unsigned ks = 0; ks < STEPS; ks++) issue_ts(leader, W::t_o, W::t_p + W::TILE / 2 + 8u * (h * STEPS + ks), v + 2u * ks * HD, idesc_o, h | ks ? 1u : 0u);
#pragma unroll
            for (unsigned ks = 0; ks < STEPS; ks++) issue_ts(leader, W::t_o, W::t_p + 8u * (h * STEPS + ks), v + 2u * ks * HD, idesc_o, W::TERMS == 2 || h | ks ? 1u : i);
            commit_if(leader, base + 8u * (B_V_FREE + b));
          }
          if (!ok) continue;
          commit_if(leader, base + 8u * B_PV_DONE);
        }
      }
      if (leader) {  // every product issued must finish before shared and tensor memory go away (bounded)
        if (!ok) *fail = 1;
        tc_commit(bar(B_DONE + t));
      }
      __syncwarp();
      mb_wait(bar(B_DONE + t), 0u, kWait);
    } else if (warp == MMA_WARP + 1u || warp == MMA_WARP + 2u) {
      // ---- codes, K and the scales by one warp, V by another: the runs of a tile that lie in one page, a lane each
      const bool keys = warp == MMA_WARP + 1;
      const unsigned kv4 = keys ? 0u : 4u;
      const uint8_t* codes = keys ? a.kc : a.vc;
      const unsigned page = 1u << a.page_log, run = min(page, (unsigned)W::TILE), runs = W::TILE / run;
      auto page_of = [&](unsigned i) -> int {  // as the table has it, -1 where no row of the block sees the run
        const int p = t_begin + (int)(i * W::TILE + lane * run);
        return i < n_tiles && lane < runs && p < seen_to && p + (int)run > seen_from ? table[(unsigned)p >> a.page_log] : -1;
      };
      auto checked = [&](unsigned i, int id) -> int {
        if ((unsigned)id < a.n_pages) return id;
        const int p = t_begin + (int)(i * W::TILE + lane * run);
        if (keys && i < n_tiles && lane < runs && p < seen_to && p + (int)run > seen_from) atomicOr(a.bad, KS_BAD_PAGE);
        return -1;
      };
      auto scales_of = [&](int id) -> float2 {  // of 16 positions
        const int gid = __shfl_sync(0xffffffffu, id, lane * 16u / run);
        const size_t at = (size_t)max(gid, 0) * a.n_kv + kvh;
        return keys && lane < W::GROUPS && gid >= 0 ? make_float2(a.ks[at], a.vs[at]) : make_float2(0.0f, 0.0f);
      };
      // a tile's pages are read two tiles ahead, its scales one
      unsigned sent = 0;
      int id = checked(0, page_of(0)), next = page_of(1);
      float2 sc = scales_of(id);
      for (unsigned i = 0; i < n_tiles; i++) {
        const unsigned st = i % W::RING;
        const int p = t_begin + (int)(i * W::TILE + lane * run);
        const unsigned there = __popc(__ballot_sync(0xffffffffu, id >= 0));
        if (i >= W::RING && !__all_sync(0xffffffffu, mb_wait(bar(B_RAW_FREE + kv4 + st), (i / W::RING - 1u) & 1u, kWait))) break;
        if (lane == 0) mb_expect(bar(B_RAW_FULL + kv4 + st), there * run * HD);
        __syncwarp();
        if (id >= 0) {
          const size_t from = ((((size_t)id * a.n_kv + kvh) << a.page_log) + ((unsigned)p & (page - 1u))) * HD;
          bulk_in(sb + W::raw + st * W::raw_bytes + (keys ? 0u : W::TILE * HD) + lane * run * HD, codes + from, run * HD, bar(B_RAW_FULL + kv4 + st));
        }
        sent++;
        if (keys && lane < W::GROUPS) {
          const float f = fmaxf(q8_scale(sc.x) * fabsf(a.scale) * 1.44269504088896340736f, 1.0e-37f);
          float4 w;
          if constexpr (W::TERMS == 1) {
            const float x = fmaxf(q8_scale(sc.y), 0x1p-60f);  // (as kLeastV: below f16's range whatever the code)
            w = make_float4(f, __log2f(x), 0.0f, 1.0f / (x * kProbs));
          } else {
            float e, mant, down;
            split_scale(q8_scale(sc.y), e, mant, down);
            w = make_float4(f, e, mant * kProbs, down);
          }
          reinterpret_cast<float4*>(smem + W::scale)[i % W::SCALES * W::GROUPS + lane] = w;
        }
        __syncwarp();
        if (keys && lane == 0) arrive1(bar(B_SCALE + i % W::SCALES));
        id = checked(i + 1u, next);
        next = page_of(i + 2u);
        sc = scales_of(id);
      }
      if (sent < n_tiles && lane == 0) *fail = 1;
      // the copies must have landed before this block's shared memory goes away (bounded)
      for (unsigned i = sent > W::RING ? sent - W::RING : 0u; i < sent; i++) mb_wait(bar(B_RAW_FULL + kv4 + i % W::RING), i / W::RING & 1u, kWait);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (tid == 0 && *fail) atomicOr(wa.err, 16u);
  if (warp == MMA_WARP) tc_dealloc(*tslot, 512);
  wait_before();
}

// Records of blocks whose tiles were split, in their order; a warp a row.
template <int HD, typename T>
__global__ void __launch_bounds__(1024) sdpa_q8_wide_merge_kernel(const __grid_constant__ ks_wide_args wa) {
  using W = Wide<HD, T>;
  if (!wa.beside) wait_before();
  start_next();
  const ks_sdpa_q8_args& a = wa.a;
  const unsigned lane = threadIdx.x & 31u, r = blockIdx.y * 32u + (threadIdx.x >> 5);
  const int4 meta = wa.meta[blockIdx.x];
  const unsigned m = (unsigned)meta.y + r, n_splits = (unsigned)meta.w >> 16, kvh = (unsigned)meta.w & 0xFFFFu;
  if (m >= (unsigned)meta.z || n_splits <= 1u) {
    wait_before();
    return;
  }
  const float* rec = wa.part + (size_t)blockIdx.x * wa.n_splits * W::record;
  float top = kNone, l = 0.0f, v[HD / 32];
  // a split's (m, l) per lane
  const float mk = lane < n_splits ? rec[lane * (size_t)W::record + r] : kNone, lk = lane < n_splits ? rec[lane * (size_t)W::record + W::ROWS + r] : 0.0f;
  top = mk;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float ek = lk == 0.0f ? 0.0f : exp2_fast(mk - top);  // (nothing seen: it may have left no values)
  l = q8_warp_sum(ek * lk);
#pragma unroll
  for (int d = 0; d < HD / 32; d++) v[d] = 0.0f;
  for (unsigned k = 0; k < n_splits; k++) {
    const float e = __shfl_sync(0xffffffffu, ek, k);
    if (e == 0.0f) continue;
    const float* x = rec + k * (size_t)W::record + 2 * W::ROWS + (size_t)r * HD + 2u * lane;
#pragma unroll
    for (int d = 0; d < HD / 32; d += 2) {
      const float2 y = *reinterpret_cast<const float2*>(x + 32 * d);
      v[d] = fmaf(e, y.x, v[d]);
      v[d + 1] = fmaf(e, y.y, v[d + 1]);
    }
  }
  const float f = over(l);
  T* o = (T*)a.out + ((size_t)(meta.x + (int)(m / a.G)) * a.n_q + kvh * a.G + m % a.G) * HD;
#pragma unroll
  for (int d = 0; d < HD / 32; d += 2) {
    const float y[2] = {v[d] * f, v[d + 1] * f};
    put_dims(o + 2u * lane + 32 * d, y, 2);
  }
  wait_before();
}

// Tiles of `rows` (row, head) pairs that the sequences above the line can make at most.
size_t wide_tiles(size_t n_seqs, size_t max_rows, size_t G, size_t rows) {
  const size_t pairs = max_rows * G, seqs = pairs / (KS_Q8_FEW + 1);
  return pairs / rows + (seqs < n_seqs ? seqs : n_seqs);
}
// Splits of the longest context: the number for which the launch should end first.  Blocks see three quarters of the longest context on the
// average (causal rows), and the last blocks leave a quarter of their time to nobody; setting up is worth `set_up` tiles, with a record to leave
// (and to merge) `set_up_split`.  blocks x splits is 4 blocks an SM at most.  Measured: 2047 rows of 8 heads (f32, 128 blocks of up to 32 tiles) 102, 89, 96, 106 us in
// 1 .. 4 splits; 4096 behind 4096 (f16, 256 blocks of up to 128) 329 and 365 in 1 and 2; eight ragged pieces through a window of 512 (f32, 40 blocks of
// up to 9) 55, 47 and 62.
constexpr unsigned kMostSplits = 32;  // a lane of the merge each
unsigned wide_splits(const ks_ctx* ctx, size_t blocks, size_t tiles, size_t set_up, size_t set_up_split, unsigned* share) {
  if (tiles < 1) tiles = 1;
  const size_t sms = (size_t)ctx->sm_count;
  size_t best = 1, least = ~size_t(0);
  for (size_t n = 1; n <= kMostSplits && n <= tiles && (n == 1 || blocks * n <= 4 * sms); n++) {
    const size_t extra = n == 1 ? set_up : set_up_split, one = (tiles + n - 1) / n + extra, even = 3 * blocks * (tiles + n * extra) / 4 / sms + one / 4, time = one > even ? one : even;
    if (time < least) {
      least = time;
      best = n;
    }
  }
  const size_t s = (tiles + best - 1) / best;
  *share = (unsigned)(s < 0x7FFFFFFFu ? s : 0x7FFFFFFFu);
  return (unsigned)((tiles + s - 1) / s);
}

// Blocks of the launch, and what its kernels get.
template <int HD, typename T>
size_t wide_plan(ks_ctx* ctx, const ks_sdpa_q8_args& a, float* tmp, size_t ctx_most, bool beside, ks_wide_args* wa) {
  using W = Wide<HD, T>;
  const size_t blocks = wide_tiles(a.n_seqs, a.max_rows, a.G, W::ROWS) * a.n_kv;
  wa->a = a;
  wa->beside = beside;
  const size_t window = a.window ? (size_t)a.window + W::ROWS / a.G + 1 : ctx_most;
  wa->n_splits = wide_splits(ctx, blocks, ((window < ctx_most ? window : ctx_most) + W::TILE - 1) / W::TILE, W::TERMS == 1 ? 4 : 2, W::TERMS == 1 ? 12 : 5, &wa->share);
  wa->meta = (int4*)tmp;
  wa->part = tmp + 4 * blocks;
  wa->err = (unsigned*)ctx->ws + KS_WS_ERR_WORD;
  return blocks;
}

template <int HD, typename T, bool FP8>
int launch_wide(ks_ctx* ctx, const ks_sdpa_q8_args& a, float* tmp, size_t ctx_most, bool beside) {
  using W = Wide<HD, T>;
  static bool set[16] = {false};
  if (!set[ctx->device & 15]) {
    cudaError_t e = cudaFuncSetAttribute(sdpa_q8_wide_kernel<HD, T, FP8>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)W::total);
    if (e != cudaSuccess) return ks_fail(ctx, KS_ERR_CUDA, "sdpa_paged_q8: cannot set %u B shared memory: %s", W::total, cudaGetErrorString(e));
    set[ctx->device & 15] = true;
  }
  ks_wide_args wa;
  const size_t blocks = wide_plan<HD, T>(ctx, a, tmp, ctx_most, beside, &wa);
  KS_REQUIRE(ctx, blocks < (1u << 31), "sdpa_paged_q8: too many rows and heads for one launch");
  KS_LAUNCH(ctx, (sdpa_q8_wide_kernel<HD, T, FP8>), dim3((unsigned)blocks, wa.n_splits), W::THREADS, W::total, wa);
  return ks_after_launch(ctx, "sdpa_paged_q8 wide");
}

template <int HD, typename T>
int launch_wide_merge(ks_ctx* ctx, const ks_sdpa_q8_args& a, float* tmp, size_t ctx_most, bool beside) {
  ks_wide_args wa;
  const size_t blocks = wide_plan<HD, T>(ctx, a, tmp, ctx_most, beside, &wa);
  if (wa.n_splits == 1) return KS_OK;
  KS_LAUNCH(ctx, (sdpa_q8_wide_merge_kernel<HD, T>), dim3((unsigned)blocks, Wide<HD, T>::ROWS / 32), 1024, 0, wa);
  return ks_after_launch(ctx, "sdpa_paged_q8 wide merge");
}

}  // namespace

size_t ks_sdpa_q8_wide_floats(const ks_ctx* ctx, size_t n_seqs, size_t max_rows, size_t n_kv, size_t G, size_t hd) {
  size_t most = 0;
  for (size_t rows = kRows; rows <= (hd == 256 ? 1 : 2) * kRows; rows += kRows) {  // either activation type
    const size_t blocks = wide_tiles(n_seqs, max_rows, G, rows) * n_kv, most_records = 4 * (size_t)ctx->sm_count;
    const size_t n = 4 * blocks + (2 * blocks <= most_records ? most_records * rows * (hd + 2) : 0);
    if (n > most) most = n;
  }
  return most;
}

int ks_launch_sdpa_q8_wide(ks_ctx* ctx, const ks_sdpa_q8_args& a, size_t hd, ks_dtype act, bool fp8, float* tmp, size_t ctx_most, bool beside) {
#define KS_WD(HD_, T_, F_) launch_wide<HD_, T_, F_>(ctx, a, tmp, ctx_most, beside)
#define KS_WD_T(HD_, F_) (act == KS_F32 ? KS_WD(HD_, float, F_) : KS_WD(HD_, __half, F_))
#define KS_WD_F(HD_) (fp8 ? KS_WD_T(HD_, true) : KS_WD_T(HD_, false))
  return hd == 256 ? KS_WD_F(256) : hd == 128 ? KS_WD_F(128) : KS_WD_F(64);
#undef KS_WD_F
#undef KS_WD_T
#undef KS_WD
}

int ks_launch_sdpa_q8_wide_merge(ks_ctx* ctx, const ks_sdpa_q8_args& a, size_t hd, ks_dtype act, float* tmp, size_t ctx_most, bool beside) {
#define KS_WM(HD_) (act == KS_F32 ? launch_wide_merge<HD_, float>(ctx, a, tmp, ctx_most, beside) : launch_wide_merge<HD_, __half>(ctx, a, tmp, ctx_most, beside))
  return hd == 256 ? KS_WM(256) : hd == 128 ? KS_WM(128) : KS_WM(64);
#undef KS_WM
}
