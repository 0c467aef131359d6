// Attention of many rows (prompt pieces, long drafts) over a paged 8-bit cache, on tcgen05.
//
// A block takes 128 query rows (row and query head of the group, counted together) of a sequence against one KV head and walks over the tiles of
// TILE positions that they see.  Five kinds of warps hand tiles on through mbarriers:
//   loader      codes of a tile, page by page, by bulk copies into a ring of two; what scores and probabilities are scaled by per 16 positions;
//   converters  codes -> f16 (exact) core matrices: K as positions x dims, V transposed as dims x positions;
//   products    one elected lane issues S = q K^T into tensor memory and O (+)= P V with P out of tensor memory;
//   softmax     eight warps, half a row a thread: S -> mask, maximum, probabilities -> P.
// The maximum that probabilities refer to moves only when a score exceeds it by 2^4, so the two threads of a row mostly agree by one vote.
// f16 activations: q as it is, P rounded to f16, O stays in tensor memory and is rescaled there when the maximum moves.  f32: q (first term in
// tensor memory, second in shared memory) and P are two f16 terms each, small terms first, and O leaves tensor memory after every tile
// for f32 registers, because its accumulator drops the low bits of what is added.
#include "ks_sdpa_q8.cuh"
#include "ks_gemm_common.cuh"

namespace {

constexpr int kRows = 128;
constexpr unsigned kWait = 1u << 20;
constexpr int kWork = 8;  // softmax warps

enum { B_RAW_FULL = 0, B_RAW_FREE = 2, B_K_FULL = 4, B_K_FREE, B_V_FULL, B_V_FREE, B_S_FULL, B_S_FREE, B_P_FULL, B_DONE, B_COUNT };

template <int HD_, typename T_>
struct Wide {
  static constexpr int HD = HD_, TERMS = sizeof(T_) == 4 ? 2 : 1, TILE = HD == 256 ? 64 : 128, GROUPS = TILE / 16, COLS = TILE / 2;
  static constexpr int CONV = TERMS == 1 ? 8 : 4, WARPS = kWork + CONV + 4, THREADS = WARPS * 32;
  static constexpr int R_WORK = TERMS == 1 ? 128 : 208, R_CONV = TERMS == 1 ? 80 : 64, R_REST = TERMS == 1 ? 64 : 32;
  static_assert(kWork * 32 * R_WORK + CONV * 32 * R_CONV + 128 * R_REST <= THREADS * (65536 / THREADS / 8 * 8), "registers: the shares fit the launch");
  // shared memory: barriers, the tensor-memory address and the failure flag; per row: scale, first and last position seen, maxima of its two
  // threads; per 16 positions of two tiles: the score's factor, log2 and mantissa of V's scale, its power's reciprocal
  static constexpr unsigned slot = 128, row = 256, best = row + 3 * kRows * 4, scale = best + 2 * kRows * 4, q = 3072;
  static_assert(scale + 2 * GROUPS * 16 <= q, "the words fit in front of the operands");
  static constexpr unsigned k = q + kRows * HD * 2, v = k + TILE * HD * 2, raw = v + TILE * HD * 2, raw_bytes = 2 * TILE * HD, total = raw + 2 * raw_bytes;
  static_assert(q % 128 == 0 && kRows * HD * 2 <= 2 * TILE * HD * 2, "q's first term passes through K's and V's place");
  static constexpr unsigned OP = HD + 2;
  static_assert(kRows * OP * 4 <= total - q, "the result fits the operands");
  // tensor memory: scores, probabilities (two terms), O, q's first term
  static constexpr unsigned t_s = 0, t_p = TILE, t_pl = t_p + (TERMS - 1) * TILE / 2, t_o = t_p + TERMS * TILE / 2, t_q = t_o + HD;
  static_assert(t_q + (TERMS == 2 ? HD / 2 : 0) <= 512, "tensor memory");
  static constexpr unsigned record = kRows * (HD + 2);  // floats: m[128], l[128], O[128][HD]
};

__device__ __forceinline__ void arrive1(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
// `threads` threads (whole warps) meet at barrier `id`: does any, do all of them say so?
__device__ __forceinline__ bool meet_any(unsigned id, unsigned threads, bool x) {
  unsigned r;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, %2, %3, p;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(r) : "r"((unsigned)x), "r"(id), "r"(threads) : "memory");
  return r != 0;
}
__device__ __forceinline__ bool meet_all(unsigned id, unsigned threads, bool x) { return !meet_any(id, threads, !x); }
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

struct ks_wide_args {
  ks_sdpa_q8_args a;
  unsigned n_splits;
  int4* meta;   // per block of split 0: first row of the sequence, first (row, head) of the tile, how many the sequence has, KV head
  float* part;
  unsigned* err;
};

template <int HD, typename T, bool FP8>
__global__ void __launch_bounds__(Wide<HD, T>::THREADS, 1) sdpa_q8_wide_kernel(const __grid_constant__ ks_wide_args wa) {
  using W = Wide<HD, T>;
  const ks_sdpa_q8_args& a = wa.a;
  extern __shared__ __align__(1024) unsigned char smem[];
  __shared__ unsigned scan[W::WARPS], mine_seq, mine_tile;
  ks_pdl_entry();
  const unsigned tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
  const unsigned kvh = blockIdx.x % a.n_kv, index = blockIdx.x / a.n_kv, split = blockIdx.y;

  // ---- which tile of which sequence: a thread counts for up to two sequences
  {
    const unsigned per = (a.n_seqs + W::THREADS - 1u) / W::THREADS;
    unsigned count[2] = {0, 0}, sum = 0;
    for (unsigned k = 0; k < per; k++) {
      const unsigned i = tid * per + k;
      Seq s;
      if (i < a.n_seqs && seq_of(a, i, s) && (unsigned)s.rows * a.G > a.few) count[k] = ((unsigned)s.rows * a.G + kRows - 1u) / kRows;
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
      return;
    }
    for (unsigned k = 0; k < per; k++) {
      if (index >= before && index - before < count[k]) {
        mine_seq = tid * per + k;
        mine_tile = count[k] - 1u - (index - before);  // the last rows see the most: they start first
      }
      before += count[k];
    }
    __syncthreads();
  }
  Seq s;
  seq_of(a, mine_seq, s);
  const unsigned m_rows = (unsigned)s.rows * a.G, m0 = mine_tile * kRows;
  const int* table = a.tables + (size_t)mine_seq * a.max_blocks;
  if (split == 0 && tid == 0) wa.meta[blockIdx.x] = make_int4(s.row0, (int)m0, (int)m_rows, (int)kvh);

  const uint32_t sb = sm32(smem);
  auto bar = [&](unsigned i) { return sb + 8u * i; };
  uint32_t* tslot = reinterpret_cast<uint32_t*>(smem + W::slot);
  volatile unsigned* fail = reinterpret_cast<volatile unsigned*>(smem + W::slot + 8);
  float* row_scale = reinterpret_cast<float*>(smem + W::row);
  int* row_lo = reinterpret_cast<int*>(smem + W::row + kRows * 4);
  int* row_hi = reinterpret_cast<int*>(smem + W::row + kRows * 8);
  float* best = reinterpret_cast<float*>(smem + W::best);

  // ---- the positions that the rows see, and this split's tiles of them
  const int tok_a = (int)(m0 / a.G), tok_b = (int)(min(m0 + kRows - 1u, m_rows - 1u) / a.G), p_row0 = s.len - s.rows;
  const int seen_from = a.window && p_row0 + tok_a >= (int)a.window ? p_row0 + tok_a - (int)a.window + 1 : 0, seen_to = p_row0 + tok_b + 1;  // (may be below 1: nothing)
  const int first = seen_from & ~(W::TILE - 1), span = seen_to > first ? (seen_to - first + W::TILE - 1) / W::TILE : 0;
  const int share = (span + (int)wa.n_splits - 1) / (int)wa.n_splits;
  const int t_begin = first + (int)split * share * W::TILE;
  const unsigned n_tiles = (unsigned)max(min(share, span - (int)split * share), 0);
  const bool whole = wa.n_splits == 1u;
  float* rec = wa.part + ((size_t)blockIdx.x * wa.n_splits + split) * W::record;
  auto out_row = [&](unsigned m) { return (T*)a.out + ((size_t)(s.row0 + (int)(m / a.G)) * a.n_q + kvh * a.G + m % a.G) * HD; };
  if (n_tiles == 0u) {  // an empty record, or rows of zeros
    if (!whole) {
      if (tid < kRows) {
        rec[tid] = kNone;
        rec[kRows + tid] = 0.0f;
      }
    } else {
      for (unsigned i = tid; i < kRows * HD; i += W::THREADS)
        if (m0 + i / HD < m_rows) out_row(m0 + i / HD)[i % HD] = (T)0.0f;
    }
    return;
  }

  if (tid == 0) {
    for (unsigned i = 0; i < 2u; i++) {
      mb_init(bar(B_RAW_FULL + i), 1);
      mb_init(bar(B_RAW_FREE + i), W::CONV + kWork);  // codes converted, scales read
    }
    mb_init(bar(B_K_FULL), W::CONV);
    mb_init(bar(B_V_FULL), W::CONV);
    mb_init(bar(B_K_FREE), 1);
    mb_init(bar(B_V_FREE), 1);
    mb_init(bar(B_S_FULL), 1);
    mb_init(bar(B_S_FREE), kWork);
    mb_init(bar(B_P_FULL), kWork);
    mb_init(bar(B_DONE), 1);
    *fail = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    proxy_fence();
  }
  if (warp == kWork + W::CONV) tc_alloc(sm32(tslot), 512);

  // ---- q: a softmax warp takes twice eight rows, lane = row lane % 8, 8 dims lane / 8 (+ 4 a step): core matrices of 8 rows x 16 bytes
  if (warp < kWork) {
    constexpr int STEPS = HD / 32, GR = kRows / 8 / kWork;
#pragma unroll 1
    for (int p = 0; p < GR; p++) {
      const unsigned r = (warp * GR + p) * 8u + (lane & 7u), m = m0 + r;
      const bool in = m < m_rows;
      const T* src = (const T*)a.q + ((size_t)(s.row0 + (int)((in ? m : m0) / a.G)) * a.n_q + kvh * a.G + (in ? m : m0) % a.G) * HD + 8u * (lane >> 3);
      if (lane < 8u) {
        const int hi = in ? p_row0 + (int)(m / a.G) : -1;
        row_hi[r] = hi;
        row_lo[r] = a.window && hi >= (int)a.window ? hi - (int)a.window + 1 : 0;
      }
      if constexpr (W::TERMS == 1) {
        uint4 v[STEPS];
#pragma unroll
        for (int k = 0; k < STEPS; k++) v[k] = in ? *reinterpret_cast<const uint4*>(src + 32 * k) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int k = 0; k < STEPS; k++) *reinterpret_cast<uint4*>(smem + W::q + ((4u * k + (lane >> 3)) * kRows + r) * 16u) = v[k];
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
          for (int e = 0; e < 8; e++) v[k][e] *= down;
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
  const unsigned quad = warp & 3u, half = warp >> 2 & 1u, row = quad * 32u + lane;  // softmax warps: half the columns of a row
  const uint32_t tlane = quad << 21;  // 32 rows a warp, in the address bits of the lane
  if (W::TERMS == 2) {
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
    if constexpr (W::TERMS == 1) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(W::R_WORK));
    else asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(W::R_WORK));
    constexpr int COLS = W::COLS, HALF = HD / 2;
    const float up = W::TERMS == 2 ? row_scale[row] : 1.0f;
    const int lo = row_lo[row], hi = row_hi[row];
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
    for (unsigned i = 0; i < n_tiles; i++) {
      ok = __all_sync(0xffffffffu, mb_wait(bar(B_RAW_FULL + (i & 1u)), i >> 1 & 1u, kWait)) && __all_sync(0xffffffffu, mb_wait(bar(B_S_FULL), i & 1u, kWait));
      float x[COLS / 16][16], top = -INFINITY;
      const float4* scale = reinterpret_cast<const float4*>(smem + W::scale) + (i & 1u) * W::GROUPS + half * (W::GROUPS / 2);
      if (ok) {
        tc_fence_after();
        uint32_t r[COLS / 16][16];
#pragma unroll
        for (int c = 0; c < COLS / 16; c++) tc_ld16(tlane + W::t_s + half * COLS + 16u * c, r[c]);
#pragma unroll
        for (int c = 0; c < COLS / 16; c++) tc_wait_ld16(r[c]);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive1(bar(B_S_FREE));
#pragma unroll
        for (int c = 0; c < COLS / 16; c++) {
          const float2 sc = *reinterpret_cast<const float2*>(scale + c);
          const float f = sc.x * up;
#pragma unroll
          for (int e = 0; e < 16; e++) x[c][e] = fmaf(__uint_as_float(r[c][e]), f, sc.y);
        }
        const int p0 = t_begin + (int)i * W::TILE + (int)half * COLS;
        if (!__all_sync(0xffffffffu, lo <= p0 && hi >= p0 + COLS - 1)) {
#pragma unroll
          for (int c = 0; c < COLS; c++)
            if (p0 + c < lo || p0 + c > hi) x[c / 16][c % 16] = -INFINITY;
        }
#pragma unroll
        for (int c = 0; c < COLS; c++) top = fmaxf(top, x[c / 16][c % 16]);
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
      uint32_t ph[COLS / 2], pl[W::TERMS == 2 ? COLS / 2 : 1];
#pragma unroll
      for (int c = 0; c < COLS / 16; c++) {
        const float2 sc = *(reinterpret_cast<const float2*>(scale + c) + 1);
        float sum = 0.0f;
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          const float y0 = exp2_fast(x[c][e] - ref), y1 = exp2_fast(x[c][e + 1] - ref);
          sum += y0 + y1;
          const __half2 h = __floats2half2_rn(y0 * sc.x, y1 * sc.x);
          ph[c * 8 + e / 2] = q8_u32(h);
          if constexpr (W::TERMS == 2) {
            const float2 f = __half22float2(h);
            pl[c * 8 + e / 2] = q8_u32(__floats2half2_rn(fmaf(y0, sc.x, -f.x), fmaf(y1, sc.x, -f.y)));
          }
        }
        l = fmaf(sum, sc.y, l);
      }
      __syncwarp();
      if (ok && lane == 0) arrive1(bar(B_RAW_FREE + (i & 1u)));
      // the tile before's values are done: P's place is free, O may be touched
      if (i > 0) ok = __all_sync(0xffffffffu, mb_wait(bar(B_V_FREE), (i - 1u) & 1u, kWait));
      if (ok && i > 0) {
        if constexpr (W::TERMS == 2) {
          fold();
          if (turned)
#pragma unroll
            for (int c = 0; c < HALF; c++) acc[c] *= turn;
        } else if (turned) {
          tc_fence_after();
#pragma unroll
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
        for (int c = 0; c < COLS / 2; c += 8) {
          const uint32_t w[8] = {ph[c], ph[c + 1], ph[c + 2], ph[c + 3], ph[c + 4], ph[c + 5], ph[c + 6], ph[c + 7]};
          tc_st8(tlane + W::t_p + half * (COLS / 2) + c, w);
          if constexpr (W::TERMS == 2) {
            const uint32_t z[8] = {pl[c], pl[c + 1], pl[c + 2], pl[c + 3], pl[c + 4], pl[c + 5], pl[c + 6], pl[c + 7]};
            tc_st8(tlane + W::t_pl + half * (COLS / 2) + c, z);
          }
        }
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive1(bar(B_P_FULL));
      }
    }
    ok = ok && __all_sync(0xffffffffu, mb_wait(bar(B_V_FREE), (n_tiles - 1u) & 1u, kWait));
    if (!ok && lane == 0) *fail = 1;
    // ---- the rows through shared memory, so that they leave in whole lines; every product that read it is done.  Column n of O is dim
    // 4 (n mod HD / 4) + n / (HD / 4)
    best[half * kRows + row] = l;
    if (meet_all(5u, kWork * 32u, ok)) {
      l = best[row] + best[kRows + row];
      const float f = whole ? over(l) : 1.0f;
      float* to = reinterpret_cast<float*>(smem + W::q) + (size_t)row * W::OP + 2u * half;
      if constexpr (W::TERMS == 2) {
        fold();
#pragma unroll
        for (int c = 0; c < HD / 4; c++) *reinterpret_cast<float2*>(to + 4 * c) = make_float2(acc[c] * f, acc[c + HD / 4] * f);
      } else {
        tc_fence_after();
#pragma unroll
        for (unsigned c = 0; c < HD / 4u; c += 8u) {
          uint32_t o0[8], o1[8];
          tc_ld8(tlane + W::t_o + half * HALF + c, o0);
          tc_ld8(tlane + W::t_o + half * HALF + HD / 4u + c, o1);
#pragma unroll
          for (int e = 0; e < 8; e++) *reinterpret_cast<float2*>(to + 4u * (c + e)) = make_float2(__uint_as_float(o0[e]) * f, __uint_as_float(o1[e]) * f);
        }
      }
      if (!whole && half == 0) {
        rec[row] = ref;
        rec[kRows + row] = l;
      }
      meet_all(5u, kWork * 32u, true);
      const float* from = reinterpret_cast<const float*>(smem + W::q);
      for (unsigned r = warp; r < kRows && m0 + r < m_rows; r += kWork) {
        float2 v[HD / 64];
#pragma unroll
        for (int k = 0; k < HD / 64; k++) v[k] = *reinterpret_cast<const float2*>(from + (size_t)r * W::OP + 2u * lane + 64 * k);
        T* o = out_row(m0 + r);
        float* rr = rec + 2 * kRows + (size_t)r * HD;
#pragma unroll
        for (int k = 0; k < HD / 64; k++) {
          const float y[2] = {v[k].x, v[k].y};
          if (whole) put_dims(o + 2u * lane + 64 * k, y, 2);
          else put_dims(rr + 2u * lane + 64 * k, y, 2);
        }
      }
    }
  } else if (warp < kWork + W::CONV) {
    // ---- codes -> f16 core matrices
    if constexpr (W::TERMS == 1) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(W::R_CONV));
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(W::R_CONV));
    const unsigned cw = warp - kWork;
    unsigned done = 0;
    for (unsigned i = 0; i < n_tiles; i++) {
      const unsigned char* raw_k = smem + W::raw + (i & 1u) * W::raw_bytes;
      const unsigned char* raw_v = raw_k + W::TILE * HD;
      if (!__all_sync(0xffffffffu, mb_wait(bar(B_RAW_FULL + (i & 1u)), i >> 1 & 1u, kWait))) break;
      if (i > 0 && !__all_sync(0xffffffffu, mb_wait(bar(B_K_FREE), (i - 1u) & 1u, kWait))) break;
      {
        // 32 rows and one 16-byte chunk of each, a different one for neighbouring lanes: neither the read nor the writes meet a bank twice
        constexpr unsigned CH = HD / 16, STEPS = W::TILE / 32 * CH, RING = HD == 64 ? 4 : 8;
#pragma unroll 4
        for (unsigned n = cw; n < STEPS; n += W::CONV) {
          const unsigned r = n / CH * 32u + lane, k = n % CH, ch = k / RING * RING + ((HD == 64 ? lane >> 1 : lane) + k) % RING;
          const uint4 w = *reinterpret_cast<const uint4*>(raw_k + r * HD + ch * 16u);
          uint4 x, y;
          widen4<FP8>(w.x, x.x, x.y);
          widen4<FP8>(w.y, x.z, x.w);
          widen4<FP8>(w.z, y.x, y.y);
          widen4<FP8>(w.w, y.z, y.w);
          *reinterpret_cast<uint4*>(smem + W::k + (2u * ch * W::TILE + r) * 16u) = x;
          *reinterpret_cast<uint4*>(smem + W::k + ((2u * ch + 1u) * W::TILE + r) * 16u) = y;
        }
      }
      proxy_fence();
      __syncwarp();
      if (lane == 0) arrive1(bar(B_K_FULL));
      if (i > 0 && !__all_sync(0xffffffffu, mb_wait(bar(B_V_FREE), (i - 1u) & 1u, kWait))) break;
      {
        // eight positions and four dims a lane; dim 4 w + j becomes column j HD / 4 + w of O, so that neighbouring lanes write neighbouring chunks
        constexpr unsigned WORDS = HD / 4, PER = HD == 64 ? 2 : 1, STEPS = W::TILE / 8 * WORDS / 32;
#pragma unroll 2
        for (unsigned n = cw; n < STEPS; n += W::CONV) {
          const unsigned w = PER == 2 ? lane & 15u : n % (WORDS / 32u ? WORDS / 32u : 1u) * 32u + lane, pg = PER == 2 ? 2u * n + (lane >> 4) : n / (WORDS / 32u ? WORDS / 32u : 1u);
          uint32_t v[8], p[4][4];
#pragma unroll
          for (int e = 0; e < 8; e++) v[e] = *reinterpret_cast<const uint32_t*>(raw_v + (8u * pg + e) * HD + 4u * w);
#pragma unroll
          for (int e = 0; e < 4; e++) widen_pairs<FP8>(v[2 * e], v[2 * e + 1], p[e]);
#pragma unroll
          for (int j = 0; j < 4; j++) *reinterpret_cast<uint4*>(smem + W::v + (pg * HD + j * WORDS + w) * 16u) = make_uint4(p[0][j], p[1][j], p[2][j], p[3][j]);
        }
      }
      proxy_fence();
      __syncwarp();
      if (lane == 0) {
        arrive1(bar(B_V_FULL));
        arrive1(bar(B_RAW_FREE + (i & 1u)));
      }
      done++;
    }
    if (done < n_tiles && lane == 0) *fail = 1;
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(W::R_REST));
    if (warp == kWork + W::CONV) {
      // ---- products
      const unsigned leader = elect_one(), tiles = __reduce_max_sync(0xffffffffu, n_tiles);
      constexpr uint32_t idesc_s = (1u << 4) | ((W::TILE >> 3) << 17) | ((kRows >> 4) << 24), idesc_o = (1u << 4) | ((HD >> 3) << 17) | ((kRows >> 4) << 24);
      const uint64_t d_q = tc_desc(sb + W::q, kRows * 16u, 128u), d_k = tc_desc(sb + W::k, W::TILE * 16u, 128u), d_v = tc_desc(sb + W::v, HD * 16u, 128u);
      auto scores = [&] {
        if (leader) {
          if constexpr (W::TERMS == 2) {
#pragma unroll
            for (unsigned ks = 0; ks < HD / 16u; ks++) tc_mma_f16(W::t_s, d_q + (uint64_t)(2u * ks * kRows), d_k + (uint64_t)(2u * ks * W::TILE), idesc_s, ks ? 1u : 0u);
#pragma unroll
            for (unsigned ks = 0; ks < HD / 16u; ks++) tc_mma_f16_ta(W::t_s, W::t_q + 8u * ks, d_k + (uint64_t)(2u * ks * W::TILE), idesc_s, 1u);
          } else {
#pragma unroll
            for (unsigned ks = 0; ks < HD / 16u; ks++) tc_mma_f16(W::t_s, d_q + (uint64_t)(2u * ks * kRows), d_k + (uint64_t)(2u * ks * W::TILE), idesc_s, ks ? 1u : 0u);
          }
          tc_commit(bar(B_S_FULL));
          tc_commit(bar(B_K_FREE));
        }
        __syncwarp();
      };
      bool ok = __all_sync(0xffffffffu, mb_wait(bar(B_K_FULL), 0u, kWait));
      if (ok) {
        tc_fence_after();
        scores();
      }
      for (unsigned i = 0; ok && i < tiles; i++) {
        if (i + 1u < tiles) {
          ok = __all_sync(0xffffffffu, mb_wait(bar(B_K_FULL), (i + 1u) & 1u, kWait)) && __all_sync(0xffffffffu, mb_wait(bar(B_S_FREE), i & 1u, kWait));
          if (!ok) break;
          tc_fence_after();
          scores();
        }
        ok = __all_sync(0xffffffffu, mb_wait(bar(B_V_FULL), i & 1u, kWait)) && __all_sync(0xffffffffu, mb_wait(bar(B_P_FULL), i & 1u, kWait));
        if (!ok) break;
        tc_fence_after();
        if (leader) {
          if constexpr (W::TERMS == 2) {
#pragma unroll
            for (unsigned ks = 0; ks < W::TILE / 16u; ks++) tc_mma_f16_ta(W::t_o, W::t_pl + 8u * ks, d_v + (uint64_t)(2u * ks * HD), idesc_o, ks ? 1u : 0u);
#pragma unroll
            for (unsigned ks = 0; ks < W::TILE / 16u; ks++) tc_mma_f16_ta(W::t_o, W::t_p + 8u * ks, d_v + (uint64_t)(2u * ks * HD), idesc_o, 1u);
          } else {
#pragma unroll
            for (unsigned ks = 0; ks < W::TILE / 16u; ks++) tc_mma_f16_ta(W::t_o, W::t_p + 8u * ks, d_v + (uint64_t)(2u * ks * HD), idesc_o, i || ks ? 1u : 0u);
          }
          tc_commit(bar(B_V_FREE));
        }
        __syncwarp();
      }
      if (leader) {  // every product issued must finish before shared and tensor memory go away (bounded)
        if (!ok) *fail = 1;
        tc_commit(bar(B_DONE));
      }
      __syncwarp();
      mb_wait(bar(B_DONE), 0u, kWait);
    } else if (warp == kWork + W::CONV + 1) {
      // ---- codes: the runs of a tile that lie in one page, a lane each
      const unsigned page = 1u << a.page_log, run = min(page, (unsigned)W::TILE), runs = W::TILE / run;
      unsigned sent = 0;
      for (unsigned i = 0; i < n_tiles; i++) {
        const unsigned st = i & 1u;
        const int p0 = t_begin + (int)i * W::TILE, p = p0 + (int)(lane * run);
        int id = -1;
        if (lane < runs && p < seen_to && p + (int)run > seen_from) {
          id = table[(unsigned)p >> a.page_log];
          if ((unsigned)id >= a.n_pages) {
            atomicOr(a.bad, KS_BAD_PAGE);
            id = -1;
          }
        }
        const int gid = __shfl_sync(0xffffffffu, id, lane * 16u / run);
        float ks = 0.0f, vs = 0.0f;
        if (lane < W::GROUPS && gid >= 0) {
          ks = a.ks[(size_t)gid * a.n_kv + kvh];
          vs = a.vs[(size_t)gid * a.n_kv + kvh];
        }
        const unsigned there = __popc(__ballot_sync(0xffffffffu, id >= 0));
        if (i >= 2u && !__all_sync(0xffffffffu, mb_wait(bar(B_RAW_FREE + st), ((i >> 1) - 1u) & 1u, kWait))) break;
        if (lane < W::GROUPS) {
          float e, factor, down;
          split_scale(q8_scale(vs), e, factor, down);
          reinterpret_cast<float4*>(smem + W::scale)[(i & 1u) * W::GROUPS + lane] = make_float4(q8_scale(ks) * a.scale * 1.44269504088896340736f, e, factor * kProbs, down);
        }
        __syncwarp();
        if (lane == 0) mb_expect(bar(B_RAW_FULL + st), there * 2u * run * HD);
        __syncwarp();
        if (id >= 0) {
          const size_t from = ((((size_t)id * a.n_kv + kvh) << a.page_log) + ((unsigned)p & (page - 1u))) * HD;
          const uint32_t to = sb + W::raw + st * W::raw_bytes + lane * run * HD;
          bulk_in(to, a.kc + from, run * HD, bar(B_RAW_FULL + st));
          bulk_in(to + W::TILE * HD, a.vc + from, run * HD, bar(B_RAW_FULL + st));
        }
        sent++;
      }
      if (sent < n_tiles && lane == 0) *fail = 1;
      // the copies must have landed before this block's shared memory goes away (bounded)
      for (unsigned i = sent > 2u ? sent - 2u : 0u; i < sent; i++) mb_wait(bar(B_RAW_FULL + (i & 1u)), i >> 1 & 1u, kWait);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (tid == 0 && *fail) atomicOr(wa.err, 16u);
  if (warp == kWork + W::CONV) tc_dealloc(*tslot, 512);
}

// Records of blocks whose tiles were split, in their order; a warp a row.
template <int HD, typename T>
__global__ void __launch_bounds__(256) sdpa_q8_wide_merge_kernel(const __grid_constant__ ks_wide_args wa) {
  using W = Wide<HD, T>;
  ks_pdl_entry();
  const ks_sdpa_q8_args& a = wa.a;
  const unsigned lane = threadIdx.x & 31u, r = blockIdx.y * 8u + (threadIdx.x >> 5);
  const int4 meta = wa.meta[blockIdx.x];
  const unsigned m = (unsigned)meta.y + r;
  if (m >= (unsigned)meta.z) return;
  const float* rec = wa.part + (size_t)blockIdx.x * wa.n_splits * W::record;
  float top = kNone, l = 0.0f, v[HD / 32];
  for (unsigned k = 0; k < wa.n_splits; k++) top = fmaxf(top, rec[k * (size_t)W::record + r]);
#pragma unroll
  for (int d = 0; d < HD / 32; d++) v[d] = 0.0f;
  for (unsigned k = 0; k < wa.n_splits; k++) {
    const float* x = rec + k * (size_t)W::record;
    const float lk = x[kRows + r];
    if (lk == 0.0f) continue;  // nothing seen: it may have left no values
    const float e = exp2_fast(x[r] - top);
    l = fmaf(e, lk, l);
#pragma unroll
    for (int d = 0; d < HD / 32; d += 2) {
      const float2 y = *reinterpret_cast<const float2*>(x + 2 * kRows + (size_t)r * HD + 2u * lane + 32 * d);
      v[d] = fmaf(e, y.x, v[d]);
      v[d + 1] = fmaf(e, y.y, v[d + 1]);
    }
  }
  const float f = over(l);
  T* o = (T*)a.out + ((size_t)(meta.x + (int)(m / a.G)) * a.n_q + (unsigned)meta.w * a.G + m % a.G) * HD;
#pragma unroll
  for (int d = 0; d < HD / 32; d += 2) {
    const float y[2] = {v[d] * f, v[d + 1] * f};
    put_dims(o + 2u * lane + 32 * d, y, 2);
  }
}

// Tiles of 128 (row, head) pairs that the sequences above `few` can make at most.
size_t wide_tiles(size_t n_seqs, size_t max_rows, size_t G) {
  const size_t pairs = max_rows * G, seqs = pairs / (KS_Q8_FEW + 1);
  return pairs / kRows + (seqs < n_seqs ? seqs : n_seqs) + 1;
}
// Blocks for every SM, as far as the contexts go: two tiles each at least.
unsigned wide_splits(const ks_ctx* ctx, size_t blocks, size_t ctx_most, size_t tile) {
  size_t n = blocks < (size_t)ctx->sm_count ? (size_t)ctx->sm_count / blocks : 1;
  const size_t by_len = (ctx_most + 2 * tile - 1) / (2 * tile);
  if (n > by_len) n = by_len;
  if (n > 16) n = 16;
  return n < 1 ? 1u : (unsigned)n;
}

template <int HD, typename T, bool FP8>
int launch_wide(ks_ctx* ctx, const ks_sdpa_q8_args& a, float* tmp, size_t ctx_most) {
  using W = Wide<HD, T>;
  static bool set[16] = {false};
  if (!set[ctx->device & 15]) {
    cudaError_t e = cudaFuncSetAttribute(sdpa_q8_wide_kernel<HD, T, FP8>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)W::total);
    if (e != cudaSuccess) return ks_fail(ctx, KS_ERR_CUDA, "sdpa_paged_q8: cannot set %u B shared memory: %s", W::total, cudaGetErrorString(e));
    set[ctx->device & 15] = true;
  }
  const size_t blocks = wide_tiles(a.n_seqs, a.max_rows, a.G) * a.n_kv;
  KS_REQUIRE(ctx, blocks < (1u << 31), "sdpa_paged_q8: too many rows and heads for one launch");
  ks_wide_args wa;
  wa.a = a;
  wa.n_splits = wide_splits(ctx, blocks, ctx_most, W::TILE);
  wa.meta = (int4*)tmp;
  wa.part = tmp + 4 * blocks;
  wa.err = (unsigned*)ctx->ws + KS_WS_ERR_WORD;
  KS_LAUNCH(ctx, (sdpa_q8_wide_kernel<HD, T, FP8>), dim3((unsigned)blocks, wa.n_splits), W::THREADS, W::total, wa);
  int rc = ks_after_launch(ctx, "sdpa_paged_q8 wide");
  if (rc || wa.n_splits == 1) return rc;
  KS_LAUNCH(ctx, (sdpa_q8_wide_merge_kernel<HD, T>), dim3((unsigned)blocks, kRows / 8), 256, 0, wa);
  return ks_after_launch(ctx, "sdpa_paged_q8 wide merge");
}

}  // namespace

size_t ks_sdpa_q8_wide_floats(const ks_ctx* ctx, size_t n_seqs, size_t max_rows, size_t n_kv, size_t G, size_t hd) {
  const size_t blocks = wide_tiles(n_seqs, max_rows, G) * n_kv;
  const unsigned n = wide_splits(ctx, blocks, ~size_t(0) / 2, 128);
  return 4 * blocks + (n > 1 ? blocks * n * kRows * (hd + 2) : 0);
}

int ks_launch_sdpa_q8_wide(ks_ctx* ctx, const ks_sdpa_q8_args& a, size_t hd, ks_dtype act, bool fp8, float* tmp, size_t ctx_most) {
#define KS_WD(HD_, T_, F_) launch_wide<HD_, T_, F_>(ctx, a, tmp, ctx_most)
#define KS_WD_T(HD_, F_) (act == KS_F32 ? KS_WD(HD_, float, F_) : KS_WD(HD_, __half, F_))
#define KS_WD_F(HD_) (fp8 ? KS_WD_T(HD_, true) : KS_WD_T(HD_, false))
  return hd == 256 ? KS_WD_F(256) : hd == 128 ? KS_WD_F(128) : KS_WD_F(64);
#undef KS_WD_F
#undef KS_WD_T
#undef KS_WD
}
