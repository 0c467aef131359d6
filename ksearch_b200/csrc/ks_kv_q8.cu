// Rows into and out of a paged 8-bit cache: append as they are, append behind the per-head norms and RoPE, read back.
//
// A block of the append takes the new rows of one page for one KV head, K or V.  With a = max |x| of its finite values it sets
//   s = 2^e, the least e with a <= qmax 2^e   (qmax 127 or 448, e in -100 .. 100),   s = max(s, scale of the page) unless the page starts here,
// writes rne(x / s), and rounds the page's earlier codes again by (old scale) / s where s grew.  Scales are powers of two so that the
// division is exact: codes depend on nothing but the values, whatever the order of the operations around them, and however often a
// scale doubles the error that re-rounding adds stays below one step in all (1/2 + 1/4 + ...); with a / qmax as the scale every new maximum
// would add half a step.  The price is up to one bit of the int8 codes (none of e4m3's mantissa).
//
// Bound by: a few tokens by latency (record of the page, rows and scale, the block's maximum, stores: 2.1 us behind another kernel).  2047 rows of 8 heads of
// 128 (f16, 12.6 MB): 5.6 us.  2048 rows behind norm and RoPE (f16, 8 query heads, 2 of 256, 25 MB): 10 us, bound by instructions, two thirds of
// them the query heads'; eight rows a warp (100 registers, half the warps) took 12.  Read-back of 20000 rows of 2 heads of 256 to f16 (61 MB): 13.7 us,
// 69 % of the measured copy rate.
#include <cuda_fp16.h>

#include "ks_q8.h"
#include "ks_q8.cuh"

namespace {

constexpr int kHeadsPerWarp = 2;  // (row, query head) pairs of a warp

struct AppendArgs {
  uint8_t *kc, *vc;      // codes [n_pages, n_kv, page, hd]
  float *ks, *vs;        // scales [n_pages, n_kv]
  const int* plan;
  ks_plan_layout at;
  unsigned max_rows, page_log, n_kv, n_jobs;
  unsigned n_slots;      // n_pages * page
  const void *k, *v;
  size_t kv_ld;
  unsigned* bad;
  // behind the norms
  const void *q, *qw, *kw;
  void* q_out;
  const float* rope;
  unsigned n_q, rope_rows;
  float eps;
};

template <int V, typename T>
__device__ __forceinline__ void load_act(const T* p, float (&x)[V]) {
  if constexpr (sizeof(T) == 4) {
    if constexpr (V == 4) {
      const float4 a = *reinterpret_cast<const float4*>(p);
      x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    } else if constexpr (V == 2) {
      const float2 a = *reinterpret_cast<const float2*>(p);
      x[0] = a.x; x[1] = a.y;
    } else {
      x[0] = *p;
    }
  } else {
    if constexpr (V == 4) {
      const uint2 a = *reinterpret_cast<const uint2*>(p);
      const float2 u = __half22float2(q8_h2(a.x)), w = __half22float2(q8_h2(a.y));
      x[0] = u.x; x[1] = u.y; x[2] = w.x; x[3] = w.y;
    } else if constexpr (V == 2) {
      const float2 u = __half22float2(*reinterpret_cast<const __half2*>(p));
      x[0] = u.x; x[1] = u.y;
    } else {
      x[0] = __half2float(*p);
    }
  }
}
template <int V, typename T>
__device__ __forceinline__ void store_act(T* p, const float (&x)[V]) {
  if constexpr (sizeof(T) == 4) {
    if constexpr (V == 4) *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    else if constexpr (V == 2) *reinterpret_cast<float2*>(p) = make_float2(x[0], x[1]);
    else *p = x[0];
  } else {
    if constexpr (V == 4) {
      uint2 a;
      a.x = q8_u32(__floats2half2_rn(x[0], x[1]));
      a.y = q8_u32(__floats2half2_rn(x[2], x[3]));
      *reinterpret_cast<uint2*>(p) = a;
    } else if constexpr (V == 2) {
      *reinterpret_cast<__half2*>(p) = __floats2half2_rn(x[0], x[1]);
    } else {
      *p = __float2half_rn(x[0]);
    }
  }
}
template <int V, bool FP8>
__device__ __forceinline__ void store_codes(uint8_t* p, const float (&x)[V], float inv) {
  if constexpr (V == 4) {
    *reinterpret_cast<uint32_t*>(p) = q8_encode2<FP8>(x[0] * inv, x[1] * inv) | q8_encode2<FP8>(x[2] * inv, x[3] * inv) << 16;
  } else if constexpr (V == 2) {
    *reinterpret_cast<unsigned short*>(p) = (unsigned short)q8_encode2<FP8>(x[0] * inv, x[1] * inv);
  } else {
    *p = (uint8_t)q8_encode2<FP8>(x[0] * inv, 0.0f);
  }
}

// What a head of a row is normed and turned by.  A lane holds dims V lane.. of both halves, so RoPE partners sit in one lane.
template <int V>
struct Turn {
  float w0[V], w1[V], c[V], s[V];
};
template <int HD, int V, typename T>
__device__ __forceinline__ void load_turn(Turn<V>& t, const T* w, const float* cs) {
  load_act<V, T>(w, t.w0);
  load_act<V, T>(w + HD / 2, t.w1);
  load_act<V, float>(cs, t.c);
  load_act<V, float>(cs + HD / 2, t.s);
}
template <int HD, int V>
__device__ __forceinline__ float norm_of(const float (&x)[2][V], float eps) {
  float ss = 0.0f;
#pragma unroll
  for (int e = 0; e < V; e++) ss = fmaf(x[0][e], x[0][e], fmaf(x[1][e], x[1][e], ss));
  ss = q8_warp_sum(ss);
  return rsqrtf(fmaf(ss, 1.0f / HD, eps));
}
template <int V>
__device__ __forceinline__ void norm_rope(float (&x)[2][V], float inv, const Turn<V>& t) {
#pragma unroll
  for (int e = 0; e < V; e++) {
    const float a = __fmul_rn(__fmul_rn(x[0][e], inv), t.w0[e]), b = __fmul_rn(__fmul_rn(x[1][e], inv), t.w1[e]);
    x[0][e] = __fsub_rn(__fmul_rn(a, t.c[e]), __fmul_rn(b, t.s[e]));
    x[1][e] = __fadd_rn(__fmul_rn(a, t.s[e]), __fmul_rn(b, t.c[e]));
  }
}

// The same for what is rounded to codes, as sums of two floats: a value that single ones move across the middle between two codes would be a whole step
// off (one in 2^20 of them).  Error terms of products by fma, of sums by the usual six operations.  All values of 2048 rows of 2 KV heads take
// 4.7 us more this way: the append makes only those rows so that need it.
struct Two {
  float hi, lo;
};
__device__ __forceinline__ Two times(Two a, float b) {
  const float p = __fmul_rn(a.hi, b);
  return {p, __fmaf_rn(a.lo, b, __fmaf_rn(a.hi, b, -p))};
}
__device__ __forceinline__ Two plus(Two a, Two b) {
  const float s = __fadd_rn(a.hi, b.hi), t = __fsub_rn(s, a.hi);
  return {s, __fadd_rn(__fadd_rn(__fsub_rn(a.hi, __fsub_rn(s, t)), __fsub_rn(b.hi, t)), __fadd_rn(a.lo, b.lo))};
}
// Rounded to one float toward the odd neighbour, so that rounding it again to 8 bits, and comparing it with a limit, give what the sum gives.  A first term
// that has passed f32's range (or is NaN) is the result as one float has it; the second one is no error of it any more.
__device__ __forceinline__ float to_odd(Two x) {
  if (!(fabsf(x.hi) < INFINITY)) return x.hi;
  const float f = __fadd_rn(x.hi, x.lo), rest = __fsub_rn(x.lo, __fsub_rn(f, x.hi));
  const uint32_t b = __float_as_uint(f);
  if (rest == 0.0f || (b & 1u) || !(fabsf(f) < INFINITY) || f == 0.0f) return f;
  return __uint_as_float((rest > 0.0f) == (f > 0.0f) ? b + 1u : b - 1u);
}
// 1 / sqrt(mean of squares + eps): the hardware's approximation r, and one Newton step r / 2 (1 - m r^2) as the second term.
template <int HD, int V>
__device__ __forceinline__ Two norm_of_two(const float (&x)[2][V], float eps) {
  Two ss = {0.0f, 0.0f};
#pragma unroll
  for (int e = 0; e < 2 * V; e++) {
    const float y = x[e / V][e % V];
    ss = plus(ss, times(Two{y, 0.0f}, y));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss = plus(ss, Two{__shfl_xor_sync(0xffffffffu, ss.hi, o), __shfl_xor_sync(0xffffffffu, ss.lo, o)});
  const Two m = plus(Two{ss.hi * (1.0f / HD), ss.lo * (1.0f / HD)}, Two{eps, 0.0f});
  const float r = rsqrtf(m.hi);
  const Two r2 = times(Two{r, 0.0f}, r), mr2 = times(r2, m.hi);
  const float rest = __fsub_rn(__fsub_rn(1.0f, mr2.hi), __fmaf_rn(r2.hi, m.lo, mr2.lo)), step = 0.5f * r * rest, hi = __fadd_rn(r, step);
  return {hi, __fsub_rn(step, __fsub_rn(hi, r))};
}
template <int V>
__device__ __forceinline__ void norm_rope_two(float (&x)[2][V], Two inv, const Turn<V>& t) {
#pragma unroll
  for (int e = 0; e < V; e++) {
    const Two a = times(times(inv, x[0][e]), t.w0[e]), b = times(times(inv, x[1][e]), t.w1[e]);
    x[0][e] = to_odd(plus(times(a, t.c[e]), times(b, -t.s[e])));
    x[1][e] = to_odd(plus(times(a, t.s[e]), times(b, t.c[e])));
  }
}

// Grid: (touched pages x n_kv x 2) blocks of page / ROWS warps, each of which keeps ROWS rows in registers between
// their maximum and their codes; K and V of a head next to each other.  NORM: behind them, which take longer, the blocks of
// the query heads.
template <int HD, typename T, bool FP8, bool NORM, int ROWS>
__global__ void __launch_bounds__(1024) append_q8_kernel(const AppendArgs a) {
  constexpr int V = HD / 64;
  __shared__ float red[32];
  ks_pdl_entry();
  const unsigned lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, nwarp = blockDim.x >> 5;
  const unsigned page = 1u << a.page_log, per_job = 2u * a.n_kv;
  if (NORM && blockIdx.x >= a.n_jobs * per_job) {
    const unsigned it0 = ((blockIdx.x - a.n_jobs * per_job) * nwarp + warp) * kHeadsPerWarp, most = a.max_rows * a.n_q;
    float x[kHeadsPerWarp][2][V];
    int pos[kHeadsPerWarp];
    const unsigned items = min((unsigned)max(a.plan[1], 0), a.max_rows) * a.n_q;
#pragma unroll
    for (int i = 0; i < kHeadsPerWarp; i++) {  // (rows behind the plan's last are in the buffers too: nothing waits for how many there are)
      const unsigned it = min(it0 + i, most - 1u);
      const T* src = (const T*)a.q + (size_t)it * HD + lane * V;
      load_act<V, T>(src, x[i][0]);
      load_act<V, T>(src + HD / 2, x[i][1]);
      pos[i] = a.plan[a.at.row_pos + it / a.n_q];
    }
    Turn<V> t[kHeadsPerWarp];
#pragma unroll
    for (int i = 0; i < kHeadsPerWarp; i++) load_turn<HD, V, T>(t[i], (const T*)a.qw + lane * V, a.rope + (size_t)min((unsigned)max(pos[i], 0), a.rope_rows - 1u) * HD + lane * V);
#pragma unroll
    for (int i = 0; i < kHeadsPerWarp; i++) {
      const unsigned it = it0 + i;
      const float inv = norm_of<HD, V>(x[i], a.eps);
      if (it >= items) continue;
      if ((unsigned)pos[i] >= a.rope_rows) {
        if (lane == 0) atomicOr(a.bad, KS_BAD_POSITION);
        continue;
      }
      norm_rope<V>(x[i], inv, t[i]);
      T* dst = (T*)a.q_out + (size_t)it * HD + lane * V;
      store_act<V, T>(dst, x[i][0]);
      store_act<V, T>(dst + HD / 2, x[i][1]);
    }
    return;
  }
  const unsigned j = blockIdx.x / per_job, head = blockIdx.x % per_job >> 1;
  const bool vals = blockIdx.x & 1u;
  const int4 job = reinterpret_cast<const int4*>(a.plan + a.at.jobs)[j];
  if (job.x < 0 || job.y == 0) return;  // (no rows: words of zeros, a plan that no step has filled yet)
  const unsigned row0 = (unsigned)job.x, rows = (unsigned)job.y, slot = (unsigned)job.z, off = slot & (page - 1u);
  if (job.z < 0 || slot >= a.n_slots || rows > page - off || row0 >= a.max_rows || rows > a.max_rows - row0) {
    if (threadIdx.x == 0) atomicOr(a.bad, KS_BAD_SLOT);
    return;
  }
  if (NORM && !vals && ((unsigned)job.w >= a.rope_rows || rows > a.rope_rows - (unsigned)job.w)) {
    if (threadIdx.x == 0) atomicOr(a.bad, KS_BAD_POSITION);
    return;
  }
  const size_t block = (size_t)(slot >> a.page_log) * a.n_kv + head;
  float* scale_at = (vals ? a.vs : a.ks) + block;
  const float held = off ? q8_scale(*scale_at) : 0.0f;
  const T* src = (const T*)(vals ? a.v : a.k) + (size_t)row0 * a.kv_ld + (size_t)head * HD + lane * V;
  float x[ROWS][2][V], amax = 0.0f;
  auto fetch = [&](int i) {
    const unsigned r = warp + (unsigned)i * nwarp;
    load_act<V, T>(src + (size_t)r * a.kv_ld, x[i][0]);
    load_act<V, T>(src + (size_t)r * a.kv_ld + HD / 2, x[i][1]);
  };
  auto turned = [&](int i, bool fine) {  // a fetched row behind its norm and RoPE, in f32 or as sums of two
    const unsigned r = warp + (unsigned)i * nwarp;
    Turn<V> t;
    if (!vals) load_turn<HD, V, T>(t, (const T*)a.kw + lane * V, a.rope + (size_t)((unsigned)job.w + r) * HD + lane * V);
    if (fine) {
      const Two inv = norm_of_two<HD, V>(x[i], a.eps);
      if (!vals) return norm_rope_two<V>(x[i], inv, t);
#pragma unroll
      for (int e = 0; e < 2 * V; e++) x[i][e / V][e % V] = to_odd(times(inv, x[i][e / V][e % V]));
    } else {
      const float inv = norm_of<HD, V>(x[i], a.eps);
      if (!vals) return norm_rope<V>(x[i], inv, t);
#pragma unroll
      for (int e = 0; e < 2 * V; e++) x[i][e / V][e % V] *= inv;
    }
  };
  auto finite_most = [&](int i) {  // the largest finite value of a row's piece; NaN becomes 0
    float most = 0.0f, odd = 0.0f;
#pragma unroll
    for (int e = 0; e < 2 * V; e++) {
      const float y = x[i][e / V][e % V];
      most = fmaxf(most, fabsf(y));
      odd = fmaf(y, 0.0f, odd);
    }
    if (odd != 0.0f) {  // an infinity or NaN among them
      most = 0.0f;
#pragma unroll
      for (int e = 0; e < 2 * V; e++) {
        float& y = x[i][e / V][e % V];
        if (y != y) y = 0.0f;
        if (fabsf(y) < INFINITY) most = fmaxf(most, fabsf(y));
      }
    }
    return most;
  };
  auto largest = [&] {  // of the block
    amax = 0.0f;
#pragma unroll
    for (int i = 0; i < ROWS; i++)
      if (warp + (unsigned)i * nwarp < rows) amax = fmaxf(amax, finite_most(i));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (lane == 0) red[warp] = amax;
    __syncthreads();
    amax = lane < nwarp ? red[lane] : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  };
#pragma unroll
  for (int i = 0; i < ROWS; i++)
    if (warp + (unsigned)i * nwarp < rows) fetch(i);
  if constexpr (NORM)
#pragma unroll
    for (int i = 0; i < ROWS; i++)
      if (warp + (unsigned)i * nwarp < rows) turned(i, false);
  largest();
  // f32 leaves a value off by a dozen roundings of its pair at most.  A maximum that near to a limit, and a row with a value that near to the middle
  // between two codes, is made again as sums of two floats
  constexpr float DOUBT = 0x1p-20f;
  bool fine = false;
  if (NORM && q8_scale_for<FP8>(amax * (1.0f - 2.0f * DOUBT)) != q8_scale_for<FP8>(amax * (1.0f + 2.0f * DOUBT))) {
    fine = true;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ROWS; i++)
      if (warp + (unsigned)i * nwarp < rows) {
        fetch(i);
        turned(i, true);
      }
    largest();
  }
  const float s = fmaxf(q8_scale_for<FP8>(amax), q8_power_above(held)), inv = 1.0f / s;  // (powers of two: exact)
  uint8_t* codes = (vals ? a.vc : a.kc) + (block << a.page_log) * HD;
  if (off && s != held) {  // the page's earlier rows under the larger scale
    const float turn = held * inv;
    for (unsigned i = threadIdx.x; i < off * (HD / 4u); i += blockDim.x) {
      uint32_t* at = reinterpret_cast<uint32_t*>(codes) + i;
      const uint32_t w = *at;
      const float2 lo = q8_decode2f<FP8>(w), hi = q8_decode2f<FP8>(w >> 16);
      *at = q8_encode2<FP8>(lo.x * turn, lo.y * turn) | q8_encode2<FP8>(hi.x * turn, hi.y * turn) << 16;
    }
  }
#pragma unroll
  for (int i = 0; i < ROWS; i++) {
    const unsigned r = warp + (unsigned)i * nwarp;
    if (r >= rows) continue;
    if (NORM && !fine) {
      uint32_t differ = 0;
      float lo[2][V], hi[2][V];
#pragma unroll
      for (int e = 0; e < V; e++) {
        const float y0 = x[i][0][e] * inv, y1 = x[i][1][e] * inv, both = fabsf(y0) + fabsf(y1), d0 = DOUBT * (vals ? fabsf(y0) : both), d1 = DOUBT * (vals ? fabsf(y1) : both);
        lo[0][e] = y0 - d0; hi[0][e] = y0 + d0;
        lo[1][e] = y1 - d1; hi[1][e] = y1 + d1;
      }
#pragma unroll
      for (int h = 0; h < 2; h++)
#pragma unroll
        for (int e = 0; e < V; e += 2) differ |= q8_encode2<FP8>(lo[h][e], lo[h][V > 1 ? e + 1 : 0]) ^ q8_encode2<FP8>(hi[h][e], hi[h][V > 1 ? e + 1 : 0]);
      if (__any_sync(0xffffffffu, differ != 0u)) {
        fetch(i);
        turned(i, true);
        finite_most(i);
      }
    }
    uint8_t* dst = codes + (size_t)(off + r) * HD + lane * V;
    store_codes<V, FP8>(dst, x[i][0], inv);
    store_codes<V, FP8>(dst + HD / 2, x[i][1], inv);
  }
  if (threadIdx.x == 0 && s != held) *scale_at = s;
}

// Eight codes at a time, kReadsPerThread such reads on their way; K and V in blockIdx.y.
constexpr int kReadsPerThread = 4;
template <typename T, bool FP8>
__global__ void __launch_bounds__(256) read_q8_kernel(const uint8_t* kc, const uint8_t* vc, const float* ks, const float* vs, unsigned hd_log, unsigned n_kv, unsigned page_log,
                                                      unsigned n_slots, unsigned n_rows, const int* slots, T* k, T* v, unsigned* bad) {
  ks_pdl_entry();
  const uint8_t* codes = blockIdx.y ? vc : kc;
  const float* scales = blockIdx.y ? vs : ks;
  T* out = blockIdx.y ? v : k;
  const unsigned chunk_log = hd_log - 3u, per_row = n_kv << chunk_log;
  const size_t n = (size_t)n_rows * per_row, step = (size_t)gridDim.x * blockDim.x;
  for (size_t i0 = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i0 < n; i0 += step * kReadsPerThread) {
    int slot[kReadsPerThread];
    unsigned rest[kReadsPerThread];
#pragma unroll
    for (int u = 0; u < kReadsPerThread; u++) {
      const size_t i = i0 + u * step;
      const size_t row = i / per_row;
      rest[u] = (unsigned)(i - row * per_row);
      slot[u] = i < n ? slots[row] : -1;
    }
    uint2 w[kReadsPerThread];
    float s[kReadsPerThread];
#pragma unroll
    for (int u = 0; u < kReadsPerThread; u++) {
      if (slot[u] != -1 && (unsigned)slot[u] >= n_slots) {
        atomicOr(bad, KS_BAD_SLOT);
        slot[u] = -1;
      }
      const unsigned at = (unsigned)max(slot[u], 0), head = rest[u] >> chunk_log, c = rest[u] & ((1u << chunk_log) - 1u);
      const size_t block = (size_t)(at >> page_log) * n_kv + head;
      w[u] = make_uint2(0u, 0u);
      s[u] = 0.0f;
      if (slot[u] >= 0) {
        s[u] = scales[block];
        w[u] = *reinterpret_cast<const uint2*>(codes + ((((block << page_log) + (at & ((1u << page_log) - 1u))) << hd_log) + 8u * c));
      }
    }
#pragma unroll
    for (int u = 0; u < kReadsPerThread; u++) {
      if (slot[u] < 0) continue;
      const float f = q8_scale(s[u]);
      const float2 f0 = q8_decode2f<FP8>(w[u].x), f1 = q8_decode2f<FP8>(w[u].x >> 16), f2 = q8_decode2f<FP8>(w[u].y), f3 = q8_decode2f<FP8>(w[u].y >> 16);
      T* to = out + (i0 + u * step) * 8;
      if constexpr (sizeof(T) == 4) {
        const float lo[4] = {f0.x * f, f0.y * f, f1.x * f, f1.y * f}, hi[4] = {f2.x * f, f2.y * f, f3.x * f, f3.y * f};
        store_act<4, T>(to, lo);
        store_act<4, T>(to + 4, hi);
      } else {
        uint4 y;
        y.x = q8_u32(__floats2half2_rn(f0.x * f, f0.y * f));
        y.y = q8_u32(__floats2half2_rn(f1.x * f, f1.y * f));
        y.z = q8_u32(__floats2half2_rn(f2.x * f, f2.y * f));
        y.w = q8_u32(__floats2half2_rn(f3.x * f, f3.y * f));
        *reinterpret_cast<uint4*>(to) = y;
      }
    }
  }
}

AppendArgs append_args(ks_ctx* ctx, const ks_q8_cache* c, const ks_page_tables* t) {
  AppendArgs a{};
  a.kc = (uint8_t*)c->k->dptr;
  a.vc = (uint8_t*)c->v->dptr;
  a.ks = (float*)c->k_scale->dptr;
  a.vs = (float*)c->v_scale->dptr;
  a.plan = (const int*)t->plan->dptr;
  a.at = ks_plan_parts(t->n_seqs, t->max_rows, t->page);
  a.max_rows = (unsigned)t->max_rows;
  a.page_log = (unsigned)__builtin_ctzll(c->page);
  a.n_kv = (unsigned)c->n_kv;
  a.n_jobs = a.at.n_jobs < a.max_rows ? a.at.n_jobs : a.max_rows;  // (a touched page has a row)
  a.n_slots = (unsigned)(c->n_pages * c->page);
  a.bad = (unsigned*)ctx->ws + KS_WS_INDEX_WORD;
  return a;
}

template <bool NORM>
int launch_append(ks_ctx* ctx, const ks_q8_cache* c, ks_dtype act, const AppendArgs& a, const char* who) {
  const int rows = c->page == 128 ? 4 : 2;  // (up to 32 warps)
  const unsigned warps = (unsigned)c->page / rows;
  const size_t q_blocks = NORM ? ((size_t)a.max_rows * a.n_q + kHeadsPerWarp * warps - 1) / (kHeadsPerWarp * warps) : 0, blocks = q_blocks + (size_t)a.n_jobs * 2 * a.n_kv;
  KS_REQUIRE(ctx, blocks < (1u << 31), "%s: too many rows and heads for one launch", who);
  KS_REQUIRE_DEVICE(ctx, who);
  ks_on_device on(ctx);
#define KS_AP(HD_, T_, F_) do { if (rows == 4) KS_LAUNCH(ctx, (append_q8_kernel<HD_, T_, F_, NORM, 4>), (unsigned)blocks, warps * 32, 0, a); else KS_LAUNCH(ctx, (append_q8_kernel<HD_, T_, F_, NORM, 2>), (unsigned)blocks, warps * 32, 0, a); } while (0)
#define KS_AP_T(HD_, F_) do { if (act == KS_F32) KS_AP(HD_, float, F_); else KS_AP(HD_, __half, F_); } while (0)
#define KS_AP_F(HD_) do { if (c->dtype == KS_E4M3) KS_AP_T(HD_, true); else KS_AP_T(HD_, false); } while (0)
  if (c->hd == 256) KS_AP_F(256);
  else if (c->hd == 128) KS_AP_F(128);
  else KS_AP_F(64);
#undef KS_AP_F
#undef KS_AP_T
#undef KS_AP
  return ks_after_launch(ctx, who);
}

}  // namespace

int ks_check_cache(ks_ctx* ctx, const char* who, const ks_q8_cache* c, const ks_page_tables* t) {
  KS_REQUIRE(ctx, c, "%s: null cache", who);
  if (c->dtype != KS_I8 && c->dtype != KS_E4M3) return ks_fail(ctx, KS_ERR_UNSUPPORTED, "%s: cache dtype %d not supported (I8, E4M3)", who, (int)c->dtype);
  if (c->hd != 64 && c->hd != 128 && c->hd != 256) return ks_fail(ctx, KS_ERR_UNSUPPORTED, "%s: head_dim %zu not supported (64, 128, 256)", who, c->hd);
  KS_REQUIRE(ctx, ks_page_ok(c->page), "%s: pages of %zu positions not supported (16, 32, 64, 128)", who, c->page);
  KS_REQUIRE(ctx, c->n_kv >= 1 && c->n_kv <= 1024, "%s: n_kv=%zu outside 1..1024", who, c->n_kv);
  KS_REQUIRE(ctx, c->n_pages >= 1 && c->n_pages <= 0x7FFFFFFFu / c->page, "%s: %zu pages: at least one, and below 2^31 positions", who, c->n_pages);
  if (t) KS_REQUIRE(ctx, t->n_pages == c->n_pages && t->page == c->page, "%s: the tables hand out %zu pages of %zu positions, the cache has %zu of %zu", who, t->n_pages, t->page, c->n_pages, c->page);
  const size_t blocks = c->n_pages * c->n_kv;
  KS_REQUIRE(ctx, ks_fits(c->k, 0, blocks * c->page * c->hd) && ks_fits(c->v, 0, blocks * c->page * c->hd), "%s: cache buffer too small for %zu pages", who, c->n_pages);
  KS_REQUIRE(ctx, ks_fits(c->k_scale, 0, blocks * 4) && ks_fits(c->v_scale, 0, blocks * 4), "%s: scale buffer too small for %zu pages", who, c->n_pages);
  KS_REQUIRE(ctx, ks_aligned(c->k, 16) && ks_aligned(c->v, 16) && ks_aligned(c->k_scale, 4) && ks_aligned(c->v_scale, 4), "%s: codes must start on 16 bytes, scales on 4", who);
  return KS_OK;
}

extern "C" {

int ks_kv_append_q8(ks_ctx* ctx, const ks_q8_cache* c, const ks_page_tables* t, ks_dtype act, const ks_buf* k, size_t k_off, const ks_buf* v, size_t v_off, size_t kv_ld) {
  if (!ctx) return KS_ERR_INVALID;
  int rc = ks_check_tables(ctx, "kv_append_q8", t);
  if (!rc) rc = ks_check_cache(ctx, "kv_append_q8", c, t);
  if (rc) return rc;
  KS_REQUIRE(ctx, ks_is_act(act), "kv_append_q8: activation dtype must be F32 or F16");
  const size_t ab = ks_act_bytes(act), width = c->n_kv * c->hd;
  KS_REQUIRE(ctx, kv_ld >= width && kv_ld % 8 == 0 && kv_ld < (size_t(1) << 32) && k_off % 8 == 0 && v_off % 8 == 0, "kv_append_q8: rows %zu apart at offsets %zu, %zu: multiples of 8, rows at least n_kv * hd = %zu apart",
             kv_ld, k_off, v_off, width);
  const size_t need = ((t->max_rows - 1) * kv_ld + width) * ab;
  KS_REQUIRE(ctx, k_off < (size_t(1) << 48) && v_off < (size_t(1) << 48) && ks_fits(k, k_off * ab, need) && ks_fits(v, v_off * ab, need), "kv_append_q8: k/v buffer too small for %zu rows", t->max_rows);
  KS_REQUIRE(ctx, ks_aligned(k, 16) && ks_aligned(v, 16), "kv_append_q8: k and v must start on 16 bytes");
  AppendArgs a = append_args(ctx, c, t);
  a.k = (const uint8_t*)k->dptr + k_off * ab;
  a.v = (const uint8_t*)v->dptr + v_off * ab;
  a.kv_ld = kv_ld;
  return launch_append<false>(ctx, c, act, a, "kv_append_q8");
}

int ks_rmsnorm_per_head_qkv_q8(ks_ctx* ctx, const ks_q8_cache* c, const ks_page_tables* t, size_t n_q, float eps, ks_dtype act, const ks_buf* q, const ks_buf* qw, const ks_buf* rope,
                               const ks_buf* k, const ks_buf* kw, const ks_buf* v, ks_buf* q_out) {
  if (!ctx) return KS_ERR_INVALID;
  static const char who[] = "rmsnorm_per_head_qkv_q8";
  int rc = ks_check_tables(ctx, who, t);
  if (!rc) rc = ks_check_cache(ctx, who, c, t);
  if (rc) return rc;
  KS_REQUIRE(ctx, ks_is_act(act), "%s: activation dtype must be F32 or F16", who);
  KS_REQUIRE(ctx, n_q >= 1 && n_q <= 65536 && n_q * t->max_rows < (1u << 30), "%s: bad query head count %zu", who, n_q);
  const size_t ab = ks_act_bytes(act), q_bytes = t->max_rows * n_q * c->hd * ab, kv_bytes = t->max_rows * c->n_kv * c->hd * ab;
  KS_REQUIRE(ctx, ks_fits(q, 0, q_bytes) && ks_fits(q_out, 0, q_bytes), "%s: q buffer too small for %zu rows", who, t->max_rows);
  KS_REQUIRE(ctx, ks_fits(k, 0, kv_bytes) && ks_fits(v, 0, kv_bytes), "%s: k/v buffer too small for %zu rows", who, t->max_rows);
  KS_REQUIRE(ctx, ks_fits(qw, 0, c->hd * ab) && ks_fits(kw, 0, c->hd * ab), "%s: norm weight too small", who);
  KS_REQUIRE(ctx, ks_fits(rope, 0, c->hd * 4), "%s: rope table too small", who);
  KS_REQUIRE(ctx, ks_aligned(q, 16) && ks_aligned(q_out, 16) && ks_aligned(k, 16) && ks_aligned(v, 16) && ks_aligned(qw, 16) && ks_aligned(kw, 16) && ks_aligned(rope, 16),
             "%s: operands must start on 16 bytes", who);
  AppendArgs a = append_args(ctx, c, t);
  a.k = k->dptr;
  a.v = v->dptr;
  a.kv_ld = c->n_kv * c->hd;
  a.q = q->dptr;
  a.qw = qw->dptr;
  a.kw = kw->dptr;
  a.q_out = q_out->dptr;
  a.rope = (const float*)rope->dptr;
  const size_t rope_rows = rope->bytes / (c->hd * 4);
  a.rope_rows = (unsigned)(rope_rows < 0x7FFFFFFFu ? rope_rows : 0x7FFFFFFFu);
  a.n_q = (unsigned)n_q;
  a.eps = eps;
  return launch_append<true>(ctx, c, act, a, who);
}

int ks_kv_read_q8(ks_ctx* ctx, const ks_q8_cache* c, size_t n_rows, const ks_buf* slots, size_t slot_off, ks_dtype act, ks_buf* k, ks_buf* v) {
  if (!ctx) return KS_ERR_INVALID;
  int rc = ks_check_cache(ctx, "kv_read_q8", c, nullptr);
  if (rc) return rc;
  KS_REQUIRE(ctx, ks_is_act(act), "kv_read_q8: activation dtype must be F32 or F16");
  KS_REQUIRE(ctx, n_rows >= 1 && n_rows < (1u << 31), "kv_read_q8: n_rows=%zu outside 1..2^31 - 1", n_rows);
  KS_REQUIRE(ctx, slot_off < (size_t(1) << 48) && ks_fits(slots, slot_off * 4, n_rows * 4) && ks_aligned(slots, 4), "kv_read_q8: slots buffer too small for %zu rows, or not on 4 bytes", n_rows);
  const size_t bytes = n_rows * c->n_kv * c->hd * ks_act_bytes(act);
  KS_REQUIRE(ctx, ks_fits(k, 0, bytes) && ks_fits(v, 0, bytes) && ks_aligned(k, 16) && ks_aligned(v, 16), "kv_read_q8: k/v buffer too small for %zu rows, or not on 16 bytes", n_rows);
  KS_REQUIRE_DEVICE(ctx, "kv_read_q8");
  ks_on_device on(ctx);
  const size_t items = n_rows * c->n_kv * c->hd / 8;
  const size_t most = (size_t)ctx->sm_count * 8, blocks = (items + 256 * kReadsPerThread - 1) / (256 * kReadsPerThread);
  const dim3 grid((unsigned)(blocks < most ? blocks : most), 2);
  const int* at = (const int*)slots->dptr + slot_off;
  const unsigned hd_log = (unsigned)__builtin_ctzll(c->hd), page_log = (unsigned)__builtin_ctzll(c->page);
  unsigned* bad = (unsigned*)ctx->ws + KS_WS_INDEX_WORD;
#define KS_RD(T_, F_) KS_LAUNCH(ctx, (read_q8_kernel<T_, F_>), grid, 256, 0, (const uint8_t*)c->k->dptr, (const uint8_t*)c->v->dptr, (const float*)c->k_scale->dptr, \
                                (const float*)c->v_scale->dptr, hd_log, (unsigned)c->n_kv, page_log, (unsigned)(c->n_pages * c->page), (unsigned)n_rows, at, (T_*)k->dptr, (T_*)v->dptr, bad)
  if (act == KS_F32) {
    if (c->dtype == KS_E4M3) KS_RD(float, true);
    else KS_RD(float, false);
  } else {
    if (c->dtype == KS_E4M3) KS_RD(__half, true);
    else KS_RD(__half, false);
  }
#undef KS_RD
  return ks_after_launch(ctx, "kv_read_q8");
}

}  // extern "C"
