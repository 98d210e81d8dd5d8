// Log-probabilities of given tokens, with the entropy and the likeliest alternatives of each row of logits, and the logits' gradient.
//
// For a row y = scale * x with largest element m:  l = sum exp(y - m),  log p_j = (y_j - m) - log l,  H = -sum p_j log p_j = log l - s / l
// with s = sum exp(y - m) (y - m).  The differences from m are what is summed, so that nothing of the size of m cancels.  With gradients g of the
// target's log-probability and h of the entropy,
//   dx_j = scale * (g ([j = target] - p_j) - h p_j (log p_j + H)).
// A logit of -inf has probability 0 and adds nothing anywhere.  A row with NaN or +inf is NaN; a row without anything above -inf has
// log-probability -inf, entropy 0 and no gradient.
//
// Forward reads a row once, in 16-byte pieces, four to eight to a thread under way: every thread sums below a maximum of its own, and the threads meet at the
// end.  The alternatives cost no second pass: the k-th largest of the threads' maxima has k elements at or above it, so it is a bound that few others
// reach, and only the threads whose maximum does read their pieces again, from L2.  Long rows of which there are few are cut over a cluster of CTAs
// that meet in distributed shared memory; short ones share a warp.  Backward is one pass.
//
// fp32 is bound by the bytes: 16384 x 32000 297 us, 7.1 TB/s.  bf16 has an exponential to every two bytes and stays behind them: 189 us, 5.6 TB/s (issue slots 58 % busy,
// the exponentials' unit 57 %), with five alternatives 229, the gradient 343 (read and written: 6.1 TB/s).  Few rows are latency: 32 x 201088 8.2 us, with
// twenty alternatives 13.5.
#include <cooperative_groups.h>

#include "common.cuh"
#include "per_device.h"
#include "api.h"

namespace oa {

namespace cg = cooperative_groups;

typedef unsigned long long u64;

constexpr int LP_MAX_TOP = 32;
constexpr int LP_BATCH = 4;                // pieces of a thread under way
constexpr float LP_LOG2E = 1.4426950408889634f;
constexpr float LP_FAR = -1e4f;            // differences from the maximum end here: e^-10000 is 0, and 0 times it is 0

struct LogprobParams {
  const void* x;
  long long stride;
  const int* targets;
  float *logprobs, *entropy, *stats, *top_logprobs;
  int* top_ids;
  int top, rows, vocab, ignore;
  float scale;
};

__device__ __forceinline__ float lp_load(const float* p) { return *p; }
__device__ __forceinline__ float lp_load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float lp_max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// 16 bytes of logits
template <typename T> struct LpPiece;
template <> struct LpPiece<__nv_bfloat16> {
  static constexpr int N = 8;
  uint32_t w[4];
  __device__ __forceinline__ u64 pair(int i) const { return f2_bf16x2(w[i]); }
  __device__ __forceinline__ float at(int i) const { return __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16); }
  __device__ __forceinline__ float largest() const {         // NaN does not count
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(w);
    const float2 m = __bfloat1622float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
    return fmaxf(m.x, m.y);
  }
  __device__ __forceinline__ void none() { w[0] = w[1] = w[2] = w[3] = 0xff80ff80u; }      // -inf
  __device__ __forceinline__ void put(int i, const __nv_bfloat16* p) {
    const uint32_t b = *reinterpret_cast<const unsigned short*>(p);
    w[i >> 1] = i & 1 ? (w[i >> 1] & 0xffffu) | b << 16 : (w[i >> 1] & 0xffff0000u) | b;
  }
  __device__ __forceinline__ void set(int i, u64 v) { w[i] = f2_bf16(v); }
  __device__ __forceinline__ void set1(int i, float v) {
    const __nv_bfloat16 r = __float2bfloat16_rn(v);
    put(i, &r);
  }
  __device__ __forceinline__ void get(int i, __nv_bfloat16* p) const { *reinterpret_cast<unsigned short*>(p) = (unsigned short)(i & 1 ? w[i >> 1] >> 16 : w[i >> 1] & 0xffffu); }
};
template <> struct LpPiece<float> {
  static constexpr int N = 4;
  uint32_t w[4];
  __device__ __forceinline__ u64 pair(int i) const { return f2_of(w[2 * i], w[2 * i + 1]); }
  __device__ __forceinline__ float at(int i) const { return __uint_as_float(w[i]); }
  __device__ __forceinline__ float largest() const { return fmax3(fmaxf(at(0), at(1)), at(2), at(3)); }
  __device__ __forceinline__ void none() { w[0] = w[1] = w[2] = w[3] = 0xff800000u; }
  __device__ __forceinline__ void put(int i, const float* p) { w[i] = __float_as_uint(*p); }
  __device__ __forceinline__ void set(int i, u64 v) { f2_to(v, w[2 * i], w[2 * i + 1]); }
  __device__ __forceinline__ void set1(int i, float v) { w[i] = __float_as_uint(v); }
  __device__ __forceinline__ void get(int i, float* p) const { *p = __uint_as_float(w[i]); }
};

// A row as aligned pieces: piece p holds elements p N - head and on.  The first and the last may reach beyond the row: those elements are not touched,
// and count as -inf.
template <typename T>
struct LpRow {
  static constexpr int N = LpPiece<T>::N;
  const T* x;                              // where the first piece begins
  int head, vocab;
  __device__ __forceinline__ LpRow(const T* row, int vocab_) : head((int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T))), vocab(vocab_) { x = row - head; }
  __device__ __forceinline__ int pieces() const { return (int)(((long long)head + vocab + N - 1) / N); }
  __device__ __forceinline__ int first(int p) const { return p * N - head; }
  __device__ __forceinline__ bool whole(int p) const { return p * N >= head && p * N <= head + vocab - N; }
  __device__ __forceinline__ bool holds(int e) const { return e >= 0 && e < vocab; }
  __device__ __forceinline__ float element(int e) const { return lp_load(x + head + e); }
  __device__ __forceinline__ void load(LpPiece<T>& to, int p) const {
    if (whole(p)) {
      const uint4 v = reinterpret_cast<const uint4*>(x)[p];
      to.w[0] = v.x; to.w[1] = v.y; to.w[2] = v.z; to.w[3] = v.w;
    } else {
      to.none();
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (holds(first(p) + i)) to.put(i, x + p * N + i);
    }
  }
};

// Sums of exponentials below a maximum
struct LpSums {
  float m, l, s;
  __device__ __forceinline__ void raise(float to) {          // to > m
    if (m != -INFINITY) {
      const float d = m - to, a = exp2f(d * LP_LOG2E);
      s = a * fmaf(l, fmaxf(d, LP_FAR), s);
      l *= a;
    }
    m = to;
  }
  __device__ __forceinline__ void join(LpSums b) {
    if (b.m > m) raise(b.m);
    else if (m > b.m) b.raise(m);
    l += b.l;
    s += b.s;
  }
};

// Whole numbers that order like the logits, NaN as -inf; with the index, the lower one of equal logits the larger
__device__ __forceinline__ uint32_t lp_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return x != x ? 0x007fffffu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float lp_unkey(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
__device__ __forceinline__ u64 lp_rank(uint32_t key, int i) { return ((u64)key << 32) | (uint32_t)~i; }

// A row is worked on by a team: a warp of a block, or a whole block (of a cluster).
template <int THREADS>
__device__ __forceinline__ void lp_sync() {
  if (THREADS == 32) __syncwarp();
  else __syncthreads();
}

template <int THREADS, bool TOP>
struct LpShared {
  static constexpr int WARPS = THREADS / 32, GROUPS = THREADS < 128 ? THREADS : 128, PER = THREADS / GROUPS;
  static constexpr int LIST = !TOP ? 1 : THREADS == 32 ? 128 : 1024;      // candidates for the alternatives
  u64 list[LIST], best[LP_MAX_TOP], red[WARPS];
  LpSums sums[WARPS], total;
  float log_l;
  uint32_t maxima[GROUPS];
  unsigned short hot[TOP ? THREADS : 1];
  int count, hots, scan[WARPS];
  uint32_t bound;
};

// s.best[rank] = element, of the n in s.list, as far as rank < top
template <int THREADS, typename S>
__device__ __forceinline__ void lp_order(S& s, int n, int top, int tid) {
  for (int i = tid; i < n; i += THREADS) {
    const u64 mine = s.list[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += s.list[j] > mine;
    if (rank < top && mine) s.best[rank] = mine;
  }
}

// The `top` first of the ranking of pieces [p0, p1) into s.best, 0 where there are fewer.  tmax: the largest key of this thread's pieces p0 + tid +
// i THREADS
template <typename T, int THREADS, typename S>
__device__ __forceinline__ void lp_top(S& s, const LpRow<T>& row, int p0, int p1, uint32_t tmax, int top, int tid) {
  constexpr int N = LpPiece<T>::N;
  constexpr uint32_t LOW = sizeof(T) == 2 ? 0xffffu : 0u;      // bits of a key that say nothing
  const int lane = tid & 31, warp = tid >> 5;
  // a bound that at least `top` elements reach: the top-th largest of the maxima of groups of threads
  uint32_t g = tmax;
#pragma unroll
  for (int o = 1; o < S::PER; o <<= 1) g = max(g, __shfl_xor_sync(0xffffffffu, g, o));
  if (tid % S::PER == 0) s.maxima[tid / S::PER] = g;
  if (tid == 0) s.count = s.hots = 0;
  if (tid < LP_MAX_TOP) s.best[tid] = 0;
  lp_sync<THREADS>();
  if (warp == 0) {
    uint32_t mine[S::GROUPS / 32], bound = 0;
#pragma unroll
    for (int i = 0; i < S::GROUPS / 32; ++i) mine[i] = s.maxima[i * 32 + lane] & ~LOW;
    uint32_t hi = mine[0], lo = mine[0];
#pragma unroll
    for (int i = 1; i < S::GROUPS / 32; ++i) { hi = max(hi, mine[i]); lo = min(lo, mine[i]); }
    hi = __reduce_max_sync(0xffffffffu, hi);
    lo = __reduce_min_sync(0xffffffffu, lo);
    uint32_t bit = top == 1 || hi == lo ? 0 : 1u << (31 - __clz(hi ^ lo));       // the first in which they differ; one alternative is at the largest maximum
    bound = bit ? hi & ~(2 * bit - 1) : hi;
#pragma unroll 1
    for (; bit > LOW; bit >>= 1) {
      const uint32_t c = bound | bit;
      int n = 0;
#pragma unroll
      for (int i = 0; i < S::GROUPS / 32; ++i) n += __popc(__ballot_sync(0xffffffffu, mine[i] >= c));
      if (n >= top) bound = c;
      if (n == top) break;                 // a closer one would leave out little more
    }
    if (lane == 0) s.bound = bound;
  }
  lp_sync<THREADS>();
  const uint32_t bound = s.bound;
  // The pieces of the threads whose maximum reaches the bound, dealt to all; elements from `from` on go into the list as far as there is room
  if (tmax >= bound) s.hot[atomicAdd(&s.hots, 1)] = (unsigned short)tid;
  lp_sync<THREADS>();
  const int hots = s.hots, steps = (p1 - p0 + THREADS - 1) / THREADS;
  const auto collect = [&](uint32_t from) {
    for (int i = tid; i < hots * steps; i += THREADS) {
      const int h = i / steps, p = p0 + s.hot[h] + (i - h * steps) * THREADS;
      if (p >= p1) continue;
      if (*static_cast<volatile int*>(&s.count) > S::LIST) break;          // too many already (a share that is masked as a whole, say)
      LpPiece<T> v;
      row.load(v, p);
      const int e = row.first(p);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const uint32_t k = lp_key(v.at(j));
        if (k >= from && row.holds(e + j)) {
          const int at = atomicAdd(&s.count, 1);
          if (at < S::LIST) s.list[at] = lp_rank(k, e + j);
        }
      }
    }
  };
  collect(bound);
  lp_sync<THREADS>();
  int n = s.count;
  if (n > S::LIST) {
    // very many equal logits, masked ones for instance: those above the bound, then of those at it the first by index
    lp_sync<THREADS>();
    if (tid == 0) s.count = 0;
    lp_sync<THREADS>();
    collect((bound | LOW) + 1);
    lp_sync<THREADS>();
    n = s.count;
    if (n <= S::LIST - LP_MAX_TOP) {
      for (int q0 = p0; q0 < p1 && n < top; q0 += THREADS) {     // a step's elements lie side by side: their order is that of threads and pieces
        int e = 0;
        unsigned hit = 0;
        uint32_t key = 0;
        if (q0 + tid < p1) {
          LpPiece<T> v;
          row.load(v, q0 + tid);
          e = row.first(q0 + tid);
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const uint32_t k = lp_key(v.at(i));
            if ((k & ~LOW) == bound && row.holds(e + i)) { hit |= 1u << i; key = k; }
          }
        }
        const int mine = __popc(hit);
        int sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int u = __shfl_up_sync(0xffffffffu, sum, o);
          if (lane >= o) sum += u;
        }
        lp_sync<THREADS>();
        if (lane == 31) s.scan[warp] = sum;
        lp_sync<THREADS>();
        int before = n + sum - mine, all = 0;
        for (int w = 0; w < S::WARPS; ++w) { if (w < warp) before += s.scan[w]; all += s.scan[w]; }
        for (; hit && before < top; hit &= hit - 1, ++before) s.list[before] = lp_rank(key, e + __ffs(hit) - 1);
        n = min(n + all, max(top, n));
      }
      lp_sync<THREADS>();
    } else {
      // few threads with more than fits above it: one after the other
      u64 last = ~0ull;
      for (int k = 0; k < top; ++k) {
        u64 best = 0;
        for (int p = p0 + tid; p < p1; p += THREADS) {
          LpPiece<T> v;
          row.load(v, p);
          const int e = row.first(p);
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const u64 r = lp_rank(lp_key(v.at(i)), e + i);
            if (r < last && r > best && row.holds(e + i)) best = r;
          }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
        lp_sync<THREADS>();
        if (lane == 0) s.red[warp] = best;
        lp_sync<THREADS>();
        for (int w = 0; w < S::WARPS; ++w) best = max(best, s.red[w]);
        last = best;
        if (tid == 0) s.best[k] = best;
      }
      lp_sync<THREADS>();
      return;
    }
  }
  lp_order<THREADS>(s, n, top, tid);
  lp_sync<THREADS>();
}

__device__ __forceinline__ LpSums lp_warp_join(LpSums a, int lanes = 32) {
  LpSums to{a.m, 0.f, 0.f};
  for (int o = lanes >> 1; o > 0; o >>= 1) to.m = fmaxf(to.m, __shfl_xor_sync(0xffffffffu, to.m, o));
  if (to.m > a.m) a.raise(to.m);
  for (int o = lanes >> 1; o > 0; o >>= 1) {
    a.l += __shfl_xor_sync(0xffffffffu, a.l, o);
    a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
  }
  return a;
}

// The sums of a piece's elements, added to l and s; NaN where an element is -inf (0 times infinity) unless FAR, which lets differences end at LP_FAR
template <bool FAR, typename T>
__device__ __forceinline__ void lp_add(const LpPiece<T>& v, u64 scale2, u64 neg_m2, u64& l2, u64& s2) {
#pragma unroll
  for (int i = 0; i < LpPiece<T>::N / 2; ++i) {
    u64 d = f2_fma(v.pair(i), scale2, neg_m2);
    if (FAR) {
      uint32_t d0, d1;
      f2_to(d, d0, d1);
      d = f2_of(__float_as_uint(lp_max_nan(__uint_as_float(d0), LP_FAR)), __float_as_uint(lp_max_nan(__uint_as_float(d1), LP_FAR)));
    }
    const u64 e = exp2_mufu2(f2_mul(d, f2_splat(LP_LOG2E)));
    l2 = f2_add(l2, e);
    s2 = f2_fma(e, d, s2);
  }
}
__device__ __forceinline__ float lp_both(u64 v) {
  uint32_t a, b;
  f2_to(v, a, b);
  return __uint_as_float(a) + __uint_as_float(b);
}

// fp32 teams of a block have more under way, as far as registers go: 16384 x 32000 with 4 / 5 / 6 / 8 322 / 315 / 309 / 297 us, with five alternatives 393 / 385 / 374 / 369 (but
// 32 x 201088 12.5 / 12.7 / 12.8 / 13.7).  bf16 with 4 / 6: one call after the other on the same logits 189 / 187 and 230 / 226, on others each time, out of memory, 4096 x 32000 with
// five alternatives 68.1 / 69.5 and 16384 x 32000 with its gradient 592 / 600.
template <typename T, int THREADS, bool TOP> constexpr int LP_DEEP = sizeof(T) == 2 || THREADS < 128 ? LP_BATCH : TOP ? 6 : 8;
// The sums of pieces p0 + tid + i THREADS below p1, and the largest logit there; BATCH: pieces of a thread under way
template <typename T, int THREADS, int BATCH>
__device__ __forceinline__ LpSums lp_sums(const LpRow<T>& row, int p0, int p1, int tid, float scale, float& tmax) {
  LpSums a{-INFINITY, 0.f, 0.f};
  const u64 scale2 = f2_splat(scale);
  tmax = -INFINITY;
  LpPiece<T> v[BATCH];
#pragma unroll
  for (int b = 0; b < BATCH; ++b)
    if (p0 + tid + b * THREADS < p1) row.load(v[b], p0 + tid + b * THREADS);
  for (int q = p0 + tid; q < p1; q += BATCH * THREADS) {
#pragma unroll
    for (int b = 0; b < BATCH; ++b)
      if (q + b * THREADS < p1) tmax = fmaxf(tmax, v[b].largest());
    const float top = tmax * scale;
    if (top > a.m) a.raise(top);
    const u64 neg_m2 = f2_splat(a.m == -INFINITY ? 0.f : -a.m);
    u64 l2 = 0, s2 = 0;
#pragma unroll
    for (int b = 0; b < BATCH; ++b)
      if (q + b * THREADS < p1) {
        lp_add<false>(v[b], scale2, neg_m2, l2, s2);
        const int next = q + (BATCH + b) * THREADS;      // the place that is free again takes the next step's piece
        if (next < p1) row.load(v[b], next);
      }
    float s1 = lp_both(s2);
    if (s1 != s1) {
      l2 = s2 = 0;
#pragma unroll 1
      for (int i = q; i < p1 && i < q + BATCH * THREADS; i += THREADS) {
        LpPiece<T> again;
        row.load(again, i);
        lp_add<true>(again, scale2, neg_m2, l2, s2);
      }
      s1 = lp_both(s2);
    }
    a.l += lp_both(l2);
    a.s += s1;
  }
  return a;
}

// +inf leaves NaN in the sums, like NaN itself
struct LpResult {
  bool none;
  float m, log_l, scale;
  __device__ __forceinline__ LpResult(LpSums a, float scale_) : none(a.m == -INFINITY && a.l == 0.f), m(a.l != a.l ? NAN : a.m), log_l(none ? 0.f : logf(a.l)), scale(scale_) {}
  __device__ __forceinline__ float logprob(float x) const { return none ? -INFINITY : fmaf(x, scale, -m) - log_l; }
};
template <typename T>
__device__ __forceinline__ void lp_write(const LogprobParams& p, const LpRow<T>& row, int r, const LpSums& a, const LpResult& to) {
  const int t = p.targets[r];
  p.logprobs[r] = t == p.ignore ? 0.f : t >= 0 && t < p.vocab ? to.logprob(row.element(t)) : NAN;
  p.entropy[r] = to.none ? 0.f : to.log_l - a.s / a.l;
  p.stats[2ll * r] = to.m;
  p.stats[2ll * r + 1] = to.log_l;
}

// A team of THREADS to a row: 32, eight rows to a block of 256, or a block, gridDim.x = rows * CTAs of a cluster
template <typename T, int THREADS, bool TOP>
__global__ void __launch_bounds__(THREADS == 128 ? 128 : 256, THREADS == 128 ? 8 : 4) logprob_kernel(const __grid_constant__ LogprobParams p) {
  using S = LpShared<THREADS, TOP>;
  constexpr int TEAMS = THREADS == 32 ? 8 : 1;
  __shared__ S shared[TEAMS];
  pdl_launch_dependents();
  pdl_wait();
  S& s = shared[TEAMS > 1 ? threadIdx.x >> 5 : 0];
  int parts = 1, part = 0;
  if constexpr (TEAMS == 1) {
    parts = cg::this_cluster().num_blocks();
    part = cg::this_cluster().block_rank();
  }
  const int r = TEAMS > 1 ? blockIdx.x * TEAMS + (threadIdx.x >> 5) : blockIdx.x / parts, tid = threadIdx.x % THREADS, lane = tid & 31, warp = tid >> 5;
  if (TEAMS > 1 && r >= p.rows) return;
  const LpRow<T> row(static_cast<const T*>(p.x) + r * p.stride, p.vocab);
  const int all = row.pieces(), per = (all + parts - 1) / parts, p0 = min(part * per, all), p1 = min(p0 + per, all);
  float tmax;                              // of the logits themselves
  LpSums a = lp_sums<T, THREADS, LP_DEEP<T, THREADS, TOP>>(row, p0, p1, tid, p.scale, tmax);
  a = lp_warp_join(a);
  if (THREADS > 32) {
    if (lane == 0) s.sums[warp] = a;
    __syncthreads();
    if (warp == 0) a = lp_warp_join(lane < S::WARPS ? s.sums[lane] : LpSums{-INFINITY, 0.f, 0.f});
    if (parts > 1 && tid == 0) s.total = a;
  }
  if constexpr (TOP) lp_top<T, THREADS>(s, row, p0, p1, lp_key(tmax), p.top, tid);
  if constexpr (TEAMS == 1) {
    if (parts > 1) {
      cg::this_cluster().sync();
      if (part == 0) {
        if (warp == 0) a = lp_warp_join(lane < parts ? cg::this_cluster().map_shared_rank(&s, lane)->total : LpSums{-INFINITY, 0.f, 0.f});
        if constexpr (TOP) {
          for (int i = tid; i < parts * p.top; i += THREADS) s.list[i] = cg::this_cluster().map_shared_rank(&s, i / p.top)->best[i % p.top];
          __syncthreads();
          lp_order<THREADS>(s, parts * p.top, p.top, tid);      // the largest of all are at least as many as this CTA's own: every place is written anew
        }
      }
      cg::this_cluster().sync();           // the others' shared memory has been read
      if (part != 0) return;
    }
  }
  if (warp == 0) {
    const LpResult to(a, p.scale);
    if (lane == 0) lp_write(p, row, r, a, to);
    if (TOP && lane < p.top) {
      const u64 v = s.best[lane];
      p.top_ids[(long long)r * p.top + lane] = (int)~(uint32_t)v;
      p.top_logprobs[(long long)r * p.top + lane] = to.logprob(lp_unkey((uint32_t)(v >> 32)));
    }
  }
}

// Short rows without alternatives: eight lanes to a row, so that what a row costs once (the join, the logarithms) is shared by four rows
constexpr int LP_LANES = 8;
template <typename T>
__global__ void __launch_bounds__(256, 4) logprob_short_kernel(const __grid_constant__ LogprobParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int r = blockIdx.x * (256 / LP_LANES) + threadIdx.x / LP_LANES, tid = threadIdx.x % LP_LANES;
  const LpRow<T> row(static_cast<const T*>(p.x) + (r < p.rows ? r : 0) * p.stride, p.vocab);
  float tmax;
  const LpSums a = lp_warp_join(lp_sums<T, LP_LANES, LP_BATCH>(row, 0, r < p.rows ? row.pieces() : 0, tid, p.scale, tmax), LP_LANES);
  if (tid == 0 && r < p.rows) lp_write(p, row, r, a, LpResult(a, p.scale));
}

struct LogprobBwdParams {
  const void* x;
  long long stride;
  const int* targets;
  const float *entropy, *stats, *dlogprobs, *dentropy;
  void* dx;
  long long d_stride;
  int rows, vocab, ignore, team_log2;
  float scale;
};

// Blocks of 2^team_log2 threads to a row and 256 / 2^team_log2 rows; blockIdx.y: which part of the row's pieces, those of the logits.  Where the gradient's rows
// lie otherwise (`apart`) their elements are written one by one.  ENTROPY: dentropy is given.
template <typename T, bool ENTROPY>
__global__ void __launch_bounds__(256, 5) logprob_bwd_kernel(const __grid_constant__ LogprobBwdParams p) {
  constexpr int N = LpPiece<T>::N;
  pdl_launch_dependents();
  pdl_wait();
  const int team = 1 << p.team_log2, r = (blockIdx.x << (8 - p.team_log2)) + (threadIdx.x >> p.team_log2);
  if (r >= p.rows) return;
  const LpRow<T> row(static_cast<const T*>(p.x) + r * p.stride, p.vocab);
  T* dx = static_cast<T*>(p.dx) + r * p.d_stride - row.head;
  const bool apart = (reinterpret_cast<uintptr_t>(dx) & 15) != 0;
  const int all = row.pieces(), step = gridDim.y * team;
  int q = blockIdx.y * team + (threadIdx.x & (team - 1));
  LpPiece<T> v[LP_BATCH];
  const auto fetch = [&] {
#pragma unroll
    for (int b = 0; b < LP_BATCH; ++b)
      if (q + b * step < all) row.load(v[b], q + b * step);
  };
  fetch();                                 // beside the row's own numbers
  const float m = p.stats[2ll * r], log_l = p.stats[2ll * r + 1];
  const int target = p.targets[r];
  const bool none = m == -INFINITY;        // no gradient at all
  const float g = none || target == p.ignore || !p.dlogprobs ? 0.f : target >= 0 && target < p.vocab ? p.dlogprobs[r] * p.scale : NAN;
  const float h = ENTROPY && !none ? p.dentropy[r] * p.scale : 0.f;
  // dx = p_j (-h log p_j - (h H + g)), and g more at the target
  const u64 scale2 = f2_splat(p.scale), neg_m2 = f2_splat(none ? 0.f : -m), neg_l2 = f2_splat(-log_l), h2 = f2_splat(-h),
            c2 = f2_splat(-(ENTROPY && !none ? fmaf(h, p.entropy[r], g) : g));
  while (q < all) {
#pragma unroll
    for (int b = 0; b < LP_BATCH; ++b) {
      const int at = q + b * step;
      if (at >= all) break;
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        u64 d = f2_add(f2_fma(v[b].pair(i), scale2, neg_m2), neg_l2), f = c2;
        if (ENTROPY) {
          uint32_t d0, d1;
          f2_to(d, d0, d1);
          d = f2_of(__float_as_uint(lp_max_nan(__uint_as_float(d0), LP_FAR)), __float_as_uint(lp_max_nan(__uint_as_float(d1), LP_FAR)));
          f = f2_fma(h2, d, c2);
        }
        v[b].set(i, f2_mul(exp2_mufu2(f2_mul(d, f2_splat(LP_LOG2E))), f));
      }
      const int hit = target - row.first(at);
      if ((unsigned)hit < (unsigned)N && row.holds(target) && !none) {      // its logit still stands where the gradient may go
        const float d = lp_max_nan(fmaf(row.element(target), p.scale, -m) - log_l, LP_FAR);
        uint32_t c, unused;
        f2_to(c2, c, unused);
        const float w = fmaf(fast_exp2(d * LP_LOG2E), fmaf(-h, d, __uint_as_float(c)), g);
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (i == hit) v[b].set1(i, w);
      }
      if (row.whole(at) && !apart) {
        reinterpret_cast<uint4*>(dx)[at] = make_uint4(v[b].w[0], v[b].w[1], v[b].w[2], v[b].w[3]);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (row.holds(row.first(at) + i)) v[b].get(i, dx + at * N + i);
      }
    }
    q += LP_BATCH * step;
    fetch();
  }
}

template <typename T, int THREADS>
static int logprob_launch(const LogprobParams& p, int parts, cudaStream_t st) {
  const long long blocks = THREADS == 32 ? ((long long)p.rows + 7) / 8 : (long long)p.rows * parts;
  if (blocks > 0x7fffffffll) return OA_ERR_TOO_LARGE;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(THREADS == 32 ? 256 : THREADS);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = parts;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_on(blocks <= PDL_SHORT_BLOCKS) ? 2 : 1;
  const cudaError_t rc = p.top > 0 ? cudaLaunchKernelEx(&cfg, logprob_kernel<T, THREADS, true>, p) : cudaLaunchKernelEx(&cfg, logprob_kernel<T, THREADS, false>, p);
  return rc == cudaSuccess ? OA_OK : OA_ERR_LAUNCH;
}

template <typename T>
static int logprob_run(const LogprobParams& p, cudaStream_t st) {
  // Otherwise a warp to a row of up to 2048 elements; for longer ones as many CTAs to a row as leave no SM without two, each with 2048 elements at least.  Smaller CTAs cover
  // one another's meetings where there are several waves of them, larger ones end sooner where there is one (bf16, five alternatives, threads 128 / 256: 32 x 201088 12.2 / 11.3
  // us, 64 x 50257 9.1 / 8.8) or a thread has many pieces, which its second look pays for by the alternatives.  4096 rows of 4000 pieces, bf16 x 32000 and fp32 x 16000, with
  // five 65 / 73 and 58 / 63, with twenty 80 / 83 and 68 / 70; of 5000 and 6000, bf16 x 40000 and fp32 x 24001, five 78 / 84 and 79 / 84, twenty 98 / 94 and 100 / 93; of 8100, five
  // 118 / 118 and 101 / 100, none 99 / 102 and 84 / 81.  Two waves, bf16 1800 x 40000, five 40 / 43; one, 600 rows of 4000 and 5000, 18.5 / 18.1 and 22 / 20.
  // Eight lanes to a row where there are rows enough for every SM's warps, or a row is one 16-byte piece or two to a lane (bf16, eight lanes / a warp to
  // a row: 200000 x 256 30 / 86 us, 60000 x 1000 28 / 36, 20000 x 2000 20 / 19, 2000 x 128 2.2 / 2.7, 2000 x 500 4.6 / 3.9; fp32, 20000 x 2000 41 / 33).
  const long long bytes = (long long)p.vocab * sizeof(T);
  if (p.top == 0 && (bytes <= 256 || (bytes <= 4096 && p.rows >= 64 * sm_count()))) {
    launch_short(logprob_short_kernel<T>, dim3((unsigned)((p.rows + 256 / LP_LANES - 1) / (256 / LP_LANES))), dim3(256), 0, st, p);
    return cudaGetLastError() == cudaSuccess ? OA_OK : OA_ERR_LAUNCH;
  }
  if (p.vocab <= 2048) return logprob_launch<T, 32>(p, 1, st);
  int parts = 1;
  while (parts < 8 && (long long)p.rows * parts <= 2 * sm_count() && p.vocab / (2 * parts) >= 2048) parts *= 2;
  if (p.rows >= 4 * sm_count() && p.vocab / LpPiece<T>::N <= (p.top <= 8 && p.rows >= 12 * sm_count() ? 7000 : 4200)) return logprob_launch<T, 128>(p, parts, st);
  return logprob_launch<T, 256>(p, parts, st);
}

template <typename T>
static int logprob_bwd_run(LogprobBwdParams& p, cudaStream_t st) {
  // threads to a row that four pieces each fill, and as many blocks side by side as it then still takes; a row that does not begin on 16 bytes has a piece more, for
  // which the loop goes round again (200000 x 256 in bf16, with threads for that piece too / without: 55 / 43 us)
  const long long pieces = ((long long)p.vocab + LpPiece<T>::N - 1) / LpPiece<T>::N;
  p.team_log2 = 3;
  while (p.team_log2 < 8 && (LP_BATCH << p.team_log2) < pieces) ++p.team_log2;
  const long long parts = (pieces + (LP_BATCH << p.team_log2) - 1) / (LP_BATCH << p.team_log2);
  const dim3 grid((unsigned)(((long long)p.rows + (256 >> p.team_log2) - 1) >> (8 - p.team_log2)), (unsigned)(parts < 65535 ? parts : 65535));
  if (p.dentropy) launch_short(logprob_bwd_kernel<T, true>, grid, dim3(256), 0, st, p);
  else launch_short(logprob_bwd_kernel<T, false>, grid, dim3(256), 0, st, p);
  return cudaGetLastError() == cudaSuccess ? OA_OK : OA_ERR_LAUNCH;
}

}  // namespace oa

using namespace oa;

extern "C" int oa_token_logprobs(int dtype, const void* logits, long long stride, const int* targets, float* logprobs, float* entropy, float* stats,
                                 float* top_logprobs, int* top_ids, int top, int rows, int vocab, float scale, int ignore_index, void* stream) {
  if (dtype != OA_F32 && dtype != OA_BF16) return OA_ERR_UNSUPPORTED;
  if (rows < 0 || vocab < 1 || top < 0 || top > vocab || stride < 0 || !(scale > 0.f)) return OA_ERR_ARG;
  if (top > LP_MAX_TOP) return OA_ERR_UNSUPPORTED;
  if (vocab > 0x7ffffff0) return OA_ERR_TOO_LARGE;
  if (rows == 0) return OA_OK;
  const LogprobParams p{logits, stride, targets, logprobs, entropy, stats, top_logprobs, top_ids, top, rows, vocab, ignore_index, scale};
  return dtype == OA_F32 ? logprob_run<float>(p, (cudaStream_t)stream) : logprob_run<__nv_bfloat16>(p, (cudaStream_t)stream);
}

extern "C" int oa_token_logprobs_bwd(int dtype, const void* logits, long long stride, const int* targets, const float* entropy, const float* stats,
                                     const float* dlogprobs, const float* dentropy, void* dlogits, long long d_stride, int rows, int vocab, float scale,
                                     int ignore_index, void* stream) {
  if (dtype != OA_F32 && dtype != OA_BF16) return OA_ERR_UNSUPPORTED;
  if (rows < 0 || vocab < 1 || stride < 0 || (rows > 1 && d_stride < vocab) || !(scale > 0.f)) return OA_ERR_ARG;
  if (vocab > 0x7ffffff0) return OA_ERR_TOO_LARGE;
  if (rows == 0) return OA_OK;
  LogprobBwdParams p{logits, stride, targets, entropy, stats, dlogprobs, dentropy, dlogits, d_stride, rows, vocab, ignore_index, 0, scale};
  return dtype == OA_F32 ? logprob_bwd_run<float>(p, (cudaStream_t)stream) : logprob_bwd_run<__nv_bfloat16>(p, (cudaStream_t)stream);
}
