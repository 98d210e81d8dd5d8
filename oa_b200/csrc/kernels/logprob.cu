// Log-probabilities of given tokens, with the entropy and the likeliest alternatives of each row of logits, and the logits' gradient.
//
// For a row y = scale * x with largest element m:  l = sum exp(y - m),  log p_j = (y_j - m) - log l,  H = -sum p_j log p_j = log l - s / l
// with s = sum exp(y - m) (y - m).  The differences from m are what is summed, so that nothing of the size of m cancels.  With gradients g of the
// target's log-probability and h of the entropy,
//   dx_j = scale * (g ([j = target] - p_j) - h p_j (log p_j + H)).
// A logit of -inf has probability 0 and adds nothing anywhere.  A row with NaN or +inf is NaN; a row without anything above -inf has
// log-probability -inf, entropy 0 and no gradient.
//
// Forward reads a row once, in 16-byte pieces, four to a thread under way: every thread sums below a maximum of its own, and the threads meet at the
// end.  The alternatives cost no second pass: the k-th largest of the threads' maxima has k elements at or above it, so it is a bound that few others
// reach, and only the threads whose maximum does read their pieces again, from L2.  Long rows of which there are few are cut over a cluster of CTAs
// that meet in distributed shared memory.  Backward is one pass.  Bound by the bytes.
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
  __device__ __forceinline__ void none() { w[0] = w[1] = w[2] = w[3] = 0xff80ff80u; }      // -inf
  __device__ __forceinline__ void put(int i, const __nv_bfloat16* p) {
    const uint32_t b = *reinterpret_cast<const unsigned short*>(p);
    w[i >> 1] = i & 1 ? (w[i >> 1] & 0xffffu) | b << 16 : (w[i >> 1] & 0xffff0000u) | b;
  }
  __device__ __forceinline__ void set(int i, u64 v) { w[i] = f2_bf16(v); }
  __device__ __forceinline__ void get(int i, __nv_bfloat16* p) const { *reinterpret_cast<unsigned short*>(p) = (unsigned short)(i & 1 ? w[i >> 1] >> 16 : w[i >> 1] & 0xffffu); }
};
template <> struct LpPiece<float> {
  static constexpr int N = 4;
  uint32_t w[4];
  __device__ __forceinline__ u64 pair(int i) const { return f2_of(w[2 * i], w[2 * i + 1]); }
  __device__ __forceinline__ float at(int i) const { return __uint_as_float(w[i]); }
  __device__ __forceinline__ void none() { w[0] = w[1] = w[2] = w[3] = 0xff800000u; }
  __device__ __forceinline__ void put(int i, const float* p) { w[i] = __float_as_uint(*p); }
  __device__ __forceinline__ void set(int i, u64 v) { f2_to(v, w[2 * i], w[2 * i + 1]); }
  __device__ __forceinline__ void get(int i, float* p) const { *p = __uint_as_float(w[i]); }
};

// A row as aligned pieces: piece p holds elements p N - head and on.  The first and the last may reach beyond the row: those elements are not touched,
// and count as -inf.
template <typename T>
struct LpRow {
  static constexpr int N = LpPiece<T>::N;
  const T* x;
  int head, vocab;
  __device__ __forceinline__ LpRow(const T* row, int vocab_) : x(row), head((int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T))), vocab(vocab_) {}
  __device__ __forceinline__ int pieces() const { return (int)(((long long)head + vocab + N - 1) / N); }
  __device__ __forceinline__ int first(int p) const { return p * N - head; }
  __device__ __forceinline__ bool whole(int e) const { return e >= 0 && e <= vocab - N; }
  __device__ __forceinline__ void load(LpPiece<T>& to, int p) const {
    const int e = first(p);
    if (whole(e)) {
      const uint4 v = *reinterpret_cast<const uint4*>(x + e);
      to.w[0] = v.x; to.w[1] = v.y; to.w[2] = v.z; to.w[3] = v.w;
    } else {
      to.none();
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (e + i >= 0 && e + i < vocab) to.put(i, x + e + i);
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

template <int THREADS, bool TOP>
struct LpShared {
  static constexpr int WARPS = THREADS / 32, GROUPS = THREADS < 128 ? THREADS : 128, PER = THREADS / GROUPS;
  static constexpr int LIST = !TOP ? 1 : THREADS == 32 ? 256 : THREADS == 128 ? 1024 : 2048;      // candidates for the alternatives
  u64 list[LIST], best[LP_MAX_TOP], red[WARPS];
  LpSums sums[WARPS];
  uint32_t maxima[GROUPS];
  int count, scan[WARPS];
  uint32_t bound;
};

// The `top` first of the ranking of pieces [p0, p1) into s.best, 0 where there are fewer.  tmax: the largest key of this thread's pieces p0 + tid +
// i THREADS
template <typename T, int THREADS, typename S>
__device__ __forceinline__ void lp_top(S& s, const LpRow<T>& row, int p0, int p1, uint32_t tmax, int top) {
  constexpr int N = LpPiece<T>::N;
  constexpr uint32_t LOW = sizeof(T) == 2 ? 0xffffu : 0u;      // bits of a key that say nothing
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // a bound that at least `top` elements reach: the top-th largest of the maxima of groups of threads
  uint32_t g = tmax;
#pragma unroll
  for (int o = 1; o < S::PER; o <<= 1) g = max(g, __shfl_xor_sync(0xffffffffu, g, o));
  if (tid % S::PER == 0) s.maxima[tid / S::PER] = g;
  if (tid == 0) s.count = 0;
  if (tid < LP_MAX_TOP) s.best[tid] = 0;
  __syncthreads();
  if (warp == 0) {
    uint32_t mine[S::GROUPS / 32], bound = 0;
#pragma unroll
    for (int i = 0; i < S::GROUPS / 32; ++i) mine[i] = s.maxima[i * 32 + lane] & ~LOW;
#pragma unroll 1
    for (uint32_t bit = 1u << 31; bit > LOW; bit >>= 1) {
      const uint32_t c = bound | bit;
      int n = 0;
#pragma unroll
      for (int i = 0; i < S::GROUPS / 32; ++i) n += __popc(__ballot_sync(0xffffffffu, mine[i] >= c));
      if (n >= top) bound = c;
    }
    if (lane == 0) s.bound = bound;
  }
  __syncthreads();
  const uint32_t bound = s.bound;
  // everything from `from` on goes into the list, as far as there is room
  const auto collect = [&](uint32_t from) {
    if (tmax < from) return;
    for (int p = p0 + tid; p < p1; p += LP_BATCH * THREADS) {
      LpPiece<T> v[LP_BATCH];
#pragma unroll
      for (int b = 0; b < LP_BATCH; ++b)
        if (p + b * THREADS < p1) row.load(v[b], p + b * THREADS);
#pragma unroll
      for (int b = 0; b < LP_BATCH; ++b) {
        if (p + b * THREADS >= p1) break;
        const int e = row.first(p + b * THREADS);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const uint32_t k = lp_key(v[b].at(i));
          if (k >= from && e + i >= 0 && e + i < row.vocab) {
            const int at = atomicAdd(&s.count, 1);
            if (at < S::LIST) s.list[at] = lp_rank(k, e + i);
          }
        }
      }
    }
  };
  collect(bound);
  __syncthreads();
  int n = s.count;
  if (n > S::LIST) {
    // very many equal logits, masked ones for instance: those above the bound, then of those at it the first by index
    __syncthreads();
    if (tid == 0) s.count = 0;
    __syncthreads();
    collect((bound | LOW) + 1);
    __syncthreads();
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
            if ((k & ~LOW) == bound && e + i >= 0 && e + i < row.vocab) { hit |= 1u << i; key = k; }
          }
        }
        const int mine = __popc(hit);
        int sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int u = __shfl_up_sync(0xffffffffu, sum, o);
          if (lane >= o) sum += u;
        }
        __syncthreads();
        if (lane == 31) s.scan[warp] = sum;
        __syncthreads();
        int before = n + sum - mine, all = 0;
        for (int w = 0; w < S::WARPS; ++w) { if (w < warp) before += s.scan[w]; all += s.scan[w]; }
        for (; hit && before < top; hit &= hit - 1, ++before) s.list[before] = lp_rank(key, e + __ffs(hit) - 1);
        n = min(n + all, max(top, n));
      }
      __syncthreads();
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
            if (r < last && r > best && e + i >= 0 && e + i < row.vocab) best = r;
          }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
        __syncthreads();
        if (lane == 0) s.red[warp] = best;
        __syncthreads();
        for (int w = 0; w < S::WARPS; ++w) best = max(best, s.red[w]);
        last = best;
        if (tid == 0) s.best[k] = best;
      }
      __syncthreads();
      return;
    }
  }
  for (int i = tid; i < n; i += THREADS) {
    const u64 mine = s.list[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += s.list[j] > mine;
    if (rank < top) s.best[rank] = mine;
  }
  __syncthreads();
}

// gridDim.x = rows * CTAs of a cluster; each cluster a row
template <typename T, int THREADS, bool TOP>
__global__ void __launch_bounds__(THREADS, THREADS == 512 ? 2 : 1) logprob_kernel(const __grid_constant__ LogprobParams p) {
  using S = LpShared<THREADS, TOP>;
  constexpr int N = LpPiece<T>::N;
  __shared__ S s;
  pdl_launch_dependents();
  pdl_wait();
  const cg::cluster_group cluster = cg::this_cluster();
  const int parts = cluster.num_blocks(), part = cluster.block_rank(), r = blockIdx.x / parts, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const LpRow<T> row(static_cast<const T*>(p.x) + r * p.stride, p.vocab);
  const int all = row.pieces(), per = (all + parts - 1) / parts, p0 = min(part * per, all), p1 = min(p0 + per, all);
  LpSums a{-INFINITY, 0.f, 0.f};
  float tmax = -INFINITY;                  // of the logits themselves
  u64 l2 = 0, s2 = 0;
  const u64 scale2 = f2_splat(p.scale), log2e2 = f2_splat(LP_LOG2E);
  for (int q = p0 + tid; q < p1; q += LP_BATCH * THREADS) {
    LpPiece<T> v[LP_BATCH];
#pragma unroll
    for (int b = 0; b < LP_BATCH; ++b) {
      if (q + b * THREADS < p1) row.load(v[b], q + b * THREADS);
      else v[b].none();
    }
    float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
    for (int b = 0; b < LP_BATCH; ++b)
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        m0 = fmax3(m0, v[b].at(i), v[b].at(i + 1));
        m1 = fmax3(m1, v[b].at(i + 2), v[b].at(i + 3));
      }
    tmax = fmax3(tmax, m0, m1);
    const float top = tmax * p.scale;
    if (top > a.m) {
      uint32_t u[4];
      f2_to(l2, u[0], u[1]);
      f2_to(s2, u[2], u[3]);
      a.l = __uint_as_float(u[0]) + __uint_as_float(u[1]);
      a.s = __uint_as_float(u[2]) + __uint_as_float(u[3]);
      a.raise(top);
      l2 = f2_of(__float_as_uint(a.l), 0);
      s2 = f2_of(__float_as_uint(a.s), 0);
    }
    const u64 neg_m2 = f2_splat(a.m == -INFINITY ? 0.f : -a.m);
#pragma unroll
    for (int b = 0; b < LP_BATCH; ++b)
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        uint32_t d0, d1;
        f2_to(f2_fma(v[b].pair(i), scale2, neg_m2), d0, d1);
        const u64 d = f2_of(__float_as_uint(lp_max_nan(__uint_as_float(d0), LP_FAR)), __float_as_uint(lp_max_nan(__uint_as_float(d1), LP_FAR)));
        const u64 e = exp2_mufu2(f2_mul(d, log2e2));
        l2 = f2_add(l2, e);
        s2 = f2_fma(e, d, s2);
      }
  }
  {
    uint32_t u[4];
    f2_to(l2, u[0], u[1]);
    f2_to(s2, u[2], u[3]);
    a.l = __uint_as_float(u[0]) + __uint_as_float(u[1]);
    a.s = __uint_as_float(u[2]) + __uint_as_float(u[3]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    a.join({__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.l, o), __shfl_xor_sync(0xffffffffu, a.s, o)});
  if (lane == 0) s.sums[warp] = a;
  if constexpr (TOP) lp_top<T, THREADS>(s, row, p0, p1, lp_key(tmax), p.top);
  if (parts > 1) cluster.sync();
  else __syncthreads();
  if (part == 0) {
    if (warp == 0) {
      // one entry to a lane: the warps of this CTA, then those of the others
      a = {-INFINITY, 0.f, 0.f};
      for (int i = lane; i < parts * S::WARPS; i += 32) {
        const int c = i / S::WARPS, w = i % S::WARPS;
        const S* from = parts > 1 ? cluster.map_shared_rank(&s, c) : &s;
        a.join(from->sums[w]);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
        a.join({__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.l, o), __shfl_xor_sync(0xffffffffu, a.s, o)});
      // +inf leaves NaN in the sums, like NaN itself
      const bool none = a.m == -INFINITY && a.l == 0.f;
      if (a.l != a.l) a.m = NAN;
      const float log_l = none ? 0.f : logf(a.l);
      const auto logprob = [&](float x) { return none ? -INFINITY : (fmaf(x, p.scale, -a.m)) - log_l; };
      if (lane == 0) {
        const int t = p.targets[r];
        p.logprobs[r] = t == p.ignore ? 0.f : t >= 0 && t < p.vocab ? logprob(lp_load(row.x + t)) : NAN;
        p.entropy[r] = none ? 0.f : log_l - a.s / a.l;
        p.stats[2ll * r] = a.m;
        p.stats[2ll * r + 1] = log_l;
      }
      if constexpr (TOP) {
        const long long out = (long long)r * p.top;
        const auto write = [&](int rank, u64 v) {
          p.top_ids[out + rank] = (int)~(uint32_t)v;
          p.top_logprobs[out + rank] = logprob(lp_unkey((uint32_t)(v >> 32)));
        };
        if (parts == 1) {
          if (lane < p.top) write(lane, s.best[lane]);
        } else {
          // the CTAs' lists are in order: an element's rank is the sum of where it would stand in each
          for (int i = lane; i < parts * p.top; i += 32) {
            const int c = i / p.top;
            const u64 mine = cluster.map_shared_rank(&s, c)->best[i % p.top];
            if (mine == 0) continue;
            int rank = i % p.top;
            for (int o = 0; o < parts && rank < p.top; ++o) {
              if (o == c) continue;
              const S* from = cluster.map_shared_rank(&s, o);
              int lo = 0, hi = p.top;
              while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (from->best[mid] > mine) lo = mid + 1;
                else hi = mid;
              }
              rank += lo;
            }
            if (rank < p.top) write(rank, mine);
          }
        }
      }
    }
  }
  if (parts > 1) cluster.sync();           // the others' shared memory has been read
}

struct LogprobBwdParams {
  const void* x;
  long long stride;
  const int* targets;
  const float *entropy, *stats, *dlogprobs, *dentropy;
  void* dx;
  long long d_stride;
  int rows, vocab, ignore;
  float scale;
};

// blockIdx.y: which part of the row's pieces.  Pieces are those of the logits; where the gradient's rows lie otherwise (`apart`) their elements are written
// one by one.
template <typename T>
__global__ void __launch_bounds__(256) logprob_bwd_kernel(const __grid_constant__ LogprobBwdParams p) {
  constexpr int N = LpPiece<T>::N;
  pdl_launch_dependents();
  pdl_wait();
  const int r = blockIdx.x;
  const LpRow<T> row(static_cast<const T*>(p.x) + r * p.stride, p.vocab);
  T* dx = static_cast<T*>(p.dx) + r * p.d_stride;
  const bool apart = ((reinterpret_cast<uintptr_t>(dx) ^ reinterpret_cast<uintptr_t>(row.x)) & 15) != 0;
  const float m = p.stats[2ll * r], log_l = p.stats[2ll * r + 1], H = p.entropy[r];
  const int target = p.targets[r];
  const float g = target == p.ignore || !p.dlogprobs ? 0.f : target >= 0 && target < p.vocab ? p.dlogprobs[r] * p.scale : NAN;
  const float h = p.dentropy ? p.dentropy[r] * p.scale : 0.f;
  const bool none = m == -INFINITY;
  const u64 scale2 = f2_splat(p.scale), neg_m2 = f2_splat(none ? 0.f : -m), neg_l2 = f2_splat(-log_l), log2e2 = f2_splat(LP_LOG2E), h2 = f2_splat(none ? 0.f : h),
            c2 = f2_splat(none ? 0.f : fmaf(h, H, g)), neg2 = f2_splat(-1.f);
  const int all = row.pieces(), step = gridDim.y * 256;
  for (int q = blockIdx.y * 256 + threadIdx.x; q < all; q += LP_BATCH * step) {
    LpPiece<T> v[LP_BATCH];
#pragma unroll
    for (int b = 0; b < LP_BATCH; ++b)
      if (q + b * step < all) row.load(v[b], q + b * step);
#pragma unroll
    for (int b = 0; b < LP_BATCH; ++b) {
      if (q + b * step >= all) break;
      const int e = row.first(q + b * step);
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        uint32_t d0, d1;
        f2_to(f2_add(f2_fma(v[b].pair(i), scale2, neg_m2), neg_l2), d0, d1);
        const u64 d = f2_of(__float_as_uint(lp_max_nan(__uint_as_float(d0), LP_FAR)), __float_as_uint(lp_max_nan(__uint_as_float(d1), LP_FAR)));
        const u64 w = f2_mul(exp2_mufu2(f2_mul(d, log2e2)), f2_fma(h2, d, c2));
        u64 out = f2_mul(w, neg2);
        if (e + 2 * i == target || e + 2 * i + 1 == target) out = f2_add(out, e + 2 * i == target ? f2_of(__float_as_uint(none ? 0.f : g), 0) : f2_of(0, __float_as_uint(none ? 0.f : g)));
        v[b].set(i, out);
      }
      if (row.whole(e) && !apart) {
        *reinterpret_cast<uint4*>(dx + e) = make_uint4(v[b].w[0], v[b].w[1], v[b].w[2], v[b].w[3]);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (e + i >= 0 && e + i < p.vocab) v[b].get(i, dx + e + i);
      }
    }
  }
}

template <typename T, int THREADS>
static int logprob_launch(const LogprobParams& p, int parts, cudaStream_t st) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)((long long)p.rows * parts));
  cfg.blockDim = dim3(THREADS);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = parts;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_on((long long)p.rows * parts <= PDL_SHORT_BLOCKS) ? 2 : 1;
  const cudaError_t rc = p.top > 0 ? cudaLaunchKernelEx(&cfg, logprob_kernel<T, THREADS, true>, p) : cudaLaunchKernelEx(&cfg, logprob_kernel<T, THREADS, false>, p);
  return rc == cudaSuccess ? OA_OK : OA_ERR_LAUNCH;
}

template <typename T>
static int logprob_run(const LogprobParams& p, cudaStream_t st) {
  // As many CTAs to a row as leave no SM without one, each with 2048 elements at least; threads by what is left for them
  int parts = 1;
  while (parts < 8 && (long long)p.rows * parts * 2 <= 2 * sm_count() && p.vocab / (2 * parts) >= 2048) parts *= 2;
  const int share = p.vocab / parts;
  if ((long long)p.rows * parts > 0x7fffffffll) return OA_ERR_TOO_LARGE;
  if (share <= 1024) return logprob_launch<T, 32>(p, parts, st);
  if (share <= 8192) return logprob_launch<T, 128>(p, parts, st);
  return logprob_launch<T, 512>(p, parts, st);
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
  const LogprobBwdParams p{logits, stride, targets, entropy, stats, dlogprobs, dentropy, dlogits, d_stride, rows, vocab, ignore_index, scale};
  // four pieces to a thread
  const int n = dtype == OA_F32 ? 4 : 8, per = 256 * LP_BATCH * n, parts = (int)(((long long)vocab + per) / per);
  const dim3 grid((unsigned)rows, (unsigned)(parts < 65535 ? parts : 65535));
  if (dtype == OA_F32) launch_short(logprob_bwd_kernel<float>, grid, dim3(256), 0, (cudaStream_t)stream, p);
  else launch_short(logprob_bwd_kernel<__nv_bfloat16>, grid, dim3(256), 0, (cudaStream_t)stream, p);
  return cudaGetLastError() == cudaSuccess ? OA_OK : OA_ERR_LAUNCH;
}
