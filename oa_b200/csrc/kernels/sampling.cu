// Sampling of the next token of each row of logits from a given random number, with temperature, top-k, top-p and min-p.
//
// For a row x with maximum m:  y = (x - m) * (1 / temperature) in fp32, w = exp(y) in (0, 1], and the mass of a token is the whole number
// floor(w * 2^40).  Masses are added as whole numbers, so that a row's sums, and with them the token, do not depend on the order in which
// they are added.  Tokens are ranked by x, of equal ones the lower index first.  Kept are
//   the first top_k of them, of these the first whose mass before them is less than top_p times the mass of all of these, and of these the
//   ones with w >= min_p (the first one always).
// With S the mass of what is kept, the token is the first in the vocabulary's order whose running mass exceeds floor(u * S), and its
// log-probability y - log(S / 2^40).  A temperature of 0 or less takes the first of the ranking, with log-probability 0.  NaN counts as
// -inf; a row without anything above -inf gives token -1 and log-probability -inf.
#include "common.cuh"
#include "api.h"

namespace oa {

typedef unsigned long long u64;

struct SampleParams {
  const void* logits;
  long long stride;
  const float *u, *temperature, *top_p, *min_p;
  const int* top_k;
  int* tokens;
  float* logprobs;
  int rows, vocab;
};

// Logits in an order that whole numbers have: larger logits have larger keys, the two zeros the same, NaN the key of -inf.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return x != x ? 0x007fffffu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
constexpr uint32_t KEY_NONE = 0x007fffffu;   // of -inf

__device__ __forceinline__ float load_logit(const float* p) { return *p; }
__device__ __forceinline__ float load_logit(const __nv_bfloat16* p) { return __bfloat162float(*p); }

struct Weigh {
  float max, inv_t;
  __device__ __forceinline__ float scaled(float x) const { return x == max ? 0.f : (x - max) * inv_t; }
  __device__ __forceinline__ float weight(float x) const { return x != x || x == -INFINITY ? 0.f : expf(scaled(x)); }
};
// floor(w * 2^40) for w in [0, 1] as two numbers of 20 bits: sums of up to 4096 of either fit 32 bits.  Adding 2^23 rounded down leaves a
// whole number in the low bits of a float.
struct Mass20 { uint32_t hi, lo; };
__device__ __forceinline__ Mass20 mass20_of(float w) {
  const float a = w * 1048576.f, h = __fadd_rd(a, 8388608.f), f = a - (h - 8388608.f);
  return {__float_as_uint(h) - 0x4b000000u, __float_as_uint(__fmaf_rd(f, 1048576.f, 8388608.f)) - 0x4b000000u};
}
__device__ __forceinline__ u64 mass_of(float w) { const Mass20 m = mass20_of(w); return ((u64)m.hi << 20) + m.lo; }

template <typename V, typename F>
__device__ __forceinline__ V block_all(V v, V* red, F op) {   // op over a block of SAMPLE_THREADS, the result to all
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
  for (int w = 1; w < (int)blockDim.x / 32; ++w) v = op(v, red[w]);
  return v;
}

constexpr int SAMPLE_THREADS = 512;

template <typename T>
__global__ void __launch_bounds__(SAMPLE_THREADS) sample_kernel(const SampleParams p) {
  __shared__ u64 s_red[SAMPLE_THREADS / 32];
  __shared__ u64 s_scan[SAMPLE_THREADS / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int row = blockIdx.x, tid = threadIdx.x, V = p.vocab;
  const T* x = static_cast<const T*>(p.logits) + row * p.stride;
  const auto sum = [](u64 a, u64 b) { return a + b; };
  const auto top = [](u64 a, u64 b) { return a > b ? a : b; };
  // the first of the ranking: largest key, lowest index
  u64 best = 0;
  for (int i = tid; i < V; i += SAMPLE_THREADS) best = top(best, ((u64)key_of(load_logit(x + i)) << 32) | (uint32_t)~i);
  best = block_all(best, s_red, top);
  const uint32_t top_key = (uint32_t)(best >> 32);
  const float t = p.temperature ? p.temperature[row] : 1.f;
  if (V == 0 || top_key <= KEY_NONE || !(t > 0.f)) {
    if (tid == 0) {
      const bool none = V == 0 || top_key <= KEY_NONE;
      p.tokens[row] = none ? -1 : (int)~(uint32_t)best;
      p.logprobs[row] = none ? -INFINITY : 0.f;
    }
    return;
  }
  const float peak = __uint_as_float((top_key & 0x80000000u) ? top_key & 0x7fffffffu : ~top_key);
  const Weigh wt{peak, peak == INFINITY ? 1.f : 1.f / t};
  // what is kept so far: keys above `key`, and of those equal to it the indices up to `idx`
  uint32_t key = KEY_NONE + 1;
  int idx = V - 1;
  const auto in = [&](uint32_t k, int i) { return k > key || (k == key && i <= idx); };
  // measure(f): the sum of f(key, index, weight) over what is kept
  const auto measure = [&](auto f) {
    u64 s = 0;
    for (int i = tid; i < V; i += SAMPLE_THREADS) {
      const float xi = load_logit(x + i);
      const uint32_t k = key_of(xi);
      if (in(k, i)) s += f(k, i, xi);
    }
    return block_all(s, s_red, sum);
  };
  // Cuts what is kept to the shortest head of the ranking for which enough(measure of it) holds, given that it holds for all of it: the
  // largest key for which it holds, and of the tokens with that key the lowest index.
  const auto cut = [&](auto f, auto enough) {
    uint32_t lo = key;                      // holds
    for (int bit = 31; bit >= 0; --bit) {
      // candidates lo + 2^bit, as far as they are keys that occur
      const uint32_t c = lo + (1u << bit);
      if (c < lo || c > top_key) continue;
      if (enough(measure([&](uint32_t k, int i, float xi) { return k >= c ? f(xi) : 0ull; }))) lo = c;
    }
    int hi = lo == key ? idx : V - 1, low = 0;
    while (low < hi) {
      const int mid = (low + hi) >> 1;
      if (enough(measure([&](uint32_t k, int i, float xi) { return k > lo || (k == lo && i <= mid) ? f(xi) : 0ull; }))) hi = mid;
      else low = mid + 1;
    }
    key = lo;
    idx = hi;
  };
  const int k = p.top_k ? p.top_k[row] : 0;
  if (k > 0 && measure([](uint32_t, int, float) { return 1ull; }) > (u64)k)
    cut([](float) { return 1ull; }, [&](u64 n) { return n >= (u64)k; });
  const auto mass = [&](float xi) { return mass_of(wt.weight(xi)); };
  const float top_p = p.top_p ? p.top_p[row] : 1.f;
  if (!(top_p >= 1.f)) {
    const double part = (double)top_p * (double)measure([&](uint32_t, int, float xi) { return mass(xi); });
    cut(mass, [&](u64 n) { return n > 0 && !((double)n < part); });
  }
  const float least = p.min_p ? fminf(p.min_p[row], 1.f) : 0.f;
  const auto kept = [&](uint32_t kk, int i, float xi) -> u64 {
    if (!in(kk, i)) return 0;
    const float w = wt.weight(xi);
    return w >= least ? mass_of(w) : 0;
  };
  const u64 S = measure([&](uint32_t kk, int i, float xi) { return kept(kk, i, xi); });
  const double at = floor((double)p.u[row] * (double)S);
  const u64 r = !(at > 0.0) ? 0 : at >= (double)S ? S - 1 : min((u64)at, S - 1);
  // the running mass in the vocabulary's order, a warp's lanes over neighbours
  const int warp = tid >> 5, lane = tid & 31, span = ((V + SAMPLE_THREADS - 1) / SAMPLE_THREADS) * 32;
  const int lo = min(warp * span, V), hi = min(lo + span, V);
  u64 mine = 0;
  for (int i = lo + lane; i < hi; i += 32) { const float xi = load_logit(x + i); mine += kept(key_of(xi), i, xi); }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  if (lane == 0) s_scan[warp] = mine;
  __syncthreads();
  u64 run = 0;
  for (int w = 0; w < warp; ++w) run += s_scan[w];
  if (r >= run && r < run + s_scan[warp]) {
    for (int i0 = lo; i0 < hi; i0 += 32) {
      const int i = i0 + lane;
      u64 m = 0;
      float xi = 0.f;
      if (i < hi) { xi = load_logit(x + i); m = kept(key_of(xi), i, xi); }
      u64 inc = m;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) { const u64 a = __shfl_up_sync(0xffffffffu, inc, o); if (lane >= o) inc += a; }
      const unsigned past = __ballot_sync(0xffffffffu, run + inc > r);
      if (past) {
        if (lane == __ffs(past) - 1) {
          p.tokens[row] = i;
          p.logprobs[row] = wt.scaled(xi) - (float)log((double)S / 1099511627776.0);
        }
        break;
      }
      run += __shfl_sync(0xffffffffu, inc, 31);
    }
  }
}

// ------------------------------------------------------------------------------------------------ a cluster of CTAs for a row
// A row is read once, by up to eight CTAs of a cluster that keep it in shared memory; every later pass is over those copies.  A warp owns
// neighbouring tokens, fetched by a bulk copy of its own, and a lane 16 bytes of them at a time.
//   1  maximum of each thread, warp, CTA, cluster.  A greedy row ends here.
//   2  top-k up to 512: the k-th largest of the threads' maxima is no larger than the k-th largest logit, so that what lies in its bin of
//      (max - x) or above holds the top k, and little more; those tokens meet in the leading CTA, which sorts them.
//   3  top-p (and larger top-k): masses in 1024 bins of y; the bin in which the wanted mass is reached goes to the leading CTA, which sorts it.
//      A token of weight below (1 - p) / (2 V) is never kept: all such ones together have less than the mass to be cut off, as the
//      maximum's weight is 1.  Those take no part.
//      Bins too full for the list (equal logits, above all) are left to a search over keys and indices, 50 passes in shared memory.
//   4  mass of what is kept for each warp, prefix sums over warps and CTAs, and the warp in whose stretch u falls looks again.
constexpr int ROW_BINS = 1024, ROW_LIST = 1024, ROW_BRIEF_K = 512;

template <typename T> struct Lane16;
template <> struct Lane16<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void get(const uint8_t* p, float* f) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
  }
};
template <> struct Lane16<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void get(const uint8_t* p, float* f) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(w[i] << 16); f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
  }
};

__device__ __forceinline__ uint32_t cluster_add(uint32_t addr, uint32_t v) {
  uint32_t r;
  asm volatile("atom.relaxed.cluster.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(r) : "r"(addr), "r"(v) : "memory");
  return r;
}
__device__ __forceinline__ void cluster_st(uint32_t addr, u64 v) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory"); }
__device__ __forceinline__ u64 cluster_ld(uint32_t addr) {
  u64 v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
  return v;
}

struct RowShared {
  u64 exchange[2][8];                      // a number of each CTA of the cluster, in two sets used in turn
  u64 red[SAMPLE_THREADS / 32];
  u64 cut;                                 // from the leader: key and index, or a bin and what lies before it
  u64 base;
  uint64_t bars[SAMPLE_THREADS / 32];
  uint32_t listed;
};

template <typename T>
__global__ void __launch_bounds__(SAMPLE_THREADS, 2) sample_row_kernel(const SampleParams p, int span, int* status) {
  constexpr int N16 = Lane16<T>::N, WARPS = SAMPLE_THREADS / 32;
  extern __shared__ __align__(16) uint8_t row_smem[];
  __shared__ RowShared sh;
  u64* bins = reinterpret_cast<u64*>(row_smem);                  // [ROW_BINS], and later, in the leader, the list [ROW_LIST]
  uint8_t* data = row_smem + ROW_BINS * sizeof(u64);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint32_t ctas;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
  const uint32_t rank = cluster_ctarank();
  const int row = blockIdx.x / ctas, V = p.vocab;
  pdl_launch_dependents();
  if (lane == 0) { mbar_init(&sh.bars[warp], 1); mbar_fence_init(); }
  __syncwarp();
  pdl_wait();

  // ---- the row's share of this CTA, [lo, hi), lies in shared memory as it does to 16 bytes in the row
  const T* x = static_cast<const T*>(p.logits) + row * p.stride;
  const int share = (V + (int)ctas - 1) / (int)ctas, lo = min((int)rank * share, V), hi = min(lo + share, V);
  const int skew = (int)((reinterpret_cast<uintptr_t>(x + lo) & 15) / sizeof(T));
  const int first = lo - skew;                                   // token at place 0
  const int s0 = warp * span, s1 = s0 + span;                    // this warp's places
  const int a = min(max(s0, skew), s1), b = max(min(s1, hi - first), a);          // of them [a, b) hold tokens
  const int a16 = min((a + N16 - 1) / N16 * N16, b), b16 = max(b / N16 * N16, a16);
  T* places = reinterpret_cast<T*>(data);
  if (b16 > a16 && lane == 0) {
    mbar_expect_tx(&sh.bars[warp], (uint32_t)(b16 - a16) * sizeof(T));
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(places + a16)), "l"(x + first + a16),
                 "r"((uint32_t)(b16 - a16) * (uint32_t)sizeof(T)), "r"(smem_u32(&sh.bars[warp])) : "memory");
  }
  const auto by_hand = [&](int i) { if (i >= a && i < b) places[i] = x[first + i]; else places[i] = T(-INFINITY); };
  for (int i = s0 + lane; i < a16; i += 32) by_hand(i);          // ends off 16 bytes, and places without a token
  for (int i = b16 + lane; i < s1; i += 32) by_hand(i);
  if (ctas > 1) cluster_sync_all();                              // every CTA of the cluster is there before anything is written to it
  __syncwarp();
  bool fine = true;
  if (b16 > a16) fine = warp_wait(&sh.bars[warp], 0);
  if (!fine && lane == 0) report_error(status, OA_KERR_WAIT_FULL);
  // every pass: f(token, logit) for the tokens of this lane, 16 bytes at a time
  const auto each = [&](auto f) {
    for (int c = s0 + lane * N16; c < s1; c += 32 * N16) {
      float v[N16];
      Lane16<T>::get(data + c * sizeof(T), v);
#pragma unroll
      for (int k = 0; k < N16; ++k) f(first + c + k, v[k]);
    }
  };
  const auto sum = [](u64 u, u64 v) { return u + v; };
  const auto top = [](u64 u, u64 v) { return u > v ? u : v; };
  int turn = 0;
  // op over the whole cluster, the result to all
  const auto cluster_all = [&](u64 v, auto op) {
    v = block_all(v, sh.red, op);
    if (ctas == 1) return v;
    turn ^= 1;
    if (tid < (int)ctas) cluster_st(map_to_cta(smem_u32(&sh.exchange[turn][rank]), tid), v);
    cluster_sync_all();
    v = sh.exchange[turn][0];
    for (uint32_t r = 1; r < ctas; ++r) v = op(v, sh.exchange[turn][r]);
    return v;
  };
  const auto meet = [&] { if (ctas > 1) cluster_sync_all(); else __syncthreads(); };

  // ---- 1
  float high = -INFINITY;                                        // of this thread; NaN is passed over
  each([&](int, float v) { high = fmaxf(high, v); });
  const uint32_t top_key = (uint32_t)cluster_all(key_of(high), top);
  const float t = p.temperature ? p.temperature[row] : 1.f;
  const bool none = top_key <= KEY_NONE;
  if (none || !(t > 0.f)) {
    u64 best = 0;
    if (!none) {
      each([&](int i, float v) { if (key_of(v) == top_key) best = top(best, (uint32_t)~i); });
      best = cluster_all(best, top);
    }
    if (rank == 0 && tid == 0) {
      p.tokens[row] = none ? -1 : (int)~(uint32_t)best;
      p.logprobs[row] = none ? -INFINITY : 0.f;
    }
    return;
  }
  const float peak = __uint_as_float((top_key & 0x80000000u) ? top_key & 0x7fffffffu : ~top_key);
  const Weigh wt{peak, peak == INFINITY ? 1.f : 1.f / t};
  uint32_t key = KEY_NONE + 1;                                   // kept: keys above, and of those equal the indices up to idx
  int idx = V - 1;
  const auto in = [&](uint32_t k, int i) { return k > key || (k == key && i <= idx); };
  const uint32_t list_at = map_to_cta(smem_u32(bins), 0), listed_at = map_to_cta(smem_u32(&sh.listed), 0);
  // Tokens for which pred holds go to the leader's list, in any order; returns how many there were (more than ROW_LIST: not all are there).
  const auto collect = [&](auto pred) {
    if (rank == 0 && tid == 0) sh.listed = 0;
    meet();
    each([&](int i, float v) {
      const uint32_t k = key_of(v);
      const bool yes = k > KEY_NONE && in(k, i) && pred(v);
      const unsigned who = __ballot_sync(0xffffffffu, yes);
      if (who) {
        uint32_t at = 0;
        if (lane == 0) at = cluster_add(listed_at, __popc(who));
        at = __shfl_sync(0xffffffffu, at, 0) + __popc(who & ((1u << lane) - 1));
        if (yes && at < ROW_LIST) cluster_st(list_at + at * 8, ((u64)k << 32) | (uint32_t)~i);
      }
    });
    meet();
    return rank == 0 ? (int)sh.listed : 0;
  };
  // The leader's list into the ranking's order.
  const auto sort_list = [&](int n) {
    int size = 64;
    while (size < n) size <<= 1;
    for (int i = n + tid; i < size; i += SAMPLE_THREADS) bins[i] = 0;
    __syncthreads();
    for (int k = 2; k <= size; k <<= 1) {
      for (int j = k >> 1; j > 0; j >>= 1) {
        if (tid < size / 2) {
          const int i = 2 * j * (tid / j) + tid % j;
          const u64 u = bins[i], v = bins[i + j];
          if ((u < v) == ((i & k) == 0)) { bins[i] = v; bins[i + j] = u; }
        }
        if (j > 32) __syncthreads(); else __syncwarp();          // up to a distance of 32 a warp's pairs lie in 64 entries of its own
      }
      __syncthreads();
    }
  };
  // Of the sorted list's first n: the mass before entry `tid` and before entry `tid + SAMPLE_THREADS`.
  const auto list_masses = [&](int n, u64* before, u64& total) {
    u64 m[2], run = 0;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int i = tid + r * SAMPLE_THREADS;
      const uint32_t k = i < n ? (uint32_t)(bins[i] >> 32) : 0;
      m[r] = i < n ? mass_of(wt.weight(__uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k))) : 0;
      u64 inc = m[r];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) { const u64 u = __shfl_up_sync(0xffffffffu, inc, o); if (lane >= o) inc += u; }
      __syncthreads();
      if (lane == 31) sh.red[warp] = inc;
      __syncthreads();
      u64 all = 0, prior = 0;
      for (int w = 0; w < WARPS; ++w) { if (w < warp) prior += sh.red[w]; all += sh.red[w]; }
      before[r] = run + prior + inc - m[r];
      run += all;
    }
    total = run;
  };
  // The leader tells where the list's first n end.
  const auto cut_after = [&](int n) {
    if (rank == 0) {
      __syncthreads();
      if (tid < (int)ctas) cluster_st(map_to_cta(smem_u32(&sh.cut), tid), bins[n - 1]);
    }
    meet();
    key = (uint32_t)(sh.cut >> 32);
    idx = (int)~(uint32_t)sh.cut;
  };
  // Slow and sure: the largest key, and of the tokens with it the lowest index, for which enough(f over what is up to there) holds.
  const auto search = [&](auto f, auto enough) {
    const auto measure = [&](auto part) {
      u64 s = 0;
      each([&](int i, float v) { const uint32_t k = key_of(v); if (k > KEY_NONE && in(k, i) && part(k, i)) s += f(v); });
      return cluster_all(s, sum);
    };
    uint32_t low = key;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t c = low + (1u << bit);
      if (c < low || c > top_key) continue;
      if (enough(measure([&](uint32_t k, int) { return k >= c; }))) low = c;
    }
    int up = low == key ? idx : V - 1, down = 0;
    while (down < up) {
      const int mid = (down + up) >> 1;
      if (enough(measure([&](uint32_t k, int i) { return k > low || (k == low && i <= mid); }))) up = mid;
      else down = mid + 1;
    }
    key = low;
    idx = up;
  };
  // From the leader to all: the list's length was too large
  const auto agreed = [&](int n) { return (int)cluster_all(rank == 0 && tid == 0 ? (u64)n : 0, sum); };
  // First bin in which a running sum over the cluster's bins meets enough(); ROW_BINS if there is none.  `base`: the sum before it.
  const auto find_bin = [&](auto enough, u64& base) {
    meet();                                                      // all bins are filled
    if (rank == 0) {
      u64 v[2], run = 0;
      if (tid == 0) { sh.cut = ROW_BINS; sh.base = 0; }
      __syncthreads();
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const uint32_t at = smem_u32(bins + tid + r * SAMPLE_THREADS);
        v[r] = 0;
        for (uint32_t c = 0; c < ctas; ++c) v[r] += cluster_ld(map_to_cta(at, c));
        u64 inc = v[r];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const u64 u = __shfl_up_sync(0xffffffffu, inc, o); if (lane >= o) inc += u; }
        __syncthreads();
        if (lane == 31) sh.red[warp] = inc;
        __syncthreads();
        u64 all = 0, prior = 0;
        for (int w = 0; w < WARPS; ++w) { if (w < warp) prior += sh.red[w]; all += sh.red[w]; }
        const u64 upto = run + prior + inc;
        if (enough(upto) && !enough(upto - v[r])) { sh.cut = tid + r * SAMPLE_THREADS; sh.base = upto - v[r]; }
        run += all;
      }
      __syncthreads();
      const u64 bin = sh.cut, before = sh.base;
      if (tid > 0 && tid < (int)ctas) { cluster_st(map_to_cta(smem_u32(&sh.cut), tid), bin); cluster_st(map_to_cta(smem_u32(&sh.base), tid), before); }
    }
    meet();
    base = sh.base;
    return (int)sh.cut;
  };
  const auto clear_bins = [&] {
    for (int i = tid; i < ROW_BINS; i += SAMPLE_THREADS) bins[i] = 0;
    __syncthreads();
  };

  // ---- 2
  const int want = p.top_k ? p.top_k[row] : 0;
  const float top_p = p.top_p ? p.top_p[row] : 1.f;
  const double dp = (double)top_p;
  bool cut_p = !(top_p >= 1.f);
  if (want > 0 && want < V) {
    const auto by_gap = [&](float v) { return v == peak ? 0 : (int)fminf((peak - v) * 32.f, (float)(ROW_BINS - 1)); };
    const auto enough = [&](u64 n) { return n >= (u64)want; };
    int n = ROW_LIST + 1;
    if (want <= ROW_BRIEF_K) {
      clear_bins();
      if (key_of(high) > KEY_NONE) atomicAdd(&bins[by_gap(high)], 1ull);
      u64 base;
      const int bin = min(find_bin(enough, base), ROW_BINS - 1);
      n = agreed(collect([&](float v) { return by_gap(v) <= bin; }));
    }
    if (n <= ROW_LIST) {
      int keep = min(want, n);                                   // fewer than wanted: the others are -inf
      if (rank == 0) {
        sort_list(n);
        if (cut_p) {
          u64 before[2], total;
          list_masses(keep, before, total);
          const double part = dp * (double)total;
          const u64 inside = (tid < keep && (double)before[0] < part) + (tid + SAMPLE_THREADS < keep && (double)before[1] < part);
          const int fewer = (int)block_all(inside, sh.red, sum);
          keep = fewer > 1 ? fewer : 1;
        }
      }
      cut_after(keep);
      cut_p = false;
    } else {
      u64 have = 0;
      each([&](int i, float v) { have += key_of(v) > KEY_NONE; });
      if (cluster_all(have, sum) > (u64)want) {
        clear_bins();
        each([&](int i, float v) { if (key_of(v) > KEY_NONE) atomicAdd(&bins[by_gap(v)], 1ull); });
        u64 base;
        const int bin = find_bin(enough, base);
        n = agreed(collect([&](float v) { return by_gap(v) == bin; }));
        if (n <= ROW_LIST) {
          if (rank == 0) sort_list(n);
          cut_after(want - (int)base);
        } else {
          search([](float) { return 1ull; }, enough);
        }
      }
    }
  }
  // ---- 3
  if (cut_p) {
    const float floor_w = fminf(fmaxf((float)(0.5 * (1.0 - dp) / V), 5e-13f), 0.5f), deep = logf(floor_w), scale = (float)ROW_BINS / -deep;
    const auto by_y = [&](float y) { return (int)fminf(-y * scale, (float)(ROW_BINS - 1)); };
    clear_bins();
    u64 mine = 0;
    each([&](int i, float v) {
      const uint32_t k = key_of(v);
      if (!(k > KEY_NONE && in(k, i))) return;
      const float y = wt.scaled(v);
      const u64 m = mass_of(expf(y));
      mine += m;
      if (y > deep) atomicAdd(&bins[by_y(y)], m);
    });
    const double part = dp * (double)cluster_all(mine, sum);
    const auto enough = [&](u64 m) { return m > 0 && !((double)m < part); };
    u64 base;
    const int bin = find_bin(enough, base);
    const int n = agreed(collect([&](float v) { const float y = wt.scaled(v); return y > deep && by_y(y) == bin; }));
    if (n > 0 && n <= ROW_LIST) {
      int keep = 1;
      if (rank == 0) {
        sort_list(n);
        u64 before[2], total;
        list_masses(n, before, total);
        const u64 inside = (tid < n && (double)(base + before[0]) < part) + (tid + SAMPLE_THREADS < n && (double)(base + before[1]) < part);
        keep = max((int)block_all(inside, sh.red, sum), 1);
      }
      cut_after(keep);
    } else {
      search([&](float v) { return mass_of(wt.weight(v)); }, enough);
    }
  }
  // ---- 4
  const float least = p.min_p ? fminf(p.min_p[row], 1.f) : 0.f;
  const auto kept = [&](int i, float v) -> u64 {
    const uint32_t k = key_of(v);
    if (!(k > KEY_NONE && in(k, i))) return 0;
    const float w = expf(wt.scaled(v));
    return w >= least ? mass_of(w) : 0;
  };
  uint32_t hi20 = 0, lo20 = 0;                                   // a lane has fewer than 4096 tokens
  each([&](int i, float v) {
    const uint32_t k = key_of(v);
    if (!(k > KEY_NONE && in(k, i))) return;
    const float w = expf(wt.scaled(v));
    if (!(w >= least)) return;
    const Mass20 m = mass20_of(w);
    hi20 += m.hi;
    lo20 += m.lo;
  });
  u64 mine = ((u64)hi20 << 20) + lo20;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  __syncthreads();
  if (lane == 0) sh.red[warp] = mine;
  __syncthreads();
  u64 before = 0, all = 0;
  for (int w = 0; w < WARPS; ++w) { if (w < warp) before += sh.red[w]; all += sh.red[w]; }
  u64 S = all;
  if (ctas > 1) {
    turn ^= 1;
    if (tid < (int)ctas) cluster_st(map_to_cta(smem_u32(&sh.exchange[turn][rank]), tid), all);
    cluster_sync_all();
    S = 0;
    for (uint32_t r = 0; r < ctas; ++r) { if (r < rank) before += sh.exchange[turn][r]; S += sh.exchange[turn][r]; }
  }
  const double at = floor((double)p.u[row] * (double)S);
  const u64 r = !(at > 0.0) ? 0 : at >= (double)S ? S - 1 : min((u64)at, S - 1);
  if (r < before || r >= before + mine) return;                  // not in this warp's stretch
  // a lane takes neighbours, then the lane's stretch is looked at token by token
  const int piece = (span + 31) / 32, p0 = min(s0 + lane * piece, s1), p1 = min(p0 + piece, s1);
  u64 part = 0;
  for (int i = p0; i < p1; ++i) part += kept(first + i, load_logit(places + i));
  u64 inc = part;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) { const u64 v = __shfl_up_sync(0xffffffffu, inc, o); if (lane >= o) inc += v; }
  const int who = __ffs(__ballot_sync(0xffffffffu, before + inc > r)) - 1;
  u64 run = before + __shfl_sync(0xffffffffu, inc - part, who);
  const int q0 = __shfl_sync(0xffffffffu, p0, who), q1 = __shfl_sync(0xffffffffu, p1, who);
  for (int c = q0; c < q1; c += 32) {
    const int i = c + lane;
    const float v = i < q1 ? load_logit(places + i) : -INFINITY;
    inc = i < q1 ? kept(first + i, v) : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const u64 u = __shfl_up_sync(0xffffffffu, inc, o); if (lane >= o) inc += u; }
    const unsigned past = __ballot_sync(0xffffffffu, run + inc > r);
    if (past) {
      if (lane == __ffs(past) - 1) {
        p.tokens[row] = first + i;
        p.logprobs[row] = wt.scaled(v) - (float)log((double)S / 1099511627776.0);
      }
      return;
    }
    run += __shfl_sync(0xffffffffu, inc, 31);
  }
}

}  // namespace oa

using namespace oa;

template <typename T>
static int launch_sample(const SampleParams& p, int* status, cudaStream_t st) {
  // As many CTAs to a row as keep its share within 104 KB (two CTAs on an SM); more, up to eight, while rows leave SMs idle and a share
  // has 4096 tokens or more.
  constexpr int UNIT = 32 * Lane16<T>::N, WARPS = SAMPLE_THREADS / 32, MOST = 216 * 1024;
  int ctas = 1;
  while (ctas < 8 && ((size_t)(p.vocab / ctas) * sizeof(T) > 104 * 1024 || (p.rows * (long long)ctas < 148 && p.vocab / ctas >= 2 * 4096))) ctas *= 2;
  const int share = (p.vocab + ctas - 1) / ctas + Lane16<T>::N;  // places: tokens, and what the first lacks to 16 bytes
  const int span = (share + WARPS * UNIT - 1) / (WARPS * UNIT) * UNIT;
  const size_t smem = ROW_BINS * sizeof(u64) + (size_t)span * WARPS * sizeof(T);
  if (smem > MOST) {                                             // beyond what eight CTAs hold
    launch_short(sample_kernel<T>, dim3((unsigned)p.rows), dim3(SAMPLE_THREADS), 0, st, p);
    return cudaGetLastError() == cudaSuccess ? OA_OK : OA_ERR_LAUNCH;
  }
  static bool set = false;
  if (!set) {
    if (cudaFuncSetAttribute(sample_row_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, MOST) != cudaSuccess) return OA_ERR_LAUNCH;
    set = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)p.rows * ctas);
  cfg.blockDim = dim3(SAMPLE_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_on((long long)p.rows * ctas <= PDL_SHORT_BLOCKS) ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, sample_row_kernel<T>, p, span, status) == cudaSuccess ? OA_OK : OA_ERR_LAUNCH;
}

extern "C" int oa_sample(int dtype, const void* logits, long long stride, const float* u, const float* temperature, const int* top_k, const float* top_p,
                         const float* min_p, int* tokens, float* logprobs, int rows, int vocab, int* status, void* stream) {
  if (dtype != OA_F32 && dtype != OA_BF16) return OA_ERR_UNSUPPORTED;
  if (rows < 0 || vocab < 0) return OA_ERR_ARG;
  if (vocab > 1 << 23) return OA_ERR_TOO_LARGE;              // 2^40 times this many fits a sum of 64 bits
  if (rows == 0) return OA_OK;
  if (rows > 0x7fffffff / 8) return OA_ERR_TOO_LARGE;
  const SampleParams p{logits, stride, u, temperature, top_p, min_p, top_k, tokens, logprobs, rows, vocab};
  return dtype == OA_F32 ? launch_sample<float>(p, status, (cudaStream_t)stream) : launch_sample<__nv_bfloat16>(p, status, (cudaStream_t)stream);
}
