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
#include "per_device.h"
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
constexpr float LOWEST = -3.402823466e38f;   // the lowest logit that counts

__device__ __forceinline__ float load_logit(const float* p) { return *p; }
__device__ __forceinline__ float load_logit(const __nv_bfloat16* p) { return __bfloat162float(*p); }

struct Weigh {
  float max, inv_t;
  __device__ __forceinline__ float scaled(float x) const { return x == max ? 0.f : __fmul_rn(x - max, inv_t); }
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
// neighbouring tokens, fetched by a bulk copy of its own, a lane 16 bytes of them at a time; warps in the order of their CTAs own the
// vocabulary in order, so that a number from each warp (a maximum, a mass), sent to every CTA, says who has the first of something.
//   1  maximum of each thread, of all warps.  A greedy row ends here.
//   2  top-k up to 256: the k-th largest of the maxima of 512 groups of threads is no larger than the k-th largest logit, so that what is not
//      below it (cut to 16 bits) contains the top k, and little more: of n tokens spread over the groups about 512 ln(512 / (512 - k)).  Those
//      tokens go to the first CTA, which sorts them, makes all cuts and samples; the other CTAs are done.
//   3  top-p (and larger top-k): masses (counts) in 1024 bins of a place that rises as x falls; the bin in which the wanted sum is reached is cut into
//      1024 again while it holds more than a list does; its tokens go to the first CTA, which sorts them and says where the cut is.
//      (The last bin of a top-k's first pass, 32 and more below the maximum, has no end, and is not cut again.)
//      A token of weight below (1 - p) / (2 V) is never kept: all such ones together have less than the mass that is cut off, as the
//      maximum's weight is 1.  Those take no part.  What no bins separate, equal logits above all, is left to a search over keys and indices, 50 passes.
//   4  mass of what is kept for each warp, and the warp in whose stretch u falls looks again.
constexpr int ROW_LIST = 512, ROW_BINS = 1024, ROW_BRIEF_K = 256, ROW_WARPS = SAMPLE_THREADS / 32;
static_assert(ROW_LIST == SAMPLE_THREADS && ROW_BINS == 2 * SAMPLE_THREADS, "an entry of the list to a thread, and two bins");

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
template <int N> __device__ __forceinline__ float highest(const float* v) {
  float m = v[0];
#pragma unroll
  for (int k = 1; k < N; ++k) m = fmaxf(m, v[k]);
  return m;
}

__device__ __forceinline__ void cluster_st(uint32_t addr, u64 v) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory"); }
__device__ __forceinline__ void cluster_st32(uint32_t addr, uint32_t v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }
__device__ __forceinline__ void cluster_ld2(uint32_t addr, u64& a, u64& b) {
  asm volatile("ld.shared::cluster.v2.u64 {%0, %1}, [%2];" : "=l"(a), "=l"(b) : "r"(addr) : "memory");
}
__device__ __forceinline__ u64 warp_scan(u64 v, int lane) {      // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) { const u64 u = __shfl_up_sync(0xffffffffu, v, o); if (lane >= o) v += u; }
  return v;
}
__device__ __forceinline__ u64 warp_total(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float logit_of(uint32_t key) { return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key); }

struct RowShared {
  u64 slots[2][8 * ROW_WARPS];             // a number of each warp of the cluster, in two sets used in turn
  u64 red[ROW_WARPS];
  u64 cut, base;                           // where a cut is; a bin and the sum before it
  u64 far_cut;                             // the first CTA's word to the others
  uint64_t bars[ROW_WARPS];
  int listed, bin;
};

template <typename T>
__global__ void __launch_bounds__(SAMPLE_THREADS, 2) sample_row_kernel(const SampleParams p, int span, int lg, int* status) {
  constexpr int N16 = Lane16<T>::N;
  extern __shared__ __align__(16) uint8_t row_smem[];
  __shared__ RowShared sh;
  u64* bins = reinterpret_cast<u64*>(row_smem);                  // [ROW_BINS]; later, in the first CTA, the list of all
  u64* own_list = bins + ROW_BINS;                               // tokens of this CTA
  uint32_t* group_tops = reinterpret_cast<uint32_t*>(own_list);  // before that, maxima of groups of threads, in the vocabulary's order by warps
  uint8_t* data = row_smem + (ROW_BINS + ROW_LIST) * sizeof(u64);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t ctas = 1u << lg, rank = cluster_ctarank();
  const int row = blockIdx.x >> lg, V = p.vocab;
  pdl_launch_dependents();
  if (lane == 0) { mbar_init(&sh.bars[warp], 1); fence_proxy_async_smem(); }
  const auto clear_bins = [&] { reinterpret_cast<ulonglong2*>(bins)[tid] = make_ulonglong2(0, 0); };
  clear_bins();
  for (int i = tid; i < 2 * 8 * ROW_WARPS; i += SAMPLE_THREADS) sh.slots[0][i] = 0;
  if (tid == 0) sh.listed = 0;
  __syncwarp();
  pdl_wait();

  // ---- the row's share of this CTA, [lo, hi), lies in shared memory as it does to 16 bytes in the row
  const T* x = static_cast<const T*>(p.logits) + row * p.stride;
  const int share = (V + (int)ctas - 1) >> lg, lo = min((int)rank * share, V), hi = min(lo + share, V);
  const int skew = (int)((reinterpret_cast<uintptr_t>(x + lo) & 15) / sizeof(T));
  const int first = lo - skew;                                   // token at place 0
  const int s0 = warp * span, s1 = s0 + span;                    // this warp's places
  T* places = reinterpret_cast<T*>(data);
  {
    const int a = min(max(s0, skew), s1), b = max(min(s1, hi - first), a);        // of them [a, b) hold tokens
    const int a16 = min((a + N16 - 1) / N16 * N16, b), b16 = max(b / N16 * N16, a16);
    if (b16 > a16 && lane == 0) {
      mbar_expect_tx(&sh.bars[warp], (uint32_t)(b16 - a16) * sizeof(T));
      asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(places + a16)), "l"(x + first + a16),
                   "r"((uint32_t)(b16 - a16) * (uint32_t)sizeof(T)), "r"(smem_u32(&sh.bars[warp])) : "memory");
    }
    const auto by_hand = [&](int i) { if (i >= a && i < b) places[i] = x[first + i]; else places[i] = T(-INFINITY); };
    for (int i = s0 + lane; i < a16; i += 32) by_hand(i);        // ends off 16 bytes, and places without a token
    for (int i = b16 + lane; i < s1; i += 32) by_hand(i);
    __syncwarp();                                                // other lanes read them, 16 bytes at a time, and a warp without a copy waits for nothing else
    // every CTA of the cluster is there before anything is written to it
    if (ctas > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
    if (b16 > a16 && !warp_wait(&sh.bars[warp], 0) && lane == 0) report_error(status, OA_KERR_WAIT_FULL);
  }
  const auto meet = [&] { if (ctas > 1) cluster_sync_all(); else __syncthreads(); };
  // a pass: f(place, N16 logits) for 16 bytes of this lane at a time
  const auto each = [&](auto f) {
    for (int c = s0 + lane * N16; c < s1; c += 32 * N16) {
      float v[N16];
      Lane16<T>::get(data + c * sizeof(T), v);
      f(c, v);
    }
  };
  // a pass for which most of 16 bytes is nothing: f(token, logit) where the logit is not below `floor`.  Four pieces are fetched before the first
  // is looked at.
  const auto each_from = [&](float floor, auto f) {
    for (int c0 = s0 + lane * N16; c0 < s1; c0 += 4 * 32 * N16) {
      float top4[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int c = c0 + q * 32 * N16;
        float v[N16];
        Lane16<T>::get(data + min(c, s1 - N16) * sizeof(T), v);
        top4[q] = c < s1 ? highest<N16>(v) : -INFINITY;
      }
      if (!(highest<4>(top4) >= floor)) continue;
#pragma unroll 1
      for (int q = 0; q < 4; ++q) {
        const int c = c0 + q * 32 * N16;
        if (c >= s1) break;
        float v[N16];
        Lane16<T>::get(data + c * sizeof(T), v);
#pragma unroll
        for (int k = 0; k < N16; ++k)
          if (v[k] >= floor && v[k] > -INFINITY) f(first + c + k, v[k]);
      }
    }
  };
  int turn = 0;
  // Every warp's number to every CTA; then, to each warp, the sum of the numbers before its own and of all.
  const auto tell = [&](u64* slots, u64 mine) {
    if (lane < (int)ctas) cluster_st(map_to_cta(smem_u32(&slots[rank * ROW_WARPS + warp]), lane), mine);
  };
  const auto hear = [&](const u64* slots, u64& before, u64& all) {
    u64 v[4], sum = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) { v[k] = lane * 4 + k < (int)ctas * ROW_WARPS ? slots[lane * 4 + k] : 0; sum += v[k]; }
    u64 at = warp_scan(sum, lane);
    all = __shfl_sync(0xffffffffu, at, 31);
    at -= sum;
    const int me = rank * ROW_WARPS + warp;
#pragma unroll
    for (int k = 0; k < 3; ++k) if (k < (me & 3)) at += v[k];
    before = __shfl_sync(0xffffffffu, at, me >> 2);
  };
  const auto share_sums = [&](u64 mine, u64& before, u64& all) {
    turn ^= 1;
    tell(sh.slots[turn], mine);
    meet();
    hear(sh.slots[turn], before, all);
  };

  // ---- 1
  uint32_t top_key, tops;                                        // tops: of the maxima of 512 groups of threads, the one of group tid
  int first_warp;                                                // the first that has the maximum
  {
    float high = -INFINITY;                                      // NaN is passed over
#pragma unroll 4
    for (int c = s0 + lane * N16; c < s1; c += 32 * N16) {
      float v[N16];
      Lane16<T>::get(data + c * sizeof(T), v);
      high = fmaxf(high, highest<N16>(v));
    }
    uint32_t mine = key_of(high);                                // groups of as many lanes as there are CTAs, so that every lane tells one CTA
    for (int o = 1; o < (int)ctas; o <<= 1) mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, o));
    cluster_st32(map_to_cta(smem_u32(&group_tops[((rank * ROW_WARPS + warp) << (5 - lg)) + (lane >> lg)]), lane & (ctas - 1)), mine);
    meet();
    tops = group_tops[tid];
    uint32_t k[16], best = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) reinterpret_cast<uint4*>(k)[i] = reinterpret_cast<const uint4*>(group_tops)[lane * 4 + i];
#pragma unroll
    for (int i = 0; i < 16; ++i) best = max(best, k[i]);
    top_key = __reduce_max_sync(0xffffffffu, best);
    int at = SAMPLE_THREADS;
#pragma unroll
    for (int i = 15; i >= 0; --i) if (k[i] == top_key) at = lane * 16 + i;
    first_warp = (int)__reduce_min_sync(0xffffffffu, (unsigned)at) >> (5 - lg);
  }
  const float t = p.temperature ? p.temperature[row] : 1.f;
  float peak = logit_of(top_key);
  if (top_key <= KEY_NONE) {
    if (rank == 0 && tid == 0) { p.tokens[row] = -1; p.logprobs[row] = -INFINITY; }
    return;
  }
  if (!(t > 0.f)) {
    if (first_warp != (int)rank * ROW_WARPS + warp) return;
    unsigned at = 0xffffffffu;
    each([&](int c, const float* v) {
#pragma unroll
      for (int k = N16 - 1; k >= 0; --k) if (v[k] == peak) at = min(at, (unsigned)(first + c + k));
    });
    at = __reduce_min_sync(0xffffffffu, at);
    if (lane == 0) { p.tokens[row] = (int)at; p.logprobs[row] = 0.f; }
    return;
  }
  const float inv_t = fminf(1.f / t, -LOWEST);
  if (peak == INFINITY) {                                        // only those that are infinite count: 0 for them, nothing for the others
    for (int i = s0 + lane; i < s1; i += 32) places[i] = load_logit(places + i) == INFINITY ? T(0.f) : T(-INFINITY);
    __syncwarp();
    tops = logit_of(tops) == INFINITY ? key_of(0.f) : KEY_NONE;
    peak = 0.f;
    top_key = key_of(0.f);
  }
  // products that are never joined with an addition behind them: bins, and the rule itself, are of the rounded numbers
  const auto scaled = [&](float v) { return __fmul_rn(v - peak, inv_t); };
  const auto weight = [&](float v) { return expf(scaled(v)); };
  float from = -INFINITY;                                        // kept: logits above, and of those equal the indices up to idx
  int idx = V - 1;
  const auto in = [&](int i, float v) { return v > from || (v == from && i <= idx); };
  const auto cut_at = [&](u64 entry) { from = logit_of((uint32_t)(entry >> 32)); idx = (int)~(uint32_t)entry; };
  // the same for logits between two that lie close together
  const auto each_between = [&](float below, float above, auto f) {
    each([&](int c, const float* v) {
      bool any = false;
#pragma unroll
      for (int k = 0; k < N16; ++k) any |= v[k] >= below && v[k] <= above;
      if (!any) return;
#pragma unroll
      for (int k = 0; k < N16; ++k)
        if (v[k] >= below && v[k] <= above) f(first + c + k, v[k]);
    });
  };
  // Tokens of a pass for which pred holds go to the first CTA's list, in any order; returns how many there are.  With more than
  // ROW_LIST the list is of no use.
  const auto collect = [&](auto pass, auto pred) {
    pass([&](int i, float v) {
      if (!in(i, v) || !pred(v)) return;
      const int at = atomicAdd(&sh.listed, 1);
      if (at < ROW_LIST) own_list[at] = ((u64)key_of(v) << 32) | (uint32_t)~i;
    });
    __syncthreads();
    const int mine = sh.listed;
    u64 before, all;
    share_sums(warp == 0 ? (u64)mine : 0, before, all);          // a CTA's number stands with its first warp
    if (tid == 0) { sh.base = before; sh.listed = 0; }
    __syncthreads();
    if (all <= ROW_LIST && tid < mine) cluster_st(map_to_cta(smem_u32(bins + sh.base + tid), 0), own_list[tid]);
    meet();
    return (int)min(all, (u64)ROW_LIST + 1);
  };
  // The first n entries of bins into falling order, by counting those above each, with four, two or one thread to an entry (64 entries: 0.4 us, by
  // exchanges 2.0; 256: 1.3 and 4.7; 512 are alike).
  const auto sort_list = [&](int n) {
    const int lt = n <= ROW_LIST / 4 ? 2 : n <= ROW_LIST / 2 ? 1 : 0, at = tid >> lt, part = tid & ((1 << lt) - 1);
    if (tid == 0) bins[n] = 0;                                   // entries are read in pairs
    __syncthreads();
    u64 e = 0;
    int above = 0;
    if (at < n) {
      e = bins[at];
#pragma unroll 4
      for (int i = 2 * part; i < n; i += 2 << lt) {
        const ulonglong2 o = *reinterpret_cast<const ulonglong2*>(bins + i);
        above += (o.x > e) + (o.y > e);
      }
    }
    if (lt > 0) above += __shfl_xor_sync(0xffffffffu, above, 1);
    if (lt > 1) above += __shfl_xor_sync(0xffffffffu, above, 2);
    __syncthreads();
    if (part == 0 && at < n) bins[above] = e;
    __syncthreads();
  };
  // Sums over a block in thread order: what is before this thread, and all.
  const auto block_scan = [&](u64 v, u64& all) {
    const u64 inc = warp_scan(v, lane);
    __syncthreads();
    if (lane == 31) sh.red[warp] = inc;
    __syncthreads();
    const u64 r = lane < ROW_WARPS ? sh.red[lane] : 0, up = warp_scan(r, lane);
    all = __shfl_sync(0xffffffffu, up, ROW_WARPS - 1);
    return __shfl_sync(0xffffffffu, up - r, warp) + inc - v;
  };
  // The sums of all CTAs' bins, two to a thread; then the first bin in which the running sum is enough, and the sum before it.  Returns
  // false when no bin is.
  const auto find_bin = [&](u64 base, auto enough, int& bin, u64& before, u64& all) {
    if (tid == 0) sh.bin = -1;
    meet();                                                      // all bins are filled
    const uint32_t at = smem_u32(bins + 2 * tid);
    u64 v0 = 0, v1 = 0;
#pragma unroll
    for (int c = 0; c < 8; ++c) {                                // all under way together
      u64 a = 0, b = 0;
      if (c < (int)ctas) cluster_ld2(map_to_cta(at, c), a, b);
      v0 += ((a >> 32) << 20) + (uint32_t)a;
      v1 += ((b >> 32) << 20) + (uint32_t)b;
    }
    const u64 run = base + block_scan(v0 + v1, all);
    if (enough(run + v0 + v1) && !enough(run)) {
      const bool second = !enough(run + v0);
      sh.bin = 2 * tid + second;
      sh.base = run + (second ? v0 : 0);
    }
    __syncthreads();
    bin = sh.bin;
    before = sh.base;
    return bin >= 0;
  };
  // What a bin holds are two sums of 32 bits, in units of 1 and 2^20.  A bin of very many large weights overflows, which shows in the sum of all.
  const uint32_t bins_at = smem_u32(bins) - (0x4b000000u << 3);
  const auto add_to_bin = [&](float s, Mass20 m) {              // s in [0, ROW_BINS): the bin is its whole part
    const uint32_t at = bins_at + (__float_as_uint(__fadd_rd(s, 8388608.f)) << 3);
    asm volatile("red.shared.add.u32 [%0], %1;" ::"r"(at), "r"(m.lo) : "memory");
    if (m.hi) asm volatile("red.shared.add.u32 [%0], %1;" ::"r"(at + 4), "r"(m.hi) : "memory");
  };
  // Slow and sure: the largest key, and of the tokens with it the lowest index, for which enough(f over what is up to there) holds.
  const auto search = [&](auto f, auto enough) {
    const auto measure = [&](float floor, auto part) {
      u64 s = 0, before, all;
      each_from(floor, [&](int i, float v) { if (in(i, v) && part(i, v)) s += f(v); });
      share_sums(warp_total(s), before, all);
      return all;
    };
    uint32_t low = key_of(from) > KEY_NONE ? key_of(from) : KEY_NONE + 1;
    const uint32_t start = low;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t c = low + (1u << bit);
      if (c < low || c > top_key) continue;
      if (enough(measure(logit_of(c), [](int, float) { return true; }))) low = c;
    }
    const float at = logit_of(low);
    int up = low == start ? idx : V - 1, down = 0;
    while (down < up) {
      const int mid = (down + up) >> 1;
      if (enough(measure(at, [&](int i, float v) { return v > at || i <= mid; }))) up = mid;
      else down = mid + 1;
    }
    from = at;
    idx = up;
    meet();                                                      // the last sums have been read everywhere: either set of slots may be written
  };
  // A logit that is surely not above peak - gap, whatever was rounded on the way to the gap
  const auto below_gap = [&](float gap, bool unbounded) { return unbounded ? LOWEST : fmaxf(peak - gap * 1.00001f - (fabsf(peak) + gap) * 0x1p-20f, LOWEST); };
  // and one that is surely not below it
  const auto above_gap = [&](float gap) { return peak - gap * 0.99999f + (fabsf(peak) + gap) * 0x1p-20f; };
  // Cuts what is kept to the shortest head of the ranking whose sum of f is enough.  place(v) rises from 0 as v falls, by 1, a bin, for `step`;
  // tokens at ROW_BINS or more of it take no part in the first pass of bins, which the caller has made (their sum: `binned`), and are not reached.
  // `open`: the last bin of that pass holds all tokens from there on, whatever their place, so that it cannot be cut again.  A list in which
  // the sum is not reached makes no cut; the search does then.  (A list's sum against its bin's would say more, but cost 2 us of 42 where 256 rows of 201088
  // take their largest logit, which comes nowhere near it.)
  const auto cut_by_bins = [&](u64 binned, auto place, float step, bool open, auto f, auto enough) {
    u64 base = 0, all;
    float origin = 0.f, zoom = 1.f;                              // bins of this pass: (place - origin) * zoom
    for (int pass = 0; pass < 3; ++pass) {
      int bin;
      u64 before;
      const bool there = find_bin(base, enough, bin, before, all);
      if (!there || all != binned) break;                        // a bin has overflowed, or all was cut off
      base = before;
      const float o = origin, z = zoom;
      const auto mine = [&](float v) { const float s = (place(v) - o) * z; return s >= (float)bin && s < (float)(bin + 1); };
      const float below = below_gap((o + (float)(bin + 1) / z) * step, o == 0.f && bin == ROW_BINS - 1), above = above_gap((o + (float)bin / z) * step);
      const int n = collect([&](auto f) { each_between(below, above, f); }, mine);
      if (n > 0 && n <= ROW_LIST) {
        if (rank == 0) {
          if (tid == 0) sh.cut = 0;                              // no entry is 0
          sort_list(n);
          u64 m = tid < n ? (u64)f(logit_of((uint32_t)(bins[tid] >> 32))) : 0, total;
          const u64 run = base + block_scan(m, total);
          if (tid < n && !enough(run) && enough(run + m)) sh.cut = bins[tid];
          __syncthreads();
          if (tid < (int)ctas) cluster_st(map_to_cta(smem_u32(&sh.far_cut), tid), sh.cut);
        }
        meet();
        if (sh.far_cut == 0) break;
        cut_at(sh.far_cut);
        return;
      }
      if (pass == 2 || n == 0 || (open && pass == 0 && bin == ROW_BINS - 1)) break;
      // the bin again, in as many: the next bits of place
      origin = o + (float)bin / z;
      zoom = z * (float)ROW_BINS;
      clear_bins();
      __syncthreads();
      u64 sum = 0, prior;
      each_between(below, above, [&](int i, float v) {
        if (!in(i, v) || !mine(v)) return;
        const u64 m = f(v);
        sum += m;
        add_to_bin((place(v) - origin) * zoom, {(uint32_t)(m >> 20), (uint32_t)m & 0xfffffu});
      });
      share_sums(warp_total(sum), prior, binned);
    }
    search(f, enough);
  };
  const float least = p.min_p ? fminf(p.min_p[row], 1.f) : 0.f;
  const float u01 = p.u[row];
  const auto target = [&](u64 S) -> u64 {
    const double at = floor((double)u01 * (double)S);
    return !(at > 0.0) ? 0 : at >= (double)S ? S - 1 : min((u64)at, S - 1);
  };
  const auto answer = [&](int token, float v, u64 S) {
    p.tokens[row] = token;
    p.logprobs[row] = scaled(v) - (float)log((double)S / 1099511627776.0);
  };

  // ---- 2
  const int want = p.top_k ? p.top_k[row] : 0;
  const float top_p = p.top_p ? p.top_p[row] : 1.f;
  const double dp = (double)top_p;
  const bool cut_p = !(top_p >= 1.f);
  const auto place_of_gap = [&](float v) { return fminf(__fmul_rn(peak - v, 32.f), (float)ROW_BINS - 0.5f); };      // 32 of logits, all beyond in the last
  bool brief = V <= ROW_LIST && ((want > 0 && want < V) || cut_p);
  float floor = LOWEST;
  if (!brief && want > 0 && want <= ROW_BRIEF_K && want < V) {
    brief = true;
    uint32_t low = 0;                                            // the largest number of 16 bits that `want` of the maxima reach
    for (int bit = 31; bit >= 16; --bit)
      if (__syncthreads_count(tops >= (low | 1u << bit)) >= want) low |= 1u << bit;
    if (low > KEY_NONE) floor = logit_of(low);
  }
  if (brief) {
    __syncthreads();                                             // the maxima have been read: the list may go over them
    const int n = collect([&](auto f) { each_from(floor, f); }, [](float) { return true; });
    if (n <= ROW_LIST) {
      if (rank != 0) return;
      sort_list(n);
      int keep = want > 0 ? min(want, n) : n;
      const float w = tid < keep ? weight(logit_of((uint32_t)(bins[tid] >> 32))) : 0.f;
      const u64 m = mass_of(w);
      u64 S;
      const u64 run = block_scan(m, S);
      const double part = dp * (double)S;
      const bool stays = tid < keep && (tid == 0 || ((!cut_p || (double)run < part) && w >= least));      // both cuts leave a head of the ranking
      keep = __syncthreads_count(stays);
      const u64 entry = tid < keep ? bins[tid] : 0;
      __syncthreads();
      if (tid < keep) bins[tid] = (entry << 32) | (entry >> 32);                             // the lowest index first
      sort_list(keep);
      const u64 e = tid < keep ? bins[tid] : 0;
      const float v = logit_of((uint32_t)e);
      const u64 mine = tid < keep ? mass_of(weight(v)) : 0, at = block_scan(mine, S), r = target(S);
      if (r >= at && r < at + mine) answer((int)~(uint32_t)(e >> 32), v, S);
      return;
    }
  }
  if (want > 0 && want < V) {
    u64 have = 0, before, all;
    clear_bins();
    __syncthreads();
    each([&](int, const float* v) {
#pragma unroll
      for (int k = 0; k < N16; ++k)
        if (v[k] > -INFINITY) {
          ++have;
          add_to_bin(place_of_gap(v[k]), {0, 1});
        }
    });
    share_sums(warp_total(have), before, all);
    if (all > (u64)want) cut_by_bins(all, place_of_gap, 1.f / 32.f, true, [](float) { return 1ull; }, [&](u64 n) { return n >= (u64)want; });
    else if (cut_p) meet();                                      // as above
  }
  // ---- 3
  if (cut_p) {
    const float never = fminf(fmaxf((float)(0.5 * (1.0 - dp) / V), 5e-13f), 0.5f), scale = (float)ROW_BINS / -logf(never);
    const auto place = [&](float v) { return __fmul_rn(-scaled(v), scale); };
    clear_bins();
    __syncthreads();
    uint32_t hi_in = 0, lo_in = 0, hi_out = 0, lo_out = 0;       // a lane has fewer than 4096 tokens
    const auto put = [&](float v) {
      const float s = place(v);
      const Mass20 m = mass20_of(fmaxf(weight(v), 0.f));         // NaN: nothing
      if (s < (float)ROW_BINS) { hi_in += m.hi; lo_in += m.lo; add_to_bin(s, m); }
      else { hi_out += m.hi; lo_out += m.lo; }
    };
    if (from == -INFINITY) {
      each([&](int, const float* v) {
#pragma unroll
        for (int k = 0; k < N16; ++k) put(v[k]);
      });
    } else {
      each_from(from, [&](int i, float v) { if (in(i, v)) put(v); });
    }
    u64 before, binned, rest;
    // Both sets: since either was read last, all have met (in `collect`, at the end of `search`, or where nothing was cut off)
    tell(sh.slots[0], warp_total(((u64)hi_in << 20) + lo_in));
    tell(sh.slots[1], warp_total(((u64)hi_out << 20) + lo_out));
    meet();
    hear(sh.slots[0], before, binned);
    hear(sh.slots[1], before, rest);
    const double part = dp * (double)(binned + rest);
    cut_by_bins(binned, place, t / scale, false, [&](float v) -> u64 { return mass_of(weight(v)); }, [&](u64 m) { return m > 0 && !((double)m < part); });
  }
  // ---- 4
  const bool all_in = from == -INFINITY && !(least > 0.f);
  const float start = fmaxf(from, least > 0.f ? peak + (logf(least) * 1.0001f - 1e-5f) * t - 1e-6f * (1.f + fabsf(peak)) : -INFINITY);    // below: weights below `least`
  uint32_t hi20 = 0, lo20 = 0;
  if (all_in) {
    each([&](int, const float* v) {
#pragma unroll
      for (int k = 0; k < N16; ++k) {
        const Mass20 m = mass20_of(fmaxf(weight(v[k]), 0.f));    // NaN: nothing
        hi20 += m.hi;
        lo20 += m.lo;
      }
    });
  } else {
    each([&](int c, const float* v) {
      if (!(highest<N16>(v) >= start)) return;
#pragma unroll
      for (int k = 0; k < N16; ++k) {
        const float w = weight(v[k]);
        const Mass20 m = mass20_of(v[k] > -INFINITY && in(first + c + k, v[k]) && w >= least ? w : 0.f);
        hi20 += m.hi;
        lo20 += m.lo;
      }
    });
  }
  const u64 mine = warp_total(((u64)hi20 << 20) + lo20);
  u64 before, S;
  share_sums(mine, before, S);
  const u64 r = target(S);
  if (r < before || r >= before + mine) return;                  // not in this warp's stretch
  const auto kept = [&](int i, float v) -> u64 {
    if (!(v > -INFINITY) || !in(i, v)) return 0;
    const float w = weight(v);
    return w >= least ? mass_of(w) : 0;
  };
  // a lane takes neighbours, then the lane's stretch is looked at token by token
  const int piece = (span + 31) / 32, p0 = min(s0 + lane * piece, s1), p1 = min(p0 + piece, s1);
  u64 part = 0;
  for (int i = p0; i < p1; ++i) part += kept(first + i, load_logit(places + i));
  const u64 upto = warp_scan(part, lane);
  const int who = __ffs(__ballot_sync(0xffffffffu, before + upto > r)) - 1;
  u64 run = before + __shfl_sync(0xffffffffu, upto - part, who);
  const int q0 = __shfl_sync(0xffffffffu, p0, who), q1 = __shfl_sync(0xffffffffu, p1, who);
  for (int c = q0; c < q1; c += 32) {
    const int i = c + lane;
    const float v = i < q1 ? load_logit(places + i) : -INFINITY;
    const u64 inc = warp_scan(kept(first + i, v), lane);
    const unsigned past = __ballot_sync(0xffffffffu, run + inc > r);
    if (past) {
      if (lane == __ffs(past) - 1) answer(first + i, v, S);
      return;
    }
    run += __shfl_sync(0xffffffffu, inc, 31);
  }
}

}  // namespace oa

using namespace oa;

template <typename T>
static int launch_sample(const SampleParams& p, int* status, cudaStream_t st) {
  // As many CTAs to a row as leave room for two on an SM (of its 228 KB each has half, less the 1 KB that the system keeps: a share of 98 KB beside bins,
  // list and slots: 256 rows of 52000 bf16 logits, top-p 81 us, plain 33, top-k 50 27, by one to an SM with twice the share 92, 40 and 26; 592 of 51000
  // fp32 231, 91 and 96, by one 238, 107 and 94); more, up to eight, while rows leave SMs idle and a share has 4096 tokens or more.
  constexpr int UNIT = Lane16<T>::N, WARPS = SAMPLE_THREADS / 32, MOST = 216 * 1024, HALF = (228 / 2 - 1) * 1024 - (int)sizeof(RowShared);
  const int sms = sm_count();
  const auto span_of = [&](int lg) {                             // places: tokens, and what the first lacks to 16 bytes
    const int share = (p.vocab + (1 << lg) - 1 >> lg) + UNIT;
    return (share + WARPS * UNIT - 1) / (WARPS * UNIT) * UNIT;
  };
  const auto bytes_of = [](int span) { return (ROW_BINS + ROW_LIST) * sizeof(u64) + (size_t)span * WARPS * sizeof(T); };
  int lg = 0;
  while (lg < 3 && (bytes_of(span_of(lg)) > HALF || ((long long)p.rows << lg < sms && p.vocab >> lg >= 2 * 4096))) ++lg;
  const int ctas = 1 << lg, span = span_of(lg);
  const size_t smem = bytes_of(span);
  if (smem > MOST) {                                             // beyond what eight CTAs hold
    launch_short(sample_kernel<T>, dim3((unsigned)p.rows), dim3(SAMPLE_THREADS), 0, st, p);
    return cudaGetLastError() == cudaSuccess ? OA_OK : OA_ERR_LAUNCH;
  }
  static std::atomic<unsigned long long> allowed{0};
  if (allow_smem(allowed, (const void*)sample_row_kernel<T>, MOST) != cudaSuccess) return OA_ERR_LAUNCH;
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
  return cudaLaunchKernelEx(&cfg, sample_row_kernel<T>, p, span, lg, status) == cudaSuccess ? OA_OK : OA_ERR_LAUNCH;
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
