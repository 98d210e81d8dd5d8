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
__device__ __forceinline__ u64 mass_of(float w) { return (u64)(w * 1099511627776.f); }

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
  const Weigh wt{__uint_as_float((top_key & 0x80000000u) ? top_key & 0x7fffffffu : ~top_key), 1.f / t};
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

}  // namespace oa

using namespace oa;

extern "C" int oa_sample(int dtype, const void* logits, long long stride, const float* u, const float* temperature, const int* top_k, const float* top_p,
                         const float* min_p, int* tokens, float* logprobs, int rows, int vocab, void* stream) {
  if (dtype != OA_F32 && dtype != OA_BF16) return OA_ERR_UNSUPPORTED;
  if (rows < 0 || vocab < 0) return OA_ERR_ARG;
  if (vocab > 1 << 23) return OA_ERR_TOO_LARGE;              // 2^40 times this many fits a sum of 64 bits
  if (rows == 0) return OA_OK;
  const SampleParams p{logits, stride, u, temperature, top_p, min_p, top_k, tokens, logprobs, rows, vocab};
  if (dtype == OA_F32) launch_short(sample_kernel<float>, dim3((unsigned)rows), dim3(SAMPLE_THREADS), 0, (cudaStream_t)stream, p);
  else launch_short(sample_kernel<__nv_bfloat16>, dim3((unsigned)rows), dim3(SAMPLE_THREADS), 0, (cudaStream_t)stream, p);
  return cudaGetLastError() == cudaSuccess ? OA_OK : OA_ERR_LAUNCH;
}
