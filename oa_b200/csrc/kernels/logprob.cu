// Log-probabilities of given tokens, with the entropy and the likeliest alternatives of each row of logits, and the logits' gradient.
//
// For a row y = scale * x with largest element m:  l = sum exp(y - m),  log p_j = (y_j - m) - log l,  H = -sum p_j log p_j = log l - s / l
// with s = sum exp(y - m) (y - m).  The differences from m are what is summed, so that nothing of the size of m cancels.  With gradients g of the
// target's log-probability and h of the entropy,
//   dx_j = scale * (g ([j = target] - p_j) - h p_j (log p_j + H)).
// A logit of -inf has probability 0 and adds nothing anywhere.  A row with NaN or +inf is NaN; a row without anything above -inf has
// log-probability -inf, entropy 0 and no gradient.
#include "common.cuh"
#include "per_device.h"
#include "api.h"

namespace oa {

constexpr int LP_THREADS = 512;
constexpr int LP_MAX_TOP = 32;

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

// Sums of exponentials below a running maximum
struct LpSums {
  float m, l, s;
  __device__ __forceinline__ void raise(float to) {          // to > m
    if (m != -INFINITY) {
      const float d = m - to, a = expf(d);
      s = a * fmaf(l, fmaxf(d, -1e4f), s);
      l *= a;
    }
    m = to;
  }
  __device__ __forceinline__ void add(float y) {
    if (y > m) raise(y);
    const float d = fmaxf(y - m, -1e4f), e = expf(d);        // a NaN, like -inf, adds nothing here: the row is marked
    if (m != -INFINITY) { l += e; s = fmaf(e, d, s); }
  }
  __device__ __forceinline__ void join(const LpSums& o) {
    LpSums b = o;
    if (b.m > m) raise(b.m);
    else if (m > b.m) b.raise(m);
    l += b.l;
    s += b.s;
  }
};

// Whole numbers that order like the logits: larger ones first, of equal ones the lower index; NaN as -inf
__device__ __forceinline__ unsigned long long lp_rank(float x, int i) {
  const uint32_t b = __float_as_uint(x + 0.f);
  const uint32_t k = x != x ? 0x007fffffu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
  return ((unsigned long long)k << 32) | (uint32_t)~i;
}

template <typename T>
__global__ void __launch_bounds__(LP_THREADS) logprob_kernel(const LogprobParams p) {
  __shared__ LpSums s_sums[LP_THREADS / 32];
  __shared__ unsigned long long s_best[LP_THREADS / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T* x = static_cast<const T*>(p.x) + row * p.stride;
  LpSums a{-INFINITY, 0.f, 0.f};
  bool bad = false;
  for (int i = tid; i < p.vocab; i += LP_THREADS) {
    const float y = lp_load(x + i) * p.scale;
    bad |= !(y <= 3.402823466e38f);
    a.add(y);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    a.join({__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.l, o), __shfl_xor_sync(0xffffffffu, a.s, o)});
  if (lane == 0) s_sums[warp] = a;
  bad = __syncthreads_or(bad);
  a = s_sums[0];
  for (int w = 1; w < LP_THREADS / 32; ++w) a.join(s_sums[w]);
  if (bad) a.m = a.l = a.s = NAN;
  const bool none = a.m == -INFINITY;
  const float log_l = none ? 0.f : logf(a.l);
  const auto logprob = [&](float xi) { return none ? -INFINITY : (xi * p.scale - a.m) - log_l; };
  if (tid == 0) {
    const int t = p.targets[row];
    p.logprobs[row] = t == p.ignore ? 0.f : t >= 0 && t < p.vocab ? logprob(lp_load(x + t)) : NAN;
    p.entropy[row] = none ? 0.f : log_l - a.s / a.l;
    p.stats[2 * row] = a.m;
    p.stats[2 * row + 1] = log_l;
  }
  // the likeliest one after the other
  unsigned long long last = ~0ull;
  for (int k = 0; k < p.top; ++k) {
    unsigned long long best = 0;
    for (int i = tid; i < p.vocab; i += LP_THREADS) {
      const unsigned long long r = lp_rank(lp_load(x + i), i);
      if (r < last && r > best) best = r;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    __syncthreads();
    if (lane == 0) s_best[warp] = best;
    __syncthreads();
    for (int w = 0; w < LP_THREADS / 32; ++w) best = max(best, s_best[w]);
    last = best;
    if (tid == 0) {
      const int id = (int)~(uint32_t)best;
      p.top_ids[(long long)row * p.top + k] = id;
      p.top_logprobs[(long long)row * p.top + k] = logprob(lp_load(x + id));
    }
  }
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

__device__ __forceinline__ float lp_max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ void lp_put(float* p, float v) { *p = v; }
__device__ __forceinline__ void lp_put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// A row's own numbers
struct LpRow {
  float m, log_l, H, g, h, scale;
  int target;
  bool none;
  __device__ __forceinline__ LpRow(const LogprobBwdParams& p, int row) {
    m = p.stats[2 * row];
    log_l = p.stats[2 * row + 1];
    H = p.entropy[row];
    target = p.targets[row];
    g = target == p.ignore || !p.dlogprobs ? 0.f : target >= 0 && target < p.vocab ? p.dlogprobs[row] : NAN;
    h = p.dentropy ? p.dentropy[row] : 0.f;
    none = m == -INFINITY;
    scale = p.scale;
  }
  __device__ __forceinline__ float grad(float x, int j) const {
    const float lp = lp_max_nan(fmaf(x, scale, -m) - log_l, -1e4f), q = expf(lp);      // a probability of 0 takes its logarithm along
    const float d = -q * fmaf(h, lp + H, g) + (j == target ? g : 0.f);
    return none ? 0.f : scale * d;
  }
};

template <typename T>
__global__ void __launch_bounds__(256) logprob_bwd_kernel(const LogprobBwdParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int row = blockIdx.x;
  const LpRow r(p, row);
  const T* x = static_cast<const T*>(p.x) + row * p.stride;
  T* dx = static_cast<T*>(p.dx) + row * p.d_stride;
  for (int i = blockIdx.y * 256 + threadIdx.x; i < p.vocab; i += gridDim.y * 256) lp_put(dx + i, r.grad(lp_load(x + i), i));
}

}  // namespace oa

using namespace oa;

extern "C" int oa_token_logprobs(int dtype, const void* logits, long long stride, const int* targets, float* logprobs, float* entropy, float* stats,
                                 float* top_logprobs, int* top_ids, int top, int rows, int vocab, float scale, int ignore_index, void* stream) {
  if (dtype != OA_F32 && dtype != OA_BF16) return OA_ERR_UNSUPPORTED;
  if (rows < 0 || vocab < 1 || top < 0 || top > vocab || stride < 0) return OA_ERR_ARG;
  if (top > LP_MAX_TOP) return OA_ERR_UNSUPPORTED;
  if (rows == 0) return OA_OK;
  const LogprobParams p{logits, stride, targets, logprobs, entropy, stats, top_logprobs, top_ids, top, rows, vocab, ignore_index, scale};
  if (dtype == OA_F32) launch_short(logprob_kernel<float>, dim3(rows), dim3(LP_THREADS), 0, (cudaStream_t)stream, p);
  else launch_short(logprob_kernel<__nv_bfloat16>, dim3(rows), dim3(LP_THREADS), 0, (cudaStream_t)stream, p);
  return cudaGetLastError() == cudaSuccess ? OA_OK : OA_ERR_LAUNCH;
}

extern "C" int oa_token_logprobs_bwd(int dtype, const void* logits, long long stride, const int* targets, const float* entropy, const float* stats,
                                     const float* dlogprobs, const float* dentropy, void* dlogits, long long d_stride, int rows, int vocab, float scale,
                                     int ignore_index, void* stream) {
  if (dtype != OA_F32 && dtype != OA_BF16) return OA_ERR_UNSUPPORTED;
  if (rows < 0 || vocab < 1 || stride < 0 || (rows > 1 && d_stride < vocab)) return OA_ERR_ARG;
  if (rows == 0) return OA_OK;
  const LogprobBwdParams p{logits, stride, targets, entropy, stats, dlogprobs, dentropy, dlogits, d_stride, rows, vocab, ignore_index, scale};
  const int pieces = (vocab + 2047) / 2048;
  const dim3 grid((unsigned)rows, (unsigned)(pieces < 64 ? pieces : 64));
  if (dtype == OA_F32) launch_short(logprob_bwd_kernel<float>, grid, dim3(256), 0, (cudaStream_t)stream, p);
  else launch_short(logprob_bwd_kernel<__nv_bfloat16>, grid, dim3(256), 0, (cudaStream_t)stream, p);
  return cudaGetLastError() == cudaSuccess ? OA_OK : OA_ERR_LAUNCH;
}
