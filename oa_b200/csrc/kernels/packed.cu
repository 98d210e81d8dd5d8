// Packed sequences: which tiles the attention kernels work on, and rotation by positions on several axes.
#include "common.cuh"
#include "packed.cuh"
#include "vec8.cuh"
#include "per_device.h"
#include "api.h"

namespace oa {

// ------------------------------------------------------------------------------------------------ plan
// Sequences are rows [starts[b], starts[b + 1]) of the packed tensors; starts that fall or leave [0, tokens] are taken as the nearest that do
// not.  Sequences of up to 64 rows go on a list of their own; of the others the attention kernels take their work from two lists, the longest first: tiles of 128
// rows of a sequence, and pairs of neighbouring tiles.  Under the causal mask tile i of a sequence sees i + 1 tiles of keys (and its mirror image, tile n - 1 - i, is seen by as many tiles of
// queries), so both lists are sorted by that index, by counting.  The order among equals is that of the atomics; nothing depends on it but
// which SM works on a tile.  One block: a batch has few thousand tiles, and one plan serves every layer of a step in both directions.  Latency: 5 us
// for one sequence of 4096 and for 16 of up to 2048, 5.6 for 64 of up to 300, 6.5 for 512 of up to 48.
constexpr int PLAN_KEPT = 1024;           // sequences whose starts are kept in shared memory, at most
constexpr int PLAN_FEW = 8;               // bins taken for 32 sequences at once

struct PackedPlanParams {
  const int* starts;
  int* plan;
  int batch, tokens, shift;               // bins of 2^shift tile indices
};

template <int THREADS, typename Op>
__device__ __forceinline__ int plan_scan(int v, int* s_warp, Op op) {   // inclusive, over the block
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v = op(v, u);
  }
  __syncthreads();                        // the last scan's reads
  if (lane == 31) s_warp[warp] = v;
  __syncthreads();
  int w = s_warp[lane < THREADS / 32 ? lane : 0];            // by every warp for itself
#pragma unroll
  for (int o = 1; o < THREADS / 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w = op(w, u);
  }
  const int before = __shfl_sync(0xffffffffu, w, warp > 0 ? warp - 1 : 0);
  return warp > 0 ? op(v, before) : v;
}

// THREADS: of the block, and bins
template <int THREADS>
__global__ void __launch_bounds__(THREADS) packed_plan_kernel(const PackedPlanParams p) {
  __shared__ int s_warp[32], s_count[2][THREADS], s_top, s_short[3], s_starts[PLAN_KEPT + 1];
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, shift = p.shift, per = 1 << shift;
  int* const out = p.plan + PACKED_HEADER;
  const bool kept = p.batch <= PLAN_KEPT;
  const int* const starts = kept ? s_starts : out;
  s_count[0][tid] = s_count[1][tid] = 0;
  if (tid < 3) s_short[tid] = 0;
  if (tid == 0) s_top = 0;
  const auto most = [](int a, int b) { return max(a, b); };
  for (int b0 = 0; b0 <= p.batch; b0 += THREADS) {
    const int b = b0 + tid;
    const int v = plan_scan<THREADS>(b <= p.batch ? min(max(p.starts[b], 0), p.tokens) : 0, s_warp, most);
    const int s = max(v, s_top);          // written below, behind a barrier
    if (b <= p.batch) {
      out[b] = s;
      if (kept) s_starts[b] = s;
    }
    __syncthreads();
    if (tid == THREADS - 1) s_top = s;
  }
  __syncthreads();
  // `team` warps to 32 sequences.  The first bins are taken for all of them at once, each by one of the warps; the others of one sequence after the other, a bin to
  // a lane, each warp its share of the sequences.
  // add(which, bin, n) is called for n indices of a bin, returns where they go; put(which, at, first index, n) follows
  int team = 1;
  while (team < THREADS / 32 && team * p.batch <= THREADS / 2) team *= 2;
  const int sub = (tid >> 5) & (team - 1);
  const auto walk = [&](auto add, auto put) {
    for (int b0 = (tid >> 5) / team * 32; b0 < p.batch; b0 += THREADS / team) {
      const int b = b0 + lane;
      const int lo = b < p.batch ? starts[b] : 0, hi = b < p.batch ? starts[b + 1] : 0;
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        const int rows = PACKED_TILE << which;
        const int n = hi - lo <= PACKED_SHORT ? 0 : (hi - lo + rows - 1) / rows;
        for (int k = sub; k < PLAN_FEW; k += team) {
          const int c = min(max(n - (k << shift), 0), per);
          const unsigned any = __ballot_sync(0xffffffffu, c > 0);
          if (!any) break;
          int sum = __popc(any & 0xffffffffu >> (31 - lane));              // of the lanes up to this one
          if (per > 1) {
            sum = c;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
              const int u = __shfl_up_sync(0xffffffffu, sum, o);
              if (lane >= o) sum += u;
            }
          }
          int base = lane == 31 ? add(which, k, sum) : 0;
          base = __shfl_sync(0xffffffffu, base, 31);
          put(which, base + sum - c, k << shift, c, lo, hi, b);
        }
        unsigned more = __ballot_sync(0xffffffffu, n > PLAN_FEW << shift);
        for (int i = 0; more; ++i) {
          const int src = __ffs(more) - 1;
          more &= more - 1;
          if ((i & (team - 1)) != sub) continue;
          const int nn = __shfl_sync(0xffffffffu, n, src), l = __shfl_sync(0xffffffffu, lo, src), h = __shfl_sync(0xffffffffu, hi, src);
          for (int k = PLAN_FEW + lane; (k << shift) < nn; k += 32) {
            const int c = min(per, nn - (k << shift));
            put(which, add(which, k, c), k << shift, c, l, h, b0 + src);
          }
        }
      }
    }
  };
  walk([&](int which, int bin, int n) { return n > 0 ? atomicAdd(&s_count[which][bin], n) : 0; }, [](int, int, int, int, int, int, int) {});
  __syncthreads();
  int4* lists[3];
  lists[0] = reinterpret_cast<int4*>(p.plan + packed_tiles_at(p.batch));
  lists[1] = lists[0] + packed_max_tiles(p.tokens, p.batch);
  lists[2] = lists[1] + packed_max_pairs(p.tokens, p.batch);
  // short sequences by their number of 16 rows, most first: counted, then placed
  for (int pass = 0; pass < 2; ++pass) {
    for (int b0 = tid - lane; b0 < p.batch; b0 += THREADS) {
      const int b = b0 + lane;
      const int lo = b < p.batch ? starts[b] : 0, hi = b < p.batch ? starts[b + 1] : 0, n = hi - lo;
      const int mine = n < 1 || n > PACKED_SHORT ? -1 : n > 32 ? 0 : n > 16 ? 1 : 2;
#pragma unroll
      for (int c = 0; c < 3; ++c) {
        const unsigned all = __ballot_sync(0xffffffffu, mine == c);
        if (!all) continue;
        int at = lane == 0 ? atomicAdd(&s_short[c], __popc(all)) : 0;
        at = __shfl_sync(0xffffffffu, at, 0);
        if (pass == 1 && mine == c) lists[2][at + __popc(all & ((1u << lane) - 1))] = make_int4(lo, hi, 0, b);
      }
    }
    __syncthreads();
    if (pass == 0 && tid == 0) {
      const int n0 = s_short[0], n1 = s_short[1];
      p.plan[4] = n0; p.plan[5] = n1; p.plan[6] = s_short[2];
      s_short[0] = 0; s_short[1] = n0; s_short[2] = n0 + n1;
    }
    __syncthreads();
  }
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    // how many have a larger index: the sums from the end
    const int mine = s_count[which][THREADS - 1 - tid];
    const int sum = plan_scan<THREADS>(mine, s_warp, [](int a, int b) { return a + b; });
    s_count[which][THREADS - 1 - tid] = sum - mine;
    if (tid == THREADS - 1) p.plan[which] = sum;
  }
  __syncthreads();
  if (tid == 0) { p.plan[2] = starts[0]; p.plan[3] = starts[p.batch]; p.plan[7] = 0; }
  walk([&](int which, int bin, int n) { return n > 0 ? atomicAdd(&s_count[which][bin], n) : 0; },
       [&](int which, int at, int first, int n, int lo, int hi, int b) {
         for (int i = 0; i < n; ++i) lists[which][at + i] = make_int4(lo, hi, first + i, b);
       });
}

// ------------------------------------------------------------------------------------------------ rotation
// y = x with each pair (j, j + half) of a head turned by the token's position on the pair's own axis, times theta^(-j / half); dimensions from
// 2 half on are copied.  A token's angles are worked out once for all its heads: position * turns in 64 bits (in 32 bits a position of 131072 leaves
// an angle 0.008 off), the whole turns taken off, and what is left in [-1/2, 1/2] turns in 32 bits.  The gradient turns the other way.
//
// Bound by the bytes: each thread takes 16 bytes of a head's first half and the 16 that belong to them, and has two such pieces on their way before the angles are
// worked out.  A block works on as many tokens as give its threads a piece each, or on a part of one where tokens alone leave SMs idle.
// 16381 rows of 72 heads of 64 in bf16 47.7 us, 6.3 TB/s; 32 rows 2.5 us.
constexpr int ROTARY_MAX_HALF = 128, ROTARY_THREADS = 256;
constexpr int ROTARY_ANGLES = 1024;       // of a block's tokens
struct RotaryParams {
  const void* x;
  long long x_stride;
  void* y;
  long long y_stride;
  const int* positions;                   // [axes, tokens]
  int tokens, heads, hd, half, backward;
  int group;                              // tokens of a block
  int per, of_head, turned;               // pieces of a token, of a head, and those of a head that are turned
  uint32_t per_inv, of_head_inv;          // 2^32 over them, rounded up: quotients of numbers below 2^16 by multiplication
  uint8_t axis[ROTARY_MAX_HALF];
  double turns[ROTARY_MAX_HALF];          // turns a position: theta^(-j / half) / (2 pi)
};

__device__ __forceinline__ void rotary_angle(const RotaryParams& p, int t, int k, float* s_cos, float* s_sin) {
  const double a = (double)p.positions[(long long)p.axis[k] * p.tokens + t] * p.turns[k];
  float s, c;
  sincospif((float)(2.0 * (a - rint(a))), &s, &c);
  *s_cos = c;
  *s_sin = p.backward ? -s : s;
}

template <typename T>
__global__ void __launch_bounds__(ROTARY_THREADS) rotary_kernel(const __grid_constant__ RotaryParams p) {
  __shared__ __align__(16) float s_cos[ROTARY_ANGLES], s_sin[ROTARY_ANGLES];
  pdl_launch_dependents();
  pdl_wait();
  const int t0 = blockIdx.x * p.group, here = min(p.group, p.tokens - t0), n = here * p.per, step = gridDim.y * blockDim.x;
  int i = blockIdx.y * blockDim.x + threadIdx.x;
  Vec8<T> a[2], b[2];
  int token[2], off[2], pair[2];          // of a piece: where in its token's row, and its first pair (-1: dimensions that are only copied)
  const auto over = [](int x, int d, uint32_t inv) { return d == 1 ? x : (int)__umulhi((uint32_t)x, inv); };
  const auto fetch = [&] {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int at = i + q * step;
      if (at >= n) continue;
      token[q] = over(at, p.per, p.per_inv);
      const int in = at - token[q] * p.per, head = over(in, p.of_head, p.of_head_inv), j = in - head * p.of_head;
      pair[q] = j < p.turned ? j * 8 : -1;
      off[q] = head * p.hd + (j < p.turned ? j * 8 : p.half + j * 8);
      const T* row = static_cast<const T*>(p.x) + (t0 + token[q]) * p.x_stride + off[q];
      a[q] = *reinterpret_cast<const Vec8<T>*>(row);
      if (pair[q] >= 0) b[q] = *reinterpret_cast<const Vec8<T>*>(row + p.half);
    }
  };
  fetch();
  for (int k = threadIdx.x; k < here * p.half; k += blockDim.x) rotary_angle(p, t0 + k / p.half, k % p.half, s_cos + k, s_sin + k);
  __syncthreads();
  while (i < n) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      if (i + q * step >= n) continue;
      T* to = static_cast<T*>(p.y) + (t0 + token[q]) * p.y_stride + off[q];
      if (pair[q] >= 0) {
        float x[8], y[8], lo[8], hi[8], c[8], s[8];
        a[q].get(x);
        b[q].get(y);
        const int k0 = token[q] * p.half + pair[q];
#pragma unroll
        for (int k = 0; k < 8; k += 4) {
          *reinterpret_cast<float4*>(c + k) = *reinterpret_cast<const float4*>(s_cos + k0 + k);
          *reinterpret_cast<float4*>(s + k) = *reinterpret_cast<const float4*>(s_sin + k0 + k);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          lo[k] = x[k] * c[k] - y[k] * s[k];
          hi[k] = y[k] * c[k] + x[k] * s[k];
        }
        a[q].set(lo);
        b[q].set(hi);
        *reinterpret_cast<Vec8<T>*>(to + p.half) = b[q];
      }
      *reinterpret_cast<Vec8<T>*>(to) = a[q];
    }
    i += 2 * step;
    fetch();
  }
}

// The same element by element: rows that lie anywhere, any number of pairs
__device__ __forceinline__ float rotary_load(const float* p) { return *p; }
__device__ __forceinline__ float rotary_load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void rotary_store(float* p, float v) { *p = v; }
__device__ __forceinline__ void rotary_store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

template <typename T>
__global__ void __launch_bounds__(ROTARY_THREADS) rotary_any_kernel(const __grid_constant__ RotaryParams p) {
  __shared__ float s_cos[ROTARY_MAX_HALF], s_sin[ROTARY_MAX_HALF];
  pdl_launch_dependents();
  pdl_wait();
  const int rest = p.hd - 2 * p.half, per = p.half + rest;       // pairs and single dimensions of a head
  for (int t = blockIdx.x; t < p.tokens; t += gridDim.x) {
    __syncthreads();
    for (int k = threadIdx.x; k < p.half; k += blockDim.x) rotary_angle(p, t, k, s_cos + k, s_sin + k);
    __syncthreads();
    const T* x = static_cast<const T*>(p.x) + t * p.x_stride;
    T* y = static_cast<T*>(p.y) + t * p.y_stride;
    for (int i = threadIdx.x; i < p.heads * per; i += blockDim.x) {
      const int h = i / per, j = i - h * per, at = h * p.hd + j;
      if (j < p.half) {
        const float a = rotary_load(x + at), b = rotary_load(x + at + p.half), c = s_cos[j], s = s_sin[j];
        rotary_store(y + at, a * c - b * s);
        rotary_store(y + at + p.half, b * c + a * s);
      } else {
        y[at + p.half] = x[at + p.half];
      }
    }
  }
}

template <typename T>
static int rotary_run(RotaryParams& p, cudaStream_t st) {
  const int rest = p.hd - 2 * p.half, unit = 16 / (int)sizeof(T);
  const bool pieces = p.half % 8 == 0 && rest % 8 == 0 && p.x_stride % unit == 0 && p.y_stride % unit == 0 &&
                      ((reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.y)) & 15) == 0 && (long long)p.heads * p.hd < (1 << 18);
  if (!pieces) {
    const dim3 grid((unsigned)(p.tokens < (1 << 20) ? p.tokens : 1 << 20));
    launch_short(rotary_any_kernel<T>, grid, dim3(ROTARY_THREADS), 0, st, p);
    return cudaGetLastError() == cudaSuccess ? OA_OK : OA_ERR_LAUNCH;
  }
  // dimensions that are only copied are left alone where they lie already
  p.turned = p.half / 8;
  p.of_head = p.turned + (p.x == p.y && p.x_stride == p.y_stride ? 0 : rest / 8);
  p.per = p.heads * p.of_head;
  p.per_inv = (uint32_t)(((1ull << 32) + p.per - 1) / p.per);
  p.of_head_inv = (uint32_t)(((1ull << 32) + p.of_head - 1) / p.of_head);
  constexpr int FULL = 2 * ROTARY_THREADS;                       // pieces of a block, two to a thread
  p.group = p.per >= FULL ? 1 : FULL / p.per;
  const int few = p.tokens / (2 * sm_count());                   // tokens of a block while every SM has two
  if (p.group > few) p.group = few > 1 ? few : 1;
  if (p.group > ROTARY_ANGLES / p.half) p.group = ROTARY_ANGLES / p.half;
  // a token over several blocks while tokens alone leave SMs idle; the threads that two pieces each keep busy, one each while they are few
  const int blocks = (p.tokens + p.group - 1) / p.group, n = p.group * p.per, room = (2 * sm_count() + blocks - 1) / blocks, want = (n + ROTARY_THREADS - 1) / ROTARY_THREADS;
  const int spread = room < want ? room : want, share = (n + spread - 1) / spread, rounds = (share + FULL - 1) / FULL;
  const int each = blocks >= 2 * sm_count() ? 2 * rounds : (share + ROTARY_THREADS - 1) / ROTARY_THREADS, threads = ((share + each - 1) / each + 31) / 32 * 32;
  launch_short(rotary_kernel<T>, dim3((unsigned)blocks, (unsigned)spread), dim3((unsigned)threads), 0, st, p);
  return cudaGetLastError() == cudaSuccess ? OA_OK : OA_ERR_LAUNCH;
}

}  // namespace oa

using namespace oa;

extern "C" size_t oa_packed_plan_bytes(int tokens, int batch) {
  return ((size_t)packed_tiles_at(batch) + 4 * ((size_t)packed_max_tiles(tokens, batch) + packed_max_pairs(tokens, batch) + batch)) * sizeof(int);
}

extern "C" int oa_packed_plan(const int* starts, int* plan, int batch, int tokens, void* stream) {
  if (batch < 0 || tokens < 0 || !starts || !plan) return OA_ERR_ARG;
  if (batch > PACKED_MAX_BATCH || tokens > PACKED_MAX_TOKENS) return OA_ERR_TOO_LARGE;
  if (reinterpret_cast<uintptr_t>(plan) & 15) return OA_ERR_ALIGN;
  // the smaller block where a bin to an index is not more than it has threads, for it gets through its barriers sooner
  const bool small = batch <= 256 && tokens / PACKED_TILE < 256;
  const int bins = small ? 256 : 1024;
  int shift = 0;
  while (((tokens / PACKED_TILE) >> shift) >= bins) ++shift;
  launch_short(small ? packed_plan_kernel<256> : packed_plan_kernel<1024>, dim3(1), dim3(bins), 0, (cudaStream_t)stream,
               PackedPlanParams{starts, plan, batch, tokens, shift});
  return cudaGetLastError() == cudaSuccess ? OA_OK : OA_ERR_LAUNCH;
}

extern "C" int oa_rotary_axes(int dtype, const void* x, long long x_stride, void* y, long long y_stride, const int* positions, const void* pair_axes,
                              const void* turns, int pairs, int tokens, int heads, int head_dim, int backward, void* stream) {
  if (dtype != OA_F32 && dtype != OA_BF16) return OA_ERR_UNSUPPORTED;
  if (pairs < 1 || pairs > ROTARY_MAX_HALF) return OA_ERR_UNSUPPORTED;
  if (tokens < 0 || heads < 1 || 2 * pairs > head_dim || !pair_axes || !turns) return OA_ERR_ARG;
  if (tokens == 0) return OA_OK;
  RotaryParams p{x, x_stride, y, y_stride, positions, tokens, heads, head_dim, pairs, backward, 1, 0, 0, 0, 0, 0, {}, {}};
  for (int j = 0; j < pairs; ++j) {
    p.axis[j] = static_cast<const uint8_t*>(pair_axes)[j];
    p.turns[j] = static_cast<const double*>(turns)[j];
  }
  return dtype == OA_F32 ? rotary_run<float>(p, (cudaStream_t)stream) : rotary_run<__nv_bfloat16>(p, (cudaStream_t)stream);
}
