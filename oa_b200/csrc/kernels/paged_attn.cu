// Attention of a batch of requests over a paged key-value cache, behind a prompt that they share.  Query token i of the n new tokens of a
// request sees all `prefix_len` keys of the prompt and the first len - n + i + 1 keys of the request's own pages:
//   o = sum_s softmax_s(scale q . k_s) v_s,   lse = log sum_s exp(scale q . k_s);   a row that sees nothing gives o = 0, lse = -inf.
// A table entry that names no page counts as keys and values of zeros.  Nothing beyond a request's length is read into a result.
#include "common.cuh"
#include "api.h"

namespace oa {

struct PagedAttnParams {
  const void* q;                           // [tokens, q_stride], head h at column h * head_dim
  const void *k, *v;                       // [pages, kv_heads, page_size, head_dim]
  void* out;                               // [tokens, q_heads * head_dim]
  float* lse;                              // [tokens, q_heads] or null
  const int *tables, *lens, *starts, *prefix_table;
  long long q_stride, k_page_stride, v_page_stride, table_stride;
  int tokens, batch, max_fresh, q_heads, kv_heads, page_log2, pages, width, prefix_len;
  float scale;
};

// The request of token t and the token's index in it, found by a whole warp: every round the lanes try 32 places of what is left.
// False for a token that belongs to no request.
__device__ __forceinline__ bool find_request(const int* __restrict__ starts, int batch, int t, int lane, int& b, int& i) {
  int lo = 0, n = batch;                   // starts[lo] <= t is known to hold when anything holds
  if (batch <= 0 || starts[0] > t || starts[batch] <= t) return false;
  while (n > 1) {
    const int step = (n + 31) / 32, at = lo + lane * step;
    const unsigned under = __ballot_sync(0xffffffffu, lane * step < n && starts[at] <= t);
    const int k = 31 - __clz(under);       // starts do not fall, so the lanes at or under t come first; lane 0 is one
    lo += k * step;
    n = min(step, n - k * step);
  }
  b = lo;
  i = t - starts[lo];
  return true;
}

template <typename T> struct Four;         // four elements of a row
template <> struct Four<float> {
  static __device__ __forceinline__ float4 load(const float* p) { return *reinterpret_cast<const float4*>(p); }
};
template <> struct Four<__nv_bfloat16> {
  static __device__ __forceinline__ float4 load(const __nv_bfloat16* p) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    const float2 a = unpack_bf16x2(u.x), b = unpack_bf16x2(u.y);
    return make_float4(a.x, a.y, b.x, b.y);
  }
};
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// One block for a query row: four warps stride over the keys with a running maximum and sum, 32 keys at a time (lane = key for q . k,
// lane = a slice of the head for p v), and join their states through shared memory.
template <typename T, int HD>
__global__ void __launch_bounds__(128) paged_attn_rows_kernel(const PagedAttnParams p) {
  constexpr int PER = HD / 32;
  __shared__ float s_q[HD];
  __shared__ float s_m[4], s_l[4];
  __shared__ float s_acc[4][HD];
  pdl_launch_dependents();
  pdl_wait();
  const int t = blockIdx.x, h = blockIdx.y, kh = h / (p.q_heads / p.kv_heads);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float sl2 = p.scale * 1.4426950408889634f;
  for (int d = threadIdx.x; d < HD; d += 128) s_q[d] = to_f32(static_cast<const T*>(p.q)[t * p.q_stride + h * HD + d]) * sl2;
  int b = 0, i = 0, len = 0, prefix = p.prefix_len;
  if (find_request(p.starts, p.batch, t, lane, b, i) && i < p.max_fresh) {
    const int own = min(p.lens[b], p.width << p.page_log2);
    len = max(own - (p.starts[b + 1] - p.starts[b]) + i + 1, 0);
  } else {
    prefix = 0;
  }
  __syncthreads();
  const int total = prefix + len;
  float m = -INFINITY, l = 0.f, acc[PER];
#pragma unroll
  for (int e = 0; e < PER; ++e) acc[e] = 0.f;
  const long long head_off = ((long long)kh << p.page_log2) * HD;
  const int mask = (1 << p.page_log2) - 1;
  for (int s0 = warp * 32; s0 < total; s0 += 128) {
    const int s = s0 + lane;
    float sc = -INFINITY;
    int page = -1, off = 0;
    if (s < total) {
      const int o = s < prefix ? s : s - prefix;
      page = s < prefix ? p.prefix_table[o >> p.page_log2] : p.tables[b * p.table_stride + (o >> p.page_log2)];
      off = o & mask;
      if (page >= p.pages) page = -1;
      sc = 0.f;
      if (page >= 0) {
        const T* kr = static_cast<const T*>(p.k) + page * p.k_page_stride + head_off + off * HD;
#pragma unroll
        for (int j = 0; j < HD; j += 4) {
          const float4 kv = Four<T>::load(kr + j);
          sc += kv.x * s_q[j] + kv.y * s_q[j + 1] + kv.z * s_q[j + 2] + kv.w * s_q[j + 3];
        }
      }
    }
    const float m_new = fmaxf(m, warp_max(sc));
    const float pr = (s < total && m_new != -INFINITY) ? fast_exp2(sc - m_new) : 0.f;
    const float corr = m == -INFINITY ? 0.f : fast_exp2(m - m_new);
    l = l * corr + warp_sum(pr);
    m = m_new;
#pragma unroll
    for (int e = 0; e < PER; ++e) acc[e] *= corr;
    const int n = min(32, total - s0);
    for (int j = 0; j < n; ++j) {
      const float pj = __shfl_sync(0xffffffffu, pr, j);
      const int pg = __shfl_sync(0xffffffffu, page, j), of = __shfl_sync(0xffffffffu, off, j);
      if (pg < 0) continue;
      const T* vr = static_cast<const T*>(p.v) + pg * p.v_page_stride + head_off + of * HD + lane;
#pragma unroll
      for (int e = 0; e < PER; ++e) acc[e] += pj * to_f32(vr[e * 32]);
    }
  }
  if (lane == 0) { s_m[warp] = m; s_l[warp] = l; }
#pragma unroll
  for (int e = 0; e < PER; ++e) s_acc[warp][e * 32 + lane] = acc[e];
  __syncthreads();
  const float M = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
  float L = 0.f, w[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) { w[k] = s_m[k] == -INFINITY ? 0.f : fast_exp2(s_m[k] - M); L += s_l[k] * w[k]; }
  for (int d = threadIdx.x; d < HD; d += 128) {
    const float v = s_acc[0][d] * w[0] + s_acc[1][d] * w[1] + s_acc[2][d] * w[2] + s_acc[3][d] * w[3];
    put(static_cast<T*>(p.out) + ((long long)t * p.q_heads + h) * HD + d, total > 0 ? v / L : 0.f);
  }
  if (p.lse && threadIdx.x == 0) p.lse[(long long)t * p.q_heads + h] = total > 0 ? (M + log2f(L)) * 0.6931471805599453f : -INFINITY;
}

}  // namespace oa

using namespace oa;

extern "C" int oa_paged_attn(int dtype, const void* q, long long q_stride, const void* k_pages, const void* v_pages, long long k_page_stride,
                             long long v_page_stride, const int* tables, long long table_stride, const int* lens, const int* starts, const int* prefix_table,
                             int prefix_len, void* out, float* lse, int tokens, int batch, int max_fresh, int q_heads, int kv_heads, int head_dim,
                             int page_size, int pages, int width, float scale, void* stream) {
  int lg = 4;
  while (lg < 7 && 1 << lg != page_size) ++lg;
  if (1 << lg != page_size || (head_dim != 32 && head_dim != 64 && head_dim != 128) || (dtype != OA_F32 && dtype != OA_BF16)) return OA_ERR_UNSUPPORTED;
  if (tokens < 0 || batch < 0 || max_fresh < 0 || q_heads < 1 || kv_heads < 1 || q_heads % kv_heads || pages < 0 || width < 0 || prefix_len < 0 ||
      table_stride < width || (prefix_len > 0 && !prefix_table) || ((long long)width << lg) > 0x7fffffffll - prefix_len)
    return OA_ERR_ARG;
  const int unit = dtype == OA_F32 ? 4 : 8;                  // elements of 16 bytes
  if (q_stride % unit || k_page_stride % unit || v_page_stride % unit ||
      ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_pages) | reinterpret_cast<uintptr_t>(v_pages) | reinterpret_cast<uintptr_t>(out)) & 15))
    return OA_ERR_ALIGN;
  if (q_heads > 65535) return OA_ERR_TOO_LARGE;
  if (tokens == 0) return OA_OK;
  const PagedAttnParams p{q, k_pages, v_pages, out, lse, tables, lens, starts, prefix_table, q_stride, k_page_stride, v_page_stride, table_stride,
                          tokens, batch, max_fresh, q_heads, kv_heads, lg, pages, width, prefix_len, scale};
  const dim3 grid((unsigned)tokens, (unsigned)q_heads);
  cudaStream_t st = (cudaStream_t)stream;
#define OA_ROWS(T, HD) launch_short(paged_attn_rows_kernel<T, HD>, grid, dim3(128), 0, st, p)
  if (dtype == OA_F32) {
    if (head_dim == 32) OA_ROWS(float, 32); else if (head_dim == 64) OA_ROWS(float, 64); else OA_ROWS(float, 128);
  } else {
    if (head_dim == 32) OA_ROWS(__nv_bfloat16, 32); else if (head_dim == 64) OA_ROWS(__nv_bfloat16, 64); else OA_ROWS(__nv_bfloat16, 128);
  }
#undef OA_ROWS
  return cudaGetLastError() == cudaSuccess ? OA_OK : OA_ERR_LAUNCH;
}
