// A paged key-value cache for requests of unequal length.  The cache of a layer is [pages, kv_heads, page_size, head_dim]; a request owns
// the pages in its row of a table, and the slot of a token is page * page_size + offset.
//   oa_paged_plan     from the requests' lengths: fresh pages into the tables, and for every new token its request, position and slot
//   oa_paged_release  pages of finished requests go back on the free stack
//   oa_paged_append   rotary embedding of q and k by each token's own position, k and v into their slots
#include "common.cuh"
#include "vec8.cuh"
#include "per_device.h"
#include "api.h"

namespace oa {

// ------------------------------------------------------------------------------------------------ plan
constexpr int PLAN_THREADS = 256;
constexpr int PLAN_MAX_BATCH = 16384;      // two prefix sums of a batch in shared memory: 128 KB

// The last i in [0, n) with a[i] <= x, for a[0] <= x; of equal entries the last, so that requests without anything are passed over.
__device__ __forceinline__ int owner_of(const int* a, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

struct PlanParams {
  const int *cached, *fresh;
  int* tables;
  long long table_stride;
  const int *free_pages, *taken;
  int *starts, *lens, *slots, *positions, *rows, *taken_out, *missing;
  int batch, width, n_free, page_log2, tokens, position0;
};

// pages that hold n tokens, and no more than a table row has room for
__device__ __forceinline__ int pages_of(long long n, const PlanParams& p) {
  return (int)min((n + (1 << p.page_log2) - 1) >> p.page_log2, (long long)p.width);
}

// One launch: every block makes the prefix sums of the whole batch for itself (a few KB that come from L2) and then takes its share of
// tokens and of fresh pages, so no block waits for another.  A token's page comes from the table where the request had it before, and
// from the free stack where it is fresh: nothing that this launch writes is read in it.  The bytes (12 a token) would take less than a
// microsecond; what counts is that it is a single launch.
__global__ void __launch_bounds__(PLAN_THREADS) paged_plan_kernel(const PlanParams p) {
  extern __shared__ int plan_smem[];
  int* s_first = plan_smem;                // [batch] fresh pages of the requests before
  int* s_start = plan_smem + p.batch;      // [batch] new tokens of the requests before
  __shared__ int s_sum[2][PLAN_THREADS / 32], s_got[PLAN_THREADS / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int per = (p.batch + PLAN_THREADS - 1) / PLAN_THREADS;
  const int b0 = min(tid * per, p.batch), b1 = min(b0 + per, p.batch);
  int pages = 0, tokens = 0;
  for (int b = b0; b < b1; ++b) {
    const int c = max(p.cached[b], 0), f = max(p.fresh[b], 0);
    const int need = max(pages_of((long long)c + f, p) - pages_of(c, p), 0);
    s_first[b] = pages;                    // within this thread's requests so far
    s_start[b] = tokens;
    pages += need;
    tokens += f;
  }
  int ip = pages, it = tokens;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, ip, o), c = __shfl_up_sync(0xffffffffu, it, o);
    if (lane >= o) { ip += a; it += c; }
  }
  if (lane == 31) { s_sum[0][warp] = ip; s_sum[1][warp] = it; }
  __syncthreads();
  int before_p = ip - pages, before_t = it - tokens, total_p = 0, total_t = 0;
#pragma unroll
  for (int w = 0; w < PLAN_THREADS / 32; ++w) {
    if (w < warp) { before_p += s_sum[0][w]; before_t += s_sum[1][w]; }
    total_p += s_sum[0][w];
    total_t += s_sum[1][w];
  }
  for (int b = b0; b < b1; ++b) { s_first[b] += before_p; s_start[b] += before_t; }
  __syncthreads();
  const int taken = min(max(*p.taken, 0), p.n_free);
  const int page = 1 << p.page_log2;

  if (blockIdx.x == 0) {                   // what there is one of for each request
    int lost = 0;
    for (int b = tid; b < p.batch; b += PLAN_THREADS) {
      const int c = max(p.cached[b], 0), f = max(p.fresh[b], 0);
      const int old = pages_of(c, p), need = max(pages_of((long long)c + f, p) - old, 0);
      const int have = min(max(p.n_free - taken - s_first[b], 0), need);
      lost += f - (int)min((long long)f, max(((long long)(old + have) << p.page_log2) - c, 0ll));
      const int on = (int)min((long long)f, ((long long)old << p.page_log2) - c);      // go to the page that is begun, which may not be there either
      if (on > 0 && p.tables[b * p.table_stride + old - 1] < 0) lost += on;
      p.starts[b] = s_start[b];
      p.lens[b] = (int)min((long long)c + f, (long long)p.width << p.page_log2);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) lost += __shfl_xor_sync(0xffffffffu, lost, o);
    if (lane == 0) s_got[warp] = lost;
    __syncthreads();
    if (tid == 0) {
      int sum = 0;
      for (int w = 0; w < PLAN_THREADS / 32; ++w) sum += s_got[w];
      p.starts[p.batch] = total_t;
      *p.taken_out = min(taken + total_p, p.n_free);
      *p.missing = sum + max(total_t - p.tokens, 0);
    }
  }
  const int step = gridDim.x * PLAN_THREADS;
  for (int t = blockIdx.x * PLAN_THREADS + tid; t < p.tokens; t += step) {
    int slot = -1, pos = -1, row = -1;
    if (t < total_t) {
      row = owner_of(s_start, p.batch, t);
      const int c = max(p.cached[row], 0);
      const long long at = (long long)c + t - s_start[row];
      const long long j = at >> p.page_log2;
      pos = (int)(at + p.position0);
      if (j < p.width) {
        const int old = pages_of(c, p);
        const long long k = (long long)taken + s_first[row] + j - old;
        const int id = j < old ? p.tables[row * p.table_stride + j] : k < p.n_free ? p.free_pages[k] : -1;
        if (id >= 0) slot = (id << p.page_log2) + (int)(at & (page - 1));
      }
    }
    p.slots[t] = slot;
    p.positions[t] = pos;
    p.rows[t] = row;
  }
  for (int i = blockIdx.x * PLAN_THREADS + tid; i < total_p; i += step) {
    const int b = owner_of(s_first, p.batch, i);
    const int j = pages_of(max(p.cached[b], 0), p) + i - s_first[b];
    const long long k = (long long)taken + i;
    p.tables[b * p.table_stride + j] = k < p.n_free ? p.free_pages[k] : -1;
  }
}

// ------------------------------------------------------------------------------------------------ release
// Pages of the requests marked done, in request order, onto the stack below `taken`; their lengths become 0 and their table entries -1.  One
// block: requests end seldom and few at a time.  Entries that are no page (the stack had run out) are left out.
__global__ void __launch_bounds__(256) paged_release_kernel(const uint8_t* __restrict__ done, int* lens, int* tables, long long table_stride, int* free_pages,
                                                            int n_free, const int* __restrict__ taken_in, int* taken_out, int batch, int width,
                                                            int page_log2) {
  __shared__ int s_count[8];
  __shared__ int s_top;
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) s_top = min(max(*taken_in, 0), n_free);
  __syncthreads();
  for (int b0 = 0; b0 < batch; b0 += 8) {                  // eight requests at a time, a warp for each
    const int b = b0 + warp;
    const bool mine = b < batch && done[b];
    const int n = mine ? (int)min(((long long)max(lens[b], 0) + (1 << page_log2) - 1) >> page_log2, (long long)width) : 0;
    int count = 0;
    for (int j0 = 0; j0 < n; j0 += 32)
      count += __popc(__ballot_sync(0xffffffffu, j0 + lane < n && tables[b * table_stride + min(j0 + lane, n - 1)] >= 0));
    if (lane == 0) s_count[warp] = count;
    __syncthreads();
    int at = s_top, all = 0;
    for (int w = 0; w < 8; ++w) { if (w <= warp) at -= s_count[w]; all += s_count[w]; }
    for (int j0 = 0; j0 < n; j0 += 32) {
      const bool in = j0 + lane < n;
      const int id = in ? tables[b * table_stride + j0 + lane] : -1;
      const unsigned live = __ballot_sync(0xffffffffu, id >= 0);
      const int to = at + __popc(live & ((1u << lane) - 1));
      if (id >= 0 && to >= 0) free_pages[to] = id;
      if (in) tables[b * table_stride + j0 + lane] = -1;
      at += __popc(live);
    }
    if (mine && lane == 0) lens[b] = 0;
    __syncthreads();
    if (threadIdx.x == 0) s_top = max(s_top - all, 0);
    __syncthreads();
  }
  if (threadIdx.x == 0) *taken_out = s_top;
}

// ------------------------------------------------------------------------------------------------ append
constexpr int APPEND_MAX_HALF = 64;
struct AppendParams {
  const void* x;                           // [tokens, row_stride]: q heads, k heads, v heads
  long long row_stride;
  void* q_out;                             // [tokens, q_heads * head_dim]
  void *k_pages, *v_pages;
  long long k_page_stride, v_page_stride;  // elements
  const int *positions, *slots;
  int tokens, q_heads, kv_heads, half, page_log2, pages, rotate;
  double turns[APPEND_MAX_HALF];           // turns a position: theta^(-j / half) / (2 pi)
};

// A token's angles are worked out once for all its heads: position * turns in 64 bits (in 32 bits a position of 131072 leaves an angle
// 0.008 off), the whole turns taken off, and what is left in [-1/2, 1/2] turns in 32 bits.  Reads the packed rows once and writes q, k and v
// once: bound by those bytes.  A thread's first two pieces are on their way before the angles are worked out.
template <typename T>
__global__ void __launch_bounds__(256) paged_append_kernel(const __grid_constant__ AppendParams p) {
  __shared__ float s_cos[APPEND_MAX_HALF], s_sin[APPEND_MAX_HALF];
  pdl_launch_dependents();
  pdl_wait();
  const int t = blockIdx.x, hd = 2 * p.half;
  const T* row = static_cast<const T*>(p.x) + t * p.row_stride;
  const int jv = p.half >> 3, heads = p.q_heads + 2 * p.kv_heads;
  const int n = heads * jv, stride = gridDim.y * blockDim.x;
  int i = blockIdx.y * blockDim.x + threadIdx.x;
  Vec8<T> a[2], b[2];
  const auto fetch = [&] {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int at = i + q * stride, head = at / jv, j = (at - head * jv) * 8;
      if (at < n) {
        a[q] = *reinterpret_cast<const Vec8<T>*>(row + (long long)head * hd + j);
        b[q] = *reinterpret_cast<const Vec8<T>*>(row + (long long)head * hd + j + p.half);
      }
    }
  };
  const int slot = p.slots[t], position = p.positions[t];
  fetch();
  for (int k = threadIdx.x; k < p.half; k += blockDim.x) {
    const double x = (double)position * p.turns[k];
    sincospif((float)(2.0 * (x - rint(x))), &s_sin[k], &s_cos[k]);
  }
  __syncthreads();
  const bool there = slot >= 0 && (slot >> p.page_log2) < p.pages;
  const long long page = slot >> p.page_log2, off = slot & ((1 << p.page_log2) - 1);
  while (i < n) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int at = i + q * stride, head = at / jv, j = (at - head * jv) * 8;
      if (at >= n) continue;
      if (p.rotate && head < p.q_heads + p.kv_heads) {
        float x[8], y[8], lo[8], hi[8];
        a[q].get(x);
        b[q].get(y);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float c = s_cos[j + k], s = s_sin[j + k];
          lo[k] = x[k] * c - y[k] * s;
          hi[k] = y[k] * c + x[k] * s;
        }
        a[q].set(lo);
        b[q].set(hi);
      }
      T* to;
      if (head < p.q_heads) {
        to = static_cast<T*>(p.q_out) + ((long long)t * p.q_heads + head) * hd + j;
      } else {
        if (!there) continue;
        const bool is_k = head < p.q_heads + p.kv_heads;
        const int h = head - p.q_heads - (is_k ? 0 : p.kv_heads);
        to = static_cast<T*>(is_k ? p.k_pages : p.v_pages) + page * (is_k ? p.k_page_stride : p.v_page_stride) +
             (((long long)h << p.page_log2) + off) * hd + j;
      }
      *reinterpret_cast<Vec8<T>*>(to) = a[q];
      *reinterpret_cast<Vec8<T>*>(to + p.half) = b[q];
    }
    i += 2 * stride;
    fetch();
  }
}

static int log2_of_page(int page_size) {
  for (int l = 4; l <= 7; ++l)
    if (page_size == 1 << l) return l;
  return -1;
}

}  // namespace oa

using namespace oa;

extern "C" int oa_paged_plan(const int* cached, const int* fresh, int* tables, long long table_stride, const int* free_pages, const int* taken,
                             int* starts, int* lens, int* slots, int* positions, int* rows, int* taken_out, int* missing, int batch, int width,
                             int n_free, int page_size, int tokens, int position0, void* stream) {
  const int lg = log2_of_page(page_size);
  if (lg < 0) return OA_ERR_UNSUPPORTED;
  if (batch < 0 || width < 0 || n_free < 0 || tokens < 0 || table_stride < width) return OA_ERR_ARG;
  if (batch > PLAN_MAX_BATCH) return OA_ERR_TOO_LARGE;
  const int smem = 2 * batch * (int)sizeof(int);
  if (smem > 48 * 1024 &&
      cudaFuncSetAttribute(paged_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * PLAN_MAX_BATCH * (int)sizeof(int)) != cudaSuccess)
    return OA_ERR_LAUNCH;
  const PlanParams p{cached, fresh, tables, table_stride, free_pages, taken, starts, lens, slots, positions, rows, taken_out, missing,
                     batch, width, n_free, lg, tokens, position0};
  const int work = tokens > batch ? tokens : batch;
  const int blocks = (work + 4 * PLAN_THREADS - 1) / (4 * PLAN_THREADS), most = 4 * sm_count();
  launch_short(paged_plan_kernel, dim3(blocks < 1 ? 1 : blocks > most ? most : blocks), dim3(PLAN_THREADS), smem, (cudaStream_t)stream, p);
  return cudaGetLastError() == cudaSuccess ? OA_OK : OA_ERR_LAUNCH;
}

extern "C" int oa_paged_release(const void* done, int* lens, int* tables, long long table_stride, int* free_pages, int n_free, const int* taken,
                                int* taken_out, int batch, int width, int page_size, void* stream) {
  const int lg = log2_of_page(page_size);
  if (lg < 0) return OA_ERR_UNSUPPORTED;
  if (batch < 0 || width < 0 || n_free < 0 || table_stride < width) return OA_ERR_ARG;
  launch_short(paged_release_kernel, dim3(1), dim3(256), 0, (cudaStream_t)stream, (const uint8_t*)done, lens, tables, table_stride, free_pages, n_free,
               taken, taken_out, batch, width, lg);
  return cudaGetLastError() == cudaSuccess ? OA_OK : OA_ERR_LAUNCH;
}

extern "C" int oa_paged_append(int dtype, const void* x, long long row_stride, void* q_out, void* k_pages, void* v_pages, long long k_page_stride,
                               long long v_page_stride, const int* positions, const int* slots, const void* turns, int tokens, int q_heads,
                               int kv_heads, int head_dim, int page_size, int pages, void* stream) {
  const int lg = log2_of_page(page_size), half = head_dim / 2;
  if (lg < 0 || head_dim < 16 || head_dim % 16 || half > APPEND_MAX_HALF || (dtype != OA_F32 && dtype != OA_BF16)) return OA_ERR_UNSUPPORTED;
  if (tokens < 0 || q_heads < 1 || kv_heads < 1 || pages < 0 || (long long)pages << lg > 0x7fffffffll) return OA_ERR_ARG;
  const int unit = dtype == OA_F32 ? 4 : 8;                  // elements of 16 bytes
  if (row_stride % unit || k_page_stride % unit || v_page_stride % unit ||
      ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(q_out) | reinterpret_cast<uintptr_t>(k_pages) | reinterpret_cast<uintptr_t>(v_pages)) & 15))
    return OA_ERR_ALIGN;
  if (tokens == 0) return OA_OK;
  AppendParams p{x, row_stride, q_out, k_pages, v_pages, k_page_stride, v_page_stride, positions, slots, tokens, q_heads, kv_heads, half, lg, pages,
                 turns != nullptr, {}};
  if (turns)
    for (int j = 0; j < half; ++j) p.turns[j] = static_cast<const double*>(turns)[j];
  // A row's pieces over several blocks while the tokens alone leave SMs idle, one to a thread; otherwise two, so that no thread is without (16381 rows
  // of 80 heads of 64: 53 us, 6.3 TB/s; 68 with 256 threads whose fetches wait for the angles).
  const int n = (q_heads + 2 * kv_heads) * (half / 8), want = (n + 255) / 256, spread = (2 * sm_count() + tokens - 1) / tokens, per = spread < want ? (n + spread - 1) / spread : n;
  const dim3 grid((unsigned)tokens, (unsigned)(spread < want ? spread : want));
  const int pieces = spread < want ? (per + 511) / 512 * 2 : 1, threads = pieces == 1 ? 256 : ((per + pieces - 1) / pieces + 31) / 32 * 32;
  if (dtype == OA_F32) launch_short(paged_append_kernel<float>, grid, dim3((unsigned)threads), 0, (cudaStream_t)stream, p);
  else launch_short(paged_append_kernel<__nv_bfloat16>, grid, dim3((unsigned)threads), 0, (cudaStream_t)stream, p);
  return cudaGetLastError() == cudaSuccess ? OA_OK : OA_ERR_LAUNCH;
}
