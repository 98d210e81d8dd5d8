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


// ------------------------------------------------------------------------------------------------ bf16 on the tensor cores
// A tile of queries is 128 rows, the group of query heads that share a key-value head times `tpt` tokens (row = token * group + head), and
// a tile of keys is 128 keys, one to eight pages.  An item is the work of one query tile on one key-value head:
//   shared form   the prompt is read once for the whole batch: its items take tokens of the batch as they come, whatever request they
//                 belong to, and each request's own keys make items of their own; every row then has two partial results or more;
//   joint form    where a request's new tokens fill a tile themselves (or there is no prompt) an item sees the prompt's keys and then its own.
// The key tiles of all items, one after the other, are cut into as many equal stretches as there are CTAs, so that a long prompt for few
// requests and short histories for many fill the chip alike.  The part of an item in one stretch is a segment.  Segments that are not a
// whole result leave (o, m, l) in fp32 in scratch, a second launch joins them.  Where everything goes follows from prefix sums over the
// batch that each CTA makes for itself; CTA 0 leaves them for the second launch.
//
// Inside a CTA, segments run through one pipeline of tiles, g = 0, 1, ..:  warp 9 loads Q (two buffers), K and V by TMA, a box for each
// page;  warp 8 issues S[g & 1] = Q K_g^T two tiles ahead of O[segment & 1] += P_g V_g, P taken from TMEM;  warps 0-7 are the softmax, two
// threads to a row.  Warps all of whose rows are empty only keep step: a request's single token fills 8 of 128 rows with 8 heads to a group,
// and its key tiles then cost what they take to arrive.
// Keys beyond a length are cut off from the scores by a select, and their values are overwritten by zeros before the product: what lies there
// (the rest of a page, or of the ring) may be anything, NaN included.
// The product P_g V_g has a barrier for even and one for odd tiles: the scores of tile g + 1 do not wait for it, so that a reader may be two
// products ahead of one barrier's phase.
constexpr int PA_M = 128, PA_N = 128, PA_THREADS = 320, PA_MAX_BATCH = 2048;
constexpr float PA_RESCALE = 8.f;          // log2: the running maximum is let be while rows grow by less

template <int HD> struct PaCfg {
  static constexpr int NK = HD == 64 ? 4 : 2, NV = HD == 64 ? 4 : 2;
  static constexpr int Q_BYTES = PA_M * HD * 2, T_BYTES = PA_N * HD * 2;
  static constexpr int OFF_Q = 0, OFF_K = 2 * Q_BYTES, OFF_V = OFF_K + NK * T_BYTES, OFF_X = OFF_V + NV * T_BYTES;
  static constexpr int OFF_BAR = OFF_X + 3 * 2 * PA_M * 4, OFF_SCAN = OFF_BAR + 512;
  static constexpr int SMEM_BYTES = OFF_SCAN + 2 * (PA_MAX_BATCH + 1) * 4;
  static constexpr int TM_S = 0, TM_O = 256;
};

struct PagedTcParams {
  PagedAttnParams a;
  int group, tpt, ts;                      // query heads to a key-value head, tokens in a tile, tokens in an own item's box
  int joint, prefix_tiles, prefix_row_tiles, prefix_work;   // prefix_work: key tiles of all prompt items (shared form)
  float* part;                             // partial o: [prompt slots][128][HD], then [own slots][ts * group][HD]
  float2* ml;                              // their (m, l), m in units of log2
  int* sums;                               // per, tiles before a request [batch + 1], query tiles before a request [batch + 1]
  long long own_slot0, part_rows;          // rows of the prompt's slots, rows in all
  int* status;
};

struct Request {
  int t0, n, fresh, own, row_tiles;        // first token, new tokens, those of them that count, own keys, query tiles
};
__device__ __forceinline__ Request request_of(const PagedTcParams& p, int b) {
  Request r;
  r.t0 = p.a.starts[b];
  r.n = max(p.a.starts[b + 1] - r.t0, 0);
  r.fresh = max(min(min(r.n, p.a.max_fresh), p.a.tokens - max(r.t0, 0)), 0);
  r.own = max(min(p.a.lens[b], p.a.width << p.a.page_log2), 0);
  r.row_tiles = (r.fresh + p.tpt - 1) / p.tpt;
  return r;
}
// keys of its own that some row of query tile rt sees
__device__ __forceinline__ int seen_by(const PagedTcParams& p, const Request& r, int rt) {
  return max(r.own - r.n + min(r.fresh, (rt + 1) * p.tpt), 0);
}
// key tiles of the item: with none at all an item of the joint form takes an empty one, which gives the rows their zeros
__device__ __forceinline__ int tiles_of(const PagedTcParams& p, const Request& r, int rt) {
  const int own = (seen_by(p, r, rt) + PA_N - 1) / PA_N;
  return p.joint ? max(p.prefix_tiles + own, 1) : own;
}

struct Segment {
  int prompt, h, b, rt;                    // of the prompt's items: rt counts tiles of the whole batch
  int tile, tiles;                         // first key tile inside the item, how many
  int item, item_tiles;
  int t0, tokens, n, own, seen, i0;        // first token and how many; own items: see Request, i0 = index of the first token in the request
};

// The segments of a stretch [pos, end) of all key tiles, in order.
struct Walk {
  const PagedTcParams& p;
  const int *tiles_before, *items_before;
  int pos, end;
  int b, h, rt, tile;                      // own items: the next one and the tile in it
  Request r;
  bool placed;
  __device__ __forceinline__ Walk(const PagedTcParams& p_, const int* tb, const int* ib, int pos_, int end_)
      : p(p_), tiles_before(tb), items_before(ib), pos(pos_), end(end_), b(0), h(0), rt(0), tile(0), placed(false) {}
  __device__ __forceinline__ void place() {
    const int u = pos - p.prefix_work;
    int lo = 0, n = p.a.batch;             // the last request whose tiles begin at or before u
    const int per_head = u / p.a.kv_heads;
    while (n > 1) {
      const int half = n >> 1;
      if (tiles_before[lo + half] <= per_head) { lo += half; n -= half; } else n = half;
    }
    b = lo;
    r = request_of(p, b);
    const int all = max(tiles_before[b + 1] - tiles_before[b], 1);
    int off = u - tiles_before[b] * p.a.kv_heads;
    h = off / all;
    off -= h * all;
    rt = 0;
    for (int t = tiles_of(p, r, 0); off >= t && rt + 1 < r.row_tiles; t = tiles_of(p, r, rt)) { off -= t; ++rt; }
    tile = off;
    placed = true;
  }
  __device__ __forceinline__ bool next(Segment& s) {
    if (pos >= end) return false;
    if (pos < p.prefix_work) {
      s.prompt = 1;
      s.item = pos / p.prefix_tiles;
      s.tile = pos - s.item * p.prefix_tiles;
      s.item_tiles = p.prefix_tiles;
      s.h = s.item / p.prefix_row_tiles;
      s.rt = s.item - s.h * p.prefix_row_tiles;
      s.t0 = s.rt * p.tpt;
      s.tokens = min(p.tpt, p.a.tokens - s.t0);
      s.b = s.n = s.own = s.seen = s.i0 = 0;
    } else {
      if (!placed) place();
      while (tiles_of(p, r, rt) <= tile || rt >= r.row_tiles) {      // on to the next item that has tiles; there is one before `end`
        tile = 0;
        if (++rt >= r.row_tiles) {
          rt = 0;
          if (++h >= p.a.kv_heads || r.row_tiles == 0) {
            h = 0;
            if (++b >= p.a.batch) return false;
            r = request_of(p, b);
          }
        }
      }
      s.prompt = 0;
      s.h = h;
      s.b = b;
      s.rt = rt;
      s.tile = tile;
      s.item_tiles = tiles_of(p, r, rt);
      s.item = items_before[b] * p.a.kv_heads + h * r.row_tiles + rt;
      s.i0 = rt * p.tpt;
      s.t0 = r.t0 + s.i0;
      s.tokens = min(p.tpt, r.fresh - s.i0);
      s.n = r.n;
      s.own = r.own;
      s.seen = seen_by(p, r, rt);
    }
    s.tiles = min(s.item_tiles - s.tile, end - pos);
    pos += s.tiles;
    if (!s.prompt) tile += s.tiles;
    return true;
  }
};

// Keys of key tile j of a segment's item: how many there are and where in their table they begin.
struct KeyTile { int prompt, first, count; };
__device__ __forceinline__ KeyTile key_tile(const PagedTcParams& p, const Segment& s, int j) {
  KeyTile k;
  k.prompt = s.prompt || (p.joint && j < p.prefix_tiles);
  k.first = (k.prompt || !p.joint ? j : j - p.prefix_tiles) * PA_N;
  k.count = max(min(PA_N, (k.prompt ? p.a.prefix_len : s.seen) - k.first), 0);
  return k;
}

// Prefix sums over the batch (a block of `threads`): key tiles for one key-value head, and query tiles, before each request.  Returns the tiles
// of all.
__device__ __forceinline__ int scan_batch(const PagedTcParams& p, int* tiles_before, int* items_before, int* warp_sums, int threads) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = threads >> 5;
  const int per = (p.a.batch + threads - 1) / threads, b0 = min(tid * per, p.a.batch), b1 = min(b0 + per, p.a.batch);
  int tiles = 0, items = 0;
  for (int b = b0; b < b1; ++b) {
    const Request r = request_of(p, b);
    tiles_before[b] = tiles;
    items_before[b] = items;
    for (int rt = 0; rt < r.row_tiles; ++rt) tiles += tiles_of(p, r, rt);
    items += r.row_tiles;
  }
  int it = tiles, ii = items;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, it, o), y = __shfl_up_sync(0xffffffffu, ii, o);
    if (lane >= o) { it += x; ii += y; }
  }
  if (lane == 31) { warp_sums[2 * warp] = it; warp_sums[2 * warp + 1] = ii; }
  __syncthreads();
  int bt = it - tiles, bi = ii - items, all_t = 0, all_i = 0;
  for (int w = 0; w < warps; ++w) {
    if (w < warp) { bt += warp_sums[2 * w]; bi += warp_sums[2 * w + 1]; }
    all_t += warp_sums[2 * w];
    all_i += warp_sums[2 * w + 1];
  }
  for (int b = b0; b < b1; ++b) { tiles_before[b] += bt; items_before[b] += bi; }
  if (tid == 0) { tiles_before[p.a.batch] = all_t; items_before[p.a.batch] = all_i; }
  return all_t;
}

// Where a partial result goes.  Shared form: every segment of every item, numbered by item + CTA (a segment begins where an item or a
// stretch does).  Joint form: only items that a stretch's end cuts, of which a CTA has its first and its last segment.
__device__ __forceinline__ long long partial_row(const PagedTcParams& p, const Segment& s, int cta, bool first) {
  if (s.prompt) return (long long)(s.item + cta) * PA_M;
  return p.own_slot0 + (p.joint ? 2ll * cta + (first ? 0 : 1) : (long long)s.item + cta) * (p.ts * p.group);
}
// Starts that do not rise would make more items than there is room for: their rows stay out of the scratch.
__device__ __forceinline__ bool has_room(const PagedTcParams& p, long long row) { return row >= 0 && row < p.part_rows; }

__device__ __forceinline__ void softmax_pair_sync(int quad) { asm volatile("bar.sync %0, 64;" ::"r"(quad + 1) : "memory"); }

template <int HD>
__global__ void __launch_bounds__(PA_THREADS, 1)
paged_attn_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmQown, const __grid_constant__ CUtensorMap tmK,
                     const __grid_constant__ CUtensorMap tmV, const __grid_constant__ PagedTcParams p) {
  using Cfg = PaCfg<HD>;
  constexpr int NK = Cfg::NK, NV = Cfg::NV, CHUNKS = HD / 64;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ int s_warp_sums[2 * PA_THREADS / 32];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::OFF_BAR);
  uint64_t *q_full = bars, *q_empty = bars + 2, *k_full = bars + 4, *k_empty = k_full + NK, *v_full = k_empty + NK, *v_empty = v_full + NV;
  uint64_t *s_full = v_empty + NV, *p_full = s_full + 2, *o_done = s_full + 4, *o_free = s_full + 6;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(s_full + 8);
  int* tiles_before = reinterpret_cast<int*>(smem + Cfg::OFF_SCAN);
  int* items_before = tiles_before + p.a.batch + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_launch_dependents();
  if ((smem_u32(smem) & 1023u) != 0) {
    if (threadIdx.x == 0) report_error(p.status, OA_KERR_BAD_ARG);
    return;
  }
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmQ); tma_prefetch_desc(&tmQown); tma_prefetch_desc(&tmK); tma_prefetch_desc(&tmV);
    for (int i = 0; i < 2; ++i) { mbar_init(&q_full[i], 1); mbar_init(&q_empty[i], 1); mbar_init(&s_full[i], 1); mbar_init(&p_full[i], 8); mbar_init(&o_done[i], 1); mbar_init(&o_free[i], 8); }
    for (int i = 0; i < NK; ++i) { mbar_init(&k_full[i], 1); mbar_init(&k_empty[i], 1); }
    for (int i = 0; i < NV; ++i) { mbar_init(&v_full[i], 1); mbar_init(&v_empty[i], 1); }
    mbar_fence_init();
  }
  if (warp == 8) { tmem_alloc<512>(tmem_slot); tmem_relinquish(); }
  pdl_wait();
  const int own_tiles = scan_batch(p, tiles_before, items_before, s_warp_sums, PA_THREADS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int work = p.prefix_work + own_tiles * p.a.kv_heads, per = max((work + (int)gridDim.x - 1) / (int)gridDim.x, 1);
  if (blockIdx.x == 0) {                   // for the second launch
    if (threadIdx.x == 0) { p.sums[0] = per; p.sums[1] = work; }
    for (int b = threadIdx.x; b <= p.a.batch; b += PA_THREADS) { p.sums[2 + b] = tiles_before[b]; p.sums[3 + p.a.batch + b] = items_before[b]; }
  }
  const long long begin = (long long)blockIdx.x * per;
  const int lo = (int)min(begin, (long long)work), hi = (int)min(begin + per, (long long)work);
  Walk walk(p, tiles_before, items_before, lo, hi);
  Segment s;

  if (warp == 9) {
    // ---------------------------------------------------------------- loads.  Lane i fetches the page that holds the tile's keys from i * page_size on.
    const int ps = 1 << p.a.page_log2;
    int g = 0, sq = 0;
    bool ok = true;
    int id1 = -1, h1 = 0, n1 = -1, id2 = -1, h2 = 0, n2 = -1;    // page, head and pages of the tiles one and two before (their values are still to come)
    const auto load = [&](uint8_t* to, const CUtensorMap* m, uint64_t* bar, int id, int h, int boxes) {
      if (elect_one()) mbar_expect_tx(bar, (uint32_t)(boxes * ps * HD * 2));
      __syncwarp();
      if (lane < boxes) {
#pragma unroll
        for (int x = 0; x < CHUNKS; ++x) tma_load_3d(to + x * (PA_N * 128) + lane * ps * 128, m, bar, x * 64, h << p.a.page_log2, id);
      }
      __syncwarp();
    };
    const auto load_v = [&](int gv, int id, int h, int boxes) {
      const int st = gv % NV;
      if (!warp_wait(&v_empty[st], ((gv / NV) & 1) ^ 1)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_EMPTY); return false; }
      load(smem + Cfg::OFF_V + st * Cfg::T_BYTES, &tmV, &v_full[st], id, h, boxes);
      return true;
    };
    while (ok && walk.next(s)) {
      const int qb = sq & 1;
      ok = warp_wait(&q_empty[qb], ((sq >> 1) & 1) ^ 1);
      if (!ok) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_EMPTY); break; }
      if (elect_one()) {
        const int tokens = s.prompt ? p.tpt : p.ts;
        mbar_expect_tx(&q_full[qb], (uint32_t)(tokens * p.group * HD * 2));
#pragma unroll
        for (int x = 0; x < CHUNKS; ++x)
          tma_load_3d(smem + Cfg::OFF_Q + qb * Cfg::Q_BYTES + x * (PA_M * 128), s.prompt ? &tmQ : &tmQown, &q_full[qb], x * 64, s.h * p.group, s.t0);
      }
      __syncwarp();
      for (int j = 0; j < s.tiles && ok; ++j, ++g) {
        const KeyTile kt = key_tile(p, s, s.tile + j);
        const int boxes = (kt.count + ps - 1) >> p.a.page_log2;
        int id = -1;
        if (lane < boxes) {
          const int at = (kt.first >> p.a.page_log2) + lane;
          id = kt.prompt ? p.a.prefix_table[at] : p.a.tables[s.b * p.a.table_stride + at];
        }
        const int st = g % NK;
        ok = warp_wait(&k_empty[st], ((g / NK) & 1) ^ 1);
        if (!ok) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_EMPTY); break; }
        load(smem + Cfg::OFF_K + st * Cfg::T_BYTES, &tmK, &k_full[st], id, s.h, boxes);
        if (n2 >= 0) ok = load_v(g - 2, id2, h2, n2);
        id2 = id1; h2 = h1; n2 = n1;
        id1 = id; h1 = s.h; n1 = boxes;
      }
      ++sq;
    }
    if (ok && n2 >= 0) ok = load_v(g - 2, id2, h2, n2);
    if (ok && n1 >= 0) load_v(g - 1, id1, h1, n1);
  } else if (warp == 8) {
    // ---------------------------------------------------------------- products
    constexpr uint32_t idesc_qk = umma_idesc_bf16(PA_M, PA_N, 0, 0), idesc_pv = umma_idesc_bf16(PA_M, HD, 0, 1);
    const uint64_t q_desc = umma_smem_desc_sw128(smem_u32(smem + Cfg::OFF_Q), 16, 1024), k_desc = umma_smem_desc_sw128(smem_u32(smem + Cfg::OFF_K), 16, 1024);
    const uint64_t v_desc = umma_smem_desc_sw128(smem_u32(smem + Cfg::OFF_V), PA_N * 128, 1024);
    Walk ahead(p, tiles_before, items_before, lo, hi);           // of the score products, two tiles ahead
    Segment sa;
    int ja = 0, na = 0, sqa = -1, ga = 0;
    const auto issue_qk = [&]() -> bool {                         // the next score product, if there is one
      if (ja == na) {
        if (!ahead.next(sa)) return true;
        ja = 0; na = sa.tiles; ++sqa;
        if (!warp_wait(&q_full[sqa & 1], (sqa >> 1) & 1)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_FULL); return false; }
      }
      const int st = ga % NK;
      if (!warp_wait(&k_full[st], (ga / NK) & 1)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_FULL); return false; }
      tc_fence_after();
      if (elect_one()) {
        const uint64_t qd = q_desc + ((sqa & 1) * Cfg::Q_BYTES >> 4), kd = k_desc + (st * Cfg::T_BYTES >> 4);
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks) {
          const uint32_t off = ((ks >> 2) * (PA_M * 128) + (ks & 3) * 32) >> 4;
          umma_f16(tmem_base + Cfg::TM_S + (ga & 1) * PA_N, qd + off, kd + off, idesc_qk, ks > 0 ? 1u : 0u);
        }
        umma_commit(&k_empty[st]);
        umma_commit(&s_full[ga & 1]);
        if (ja + 1 == na) umma_commit(&q_empty[sqa & 1]);
      }
      __syncwarp();
      ++ja; ++ga;
      return true;
    };
    bool ok = issue_qk();
    if (ok) ok = issue_qk();
    int g = 0, sq = 0;
    while (ok && walk.next(s)) {
      ok = warp_wait(&o_free[sq & 1], ((sq >> 1) & 1) ^ 1);       // the result before the last has been read
      if (!ok) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_TMEM_EMPTY); break; }
      for (int j = 0; j < s.tiles; ++j, ++g) {
        const int st = g % NV;
        ok = warp_wait(&v_full[st], (g / NV) & 1);
        if (!ok) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_FULL); break; }
        ok = warp_wait(&p_full[g & 1], (g >> 1) & 1);
        if (!ok) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_SOFTMAX); break; }
        tc_fence_after();
        if (elect_one()) {
          const uint64_t vd = v_desc + (st * Cfg::T_BYTES >> 4);
#pragma unroll
          for (int ks = 0; ks < PA_N / 16; ++ks)
            umma_f16_ts(tmem_base + Cfg::TM_O + (sq & 1) * HD, tmem_base + Cfg::TM_S + (g & 1) * PA_N + ks * 8, vd + (ks * 2048 >> 4), idesc_pv,
                        (j > 0 || ks > 0) ? 1u : 0u);
          umma_commit(&v_empty[st]);
          umma_commit(&o_done[g & 1]);
        }
        __syncwarp();
        ok = issue_qk();                                          // over S[g & 1] = P_g: behind its product in the pipe
        if (!ok) break;
      }
      ++sq;
    }
  } else {
    // ---------------------------------------------------------------- softmax: warp w has rows 32 (w % 4).., keys 64 (w / 4).. of a tile
    constexpr int OC = HD / 2;
    const int quad = warp & 3, half = warp >> 2, r = quad * 32 + lane;
    const uint32_t t_lane = (uint32_t)(quad * 32) << 16;
    const float sl2 = p.a.scale * 1.4426950408889634f;
    float* xch = reinterpret_cast<float*>(smem + Cfg::OFF_X);
    const int i_row = r / p.group;                                // token of this row in the tile
    int g = 0, sq = 0;
    bool ok = true;
    while (ok && walk.next(s)) {
      const int rows = s.tokens * p.group;
      const bool live = quad * 32 < rows;                         // of this warp: some row is there
      float m_run = -INFINITY, l_run = 0.f;
      const uint32_t o_addr = tmem_base + t_lane + Cfg::TM_O + (sq & 1) * HD + half * OC;
      for (int j = 0; j < s.tiles; ++j, ++g) {
        const KeyTile kt = key_tile(p, s, s.tile + j);
        ok = warp_wait(&s_full[g & 1], (g >> 1) & 1);
        if (!ok) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_TMEM_FULL); break; }
        tc_fence_after();
        if (live) {
          const uint32_t s_addr = tmem_base + t_lane + Cfg::TM_S + (g & 1) * PA_N;
          uint32_t sv[64];
          tmem_ld32(s_addr + half * 64, sv);
          tmem_ld32(s_addr + half * 64 + 32, sv + 32);
          tmem_ld_wait();
          // columns up to lim are seen: the keys that there are, and of a request's own keys those up to the row's token
          const int last = kt.prompt ? kt.count - 1 : min(kt.count - 1, s.own - s.n + s.i0 + i_row - kt.first);
          const int first_last = kt.prompt ? kt.count - 1 : min(kt.count - 1, s.own - s.n + s.i0 - kt.first);
          if (first_last < PA_N - 1) {
            const int lim = last - half * 64;
#pragma unroll
            for (int i = 0; i < 64; ++i) sv[i] = i <= lim ? sv[i] : 0xff800000u;
          }
          float m0 = __uint_as_float(sv[0]), m1 = __uint_as_float(sv[1]), m2 = __uint_as_float(sv[2]), m3 = __uint_as_float(sv[3]);
#pragma unroll
          for (int i = 4; i < 64; i += 4) {
            m0 = fmaxf(m0, __uint_as_float(sv[i])); m1 = fmaxf(m1, __uint_as_float(sv[i + 1]));
            m2 = fmaxf(m2, __uint_as_float(sv[i + 2])); m3 = fmaxf(m3, __uint_as_float(sv[i + 3]));
          }
          float mx = fmaxf(fmaxf(m0, m1), fmaxf(m2, m3));
          float* slots = xch + (g & 1) * (2 * PA_M);
          slots[(half ^ 1) * PA_M + r] = mx;
          softmax_pair_sync(quad);                                // both halves are in registers: P may go over S
          mx = fmaxf(mx, slots[half * PA_M + r]) * sl2;
          const float m_new = fmaxf(m_run, mx);
          const bool grow = (m_new - m_run) > PA_RESCALE;         // the first time: from -inf
          const float m_cand = grow ? m_new : m_run;
          const float m_use = m_cand == -INFINITY ? 0.f : m_cand; // a row that has seen nothing yet
          const float alpha = grow ? fast_exp2(m_run - m_use) : 1.f;
          const float neg_m = -m_use;
          float l0 = 0.f, l1 = 0.f, l2 = 0.f, l3 = 0.f;
          uint32_t pk[32];
#pragma unroll
          for (int i = 0; i < 64; i += 4) {
            const float e0 = fast_exp2(fmaf(__uint_as_float(sv[i]), sl2, neg_m)), e1 = fast_exp2(fmaf(__uint_as_float(sv[i + 1]), sl2, neg_m));
            const float e2 = fast_exp2(fmaf(__uint_as_float(sv[i + 2]), sl2, neg_m)), e3 = fast_exp2(fmaf(__uint_as_float(sv[i + 3]), sl2, neg_m));
            l0 += e0; l1 += e1; l2 += e2; l3 += e3;
            pk[i >> 1] = pack_bf16x2(e0, e1);                     // weights to bf16, as the tensor cores take them; their sum stays fp32
            pk[(i >> 1) + 1] = pack_bf16x2(e2, e3);
          }
          tmem_st32(s_addr + half * 32, pk);
          l_run = l_run * alpha + ((l0 + l1) + (l2 + l3));
          m_run = m_cand;
          if (j > 0 && __any_sync(0xffffffffu, grow)) {           // O again to the new maximum, behind the product before
            ok = warp_wait(&o_done[(g - 1) & 1], ((g - 1) >> 1) & 1);
            if (!ok) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_TMEM_FULL); break; }
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < OC / 32; ++c) {
              uint32_t o[32];
              tmem_ld32(o_addr + c * 32, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              tmem_st32(o_addr + c * 32, o);
            }
          }
          tmem_st_wait();
          tc_fence_before();
        }
        if (kt.count < PA_N) {                                    // values that no key goes with: zeros, whatever lies there
          const int st = g % NV;
          ok = warp_wait(&v_full[st], (g / NV) & 1);
          if (!ok) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_FULL); break; }
          const uint32_t base = smem_u32(smem + Cfg::OFF_V + st * Cfg::T_BYTES);
          for (int i = threadIdx.x; i < (PA_N - kt.count) * CHUNKS * 8; i += 256) {
            const int row = kt.count + i / (CHUNKS * 8), c = i % (CHUNKS * 8);
            st_shared_v4(base + (c >> 3) * (PA_N * 128) + row * 128 + (c & 7) * 16, make_uint4(0, 0, 0, 0));
          }
          fence_proxy_async_smem();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[g & 1]);
      }
      if (!ok) break;
      if (live) {                                                 // the two halves' sums, in slots of their own: the next tile's maxima may come at once
        float* slots = xch + 2 * (2 * PA_M);
        slots[(half ^ 1) * PA_M + r] = l_run;
        softmax_pair_sync(quad);
        l_run += slots[half * PA_M + r];
      }
      ok = warp_wait(&o_done[(g - 1) & 1], ((g - 1) >> 1) & 1);
      if (!ok) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_TMEM_FULL); break; }
      tc_fence_after();
      if (live) {
        uint32_t o[OC];
#pragma unroll
        for (int c = 0; c < OC / 32; ++c) tmem_ld32(o_addr + c * 32, o + c * 32);
        tmem_ld_wait();
        const int r0 = quad * 32 + (lane & ~3);                   // after an exchange among four lanes a lane has 16 bytes of four rows
        if (p.joint && s.tiles == s.item_tiles) {                 // the whole result
          const float inv = l_run > 0.f ? 1.f / l_run : l_run == 0.f ? 0.f : l_run;      // NaN stays NaN
#pragma unroll
          for (int c = 0; c < OC / 32; ++c) {
            uint4 v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float* f = reinterpret_cast<const float*>(o) + c * 32 + k * 8;
              v[k] = make_uint4(pack_bf16x2(f[0] * inv, f[1] * inv), pack_bf16x2(f[2] * inv, f[3] * inv), pack_bf16x2(f[4] * inv, f[5] * inv), pack_bf16x2(f[6] * inv, f[7] * inv));
            }
            exchange4(v, lane);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int row = r0 + k, t = s.t0 + row / p.group;
              if (row < rows && t >= 0 && t < p.a.tokens)
                *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.a.out) + ((long long)t * p.a.q_heads + s.h * p.group + row % p.group) * HD + half * OC +
                                          c * 32 + (lane & 3) * 8) = v[k];
            }
          }
          const int t = s.t0 + i_row;
          if (p.a.lse && half == 0 && r < rows && t >= 0 && t < p.a.tokens)
            p.a.lse[(long long)t * p.a.q_heads + s.h * p.group + r % p.group] = l_run == 0.f ? -INFINITY : (m_run + log2f(l_run)) * 0.6931471805599453f;
        } else {
          const long long at = partial_row(p, s, blockIdx.x, s.tile > 0 || walk.pos - s.tiles == lo);
#pragma unroll
          for (int c = 0; c < OC / 16; ++c) {
            uint4 v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = make_uint4(o[c * 16 + k * 4], o[c * 16 + k * 4 + 1], o[c * 16 + k * 4 + 2], o[c * 16 + k * 4 + 3]);
            exchange4(v, lane);
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (r0 + k < rows && has_room(p, at + r0 + k)) *reinterpret_cast<uint4*>(p.part + (at + r0 + k) * HD + half * OC + c * 16 + (lane & 3) * 4) = v[k];
          }
          if (half == 0 && r < rows && has_room(p, at + r)) p.ml[at + r] = make_float2(m_run, l_run);
        }
        tc_fence_before();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&o_free[sq & 1]);
      ++sq;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) { tc_fence_after(); tmem_dealloc<512>(tmem_base); }
}

// Joins partial results (acc, m, l) of one row, a warp to a row, a lane to HD / 32 neighbouring columns.
template <int HD>
struct RowJoin {
  static constexpr int PER = HD / 32;
  float m = -INFINITY, l = 0.f, acc[PER] = {};
  __device__ __forceinline__ void add(const PagedTcParams& p, long long row, int lane) {
    if (!has_room(p, row)) return;
    const float2 ml = p.ml[row];
    float v[PER];
    if (PER == 4) *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(p.part + row * HD + lane * PER);
    else *reinterpret_cast<float2*>(v) = *reinterpret_cast<const float2*>(p.part + row * HD + lane * PER);
    if (ml.y == 0.f) return;                                     // a piece of which this row saw nothing
    const float m_new = fmaxf(m, ml.x);
    const float a = m == -INFINITY ? 0.f : fast_exp2(m - m_new), b = ml.x == -INFINITY ? 1.f : fast_exp2(ml.x - m_new);
    l = l * a + ml.y * b;
#pragma unroll
    for (int e = 0; e < PER; ++e) acc[e] = acc[e] * a + v[e] * b;
    m = m_new;
  }
  __device__ __forceinline__ void write(const PagedTcParams& p, int t, int hq, int lane) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    __nv_bfloat16* to = static_cast<__nv_bfloat16*>(p.a.out) + ((long long)t * p.a.q_heads + hq) * HD + lane * PER;
    if (PER == 4) *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[PER - 2] * inv, acc[PER - 1] * inv));
    else *reinterpret_cast<uint32_t*>(to) = pack_bf16x2(acc[0] * inv, acc[1] * inv);
    if (p.a.lse && lane == 0) p.a.lse[(long long)t * p.a.q_heads + hq] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
  }
};

// Shared form: every row from the pieces of its prompt item and of its own item.
template <int HD>
__global__ void __launch_bounds__(256) paged_join_rows_kernel(const __grid_constant__ PagedTcParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= (long long)p.a.tokens * p.a.q_heads) return;
  const int t = (int)(row / p.a.q_heads), hq = (int)(row - (long long)t * p.a.q_heads), h = hq / p.group, head = hq - h * p.group;
  const int per = p.sums[0];
  RowJoin<HD> join;
  int b = 0, i = 0;
  if (find_request(p.a.starts, p.a.batch, t, lane, b, i) && i < p.a.max_fresh) {
    {
      const int rt = t / p.tpt, item = h * p.prefix_row_tiles + rt, a = item * p.prefix_tiles;
      for (int c = a / per; c <= (a + p.prefix_tiles - 1) / per; ++c) join.add(p, (long long)(item + c) * PA_M + (t - rt * p.tpt) * p.group + head, lane);
    }
    const Request r = request_of(p, b);
    const int rt = i / p.tpt, tiles = tiles_of(p, r, rt);
    if (tiles > 0) {
      const int before = p.sums[2 + b], all = p.sums[3 + b] - before;
      int a = p.prefix_work + before * p.a.kv_heads + h * all;
      for (int k = 0; k < rt; ++k) a += tiles_of(p, r, k);
      const int item = p.sums[3 + p.a.batch + b] * p.a.kv_heads + h * r.row_tiles + rt;
      for (int c = a / per; c <= (a + tiles - 1) / per; ++c)
        join.add(p, p.own_slot0 + (long long)(item + c) * (p.ts * p.group) + (i - rt * p.tpt) * p.group + head, lane);
    }
  }
  join.write(p, t, hq, lane);
}

// Joint form: the items that a stretch's end cuts (block c: the one that begins in stretch c and goes beyond it), and zeros for the rows of
// no request.
template <int HD>
__global__ void __launch_bounds__(256) paged_join_cuts_kernel(const __grid_constant__ PagedTcParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, per = p.sums[0], work = p.sums[1];
  const long long cut = (long long)(blockIdx.x + 1) * per;       // the first tile of the next stretch
  if (cut < work) {
    Walk walk(p, p.sums + 2, p.sums + 3 + p.a.batch, (int)cut, work);
    Segment s;
    if (walk.next(s) && s.tile > 0 && s.tile <= per) {           // begins in this stretch (at its very first tile at the earliest)
      const int a = (int)cut - s.tile, last = (a + s.item_tiles - 1) / per;
      for (int r = warp; r < s.tokens * p.group; r += 8) {
        RowJoin<HD> join;
        for (int c = blockIdx.x; c <= last; ++c) {
          const bool first = (long long)c * per >= a;             // the piece is the first of its CTA
          join.add(p, p.own_slot0 + (2ll * c + (first ? 0 : 1)) * (p.ts * p.group) + r, lane);
        }
        const int t = s.t0 + r / p.group;
        if (t >= 0 && t < p.a.tokens) join.write(p, t, s.h * p.group + r % p.group, lane);
      }
    }
  }
  const auto zero = [&](long long from, long long to) {
    for (long long t = max(from, 0ll); t < min(to, (long long)p.a.tokens); ++t)
      for (int hq = warp; hq < p.a.q_heads; hq += 8) RowJoin<HD>().write(p, (int)t, hq, lane);
  };
  for (int b = blockIdx.x; b < p.a.batch; b += gridDim.x) zero((long long)p.a.starts[b] + p.a.max_fresh, p.a.starts[b + 1]);
  const long long behind = p.a.batch > 0 ? max(p.a.starts[p.a.batch], 0) : 0, rest = max((long long)p.a.tokens - behind, 0ll), share = (rest + gridDim.x - 1) / gridDim.x;
  zero(behind + blockIdx.x * share, behind + (blockIdx.x + 1) * share);
  if (blockIdx.x == 0 && p.a.batch > 0) zero(0, p.a.starts[0]);
}

}  // namespace oa

using namespace oa;

// The sizes that follow from a call's arguments: which form, how many items there can be, what they need in scratch.
struct PagedTcPlan {
  int group, tpt, ts, joint, prefix_tiles, prefix_row_tiles, grid;
  long long prompt_rows, own_rows, items;
  size_t o_bytes, ml_bytes, bytes;
};
static int sm_count() {
  static int sms = 0;
  if (sms == 0) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) sms = 0;
  }
  return sms > 0 ? sms : 148;
}
static PagedTcPlan plan_tc(int tokens, int batch, int max_fresh, int q_heads, int kv_heads, int head_dim, int prefix_len) {
  PagedTcPlan c;
  c.group = q_heads / kv_heads;
  c.tpt = PA_M / c.group;
  c.ts = max_fresh < c.tpt ? (max_fresh > 0 ? max_fresh : 1) : c.tpt;
  c.prefix_tiles = (prefix_len + PA_N - 1) / PA_N;
  c.prefix_row_tiles = (tokens + c.tpt - 1) / c.tpt;
  // The prompt for the whole batch at once where that reads it at most half as often as request by request.
  c.joint = prefix_len == 0 || 2ll * c.prefix_row_tiles > batch;
  c.grid = sm_count();
  c.items = ((long long)batch + tokens / c.tpt) * kv_heads;                    // query tiles of single requests, at most
  c.prompt_rows = c.joint ? 0 : ((long long)c.prefix_row_tiles * kv_heads + c.grid) * PA_M;
  c.own_rows = (c.joint ? 2ll * c.grid : c.items + c.grid) * (c.ts * c.group);
  c.o_bytes = (size_t)(c.prompt_rows + c.own_rows) * head_dim * sizeof(float);
  c.ml_bytes = (size_t)(c.prompt_rows + c.own_rows) * sizeof(float2);
  c.bytes = c.o_bytes + c.ml_bytes + (2 * ((size_t)batch + 1) + 2) * sizeof(int);
  return c;
}
// Which calls the tensor-core kernel takes: bf16, head dims of whole 128-byte rows, a batch whose prefix sums fit in shared memory beside the
// rings, a positive scale (the running maximum is taken before the scale).  The others run a block for each row.
static bool takes_tc(int dtype, int tokens, int batch, int q_heads, int kv_heads, int head_dim, int pages, float scale) {
  return dtype == OA_BF16 && (head_dim == 64 || head_dim == 128) && q_heads / kv_heads <= PA_M && batch > 0 && batch <= PA_MAX_BATCH && pages > 0 &&
         scale > 0.f && tokens > 0;
}

extern "C" size_t oa_paged_attn_scratch_bytes(int dtype, int tokens, int batch, int max_fresh, int q_heads, int kv_heads, int head_dim, int pages,
                                              int prefix_len, float scale) {
  if (kv_heads < 1 || q_heads < kv_heads || !takes_tc(dtype, tokens, batch, q_heads, kv_heads, head_dim, pages, scale)) return 0;
  return plan_tc(tokens, batch, max_fresh, q_heads, kv_heads, head_dim, prefix_len).bytes;
}

namespace oa {
int make_tmap_box3_bf16(CUtensorMap* out, const void* ptr, const uint64_t* dims, const uint64_t* strides, const uint32_t* box);
}

template <int HD>
static int launch_tc(const PagedAttnParams& a, void* scratch, int* status, cudaStream_t st) {
  using Cfg = PaCfg<HD>;
  static bool set = false;
  if (!set) {
    if (cudaFuncSetAttribute(paged_attn_tc_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM_BYTES) != cudaSuccess) return OA_ERR_LAUNCH;
    set = true;
  }
  const PagedTcPlan c = plan_tc(a.tokens, a.batch, a.max_fresh, a.q_heads, a.kv_heads, HD, a.prefix_len);
  const int ps = 1 << a.page_log2;
  const long long own_tiles = ((long long)a.width * ps + PA_N - 1) / PA_N;
  const long long work = (c.joint ? 0 : (long long)a.kv_heads * c.prefix_row_tiles * c.prefix_tiles);
  if (work + c.items * (own_tiles + c.prefix_tiles + 1) > 0x7fffffffll) return OA_ERR_TOO_LARGE;
  PagedTcParams p;
  p.a = a;
  p.group = c.group; p.tpt = c.tpt; p.ts = c.ts;
  p.joint = c.joint; p.prefix_tiles = c.prefix_tiles; p.prefix_row_tiles = c.prefix_row_tiles; p.prefix_work = (int)work;
  p.part = static_cast<float*>(scratch);
  p.ml = reinterpret_cast<float2*>(static_cast<char*>(scratch) + c.o_bytes);
  p.sums = reinterpret_cast<int*>(static_cast<char*>(scratch) + c.o_bytes + c.ml_bytes);
  p.own_slot0 = c.prompt_rows;
  p.part_rows = c.prompt_rows + c.own_rows;
  p.status = status;
  CUtensorMap tq, tqo, tk, tv;
  int rc;
  {
    const uint64_t dims[3] = {HD, (uint64_t)a.q_heads, (uint64_t)a.tokens}, strides[2] = {HD * 2, (uint64_t)a.q_stride * 2};
    const uint32_t box[3] = {64, (uint32_t)c.group, (uint32_t)c.tpt}, own[3] = {64, (uint32_t)c.group, (uint32_t)c.ts};
    if ((rc = make_tmap_box3_bf16(&tq, a.q, dims, strides, box)) || (rc = make_tmap_box3_bf16(&tqo, a.q, dims, strides, own))) return rc;
  }
  const uint64_t packed = (uint64_t)a.kv_heads * ps * HD;
  const uint64_t dims[3] = {HD, (uint64_t)a.kv_heads * ps, (uint64_t)a.pages};
  const uint32_t box[3] = {64, (uint32_t)ps, 1};
  const uint64_t ks[2] = {HD * 2, (a.pages > 1 ? (uint64_t)a.k_page_stride : packed) * 2}, vs[2] = {HD * 2, (a.pages > 1 ? (uint64_t)a.v_page_stride : packed) * 2};
  if ((rc = make_tmap_box3_bf16(&tk, a.k, dims, ks, box)) || (rc = make_tmap_box3_bf16(&tv, a.v, dims, vs, box))) return rc;
  launch_short(paged_attn_tc_kernel<HD>, dim3((unsigned)c.grid), dim3(PA_THREADS), Cfg::SMEM_BYTES, st, tq, tqo, tk, tv, p);
  if (c.joint) launch_short(paged_join_cuts_kernel<HD>, dim3((unsigned)c.grid), dim3(256), 0, st, p);
  else launch_short(paged_join_rows_kernel<HD>, dim3((unsigned)(((long long)a.tokens * a.q_heads + 7) / 8)), dim3(256), 0, st, p);
  return cudaGetLastError() == cudaSuccess ? OA_OK : OA_ERR_LAUNCH;
}

extern "C" int oa_paged_attn(int dtype, const void* q, long long q_stride, const void* k_pages, const void* v_pages, long long k_page_stride,
                             long long v_page_stride, const int* tables, long long table_stride, const int* lens, const int* starts, const int* prefix_table,
                             int prefix_len, void* out, float* lse, int tokens, int batch, int max_fresh, int q_heads, int kv_heads, int head_dim,
                             int page_size, int pages, int width, float scale, void* scratch, int* status, void* stream) {
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
  cudaStream_t st = (cudaStream_t)stream;
  if (takes_tc(dtype, tokens, batch, q_heads, kv_heads, head_dim, pages, scale))
    return head_dim == 64 ? launch_tc<64>(p, scratch, status, st) : launch_tc<128>(p, scratch, status, st);
  const dim3 grid((unsigned)tokens, (unsigned)q_heads);
#define OA_ROWS(T, HD) launch_short(paged_attn_rows_kernel<T, HD>, grid, dim3(128), 0, st, p)
  if (dtype == OA_F32) {
    if (head_dim == 32) OA_ROWS(float, 32); else if (head_dim == 64) OA_ROWS(float, 64); else OA_ROWS(float, 128);
  } else {
    if (head_dim == 32) OA_ROWS(__nv_bfloat16, 32); else if (head_dim == 64) OA_ROWS(__nv_bfloat16, 64); else OA_ROWS(__nv_bfloat16, 128);
  }
#undef OA_ROWS
  return cudaGetLastError() == cudaSuccess ? OA_OK : OA_ERR_LAUNCH;
}
