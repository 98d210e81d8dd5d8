// Attention of a batch of requests over a paged key-value cache, behind a prompt that they share.  Query token i of the n new tokens of a
// request sees all `prefix_len` keys of the prompt and the first len - n + i + 1 keys of the request's own pages:
//   o = sum_s softmax_s(scale q . k_s) v_s,   lse = log sum_s exp(scale q . k_s);   a row that sees nothing gives o = 0, lse = -inf.
// A table entry that names no page counts as keys and values of zeros.  Nothing beyond a request's length is read into a result.
#include <type_traits>
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
// A tile of queries is up to 128 rows, the group of query heads that share a key-value head times `tpt` tokens (row = token * group +
// head), and a tile of keys is 128 keys, one to eight pages.  An item is the work of one query tile on one key-value head:
//   shared form   the prompt is read once for the whole batch: its items take tokens of the batch as they come, whatever request they
//                 belong to, and each request's own keys make items of their own; every row then has two partial results or more;
//   joint form    where a request's new tokens fill a tile themselves (or there is no prompt) an item sees the prompt's keys and then its own.
// The key tiles of all items, one after the other, are cut into as many equal stretches as there are CTAs for them (in the shared form some
// CTAs have the prompt's items and the others the requests'), so that a long prompt for few requests and short histories for many fill the chip
// alike.  The part of an item in one stretch is a segment.  Segments that are not a whole result leave (o, m, l) in fp32 in scratch, and a
// second launch joins them.  Where everything goes follows from prefix sums over the batch that each CTA makes for itself; CTA 0 leaves them
// for the second launch.
//
// Inside a CTA, warp 15 works out the segments, one after the other, and leaves them in a list of eight in shared memory (every warp on
// its own needed so much code that the warps waited for instructions: 32 requests behind 2048 tokens 59 us).  They run through one pipeline of tiles,
// g = 0, 1, ..:  warps 13 and 14 load Q (two buffers) and K, and V, by TMA, a box for each page;  warp 12 issues S[g & 1] = Q K_g^T two tiles ahead of O[segment & 1] += P_g V_g, P taken from TMEM;  warps 0-7 are the
// softmax, two threads to a row;  warps 8-11 write a segment's result out while the next one runs.
//
// Few rows: a warp reaches only its own quarter of the TMEM lanes, and the two warps of a quarter share a scheduler, so that 32 rows alone
// would take as long as 128 (0.9 us a tile, where the products need 0.55).  Up to 32 rows therefore lie in the tile four times, and copy c
// takes a quarter of a tile's keys, its other weights being zeros; the copies' results are joined on the way out.
//
// Keys beyond a length are cut off from the scores by a select, and their values are overwritten by zeros before the product: what lies there
// (the rest of a page, or of the ring) may be anything, NaN included.
// The product P_g V_g has a barrier for even and one for odd tiles: the scores of tile g + 1 do not wait for it, so that a reader may be two
// products ahead of one barrier's phase.
constexpr int PA_M = 128, PA_N = 128, PA_THREADS = 512, PA_MAX_BATCH = 1024, PA_LIST = 8;
constexpr float PA_RESCALE = 8.f;          // log2: the running maximum is let be while rows grow by less

template <int HD> struct PaCfg {
  static constexpr int NK = HD == 64 ? 4 : 2, NV = HD == 64 ? 4 : 2;
  static constexpr int Q_BYTES = PA_M * HD * 2, T_BYTES = PA_N * HD * 2;
  static constexpr int OFF_Q = 0, OFF_K = 2 * Q_BYTES, OFF_V = OFF_K + NK * T_BYTES;
  static constexpr int OFF_X = OFF_V + NV * T_BYTES;             // float[2 parities][2 halves][128]: maxima of a tile's halves
  static constexpr int OFF_ML = OFF_X + 2 * 2 * PA_M * 4;        // float[2 segments][3][128]: m, and l of either half
  static constexpr int OFF_STAGE = OFF_ML + 2 * 3 * PA_M * 4;    // float[128][36] (or [32][HD + 8]): results of copies on the way out
  static constexpr int OFF_BAR = OFF_STAGE + PA_M * 36 * 4, OFF_LIST = OFF_BAR + 512, OFF_SCAN = OFF_LIST + PA_LIST * 48;
  static constexpr int SMEM_BYTES = OFF_SCAN + 2 * (PA_MAX_BATCH + 1) * 4;
  static constexpr int TM_S = 0, TM_O = 256;
};

struct PagedTcParams {
  PagedAttnParams a;
  int group, group_mul, tpt;               // query heads to a key-value head (and 65536 / group + 1: see token_of), tokens in a tile
  int ts, tb;                              // tokens in a box of an own item, of a prompt's item
  int copies, copies_prompt;
  int joint, prefix_tiles, prefix_row_tiles, prefix_work;   // prefix_work: key tiles of all prompt items (shared form)
  float* part;                             // partial o: [prompt slots][tb * group][HD], then [own slots][ts * group][HD]
  float2* ml;                              // their (m, l), m in units of log2
  int* sums;                               // Stretches, tiles before a request [batch + 1], query tiles before a request [batch + 1]
  long long own_slot0, part_rows;          // rows of the prompt's slots, rows in all
  int* status;
};
constexpr int PA_SUMS = 4;                 // ints in front of the prefix sums

// row / group for rows of a tile
__device__ __forceinline__ int token_of(const PagedTcParams& p, int row) { return row * p.group_mul >> 16; }

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

// How the tiles are dealt: CTAs [0, prompt_ctas) have stretches of `per_prompt` of the prompt's, the others of `per` of the requests'.  With
// both there, in proportion to what they cost: tiles and items of a request's own, tiles of the prompt's by the rows in them.
// Relative: a full tile waits for its exponentials, one of few rows for its products or its bytes, and an item for its first bytes.
constexpr float PA_COST_FULL = 1.f, PA_COST_FEW = 0.6f, PA_COST_ITEM = 0.3f;
struct Stretches { int prompt_ctas, per_prompt, per, own_work; };
__device__ __forceinline__ Stretches stretches_of(const PagedTcParams& p, int own_work, int own_items, int ctas) {
  Stretches d;
  d.own_work = own_work;
  d.prompt_ctas = 0;
  if (p.prefix_work > 0) {
    const float prompt = (float)p.prefix_work * (p.copies_prompt == 1 ? PA_COST_FULL : PA_COST_FEW);
    const float own = (float)own_work * (p.copies == 1 ? PA_COST_FULL : PA_COST_FEW) + (float)own_items * PA_COST_ITEM;
    d.prompt_ctas = own_work > 0 ? min(max((int)((float)ctas * prompt / (prompt + own) + 0.5f), 1), ctas - 1) : ctas;
  }
  d.per_prompt = max((p.prefix_work + max(d.prompt_ctas, 1) - 1) / max(d.prompt_ctas, 1), 1);
  d.per = max((own_work + max(ctas - d.prompt_ctas, 1) - 1) / max(ctas - d.prompt_ctas, 1), 1);
  return d;
}

// The segments of a stretch [pos, end) of the prompt's or the requests' key tiles, in order.
struct Walk {
  const PagedTcParams& p;
  const int *tiles_before, *items_before;
  int pos, end;
  int b, h, rt, tile;                      // own items: the next one and the tile in it
  Request r;
  bool prompt, placed;
  __device__ __forceinline__ Walk(const PagedTcParams& p_, const int* tb, const int* ib, bool prompt_, int pos_, int end_)
      : p(p_), tiles_before(tb), items_before(ib), pos(pos_), end(end_), b(0), h(0), rt(0), tile(0), prompt(prompt_), placed(false) {}
  __device__ __forceinline__ int find() const {      // the last request whose tiles begin at or before pos
    int lo = 0, n = p.a.batch;
    const int per_head = pos / p.a.kv_heads;
    while (n > 1) {
      const int half = n >> 1;
      if (tiles_before[lo + half] <= per_head) { lo += half; n -= half; } else n = half;
    }
    return lo;
  }
  __device__ __forceinline__ void place(int at, const Request& its) {
    b = at;
    r = its;
    const int all = max(tiles_before[b + 1] - tiles_before[b], 1);
    int off = pos - tiles_before[b] * p.a.kv_heads;
    h = off / all;
    off -= h * all;
    rt = 0;
    for (int t = tiles_of(p, r, 0); off >= t && rt + 1 < r.row_tiles; t = tiles_of(p, r, rt)) { off -= t; ++rt; }
    tile = off;
    placed = true;
  }
  __device__ __forceinline__ bool next(Segment& s) {
    if (pos >= end) return false;
    if (prompt) {
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
      if (!placed) { const int at = find(); place(at, request_of(p, at)); }
      while (rt >= r.row_tiles || tiles_of(p, r, rt) <= tile) {      // on to the next item that has tiles; there is one before `end`
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

// What the warps have to know of a segment, as it lies in the list.
struct __align__(16) Listed {
  int tiles;                               // 0: no more
  int tile, flags, h, b;                   // first key tile in the item; 1: of the prompt, 2: a whole result
  int t0, rows;                            // first token, rows
  int seen, shift;                         // own keys that some row sees; the row of token i sees own keys up to shift + i
  int pad;
  long long at;                            // where its partial rows go
};
static_assert(sizeof(Listed) == 48, "a list entry");

// Keys of key tile j of a segment's item: how many there are and where in their table they begin.
struct KeyTile { int prompt, first, count; };
__device__ __forceinline__ KeyTile key_tile(const PagedTcParams& p, int flags, int seen, int j) {
  KeyTile k;
  k.prompt = (flags & 1) || (p.joint && j < p.prefix_tiles);
  k.first = (k.prompt || !p.joint ? j : j - p.prefix_tiles) * PA_N;
  k.count = max(min(PA_N, (k.prompt ? p.a.prefix_len : seen) - k.first), 0);
  return k;
}
// The page, for lane i, that holds the tile's keys from i * page_size on; -1 for lanes without one.  `boxes`: how many there are.
__device__ __forceinline__ int page_for(const PagedTcParams& p, const Listed& s, int j, int lane, int& boxes) {
  const KeyTile k = key_tile(p, s.flags, s.seen, j);
  boxes = (k.count + (1 << p.a.page_log2) - 1) >> p.a.page_log2;
  if (lane >= boxes) return -1;
  const int at = (k.first >> p.a.page_log2) + lane;
  return k.prompt ? p.a.prefix_table[at] : p.a.tables[s.b * p.a.table_stride + at];
}

// Prefix sums over the batch (a block of PA_THREADS): key tiles for one key-value head, and query tiles, before each request.
__device__ __forceinline__ void scan_batch(const PagedTcParams& p, int* tiles_before, int* items_before, int* warp_sums, int& all_tiles, int& all_items) {
  constexpr int WARPS = PA_THREADS / 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (p.a.batch + PA_THREADS - 1) / PA_THREADS, b0 = min(tid * per, p.a.batch), b1 = min(b0 + per, p.a.batch);
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
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    const int x = warp_sums[2 * w], y = warp_sums[2 * w + 1];
    if (w < warp) { bt += x; bi += y; }
    all_t += x;
    all_i += y;
  }
  for (int b = b0; b < b1; ++b) { tiles_before[b] += bt; items_before[b] += bi; }
  if (tid == 0) { tiles_before[p.a.batch] = all_t; items_before[p.a.batch] = all_i; }
  all_tiles = all_t;
  all_items = all_i;
}

// Where a partial result goes.  Shared form: every segment of every item, numbered by item + CTA (a segment begins where an item or a
// stretch does).  Joint form: only items that a stretch's end cuts, of which a CTA has its first and its last segment.
__device__ __forceinline__ long long own_row(const PagedTcParams& p, long long slot) { return p.own_slot0 + slot * (p.ts * p.group); }
__device__ __forceinline__ long long prompt_row(const PagedTcParams& p, long long slot) { return slot * (p.tb * p.group); }
// Starts that do not rise would make more items than there is room for: their rows stay out of the scratch.
__device__ __forceinline__ bool has_room(const PagedTcParams& p, long long row) { return row >= 0 && row < p.part_rows; }

// Whether the phase is complete, without waiting for it.
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred P;\n\tmbarrier.test_wait.parity.shared::cta.b64 P, [%1], %2;\n\tselp.b32 %0, 1, 0, P;\n\t}\n" : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
  return ok != 0;
}
// Out of the way until the phase completes, for at most about `ns`: a loop over several barriers that only tests them takes issue slots from
// the warps beside it.
__device__ __forceinline__ void mbar_nap(uint64_t* bar, uint32_t parity, uint32_t ns) {
  asm volatile("{\n\t.reg .pred P;\n\tmbarrier.try_wait.parity.shared::cta.b64 P, [%0], %1, %2;\n\t}\n" ::"r"(smem_u32(bar)), "r"(parity), "r"(ns) : "memory");
}
__device__ __forceinline__ void softmax_pair_sync(int quad) { asm volatile("bar.sync %0, 64;" ::"r"(quad + 1) : "memory"); }
__device__ __forceinline__ void out_sync() { asm volatile("bar.sync 5, 128;" ::: "memory"); }
// Lanes 0-15 of the quarter, 64 columns: lane l of the warp receives columns 8 k + 2 (l % 4) and the next of row l / 4 in r[4 k], r[4 k + 1], of
// row 8 + l / 4 in r[4 k + 2], r[4 k + 3].
__device__ __forceinline__ void tmem_ld_16x256b_x8(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x8.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
               "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

template <int HD>
__global__ void __launch_bounds__(PA_THREADS, 1)
paged_attn_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmQown, const __grid_constant__ CUtensorMap tmK,
                     const __grid_constant__ CUtensorMap tmV, const __grid_constant__ PagedTcParams p) {
  using Cfg = PaCfg<HD>;
  constexpr int NK = Cfg::NK, NV = Cfg::NV, CHUNKS = HD / 64;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ int s_warp_sums[2 * PA_THREADS / 32];
  __shared__ float s_inv[PA_M];
  __shared__ int s_fail, s_first;
  __shared__ Request s_request;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::OFF_BAR);
  uint64_t *q_full = bars, *q_empty = bars + 2, *k_full = bars + 4, *k_empty = k_full + NK, *v_full = k_empty + NK, *v_empty = v_full + NV;
  uint64_t *s_full = v_empty + NV, *p_full = s_full + 2, *o_done = s_full + 4, *o_free = s_full + 6, *seg_done = s_full + 8, *o_full = s_full + 10;
  uint64_t *listed = s_full + 12, *list_free = listed + PA_LIST;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(list_free + PA_LIST);
  const Listed* list = reinterpret_cast<const Listed*>(smem + Cfg::OFF_LIST);
  int* tiles_before = reinterpret_cast<int*>(smem + Cfg::OFF_SCAN);
  int* items_before = tiles_before + p.a.batch + 1;
  float* s_ml = reinterpret_cast<float*>(smem + Cfg::OFF_ML);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_launch_dependents();
  if ((smem_u32(smem) & 1023u) != 0) {
    if (threadIdx.x == 0) report_error(p.status, OA_KERR_BAD_ARG);
    return;
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1); mbar_init(&q_empty[i], 1); mbar_init(&s_full[i], 1); mbar_init(&p_full[i], 8);
      mbar_init(&o_done[i], 1); mbar_init(&o_full[i], 1); mbar_init(&o_free[i], 4); mbar_init(&seg_done[i], 8);
    }
    for (int i = 0; i < NK; ++i) { mbar_init(&k_full[i], 1); mbar_init(&k_empty[i], 1); }
    for (int i = 0; i < NV; ++i) { mbar_init(&v_full[i], 1); mbar_init(&v_empty[i], 1); }
    for (int i = 0; i < PA_LIST; ++i) { mbar_init(&listed[i], 1); mbar_init(&list_free[i], 15); }
    mbar_fence_init();
    s_fail = 0;
  }
  if (warp == 12) { tmem_alloc<512>(tmem_slot); tmem_relinquish(); }
  if (warp == 13 && lane == 0) { tma_prefetch_desc(&tmQ); tma_prefetch_desc(&tmQown); tma_prefetch_desc(&tmK); tma_prefetch_desc(&tmV); }
  __syncwarp();
  pdl_wait();
  {                                        // tables on their way to L2 while the lengths arrive: 128 bytes to a thread
    const int lines = (p.a.width + 31) / 32, at = blockIdx.x * PA_THREADS + threadIdx.x;
    for (int i = at; i < p.a.batch * lines; i += gridDim.x * PA_THREADS)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(p.a.tables + (long long)(i / lines) * p.a.table_stride + min(i % lines * 32, p.a.width - 1)));
    if (at * 32 < p.a.prefix_len >> p.a.page_log2) asm volatile("prefetch.global.L2 [%0];" ::"l"(p.a.prefix_table + at * 32));
  }
  int own_tiles, own_items;
  scan_batch(p, tiles_before, items_before, s_warp_sums, own_tiles, own_items);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const Stretches deal = stretches_of(p, own_tiles * p.a.kv_heads, own_items * p.a.kv_heads, gridDim.x);
  const bool on_prompt = (int)blockIdx.x < deal.prompt_ctas;
  const int cta = on_prompt ? blockIdx.x : blockIdx.x - deal.prompt_ctas, per = on_prompt ? deal.per_prompt : deal.per;
  const int work = on_prompt ? p.prefix_work : deal.own_work;
  const int lo = (int)min((long long)cta * per, (long long)work), hi = (int)min((long long)(cta + 1) * per, (long long)work);
  if (!on_prompt)                          // the request in which the stretch begins, by the thread that has scanned it
    for (int b = threadIdx.x * ((p.a.batch + PA_THREADS - 1) / PA_THREADS), k = 0; k < (p.a.batch + PA_THREADS - 1) / PA_THREADS && b < p.a.batch; ++k, ++b)
      if (lo >= tiles_before[b] * p.a.kv_heads && lo < tiles_before[b + 1] * p.a.kv_heads) { s_first = b; s_request = request_of(p, b); }
  __syncthreads();
  const int copies = on_prompt ? p.copies_prompt : p.copies, copy_rows = PA_M / copies;     // 1 and 128, or 4 and 32

  // The next entry of the list.  Every warp reads each once, in order, and lets go of it when it has what it needs.
  int li = 0;
  uint32_t lphase = 0;
  const auto take = [&](Listed& s, bool& ok) -> bool {
    ok = warp_wait(&listed[li], lphase);
    if (!ok) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_FULL); return false; }
    s = list[li];
    return s.tiles > 0;
  };
  const auto let_go = [&] {
    __syncwarp();
    if (lane == 0) mbar_arrive(&list_free[li]);
    if (++li == PA_LIST) { li = 0; lphase ^= 1; }
  };
  Listed s;
  bool ok = true;

  if (warp == 15) {
    // ---------------------------------------------------------------- segments
    if (blockIdx.x == 0) {                 // for the second launch
      if (lane == 0) { p.sums[0] = deal.prompt_ctas; p.sums[1] = deal.per_prompt; p.sums[2] = deal.per; p.sums[3] = deal.own_work; }
      for (int b = lane; b <= p.a.batch; b += 32) { p.sums[PA_SUMS + b] = tiles_before[b]; p.sums[PA_SUMS + 1 + p.a.batch + b] = items_before[b]; }
    }
    if (lane == 0) {
      Walk walk(p, tiles_before, items_before, on_prompt, lo, hi);
      if (!on_prompt && lo < hi) walk.place(s_first, s_request);
      Segment g;
      bool more = true;
      while (more) {
        more = walk.next(g);
        if (!mbar_wait(&list_free[li], lphase ^ 1)) { report_error(p.status, OA_KERR_WAIT_EMPTY); break; }
        Listed e;
        e.tiles = more ? g.tiles : 0;
        e.tile = g.tile;
        e.flags = (g.prompt ? 1 : 0) | (p.joint && g.tiles == g.item_tiles ? 2 : 0);
        e.h = g.h;
        e.b = g.b;
        e.t0 = g.t0;
        e.rows = g.tokens * p.group;
        e.seen = g.seen;
        e.shift = g.own - g.n + g.i0;
        const bool first = g.tile > 0 || walk.pos - g.tiles == lo;
        const long long slot = p.joint ? 2ll * cta + (first ? 0 : 1) : (long long)g.item + cta;
        e.at = g.prompt ? prompt_row(p, slot) : own_row(p, slot);
        reinterpret_cast<Listed*>(smem + Cfg::OFF_LIST)[li] = e;
        mbar_arrive(&listed[li]);
        if (++li == PA_LIST) { li = 0; lphase ^= 1; }
      }
    }
    __syncwarp();
  } else if (warp == 13 || warp == 14) {
    // ---------------------------------------------------------------- loads: warp 13 Q and K, warp 14 V
    const bool is_k = warp == 13;
    const int ps = 1 << p.a.page_log2, ring = is_k ? NK : NV;
    uint64_t *full = is_k ? k_full : v_full, *empty = is_k ? k_empty : v_empty;
    uint8_t* tiles = smem + (is_k ? Cfg::OFF_K : Cfg::OFF_V);
    const CUtensorMap* map = is_k ? &tmK : &tmV;
    int st = 0, sq = 0, boxes = 0, id = -1;
    uint32_t phase = 1;                                           // of the slot to fill: free at first
    bool more = take(s, ok);
    if (more) { let_go(); id = page_for(p, s, s.tile, lane, boxes); }
    while (ok && more) {
      const int n = s.tiles, h = s.h;
      if (is_k) {
        const int qb = sq & 1;
        ok = warp_wait(&q_empty[qb], ((sq >> 1) & 1) ^ 1);
        if (!ok) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_EMPTY); break; }
        if (elect_one()) {
          const CUtensorMap* mq = (s.flags & 1) ? &tmQ : &tmQown;
          mbar_expect_tx(&q_full[qb], (uint32_t)(copies * ((s.flags & 1) ? p.tb : p.ts) * p.group * HD * 2));
#pragma unroll 1
          for (int c = 0; c < copies; ++c)
#pragma unroll
            for (int x = 0; x < CHUNKS; ++x)
              tma_load_3d(smem + Cfg::OFF_Q + qb * Cfg::Q_BYTES + x * (PA_M * 128) + c * copy_rows * 128, mq, &q_full[qb], x * 64, h * p.group, s.t0);
        }
        __syncwarp();
        ++sq;
      }
#pragma unroll 1
      for (int j = 0; j < n; ++j) {
        const int now = id, now_boxes = boxes;                    // and the next tile's page, of the next segment's first where this is the last
        int next = s.tile + j + 1;
        if (j + 1 == n) {
          more = take(s, ok);
          if (more) let_go();
          next = s.tile;
        }
        if (more) id = page_for(p, s, next, lane, boxes);
        if (ok) ok = warp_wait(&empty[st], phase);
        if (!ok) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_EMPTY); break; }
        if (elect_one()) mbar_expect_tx(&full[st], (uint32_t)(now_boxes * ps * HD * 2));
        __syncwarp();
        if (lane < now_boxes) {
#pragma unroll
          for (int x = 0; x < CHUNKS; ++x)
            tma_load_3d(tiles + st * Cfg::T_BYTES + x * (PA_N * 128) + lane * ps * 128, map, &full[st], x * 64, h << p.a.page_log2, now);
        }
        __syncwarp();
        if (++st == ring) { st = 0; phase ^= 1; }
      }
    }
  } else if (warp == 12) {
    // ---------------------------------------------------------------- products: the next scores or the next P V, whichever has what it needs
    constexpr uint32_t idesc_qk = umma_idesc_bf16(PA_M, PA_N, 0, 0), idesc_pv = umma_idesc_bf16(PA_M, HD, 0, 1);
    const uint64_t q_desc = umma_smem_desc_sw128(smem_u32(smem + Cfg::OFF_Q), 16, 1024), k_desc = umma_smem_desc_sw128(smem_u32(smem + Cfg::OFF_K), 16, 1024);
    const uint64_t v_desc = umma_smem_desc_sw128(smem_u32(smem + Cfg::OFF_V), PA_N * 128, 1024);
    const auto ready = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_test(bar, parity)); };
    int gq = 0, jq = 0, nq = 0, sqq = -1, lq = 0;                 // of the score products: tile, tile in the segment, its tiles, segment, list entry
    uint32_t lqphase = 0;
    bool q_there = false, q_end = false;
    int g = 0, sq = 0, j = 0, n = 0;                              // of P V
    bool o_there = false;
    uint64_t since = 0;
    uint32_t idle = 0;
    for (;;) {
      bool moved = false;
      // scores, over P of the tile before the last: behind its product in the pipe
      if (!q_end && gq < g + 2) {
        if (jq == nq && ready(&listed[lq], lqphase)) {
          nq = list[lq].tiles;
          jq = 0;
          q_there = false;
          q_end = nq == 0;
          if (!q_end) { ++sqq; if (++lq == PA_LIST) { lq = 0; lqphase ^= 1; } }
          moved = true;
        }
        if (jq < nq) {
          const int st = gq % NK;
          if (!q_there) q_there = ready(&q_full[sqq & 1], (sqq >> 1) & 1);
          if (q_there && ready(&k_full[st], (gq / NK) & 1)) {
            tc_fence_after();
            if (elect_one()) {
              const uint64_t qd = q_desc + ((sqq & 1) * Cfg::Q_BYTES >> 4), kd = k_desc + (st * Cfg::T_BYTES >> 4);
#pragma unroll
              for (int ks = 0; ks < HD / 16; ++ks) {
                const uint32_t off = ((ks >> 2) * (PA_M * 128) + (ks & 3) * 32) >> 4;
                umma_f16(tmem_base + Cfg::TM_S + (gq & 1) * PA_N, qd + off, kd + off, idesc_qk, ks > 0 ? 1u : 0u);
              }
              umma_commit(&k_empty[st]);
              umma_commit(&s_full[gq & 1]);
              if (jq + 1 == nq) umma_commit(&q_empty[sqq & 1]);
            }
            __syncwarp();
            ++jq; ++gq;
            moved = true;
          }
        }
      }
      if (g < gq || (q_end && j == n)) {
        if (j == n) {                                             // the segment of the next product
          if (g == gq) break;                                     // there is none
          if (!take(s, ok)) break;                                // listed already
          let_go();
          n = s.tiles;
          j = 0;
          o_there = false;
        }
        const int st = g % NV;
        if (!o_there) o_there = ready(&o_free[sq & 1], ((sq >> 1) & 1) ^ 1);      // the result before the last has been read
        if (o_there && ready(&p_full[g & 1], (g >> 1) & 1) && ready(&v_full[st], (g / NV) & 1)) {
          tc_fence_after();
          if (elect_one()) {
            const uint64_t vd = v_desc + (st * Cfg::T_BYTES >> 4);
#pragma unroll
            for (int ks = 0; ks < PA_N / 16; ++ks)
              umma_f16_ts(tmem_base + Cfg::TM_O + (sq & 1) * HD, tmem_base + Cfg::TM_S + (g & 1) * PA_N + ks * 8, vd + (ks * 2048 >> 4), idesc_pv,
                          (j > 0 || ks > 0) ? 1u : 0u);
            umma_commit(&v_empty[st]);
            umma_commit(&o_done[g & 1]);
            if (j + 1 == n) umma_commit(&o_full[sq & 1]);
          }
          __syncwarp();
          ++g;
          if (++j == n) ++sq;
          moved = true;
        }
      }
      if (moved) { idle = 0; since = 0; continue; }
      if (g < gq) mbar_nap(&p_full[g & 1], (g >> 1) & 1, 64);
      else if (jq < nq) mbar_nap(&k_full[gq % NK], (gq / NK) & 1, 64);
      else mbar_nap(&listed[lq], lqphase, 64);
      if ((++idle & 0xff) == 0) {                                 // bounded like every wait: by wall time
        const uint64_t now = global_timer_ns();
        if (since == 0) since = now;
        else if (__any_sync(0xffffffffu, now - since > OA_WAIT_LIMIT_NS)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_SOFTMAX); break; }
      }
    }
  } else if (warp < 8) {
    // ---------------------------------------------------------------- softmax: warp w has TMEM lanes 32 (w % 4).. and the keys of half w / 4 of a tile
    constexpr int OC = HD / 2;
    const int quad = warp & 3, half = warp >> 2, r = quad * 32 + lane;
    const int copy = copies == 1 ? 0 : quad, row = copies == 1 ? r : lane, i_row = token_of(p, row);      // i_row: token of this row in the tile
    const uint32_t t_lane = (uint32_t)(quad * 32) << 16;
    const float sl2 = p.a.scale * 1.4426950408889634f;
    const unsigned long long sl22 = f2_splat(sl2);
    float* xch = reinterpret_cast<float*>(smem + Cfg::OFF_X);
    int g = 0, sq = 0;
#pragma unroll 1
    while (ok && take(s, ok)) {
      let_go();
      const bool live = copies > 1 || quad * 32 < s.rows;         // of this warp: some row is there
      float m_run = -INFINITY, l_run = 0.f;
      const uint32_t o_addr = tmem_base + t_lane + Cfg::TM_O + (sq & 1) * HD + half * OC;
#pragma unroll 1
      for (int j = 0; j < s.tiles; ++j, ++g) {
        const KeyTile kt = key_tile(p, s.flags, s.seen, s.tile + j);
        ok = warp_wait(&s_full[g & 1], (g >> 1) & 1);
        if (!ok) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_TMEM_FULL); break; }
        tc_fence_after();
        if (live) {
          const uint32_t s_addr = tmem_base + t_lane + Cfg::TM_S + (g & 1) * PA_N;
          // columns up to `last` are seen: the keys that there are, and of a request's own keys those up to the row's token
          const int last = kt.prompt ? kt.count - 1 : min(kt.count - 1, s.shift + i_row - kt.first);
          const bool cut = (kt.prompt ? kt.count - 1 : min(kt.count - 1, s.shift - kt.first)) < PA_N - 1;
          float alpha = 1.f;
          bool grow = false;
          const auto tile = [&](auto copies_of) {                 // 64 / C keys of this thread: half * 64 + copy * W ..
            constexpr int C = decltype(copies_of)::value, W = 64 / C;
            uint32_t sv[W];
            if constexpr (C == 1) { tmem_ld32(s_addr + half * 64, sv); tmem_ld32(s_addr + half * 64 + 32, sv + 32); }
            else tmem_ld16(s_addr + half * 64 + copy * 16, sv);
            tmem_ld_wait();
            if (cut) {
              const int lim = last - half * 64 - copy * W;
#pragma unroll
              for (int i = 0; i < W; ++i) sv[i] = i <= lim ? sv[i] : 0xff800000u;
            }
            float m0 = __uint_as_float(sv[0]), m1 = __uint_as_float(sv[1]);
#pragma unroll
            for (int i = 2; i < W - 2; i += 4) {
              m0 = fmax3(m0, __uint_as_float(sv[i]), __uint_as_float(sv[i + 1]));
              m1 = fmax3(m1, __uint_as_float(sv[i + 2]), __uint_as_float(sv[i + 3]));
            }
            float mx = fmax3(m0, m1, fmaxf(__uint_as_float(sv[W - 2]), __uint_as_float(sv[W - 1])));
            float* slots = xch + (g & 1) * (2 * PA_M);
            slots[(half ^ 1) * PA_M + r] = mx;
            softmax_pair_sync(quad);                              // both halves are in registers: P may go over S
            mx = fmaxf(mx, slots[half * PA_M + r]) * sl2;
            const float m_new = fmaxf(m_run, mx);
            grow = row < s.rows && (m_new - m_run) > PA_RESCALE;  // the first time: from -inf.  Not for rows that are not there, whose scores are anything
            const float m_cand = grow ? m_new : m_run;
            const float m_use = m_cand == -INFINITY ? 0.f : m_cand;       // a row that has seen nothing yet
            alpha = grow ? fast_exp2(m_run - m_use) : 1.f;
            m_run = m_cand;
            const unsigned long long neg_m = f2_splat(-m_use);
            unsigned long long l01 = 0, l23 = 0;
            uint32_t pk[W / 2];
#pragma unroll
            for (int i = 0; i < W; i += 4) {
              const unsigned long long x01 = f2_fma(f2_of(sv[i], sv[i + 1]), sl22, neg_m), x23 = f2_fma(f2_of(sv[i + 2], sv[i + 3]), sl22, neg_m);
              // one of eight pairs on the multiply-add pipe, where the special-function units are what a full tile waits for
              const unsigned long long e01 = exp2_mufu2(x01), e23 = C == 1 && (i >> 2) % 4 == 0 ? exp2_fma2(x23) : exp2_mufu2(x23);
              l01 = f2_add(l01, e01);
              l23 = f2_add(l23, e23);
              pk[i >> 1] = f2_bf16(e01);                          // weights to bf16, as the tensor cores take them; their sum stays fp32
              pk[(i >> 1) + 1] = f2_bf16(e23);
            }
            uint32_t a, b;
            f2_to(f2_add(l01, l23), a, b);
            l_run = l_run * alpha + (__uint_as_float(a) + __uint_as_float(b));
            const uint32_t p_addr = s_addr + half * 32;           // this half's 64 keys: the copy's own, zeros elsewhere
            if constexpr (C == 1) tmem_st32(p_addr, pk);
            else {
              uint32_t all[32];
#pragma unroll
              for (int i = 0; i < 32; ++i) all[i] = (i >> 3) == copy ? pk[i & 7] : 0u;
              tmem_st32(p_addr, all);
            }
          };
          if (copies > 1) tile(std::integral_constant<int, 4>());
          else tile(std::integral_constant<int, 1>());
          if (j > 0 && __any_sync(0xffffffffu, grow)) {           // O again to the new maximum, behind the product before
            ok = warp_wait(&o_done[(g - 1) & 1], ((g - 1) >> 1) & 1);
            if (!ok) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_TMEM_FULL); break; }
            tc_fence_after();
#pragma unroll 1
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
#pragma unroll 1
          for (int i = threadIdx.x; i < (PA_N - kt.count) * CHUNKS * 8; i += 256) {
            const int at = kt.count + i / (CHUNKS * 8), c = i % (CHUNKS * 8);
            st_shared_v4(base + (c >> 3) * (PA_N * 128) + at * 128 + (c & 7) * 16, make_uint4(0, 0, 0, 0));
          }
          fence_proxy_async_smem();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[g & 1]);
      }
      if (!ok) break;
      ok = warp_wait(&o_free[sq & 1], ((sq >> 1) & 1) ^ 1);       // m and l of the segment before the last have been read
      if (!ok) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_TMEM_EMPTY); break; }
      float* ml = s_ml + (sq & 1) * 3 * PA_M;
      if (half == 0) ml[r] = m_run;
      ml[(1 + half) * PA_M + r] = l_run;
      __syncwarp();
      if (lane == 0) mbar_arrive(&seg_done[sq & 1]);
      ++sq;
    }
  } else {
    // ---------------------------------------------------------------- results: warp 8 + q has TMEM lanes 32 q..
    const int quad = warp & 3, r = quad * 32 + lane, et = threadIdx.x - 256;
    const int copy = copies == 1 ? 0 : quad, row = copies == 1 ? r : lane, i_row = token_of(p, row);
    const uint32_t t_lane = tmem_base + ((uint32_t)(quad * 32) << 16);
    float* stage = reinterpret_cast<float*>(smem + Cfg::OFF_STAGE);
    int sq = 0;
    bool met = false;
#pragma unroll 1
    while (take(s, ok)) {
      let_go();
      // barriers of segments, of which at most two are under way: this warp may be behind by many tiles
      ok = warp_wait(&seg_done[sq & 1], (sq >> 1) & 1) && warp_wait(&o_full[sq & 1], (sq >> 1) & 1);
      if (!ok && lane == 0) { report_error(p.status, OA_KERR_WAIT_TMEM_FULL); s_fail = 1; }
      if (copies > 1) { out_sync(); ok = s_fail == 0; }           // what was staged before has been read; and the four warps leave together
      if (!ok) { met = true; break; }
      tc_fence_after();
      const float* ml = s_ml + (sq & 1) * 3 * PA_M;
      const uint32_t o_addr = t_lane + Cfg::TM_O + (sq & 1) * HD;
      const bool whole = s.flags & 2;                             // nothing to be joined
      // the row's m, l and the factor of this copy's part
      float m = ml[r], l = ml[PA_M + r] + ml[2 * PA_M + r], f = 1.f;
      if (copies > 1) {
        const float mine = m;
        float mc[4], sum = 0.f;
#pragma unroll
        for (int c = 0; c < 4; ++c) { mc[c] = ml[c * 32 + lane]; m = fmaxf(m, mc[c]); }
#pragma unroll
        for (int c = 0; c < 4; ++c)
          sum += (ml[PA_M + c * 32 + lane] + ml[2 * PA_M + c * 32 + lane]) * (mc[c] == -INFINITY ? (m == -INFINITY ? 1.f : 0.f) : fast_exp2(mc[c] - m));
        f = mine == -INFINITY ? 0.f : fast_exp2(mine - m);
        l = sum;
      }
      const float inv = l == 0.f ? 0.f : 1.f / l;                 // NaN stays NaN
      const int t = s.t0 + i_row;
      const bool there = row < s.rows && (whole ? t >= 0 && t < p.a.tokens : has_room(p, s.at + row));
      const long long out_row = (long long)t * p.a.q_heads + s.h * p.group + row - i_row * p.group;
      if (copy == 0 && there) {
        if (!whole) p.ml[s.at + row] = make_float2(m, l);
        else if (p.a.lse) p.a.lse[out_row] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
      }
      const auto release = [&] {                                  // all has been read
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&o_free[sq & 1]);
      };
      if (copies == 1) {                                          // a row to a lane
        if (quad * 32 < s.rows) {
#pragma unroll 1
          for (int c = 0; c < HD; c += 32) {
            uint32_t o[32];
            tmem_ld32(o_addr + c, o);
            tmem_ld_wait();
            const float* x = reinterpret_cast<const float*>(o);
            if (!there) {
            } else if (whole) {
              uint4* to = reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.a.out) + out_row * HD + c);
#pragma unroll
              for (int k = 0; k < 4; ++k, x += 8)
                to[k] = make_uint4(pack_bf16x2(x[0] * inv, x[1] * inv), pack_bf16x2(x[2] * inv, x[3] * inv), pack_bf16x2(x[4] * inv, x[5] * inv), pack_bf16x2(x[6] * inv, x[7] * inv));
            } else {
              uint4* to = reinterpret_cast<uint4*>(p.part + (s.at + row) * HD + c);
#pragma unroll
              for (int k = 0; k < 8; ++k) to[k] = make_uint4(o[k * 4], o[k * 4 + 1], o[k * 4 + 2], o[k * 4 + 3]);
            }
            __syncwarp();
          }
        }
        release();
      } else {
        // copies meet in shared memory
        if (copy == 0) s_inv[row] = inv;
        const auto emit = [&](int rw, int c, float4 sum) {        // four columns of a row
          if (!whole) {
            if (has_room(p, s.at + rw)) *reinterpret_cast<float4*>(p.part + (s.at + rw) * HD + c) = sum;
            return;
          }
          const int i = token_of(p, rw), tr = s.t0 + i;
          if (tr < 0 || tr >= p.a.tokens) return;
          const float q = s_inv[rw];
          *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.a.out) + ((long long)tr * p.a.q_heads + s.h * p.group + rw - i * p.group) * HD + c) =
              make_uint2(pack_bf16x2(sum.x * q, sum.y * q), pack_bf16x2(sum.z * q, sum.w * q));
        };
        if (s.rows <= 8) {
          // Up to eight rows: a load that gives lane l two neighbouring columns of row l / 4, so that every lane has some of them.  A row to a
          // lane left 24 lanes or more idle and made a request's single token 1.5 us of it.
          const float fr = __shfl_sync(0xffffffffu, f, lane >> 2);
          float* to = stage + (copy * 8 + (lane >> 2)) * (HD + 8) + (lane & 3) * 2;
          uint32_t o[HD / 2];
#pragma unroll
          for (int c = 0; c < HD / 64; ++c) tmem_ld_16x256b_x8(o_addr + c * 64, o + c * 32);
          tmem_ld_wait();
          release();
#pragma unroll
          for (int c = 0; c < HD / 8; ++c)
            *reinterpret_cast<float2*>(to + c * 8) = fr == 0.f ? make_float2(0.f, 0.f) : make_float2(__uint_as_float(o[c * 4]) * fr, __uint_as_float(o[c * 4 + 1]) * fr);
          out_sync();
          constexpr int PER_ROW = HD / 4;
#pragma unroll 1
          for (int i = et; i < s.rows * PER_ROW; i += 128) {
            const int rw = i / PER_ROW, c = (i % PER_ROW) * 4;
            float4 x[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) x[k] = *reinterpret_cast<const float4*>(stage + (k * 8 + rw) * (HD + 8) + c);
            emit(rw, c, make_float4((x[0].x + x[1].x) + (x[2].x + x[3].x), (x[0].y + x[1].y) + (x[2].y + x[3].y), (x[0].z + x[1].z) + (x[2].z + x[3].z),
                                    (x[0].w + x[1].w) + (x[2].w + x[3].w)));
          }
        } else {
#pragma unroll 1
          for (int c0 = 0; c0 < HD; c0 += 32) {                   // 32 columns at a time
            if (c0 > 0) out_sync();                               // the columns before have been read
            uint32_t o[32];
            tmem_ld32(o_addr + c0, o);
            tmem_ld_wait();
            if (c0 + 32 == HD) release();
            if (row < s.rows) {
              float4* to = reinterpret_cast<float4*>(stage + r * 36);
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                const float* x = reinterpret_cast<const float*>(o) + k * 4;
                to[k] = f == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(x[0] * f, x[1] * f, x[2] * f, x[3] * f);
              }
            }
            out_sync();
#pragma unroll 1
            for (int i = et; i < s.rows * 8; i += 128) {
              const int rw = i >> 3, c = (i & 7) * 4;
              float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const float4 x = *reinterpret_cast<const float4*>(stage + (k * 32 + rw) * 36 + c);
                sum.x += x.x; sum.y += x.y; sum.z += x.z; sum.w += x.w;
              }
              emit(rw, c0 + c, sum);
            }
          }
        }
      }
      ++sq;
    }
    if (!ok && copies > 1 && !met) { s_fail = 1; out_sync(); }    // the entry never came: the others, who meet once more, do not wait for this warp
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 12) { tc_fence_after(); tmem_dealloc<512>(tmem_base); }
}

// Joins partial results (acc, m, l) of one row, a warp to a row, a lane to HD / 32 neighbouring columns.
template <int HD>
struct RowJoin {
  static constexpr int PER = HD / 32;
  float m = -INFINITY, l = 0.f, acc[PER] = {};
  // `count` pieces, of which row_of(i) is the i-th: the weights of 32 at a time, one to a lane, then their rows, four under way at once
  template <typename F>
  __device__ __forceinline__ void add(const PagedTcParams& p, int count, F row_of, int lane) {
    for (int i0 = 0; i0 < count; i0 += 32) {
      const int i = i0 + lane;
      const long long mine = i < count ? row_of(i) : -1;
      const float2 ml = has_room(p, mine) ? p.ml[mine] : make_float2(-INFINITY, 0.f);
      const bool some = ml.y != 0.f;                             // otherwise a piece of which this row saw nothing
      const float m_new = fmaxf(m, warp_max(some ? ml.x : -INFINITY));
      const float a = m == -INFINITY ? 0.f : fast_exp2(m - m_new), w = some ? (ml.x == -INFINITY ? 1.f : fast_exp2(ml.x - m_new)) : 0.f;
      l = l * a + warp_sum(ml.y * w);
#pragma unroll
      for (int e = 0; e < PER; ++e) acc[e] *= a;
      m = m_new;
      const int n = min(count - i0, 32);
      for (int j0 = 0; j0 < n; j0 += 4) {
        float v[4][PER], wj[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const long long row = __shfl_sync(0xffffffffu, mine, min(j0 + k, 31));
          wj[k] = j0 + k < n ? __shfl_sync(0xffffffffu, w, min(j0 + k, 31)) : 0.f;
#pragma unroll
          for (int e = 0; e < PER; ++e) v[k][e] = 0.f;
          if (wj[k] != 0.f) {
            if (PER == 4) *reinterpret_cast<float4*>(v[k]) = *reinterpret_cast<const float4*>(p.part + row * HD + lane * PER);
            else *reinterpret_cast<float2*>(v[k]) = *reinterpret_cast<const float2*>(p.part + row * HD + lane * PER);
          }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int e = 0; e < PER; ++e) acc[e] += v[k][e] * wj[k];
      }
    }
  }
  __device__ __forceinline__ void write(const PagedTcParams& p, int t, int hq, int lane) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    __nv_bfloat16* to = static_cast<__nv_bfloat16*>(p.a.out) + ((long long)t * p.a.q_heads + hq) * HD + lane * PER;
    if (PER == 4) *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[PER - 2] * inv, acc[PER - 1] * inv));
    else *reinterpret_cast<uint32_t*>(to) = pack_bf16x2(acc[0] * inv, acc[1] * inv);
    if (p.a.lse && lane == 0) p.a.lse[(long long)t * p.a.q_heads + hq] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
  }
};

// Shared form: every row from the pieces of its prompt item and of its own item.  Block (b, y) has rows 8 y .. of request b, a warp to each, so that
// all it has to know of the request arrives at once; blocks of b = batch the rows of no request, zeros.
template <int HD>
__global__ void __launch_bounds__(256) paged_join_rows_kernel(const __grid_constant__ PagedTcParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, b = blockIdx.x;
  if (b == p.a.batch) {
    const int t0 = p.a.starts[0], t1 = p.a.starts[p.a.batch];
    for (int t = blockIdx.y * 8 + warp; t < p.a.tokens; t += gridDim.y * 8)
      if (t < t0 || t >= t1)
        for (int hq = 0; hq < p.a.q_heads; ++hq) RowJoin<HD>().write(p, t, hq, lane);
    return;
  }
  const int per_prompt = p.sums[1], per = p.sums[2], before = p.sums[PA_SUMS + b], all = p.sums[PA_SUMS + b + 1] - before;
  const int items = p.sums[PA_SUMS + 1 + p.a.batch + b];
  const Request r = request_of(p, b);
  for (int w = blockIdx.y * 8 + warp; w < r.n * p.a.q_heads; w += gridDim.y * 8) {
    const int i = w / p.a.q_heads, hq = w - i * p.a.q_heads, t = r.t0 + i, h = hq / p.group, head = hq - h * p.group;
    if (t < 0 || t >= p.a.tokens) continue;
    RowJoin<HD> join;
    if (i < r.fresh) {
      const int prt = t / p.tpt, p_item = h * p.prefix_row_tiles + prt, pa = p_item * p.prefix_tiles;
      const int p_first = pa / per_prompt, p_count = (pa + p.prefix_tiles - 1) / per_prompt - p_first + 1;
      const int rt = i / p.tpt, tiles = tiles_of(p, r, rt), item = items * p.a.kv_heads + h * r.row_tiles + rt;
      int first = 0, count = 0;
      if (tiles > 0) {
        int a = before * p.a.kv_heads + h * all;
        for (int k = 0; k < rt; ++k) a += tiles_of(p, r, k);
        first = a / per;
        count = (a + tiles - 1) / per - first + 1;
      }
      join.add(p, p_count + count, [&](int k) -> long long {
        return k < p_count ? prompt_row(p, (long long)p_item + p_first + k) + (t - prt * p.tpt) * p.group + head
                           : own_row(p, (long long)item + first + k - p_count) + (i - rt * p.tpt) * p.group + head;
      }, lane);
    }
    join.write(p, t, hq, lane);
  }
}

// Joint form: the items that a stretch's end cuts (block c: the one that begins in stretch c and goes beyond it), and zeros for the rows of
// no request.
template <int HD>
__global__ void __launch_bounds__(256) paged_join_cuts_kernel(const __grid_constant__ PagedTcParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, per = p.sums[2], work = p.sums[3];
  const long long cut = (long long)(blockIdx.x + 1) * per;       // the first tile of the next stretch
  if (cut < work) {
    Walk walk(p, p.sums + PA_SUMS, p.sums + PA_SUMS + 1 + p.a.batch, false, (int)cut, work);
    Segment s;
    if (walk.next(s) && s.tile > 0 && s.tile <= per) {           // begins in this stretch (at its very first tile at the earliest)
      const int a = (int)cut - s.tile, last = (a + s.item_tiles - 1) / per, c0 = blockIdx.x;
      for (int r = warp; r < s.tokens * p.group; r += 8) {
        RowJoin<HD> join;
        join.add(p, last - c0 + 1, [&](int k) -> long long {      // the piece is the first of its CTA, but for an item that begins inside
          return own_row(p, 2ll * (c0 + k) + ((long long)(c0 + k) * per >= a ? 0 : 1)) + r;
        }, lane);
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
  int group, tpt, ts, tb, copies, copies_prompt, joint, prefix_tiles, prefix_row_tiles, grid;
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
  c.tb = tokens < c.tpt ? tokens : c.tpt;
  c.copies = c.ts * c.group <= 32 ? 4 : 1;
  c.copies_prompt = c.tb * c.group <= 32 ? 4 : 1;
  c.prefix_tiles = (prefix_len + PA_N - 1) / PA_N;
  c.prefix_row_tiles = (tokens + c.tpt - 1) / c.tpt;
  // The prompt for the whole batch at once where that reads it at most half as often as request by request.
  c.joint = prefix_len == 0 || 2ll * c.prefix_row_tiles > batch;
  c.grid = sm_count();
  c.items = ((long long)batch + tokens / c.tpt) * kv_heads;                    // query tiles of single requests, at most
  c.prompt_rows = c.joint ? 0 : ((long long)c.prefix_row_tiles * kv_heads + c.grid) * (c.tb * c.group);
  c.own_rows = (c.joint ? 2ll * c.grid : c.items + c.grid) * (c.ts * c.group);
  c.o_bytes = (size_t)(c.prompt_rows + c.own_rows) * head_dim * sizeof(float);
  c.ml_bytes = (size_t)(c.prompt_rows + c.own_rows) * sizeof(float2);
  c.bytes = c.o_bytes + c.ml_bytes + (2 * ((size_t)batch + 1) + PA_SUMS) * sizeof(int);
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
  p.group = c.group; p.group_mul = 65536 / c.group + 1; p.tpt = c.tpt; p.ts = c.ts; p.tb = c.tb;
  p.copies = c.copies; p.copies_prompt = c.copies_prompt;
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
    const uint32_t box[3] = {64, (uint32_t)c.group, (uint32_t)c.tb}, own[3] = {64, (uint32_t)c.group, (uint32_t)c.ts};
    if ((rc = make_tmap_box3_bf16(&tq, a.q, dims, strides, box)) || (rc = make_tmap_box3_bf16(&tqo, a.q, dims, strides, own))) return rc;
  }
  const uint64_t packed = (uint64_t)a.kv_heads * ps * HD;
  const uint64_t dims[3] = {HD, (uint64_t)a.kv_heads * ps, (uint64_t)a.pages};
  const uint32_t box[3] = {64, (uint32_t)ps, 1};
  const uint64_t ks[2] = {HD * 2, (a.pages > 1 ? (uint64_t)a.k_page_stride : packed) * 2}, vs[2] = {HD * 2, (a.pages > 1 ? (uint64_t)a.v_page_stride : packed) * 2};
  if ((rc = make_tmap_box3_bf16(&tk, a.k, dims, ks, box)) || (rc = make_tmap_box3_bf16(&tv, a.v, dims, vs, box))) return rc;
  launch_short(paged_attn_tc_kernel<HD>, dim3((unsigned)c.grid), dim3(PA_THREADS), Cfg::SMEM_BYTES, st, tq, tqo, tk, tv, p);
  if (c.joint) launch_short(paged_join_cuts_kernel<HD>, dim3((unsigned)c.grid), dim3(256), 0, st, p);
  else {
    const long long rows = (long long)(a.max_fresh > 0 ? a.max_fresh : 1) * a.q_heads;           // of a request, at most
    launch_short(paged_join_rows_kernel<HD>, dim3((unsigned)a.batch + 1, (unsigned)(rows < 8 * 1024 ? (rows + 7) / 8 : 1024)), dim3(256), 0, st, p);
  }
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
