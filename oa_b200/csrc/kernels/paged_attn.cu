// Attention of a batch of requests over a paged key-value cache, behind a prompt that they share.  Query token i of the n new tokens of a
// request sees all `prefix_len` keys of the prompt and the first len - n + i + 1 keys of the request's own pages:
//   o = sum_s softmax_s(scale q . k_s) v_s,   lse = log sum_s exp(scale q . k_s);   a row that sees nothing gives o = 0, lse = -inf.
// A table entry that names no page counts as keys and values of zeros.  Nothing beyond a request's length is read into a result.
#include <type_traits>
#include "common.cuh"
#include "per_device.h"
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
// A query tile is the group of query heads that share a key-value head times tokens, row = token * group + head.  An item is the work of one
// query tile on one key-value head:
//   shared form   the prompt is read once for the whole batch: its items take tokens of the batch as they come, whatever request they
//                 belong to, and each request's own keys make items of their own; every row then has two partial results or more;
//   joint form    where a request's new tokens fill a tile themselves an item sees the prompt's keys and then its own.
// The key tiles of all items, one after the other, are cut into equal stretches, so that a long prompt for few requests and short histories
// for many fill the chip alike.  The part of an item in one stretch is a segment.  Segments that are not a whole result leave (o, m, l) in fp32
// in scratch, and a second launch joins them.  Where everything goes follows from prefix sums over the batch that each CTA makes for
// itself; what the second launch has to know of them is left in scratch.
//
// There are two kinds of CTAs.
//   Many rows (a tile of up to 128, tiles of 128 keys, a stretch to a CTA): tcgen05 with scores, weights and results in TMEM, below.
//   Few rows (up to 8 or 16, the single tokens of decoding above all; tiles of 16 or 32 keys): what counts is that bytes arrive.  A CTA's
//   stretch is dealt to eight warps, each with a ring of three tiles that a warp beside it fills by TMA, one box to a page; no warp waits for
//   another until they join what they have in shared memory.  Scores are K Q^T on mma.sync, keys along M and up to eight rows along N, so
//   that a row is an eighth of an instruction and not 1/128 of a tile, and stay in registers: their exponentials turn into an operand of
//   V^T P^T by a transpose among lanes.  128 requests behind 8191 shared keys with 1024 of their own on average, 8 key-value heads of 64, group 8:
//   own keys arrive at 95 bytes a nanosecond and SM where 72 SMs take them, which is what the memory gives; a tcgen05 tile with 8 of its 128 rows
//   alive took 3300 instructions and 0.75 us for 128 keys (46 bytes a nanosecond and SM).  With all items as tiles of many rows: 109 us, 71 so; 32 requests 41.4
//   and 32.3, 4 requests 22.8 and 19.8.
//   More than 16 rows would need more registers than a thread has.
//
// Keys beyond a length are cut off from the scores by a select, and their values are overwritten by zeros before the product: what lies there
// (the rest of a page, or of the ring) may be anything, NaN included.  Among a request's new tokens the cut is the score's alone: a value that is
// infinite or NaN reaches the earlier tokens in its tile as well, as 0 times it.
//
// Weights are rounded to bf16 before they meet the values: both operands of a product have one type, and values are bf16.  That is 2^-9 of each weight, and
// results are 2.3e-3 from 64 bits (relative, over a whole output) where the rounding of the result alone gives 1.7e-3; weights as two bf16 numbers
// would take the product twice.  Maxima, sums of weights and partial results are fp32.
//
// Many rows.  Warp 15 works out the segments, one after the other, and leaves them in a list of eight in shared memory (every warp on its
// own needed so much code that the warps waited for instructions).  They run through one pipeline of tiles, g = 0, 1, ..:  warps 13 and 14
// load Q (two buffers) and K, and V, by TMA, a box for each page;  warp 12 issues S[g & 1] = Q K_g^T two tiles ahead, and O += P_g V_g, P[g & 1] taken from
// TMEM;  warps 0-3 are the softmax of even tiles, warps 4-7 of odd ones, a thread to a row: the exponentials of one tile run beside the
// waits of the other.  A row's maximum in use goes from tile to tile through shared memory, ahead of the exponentials, so that both sides
// share O;  warps 8-11 write a segment's result out while the next one runs.  The product P_g V_g has a barrier for even and one for odd
// tiles, so that no reader is more than one phase behind.  Scores are read twice, 32 at a time in loops
// that are not unrolled: the code has to fit (128 requests behind 8191 shared keys: 73 us; 64 at a time 80; unrolled, the next 32 on their way
// while these are worked on, 93).  A tile of 128 x 128 takes about 1700 cycles (two threads to a row, all eight warps in the same tile: 2000 and more), of
// which the exponentials keep the special-function units busy for 1000; the rest are round trips to barriers and TMEM (200 each) that two warps to
// a scheduler do not hide.
constexpr int PA_M = 128, PA_N = 128, PA_THREADS = 512, PA_MAX_BATCH = 2048, PA_LIST = 8;
constexpr int PF_WARPS = 8, PF_STAGES = 3, PF_STAGE_BYTES = 8192, PF_KEPT_BYTES = 792;    // few rows: warps, tiles in a warp's ring, K and V of a tile
template <int HD> constexpr int PF_KEYS_LOG2 = HD == 64 ? 5 : 4;       // keys of such a tile
constexpr int PF_ROWS = 16;                                             // and the most rows: what a thread's registers hold
constexpr float PA_RESCALE = 8.f;          // log2: the running maximum is let be while rows grow by less

template <int HD> struct PaCfg {
  static constexpr int NK = HD == 64 ? 4 : 2, NV = HD == 64 ? 4 : 2;
  static constexpr int Q_BYTES = PA_M * HD * 2, T_BYTES = PA_N * HD * 2;
  static constexpr int OFF_Q = 0, OFF_K = 2 * Q_BYTES, OFF_V = OFF_K + NK * T_BYTES;
  static constexpr int OFF_X = PF_WARPS * PF_STAGES * PF_STAGE_BYTES;         // float[2 parities][128]: maxima in use
  static constexpr int OFF_ML = OFF_X + 2 * PA_M * 4;            // float[2 segments][even, odd][m, l][128]
  static constexpr int OFF_BAR = OFF_ML + 2 * 2 * 2 * PA_M * 4, OFF_LIST = OFF_BAR + 512, OFF_SCAN = OFF_LIST + PA_LIST * 48;
  static constexpr int OFF_FEW = OFF_SCAN + 2 * (PA_MAX_BATCH + 1) * 4;        // FewWarp[8]
  static constexpr int SMEM_BYTES = OFF_FEW + PF_WARPS * PF_KEPT_BYTES;
  static_assert(OFF_V + NV * T_BYTES <= OFF_X, "both kinds' rings");
  static constexpr int TM_S = 0, TM_P = 256, TM_O = 384, SETS = HD == 64 ? 2 : 1;      // S and P of two tiles, O of so many segments
};

// Where a token's partial results over its own keys are (shared form): those of key-value head h begin at tile pos + h * all, in item + h * row_tiles.
struct __align__(16) PagedOwn {
  int pos, all, tiles, item, row_tiles;
  int inner;                               // the token in its tile; -1: of no request, or beyond those that one may have
  int pad[2];
};

struct PagedTcParams {
  PagedAttnParams a;
  int group, group_mul, tpt;               // query heads to a key-value head (and 65536 / group + 1: see token_of), tokens in a tile
  int ts, tb;                              // tokens in a box of an own item, of a prompt's item
  int few, few_prompt;                     // few rows: 8 or 16, the most of an item; or 0
  int many;                                // some CTA has a tile of more rows
  int own_log2;                            // keys of a tile of a request's own
  int over;                                // what an item of a request's own costs beside its tiles, in tiles
  int joint, prefix_tiles, prefix_row_tiles, prefix_work;   // prefix_work: key tiles of all prompt items (shared form)
  float* part;                             // partial o: [prompt slots][tb * group][HD], then [own slots][ts * group][HD]
  float2* ml;                              // their (m, l), m in units of log2
  int* sums;                               // Stretches, tiles before a request [batch + 1], query tiles before a request [batch + 1]
  PagedOwn* owns;                          // [tokens], shared form
  long long own_slot0, part_rows;          // rows of the prompt's slots, rows in all
  int ctas;                                // of the first launch: no row has more pieces of one kind
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
  const int own = (seen_by(p, r, rt) + (1 << p.own_log2) - 1) >> p.own_log2;
  return p.joint ? max(p.prefix_tiles + own, 1) : own;
}

// what the item counts in a stretch: units in front that are no tiles, and its tiles
__device__ __forceinline__ int units_of(const PagedTcParams& p, const Request& r, int rt) {
  const int tiles = tiles_of(p, r, rt);
  return tiles > 0 ? tiles + p.over : 0;
}

struct Segment {
  int prompt, h, b, rt;                    // of the prompt's items: rt counts tiles of the whole batch
  int tile, tiles;                         // first key tile inside the item, how many
  int item, item_tiles;
  int t0, tokens, n, own, seen, i0;        // first token and how many; own items: see Request, i0 = index of the first token in the request
};

// How the tiles are dealt: CTAs [0, prompt_ctas) have stretches of `per_prompt` of the prompt's, the others of `per` of the requests'
// each, in which an item counts some tiles more than it has (`over`) for its beginning and its end (few rows 3, many 1, against none: 32 requests 32.2
// and 33.6 us, 128 70.8 and 73.9, ragged pieces 37.4 and 39.4).  With both there, CTAs are dealt in proportion to what the tiles cost: 128 keys of few rows,
// which wait for memory, relative to a tile of 128 keys and many rows (0.31 and 0.4: up to 4% slower at 32 to 128 requests).
constexpr float PA_COST_FEW = 0.37f;
struct Stretches { int prompt_ctas, per_prompt, per, own_work; };
template <int HD>
__device__ __forceinline__ Stretches stretches_of(const PagedTcParams& p, int own_work, int ctas) {
  Stretches d;
  d.own_work = own_work;
  d.prompt_ctas = 0;
  const float few = PA_COST_FEW * (1 << PF_KEYS_LOG2<HD>) / PA_N;      // of a tile of few rows
  if (p.prefix_work > 0) {
    const float prompt = (float)p.prefix_work * (p.few_prompt ? few : 1.f);
    const float own = (float)own_work * (p.few ? few : 1.f);
    d.prompt_ctas = own_work > 0 ? min(max((int)((float)ctas * prompt / (prompt + own) + 0.5f), 1), ctas - 1) : ctas;
  }
  d.per_prompt = max((p.prefix_work + max(d.prompt_ctas, 1) - 1) / max(d.prompt_ctas, 1), 1);
  d.per = max((own_work + ctas - d.prompt_ctas - 1) / max(ctas - d.prompt_ctas, 1), 1);
  return d;
}

// The segments of a stretch [pos, end) of the prompt's or the requests' key tiles, in order.
struct Walk {
  const PagedTcParams& p;
  const int *tiles_before, *items_before;
  int pos, end;
  int b, h, rt, unit;                      // own items: the next one and the unit in it
  Request r;
  bool prompt, placed;
  __device__ __forceinline__ Walk(const PagedTcParams& p_, const int* tb, const int* ib, bool prompt_, int pos_, int end_)
      : p(p_), tiles_before(tb), items_before(ib), pos(pos_), end(end_), b(0), h(0), rt(0), unit(0), prompt(prompt_), placed(false) {}
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
    for (int t = units_of(p, r, 0); off >= t && rt + 1 < r.row_tiles; t = units_of(p, r, rt)) { off -= t; ++rt; }
    unit = off;
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
      s.tiles = min(s.item_tiles - s.tile, end - pos);
      pos += s.tiles;
      return true;
    }
    if (!placed) { const int at = find(); place(at, request_of(p, at)); }
    while (rt >= r.row_tiles || units_of(p, r, rt) <= unit) {        // on to the next item that has tiles; there is one before `end`
      unit = 0;
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
    s.item_tiles = tiles_of(p, r, rt);
    s.item = items_before[b] * p.a.kv_heads + h * r.row_tiles + rt;
    s.i0 = rt * p.tpt;
    s.t0 = r.t0 + s.i0;
    s.tokens = min(p.tpt, r.fresh - s.i0);
    s.n = r.n;
    s.own = r.own;
    s.seen = seen_by(p, r, rt);
    const int step = min(s.item_tiles + p.over - unit, end - pos);
    s.tile = max(unit - p.over, 0);
    s.tiles = max(unit + step - p.over, 0) - s.tile;
    pos += step;
    unit += step;
    return s.tiles > 0;                    // none: the stretch ends in front of the item's tiles
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
__device__ __forceinline__ void scan_batch(const PagedTcParams& p, int* tiles_before, int* items_before, int* warp_sums, int& all_tiles) {
  constexpr int WARPS = PA_THREADS / 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (p.a.batch + PA_THREADS - 1) / PA_THREADS, b0 = min(tid * per, p.a.batch), b1 = min(b0 + per, p.a.batch);
  int tiles = 0, items = 0;
  for (int b = b0; b < b1; ++b) {
    const Request r = request_of(p, b);
    tiles_before[b] = tiles;
    items_before[b] = items;
    for (int rt = 0; rt < r.row_tiles; ++rt) tiles += units_of(p, r, rt);
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
}

// Where a partial result goes.  Shared form: every segment of every item, numbered by item + stretch (a segment begins where an item or a
// stretch does).  Joint form: only items that a stretch's end cuts, of which a CTA has its first and its last segment.
__device__ __forceinline__ long long own_row(const PagedTcParams& p, long long slot) { return p.own_slot0 + slot * (p.ts * p.group); }
__device__ __forceinline__ long long prompt_row(const PagedTcParams& p, long long slot) { return slot * (p.tb * p.group); }
// Starts that do not rise would make more items than there is room for: their rows stay out of the scratch.
__device__ __forceinline__ bool has_room(const PagedTcParams& p, long long row) { return row >= 0 && row < p.part_rows; }

// ---- few rows
__device__ __forceinline__ void ldmatrix_x4(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_t(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {      // an 8 x 8 matrix of 16 bits, a row to four lanes
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ void mma_16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// What a warp keeps in shared memory beside its ring.
// tiles: 0, no more; shift: the row of token i sees own keys before shift + i; flags: 1 begins in a warp before, 2 goes on in the next, 4 the slot of its last tile
// is kept for its results
struct FewSegment { int tile, tiles, item, h, t0, rows, seen, shift, flags, pad[3]; };
struct FewPart { int rows, goes_on, at; float2 ml[PF_ROWS]; };                   // rows 0: none; `at`: where its o lies in the ring
struct FewWarp {
  uint64_t full[PF_STAGES], empty[PF_STAGES], listed[8];
  FewSegment list[8];                      // of which the warp is in one, and its loads at most five ahead: none is written before it has been read
  FewPart front, back;                     // what is to be joined with the warp before, and with the warp behind
  int item;                                // of `back`
  int pad;
};
static_assert(sizeof(FewWarp) == PF_KEPT_BYTES, "what is set aside for it");

__device__ __forceinline__ int few_step(int x, int hole) {        // the next slot of a ring
  x = x + 1 == PF_STAGES ? 0 : x + 1;
  if (x == hole) x = x + 1 == PF_STAGES ? 0 : x + 1;
  return x;
}
// The loads of warp `warp`, whose part of the CTA's stretch [lo, hi) is an eighth, by a warp beside it: chunks of up to 32 pages of a segment, the pages of the next chunk looked up while this one's
// tiles are loaded.
template <int HD>
__device__ __forceinline__ void few_loads(const PagedTcParams& p, const CUtensorMap* tmK, const CUtensorMap* tmV, uint8_t* ring, FewWarp& mine, int warp,
                                          const int* tiles_before, const int* items_before, bool prompt, int lo, int hi) {
  constexpr int UL = PF_KEYS_LOG2<HD>, U = 1 << UL, CHUNKS = HD / 64, KV = U * HD * 2;
  const int lane = threadIdx.x & 31;
  const int lg = p.a.page_log2, box = min(1 << lg, U), boxes_log2 = max(UL - lg, 0);         // rows of a box; boxes of a tile
  const int part = (hi - lo + PF_WARPS - 1) / PF_WARPS, from = min(lo + warp * part, hi), to = min(from + part, hi);
  struct Chunk { int n, k0, end, h, id; };
  Walk walk(p, tiles_before, items_before, prompt, from, to);
  Chunk now{0, 0, 0, 0, 0}, then{0, 0, 0, 0, 0};
  int seg_h = 0, seg_b = 0, seg_tile = 0, seg_left = 0, seg_end = 0, seg_at = 0, used = 0, st = 0, hole = -1;
  bool ended = false;
  int keeps = 0;                           // the tile whose slot the warp keeps, counted from 1; 0: none
  const auto fetch = [&](Chunk& c) {
    c.n = 0;
    if (seg_left == 0) {
      Segment s{};
      if (ended) return;
      ended = !walk.next(s);
      const bool front = seg_at == 0 && s.tile > 0 && from > lo, back = walk.pos == to && to < hi && s.tile + s.tiles < s.item_tiles, kept = front && walk.pos < to;
      if (lane == 0) {
        mine.list[seg_at & 7] = FewSegment{s.tile, ended ? 0 : s.tiles, s.item, s.h, s.t0, s.tokens * p.group, s.seen, s.own - s.n + s.i0 + 1, (front ? 1 : 0) | (back ? 2 : 0) | (kept ? 4 : 0)};
        mbar_arrive(&mine.listed[seg_at & 7]);
      }
      if (ended) return;
      if (kept) keeps = s.tiles;
      ++seg_at;
      seg_h = s.h; seg_b = s.b; seg_tile = s.tile; seg_left = s.tiles;
      seg_end = prompt ? p.a.prefix_len : s.seen;
      const int t = s.t0 + lane / (p.group * CHUNKS), off = lane % (p.group * CHUNKS) * 64;           // its queries on their way to L2
      if (lane < s.tokens * p.group * CHUNKS && t >= 0 && t < p.a.tokens)
        asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const __nv_bfloat16*>(p.a.q) + (long long)t * p.a.q_stride + s.h * p.group * HD + off));
    }
    c.n = min(seg_left, 32 >> boxes_log2);
    c.k0 = seg_tile << UL;
    c.end = seg_end;
    c.h = seg_h;
    c.id = -1;
    if (lane * box < min(c.n << UL, c.end - c.k0)) {
      const int at = (c.k0 + lane * box) >> lg;
      c.id = prompt ? p.a.prefix_table[at] : p.a.tables[seg_b * p.a.table_stride + at];
    }
    seg_tile += c.n;
    seg_left -= c.n;
  };
  fetch(now);
  if (now.n > 0) fetch(then);
  uint32_t phases = (1u << PF_STAGES) - 1;                       // a bit for each slot: free at first
#pragma unroll 1
  while (now.n > 0) {
    const int boxes = (min(U, now.end - now.k0) + box - 1) / box, id = __shfl_sync(0xffffffffu, now.id, (used << boxes_log2) + lane);
    if (!warp_wait(&mine.empty[st], phases >> st & 1)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_EMPTY); return; }
    phases ^= 1u << st;
    if (lane == 0) mbar_expect_tx(&mine.full[st], (uint32_t)(boxes * box * HD * 4));
    __syncwarp();
    if (lane < boxes) {
      uint8_t* at = ring + st * PF_STAGE_BYTES + lane * box * 128;
      const int y = (now.h << lg) + ((now.k0 + lane * box) & ((1 << lg) - 1));
#pragma unroll
      for (int x = 0; x < CHUNKS; ++x) {
        tma_load_3d(at + x * (U * 128), tmK, &mine.full[st], x * 64, y, id);
        tma_load_3d(at + KV + x * (U * 128), tmV, &mine.full[st], x * 64, y, id);
      }
    }
    __syncwarp();
    if (--keeps == 0) hole = st;
    st = few_step(st, hole);
    now.k0 += U;
    ++used;
    if (--now.n == 0) {
      now = then;
      used = 0;
      if (now.n > 0) fetch(then);
    }
  }
}

// Warp `warp` of eight, NT groups of eight rows.
template <int HD, int NT>
__device__ __forceinline__ void few_rows(const PagedTcParams& p, uint8_t* rings, FewWarp* all, bool prompt, int cta) {
  constexpr int UL = PF_KEYS_LOG2<HD>, U = 1 << UL, MT = U / 16, KC = HD / 16, KV = U * HD * 2, PER = HD / 32;
  static_assert(2 * KV == PF_STAGE_BYTES && NT * 8 * HD * 4 <= PF_STAGE_BYTES, "a tile of K and of V, or results");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, quad = lane >> 2, pair = (lane & 3) * 2;
  const float sl2 = p.a.scale * 1.4426950408889634f;
  uint8_t* ring = rings + warp * (PF_STAGES * PF_STAGE_BYTES);
  FewWarp& mine = all[warp];
  int st = 0, sg = 0, hole = -1;
  uint32_t phases = 0;                     // a bit for each slot
  bool ok = true;
  if (lane == 0) mine.front.rows = mine.back.rows = 0;
#pragma unroll 1
  while (ok) {
    if (!warp_wait(&mine.listed[sg & 7], sg >> 3 & 1)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_FULL); break; }
    const FewSegment s = mine.list[sg & 7];
    if (s.tiles == 0) break;
    ++sg;
    uint32_t q[KC][NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int row = n * 8 + quad, i = token_of(p, row), t = s.t0 + i;
      const bool there = row < s.rows && t >= 0 && t < p.a.tokens;
      const __nv_bfloat16* at = static_cast<const __nv_bfloat16*>(p.a.q) + (long long)t * p.a.q_stride + (s.h * p.group + row - i * p.group) * HD + pair;
#pragma unroll
      for (int k = 0; k < KC; ++k) {
        q[k][n][0] = there ? *reinterpret_cast<const uint32_t*>(at + k * 16) : 0u;
        q[k][n][1] = there ? *reinterpret_cast<const uint32_t*>(at + k * 16 + 8) : 0u;
      }
    }
    float o[KC][NT][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) { m[n][e] = -INFINITY; l[n][e] = 0.f; }
#pragma unroll
    for (int k = 0; k < KC; ++k)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[k][n][e] = 0.f;
    const int most = prompt ? p.a.prefix_len : s.seen, least = prompt ? most : min(s.shift, most);
    const bool front = s.flags & 1, back = s.flags & 2;
#pragma unroll 1
    for (int j = 0; j < s.tiles; ++j) {
      const int k0 = (s.tile + j) << UL;
      if (!warp_wait(&mine.full[st], phases >> st & 1)) {
        if (lane == 0) report_error(p.status, OA_KERR_WAIT_FULL);
        for (int i = 1; i < PF_STAGES; ++i) {                    // copies that may still be under way
          st = few_step(st, hole);
          warp_wait(&mine.full[st], phases >> st & 1);
        }
        ok = false;
        break;
      }
      phases ^= 1u << st;
      const uint32_t kt = smem_u32(ring + st * PF_STAGE_BYTES), vt = kt + KV;
      float c[MT][NT][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) c[mt][n][e] = 0.f;
        const int row = mt * 16 + (lane & 15);
#pragma unroll
        for (int k = 0; k < KC; ++k) {
          uint32_t a[4];
          ldmatrix_x4(kt + (k >> 2) * (U * 128) + row * 128 + ((((k & 3) * 2 + (lane >> 4)) ^ (row & 7)) << 4), a);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_16816(c[mt][n], a, q[k][n][0], q[k][n][1]);
        }
      }
      if (k0 + U > least) {                // -inf for what is not seen, zeros over values that no key goes with
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int see = prompt ? most : min(s.shift + token_of(p, n * 8 + pair + e), most);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              if (k0 + mt * 16 + quad >= see) c[mt][n][e] = -INFINITY;
              if (k0 + mt * 16 + quad + 8 >= see) c[mt][n][e + 2] = -INFINITY;
            }
          }
        if (k0 + U > most) {
          for (int i = lane; i < (k0 + U - most) * (HD / 8); i += 32) {
            const int key = most - k0 + i / (HD / 8), x = i % (HD / 8);
            st_shared_v4(vt + (x >> 3) * (U * 128) + key * 128 + (x & 7) * 16, make_uint4(0, 0, 0, 0));
          }
          fence_proxy_async_smem();        // before the copy that comes here next
          __syncwarp();
        }
      }
      // the running maximum is let be while no row of the warp grows by more than 2^8
      float top[NT][2];
      bool grow = false;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float t = fmaxf(c[0][n][e], c[0][n][e + 2]);
#pragma unroll
          for (int mt = 1; mt < MT; ++mt) t = fmax3(t, c[mt][n][e], c[mt][n][e + 2]);
          top[n][e] = t * sl2;
          grow |= top[n][e] - m[n][e] > PA_RESCALE;
        }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float t = top[n][e];
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, x));
            if (t > m[n][e]) {
              const float alpha = fast_exp2(m[n][e] - t);        // 0 from -inf
              m[n][e] = t;
              l[n][e] *= alpha;
#pragma unroll
              for (int k = 0; k < KC; ++k) { o[k][n][e] *= alpha; o[k][n][e + 2] *= alpha; }
            }
          }
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        uint32_t w[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float base = m[n][e & 1] == -INFINITY ? 0.f : m[n][e & 1];     // a row that has seen nothing yet
            c[mt][n][e] = fast_exp2(fmaf(c[mt][n][e], sl2, -base));
            l[n][e & 1] += c[mt][n][e];
          }
          // weights to bf16, as the products take them; their sum stays fp32
          w[n][0] = transpose8(pack_bf16x2(c[mt][n][0], c[mt][n][1]));
          w[n][1] = transpose8(pack_bf16x2(c[mt][n][2], c[mt][n][3]));
        }
        const int key = mt * 16 + (lane & 7) + (lane >> 4) * 8;
#pragma unroll
        for (int k = 0; k < KC; ++k) {
          uint32_t a[4];
          ldmatrix_x4_t(vt + (k >> 2) * (U * 128) + key * 128 + ((((k & 3) * 2 + ((lane >> 3) & 1)) ^ (key & 7)) << 4), a);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_16816(o[k][n], a, w[n][0], w[n][1]);
        }
      }
      __syncwarp();
      if (j + 1 == s.tiles && (s.flags & 4)) hole = st;          // this slot keeps the results that another warp joins
      else if (lane == 0) mbar_arrive(&mine.empty[st]);
      st = few_step(st, hole);
    }
    // Results: a segment that ends where another warp goes on waits for it in shared memory, the others go to scratch.
    const long long at = prompt ? prompt_row(p, (long long)s.item + cta) : own_row(p, (long long)s.item + cta);
    FewPart& kept = front ? mine.front : mine.back;
    const int slot = front ? (hole >= 0 ? hole : 0) : (hole == 0 ? 1 : 0);       // of the ring, in which nothing is under way
    if ((front || back) && lane == 0) {
      kept.rows = s.rows;
      kept.goes_on = back;
      kept.at = slot * PF_STAGE_BYTES;
      mine.item = s.item;
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = n * 8 + pair + e;
        float sum = l[n][e];
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
        if (row < s.rows) {
          float* to_o;
          float2* to_ml;
          if (front || back) { to_o = reinterpret_cast<float*>(ring + slot * PF_STAGE_BYTES) + row * HD; to_ml = &kept.ml[row]; }
          else { to_o = p.part + (at + row) * HD; to_ml = p.ml + at + row; }
          if (front || back || has_room(p, at + row)) {
            if (quad == 0) *to_ml = make_float2(m[n][e], sum);
#pragma unroll
            for (int k = 0; k < KC; ++k) { to_o[k * 16 + quad] = o[k][n][e]; to_o[k * 16 + quad + 8] = o[k][n][e + 2]; }
          }
        }
      }
  }
  // Joins what the warps have left, a row to a warp, in the order of the keys.
  asm volatile("bar.sync 1, 256;" ::: "memory");
#pragma unroll 1
  for (int w = 0; w < PF_WARPS; ++w) {
    if (all[w].back.rows == 0) continue;
    const long long at = prompt ? prompt_row(p, (long long)all[w].item + cta) : own_row(p, (long long)all[w].item + cta);
#pragma unroll 1
    for (int row = warp; row < all[w].back.rows; row += PF_WARPS) {
      float m = -INFINITY, l = 0.f, acc[PER] = {};
#pragma unroll 1
      for (int x = w; x < PF_WARPS; ++x) {
        const FewPart& f = x == w ? all[x].back : all[x].front;
        if (x > w && f.rows == 0) break;
        const float2 ml = f.ml[row];
        const float* o = reinterpret_cast<const float*>(rings + x * (PF_STAGES * PF_STAGE_BYTES) + f.at) + row * HD + lane * PER;
        if (ml.y != 0.f) {                 // otherwise a part of which this row saw nothing
          const float top = fmaxf(m, ml.x), a = m == -INFINITY ? 0.f : fast_exp2(m - top), b = ml.x == -INFINITY ? 1.f : fast_exp2(ml.x - top);
          l = l * a + ml.y * b;
#pragma unroll
          for (int e = 0; e < PER; ++e) acc[e] = acc[e] * a + o[e] * b;
          m = top;
        }
        if (x > w && !f.goes_on) break;
      }
      if (!has_room(p, at + row)) continue;
      if (lane == 0) p.ml[at + row] = make_float2(m, l);
      float* part_o = p.part + (at + row) * HD + lane * PER;
      if (PER == 4) *reinterpret_cast<float4*>(part_o) = make_float4(acc[0], acc[1], acc[PER - 2], acc[PER - 1]);
      else *reinterpret_cast<float2*>(part_o) = make_float2(acc[0], acc[1]);
    }
  }
}

// NT: 1, or 2 where some item may have 9 to 16 rows (the registers of which, at head dim 128, spill: 3% of a call that does without)
template <int HD, int NT>
__global__ void __launch_bounds__(PA_THREADS, 1)
paged_attn_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmQown, const __grid_constant__ CUtensorMap tmK,
                     const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmKfew, const __grid_constant__ CUtensorMap tmVfew,
                     const __grid_constant__ PagedTcParams p) {
  using Cfg = PaCfg<HD>;
  constexpr int NK = Cfg::NK, NV = Cfg::NV, CHUNKS = HD / 64;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ int s_warp_sums[2 * PA_THREADS / 32];
  __shared__ int s_first;
  __shared__ Request s_request;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::OFF_BAR);
  uint64_t *q_full = bars, *q_empty = bars + 2, *k_full = bars + 4, *k_empty = k_full + NK, *v_full = k_empty + NK, *v_empty = v_full + NV;
  uint64_t *s_full = v_empty + NV, *p_full = s_full + 2, *o_done = s_full + 4, *o_free = s_full + 6, *seg_done = s_full + 8, *o_full = s_full + 10, *s_free = s_full + 12, *seg_free = s_full + 14;
  uint64_t *listed = s_full + 16, *list_free = listed + PA_LIST, *m_there = list_free + PA_LIST;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(m_there + 8);
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
  // `many`: some CTA may have many rows
  if (p.many && threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1); mbar_init(&q_empty[i], 1); mbar_init(&s_full[i], 1); mbar_init(&s_free[i], 4); mbar_init(&p_full[i], 4);
      mbar_init(&o_done[i], 1); mbar_init(&o_full[i], 1); mbar_init(&o_free[i], 4); mbar_init(&seg_done[i], 8); mbar_init(&seg_free[i], 4);
    }
    for (int i = 0; i < NK; ++i) { mbar_init(&k_full[i], 1); mbar_init(&k_empty[i], 1); }
    for (int i = 0; i < NV; ++i) { mbar_init(&v_full[i], 1); mbar_init(&v_empty[i], 1); }
    for (int i = 0; i < 8; ++i) mbar_init(&m_there[i], 1);
    for (int i = 0; i < PA_LIST; ++i) { mbar_init(&listed[i], 1); mbar_init(&list_free[i], 15); }
    mbar_fence_init();
  }
  if (p.many && warp == 12) { tmem_alloc<512>(tmem_slot); tmem_relinquish(); }
  if (p.many && warp == 13 && lane == 0) { tma_prefetch_desc(&tmQ); tma_prefetch_desc(&tmQown); tma_prefetch_desc(&tmK); tma_prefetch_desc(&tmV); }
  if (warp >= 16 - PF_WARPS && lane == 0 && (p.few || p.few_prompt)) {           // barriers of the few rows' rings
    FewWarp& f = reinterpret_cast<FewWarp*>(smem + Cfg::OFF_FEW)[warp - (16 - PF_WARPS)];
    for (int i = 0; i < PF_STAGES; ++i) { mbar_init(&f.full[i], 1); mbar_init(&f.empty[i], 1); }
    for (int i = 0; i < 8; ++i) mbar_init(&f.listed[i], 1);
    mbar_fence_init();
    tma_prefetch_desc(&tmKfew);
    tma_prefetch_desc(&tmVfew);
  }
  pdl_wait();
  {                                        // tables on their way to L2 while the lengths arrive: 128 bytes to a thread
    const int lines = (p.a.width + 31) / 32, at = blockIdx.x * PA_THREADS + threadIdx.x;
    for (int i = at; i < p.a.batch * lines; i += gridDim.x * PA_THREADS)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(p.a.tables + (long long)(i / lines) * p.a.table_stride + min(i % lines * 32, p.a.width - 1)));
    if (at * 32 < p.a.prefix_len >> p.a.page_log2) asm volatile("prefetch.global.L2 [%0];" ::"l"(p.a.prefix_table + at * 32));
  }
  int own_tiles;
  scan_batch(p, tiles_before, items_before, s_warp_sums, own_tiles);
  __syncthreads();
  const Stretches deal = stretches_of<HD>(p, own_tiles * p.a.kv_heads, gridDim.x);
  const bool on_prompt = (int)blockIdx.x < deal.prompt_ctas;
  const int cta = on_prompt ? blockIdx.x : blockIdx.x - deal.prompt_ctas, per = on_prompt ? deal.per_prompt : deal.per;
  const int work = on_prompt ? p.prefix_work : deal.own_work;
  // for the second launch
  if (blockIdx.x == 0 && threadIdx.x == 0) { p.sums[0] = deal.prompt_ctas; p.sums[1] = deal.per_prompt; p.sums[2] = deal.per; p.sums[3] = deal.own_work; }
  if (p.joint) {
    if (blockIdx.x == 0)
      for (int b = threadIdx.x; b <= p.a.batch; b += PA_THREADS) { p.sums[PA_SUMS + b] = tiles_before[b]; p.sums[PA_SUMS + 1 + p.a.batch + b] = items_before[b]; }
  } else {
    const auto none = [&](int from, int to) {                    // tokens of no request
      for (int t = max(from, 0) + threadIdx.x; t < min(to, p.a.tokens); t += PA_THREADS) p.owns[t].inner = -1;
    };
    for (int b = blockIdx.x; b < p.a.batch; b += gridDim.x) {
      const Request r = request_of(p, b);
      if (b == 0) none(0, r.t0);
      if (b == p.a.batch - 1) none(r.t0 + r.n, p.a.tokens);
      for (int i = threadIdx.x; i < r.n; i += PA_THREADS) {
        if (r.t0 + i < 0 || r.t0 + i >= p.a.tokens) continue;
        const int rt = i / p.tpt;
        PagedOwn o{tiles_before[b] * p.a.kv_heads + p.over, tiles_before[b + 1] - tiles_before[b], tiles_of(p, r, rt), items_before[b] * p.a.kv_heads + rt, r.row_tiles,
                   i < r.fresh ? i - rt * p.tpt : -1, {0, 0}};
        for (int k = 0; k < rt; ++k) o.pos += units_of(p, r, k);
        p.owns[r.t0 + i] = o;
      }
    }
  }
  if (const int few = on_prompt ? p.few_prompt : p.few) {
    if (p.many && warp == 12) tmem_dealloc<512>(*tmem_slot);
    const int from = (int)min((long long)cta * per, (long long)work), to = (int)min((long long)(cta + 1) * per, (long long)work);
    FewWarp* all = reinterpret_cast<FewWarp*>(smem + Cfg::OFF_FEW);
    if (warp >= PF_WARPS) {
      few_loads<HD>(p, &tmKfew, &tmVfew, smem + (warp - PF_WARPS) * (PF_STAGES * PF_STAGE_BYTES), all[warp - PF_WARPS], warp - PF_WARPS, tiles_before, items_before,
                    on_prompt, from, to);
    } else if (NT == 1 || few == 8) {
      few_rows<HD, 1>(p, smem, all, on_prompt, cta);
    } else {
      few_rows<HD, NT>(p, smem, all, on_prompt, cta);
    }
    return;
  }
  const int lo = (int)min((long long)cta * per, (long long)work), hi = (int)min((long long)(cta + 1) * per, (long long)work);
  if (!on_prompt)                          // the request in which the stretch begins, by the thread that has scanned it
    for (int b = threadIdx.x * ((p.a.batch + PA_THREADS - 1) / PA_THREADS), k = 0; k < (p.a.batch + PA_THREADS - 1) / PA_THREADS && b < p.a.batch; ++k, ++b)
      if (lo >= tiles_before[b] * p.a.kv_heads && lo < tiles_before[b + 1] * p.a.kv_heads) { s_first = b; s_request = request_of(p, b); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

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
          mbar_expect_tx(&q_full[qb], (uint32_t)(((s.flags & 1) ? p.tb : p.ts) * p.group * HD * 2));
#pragma unroll
          for (int x = 0; x < CHUNKS; ++x) tma_load_3d(smem + Cfg::OFF_Q + qb * Cfg::Q_BYTES + x * (PA_M * 128), mq, &q_full[qb], x * 64, h * p.group, s.t0);
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
    // ---------------------------------------------------------------- products, in the order in which the softmax comes to want them: S of g + 2, P V of g
    constexpr uint32_t idesc_qk = umma_idesc_bf16(PA_M, PA_N, 0, 0), idesc_pv = umma_idesc_bf16(PA_M, HD, 0, 1);
    const uint64_t q_desc = umma_smem_desc_sw128(smem_u32(smem + Cfg::OFF_Q), 16, 1024), k_desc = umma_smem_desc_sw128(smem_u32(smem + Cfg::OFF_K), 16, 1024);
    const uint64_t v_desc = umma_smem_desc_sw128(smem_u32(smem + Cfg::OFF_V), PA_N * 128, 1024);
    int gq = 0, jq = 0, nq = 0, sqq = -1, lq = 0;                 // of the score products: tile, tile in the segment, its tiles, segment, list entry
    uint32_t lqphase = 0;
    bool q_end = false;
    const auto product_qk = [&] {
      if (q_end) return;
      const int st = gq % NK;
      bool there = true;
      if (jq == nq) {
        there = mbar_wait(&listed[lq], lqphase);
        nq = there ? list[lq].tiles : 0;
        jq = 0;
        if (nq == 0) { q_end = true; ok = __all_sync(0xffffffffu, there) && ok; return; }
        ++sqq;
        if (++lq == PA_LIST) { lq = 0; lqphase ^= 1; }
        there = mbar_wait(&q_full[sqq & 1], (sqq >> 1) & 1);
      }
      there = there && mbar_wait(&k_full[st], (gq / NK) & 1) && mbar_wait(&s_free[gq & 1], ((gq >> 1) & 1) ^ 1);
      ok = __all_sync(0xffffffffu, there) && ok;
      if (!ok) return;
      tc_fence_after();
      if (elect_one()) {
        const uint64_t qd = q_desc + ((sqq & 1) * Cfg::Q_BYTES >> 4), kd = k_desc + (st * Cfg::T_BYTES >> 4);
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks) {
          const uint32_t off = ((ks >> 2) * (PA_M * 128) + (ks & 3) * 32) >> 4;
          umma_f16(tmem_base + Cfg::TM_S + (gq & 1) * PA_N, qd + off, kd + off, idesc_qk, ks > 0 ? 1u : 0u);
        }
        umma_commit(&s_full[gq & 1]);
        umma_commit(&k_empty[st]);
        if (jq + 1 == nq) umma_commit(&q_empty[sqq & 1]);
      }
      __syncwarp();
      ++jq; ++gq;
    };
    int g = 0, sq = 0, j = 0, n = 0;                              // of P V
#pragma unroll 1
    for (int ahead = 0; ok; ++ahead) {
      product_qk();
      if (ahead < 2 && !q_end) continue;                          // two scores before the first P V
      if (!ok) break;
      if (j == n) {                                               // the segment of the next product
        if (!take(s, ok)) break;
        let_go();
        n = s.tiles;
        j = 0;
      }
      const int st = g % NV, set = sq % Cfg::SETS;
      bool there = j > 0 || mbar_wait(&o_free[set], ((sq / Cfg::SETS) & 1) ^ 1);        // the result there before has been read
      there = there && mbar_wait(&v_full[st], (g / NV) & 1) && mbar_wait(&p_full[g & 1], (g >> 1) & 1);
      ok = __all_sync(0xffffffffu, there);
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
        const uint64_t vd = v_desc + (st * Cfg::T_BYTES >> 4);
#pragma unroll
        for (int ks = 0; ks < PA_N / 16; ++ks)
          umma_f16_ts(tmem_base + Cfg::TM_O + set * HD, tmem_base + Cfg::TM_P + (g & 1) * 64 + ks * 8, vd + (ks * 2048 >> 4), idesc_pv, (j > 0 || ks > 0) ? 1u : 0u);
        umma_commit(&o_done[g & 1]);
        umma_commit(&v_empty[st]);
        if (j + 1 == n) umma_commit(&o_full[sq & 1]);
      }
      __syncwarp();
      ++g;
      if (++j == n) ++sq;
    }
    if (!ok && lane == 0) report_error(p.status, OA_KERR_WAIT_SOFTMAX);
  } else if (warp < 8) {
    // ---------------------------------------------------------------- softmax: warp w has TMEM lanes 32 (w % 4).. of even (w < 4) or odd tiles
    const int quad = warp & 3, grp = warp >> 2, r = quad * 32 + lane;
    const int i_row = token_of(p, r);                             // token of this row in the tile
    const uint32_t t_lane = tmem_base + ((uint32_t)(quad * 32) << 16);
    const uint32_t s_addr = t_lane + Cfg::TM_S + grp * PA_N, p_addr = t_lane + Cfg::TM_P + grp * (PA_N / 2);
    const float sl2 = p.a.scale * 1.4426950408889634f;
    const unsigned long long sl22 = f2_splat(sl2);
    float* xch = reinterpret_cast<float*>(smem + Cfg::OFF_X);     // a row's maximum in use, by the even or odd tile that has set it
    int g0 = 0, sq = 0;
#pragma unroll 1
    while (ok && take(s, ok)) {
      let_go();
      const bool live = quad * 32 < s.rows;                       // of this warp: some row is there
      float m_run = -INFINITY, l_run = 0.f;
      const uint32_t o_addr = t_lane + Cfg::TM_O + sq % Cfg::SETS * HD;
#pragma unroll 1
      for (int j = (g0 ^ grp) & 1; j < s.tiles; j += 2) {
        const int g = g0 + j;
        const KeyTile kt = key_tile(p, s.flags, s.seen, s.tile + j);
        ok = warp_wait(&s_full[grp], (g >> 1) & 1);
        if (!ok) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_TMEM_FULL); break; }
        tc_fence_after();
        // columns up to `last` are seen: the keys that there are, and of a request's own keys those up to the row's token
        const int last = kt.prompt ? kt.count - 1 : min(kt.count - 1, s.shift + i_row - kt.first);
        const bool cut = (kt.prompt ? kt.count - 1 : min(kt.count - 1, s.shift - kt.first)) < PA_N - 1;
        float mx = -INFINITY;
        if (live) {
#pragma unroll 1
          for (int c0 = 0; c0 < PA_N; c0 += 32) {
            uint32_t sv[32];
            tmem_ld32(s_addr + c0, sv);
            tmem_ld_wait();
            if (cut) {                                            // -inf for those that are not seen, here and for the weights
              const int lim = last - c0;
#pragma unroll
              for (int i = 0; i < 32; ++i) sv[i] = i <= lim ? sv[i] : 0xff800000u;
              tmem_st32(s_addr + c0, sv);
              tmem_st_wait();
            }
            float m1 = __uint_as_float(sv[0]);
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              mx = fmax3(mx, __uint_as_float(sv[i]), __uint_as_float(sv[i + 1]));
              m1 = fmax3(m1, __uint_as_float(sv[i + 2]), __uint_as_float(sv[i + 3]));
            }
            mx = fmaxf(mx, m1);
          }
        }
        // the maximum in use goes from tile to tile: from the other warps' to this one, and on
        ok = g == 0 || mbar_wait(&m_there[(grp ^ 1) * 4 + quad], ((g - 1) >> 1) & 1);
        const float m_old = j == 0 ? -INFINITY : xch[(grp ^ 1) * PA_M + r];
        const float m_new = fmaxf(m_old, mx * sl2);
        const bool grow = r < s.rows && (m_new - m_old) > PA_RESCALE;           // the first time: from -inf.  Not for rows that are not there, whose scores are anything
        const float m_cand = grow ? m_new : m_old;
        xch[grp * PA_M + r] = m_cand;
        __syncwarp();
        if (lane == 0) mbar_arrive(&m_there[grp * 4 + quad]);
        // P of the tile before the last has been used: its place is free
        ok = ok && (g < 2 || mbar_wait(&o_done[grp], ((g - 2) >> 1) & 1));
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_SOFTMAX); break; }
        tc_fence_after();
        if (!live) {
          if (lane == 0) mbar_arrive(&s_free[grp]);
        } else {
          const float m_use = m_cand == -INFINITY ? 0.f : m_cand; // a row that has seen nothing yet
          const unsigned long long neg_m = f2_splat(-m_use);
          unsigned long long l01 = 0, l23 = 0;
#pragma unroll 1
          for (int c0 = 0; c0 < PA_N; c0 += 32) {
            uint32_t sv[32], pk[16];
            tmem_ld32(s_addr + c0, sv);
            tmem_ld_wait();
            if (c0 + 32 == PA_N) {                                // all have been read
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&s_free[grp]);
            }
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              const unsigned long long e01 = exp2_mufu2(f2_fma(f2_of(sv[i], sv[i + 1]), sl22, neg_m)), e23 = exp2_mufu2(f2_fma(f2_of(sv[i + 2], sv[i + 3]), sl22, neg_m));
              l01 = f2_add(l01, e01);
              l23 = f2_add(l23, e23);
              pk[i >> 1] = f2_bf16(e01);                          // weights to bf16, as the tensor cores take them; their sum stays fp32
              pk[(i >> 1) + 1] = f2_bf16(e23);
            }
            tmem_st16(p_addr + (c0 >> 1), pk);
          }
          uint32_t a, b;
          f2_to(f2_add(l01, l23), a, b);
          l_run = (m_run == m_cand ? l_run : l_run * fast_exp2(m_run - m_use)) + (__uint_as_float(a) + __uint_as_float(b));
          m_run = m_cand;
          if (j > 0 && __any_sync(0xffffffffu, grow)) {           // O again to the new maximum, behind the product before
            const float alpha = grow ? fast_exp2(m_old - m_use) : 1.f;
            ok = warp_wait(&o_done[grp ^ 1], ((g - 1) >> 1) & 1);
            if (!ok) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_TMEM_FULL); break; }
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < HD; c += 32) {
              uint32_t o[32];
              tmem_ld32(o_addr + c, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              tmem_st32(o_addr + c, o);
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
          for (int i = threadIdx.x & 127; i < (PA_N - kt.count) * CHUNKS * 8; i += 128) {
            const int at = kt.count + i / (CHUNKS * 8), c = i % (CHUNKS * 8);
            st_shared_v4(base + (c >> 3) * (PA_N * 128) + at * 128 + (c & 7) * 16, make_uint4(0, 0, 0, 0));
          }
          fence_proxy_async_smem();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[grp]);
      }
      if (!ok) break;
      ok = warp_wait(&seg_free[sq & 1], ((sq >> 1) & 1) ^ 1);     // m and l of the segment before the last have been read
      if (!ok) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_TMEM_EMPTY); break; }
      float* ml = s_ml + ((sq & 1) * 2 + grp) * 2 * PA_M;
      ml[r] = m_run;
      ml[PA_M + r] = l_run;
      __syncwarp();
      if (lane == 0) mbar_arrive(&seg_done[sq & 1]);
      ++sq;
      g0 += s.tiles;
    }
  } else {
    // ---------------------------------------------------------------- results: warp 8 + q has TMEM lanes 32 q..
    const int quad = warp & 3, r = quad * 32 + lane;
    const uint32_t t_lane = tmem_base + ((uint32_t)(quad * 32) << 16);
    int sq = 0;
#pragma unroll 1
    while (take(s, ok)) {
      let_go();
      // barriers of segments, of which at most two are under way: this warp may be behind by many tiles
      ok = warp_wait(&seg_done[sq & 1], (sq >> 1) & 1) && warp_wait(&o_full[sq & 1], (sq >> 1) & 1);
      if (!ok) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_TMEM_FULL); break; }
      tc_fence_after();
      const int set = sq % Cfg::SETS;
      const uint32_t o_addr = t_lane + Cfg::TM_O + set * HD;
      const float* ml = s_ml + (sq & 1) * 4 * PA_M + r;           // sums of even and odd tiles, each to the maximum that it has seen last; O is to the last of all
      const float m_even = ml[0], m_odd = ml[2 * PA_M], m = fmaxf(m_even, m_odd);
      const float l = ml[PA_M] * (m_even == m ? 1.f : fast_exp2(m_even - m)) + ml[3 * PA_M] * (m_odd == m ? 1.f : fast_exp2(m_odd - m));
      __syncwarp();
      if (lane == 0) mbar_arrive(&seg_free[sq & 1]);
      const auto release = [&] {                                  // all has been read
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&o_free[set]);
      };
      const bool whole = s.flags & 2;                           // nothing to be joined
      const float inv = whole ? (l == 0.f ? 0.f : 1.f / l) : 1.f;           // NaN stays NaN
      if (whole) {
        const int i = token_of(p, r), t = s.t0 + i;
        if (p.a.lse && r < s.rows && t >= 0 && t < p.a.tokens)
          p.a.lse[(long long)t * p.a.q_heads + s.h * p.group + r - i * p.group] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
      } else if (r < s.rows && has_room(p, s.at + r)) {
        p.ml[s.at + r] = make_float2(m, l);
      }
      if (quad * 32 < s.rows) {
        const int row0 = quad * 32 + (lane & ~3);               // after an exchange among four lanes a lane has 16 bytes of four rows
#pragma unroll 1
        for (int c = 0; c < HD; c += 32) {
          uint32_t x[32];
          tmem_ld32(o_addr + c, x);
          tmem_ld_wait();
          if (c + 32 == HD) release();
          if (whole) {
            uint4 v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const auto pair = [&](int i) { return pack_bf16x2(__uint_as_float(x[k * 8 + i]) * inv, __uint_as_float(x[k * 8 + i + 1]) * inv); };
              v[k] = make_uint4(pair(0), pair(2), pair(4), pair(6));
            }
            exchange4(v, lane);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int row = row0 + k, i = token_of(p, row), t = s.t0 + i;
              if (row < s.rows && t >= 0 && t < p.a.tokens)
                *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.a.out) + ((long long)t * p.a.q_heads + s.h * p.group + row - i * p.group) * HD + c + (lane & 3) * 8) = v[k];
            }
          } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint4 v[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) v[k] = make_uint4(x[h * 16 + k * 4], x[h * 16 + k * 4 + 1], x[h * 16 + k * 4 + 2], x[h * 16 + k * 4 + 3]);
              exchange4(v, lane);
#pragma unroll
              for (int k = 0; k < 4; ++k)
                if (row0 + k < s.rows && has_room(p, s.at + row0 + k)) *reinterpret_cast<uint4*>(p.part + (s.at + row0 + k) * HD + c + h * 16 + (lane & 3) * 4) = v[k];
            }
          }
          __syncwarp();
        }
      } else {
        release();
      }
      ++sq;
    }
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
  // `count` pieces, of which row_of(i) is the i-th: the weights of 32 at a time, one to a lane, then their rows, eight under way at once
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
      for (int j0 = 0; j0 < n; j0 += 8) {
        float v[8][PER], wj[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
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
        for (int k = 0; k < 8; ++k)
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

// Shared form: every row from the pieces of its prompt item and of its own item, HD / 4 lanes to a row.  The first four pieces, of which there are seldom
// more, are fetched together with their (m, l), before it is known whether they count.
template <int HD>
__global__ void __launch_bounds__(256) paged_join_rows_kernel(const __grid_constant__ PagedTcParams p) {
  constexpr int LANES = HD / 4, AT_ONCE = 4;
  pdl_launch_dependents();
  pdl_wait();
  const long long row = (long long)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  const int t = (int)(row / p.a.q_heads), hq = (int)(row - (long long)t * p.a.q_heads), h = hq / p.group, head = hq - h * p.group, x = threadIdx.x % LANES * 4;
  if (t >= p.a.tokens) return;
  const PagedOwn own = p.owns[t];
  const int per_prompt = p.sums[1], per = p.sums[2];
  const int prt = t / p.tpt, p_item = h * p.prefix_row_tiles + prt, pa = p_item * p.prefix_tiles, p_first = pa / per_prompt;
  const int p_count = own.inner >= 0 && p.prefix_tiles > 0 ? min((pa + p.prefix_tiles - 1) / per_prompt - p_first + 1, p.ctas) : 0;
  const int a = own.pos + h * own.all, first = a / per, count = own.inner >= 0 && own.tiles > 0 ? min((a + own.tiles - 1) / per - first + 1, p.ctas) : 0;
  // rows of the scratch, which is far from 2^31 of them
  const int p_step = p.tb * p.group, o_step = p.ts * p.group, room = (int)p.part_rows;
  int at = (p_item + p_first) * p_step + (t - prt * p.tpt) * p.group + head;     // the next piece's row
  const int o_row = (int)p.own_slot0 + (own.item + h * own.row_tiles + first) * o_step + own.inner * p.group + head;
  if (p_count == 0) at = o_row;
  float m = -INFINITY, l = 0.f, acc[4] = {};
#pragma unroll 1
  for (int k0 = 0; k0 < p_count + count; k0 += AT_ONCE) {
    float2 ml[AT_ONCE];
    float4 v[AT_ONCE];
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k) {
      ml[k] = make_float2(-INFINITY, 0.f);
      v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (k0 + k < p_count + count && at >= 0 && at < room) {
        ml[k] = p.ml[at];
        v[k] = *reinterpret_cast<const float4*>(p.part + (long long)at * HD + x);
      }
      at = k0 + k + 1 == p_count ? o_row : at + (k0 + k + 1 < p_count ? p_step : o_step);
    }
    float top = m;
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k)
      if (ml[k].y != 0.f) top = fmaxf(top, ml[k].x);             // otherwise a piece of which this row saw nothing
    const float keep = m == -INFINITY ? 0.f : fast_exp2(m - top);
    l *= keep;
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] *= keep;
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k) {
      if (ml[k].y == 0.f) continue;
      const float w = ml[k].x == -INFINITY ? 1.f : fast_exp2(ml[k].x - top);
      l += ml[k].y * w;
      acc[0] += v[k].x * w; acc[1] += v[k].y * w; acc[2] += v[k].z * w; acc[3] += v[k].w * w;
    }
    m = top;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.a.out) + ((long long)t * p.a.q_heads + hq) * HD + x) =
      make_uint2(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv));
  if (p.a.lse && x == 0) p.a.lse[(long long)t * p.a.q_heads + hq] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

// Joint form: the items that a stretch's end cuts (blocks (c, y): the one that begins in stretch c and goes beyond it, rows dealt to four blocks: four
// requests of up to 2048 tokens 88 us, 112 with one), and zeros for the rows of no request.
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
      for (int r = blockIdx.y * 8 + warp; r < s.tokens * p.group; r += 8 * gridDim.y) {
        RowJoin<HD> join;
        join.add(p, last - c0 + 1, [&](int k) -> long long {      // the piece is the first of its CTA, but for an item that begins inside
          return own_row(p, 2ll * (c0 + k) + ((long long)(c0 + k) * per >= a ? 0 : 1)) + r;
        }, lane);
        const int t = s.t0 + r / p.group;
        if (t >= 0 && t < p.a.tokens) join.write(p, t, s.h * p.group + r % p.group, lane);
      }
    }
  }
  if (blockIdx.y > 0) return;
  const auto zero = [&](long long from, long long to) {
    for (long long t = max(from, 0ll); t < min(to, (long long)p.a.tokens); ++t)
      for (int hq = warp; hq < p.a.q_heads; hq += 8) RowJoin<HD>().write(p, (int)t, hq, lane);
  };
  for (int b = blockIdx.x; b < p.a.batch; b += gridDim.x) zero((long long)p.a.starts[b] + p.a.max_fresh, p.a.starts[b + 1]);
  const int behind = p.a.batch > 0 ? max(p.a.starts[p.a.batch], 0) : 0;
  const long long share = ((unsigned)max(p.a.tokens - behind, 0) + gridDim.x - 1) / gridDim.x;
  zero(behind + blockIdx.x * share, behind + (blockIdx.x + 1) * share);
  if (blockIdx.x == 0 && p.a.batch > 0) zero(0, p.a.starts[0]);
}

}  // namespace oa

using namespace oa;

// The sizes that follow from a call's arguments: which form, how many items there can be, what they need in scratch.
struct PagedTcPlan {
  int group, tpt, ts, tb, few, few_prompt, own_log2, over, joint, prefix_tiles, prefix_row_tiles, grid;
  long long prompt_rows, own_rows, items;
  size_t o_bytes, owns_bytes, ml_bytes, bytes;
};
static PagedTcPlan plan_tc(int tokens, int batch, int max_fresh, int q_heads, int kv_heads, int head_dim, int prefix_len) {
  PagedTcPlan c;
  c.group = q_heads / kv_heads;
  c.tpt = PA_M / c.group;
  c.ts = max_fresh < c.tpt ? (max_fresh > 0 ? max_fresh : 1) : c.tpt;
  c.tb = tokens < c.tpt ? tokens : c.tpt;
  const int few_log2 = head_dim == 64 ? PF_KEYS_LOG2<64> : PF_KEYS_LOG2<128>;
  const auto few = [&](int rows) { return rows > PF_ROWS ? 0 : rows <= 8 ? 8 : 16; };       // 32 requests of 2048, group 16, heads of 128: 19.0 us, 22.5 as tiles of many
  c.few = few(c.ts * c.group);
  // 16 requests, 32 heads of 128, behind 4096 shared keys: 33.1 us with few rows, 30.7 without; heads of 64, 4000: 21.2 and 26.7
  c.few_prompt = head_dim == 128 && c.tb * c.group > 8 ? 0 : few(c.tb * c.group);
  c.own_log2 = c.few ? few_log2 : 7;
  c.prefix_row_tiles = (tokens + c.tpt - 1) / c.tpt;
  // With a prompt, its keys and a request's own in one item only where requests fill many query tiles: results need not be joined then, but the
  // prompt is read by each request's (8 requests of up to 1000 tokens behind 500: 141 us, 201 apart; 2 of up to 4000 behind 2048: 178 and 197; 4 of
  // up to 512: 61 and 55; 64 of up to 16 behind 4000: 141 and 92).  Without a prompt always (32 of up to 300: 102 and 129).
  c.joint = !c.few && (prefix_len == 0 || c.prefix_row_tiles > 9ll * batch);
  c.over = c.joint ? 0 : c.few ? 3 : 1;
  const int prefix_log2 = c.few_prompt && !c.joint ? few_log2 : 7;
  c.prefix_tiles = (int)(((long long)prefix_len + (1 << prefix_log2) - 1) >> prefix_log2);
  c.grid = sm_count();
  c.items = ((long long)batch + tokens / c.tpt) * kv_heads;                    // query tiles of single requests, at most
  c.prompt_rows = c.joint || prefix_len == 0 ? 0 : ((long long)c.prefix_row_tiles * kv_heads + c.grid) * (c.tb * c.group);
  c.own_rows = (c.joint ? 2ll * c.grid : c.items + c.grid) * (c.ts * c.group);
  c.o_bytes = (size_t)(c.prompt_rows + c.own_rows) * head_dim * sizeof(float);
  c.ml_bytes = (size_t)(c.prompt_rows + c.own_rows) * sizeof(float2);
  c.owns_bytes = c.joint ? 0 : (size_t)tokens * sizeof(PagedOwn);
  c.bytes = c.o_bytes + c.owns_bytes + c.ml_bytes + (2 * ((size_t)batch + 1) + PA_SUMS) * sizeof(int);
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
  static std::atomic<unsigned long long> allowed[2];
  const PagedTcPlan c = plan_tc(a.tokens, a.batch, a.max_fresh, a.q_heads, a.kv_heads, HD, a.prefix_len);
  const int ps = 1 << a.page_log2;
  const long long own_tiles = (((long long)a.width * ps) >> c.own_log2) + 1;
  const long long work = (c.joint ? 0 : (long long)a.kv_heads * c.prefix_row_tiles * c.prefix_tiles);
  if (work + c.items * (own_tiles + c.over + c.prefix_tiles + 1) > 0x7fffffffll) return OA_ERR_TOO_LARGE;
  PagedTcParams p;
  p.a = a;
  p.group = c.group; p.group_mul = 65536 / c.group + 1; p.tpt = c.tpt; p.ts = c.ts; p.tb = c.tb;
  p.few = c.few; p.few_prompt = c.few_prompt; p.own_log2 = c.own_log2; p.over = c.over;
  p.many = !c.few || (work > 0 && !c.few_prompt);
  p.joint = c.joint; p.prefix_tiles = c.prefix_tiles; p.prefix_row_tiles = c.prefix_row_tiles; p.prefix_work = (int)work;
  p.part = static_cast<float*>(scratch);
  p.owns = reinterpret_cast<PagedOwn*>(static_cast<char*>(scratch) + c.o_bytes);
  p.ml = reinterpret_cast<float2*>(static_cast<char*>(scratch) + c.o_bytes + c.owns_bytes);
  p.sums = reinterpret_cast<int*>(static_cast<char*>(scratch) + c.o_bytes + c.owns_bytes + c.ml_bytes);
  p.own_slot0 = c.prompt_rows;
  p.part_rows = c.prompt_rows + c.own_rows;
  p.ctas = c.grid;
  p.status = status;
  // descriptors of what the call's kinds of CTAs load; the others' are never used
  CUtensorMap tq = {}, tqo = {}, tk = {}, tv = {}, tkf = {}, tvf = {};
  int rc;
  const uint64_t packed = (uint64_t)a.kv_heads * ps * HD;
  const uint64_t dims[3] = {HD, (uint64_t)a.kv_heads * ps, (uint64_t)a.pages};
  const uint64_t ks[2] = {HD * 2, (a.pages > 1 ? (uint64_t)a.k_page_stride : packed) * 2}, vs[2] = {HD * 2, (a.pages > 1 ? (uint64_t)a.v_page_stride : packed) * 2};
  if (p.many) {
    const uint64_t q_dims[3] = {HD, (uint64_t)a.q_heads, (uint64_t)a.tokens}, strides[2] = {HD * 2, (uint64_t)a.q_stride * 2};
    const uint32_t box[3] = {64, (uint32_t)c.group, (uint32_t)c.tb}, own[3] = {64, (uint32_t)c.group, (uint32_t)c.ts}, page[3] = {64, (uint32_t)ps, 1};
    if ((rc = make_tmap_box3_bf16(&tq, a.q, q_dims, strides, box)) || (rc = make_tmap_box3_bf16(&tqo, a.q, q_dims, strides, own)) ||
        (rc = make_tmap_box3_bf16(&tk, a.k, dims, ks, page)) || (rc = make_tmap_box3_bf16(&tv, a.v, dims, vs, page)))
      return rc;
  }
  if (c.few || c.few_prompt) {                                     // a tile's keys, or a page's where it has fewer
    const uint32_t box[3] = {64, (uint32_t)(ps < 1 << PF_KEYS_LOG2<HD> ? ps : 1 << PF_KEYS_LOG2<HD>), 1};
    if ((rc = make_tmap_box3_bf16(&tkf, a.k, dims, ks, box)) || (rc = make_tmap_box3_bf16(&tvf, a.v, dims, vs, box))) return rc;
  }
  const bool two = c.few > 8 || (work > 0 && c.few_prompt > 8);
  const auto kernel = two ? paged_attn_tc_kernel<HD, 2> : paged_attn_tc_kernel<HD, 1>;
  if (allow_smem(allowed[two], (const void*)kernel, Cfg::SMEM_BYTES) != cudaSuccess) return OA_ERR_LAUNCH;
  launch_short(kernel, dim3((unsigned)c.grid), dim3(PA_THREADS), Cfg::SMEM_BYTES, st, tq, tqo, tk, tv, tkf, tvf, p);
  if (c.joint) launch_short(paged_join_cuts_kernel<HD>, dim3((unsigned)c.grid, 4), dim3(256), 0, st, p);
  else {
    const long long rows = (long long)a.tokens * a.q_heads, rows_of_block = 1024 / HD;
    launch_short(paged_join_rows_kernel<HD>, dim3((unsigned)((rows + rows_of_block - 1) / rows_of_block)), dim3(256), 0, st, p);
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
