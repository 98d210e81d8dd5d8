// Causal attention over packed sequences of up to 64 rows, forward and backward, bf16 in / fp32 accumulate: the sequences that a tile of 128 x 128 would be
// mostly empty for (packed_attn.cu has the mathematics and the longer ones).
//
// A block of four warps works on one sequence and as many heads as give every warp 16 rows of one (backward: key-value heads, each with its query heads in turn).  The
// rows come to shared memory by cp.async, in 16-byte pieces swizzled over eight banks' groups; rows behind the sequence up to the next 16 are zeros.  A warp
// takes 16 queries (forward, dQ) or 16 keys (dK, dV) and the products run on mma.sync, whose accumulators are the next product's operand as they stand: tiles this small cannot
// fill a tcgen05 instruction.  Backward, scores are worked out twice, with the keys as rows for dK and dV and with the queries as rows for dQ.  Bound by latency: loads,
// a chain of products and exponentials, stores, one after the other, which as many blocks as fit on an SM cover for one another (issue slots 56 % busy, memory 35 %).  512 sequences of up to 48 rows, 16 heads of
// 64: 31 us, gradients 77; the bytes would take 15 and 30.
#include "common.cuh"
#include "packed.cuh"
#include "per_device.h"
#include "api.h"
#include "packed_short.h"

namespace oa {

constexpr int PS_THREADS = 128;
constexpr float PS_LOG2E = 1.4426950408889634f;

// [64][HD] bf16 in shared memory, at a multiple of 256 bytes: piece c of row r stands at place c ^ (r & 7).  A lane's address is worked out once for a set of rows;
// another pair of pieces 2 k, 2 k + 1 of the same rows is that with 32 k exclusive-or'ed into it, 16 rows on are 16 STRIDE.
template <int HD>
struct ShortTile {
  static constexpr int STRIDE = HD * 2, BYTES = PACKED_SHORT * STRIDE, CHUNKS = HD / 8;
  // of a left operand [16 rows x 16 dimensions], and of a right one whose reduction runs along the 16 rows
  static __device__ __forceinline__ uint32_t rows_first(int lane) { return (lane & 15) * STRIDE + (((lane >> 4) ^ (lane & 7)) << 4); }
  // of two right operands of 8 columns each, where columns are rows and the reduction runs along dimensions
  static __device__ __forceinline__ uint32_t columns_first(int lane) { return ((lane & 7) + ((lane >> 4) << 3)) * STRIDE + ((((lane >> 3) & 1) ^ (lane & 7)) << 4); }
  // rows [0, n) of each of `heads` heads from memory, with zeros up to 16 `tiles` behind each; first(u): where head u's first row begins.  A pass of the
  // block covers 16 rows (8 at head dim 128), so that its head is one for all threads.
  template <typename F>
  static __device__ __forceinline__ void fetch(uint32_t base, long long stride, int n, int tiles, int heads, F first) {
    constexpr int ROWS = PS_THREADS / CHUNKS;
    const int r0 = threadIdx.x / CHUNKS, c = threadIdx.x % CHUNKS;
    uint32_t to = base + r0 * STRIDE + ((c ^ (r0 & 7)) << 4);
    const long long at = r0 * stride + c * 8;
    for (int u = 0; u < heads; ++u) {
      const __nv_bfloat16* src = first(u) + at;
#pragma unroll
      for (int row = 0; row < PACKED_SHORT; row += ROWS) {
        if (row >= tiles * 16) break;
        // a row that is not there is not read: zeros
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(row + r0 < n ? src : first(u)), "r"(row + r0 < n ? 16 : 0) : "memory");
        to += ROWS * STRIDE;
        src += ROWS * stride;
      }
    }
  }
};

__device__ __forceinline__ void short_ld4(uint32_t (&a)[4], uint32_t p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3]) : "r"(p) : "memory");
}
__device__ __forceinline__ void short_ld4_t(uint32_t (&a)[4], uint32_t p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3]) : "r"(p) : "memory");
}
__device__ __forceinline__ void short_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void short_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void short_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// [16 x 16] = rows of x (their address as a left operand) times rows of y (as right ones), over HD dimensions: d[0], d[1] are the halves of 8 columns
template <int HD>
__device__ __forceinline__ void short_scores(float (&d)[2][4], uint32_t x, uint32_t y) {
#pragma unroll
  for (int u = 0; u < 4; ++u) d[0][u] = d[1][u] = 0.f;
#pragma unroll
  for (int k = 0; k < HD / 16; ++k) {
    uint32_t a[4], b[4];
    short_ld4(a, x ^ (k << 5));
    short_ld4(b, y ^ (k << 5));
    short_mma(d[0], a, b[0], b[1]);
    short_mma(d[1], a, b[2], b[3]);
  }
}
// acc[16 x HD] += w[16 x 16] times 16 rows of y
template <int HD>
__device__ __forceinline__ void short_weigh(float (&acc)[HD / 8][4], const uint32_t (&w)[4], uint32_t y) {
#pragma unroll
  for (int c = 0; c < HD / 16; ++c) {
    uint32_t b[4];
    short_ld4_t(b, y ^ (c << 5));
    short_mma(acc[2 * c], w, b[0], b[1]);
    short_mma(acc[2 * c + 1], w, b[2], b[3]);
  }
}
// two [16 x 8] accumulators as a left operand
__device__ __forceinline__ void short_operand(uint32_t (&w)[4], const float (&d)[2][4]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    w[2 * h] = pack_bf16x2(d[h][0], d[h][1]);
    w[2 * h + 1] = pack_bf16x2(d[h][2], d[h][3]);
  }
}
// ... and what its rounding leaves
__device__ __forceinline__ void short_remainder(uint32_t (&w)[4], const float (&d)[2][4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float* v = &d[i >> 1][(i & 1) * 2];
    w[i] = pack_bf16x2(v[0] - __uint_as_float(w[i] << 16), v[1] - __uint_as_float(w[i] & 0xffff0000u));
  }
}
// A warp's 16 rows of an accumulator, times mul0 / mul1 for its rows lane / 4 and + 8, to memory through 16 rows of a tile (their address) that only this warp
// uses: the first `n`, in 16-byte pieces
template <int HD>
__device__ __forceinline__ void short_store(const float (&acc)[HD / 8][4], float mul0, float mul1, uint32_t rows, int n, __nv_bfloat16* to, long long stride, int lane) {
  constexpr int STRIDE = ShortTile<HD>::STRIDE, CHUNKS = HD / 8;
  const uint32_t put = rows + (lane >> 2) * STRIDE + (((lane >> 2) & 7) << 4) + (lane & 3) * 4;
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    asm volatile("st.shared.b32 [%0], %1;" ::"r"(put ^ (c << 4)), "r"(pack_bf16x2(acc[c][0] * mul0, acc[c][1] * mul0)) : "memory");
    asm volatile("st.shared.b32 [%0], %1;" ::"r"((put ^ (c << 4)) + 8 * STRIDE), "r"(pack_bf16x2(acc[c][2] * mul1, acc[c][3] * mul1)) : "memory");
  }
  __syncwarp();
  constexpr int ROWS = 32 / CHUNKS;                                    // of a pass
  const int r0 = lane / CHUNKS, c = lane % CHUNKS;
  to += r0 * stride + c * 8;
#pragma unroll
  for (int r = 0; r < 16; r += ROWS, to += ROWS * stride) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(rows + (r + r0) * STRIDE + ((c ^ ((r + r0) & 7)) << 4)) : "memory");
    if (r + r0 < n) *reinterpret_cast<uint4*>(to) = v;
  }
  __syncwarp();
}

// A block's task: a sequence and as many of its heads as make four 16-row tiles at most.  Tasks with three or four tiles to a head come first, then those with two,
// then one; sets of heads one after the other.
struct ShortTask {
  int lo, n, tiles, head, heads;           // head: the first
};
struct ShortWalk {
  const PackedPlan& plan;
  const int all_heads, n0, n1, n2, end0, end1, end;
  int task, set, sets;
  int4 ahead;                              // the next task's entry, on its way; its set of heads, and how many there are to a set
  __device__ __forceinline__ ShortWalk(const PackedPlan& p, int heads)
      : plan(p), all_heads(heads), n0(p.words[4]), n1(p.words[5]), n2(p.words[6]), end0(n0 * heads), end1(end0 + n1 * ((heads + 1) >> 1)),
        end(end1 + n2 * ((heads + 3) >> 2)), task(blockIdx.x) { fetch(); }
  __device__ __forceinline__ void fetch() {
    if (task >= end) return;
    const int from = task < end0 ? 0 : task < end1 ? end0 : end1, n = task < end0 ? n0 : task < end1 ? n1 : n2;
    set = (int)((unsigned)(task - from) / (unsigned)n);
    ahead = plan.brief((task < end0 ? 0 : task < end1 ? n0 : n0 + n1) + task - from - set * n);
    sets = task < end0 ? 1 : task < end1 ? 2 : 4;
  }
  __device__ __forceinline__ bool next(ShortTask& e) {
    if (task >= end) return false;
    e.lo = ahead.x;
    e.n = ahead.y - ahead.x;
    e.tiles = (e.n + 15) >> 4;
    e.head = set * sets;
    e.heads = min(sets, all_heads - e.head);
    task += gridDim.x;
    fetch();
    return true;
  }
};

template <int HD>
__global__ void __launch_bounds__(PS_THREADS, HD == 64 ? 4 : 2) packed_short_fwd_kernel(const PackedShortFwd p) {
  using Tile = ShortTile<HD>;
  extern __shared__ __align__(1024) uint8_t smem[];      // two stages of Q, K, V
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float sl2 = p.scale * PS_LOG2E;
  const uint32_t rows_at = Tile::rows_first(lane), columns_at = Tile::columns_first(lane), stages = smem_u32(smem);
  const auto fetch = [&](uint32_t to, const ShortTask& e) {
    const __nv_bfloat16* q = p.q + e.lo * p.qs + e.head * HD;
    Tile::fetch(to, p.qs, e.n, e.tiles, e.heads, [&](int u) { return q + u * HD; });
    const auto kv = [&](int u) { return (p.group == 1 ? e.head + u : (int)((unsigned)(e.head + u) / (unsigned)p.group)) * HD; };
    const __nv_bfloat16 *k = p.k + e.lo * p.ks, *v = p.v + e.lo * p.vs;
    Tile::fetch(to + Tile::BYTES, p.ks, e.n, e.tiles, e.heads, [&](int u) { return k + kv(u); });
    Tile::fetch(to + 2 * Tile::BYTES, p.vs, e.n, e.tiles, e.heads, [&](int u) { return v + kv(u); });
  };
  ShortWalk walk(p.plan, p.q_heads);
  ShortTask e, then;
  if (!walk.next(e)) return;
  fetch(stages, e);
  short_commit();
  for (int stage = 0;; stage ^= 1) {
    const bool more = walk.next(then);
    if (more) fetch(stages + (stage ^ 1) * 3 * Tile::BYTES, then);
    short_commit();
    short_wait<1>();
    __syncthreads();
    const uint32_t sq = stages + stage * 3 * Tile::BYTES, sk = sq + Tile::BYTES, sv = sk + Tile::BYTES;
    const int u = e.tiles == 1 ? warp : e.tiles == 2 ? warp >> 1 : 0, tile = warp - u * e.tiles, base = u * e.tiles * 16, r0 = base + tile * 16;
    if (u < e.heads && tile < e.tiles) {
      // scores of 16 queries and the keys up to them, at most 64
      constexpr int STEP = 16 * Tile::STRIDE;
      float s[4][2][4];
      const int i0 = tile * 16 + (lane >> 2), i1 = i0 + 8;             // this thread's queries
      float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        if (t > tile) break;
        short_scores<HD>(s[t], sq + r0 * Tile::STRIDE + rows_at, sk + base * Tile::STRIDE + t * STEP + columns_at);
        if (t == tile) {
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const int j = t * 16 + c * 8 + (lane & 3) * 2 + x;
              s[t][c][x] = j <= i0 ? s[t][c][x] : -INFINITY;
              s[t][c][2 + x] = j <= i1 ? s[t][c][2 + x] : -INFINITY;
            }
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          m0 = fmax3(m0, s[t][c][0], s[t][c][1]);
          m1 = fmax3(m1, s[t][c][2], s[t][c][3]);
        }
      }
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, o));
        m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, o));
      }
      m0 = m0 == -INFINITY ? 0.f : m0 * sl2;                           // every score is -inf
      m1 = m1 == -INFINITY ? 0.f : m1 * sl2;
      float l0 = 0.f, l1 = 0.f, o[HD / 8][4];
#pragma unroll
      for (int c = 0; c < HD / 8; ++c) o[c][0] = o[c][1] = o[c][2] = o[c][3] = 0.f;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        if (t > tile) break;
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            l0 += s[t][c][u] = fast_exp2(fmaf(s[t][c][u], sl2, -m0));
            l1 += s[t][c][2 + u] = fast_exp2(fmaf(s[t][c][2 + u], sl2, -m1));
          }
        uint32_t w[4];
        short_operand(w, s[t]);
        short_weigh<HD>(o, w, sv + base * Tile::STRIDE + t * STEP + rows_at);
      }
#pragma unroll
      for (int q = 1; q < 4; q <<= 1) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, q);
        l1 += __shfl_xor_sync(0xffffffffu, l1, q);
      }
      if (p.lse && (lane & 3) == 0) {
        float* to = p.lse + (long long)(e.head + u) * p.plan.tokens + e.lo;
        if (i0 < e.n) to[i0] = (m0 + log2f(l0)) / PS_LOG2E;
        if (i1 < e.n) to[i1] = (m1 + log2f(l1)) / PS_LOG2E;
      }
      short_store<HD>(o, 1.f / l0, 1.f / l1, sq + r0 * Tile::STRIDE, e.n - tile * 16, p.o + (e.lo + tile * 16) * p.os + (e.head + u) * HD, p.os, lane);
    }
    if (!more) break;
    __syncthreads();                                                   // the stage is free
    e = then;
  }
}

// STAGES: 2 where the next rows are on their way during the work on these
template <int HD> constexpr int PS_STAGES = HD == 64 ? 2 : 1;
template <int HD> constexpr int PS_BWD_BYTES = PS_STAGES<HD> * (4 * ShortTile<HD>::BYTES + 2 * PACKED_SHORT * 4);

template <int HD>
__global__ void __launch_bounds__(PS_THREADS, HD == 64 ? 3 : 2) packed_short_bwd_kernel(const PackedShortBwd p) {
  using Tile = ShortTile<HD>;
  constexpr int STAGES = PS_STAGES<HD>;
  extern __shared__ __align__(1024) uint8_t smem[];      // stages of Q and dO, of K and V, of log-sum-exp and delta
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float sl2 = p.scale * PS_LOG2E, scale = p.scale;
  const uint32_t rows_at = Tile::rows_first(lane), columns_at = Tile::columns_first(lane), stages = smem_u32(smem);
  const uint32_t kv_stages = stages + STAGES * 2 * Tile::BYTES;
  float* const stats = reinterpret_cast<float*>(smem + STAGES * 4 * Tile::BYTES);
  // query head g of every key-value head of a task, and with the first of them the keys and values
  const auto fetch = [&](int stage, int kv_stage, const ShortTask& e, int g) {
    const uint32_t sq = stages + stage * 2 * Tile::BYTES;
    const int col = (e.head * p.group + g) * HD, apart = p.group * HD;
    const __nv_bfloat16 *q = p.q + e.lo * p.qs + col, *dout = p.dout + e.lo * p.dos + col;
    Tile::fetch(sq, p.qs, e.n, e.tiles, e.heads, [&](int u) { return q + u * apart; });
    Tile::fetch(sq + Tile::BYTES, p.dos, e.n, e.tiles, e.heads, [&](int u) { return dout + u * apart; });
    if (g == 0) {
      const uint32_t sk = kv_stages + kv_stage * 2 * Tile::BYTES;
      const __nv_bfloat16 *k = p.k + e.lo * p.ks + e.head * HD, *v = p.v + e.lo * p.vs + e.head * HD;
      Tile::fetch(sk, p.ks, e.n, e.tiles, e.heads, [&](int u) { return k + u * HD; });
      Tile::fetch(sk + Tile::BYTES, p.vs, e.n, e.tiles, e.heads, [&](int u) { return v + u * HD; });
    }
    const int row = threadIdx.x, v = e.tiles == 1 ? row >> 4 : e.tiles == 2 ? row >> 5 : 0, in = row - v * e.tiles * 16;
    if (row < PACKED_SHORT && v < e.heads) {
      const long long at = (long long)((e.head + v) * p.group + g) * p.plan.tokens + e.lo;
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(stats + stage * 2 * PACKED_SHORT + row)), "l"(p.lse + at + (in < e.n ? in : 0)), "r"(in < e.n ? 4 : 0) : "memory");
    }
  };
  ShortWalk walk(p.plan, p.kv_heads);
  ShortTask e, then;
  if (!walk.next(e)) return;
  int g = 0, kv_stage = 0;
  float dk[HD / 8][4], dv[HD / 8][4];
  if (STAGES == 2) fetch(0, 0, e, 0);
  short_commit();
  for (int stage = 0;; stage ^= STAGES - 1) {
    const bool last = g + 1 == p.group;
    bool more = true;
    if (last) more = walk.next(then);
    if (STAGES == 2) {
      if (!last) fetch(stage ^ 1, kv_stage, e, g + 1);
      else if (more) fetch(stage ^ 1, kv_stage ^ 1, then, 0);
      short_commit();
      short_wait<1>();
    } else {
      fetch(0, 0, e, g);
      short_commit();
      short_wait<0>();
    }
    __syncthreads();
    const uint32_t sq = stages + stage * 2 * Tile::BYTES, sdo = sq + Tile::BYTES, sk = kv_stages + kv_stage * 2 * Tile::BYTES, sv = sk + Tile::BYTES;
    float* stat = stats + stage * 2 * PACKED_SHORT;                      // log-sum-exp, and delta from this kernel
    const int n = e.n, u = e.tiles == 1 ? warp : e.tiles == 2 ? warp >> 1 : 0, tile = warp - u * e.tiles, base = u * e.tiles * 16, r0 = base + tile * 16;
    const bool mine_too = u < e.heads && tile < e.tiles;
    // dS goes to its products rounded, and up to 32 rows, whose roundings are too few to even out (gradients of sequences of two tokens up to 1.6 times as far off as
    // by the rounding of the result alone), what that leaves as well: 512 sequences of up to 48 rows take 76.8 us, with it for all of them 80.9
    const bool few = e.tiles <= 2;
    const long long row0 = e.lo + tile * 16;
    float dq[HD / 8][4];
    if (g == 0) {
#pragma unroll
      for (int c = 0; c < HD / 8; ++c)
#pragma unroll
        for (int x = 0; x < 4; ++x) dk[c][x] = dv[c][x] = 0.f;
    }
    if (mine_too) {
      constexpr int STEP = 16 * Tile::STRIDE;
      const uint32_t mine = r0 * Tile::STRIDE, all = base * Tile::STRIDE;
      const int j0 = tile * 16 + (lane >> 2), j1 = j0 + 8;                // this thread's queries, then its keys
      // queries as rows: dS, for the keys up to them
#pragma unroll
      for (int c = 0; c < HD / 8; ++c) dq[c][0] = dq[c][1] = dq[c][2] = dq[c][3] = 0.f;
      const float nl0 = -stat[base + j0] * PS_LOG2E, nl1 = -stat[base + j1] * PS_LOG2E;
      // delta = sum p dP, in 32 bits; from the rounded output it would be off by as much as everything else together
      float nd0 = 0.f, nd1 = 0.f, s[2][4], dp[2][4];                      // s: then the weights
      const auto weights = [&](int t) {
        short_scores<HD>(s, sq + mine + rows_at, sk + all + t * STEP + columns_at);
        short_scores<HD>(dp, sdo + mine + rows_at, sv + all + t * STEP + columns_at);
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int j = t * 16 + c * 8 + (lane & 3) * 2 + x;
            s[c][x] = j <= j0 ? fast_exp2(fmaf(s[c][x], sl2, nl0)) : 0.f;
            s[c][2 + x] = j <= j1 ? fast_exp2(fmaf(s[c][2 + x], sl2, nl1)) : 0.f;
          }
      };
#pragma unroll 1
      for (int t = 0; t <= tile; ++t) {
        weights(t);
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            nd0 -= s[c][x] * dp[c][x];
            nd1 -= s[c][2 + x] * dp[c][2 + x];
          }
      }
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        nd0 += __shfl_xor_sync(0xffffffffu, nd0, o);
        nd1 += __shfl_xor_sync(0xffffffffu, nd1, o);
      }
      nd0 *= scale;
      nd1 *= scale;
      if ((lane & 3) == 0) {
        stat[PACKED_SHORT + base + j0] = nd0;
        stat[PACKED_SHORT + base + j1] = nd1;
      }
#pragma unroll 1
      for (int t = tile;; weights(t)) {                                   // the last keys' are still there
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            dp[c][x] = s[c][x] * fmaf(dp[c][x], scale, nd0);
            dp[c][2 + x] = s[c][2 + x] * fmaf(dp[c][2 + x], scale, nd1);
          }
        uint32_t w[4];
        short_operand(w, dp);
        short_weigh<HD>(dq, w, sk + all + t * STEP + rows_at);
        if (few) {
          short_remainder(w, dp);
          short_weigh<HD>(dq, w, sk + all + t * STEP + rows_at);
        }
        if (--t < 0) break;
      }
    }
    __syncthreads();                                                   // delta of every query
    if (mine_too) {
      constexpr int STEP = 16 * Tile::STRIDE;
      const uint32_t mine = r0 * Tile::STRIDE, all = base * Tile::STRIDE;
      const int j0 = tile * 16 + (lane >> 2), j1 = j0 + 8;
      // keys as rows: P^T and dS^T, for the queries from them on
#pragma unroll 1
      for (int t = tile; t < e.tiles; ++t) {
        float s[2][4], dp[2][4];
        short_scores<HD>(s, sk + mine + rows_at, sq + all + t * STEP + columns_at);
        short_scores<HD>(dp, sv + mine + rows_at, sdo + all + t * STEP + columns_at);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int i = t * 16 + c * 8 + (lane & 3) * 2;
          const float2 L = *reinterpret_cast<const float2*>(stat + base + i), D = *reinterpret_cast<const float2*>(stat + PACKED_SHORT + base + i);
          const float2 nl = make_float2(-L.x * PS_LOG2E, -L.y * PS_LOG2E), nd = D;
          s[c][0] = fast_exp2(fmaf(s[c][0], sl2, nl.x));
          s[c][1] = fast_exp2(fmaf(s[c][1], sl2, nl.y));
          s[c][2] = fast_exp2(fmaf(s[c][2], sl2, nl.x));
          s[c][3] = fast_exp2(fmaf(s[c][3], sl2, nl.y));
          dp[c][0] = s[c][0] * fmaf(dp[c][0], scale, nd.x);
          dp[c][1] = s[c][1] * fmaf(dp[c][1], scale, nd.y);
          dp[c][2] = s[c][2] * fmaf(dp[c][2], scale, nd.x);
          dp[c][3] = s[c][3] * fmaf(dp[c][3], scale, nd.y);
          if (t == tile || t + 1 == e.tiles) {                       // queries before the key, and behind the sequence
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const bool a0 = j0 <= i + x && i + x < n, a1 = j1 <= i + x && i + x < n;
              s[c][x] = a0 ? s[c][x] : 0.f;
              s[c][2 + x] = a1 ? s[c][2 + x] : 0.f;
              dp[c][x] = a0 ? dp[c][x] : 0.f;
              dp[c][2 + x] = a1 ? dp[c][2 + x] : 0.f;
            }
          }
        }
        uint32_t w[4];
        short_operand(w, s);
        short_weigh<HD>(dv, w, sdo + all + t * STEP + rows_at);
        short_operand(w, dp);
        short_weigh<HD>(dk, w, sq + all + t * STEP + rows_at);
        if (few) {
          short_remainder(w, dp);
          short_weigh<HD>(dk, w, sq + all + t * STEP + rows_at);
        }
      }
    }
    __syncthreads();                                                   // every warp has read what it needs of these rows
    if (mine_too) {
      short_store<HD>(dq, 1.f, 1.f, sq + r0 * Tile::STRIDE, n - tile * 16, p.dq + row0 * p.dqs + ((e.head + u) * p.group + g) * HD, p.dqs, lane);
      if (last) {
        short_store<HD>(dk, 1.f, 1.f, sk + r0 * Tile::STRIDE, n - tile * 16, p.dk + row0 * p.dks + (e.head + u) * HD, p.dks, lane);
        short_store<HD>(dv, 1.f, 1.f, sv + r0 * Tile::STRIDE, n - tile * 16, p.dv + row0 * p.dvs + (e.head + u) * HD, p.dvs, lane);
      }
    }
    if (!more) break;
    __syncthreads();                                                   // the stages may be written over
    g = last ? 0 : g + 1;
    if (last) {
      e = then;
      kv_stage ^= STAGES - 1;
    }
  }
}

// As many blocks as the device holds at once, each with tasks in turn
template <typename P>
static int short_launch(void (*kernel)(const P), int smem, std::atomic<unsigned long long>& allowed, int per_sm, long long most, const P& p, cudaStream_t st) {
  if (allow_smem(allowed, (const void*)kernel, smem) != cudaSuccess) return OA_ERR_LAUNCH;
  const long long room = (long long)per_sm * sm_count();
  launch_short(kernel, dim3((unsigned)(most < 1 ? 1 : most < room ? most : room)), dim3(PS_THREADS), smem, st, p);
  return cudaGetLastError() == cudaSuccess ? OA_OK : OA_ERR_LAUNCH;
}

int packed_short_fwd(const PackedShortFwd& p, int head_dim, cudaStream_t st) {
  static std::atomic<unsigned long long> a64, a128;
  const long long most = (long long)p.plan.batch * p.q_heads;
  return head_dim == 64 ? short_launch(packed_short_fwd_kernel<64>, 6 * ShortTile<64>::BYTES, a64, 4, most, p, st)
                        : short_launch(packed_short_fwd_kernel<128>, 6 * ShortTile<128>::BYTES, a128, 2, most, p, st);
}

int packed_short_bwd(const PackedShortBwd& p, int head_dim, cudaStream_t st) {
  static std::atomic<unsigned long long> a64, a128;
  const long long most = (long long)p.plan.batch * p.kv_heads;
  return head_dim == 64 ? short_launch(packed_short_bwd_kernel<64>, PS_BWD_BYTES<64>, a64, 3, most, p, st)
                        : short_launch(packed_short_bwd_kernel<128>, PS_BWD_BYTES<128>, a128, 2, most, p, st);
}

}  // namespace oa
