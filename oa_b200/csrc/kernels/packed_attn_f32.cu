// Causal attention over packed sequences in fp32, with grouped heads, forward and backward: the engine's exact precision, and gradient checks.
//
// packed_attn.cu has the mathematics; here every product is fp32 multiply-adds.  A block of 256 threads owns 64 rows of one head of a sequence (forward and dQ: queries;
// dK and dV: keys of a key-value head) and the other side streams through shared memory 64 rows at a time.  A thread works on 4 x 4 of the 64 x 64
// scores, rows ty + 16 i and columns tx + 16 j, so that it takes 8 loads of 16 bytes for 64 multiply-adds and no two rows of a warp's loads meet in a
// bank; the weights go to shared memory and the second product is dealt out the same way, over the head's dimensions.  The next tile's first operand is on its
// way (cp.async) while the second product of this one runs.  Rows of other sequences are never read: what a sequence holds does not reach another.  dK and
// dV of a key-value head add up over the query heads that share it: up to eight of them are a cluster of blocks, a head to each, whose sums meet in distributed
// shared memory in the heads' order; more are worked on by one block one after the other.  Either way there is one writer and one order.
// 16 x 512 rows of 4 heads of 32 take 63 us (17 TFLOP/s) and 175 for the gradients (15), 512 of 8 heads over 2 of 64 46 and 109; 16 of up to 128 of 4 of 32, a few
// tiles to an SM, 12 and 23.  There what the warps wait for is shared memory and one another (issue slots 43 % busy, multiply-add pipe 26 %).
#include <cooperative_groups.h>

#include "common.cuh"
#include "packed.cuh"
#include "per_device.h"
#include "api.h"

namespace oa {

namespace cg = cooperative_groups;

constexpr int PF32_CLUSTER = 8;                        // blocks of a cluster, at most
constexpr int PF32_THREADS = 256, PF32_ROWS = 64;
constexpr int PF32_LDW = PF32_ROWS + 4;                // floats between rows of weights

struct PackedF32Params {
  const float *q, *k, *v, *o, *dout, *lse;
  float *out, *lse_out, *dq, *dk, *dv;
  long long qs, ks, vs, os, dos, dqs, dks, dvs;      // elements between rows
  PackedPlan plan;
  int q_heads, kv_heads, group, hd, vec;
  float scale;
};

// Where a block's rows are: sequence rows [lo, lo + n), its own from i0 on; i0 >= n: none.  MIRROR: tiles counted from the sequence's end
struct PackedRows { int lo, n, i0; };
template <bool MIRROR>
__device__ __forceinline__ PackedRows packed_rows(const PackedPlan& plan, int block) {
  constexpr int SUBS = PACKED_TILE / PF32_ROWS;
  const int at = block / SUBS, sub = block % SUBS, tiles = plan.tiles();
  if (at >= tiles + plan.shorts()) return {0, 0, 0};
  const int4 t = at < tiles ? plan.tile(at) : plan.brief(at - tiles);
  const int n = t.y - t.x, idx = MIRROR ? (n + PACKED_TILE - 1) / PACKED_TILE - 1 - t.z : t.z;
  return {t.x, n, idx * PACKED_TILE + (MIRROR ? sub : SUBS - 1 - sub) * PF32_ROWS};       // the longer half first
}

// HD: the head's dimensions rounded up to 32, 64 or 128
template <int HD>
struct F32Tile {
  static constexpr int LD = HD + 4, FLOATS = PF32_ROWS * LD;
  static constexpr int WIDE = HD == 32 ? 4 : HD / 16;           // dimensions of a thread in a second product
  // rows [r0, r0 + 64) of a sequence from lo on, columns [col, col + hd); rows from n and dimensions from hd on become 0
  static __device__ __forceinline__ void fetch(float* sm, const float* __restrict__ g, long long stride, int lo, int r0, int n, int col, int hd, bool vec) {
    if (vec) {
      constexpr int C = HD / 4;
#pragma unroll
      for (int i = threadIdx.x; i < PF32_ROWS * C; i += PF32_THREADS) {
        const int r = i / C, c = i % C * 4;
        const bool there = r0 + r < n && c < hd;
        const float* src = there ? g + (lo + r0 + r) * stride + col + c : g;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(sm + r * LD + c)), "l"(src), "r"(there ? 16 : 0) : "memory");
      }
    } else {
#pragma unroll 4
      for (int i = threadIdx.x; i < PF32_ROWS * HD; i += PF32_THREADS) {
        const int r = i / HD, c = i % HD;
        sm[r * LD + c] = r0 + r < n && c < hd ? g[(lo + r0 + r) * stride + col + c] : 0.f;
      }
    }
  }
  // s[i][j] = row ty + 16 i of x times row tx + 16 j of y
  static __device__ __forceinline__ void scores(float (&s)[4][4], const float* x, const float* y, int tx, int ty) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
#pragma unroll 4
    for (int k = 0; k < HD; k += 4) {
      float4 a[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        a[i] = *reinterpret_cast<const float4*>(x + (ty + 16 * i) * LD + k);
        b[i] = *reinterpret_cast<const float4*>(y + (tx + 16 * i) * LD + k);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][j] = fmaf(a[i].w, b[j].w, fmaf(a[i].z, b[j].z, fmaf(a[i].y, b[j].y, fmaf(a[i].x, b[j].x, s[i][j]))));
    }
  }
  // acc[i] += row ty + 16 i of w (over the first `rows` rows of y) times this thread's dimensions of y: 4 tx.. (and 64 on), or, where a head has 32, 4 (tx % 8).. of the
  // rows whose fourth has this half's parity
  static __device__ __forceinline__ void weigh(float (&acc)[4][WIDE], const float* w, const float* y, int rows, int tx, int ty) {
    const int from = HD == 32 ? (tx >> 3) * 4 : 0, at = (HD == 32 ? tx & 7 : tx) * 4;
#pragma unroll 2
    for (int k = from; k < rows; k += HD == 32 ? 8 : 4) {
      float4 a[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = *reinterpret_cast<const float4*>(w + (ty + 16 * i) * PF32_LDW + k);
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int c = 0; c < WIDE; c += 4) {
          const float4 b = *reinterpret_cast<const float4*>(y + (k + u) * LD + at + c * 16);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float x = u == 0 ? a[i].x : u == 1 ? a[i].y : u == 2 ? a[i].z : a[i].w;
            acc[i][c] = fmaf(x, b.x, acc[i][c]);
            acc[i][c + 1] = fmaf(x, b.y, acc[i][c + 1]);
            acc[i][c + 2] = fmaf(x, b.z, acc[i][c + 2]);
            acc[i][c + 3] = fmaf(x, b.w, acc[i][c + 3]);
          }
        }
    }
  }
  // rows i0 + ty + 16 i below n of the result, times mul[i]
  static __device__ __forceinline__ void store(float (&acc)[4][WIDE], const float (&mul)[4], float* g, long long stride, int lo, int i0, int n, int col, int hd, int tx, int ty) {
    const bool pieces = ((hd | (int)(stride & 3) | col) & 3) == 0 && (reinterpret_cast<uintptr_t>(g) & 15) == 0;
    const int at = (HD == 32 ? tx & 7 : tx) * 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = i0 + ty + 16 * i;
      float* to = g + (lo + row) * stride + col;
#pragma unroll
      for (int c = 0; c < WIDE; c += 4) {
        float v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          v[u] = acc[i][c + u];
          if (HD == 32) v[u] += __shfl_xor_sync(0xffffffffu, v[u], 8);
          v[u] *= mul[i];
        }
        const int d = at + c * 16;
        if (row >= n || (HD == 32 && tx >= 8)) continue;
        if (pieces) {
          if (d < hd) *reinterpret_cast<float4*>(to + d) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
#pragma unroll
          for (int u = 0; u < 4; ++u)
            if (d + u < hd) to[d + u] = v[u];
        }
      }
    }
  }
};

__device__ __forceinline__ void f32_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void f32_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <int HD>
__global__ void __launch_bounds__(PF32_THREADS) packed_f32_fwd_kernel(const __grid_constant__ PackedF32Params p) {
  using Tile = F32Tile<HD>;
  extern __shared__ __align__(16) float sm[];
  float *sQ = sm, *sK = sQ + Tile::FLOATS, *sV = sK + Tile::FLOATS, *sP = sV + Tile::FLOATS;
  pdl_launch_dependents();
  pdl_wait();
  const int h = blockIdx.y, hk = h / p.group, hd = p.hd, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  p.plan.others(blockIdx.x, gridDim.x, [&](int r) {
    for (int d = threadIdx.x; d < hd; d += PF32_THREADS) p.out[r * p.os + h * hd + d] = 0.f;
    if (threadIdx.x == 0 && p.lse_out) p.lse_out[(long long)h * p.plan.tokens + r] = -INFINITY;
  });
  const PackedRows t = packed_rows<false>(p.plan, blockIdx.x);
  if (t.i0 >= t.n) return;
  const bool vec = p.vec;
  Tile::fetch(sQ, p.q, p.qs, t.lo, t.i0, t.n, h * hd, hd, vec);
  Tile::fetch(sK, p.k, p.ks, t.lo, 0, t.n, hk * hd, hd, vec);
  f32_commit();
  Tile::fetch(sV, p.v, p.vs, t.lo, 0, t.n, hk * hd, hd, vec);
  f32_commit();
  float acc[4][Tile::WIDE] = {}, m[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) { m[i] = -INFINITY; l[i] = 0.f; }
  const int end = min(t.n, t.i0 + PF32_ROWS);
  for (int j0 = 0; j0 < end; j0 += PF32_ROWS) {
    const bool more = j0 + PF32_ROWS < end;
    f32_wait<1>();
    __syncthreads();                                          // K is there; the last weights have been read
    float s[4][4];
    Tile::scores(s, sQ, sK, tx, ty);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = t.i0 + ty + 16 * i;
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = j0 + tx + 16 * j <= row ? s[i][j] * p.scale : -INFINITY;
        top = fmaxf(top, s[i][j]);
      }
#pragma unroll
      for (int o = 1; o < 16; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float mn = fmaxf(m[i], top), mu = mn == -INFINITY ? 0.f : mn, alpha = __expf(m[i] - mu);
      m[i] = mn;
      l[i] *= alpha;
#pragma unroll
      for (int c = 0; c < Tile::WIDE; ++c) acc[i][c] *= alpha;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float e = __expf(s[i][j] - mu);
        l[i] += e;
        sP[(ty + 16 * i) * PF32_LDW + tx + 16 * j] = e;
      }
    }
    f32_wait<0>();
    __syncthreads();                                          // V and the weights are there, K has been read
    if (more) Tile::fetch(sK, p.k, p.ks, t.lo, j0 + PF32_ROWS, t.n, hk * hd, hd, vec);
    f32_commit();
    Tile::weigh(acc, sP, sV, min(PF32_ROWS, end - j0), tx, ty);
    __syncthreads();                                          // V has been read
    if (more) Tile::fetch(sV, p.v, p.vs, t.lo, j0 + PF32_ROWS, t.n, hk * hd, hd, vec);
    f32_commit();
  }
  float mul[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], o);
    mul[i] = 1.f / l[i];
    const int row = t.i0 + ty + 16 * i;
    if (tx == 0 && row < t.n && p.lse_out) p.lse_out[(long long)h * p.plan.tokens + t.lo + row] = m[i] + logf(l[i]);
  }
  Tile::store(acc, mul, p.out, p.os, t.lo, t.i0, t.n, h * hd, hd, tx, ty);
}

// dQ: rows are queries
template <int HD>
__device__ __forceinline__ void packed_f32_bwd_q(float* sm, const PackedF32Params& p) {
  using Tile = F32Tile<HD>;
  float *sQ = sm, *sDO = sQ + Tile::FLOATS, *sK = sDO + Tile::FLOATS, *sV = sK + Tile::FLOATS, *sW = sV + Tile::FLOATS;
  const int h = blockIdx.y, hk = h / p.group, hd = p.hd, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  p.plan.others(blockIdx.x, gridDim.x, [&](int r) {
    for (int d = threadIdx.x; d < hd; d += PF32_THREADS) p.dq[r * p.dqs + h * hd + d] = 0.f;
  });
  const PackedRows t = packed_rows<false>(p.plan, blockIdx.x);
  if (t.i0 >= t.n) return;
  const bool vec = p.vec;
  Tile::fetch(sQ, p.q, p.qs, t.lo, t.i0, t.n, h * hd, hd, vec);
  Tile::fetch(sDO, p.dout, p.dos, t.lo, t.i0, t.n, h * hd, hd, vec);
  Tile::fetch(sK, p.k, p.ks, t.lo, 0, t.n, hk * hd, hd, vec);
  f32_commit();
  Tile::fetch(sV, p.v, p.vs, t.lo, 0, t.n, hk * hd, hd, vec);
  f32_commit();
  float L[4], delta[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = t.i0 + ty + 16 * i;
    L[i] = row < t.n ? p.lse[(long long)h * p.plan.tokens + t.lo + row] : 0.f;
    delta[i] = 0.f;
    if (row < t.n)
      for (int d = tx; d < hd; d += 16) delta[i] = fmaf(p.dout[(t.lo + row) * p.dos + h * hd + d], p.o[(t.lo + row) * p.os + h * hd + d], delta[i]);
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) delta[i] += __shfl_xor_sync(0xffffffffu, delta[i], o);
  }
  float acc[4][Tile::WIDE] = {};
  const int end = min(t.n, t.i0 + PF32_ROWS);
  for (int j0 = 0; j0 < end; j0 += PF32_ROWS) {
    const bool more = j0 + PF32_ROWS < end;
    f32_wait<1>();
    __syncthreads();
    float s[4][4], dp[4][4];
    Tile::scores(s, sQ, sK, tx, ty);
    f32_wait<0>();
    __syncthreads();
    Tile::scores(dp, sDO, sV, tx, ty);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = t.i0 + ty + 16 * i;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool alive = j0 + tx + 16 * j <= row && row < t.n;
        sW[(ty + 16 * i) * PF32_LDW + tx + 16 * j] = alive ? __expf(s[i][j] * p.scale - L[i]) * (dp[i][j] - delta[i]) : 0.f;
      }
    }
    __syncthreads();                                          // the weights are there, V has been read
    if (more) Tile::fetch(sV, p.v, p.vs, t.lo, j0 + PF32_ROWS, t.n, hk * hd, hd, vec);
    Tile::weigh(acc, sW, sK, min(PF32_ROWS, end - j0), tx, ty);
    __syncthreads();                                          // K has been read
    if (more) Tile::fetch(sK, p.k, p.ks, t.lo, j0 + PF32_ROWS, t.n, hk * hd, hd, vec);
    f32_commit();
    f32_commit();                                             // both in the older group: neither is waited for without the other
  }
  const float mul[4] = {p.scale, p.scale, p.scale, p.scale};
  Tile::store(acc, mul, p.dq, p.dqs, t.lo, t.i0, t.n, h * hd, hd, tx, ty);
}

// dK, dV: rows are keys; the queries of the group's heads stream by with their log-sum-exp and delta = rowsum(dO * O).  blockIdx.y: the query head that this block of
// a cluster works on; without a cluster the first of a group stands for all.
template <int HD>
__device__ __forceinline__ void packed_f32_bwd_kv(float* sm, const PackedF32Params& p) {
  using Tile = F32Tile<HD>;
  float *sK = sm, *sV = sK + Tile::FLOATS, *sQ = sV + Tile::FLOATS, *sDO = sQ + Tile::FLOATS, *sW = sDO + Tile::FLOATS;
  __shared__ float sL[PF32_ROWS], sDelta[PF32_ROWS];
  const int hk = blockIdx.y / p.group, first = blockIdx.y % p.group, hd = p.hd, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int parts = p.group <= PF32_CLUSTER ? p.group : 1, heads = p.group / parts;
  if (first >= parts) return;
  if (first == 0) p.plan.others(blockIdx.x, gridDim.x, [&](int r) {
    for (int d = threadIdx.x; d < hd; d += PF32_THREADS) p.dk[r * p.dks + hk * hd + d] = p.dv[r * p.dvs + hk * hd + d] = 0.f;
  });
  const PackedRows t = packed_rows<true>(p.plan, blockIdx.x);
  if (t.i0 >= t.n) return;
  const bool vec = p.vec;
  Tile::fetch(sK, p.k, p.ks, t.lo, t.i0, t.n, hk * hd, hd, vec);
  Tile::fetch(sV, p.v, p.vs, t.lo, t.i0, t.n, hk * hd, hd, vec);
  float dk[4][Tile::WIDE] = {}, dv[4][Tile::WIDE] = {};
  // steps: tiles of queries from the block's own rows on, of one head after the other
  const int per = (t.n - t.i0 + PF32_ROWS - 1) / PF32_ROWS, steps = per * heads, h0 = blockIdx.y;
  const auto fetch = [&](int step) {
    const int h = h0 + step / per, q0 = t.i0 + step % per * PF32_ROWS;
    Tile::fetch(sQ, p.q, p.qs, t.lo, q0, t.n, h * hd, hd, vec);
    Tile::fetch(sDO, p.dout, p.dos, t.lo, q0, t.n, h * hd, hd, vec);
    f32_commit();
  };
  fetch(0);
  for (int step = 0; step < steps; ++step) {
    const int h = h0 + step / per, q0 = t.i0 + step % per * PF32_ROWS;
    {                                                         // four threads to a query
      const int r = threadIdx.x >> 2, part = threadIdx.x & 3, row = q0 + r;
      float delta = 0.f, L = INFINITY;
      if (row < t.n) {
        L = p.lse[(long long)h * p.plan.tokens + t.lo + row];
        const float *pd = p.dout + (t.lo + row) * p.dos + h * hd, *po = p.o + (t.lo + row) * p.os + h * hd;
        if (vec) {
#pragma unroll 4
          for (int d = part * 4; d < hd; d += 16) {
            const float4 a = *reinterpret_cast<const float4*>(pd + d), c = *reinterpret_cast<const float4*>(po + d);
            delta = fmaf(a.x, c.x, fmaf(a.y, c.y, fmaf(a.z, c.z, fmaf(a.w, c.w, delta))));
          }
        } else {
          for (int d = part * 4; d < hd; d += 16)              // in the same order
            for (int u = 3; u >= 0; --u)
              if (d + u < hd) delta = fmaf(pd[d + u], po[d + u], delta);
        }
      }
      delta += __shfl_xor_sync(0xffffffffu, delta, 1);
      delta += __shfl_xor_sync(0xffffffffu, delta, 2);
      if (part == 0) {
        sDelta[r] = delta;
        sL[r] = L;
      }
    }
    f32_wait<0>();
    __syncthreads();
    float s[4][4], dp[4][4];
    Tile::scores(s, sK, sQ, tx, ty);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int key = t.i0 + ty + 16 * i;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int query = q0 + tx + 16 * j;
        s[i][j] = key <= query && query < t.n && key < t.n ? __expf(s[i][j] * p.scale - sL[tx + 16 * j]) : 0.f;
        sW[(ty + 16 * i) * PF32_LDW + tx + 16 * j] = s[i][j];
      }
    }
    __syncthreads();
    const int rows = min(PF32_ROWS, (t.n - q0 + 3) & ~3);
    Tile::weigh(dv, sW, sDO, rows, tx, ty);
    Tile::scores(dp, sV, sDO, tx, ty);
    __syncthreads();                                          // P has been read
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int key = t.i0 + ty + 16 * i;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int query = q0 + tx + 16 * j;
        const bool alive = key <= query && query < t.n && key < t.n;
        sW[(ty + 16 * i) * PF32_LDW + tx + 16 * j] = alive ? s[i][j] * (dp[i][j] - sDelta[tx + 16 * j]) : 0.f;
      }
    }
    __syncthreads();
    Tile::weigh(dk, sW, sQ, rows, tx, ty);
    __syncthreads();                                          // Q and dO have been read
    if (step + 1 < steps) fetch(step + 1);
  }
  if (parts > 1) {
    // every block's sums to its shared memory, in the order of its threads; each then adds up a share of the places over the cluster
    constexpr int PLACES = 4 * Tile::WIDE;                    // of a thread, for dK and for dV
    const cg::cluster_group cluster = cg::this_cluster();
#pragma unroll
    for (int c = 0; c < PLACES; ++c) {
      sm[c * PF32_THREADS + threadIdx.x] = dk[c / Tile::WIDE][c % Tile::WIDE];
      sm[(PLACES + c) * PF32_THREADS + threadIdx.x] = dv[c / Tile::WIDE][c % Tile::WIDE];
    }
    cluster.sync();
    for (int c = first; c < 2 * PLACES; c += parts) {
      float sum = 0.f;
      for (int b = 0; b < parts; ++b) sum += cluster.map_shared_rank(sm, b)[c * PF32_THREADS + threadIdx.x];
      cluster.map_shared_rank(sm, 0)[c * PF32_THREADS + threadIdx.x] = sum;      // nobody else reads this place of any block
    }
    cluster.sync();
    if (first > 0) return;
#pragma unroll
    for (int c = 0; c < PLACES; ++c) {
      dk[c / Tile::WIDE][c % Tile::WIDE] = sm[c * PF32_THREADS + threadIdx.x];
      dv[c / Tile::WIDE][c % Tile::WIDE] = sm[(PLACES + c) * PF32_THREADS + threadIdx.x];
    }
  }
  const float one[4] = {1.f, 1.f, 1.f, 1.f}, mul[4] = {p.scale, p.scale, p.scale, p.scale};
  Tile::store(dk, mul, p.dk, p.dks, t.lo, t.i0, t.n, hk * hd, hd, tx, ty);
  Tile::store(dv, one, p.dv, p.dvs, t.lo, t.i0, t.n, hk * hd, hd, tx, ty);
}

// Both gradients in one launch: the first half of the grid takes dK and dV, the second dQ
template <int HD>
__global__ void __launch_bounds__(PF32_THREADS) packed_f32_bwd_kernel(const __grid_constant__ PackedF32Params p) {
  extern __shared__ __align__(16) float sm[];
  pdl_launch_dependents();
  pdl_wait();
  if (blockIdx.z == 0) packed_f32_bwd_kv<HD>(sm, p);
  else packed_f32_bwd_q<HD>(sm, p);
}

static bool packed_f32_vec(const PackedF32Params& p) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v) | reinterpret_cast<uintptr_t>(p.o) |
                       reinterpret_cast<uintptr_t>(p.dout);
  return ((p.hd | p.qs | p.ks | p.vs | p.os | p.dos) & 3) == 0 && (at & 15) == 0;
}

template <int HD, bool BWD>
static int packed_f32_run(const PackedF32Params& p, dim3 grid, cudaStream_t st) {
  static std::atomic<unsigned long long> allowed;
  constexpr int BYTES = ((BWD ? 4 : 3) * F32Tile<HD>::FLOATS + PF32_ROWS * PF32_LDW) * (int)sizeof(float);
  static_assert(!BWD || BYTES >= 8 * F32Tile<HD>::WIDE * PF32_THREADS * (int)sizeof(float), "a cluster's sums");
  void (*const kernel)(const PackedF32Params) = BWD ? packed_f32_bwd_kernel<HD> : packed_f32_fwd_kernel<HD>;
  if (allow_smem(allowed, (const void*)kernel, BYTES) != cudaSuccess) return OA_ERR_LAUNCH;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(PF32_THREADS);
  cfg.dynamicSmemBytes = BYTES;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = attr[0].val.clusterDim.z = 1;
  attr[0].val.clusterDim.y = BWD && p.group <= PF32_CLUSTER ? p.group : 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_on((long long)grid.x * grid.y * grid.z <= PDL_SHORT_BLOCKS) ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, p) == cudaSuccess ? OA_OK : OA_ERR_LAUNCH;
}

template <bool BWD>
static int packed_f32_launch(PackedF32Params& p, cudaStream_t st) {
  p.vec = packed_f32_vec(p);
  const long long blocks = packed_max_tiles(p.plan.tokens, p.plan.batch) * (long long)(PACKED_TILE / PF32_ROWS);
  if (blocks > 0x7fffffffll) return OA_ERR_TOO_LARGE;
  const dim3 grid((unsigned)(blocks > 0 ? blocks : 1), (unsigned)p.q_heads, BWD ? 2 : 1);
  return p.hd <= 32 ? packed_f32_run<32, BWD>(p, grid, st) : p.hd <= 64 ? packed_f32_run<64, BWD>(p, grid, st) : packed_f32_run<128, BWD>(p, grid, st);
}

}  // namespace oa

using namespace oa;

static int packed_f32_check(int tokens, int batch, int q_heads, int kv_heads, int head_dim, float scale) {
  if (tokens < 0 || batch < 0 || !(scale > 0.f) || kv_heads < 1 || q_heads < 1 || q_heads % kv_heads) return OA_ERR_ARG;
  if (tokens > PACKED_MAX_TOKENS || batch > PACKED_MAX_BATCH || q_heads > 65535) return OA_ERR_TOO_LARGE;
  return head_dim < 1 || head_dim > 128 ? OA_ERR_UNSUPPORTED : OA_OK;
}

extern "C" int oa_packed_attn_f32(const float* q, const float* k, const float* v, const int* plan, float* o, float* lse, int tokens, int batch, int q_heads,
                                  int kv_heads, int head_dim, long long q_stride, long long k_stride, long long v_stride, long long o_stride, float scale,
                                  void* stream) {
  if (int rc = packed_f32_check(tokens, batch, q_heads, kv_heads, head_dim, scale)) return rc;
  if (tokens == 0) return OA_OK;
  PackedF32Params p{};
  p.q = q; p.k = k; p.v = v; p.out = o; p.lse_out = lse;
  p.qs = q_stride; p.ks = k_stride; p.vs = v_stride; p.os = o_stride;
  p.plan = {plan, batch, tokens};
  p.q_heads = q_heads; p.kv_heads = kv_heads; p.group = q_heads / kv_heads; p.hd = head_dim; p.scale = scale;
  return packed_f32_launch<false>(p, (cudaStream_t)stream);
}

extern "C" int oa_packed_attn_f32_bwd(const float* q, const float* k, const float* v, const float* o, const float* dout, const float* lse, const int* plan,
                                      float* dq, float* dk, float* dv, int tokens, int batch, int q_heads, int kv_heads, int head_dim, long long q_stride,
                                      long long k_stride, long long v_stride, long long o_stride, long long do_stride, long long dq_stride,
                                      long long dk_stride, long long dv_stride, float scale, void* stream) {
  if (int rc = packed_f32_check(tokens, batch, q_heads, kv_heads, head_dim, scale)) return rc;
  if (tokens == 0) return OA_OK;
  PackedF32Params p{};
  p.q = q; p.k = k; p.v = v; p.o = o; p.dout = dout; p.lse = lse; p.dq = dq; p.dk = dk; p.dv = dv;
  p.qs = q_stride; p.ks = k_stride; p.vs = v_stride; p.os = o_stride; p.dos = do_stride; p.dqs = dq_stride; p.dks = dk_stride; p.dvs = dv_stride;
  p.plan = {plan, batch, tokens};
  p.q_heads = q_heads; p.kv_heads = kv_heads; p.group = q_heads / kv_heads; p.hd = head_dim; p.scale = scale;
  return packed_f32_launch<true>(p, (cudaStream_t)stream);
}
