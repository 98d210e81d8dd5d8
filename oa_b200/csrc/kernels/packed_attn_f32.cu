// Causal attention over packed sequences in fp32, with grouped heads, forward and backward: the engine's exact precision, and gradient checks.
//
// Query head h reads key-value head h / group.  Within a sequence the work is that of attn_f32.cu: a block of 128 threads owns 128 / (DS KS) rows of one
// head, the other side streams through shared memory 32 rows at a time.  A block finds its rows in the plan's lists, of tiles (128 rows of a sequence,
// the longest first) and of short sequences: a tile is KS DS blocks.  Rows of other sequences are never read: what a sequence holds does not reach another.  dK and
// dV of a key-value head add up over the query heads that share it, one after the other in one block, so that there is one writer and one order.
#include "attn_f32.cuh"
#include "packed.cuh"
#include "per_device.h"
#include "api.h"

namespace oa {

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
template <int ROWS, bool MIRROR>
__device__ __forceinline__ PackedRows packed_rows(const PackedPlan& plan, int block) {
  constexpr int SUBS = PACKED_TILE / ROWS;
  const int at = block / SUBS, sub = block % SUBS;
  const int tiles = plan.tiles();
  if (at >= tiles + plan.shorts()) return {0, 0, 0};
  const int4 t = at < tiles ? plan.tile(at) : plan.brief(at - tiles);
  const int n = t.y - t.x, idx = MIRROR ? (n + PACKED_TILE - 1) / PACKED_TILE - 1 - t.z : t.z;
  return {t.x, n, idx * PACKED_TILE + sub * ROWS};
}

template <int DS, int KS>
__global__ void __launch_bounds__(AF_THREADS) packed_f32_fwd_kernel(const PackedF32Params p) {
  using Cfg = AfCfg<DS, KS>;
  constexpr int NJ = AF_TILE / KS;
  __shared__ __align__(16) float sK[Cfg::BUFS * Cfg::TILE], sV[Cfg::BUFS * Cfg::TILE];
  pdl_wait();
  const int h = blockIdx.y, hk = h / p.group, hd = p.hd;
  p.plan.others(blockIdx.x, gridDim.x, [&](int r) {
    for (int d = threadIdx.x; d < hd; d += AF_THREADS) p.out[r * p.os + h * hd + d] = 0.f;
    if (threadIdx.x == 0 && p.lse_out) p.lse_out[(long long)h * p.plan.tokens + r] = -INFINITY;
  });
  const PackedRows t = packed_rows<Cfg::ROWS, false>(p.plan, blockIdx.x);
  if (t.i0 >= t.n) return;
  const int i = t.i0 + threadIdx.x / Cfg::TPR, seg = threadIdx.x % DS, ks = threadIdx.x % Cfg::TPR / DS;
  const bool row_ok = i < t.n;
  const long long row = t.lo + (row_ok ? i : 0);
  float qr[AF_W], acc[AF_W];
  af_own(qr, p.q + row * p.qs + h * hd + seg * AF_W, hd - seg * AF_W, row_ok, p.vec);
#pragma unroll
  for (int d = 0; d < AF_W; ++d) {
    qr[d] *= p.scale;
    acc[d] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  const int kend = min(t.n, t.i0 + Cfg::ROWS);
  af_stream<DS, KS>(sK, sV, p.k, p.ks, p.v, p.vs, t.lo, 0, kend, t.n, hk * hd, hd, p.vec, [&](int j0, const float* tk, const float* tv) {
    float s[NJ];
    float mt = -INFINITY;
#pragma unroll
    for (int jj = 0; jj < NJ; ++jj) {
      const int j = jj * KS + ks;
      const float d = af_reduce<DS>(af_dot(qr, tk + (j * DS + seg) * AF_SEG));
      s[jj] = j0 + j <= i ? d : -INFINITY;
      mt = fmaxf(mt, s[jj]);
    }
    const float mn = fmaxf(m, mt), mu = mn == -INFINITY ? 0.f : mn;
    const float alpha = __expf(m - mu);
    float ls = 0.f;
#pragma unroll
    for (int d = 0; d < AF_W; ++d) acc[d] *= alpha;
#pragma unroll
    for (int jj = 0; jj < NJ; ++jj) {
      const float e = __expf(s[jj] - mu);
      ls += e;
      af_axpy(acc, e, tv + ((jj * KS + ks) * DS + seg) * AF_SEG);
    }
    l = l * alpha + ls;
    m = mn;
  });
  if constexpr (KS == 4) {                                     // the groups' maxima and sums meet
    float mx = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, DS));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2 * DS));
    const float w = __expf(m - (mx == -INFINITY ? 0.f : mx));
    l *= w;
    l += __shfl_xor_sync(0xffffffffu, l, DS);
    l += __shfl_xor_sync(0xffffffffu, l, 2 * DS);
#pragma unroll
    for (int d = 0; d < AF_W; ++d) acc[d] *= w;
    m = mx;
    af_scatter_sum<DS, KS>(acc, ks);
  }
  if (!row_ok) return;
  const float inv = 1.f / l;
#pragma unroll
  for (int u = 0; u < AF_W / KS; ++u) {
    const int d = seg * AF_W + af_first<KS>(ks) + u;
    if (d < hd) p.out[row * p.os + h * hd + d] = acc[u] * inv;
  }
  if (seg == 0 && ks == 0 && p.lse_out) p.lse_out[(long long)h * p.plan.tokens + row] = m + logf(l);
}

// dQ: rows are queries
template <int DS, int KS>
__device__ __forceinline__ void packed_f32_bwd_q(float* sK, float* sV, const PackedF32Params& p) {
  using Cfg = AfCfg<DS, KS>;
  constexpr int NJ = AF_TILE / KS;
  const int h = blockIdx.y, hk = h / p.group, hd = p.hd;
  p.plan.others(blockIdx.x, gridDim.x, [&](int r) {
    for (int d = threadIdx.x; d < hd; d += AF_THREADS) p.dq[r * p.dqs + h * hd + d] = 0.f;
  });
  const PackedRows t = packed_rows<Cfg::ROWS, false>(p.plan, blockIdx.x);
  if (t.i0 >= t.n) return;
  const int i = t.i0 + threadIdx.x / Cfg::TPR, seg = threadIdx.x % DS, ks = threadIdx.x % Cfg::TPR / DS;
  const bool row_ok = i < t.n;
  const long long row = t.lo + (row_ok ? i : 0);
  const int left = hd - seg * AF_W, col = h * hd + seg * AF_W;
  float qr[AF_W], dor[AF_W], acc[AF_W];
  float delta = 0.f;
  af_own(acc, p.o + row * p.os + col, left, row_ok, p.vec);
  af_own(dor, p.dout + row * p.dos + col, left, row_ok, p.vec);
  af_own(qr, p.q + row * p.qs + col, left, row_ok, p.vec);
#pragma unroll
  for (int d = 0; d < AF_W; ++d) {
    qr[d] *= p.scale;
    if (d < left) delta = fmaf(dor[d], acc[d], delta);
    acc[d] = 0.f;
  }
  delta = af_reduce<DS>(delta);
  const float L = row_ok ? p.lse[(long long)h * p.plan.tokens + row] : 0.f;
  const int kend = min(t.n, t.i0 + Cfg::ROWS);
  af_stream<DS, KS>(sK, sV, p.k, p.ks, p.v, p.vs, t.lo, 0, kend, t.n, hk * hd, hd, p.vec, [&](int j0, const float* tk, const float* tv) {
#pragma unroll 4
    for (int jj = 0; jj < NJ; ++jj) {
      const int j = jj * KS + ks;
      const float* kr = tk + (j * DS + seg) * AF_SEG;
      const float d = af_reduce<DS>(af_dot(qr, kr));
      const float dp = af_reduce<DS>(af_dot(dor, tv + (j * DS + seg) * AF_SEG));
      const float ds = row_ok && j0 + j <= i ? __expf(d - L) * (dp - delta) * p.scale : 0.f;
      af_axpy(acc, ds, kr);
    }
  });
  af_scatter_sum<DS, KS>(acc, ks);
  if (!row_ok) return;
#pragma unroll
  for (int u = 0; u < AF_W / KS; ++u) {
    const int d = seg * AF_W + af_first<KS>(ks) + u;
    if (d < hd) p.dq[row * p.dqs + h * hd + d] = acc[u];
  }
}

// dK, dV: rows are keys; the queries of every head of the group stream by with their log-sum-exp and delta = rowsum(dO * O)
template <int DS, int KS>
__device__ __forceinline__ void packed_f32_bwd_kv(float* sQ, float* sDO, const PackedF32Params& p) {
  using Cfg = AfCfg<DS, KS>;
  constexpr int NI = AF_TILE / KS;
  __shared__ float sL[2][AF_TILE], sDelta[2][AF_TILE];
  const int hk = blockIdx.y, hd = p.hd;
  if (hk >= p.kv_heads) return;
  p.plan.others(blockIdx.x, gridDim.x, [&](int r) {
    for (int d = threadIdx.x; d < hd; d += AF_THREADS) p.dk[r * p.dks + hk * hd + d] = p.dv[r * p.dvs + hk * hd + d] = 0.f;
  });
  const PackedRows t = packed_rows<Cfg::ROWS, true>(p.plan, blockIdx.x);
  if (t.i0 >= t.n) return;
  const int j = t.i0 + threadIdx.x / Cfg::TPR, seg = threadIdx.x % DS, ks = threadIdx.x % Cfg::TPR / DS;
  const bool row_ok = j < t.n;
  const long long row = t.lo + (row_ok ? j : 0);
  const int left = hd - seg * AF_W, col = hk * hd + seg * AF_W;
  float kr[AF_W], vr[AF_W], acck[AF_W], accv[AF_W];
  af_own(kr, p.k + row * p.ks + col, left, row_ok, p.vec);
  af_own(vr, p.v + row * p.vs + col, left, row_ok, p.vec);
#pragma unroll
  for (int d = 0; d < AF_W; ++d) {
    kr[d] *= p.scale;
    acck[d] = 0.f; accv[d] = 0.f;
  }
  const int istart = t.i0 / AF_TILE * AF_TILE;               // first query tile that any key of this block is seen by
  for (int h = hk * p.group; h < (hk + 1) * p.group; ++h) {
    // delta and log-sum-exp of the 32 queries of a tile: four threads to a query.  Fetched before a tile is worked on, those of the next one are written behind
    // it, to the other of two slots: the last warps may still read this one's.
    const int r = threadIdx.x >> 2, part = threadIdx.x & 3;
    float delta = 0.f, lse = INFINITY;
    const auto fetch = [&](int i0) {
      delta = 0.f;
      lse = INFINITY;
      if (i0 + r < t.n) {
        const float *pd = p.dout + (t.lo + i0 + r) * p.dos + h * hd, *po = p.o + (t.lo + i0 + r) * p.os + h * hd;
        lse = p.lse[(long long)h * p.plan.tokens + t.lo + i0 + r];
        if (p.vec) {
#pragma unroll
          for (int d = part * 4; d < DS * AF_W; d += 16)
            if (d < hd) {
              const float4 a = *reinterpret_cast<const float4*>(pd + d), c = *reinterpret_cast<const float4*>(po + d);
              delta = fmaf(a.x, c.x, fmaf(a.y, c.y, fmaf(a.z, c.z, fmaf(a.w, c.w, delta))));
            }
        } else {
          for (int d = part * 4; d < hd; d += 16)              // in the same order
            for (int u = 3; u >= 0; --u)
              if (d + u < hd) delta = fmaf(pd[d + u], po[d + u], delta);
        }
      }
    };
    const auto keep = [&](int slot) {
      delta += __shfl_xor_sync(0xffffffffu, delta, 1);
      delta += __shfl_xor_sync(0xffffffffu, delta, 2);
      if (part == 0) {
        sDelta[slot][r] = delta;
        sL[slot][r] = lse;
      }
    };
    int slot = 0;
    __syncthreads();                                          // the last head's last tile has been read
    fetch(istart);
    keep(0);
    af_stream<DS, KS>(sQ, sDO, p.q, p.qs, p.dout, p.dos, t.lo, istart, t.n, t.n, h * hd, hd, p.vec, [&](int i0, const float* tq, const float* td) {
      fetch(i0 + AF_TILE);
#pragma unroll 4
      for (int jj = 0; jj < NI; ++jj) {
        const int ii = jj * KS + ks;
        const float* qrow = tq + (ii * DS + seg) * AF_SEG;
        const float* dorow = td + (ii * DS + seg) * AF_SEG;
        const float d = af_reduce<DS>(af_dot(kr, qrow));
        const float dp = af_reduce<DS>(af_dot(vr, dorow));
        const int qi = i0 + ii;
        const bool alive = row_ok && qi < t.n && j <= qi;
        const float e = alive ? __expf(d - sL[slot][ii]) : 0.f;
        const float ds = alive ? e * (dp - sDelta[slot][ii]) : 0.f;
        af_axpy(accv, e, dorow);
        af_axpy(acck, ds, qrow);
      }
      keep(slot ^ 1);
      slot ^= 1;
    });
  }
  af_scatter_sum<DS, KS>(acck, ks);
  af_scatter_sum<DS, KS>(accv, ks);
  if (!row_ok) return;
#pragma unroll
  for (int u = 0; u < AF_W / KS; ++u) {
    const int d = seg * AF_W + af_first<KS>(ks) + u;
    if (d < hd) {
      p.dk[row * p.dks + hk * hd + d] = acck[u] * p.scale;
      p.dv[row * p.dvs + hk * hd + d] = accv[u];
    }
  }
}

// Both gradients in one launch: the first half of the grid takes dK and dV, the second dQ
template <int DS, int KS>
__global__ void __launch_bounds__(AF_THREADS) packed_f32_bwd_kernel(const PackedF32Params p) {
  using Cfg = AfCfg<DS, KS>;
  __shared__ __align__(16) float sx[Cfg::BUFS * Cfg::TILE], sy[Cfg::BUFS * Cfg::TILE];
  pdl_wait();
  if (blockIdx.z == 0) packed_f32_bwd_kv<DS, KS>(sx, sy, p);
  else packed_f32_bwd_q<DS, KS>(sx, sy, p);
}

// DS, or -4 DS for KS = 4, by the rule of attn_f32.cu
static int packed_f32_split(int hd, long long tiles, int heads) {
  const int wide = hd <= 32 ? 1 : hd <= 64 ? 2 : 4;
  return hd <= 64 && tiles * wide * heads <= 300 ? -4 * wide : wide;
}

static bool packed_f32_vec(const PackedF32Params& p) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v) | reinterpret_cast<uintptr_t>(p.o) |
                       reinterpret_cast<uintptr_t>(p.dout);
  return ((p.hd | p.qs | p.ks | p.vs | p.os | p.dos) & 3) == 0 && (at & 15) == 0;
}

template <bool BWD>
static int packed_f32_launch(PackedF32Params& p, cudaStream_t st) {
  p.vec = packed_f32_vec(p);
  const long long tiles = packed_max_tiles(p.plan.tokens, p.plan.batch);
  const int split = packed_f32_split(p.hd, tiles, p.q_heads), subs = split < 0 ? -split : split;
  if (tiles * subs > 0x7fffffffll) return OA_ERR_TOO_LARGE;
  const dim3 grid((unsigned)(tiles * subs > 0 ? tiles * subs : 1), (unsigned)p.q_heads, BWD ? 2 : 1);
#define PACKED_F32(D, S)                                                                                         \
  (BWD ? launch_short(packed_f32_bwd_kernel<D, S>, grid, dim3(AF_THREADS), 0, st, p)                             \
       : launch_short(packed_f32_fwd_kernel<D, S>, grid, dim3(AF_THREADS), 0, st, p))
  if (split == -4) PACKED_F32(1, 4);
  else if (split == -8) PACKED_F32(2, 4);
  else if (split == 1) PACKED_F32(1, 1);
  else if (split == 2) PACKED_F32(2, 1);
  else PACKED_F32(4, 1);
#undef PACKED_F32
  return cudaGetLastError() == cudaSuccess ? OA_OK : OA_ERR_LAUNCH;
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
