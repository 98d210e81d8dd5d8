// Causal attention over packed sequences of up to 64 rows, forward and backward, bf16 in / fp32 accumulate: the sequences that a tile of 128 x 128 would be
// mostly empty for (packed_attn.cu has the mathematics and the longer ones).
//
// A block of four warps works on one sequence and one head (backward: one key-value head with its query heads in turn).  Its rows come to shared memory by
// cp.async, in 16-byte pieces swizzled over eight banks' groups; rows behind the sequence up to the next 16 are zeros.  A warp takes 16 queries (forward, dQ)
// or 16 keys (dK, dV) and the products run on mma.sync, whose accumulators are the next product's operand as they stand: tiles this small cannot
// fill a tcgen05 instruction.  Backward, scores are worked out twice, with the keys as rows for dK and dV and with the queries as rows for dQ.  Bound by latency: loads,
// a chain of products and exponentials, stores, one after the other, which as many blocks as fit on an SM cover for one another.
#include "common.cuh"
#include "packed.cuh"
#include "per_device.h"
#include "api.h"
#include "packed_short.h"

namespace oa {

constexpr int PS_THREADS = 128;
constexpr float PS_LOG2E = 1.4426950408889634f;

// [64][HD] bf16 in shared memory
template <int HD>
struct ShortTile {
  static constexpr int BYTES = PACKED_SHORT * HD * 2, CHUNKS = HD / 8;
  static __device__ __forceinline__ uint32_t at(uint32_t base, int row, int chunk) { return base + row * (HD * 2) + ((chunk ^ (row & 7)) << 4); }
  // rows [0, n) from memory, zeros up to `rows`
  static __device__ __forceinline__ void fetch(uint32_t base, const __nv_bfloat16* from, long long stride, int n, int rows) {
    for (int i = threadIdx.x; i < rows * CHUNKS; i += PS_THREADS) {
      const int r = i / CHUNKS, c = i % CHUNKS;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at(base, r, c)), "l"(from + (r < n ? r : 0) * stride + c * 8), "r"(r < n ? 16 : 0) : "memory");
    }
  }
  // [16 rows x 16 dimensions] as the left operand, rows r0.., dimensions 16 k..
  static __device__ __forceinline__ void left(uint32_t (&a)[4], uint32_t base, int r0, int k, int lane) {
    ld4(a, at(base, r0 + (lane & 15), 2 * k + (lane >> 4)));
  }
  // the same rows as the right operand of two products of 8 columns each (columns are rows here, the reduction runs along dimensions)
  static __device__ __forceinline__ void right(uint32_t (&b)[4], uint32_t base, int r0, int k, int lane) {
    ld4(b, at(base, r0 + (lane & 7) + ((lane >> 4) << 3), 2 * k + ((lane >> 3) & 1)));
  }
  // ... and where the reduction runs along the 16 rows r0.., the columns are dimensions 16 c..
  static __device__ __forceinline__ void right_t(uint32_t (&b)[4], uint32_t base, int r0, int c, int lane) {
    const uint32_t p = at(base, r0 + (lane & 15), 2 * c + (lane >> 4));
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(b[0]), "=r"(b[1]), "=r"(b[2]), "=r"(b[3]) : "r"(p) : "memory");
  }
  static __device__ __forceinline__ void ld4(uint32_t (&a)[4], uint32_t p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3]) : "r"(p) : "memory");
  }
};

__device__ __forceinline__ void short_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void short_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void short_wait() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }

// [16 x 16] += rows of x times rows of y, over HD dimensions: d[0], d[1] are the halves of 8 columns
template <int HD>
__device__ __forceinline__ void short_scores(float (&d)[2][4], uint32_t x, int x0, uint32_t y, int y0, int lane) {
#pragma unroll
  for (int k = 0; k < HD / 16; ++k) {
    uint32_t a[4], b[4];
    ShortTile<HD>::left(a, x, x0, k, lane);
    ShortTile<HD>::right(b, y, y0, k, lane);
    short_mma(d[0], a, b[0], b[1]);
    short_mma(d[1], a, b[2], b[3]);
  }
}
// acc[16 x HD] += w[16 x 16] times rows y0.. of y
template <int HD>
__device__ __forceinline__ void short_weigh(float (&acc)[HD / 8][4], const uint32_t (&w)[4], uint32_t y, int y0, int lane) {
#pragma unroll
  for (int c = 0; c < HD / 16; ++c) {
    uint32_t b[4];
    ShortTile<HD>::right_t(b, y, y0, c, lane);
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
// A warp's 16 rows r0.. of an accumulator, times mul0 / mul1 for its rows lane / 4 and + 8, to memory through the rows of a tile that only this warp uses: those
// below `n`, in 16-byte pieces
template <int HD>
__device__ __forceinline__ void short_store(const float (&acc)[HD / 8][4], float mul0, float mul1, uint8_t* smem, uint32_t base, int r0, int n, __nv_bfloat16* to,
                                            long long stride, int lane) {
  const uint32_t off = base - smem_u32(smem);
#pragma unroll
  for (int c = 0; c < HD / 8; ++c) {
    *reinterpret_cast<uint32_t*>(smem + ShortTile<HD>::at(off, r0 + (lane >> 2), c) + (lane & 3) * 4) = pack_bf16x2(acc[c][0] * mul0, acc[c][1] * mul0);
    *reinterpret_cast<uint32_t*>(smem + ShortTile<HD>::at(off, r0 + 8 + (lane >> 2), c) + (lane & 3) * 4) = pack_bf16x2(acc[c][2] * mul1, acc[c][3] * mul1);
  }
  __syncwarp();
#pragma unroll
  for (int i = lane; i < 16 * HD / 8; i += 32) {
    const int r = r0 + i / (HD / 8), c = i % (HD / 8);
    if (r < n) *reinterpret_cast<uint4*>(to + r * stride + c * 8) = *reinterpret_cast<const uint4*>(smem + ShortTile<HD>::at(off, r, c));
  }
  __syncwarp();
}

template <int HD>
__global__ void __launch_bounds__(PS_THREADS) packed_short_fwd_kernel(const PackedShortFwd p) {
  using Tile = ShortTile<HD>;
  extern __shared__ __align__(128) uint8_t smem[];
  const uint32_t sq = smem_u32(smem), sk = sq + Tile::BYTES, sv = sk + Tile::BYTES;
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tasks = p.plan.shorts() * p.q_heads;
  const float sl2 = p.scale * PS_LOG2E;
  for (int task = blockIdx.x; task < tasks; task += gridDim.x) {
    const int4 e = p.plan.brief(task / p.q_heads);
    const int h = task % p.q_heads, hk = h / p.group, n = e.y - e.x, rows = (n + 15) & ~15;
    Tile::fetch(sq, p.q + e.x * p.qs + h * HD, p.qs, n, rows);
    Tile::fetch(sk, p.k + e.x * p.ks + hk * HD, p.ks, n, rows);
    Tile::fetch(sv, p.v + e.x * p.vs + hk * HD, p.vs, n, rows);
    short_commit();
    short_wait();
    __syncthreads();
    const int r0 = warp * 16;
    if (r0 < n) {
      // scores of 16 queries and the keys up to them, at most 64
      float s[4][2][4];
      const int i0 = r0 + (lane >> 2), i1 = i0 + 8;                    // this thread's queries
      float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        if (t > warp) break;
#pragma unroll
        for (int c = 0; c < 2; ++c) s[t][c][0] = s[t][c][1] = s[t][c][2] = s[t][c][3] = 0.f;
        short_scores<HD>(s[t], sq, r0, sk, t * 16, lane);
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int j = t * 16 + c * 8 + (lane & 3) * 2 + u;
            s[t][c][u] = j <= i0 ? s[t][c][u] : -INFINITY;
            s[t][c][2 + u] = j <= i1 ? s[t][c][2 + u] : -INFINITY;
            m0 = fmaxf(m0, s[t][c][u]);
            m1 = fmaxf(m1, s[t][c][2 + u]);
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
        if (t > warp) break;
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            l0 += s[t][c][u] = fast_exp2(fmaf(s[t][c][u], sl2, -m0));
            l1 += s[t][c][2 + u] = fast_exp2(fmaf(s[t][c][2 + u], sl2, -m1));
          }
        uint32_t w[4];
        short_operand(w, s[t]);
        short_weigh<HD>(o, w, sv, t * 16, lane);
      }
#pragma unroll
      for (int q = 1; q < 4; q <<= 1) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, q);
        l1 += __shfl_xor_sync(0xffffffffu, l1, q);
      }
      if (p.lse && (lane & 3) == 0) {
        float* to = p.lse + (long long)h * p.plan.tokens + e.x;
        if (i0 < n) to[i0] = (m0 + log2f(l0)) / PS_LOG2E;
        if (i1 < n) to[i1] = (m1 + log2f(l1)) / PS_LOG2E;
      }
      short_store<HD>(o, 1.f / l0, 1.f / l1, smem, sq, r0, n, p.o + e.x * p.os + h * HD, p.os, lane);
    }
    __syncthreads();                                                   // the tiles are free
  }
}

template <int HD>
__global__ void __launch_bounds__(PS_THREADS) packed_short_bwd_kernel(const PackedShortBwd p) {
  using Tile = ShortTile<HD>;
  extern __shared__ __align__(128) uint8_t smem[];
  const uint32_t sq = smem_u32(smem), sdo = sq + Tile::BYTES, sk = sdo + Tile::BYTES, sv = sk + Tile::BYTES;
  float* stat = reinterpret_cast<float*>(smem + 4 * Tile::BYTES);      // [2][64]: -lse log2(e), -delta scale
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tasks = p.plan.shorts() * p.kv_heads, r0 = warp * 16;
  const float sl2 = p.scale * PS_LOG2E, scale = p.scale;
  for (int task = blockIdx.x; task < tasks; task += gridDim.x) {
    const int4 e = p.plan.brief(task / p.kv_heads);
    const int hk = task % p.kv_heads, n = e.y - e.x, rows = (n + 15) & ~15;
    Tile::fetch(sk, p.k + e.x * p.ks + hk * HD, p.ks, n, rows);
    Tile::fetch(sv, p.v + e.x * p.vs + hk * HD, p.vs, n, rows);
    float dk[HD / 8][4], dv[HD / 8][4];
#pragma unroll
    for (int c = 0; c < HD / 8; ++c)
#pragma unroll
      for (int u = 0; u < 4; ++u) dk[c][u] = dv[c][u] = 0.f;
    for (int g = 0; g < p.group; ++g) {
      const int h = hk * p.group + g;
      Tile::fetch(sq, p.q + e.x * p.qs + h * HD, p.qs, n, rows);
      Tile::fetch(sdo, p.dout + e.x * p.dos + h * HD, p.dos, n, rows);
      short_commit();
      if (threadIdx.x < PACKED_SHORT) {
        const bool there = (int)threadIdx.x < n;
        const long long at = (long long)h * p.plan.tokens + e.x + threadIdx.x;
        stat[threadIdx.x] = there ? -p.lse[at] * PS_LOG2E : -INFINITY;
        stat[PACKED_SHORT + threadIdx.x] = there ? -p.delta[at] * scale : 0.f;
      }
      short_wait();
      __syncthreads();
      if (r0 < n) {
        // keys as rows: P^T and dS^T, for the queries from them on
        const int j0 = r0 + (lane >> 2), j1 = j0 + 8;
#pragma unroll 1
        for (int t = warp; t * 16 < n; ++t) {
          float s[2][4] = {}, dp[2][4] = {};
          short_scores<HD>(s, sk, r0, sq, t * 16, lane);
          short_scores<HD>(dp, sv, r0, sdo, t * 16, lane);
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const int i = t * 16 + c * 8 + (lane & 3) * 2 + u;
              const float nl = stat[i], nd = stat[PACKED_SHORT + i];
              const bool a0 = j0 <= i && i < n, a1 = j1 <= i && i < n;
              s[c][u] = a0 ? fast_exp2(fmaf(s[c][u], sl2, nl)) : 0.f;
              s[c][2 + u] = a1 ? fast_exp2(fmaf(s[c][2 + u], sl2, nl)) : 0.f;
              dp[c][u] = a0 ? s[c][u] * fmaf(dp[c][u], scale, nd) : 0.f;
              dp[c][2 + u] = a1 ? s[c][2 + u] * fmaf(dp[c][2 + u], scale, nd) : 0.f;
            }
          uint32_t w[4];
          short_operand(w, s);
          short_weigh<HD>(dv, w, sdo, t * 16, lane);
          short_operand(w, dp);
          short_weigh<HD>(dk, w, sq, t * 16, lane);
        }
        // queries as rows: dS, for the keys up to them
        float dq[HD / 8][4];
#pragma unroll
        for (int c = 0; c < HD / 8; ++c) dq[c][0] = dq[c][1] = dq[c][2] = dq[c][3] = 0.f;
        const float nl0 = stat[j0], nl1 = stat[j1], nd0 = stat[PACKED_SHORT + j0], nd1 = stat[PACKED_SHORT + j1];
#pragma unroll 1
        for (int t = 0; t <= warp; ++t) {
          float s[2][4] = {}, dp[2][4] = {};
          short_scores<HD>(s, sq, r0, sk, t * 16, lane);
          short_scores<HD>(dp, sdo, r0, sv, t * 16, lane);
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const int j = t * 16 + c * 8 + (lane & 3) * 2 + u;
              dp[c][u] = j <= j0 ? fast_exp2(fmaf(s[c][u], sl2, nl0)) * fmaf(dp[c][u], scale, nd0) : 0.f;
              dp[c][2 + u] = j <= j1 ? fast_exp2(fmaf(s[c][2 + u], sl2, nl1)) * fmaf(dp[c][2 + u], scale, nd1) : 0.f;
            }
          uint32_t w[4];
          short_operand(w, dp);
          short_weigh<HD>(dq, w, sk, t * 16, lane);
        }
        __syncwarp();
        // this warp's rows of dO have other readers, and Q's too: both are done with behind the barrier
        __syncthreads();
        short_store<HD>(dq, 1.f, 1.f, smem, sq, r0, n, p.dq + e.x * p.dqs + h * HD, p.dqs, lane);
      } else {
        __syncthreads();
      }
      __syncthreads();                                                 // Q and dO may be written over
    }
    if (r0 < n) {
      short_store<HD>(dk, 1.f, 1.f, smem, sk, r0, n, p.dk + e.x * p.dks + hk * HD, p.dks, lane);
      short_store<HD>(dv, 1.f, 1.f, smem, sv, r0, n, p.dv + e.x * p.dvs + hk * HD, p.dvs, lane);
    }
    __syncthreads();
  }
}

// As many blocks as the device holds at once, each with tasks in turn
template <typename P>
static int short_launch(void (*kernel)(const P), int smem, std::atomic<unsigned long long>& allowed, int per_sm, long long most, const P& p, cudaStream_t st) {
  if (allow_smem(allowed, (const void*)kernel, smem) != cudaSuccess) return OA_ERR_LAUNCH;
  const long long room = (long long)per_sm * sm_count();
  launch_pdl(kernel, dim3((unsigned)(most < 1 ? 1 : most < room ? most : room)), dim3(PS_THREADS), smem, st, p);
  return cudaGetLastError() == cudaSuccess ? OA_OK : OA_ERR_LAUNCH;
}

int packed_short_fwd(const PackedShortFwd& p, int head_dim, cudaStream_t st) {
  static std::atomic<unsigned long long> a64, a128;
  const long long most = (long long)p.plan.batch * p.q_heads;
  return head_dim == 64 ? short_launch(packed_short_fwd_kernel<64>, 3 * ShortTile<64>::BYTES, a64, 4, most, p, st)
                        : short_launch(packed_short_fwd_kernel<128>, 3 * ShortTile<128>::BYTES, a128, 4, most, p, st);
}

int packed_short_bwd(const PackedShortBwd& p, int head_dim, cudaStream_t st) {
  static std::atomic<unsigned long long> a64, a128;
  const long long most = (long long)p.plan.batch * p.kv_heads;
  return head_dim == 64 ? short_launch(packed_short_bwd_kernel<64>, 4 * ShortTile<64>::BYTES + 512, a64, 4, most, p, st)
                        : short_launch(packed_short_bwd_kernel<128>, 4 * ShortTile<128>::BYTES + 512, a128, 2, most, p, st);
}

}  // namespace oa
