// Parts of the fp32 attention kernels (attn_f32.cu says how they work): tiles of 32 streamed rows in shared memory, a row's dimensions dealt to threads.
#pragma once
#include "common.cuh"

namespace oa {

constexpr int AF_THREADS = 128;
constexpr int AF_TILE = 32;     // streamed rows per step

constexpr int AF_W = 32;        // head dimensions per thread
constexpr int AF_SEG = AF_W + 4;   // floats per such segment in shared memory (padded: rows and segments land in different banks)

// A streamed tile of rows [r0, r0 + 32) of a [rows, stride] matrix, columns [col0, col0 + hd), as [32][DS][AF_SEG]; rows >= limit and
// dimensions >= hd become 0.  `vec`: 16-byte pieces (hd, stride and the pointer allow it), asynchronously when ASYNC.
template <int DS, bool ASYNC>
__device__ __forceinline__ void af_load_tile(float* sm, const float* __restrict__ g, long long stride, long long row_base, int r0, int limit, int col0,
                                             int hd, bool vec) {
  constexpr int COLS = DS * AF_W;
  if (vec) {
#pragma unroll
    for (int idx = threadIdx.x; idx < AF_TILE * COLS / 4; idx += AF_THREADS) {
      const int r = idx / (COLS / 4), c = idx % (COLS / 4) * 4;
      const bool ok = r0 + r < limit && c < hd;
      const float* src = ok ? g + (row_base + r0 + r) * stride + col0 + c : g;
      float* dst = sm + (r * DS + c / AF_W) * AF_SEG + c % AF_W;
      if (ASYNC) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(ok ? 16 : 0) : "memory");
      else *reinterpret_cast<float4*>(dst) = ok ? *reinterpret_cast<const float4*>(src) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  } else {
#pragma unroll 4
    for (int idx = threadIdx.x; idx < AF_TILE * COLS; idx += AF_THREADS) {
      const int r = idx / COLS, c = idx % COLS;
      float x = 0.f;
      if (r0 + r < limit && c < hd) x = g[(row_base + r0 + r) * stride + col0 + c];
      sm[(r * DS + c / AF_W) * AF_SEG + c % AF_W] = x;
    }
  }
}
__device__ __forceinline__ void af_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void af_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// A thread's 32 dimensions of its own row, zeros beyond hd and for rows that are not there
__device__ __forceinline__ void af_own(float* dst, const float* __restrict__ row, int left, bool ok, bool vec) {
  if (!ok) left = 0;
  if (vec) {
#pragma unroll
    for (int t = 0; t < AF_W; t += 4) *reinterpret_cast<float4*>(dst + t) = t < left ? *reinterpret_cast<const float4*>(row + t) : make_float4(0.f, 0.f, 0.f, 0.f);
  } else {
#pragma unroll
    for (int t = 0; t < AF_W; ++t) dst[t] = t < left ? row[t] : 0.f;
  }
}

// sum over the DS threads that share a row's dot products (neighbouring lanes)
template <int DS>
__device__ __forceinline__ float af_reduce(float x) {
  if (DS >= 2) x += __shfl_xor_sync(0xffffffffu, x, 1);
  if (DS >= 4) x += __shfl_xor_sync(0xffffffffu, x, 2);
  return x;
}
// Sums of v[0..31] over the KS groups of a row: every group ends up with 32 / KS of them, v[0 .. 32 / KS), which are dimensions
// af_first<KS>(ks) and on.
template <int DS, int KS>
__device__ __forceinline__ void af_scatter_sum(float* v, int ks) {
  if constexpr (KS == 4) {
#pragma unroll
    for (int t = 0; t < 16; ++t) {
      const float mine = ks & 1 ? v[t + 16] : v[t], theirs = ks & 1 ? v[t] : v[t + 16];
      v[t] = mine + __shfl_xor_sync(0xffffffffu, theirs, DS);
    }
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      const float mine = ks & 2 ? v[t + 8] : v[t], theirs = ks & 2 ? v[t] : v[t + 8];
      v[t] = mine + __shfl_xor_sync(0xffffffffu, theirs, 2 * DS);
    }
  }
}
template <int KS>
__device__ __forceinline__ int af_first(int ks) { return KS == 4 ? (ks & 1) * 16 + (ks >> 1) * 8 : 0; }

__device__ __forceinline__ float af_dot(const float* a, const float* __restrict__ sm_row) {
  float d0 = 0.f, d1 = 0.f, d2 = 0.f, d3 = 0.f;
#pragma unroll
  for (int t = 0; t < AF_W; t += 4) {
    const float4 x = *reinterpret_cast<const float4*>(sm_row + t);
    d0 = fmaf(a[t], x.x, d0); d1 = fmaf(a[t + 1], x.y, d1); d2 = fmaf(a[t + 2], x.z, d2); d3 = fmaf(a[t + 3], x.w, d3);
  }
  return (d0 + d1) + (d2 + d3);
}

__device__ __forceinline__ void af_axpy(float* acc, float a, const float* __restrict__ sm_row) {
#pragma unroll
  for (int t = 0; t < AF_W; t += 4) {
    const float4 x = *reinterpret_cast<const float4*>(sm_row + t);
    acc[t] = fmaf(a, x.x, acc[t]); acc[t + 1] = fmaf(a, x.y, acc[t + 1]);
    acc[t + 2] = fmaf(a, x.z, acc[t + 2]); acc[t + 3] = fmaf(a, x.w, acc[t + 3]);
  }
}

template <int DS, int KS>
struct AfCfg {
  static constexpr int TPR = DS * KS, ROWS = AF_THREADS / TPR;
  static constexpr bool ASYNC = KS > 1;                        // two buffers, the next tile in flight
  static constexpr int BUFS = ASYNC ? 2 : 1, TILE = AF_TILE * DS * AF_SEG;
};

// The two streamed matrices of each pass, tile by tile: body(j0, x tile, y tile) for j0 in [lo, hi) in steps of 32.
template <int DS, int KS, typename Body>
__device__ __forceinline__ void af_stream(float* sx, float* sy, const float* __restrict__ x, long long xs, const float* __restrict__ y, long long ys,
                                          long long row0, int lo, int hi, int limit, int col0, int hd, bool vec, Body body) {
  using Cfg = AfCfg<DS, KS>;
  auto load = [&](int j0, int buf) {
    af_load_tile<DS, Cfg::ASYNC>(sx + buf * Cfg::TILE, x, xs, row0, j0, limit, col0, hd, vec);
    af_load_tile<DS, Cfg::ASYNC>(sy + buf * Cfg::TILE, y, ys, row0, j0, limit, col0, hd, vec);
    if (Cfg::ASYNC) af_commit();
  };
  if constexpr (Cfg::ASYNC) {
    load(lo, 0);
    for (int j0 = lo, buf = 0; j0 < hi; j0 += AF_TILE, buf ^= 1) {
      if (j0 + AF_TILE < hi) { load(j0 + AF_TILE, buf ^ 1); af_wait<1>(); } else { af_wait<0>(); }
      __syncthreads();
      body(j0, sx + buf * Cfg::TILE, sy + buf * Cfg::TILE);
      __syncthreads();                                         // the buffer may be filled again
    }
  } else {
    for (int j0 = lo; j0 < hi; j0 += AF_TILE) {
      __syncthreads();
      load(j0, 0);
      __syncthreads();
      body(j0, sx, sy);
    }
  }
}

}  // namespace oa
