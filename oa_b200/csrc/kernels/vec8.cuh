// Eight elements in registers, loaded and stored as 16-byte words, worked on in fp32.
#pragma once
#include "common.cuh"

namespace oa {

template <typename T> struct Vec8;         // eight elements as 16-byte words
template <> struct Vec8<__nv_bfloat16> {
  uint4 w[1];
  __device__ __forceinline__ void get(float* f) const {
    const uint32_t u[4] = {w[0].x, w[0].y, w[0].z, w[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { const float2 a = unpack_bf16x2(u[i]); f[2 * i] = a.x; f[2 * i + 1] = a.y; }
  }
  __device__ __forceinline__ void set(const float* f) {
    w[0] = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  }
};
template <> struct Vec8<float> {
  uint4 w[2];
  __device__ __forceinline__ void get(float* f) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      f[4 * i] = __uint_as_float(w[i].x); f[4 * i + 1] = __uint_as_float(w[i].y); f[4 * i + 2] = __uint_as_float(w[i].z); f[4 * i + 3] = __uint_as_float(w[i].w);
    }
  }
  __device__ __forceinline__ void set(const float* f) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      w[i] = make_uint4(__float_as_uint(f[4 * i]), __float_as_uint(f[4 * i + 1]), __float_as_uint(f[4 * i + 2]), __float_as_uint(f[4 * i + 3]));
  }
};

}  // namespace oa
