// Parts of the attention kernels on tcgen05 (flash_attn.cu, packed_attn.cu): tiles of 128 x 128, operand descriptors, exponentials, rows to memory.
#pragma once
#include "common.cuh"

namespace oa {

constexpr int FA_BM = 128;   // queries per tile
constexpr int FA_BN = 128;   // keys per tile
constexpr float LOG2E = 1.4426950408889634f;

// The descriptor of an operand that starts `bytes` further (the address is in units of 16 bytes in the low bits): an issuing warp makes
// its descriptors once and only adds to them between products.
__device__ __forceinline__ uint64_t desc_at(uint64_t desc, uint32_t bytes) { return desc + (bytes >> 4); }
__device__ __forceinline__ uint64_t desc_k(const void* smem) { return umma_smem_desc_sw128(smem_u32(smem), 16, 1024); }             // reduction contiguous
__device__ __forceinline__ uint64_t desc_mn(const void* smem) { return umma_smem_desc_sw128(smem_u32(smem), FA_BN * 128, 1024); }   // 128 rows of the reduction

// Two exponentials 2^x on the multiply-add pipe: x = n + f with n the nearest integer (added and taken off at 1.5 * 2^23), 2^f by the
// minimax polynomial of degree 5 on [-1/2, 1/2] (Remez exchange on the relative error: 7.5e-8, with coefficients rounded to fp32 1.55e-7,
// 2.1e-7 with the rounding of its steps; ex2.approx states 2^-22 = 2.4e-7), 2^n as an exponent field, which is zero at n = -127: below that, -inf included, the result is 0 as ex2.approx.ftz gives it.
// NaN stays NaN; x up to 127.
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ unsigned long long exp2_fma2(unsigned long long x) {
  uint32_t a, b;
  f2_to(x, a, b);
  x = f2_of(__float_as_uint(max_nan(__uint_as_float(a), -127.f)), __float_as_uint(max_nan(__uint_as_float(b), -127.f)));
  const unsigned long long t = f2_add(x, f2_splat(12582912.f));
  const unsigned long long f = f2_fma(f2_add(t, f2_splat(-12582912.f)), f2_splat(-1.f), x);
  unsigned long long r = f2_fma(f2_splat(0.00132764725f), f, f2_splat(0.00967554096f));
  r = f2_fma(r, f, f2_splat(0.0555071309f));
  r = f2_fma(r, f, f2_splat(0.240221202f));
  r = f2_fma(r, f, f2_splat(0.693146944f));
  r = f2_fma(r, f, f2_splat(1.00000012f));
  f2_to(t, a, b);
  return f2_mul(r, f2_of((a << 23) + 0x3f800000u, (b << 23) + 0x3f800000u));
}

// 32 fp32 columns of a warp's 32 rows (one row to a lane) as bf16, 64 bytes of eight rows to a store (the rows lie apart by a whole
// projection).  `at`: the row of this warp's first lane; rows from `rows` on are not written.
__device__ __forceinline__ void store_rows(__nv_bfloat16* at, long long stride, int rows, const uint32_t* a, float mul, int lane) {
  uint4 v[4];
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const float* f = reinterpret_cast<const float*>(a) + g * 8;
    v[g] = make_uint4(pack_bf16x2(f[0] * mul, f[1] * mul), pack_bf16x2(f[2] * mul, f[3] * mul), pack_bf16x2(f[4] * mul, f[5] * mul), pack_bf16x2(f[6] * mul, f[7] * mul));
  }
  exchange4(v, lane);
  const int r0 = lane & ~3;
  at += (long long)r0 * stride + (lane & 3) * 8;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (r0 + k < rows) *reinterpret_cast<uint4*>(at + k * stride) = v[k];
}

constexpr float FA_RESCALE_THRESHOLD = 8.f;                // log2 units

// Two probabilities exp2(s sl2 + nl), over the scores; two p (dp scale + nd), over the probabilities
template <bool FMA = false>
__device__ __forceinline__ void bwd_prob2(uint32_t& a, uint32_t& b, unsigned long long sl2, unsigned long long nl) {
  const unsigned long long x = f2_fma(f2_of(a, b), sl2, nl);
  f2_to(FMA ? exp2_fma2(x) : exp2_mufu2(x), a, b);
}
__device__ __forceinline__ void bwd_ds2(uint32_t& a, uint32_t& b, uint32_t d0, uint32_t d1, unsigned long long scale, unsigned long long nd) {
  f2_to(f2_mul(f2_of(a, b), f2_fma(f2_of(d0, d1), scale, nd)), a, b);
}
// 32 values of a lane as bf16 over 16 columns
__device__ __forceinline__ void bwd_store16(uint32_t taddr, const uint32_t* v) {
  uint32_t w[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) w[i] = pack_bf16x2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
  tmem_st16(taddr, w);
}

}  // namespace oa
