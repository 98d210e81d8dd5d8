// Attention over the packed sequences of up to 64 rows (packed_short.cu), launched beside that over the longer ones (packed_attn.cu).
#pragma once
#include <cuda_bf16.h>

#include "packed.cuh"

namespace oa {

struct PackedShortFwd {
  PackedPlan plan;
  const __nv_bfloat16 *q, *k, *v;
  __nv_bfloat16* o;
  float* lse;                              // [q_heads, tokens] or null
  long long qs, ks, vs, os;                // elements between rows
  int q_heads, group;
  float scale;
};
struct PackedShortBwd {
  PackedPlan plan;
  const __nv_bfloat16 *q, *k, *v, *dout;
  const float* lse;                        // [q_heads, tokens]
  __nv_bfloat16 *dq, *dk, *dv;
  long long qs, ks, vs, dos, dqs, dks, dvs;
  int kv_heads, group;
  float scale;
};

int packed_short_fwd(const PackedShortFwd& p, int head_dim, cudaStream_t st);
int packed_short_bwd(const PackedShortBwd& p, int head_dim, cudaStream_t st);

}  // namespace oa
