// The plan of a batch of packed sequences, in int32 words: [tiles, pairs, first row, row behind the last, short sequences of 33 to 64 rows, of 17 to 32, of up to 16, -,
// starts.., tiles.., pairs.., short sequences..].  A tile (128 rows) or a pair of tiles of a sequence of more than 64 rows is (first row of its sequence, row behind it, index in the sequence,
// sequence), the largest index first; a short sequence is (first row, row behind it, 0, sequence), in the order
// of the three counts.
#pragma once
#include <cuda_runtime.h>

namespace oa {

constexpr int PACKED_TILE = 128;
constexpr int PACKED_SHORT = 64;           // rows of a short sequence, at most
constexpr int PACKED_HEADER = 8;
constexpr int PACKED_MAX_BATCH = 1 << 24, PACKED_MAX_TOKENS = 1 << 30;   // numbers of tiles, rows and words stay far below 2^31
__host__ __device__ inline int packed_tiles_at(int batch) { return (PACKED_HEADER + batch + 1 + 3) & ~3; }
__host__ __device__ inline int packed_max_tiles(int tokens, int batch) { return tokens / PACKED_TILE + batch; }
__host__ __device__ inline int packed_max_pairs(int tokens, int batch) { return tokens / (2 * PACKED_TILE) + batch; }

// Words of a plan
struct PackedPlan {
  const int* words;
  int batch, tokens;
  __device__ __forceinline__ int tiles() const { return words[0]; }
  __device__ __forceinline__ int pairs() const { return words[1]; }
  __device__ __forceinline__ int shorts() const { return words[4] + words[5] + words[6]; }
  __device__ __forceinline__ int4 tile(int i) const { return reinterpret_cast<const int4*>(words + packed_tiles_at(batch))[i]; }
  __device__ __forceinline__ int4 pair(int i) const {
    return reinterpret_cast<const int4*>(words + packed_tiles_at(batch))[packed_max_tiles(tokens, batch) + i];
  }
  __device__ __forceinline__ int4 brief(int i) const {
    return reinterpret_cast<const int4*>(words + packed_tiles_at(batch))[packed_max_tiles(tokens, batch) + packed_max_pairs(tokens, batch) + i];
  }
  // f(row) for this worker's share of the rows that belong to no sequence
  template <typename F>
  __device__ __forceinline__ void others(int worker, int workers, F f) const {
    const int first = words[2], end = words[3];
    for (int r = worker; r < first; r += workers) f(r);
    for (int r = end + worker; r < tokens; r += workers) f(r);
  }
};

}  // namespace oa
