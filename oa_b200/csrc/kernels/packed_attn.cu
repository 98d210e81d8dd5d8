// Causal attention over packed sequences with grouped heads for sm_100a, forward and backward, bf16 in / fp32 accumulate.  Sequences of up to 64 rows are worked on
// by packed_short.cu, whose launches stand beside these.
//
// Query head h reads key-value head h / group; o_i = sum_j p_ij v_j over the keys j <= i of i's own sequence, p_ij = exp(scale q_i k_j - lse_i).  Backward,
// with delta_i = dO_i O_i:  dV_j = sum p_ij dO_i,  dS_ij = scale p_ij (dO_i v_j - delta_i),  dQ_i = sum dS_ij k_j,  dK_j = sum dS_ij q_i, where those of a
// key-value head add up over its group's query heads.
//
// The tiles are those of flash_attn.cu: 128 queries x 128 keys on tcgen05 with scores, weights and accumulators in TMEM, operands through TMA, a running
// maximum that moves when a row outgrows it by 2^8.  What differs: tiles begin at a sequence's first row and come from the plan's list, the longest first,
// dealt to one CTA per SM in snake order; the two tiles of a forward CTA are two heads of one group where groups are even, so that both need the same
// blocks of keys and values, and neighbouring tiles of one head otherwise; dK and dV of a key-value head stay in TMEM over all query tiles of all
// heads of its group, so that there is one writer and one order.  A sequence's last block may reach into the next sequence, or into rows that nobody
// wrote: a warp of its own puts zeros in place of those rows (of values forward, of everything that is a product's second operand backward),
// because a weight of 0 times NaN is NaN.
//
// Forward is bound by the softmax warps: about 1700 cycles for a tile of 128 x 128, of which the exponentials need 900 (two warps to a scheduler, each a chain of
// loads from TMEM, maximum, exponentials, stores).  Backward is two kernels, dQ and then dK and dV, which work out scores and dP twice: seven products for
// five, but sums of one order, no atomics, and little in memory between them: two numbers to a row (delta, and delta put right), and where the heads of a group go over
// several CTAs their fp32 sums of dK and dV.  They too are bound by their softmax warps (issue slots 45 to 50 %
// busy, tensor pipe 40 % at head dim 64).  Measured: 8 x 2048 rows of 16 heads of 64 109 us (630 TFLOP/s of what the mask leaves) and 353 for the gradients
// (487); 4096 of 32 of 128 120 (1149) and 457 (751); 8192 of 32 over 8 of 128 415 (1326) and 1653 (831).  Where tiles are few the heads of a group go over several CTAs
// whose dK and dV are joined by a third kernel.
//
// Every wait is bounded and reports to a status word.
#include "attn_tile.cuh"
#include "packed_short.h"
#include "per_device.h"
#include "api.h"

namespace oa {

// A CTA's work items: (tile or pair of tiles, one of `per` heads or pairs of heads), all of the longest tiles first, in snake order over the
// CTAs (round r: CTA c takes item r G + c, or r G + G - 1 - c when r is odd).  Every warp walks them alike.  The plan's entries of the first rounds are
// fetched to shared memory at the start: a load from L2 for each item, sent for during the one before, cost 2 to 3 %.
constexpr int PACKED_ROUNDS = 96;
template <bool PAIRS>
struct PackedWalk {
  const PackedPlan& plan;
  const int4* kept;
  const int per, n;
  int round, item, index;                 // index: of the entry last handed out
  __device__ __forceinline__ PackedWalk(const PackedPlan& p, int heads, int4* room)
      : plan(p), kept(room), per(heads), n((PAIRS ? p.pairs() : p.tiles()) * heads), round(0), item(blockIdx.x), index(0) {
    for (int r = threadIdx.x; r < PACKED_ROUNDS; r += blockDim.x) {
      const int i = at(r);
      if (i < n) room[r] = entry_of(i);
    }
    __syncthreads();
  }
  __device__ __forceinline__ int at(int r) const {
    const int g = gridDim.x;
    return r * g + ((r & 1) ? g - 1 - (int)blockIdx.x : (int)blockIdx.x);
  }
  __device__ __forceinline__ int4 entry_of(int i) const { return PAIRS ? plan.pair(i / per) : plan.tile(i / per); }
  // false: no item left; otherwise the plan's entry and which of the heads
  __device__ __forceinline__ bool next(int4& entry, int& which) {
    if (item >= n) return false;
    entry = round < PACKED_ROUNDS ? kept[round] : entry_of(item);
    index = item / per;
    which = item - index * per;
    item = at(++round);
    return true;
  }
};

__device__ __forceinline__ float lo_of(unsigned long long v) {
  uint32_t a, b;
  f2_to(v, a, b);
  return __uint_as_float(a);
}
__device__ __forceinline__ float f2_sum(unsigned long long v) {
  uint32_t a, b;
  f2_to(v, a, b);
  return __uint_as_float(a) + __uint_as_float(b);
}

// Zeros in place of rows `from` .. 127 of a tile of 128 rows of HD values that a TMA load has left in shared memory (a row is 128 bytes of each
// slab of 64 columns, however its pieces are swizzled)
template <int HD>
__device__ __forceinline__ void clear_rows(uint8_t* tile, int from, int lane) {
#pragma unroll
  for (int x = 0; x < HD / 64; ++x)
    for (int i = from * 8 + lane; i < FA_BM * 8; i += 32) reinterpret_cast<uint4*>(tile + x * (FA_BM * 128))[i] = make_uint4(0, 0, 0, 0);
}

// A wait that spans other warps' work on whole items (their blocks may be so many that it outlasts the limit of a wait for one): the limit runs anew
// as long as `pulse`, in shared memory, moves with the blocks that the loading warp sends for.  Its own waits are for one block each, so this one ends too.
__device__ __forceinline__ bool idle_wait(uint64_t* bar, uint32_t parity, const volatile uint32_t* pulse) {
  uint32_t seen = __shfl_sync(0xffffffffu, *pulse, 0);
  while (!warp_wait(bar, parity)) {
    const uint32_t now = __shfl_sync(0xffffffffu, *pulse, 0);
    if (now == seen) return false;
    seen = now;
  }
  return true;
}

// Rows that belong to no sequence become zeros: `cols` bf16, a multiple of 8, by `threads` threads of every CTA
__device__ __forceinline__ void clear_others(const PackedPlan& plan, __nv_bfloat16* base, long long stride, int cols, int tid, int threads) {
  plan.others(blockIdx.x, gridDim.x, [&](int r) {
    for (int c = tid * 8; c < cols; c += threads * 8) *reinterpret_cast<uint4*>(base + r * stride + c) = make_uint4(0, 0, 0, 0);
  });
}

// Eight warps of 128 x 128 scores want more than the 168 registers that each of 384 threads can have; the issuing and loading warps do with 104, which leaves
// 200.  Head dim 64: forward 113 -> 108.5 us, backward 372 -> 363 us for 8 x 2048 rows of 16 heads.  Head dim 128: 119 -> 120 and 450 -> 447 us
// for 4096 of 32, its MMA warps spill; left alone.
template <int HD>
__device__ __forceinline__ void more_registers() {
  if constexpr (HD == 64) asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
}
template <int HD>
__device__ __forceinline__ void fewer_registers() {
  if constexpr (HD == 64) asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
}

struct PackedFwdParams {
  PackedPlan plan;
  int q_heads, group;
  float scale;
  __nv_bfloat16* o;
  float* lse;                         // [q_heads, tokens] or null
  int* status;
};

// How many of eight pairs of exponentials go to the multiply-add pipe.  8 x 2048 rows of 16 heads of 64 with 0 / 1 / 2 / 3: 118 / 109 / 111 / 117 us; 4096 of
// 32 of 128 with 0 / 1 / 2: 119 / 121.5 / 125.
template <int HD> constexpr int PF_FMA_PAIRS = HD == 64 ? 1 : 0;

template <int HD_>
struct PackedFwdCfg {
  static constexpr int HD = HD_;
  static constexpr bool ALIAS = HD == 128;                 // P over S: the columns of O are wanted
  static constexpr int NS = ALIAS ? 2 : 3;
  static constexpr int Q_BYTES = FA_BM * HD * 2;
  static constexpr int KV_BYTES = FA_BN * HD * 2;
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_K = OFF_Q + 2 * Q_BYTES;
  static constexpr int OFF_V = OFF_K + NS * KV_BYTES;
  static constexpr int OFF_BAR = OFF_V + NS * KV_BYTES;
  static constexpr int OFF_ITEMS = OFF_BAR + 256;
  static constexpr int SMEM_BYTES = OFF_ITEMS + PACKED_ROUNDS * 16;
  static constexpr int TMEM_COLS = 512;
  static constexpr int TM_S = 0, TM_P = ALIAS ? 0 : 256, P_STEP = ALIAS ? FA_BN : 64, TM_O = ALIAS ? 256 : 384;   // S: + 128 * tile, O: + HD * tile
  static constexpr int MMA_WARPS = ALIAS ? 1 : 2, TMA_WARP = 8 + MMA_WARPS, CLEAR_WARP = TMA_WARP + 1;   // after 8 softmax warps
  static constexpr int THREADS = (CLEAR_WARP + 1) * 32;
};

// What an item of the forward kernel is: up to two tiles of queries and their blocks of keys
template <bool HEADS>
struct PackedFwdItem {
  int lo, hi, kv_head;
  int row[2], head[2], n[2];          // first query in the sequence, head, blocks of keys (0: no such tile)
  __device__ __forceinline__ PackedFwdItem(const PackedFwdParams& p, const int4& e, int which) : lo(e.x), hi(e.y) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int tile = HEADS ? e.z : 2 * e.z + t;
      head[t] = HEADS ? 2 * which + t : which;
      row[t] = tile * FA_BM;
      n[t] = row[t] < hi - lo ? tile + 1 : 0;
    }
    kv_head = head[0] / p.group;
  }
};

// HEADS: a CTA's two tiles are two heads of a group, otherwise neighbouring tiles of one head
template <int HD, bool HEADS>
__global__ void __launch_bounds__(PackedFwdCfg<HD>::THREADS, 1)
packed_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                  const PackedFwdParams p) {
  using Cfg = PackedFwdCfg<HD>;
  constexpr int NS = Cfg::NS;
  constexpr bool ALIAS = Cfg::ALIAS;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::OFF_BAR);
  uint64_t* q_full = bars + 0;
  uint64_t* q_empty = bars + 1;            // the MMA warps are done with the Q tiles of the item
  uint64_t* k_full = bars + 2;             // [NS]
  uint64_t* k_empty = k_full + NS;         // [NS]  one arrival per MMA warp
  uint64_t* v_full = k_empty + NS;         // [NS]
  uint64_t* v_empty = v_full + NS;         // [NS]  one arrival per MMA warp
  uint64_t* s_full = v_empty + NS;         // [2]   S_t holds Q_t K_j^T
  uint64_t* s_empty = s_full + 2;          // [2]   ... and is in registers (4 warps)
  uint64_t* p_full = s_full + 4;           // [2][2]  P_t written, by half of the keys (the first: O_t rescaled if needed) (4 warps)
  uint64_t* o_done = s_full + 8;           // [2]   O_t += P_t V_j finished: P_t may be overwritten, O_t may be rescaled
  uint64_t* v_part = s_full + 10;          // [NS]  the values of a sequence's last block are there, and some rows of others
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(v_part + NS);
  volatile uint32_t* pulse = tmem_slot + 1;   // blocks sent for

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if ((smem_u32(smem) & 1023u) != 0) {
    if (threadIdx.x == 0) report_error(p.status, OA_KERR_BAD_ARG);
    return;
  }
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmQ); tma_prefetch_desc(&tmK); tma_prefetch_desc(&tmV);
    mbar_init(q_full, 1);
    mbar_init(q_empty, Cfg::MMA_WARPS);
    for (int s = 0; s < NS; ++s) { mbar_init(&k_full[s], 1); mbar_init(&v_full[s], 1); mbar_init(&k_empty[s], Cfg::MMA_WARPS); mbar_init(&v_empty[s], Cfg::MMA_WARPS); }
    for (int t = 0; t < 2; ++t) { mbar_init(&s_full[t], 1); mbar_init(&s_empty[t], 4); mbar_init(&p_full[2 * t], 4); mbar_init(&p_full[2 * t + 1], 4); mbar_init(&o_done[t], 1); }
    for (int s = 0; s < NS; ++s) mbar_init(&v_part[s], 1);
    *pulse = 0;
    mbar_fence_init();
  }
  if (warp == 8) { tmem_alloc<Cfg::TMEM_COLS>(tmem_slot); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();                            // the prologue above ran under the previous kernel's tail; global memory from here on

  PackedWalk<!HEADS> walk(p.plan, HEADS ? p.q_heads >> 1 : p.q_heads, reinterpret_cast<int4*>(smem + Cfg::OFF_ITEMS));
  int4 entry;
  int which;

  if (warp >= 8) {
    fewer_registers<HD>();
    if (warp == Cfg::TMA_WARP) {
      // ------------- producer
      uint32_t blk = 0, itc = 0;   // K / V blocks and items loaded so far
      bool ok = true;
      while (ok && walk.next(entry, which)) {
        const PackedFwdItem<HEADS> it(p, entry, which);
        const int n_it = max(it.n[0], it.n[1]);
        if (!warp_wait(q_empty, (itc & 1) ^ 1)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_EMPTY); break; }
        if (elect_one()) {
          const int tiles = it.n[1] > 0 ? 2 : 1;
          mbar_expect_tx(q_full, tiles * Cfg::Q_BYTES);
          for (int t = 0; t < tiles; ++t)
#pragma unroll
            for (int x = 0; x < HD / 64; ++x)
              tma_load_2d(smem + Cfg::OFF_Q + t * Cfg::Q_BYTES + x * (FA_BM * 128), &tmQ, q_full, it.head[t] * HD + x * 64, it.lo + it.row[t]);
        }
        for (int j = 0; j < n_it; ++j, ++blk) {
          const int st = blk % NS, row = it.lo + j * FA_BN;
          const uint32_t ph = (blk / NS) & 1;
          if (!warp_wait(&k_empty[st], ph ^ 1)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_EMPTY); ok = false; break; }
          if (elect_one()) {
            mbar_expect_tx(&k_full[st], Cfg::KV_BYTES);
#pragma unroll
            for (int x = 0; x < HD / 64; ++x)
              tma_load_2d(smem + Cfg::OFF_K + st * Cfg::KV_BYTES + x * (FA_BN * 128), &tmK, &k_full[st], it.kv_head * HD + x * 64, row);
          }
          if (!warp_wait(&v_empty[st], ph ^ 1)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_EMPTY); ok = false; break; }
          if (elect_one()) {
            uint64_t* bar = row + FA_BN > it.hi ? &v_part[st] : &v_full[st];
            *pulse = blk + 1;
            mbar_expect_tx(bar, Cfg::KV_BYTES);
#pragma unroll
            for (int x = 0; x < HD / 64; ++x)
              tma_load_2d(smem + Cfg::OFF_V + st * Cfg::KV_BYTES + x * (FA_BN * 128), &tmV, bar, it.kv_head * HD + x * 64, row);
          }
          __syncwarp();
        }
        ++itc;
      }
    } else if (warp == Cfg::CLEAR_WARP) {
      // ------------- zeros in place of rows behind a sequence, which only an item's last block can have
      uint32_t blk = 0, phases = 0;
      while (walk.next(entry, which)) {
        const PackedFwdItem<HEADS> it(p, entry, which);
        const int n_it = max(it.n[0], it.n[1]), row = it.lo + (n_it - 1) * FA_BN;
        blk += n_it;
        if (row + FA_BN <= it.hi) continue;
        const int st = (blk - 1) % NS;
        // from the last such item to this one's last block
        if (!idle_wait(&v_part[st], (phases >> st) & 1, pulse)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_FULL); break; }
        phases ^= 1u << st;
        clear_rows<HD>(smem + Cfg::OFF_V + st * Cfg::KV_BYTES, it.hi - row, lane);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_full[st]);
      }
    } else if (ALIAS && warp == 8) {
      // ------------- MMA issuer of both tiles, in turn (warp-uniform waits, one lane issues)
      constexpr uint32_t idesc_qk = umma_idesc_bf16(FA_BM, FA_BN, 0, 0);
      constexpr uint32_t idesc_pv = umma_idesc_bf16(FA_BM, HD, 0, 1);
      uint32_t base = 0, itc = 0, pc[2] = {0, 0};   // K / V blocks before this item, items, P V products of each tile so far
      bool ok = true;
      const uint64_t q_desc = desc_k(smem + Cfg::OFF_Q), k_desc = desc_k(smem + Cfg::OFF_K), v_desc = desc_mn(smem + Cfg::OFF_V);
      // S_t = Q_t K^T of ring block `blk`; `first` / `last`: of the tiles that read it, `end`: nothing reads Q after it
      auto issue_qk = [&](int t, uint32_t blk, bool first, bool last, bool end) -> bool {
        const int st = blk % NS;
        if (first && !warp_wait(&k_full[st], (blk / NS) & 1)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_FULL); return false; }
        tc_fence_after();
        if (elect_one()) {
          const uint64_t qd = desc_at(q_desc, t * Cfg::Q_BYTES), kd = desc_at(k_desc, st * Cfg::KV_BYTES);
#pragma unroll
          for (int ks = 0; ks < HD / 16; ++ks) {
            const uint32_t off = (ks >> 2) * (FA_BM * 128) + (ks & 3) * 32;
            umma_f16(tmem_base + Cfg::TM_S + t * FA_BN, desc_at(qd, off), desc_at(kd, off), idesc_qk, ks > 0 ? 1u : 0u);
          }
          umma_commit(&s_full[t]);
          if (last) umma_commit(&k_empty[st]);
          if (end) umma_commit(q_empty);
        }
        __syncwarp();
        return true;
      };
      while (ok && walk.next(entry, which)) {
        const PackedFwdItem<HEADS> item(p, entry, which);
        const int n[2] = {item.n[0], item.n[1]}, n_it = max(n[0], n[1]);
        if (!warp_wait(q_full, itc & 1)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_FULL); break; }
        // a block's tiles: both, or the one whose row of blocks is longer (tile 1, unless it is absent)
        auto qk = [&](int t, int j) -> bool {
          const bool last = j >= n[1 - t] || t == 1;
          return issue_qk(t, base + j, t == 0 || j >= n[0], last, last && j + 1 == n_it);
        };
        if (n[0] > 0) ok = qk(0, 0);
        if (ok && n[1] > 0) ok = qk(1, 0);
        for (int j = 0; j < n_it && ok; ++j) {
          const int st = (base + j) % NS;
          if (!warp_wait(&v_full[st], ((base + j) / NS) & 1)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_FULL); ok = false; break; }
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (j >= n[t]) continue;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              if (!warp_wait(&p_full[2 * t + half], pc[t] & 1)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_SOFTMAX); ok = false; break; }
              tc_fence_after();
              if (elect_one()) {
                const uint64_t vd = desc_at(v_desc, st * Cfg::KV_BYTES);
                const uint32_t p_tm = tmem_base + Cfg::TM_P + t * Cfg::P_STEP, o_tm = tmem_base + Cfg::TM_O + t * HD;
#pragma unroll
                for (int ks = half * 4; ks < half * 4 + 4; ++ks)
                  umma_f16_ts(o_tm, p_tm + ks * 8, desc_at(vd, ks * 2048), idesc_pv, (j > 0 || ks > 0) ? 1u : 0u);
                if (half == 1) {
                  if (t == 1 || j >= n[1]) umma_commit(&v_empty[st]);
                  if (j + 1 == n[t]) umma_commit(&o_done[t]);
                }
              }
              __syncwarp();
            }
            if (!ok) break;
            ++pc[t];
            if (j + 1 < n[t]) { ok = qk(t, j + 1); if (!ok) break; }   // overwrites P_j: ordered after P_j V_j by the pipe
          }
        }
        base += n_it;
        ++itc;
      }
    } else if (!ALIAS && warp < 8 + Cfg::MMA_WARPS) {
      // ------------- MMA issuer of tile t (warp-uniform waits, one lane issues)
      const int t = warp - 8;
      constexpr uint32_t idesc_qk = umma_idesc_bf16(FA_BM, FA_BN, 0, 0);
      constexpr uint32_t idesc_pv = umma_idesc_bf16(FA_BM, HD, 0, 1);
      const uint64_t qd = desc_k(smem + Cfg::OFF_Q + t * Cfg::Q_BYTES), k_desc = desc_k(smem + Cfg::OFF_K), v_desc = desc_mn(smem + Cfg::OFF_V);
      const uint32_t s_tm = tmem_base + Cfg::TM_S + t * FA_BN, p_tm = tmem_base + Cfg::TM_P + t * Cfg::P_STEP, o_tm = tmem_base + Cfg::TM_O + t * HD;
      uint32_t base = 0, itc = 0, sc = 0, pc = 0;   // K / V blocks before this item, items, S products and P V products of this tile so far
      bool ok = true;
      auto issue_qk = [&](uint32_t blk, bool last) -> bool {       // S_t = Q_t K^T of ring block `blk`
        const int st = blk % NS;
        if (!warp_wait(&k_full[st], (blk / NS) & 1)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_FULL); return false; }
        if (sc > 0 && !warp_wait(&s_empty[t], (sc - 1) & 1)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_TMEM_EMPTY); return false; }
        tc_fence_after();
        if (elect_one()) {
          const uint64_t kd = desc_at(k_desc, st * Cfg::KV_BYTES);
#pragma unroll
          for (int ks = 0; ks < HD / 16; ++ks) {
            const uint32_t off = (ks >> 2) * (FA_BM * 128) + (ks & 3) * 32;
            umma_f16(s_tm, desc_at(qd, off), desc_at(kd, off), idesc_qk, ks > 0 ? 1u : 0u);
          }
          umma_commit(&k_empty[st]);
          umma_commit(&s_full[t]);
          if (last) umma_commit(q_empty);
        }
        __syncwarp();
        ++sc;
        return true;
      };
      while (ok && walk.next(entry, which)) {
        const PackedFwdItem<HEADS> item(p, entry, which);
        const int n_it = max(item.n[0], item.n[1]), n = t == 0 ? item.n[0] : item.n[1];
        if (!warp_wait(q_full, itc & 1)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_FULL); break; }
        if (n > 0) ok = issue_qk(base, n == 1);
        for (int j = 0; j < n && ok; ++j) {
          if (j + 1 < n) { ok = issue_qk(base + j + 1, j + 2 == n); if (!ok) break; }
          const int st = (base + j) % NS;
          if (!warp_wait(&v_full[st], ((base + j) / NS) & 1)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_FULL); ok = false; break; }
          if (!warp_wait(&p_full[2 * t], pc & 1)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_SOFTMAX); ok = false; break; }
          tc_fence_after();
          if (elect_one()) {
            const uint64_t vd = desc_at(v_desc, st * Cfg::KV_BYTES);
#pragma unroll
            for (int ks = 0; ks < FA_BN / 16; ++ks)
              umma_f16_ts(o_tm, p_tm + ks * 8, desc_at(vd, ks * 2048), idesc_pv, (j > 0 || ks > 0) ? 1u : 0u);
            umma_commit(&v_empty[st]);
            umma_commit(&o_done[t]);
          }
          __syncwarp();
          ++pc;
        }
        // blocks of this item that this tile does not use (the last one of the pair's shorter tile, or all of an absent tile):
        // the rings still expect one arrival per MMA warp, given once the block has landed
        for (int j = n; j < n_it && ok; ++j) {
          const int st = (base + j) % NS;
          const uint32_t ph = ((base + j) / NS) & 1;
          if (!warp_wait(&k_full[st], ph)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_FULL); ok = false; break; }
          if (lane == 0) mbar_arrive(&k_empty[st]);
          if (!warp_wait(&v_full[st], ph)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_FULL); ok = false; break; }
          if (lane == 0) mbar_arrive(&v_empty[st]);
          __syncwarp();
        }
        if (n == 0 && ok && lane == 0) mbar_arrive(q_empty);
        __syncwarp();
        base += n_it;
        ++itc;
      }
    }
  } else {
    more_registers<HD>();
    // ------------- softmax + output of tile t: one thread per query row
    const int t = warp >> 2;
    const int quad = warp & 3;
    const int r = quad * 32 + lane;
    const uint32_t t_lane = (uint32_t)(quad * 32) << 16;
    const uint32_t s_addr = tmem_base + t_lane + Cfg::TM_S + t * FA_BN;
    const uint32_t p_addr = tmem_base + t_lane + Cfg::TM_P + t * Cfg::P_STEP;
    const uint32_t o_addr = tmem_base + t_lane + Cfg::TM_O + t * HD;
    const float sl2 = p.scale * LOG2E;
    const int o_stride = p.q_heads * HD;
    uint32_t sc = 0, pc = 0;     // score tiles consumed and P V completions awaited so far
    bool ok = true, idle = false;
    clear_others(p.plan, p.o, o_stride, o_stride, threadIdx.x, 256);
    if (p.lse)
      p.plan.others(blockIdx.x, gridDim.x, [&](int row) {
        for (int h = threadIdx.x; h < p.q_heads; h += 256) p.lse[(long long)h * p.plan.tokens + row] = -INFINITY;
      });
    while (ok && walk.next(entry, which)) {
      const int tile = HEADS ? entry.z : 2 * entry.z + t, head = HEADS ? 2 * which + t : which, hi = entry.y;
      const int q0 = entry.x + tile * FA_BM + quad * 32;    // this warp's first row
      if (entry.x + tile * FA_BM >= hi) { idle = true; continue; }
      if (!HEADS && idle) {          // the other tile alone has been worked on since
        idle = false;
        ok = idle_wait(&s_full[t], sc & 1, pulse);
        if (!ok) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_TMEM_FULL); break; }
      }
      const int n = tile + 1;
      float m_run = -INFINITY, l_run = 0.f;
      for (int j = 0; j < n; ++j, ++sc) {
        ok = warp_wait(&s_full[t], sc & 1);
        if (!ok) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_TMEM_FULL); break; }
        tc_fence_after();
        uint32_t sv[FA_BN];
#pragma unroll
        for (int c = 0; c < FA_BN / 32; ++c) tmem_ld32(s_addr + c * 32, sv + c * 32);
        tmem_ld_wait();
        if (!ALIAS) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s_empty[t]);   // the next block's scores may overwrite S_t now
        }
        // only the last block is on the diagonal, and only it can reach behind the sequence: keys up to the query's own
        if (j + 1 == n) {
#pragma unroll
          for (int i = 0; i < FA_BN; ++i) sv[i] = i <= r ? sv[i] : 0xff800000u;  // -inf
        }
        float m0 = __uint_as_float(sv[0]), m1 = __uint_as_float(sv[1]);
#pragma unroll
        for (int i = 2; i < FA_BN - 2; i += 4) {
          m0 = fmax3(m0, __uint_as_float(sv[i]), __uint_as_float(sv[i + 1]));
          m1 = fmax3(m1, __uint_as_float(sv[i + 2]), __uint_as_float(sv[i + 3]));
        }
        const float mx = fmax3(m0, m1, fmaxf(__uint_as_float(sv[FA_BN - 2]), __uint_as_float(sv[FA_BN - 1]))) * sl2;
        const float m_new = fmaxf(m_run, mx);
        const bool grow = (m_new - m_run) > FA_RESCALE_THRESHOLD;           // first block: m_run = -inf -> true
        const float m_cand = grow ? m_new : m_run;
        const float m_use = (m_cand == -INFINITY) ? 0.f : m_cand;           // every score so far is -inf
        const float alpha = grow ? fast_exp2(m_run - m_use) : 1.f;           // m_run = -inf -> 0
        const float neg_m = -m_use;
        // P_t is free and O_t is complete once the previous P V has finished (head dim 128: s_full already says so, the scores were
        // issued behind it)
        if (!ALIAS && j > 0) {
          ok = warp_wait(&o_done[t], pc & 1);
          if (!ok) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_TMEM_FULL); break; }
          ++pc;
          tc_fence_after();
        }
        auto rescale = [&]() {                               // some row of this warp moved its maximum: rescale O
          if (j == 0 || !__any_sync(0xffffffffu, grow)) return;
#pragma unroll 1
          for (int q = 0; q < HD / 32; ++q) {
            uint32_t o[32];
            tmem_ld32(o_addr + q * 32, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st32(o_addr + q * 32, o);
          }
        };
        auto hand_over = [&](int half) {
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[2 * t + half]);
        };
        unsigned long long l01 = 0, l23 = 0;
        const unsigned long long sl22 = f2_splat(sl2), neg_m2 = f2_splat(neg_m);
#pragma unroll
        for (int c = 0; c < FA_BN / 32; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const uint32_t* sc4 = sv + c * 32 + i;
            const unsigned long long x01 = f2_fma(f2_of(sc4[0], sc4[1]), sl22, neg_m2), x23 = f2_fma(f2_of(sc4[2], sc4[3]), sl22, neg_m2);
            const unsigned long long e01 = exp2_mufu2(x01), e23 = (i >> 2) % 4 < PF_FMA_PAIRS<HD> ? exp2_fma2(x23) : exp2_mufu2(x23);
            l01 = f2_add(l01, e01);
            l23 = f2_add(l23, e23);
            pk[i >> 1] = f2_bf16(e01);
            pk[(i >> 1) + 1] = f2_bf16(e23);
          }
          tmem_st16(p_addr + c * 16, pk);
          if (ALIAS && (c & 1)) {                        // the products of half of the keys start under the other half's exponentials
            if (c == 1) rescale();
            hand_over(c >> 1);
          }
        }
        if (!ALIAS) {
          rescale();
          hand_over(0);
        }
        uint32_t lw[4];
        f2_to(l01, lw[0], lw[1]);
        f2_to(l23, lw[2], lw[3]);
        l_run = l_run * alpha + ((__uint_as_float(lw[0]) + __uint_as_float(lw[1])) + (__uint_as_float(lw[2]) + __uint_as_float(lw[3])));
        m_run = m_cand;
      }
      if (!ok) break;
      ok = warp_wait(&o_done[t], pc & 1);
      if (!ok) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_TMEM_FULL); break; }
      ++pc;
      tc_fence_after();
      const float inv = 1.f / l_run;
      __nv_bfloat16* op = p.o + (long long)q0 * o_stride + head * HD;
#pragma unroll
      for (int c = 0; c < HD / 32; ++c) {
        uint32_t o[32];
        tmem_ld32(o_addr + c * 32, o);
        tmem_ld_wait();
        // At head dim 64 a row's 16 bytes to a lane are the faster (flash_attn.cu)
        if (ALIAS) store_rows(op + c * 32, o_stride, hi - q0, o, inv, lane);
        else if (q0 + lane < hi) {
          __nv_bfloat16* od = op + (long long)lane * o_stride + c * 32;
#pragma unroll
          for (int g = 0; g < 4; ++g)
            *reinterpret_cast<uint4*>(od + g * 8) = make_uint4(
                pack_bf16x2(__uint_as_float(o[g * 8]) * inv, __uint_as_float(o[g * 8 + 1]) * inv),
                pack_bf16x2(__uint_as_float(o[g * 8 + 2]) * inv, __uint_as_float(o[g * 8 + 3]) * inv),
                pack_bf16x2(__uint_as_float(o[g * 8 + 4]) * inv, __uint_as_float(o[g * 8 + 5]) * inv),
                pack_bf16x2(__uint_as_float(o[g * 8 + 6]) * inv, __uint_as_float(o[g * 8 + 7]) * inv));
        }
      }
      if (p.lse && q0 + lane < hi) p.lse[(long long)head * p.plan.tokens + q0 + lane] = (m_run + log2f(l_run)) / LOG2E;
      tc_fence_before();   // the O reads above complete before this warp's next p_full arrival lets the next item's first P V overwrite O
    }
  }
  pdl_launch_dependents();
  tc_fence_before();
  __syncthreads();
  if (warp == 8) { tc_fence_after(); tmem_dealloc<Cfg::TMEM_COLS>(tmem_base); }
}

// ===================================================================================== backward
struct PackedBwdParams {
  PackedPlan plan;
  int q_heads, kv_heads, group;
  float scale;
  const float* lse;      // [q_heads, tokens]
  const float* delta;    // [q_heads, tokens]  sum_d dO * O
  float* ndelta;         // [q_heads, tokens]  -scale times the delta that the rows' sums of dS lead to
  __nv_bfloat16 *dq, *dk, *dv;
  long long dq_stride, dk_stride, dv_stride;
  int* status;
  int parts, heads;      // CTAs that share the query heads of a key-value head's tile, and how many each takes
  float4* partial;       // [parts][tiles, at most][kv_heads][dV, dK][HD / 4][128 rows], where there are several
  __device__ __forceinline__ long long partial_at(int part, int tile, int kv_head, int w, int hd) const {
    return ((((long long)part * packed_max_tiles(plan.tokens, plan.batch) + tile) * kv_heads + kv_head) * 2 + w) * (hd / 4 * FA_BM);
  }
};

// delta[h, i] = sum_d dO[i, h*hd + d] * O[i, h*hd + d] of the rows in tiles (short sequences work out their own): HD / 8 lanes to a head, each with 16 bytes of four
// rows under way.  Bound by the bytes: 12 us for 16384 rows of 16 heads of 64, 5.6 TB/s.
constexpr int DELTA_ROWS = 4, DELTA_THREADS = 256;
template <int HD>
__global__ void __launch_bounds__(DELTA_THREADS)
packed_delta_kernel(const __nv_bfloat16* __restrict__ o, const __nv_bfloat16* __restrict__ dout, float* __restrict__ delta, const PackedPlan plan, int heads,
                    long long o_stride, long long do_stride) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int LANES = HD / 8, GROUPS = FA_BM / DELTA_ROWS;
  const int per = heads * LANES, chunks = (GROUPS * per + DELTA_THREADS - 1) / DELTA_THREADS;
  const long long units = (long long)plan.tiles() * chunks;
  for (long long u = blockIdx.x; u < units; u += gridDim.x) {
    const int tile = (int)(u / chunks), i = (int)(u - (long long)tile * chunks) * DELTA_THREADS + threadIdx.x;
    const int4 e = plan.tile(tile);
    const int group = i / per, h = (i - group * per) / LANES, sub = threadIdx.x % LANES;
    const int row0 = e.x + e.z * FA_BM + group * DELTA_ROWS, rows = group < GROUPS ? min(DELTA_ROWS, e.y - row0) : 0;
    uint4 a[DELTA_ROWS], b[DELTA_ROWS];
#pragma unroll
    for (int r = 0; r < DELTA_ROWS; ++r) {
      a[r] = b[r] = make_uint4(0, 0, 0, 0);
      if (r < rows) {
        a[r] = *reinterpret_cast<const uint4*>(o + (row0 + r) * o_stride + h * HD + sub * 8);
        b[r] = *reinterpret_cast<const uint4*>(dout + (row0 + r) * do_stride + h * HD + sub * 8);
      }
    }
#pragma unroll
    for (int r = 0; r < DELTA_ROWS; ++r) {
      unsigned long long sum = f2_mul(f2_bf16x2(a[r].x), f2_bf16x2(b[r].x));
      sum = f2_fma(f2_bf16x2(a[r].y), f2_bf16x2(b[r].y), sum);
      sum = f2_fma(f2_bf16x2(a[r].z), f2_bf16x2(b[r].z), sum);
      sum = f2_fma(f2_bf16x2(a[r].w), f2_bf16x2(b[r].w), sum);
      float s = f2_sum(sum);
#pragma unroll
      for (int off = LANES >> 1; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
      if (sub == 0 && r < rows) delta[(long long)h * plan.tokens + row0 + r] = s;
    }
  }
}

constexpr int PB_THREADS = 384;   // 8 softmax warps, 2 MMA issuer warps, a TMA warp and one that clears rows and stages statistics
// Of eight pairs of exponentials, those on the multiply-add pipe.  The same rows' gradients at head dim 64 with 1 / 2 / 3 / 4: 366 / 362 / 360 / 376 us, at 128
// with 0 / 1 / 2: 459 / 456 / 462.
template <int HD> constexpr int PB_FMA_PAIRS = HD == 64 ? 3 : 1;

// The pipeline of both kernels is that of flash_attn.cu, whose comment says why: a tile passes through two phases in the eight softmax warps (two
// threads per TMEM lane, 64 columns each), scores -> probabilities, then dP -> dS, with barriers of their own; one warp issues the products that hang on
// the probabilities, another those that hang on dS; at head dim 128 the second waits its turn until the next tile's scores are in the pipe.
// The dK/dV kernel works on the TRANSPOSED tile, S^T = K Q^T with keys on the TMEM lanes; per-query statistics are then per column and
// are staged in shared memory beside the Q tile.
template <int HD>
struct PackedKvCfg {
  static constexpr int NST = (HD == 64) ? 3 : 2;       // Q and dO rings
  static constexpr int NS = (HD == 64) ? 2 : 1;        // score buffers in TMEM (P^T lies over S^T, dS^T over dP^T)
  static constexpr int T_BYTES = FA_BM * HD * 2;        // one [128 x HD] tile
  static constexpr int OFF_K = 0;
  static constexpr int OFF_V = OFF_K + T_BYTES;
  static constexpr int OFF_Q = OFF_V + T_BYTES;
  static constexpr int OFF_DO = OFF_Q + NST * T_BYTES;
  static constexpr int OFF_STAT = OFF_DO + NST * T_BYTES;   // float[NST][256]: -lse*log2e | -delta*scale of the query block
  static constexpr int OFF_BAR = OFF_STAT + NST * 256 * 4;
  static constexpr int OFF_ITEMS = OFF_BAR + 272;
  static constexpr int SMEM_BYTES = OFF_ITEMS + PACKED_ROUNDS * 16;
  static constexpr int TMEM_COLS = 512;
  static constexpr int TM_S = 0, TM_DP = NS * FA_BN, TM_DV = TM_DP + FA_BN, TM_DK = TM_DV + HD;
};

// An item of the dK/dV kernel: a tile of keys of one key-value head, and how many tiles of queries see it, of each of the group's heads.  The list has the
// tiles of queries with the longest rows first; tiles of keys are their mirror images.
template <bool SPLIT>
struct PackedKvItem {
  int lo, hi, key0, blocks, kv_head, part, head0, heads;      // the query heads: `heads` from head0 on
  __device__ __forceinline__ PackedKvItem(const PackedBwdParams& p, const int4& e, int which) : lo(e.x), hi(e.y) {
    kv_head = SPLIT ? which / p.parts : which;
    part = SPLIT ? which - kv_head * p.parts : 0;
    heads = SPLIT ? p.heads : p.group;
    head0 = which * heads;
    blocks = e.z + 1;
    key0 = ((e.y - e.x + FA_BN - 1) / FA_BN - blocks) * FA_BN;
  }
};

// SPLIT: the group's heads are several CTAs' (a template, because the code for it cost the others 2 %)
template <int HD, bool SPLIT>
__global__ void __launch_bounds__(PB_THREADS, 1)
packed_bwd_kv_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                     const __grid_constant__ CUtensorMap tmDO, const PackedBwdParams p) {
  using Cfg = PackedKvCfg<HD>;
  constexpr int NST = Cfg::NST, NS = Cfg::NS;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::OFF_BAR);
  uint64_t* kv_full = bars + 0;
  uint64_t* kv_empty = bars + 1;   // the item's last score and dP products have read K, V
  uint64_t* q_full = bars + 2;     // [3]  Q bytes and the statistics
  uint64_t* q_empty = bars + 5;    // [3]  dK has read Q (the scores and the statistics were read before)
  uint64_t* do_full = bars + 8;    // [3]
  uint64_t* do_empty = bars + 11;  // [3]  dP and dV have read dO
  uint64_t* s_full = bars + 14;    // [2]  S^T of this tile is in TMEM
  uint64_t* p_full = bars + 16;    // [2][2]  P^T, by score buffer and column half (4 warps each)
  uint64_t* dp_full = bars + 20;   // dP^T
  uint64_t* ds_full = bars + 21;   // [2]  dS^T, by column half (4 warps each)
  uint64_t* fin_full = bars + 23;  // dV, dK of the item are complete (both issuers arrive)
  uint64_t* turn = bars + 24;      // NS == 1: the next tile's scores are in the pipe, dK and dP may follow (not for an item's last tile)
  uint64_t* part_full = bars + 25; // [3]  Q and dO of a sequence's last block are there, and some rows of others
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 28);
  float* stat = reinterpret_cast<float*>(smem + Cfg::OFF_STAT);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if ((smem_u32(smem) & 1023u) != 0) {
    if (threadIdx.x == 0) report_error(p.status, OA_KERR_BAD_ARG);
    return;
  }
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmQ); tma_prefetch_desc(&tmK); tma_prefetch_desc(&tmV); tma_prefetch_desc(&tmDO);
    mbar_init(kv_full, 1);
    mbar_init(kv_empty, 2);
    for (int s = 0; s < NST; ++s) { mbar_init(&q_full[s], 2); mbar_init(&q_empty[s], 1); mbar_init(&do_full[s], 1); mbar_init(&do_empty[s], 2); }
    for (int s = 0; s < 2; ++s) { mbar_init(&s_full[s], 1); mbar_init(&ds_full[s], 4); }
    for (int s = 0; s < 4; ++s) mbar_init(&p_full[s], 4);
    mbar_init(dp_full, 1);
    mbar_init(fin_full, 2);
    mbar_init(turn, 1);
    for (int s = 0; s < NST; ++s) mbar_init(&part_full[s], 1);
    mbar_fence_init();
  }
  if (warp == 8) { tmem_alloc<Cfg::TMEM_COLS>(tmem_slot); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();                            // the prologue above ran under the previous kernel's tail; global memory from here on

  PackedWalk<false> walk(p.plan, SPLIT ? p.kv_heads * p.parts : p.kv_heads, reinterpret_cast<int4*>(smem + Cfg::OFF_ITEMS));
  int4 entry;
  int which;

  if (warp >= 8) {
    fewer_registers<HD>();
    if (warp == 10) {
      // ------------- TMA producer
      uint32_t itc = 0, qc = 0;       // items and Q / dO blocks loaded so far
      bool ok = true;
      while (ok && walk.next(entry, which)) {
        const PackedKvItem<SPLIT> it(p, entry, which);
        if (!warp_wait(kv_empty, (itc & 1) ^ 1)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_EMPTY); break; }
        if (elect_one()) {
          mbar_expect_tx(kv_full, 2 * Cfg::T_BYTES);
#pragma unroll
          for (int x = 0; x < HD / 64; ++x) {
            tma_load_2d(smem + Cfg::OFF_K + x * (FA_BN * 128), &tmK, kv_full, it.kv_head * HD + x * 64, it.lo + it.key0);
            tma_load_2d(smem + Cfg::OFF_V + x * (FA_BN * 128), &tmV, kv_full, it.kv_head * HD + x * 64, it.lo + it.key0);
          }
        }
        for (int g = 0; g < it.heads && ok; ++g) {
          const int h = it.head0 + g;
          for (int i = 0; i < it.blocks; ++i, ++qc) {
            const int st = qc % NST;
            const uint32_t ph = (qc / NST) & 1;
            const int qrow = it.lo + it.key0 + i * FA_BM;
            const bool part = qrow + FA_BM > it.hi;
            uint8_t *q_tile = smem + Cfg::OFF_Q + st * Cfg::T_BYTES, *do_tile = smem + Cfg::OFF_DO + st * Cfg::T_BYTES;
            if (!warp_wait(&q_empty[st], ph ^ 1)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_EMPTY); ok = false; break; }
            if (elect_one()) {
              uint64_t* bar = part ? &part_full[st] : &q_full[st];
              mbar_expect_tx(bar, part ? 2 * Cfg::T_BYTES : Cfg::T_BYTES);
#pragma unroll
              for (int x = 0; x < HD / 64; ++x) tma_load_2d(q_tile + x * (FA_BM * 128), &tmQ, bar, h * HD + x * 64, qrow);
            }
            if (!warp_wait(&do_empty[st], ph ^ 1)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_EMPTY); ok = false; break; }
            if (elect_one()) {
              uint64_t* bar = part ? &part_full[st] : &do_full[st];
              if (!part) mbar_expect_tx(bar, Cfg::T_BYTES);
#pragma unroll
              for (int x = 0; x < HD / 64; ++x) tma_load_2d(do_tile + x * (FA_BM * 128), &tmDO, bar, h * HD + x * 64, qrow);
            }
            __syncwarp();
          }
        }
        ++itc;
      }
    } else if (warp == 11) {
      // ------------- the per-query statistics of each block, and zeros in place of rows behind a sequence, which only a head's last block can have
      uint32_t qc = 0, phases = 0;
      bool ok = true;
      while (ok && walk.next(entry, which)) {
        const PackedKvItem<SPLIT> it(p, entry, which);
        for (int g = 0; g < it.heads && ok; ++g) {
          const long long stat_base = (long long)(it.head0 + g) * p.plan.tokens;
          for (int i = 0; i < it.blocks; ++i, ++qc) {
            const int st = qc % NST, qrow = it.lo + it.key0 + i * FA_BM;
            // lane l stages queries 4l .. 4l+3; sent for before their place is free
            float4 nl, nd;
            float* nlp = reinterpret_cast<float*>(&nl);
            float* ndp = reinterpret_cast<float*>(&nd);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              const int qi = qrow + lane * 4 + u;
              const bool okq = qi < it.hi;
              nlp[u] = okq ? -p.lse[stat_base + qi] * LOG2E : -INFINITY;
              ndp[u] = okq ? p.ndelta[stat_base + qi] : 0.f;
            }
            if (!warp_wait(&q_empty[st], ((qc / NST) & 1) ^ 1)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_EMPTY); ok = false; break; }
            float* dst = stat + st * 256;
            reinterpret_cast<float4*>(dst)[lane] = nl;
            reinterpret_cast<float4*>(dst + 128)[lane] = nd;
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_full[st]);
            if (qrow + FA_BM <= it.hi) continue;
            if (!warp_wait(&part_full[st], (phases >> st) & 1)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_FULL); ok = false; break; }
            phases ^= 1u << st;
            clear_rows<HD>(smem + Cfg::OFF_Q + st * Cfg::T_BYTES, it.hi - qrow, lane);
            clear_rows<HD>(smem + Cfg::OFF_DO + st * Cfg::T_BYTES, it.hi - qrow, lane);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) { mbar_arrive(&q_full[st]); mbar_arrive(&do_full[st]); }
          }
        }
      }
    } else if (warp == 8) {
      // ------------- MMA issuer A: S^T = K Q^T and dV += P^T dO.  S^T of a tile goes over the P^T that dV read NS tiles ago.
      constexpr uint32_t idesc_s = umma_idesc_bf16(FA_BN, FA_BM, 0, 0);
      constexpr uint32_t idesc_g = umma_idesc_bf16(FA_BN, HD, 0, 1);   // [keys x HD] += X^T[keys x q] (TMEM) * Y[q x HD]
      const uint64_t k_desc = desc_k(smem + Cfg::OFF_K), q_desc = desc_k(smem + Cfg::OFF_Q), do_desc = desc_mn(smem + Cfg::OFF_DO);
      uint32_t itc = 0, qc = 0;
      bool ok = true;
      auto issue_s = [&](uint32_t n, bool last) -> bool {
        const int st = n % NST;
        if (!warp_wait(&q_full[st], (n / NST) & 1)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_FULL); return false; }
        tc_fence_after();
        if (elect_one()) {
          const uint64_t qd = desc_at(q_desc, st * Cfg::T_BYTES);
          const uint32_t s_tm = tmem_base + Cfg::TM_S + (n % NS) * FA_BN;
#pragma unroll
          for (int ks = 0; ks < HD / 16; ++ks) {
            const uint32_t off = (ks >> 2) * (FA_BM * 128) + (ks & 3) * 32;
            umma_f16(s_tm, desc_at(k_desc, off), desc_at(qd, off), idesc_s, ks > 0 ? 1u : 0u);
          }
          umma_commit(&s_full[n % NS]);
          if (last) umma_commit(kv_empty);
        }
        __syncwarp();
        return true;
      };
      while (ok && walk.next(entry, which)) {
        const int n_it = (entry.z + 1) * (SPLIT ? p.heads : p.group);
        if (!warp_wait(kv_full, itc & 1)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_FULL); break; }
        ok = issue_s(qc, n_it == 1);
        // the previous item's dV / dK were read by the softmax warps before they produced this item's first P^T, dS^T
        for (int it = 0; it < n_it && ok; ++it, ++qc) {
          if (NS == 2 && it + 1 < n_it) { ok = issue_s(qc + 1, it + 2 == n_it); if (!ok) break; }
          const int st = qc % NST;
          if (!warp_wait(&do_full[st], (qc / NST) & 1)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_FULL); ok = false; break; }
          const uint64_t bd = desc_at(do_desc, st * Cfg::T_BYTES);
          const uint32_t a_addr = tmem_base + Cfg::TM_S + (qc % NS) * FA_BN;
          for (int half = 0; half < 2; ++half) {
            // an item's first product replaces the accumulator: wait until both halves' warps have read the previous item's
            if (it == 0 && half == 0) ok = warp_wait(&p_full[(qc % NS) * 2 + 1], (qc / NS) & 1);
            if (!ok || !warp_wait(&p_full[(qc % NS) * 2 + half], (qc / NS) & 1)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_SOFTMAX); ok = false; break; }
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
              for (int ks = 0; ks < 4; ++ks)    // reduction over the 64 queries of this half
                umma_f16_ts(tmem_base + Cfg::TM_DV, a_addr + half * 64 + ks * 8, desc_at(bd, (half * 4 + ks) * 2048),
                            idesc_g, (it > 0 || half > 0 || ks > 0) ? 1u : 0u);
              if (half == 1) {
                umma_commit(&do_empty[st]);
                if (it + 1 == n_it) umma_commit(fin_full);
              }
            }
            __syncwarp();
          }
          if (!ok) break;
          if (NS == 1 && it + 1 < n_it) {
            ok = issue_s(qc + 1, it + 2 == n_it);
            if (lane == 0) mbar_arrive(turn);
          }
        }
        ++itc;
      }
    } else if (warp == 9) {
      // ------------- MMA issuer B: dP^T = V dO^T and dK += dS^T Q.  dP^T of a tile goes over the dS^T that dK has read.
      constexpr uint32_t idesc_s = umma_idesc_bf16(FA_BN, FA_BM, 0, 0);
      constexpr uint32_t idesc_g = umma_idesc_bf16(FA_BN, HD, 0, 1);
      const uint64_t v_desc = desc_k(smem + Cfg::OFF_V), do_desc = desc_k(smem + Cfg::OFF_DO), q_desc = desc_mn(smem + Cfg::OFF_Q);
      const uint32_t dp_tm = tmem_base + Cfg::TM_DP;
      uint32_t itc = 0, qc = 0, turns = 0;
      bool ok = true;
      auto issue_dp = [&](uint32_t n, bool last) -> bool {
        const int st = n % NST;
        if (!warp_wait(&do_full[st], (n / NST) & 1)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_FULL); return false; }
        tc_fence_after();
        if (elect_one()) {
          const uint64_t dd = desc_at(do_desc, st * Cfg::T_BYTES);
#pragma unroll
          for (int ks = 0; ks < HD / 16; ++ks) {
            const uint32_t off = (ks >> 2) * (FA_BM * 128) + (ks & 3) * 32;
            umma_f16(dp_tm, desc_at(v_desc, off), desc_at(dd, off), idesc_s, ks > 0 ? 1u : 0u);
          }
          umma_commit(dp_full);
          umma_commit(&do_empty[st]);
          if (last) umma_commit(kv_empty);
        }
        __syncwarp();
        return true;
      };
      while (ok && walk.next(entry, which)) {
        const int n_it = (entry.z + 1) * (SPLIT ? p.heads : p.group);
        if (!warp_wait(kv_full, itc & 1)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_FULL); break; }
        ok = issue_dp(qc, n_it == 1);
        for (int it = 0; it < n_it && ok; ++it, ++qc) {
          const int st = qc % NST;
          if (!warp_wait(&q_full[st], (qc / NST) & 1)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_FULL); ok = false; break; }
          const uint64_t bd = desc_at(q_desc, st * Cfg::T_BYTES);
          if (NS == 1 && it + 1 < n_it) {
            if (!warp_wait(turn, turns & 1)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_EMPTY); ok = false; break; }
            ++turns;
          }
          for (int half = 0; half < 2; ++half) {
            if (it == 0 && half == 0) ok = warp_wait(&ds_full[1], qc & 1);   // as for dV
            if (!ok || !warp_wait(&ds_full[half], qc & 1)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_SOFTMAX); ok = false; break; }
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
              for (int ks = 0; ks < 4; ++ks)
                umma_f16_ts(tmem_base + Cfg::TM_DK, dp_tm + half * 64 + ks * 8, desc_at(bd, (half * 4 + ks) * 2048),
                            idesc_g, (it > 0 || half > 0 || ks > 0) ? 1u : 0u);
              if (half == 1) {
                umma_commit(&q_empty[st]);
                if (it + 1 == n_it) umma_commit(fin_full);
              }
            }
            __syncwarp();
          }
          if (!ok) break;
          if (it + 1 < n_it) ok = issue_dp(qc + 1, it + 2 == n_it);
        }
        ++itc;
      }
    }
  } else {
    more_registers<HD>();
    const int quad = warp & 3;
    const int half = warp >> 2;                  // this thread owns query columns [64*half, 64*half+64) of the tile
    const int r = quad * 32 + lane;              // key row inside the block = TMEM lane
    const uint32_t t_lane = tmem_base + ((uint32_t)(quad * 32) << 16);
    const unsigned long long sl22 = f2_splat(p.scale * LOG2E), scale2 = f2_splat(p.scale);
    uint32_t itc = 0, qc = 0;
    bool ok = true;
    clear_others(p.plan, p.dk, p.dk_stride, p.kv_heads * HD, threadIdx.x, 256);
    clear_others(p.plan, p.dv, p.dv_stride, p.kv_heads * HD, threadIdx.x, 256);
    while (ok && walk.next(entry, which)) {
      const PackedKvItem<SPLIT> item(p, entry, which);
      const int n_it = item.blocks * item.heads;
      for (int it = 0, i = 0; it < n_it; ++it, ++qc, i = i + 1 < item.blocks ? i + 1 : 0) {
        const int st = qc % NST;
        const float* st_cur = stat + st * 256 + half * 64;
        ok = warp_wait(&q_full[st], (qc / NST) & 1);   // statistics of this block are staged
        if (ok) ok = warp_wait(&s_full[qc % NS], (qc / NS) & 1);
        if (!ok) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_TMEM_FULL); break; }
        tc_fence_after();
        const uint32_t s_addr = t_lane + Cfg::TM_S + (qc % NS) * FA_BN + half * 64;
        const uint32_t dp_addr = t_lane + Cfg::TM_DP + half * 64;
        uint32_t s[64];
        tmem_ld32(s_addr, s);
        tmem_ld32(s_addr + 32, s + 32);
        tmem_ld_wait();
        const ulonglong2* nl4 = reinterpret_cast<const ulonglong2*>(st_cur);
        const ulonglong2* nd4 = reinterpret_cast<const ulonglong2*>(st_cur + 128);
        const bool diag = i == 0;                  // alive iff key <= query: column >= row
        const int first = r - half * 64;           // first alive column of this thread on the diagonal tile
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
          for (int u = 0; u < 32; u += 4) {
            const ulonglong2 nl = nl4[c * 8 + (u >> 2)];
            uint32_t* sc = s + c * 32 + u;
            bwd_prob2(sc[0], sc[1], sl22, nl.x);
            if ((u >> 2) % 4 < PB_FMA_PAIRS<HD>) bwd_prob2<true>(sc[2], sc[3], sl22, nl.y);
            else bwd_prob2(sc[2], sc[3], sl22, nl.y);
          }
          if (diag) {
#pragma unroll
            for (int u = 0; u < 32; ++u) s[c * 32 + u] = (c * 32 + u >= first) ? s[c * 32 + u] : 0u;
          }
          bwd_store16(s_addr + c * 16, s + c * 32);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[(qc % NS) * 2 + half]);
        ok = warp_wait(dp_full, qc & 1);
        if (!ok) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_TMEM_FULL); break; }
        tc_fence_after();
        uint32_t dp[64];
        tmem_ld32(dp_addr, dp);
        tmem_ld32(dp_addr + 32, dp + 32);
        tmem_ld_wait();
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
          for (int u = 0; u < 32; u += 4) {
            const ulonglong2 nd = nd4[c * 8 + (u >> 2)];
            uint32_t *sc = s + c * 32 + u, *dc = dp + c * 32 + u;
            bwd_ds2(sc[0], sc[1], dc[0], dc[1], scale2, nd.x);
            bwd_ds2(sc[2], sc[3], dc[2], dc[3], scale2, nd.y);
          }
          bwd_store16(dp_addr + c * 16, s + c * 32);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ds_full[half]);
      }
      if (!ok) break;
      ok = warp_wait(fin_full, itc & 1);
      if (!ok) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_TMEM_FULL); break; }
      ++itc;
      tc_fence_after();
      const int k0 = item.lo + item.key0 + quad * 32;   // accumulator rows are keys
#pragma unroll 1
      for (int w = 0; w < 2; ++w) {
        const long long stride = w == 0 ? p.dv_stride : p.dk_stride;
        __nv_bfloat16* base = (w == 0 ? p.dv : p.dk) + k0 * stride + item.kv_head * HD + half * (HD / 2);
        const uint32_t tcol = t_lane + (w == 0 ? Cfg::TM_DV : Cfg::TM_DK) + half * (HD / 2);
        uint32_t a[HD / 2];
#pragma unroll
        for (int c = 0; c < HD / 64; ++c) tmem_ld32(tcol + c * 32, a + c * 32);
        tmem_ld_wait();
        if constexpr (SPLIT) {                       // a row to a lane, side by side
          float4* to = p.partial + p.partial_at(item.part, walk.index, item.kv_head, w, HD) + half * (HD / 8) * FA_BM + r;
#pragma unroll
          for (int c = 0; c < HD / 8; ++c) to[c * FA_BM] = *reinterpret_cast<const float4*>(a + 4 * c);
        } else {
#pragma unroll
          for (int c = 0; c < HD / 64; ++c) store_rows(base + c * 32, stride, item.hi - k0, a + c * 32, 1.f, lane);
        }
      }
      tc_fence_before();   // dV / dK are read before this warp's next p_full / ds_full arrivals let the next item's products overwrite them
    }
  }
  pdl_launch_dependents();
  tc_fence_before();
  __syncthreads();
  if (warp == 8) { tc_fence_after(); tmem_dealloc<Cfg::TMEM_COLS>(tmem_base); }
}

template <int HD>
struct PackedQCfg {
  static constexpr int NK = (HD == 64) ? 4 : 3;        // K ring: a tile is held from its scores to dQ
  static constexpr int NV = (HD == 64) ? 3 : 2;        // V ring: held for dP only
  static constexpr int T_BYTES = FA_BM * HD * 2;
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_DO = OFF_Q + T_BYTES;
  static constexpr int OFF_K = OFF_DO + T_BYTES;
  static constexpr int OFF_V = OFF_K + NK * T_BYTES;
  static constexpr int OFF_BAR = OFF_V + NV * T_BYTES;
  static constexpr int OFF_ITEMS = OFF_BAR + 304;
  static constexpr int OFF_X = OFF_ITEMS + PACKED_ROUNDS * 16;   // float[2 halves][128 rows]
  static constexpr int SMEM_BYTES = OFF_X + 2 * FA_BM * 4;
  static constexpr int TMEM_COLS = 512;
  static constexpr int TM_S = 0, TM_DP = FA_BN, TM_DQ = 3 * FA_BN;   // two buffers of dP, dS over it: 32 columns of each half, its remainder in the next 32
};

// Items are (tile of queries, query head), the longest rows first; dQ of an item accumulates in TMEM over its key blocks.  P is needed in registers only, so
// the one score buffer is free once it has been read; dP has two, so that the next tile's is formed while this one's becomes dS and a product (with two buffers
// of scores and one of dP, dP -> dS -> dQ -> the next dP stood one behind the other).
// delta comes from the rounded output of weights that were rounded: what it is off by adds the same multiple of p_ij to a whole row of dS, and rounding dS to bf16
// adds as much again.  Together 1.6 to 2 times the rounding of the result itself.  So dS goes to the products as two bf16 numbers, its rounding and what that
// leaves; the rows' sums of dS, which are 0 for the right delta, go to the dK / dV kernel, which then has the right one; and where a row has one block of
// keys, the right one is there before dS is (shorter rows suffer most).
template <int HD>
__global__ void __launch_bounds__(PB_THREADS, 1)
packed_bwd_q_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                    const __grid_constant__ CUtensorMap tmDO, const PackedBwdParams p) {
  using Cfg = PackedQCfg<HD>;
  constexpr int NK = Cfg::NK, NV = Cfg::NV;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::OFF_BAR);
  uint64_t* q_full = bars + 0;
  uint64_t* q_empty = bars + 1;    // the item's last score and dP products have read Q, dO
  uint64_t* k_full = bars + 2;     // [4]
  uint64_t* k_empty = bars + 6;    // [4]  dQ has read K
  uint64_t* v_full = bars + 10;    // [3]
  uint64_t* v_empty = bars + 13;   // [3]
  uint64_t* s_full = bars + 16;
  uint64_t* s_empty = bars + 17;   // (8 warps)
  uint64_t* dp_full = bars + 18;   // [2]
  uint64_t* ds_full = bars + 20;   // [2][2]  by buffer and column half (4 warps each)
  uint64_t* fin_full = bars + 24;
  uint64_t* k_part = bars + 25;    // [4]  K, V of a sequence's last block are there, and some rows of others
  uint64_t* v_part = bars + 29;    // [3]
  uint64_t* x_full = bars + 32;    // [4]  sums of the two warps that share 32 rows are in xch
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 36);
  volatile uint32_t* pulse = tmem_slot + 1;   // blocks sent for

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if ((smem_u32(smem) & 1023u) != 0) {
    if (threadIdx.x == 0) report_error(p.status, OA_KERR_BAD_ARG);
    return;
  }
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmQ); tma_prefetch_desc(&tmK); tma_prefetch_desc(&tmV); tma_prefetch_desc(&tmDO);
    mbar_init(q_full, 1);
    mbar_init(q_empty, 2);
    for (int s = 0; s < 4; ++s) mbar_init(&x_full[s], 2);
    for (int s = 0; s < NK; ++s) { mbar_init(&k_full[s], 1); mbar_init(&k_empty[s], 1); }
    for (int s = 0; s < NV; ++s) { mbar_init(&v_full[s], 1); mbar_init(&v_empty[s], 1); }
    mbar_init(s_full, 1);
    mbar_init(s_empty, 8);
    for (int s = 0; s < 2; ++s) mbar_init(&dp_full[s], 1);
    for (int s = 0; s < 4; ++s) mbar_init(&ds_full[s], 4);
    mbar_init(fin_full, 1);
    for (int s = 0; s < NK; ++s) mbar_init(&k_part[s], 1);
    for (int s = 0; s < NV; ++s) mbar_init(&v_part[s], 1);
    *pulse = 0;
    mbar_fence_init();
  }
  if (warp == 8) { tmem_alloc<Cfg::TMEM_COLS>(tmem_slot); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();                            // the prologue above ran under the previous kernel's tail; global memory from here on

  PackedWalk<false> walk(p.plan, p.q_heads, reinterpret_cast<int4*>(smem + Cfg::OFF_ITEMS));
  int4 entry;
  int which;

  if (warp >= 8) {
    fewer_registers<HD>();
    if (warp == 10) {
      uint32_t itc = 0, kc = 0;
      bool ok = true;
      while (ok && walk.next(entry, which)) {
        const int lo = entry.x, hi = entry.y, n_kv = entry.z + 1, h = which, hk = which / p.group, qrow = lo + entry.z * FA_BM;
        if (!warp_wait(q_empty, (itc & 1) ^ 1)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_EMPTY); break; }
        if (elect_one()) {
          mbar_expect_tx(q_full, 2 * Cfg::T_BYTES);
#pragma unroll
          for (int x = 0; x < HD / 64; ++x) {
            tma_load_2d(smem + Cfg::OFF_Q + x * (FA_BM * 128), &tmQ, q_full, h * HD + x * 64, qrow);
            tma_load_2d(smem + Cfg::OFF_DO + x * (FA_BM * 128), &tmDO, q_full, h * HD + x * 64, qrow);
          }
        }
        for (int j = 0; j < n_kv; ++j, ++kc) {
          const int sk = kc % NK, sv = kc % NV, row = lo + j * FA_BN;
          const bool part = row + FA_BN > hi;
          uint8_t *k_tile = smem + Cfg::OFF_K + sk * Cfg::T_BYTES, *v_tile = smem + Cfg::OFF_V + sv * Cfg::T_BYTES;
          if (!warp_wait(&k_empty[sk], ((kc / NK) & 1) ^ 1)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_EMPTY); ok = false; break; }
          if (elect_one()) {
            uint64_t* bar = part ? &k_part[sk] : &k_full[sk];
            *pulse = kc + 1;
            mbar_expect_tx(bar, Cfg::T_BYTES);
#pragma unroll
            for (int x = 0; x < HD / 64; ++x) tma_load_2d(k_tile + x * (FA_BN * 128), &tmK, bar, hk * HD + x * 64, row);
          }
          if (!warp_wait(&v_empty[sv], ((kc / NV) & 1) ^ 1)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_EMPTY); ok = false; break; }
          if (elect_one()) {
            uint64_t* bar = part ? &v_part[sv] : &v_full[sv];
            mbar_expect_tx(bar, Cfg::T_BYTES);
#pragma unroll
            for (int x = 0; x < HD / 64; ++x) tma_load_2d(v_tile + x * (FA_BN * 128), &tmV, bar, hk * HD + x * 64, row);
          }
          __syncwarp();
        }
        ++itc;
      }
    } else if (warp == 11) {
      // ------------- zeros in place of rows behind a sequence, which only an item's last block can have
      uint32_t kc = 0, k_phases = 0, v_phases = 0;
      while (walk.next(entry, which)) {
        const int row = entry.x + entry.z * FA_BN, from = entry.y - row;
        kc += entry.z + 1;
        if (from >= FA_BN) continue;
        const int sk = (kc - 1) % NK, sv = (kc - 1) % NV;
        // from the last such item to this one's last block
        if (!idle_wait(&k_part[sk], (k_phases >> sk) & 1, pulse)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_FULL); break; }
        clear_rows<HD>(smem + Cfg::OFF_K + sk * Cfg::T_BYTES, from, lane);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&k_full[sk]);
        if (!warp_wait(&v_part[sv], (v_phases >> sv) & 1)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_FULL); break; }
        clear_rows<HD>(smem + Cfg::OFF_V + sv * Cfg::T_BYTES, from, lane);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_full[sv]);
        k_phases ^= 1u << sk;
        v_phases ^= 1u << sv;
      }
    } else if (warp == 8) {
      // ------------- MMA issuer A: S = Q K_j^T
      constexpr uint32_t idesc_s = umma_idesc_bf16(FA_BM, FA_BN, 0, 0);
      const uint64_t q_desc = desc_k(smem + Cfg::OFF_Q), k_desc = desc_k(smem + Cfg::OFF_K);
      uint32_t itc = 0, kc = 0;
      bool ok = true;
      while (ok && walk.next(entry, which)) {
        const int n_kv = entry.z + 1;
        if (!warp_wait(q_full, itc & 1)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_FULL); break; }
        for (int j = 0; j < n_kv; ++j, ++kc) {
          const int st = kc % NK;
          if (!warp_wait(&k_full[st], (kc / NK) & 1)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_FULL); ok = false; break; }
          if (kc > 0 && !warp_wait(s_empty, (kc - 1) & 1)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_TMEM_EMPTY); ok = false; break; }
          tc_fence_after();
          if (elect_one()) {
            const uint64_t kd = desc_at(k_desc, st * Cfg::T_BYTES);
#pragma unroll
            for (int ks = 0; ks < HD / 16; ++ks) {
              const uint32_t off = (ks >> 2) * (FA_BM * 128) + (ks & 3) * 32;
              umma_f16(tmem_base + Cfg::TM_S, desc_at(q_desc, off), desc_at(kd, off), idesc_s, ks > 0 ? 1u : 0u);
            }
            umma_commit(s_full);
            if (j + 1 == n_kv) umma_commit(q_empty);
          }
          __syncwarp();
        }
        ++itc;
      }
    } else if (warp == 9) {
      // ------------- MMA issuer B: dP = dO V_j^T and dQ += dS K_j (dS from TMEM, over dP)
      constexpr uint32_t idesc_s = umma_idesc_bf16(FA_BM, FA_BN, 0, 0);
      constexpr uint32_t idesc_q = umma_idesc_bf16(FA_BM, HD, 0, 1);   // dQ[q x HD] += dS[q x keys] * K[keys x HD]
      const uint64_t do_desc = desc_k(smem + Cfg::OFF_DO), v_desc = desc_k(smem + Cfg::OFF_V), k_desc = desc_mn(smem + Cfg::OFF_K);
      uint32_t itc = 0, kc = 0;
      bool ok = true;
      auto issue_dp = [&](uint32_t n, bool last) -> bool {
        const int st = n % NV;
        if (!warp_wait(&v_full[st], (n / NV) & 1)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_FULL); return false; }
        tc_fence_after();
        if (elect_one()) {
          const uint64_t vd = desc_at(v_desc, st * Cfg::T_BYTES);
#pragma unroll
          for (int ks = 0; ks < HD / 16; ++ks) {
            const uint32_t off = (ks >> 2) * (FA_BM * 128) + (ks & 3) * 32;
            umma_f16(tmem_base + Cfg::TM_DP + (n & 1) * FA_BN, desc_at(do_desc, off), desc_at(vd, off), idesc_s, ks > 0 ? 1u : 0u);
          }
          umma_commit(&dp_full[n & 1]);
          umma_commit(&v_empty[st]);
          if (last) umma_commit(q_empty);
        }
        __syncwarp();
        return true;
      };
      while (ok && walk.next(entry, which)) {
        const int n_kv = entry.z + 1;
        if (!warp_wait(q_full, itc & 1)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_FULL); break; }
        ok = issue_dp(kc, n_kv == 1);
        if (ok && n_kv > 1) ok = issue_dp(kc + 1, n_kv == 2);
        for (int j = 0; j < n_kv && ok; ++j, ++kc) {
          const int st = kc % NK;
          if (!warp_wait(&k_full[st], (kc / NK) & 1)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_FULL); ok = false; break; }
          const uint64_t kd = desc_at(k_desc, st * Cfg::T_BYTES);
          const uint32_t ds_tm = tmem_base + Cfg::TM_DP + (kc & 1) * FA_BN;
          uint64_t* ready = ds_full + (kc & 1) * 2;
          for (int half = 0; half < 2; ++half) {
            // an item's first product replaces the accumulator: wait until both halves' warps have read the previous item's
            if (j == 0 && half == 0) ok = warp_wait(&ready[1], (kc >> 1) & 1);
            if (!ok || !warp_wait(&ready[half], (kc >> 1) & 1)) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_SOFTMAX); ok = false; break; }
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
              for (int ks = 0; ks < 8; ++ks)           // dS, then its remainder
                umma_f16_ts(tmem_base + Cfg::TM_DQ, ds_tm + half * 64 + ks * 8, desc_at(kd, (half * 4 + (ks & 3)) * 2048),
                            idesc_q, (j > 0 || half > 0 || ks > 0) ? 1u : 0u);
              if (half == 1) {
                umma_commit(&k_empty[st]);
                if (j + 1 == n_kv) umma_commit(fin_full);
              }
            }
            __syncwarp();
          }
          if (!ok) break;
          if (j + 2 < n_kv) ok = issue_dp(kc + 2, j + 3 == n_kv);      // over dS_j: ordered after its product by the pipe
        }
        ++itc;
      }
    }
  } else {
    more_registers<HD>();
    const int quad = warp & 3;
    const int half = warp >> 2;
    const int r = quad * 32 + lane;
    const uint32_t t_lane = tmem_base + ((uint32_t)(quad * 32) << 16);
    const unsigned long long sl22 = f2_splat(p.scale * LOG2E), scale2 = f2_splat(p.scale);
    uint32_t itc = 0, kc = 0;
    bool ok = true;
    float* xch = reinterpret_cast<float*>(smem + Cfg::OFF_X);
    uint32_t met = 0;
    const auto rows_met = [&]() -> bool {          // both warps of these 32 rows have written their sums
      __syncwarp();
      if (lane == 0) mbar_arrive(&x_full[quad]);
      return warp_wait(&x_full[quad], met++ & 1);
    };
    clear_others(p.plan, p.dq, p.dq_stride, p.q_heads * HD, threadIdx.x, 256);
    while (ok && walk.next(entry, which)) {
      const int hi = entry.y, n_kv = entry.z + 1, h = which, q0 = entry.x + entry.z * FA_BM + quad * 32, qi = q0 + lane;
      const long long stat_at = (long long)h * p.plan.tokens + qi;
      const unsigned long long nlse2 = f2_splat(qi < hi ? -p.lse[stat_at] * LOG2E : -INFINITY);
      unsigned long long ndlt2 = f2_splat(qi < hi ? -p.delta[stat_at] * p.scale : 0.f), sum2 = 0;
      for (int j = 0; j < n_kv; ++j, ++kc) {
        ok = warp_wait(s_full, kc & 1);
        if (!ok) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_TMEM_FULL); break; }
        tc_fence_after();
        const uint32_t s_addr = t_lane + Cfg::TM_S + half * 64;
        const uint32_t dp_addr = t_lane + Cfg::TM_DP + (kc & 1) * FA_BN + half * 64;
        uint32_t s[64];
        tmem_ld32(s_addr, s);
        tmem_ld32(s_addr + 32, s + 32);
        tmem_ld_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(s_empty);
#pragma unroll
        for (int i = 0; i < 64; i += 4) {
          bwd_prob2(s[i], s[i + 1], sl22, nlse2);
          if ((i >> 2) % 4 < PB_FMA_PAIRS<HD>) bwd_prob2<true>(s[i + 2], s[i + 3], sl22, nlse2);
          else bwd_prob2(s[i + 2], s[i + 3], sl22, nlse2);
        }
        if (j + 1 == n_kv) {                       // the diagonal block: keys up to the query's own
          const int lim = r - half * 64;
#pragma unroll
          for (int i = 0; i < 64; ++i) s[i] = (i <= lim) ? s[i] : 0u;
        }
        ok = warp_wait(&dp_full[kc & 1], (kc >> 1) & 1);
        if (!ok) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_TMEM_FULL); break; }
        tc_fence_after();
        uint32_t dp[64];
        tmem_ld32(dp_addr, dp);
        tmem_ld32(dp_addr + 32, dp + 32);
        tmem_ld_wait();
        if (n_kv == 1) {                           // the whole row is here: delta is its sum of p dP
          unsigned long long mine2 = 0;
#pragma unroll
          for (int i = 0; i < 64; i += 2) mine2 = f2_fma(f2_of(s[i], s[i + 1]), f2_of(dp[i], dp[i + 1]), mine2);
          xch[half * FA_BM + r] = f2_sum(mine2);
          ok = rows_met();
          if (!ok) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_SOFTMAX); break; }
          ndlt2 = f2_splat(-(xch[r] + xch[FA_BM + r]) * p.scale);
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t w[16], rest[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            uint32_t *a = s + c * 32 + 2 * i, *b = dp + c * 32 + 2 * i;
            bwd_ds2(a[0], a[1], b[0], b[1], scale2, ndlt2);
            const unsigned long long ds = f2_of(a[0], a[1]);
            sum2 = f2_add(sum2, ds);
            w[i] = f2_bf16(ds);
            rest[i] = f2_bf16(f2_fma(f2_bf16x2(w[i]), f2_splat(-1.f), ds));
          }
          tmem_st16(dp_addr + c * 16, w);
          tmem_st16(dp_addr + 32 + c * 16, rest);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ds_full[(kc & 1) * 2 + half]);
      }
      if (!ok) break;
      ok = warp_wait(fin_full, itc & 1);
      if (!ok) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_TMEM_FULL); break; }
      ++itc;
      tc_fence_after();
      // Into the first half's own place: it has read the second's by now (dQ holds its dS), and the second half writes there again only when dQ holds the
      // next item's
      if (half == 1) xch[r] = f2_sum(sum2);
      ok = rows_met();
      if (!ok) { if (lane == 0) report_error(p.status, OA_KERR_WAIT_SOFTMAX); break; }
      if (half == 0 && qi < hi) p.ndelta[stat_at] = lo_of(ndlt2) - (f2_sum(sum2) + xch[r]);
      __nv_bfloat16* base = p.dq + q0 * p.dq_stride + h * HD + half * (HD / 2);
      uint32_t a[HD / 2];
#pragma unroll
      for (int c = 0; c < HD / 64; ++c) tmem_ld32(t_lane + Cfg::TM_DQ + half * (HD / 2) + c * 32, a + c * 32);
      tmem_ld_wait();
#pragma unroll
      for (int c = 0; c < HD / 64; ++c) store_rows(base + c * 32, p.dq_stride, hi - q0, a + c * 32, 1.f, lane);
      tc_fence_before();   // dQ is read before this warp's next ds_full arrival lets the next item's products overwrite it
    }
  }
  pdl_launch_dependents();
  tc_fence_before();
  __syncthreads();
  if (warp == 8) { tc_fence_after(); tmem_dealloc<Cfg::TMEM_COLS>(tmem_base); }
}

// dK and dV of the tiles whose query heads several CTAs shared: their sums added up in order.  A warp takes four rows of 64 columns
constexpr int JOIN_THREADS = 256;
template <int HD>
__global__ void __launch_bounds__(JOIN_THREADS) packed_join_kernel(const PackedBwdParams p) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int CHUNKS = FA_BM * HD / 8 / JOIN_THREADS;       // of dK or dV of a tile and head, 8 columns to a thread
  const long long units = (long long)p.plan.tiles() * p.kv_heads * 2 * CHUNKS;
  for (long long u = blockIdx.x; u < units; u += gridDim.x) {
    const int chunk = (int)(u % CHUNKS), w = (int)(u / CHUNKS) & 1;
    const long long at = u / (2 * CHUNKS);
    const int tile = (int)(at / p.kv_heads), kv_head = (int)(at - (long long)tile * p.kv_heads);
    const PackedKvItem<true> item(p, p.plan.tile(tile), kv_head * p.parts);
    const int i = chunk * JOIN_THREADS + threadIdx.x, col = (i & 7) + i / (8 * FA_BM) * 8, row = i / 8 % FA_BM;
    float v[8] = {};
    for (int part = 0; part < p.parts; ++part) {
      const float4* from = p.partial + p.partial_at(part, tile, kv_head, w, HD) + 2 * col * FA_BM + row;
      const float4 a = from[0], b = from[FA_BM];
      v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
      v[4] += b.x; v[5] += b.y; v[6] += b.z; v[7] += b.w;
    }
    const int key = item.lo + item.key0 + row;
    if (key >= item.hi) continue;
    __nv_bfloat16* to = (w == 0 ? p.dv + key * p.dv_stride : p.dk + key * p.dk_stride) + kv_head * HD + col * 8;
    *reinterpret_cast<uint4*>(to) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
  }
}

int make_tmap_2d_bf16(CUtensorMap* out, const void* ptr, uint64_t inner, uint64_t outer, uint64_t ld,
                      uint32_t box_inner, uint32_t box_outer);

static int packed_ctas(long long items) {
  const int sms = sm_count();
  return (int)(items < 1 ? 1 : items < sms ? items : sms);      // persistent: one CTA per SM walks its items
}

// Over how many CTAs the query heads of a key-value head go.  A tile of keys is as long as all the queries behind it times the group, and with few tiles the first
// ones are most of the kernel: more as long as the longest item, were the sequences equally long, is more than 5/4 of an SM's share, at head dim 128, where
// partial sums are twice as many, 8/5.  Gradients of 64 heads over 8 of 64 with 1 / 2 / 4 CTAs: one sequence of 1000 rows 111 / 81 / 68 us, of 2000 251 / 187 / 196, of 3000 417 / 378;
// 4 of 375 (2.3 shares) 72 / 66 / 73, of 500 (1.9) 95 / 96, of 750 (1.3) 147 / 155, of rising lengths up to 1200 197 / 192, 1800 beside 3 of 400 262 / 239.  Of 32 over 8 of 128: one of 1500 131 /
// 109 / 115, of 3000 (1.5) 295 / 287; 2 of 750 97 / 80 / 90; 8 of 250 (1.5) 52 / 69, of rising lengths up to 444 115 / 136, 1200 beside 7 of 114 116 / 107.
// The host knows the number of sequences, not their lengths: where one is much longer than the others, or many are empty, more would be better than it takes.
static int packed_parts(int tokens, int batch, int kv_heads, int group, int head_dim) {
  const long long seqs = batch > 0 ? batch : 1, n = tokens / (FA_BM * seqs) + 1;
  const long long share = head_dim == 64 ? 32 : 25;                  // 2 / (5/4), 2 / (8/5), in twentieths
  int parts = 1;
  for (int d = 2; tokens > PACKED_SHORT && d <= group && d <= 64 && 20 * parts * kv_heads * seqs * (n + 1) < share * sm_count(); ++d)
    if (group % d == 0) parts = d;
  return parts;
}
static size_t packed_delta_floats(int tokens, int q_heads) { return (2 * (size_t)q_heads * tokens + 3) & ~(size_t)3; }

static int packed_check(int tokens, int batch, int q_heads, int kv_heads, int head_dim) {
  if (tokens < 0 || batch < 0 || kv_heads < 1 || q_heads < 1 || q_heads % kv_heads) return OA_ERR_ARG;
  if (head_dim != 64 && head_dim != 128) return OA_ERR_UNSUPPORTED;
  if (tokens > PACKED_MAX_TOKENS || batch > PACKED_MAX_BATCH || (long long)packed_max_tiles(tokens, batch) * q_heads > 0x3fffffffll || q_heads > (1 << 19)) return OA_ERR_TOO_LARGE;
  return OA_OK;
}

template <int HD, bool HEADS>
static int packed_fwd(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const PackedFwdParams& p, cudaStream_t st) {
  static std::atomic<unsigned long long> allowed;
  if (allow_smem(allowed, (const void*)packed_fwd_kernel<HD, HEADS>, PackedFwdCfg<HD>::SMEM_BYTES) != cudaSuccess) return OA_ERR_LAUNCH;
  // starts under the launch for short sequences, which is over at once where there are none
  const long long items = HEADS ? (long long)packed_max_tiles(p.plan.tokens, p.plan.batch) * (p.q_heads / 2)
                                     : (long long)packed_max_pairs(p.plan.tokens, p.plan.batch) * p.q_heads;
  launch_pdl_if(pdl_on(true), packed_fwd_kernel<HD, HEADS>, dim3(packed_ctas(items)), dim3(PackedFwdCfg<HD>::THREADS), PackedFwdCfg<HD>::SMEM_BYTES, st, tq, tk, tv, p);
  return cudaGetLastError() == cudaSuccess ? OA_OK : OA_ERR_LAUNCH;
}

template <int HD>
static int packed_bwd(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& tdo, const PackedBwdParams& p, cudaStream_t st) {
  static std::atomic<unsigned long long> allowed_kv, allowed_split, allowed_q;
  const auto kv_kernel = p.parts > 1 ? packed_bwd_kv_kernel<HD, true> : packed_bwd_kv_kernel<HD, false>;
  if (allow_smem(p.parts > 1 ? allowed_split : allowed_kv, (const void*)kv_kernel, PackedKvCfg<HD>::SMEM_BYTES) != cudaSuccess) return OA_ERR_LAUNCH;
  if (allow_smem(allowed_q, (const void*)packed_bwd_q_kernel<HD>, PackedQCfg<HD>::SMEM_BYTES) != cudaSuccess) return OA_ERR_LAUNCH;
  const long long tiles = packed_max_tiles(p.plan.tokens, p.plan.batch);
  // dQ first: it works out what delta is off by.  It starts under the launch for short sequences, which is over at once where there are none
  launch_pdl_if(pdl_on(true), packed_bwd_q_kernel<HD>, dim3(packed_ctas(tiles * p.q_heads)), dim3(PB_THREADS), PackedQCfg<HD>::SMEM_BYTES, st, tq, tk, tv, tdo, p);
  launch_pdl(kv_kernel, dim3(packed_ctas(tiles * p.kv_heads * p.parts)), dim3(PB_THREADS), PackedKvCfg<HD>::SMEM_BYTES, st, tq, tk, tv, tdo, p);
  if (p.parts > 1) {
    const long long units = tiles * p.kv_heads * 2 * (FA_BM * HD / 8 / JOIN_THREADS);
    launch_short(packed_join_kernel<HD>, dim3((unsigned)(units < 8 * sm_count() ? units : 8 * sm_count())), dim3(JOIN_THREADS), 0, st, p);
  }
  return cudaGetLastError() == cudaSuccess ? OA_OK : OA_ERR_LAUNCH;
}

}  // namespace oa

using namespace oa;

extern "C" int oa_packed_attn(const void* q, const void* k, const void* v, const int* plan, void* o, float* lse, int tokens, int batch, int q_heads,
                              int kv_heads, int head_dim, long long q_stride, long long k_stride, long long v_stride, long long o_stride, float scale,
                              int* status, void* stream) {
  if (int rc = packed_check(tokens, batch, q_heads, kv_heads, head_dim)) return rc;
  if (o_stride != (long long)q_heads * head_dim || !(scale > 0.f)) return OA_ERR_ARG;
  if (reinterpret_cast<uintptr_t>(o) & 15) return OA_ERR_ALIGN;
  if (tokens == 0) return OA_OK;
  CUtensorMap tq, tk, tv;
  int rc;
  if ((rc = make_tmap_2d_bf16(&tq, q, (uint64_t)q_heads * head_dim, tokens, (uint64_t)q_stride, 64, FA_BM))) return rc;
  if ((rc = make_tmap_2d_bf16(&tk, k, (uint64_t)kv_heads * head_dim, tokens, (uint64_t)k_stride, 64, FA_BN))) return rc;
  if ((rc = make_tmap_2d_bf16(&tv, v, (uint64_t)kv_heads * head_dim, tokens, (uint64_t)v_stride, 64, FA_BN))) return rc;
  const int group = q_heads / kv_heads;
  const PackedFwdParams p{{plan, batch, tokens}, q_heads, group, scale, (__nv_bfloat16*)o, lse, status};
  cudaStream_t st = (cudaStream_t)stream;
  const PackedShortFwd brief{p.plan, (const __nv_bfloat16*)q, (const __nv_bfloat16*)k, (const __nv_bfloat16*)v, (__nv_bfloat16*)o, lse, q_stride, k_stride, v_stride,
                             o_stride, q_heads, group, scale};
  if ((rc = packed_short_fwd(brief, head_dim, st))) return rc;
  if (group % 2 == 0) return head_dim == 64 ? packed_fwd<64, true>(tq, tk, tv, p, st) : packed_fwd<128, true>(tq, tk, tv, p, st);
  return head_dim == 64 ? packed_fwd<64, false>(tq, tk, tv, p, st) : packed_fwd<128, false>(tq, tk, tv, p, st);
}

// scratch: float[2][q_heads, tokens], delta from the output and from the rows' sums; then what CTAs that share a group's heads add up to
extern "C" size_t oa_packed_attn_bwd_scratch_bytes(int tokens, int batch, int q_heads, int kv_heads, int head_dim) {
  if (packed_check(tokens, batch, q_heads, kv_heads, head_dim)) return 0;
  const int parts = packed_parts(tokens, batch, kv_heads, q_heads / kv_heads, head_dim);
  const size_t sums = parts > 1 ? (size_t)parts * packed_max_tiles(tokens, batch) * kv_heads * 2 * FA_BM * head_dim : 0;
  return (packed_delta_floats(tokens, q_heads) + sums) * sizeof(float);
}

extern "C" int oa_packed_attn_bwd(const void* q, const void* k, const void* v, const void* o, const void* dout, const float* lse, const int* plan, void* dq,
                                  void* dk, void* dv, int tokens, int batch, int q_heads, int kv_heads, int head_dim, long long q_stride,
                                  long long k_stride, long long v_stride, long long o_stride, long long do_stride, long long dq_stride,
                                  long long dk_stride, long long dv_stride, float scale, void* scratch, int* status, void* stream) {
  if (int rc = packed_check(tokens, batch, q_heads, kv_heads, head_dim)) return rc;
  if (!(scale > 0.f)) return OA_ERR_ARG;
  if (((dq_stride | dk_stride | dv_stride | o_stride | do_stride) & 7) ||
      ((reinterpret_cast<uintptr_t>(dq) | reinterpret_cast<uintptr_t>(dk) | reinterpret_cast<uintptr_t>(dv) | reinterpret_cast<uintptr_t>(o) |
        reinterpret_cast<uintptr_t>(dout) | reinterpret_cast<uintptr_t>(scratch)) & 15))
    return OA_ERR_ALIGN;
  if (tokens == 0) return OA_OK;
  cudaStream_t st = (cudaStream_t)stream;
  CUtensorMap tq, tk, tv, tdo;
  int rc;
  const uint64_t q_cols = (uint64_t)q_heads * head_dim, kv_cols = (uint64_t)kv_heads * head_dim;
  if ((rc = make_tmap_2d_bf16(&tq, q, q_cols, tokens, (uint64_t)q_stride, 64, FA_BM))) return rc;
  if ((rc = make_tmap_2d_bf16(&tk, k, kv_cols, tokens, (uint64_t)k_stride, 64, FA_BN))) return rc;
  if ((rc = make_tmap_2d_bf16(&tv, v, kv_cols, tokens, (uint64_t)v_stride, 64, FA_BN))) return rc;
  if ((rc = make_tmap_2d_bf16(&tdo, dout, q_cols, tokens, (uint64_t)do_stride, 64, FA_BM))) return rc;
  const long long units = (long long)packed_max_tiles(tokens, batch) * ((FA_BM / DELTA_ROWS * (long long)q_heads * (head_dim / 8) + DELTA_THREADS - 1) / DELTA_THREADS);
  const int fill = 8 * sm_count();
  launch_pdl(head_dim == 64 ? packed_delta_kernel<64> : packed_delta_kernel<128>, dim3((unsigned)(units < 1 ? 1 : units < fill ? units : fill)), dim3(DELTA_THREADS), 0, st,
             (const __nv_bfloat16*)o, (const __nv_bfloat16*)dout, (float*)scratch, PackedPlan{plan, batch, tokens}, q_heads, o_stride, do_stride);
  const int parts = packed_parts(tokens, batch, kv_heads, q_heads / kv_heads, head_dim);
  const PackedBwdParams p{{plan, batch, tokens}, q_heads, kv_heads, q_heads / kv_heads, scale, lse, (const float*)scratch, (float*)scratch + (size_t)q_heads * tokens, (__nv_bfloat16*)dq,
                          (__nv_bfloat16*)dk, (__nv_bfloat16*)dv, dq_stride, dk_stride, dv_stride, status, parts, q_heads / kv_heads / parts,
                          reinterpret_cast<float4*>((float*)scratch + packed_delta_floats(tokens, q_heads))};
  const PackedShortBwd brief{p.plan, (const __nv_bfloat16*)q, (const __nv_bfloat16*)k, (const __nv_bfloat16*)v, (const __nv_bfloat16*)dout, lse, p.dq, p.dk, p.dv,
                             q_stride, k_stride, v_stride, do_stride, dq_stride, dk_stride, dv_stride, kv_heads, p.group, scale};
  if ((rc = packed_short_bwd(brief, head_dim, st))) return rc;
  return head_dim == 64 ? packed_bwd<64>(tq, tk, tv, tdo, p, st) : packed_bwd<128>(tq, tk, tv, tdo, p, st);
}
