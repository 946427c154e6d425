// opc_i8_gemm.cuh -- Y[t][r] = sx[t] * sw[r] * sum_k X[t][k] W[r][k] (+ bias[r]) over 8-bit integers.
//
// Two kernels, both with exact 32-bit sums, so a result depends on neither the kernel nor the split:
//
// i8_gemm_kernel  the 5th-generation tensor cores (tcgen05.mma, kind::i8), two SMs to a tile
//                 (cta_group::2): 256 channels x N tokens, N = 32 .. 256 by the number of tokens.
//                 Each CTA of a pair stages its 128 channels and half of the tokens, 128 values deep,
//                 by TMA (128-byte swizzle); the hardware reads both halves, so a CTA's shared memory
//                 takes 8 KB instead of 12 KB per 128 x 256 x 32 step -- alone, a CTA would need
//                 96 bytes a clock from L2 and as many from shared memory.
//                 Persistent: pairs take whole tiles in turn (a group of 8 channel tiles at a time, so
//                 that what they read stays in L2), then share the rest out along K in equal ranges.
//                 Tiles cut by a range are summed through the workspace by whoever comes last.
//                   warp 0     TMA
//                   warp 1     tensor memory; in the pair's first CTA it issues the MMAs
//                   warps 2-9  epilogue: two warps per TMEM lane quarter, half of the columns each;
//                              it reads one accumulator while the MMAs fill the other
// i8_gemv_kernel  up to 8 tokens: mma.sync fragments straight from global memory; bound by the reading
//                 of W.  16 channels per CTA, K dealt to its warps 128 bytes at a time.
#pragma once

#include <cuda.h>

#include "opc_i8_rows.cuh"
#include "opc_tcgen05.cuh"

namespace opc {

constexpr int kI8Block = 128;                 // values of K per stage (one 128-byte swizzled row)
constexpr int kI8ABytes = 128 * kI8Block;     // a CTA's channels of a stage
constexpr int kI8Epi = 8;                     // epilogue warps of a CTA
constexpr int kI8Threads = 64 + 32 * kI8Epi;
constexpr int kI8Group = 8;                   // channel tiles taken together
constexpr int kI8MaxStages = 12;
constexpr int kI8SmemBudget = 227 * 1024 - 1024 - 512;  // less alignment slack and barriers

// A stage holds `sub` blocks of 128 values of K: the channels' block, then half of the tokens'.
__host__ __device__ constexpr int i8_block_bytes(int n) { return kI8ABytes + n * (kI8Block / 2); }
__host__ __device__ constexpr int i8_stages(int n, int sub) {
  return kI8SmemBudget / (sub * i8_block_bytes(n)) > kI8MaxStages ? kI8MaxStages : kI8SmemBudget / (sub * i8_block_bytes(n));
}

struct I8Out {
  const float *sx, *sw;
  const void* bias;
  void* y;
  int64_t ldy;
  int32_t rows, M, bias_type, y_type;
};

// How the tiles are dealt to the pairs of CTAs.
struct I8Deal {
  int32_t tile_n;              // tokens of a tile
  int32_t m_tiles, n_tiles;    // tiles of 256 channels, of tile_n tokens
  int32_t sub;                 // blocks of 128 values of K in a stage
  int32_t nk;                  // stages of a tile
  int32_t full;                // tiles taken whole, in turn (a multiple of the pairs)
  int32_t rest;                // tiles after them, cut along K into `sharers` equal ranges
  int32_t sharers;             // rest .. pairs (== rest: none is cut); a range lies in at most 2 tiles
};

struct I8GemmArgs {
  I8Out o;
  I8Deal d;
  int32_t* count;              // [rest][2 CTAs][epilogue warps] arrivals at cut tiles; 0 between calls
  int32_t* part;               // [sharers][2][2 CTAs][tile_n / 4][128][4] sums of cut tiles
  int* err;
};

__device__ __forceinline__ float i8_load1(int type, const void* p, int64_t i) {
  if (type == kI8F16) return __half2float(static_cast<const __half*>(p)[i]);
  if (type == kI8BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return static_cast<const float*>(p)[i];
}
template <int kY>
__device__ __forceinline__ void i8_store1(void* p, int64_t i, float v) {
  if constexpr (kY == kI8F16) static_cast<__half*>(p)[i] = __float2half_rn(v);
  else if constexpr (kY == kI8BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else static_cast<float*>(p)[i] = v;
}
// The one way from a sum to a result: fp32 operations in this order, no fused ones.  Without a bias it
// is -0, which changes nothing.
__device__ __forceinline__ float i8_result(int32_t sum, float sx, float sw, float bias) {
  return __fadd_rn(__fmul_rn(__fmul_rn(static_cast<float>(sum), sx), sw), bias);
}
__device__ __forceinline__ float i8_bias(const I8Out& o, int32_t r) { return o.bias ? i8_load1(o.bias_type, o.bias, r) : -0.f; }

// ------------------------------------------------------------------------------------------------
// Pairs of CTAs
// ------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;" ::: "memory");
}
// Shared-memory address of the same variable in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t map_to_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// The asynchronous operations are issued by one lane (`leader`) of a converged warp: outside a divergent
// branch their operands can stay in uniform registers.
// A TMA load into this CTA's shared memory that completes on a barrier of either CTA of the pair.
__device__ __forceinline__ void tma_load_2d_pair(uint32_t leader, uint32_t dst, const CUtensorMap* map, int32_t x, int32_t y, uint32_t bar) {
  asm volatile(
      "{\n .reg .pred l;\n setp.ne.b32 l, %5, 0;\n"
      " @l cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n}\n" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(bar), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void mbar_expect_tx_by(uint32_t leader, uint32_t bar, uint32_t bytes) {
  asm volatile(
      "{\n .reg .pred l;\n setp.ne.b32 l, %2, 0;\n @l mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n}\n" ::"r"(bar), "r"(bytes),
      "r"(leader)
      : "memory");
}
__device__ __forceinline__ void umma_i8_pair(uint32_t leader, uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n .reg .pred p, l;\n setp.ne.b32 l, %5, 0;\n setp.ne.b32 p, %4, 0;\n"
      " @l tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accum), "r"(leader)
      : "memory");
}
// Arrives at the barrier of both CTAs once the MMAs issued so far are done.
__device__ __forceinline__ void umma_commit_pair(uint32_t leader, uint32_t bar) {
  asm volatile(
      "{\n .reg .pred l;\n setp.ne.b32 l, %2, 0;\n"
      " @l tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n}\n" ::"r"(bar),
      "h"(static_cast<uint16_t>(3)), "r"(leader)
      : "memory");
}
// kind::i8, A and B signed, D 32-bit integers, both K-major, 256 channels x n tokens.
__device__ __forceinline__ uint32_t i8_idesc(int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(256 >> 4) << 24);
}

// One pair's work, item by item: a tile, and the stages of it that are the pair's.
struct I8Walk {
  const I8Deal& d;
  int32_t pair, pairs, next;   // next whole tile
  int64_t u, u1;               // the pair's range of the rest, in stages
  int32_t tile, k0, k1;
  __device__ I8Walk(const I8Deal& deal, int32_t p, int32_t n) : d(deal), pair(p), pairs(n), next(p), tile(0), k0(0), k1(0) {
    const int64_t all = static_cast<int64_t>(d.rest) * d.nk;
    u = p < d.sharers ? all * p / d.sharers : 0;
    u1 = p < d.sharers ? all * (p + 1) / d.sharers : 0;
  }
  __device__ bool step() {
    if (next < d.full) {
      tile = next;
      next += pairs;
      k0 = 0;
      k1 = d.nk;
      return true;
    }
    if (u >= u1) return false;
    const int32_t j = static_cast<int32_t>(u / d.nk);
    tile = d.full + j;
    k0 = static_cast<int32_t>(u - static_cast<int64_t>(j) * d.nk);
    k1 = static_cast<int32_t>(min(static_cast<int64_t>(d.nk), k0 + (u1 - u)));
    u += k1 - k0;
    return true;
  }
  __device__ bool cut() const { return k0 > 0 || k1 < d.nk; }
  // Channel and token tile: groups of kI8Group channel tiles, channels first.
  __device__ void place(int32_t* mi, int32_t* ni) const {
    const int32_t per = kI8Group * d.n_tiles, g = tile / per, in = tile - g * per;
    const int32_t width = min(kI8Group, d.m_tiles - g * kI8Group);
    *mi = g * kI8Group + in % width;
    *ni = in / width;
  }
  // Who shares the cut tile `tile`: the pairs first .. last.
  __device__ int32_t owner(int64_t unit) const {
    return static_cast<int32_t>(((unit + 1) * d.sharers - 1) / (static_cast<int64_t>(d.rest) * d.nk));
  }
  __device__ void sharers(int32_t* first, int32_t* last) const {
    const int64_t a = static_cast<int64_t>(tile - d.full) * d.nk;
    *first = owner(a);
    *last = owner(a + d.nk - 1);
  }
  // Where pair p keeps its part of `tile`: of the two places, the second if its range began in the tile before.
  __device__ int32_t slot(int32_t p) const {
    const int64_t begin = static_cast<int64_t>(d.rest) * d.nk * p / d.sharers;
    return 2 * p + (begin / d.nk != tile - d.full ? 1 : 0);
  }
};

// tw: w [M][K], box 128 bytes x 128 channels; tx: x [rows][K], box 128 bytes x tile_n / 2 tokens; both
// with the 128-byte swizzle, zeros beyond the edges.
template <int kY>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kI8Threads, 1)
    i8_gemm_kernel(const __grid_constant__ CUtensorMap tw, const __grid_constant__ CUtensorMap tx, const I8GemmArgs a) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  const int kN = a.d.tile_n;
  const int sub = a.d.sub, stages = i8_stages(kN, sub);
  const uint32_t block_bytes = i8_block_bytes(kN), stage_bytes = sub * block_bytes;
  const uint32_t bars = base + stages * stage_bytes;
  const uint32_t full_b = bars, empty_b = full_b + 8 * kI8MaxStages, accf_b = empty_b + 8 * kI8MaxStages, acce_b = accf_b + 16,
                 drain_b = acce_b + 16, tmem_slot = drain_b + 8;
  unsigned char* tmem_slot_ptr = smem_raw + (tmem_slot - raw);

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int cols = kN <= 16 ? 32 : kN <= 32 ? 64 : kN <= 64 ? 128 : kN <= 128 ? 256 : 512;  // two accumulators

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(full_b + 8 * s, 1);
      mbar_init(empty_b + 8 * s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(accf_b + 8 * b, 1);
      mbar_init(acce_b + 8 * b, 2 * kI8Epi);  // both CTAs' epilogue warps
    }
    mbar_init(drain_b, 1);
    fence_mbar_init();
  }
  griddep_wait();  // everything before has ended: its tensor memory is free again, its results are there
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_slot), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // both CTAs' barriers are set up
  tc_fence_after();
  griddep_launch_dependents();  // every CTA that has come this far holds its tensor memory
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tmem_slot_ptr);
  bool ok = true;
  I8Walk walk(a.d, pair, pairs);

  if (warp == 0) {
    // ---------------------------------------------------------------- TMA
    const uint32_t leader = elect_leader();
    const uint32_t full0 = map_to_rank(full_b, 0);  // the first CTA's MMA warp waits for both CTAs' loads
    int g = 0, st = 0;
    uint32_t par = 1;  // of the stage's use before (the first round waits for nothing)
    while (ok && walk.step()) {
      int32_t mi, ni;
      walk.place(&mi, &ni);
      const int32_t r0 = mi * 256 + static_cast<int32_t>(rank) * 128, t0 = ni * kN + static_cast<int32_t>(rank) * (kN / 2);
      for (int k = walk.k0; k < walk.k1; ++k, ++g) {
        if (g >= stages) {
          ok = __all_sync(0xffffffffu, mbar_wait_bounded(empty_b + 8 * st, par));
          if (!ok) break;
        }
        if (rank == 0) mbar_expect_tx_by(leader, full_b + 8 * st, 2 * stage_bytes);
        uint32_t at = base + st * stage_bytes;
        int32_t x = k * sub * kI8Block;
        for (int j = 0; j < sub; ++j, at += block_bytes, x += kI8Block) {
          tma_load_2d_pair(leader, at, &tw, x, r0, full0 + 8 * st);
          tma_load_2d_pair(leader, at + kI8ABytes, &tx, x, t0, full0 + 8 * st);
        }
        if (++st == stages) {
          st = 0;
          par ^= 1;
        }
      }
    }
    // what is under way to this CTA's shared memory arrives before it ends: the loads (which the first
    // CTA's barriers count, for both) where a role gave up, and the last signals of the MMAs
    for (int i = 0; i < stages && i < g; ++i) {
      const uint32_t last = ((g - 1 - ((g - 1 - i) % stages)) / stages) & 1;  // parity of the stage's last use
      if (rank == 0) mbar_wait_bounded(full_b + 8 * i, last);
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait_bounded(empty_b + 8 * i, last));
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMAs
    if (rank == 0) {
      const uint32_t leader = elect_leader();
      const uint32_t idesc = i8_idesc(kN);
      int st = 0, tl = 0;
      uint32_t par = 0;
      while (ok && walk.step()) {
        const int b = tl & 1;
        if (tl >= 2) {
          ok = __all_sync(0xffffffffu, mbar_wait_bounded(acce_b + 8 * b, ((tl >> 1) - 1) & 1));
          if (!ok) break;
        }
        tc_fence_after();
        const uint32_t acc = tmem + static_cast<uint32_t>(b * (cols / 2));
        uint32_t more = 0;  // the tile's first MMA clears the accumulator
        for (int k = walk.k0; k < walk.k1; ++k) {
          ok = __all_sync(0xffffffffu, mbar_wait_bounded(full_b + 8 * st, par));
          if (!ok) break;
          tc_fence_after();
          uint32_t at = base + st * stage_bytes;
          for (int j = 0; j < sub; ++j, at += block_bytes) {
            const uint64_t ad = umma_desc_sw128(at), bd = umma_desc_sw128(at + kI8ABytes);
#pragma unroll
            for (int kk = 0; kk < kI8Block / 32; ++kk) {  // 32 bytes further in the swizzled rows
              umma_i8_pair(leader, acc, ad + 2 * kk, bd + 2 * kk, idesc, more);
              more = 1;
            }
          }
          umma_commit_pair(leader, empty_b + 8 * st);
          if (++st == stages) {
            st = 0;
            par ^= 1;
          }
        }
        if (!ok) break;
        umma_commit_pair(leader, accf_b + 8 * b);
        ++tl;
      }
      // no MMA of this pair is in flight past this point
      if (leader) asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(drain_b) : "memory");
      mbar_wait_bounded(drain_b, 0);
    }
  } else {
    // ---------------------------------------------------------------- epilogue
    const int e = warp - 2, quarter = warp & 3, half = e >> 2;
    const int row = 32 * quarter + lane;  // channel of the CTA's 128 = TMEM lane
    const uint32_t lanes = tmem + (static_cast<uint32_t>(32 * quarter) << 16);
    const uint32_t acce0 = map_to_rank(acce_b, 0);
    const int c0 = half * (kN / 2), c1 = c0 + kN / 2;  // this warp's columns, 16 at a time
    int tl = 0;
    while (walk.step()) {
      int32_t mi, ni;
      walk.place(&mi, &ni);
      const int32_t r = mi * 256 + static_cast<int32_t>(rank) * 128 + row, t0 = ni * kN;
      const bool live = r < a.o.M, cut = walk.cut();
      const int b = tl & 1;
      const uint32_t acc = lanes + static_cast<uint32_t>(b * (cols / 2));
      // before the wait: what the results take from memory (lane l has the scales of columns l, l + 32, ...)
      float sx[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = c0 + 32 * j + lane;
        sx[j] = c < c1 && t0 + c < a.o.rows ? a.o.sx[t0 + c] : 0.f;
      }
      const float sw = live ? a.o.sw[r] : 0.f;
      const float bias = live ? i8_bias(a.o, r) : 0.f;
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait_bounded(accf_b + 8 * b, (tl >> 1) & 1));
      tc_fence_after();
      int32_t first = 0, last = 0;
      bool finish = ok;
      if (cut) {
        walk.sharers(&first, &last);
        int32_t* mine = a.part + (static_cast<int64_t>(walk.slot(pair)) * 2 + rank) * (128 * kN);
        if (ok)
          for (int c = c0; c < c1; c += 16) {
            uint32_t v[16];
            tmem_ld16(acc + c, v);
#pragma unroll
            for (int i = 0; i < 16; i += 4)
              *reinterpret_cast<uint4*>(mine + ((c + i) / 4 * 128 + row) * 4) = make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
          }
        __syncwarp();  // the lanes' stores are ordered before lane 0's release
        // (a warp that gave up arrives too, so that the counts are 0 for the next call)
        int32_t* n = a.count + (static_cast<int64_t>(walk.tile - a.d.full) * 2 + rank) * kI8Epi + e;
        int old = 0;
        if (lane == 0) {
          old = atom_add_acq_rel_gpu(n, 1);
          if (old == last - first) *n = 0;
        }
        old = __shfl_sync(0xffffffffu, old, 0);
        __syncwarp();
        finish = ok && old == last - first;
      }
      if (finish) {
        for (int c = c0; c < c1; c += 16) {
          uint32_t v[16];
          tmem_ld16(acc + c, v);
          if (cut)
            for (int p0 = first; p0 <= last; p0 += 4) {  // four pairs' loads in flight
              uint4 q[4][4];
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const int p = p0 + j;
                const bool other = p <= last && p != pair;
                const int32_t* from = a.part + (static_cast<int64_t>(walk.slot(other ? p : pair)) * 2 + rank) * (128 * kN);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  q[j][i] = other ? ld_cg_v4(from + ((c / 4 + i) * 128 + row) * 4) : make_uint4(0, 0, 0, 0);
              }
#pragma unroll
              for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  v[4 * i] += q[j][i].x;
                  v[4 * i + 1] += q[j][i].y;
                  v[4 * i + 2] += q[j][i].z;
                  v[4 * i + 3] += q[j][i].w;
                }
            }
          const int j = (c - c0) >> 4;
          const float sc = __shfl_sync(0xffffffffu, j < 4 ? (j < 2 ? sx[0] : sx[1]) : (j < 6 ? sx[2] : sx[3]), (lane & 15) + 16 * (j & 1));
          float f[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) f[i] = i8_result(static_cast<int32_t>(v[i]), __shfl_sync(0xffffffffu, sc, i), sw, bias);
          const int32_t left = a.o.rows - (t0 + c);
          const int64_t at = static_cast<int64_t>(t0 + c) * a.o.ldy + r;
          if (live && left >= 16) {  // (without a branch per value, so that their chains overlap)
#pragma unroll
            for (int i = 0; i < 16; ++i) i8_store1<kY>(a.o.y, at + i * a.o.ldy, f[i]);
          } else if (live) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (i < left) i8_store1<kY>(a.o.y, at + i * a.o.ldy, f[i]);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(acce0 + 8 * b);
      ++tl;
    }
  }
  if (!ok && lane == 0) atomicCAS(a.err, 0, kDevErrTmaTimeout);
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // neither CTA ends while the other may still signal its barriers or read its memory
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols) : "memory");
  }
}

// ------------------------------------------------------------------------------------------------
// Up to 8 tokens
// ------------------------------------------------------------------------------------------------
constexpr int kI8GemvRows = 8;
constexpr int kI8GemvWarps = 8;

// m16n8k32, both signed, 32-bit sums.
__device__ __forceinline__ void imma16832_s8(int32_t c[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 16 bytes.  Not through the read-only path: the kernel may have started while they were being written.
template <bool kOnce>
__device__ __forceinline__ uint4 i8_ld16(const void* p) {
  uint4 v;
  if constexpr (kOnce)
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  else
    asm volatile("ld.global.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
// 16 bytes of a row from byte k on, those from K on as zeros (rows start on 16 bytes, k too).
template <bool kOnce>
__device__ __forceinline__ uint4 i8_piece(const int8_t* row, int k, int K, bool live) {
  if (live && k + 16 <= K) return i8_ld16<kOnce>(row + k);
  uint32_t v[4] = {0, 0, 0, 0};
  if (live)
    for (int i = 0; i < 16 && k + i < K; ++i) v[i >> 2] |= static_cast<uint32_t>(static_cast<uint8_t>(row[k + i])) << (8 * (i & 3));
  return make_uint4(v[0], v[1], v[2], v[3]);
}

// A fragment's order along K is free as long as both operands have the same: lane 4g + q takes bytes
// 32q .. 32q + 31 of every 128 of rows g and g + 8 (and of token g), which are four k32 steps.
template <int kY>
__global__ void __launch_bounds__(kI8GemvWarps * 32) i8_gemv_kernel(const int8_t* x, int64_t ldx, const int8_t* w,
                                                                   int64_t ldw, int32_t K, const I8Out o) {
  __shared__ int32_t sums[kI8GemvWarps][128];
  griddep_wait();
  griddep_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int r0 = blockIdx.x * 16;
  const bool lo = r0 + g < o.M, hi = r0 + g + 8 < o.M, tok = g < o.rows;
  const int8_t* wl = w + static_cast<int64_t>(r0 + g) * ldw;
  const int8_t* wh = wl + 8 * ldw;
  const int8_t* xr = x + static_cast<int64_t>(g) * ldx;
  int32_t c[4] = {0, 0, 0, 0};
  constexpr int kStep = 128 * kI8GemvWarps;
  for (int k0 = 128 * warp; k0 < K; k0 += 2 * kStep) {
    uint4 a[2][2], b[2][2], t[2][2];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int at = k0 + j * kStep + 32 * q + 16 * h;
        a[j][h] = i8_piece<true>(wl, at, K, lo);
        b[j][h] = i8_piece<true>(wh, at, K, hi);
        t[j][h] = i8_piece<false>(xr, at, K, tok);
      }
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        imma16832_s8(c, a[j][h].x, b[j][h].x, a[j][h].y, b[j][h].y, t[j][h].x, t[j][h].y);
        imma16832_s8(c, a[j][h].z, b[j][h].z, a[j][h].w, b[j][h].w, t[j][h].z, t[j][h].w);
      }
  }
  // c: channel g (0, 1) and g + 8 (2, 3) of tokens 2q and 2q + 1
  sums[warp][(2 * q) * 16 + g] = c[0];
  sums[warp][(2 * q + 1) * 16 + g] = c[1];
  sums[warp][(2 * q) * 16 + g + 8] = c[2];
  sums[warp][(2 * q + 1) * 16 + g + 8] = c[3];
  __syncthreads();
  const int t = threadIdx.x >> 4, r = r0 + (threadIdx.x & 15);
  if (threadIdx.x < 128 && t < o.rows && r < o.M) {
    int32_t s = 0;
#pragma unroll
    for (int i = 0; i < kI8GemvWarps; ++i) s += sums[i][threadIdx.x];
    i8_store1<kY>(o.y, static_cast<int64_t>(t) * o.ldy + r,
                  i8_result(s, o.sx[t], o.sw[r], i8_bias(o, r)));
  }
}

}  // namespace opc
