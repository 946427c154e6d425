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
//                 Persistent: pairs take tiles in turn, 8 channel tiles at a time, so that what they
//                 read stays in L2.  Where there are few tiles, a cluster of 2 to 4 pairs shares one
//                 along K and adds its sums through distributed shared memory.
//                   warp 0     TMA
//                   warp 1     tensor memory; in a pair's first CTA it issues the MMAs
//                   warps 2-9  epilogue: two warps per TMEM lane quarter, half of the columns each;
//                              it reads one accumulator while the MMAs fill the other
//                 Measured (device time in a graph, weights from memory): 8191 tokens 4096 -> 28672 581 us,
//                 3.31 PFLOP/s at the clocks of a short run; in a loop the power limit brings the clock to
//                 1.27 GHz, of whose 3.07 PFLOP/s it reaches 2.87.  512 tokens 4096 -> 6144 14.7 us: 72 of 74
//                 pairs for one tile of 192 tokens, 8 us of MMAs behind 4 us of launch and first loads,
//                 then 2 us of results.  24 tokens 14336 -> 4096 15.2 us, 3.9 TB/s: the reading of W at
//                 6.8 TB/s, behind the same and the exchange of sums.
// i8_gemv_kernel  few tokens: mma.sync fragments straight from global memory; bound by the reading of W.
//                 One token 4096 -> 28672 20.6 us, 5.7 TB/s; 4096 -> 128256 77 us, 6.8 TB/s.  (tcgen05
//                 would wait for tensor memory, barriers and a transposed staging of W: 8.7 us instead of
//                 5.3 for 4096 -> 4096.)
#pragma once

#include <cuda.h>

#include "opc_i8_plan.h"
#include "opc_i8_rows.cuh"
#include "opc_tcgen05.cuh"

namespace opc {

constexpr int kI8Epi = 8;                     // epilogue warps of a CTA
constexpr int kI8Threads = 64 + 32 * kI8Epi;

struct I8Out {
  const float *sx, *sw;
  const void* bias;
  void* y;
  int64_t ldy;
  int32_t rows, M, bias_type;
};

struct I8GemmArgs {
  I8Out o;
  I8Deal d;
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
__device__ __forceinline__ uint4 ld_cluster_v4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared::cluster.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
// The asynchronous operations are issued by one lane (`leader`) of a converged warp: outside a divergent
// branch their operands can stay in uniform registers (8191 tokens 4096 -> 28672: 725 -> 647 us).
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
__device__ __forceinline__ void umma_commit_pair(uint32_t leader, uint32_t bar, uint32_t first) {
  asm volatile(
      "{\n .reg .pred l;\n setp.ne.b32 l, %2, 0;\n"
      " @l tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n}\n" ::"r"(bar),
      "h"(static_cast<uint16_t>(3u << first)), "r"(leader)
      : "memory");
}
// kind::i8, A and B signed, D 32-bit integers, both K-major, 256 channels x n tokens.
__device__ __forceinline__ uint32_t i8_idesc(int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(256 >> 4) << 24);
}

// One pair's work: tile after tile, and the stages of each that are the pair's.
struct I8Walk {
  const I8Deal& d;
  int32_t next, step_, tile, k0, k1;
  // `unit`: the pair, or with split > 1 the cluster, of `units`; `part`: the pair's place in its cluster
  __device__ I8Walk(const I8Deal& deal, int32_t unit, int32_t units, int32_t part) : d(deal), next(unit), step_(units), tile(0) {
    k0 = i8_cut(d, part);
    k1 = i8_cut(d, part + 1);
  }
  __device__ bool step() {
    if (next >= d.m_tiles * d.n_tiles) return false;
    tile = next;
    next += step_;
    return true;
  }
  __device__ void place(int32_t* mi, int32_t* ni) const { i8_place(d, tile, mi, ni); }
};

// kNum results of one channel, for tokens t, t + 1, ... of which `left` exist.
template <int kY, int kNum>
__device__ __forceinline__ void i8_store_column(const I8Out& o, const float (&f)[kNum], int32_t t, int32_t r, int32_t left) {
  const int64_t at = static_cast<int64_t>(t) * o.ldy + r;
  if (left >= kNum) {  // (without a branch per value, so that their chains overlap: 256 tokens of a tile 6 -> 2 us)
#pragma unroll
    for (int i = 0; i < kNum; ++i) i8_store1<kY>(o.y, at + i * o.ldy, f[i]);
  } else {
#pragma unroll
    for (int i = 0; i < kNum; ++i)
      if (i < left) i8_store1<kY>(o.y, at + i * o.ldy, f[i]);
  }
}

// tw: w [M][K], box 128 bytes x 128 channels; tx: x [rows][K], box 128 bytes x tile_n / 2 tokens; both
// with the 128-byte swizzle, zeros beyond the edges.  Clusters of 2 * split CTAs; dynamic shared memory for
// the stages, which later hold a split tile's sums, and the barriers.
template <int kY>
__global__ void __launch_bounds__(kI8Threads, 1)
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
  const uint32_t in_cluster = cluster_rank(), first = in_cluster & ~1u, rank = in_cluster & 1u;  // `first`: the pair's first CTA
  const int split = a.d.split;
  const int cols = kN <= 32 ? 64 : kN <= 64 ? 128 : kN <= 128 ? 256 : 512;  // two accumulators

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
  __syncthreads();
  cluster_sync();  // every CTA's barriers are set up
  griddep_wait();  // everything before has ended: its tensor memory is free again, its results are there
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_slot), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();  // (a pair's first MMA waits for both CTAs' loads, which come after this in either)
  tc_fence_after();
  griddep_launch_dependents();  // every CTA that has come this far holds its tensor memory
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tmem_slot_ptr);
  bool ok = true;
  const int quarter = warp & 3, half = (warp - 2) >> 2;  // epilogue warps: TMEM lanes, and which half of the columns
  const int row = 32 * quarter + lane;                   // channel of the CTA's 128 = TMEM lane
  const uint32_t lanes = tmem + (static_cast<uint32_t>(32 * quarter) << 16);
  I8Walk walk(a.d, static_cast<int>(blockIdx.x) / (2 * split), static_cast<int>(gridDim.x) / (2 * split), static_cast<int>(first >> 1));

  if (warp == 0) {
    // ---------------------------------------------------------------- TMA
    const uint32_t leader = elect_leader();
    const uint32_t full0 = map_to_rank(full_b, first);  // the first CTA's MMA warp waits for both CTAs' loads
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
          umma_commit_pair(leader, empty_b + 8 * st, first);
          if (++st == stages) {
            st = 0;
            par ^= 1;
          }
        }
        if (!ok) break;
        umma_commit_pair(leader, accf_b + 8 * b, first);
        ++tl;
      }
      // no MMA of this pair is in flight past this point
      if (leader) asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(drain_b) : "memory");
      mbar_wait_bounded(drain_b, 0);
    }
  } else {
    // ---------------------------------------------------------------- epilogue
    const uint32_t acce0 = map_to_rank(acce_b, first);
    const int c0 = half * (kN / 2), c1 = c0 + kN / 2;  // this warp's columns, 16 at a time
    int tl = 0;
    while (walk.step()) {
      int32_t mi, ni;
      walk.place(&mi, &ni);
      const int32_t r = mi * 256 + static_cast<int32_t>(rank) * 128 + row, t0 = ni * kN;
      const bool live = r < a.o.M;
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
      if (ok) {
        for (int c = c0; c < c1; c += 16) {
          uint32_t v[16];
          tmem_ld16(acc + c, v);
          if (split > 1) {  // (every MMA of the pair has ended: the stages are free)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              sts128(base + ((c / 4 + i) * 128 + row) * 16, make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]));
          } else {
            const int j = (c - c0) >> 4;
            const float sc = __shfl_sync(0xffffffffu, j < 4 ? (j < 2 ? sx[0] : sx[1]) : (j < 6 ? sx[2] : sx[3]), (lane & 15) + 16 * (j & 1));
            float f[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) f[i] = i8_result(static_cast<int32_t>(v[i]), __shfl_sync(0xffffffffu, sc, i), sw, bias);
            if (live) i8_store_column<kY>(a.o, f, t0 + c, r, a.o.rows - (t0 + c));
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
  cluster_sync();  // (split: every pair's sums lie in shared memory)
  if (split > 1) {
    if (warp >= 2) {
      // The pair's share of the columns, 8 at a time for each warp, from all pairs of the cluster.
      int32_t mi, ni;
      walk.place(&mi, &ni);
      const int32_t r = mi * 256 + static_cast<int32_t>(rank) * 128 + row, t0 = ni * kN;
      const bool live = r < a.o.M;
      const float sw = live ? a.o.sw[r] : 0.f;
      const float bias = live ? i8_bias(a.o, r) : 0.f;
#pragma unroll 2
      for (int c = 8 * (static_cast<int>(first) + half); c < kN; c += 16 * split) {
        const int32_t t = t0 + c;
        const float sx = t + (lane & 7) < a.o.rows ? a.o.sx[t + (lane & 7)] : 0.f;
        uint4 q[4][2];
#pragma unroll
        for (int p = 0; p < 4; ++p)  // (all under way before the first is used)
          if (p < split) {
            const uint32_t from = map_to_rank(base, 2 * p + rank) + ((c / 4) * 128 + row) * 16;
            q[p][0] = ld_cluster_v4(from);
            q[p][1] = ld_cluster_v4(from + 128 * 16);
          }
        uint32_t v[8] = {q[0][0].x, q[0][0].y, q[0][0].z, q[0][0].w, q[0][1].x, q[0][1].y, q[0][1].z, q[0][1].w};
#pragma unroll
        for (int p = 1; p < 4; ++p)
          if (p < split) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              v[4 * h] += q[p][h].x;
              v[4 * h + 1] += q[p][h].y;
              v[4 * h + 2] += q[p][h].z;
              v[4 * h + 3] += q[p][h].w;
            }
          }
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = i8_result(static_cast<int32_t>(v[i]), __shfl_sync(0xffffffffu, sx, i), sw, bias);
        if (live) i8_store_column<kY>(a.o, f, t, r, a.o.rows - t);
      }
    }
    __syncthreads();
    cluster_sync();  // nobody ends while another reads its sums
  }
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols) : "memory");
  }
}

// ------------------------------------------------------------------------------------------------
// Few tokens
// ------------------------------------------------------------------------------------------------
constexpr int kI8GemvRows = 8;

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
template <int kY, int kTok, int kWarps, int kDeep>
__global__ void __launch_bounds__(kWarps * 32) i8_gemv_kernel(const int8_t* x, int64_t ldx, const int8_t* w, int64_t ldw, int32_t K, const I8Out o) {
  __shared__ int32_t sums[kWarps][kTok * 128];
  griddep_wait();
  griddep_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int r0 = blockIdx.x * 16;
  const bool lo = r0 + g < o.M, hi = r0 + g + 8 < o.M;
  const int8_t* wl = w + static_cast<int64_t>(r0 + g) * ldw;
  const int8_t* wh = wl + 8 * ldw;
  const int8_t* xr = x + static_cast<int64_t>(g) * ldx;
  int32_t c[kTok][4] = {};
  constexpr int kStep = 128 * kWarps;
  for (int k0 = 128 * warp; k0 < K; k0 += kDeep * kStep) {
    uint4 a[kDeep][2], b[kDeep][2];  // the weights of kDeep steps are under way together; tokens come from L1
#pragma unroll
    for (int j = 0; j < kDeep; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int at = k0 + j * kStep + 32 * q + 16 * h;
        a[j][h] = i8_piece<true>(wl, at, K, lo);
        b[j][h] = i8_piece<true>(wh, at, K, hi);
      }
#pragma unroll
    for (int j = 0; j < kDeep; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int n = 0; n < kTok; ++n) {
          const uint4 t = i8_piece<false>(xr + 8 * n * ldx, k0 + j * kStep + 32 * q + 16 * h, K, g + 8 * n < o.rows);
          imma16832_s8(c[n], a[j][h].x, b[j][h].x, a[j][h].y, b[j][h].y, t.x, t.y);
          imma16832_s8(c[n], a[j][h].z, b[j][h].z, a[j][h].w, b[j][h].w, t.z, t.w);
        }
      }
  }
  // c: channel g (0, 1) and g + 8 (2, 3) of tokens 2q and 2q + 1
#pragma unroll
  for (int n = 0; n < kTok; ++n) {
    int32_t* to = sums[warp] + 128 * n;
    to[(2 * q) * 16 + g] = c[n][0];
    to[(2 * q + 1) * 16 + g] = c[n][1];
    to[(2 * q) * 16 + g + 8] = c[n][2];
    to[(2 * q + 1) * 16 + g + 8] = c[n][3];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kTok * 128; i += kWarps * 32) {
    const int t = i >> 4, r = r0 + (i & 15);
    if (t >= o.rows || r >= o.M) continue;
    int32_t s = 0;
#pragma unroll
    for (int j = 0; j < kWarps; ++j) s += sums[j][i];
    i8_store1<kY>(o.y, static_cast<int64_t>(t) * o.ldy + r, i8_result(s, o.sx[t], o.sw[r], i8_bias(o, r)));
  }
}

}  // namespace opc
