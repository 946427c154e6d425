// opc_kv_attention.cuh -- attention over the 4-bit paged cache (opc_kv.cuh).
#pragma once

#include "opc_kv.cuh"

namespace opc {

struct KvAttnArgs {
  KvGeom C;
  KvRows B;
  const uint16_t* q;
  uint16_t* out;
  float* lse;
  int64_t ldq, ldo;
  float scale;
  int32_t heads, group;  // group = heads / kv_heads
  int32_t bf16;          // type of q and out
  int32_t vec;           // q and out allow 16-byte accesses at multiples of 8 elements
  int32_t lo_q, hi_q;    // the launch takes the sequences with lo_q to hi_q rows
};

// ------------------------------------------------------------------------------------------------
// Steps: few query rows per sequence (a generated token, a draft).
//
// For one sequence and kv head the rows (query token i, head j of the group; row i * group + j,
// at most 8 * kNT) attend to n keys.  Memory bound: every stored byte is read once, head_dim + 8
// bytes per key for 4 * head_dim * rows operations.  At HBM's rate an SM sub-partition has about 22
// issue slots per 256 stored values, so the codes go to the tensor cores as they are:
//
//   codes     w & 0x000f000f of a 32-bit word of eight codes is a pair of fp16 subnormals
//             code * 2^-24, w & 0x00f000f0 a pair code * 2^-20: exact mma.sync operands for one
//             logical instruction per two values, no conversion.
//   scores    A = 16 keys x 16 dimensions of codes, B = 16 dimensions x 8 rows of q; then
//             score = scale_k * (q . code + zero_k * sum q), the sums in fp32.  q is multiplied by a
//             power of two per row (its largest value near 2^14), and by 1/16 where it meets the
//             2^-20 codes, so fp16 and bf16 queries enter exactly down to 2^-39 of their row's largest.
//   values    A = 16 dimensions x 16 keys (the codes of two keys interleaved by byte permutes),
//             B = 16 keys x 8 rows of weights: the score tile's accumulators are already the
//             transposed fragments that movmatrix turns into B.  A weight carries its key's scale,
//             p = exp2(x - m) * scale_v * 2^-e, and is rounded once to fp16; the zeros' share
//             sum p * zero_v is summed in fp32 from the rounded weights, so the rounding acts on
//             the values themselves (code + zero), not on the all-positive codes.  (What lies 2^-24
//             below the largest product, for which a code counts as 2^-14, is cut: up to 2^-10 code
//             steps of the largest weight of 16 keys.)  Their sums only
//             grow, while the results of long contexts are small differences of them and the zeros'
//             share, and the tensor cores cut what they add: so the share goes into the sums every
//             kKvFold stages, with half of the next stages' expected share in advance, so that they
//             run through 0 and what is cut cancels (131071 keys: results off by 4.2e-4 of their norm
//             without, 3.0e-4 with, 2.8e-4 being the roundings of the weights and of the result).
//   maximum   m and e move only when a score passes m + 7 or a scale 2^(e+8), 8 times the largest so far
//             (one vote per tile): the common tile has no shuffles and no rescaling.  At a move 2^(e+5) lies
//             above the largest scale, so that weights stay below 2^15 and a row's largest is near 2^5
//             (kKvLift): what fp16 cannot hold, 2^-25, is 2^-30 of it (at 2^0 a key with nearly all of the
//             weight and a value near 0 takes n * 2^-25 of the others' mean value away).
//
// The work -- for every sequence and kv head the stages of 128 keys -- is one line that the CTAs
// (persistent, two or three per SM) cut into equal contiguous ranges, whatever the sequences'
// lengths.  A producer warp walks the CTA's range: per item (the part of one sequence and kv head)
// it leaves a description and the item's q rows in one of two slots, and streams the keys through
// a ring (one bulk copy per page, or four where a page is larger than a stage), running ahead of
// the consumers across items.  Four consumer warps take 32 keys of a stage each and merge in shared
// memory at the end of the item.  An item that is a whole sequence and head is written out; else
// its record (m, sum, weighted sums) goes to the workspace -- a CTA has at most two -- and the last
// CTA of that sequence and head to arrive merges the records in order.
//
// Measured: 64 sequences of up to 8192 keys, 64/8 heads of 128: 74 us, 4.0 TB/s; one of 131071 keys, 32/8
// heads: 40 us, 3.6 TB/s; one of 4000 keys: 11 us, latency (lengths, pages, keys, records, one after the
// other).  Nothing is full in the large ones (logic units 48%, issue 49%, memory 60% of what a copy reaches):
// with three CTAs per SM, the registers' limit, a scheduler has three consumer warps to hide the chain of a
// tile's loads, products, exponentials and products behind.
// ------------------------------------------------------------------------------------------------
constexpr int kKvStage = 128;                 // keys per stage, 32 for each consumer
constexpr int kKvStageShift = 7;
constexpr int kKvStepWarps = 4;               // consumers
constexpr int kKvStepThreads = (kKvStepWarps + 1) * 32;
constexpr int kKvMinStages = 2;               // stages per CTA below which fewer CTAs take part
constexpr int kKvFold = 8;                    // stages between two foldings of the zeros' share
constexpr int kKvLift = 5;                    // log2 of a row's largest weight in fp16 when its reference is set
constexpr float kKvNone = -3.402823466e38f;   // the maximum of no keys: below every finite score
constexpr int kKvItemCost = 3;                // what an item costs beside its stages, in stages
__host__ __device__ constexpr int kv_stage_bytes(int hd) { return kKvStage * (hd + 8); }
// CTAs per SM: bounded by the accumulators' registers and the shared memory of a record.  (Heads of 128 with
// two row tiles keep 32 bytes of a thread in local memory: four rows of four heads over 4000 keys 20 us.)
__host__ __device__ constexpr int kv_step_ctas(int hd, int nt) { return hd <= 128 && nt == 1 ? 3 : 2; }
__host__ __device__ constexpr int kv_rec_bytes(int hd, int nt) { return kKvStepWarps * 8 * nt * (hd + 4) * 4; }
__host__ __device__ constexpr int kv_slot_bytes(int hd, int nt) { return 8 * nt * (hd * 2 + 8) + 64; }  // q, its factors, description
__host__ __device__ constexpr int kv_stages(int hd, int nt) {
  const int room = (kv_step_ctas(hd, nt) == 3 ? 75000 : 113000) - kv_rec_bytes(hd, nt) - 2 * kv_slot_bytes(hd, nt) - 512;
  return room / kv_stage_bytes(hd) > 8 ? 8 : room / kv_stage_bytes(hd);
}
__host__ __device__ constexpr int kv_step_smem(int hd, int nt) {
  return kv_stages(hd, nt) * kv_stage_bytes(hd) + kv_rec_bytes(hd, nt) + 2 * kv_slot_bytes(hd, nt) + 512;
}

struct KvSplit {
  float* part;      // [CTAs][2][rows][head_dim + 4]: weighted sums, then m, sum, -, -
  int32_t* count;   // [CTAs], zero between calls
  int32_t rows;
};

__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(x));
  return d;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127

__device__ __forceinline__ float2 unpack_half2(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }

// kW consecutive 32-bit words of shared memory.
template <int kW>
__device__ __forceinline__ void lds_words(uint32_t addr, uint32_t* w) {
  if constexpr (kW % 4 == 0) {
#pragma unroll
    for (int i = 0; i < kW; i += 4) {
      const uint4 v = lds128(addr + 4 * i);
      w[i] = v.x;
      w[i + 1] = v.y;
      w[i + 2] = v.z;
      w[i + 3] = v.w;
    }
  } else if constexpr (kW % 2 == 0) {
#pragma unroll
    for (int i = 0; i < kW; i += 2) {
      const uint2 v = lds64(addr + 4 * i);
      w[i] = v.x;
      w[i + 1] = v.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kW; ++i) w[i] = lds32(addr + 4 * i);
  }
}
__device__ __forceinline__ uint32_t lds16(uint32_t addr) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr));
  return v;
}

// The logarithm of a row's sum T of weights at maximum M (log2 units): ln 2 in two parts, so that the
// product with M adds no rounding.
__device__ __forceinline__ float kv_lse(float M, float T) {
  return T == 0.f ? -INFINITY : fmaf(M, 0.693147182f, fmaf(M, -1.90465421e-9f, logf(T)));
}

// Write 4 dimensions d.. of the result of row `row` (query token row / group, head row % group of
// the kv head): the weighted sums o over the sum T of weights at maximum M (log2 units).
__device__ __forceinline__ void kv_finish_row(const KvAttnArgs& a, int r0, int kvh, int row, int d, const float4& o, float M,
                                              float T) {
  const int i = row / a.group, head = kvh * a.group + row - i * a.group;
  const float inv = T == 0.f ? 0.f : 1.0f / T;  // a row that sees nothing: 0 (a NaN sum stays NaN)
  uint16_t* dst = a.out + static_cast<int64_t>(r0 + i) * a.ldo + head * a.C.hd + d;
  const uint32_t lo = a.bf16 ? pack_halves<true>(o.x * inv, o.y * inv) : pack_halves<false>(o.x * inv, o.y * inv);
  const uint32_t hi = a.bf16 ? pack_halves<true>(o.z * inv, o.w * inv) : pack_halves<false>(o.z * inv, o.w * inv);
  if (a.vec) {
    *reinterpret_cast<uint2*>(dst) = make_uint2(lo, hi);
  } else {
    dst[0] = static_cast<uint16_t>(lo & 0xffffu);
    dst[1] = static_cast<uint16_t>(lo >> 16);
    dst[2] = static_cast<uint16_t>(hi & 0xffffu);
    dst[3] = static_cast<uint16_t>(hi >> 16);
  }
  if (d == 0 && a.lse)
    a.lse[static_cast<int64_t>(r0 + i) * a.heads + head] = kv_lse(M, T);
}

// Merge the records of an item that `n` CTAs share, the first of them `c_first`, in order (record 1
// of the first CTA, record 0 of the others), by the kThreads consumer threads (barrier 1).  Records
// are brought to shared memory, as many as `smem` holds, by asynchronous copies that are all in
// flight together; what they merge to takes the place of the first, and the next ones follow it.
// The code is kept small (one short loop each for the copies and for the sums): it runs once per
// launch and SM, and fetching it is what it costs -- unrolled by 14 and 20 records it took 7 and 15 us
// for the 56 records of 131071 keys over 8 heads.
template <int kHd, int kThreads>
__device__ __forceinline__ void kv_merge_records(const KvAttnArgs& a, const KvSplit& sp, int r0, int kvh, int c_first, int n,
                                                 int R, float* smem, int smem_floats) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int kRec = kHd + 4, kQ = kHd / 4;
  const int size = R * kRec, most = smem_floats / size;  // floats per record here, records at once
  const int64_t stride = static_cast<int64_t>(sp.rows) * kRec;
  const float* part = sp.part + static_cast<int64_t>(c_first) * 2 * stride;
  const uint32_t base = smem_u32(smem);
  // (the first place's (m, sum) alternate between two spots, so that a row's threads need not agree on
  // when to overwrite them)
  for (int c0 = 0, have = 0, spot = 0; c0 < n; have = 1, spot ^= 2) {
    const int m = min(most - have, n - c0);
#pragma unroll 1
    for (int c = warp; c < m; c += kThreads / 32) {
      const float* src = part + (2 * (c0 + c) + (c0 + c == 0)) * stride;
#pragma unroll 1
      for (int x = 4 * lane; x < size; x += 128)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(base + 4 * ((have + c) * size + x)), "l"(src + x) : "memory");
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    named_barrier(1, kThreads);
    c0 += m;
#pragma unroll 1
    for (int i = tid; i < R * kQ; i += kThreads) {
      const int row = i / kQ, d = 4 * (i - row * kQ);
      float M = kKvNone, T = 0.f;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      const float* src = smem + row * kRec;
#pragma unroll 4
      for (int c = 0; c < have + m; ++c) M = fmaxf(M, src[c * size + kHd + (c == 0 ? spot : 0)]);
#pragma unroll 4
      for (int c = 0; c < have + m; ++c) {
        const float2 w = *reinterpret_cast<const float2*>(src + c * size + kHd + (c == 0 ? spot : 0));
        const float4 v = *reinterpret_cast<const float4*>(src + c * size + d);
        const float f = ex2(w.x - M);
        T += f * w.y;
        o.x += f * v.x;
        o.y += f * v.y;
        o.z += f * v.z;
        o.w += f * v.w;
      }
      if (c0 == n) {
        kv_finish_row(a, r0, kvh, row, d, o, M, T);
      } else {
        *reinterpret_cast<float4*>(smem + row * kRec + d) = o;
        if (d == 0) *reinterpret_cast<float2*>(smem + row * kRec + kHd + (spot ^ 2)) = make_float2(M, T);
      }
    }
    named_barrier(1, kThreads);
  }
}

// An item that the CTA shares with others.
struct KvShared {
  int32_t r0, kvh, c_first, contributors, rows;
};

// One thread's arrival for a record: it releases what the CTA's threads wrote before their last
// barrier; the arrival that completes the count has acquired the others' records.
__device__ __forceinline__ void kv_arrive(const KvSplit& sp, const KvShared& sh, int* last) {
  const bool all = atom_add_acq_rel_gpu(sp.count + sh.c_first, 1) == sh.contributors - 1;
  if (all) sp.count[sh.c_first] = 0;
  *last = all;
}

// What the producer tells the consumers of an item.
struct KvItem {
  int32_t n_st;       // stages here; -1: no more items
  int32_t k0, k1;     // keys [k0, k1)
  int32_t seq_end;    // keys the sequence holds (the last row's limit)
  int32_t hidden;     // seq_end - (position of row 0 + 1): row i sees keys below seq_end - hidden + i
  int32_t r0, rows, kvh;
  int32_t contributors, record;
};

// The rows of q as B fragments in an item's slot, from the elements each lane holds (row g of each
// row tile, dimensions q*kHd/4 + 8d + 0..7): multiplication s of code word d meets codes (2s, 2s + 4)
// in the first register, (2s + 1, 2s + 5), which are 16 times larger, in the second and so have to go in
// by the sixteenth.  A row is first multiplied by the power of two that puts its largest near 2^14 (fp16
// ones only upwards): what is rounded then, of elements below 2^-10, lies 2^-39 below the row's largest.
// Behind the fragments, per row: the factor of its scores (log2 units) and the sum of its elements.
template <int kHd, int kNT, bool kBf>
__device__ __forceinline__ void kv_stage_q(const uint4 (&raw)[kNT][kHd / 32], uint32_t slot_s, float scale, int lane) {
  const __half2 sixteenth = __float2half2_rn(0.0625f);
#pragma unroll
  for (int t = 0; t < kNT; ++t) {
    float big = 0.f;
#pragma unroll
    for (int d = 0; d < kHd / 32; ++d) {
      float x[8];
      unpack_halves<kBf>(raw[t][d], x);
#pragma unroll
      for (int e = 0; e < 8; ++e) big = fmaxf(big, fabsf(x[e]));
    }
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
    // |e2| is kept below 100 (a query beyond fp32's reach overflows)
    const int e2 = max(kBf ? -99 : 0, min(99, big > 0.f ? 14 - ((__float_as_int(big) >> 23) - 127) : 0));
    const float up = pow2i(e2);
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int d = 0; d < kHd / 32; ++d) {
      uint32_t w[4] = {raw[t][d].x, raw[t][d].y, raw[t][d].z, raw[t][d].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = pack_halves<false>(half_lo<kBf>(w[i]) * up, half_hi<kBf>(w[i]) * up);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = unpack_half2(w[i]);
        sum[0] += f.x;
        sum[1] += f.y;
      }
      const uint32_t lo0 = prmt(w[0], w[2], 0x5410u), hi0 = prmt(w[0], w[2], 0x7632u);
      const uint32_t lo1 = prmt(w[1], w[3], 0x5410u), hi1 = prmt(w[1], w[3], 0x7632u);
      const __half2 h0 = __hmul2(*reinterpret_cast<const __half2*>(&hi0), sixteenth);
      const __half2 h1 = __hmul2(*reinterpret_cast<const __half2*>(&hi1), sixteenth);
      sts128(slot_s + ((t * (kHd / 32) + d) * 32 + lane) * 16,
             make_uint4(lo0, *reinterpret_cast<const uint32_t*>(&h0), lo1, *reinterpret_cast<const uint32_t*>(&h1)));
    }
    float total = sum[0] + sum[1];
    total += __shfl_xor_sync(0xffffffffu, total, 1);
    total += __shfl_xor_sync(0xffffffffu, total, 2);
    if ((lane & 3) == 0)  // (q carries 2^e2, the codes 2^-24)
      sts64(slot_s + 8 * kNT * kHd * 2 + 8 * (8 * t + (lane >> 2)),
            __float_as_uint(scale * 1.4426950408889634f * pow2i(12 - e2) * 4096.0f), __float_as_uint(total * 0x1p-24f));
  }
}

template <int kHd, int kNT>
__global__ void __launch_bounds__(kKvStepThreads, kv_step_ctas(kHd, kNT))
kv_attention_step_kernel(const KvAttnArgs a, const KvSplit sp) {
  constexpr int kS = kv_stages(kHd, kNT), kStageBytes = kv_stage_bytes(kHd);
  static_assert(kS >= 2, "two stages at least");
  constexpr int kRow = kHd / 2;          // bytes of one key's codes
  constexpr int kKW = kHd / 32;          // words of a key row per lane (4 lanes per row)
  constexpr int kMt = kHd / 16;          // 16-dimension tiles of the values
  constexpr int kRows = 8 * kNT;
  constexpr int kSlotBytes = kv_slot_bytes(kHd, kNT);
  constexpr int kItemAt = kRows * (kHd * 2 + 8);  // of a slot: the fragments of q, (factor, sum) per row, the description
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ int sm_last[2];
  __shared__ volatile int sm_failed;
  __shared__ KvShared sm_shared[2];  // of the CTA's items those that it shares with others
  __shared__ volatile int sm_n_shared;
  float* rec = reinterpret_cast<float*>(smem + kS * kStageBytes);  // [warp][row][kHd + 4]
  unsigned char* slots = smem + kS * kStageBytes + kv_rec_bytes(kHd, kNT);
  const uint32_t ring = smem_u32(smem), bars = smem_u32(slots) + 2 * kSlotBytes;
  const uint32_t full_b = bars, empty_b = bars + 8 * kS, item_b = bars + 16 * kS, free_b = item_b + 16;
  const uint32_t valid_s = free_b + 16;  // [kS] masks of the pieces that are there
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;

  if (tid == 0) {
    sm_failed = 0;
    for (int s = 0; s < kS; ++s) {
      mbar_init(full_b + 8 * s, 1);
      mbar_init(empty_b + 8 * s, kKvStepWarps);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(item_b + 8 * s, 1);
      mbar_init(free_b + 8 * s, kKvStepWarps);
    }
    fence_mbar_init();
  }
  __syncthreads();
  griddep_wait();
  griddep_launch_dependents();
  const int pe = min(a.C.page_size, kKvStage), pe_shift = min(a.C.page_shift, kKvStageShift);  // keys per piece of a stage
  bool ok = true;

  if (warp == kKvStepWarps) {
    // ---------------------------------------------------------------- producer
    const int n_seqs = a.B.n_seqs, kvh_n = a.C.kv_heads;
    const uint64_t once = l2_policy_evict_first();  // every key is read once
    // lane i: sequence s0 + i; its stages (one at least, so that rows without keys are written), 0
    // when the launch does not take it
    int my_r0 = 0, my_q = 0, my_kv = 0, my_n = 0, my_st = 0;
    auto load_seqs = [&](int s0) {
      const int s = s0 + lane;
      my_st = 0;
      if (s < n_seqs) {
        my_r0 = __ldg(a.B.q_start + s);
        const int all = __ldg(a.B.q_start + s + 1) - my_r0;
        my_kv = __ldg(a.B.kv_len + s);
        my_q = min(all, a.B.max_q);  // rows beyond the batch's bound are skipped
        my_n = max(0, min(my_kv, a.B.max_kv));
        my_kv -= all;                // the position of row 0
        if (my_q >= a.lo_q && my_q <= a.hi_q) {
          const bool inside = my_r0 >= 0 && my_r0 <= a.B.n_tokens - my_q;
          if (blockIdx.x == 0 && (all > a.B.max_q || my_kv + all > a.B.max_kv || !inside)) kv_bad_index(a.B);
          if (inside) my_st = max(1, (my_n + kKvStage - 1) >> kKvStageShift);
        }
      }
    };
    // The line of work: a (sequence, kv head) takes its stages and kKvItemCost places before them, for
    // what an item costs beside its stages.  CTA c takes the stages at places [place(c), place(c + 1)).
    uint32_t W = 0;
    for (int s0 = 0; s0 < n_seqs; s0 += 32) {
      load_seqs(s0);
      W += __reduce_add_sync(0xffffffffu, my_st ? my_st + kKvItemCost : 0);
    }
    W *= kvh_n;
    const uint32_t G = min(static_cast<uint32_t>(gridDim.x), max(1u, W / kKvMinStages));
    const uint32_t per = W / G, rest = W - per * G;  // the first `rest` CTAs take one place more
    const auto place_of = [&](uint32_t c) { return c * per + min(c, rest); };
    const auto cta_of = [&](uint32_t x) {
      return static_cast<int>(x < rest * (per + 1) ? x / (per + 1) : rest + (x - rest * (per + 1)) / per);
    };
    const uint32_t c = blockIdx.x;
    uint32_t w = 0, w_end = 0;
    if (c < G) {
      w = place_of(c);
      w_end = place_of(c + 1);
    }
    // the first sequence of the range: base = places before sequence s0 + i
    int s0 = 0, i = 0, n_items = 0, n_shared = 0;
    uint32_t base = 0;
    if (w < w_end) {
      for (;; s0 += 32) {
        if (n_seqs > 32) load_seqs(s0);
        const uint32_t sum = __reduce_add_sync(0xffffffffu, my_st ? my_st + kKvItemCost : 0) * kvh_n;
        if (base + sum > w) break;
        base += sum;
      }
    }
    int st_all = 0;  // stages issued
    while (w < w_end) {
      const uint32_t st = __shfl_sync(0xffffffffu, my_st, i), cost = st ? st + kKvItemCost : 0;
      if (base + cost * kvh_n <= w) {  // the next sequence
        base += cost * kvh_n;
        if (++i == 32) {
          i = 0;
          s0 += 32;
          load_seqs(s0);
        }
        continue;
      }
      const int head = static_cast<int>((w - base) / cost), seq = s0 + i;
      const uint32_t pair0 = base + head * cost + kKvItemCost, pair1 = pair0 + st;  // the places of its stages
      const uint32_t begin = max(w, pair0), end = min(w_end, pair1);
      if (begin >= end) break;  // (only the places before an item's stages: another CTA's item)
      const int r0 = __shfl_sync(0xffffffffu, my_r0, i), q_len = __shfl_sync(0xffffffffu, my_q, i);
      const int n = __shfl_sync(0xffffffffu, my_n, i), pos0 = __shfl_sync(0xffffffffu, my_kv, i);
      const int k0 = static_cast<int>(begin - pair0) * kKvStage, n_st = static_cast<int>(end - begin);
      const int k1 = min(n, k0 + n_st * kKvStage);
      const int is = n_items & 1, R = q_len * a.group;
      const int c_first = cta_of(pair0), contributors = cta_of(pair1 - 1) - c_first + 1;
      if (contributors > 1) {  // (two at most: the items that the range's ends cut)
        if (lane == 0) sm_shared[n_shared] = {r0, head, c_first, contributors, R};
        ++n_shared;
      }
      w = end;
      if (!ok) continue;  // (a wait gave up: only what the CTA shares is still of interest)
      uint4 raw[kNT][kHd / 32];
#pragma unroll
      for (int t = 0; t < kNT; ++t) {
        const int row = 8 * t + g, tok = row / a.group;
        const uint16_t* src = a.q + static_cast<int64_t>(r0 + tok) * a.ldq + (head * a.group + row - tok * a.group) * kHd + q * (kHd / 4);
#pragma unroll
        for (int d = 0; d < kHd / 32; ++d) {
          raw[t][d] = make_uint4(0, 0, 0, 0);
          if (row < R) raw[t][d] = a.vec ? ld_row8<true>(src + 8 * d) : ld_row8<false>(src + 8 * d);
        }
      }
      // Its stages.  Those whose slots are surely free (all of the ring for the first item, one for
      // the others) are requested before q is turned into fragments.
      const int pieces = kKvStage >> pe_shift;                   // per stage
      const int ahead = 32 >> (kKvStageShift - pe_shift);        // stages whose page numbers the warp holds
      const uint32_t piece_bytes = static_cast<uint32_t>(pe) * (kHd + 8);
      int pages = -1;
      const auto issue = [&](int t) {
        if (t % ahead == 0) {  // lane l: the page of piece l from here on
          const int pos = k0 + t * kKvStage + lane * pe;
          pages = -1;
          if (pos < k1) {
            pages = __ldg(a.B.table + seq * a.B.table_stride + (pos >> a.C.page_shift));
            if (static_cast<uint32_t>(pages) >= static_cast<uint32_t>(a.C.n_pages)) {
              kv_bad_index(a.B);
              pages = -1;
            }
          }
        }
        const int slot = st_all % kS;
        if (st_all >= kS && !mbar_wait_bounded(empty_b + 8 * slot, ((st_all / kS) - 1) & 1)) {
          ok = false;
          return;
        }
        const int page = __shfl_sync(0xffffffffu, pages, ((t % ahead) << (kKvStageShift - pe_shift)) + min(lane, pieces - 1));
        const uint32_t mask = __ballot_sync(0xffffffffu, lane < pieces && page >= 0);
        if (lane == 0) {
          asm volatile("st.shared.u32 [%0], %1;" ::"r"(valid_s + 4 * slot), "r"(mask) : "memory");
          mbar_expect_tx(full_b + 8 * slot, piece_bytes * __popc(mask));
        }
        __syncwarp();
        if (lane < pieces && page >= 0) {
          const uint8_t* block = a.C.pages + (static_cast<int64_t>(page) * kvh_n + head) * a.C.head_bytes;
          const uint32_t dst = ring + slot * kStageBytes + lane * piece_bytes, bar = full_b + 8 * slot;
          if (a.C.page_size <= kKvStage) {
            bulk_g2s_hint(dst, block, piece_bytes, bar, once);
          } else {  // part of a larger page
            const int off = (k0 + t * kKvStage) & (a.C.page_size - 1);
            const uint8_t* pairs = block + a.C.page_size * kHd;
            bulk_g2s_hint(dst, block + off * kRow, kKvStage * kRow, bar, once);
            bulk_g2s_hint(dst + kKvStage * kRow, block + (a.C.page_size + off) * kRow, kKvStage * kRow, bar, once);
            bulk_g2s_hint(dst + kKvStage * kHd, pairs + 4 * off, 4 * kKvStage, bar, once);
            bulk_g2s_hint(dst + kKvStage * (kHd + 4), pairs + 4 * (a.C.page_size + off), 4 * kKvStage, bar, once);
          }
        }
        ++st_all;
      };
      const int first = min(n_st, st_all == 0 ? kS : 1);
      for (int t = 0; t < first && ok; ++t) issue(t);
      if (!ok) continue;
      // The item's slot: the description, and q as fragments (once per item here instead of once per
      // consumer; the consumers read them back for every 32 keys, which costs them less than holding
      // them in registers).
      if (n_items >= 2 && !mbar_wait_bounded(free_b + 8 * is, ((n_items >> 1) - 1) & 1)) {
        ok = false;
        continue;
      }
      if (lane == 0) {
        KvItem it;
        it.n_st = n_st;
        it.k0 = k0;
        it.k1 = k1;
        it.seq_end = n;
        it.hidden = n - (pos0 + 1);
        it.r0 = r0;
        it.rows = R;
        it.kvh = head;
        it.contributors = contributors;
        it.record = 2 * c + (static_cast<int>(c) == c_first);
        *reinterpret_cast<KvItem*>(slots + is * kSlotBytes + kItemAt) = it;
      }
      const uint32_t slot_s = smem_u32(slots) + is * kSlotBytes;
      if (a.bf16) kv_stage_q<kHd, kNT, true>(raw, slot_s, a.scale, lane);
      else kv_stage_q<kHd, kNT, false>(raw, slot_s, a.scale, lane);
      __syncwarp();
      if (lane == 0) mbar_arrive(item_b + 8 * is);
      ++n_items;
      for (int t = first; t < n_st && ok; ++t) issue(t);
    }
    // no more items
    const int is = n_items & 1;
    if (ok && n_items >= 2) ok = mbar_wait_bounded(free_b + 8 * is, ((n_items >> 1) - 1) & 1);
    if (ok && lane == 0) {
      reinterpret_cast<KvItem*>(slots + is * kSlotBytes + kItemAt)->n_st = -1;
      mbar_arrive(item_b + 8 * is);
    }
    // every copy has landed before the CTA can end, whatever its consumers did
    for (int t = max(0, st_all - kS); t < st_all; ++t) ok = mbar_wait_bounded(full_b + 8 * (t % kS), (t / kS) & 1) && ok;
    if (lane == 0) {
      if (!ok) atomicCAS(a.B.err, 0, kDevErrTmaTimeout);
      sm_n_shared = n_shared;
    }
    named_barrier(2, kKvStepThreads);
    return;
  }

  // ------------------------------------------------------------------ consumers
  // Score row r of 16 keys is key r ^ ((r >> 1) & 1), an order in which both code reads spread over
  // the banks: rows g and 8 + g are keys perm and 8 + perm, the weights 2q and 2q + 1 the keys pk and
  // pk +- 1.
  const int perm = g ^ ((g >> 1) & 1), pk = 2 * q + (q & 1);
  const int vnext = (q & 1) ? -kRow : kRow;
  // This lane's addresses for the first 16 of the warp's 32 keys of a stage, and the way to the others
  // (the same piece of the stage, or with pages of 16 the next).
  const uint32_t piece = ring + ((32 * warp) >> pe_shift) * pe * (kHd + 8);
  const int place = (32 * warp) & (pe - 1);
  const uint32_t ka = piece + (place + perm) * kRow + q * (kHd / 8);
  const uint32_t pa = piece + pe * kHd + 4 * (place + perm);
  const uint32_t va = piece + (pe + place + pk) * kRow + g * (kHd / 16);
  const uint32_t next_code = pe == 16 ? 16 * (kHd + 8) : 16 * kRow, next_pair = pe == 16 ? 16 * (kHd + 8) : 64;
  int slot = 0, n_shared = 0, n_arrived = 0;
  uint32_t phase = 0;
#pragma unroll 1
  for (int item = 0;; ++item) {
  // (a wait that gives up is told to all four warps, which leave together: none waits at a barrier for another)
  if (!mbar_wait_bounded(item_b + 8 * (item & 1), (item >> 1) & 1)) sm_failed = 1;
  named_barrier(1, kKvStepWarps * 32);  // ... and the last item's records have been read
  if (sm_failed) break;
  if (n_arrived < n_shared) {  // the last item's record is complete
    if (tid == 0) kv_arrive(sp, sm_shared[n_arrived], &sm_last[n_arrived]);
    ++n_arrived;
  }
  const unsigned char* slot_p = slots + (item & 1) * kSlotBytes;
  // (the description is read where it is needed: it stays in its slot until the item's end)
  const volatile KvItem& it = *reinterpret_cast<const volatile KvItem*>(slot_p + kItemAt);
  int left = it.n_st;
  if (left < 0) break;
  int kb = it.k0 + 32 * warp;  // this warp's first key of a stage
  const int k1 = it.k1;
  const uint32_t bq = smem_u32(slot_p) + lane * 16;  // q's fragments
  float cf[kNT][2], qs[kNT][2];  // of rows 2q, 2q + 1: factor of the scores, sum of q
#pragma unroll
  for (int t = 0; t < kNT; ++t) {
    const float4 v = *reinterpret_cast<const float4*>(slot_p + kRows * kHd * 2 + 8 * (8 * t + 2 * q));
    cf[t][0] = v.x;
    qs[t][0] = v.y;
    cf[t][1] = v.z;
    qs[t][1] = v.w;
  }
  // keys that row r sees (none where there is no row)
  const auto limit = [&](int r) { return r < it.rows ? min(it.seq_end, it.seq_end - it.hidden + r / a.group) : 0; };
  // keys below this need no mask: every live row sees them
  const int plain_end = min(k1, it.seq_end - it.hidden);

  float acc[kNT][kMt][4], az[kNT][2], ahead[kNT][2], sum[kNT][2], m[kNT][2];
#pragma unroll
  for (int t = 0; t < kNT; ++t) {
#pragma unroll
    for (int i = 0; i < kMt; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[t][i][c] = 0.f;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      az[t][c] = ahead[t][c] = sum[t][c] = 0.f;
      m[t][c] = kKvNone;
    }
  }
  int ve = -30;             // the weights carry scale_v * 2^-ve
  float vinv = 0x1p30f;
  for (; left > 0; --left, kb += kKvStage) {
    if (!mbar_wait_bounded(full_b + 8 * slot, phase)) {
      sm_failed = 1;
      break;
    }
    const uint32_t so = slot * kStageBytes;
    const uint32_t valid = lds32(valid_s + 4 * slot);
    const bool v0 = (valid >> ((32 * warp) >> pe_shift)) & 1u, v1 = (valid >> ((32 * warp + 16) >> pe_shift)) & 1u;
    if (kb < k1 && (v0 || v1)) {
      const bool whole = kb + 32 <= plain_end && v0 && v1;  // no mask (rows that are not live see garbage)
      uint32_t kp[2][2], vp[2][2];
      float s[2][kNT][4];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t pairs = pa + so + j * next_pair;
        kp[j][0] = lds32(pairs);
        kp[j][1] = lds32(pairs + 32);
        vp[j][0] = lds32(pairs + 4 * pe);
        vp[j][1] = lds32(pairs + 4 * pe + 32);
#pragma unroll
        for (int t = 0; t < kNT; ++t)
#pragma unroll
          for (int c = 0; c < 4; ++c) s[j][t][c] = 0.f;
      }
      // ---- scores
      {
        uint32_t w[2][2][kKW];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          lds_words<kKW>(ka + so + j * next_code, w[j][0]);
          lds_words<kKW>(ka + so + j * next_code + 8 * kRow, w[j][1]);
        }
#pragma unroll
        for (int i = 0; i < kKW; ++i) {
          uint4 b[kNT];
#pragma unroll
          for (int t = 0; t < kNT; ++t) b[t] = lds128(bq + (t * (kHd / 32) + i) * 512);
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t u0 = w[j][0][i] >> (8 * h), u1 = w[j][1][i] >> (8 * h);
              const uint32_t A[4] = {u0 & 0x000f000fu, u1 & 0x000f000fu, u0 & 0x00f000f0u, u1 & 0x00f000f0u};
#pragma unroll
              for (int t = 0; t < kNT; ++t) mma16816(s[j][t], A, h ? b[t].z : b[t].x, h ? b[t].w : b[t].y);
            }
        }
      }
      if (!whole) {  // places past the end, or of a page that does not exist, hold anything
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (kb + 16 * j + perm + 8 * e >= k1 || !(j ? v1 : v0)) kp[j][e] = vp[j][e] = 0;
      }
      float2 vf[2][2];  // (scale, zero) of the values
      float top[kNT][2], vmax = 0.f;
#pragma unroll
      for (int t = 0; t < kNT; ++t) top[t][0] = top[t][1] = -INFINITY;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float2 kf = unpack_half2(kp[j][e]);
          vf[j][e] = unpack_half2(vp[j][e]);
          vmax = fmaxf(vmax, fabsf(vf[j][e].x));
#pragma unroll
          for (int t = 0; t < kNT; ++t)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float x = (s[j][t][2 * e + c] + kf.y * qs[t][c]) * (kf.x * cf[t][c]);
              if (!whole && (kb + 16 * j + perm + 8 * e >= limit(8 * t + 2 * q + c) || !(j ? v1 : v0))) x = -INFINITY;
              s[j][t][2 * e + c] = x;
              top[t][c] = fmaxf(top[t][c], x);
            }
        }
      bool move = vmax * vinv > 256.f;
#pragma unroll
      for (int t = 0; t < kNT; ++t) move |= top[t][0] > m[t][0] + 7.f || top[t][1] > m[t][1] + 7.f;
      if (__any_sync(0xffffffffu, move)) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, o));
        const int e = max(ve, min(17, (__float_as_int(vmax) >> 23) - 126) - kKvLift);  // 2^(e + kKvLift) above every scale so far
        const float drop = pow2i(max(-126, ve - e));
        ve = e;
        vinv = pow2i(-e);
#pragma unroll
        for (int t = 0; t < kNT; ++t)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float x = top[t][c];
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
            const float mn = fmaxf(m[t][c], x), corr = ex2(m[t][c] - mn);
            m[t][c] = mn;
            sum[t][c] *= corr;
            az[t][c] *= corr * drop;
            ahead[t][c] *= corr * drop;
#pragma unroll
            for (int i = 0; i < kMt; ++i) {
              acc[t][i][c] *= corr * drop;
              acc[t][i][c + 2] *= corr * drop;
            }
          }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        // ---- weights
        const float u0 = vf[j][0].x * vinv, u1 = vf[j][1].x * vinv;
        uint32_t bp[kNT][2];
#pragma unroll
        for (int t = 0; t < kNT; ++t) {
          float p[4], w[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            p[c] = ex2(s[j][t][c] - m[t][c & 1]);
            w[c] = p[c] * (c < 2 ? u0 : u1);
            if (!whole && s[j][t][c] == -INFINITY) w[c] = 0.f;  // (a hidden key's scale may be NaN)
          }
          sum[t][0] += p[0] + p[2];
          sum[t][1] += p[1] + p[3];
          const uint32_t h0 = pack_halves<false>(w[0], w[1]), h1 = pack_halves<false>(w[2], w[3]);
          const float2 r0 = unpack_half2(h0), r1 = unpack_half2(h1);
          az[t][0] += r0.x * vf[j][0].y + r1.x * vf[j][1].y;
          az[t][1] += r0.y * vf[j][0].y + r1.y * vf[j][1].y;
          bp[t][0] = movmatrix_trans(h0);
          bp[t][1] = movmatrix_trans(h1);
        }
        // ---- values: half word h (4 dimensions) of the lane's kHd/8 dimensions, of four keys
        const uint32_t v0a = va + so + j * next_code, v1a = v0a + vnext;
        constexpr int kH = kHd / 32;  // half words per key
        uint32_t lo[kH], hi[kH];      // (key pk | key pk +- 1) of the first and the second eight keys
        if constexpr (kH % 2 == 0) {
          uint32_t x[4][kH / 2];
          lds_words<kH / 2>(v0a, x[0]);
          lds_words<kH / 2>(v1a, x[1]);
          lds_words<kH / 2>(v0a + 8 * kRow, x[2]);
          lds_words<kH / 2>(v1a + 8 * kRow, x[3]);
#pragma unroll
          for (int h = 0; h < kH; ++h) {
            const uint32_t sel = (h & 1) ? 0x7632u : 0x5410u;
            lo[h] = prmt(x[0][h >> 1], x[1][h >> 1], sel);
            hi[h] = prmt(x[2][h >> 1], x[3][h >> 1], sel);
          }
        } else {
#pragma unroll
          for (int h = 0; h < kH; ++h) {
            lo[h] = lds16(v0a + 2 * h) | (lds16(v1a + 2 * h) << 16);
            hi[h] = lds16(v0a + 8 * kRow + 2 * h) | (lds16(v1a + 8 * kRow + 2 * h) << 16);
          }
        }
#pragma unroll
        for (int h = 0; h < kH; ++h)
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            const uint32_t u = lo[h] >> (8 * z), v = hi[h] >> (8 * z);
            const uint32_t A[4] = {u & 0x000f000fu, u & 0x00f000f0u, v & 0x000f000fu, v & 0x00f000f0u};
#pragma unroll
            for (int t = 0; t < kNT; ++t) mma16816(acc[t][2 * h + z], A, bp[t][0], bp[t][1]);
          }
      }
      if ((left & (kKvFold - 1)) == 0) {
#pragma unroll
        for (int t = 0; t < kNT; ++t)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float z = az[t][c];
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
            const float half = 0.5f * (z + ahead[t][c]);  // of these stages' share, now for the next ones'
            ahead[t][c] = half;
            az[t][c] = g == 0 ? -half : 0.f;
            z += half;
#pragma unroll
            for (int i = 0; i < kMt; ++i) {
              acc[t][i][c] += z * 0x1p-24f;
              acc[t][i][c + 2] += z * 0x1p-20f;
            }
          }
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(empty_b + 8 * slot);
    if (++slot == kS) {
      slot = 0;
      phase ^= 1u;
    }
  }
  // ------------------------------------------------------------------ merge of the four warps
  constexpr int kRec = kHd + 4;
  const int R = it.rows;
  const float back = pow2i(ve);
#pragma unroll
  for (int t = 0; t < kNT; ++t) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        sum[t][c] += __shfl_xor_sync(0xffffffffu, sum[t][c], o);
        az[t][c] += __shfl_xor_sync(0xffffffffu, az[t][c], o);
      }
      const int row = 8 * t + 2 * q + c;
      float* dst = rec + (warp * kRows + row) * kRec;
      if (row < R) {
#pragma unroll
        for (int i = 0; i < kMt; ++i) {
          // tile 2h + z, lane g: dimensions g * kHd/8 + 4h + 2z, + 1
          float2 v;
          v.x = (acc[t][i][c] * 0x1p24f + az[t][c]) * back;
          v.y = (acc[t][i][c + 2] * 0x1p20f + az[t][c]) * back;
          *reinterpret_cast<float2*>(dst + g * (kHd / 8) + 2 * i) = v;
        }
        if (g == 0) {
          dst[kHd] = m[t][c];
          dst[kHd + 1] = sum[t][c];
        }
      }
    }
  }
  named_barrier(1, kKvStepWarps * 32);
  const int r0 = it.r0, kvh = it.kvh;
  const bool single = it.contributors == 1;
  float* part = sp.part + static_cast<int64_t>(it.record) * sp.rows * kRec;
  __syncwarp();
  if (lane == 0) mbar_arrive(free_b + 8 * (item & 1));
  constexpr int kQ = kHd / 4;  // float4 columns of a row
  for (int i = tid; i < R * kQ; i += kKvStepWarps * 32) {
    const int row = i / kQ, d = 4 * (i - row * kQ);
    float M = kKvNone, T = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float mw[kKvStepWarps];
#pragma unroll
    for (int w = 0; w < kKvStepWarps; ++w) {
      mw[w] = rec[(w * kRows + row) * kRec + kHd];
      M = fmaxf(M, mw[w]);
    }
#pragma unroll
    for (int w = 0; w < kKvStepWarps; ++w) {
      const float f = ex2(mw[w] - M);
      const float* src = rec + (w * kRows + row) * kRec;
      const float4 v = *reinterpret_cast<const float4*>(src + d);
      T += f * src[kHd + 1];
      o.x += f * v.x;
      o.y += f * v.y;
      o.z += f * v.z;
      o.w += f * v.w;
    }
    if (single) {
      kv_finish_row(a, r0, kvh, row, d, o, M, T);
    } else {
      *reinterpret_cast<float4*>(part + row * kRec + d) = o;
      if (d == 0) *reinterpret_cast<float2*>(part + row * kRec + kHd) = make_float2(M, T);
    }
  }
  n_shared += !single;
  }
  // Merges come after the loop: in it their registers would push the tile's to local memory
  // (attention over 131071 keys 44 -> 68 us).
  named_barrier(2, kKvStepThreads);  // sm_shared and sm_failed are final; rec may be overwritten
  if (sm_failed) {  // arrive for every shared item all the same: the counts go back to zero for the calls to come
    if (tid == 0) {
      atomicCAS(a.B.err, 0, kDevErrTmaTimeout);
      for (int i = n_arrived; i < sm_n_shared; ++i) kv_arrive(sp, sm_shared[i], &sm_last[i]);
    }
    return;
  }
  if (tid == 0 && n_arrived < n_shared) kv_arrive(sp, sm_shared[n_arrived], &sm_last[n_arrived]);
  named_barrier(1, kKvStepWarps * 32);
  for (int i = 0; i < n_shared; ++i) {
    if (!sm_last[i]) continue;
    const KvShared& sh = sm_shared[i];
    kv_merge_records<kHd, kKvStepWarps * 32>(a, sp, sh.r0, sh.kvh, sh.c_first, sh.contributors, sh.rows,
                                             reinterpret_cast<float*>(smem), (kS * kStageBytes + kv_rec_bytes(kHd, kNT)) / 4);
  }
}

}  // namespace opc
