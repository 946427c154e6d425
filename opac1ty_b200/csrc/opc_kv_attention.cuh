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

constexpr int kKvPlainThreads = 128;
constexpr int kKvPlainTile = 128;

__device__ __forceinline__ float ld_elem(const uint16_t* p, int bf16) {
  const uint32_t w = *p;
  return bf16 ? half_lo<true>(w) : half_lo<false>(w);
}
__device__ __forceinline__ void st_elem(uint16_t* p, float v, int bf16) {
  *p = bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
}

// One CTA per row and query head.  The visible positions are walked in tiles with a running
// maximum and sum: a thread takes one position's score, then one dimension's (or two dimensions')
// weighted sum of the values.
__global__ void __launch_bounds__(kKvPlainThreads) kv_attention_plain_kernel(const KvAttnArgs a) {
  __shared__ float sq[kKvMaxHd], sw[kKvPlainTile], red[kKvPlainThreads / 32];
  __shared__ int sm_seq, sm_pos;
  const int r = blockIdx.x, head = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (warp == 0) {
    const KvRowPlace p = kv_row_place(a.B, r, lane);
    if (lane == 0) {
      sm_seq = p.seq;
      sm_pos = p.pos;
    }
  }
  const int hd = a.C.hd;
  for (int d = tid; d < hd; d += kKvPlainThreads) sq[d] = ld_elem(a.q + r * a.ldq + head * hd + d, a.bf16) * a.scale;
  __syncthreads();
  const int seq = sm_seq;
  if (seq < 0) return;
  const int r0 = __ldg(a.B.q_start + seq), q_all = __ldg(a.B.q_start + seq + 1) - r0, q_len = min(q_all, a.B.max_q);
  if (q_len < a.lo_q || q_len > a.hi_q) return;
  if (r - r0 >= a.B.max_q) {
    if (tid == 0) kv_bad_index(a.B);
    return;
  }
  const int n = min(min(sm_pos + 1, a.B.max_kv), a.B.max_pages << a.C.page_shift);  // visible positions
  const int kvh = head / a.group, codes = a.C.page_size * (hd >> 1);
  float M = -INFINITY, T = 0.f, acc[2] = {0.f, 0.f};
  for (int t0 = 0; t0 < n; t0 += kKvPlainTile) {
    const int pos = t0 + tid;
    float s = -INFINITY, vs = 0.f, vz = 0.f;
    if (pos < n) {
      const int64_t place = kv_page_offset(a.C, a.B, seq, pos >> a.C.page_shift);
      if (place >= 0) {
        const uint8_t* block = a.C.pages + place + kvh * a.C.head_bytes;
        const int off = pos & (a.C.page_size - 1);
        const uint32_t pair = *reinterpret_cast<const uint32_t*>(block + 2 * codes + 4 * off);
        const uint32_t* w = reinterpret_cast<const uint32_t*>(block + off * (hd >> 1));
        float dot = 0.f;
        for (int i = 0; i < (hd >> 3); ++i)
          for (int e = 0; e < 8; ++e) dot += sq[8 * i + e] * (static_cast<float>((w[i] >> (4 * e)) & 15u) + half_hi<false>(pair));
        s = dot * half_lo<false>(pair);
      }
    }
    float m = s;
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) red[warp] = m;
    __syncthreads();
    float Mn = M;
    for (int i = 0; i < kKvPlainThreads / 32; ++i) Mn = fmaxf(Mn, red[i]);
    // (a NaN score leaves the maximum alone and turns the sums to NaN; nothing visible yet: no scale)
    const float base = Mn == -INFINITY ? 0.f : Mn, corr = M == -INFINITY ? 0.f : expf(M - base);
    sw[tid] = s == -INFINITY ? 0.f : expf(s - base);
    M = Mn;
    __syncthreads();
    T *= corr;
    acc[0] *= corr;
    acc[1] *= corr;
    const int tn = min(kKvPlainTile, n - t0);
    for (int j = 0; j < tn; ++j) {
      const float w = sw[j];
      T += w;
      const int p = t0 + j;
      const int page = __ldg(a.B.table + seq * a.B.table_stride + (p >> a.C.page_shift));
      if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(a.C.n_pages)) continue;
      const uint8_t* block = a.C.pages + (static_cast<int64_t>(page) * a.C.kv_heads + kvh) * a.C.head_bytes;
      const int off = p & (a.C.page_size - 1);
      const uint32_t pair = *reinterpret_cast<const uint32_t*>(block + 2 * codes + 4 * (a.C.page_size + off));
      vs = half_lo<false>(pair);
      vz = half_hi<false>(pair);
      for (int i = 0; i < 2; ++i) {
        const int d = tid + i * kKvPlainThreads;
        if (d < hd) {
          const uint32_t b = block[codes + off * (hd >> 1) + (d >> 1)];
          acc[i] += w * (vs * (static_cast<float>((b >> (4 * (d & 1))) & 15u) + vz));
        }
      }
    }
    __syncthreads();
  }
  const bool none = T == 0.f;
  for (int i = 0; i < 2; ++i) {
    const int d = tid + i * kKvPlainThreads;
    if (d < hd) st_elem(a.out + r * a.ldo + head * hd + d, none ? 0.f : acc[i] / T, a.bf16);
  }
  if (tid == 0 && a.lse) a.lse[static_cast<int64_t>(r) * a.heads + head] = none ? -INFINITY : M + logf(T);
}

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
//             2^-20 codes, so fp16 and bf16 queries enter exactly.
//   values    A = 16 dimensions x 16 keys (the codes of two keys interleaved by byte permutes),
//             B = 16 keys x 8 rows of weights: the score tile's accumulators are already the
//             transposed fragments that movmatrix turns into B.  A weight carries its key's scale,
//             p = exp2(x - m) * scale_v * 2^-e, and is rounded once to fp16; the zeros' share
//             sum p * zero_v is summed in fp32 from the rounded weights, so the rounding acts on
//             the values themselves (code + zero), not on the all-positive codes.
//   maximum   m and e move only when a score passes m + 8 or a scale 2^(e+5) (one vote per tile):
//             weights stay below 2^13, and the common tile has no shuffles and no rescaling.
//
// A CTA takes one chunk of the keys: a producer warp brings 64 keys per stage (one bulk copy per
// page and head, or four where a page is larger than a stage) into a ring, four consumer warps take
// 16 keys each.  Their results are merged in shared memory; where a sequence has several chunks
// the records (m, sum, weighted sums) go to the workspace and the last CTA to arrive merges them in
// order.
// ------------------------------------------------------------------------------------------------
constexpr int kKvStage = 64;                  // keys per stage
constexpr int kKvStepWarps = 4;               // consumers
constexpr int kKvStepThreads = (kKvStepWarps + 1) * 32;
constexpr int kKvCounters = 65536;            // (sequence, kv head) pairs that may be split
__host__ __device__ constexpr int kv_stage_bytes(int hd) { return kKvStage * (hd + 8); }
// As many stages as fit four CTAs into an SM's shared memory, 3 to 10.
__host__ __device__ constexpr int kv_stages(int hd) {
  return 53000 / kv_stage_bytes(hd) > 10 ? 10 : 53000 / kv_stage_bytes(hd);
}
__host__ __device__ constexpr int kv_step_smem(int hd) { return kv_stages(hd) * kv_stage_bytes(hd) + 256; }

struct KvSplit {
  int32_t chunk;    // keys per CTA, a multiple of kKvStage
  int32_t chunks;   // records per (sequence, kv head) in the workspace
  int32_t rows;     // rows of a record
  float* part;      // [n_seqs][kv_heads][chunks][rows][head_dim + 4]: weighted sums, then m, sum, -, -
  int32_t* count;   // [n_seqs * kv_heads], zero between calls
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
    a.lse[static_cast<int64_t>(r0 + i) * a.heads + head] = T == 0.f ? -INFINITY : M * 0.6931471805599453f + logf(T);
}

// The CTA has written its record; the last one of its (sequence, kv head) merges all of them, in
// order, and leaves the count at 0.  Called by the kThreads consumer threads, barrier 1; smem holds
// chunks * R + R float2.
template <int kHd, int kThreads>
__device__ __forceinline__ void kv_merge_chunks(const KvAttnArgs& a, const KvSplit& sp, int r0, int kvh, int64_t pair_id,
                                                int n_chunks, int R, unsigned char* smem, int* sm_last) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  __threadfence();
  named_barrier(1, kThreads);
  if (tid == 0) *sm_last = atom_add_acq_rel_gpu(sp.count + pair_id, 1) == n_chunks - 1;
  named_barrier(1, kThreads);
  if (!*sm_last) return;
  __threadfence();
  if (tid == 0) sp.count[pair_id] = 0;
  constexpr int kRec = kHd + 4;
  const int64_t stride = static_cast<int64_t>(sp.rows) * kRec;
  const float* part = sp.part + pair_id * sp.chunks * stride;
  float2* f = reinterpret_cast<float2*>(smem);  // [row][chunk]: (m, sum), then (factor, sum)
  float2* total = f + R * n_chunks;             // [row]: (M, T)
  for (int i = tid; i < R * n_chunks; i += kThreads) {
    const int row = i / n_chunks, c = i - row * n_chunks;
    f[i] = __ldcg(reinterpret_cast<const float2*>(part + c * stride + row * kRec + kHd));
  }
  named_barrier(1, kThreads);
  for (int row = warp; row < R; row += kThreads / 32) {
    float M = -1e30f, T = 0.f;
    for (int c = lane; c < n_chunks; c += 32) M = fmaxf(M, f[row * n_chunks + c].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    for (int c = lane; c < n_chunks; c += 32) {
      const float w = ex2(f[row * n_chunks + c].x - M);
      T += w * f[row * n_chunks + c].y;
      f[row * n_chunks + c].x = w;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) T += __shfl_xor_sync(0xffffffffu, T, o);
    if (lane == 0) total[row] = make_float2(M, T);
  }
  named_barrier(1, kThreads);
  constexpr int kQ = kHd / 4;
  for (int i = tid; i < R * kQ; i += kThreads) {
    const int row = i / kQ, d = 4 * (i - row * kQ);
    const float* src = part + row * kRec + d;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int c = 0; c < n_chunks; ++c) {
      const float4 v = __ldcg(reinterpret_cast<const float4*>(src + c * stride));
      const float w = f[row * n_chunks + c].x;
      o.x += w * v.x;
      o.y += w * v.y;
      o.z += w * v.z;
      o.w += w * v.w;
    }
    kv_finish_row(a, r0, kvh, row, d, o, total[row].x, total[row].y);
  }
}

template <int kHd, int kNT>
__global__ void __launch_bounds__(kKvStepThreads) kv_attention_step_kernel(const KvAttnArgs a, const KvSplit sp) {
  constexpr int kS = kv_stages(kHd), kStageBytes = kv_stage_bytes(kHd);
  constexpr int kRow = kHd / 2;          // bytes of one key's codes
  constexpr int kKW = kHd / 32;          // words of a key row per lane (4 lanes per row)
  constexpr int kMt = kHd / 16;          // 16-dimension tiles of the values
  constexpr int kRows = 8 * kNT;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ int sm_last;
  const uint32_t ring = smem_u32(smem), bars = ring + kS * kStageBytes;
  const uint32_t full_b = bars, empty_b = bars + 8 * kS, valid_s = bars + 16 * kS;  // valid_s: [kS] masks
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
  const int chunk = blockIdx.x, kvh = blockIdx.y, seq = blockIdx.z;

  if (tid == 0) {
    for (int s = 0; s < kS; ++s) {
      mbar_init(full_b + 8 * s, 1);
      mbar_init(empty_b + 8 * s, kKvStepWarps);
    }
    fence_mbar_init();
  }
  griddep_wait();
  griddep_launch_dependents();
  const int r0 = __ldg(a.B.q_start + seq), q_all = __ldg(a.B.q_start + seq + 1) - r0, kv_all = __ldg(a.B.kv_len + seq);
  const int q_len = min(q_all, a.B.max_q);  // rows beyond the batch's bound are skipped
  if (q_len < a.lo_q || q_len > a.hi_q) return;
  if (r0 < 0 || r0 > a.B.n_tokens - q_len) {  // starts that lead outside q and out
    if (tid == 0) kv_bad_index(a.B);
    return;
  }
  const int n = max(0, min(kv_all, a.B.max_kv));
  if ((q_all > a.B.max_q || kv_all > a.B.max_kv) && chunk == 0 && kvh == 0 && tid == 0) kv_bad_index(a.B);
  const int n_chunks = max(1, (n + sp.chunk - 1) / sp.chunk);
  if (chunk >= n_chunks) return;
  const int k0 = chunk * sp.chunk, k1 = min(n, k0 + sp.chunk);
  const int n_st = (k1 - k0 + kKvStage - 1) / kKvStage;
  const int pe = min(a.C.page_size, kKvStage), pe_shift = min(a.C.page_shift, 6);  // keys per piece of a stage
  __syncthreads();
  bool ok = true;

  if (warp == kKvStepWarps) {
    // ---------------------------------------------------------------- producer
    const int pieces = kKvStage >> pe_shift;          // per stage
    const int ahead = 32 >> (6 - pe_shift);           // stages whose page numbers the warp holds
    const uint32_t piece_bytes = static_cast<uint32_t>(pe) * (kHd + 8);
    int pages = -1;
    for (int st = 0; st < n_st && ok; ++st) {
      if (st % ahead == 0) {  // lane i: the page of piece i from here on
        const int pos = k0 + st * kKvStage + lane * pe;
        pages = -1;
        if (pos < k1) {
          pages = __ldg(a.B.table + seq * a.B.table_stride + (pos >> a.C.page_shift));
          if (static_cast<uint32_t>(pages) >= static_cast<uint32_t>(a.C.n_pages)) {
            kv_bad_index(a.B);
            pages = -1;
          }
        }
      }
      const int slot = st % kS;
      if (st >= kS && !mbar_wait_bounded(empty_b + 8 * slot, ((st / kS) - 1) & 1)) {
        ok = false;
        break;
      }
      const int page = __shfl_sync(0xffffffffu, pages, ((st % ahead) << (6 - pe_shift)) + min(lane, pieces - 1));
      const uint32_t mask = __ballot_sync(0xffffffffu, lane < pieces && page >= 0);
      if (lane == 0) {
        asm volatile("st.shared.u32 [%0], %1;" ::"r"(valid_s + 4 * slot), "r"(mask) : "memory");
        mbar_expect_tx(full_b + 8 * slot, piece_bytes * __popc(mask));
      }
      __syncwarp();
      if (lane < pieces && page >= 0) {
        const uint8_t* block = a.C.pages + (static_cast<int64_t>(page) * a.C.kv_heads + kvh) * a.C.head_bytes;
        const uint32_t dst = ring + slot * kStageBytes + lane * piece_bytes, bar = full_b + 8 * slot;
        if (a.C.page_size <= kKvStage) {
          bulk_g2s(dst, block, piece_bytes, bar);
        } else {  // part of a larger page
          const int off = (k0 + st * kKvStage) & (a.C.page_size - 1);
          const uint8_t* pairs = block + a.C.page_size * kHd;
          bulk_g2s(dst, block + off * kRow, kKvStage * kRow, bar);
          bulk_g2s(dst + kKvStage * kRow, block + (a.C.page_size + off) * kRow, kKvStage * kRow, bar);
          bulk_g2s(dst + kKvStage * kHd, pairs + 4 * off, 4 * kKvStage, bar);
          bulk_g2s(dst + kKvStage * (kHd + 4), pairs + 4 * (a.C.page_size + off), 4 * kKvStage, bar);
        }
      }
    }
    if (ok)  // every copy has landed before the CTA can end, whatever its consumers did
      for (int st = max(0, n_st - kS); st < n_st; ++st) ok = mbar_wait_bounded(full_b + 8 * (st % kS), (st / kS) & 1) && ok;
    if (!ok && lane == 0) atomicCAS(a.B.err, 0, kDevErrTmaTimeout);
    return;
  }

  // ------------------------------------------------------------------ consumers
  const int R = q_len * a.group;  // live rows
  // q as B fragments: lane (g, q) has row g of each row tile at dimensions q*kHd/4 + 8w + i, word w;
  // multiplication s of a word meets codes (2s, 2s + 4) in the first register, (2s + 1, 2s + 5) in
  // the second
  uint32_t bq[kNT][2 * kKW][2];
  float cf[kNT][2], qs[kNT][2];  // of rows 2q, 2q + 1: factor of the scores (log2 units), sum of q
  int lim[kNT][2];               // keys that the row sees
#pragma unroll
  for (int t = 0; t < kNT; ++t) {
    const int row = 8 * t + g, i = row / a.group;
    float x[kHd / 4];
    float big = 0.f, sum = 0.f;
    const uint16_t* src = a.q + static_cast<int64_t>(r0 + i) * a.ldq + (kvh * a.group + row - i * a.group) * kHd + q * (kHd / 4);
#pragma unroll
    for (int d = 0; d < kHd / 4; d += 8) {
      uint4 v = make_uint4(0, 0, 0, 0);
      if (row < R) v = a.vec ? ld_row8<true>(src + d) : ld_row8<false>(src + d);
      if (a.bf16) unpack_halves<true>(v, x + d);
      else unpack_halves<false>(v, x + d);
    }
#pragma unroll
    for (int d = 0; d < kHd / 4; ++d) big = fmaxf(big, fabsf(x[d]));
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
    // e with big * 2^e in [2^14, 2^15); |e| is kept below 100 (a query beyond fp32's reach overflows)
    const int e = max(-99, min(99, big > 0.f ? 14 - ((__float_as_int(big) >> 23) - 127) : 0));
    const float up = pow2i(e);
#pragma unroll
    for (int d = 0; d < kHd / 4; ++d) {
      x[d] = __half2float(__float2half_rn(x[d] * up));
      sum += x[d];
    }
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
    for (int w = 0; w < kKW; ++w)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        bq[t][2 * w + s][0] = pack_halves<false>(x[8 * w + 2 * s], x[8 * w + 2 * s + 4]);
        bq[t][2 * w + s][1] = pack_halves<false>(x[8 * w + 2 * s + 1] * 0.0625f, x[8 * w + 2 * s + 5] * 0.0625f);
      }
    // the scores' rows are 2q and 2q + 1 of the tile: fetch their numbers from the lanes of those rows
    const float f = a.scale * 1.4426950408889634f * pow2i(12 - e);  // the other half of 2^(24 - e): below
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      cf[t][c] = __shfl_sync(0xffffffffu, f, (2 * q + c) * 4) * 4096.0f;
      qs[t][c] = __shfl_sync(0xffffffffu, sum, (2 * q + c) * 4) * 0x1p-24f;
      const int rr = 8 * t + 2 * q + c;
      lim[t][c] = rr < R ? max(0, min(n, kv_all - q_all + rr / a.group + 1)) : 0;
    }
  }
  const int all_see = max(0, min(n, kv_all - q_all + 1));  // keys below this are seen by every live row

  float acc[kNT][kMt][4], az[kNT][2], sum[kNT][2], m[kNT][2];
#pragma unroll
  for (int t = 0; t < kNT; ++t) {
#pragma unroll
    for (int i = 0; i < kMt; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[t][i][c] = 0.f;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      az[t][c] = sum[t][c] = 0.f;
      m[t][c] = -1e30f;
    }
  }
  int ve = -30;             // the weights carry scale_v * 2^-ve
  float vinv = 0x1p30f;
  const int perm = g ^ ((g >> 1) & 1);      // the key of score row g (and 8 + perm of row 8 + g): an
  const int pk = 2 * q + (q & 1);           // order in which both code reads spread over the banks;
  const int pk1 = 2 * q + 1 - (q & 1);      // the keys of weights 2q, 2q + 1
  const uint32_t woff = static_cast<uint32_t>(((16 * warp) >> pe_shift) * pe * (kHd + 8));
  const int koff = (16 * warp) & (pe - 1);

  for (int st = 0; st < n_st; ++st) {
    const int slot = st % kS;
    if (!mbar_wait_bounded(full_b + 8 * slot, (st / kS) & 1)) {
      ok = false;
      break;
    }
    const int kb = k0 + st * kKvStage + 16 * warp;  // this warp's first key
    const uint32_t base = ring + slot * kStageBytes + woff;
    if (kb < k1 && ((lds32(valid_s + 4 * slot) >> ((16 * warp) >> pe_shift)) & 1u)) {
      const uint32_t pairs = base + pe * kHd + 4 * (koff + perm);
      uint32_t kp[2], vp[2];
      kp[0] = lds32(pairs);
      kp[1] = lds32(pairs + 32);
      vp[0] = lds32(pairs + 4 * pe);
      vp[1] = lds32(pairs + 4 * pe + 32);
      const bool whole = kb + 16 <= min(k1, all_see);  // no mask in this tile (rows that are not live see garbage)
      if (kb + perm >= k1) kp[0] = vp[0] = 0;           // places past the end hold anything
      if (kb + perm + 8 >= k1) kp[1] = vp[1] = 0;
      // ---- scores
      float s[kNT][4];
#pragma unroll
      for (int t = 0; t < kNT; ++t)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[t][c] = 0.f;
      {
        uint32_t w0[kKW], w1[kKW];
        const uint32_t ka = base + (koff + perm) * kRow + q * (kHd / 8);
        lds_words<kKW>(ka, w0);
        lds_words<kKW>(ka + 8 * kRow, w1);
#pragma unroll
        for (int w = 0; w < kKW; ++w)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t u0 = w0[w] >> (8 * h), u1 = w1[w] >> (8 * h);
            const uint32_t A[4] = {u0 & 0x000f000fu, u1 & 0x000f000fu, u0 & 0x00f000f0u, u1 & 0x00f000f0u};
#pragma unroll
            for (int t = 0; t < kNT; ++t) mma16816(s[t], A, bq[t][2 * w + h][0], bq[t][2 * w + h][1]);
          }
      }
      const float ks0 = half_lo<false>(kp[0]), kz0 = half_hi<false>(kp[0]), ks1 = half_lo<false>(kp[1]), kz1 = half_hi<false>(kp[1]);
      const float vs0 = half_lo<false>(vp[0]), vz0 = half_hi<false>(vp[0]), vs1 = half_lo<false>(vp[1]), vz1 = half_hi<false>(vp[1]);
      bool move = fmaxf(fabsf(vs0), fabsf(vs1)) * vinv > 32.f;
#pragma unroll
      for (int t = 0; t < kNT; ++t) {
        s[t][0] = (s[t][0] + kz0 * qs[t][0]) * (ks0 * cf[t][0]);
        s[t][1] = (s[t][1] + kz0 * qs[t][1]) * (ks0 * cf[t][1]);
        s[t][2] = (s[t][2] + kz1 * qs[t][0]) * (ks1 * cf[t][0]);
        s[t][3] = (s[t][3] + kz1 * qs[t][1]) * (ks1 * cf[t][1]);
        if (!whole) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (kb + perm + 8 * (c >> 1) >= lim[t][c & 1]) s[t][c] = -INFINITY;
        }
        move |= fmaxf(s[t][0], s[t][2]) > m[t][0] + 8.f || fmaxf(s[t][1], s[t][3]) > m[t][1] + 8.f;
      }
      if (__any_sync(0xffffffffu, move)) {
        float vmax = fmaxf(fmaxf(fabsf(vs0), fabsf(vs1)), 0.f);  // (NaN scales have no size)
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, o));
        const int e = max(ve, min(17, (__float_as_int(vmax) >> 23) - 126));  // 2^e above every scale so far
        const float drop = pow2i(max(-126, ve - e));
        ve = e;
        vinv = pow2i(-e);
#pragma unroll
        for (int t = 0; t < kNT; ++t)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float x = fmaxf(s[t][c], s[t][c + 2]);
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
            const float mn = fmaxf(m[t][c], x), corr = ex2(m[t][c] - mn);
            m[t][c] = mn;
            sum[t][c] *= corr;
            az[t][c] *= corr * drop;
#pragma unroll
            for (int i = 0; i < kMt; ++i) {
              acc[t][i][c] *= corr * drop;
              acc[t][i][c + 2] *= corr * drop;
            }
          }
      }
      // ---- weights
      const float u0 = vs0 * vinv, u1 = vs1 * vinv;
      uint32_t bp[kNT][2];
#pragma unroll
      for (int t = 0; t < kNT; ++t) {
        float p[4], w[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          p[c] = ex2(s[t][c] - m[t][c & 1]);
          w[c] = p[c] * (c < 2 ? u0 : u1);
          // (a hidden key's scale may be NaN)
          if (!whole && kb + perm + 8 * (c >> 1) >= lim[t][c & 1]) p[c] = w[c] = 0.f;
        }
        sum[t][0] += p[0] + p[2];
        sum[t][1] += p[1] + p[3];
        const uint32_t h0 = pack_halves<false>(w[0], w[1]), h1 = pack_halves<false>(w[2], w[3]);
        az[t][0] += half_lo<false>(h0) * vz0 + half_lo<false>(h1) * vz1;
        az[t][1] += half_hi<false>(h0) * vz0 + half_hi<false>(h1) * vz1;
        bp[t][0] = movmatrix_trans(h0);
        bp[t][1] = movmatrix_trans(h1);
      }
      // ---- values: half word h (4 dimensions) of the lane's kHd/8 dimensions, of four keys
      const uint32_t va = base + pe * kRow + koff * kRow + g * (kHd / 16);
      constexpr int kH = kHd / 32;  // half words per key
      uint32_t lo[kH], hi[kH];      // (key pk | key pk1) of the first and the second eight keys
      if constexpr (kH % 2 == 0) {
        uint32_t x[4][kH / 2];
        lds_words<kH / 2>(va + pk * kRow, x[0]);
        lds_words<kH / 2>(va + pk1 * kRow, x[1]);
        lds_words<kH / 2>(va + (8 + pk) * kRow, x[2]);
        lds_words<kH / 2>(va + (8 + pk1) * kRow, x[3]);
#pragma unroll
        for (int h = 0; h < kH; ++h) {
          const uint32_t sel = (h & 1) ? 0x7632u : 0x5410u;
          lo[h] = prmt(x[0][h >> 1], x[1][h >> 1], sel);
          hi[h] = prmt(x[2][h >> 1], x[3][h >> 1], sel);
        }
      } else {
#pragma unroll
        for (int h = 0; h < kH; ++h) {
          lo[h] = lds16(va + pk * kRow + 2 * h) | (lds16(va + pk1 * kRow + 2 * h) << 16);
          hi[h] = lds16(va + (8 + pk) * kRow + 2 * h) | (lds16(va + (8 + pk1) * kRow + 2 * h) << 16);
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
    __syncwarp();
    if (lane == 0) mbar_arrive(empty_b + 8 * slot);
  }
  if (!ok && lane == 0) atomicCAS(a.B.err, 0, kDevErrTmaTimeout);

  // ------------------------------------------------------------------ merge of the four warps
  // (the ring is free: every copy was waited for)
  named_barrier(1, kKvStepWarps * 32);
  float* rec = reinterpret_cast<float*>(smem);  // [warp][row][kHd + 4]: the sums, then m and the sum of weights
  constexpr int kRec = kHd + 4;
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
  const bool single = n_chunks == 1;
  const int64_t pair_id = static_cast<int64_t>(seq) * a.C.kv_heads + kvh;
  float* part = single ? nullptr : sp.part + (pair_id * sp.chunks + chunk) * (static_cast<int64_t>(sp.rows) * (kHd + 4));
  constexpr int kQ = kHd / 4;  // float4 columns of a row
  for (int i = tid; i < R * kQ; i += kKvStepWarps * 32) {
    const int row = i / kQ, d = 4 * (i - row * kQ);
    float M = -1e30f, T = 0.f;
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
      *reinterpret_cast<float4*>(part + row * (kHd + 4) + d) = o;
      if (d == 0) *reinterpret_cast<float2*>(part + row * (kHd + 4) + kHd) = make_float2(M, T);
    }
  }
  if (single) return;
  kv_merge_chunks<kHd, kKvStepWarps * 32>(a, sp, r0, kvh, pair_id, n_chunks, R, smem, &sm_last);
}

}  // namespace opc
