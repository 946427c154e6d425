// opc_kv_prompt.cuh -- attention over the 4-bit paged cache for many query rows (prompts and their
// chunks), on the 5th-generation tensor cores.
#pragma once

#include "opc_kv_attention.cuh"
#include "opc_tcgen05.cuh"

namespace opc {

// The rows of one sequence and kv head (query token i, head j of the group: row i * group + j) in
// tiles of 128; a CTA takes kQt tiles against the keys they see, 128 at a time:
//
//   S = Q K'^T     K' = code + zero in fp16: exact for |zero| < 8, one rounding otherwise.  The key's
//                  scale multiplies its column of S in fp32, so nothing of a key is rounded.
//   P = exp2(S * scale_k - m) * scale_v, rounded once to fp16, written over S in tensor memory
//   O += P V'      V' = code + zero in fp16, as above
//
// 4 * 128 * 128 * head_dim operations per tile pair, against 128 * 128 exponentials, which the
// special-function units take as long for as the tensor cores for the products at head_dim 128: two
// row tiles alternate, one in the tensor cores while the other is in the softmax.  Roles:
//   warps 0..3, 4..7  softmax of row tile 0 and 1: thread = row (TMEM lane).  The reference m of a row
//                     moves only when a score passes m + 12 (with the largest scale_v of the tile):
//                     the tile is first evaluated with the old m, and again, with O rescaled, where a
//                     row of the warp passed it -- always in the first tile, hardly ever later.
//   warps 8..11       thread = key: reads its codes (one tile ahead, in registers), writes K' and V'
//                     rows in the 128-byte-swizzled layout -- the same bytes are K-major for K' (rows
//                     are the N dimension) and MN-major for V' (rows are the K dimension)
//   warp 12           one lane issues the MMAs and commits them to the roles' barriers (13..15 idle)
// The warpgroups trade registers: 128 a thread at the launch, then 192 for the softmax (which holds a
// tile's weights until it knows that m stands), 88 and 40 for the others.
// The codes of a word come out in the order 0 4 1 5 2 6 3 7 (one mask per pair); q is staged in that
// order too, and the output columns are put back in order by the epilogue.
// Few CTAs are split over the keys: the partial results go to the workspace as records of the step
// kernel's form, merged by the last CTA of a row tile pair.
constexpr int kKvPM = 128, kKvPN = 128;            // rows per tile, keys per tile
constexpr int kKvPThreads = 16 * 32;
constexpr int kKvPScales = 4;                      // ring of the tiles' scales
__host__ __device__ constexpr int kv_p_hdp(int hd) { return (hd + 63) / 64 * 64; }       // whole swizzle blocks
__host__ __device__ constexpr int kv_p_qt(int hd) { return hd <= 128 ? 2 : 1; }          // row tiles per CTA
__host__ __device__ constexpr int kv_p_st(int hd) { return hd <= 128 ? 2 : 1; }          // K' and V' stages
__host__ __device__ constexpr int kv_p_tile(int hd) { return 128 * kv_p_hdp(hd) * 2; }   // bytes of Q, K', V' tiles
__host__ __device__ constexpr int kv_p_smem(int hd) {
  return 1024 + (kv_p_qt(hd) + 2 * kv_p_st(hd)) * kv_p_tile(hd) + kKvPScales * (kKvPN * 8 + 16) + 256;
}

struct KvPromptSplit {
  int32_t tiles;      // key tiles per CTA
  int32_t splits;
  float* part;        // [items][splits][kQt * 128][head_dim + 4]
  int32_t* count;     // [items]
};

// D[tmem] (+)= A[tmem] * B[smem]: kind::f16, A fp16 packed in pairs along K.
__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accum)
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
      "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
      "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
template <int kRegs>
__device__ __forceinline__ void regs_up() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
}
template <int kRegs>
__device__ __forceinline__ void regs_down() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Shared-memory descriptors of a tile of rows of 64 fp16 (128 bytes, 128-byte swizzle, 8-row groups
// 1024 bytes apart; further blocks of 64 columns 16 KB on).  K-major: rows are M or N.  MN-major: rows
// are K, the stride between the 64-column blocks is the leading offset.
__device__ __forceinline__ uint64_t kv_desc_k(uint32_t saddr) { return umma_desc_sw128(saddr); }
__device__ __forceinline__ uint64_t kv_desc_mn(uint32_t saddr) {
  return static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4) | (1024ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
__host__ __device__ constexpr uint32_t kv_idesc(int n, bool b_mn) {
  return (1u << 4) | (b_mn ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(kKvPM >> 4) << 24);
}

// Eight codes of a word plus the zero, as four pairs of fp16 in the order 04 15 26 37.
__device__ __forceinline__ uint4 kv_codes_plus(uint32_t w, __half2 zero) {
  const __half2 big = __float2half2_rn(-1024.f), small = __float2half2_rn(-64.f), sixteenth = __float2half2_rn(0.0625f);
  uint32_t r[4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t u = w >> (8 * h);
    const uint32_t a = (u & 0x000f000fu) | 0x64006400u, b = (u & 0x00f000f0u) | 0x64006400u;  // 1024 + c, 1024 + 16 c
    const __half2 x = __hadd2(__hadd2(*reinterpret_cast<const __half2*>(&a), big), zero);
    const __half2 y = __hadd2(__hfma2(*reinterpret_cast<const __half2*>(&b), sixteenth, small), zero);
    r[2 * h] = *reinterpret_cast<const uint32_t*>(&x);
    r[2 * h + 1] = *reinterpret_cast<const uint32_t*>(&y);
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}
// Eight elements in natural order to that order.
__device__ __forceinline__ uint4 kv_order8(const uint4& v) {
  return make_uint4(prmt(v.x, v.z, 0x5410u), prmt(v.x, v.z, 0x7632u), prmt(v.y, v.w, 0x5410u), prmt(v.y, v.w, 0x7632u));
}

template <int kHd>
__global__ void __launch_bounds__(kKvPThreads, 1) kv_attention_prompt_kernel(const KvAttnArgs a, const KvPromptSplit sp) {
  constexpr int kQt = kv_p_qt(kHd), kSt = kv_p_st(kHd), kTile = kv_p_tile(kHd), kHdp = kv_p_hdp(kHd);
  constexpr int kBlock = 16384;                 // bytes of 128 rows x 64 columns
  constexpr int kRaw = kHd / 32;                // 16-byte pieces of a key's codes
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  __shared__ uint32_t sm_big, sm_tmem;
  __shared__ int sm_last;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t sQ = base, sK = sQ + kQt * kTile, sV = sK + kSt * kTile, sScale = sV + kSt * kTile;
  const uint32_t sTop = sScale + kKvPScales * kKvPN * 8;  // [ring][4] largest scale_v of the warps' keys
  const uint32_t bars = sTop + kKvPScales * 16;
  const uint32_t kfull_b = bars, kempty_b = bars + 16, vfull_b = bars + 32, vempty_b = bars + 48;
  // (per row tile t and half h of a key tile: [t][h], one phase per key tile each)
  const uint32_t sfull_b = bars + 64, pfull_b = bars + 80, odone_b = bars + 112, drain_b = bars + 144;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(kfull_b + 8 * i, 4);
      mbar_init(kempty_b + 8 * i, 1);
      mbar_init(vfull_b + 8 * i, 4);
      mbar_init(vempty_b + 8 * i, 1);
      mbar_init(sfull_b + 8 * i, 1);
      for (int h = 0; h < 2; ++h) {
        mbar_init(pfull_b + 16 * i + 8 * h, 4);
        mbar_init(odone_b + 16 * i + 8 * h, 1);
      }
    }
    mbar_init(drain_b, 1);
    fence_mbar_init();
    sm_big = 0;
  }
  griddep_wait();
  griddep_launch_dependents();
  // ---------------------------------------------------------------- which rows and keys
  // (later rows see more keys: the tiles of a sequence are taken from the last)
  const int seq = blockIdx.z, kvh = blockIdx.y, split = blockIdx.x % sp.splits, pair_from_end = blockIdx.x / sp.splits;
  const int r0 = __ldg(a.B.q_start + seq), q_all = __ldg(a.B.q_start + seq + 1) - r0, kv_all = __ldg(a.B.kv_len + seq);
  const int q_len = min(q_all, a.B.max_q);
  if (q_len < a.lo_q || q_len > a.hi_q) return;
  if (r0 < 0 || r0 > a.B.n_tokens - q_len) {  // starts that lead outside q and out
    if (tid == 0) kv_bad_index(a.B);
    return;
  }
  const int R = q_len * a.group, pairs = (R + kQt * kKvPM - 1) / (kQt * kKvPM);
  const int pair = pairs - 1 - pair_from_end;
  if (pair < 0) return;
  if ((q_all > a.B.max_q || kv_all > a.B.max_kv) && pair_from_end == 0 && split == 0 && kvh == 0 && tid == 0) kv_bad_index(a.B);
  const int n = max(0, min(kv_all, a.B.max_kv));
  const int row0 = pair * kQt * kKvPM, pos0 = kv_all - q_all;
  const int row_end = min(R, row0 + kQt * kKvPM);
  const int see = max(0, min(n, pos0 + (row_end - 1) / a.group + 1));      // keys that the last row sees
  const int tiles = (see + kKvPN - 1) / kKvPN;
  const int splits = max(1, (tiles + sp.tiles - 1) / sp.tiles);            // CTAs that share this pair
  if (split >= splits) return;
  const int t0 = split * sp.tiles, nt = min(tiles, t0 + sp.tiles) - t0;    // key tiles [t0, t0 + nt)

  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm_tmem)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  __syncthreads();

  // ---------------------------------------------------------------- q: thread = row
  const bool softmax = warp < 4 * kQt;
  const int my_row = row0 + tid;  // of the softmax threads
  const bool live = softmax && my_row < R;
  const int tok = my_row / a.group;
  float qf = a.scale * 1.4426950408889634f;  // factor of the scores (log2 units)
  if (softmax) {
    const uint16_t* src = a.q + static_cast<int64_t>(r0 + tok) * a.ldq + (kvh * a.group + my_row - tok * a.group) * kHd;
    const uint32_t dst = sQ + (tid >> 7) * kTile;
    const int r = tid & 127;
    float up = 1.f;
    if (a.bf16) {  // fp16 has less range: a power of two for the whole tile pair puts its largest near 2^14
      float big = 0.f;
      if (live) {
        for (int c = 0; c < kHd / 8; ++c) {
          float x[8];
          unpack_halves<true>(a.vec ? ld_row8<true>(src + 8 * c) : ld_row8<false>(src + 8 * c), x);
#pragma unroll
          for (int e = 0; e < 8; ++e) big = fmaxf(big, fabsf(x[e]));
        }
      }
      atomicMax(&sm_big, __float_as_uint(big));
      named_barrier(2, kQt * 128);
      const float top = __uint_as_float(sm_big);
      const int e = max(-99, min(99, top > 0.f ? 14 - ((__float_as_int(top) >> 23) - 127) : 0));
      up = pow2i(e);
      qf *= pow2i(-e);
    }
#pragma unroll 4
    for (int c = 0; c < kHd / 8; ++c) {
      uint4 v = make_uint4(0, 0, 0, 0);
      if (live) {
        v = a.vec ? ld_row8<true>(src + 8 * c) : ld_row8<false>(src + 8 * c);
        if (a.bf16) {
          float x[8];
          unpack_halves<true>(v, x);
          v = make_uint4(pack_halves<false>(x[0] * up, x[1] * up), pack_halves<false>(x[2] * up, x[3] * up),
                         pack_halves<false>(x[4] * up, x[5] * up), pack_halves<false>(x[6] * up, x[7] * up));
        }
      }
      sts128(dst + (c >> 3) * kBlock + sw128_off(r, c & 7), kv_order8(v));
    }
    fence_proxy_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm_tmem;
  const uint32_t tS = tmem, tO = tmem + kQt * kKvPN;  // row tile t: S at + 128 t, O at + kHdp t
  bool ok = true;

  // (every warpgroup trades before its role: two at 192, 88 and 40, or with one row tile 192, 24, 168, 40
  // -- at most 512 = 4 * 128 together)
  if (softmax) {
    // ---------------------------------------------------------------- softmax
    regs_up<192>();
    float m = -1e30f, T = 0.f;
    const int t = tid >> 7;
    const uint32_t lanes = static_cast<uint32_t>(32 * (warp & 3)) << 16;
    const uint32_t s_addr = tS + t * kKvPN + lanes, o_addr = tO + t * kHdp + lanes;
    const int lim = live ? max(0, min(n, pos0 + tok + 1)) : 0;   // keys below it are seen by this row
    // (rows that do not exist see nothing; a warp's first live row sees the fewest)
    const int first_row = row0 + (tid & ~31);
    const int plain = first_row + 31 < R ? max(0, min(n, pos0 + first_row / a.group + 1)) : 0;  // tiles below need no mask
    for (int kt = 0; kt < nt; ++kt) {
      const int kb = (t0 + kt) * kKvPN, ring = kt % kKvPScales;
      if (!mbar_wait_bounded(sfull_b + 8 * t, kt & 1)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint32_t sc = sScale + ring * kKvPN * 8;
      const uint4 tops = lds128(sTop + ring * 16);
      // log2 of the largest scale_v of the tile, rounded up (NaN scales are left out; all zero: 2^-30)
      const uint32_t top = max(max(tops.x, tops.y), max(tops.z, tops.w));
      const float ev = static_cast<float>(max(-30, static_cast<int>(top >> 23) - 126));
      const bool whole = kb + kKvPN <= plain;
      // in halves of 64 keys: the weights of the first are multiplied while the second is evaluated
#pragma unroll 1
      for (int h = 0; h < 2 && ok; ++h) {
        uint32_t pk[32];
        float add;
#pragma unroll 1
        for (int pass = 0; pass < 2; ++pass) {
          float mx = -INFINITY;
          add = 0.f;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t v[32];
            tmem_ld32(s_addr + 64 * h + 32 * c, v);
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              const int j = 32 * c + e;  // of the half
              const uint4 f = lds128(sc + (64 * h + j) * 8);  // (scale_k, scale_v) of two keys
              float x0 = __uint_as_float(v[e]) * (__uint_as_float(f.x) * qf), x1 = __uint_as_float(v[e + 1]) * (__uint_as_float(f.z) * qf);
              if (!whole) {
                if (kb + 64 * h + j >= lim) x0 = -INFINITY;
                if (kb + 64 * h + j + 1 >= lim) x1 = -INFINITY;
              }
              mx = fmaxf(mx, fmaxf(x0, x1));
              const float p0 = ex2(x0 - m), p1 = ex2(x1 - m);
              add += p0 + p1;
              float w0 = p0 * __uint_as_float(f.y), w1 = p1 * __uint_as_float(f.w);
              if (!whole) {  // (a hidden key's scale may be NaN)
                if (x0 == -INFINITY) w0 = 0.f;
                if (x1 == -INFINITY) w1 = 0.f;
              }
              pk[j >> 1] = pack_halves<false>(w0, w1);
            }
          }
          if (pass || !__any_sync(0xffffffffu, mx + ev > m + 12.f)) break;
          const float mn = fmaxf(m, mx + ev), corr = ex2(m - mn);
          m = mn;
          T *= corr;
          if (kt + h > 0) {  // O holds the halves before
            if (!mbar_wait_bounded(odone_b + 16 * t + 8 * (1 - h), (kt + h - 1) & 1)) {
              ok = false;
              break;
            }
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < kHd / 32; ++c) {
              uint32_t v[32];
              tmem_ld32(o_addr + 32 * c, v);
#pragma unroll
              for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * corr);
              tmem_st32(o_addr + 32 * c, v);
            }
          }
        }
        T += add;
        tmem_st32(s_addr + 32 * h, pk);  // over scores that have been read
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(pfull_b + 16 * t + 8 * h);
      }
      if (!ok) break;
    }
    // -------------------------------------------------------------- results
    if (ok && nt > 0) ok = mbar_wait_bounded(odone_b + 16 * t + 8, (nt - 1) & 1);
    tc_fence_after();
    const bool single = splits == 1;
    const int64_t item = (static_cast<int64_t>(seq) * gridDim.y + kvh) * (gridDim.x / sp.splits) + pair_from_end;
    constexpr int kRec = kHd + 4;
    float* rec = single ? nullptr : sp.part + ((item * sp.splits + split) * (kQt * kKvPM) + tid) * kRec;
    const int row = my_row;  // of the sequence and kv head
#pragma unroll 1
    for (int c = 0; c < kHd / 32; ++c) {
      uint32_t v[32];
      if (nt > 0) {
        tmem_ld32(o_addr + 32 * c, v);
      } else {
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = 0;
      }
      if (live && ok) {
#pragma unroll
        for (int e = 0; e < 32; e += 8) {  // columns 0 4 1 5 2 6 3 7 of eight dimensions
          const float x[8] = {__uint_as_float(v[e]),     __uint_as_float(v[e + 2]), __uint_as_float(v[e + 4]), __uint_as_float(v[e + 6]),
                              __uint_as_float(v[e + 1]), __uint_as_float(v[e + 3]), __uint_as_float(v[e + 5]), __uint_as_float(v[e + 7])};
          const float4 lo = make_float4(x[0], x[1], x[2], x[3]), hi = make_float4(x[4], x[5], x[6], x[7]);
          const int d = 32 * c + e;
          if (single) {
            kv_finish_row(a, r0, kvh, row, d, lo, m, T);
            kv_finish_row(a, r0, kvh, row, d + 4, hi, m, T);
          } else {
            *reinterpret_cast<float4*>(rec + d) = lo;
            *reinterpret_cast<float4*>(rec + d + 4) = hi;
          }
        }
      }
    }
    if (!single) {
      if (live) *reinterpret_cast<float2*>(rec + kHd) = make_float2(m, T);
      named_barrier(2, kQt * 128);
      if (tid == 0) {
        const bool last = atom_add_acq_rel_gpu(sp.count + item, 1) == splits - 1;
        if (last) sp.count[item] = 0;
        sm_last = last;
      }
      named_barrier(2, kQt * 128);
      if (sm_last && ok) {  // merge, in order: thread = (row, four dimensions)
        const float* part = sp.part + item * sp.splits * (kQt * kKvPM) * kRec;
        const int rows = row_end - row0;
        for (int i = tid; i < rows * (kHd / 4); i += kQt * 128) {
          const int r = i / (kHd / 4), d = 4 * (i - r * (kHd / 4));
          float M = -1e30f, S = 0.f;
          float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int s = 0; s < splits; ++s) M = fmaxf(M, __ldcg(part + (static_cast<int64_t>(s) * kQt * kKvPM + r) * kRec + kHd));
          for (int s = 0; s < splits; ++s) {
            const float* src = part + (static_cast<int64_t>(s) * kQt * kKvPM + r) * kRec;
            const float2 w = __ldcg(reinterpret_cast<const float2*>(src + kHd));
            const float4 v = __ldcg(reinterpret_cast<const float4*>(src + d));
            const float f = ex2(w.x - M);
            S += f * w.y;
            o.x += f * v.x;
            o.y += f * v.y;
            o.z += f * v.z;
            o.w += f * v.w;
          }
          kv_finish_row(a, r0, kvh, row0 + r, d, o, M, S);
        }
      }
    }
    } else if (warp < 8) {
    regs_down<24>();
  } else if (warp < 12) {
    // ---------------------------------------------------------------- keys: thread = key of the tile
    if constexpr (kQt == 2) regs_down<88>();
    else regs_up<168>();
    const int key = tid - 8 * 32, w4 = warp - 8;
    const int codes = a.C.page_size * (kHd / 2);
    uint4 rk[kRaw], rv[kRaw];
    uint32_t pk = 0, pv = 0;
    int64_t off = -1;  // the key's page in the tile to load next
    const auto find = [&](int kt) {
      const int pos = (t0 + kt) * kKvPN + key;
      off = kt < nt && pos < n ? kv_page_offset(a.C, a.B, seq, pos >> a.C.page_shift) : -1;
    };
    const auto load = [&](int kt) {
#pragma unroll
      for (int i = 0; i < kRaw; ++i) rk[i] = rv[i] = make_uint4(0, 0, 0, 0);
      pk = pv = 0;  // places past the end: scale and zero 0
      if (off >= 0) {
        const int in = ((t0 + kt) * kKvPN + key) & (a.C.page_size - 1);
        const uint8_t* block = a.C.pages + off + kvh * a.C.head_bytes;
#pragma unroll
        for (int i = 0; i < kRaw; ++i) {
          rk[i] = __ldg(reinterpret_cast<const uint4*>(block + in * (kHd / 2) + 16 * i));
          rv[i] = __ldg(reinterpret_cast<const uint4*>(block + codes + in * (kHd / 2) + 16 * i));
        }
        pk = __ldg(reinterpret_cast<const uint32_t*>(block + 2 * codes + 4 * in));
        pv = __ldg(reinterpret_cast<const uint32_t*>(block + 2 * codes + 4 * (a.C.page_size + in)));
      }
    };
    const auto convert = [&](const uint4 (&raw)[kRaw], uint32_t pair, uint32_t tile) {
      const __half2 zero = __half2half2(__ushort_as_half(static_cast<unsigned short>(pair >> 16)));
#pragma unroll
      for (int i = 0; i < kRaw; ++i) {
        const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int c = 4 * i + j;  // 8 dimensions
          sts128(tile + (c >> 3) * kBlock + sw128_off(key, c & 7), kv_codes_plus(w[j], zero));
        }
      }
    };
    find(0);
    load(0);
    find(1);
    for (int kt = 0; kt < nt; ++kt) {
      const int st = kt % kSt, ring = kt % kKvPScales;
      const uint32_t par = ((kt / kSt) - 1) & 1;
      if (kt >= kSt && !mbar_wait_bounded(kempty_b + 8 * st, par)) {
        ok = false;
        break;
      }
      const float2 kf = unpack_half2(pk), vf = unpack_half2(pv);
      sts64(sScale + (ring * kKvPN + key) * 8, __float_as_uint(kf.x), __float_as_uint(vf.x));
      const float size = fminf(fmaxf(fabsf(vf.x), 0.f), 65504.f);  // (a NaN has no size)
      const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(size));
      if (lane == 0) asm volatile("st.shared.u32 [%0], %1;" ::"r"(sTop + ring * 16 + 4 * w4), "r"(top) : "memory");
      convert(rk, pk, sK + st * kTile);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(kfull_b + 8 * st);
      if (kt >= kSt && !mbar_wait_bounded(vempty_b + 8 * st, par)) {
        ok = false;
        break;
      }
      convert(rv, pv, sV + st * kTile);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(vfull_b + 8 * st);
      load(kt + 1);
      find(kt + 2);
    }
  } else {
    // ---------------------------------------------------------------- MMA issuer
    regs_down<40>();
    if (warp == 12 && lane == 0) {
      const auto scores = [&](int t, int kt) {
        const int st = kt % kSt;
#pragma unroll 2
        for (int k = 0; k < kHd / 16; ++k) {
          const uint32_t o = (k >> 2) * kBlock + (k & 3) * 32;
          umma_f16(tS + t * kKvPN, kv_desc_k(sQ + t * kTile + o), kv_desc_k(sK + st * kTile + o), kv_idesc(kKvPN, false), k > 0);
        }
        umma_commit(sfull_b + 8 * t);
        if (t == kQt - 1) umma_commit(kempty_b + 8 * st);
      };
      const auto wait = [&](uint32_t bar, uint32_t par) {
        if (ok) ok = mbar_wait_bounded(bar, par);
        tc_fence_after();
        return ok;
      };
      if (nt > 0 && wait(kfull_b, 0))
        for (int t = 0; t < kQt; ++t) scores(t, 0);
      for (int kt = 0; kt < nt && ok; ++kt) {
        const int st = kt % kSt;
        if (!wait(vfull_b + 8 * st, (kt / kSt) & 1)) break;
        for (int t = 0; t < kQt && ok; ++t) {
          for (int h = 0; h < 2 && wait(pfull_b + 16 * t + 8 * h, kt & 1); ++h) {
#pragma unroll 1
            for (int k = 0; k < kKvPN / 32; ++k)
              umma_f16_ts(tO + t * kHdp, tS + t * kKvPN + 32 * h + 8 * k, kv_desc_mn(sV + st * kTile + 8192 * h + 2048 * k),
                          kv_idesc(kHdp, true), kt > 0 || h > 0 || k > 0);
            umma_commit(odone_b + 16 * t + 8 * h);
          }
          if (!ok) break;
          if (t == kQt - 1) umma_commit(vempty_b + 8 * st);
          if (kt + 1 < nt && wait(kfull_b + 8 * ((kt + 1) % kSt), ((kt + 1) / kSt) & 1)) scores(t, kt + 1);
        }
      }
      // no tensor-core operation of this CTA is in flight past this point
      umma_commit(drain_b);
      mbar_wait_bounded(drain_b, 0);
    }
  }

  if (!ok && lane == 0) atomicCAS(a.B.err, 0, kDevErrTmaTimeout);
  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

}  // namespace opc
