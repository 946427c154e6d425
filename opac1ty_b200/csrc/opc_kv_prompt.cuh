// opc_kv_prompt.cuh -- attention over the 4-bit paged cache for many query rows (prompts and their
// chunks), on the 5th-generation tensor cores.
#pragma once

#include "opc_kv_attention.cuh"
#include "opc_tcgen05.cuh"

namespace opc {

// The rows of one sequence and kv head (query token i, head j of the group: row i * group + j) in
// tiles of 128; a CTA takes kQt tiles against the keys they see, 128 at a time:
//
//   S = Q K'^T     (in halves of 64 keys, so that the next half's scores are there while one is evaluated)
//                  K' = code - 8, exact in fp16; what is left of the zeros, (zero + 8) sum q, is added by
//                  one more product in tf32, with both factors in parts of 11 bits (sum q three, zero + 8
//                  two).  The key's scale multiplies its column of S in fp32: nothing of a key is rounded.
//                  (K' = code + zero in fp16 would save 3% of the prompts below, but round the keys' largest
//                  elements: log sums off by 1e-6 of their value instead of 4e-8.)
//   P = exp2(S * scale_k - m) * scale_v, rounded once to fp16, written over S in tensor memory
//   O += P V'      V' = code + zero in fp16: exact where no value is larger than |zero|, else one rounding
//                  (2^-11 of the value, as for P and the result)
//
// 4 * 128 * 128 * head_dim operations per tile pair, against 128 * 128 exponentials, which the
// special-function units take as long for as the tensor cores for the products at head_dim 128: two
// row tiles alternate, one in the tensor cores while the other is in the softmax.  Roles:
//   warps 0..15   softmax: four warps for rows 0..15 of each 32 TMEM lanes of row tile 0, four for rows
//                 16..31, then the same for row tile 1.  In the 16-row fragment shapes a lane has a
//                 quarter of the columns of two rows, so that it reads a quarter of the keys' scales
//                 from shared memory (with thread = row every thread would read all of them), and four
//                 warps per SM sub-partition hide each other's latencies (two took twice as long).
//                 The reference m of a row moves only when the sum of a half's weights says that one
//                 times the tile's largest scale_v may pass 2^15: then the row's maximum is looked for,
//                 O rescaled and the half evaluated again, its largest weight times that scale at 2^5
//                 (kKvLift) -- always in the first tile, hardly ever later.
//   warps 16..19  thread = key: reads its key codes (one tile ahead, in registers) and writes the K' row
//                 in the 128-byte-swizzled layout, the scales, and a bit for each key of a missing page (the
//                 softmax then keeps them out of maximum and sum)
//   warps 20..23  the same for V' -- the same layout is K-major for K' (rows are the N dimension) and
//                 MN-major for V' (rows are the K dimension).  (Four warps for both took 1% longer.)
//   warp 24       issues the MMAs and commits them to the roles' barriers (25..27 idle)
// The warpgroups trade registers: 72 a thread at the launch, then 88 for the softmax, 56 for the
// converters, 40 for the MMA warp; with one row tile (head_dim 192 and 256) two warpgroups less are
// in the softmax and the converters take more.
// The codes of a word come out in the order 0 4 1 5 2 6 3 7 (one mask per pair); q is staged in that
// order too, and the output columns are put back in order by the epilogue.
// An item is a tile pair of one sequence and kv head.  How many there are is known on the device only
// (the host knows bounds, which a batch of a few prompts among many single tokens is far below), so each
// CTA counts them from q_start (a grid of sequences times the longest one's tiles, most of it empty, would
// take twice as long for a prompt of 2000 among 100 single tokens, 161 us); where they are fewer than the SMs,
// several CTAs share an item's keys, evenly, and their partial results go to the workspace as records,
// merged by the item's last CTA.  The tiles with the most keys come first (one prompt of 2000 tokens, 256
// items over 148 SMs, 57 us: a fifth less than in order).
// Measured, 32 heads of 128 over 8, fp16: 359 us for three prompts of 1500 to 4097 tokens, 705 TFLOP/s; 59 us
// for 512 tokens behind 3584, 547 TFLOP/s; bf16 371 and 60 us, with the look at q's rows in every CTA.  No unit is
// full (tensor cores 37%, issue 59%, special functions 37%): leaving out the exponentials or most of the products
// of Q K' changes nothing, so what bounds it is the latency of the chain scores - weights - products in each of
// the four half tiles in flight, and about 8 us per CTA to fill and drain it.
constexpr int kKvPM = 128, kKvPN = 128;            // rows per tile, keys per tile
constexpr int kKvPThreads = 28 * 32;
constexpr int kKvPConv = 16, kKvPMma = 24;         // first converter warp, the MMA warp
constexpr int kKvPZero = 128 * 32;                 // bytes of a tile's factors of the tf32 product
constexpr int kKvPScales = 4;                      // ring of the tiles' scales
__host__ __device__ constexpr int kv_p_hdp(int hd) { return (hd + 63) / 64 * 64; }       // whole swizzle blocks
__host__ __device__ constexpr int kv_p_qt(int hd) { return hd <= 128 ? 2 : 1; }          // row tiles per CTA
__host__ __device__ constexpr int kv_p_st(int hd) { return hd <= 128 ? 2 : 1; }          // K' and V' stages
__host__ __device__ constexpr int kv_p_tile(int hd) { return 128 * kv_p_hdp(hd) * 2; }   // bytes of Q, K', V' tiles
__host__ __device__ constexpr int kv_p_smem(int hd) {
  return 1024 + (kv_p_qt(hd) + 2 * kv_p_st(hd)) * kv_p_tile(hd) + (kv_p_qt(hd) + kv_p_st(hd)) * kKvPZero + kKvPScales * (kKvPN * 8 + 32) + 256;
}

struct KvPromptSplit {
  uint32_t ctas;      // that may share their items' keys; 1: none do
  float* part;        // [items][CTAs per item][kQt * 128][head_dim + 4]
  int32_t* count;     // [items], zero between calls
};

// MMAs issued by one lane of a converged warp (`leader`, from elect.sync): outside a divergent branch
// their operands can be formed in uniform registers, which brought a key tile's 48 instructions and
// their barriers from ~6300 cycles to what the tensor cores take.
__device__ __forceinline__ uint32_t elect_leader() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
  return p;
}
__device__ __forceinline__ void umma_f16_by(uint32_t leader, uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n .reg .pred p, l;\n setp.ne.b32 l, %5, 0;\n setp.ne.b32 p, %4, 0;\n"
      " @l tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accum), "r"(leader)
      : "memory");
}
// tf32, 8 along K: tiles of 128 rows of 32 bytes without swizzle, in blocks of 8 rows x 16 bytes (the two of
// a row 128 bytes apart, the next 8 rows 256).
__device__ __forceinline__ void umma_tf32_by(uint32_t leader, uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n .reg .pred p, l;\n setp.ne.b32 l, %5, 0;\n setp.ne.b32 p, %4, 0;\n"
      " @l tcgen05.mma.cta_group::1.kind::tf32 [%0], %1, %2, %3, p;\n}\n" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accum), "r"(leader)
      : "memory");
}
__device__ __forceinline__ uint64_t kv_desc_rows32(uint32_t saddr) {
  return static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4) | (8ull << 16) | (16ull << 32) | (1ull << 46);
}
__device__ __forceinline__ uint32_t kv_rows32_off(int row) { return static_cast<uint32_t>((row >> 3) * 256 + (row & 7) * 16); }
__device__ __forceinline__ float high11(float x) { return __uint_as_float(__float_as_uint(x) & 0xffffe000u); }
// The same with A in tensor memory, fp16 packed in pairs along K.
__device__ __forceinline__ void umma_f16_ts_by(uint32_t leader, uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc,
                                               uint32_t accum) {
  asm volatile(
      "{\n .reg .pred p, l;\n setp.ne.b32 l, %5, 0;\n setp.ne.b32 p, %4, 0;\n"
      " @l tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accum), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void umma_commit_by(uint32_t leader, uint32_t bar) {
  asm volatile(
      "{\n .reg .pred l;\n setp.ne.b32 l, %1, 0;\n"
      " @l tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(bar), "r"(leader)
      : "memory");
}
template <typename T>
__device__ __forceinline__ void swap_values(T& a, T& b) {
  const T t = a;
  a = b;
  b = t;
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

__host__ __device__ constexpr uint32_t kv_idesc_tf32(int n) {
  return (1u << 4) | (2u << 7) | (2u << 10) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(kKvPM >> 4) << 24);
}

// The 16-row fragment shapes: of 8 fp32 columns lane (g, q) = (lane / 4, lane % 4) holds (row g, columns
// 2q, 2q + 1) and (row g + 8, the same); of 4 32-bit columns (16x128b) column q of rows g and g + 8.
__device__ __forceinline__ void tmem_ld_rows32(uint32_t taddr, uint32_t* v) {  // 32 columns
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
      "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st_rows32(uint32_t taddr, const uint32_t* v) {  // 32 columns
  asm volatile(
      "tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15,"
      "%16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_pairs32(uint32_t taddr, const uint32_t* v) {  // 32 columns of fp16 pairs
  asm volatile(
      "tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15,"
      "%16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// The weights of 16 rows (lane (g, q): rows g and g + 8) for 64 keys: pk the fp16 pairs
// exp2(S * scale_k - m) * scale_v; the lane's share of the rows' sums of the weights without scale_v.
// sk, sv: shared-memory addresses of the scales of the lane's 16 keys (8i + 2q, 8i + 2q + 1).  kMode 1: a
// row sees its first `seen` keys only.  2: and of those none whose bit is set in the two words at sg; its
// scores are multiplied by its factor, at sf (row g + 8: sf + 64), and rounded as in kv_row_max, so that a
// maximum of any size meets itself.
template <int kMode>
__device__ __forceinline__ void kv_weights(uint32_t s_addr, uint32_t sk, uint32_t sv, const float* m, const int* seen, uint32_t sg,
                                           uint32_t sf, int q, uint32_t* pk, float* add) {
  const uint64_t minus[2] = {pack2(-m[0], -m[0]), pack2(-m[1], -m[1])};
  float factor[2] = {1.f, 1.f};
  if (kMode == 2) {
    factor[0] = __uint_as_float(lds32(sf));
    factor[1] = __uint_as_float(lds32(sf + 64));
  }
  uint64_t sum[2] = {0, 0};
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    uint32_t v[16];
    tmem_ld_rows32(s_addr + 32 * c, v);
    const uint4 k4[2] = {lds128(sk + 32 * c), lds128(sk + 32 * c + 16)}, v4[2] = {lds128(sv + 32 * c), lds128(sv + 32 * c + 16)};
    const uint32_t out = kMode == 2 ? lds32(sg + 4 * c) >> (2 * q) : 0;  // bits 8j, 8j + 1: the lane's keys
    tmem_wait_ld();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int col = 32 * c + 8 * j + 2 * q;
      const uint4 &kk = k4[j >> 1], &vv = v4[j >> 1];
      const uint64_t ks = pack2(__uint_as_float((j & 1) ? kk.z : kk.x), __uint_as_float((j & 1) ? kk.w : kk.y));
      const uint64_t vs = pack2(__uint_as_float((j & 1) ? vv.z : vv.x), __uint_as_float((j & 1) ? vv.w : vv.y));
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        const float s0 = __uint_as_float(v[4 * j + 2 * a]), s1 = __uint_as_float(v[4 * j + 2 * a + 1]);
        float2 y;
        if (kMode == 2) {
          const float2 k = unpack2(ks);
          y.x = __fsub_rn(__fmul_rn(s0, k.x * factor[a]), m[a]);
          y.y = __fsub_rn(__fmul_rn(s1, k.y * factor[a]), m[a]);
        } else {
          y = unpack2(fma2(pack2(s0, s1), ks, minus[a]));
        }
        if (kMode) {
          if (col >= seen[a] || (out >> (8 * j) & 1u)) y.x = -INFINITY;
          if (col + 1 >= seen[a] || (out >> (8 * j) & 2u)) y.y = -INFINITY;
        }
        const uint64_t p = pack2(ex2(y.x), ex2(y.y));
        sum[a] = add2(sum[a], p);
        float2 w = unpack2(mul2(p, vs));
        if (kMode) {  // (a hidden key's scale may be NaN)
          if (col >= seen[a] || (out >> (8 * j) & 1u)) w.x = 0.f;
          if (col + 1 >= seen[a] || (out >> (8 * j) & 2u)) w.y = 0.f;
        }
        pk[8 * c + 2 * j + a] = pack_halves<false>(w.x, w.y);
      }
    }
  }
#pragma unroll
  for (int a = 0; a < 2; ++a) {
    const float2 x = unpack2(sum[a]);
    add[a] = x.x + x.y;
  }
}
// The largest S * scale_k (kAny: * factor, as in kv_weights) of the two rows over the 64 keys (whole rows: all four lanes get it).
template <bool kAny>
__device__ __forceinline__ void kv_row_max(uint32_t s_addr, uint32_t sk, const int* seen, uint32_t sg, uint32_t sf, int q, float* mx) {
  mx[0] = mx[1] = -INFINITY;
  float f[2] = {1.f, 1.f};
  if (kAny) {
    f[0] = __uint_as_float(lds32(sf));
    f[1] = __uint_as_float(lds32(sf + 64));
  }
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    uint32_t v[16];
    tmem_ld_rows32(s_addr + 32 * c, v);
    const uint32_t out = kAny ? lds32(sg + 4 * c) >> (2 * q) : 0;
    tmem_wait_ld();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint2 k = lds64(sk + 32 * c + 8 * j);
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        const int col = 32 * c + 8 * j + 2 * q;
        if (col < seen[a] && !(out >> (8 * j) & 1u)) mx[a] = fmaxf(mx[a], __uint_as_float(v[4 * j + 2 * a]) * (__uint_as_float(k.x) * f[a]));
        if (col + 1 < seen[a] && !(out >> (8 * j) & 2u)) mx[a] = fmaxf(mx[a], __uint_as_float(v[4 * j + 2 * a + 1]) * (__uint_as_float(k.y) * f[a]));
      }
    }
  }
#pragma unroll
  for (int a = 0; a < 2; ++a) {
    mx[a] = fmaxf(mx[a], __shfl_xor_sync(0xffffffffu, mx[a], 1));
    mx[a] = fmaxf(mx[a], __shfl_xor_sync(0xffffffffu, mx[a], 2));
  }
}

// Eight codes of a word minus 8, as four pairs of fp16 in the order 04 15 26 37.
__device__ __forceinline__ uint4 kv_codes_minus8(uint32_t w) {
  const __half2 big = __float2half2_rn(-1032.f), small = __float2half2_rn(-72.f), sixteenth = __float2half2_rn(0.0625f);
  uint32_t r[4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t u = w >> (8 * h);
    const uint32_t a = (u & 0x000f000fu) | 0x64006400u, b = (u & 0x00f000f0u) | 0x64006400u;  // 1024 + c, 1024 + 16 c
    const __half2 x = __hadd2(*reinterpret_cast<const __half2*>(&a), big);
    const __half2 y = __hfma2(*reinterpret_cast<const __half2*>(&b), sixteenth, small);
    r[2 * h] = *reinterpret_cast<const uint32_t*>(&x);
    r[2 * h + 1] = *reinterpret_cast<const uint32_t*>(&y);
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
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
// Eight results times a factor, as 16-bit elements.
__device__ __forceinline__ uint4 kv_out8(const float* x, float f, int bf16) {
  return bf16 ? make_uint4(pack_halves<true>(x[0] * f, x[1] * f), pack_halves<true>(x[2] * f, x[3] * f),
                           pack_halves<true>(x[4] * f, x[5] * f), pack_halves<true>(x[6] * f, x[7] * f))
              : make_uint4(pack_halves<false>(x[0] * f, x[1] * f), pack_halves<false>(x[2] * f, x[3] * f),
                           pack_halves<false>(x[4] * f, x[5] * f), pack_halves<false>(x[6] * f, x[7] * f));
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
  __shared__ uint32_t sm_tmem, sm_top, sm_low;
  __shared__ int sm_power, sm_uneven;  // of q as staged (below)
  __shared__ int sm_last;
  __shared__ struct {
    uint32_t item, first, rec;  // the item, its first record, this CTA's record
    int splits, r0;
  } sm_item;  // what the results need (in registers it would cost the loop between)
  __shared__ float2 sm_rows[kQt * kKvPM];  // of the rows: (largest |q|, factor of the scores), then (m, sum)
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t sQ = base, sK = sQ + kQt * kTile, sV = sK + kSt * kTile, sQz = sV + kSt * kTile;
  const uint32_t sKz = sQz + kQt * kKvPZero, sScale = sKz + kSt * kKvPZero;
  const uint32_t sTop = sScale + kKvPScales * kKvPN * 8;  // [ring][4] largest scale_v of the warps' keys
  const uint32_t sGone = sTop + kKvPScales * 16;          // [ring] 128 bits: the keys of missing pages
  const uint32_t bars = sGone + kKvPScales * 16;
  const uint32_t kfull_b = bars, kempty_b = bars + 16, vfull_b = bars + 32, vempty_b = bars + 48;
  // (per row tile t and half h of a key tile: [t][h], one phase per key tile each)
  const uint32_t sfull_b = bars + 64, pfull_b = bars + 96, odone_b = bars + 128, drain_b = bars + 160, qsum_b = bars + 168;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(kfull_b + 8 * i, 4);
      mbar_init(kempty_b + 8 * i, 1);
      mbar_init(vfull_b + 8 * i, 4);
      mbar_init(vempty_b + 8 * i, 1);
      for (int h = 0; h < 2; ++h) {
        mbar_init(sfull_b + 16 * i + 8 * h, 1);
        mbar_init(pfull_b + 16 * i + 8 * h, 8);
        mbar_init(odone_b + 16 * i + 8 * h, 1);
      }
    }
    mbar_init(drain_b, 1);
    mbar_init(qsum_b, 4 * kQt);
    fence_mbar_init();
    sm_power = sm_uneven = 0;
    sm_top = 0;
    sm_low = 0x7f800000u;
  }
  griddep_wait();
  // ---------------------------------------------------------------- which rows and keys
  // (by every warp for itself; the tile pairs of sequence s: none when the launch does not take it)
  const int kvh_n = a.C.kv_heads;
  int my_r0 = 0, my_q = 0, my_kv = 0;  // of sequence s0 + lane
  const auto load_seqs = [&](int s0) {  // their tile pairs
    const int s = s0 + lane;
    if (s >= a.B.n_seqs) return 0;
    my_r0 = __ldg(a.B.q_start + s);
    my_q = __ldg(a.B.q_start + s + 1) - my_r0;
    my_kv = __ldg(a.B.kv_len + s);
    const int len = min(my_q, a.B.max_q);
    return len < a.lo_q || len > a.hi_q ? 0 : (len * a.group + kQt * kKvPM - 1) / (kQt * kKvPM);
  };
  uint32_t items = 0;
  for (int s0 = 32; s0 < a.B.n_seqs; s0 += 32) items += load_seqs(s0);
  int n_pairs = load_seqs(0);
  items = __reduce_add_sync(0xffffffffu, items + n_pairs) * kvh_n;
  if (items == 0) return;
  uint32_t most = 1, item = blockIdx.x, split = 0;  // most: CTAs that may share an item
  if (2 * items <= sp.ctas) {
    most = sp.ctas / items;
    item = blockIdx.x / most;
    split = blockIdx.x - item * most;
  }
  if (item >= items) return;
  // The item's sequence; of a sequence the last tile pairs, which see the most keys, come first.
  int src = 0, local = 0, s0 = 0;
  for (int before = 0;;) {
    int upto = n_pairs;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    const uint32_t here = __ballot_sync(0xffffffffu, static_cast<uint32_t>((before + upto) * kvh_n) > item);
    if (here) {
      src = __ffs(here) - 1;
      local = static_cast<int>(item) - (before + __shfl_sync(0xffffffffu, upto - n_pairs, src)) * kvh_n;
      break;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
    s0 += 32;
    if (s0 >= a.B.n_seqs) return;  // (starts that go up and down, so that the sum did not fit)
    n_pairs = load_seqs(s0);
  }
  const int seq = s0 + src, pairs = __shfl_sync(0xffffffffu, n_pairs, src), r0 = __shfl_sync(0xffffffffu, my_r0, src);
  const int q_all = __shfl_sync(0xffffffffu, my_q, src), kv_all = __shfl_sync(0xffffffffu, my_kv, src);
  const int pair_from_end = local / kvh_n, kvh = local - pair_from_end * kvh_n, pair = pairs - 1 - pair_from_end;
  const int q_len = min(q_all, a.B.max_q), R = q_len * a.group;
  if (r0 < 0 || r0 > a.B.n_tokens - q_len) {  // starts that lead outside q and out
    if (tid == 0) kv_bad_index(a.B);
    return;
  }
  if ((q_all > a.B.max_q || kv_all > a.B.max_kv) && local == 0 && split == 0 && tid == 0) kv_bad_index(a.B);
  const int n = max(0, min(kv_all, a.B.max_kv));
  const int row0 = pair * kQt * kKvPM, pos0 = kv_all - q_all;
  const int row_end = min(R, row0 + kQt * kKvPM);
  const int see = max(0, min(n, pos0 + (row_end - 1) / a.group + 1));      // keys that the last row sees
  const int tiles = (see + kKvPN - 1) / kKvPN;
  int per = tiles, splits = 1;
  if (most > 1 && tiles >= 4) {  // two key tiles a CTA at least
    const int share = min(static_cast<int>(most), tiles / 2);
    per = (tiles + share - 1) / share;
    splits = (tiles + per - 1) / per;
  }
  if (split >= splits) return;
  if (tid == 0) sm_item = {item, item * most, item * most + split, splits, r0};
  const int t0 = split * per, nt = min(tiles, t0 + per) - t0;              // key tiles [t0, t0 + nt)

  if (warp == kKvPMma) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm_tmem)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (tid < kQt * kKvPM) sm_rows[tid] = make_float2(0.f, 1.f);
  __syncthreads();
  // (after the allocation: a kernel that allocates tensor memory before it waits for this one could otherwise
  // take, on this SM, the columns that this CTA goes on to ask for, and neither would end; that this CTA's
  // registers leave hardly any room for another is not what this should rest on)
  griddep_launch_dependents();

  // ---------------------------------------------------------------- the converters' first loads
  const bool softmax = warp < 8 * kQt, converter = warp >= kKvPConv && warp < kKvPMma;
  const int key = tid & 127;  // of the tile
  const int codes = a.C.page_size * (kHd / 2);
  const bool is_v = warp >= kKvPConv + 4;
  uint4 raw[kRaw];
  uint32_t pk = 0, pv = 0;
  bool gone = false;   // whether the key in raw, pk and pv is of a missing page
  int64_t off = -1;    // the key's page in the tile to load next
  const auto find = [&](int kt) {
    const int pos = (t0 + kt) * kKvPN + key;
    off = kt < nt && pos < n ? kv_page_offset(a.C, a.B, seq, pos >> a.C.page_shift) : -1;
  };
  const auto load = [&](int kt) {
#pragma unroll
    for (int i = 0; i < kRaw; ++i) raw[i] = make_uint4(0, 0, 0, 0);
    pk = pv = 0;  // places past the end and of missing pages: scale and zero 0
    gone = off < 0 && (t0 + kt) * kKvPN + key < n;
    if (off >= 0) {
      const int in = ((t0 + kt) * kKvPN + key) & (a.C.page_size - 1);
      const uint8_t* block = a.C.pages + off + kvh * a.C.head_bytes;
#pragma unroll
      for (int i = 0; i < kRaw; ++i)
        raw[i] = __ldg(reinterpret_cast<const uint4*>(block + (is_v ? codes : 0) + in * (kHd / 2) + 16 * i));
      pk = __ldg(reinterpret_cast<const uint32_t*>(block + 2 * codes + 4 * in));
      pv = __ldg(reinterpret_cast<const uint32_t*>(block + 2 * codes + 4 * (a.C.page_size + in)));
    }
  };
  if (converter) find(0);

  // ---------------------------------------------------------------- q, by all threads
  // bf16 q goes in multiplied by a power of two that puts its largest near 2^14 (fp16 has less range): one
  // for the whole tile pair, which the keys' scales take back, where every row's largest reaches 2^-12 of the
  // pair's (what is rounded then lies 2^-27 below its row's largest, less than the sums in fp32 round).  Else
  // each row has its own, and its scores are multiplied by its factor (kMode 2).  Rows with an infinity or
  // NaN stay out of the choice: they give NaN with any factor.
  const auto power_of = [](uint32_t big) {
    return big ? max(-99, min(99, 14 - (static_cast<int>(big >> 23) - 127))) : 0;
  };
  {
    constexpr int kChunks = kHd / 8, kAll = kQt * kKvPM * kChunks, kMine = (kAll + kKvPThreads - 1) / kKvPThreads;
    uint4 v[kMine];
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int x = i * kKvPThreads + tid, row = row0 + x / kChunks, c = x % kChunks, tok = row / a.group;
      const uint16_t* src = a.q + static_cast<int64_t>(r0 + tok) * a.ldq + (kvh * a.group + row - tok * a.group) * kHd + 8 * c;
      v[i] = make_uint4(0, 0, 0, 0);
      if (x < kAll && row < R) v[i] = a.vec ? ld_row8<true>(src) : ld_row8<false>(src);
    }
    if (a.bf16) {
      uint32_t top = 0, low = 0x7f800000u;  // of finite chunks of 8; of chunks that are not 0
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        float x[8], big = 0.f;
        unpack_halves<true>(v[i], x);
#pragma unroll
        for (int e = 0; e < 8; ++e) big = fmaxf(big, fabsf(x[e]));
        const uint32_t b = __float_as_uint(big);
        if (b < 0x7f800000u) top = max(top, b);
        if (b) low = min(low, b);
      }
      top = __reduce_max_sync(0xffffffffu, top);
      low = __reduce_min_sync(0xffffffffu, low);
      if (lane == 0) {
        atomicMax(&sm_top, top);
        atomicMin(&sm_low, low);
      }
      __syncthreads();
      top = *const_cast<volatile uint32_t*>(&sm_top);
      bool uneven = *const_cast<volatile uint32_t*>(&sm_low) + (12u << 23) < top;
      if (uneven) {  // some chunk is that small: is a whole row?
        // (a row's chunks are kChunks lanes in a row: those of an aligned span of them meet in registers)
        constexpr int kSpan = kChunks % 32 == 0 ? 32 : kChunks % 16 == 0 ? 16 : kChunks % 8 == 0 ? 8 : 4;
        static_assert(kChunks % kSpan == 0 && kAll % 32 == 0, "a span of lanes is of one row");
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
          float x[8], big = 0.f;
          unpack_halves<true>(v[i], x);
#pragma unroll
          for (int e = 0; e < 8; ++e) big = fmaxf(big, fabsf(x[e]));
#pragma unroll
          for (int o = 1; o < kSpan; o <<= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
          const int at = i * kKvPThreads + tid;
          if (at < kAll && (lane & (kSpan - 1)) == 0) atomicMax(reinterpret_cast<uint32_t*>(&sm_rows[at / kChunks].x), __float_as_uint(big));
        }
        __syncthreads();
        low = 0x7f800000u;
#pragma unroll
        for (int i = 0; i < kQt * kKvPM; i += 32) {
          const uint32_t big = __float_as_uint(sm_rows[i + lane].x);
          if (big) low = min(low, big);
        }
        uneven = __reduce_min_sync(0xffffffffu, low) + (12u << 23) < top;
      }
      if (tid == 0) {
        sm_power = uneven ? 0 : power_of(top);
        sm_uneven = uneven;
      }
      if (uneven && tid < kQt * kKvPM) sm_rows[tid].y = pow2i(-power_of(__float_as_uint(sm_rows[tid].x)));
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const int at = i * kKvPThreads + tid;
        const float up = pow2i(power_of(uneven && at < kAll ? __float_as_uint(sm_rows[at / kChunks].x) : top));
        float x[8];
        unpack_halves<true>(v[i], x);
        v[i] = make_uint4(pack_halves<false>(x[0] * up, x[1] * up), pack_halves<false>(x[2] * up, x[3] * up),
                          pack_halves<false>(x[4] * up, x[5] * up), pack_halves<false>(x[6] * up, x[7] * up));
      }
    }
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int x = i * kKvPThreads + tid, row = x / kChunks, c = x % kChunks;
      if (x < kAll) sts128(sQ + (row >> 7) * kTile + (c >> 3) * kBlock + sw128_off(row & 127, c & 7), kv_order8(v[i]));
    }
    fence_proxy_async_smem();
  }
  if (kQt == 2 && converter) load(0);  // (large heads: when the converters have their registers)
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm_tmem;
  const uint32_t tS = tmem, tO = tmem + kQt * kKvPN;  // row tile t: S at + 128 t, O at + kHdp t
  bool ok = true;

  // (every warpgroup trades before its role: 4 * 88 + 2 * 56 + 40 = 7 * 72, or with one row tile
  // 2 * 96 + 2 * 24 + 2 * 112 + 40)
  if (softmax) {
    // ---------------------------------------------------------------- softmax
    regs_up<kQt == 2 ? 88 : 96>();
    const int t = warp >> 3, b = (warp >> 2) & 1, g = lane >> 2, q = lane & 3;
    const int lane0 = 32 * (warp & 3) + 16 * b;  // the warp's first row (TMEM lane) of the tile
    const uint32_t lanes = static_cast<uint32_t>(lane0) << 16;
    const uint32_t s_addr = tS + t * kKvPN + lanes, o_addr = tO + t * kHdp + lanes;
    const int first_row = row0 + t * kKvPM + lane0;
    if (b == 0) {  // thread = row: the sum of its q, as staged
      const int in = tid & 127;
      float x = 0.f;
#pragma unroll 4
      for (int c = 0; c < kHd / 8; ++c) {
        const uint4 w = lds128(sQ + t * kTile + (c >> 3) * kBlock + sw128_off(in, c & 7));
        const float2 e0 = unpack_half2(w.x), e1 = unpack_half2(w.y), e2 = unpack_half2(w.z), e3 = unpack_half2(w.w);
        x += ((e0.x + e0.y) + (e1.x + e1.y)) + ((e2.x + e2.y) + (e3.x + e3.y));
      }
      const float x1 = high11(x), x2 = high11(x - x1), x3 = x - x1 - x2;
      const uint32_t at = sQz + t * kKvPZero + kv_rows32_off(in);
      sts128(at, make_uint4(__float_as_uint(x1), __float_as_uint(x1), __float_as_uint(x2), __float_as_uint(x2)));
      sts128(at + 128, make_uint4(__float_as_uint(x3), 0, 0, 0));
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(qsum_b);
    }
    float m[2], T[2];   // of rows g and g + 8
    int lim[2];         // keys below it are seen by the row
    bool fresh[2];      // no key seen yet, but one will be: m means nothing
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      m[r] = T[r] = 0.f;
      const int row = first_row + 8 * r + g;
      lim[r] = row < R ? max(0, min(n, pos0 + row / a.group + 1)) : 0;
      fresh[r] = lim[r] > 0;
    }
    // tiles below need no mask (rows that do not exist see nothing; the first row sees the fewest)
    const int plain = first_row + 15 < R ? max(0, min(n, pos0 + first_row / a.group + 1)) : 0;
    bool any = sm_uneven != 0;  // everything in kMode 2
    const uint32_t factors = smem_u32(&sm_rows[t * kKvPM + lane0 + g].y);  // of row g; of g + 8 64 bytes on
    for (int kt = 0; kt < nt; ++kt) {
      const int kb = (t0 + kt) * kKvPN, ring = kt % kKvPScales;
      const uint32_t sc = sScale + ring * kKvPN * 8;
      const bool whole = kb + kKvPN <= plain;
      // in halves of 64 keys: the weights of the first are multiplied while the second is evaluated
#pragma unroll 1
      for (int h = 0; h < 2; ++h) {
        if (!mbar_wait_bounded(sfull_b + 16 * t + 8 * h, kt & 1)) {
          ok = false;
          break;
        }
        tc_fence_after();
        // log2 of the largest scale_v of the tile, rounded up (NaN scales are left out; all zero: 2^-30); bit 31
        // of a word says that some of its keys are gone
        const uint4 tops = lds128(sTop + ring * 16);
        uint32_t top = max(max(tops.x, tops.y), max(tops.z, tops.w));
        bool full = any;
        if (top >> 31) {
          full = true;
          constexpr uint32_t kSize = 0x7fffffffu;
          top = max(max(tops.x & kSize, tops.y & kSize), max(tops.z & kSize, tops.w & kSize));
        }
        const float ev = static_cast<float>(max(-30, static_cast<int>(top >> 23) - 126));
        uint32_t pk[16];
        float add[2];
        const uint32_t addr = s_addr + 64 * h, sk = sc + 256 * h + 64 * q, sv = sk + 512, sg = sGone + ring * 16 + 8 * h;
        const int seen[2] = {lim[0] - kb - 64 * h, lim[1] - kb - 64 * h};
        // A row moves m when its weights' sum (the lane's share) says that one times scale_v may pass 2^15,
        // or when it has seen no key yet.
        bool moved = __any_sync(0xffffffffu, (fresh[0] && seen[0] > 0) || (fresh[1] && seen[1] > 0));
#pragma unroll 1
        for (;;) {
          if (moved) {
            float mx[2], corr[2];
            if (full) kv_row_max<true>(addr, sk, seen, sg, factors, q, mx);
            else kv_row_max<false>(addr, sk, seen, sg, factors, q, mx);
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const bool first = fresh[r] && mx[r] > -INFINITY;
              const float at = mx[r] + (ev - kKvLift), to = first || at > m[r] ? at : m[r];
              corr[r] = first ? 1.f : ex2(m[r] - to);
              m[r] = to;
              T[r] *= corr[r];
              fresh[r] = fresh[r] && !first;
            }
            // scores so large that products which are not rounded may differ from the maximum by more than the
            // weights' range
            if (__any_sync(0xffffffffu, fmaxf(fabsf(m[0]), fabsf(m[1])) > 1e6f)) full = any = true;
            if (kt + h > 0) {  // O holds the halves before
              if (!mbar_wait_bounded(odone_b + 16 * t + 8 * (1 - h), (kt + h - 1) & 1)) ok = false;
              tc_fence_after();
#pragma unroll 1
              for (int c = 0; c < kHd / 32; ++c) {
                uint32_t v[16];
                tmem_ld_rows32(o_addr + 32 * c, v);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 16; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * corr[(e >> 1) & 1]);
                tmem_st_rows32(o_addr + 32 * c, v);
              }
            }
          }
          if (full) kv_weights<2>(addr, sk, sv, m, seen, sg, factors, q, pk, add);
          else if (whole) kv_weights<0>(addr, sk, sv, m, seen, sg, factors, q, pk, add);
          else kv_weights<1>(addr, sk, sv, m, seen, sg, factors, q, pk, add);
          if (moved || !__any_sync(0xffffffffu, fmaxf(add[0], add[1]) > ex2(15.f - ev))) break;
          moved = true;
        }
        T[0] += add[0];
        T[1] += add[1];
        tmem_st_pairs32(addr, pk);  // over the half's scores, which have been read
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
    // From here on thread = row of the tile, the tile's second four warps taking other columns than the
    // first: (m, sum) of the rows through shared memory.
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      T[r] += __shfl_xor_sync(0xffffffffu, T[r], 1);
      T[r] += __shfl_xor_sync(0xffffffffu, T[r], 2);
      if (q == 0) sm_rows[t * kKvPM + lane0 + 8 * r + g] = make_float2(lim[r] > 0 && !fresh[r] ? m[r] : kKvNone, T[r]);
    }
    named_barrier(2 + t, 256);
    const int in = tid & 127, tile_row = t * kKvPM + in;
    const float row_m = sm_rows[tile_row].x, row_T = sm_rows[tile_row].y;
    const uint32_t row_addr = tO + t * kHdp + (static_cast<uint32_t>(32 * (warp & 3)) << 16);
    const int row = row0 + tile_row;
    const bool live = row < R;
    const int n_rec = *const_cast<volatile int*>(&sm_item.splits), first_token = *const_cast<volatile int*>(&sm_item.r0);
    const bool single = n_rec == 1;
    // a record: the weighted sums [head_dim / 4][rows] x 4, then (m, sum) [rows]
    constexpr int kRows = kQt * kKvPM;
    float* rec = sp.part + static_cast<int64_t>(sm_item.rec) * (kRows * (kHd + 4));
    const uint32_t out_s = sQ + t * kTile;  // the row tile's output, laid out like q, which is no longer needed
    const float inv = row_T == 0.f ? 0.f : 1.0f / row_T;  // a row that sees nothing: 0 (a NaN sum stays NaN)
#pragma unroll 1
    for (int c = b; c < kHd / 16; c += 2) {
      uint32_t v[16];
      if (nt > 0) {
        tmem_ld16(row_addr + 16 * c, v);
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = 0;
      }
#pragma unroll
      for (int e = 0; e < 16; e += 8) {  // columns 0 4 1 5 2 6 3 7 of eight dimensions
        const int d = 16 * c + e;
        const float x[8] = {__uint_as_float(v[e]),     __uint_as_float(v[e + 2]), __uint_as_float(v[e + 4]), __uint_as_float(v[e + 6]),
                            __uint_as_float(v[e + 1]), __uint_as_float(v[e + 3]), __uint_as_float(v[e + 5]), __uint_as_float(v[e + 7])};
        if (single) {
          sts128(out_s + (d >> 6) * kBlock + sw128_off(in, (d >> 3) & 7), kv_out8(x, inv, a.bf16));
        } else if (live) {
          *reinterpret_cast<float4*>(rec + (d / 4 * kRows + tile_row) * 4) = make_float4(x[0], x[1], x[2], x[3]);
          *reinterpret_cast<float4*>(rec + (d / 4 * kRows + kRows + tile_row) * 4) = make_float4(x[4], x[5], x[6], x[7]);
        }
      }
    }
    const int tok = row / a.group, head = kvh * a.group + row - tok * a.group;
    uint16_t* dst = a.out + static_cast<int64_t>(first_token + tok) * a.ldo + static_cast<int64_t>(head) * kHd;
    if (single) {
      if (b == 0 && live && ok && a.lse)
        a.lse[static_cast<int64_t>(first_token + tok) * a.heads + head] = kv_lse(row_m, row_T);
      named_barrier(2 + t, 256);
      constexpr int kChunks = kHd / 8;
#pragma unroll 2
      for (int i = 0; i < kChunks / 2; ++i) {  // whole rows at a time, of the warp's 16 (in lanes 16b..16b + 15)
        const int x = i * 32 + lane, r = 16 * b + x / kChunks, c = x % kChunks;
        const uint64_t to = __shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(dst), r);
        const uint4 w = lds128(out_s + (c >> 3) * kBlock + sw128_off((in & 96) + r, c & 7));
        uint16_t* o = reinterpret_cast<uint16_t*>(to) + 8 * c;
        if (row - lane + r < R && ok) {
          if (a.vec) st_row8<true>(o, w);
          else st_row8<false>(o, w);
        }
      }
    } else {
      if (b == 0 && live) *reinterpret_cast<float2*>(rec + kRows * kHd + 2 * tile_row) = make_float2(row_m, row_T);
      named_barrier(4, 2 * kRows);
      if (tid == 0) {
        const bool last = atom_add_acq_rel_gpu(sp.count + sm_item.item, 1) == n_rec - 1;
        if (last) sp.count[sm_item.item] = 0;
        sm_last = last;
      }
      named_barrier(4, 2 * kRows);
      if (sm_last && live && ok) {  // merge, in order: thread = row and every other 16 dimensions
        const float* part = sp.part + static_cast<int64_t>(sm_item.first) * (kRows * (kHd + 4));
        float M = kKvNone, S = 0.f;
#pragma unroll 4
        for (int i = 0; i < n_rec; ++i) {
          const float2 w = __ldcg(reinterpret_cast<const float2*>(part + i * (kRows * (kHd + 4)) + kRows * kHd + 2 * tile_row));
          const float up = fmaxf(M, w.x);
          S = S * ex2(M - up) + w.y * ex2(w.x - up);
          M = up;
        }
        const float scale = S == 0.f ? 0.f : 1.0f / S;
#pragma unroll 1
        for (int d = 16 * b; d < kHd; d += 32) {
          float o[16] = {};
#pragma unroll 2
          for (int i = 0; i < n_rec; ++i) {
            const float* src = part + i * (kRows * (kHd + 4));
            const float f = ex2(__ldcg(src + kRows * kHd + 2 * tile_row) - M);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float4 v = __ldcg(reinterpret_cast<const float4*>(src + ((d / 4 + e) * kRows + tile_row) * 4));
              o[4 * e] += f * v.x;
              o[4 * e + 1] += f * v.y;
              o[4 * e + 2] += f * v.z;
              o[4 * e + 3] += f * v.w;
            }
          }
#pragma unroll
          for (int e = 0; e < 16; e += 8) {
            const uint4 w = kv_out8(o + e, scale, a.bf16);
            if (a.vec) st_row8<true>(dst + d + e, w);
            else st_row8<false>(dst + d + e, w);
          }
        }
        if (b == 0 && a.lse)
          a.lse[static_cast<int64_t>(first_token + tok) * a.heads + head] = kv_lse(M, S);
      }
    }
  } else if (warp < kKvPConv) {
    regs_down<24>();
  } else if (warp < kKvPMma) {
    // ---------------------------------------------------------------- keys: thread = key of the tile
    if constexpr (kQt == 2) {
      regs_down<56>();
    } else {
      regs_up<112>();
      load(0);
    }
    find(1);
    const float qf = a.scale * 1.4426950408889634f * pow2i(-sm_power);  // factor of the scores (log2 units)
    for (int kt = 0; kt < nt; ++kt) {
      const int st = kt % kSt, ring = kt % kKvPScales;
      if (kt >= kSt && !mbar_wait_bounded((is_v ? vempty_b : kempty_b) + 8 * st, ((kt / kSt) - 1) & 1)) {
        ok = false;
        break;
      }
      if (!is_v) {
        const float2 kf = unpack_half2(pk), vf = unpack_half2(pv);
        // (in the order of the softmax's lanes: by half, then (key % 8) / 2, key / 8, key % 2)
        const uint32_t at = sScale + ring * kKvPN * 8 + 4 * ((key & 64) + 16 * ((key >> 1) & 3) + 2 * ((key >> 3) & 7) + (key & 1));
        asm volatile("st.shared.f32 [%0], %1;" ::"r"(at), "f"(kf.x * qf) : "memory");
        asm volatile("st.shared.f32 [%0], %1;" ::"r"(at + 512), "f"(vf.x) : "memory");
        const float size = fminf(fmaxf(fabsf(vf.x), 0.f), 65504.f);  // (a NaN has no size)
        const float z = kf.y + 8.f, z1 = high11(z), z2 = z - z1;
        const uint32_t z_at = sKz + st * kKvPZero + kv_rows32_off(key);
        sts128(z_at, make_uint4(__float_as_uint(z1), __float_as_uint(z2), __float_as_uint(z1), __float_as_uint(z2)));
        sts128(z_at + 128, make_uint4(__float_as_uint(z1), 0, 0, 0));
        const uint32_t out = __ballot_sync(0xffffffffu, gone);
        const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(size)) | (out ? 0x80000000u : 0u);
        if (lane == 0) {
          asm volatile("st.shared.u32 [%0], %1;" ::"r"(sTop + ring * 16 + 4 * (warp - kKvPConv)), "r"(top) : "memory");
          asm volatile("st.shared.u32 [%0], %1;" ::"r"(sGone + ring * 16 + 4 * (warp - kKvPConv)), "r"(out) : "memory");
        }
      }
      const __half2 zero = __half2half2(__ushort_as_half(static_cast<unsigned short>(pv >> 16)));
      const uint32_t tile = (is_v ? sV : sK) + st * kTile;
#pragma unroll
      for (int i = 0; i < kRaw; ++i) {
        const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int c = 4 * i + j;  // 8 dimensions
          sts128(tile + (c >> 3) * kBlock + sw128_off(key, c & 7), is_v ? kv_codes_plus(w[j], zero) : kv_codes_minus8(w[j]));
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive((is_v ? vfull_b : kfull_b) + 8 * st);
      load(kt + 1);
      find(kt + 2);
    }
  } else {
    // ---------------------------------------------------------------- MMA issuer
    regs_down<40>();
    if (warp == kKvPMma) {  // (all lanes wait and count, one issues)
      const uint32_t leader = elect_leader();
      // the scores of row tile t for half h of key tile kt
      const auto scores = [&](int t, int kt, int h) {
        const int st = kt % kSt;
        const uint64_t qd = kv_desc_k(sQ + t * kTile), kd = kv_desc_k(sK + st * kTile + 8192 * h);  // (in units of 16 bytes)
#pragma unroll
        for (int k = 0; k < kHd / 16; ++k) {
          constexpr int kB = kBlock / 16;
          umma_f16_by(leader, tS + t * kKvPN + 64 * h, qd + ((k >> 2) * kB + (k & 3) * 2), kd + ((k >> 2) * kB + (k & 3) * 2),
                   kv_idesc(kKvPN / 2, false), k > 0);
        }
        umma_tf32_by(leader, tS + t * kKvPN + 64 * h, kv_desc_rows32(sQz + t * kKvPZero), kv_desc_rows32(sKz + st * kKvPZero) + 128 * h,
                     kv_idesc_tf32(kKvPN / 2), 1);
        umma_commit_by(leader, sfull_b + 16 * t + 8 * h);
        if (t == kQt - 1 && h == 1) umma_commit_by(leader, kempty_b + 8 * st);
      };
      const auto wait = [&](uint32_t bar, uint32_t par) {
        if (ok) ok = mbar_wait_bounded(bar, par);
        tc_fence_after();
        return ok;
      };
      if (nt > 0 && wait(qsum_b, 0) && wait(kfull_b, 0))
        for (int i = 0; i < 2 * kQt; ++i) scores(i % kQt, 0, i / kQt);
      for (int kt = 0; kt < nt && ok; ++kt) {
        const int st = kt % kSt;
        if (!wait(vfull_b + 8 * st, (kt / kSt) & 1)) break;
        if (kt + 1 < nt && kSt > 1 && !wait(kfull_b + 8 * ((kt + 1) % kSt), ((kt + 1) / kSt) & 1)) break;
        for (int i = 0; i < 2 * kQt; ++i) {
          const int t = i % kQt, h = i / kQt;
          if (!wait(pfull_b + 16 * t + 8 * h, kt & 1)) break;
          const uint64_t vd = kv_desc_mn(sV + st * kTile + 8192 * h);
#pragma unroll
          for (int k = 0; k < kKvPN / 32; ++k)
            umma_f16_ts_by(leader, tO + t * kHdp, tS + t * kKvPN + 64 * h + 8 * k, vd + 128 * k, kv_idesc(kHdp, true), kt + h + k > 0);
          umma_commit_by(leader, odone_b + 16 * t + 8 * h);
          if (t == kQt - 1 && h == 1) umma_commit_by(leader, vempty_b + 8 * st);
          if (kt + 1 < nt) {
            if (kSt == 1 && i == 0 && !wait(kfull_b, (kt + 1) & 1)) break;
            scores(t, kt + 1, h);
          }
        }
      }
      // no tensor-core operation of this CTA is in flight past this point
      umma_commit_by(leader, drain_b);
      mbar_wait_bounded(drain_b, 0);
    }
  }

  if (!ok && lane == 0) atomicCAS(a.B.err, 0, kDevErrTmaTimeout);
  tc_fence_before();
  __syncthreads();
  if (warp == kKvPMma) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

}  // namespace opc
