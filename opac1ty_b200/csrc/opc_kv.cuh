// opc_kv.cuh -- the paged key/value cache held in 4 bits: its layout, appending rows to it with
// the rotary embedding, and reading them back (layout and rules: include/opc_b200.h).
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "opc_device.cuh"

namespace opc {

// The cache of one call.  `pages` holds n_pages * kv_heads blocks of head_bytes.
struct KvGeom {
  uint8_t* pages;
  int64_t head_bytes;
  int32_t kv_heads, hd, page_size, page_shift, n_pages;
};

// The batch of one call (opc_kv_batch) and the device error word.
struct KvRows {
  const int32_t* q_start;
  const int32_t* kv_len;
  const int32_t* table;
  int64_t table_stride;
  int32_t n_seqs, n_tokens, max_q, max_kv, max_pages;
  int* err;
};

__device__ __forceinline__ void kv_bad_index(const KvRows& B) { atomicCAS(B.err, 0, kDevErrBadIndex); }

// Where the batch puts row r, found by one whole warp (all lanes get the answer): the sequence is
// the number of starts q_start[1..] at or before r, counted by all lanes at once -- one round of
// independent loads instead of a chain of log2(n_seqs) dependent ones.
struct KvRowPlace {
  int seq;    // -1: the row belongs to no sequence
  int pos;    // position in the sequence (may be negative: kv_len < q_len)
};
__device__ __forceinline__ KvRowPlace kv_row_place(const KvRows& B, int r, int lane) {
  int n = 0;
  for (int i = 1 + lane; i <= B.n_seqs; i += 32) n += __ldg(B.q_start + i) <= r;
  n = __reduce_add_sync(0xffffffffu, n);
  KvRowPlace p;
  p.seq = -1;
  p.pos = -1;
  if (n < B.n_seqs && __ldg(B.q_start) <= r) {
    p.seq = n;
    p.pos = __ldg(B.kv_len + n) - (__ldg(B.q_start + n + 1) - r);
  }
  return p;
}

// Byte offset of page `index` of sequence `seq` in the cache (kv head 0), -1 when the table names
// no page of it (recorded in the error word).
__device__ __forceinline__ int64_t kv_page_offset(const KvGeom& C, const KvRows& B, int seq, int index) {
  const int page = __ldg(B.table + seq * B.table_stride + index);
  if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(C.n_pages)) {
    kv_bad_index(B);
    return -1;
  }
  return static_cast<int64_t>(page) * C.kv_heads * C.head_bytes;
}
// The place of position `pos`: its page's offset, -1 when it has none.
__device__ __forceinline__ int64_t kv_place(const KvGeom& C, const KvRows& B, const KvRowPlace& p) {
  if (p.seq < 0 || p.pos < 0) return -1;
  if (p.pos >= B.max_kv || (p.pos >> C.page_shift) >= B.max_pages) {
    kv_bad_index(B);
    return -1;
  }
  return kv_page_offset(C, B, p.seq, p.pos >> C.page_shift);
}

// Two fp32 values per instruction.
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
  float2 d;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(v));
  return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// 16-bit elements as fp32 and back; kBf: bf16, else fp16.
template <bool kBf>
__device__ __forceinline__ float half_lo(uint32_t w) {
  if constexpr (kBf) return __uint_as_float(w << 16);
  return __half2float(__ushort_as_half(static_cast<unsigned short>(w & 0xffffu)));
}
template <bool kBf>
__device__ __forceinline__ float half_hi(uint32_t w) {
  if constexpr (kBf) return __uint_as_float(w & 0xffff0000u);
  return __half2float(__ushort_as_half(static_cast<unsigned short>(w >> 16)));
}
template <bool kBf>
__device__ __forceinline__ uint32_t pack_halves(float lo, float hi) {
  if constexpr (kBf) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <bool kBf>
__device__ __forceinline__ void unpack_halves(const uint4& w, float x[8]) {
  const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (kBf) {
      x[2 * i] = half_lo<true>(v[i]);
      x[2 * i + 1] = half_hi<true>(v[i]);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
}

// Eight 16-bit elements at p: one 16-byte access where the tensor's base and leading dimension
// allow it (kVec), else one by one.
template <bool kVec>
__device__ __forceinline__ uint4 ld_row8(const uint16_t* p) {
  if constexpr (kVec) {
    return *reinterpret_cast<const uint4*>(p);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = static_cast<uint32_t>(p[2 * i]) | (static_cast<uint32_t>(p[2 * i + 1]) << 16);
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
}
template <bool kVec>
__device__ __forceinline__ void st_row8(uint16_t* p, const uint4& v) {
  if constexpr (kVec) {
    *reinterpret_cast<uint4*>(p) = v;
  } else {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      p[2 * i] = static_cast<uint16_t>(w[i] & 0xffffu);
      p[2 * i + 1] = static_cast<uint16_t>(w[i] >> 16);
    }
  }
}

// ------------------------------------------------------------------------------------------------
// Append
// ------------------------------------------------------------------------------------------------
constexpr int kKvAppendThreads = 256;
constexpr int kKvMaxHd = 256;

struct KvAppendArgs {
  KvGeom C;
  KvRows B;
  const uint16_t *k, *v, *q;
  uint16_t* q_out;
  int64_t ldk, ldv, ldq, ldqo;
  int32_t heads;          // 0: no q
  int32_t rot_dim, interleaved;  // rot_dim 0: no rotation
  const uint64_t* turns;
};

// One CTA takes kTok rows (tokens); kLpr lanes (a power of two, head_dim / 8 of them at work) take
// one head with 16 bytes each, one after the other of the CTA's heads, with the loads of the next
// kAhead heads in flight (one load at a time held 16 KB in flight on an SM, a third of what HBM's
// latency asks for).  Memory bound for prompts (2 bytes in and out per element of q, 2 in and 0.5 out
// per element of k and v), latency bound for steps: there gridDim.y spreads a row's heads over CTAs so
// that each group of lanes has one head, loaded before the row's place is looked up (three dependent
// loads: starts, length, page table).  Measured, 32/8 heads of 128: one row 3.4 us; 5217 rows 37 us, where
// issue (79%) and no longer memory (1.8 TB/s of DRAM traffic, the rest in L2) is the bound.
//
// Angles: position * turns (64-bit product) is the angle in turns modulo 1, exact; sine and cosine
// are formed in double from it, once per row and pair, shared by all heads, and rounded to fp32.
// The products are rounded one by one (no fused multiply-add), so a stored code is the same
// whatever lane computes it and equals the one an elementwise fp32 evaluation gives.
template <int kLpr, int kTok, bool kBf, bool kVec>
__global__ void __launch_bounds__(kKvAppendThreads) kv_append_kernel(const KvAppendArgs a) {
  // per row and turned dimension e: (cos, sin) of its pair, sin with the sign that its partner enters
  // with; in the order [e % 8][lane], which a head's lanes read without bank conflicts
  __shared__ float2 cs[kTok][8][kKvMaxHd / 8];
  __shared__ int64_t place[kTok];
  __shared__ int place_pos[kTok], place_seq[kTok];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  constexpr int kGroups = kKvAppendThreads / kLpr, kAhead = kTok == 1 ? 1 : 3;
  const int grp = tid / kLpr, c = tid % kLpr;
  const int hd = a.C.hd, kvh = a.C.kv_heads, chunks = hd >> 3;
  const bool on = c < chunks;
  const int heads_all = 2 * kvh + a.heads;  // a row's heads: k, then v, then q
  const int r0 = blockIdx.x * kTok, rows = min(kTok, a.B.n_tokens - r0);
  const uint32_t gmask = kLpr == 32 ? 0xffffffffu : ((1u << (kLpr & 31)) - 1u) << (lane & ~(kLpr - 1));

  // this group's heads: (row t, head h) in steps of the CTAs' groups
  const int step = kGroups * gridDim.y;
  struct At {
    int t, h;
  };
  const auto advance = [&](At& x) {
    x.h += step;
    while (x.h >= heads_all && x.t < rows) {
      x.h -= heads_all;
      ++x.t;
      if (kTok == 1) x.t = rows;  // (one row: its heads are spread over the CTAs)
    }
  };
  const auto load = [&](const At& x) {
    if (!on || x.t >= rows) return make_uint4(0, 0, 0, 0);
    const int64_t r = r0 + x.t;
    const uint16_t* p = x.h < kvh ? a.k + r * a.ldk + x.h * hd
                                  : x.h < 2 * kvh ? a.v + r * a.ldv + (x.h - kvh) * hd : a.q + r * a.ldq + (x.h - 2 * kvh) * hd;
    return ld_row8<kVec>(p + 8 * c);
  };
  At cur{0, static_cast<int>(blockIdx.y) * kGroups + grp}, ahead;
  while (cur.h >= heads_all && cur.t < rows) {
    cur.h -= heads_all;
    cur.t = kTok == 1 ? rows : cur.t + 1;
  }
  griddep_wait();
  griddep_launch_dependents();
  uint4 raws[kAhead];
  ahead = cur;
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    raws[i] = load(ahead);
    advance(ahead);
  }

  if (warp < kTok) {
    KvRowPlace p;
    p.seq = p.pos = -1;
    if (r0 + warp < a.B.n_tokens) p = kv_row_place(a.B, r0 + warp, lane);
    if (lane == 0) {
      place_pos[warp] = p.pos;
      place_seq[warp] = p.seq;
      place[warp] = kv_place(a.C, a.B, p);
    }
  }
  __syncthreads();
  const int half = a.rot_dim >> 1;
  for (int i = tid; i < kTok * half; i += kKvAppendThreads) {
    const int t = i / half, j = i - t * half;
    if (place_seq[t] >= 0 && place_pos[t] >= 0) {
      const uint64_t turn = static_cast<uint64_t>(place_pos[t]) * __ldg(a.turns + j);
      double s, co;  // the signed 64-bit fraction of a turn, in half turns
      sincospi(static_cast<double>(static_cast<int64_t>(turn)) * 0x1p-63, &s, &co);
      const int e0 = a.interleaved ? 2 * j : j, e1 = a.interleaved ? 2 * j + 1 : j + half;
      cs[t][e0 & 7][e0 >> 3] = make_float2(static_cast<float>(co), -static_cast<float>(s));
      cs[t][e1 & 7][e1 >> 3] = make_float2(static_cast<float>(co), static_cast<float>(s));
    }
  }
  __syncthreads();

  const int hc = a.rot_dim >> 4;  // lanes holding the first halves of the pairs (not interleaved)
  const bool turned = on && c < (a.rot_dim >> 3);
  // the lane with the other half of the pairs
  const int src = (lane & ~(kLpr - 1)) + (a.interleaved || c >= 2 * hc ? c : c < hc ? c + hc : c - hc);
#pragma unroll 1
  while (cur.t < rows) {
    const uint4 raw = raws[0];
#pragma unroll
    for (int i = 0; i + 1 < kAhead; ++i) raws[i] = raws[i + 1];
    raws[kAhead - 1] = load(ahead);
    advance(ahead);
    const int t = cur.t, h = cur.h;
    advance(cur);
    // a row without a position is left alone; one without a page is not stored, its q still turned
    if (place_seq[t] < 0 || place_pos[t] < 0) continue;
    const int64_t r = r0 + t;
    float x[8];
    unpack_halves<kBf>(raw, x);
    const bool is_v = h >= kvh && h < 2 * kvh;
    if (!is_v && a.rot_dim) {  // x cos + partner (-+ sin)
      uint4 other;
      other.x = __shfl_sync(gmask, raw.x, src);
      other.y = __shfl_sync(gmask, raw.y, src);
      other.z = __shfl_sync(gmask, raw.z, src);
      other.w = __shfl_sync(gmask, raw.w, src);
      if (a.interleaved) {  // the partners are the neighbours
        other.x = __funnelshift_l(other.x, other.x, 16);
        other.y = __funnelshift_l(other.y, other.y, 16);
        other.z = __funnelshift_l(other.z, other.z, 16);
        other.w = __funnelshift_l(other.w, other.w, 16);
      }
      if (turned) {
        float y[8];
        unpack_halves<kBf>(other, y);
#pragma unroll
        for (int e = 0; e < 8; ++e) {  // (one by one: the packed forms are contracted to a fused multiply-add)
          const float2 f = cs[t][e][c];
          x[e] = __fadd_rn(__fmul_rn(x[e], f.x), __fmul_rn(y[e], f.y));
        }
      }
    }
    if (h >= 2 * kvh) {  // q
      if (on)
        st_row8<kVec>(a.q_out + r * a.ldqo + (h - 2 * kvh) * hd + 8 * c,
                      make_uint4(pack_halves<kBf>(x[0], x[1]), pack_halves<kBf>(x[2], x[3]), pack_halves<kBf>(x[4], x[5]),
                                 pack_halves<kBf>(x[6], x[7])));
      continue;
    }
    if (place[t] < 0) continue;
    // scale, zero and codes of the head
    float lo = INFINITY, hi = -INFINITY;
    bool bad = false;
    if (on) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        lo = fminf(lo, x[e]);
        hi = fmaxf(hi, x[e]);
        bad |= !(fabsf(x[e]) < INFINITY);
      }
    }
#pragma unroll
    for (int o = kLpr / 2; o > 0; o >>= 1) {
      lo = fminf(lo, __shfl_xor_sync(gmask, lo, o));
      hi = fmaxf(hi, __shfl_xor_sync(gmask, hi, o));
    }
    bad = (__ballot_sync(gmask, bad) & gmask) != 0;
    const float big = fmaxf(fabsf(lo), fabsf(hi));
    const float want = fmaxf(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f), big * 0x1p-10f);
    const float scale = fmaxf(__half2float(__float2half_rn(want)), 0x1p-24f);
    bad |= !(scale < INFINITY);
    const __half zero16 = __float2half_rn(__fdiv_rn(lo, scale));
    const float zero = __half2float(zero16), inv = __frcp_rn(scale);
    // code = round(x / scale - zero) clamped: 2^23 + n has n in its low bits, and its other bits add up to
    // a constant over the word
    uint32_t word = 0;
#pragma unroll
    for (int e = 7; e >= 0; --e) {
      const float n = fminf(fmaxf(__fsub_rn(__fmul_rn(x[e], inv), zero), 0.f), 15.f);
      word = word * 16u + __float_as_uint(__fadd_rn(n, 8388608.f));
    }
    word -= 0x4b000000u * 0x11111111u;
    uint32_t pair = static_cast<uint32_t>(__half_as_ushort(__float2half_rn(scale))) |
                    (static_cast<uint32_t>(__half_as_ushort(zero16)) << 16);
    if (bad) {  // an infinity, a NaN, or values beyond the scale's range
      word = 0;
      pair = 0x00007fffu;  // scale NaN, zero 0
    }
    const int head = is_v ? h - kvh : h;
    const int off = place_pos[t] & (a.C.page_size - 1);
    uint8_t* block = a.C.pages + place[t] + head * a.C.head_bytes;
    const int codes = a.C.page_size * (hd >> 1);
    if (on) *reinterpret_cast<uint32_t*>(block + (is_v ? codes : 0) + off * (hd >> 1) + 4 * c) = word;
    if (c == 0) *reinterpret_cast<uint32_t*>(block + 2 * codes + (is_v ? 4 * a.C.page_size : 0) + 4 * off) = pair;
  }
}

// ------------------------------------------------------------------------------------------------
// Read back
// ------------------------------------------------------------------------------------------------
struct KvReadArgs {
  KvGeom C;
  KvRows B;
  uint16_t *k, *v;
  int64_t ldk, ldv;
};

// The batch's rows as the cache holds them: one CTA per row, kLpr lanes per head (k heads, then v).
// Measured, 8 kv heads of 128: one row 2.7 us; 5217 rows 12.0 us, 2.3 TB/s of what is read and written: each
// of the four to five waves of CTAs is a chain of dependent loads (starts, length, page table, codes).
template <int kLpr, bool kBf, bool kVec>
__global__ void __launch_bounds__(kKvAppendThreads) kv_read_kernel(const KvReadArgs a) {
  __shared__ int64_t sm_place;
  __shared__ int sm_off;
  const int tid = threadIdx.x, lane = tid & 31, r = blockIdx.x;
  griddep_wait();
  griddep_launch_dependents();
  if (tid < 32) {
    const KvRowPlace p = kv_row_place(a.B, r, lane);
    if (lane == 0) {
      sm_place = kv_place(a.C, a.B, p);
      sm_off = p.pos & (a.C.page_size - 1);
    }
  }
  __syncthreads();
  if (sm_place < 0) return;
  const int hd = a.C.hd, kvh = a.C.kv_heads, c = tid % kLpr;
  if (c >= (hd >> 3)) return;
  const int codes = a.C.page_size * (hd >> 1), off = sm_off;
  for (int h = tid / kLpr; h < 2 * kvh; h += kKvAppendThreads / kLpr) {
    const bool is_v = h >= kvh;
    const int head = is_v ? h - kvh : h;
    const uint8_t* block = a.C.pages + sm_place + head * a.C.head_bytes;
    const uint32_t word = *reinterpret_cast<const uint32_t*>(block + (is_v ? codes : 0) + off * (hd >> 1) + 4 * c);
    const uint32_t pair =
        *reinterpret_cast<const uint32_t*>(block + 2 * codes + (is_v ? 4 * a.C.page_size : 0) + 4 * off);
    const float scale = half_lo<false>(pair), zero = half_hi<false>(pair);
    uint32_t w[4];
    const auto value = [&](int n) {
      const float x = scale * (static_cast<float>((word >> (4 * n)) & 15u) + zero);
      if (kBf) return x;
      return x > 65504.f ? 65504.f : x < -65504.f ? -65504.f : x;  // (a NaN stays one)
    };
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pack_halves<kBf>(value(2 * i), value(2 * i + 1));
    uint16_t* dst = is_v ? a.v + r * a.ldv : a.k + r * a.ldk;
    st_row8<kVec>(dst + head * hd + 8 * c, make_uint4(w[0], w[1], w[2], w[3]));
  }
}

}  // namespace opc
