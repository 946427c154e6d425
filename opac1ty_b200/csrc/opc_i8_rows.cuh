// opc_i8_rows.cuh -- rows of 16- or 32-bit values brought into 8 bits with one scale a row, fused
// with what comes before them in a transformer block:
//   kI8Quant  v = x
//   kI8Norm   t = h + y, h_out = t, v = t * w, and the scale also divided by sqrt(mean t^2 + eps)
//   kI8Silu   v = g / (1 + exp(-g)) * u
// each followed by  a = max |v|, scale = a / 127, code = round(v * 127 / a).
//
// The norm's factor is the same for a whole row, so the codes do not depend on it: the sum of
// squares and the largest magnitude come out of ONE reduction, and every value is read once and kept
// in registers between the reduction and the rounding.  Bound by memory for large calls, which takes
// few enough instructions per value that it stays so: pairs of values in packed fp32 operations, one
// maximum of three per two values (device time with L2 flushed by the inputs: 8191 x 4096 fp32 + fp16 norms
// with values 67 us, 6.5 TB/s; 4097 x 14336 fp16 gated with values 61 us, 6.8 TB/s; 28672 x 4096 fp16
// quantized with values 87 us, 6.8 TB/s: of bytes read and written, part of which are still in L2 at the end; memory
// itself moves 5.8 to 6.0).  opc_i8.cu has how rows are dealt to threads.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>

#include "opc_device.cuh"

namespace opc {

enum : int { kI8Quant = 0, kI8Norm = 1, kI8Silu = 2 };
enum : int { kI8F16 = 0, kI8BF16 = 1, kI8F32 = 2, kI8None = 3 };  // element types (OPC_F16, ...)

constexpr float kI8Least = 7.888609052210118e-31f;  // 2^-100: rows below it are zeros

struct I8RowsArgs {
  const void* x;      // quantize: x; norm: h; silu: gate
  const void* u;      // norm: y (or NULL); silu: up
  const void* w;      // norm: weight (or NULL), element type w_type
  void* h_out;        // norm: h + y (or NULL)
  int8_t* codes;
  float* scales;
  void* values;       // what the codes stand for (or NULL), element type v_type
  void* plain;        // norm (kPlain): the normalized row as formed, element type v_type, rows ldv apart
  int64_t ldx, ldu, ldh, ldc, ldv;
  int32_t rows, n, w_type, v_type;
  float eps, inv_n;   // norm: 1 / n
};

// Two fp32 values, one instruction for both.
using I8Pair = unsigned long long;
__device__ __forceinline__ I8Pair i8_pair(float a, float b) {
  I8Pair p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(a), "f"(b));
  return p;
}
__device__ __forceinline__ float2 i8_both(I8Pair p) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p));
  return f;
}
__device__ __forceinline__ I8Pair i8_mul2(I8Pair a, I8Pair b) {
  I8Pair d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ I8Pair i8_add2(I8Pair a, I8Pair b) {
  I8Pair d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ I8Pair i8_sub2(I8Pair a, I8Pair b) {
  I8Pair d;
  asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ I8Pair i8_fma2(I8Pair a, I8Pair b, I8Pair c) {
  I8Pair d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
// max(|a|, |b|, |c|), NaN if one of them is.
__device__ __forceinline__ float i8_max3(float a, float b, float c) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// A thread's group of 8 values: with kVec, 8 in a row, moved 16 bytes at a time (every row of every operand
// starts on 16 bytes); else every 32nd of 256, so that a warp's loads and stores of single values are still
// of neighbours (4096 x 4097 fp16 quantized: 47.8 us with 8 in a row, 20.8 so).
template <bool kVec>
__device__ __forceinline__ int i8_first(int group) {
  return kVec ? 8 * group : 256 * (group >> 5) + (group & 31);
}
template <bool kVec>
constexpr int i8_stride() {
  return kVec ? 1 : 32;
}
template <bool kVec>
__device__ __forceinline__ bool i8_whole(int left) {  // `left`: values of the row from the group's first on
  return left > 7 * i8_stride<kVec>();
}

// 8 values as they lie in memory.
template <int kT>
struct I8Raw {
  uint4 a, b;  // (b: the second half of 32-bit values)
};

// Zeros for those beyond the row.
template <int kT, bool kVec>
__device__ __forceinline__ void i8_load8(const void* base, int64_t at, int left, I8Raw<kT>& r) {
  constexpr int kStep = i8_stride<kVec>();
  using T = typename std::conditional<kT == kI8F32, uint32_t, uint16_t>::type;
  const T* p = static_cast<const T*>(base) + at;
  if (kVec && i8_whole<kVec>(left)) {
    r.a = *reinterpret_cast<const uint4*>(p);
    if constexpr (kT == kI8F32) r.b = *reinterpret_cast<const uint4*>(p + 4);
    return;
  }
  uint32_t v[8];
  if (i8_whole<kVec>(left)) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = p[kStep * i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = kStep * i < left ? p[kStep * i] : 0u;
  }
  if constexpr (kT == kI8F32) {
    r.a = make_uint4(v[0], v[1], v[2], v[3]);
    r.b = make_uint4(v[4], v[5], v[6], v[7]);
  } else {
    r.a = make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
  }
}
template <int kT>
__device__ __forceinline__ void i8_open8(const I8Raw<kT>& r, I8Pair (&v)[4]) {
  const uint32_t a[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
  if constexpr (kT == kI8F32) {
    const uint32_t b[4] = {r.b.x, r.b.y, r.b.z, r.b.w};
    v[0] = i8_pair(__uint_as_float(a[0]), __uint_as_float(a[1]));
    v[1] = i8_pair(__uint_as_float(a[2]), __uint_as_float(a[3]));
    v[2] = i8_pair(__uint_as_float(b[0]), __uint_as_float(b[1]));
    v[3] = i8_pair(__uint_as_float(b[2]), __uint_as_float(b[3]));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (kT == kI8BF16) {  // a bf16 is the upper half of an fp32
        v[i] = i8_pair(__uint_as_float(a[i] << 16), __uint_as_float(a[i] & 0xffff0000u));
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&a[i]));
        v[i] = i8_pair(f.x, f.y);
      }
    }
  }
}
template <bool kVec>
__device__ __forceinline__ void i8_load8_of(int type, const void* base, int64_t at, int left, I8Pair (&v)[4]) {
  if (type == kI8F16) {
    I8Raw<kI8F16> r;
    i8_load8<kI8F16, kVec>(base, at, left, r);
    i8_open8(r, v);
  } else if (type == kI8BF16) {
    I8Raw<kI8BF16> r;
    i8_load8<kI8BF16, kVec>(base, at, left, r);
    i8_open8(r, v);
  } else {
    I8Raw<kI8F32> r;
    i8_load8<kI8F32, kVec>(base, at, left, r);
    i8_open8(r, v);
  }
}

template <int kT, bool kVec>
__device__ __forceinline__ void i8_store8(void* base, int64_t at, int left, const I8Pair (&v)[4]) {
  constexpr int kStep = i8_stride<kVec>();
  using T = typename std::conditional<kT == kI8F32, uint32_t, uint16_t>::type;
  T* p = static_cast<T*>(base) + at;
  uint32_t w[8];  // fp32 values, or pairs of 16-bit ones in the first four
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = i8_both(v[i]);
    if constexpr (kT == kI8F32) {
      w[2 * i] = __float_as_uint(f.x);
      w[2 * i + 1] = __float_as_uint(f.y);
    } else if constexpr (kT == kI8BF16) {
      const __nv_bfloat162 b = __floats2bfloat162_rn(f.x, f.y);
      w[i] = *reinterpret_cast<const uint32_t*>(&b);
    } else {
      const __half2 b = __floats2half2_rn(f.x, f.y);
      w[i] = *reinterpret_cast<const uint32_t*>(&b);
    }
  }
  const bool whole = i8_whole<kVec>(left);
  if (kVec && whole) {
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    if constexpr (kT == kI8F32) *reinterpret_cast<uint4*>(p + 4) = make_uint4(w[4], w[5], w[6], w[7]);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (whole || kStep * i < left) {
      if constexpr (kT == kI8F32) p[kStep * i] = w[i];
      else p[kStep * i] = static_cast<uint16_t>(w[i >> 1] >> (16 * (i & 1)));
    }
}
template <bool kVec>
__device__ __forceinline__ void i8_store8_of(int type, void* base, int64_t at, int left, const I8Pair (&v)[4]) {
  if (type == kI8F16) i8_store8<kI8F16, kVec>(base, at, left, v);
  else if (type == kI8BF16) i8_store8<kI8BF16, kVec>(base, at, left, v);
  else i8_store8<kI8F32, kVec>(base, at, left, v);
}

// What a row's reduction carries: max |v| (NaN if a value is), and for the norm two sums of squares,
// of t and of t * 2^-80; the second holds where the first leaves the range of fp32.
struct I8Stat {
  float big;
  I8Pair ss, small;  // sums of even and odd places
};
struct I8Row {
  float big, ss, small;
};

__device__ __forceinline__ void i8_warp_reduce(I8Row& s, bool norm) {
  s.big = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(s.big)));  // (not negative; a NaN's bits are the largest)
  if (norm) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      s.ss += __shfl_xor_sync(0xffffffffu, s.ss, o);
      s.small += __shfl_xor_sync(0xffffffffu, s.small, o);
    }
  }
}
// Over the row's threads; every one gets the result.  Sums in one order, whatever the timing.
template <bool kWarpRow>
__device__ __forceinline__ I8Row i8_reduce(const I8Stat& p, bool norm) {
  I8Row s;
  s.big = p.big;
  s.ss = s.small = 0.f;
  if (norm) {
    const float2 a = i8_both(p.ss), b = i8_both(p.small);
    s.ss = a.x + a.y;
    s.small = b.x + b.y;
  }
  i8_warp_reduce(s, norm);
  if constexpr (kWarpRow) return s;
  __shared__ float part_big[32], part_ss[32], part_small[32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  if (lane == 0) {
    part_big[warp] = s.big;
    if (norm) {
      part_ss[warp] = s.ss;
      part_small[warp] = s.small;
    }
  }
  __syncthreads();
  s.big = lane < warps ? part_big[lane] : 0.f;
  if (norm) {
    s.ss = lane < warps ? part_ss[lane] : 0.f;
    s.small = lane < warps ? part_small[lane] : 0.f;
  }
  i8_warp_reduce(s, norm);
  return s;
}

// How a code is made of a value.  kI8Product: round(v * mul).  The others: round(q), q nearly the quotient (v * c) / a with
// c = 127 and a the largest magnitude, or both times 2^-32 where v * 127 could leave fp32; inv = 1 / a.  kI8Quotient
// takes v * c as rounded to fp32 (v of 16 bits: it needs no rounding), kI8Quotient2 with what the rounding left out.
enum : int { kI8Product = 0, kI8Quotient = 1, kI8Quotient2 = 2 };
// What the codes are made with.
// `live` is false for rows of zeros and rows that hold an infinity or NaN, whose codes are 0 whatever v is.
// Every thread forms them, so they cost as much as several values do: reciprocals to a step or two of
// fp32 and their products instead of divisions (4097 x 14336 gated 77 -> 47 us).
struct I8Scale {
  float scale, mul, c, a, inv;
  float factor;  // norm: 1 / sqrt(mean t^2 + eps)
  bool live;
};
__device__ __forceinline__ float i8_recip(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ I8Scale i8_scale_of(const I8Row& s, const I8RowsArgs& a, bool norm) {
  I8Scale r;
  const bool bad = !(s.big < __uint_as_float(0x7f800000u));
  r.live = !bad && s.big >= kI8Least;
  const bool huge = s.big >= 0x1p97f;
  r.c = huge ? 127.0f * 0x1p-32f : 127.0f;
  r.a = huge ? s.big * 0x1p-32f : s.big;
  r.inv = i8_recip(r.a);
  r.mul = r.c * r.inv;
  const float q = s.big * (1.0f / 127.0f);
  r.scale = fmaf(fmaf(-q, 127.0f, s.big), 1.0f / 127.0f, q);  // big / 127, the nearest fp32
  if (norm) {
    // a finite row whose squares leave fp32: mean (t 2^-80)^2 (eps is nothing beside it)
    const bool far = !(s.ss < __uint_as_float(0x7f800000u));
    float root;
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(root) : "f"(far ? s.small * a.inv_n : fmaf(s.ss, a.inv_n, a.eps)));
    r.factor = far ? root * 0x1p-80f : root;
    r.scale *= r.factor;
  }
  r.scale = bad ? __uint_as_float(0x7fffffffu) : r.live ? r.scale : 0.f;
  return r;
}

// Codes (and values) of 8 values.  Adding 1.5 * 2^23 rounds to a whole number, to even, whose lowest
// byte is the code.  A quotient is v * c times inv, off by two steps at most, corrected once by its remainder: within
// 2^-21 steps of the true one before its last rounding, so the nearest fp32 but where two are that nearly as near.  For
// values of 16 bits, whose quotients are halves or 2^-12 away from them, a half is a half and goes to even (with v *
// (127 / a) every half of a row goes the way that 127 / a was rounded).  kI8Quotient2 costs nothing where rows are
// read from memory and quantized (16384 x 4096 fp32: 69.4 us with and without), but two registers a thread, which a
// norm of fp32 rows would pay with a CTA an SM (8191 x 4096: 38.6 -> 41.3 us): its v * c keeps its rounding.  Rows
// that were added or gated, whose values are rounded themselves, take the product; so do 16-bit rows whose sum happened
// to be exact.
template <bool kLive, int kHow, bool kVec>
__device__ __forceinline__ void i8_write8(const I8RowsArgs& a, int row, int i, int left, const I8Pair (&v)[4], const I8Scale& s) {
  constexpr float kMagic = 12582912.0f;
  const I8Pair magic = i8_pair(kMagic, kMagic);
  I8Pair f[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (!kLive) {
      f[e] = magic;
    } else if constexpr (kHow != kI8Product) {
      const I8Pair inv = i8_pair(s.inv, s.inv), t = i8_mul2(v[e], i8_pair(s.c, s.c)), q = i8_mul2(t, inv);
      I8Pair r = i8_fma2(q, i8_pair(-s.a, -s.a), t);
      if constexpr (kHow == kI8Quotient2) r = i8_sub2(r, i8_fma2(v[e], i8_pair(-s.c, -s.c), t));
      f[e] = i8_add2(i8_fma2(r, inv, q), magic);
    } else {
      f[e] = i8_fma2(v[e], i8_pair(s.mul, s.mul), magic);
    }
  }
  uint32_t q[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const float2 lo = i8_both(f[2 * e]), hi = i8_both(f[2 * e + 1]);
    q[e] = __byte_perm(__byte_perm(__float_as_uint(lo.x), __float_as_uint(lo.y), 0x0040),
                       __byte_perm(__float_as_uint(hi.x), __float_as_uint(hi.y), 0x0040), 0x5410);
  }
  int8_t* c = a.codes + static_cast<int64_t>(row) * a.ldc + i;
  const bool whole = i8_whole<kVec>(left);
  if (kVec && whole) {
    *reinterpret_cast<uint2*>(c) = make_uint2(q[0], q[1]);  // (codes start on 16 bytes, rows too)
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (whole || i8_stride<kVec>() * e < left) c[i8_stride<kVec>() * e] = static_cast<int8_t>(q[e >> 2] >> (8 * (e & 3)));
  }
  if (a.values) {
    I8Pair o[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = i8_mul2(i8_add2(f[e], i8_pair(-kMagic, -kMagic)), i8_pair(s.scale, s.scale));
    i8_store8_of<kVec>(a.v_type, a.values, static_cast<int64_t>(row) * a.ldv + i, left, o);
  }
}

// 8 normalized values, not brought into 8 bits.
template <bool kVec>
__device__ __forceinline__ void i8_write_plain(const I8RowsArgs& a, int row, int i, int left, const I8Pair (&v)[4], float factor) {
  I8Pair o[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = i8_mul2(v[e], i8_pair(factor, factor));
  i8_store8_of<kVec>(a.v_type, a.plain, static_cast<int64_t>(row) * a.ldv + i, left, o);
}

__device__ __forceinline__ float i8_ex2(float x) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x));
  return e;
}
// silu(g) * u.  exp(-g) = 2^(-g log2 e): the rounded product is off by |g log2 e| 2^-24 at most and its constant by a
// quarter of that, so the power by |g| 2^-23.6 of itself, which next to the row's largest value is nothing where |g|
// is large; 1 / (1 + it) to one step of fp32.  Below -44 that quotient is 1 / power to fp32, but it would be flushed to 0
// from -87.4 on and its power infinite from -88.8 on, while a large u brings the product back into the range of live
// rows: there it is the square of 1 / (1 + 2^(-g log2 e / 2)), one factor before u and one after, normal down to -174
// (where the product is below 2^-100, whatever u is).  Two predicated products a value: 4097 x 14336 gated 60.6 us with
// and without, 2048 x 28672 91.9 and 89.0 us.
__device__ __forceinline__ I8Pair i8_silu_mul2(I8Pair g, I8Pair u) {
  const float2 f = i8_both(g);
  float2 z = i8_both(i8_mul2(g, i8_pair(-1.4426950408889634f, -1.4426950408889634f)));
  const bool far0 = f.x < -44.0f, far1 = f.y < -44.0f;
  if (far0) z.x *= 0.5f;
  if (far1) z.y *= 0.5f;
  const float2 d = i8_both(i8_add2(i8_pair(i8_ex2(z.x), i8_ex2(z.y)), i8_pair(1.0f, 1.0f)));
  const float r0 = i8_recip(d.x), r1 = i8_recip(d.y);
  float2 v = i8_both(i8_mul2(i8_mul2(g, i8_pair(r0, r1)), u));
  if (far0) v.x *= r0;
  if (far1) v.y *= r1;
  return i8_pair(v.x, v.y);
}

// 8 values of a row before its scale from what was loaded, their part of the statistics, and (norm) h_out.
template <int kOp, int kTX, int kTU, bool kVec, bool kWriteH>
__device__ __forceinline__ void i8_make8(const I8RowsArgs& a, int row, int i, const I8Raw<kTX>& rx, const I8Raw<kTU>& ru, I8Pair (&v)[4],
                                         I8Stat& s) {
  const int left = a.n - i;
  i8_open8(rx, v);
  if constexpr (kTU != kI8None) {
    I8Pair u[4];
    i8_open8(ru, u);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (kOp == kI8Silu) {
        v[e] = i8_silu_mul2(v[e], u[e]);
      } else {
        v[e] = i8_add2(v[e], u[e]);
      }
    }
  }
  if constexpr (kOp == kI8Norm) {
    if (kWriteH && a.h_out) i8_store8<kTX, kVec>(a.h_out, static_cast<int64_t>(row) * a.ldh + i, left, v);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      s.ss = i8_fma2(v[e], v[e], s.ss);
      const I8Pair t = i8_mul2(v[e], i8_pair(0x1p-80f, 0x1p-80f));
      s.small = i8_fma2(t, t, s.small);
    }
    if (a.w) {
      I8Pair w[4];
      i8_load8_of<kVec>(a.w_type, a.w, i, left, w);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = i8_mul2(v[e], w[e]);
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 f = i8_both(v[e]);
    s.big = i8_max3(s.big, f.x, f.y);
  }
}

// CTAs of 1024 threads that an SM is to hold, where 32 registers a thread do for that: a CTA alone leaves
// the memory idle while it reduces (4097 x 14336 gated: 72 us with one CTA an SM, 48 with two).
constexpr int i8_resident(int op, int x, int per, bool warp_row) {
  return !warp_row && per < 4 && (op == kI8Quant || (op == kI8Silu && x != kI8F32)) ? 2 : 1;
}

// One row per CTA (kWarpRow: per warp), kPer groups of 8 values per thread in registers; kPer 0: rows
// of any length, read once for the statistics and once more for the codes.  kPlain (kPer 0): the normalized row is
// written too, as formed.
template <int kOp, int kTX, int kTU, int kPer, bool kWarpRow, bool kVec, bool kPlain = false>
__global__ void __launch_bounds__(kWarpRow ? 128 : 1024, i8_resident(kOp, kTX, kPer, kWarpRow)) i8_rows_kernel(const I8RowsArgs a) {
  griddep_wait();
  griddep_launch_dependents();
  const int threads = kWarpRow ? 32 : blockDim.x;
  const int t = kWarpRow ? threadIdx.x & 31 : threadIdx.x;
  const int row = kWarpRow ? blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
  if (kWarpRow && row >= a.rows) return;
  constexpr bool kNorm = kOp == kI8Norm;
  constexpr int kHow = kOp == kI8Silu || kTU != kI8None ? kI8Product : kOp == kI8Quant && kTX == kI8F32 ? kI8Quotient2 : kI8Quotient;
  I8Stat s{0.f, 0ull, 0ull};
  // groups whose loads are all under way before the first is used (two of 64 registers would not stay in them)
  constexpr int kBatch = kPer < 2 || (kPer == 4 && kTX == kI8F32 && kTU == kI8F32) ? 1 : 2;
  I8Raw<kTX> rx[kBatch];
  I8Raw<kTU> ru[kBatch];
  const auto load = [&](int i, int j) {
    i8_load8<kTX, kVec>(a.x, static_cast<int64_t>(row) * a.ldx + i, a.n - i, rx[j]);
    if constexpr (kTU != kI8None) i8_load8<kTU, kVec>(a.u, static_cast<int64_t>(row) * a.ldu + i, a.n - i, ru[j]);
  };
  if constexpr (kPer > 0) {
    I8Pair v[kPer][4];
#pragma unroll
    for (int j0 = 0; j0 < kPer; j0 += kBatch) {
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int i = i8_first<kVec>(t + (j0 + j) * threads);
        if (i < a.n) load(i, j);
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int i = i8_first<kVec>(t + (j0 + j) * threads);
        if (i < a.n) i8_make8<kOp, kTX, kTU, kVec, true>(a, row, i, rx[j], ru[j], v[j0 + j], s);
      }
    }
    const I8Scale sc = i8_scale_of(i8_reduce<kWarpRow>(s, kNorm), a, kNorm);
    if (t == 0) a.scales[row] = sc.scale;
    if (sc.live) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const int i = i8_first<kVec>(t + j * threads);
        if (i < a.n) i8_write8<true, kHow, kVec>(a, row, i, a.n - i, v[j], sc);
      }
    } else {
#pragma unroll 1
      for (int g = t, i; (i = i8_first<kVec>(g)) < a.n; g += threads) i8_write8<false, kHow, kVec>(a, row, i, a.n - i, v[0], sc);
    }
  } else {
    I8Pair v[4];
    for (int g = t, i; (i = i8_first<kVec>(g)) < a.n; g += threads) {
      load(i, 0);
      i8_make8<kOp, kTX, kTU, kVec, false>(a, row, i, rx[0], ru[0], v, s);
    }
    const I8Scale sc = i8_scale_of(i8_reduce<kWarpRow>(s, kNorm), a, kNorm);
    if (t == 0) a.scales[row] = sc.scale;
    I8Stat none{0.f, 0ull, 0ull};
    for (int g = t, i; (i = i8_first<kVec>(g)) < a.n; g += threads) {  // (h_out may be h: each thread reads a place before it writes it)
      load(i, 0);
      i8_make8<kOp, kTX, kTU, kVec, true>(a, row, i, rx[0], ru[0], v, none);
      if constexpr (kPlain) i8_write_plain<kVec>(a, row, i, a.n - i, v, sc.factor);
      if (sc.live) i8_write8<true, kHow, kVec>(a, row, i, a.n - i, v, sc);
      else i8_write8<false, kHow, kVec>(a, row, i, a.n - i, v, sc);
    }
  }
}

}  // namespace opc
