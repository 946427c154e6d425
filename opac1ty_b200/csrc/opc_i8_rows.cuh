// opc_i8_rows.cuh -- rows of 16- or 32-bit values brought into 8 bits with one scale a row, fused
// with what comes before them in a transformer block:
//   kI8Quant  v = x
//   kI8Norm   t = h + y, h_out = t, v = t * w, and the scale also divided by sqrt(mean t^2 + eps)
//   kI8Silu   v = g / (1 + exp(-g)) * u
// each followed by  a = max |v|, scale = a / 127, code = round(v * 127 / a).
//
// The norm's factor is the same for a whole row, so the codes do not depend on it: the sum of
// squares and the largest magnitude come out of ONE reduction, and every value is read once and kept
// in registers between the reduction and the rounding.  Memory bound; see opc_i8.cu for how rows are
// dealt to threads.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "opc_device.cuh"

namespace opc {

enum : int { kI8Quant = 0, kI8Norm = 1, kI8Silu = 2 };
enum : int { kI8F16 = 0, kI8BF16 = 1, kI8F32 = 2, kI8None = 3 };  // element types (OPC_F16, ...)

constexpr float kI8Least = 7.888609052210118e-31f;  // 2^-100: rows below it are zeros
constexpr int kI8MaxPer = 4;                         // most groups of 8 values a thread keeps in registers

struct I8RowsArgs {
  const void* x;      // quantize: x; norm: h; silu: gate
  const void* u;      // norm: y (or NULL); silu: up
  const void* w;      // norm: weight (or NULL), element type w_type
  void* h_out;        // norm: h + y (or NULL)
  int8_t* codes;
  float* scales;
  void* values;       // what the codes stand for (or NULL), element type v_type
  int64_t ldx, ldu, ldh, ldc, ldv;
  int32_t rows, n, w_type, v_type;
  // groups of 8 values that may be moved 16 bytes at a time (else one value at a time)
  int32_t vec_x, vec_u, vec_w, vec_h, vec_v, vec_c;
  float eps;
};

// 8 values at p (element type kT) as fp32; with !vec, or fewer than 8 left, one at a time, zeros after them.
template <int kT>
__device__ __forceinline__ void i8_load8(const void* base, int64_t at, int left, bool vec, float (&v)[8]) {
  if constexpr (kT == kI8F32) {
    const float* p = static_cast<const float*>(base) + at;
    if (vec && left >= 8) {
      const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = i < left ? p[i] : 0.f;
    }
  } else {
    const uint16_t* p = static_cast<const uint16_t*>(base) + at;
    uint32_t h[4];
    if (vec && left >= 8) {
      const uint4 a = *reinterpret_cast<const uint4*>(p);
      h[0] = a.x; h[1] = a.y; h[2] = a.z; h[3] = a.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        h[i] = (2 * i < left ? p[2 * i] : 0u) | (2 * i + 1 < left ? static_cast<uint32_t>(p[2 * i + 1]) << 16 : 0u);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (kT == kI8BF16) {  // a bf16 is the upper half of an fp32
        v[2 * i] = __uint_as_float(h[i] << 16);
        v[2 * i + 1] = __uint_as_float(h[i] & 0xffff0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      }
    }
  }
}
__device__ __forceinline__ void i8_load8_of(int type, const void* base, int64_t at, int left, bool vec, float (&v)[8]) {
  if (type == kI8F16) i8_load8<kI8F16>(base, at, left, vec, v);
  else if (type == kI8BF16) i8_load8<kI8BF16>(base, at, left, vec, v);
  else i8_load8<kI8F32>(base, at, left, vec, v);
}

template <int kT>
__device__ __forceinline__ void i8_store8(void* base, int64_t at, int left, bool vec, const float (&v)[8]) {
  if constexpr (kT == kI8F32) {
    float* p = static_cast<float*>(base) + at;
    if (vec && left >= 8) {
      *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < left) p[i] = v[i];
    }
  } else {
    uint16_t* p = static_cast<uint16_t*>(base) + at;
    uint32_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (kT == kI8BF16) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        h[i] = *reinterpret_cast<const uint32_t*>(&b);
      } else {
        const __half2 b = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        h[i] = *reinterpret_cast<const uint32_t*>(&b);
      }
    }
    if (vec && left >= 8) {
      *reinterpret_cast<uint4*>(p) = make_uint4(h[0], h[1], h[2], h[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < left) p[i] = static_cast<uint16_t>(h[i >> 1] >> (16 * (i & 1)));
    }
  }
}
__device__ __forceinline__ void i8_store8_of(int type, void* base, int64_t at, int left, bool vec, const float (&v)[8]) {
  if (type == kI8F16) i8_store8<kI8F16>(base, at, left, vec, v);
  else if (type == kI8BF16) i8_store8<kI8BF16>(base, at, left, vec, v);
  else i8_store8<kI8F32>(base, at, left, vec, v);
}

// What a row's reduction carries: max |v| as bits (a NaN's are above infinity's, so it is kept), the
// sum of t^2, and the same of t * 2^-80, which holds where the first one leaves the range of fp32.
struct I8Stat {
  uint32_t big;
  float ss, small;
};

__device__ __forceinline__ void i8_warp_reduce(I8Stat& s, bool norm) {
  s.big = __reduce_max_sync(0xffffffffu, s.big);
  if (norm) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      s.ss += __shfl_xor_sync(0xffffffffu, s.ss, o);
      s.small += __shfl_xor_sync(0xffffffffu, s.small, o);
    }
  }
}
// Over the CTA; every thread gets the result.  Sums in one order, whatever the timing.
__device__ __forceinline__ void i8_block_reduce(I8Stat& s, bool norm) {
  __shared__ uint32_t part_big[32];
  __shared__ float part_ss[32], part_small[32];
  i8_warp_reduce(s, norm);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  if (lane == 0) {
    part_big[warp] = s.big;
    if (norm) {
      part_ss[warp] = s.ss;
      part_small[warp] = s.small;
    }
  }
  __syncthreads();
  s.big = lane < warps ? part_big[lane] : 0u;
  if (norm) {
    s.ss = lane < warps ? part_ss[lane] : 0.f;
    s.small = lane < warps ? part_small[lane] : 0.f;
  }
  i8_warp_reduce(s, norm);
}

// What the codes are made with: code = round((v * c) / a) with c = 127 and a the largest magnitude, or
// both times 2^-32 where v * 127 could leave fp32; inv = 1 / a.  `live` is false for rows of zeros and
// rows that hold an infinity or NaN, whose codes are 0 whatever v is.
struct I8Scale {
  float scale, c, a, inv;
  bool live;
};
__device__ __forceinline__ I8Scale i8_scale_of(const I8Stat& s, bool norm, int n, float eps) {
  I8Scale r;
  const float big = __uint_as_float(s.big);
  const bool bad = s.big >= 0x7f800000u;
  r.live = !bad && big >= kI8Least;
  const bool huge = s.big >= 0x70000000u;  // 2^97
  r.c = huge ? 127.0f * 0x1p-32f : 127.0f;
  r.a = huge ? big * 0x1p-32f : big;
  r.inv = 1.0f / r.a;
  r.scale = bad ? __uint_as_float(0x7fffffffu) : r.live ? big / 127.0f : 0.f;
  if (norm && r.live) {
    const float len = static_cast<float>(n);
    // a finite row whose squares leave fp32: sqrt(mean (t 2^-80)^2) 2^80 (eps is nothing beside it)
    const float rms = s.ss < __uint_as_float(0x7f800000u) ? sqrtf(s.ss / len + eps) : sqrtf(s.small / len) * 0x1p80f;
    r.scale = r.scale / rms;
  }
  return r;
}

// Codes (and values) of 8 values.  The quotient is corrected once by its remainder, so it is the
// nearest fp32: a half that 16-bit inputs often meet is a half and goes to even (with v * (127 / a)
// every half of a row goes the way that 127 / a was rounded).  Adding 1.5 * 2^23 rounds it to a whole
// number; the lowest byte is the code.
__device__ __forceinline__ void i8_write8(const I8RowsArgs& a, int row, int i, int left, const float (&v)[8], const I8Scale& s) {
  constexpr float kMagic = 12582912.0f;
  float f[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float t = v[e] * s.c, q0 = t * s.inv;
    f[e] = s.live ? __fadd_rn(fmaf(fmaf(-q0, s.a, t), s.inv, q0), kMagic) : kMagic;
  }
  uint32_t q[2];
#pragma unroll
  for (int e = 0; e < 2; ++e)
    q[e] = __byte_perm(__byte_perm(__float_as_uint(f[4 * e]), __float_as_uint(f[4 * e + 1]), 0x0040),
                       __byte_perm(__float_as_uint(f[4 * e + 2]), __float_as_uint(f[4 * e + 3]), 0x0040), 0x5410);
  int8_t* c = a.codes + static_cast<int64_t>(row) * a.ldc + i;
  if (left >= 8) {
    *reinterpret_cast<uint2*>(c) = make_uint2(q[0], q[1]);  // (codes start on 16 bytes, rows too)
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < left) c[e] = static_cast<int8_t>(q[e >> 2] >> (8 * (e & 3)));
  }
  if (a.values) {
    float o[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = (f[e] - kMagic) * s.scale;
    i8_store8_of(a.v_type, a.values, static_cast<int64_t>(row) * a.ldv + i, left, a.vec_v, o);
  }
}

// The 8 values from i on of a row before its scale, their part of the statistics, and (norm) h_out.
template <int kOp, int kTX, int kTU>
__device__ __forceinline__ void i8_make8(const I8RowsArgs& a, int row, int i, float (&v)[8], I8Stat& s, bool write_h) {
  const int left = a.n - i;
  i8_load8<kTX>(a.x, static_cast<int64_t>(row) * a.ldx + i, left, a.vec_x, v);
  if constexpr (kTU != kI8None) {
    float u[8];
    i8_load8<kTU>(a.u, static_cast<int64_t>(row) * a.ldu + i, left, a.vec_u, u);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (kOp == kI8Silu) v[e] = __fdividef(v[e], 1.0f + expf(-v[e])) * u[e];
      else v[e] += u[e];
    }
  }
  if constexpr (kOp == kI8Norm) {
    if (write_h && a.h_out) i8_store8<kTX>(a.h_out, static_cast<int64_t>(row) * a.ldh + i, left, a.vec_h, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      s.ss = fmaf(v[e], v[e], s.ss);
      const float t = v[e] * 0x1p-80f;
      s.small = fmaf(t, t, s.small);
    }
    if (a.w) {
      float w[8];
      i8_load8_of(a.w_type, a.w, i, left, a.vec_w, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= w[e];
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) s.big = max(s.big, __float_as_uint(v[e]) & 0x7fffffffu);
}

// One row per CTA (kWarpRow: per warp), kPer groups of 8 values per thread in registers; kPer 0: rows
// of any length, read once for the statistics and once more for the codes.
template <int kOp, int kTX, int kTU, int kPer, bool kWarpRow>
__global__ void i8_rows_kernel(const I8RowsArgs a) {
  griddep_wait();
  griddep_launch_dependents();
  const int threads = kWarpRow ? 32 : blockDim.x;
  const int t = kWarpRow ? threadIdx.x & 31 : threadIdx.x;
  const int row = kWarpRow ? blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
  if (kWarpRow && row >= a.rows) return;
  constexpr bool kNorm = kOp == kI8Norm;
  I8Stat s{0u, 0.f, 0.f};
  if constexpr (kPer > 0) {
    float v[kPer][8];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int i = 8 * (t + j * threads);
      if (i < a.n) i8_make8<kOp, kTX, kTU>(a, row, i, v[j], s, true);
    }
    if (kWarpRow) i8_warp_reduce(s, kNorm);
    else i8_block_reduce(s, kNorm);
    const I8Scale sc = i8_scale_of(s, kNorm, a.n, a.eps);
    if (t == 0) a.scales[row] = sc.scale;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int i = 8 * (t + j * threads);
      if (i < a.n) i8_write8(a, row, i, a.n - i, v[j], sc);
    }
  } else {
    float v[8];
    for (int i = 8 * t; i < a.n; i += 8 * threads) i8_make8<kOp, kTX, kTU>(a, row, i, v, s, false);
    i8_block_reduce(s, kNorm);
    const I8Scale sc = i8_scale_of(s, kNorm, a.n, a.eps);
    if (t == 0) a.scales[row] = sc.scale;
    I8Stat none{0u, 0.f, 0.f};
    for (int i = 8 * t; i < a.n; i += 8 * threads) {  // (h_out may be h: each thread reads a place before it writes it)
      i8_make8<kOp, kTX, kTU>(a, row, i, v, none, true);
      i8_write8(a, row, i, a.n - i, v, sc);
    }
  }
}

}  // namespace opc
