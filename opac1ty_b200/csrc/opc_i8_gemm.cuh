// opc_i8_gemm.cuh -- Y[t][r] = sx[t] * sw[r] * sum_k X[t][k] W[r][k] (+ bias[r]) over 8-bit integers.
#pragma once

#include "opc_i8_rows.cuh"

namespace opc {

struct I8GemmArgs {
  const int8_t *x, *w;
  const float *sx, *sw;
  const void* bias;
  void* y;
  int64_t ldx, ldw, ldy;
  int32_t rows, M, K, bias_type, y_type;
};

__device__ __forceinline__ float i8_load1(int type, const void* p, int64_t i) {
  if (type == kI8F16) return __half2float(static_cast<const __half*>(p)[i]);
  if (type == kI8BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return static_cast<const float*>(p)[i];
}
__device__ __forceinline__ void i8_store1(int type, void* p, int64_t i, float v) {
  if (type == kI8F16) static_cast<__half*>(p)[i] = __float2half_rn(v);
  else if (type == kI8BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else static_cast<float*>(p)[i] = v;
}

// 64 tokens x 64 channels per CTA, K 64 at a time through shared memory, 4 x 4 sums a thread.
__global__ void __launch_bounds__(256) i8_gemm_simple(const I8GemmArgs a) {
  __shared__ int32_t sx[64][17], sw[64][17];
  griddep_wait();
  griddep_launch_dependents();
  const int r0 = blockIdx.x * 64, t0 = blockIdx.y * 64;
  const int tr = threadIdx.x & 15, tt = threadIdx.x >> 4;
  int32_t acc[4][4] = {};
  for (int k0 = 0; k0 < a.K; k0 += 64) {
    for (int i = threadIdx.x; i < 64 * 16; i += 256) {
      const int row = i >> 4, c = i & 15;
      uint32_t xv = 0, wv = 0;
      for (int b = 0; b < 4; ++b) {
        const int k = k0 + 4 * c + b;
        if (k < a.K && t0 + row < a.rows) xv |= static_cast<uint32_t>(static_cast<uint8_t>(a.x[static_cast<int64_t>(t0 + row) * a.ldx + k])) << (8 * b);
        if (k < a.K && r0 + row < a.M) wv |= static_cast<uint32_t>(static_cast<uint8_t>(a.w[static_cast<int64_t>(r0 + row) * a.ldw + k])) << (8 * b);
      }
      sx[row][c] = static_cast<int32_t>(xv);
      sw[row][c] = static_cast<int32_t>(wv);
    }
    __syncthreads();
    for (int c = 0; c < 16; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(sx[tt + 16 * i][c], sw[tr + 16 * j][c], acc[i][j]);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int t = t0 + tt + 16 * i, r = r0 + tr + 16 * j;
      if (t >= a.rows || r >= a.M) continue;
      float v = __fmul_rn(__fmul_rn(static_cast<float>(acc[i][j]), a.sx[t]), a.sw[r]);
      if (a.bias) v = __fadd_rn(v, i8_load1(a.bias_type, a.bias, r));
      i8_store1(a.y_type, a.y, static_cast<int64_t>(t) * a.ldy + r, v);
    }
}

}  // namespace opc
