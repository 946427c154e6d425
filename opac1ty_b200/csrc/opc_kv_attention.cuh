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
  int32_t bf16;
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
  if (r - __ldg(a.B.q_start + seq) >= a.B.max_q) {
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

}  // namespace opc
