// opc_score.cuh -- log probabilities of given tokens, entropy and top alternatives of logits rows.
#pragma once

#include <cstdint>

#include "opc_kv.cuh"

namespace opc {

constexpr int kScoreThreads = 256;
constexpr int kScoreMaxTop = 32;

struct ScoreArgs {
  const void* x;
  int64_t ld;
  int32_t dtype;  // OPC_F16, OPC_BF16, OPC_F32
  int32_t rows, vocab, top_k;
  const int32_t* targets;
  float *logprob, *entropy, *top_logprobs;
  int32_t* top_ids;
  int* err;
};

__device__ __forceinline__ float score_load(const ScoreArgs& a, int64_t row, int i) {
  if (a.dtype == 2) return static_cast<const float*>(a.x)[row * a.ld + i];
  const uint32_t w = static_cast<const uint16_t*>(a.x)[row * a.ld + i];
  return a.dtype == 1 ? half_lo<true>(w) : half_lo<false>(w);
}

// Order of candidates as one number: larger logits first, then lower ids; NaN below everything.
__device__ __forceinline__ uint64_t score_key(float x, int id) {
  uint32_t b = __float_as_uint(x == 0.f ? 0.f : x);
  b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  if (x != x) b = 0;
  return (static_cast<uint64_t>(b) << 32) | static_cast<uint32_t>(~id);
}

template <typename T, typename F>
__device__ __forceinline__ T score_block_reduce(T v, F f, T* buf) {
  for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  v = buf[0];
  for (int i = 1; i < kScoreThreads / 32; ++i) v = f(v, buf[i]);
  return v;
}

// One CTA per row: the maximum, then the sums, then top_k rounds that each find the largest
// candidate below the last one.
__global__ void __launch_bounds__(kScoreThreads) score_plain_kernel(const ScoreArgs a) {
  __shared__ float fbuf[kScoreThreads / 32];
  __shared__ uint64_t kbuf[kScoreThreads / 32];
  const int64_t r = blockIdx.x;
  const auto fmax_ = [](float u, float v) { return fmaxf(u, v); };
  const auto add = [](float u, float v) { return u + v; };
  const auto kmax = [](uint64_t u, uint64_t v) { return u > v ? u : v; };
  float m = -INFINITY, bad = 0.f;
  for (int i = threadIdx.x; i < a.vocab; i += kScoreThreads) {
    const float x = score_load(a, r, i);
    m = fmaxf(m, x);
    if (!(x < INFINITY)) bad = 1.f;
  }
  m = score_block_reduce(m, fmax_, fbuf);
  bad = score_block_reduce(bad, fmax_, fbuf);
  const float base = m == -INFINITY ? 0.f : m;
  float z = 0.f, w = 0.f;
  for (int i = threadIdx.x; i < a.vocab; i += kScoreThreads) {
    const float y = score_load(a, r, i) - base, e = expf(y);
    z += e;
    if (e > 0.f) w += e * y;
  }
  z = score_block_reduce(z, add, fbuf);
  w = score_block_reduce(w, add, fbuf);
  const float lse = logf(z), nan = __int_as_float(0x7fffffff);
  const auto value = [&](float x) { return bad > 0.f ? nan : x == -INFINITY ? -INFINITY : (x - base) - lse; };
  if (threadIdx.x == 0) {
    if (a.logprob) {
      const int t = a.targets[r];
      float v = 0.f;
      if (t >= a.vocab) {
        atomicCAS(a.err, 0, kDevErrBadIndex);
        v = nan;
      } else if (t >= 0) {
        v = value(score_load(a, r, t));
      }
      a.logprob[r] = v;
    }
    if (a.entropy) a.entropy[r] = bad > 0.f ? nan : z > 0.f ? lse - w / z : 0.f;
  }
  uint64_t last = ~0ull;
  for (int k = 0; k < a.top_k; ++k) {
    uint64_t best = 0;
    for (int i = threadIdx.x; i < a.vocab; i += kScoreThreads) {
      const uint64_t key = score_key(score_load(a, r, i), i);
      if (key < last && key > best) best = key;
    }
    best = last = score_block_reduce(best, kmax, kbuf);
    if (threadIdx.x == 0) {
      const int id = static_cast<int>(~static_cast<uint32_t>(best));
      a.top_ids[r * a.top_k + k] = id;
      a.top_logprobs[r * a.top_k + k] = value(score_load(a, r, id));
    }
  }
}

}  // namespace opc
