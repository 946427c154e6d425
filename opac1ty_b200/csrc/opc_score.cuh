// opc_score.cuh -- log probabilities of given tokens, entropy and top alternatives of logits rows.
//
// Memory bound: every logit is read once.  Per row, with y = (x - m) log2(e):
//   m = max x,  Z = sum 2^y,  W = sum 2^y y
//   logprob = x_t - m - ln2 log2 Z,  entropy = ln2 (log2 Z - W / Z)
// in one pass: a thread takes groups of 16 bytes, and moves its own m only when a group passes it (the
// sums are then rescaled); the threads' (m, Z, W) are joined at the end.  At 2 bytes a logit HBM leaves
// about 11 issue slots per logit on an SM; the pass takes about 8 (unpack, maximum, difference, product,
// clamp, exp2, sum, fma).
//
// Top alternatives without a second pass: every thread also keeps the largest logit of its share.  The
// top_k-th largest of these maxima bounds the answer from below (top_k different logits reach it), so
// only the shares whose maximum reaches it -- about top_k of them -- are read again (from L2), by the
// whole CTA, and the logits at or above the bound collected and sorted.  Where more logits reach it
// than fit (ties, mostly), the answer is found by top_k rounds of a maximum below the last one over
// those shares.
//
// Few rows are split over several CTAs: each leaves its sums and its own top_k candidates in the
// workspace, the last one of the row joins them.
#pragma once

#include <cstdint>

#include "opc_kv.cuh"

namespace opc {

constexpr int kScoreThreads = 256;
constexpr int kScoreMaxTop = 32;
constexpr int kScoreCand = 1024;    // candidates a CTA can collect
constexpr int kScoreMaxRows = 1024; // rows that may be split (workspace counters)
constexpr int kScoreMaxSplit = 64;

struct ScoreArgs {
  const void* x;
  int64_t ld;
  int32_t rows, vocab, top_k;
  const int32_t* targets;
  float *logprob, *entropy, *top_logprobs;
  int32_t* top_ids;
  int* err;
  int32_t split, chunk;   // CTAs per row, logits of each (a multiple of a group)
  int32_t* count;         // [rows], zero between calls
  float4* part;           // [rows][split]: (m, Z, W, whether a NaN or +infinity was seen)
  uint64_t* cand;         // [rows][split][kScoreMaxTop], in order
};

// One logit; kType: OPC_F16, OPC_BF16, OPC_F32.
template <int kType>
__device__ __forceinline__ float score_load(const void* row, int i) {
  if constexpr (kType == 2) return __ldg(static_cast<const float*>(row) + i);
  const uint32_t w = __ldg(static_cast<const uint16_t*>(row) + i);
  return kType == 1 ? half_lo<true>(w) : half_lo<false>(w);
}
// A group of 16 bytes (8 or 4 logits).
template <int kType>
__device__ __forceinline__ void score_unpack(const uint4& w, float* x) {
  if constexpr (kType == 2) {
    x[0] = __uint_as_float(w.x);
    x[1] = __uint_as_float(w.y);
    x[2] = __uint_as_float(w.z);
    x[3] = __uint_as_float(w.w);
  } else {
    unpack_halves<kType == 1>(w, x);
  }
}

// The order of candidates as one number: larger logits first, then lower ids; NaN below everything.
__device__ __forceinline__ uint32_t score_order(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);  // (-0 counts as 0)
  return x != x ? 0u : (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ uint64_t score_key(float x, int id) {
  return (static_cast<uint64_t>(score_order(x)) << 32) | static_cast<uint32_t>(~id);
}
__device__ __forceinline__ float score_value(uint64_t key) {  // (NaN comes back as NaN)
  const uint32_t o = static_cast<uint32_t>(key >> 32);
  return o == 0 ? __int_as_float(0x7fffffff) : __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
__device__ __forceinline__ int score_id(uint64_t key) { return static_cast<int>(~static_cast<uint32_t>(key)); }

struct ScoreSums {
  float m, z, w, bad;  // m = -inf: nothing but -infinity so far
};
__device__ __forceinline__ ScoreSums score_join(const ScoreSums& a, const ScoreSums& b) {
  ScoreSums r;
  r.m = fmaxf(a.m, b.m);
  const float base = r.m == -INFINITY ? 0.f : r.m;
  // against the larger m every y falls by d = (r.m - m) log2(e): 2^(y-d) (y-d) = 2^-d (2^y y - d 2^y)
  constexpr float kLog2e = 1.4426950408889634f;
  const float da = a.m == -INFINITY ? 0.f : (a.m - base) * kLog2e, db = b.m == -INFINITY ? 0.f : (b.m - base) * kLog2e;
  const float fa = a.m == -INFINITY ? 0.f : exp2f(da), fb = b.m == -INFINITY ? 0.f : exp2f(db);
  r.z = fa * a.z + fb * b.z;
  // (far below: nothing, and 0 * infinity is kept out)
  r.w = (fa > 0.f ? fa * (a.w + da * a.z) : 0.f) + (fb > 0.f ? fb * (b.w + db * b.z) : 0.f);
  r.bad = fmaxf(a.bad, b.bad);
  return r;
}
__device__ __forceinline__ ScoreSums score_shfl(const ScoreSums& s, int o) {
  ScoreSums r;
  r.m = __shfl_xor_sync(0xffffffffu, s.m, o);
  r.z = __shfl_xor_sync(0xffffffffu, s.z, o);
  r.w = __shfl_xor_sync(0xffffffffu, s.w, o);
  r.bad = __shfl_xor_sync(0xffffffffu, s.bad, o);
  return r;
}
__device__ __forceinline__ uint64_t score_shfl64(uint64_t v, int o) { return __shfl_xor_sync(0xffffffffu, v, o); }

// 32 keys of a warp in descending order (bitonic).
__device__ __forceinline__ uint64_t score_sort32(uint64_t v, int lane) {
#pragma unroll
  for (int k = 2; k <= 32; k *= 2) {
#pragma unroll
    for (int j = k / 2; j > 0; j /= 2) {
      const uint64_t o = score_shfl64(v, j);
      const bool up = (lane & k) != 0, low = (lane & j) == 0;  // descending blocks, ascending where up
      v = (low != up) ? (v > o ? v : o) : (v < o ? v : o);
    }
  }
  return v;
}
// Two descending sequences of 32 (lane i: element i of each) to the 32 largest of both, descending.
__device__ __forceinline__ uint64_t score_merge32(uint64_t a, uint64_t b, int lane) {
  const uint64_t r = __shfl_sync(0xffffffffu, b, 31 - lane);
  uint64_t v = a > r ? a : r;
#pragma unroll
  for (int j = 16; j > 0; j /= 2) {
    const uint64_t o = score_shfl64(v, j);
    v = (lane & j) == 0 ? (v > o ? v : o) : (v < o ? v : o);
  }
  return v;
}

// The outputs of a row from its sums and its ordered candidates (lane i of the first warp: key i).
template <int kType>
__device__ __forceinline__ void score_write(const ScoreArgs& a, int64_t r, const void* row, const ScoreSums& s, uint64_t key, int lane) {
  constexpr float kLn2 = 0.6931471805599453f;
  const bool bad = s.bad != 0.f, none = s.m == -INFINITY;
  const float nan = __int_as_float(0x7fffffff), lz = log2f(s.z);
  // (x - m first: log Z may be small beside them)
  const auto logprob = [&](float x) {
    return bad ? nan : x == -INFINITY || none ? -INFINITY : (x - s.m) - kLn2 * lz;
  };
  if (lane == 0) {
    if (a.logprob) {
      const int t = __ldg(a.targets + r);
      float v = 0.f;
      if (t >= a.vocab) {
        atomicCAS(a.err, 0, kDevErrBadIndex);
        v = nan;
      } else if (t >= 0) {
        v = logprob(score_load<kType>(row, t));
      }
      a.logprob[r] = v;
    }
    if (a.entropy) a.entropy[r] = bad ? nan : none ? 0.f : fmaxf(0.f, kLn2 * (lz - s.w / s.z));
  }
  if (lane < a.top_k) {
    a.top_ids[r * a.top_k + lane] = score_id(key);
    a.top_logprobs[r * a.top_k + lane] = logprob(score_value(key));
  }
}

template <int kType, bool kVec, bool kTop>
__global__ void __launch_bounds__(kScoreThreads) score_kernel(const ScoreArgs a) {
  constexpr int kN = kType == 2 ? 4 : 8, kWarps = kScoreThreads / 32, kU = 4;  // groups in flight per thread
  constexpr int kSize = kType == 2 ? 4 : 2;
  __shared__ ScoreSums sm_sums[kWarps];
  __shared__ uint64_t sm_keys[kWarps][32];
  __shared__ uint64_t sm_cand[kTop ? kScoreCand : 1];
  __shared__ uint32_t sm_share[kScoreThreads];
  __shared__ int sm_n, sm_shares;
  __shared__ uint64_t sm_best[kWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t r = blockIdx.x / a.split;
  const int part = blockIdx.x - static_cast<int>(r) * a.split;
  const char* row = static_cast<const char*>(a.x) + r * a.ld * kSize;
  const int begin = part * a.chunk, end = min(a.vocab, begin + a.chunk);  // this CTA's logits
  const int groups = max(0, end - begin) / kN, tail = begin + groups * kN;   // whole groups, then single ones
  griddep_wait();
  griddep_launch_dependents();
  if (kTop && tid == 0) sm_n = sm_shares = 0;

  // ---------------------------------------------------------------- one pass over the logits
  ScoreSums s = {-INFINITY, 0.f, 0.f, 0.f};
  float top = -INFINITY;  // largest logit of this thread's share (thread t: groups t, t + 256, ..., and the tail's)
  bool any = false;       // whether the share holds anything but NaN
  const auto take = [&](const float* x, int n) {
    constexpr float kLog2e = 1.4426950408889634f;
    float big = x[0];
    bool nan = !(x[0] < INFINITY);
#pragma unroll
    for (int i = 1; i < kN; ++i)
      if (i < n) {
        big = fmaxf(big, x[i]);
        nan |= !(x[i] < INFINITY);
      }
    if (nan) s.bad = 1.f;
    if (big > top || !any) {  // the share's maximum moves (seldom after the first groups)
      top = fmaxf(top, big);
      any |= big == big;
      if (big > s.m && big < INFINITY) {
        if (s.m > -INFINITY) {
          const float d = fmaxf((s.m - big) * kLog2e, -200.f), f = exp2f(d);
          s.w = f * (s.w + d * s.z);
          s.z *= f;
        }
        s.m = big;
      }
    }
    if (s.m > -INFINITY) {
#pragma unroll
      for (int i = 0; i < kN; ++i)
        if (i < n) {
          const float y = fmaxf((x[i] - s.m) * kLog2e, -200.f);  // (2^-200 is 0, and so is its product with y)
          float e;
          asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(y));
          s.z += e;
          s.w = fmaf(e, y, s.w);
        }
    }
  };
  const auto group = [&](int g) {
    const char* p = row + static_cast<int64_t>(begin + g * kN) * kSize;
    if constexpr (kVec) {
      return ld_nc_v4(p);
    } else if constexpr (kType == 2) {
      const uint32_t* q = reinterpret_cast<const uint32_t*>(p);
      return make_uint4(q[0], q[1], q[2], q[3]);
    } else {
      return ld_row8<false>(reinterpret_cast<const uint16_t*>(p));
    }
  };
  int g = tid;
  for (; g + (kU - 1) * kScoreThreads < groups; g += kU * kScoreThreads) {
    uint4 w[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) w[u] = group(g + u * kScoreThreads);
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      float x[kN];
      score_unpack<kType>(w[u], x);
      take(x, kN);
    }
  }
  for (; g < groups; g += kScoreThreads) {
    float x[kN];
    score_unpack<kType>(group(g), x);
    take(x, kN);
  }
  for (int i = tail + tid; i < end; i += kScoreThreads) {
    const float x[kN] = {score_load<kType>(row, i)};
    take(x, 1);
  }

  // ---------------------------------------------------------------- join the threads
  ScoreSums all = s;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) all = score_join(all, score_shfl(all, o));
  if (lane == 0) sm_sums[warp] = all;
  uint64_t mine = 0;
  if (kTop) {
    // the maxima in order: the top_k-th bounds the answer from below.  (id: the thread, so that keys
    // differ; a share of NaN alone counts as the lowest)
    const uint64_t own = (static_cast<uint64_t>(any ? score_order(top) : 0u) << 32) | static_cast<uint32_t>(~tid);
    sm_keys[warp][lane] = score_sort32(own, lane);
  }
  __syncthreads();
  all = sm_sums[0];
  for (int i = 1; i < kWarps; ++i) all = score_join(all, sm_sums[i]);
  if (kTop) {
#pragma unroll 1
    for (int h = kWarps / 2; h > 0; h /= 2) {  // merge the warps' lists pairwise
      uint64_t v = 0;
      if (warp < h) v = score_merge32(sm_keys[warp][lane], sm_keys[warp + h][lane], lane);
      __syncthreads();
      if (warp < h) sm_keys[warp][lane] = v;
      __syncthreads();
    }
    const int want = min(a.top_k, max(0, end - begin));
    // (where fewer shares hold something it is 0: everything is a candidate)
    const uint32_t bound = want > 0 ? static_cast<uint32_t>(sm_keys[0][want - 1] >> 32) : ~0u;
    // the shares that reach it
    if ((any ? score_order(top) : 0u) >= bound) sm_share[atomicAdd(&sm_shares, 1)] = tid;
    __syncthreads();
    const int shares = sm_shares, per = (groups + kScoreThreads - 1) / kScoreThreads;
    const int n_tail = end - tail;
    // element k of the shares: group k of them all, and the tail (once)
    const auto scan = [&](auto&& f) {
      for (int i = tid; i < shares * per; i += kScoreThreads) {
        const int gg = static_cast<int>(sm_share[i / per]) + (i % per) * kScoreThreads;
        if (gg < groups) {
          float x[kN];
          score_unpack<kType>(group(gg), x);
#pragma unroll
          for (int e = 0; e < kN; ++e) f(x[e], begin + gg * kN + e);
        }
      }
      for (int i = tid; i < n_tail; i += kScoreThreads) f(score_load<kType>(row, tail + i), tail + i);
    };
    scan([&](float x, int id) {
      if (score_order(x) >= bound) {
        const int at = atomicAdd(&sm_n, 1);
        if (at < kScoreCand) sm_cand[at] = score_key(x, id);
      }
    });
    __syncthreads();
    const int n = sm_n;
    if (n <= kScoreCand) {  // order them: sorted lists of 32 per warp, merged
      for (int i = tid + n; i < kScoreCand; i += kScoreThreads) sm_cand[i] = 0;
      __syncthreads();
      uint64_t v = 0;
      for (int i = 32 * warp; i < n; i += kScoreThreads) v = score_merge32(v, score_sort32(sm_cand[i + lane], lane), lane);
      sm_keys[warp][lane] = v;
      __syncthreads();
      if (warp == 0) {
        for (int w = 1; w < kWarps; ++w) v = score_merge32(v, sm_keys[w][lane], lane);
        mine = v;
      }
    } else {  // too many (ties): the largest below the last one, top_k times
      uint64_t last = ~0ull;
#pragma unroll 1
      for (int k = 0; k < want; ++k) {
        uint64_t best = 0;
        scan([&](float x, int id) {
          const uint64_t key = score_key(x, id);
          if (key < last && key > best) best = key;
        });
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const uint64_t o64 = score_shfl64(best, o);
          best = best > o64 ? best : o64;
        }
        if (lane == 0) sm_best[warp] = best;
        __syncthreads();
        last = sm_best[0];
        for (int w = 1; w < kWarps; ++w) last = last > sm_best[w] ? last : sm_best[w];
        __syncthreads();
        if (warp == 0 && lane == k) mine = last;
      }
    }
  }

  // ---------------------------------------------------------------- the row's outputs
  if (a.split == 1) {
    if (warp == 0) score_write<kType>(a, r, row, all, mine, lane);
    return;
  }
  if (warp == 0) {
    if (lane == 0) a.part[r * a.split + part] = make_float4(all.m, all.z, all.w, all.bad);
    if (kTop) a.cand[(r * a.split + part) * kScoreMaxTop + lane] = mine;
    __syncwarp();
    int last = 0;
    if (lane == 0) last = atom_add_acq_rel_gpu(a.count + r, 1) == a.split - 1;
    if (__shfl_sync(0xffffffffu, last, 0)) {
      __syncwarp();
      if (lane == 0) a.count[r] = 0;
      ScoreSums sums = {-INFINITY, 0.f, 0.f, 0.f};
      for (int i = lane; i < a.split; i += 32) {  // (at most two each; lanes joined in a fixed order)
        const float4 p = __ldcg(a.part + r * a.split + i);
        sums = score_join(sums, ScoreSums{p.x, p.y, p.z, p.w});
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sums = score_join(sums, score_shfl(sums, o));
      uint64_t v = 0;
      if (kTop) {
        const uint64_t* c = a.cand + r * a.split * kScoreMaxTop;
#pragma unroll 4
        for (int i = 0; i < a.split; ++i) v = score_merge32(v, __ldcg(c + i * kScoreMaxTop + lane), lane);
      }
      score_write<kType>(a, r, row, sums, v, lane);
    }
  }
}

}  // namespace opc
