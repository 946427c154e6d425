// opc_score.cuh -- log probabilities of given tokens, entropy and top alternatives of logits rows.
//
// Memory bound: every logit is read once.  Per row, with y = (x - m) log2(e):
//   m = max x,  Z = sum 2^y,  W = sum 2^y y
//   logprob = x_t - m - ln2 log2 Z,  entropy = ln2 (log2 Z - W / Z)
// in one pass: a thread takes groups of 16 bytes, and moves its own m only when a group passes it (the
// sums are then rescaled); the threads' (m, Z, W) are joined at the end.  At 2 bytes a logit HBM leaves
// about 11 issue slots per logit on an SM; two 16-bit logits take about 9 instructions (packed maximum
// and clamp, unpack, packed fp32 fma, two exp2, packed sum and fma).
//
// Top alternatives without a second pass: every thread also keeps the largest logit of its share.  The
// top_k-th largest of these maxima bounds the answer from below (top_k different logits reach it), so
// only the shares whose maximum reaches it -- about top_k of them -- are read again (from L2), by the
// whole CTA, and the logits at or above the bound collected and sorted.  Where more logits reach it
// than fit (ties, mostly), the answer is found by top_k rounds of a maximum below the last one over
// those shares.
//
// Measured: 2048 rows of 128256 bf16 logits with 8 alternatives 118 us, 4.5 TB/s; 1024 rows of fp32 112 us,
// 4.7 TB/s; one row with 20 alternatives 9 us.  Rows of which a mask leaves fewer logits than alternatives are
// read once for each of these: 2048 rows with three logits left and 20 alternatives 5.2 ms, 64 rows 244 us.
// The pass over the logits alone takes 105 us, in the arithmetic of which (two exp2 per pair of logits, half of
// the special-function units' rate) loads do not hide completely; finding and ordering the alternatives is the
// rest.
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

// The larger of two pairs of 16-bit elements, ignoring NaN, or handing it on.
template <bool kBf>
__device__ __forceinline__ uint32_t max_pair(uint32_t a, uint32_t b) {
  uint32_t d;
  if constexpr (kBf) asm("max.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  else asm("max.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
template <bool kBf>
__device__ __forceinline__ uint32_t max_pair_nan(uint32_t a, uint32_t b) {
  uint32_t d;
  if constexpr (kBf) asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  else asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// The largest of a group, ignoring NaN.
template <int kType>
__device__ __forceinline__ float score_max(const uint4& w) {
  if constexpr (kType == 2) {
    return fmaxf(fmaxf(__uint_as_float(w.x), __uint_as_float(w.y)), fmaxf(__uint_as_float(w.z), __uint_as_float(w.w)));
  } else {
    const uint32_t b = max_pair<kType == 1>(max_pair<kType == 1>(w.x, w.y), max_pair<kType == 1>(w.z, w.w));
    return fmaxf(half_lo<kType == 1>(b), half_hi<kType == 1>(b));
  }
}

struct ScoreSums {
  float m, z, w, bad;  // bad: a NaN or +infinity was seen; m = -inf: nothing but -infinity so far
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
// The sums of a warp's lanes: the largest m first, so that each lane is scaled once.
__device__ __forceinline__ ScoreSums score_join_warp(const ScoreSums& s) {
  ScoreSums r;
  const uint32_t o = __reduce_max_sync(0xffffffffu, score_order(s.m));
  r.m = __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
  r.bad = __any_sync(0xffffffffu, s.bad != 0.f) ? 1.f : 0.f;
  const float d = s.m == -INFINITY ? 0.f : (s.m - r.m) * 1.4426950408889634f, f = s.m == -INFINITY ? 0.f : exp2f(d);
  r.z = f * s.z;
  r.w = f > 0.f ? f * (s.w + d * s.z) : 0.f;
#pragma unroll
  for (int i = 16; i > 0; i >>= 1) {
    r.z += __shfl_xor_sync(0xffffffffu, r.z, i);
    r.w += __shfl_xor_sync(0xffffffffu, r.w, i);
  }
  return r;
}
// 32 keys of a warp in descending order (bitonic).
template <typename T>
__device__ __forceinline__ T score_sort32(T v, int lane) {
#pragma unroll
  for (int k = 2; k <= 32; k *= 2) {
#pragma unroll
    for (int j = k / 2; j > 0; j /= 2) {
      const T o = __shfl_xor_sync(0xffffffffu, v, j);
      const bool up = (lane & k) != 0, low = (lane & j) == 0;  // descending blocks, ascending where up
      v = (low != up) ? (v > o ? v : o) : (v < o ? v : o);
    }
  }
  return v;
}
// Two descending sequences of 32 (lane i: element i of each) to the 32 largest of both, descending.
template <typename T>
__device__ __forceinline__ T score_merge32(T a, T b, int lane) {
  const T r = __shfl_sync(0xffffffffu, b, 31 - lane);
  T v = a > r ? a : r;
#pragma unroll
  for (int j = 16; j > 0; j /= 2) {
    const T o = __shfl_xor_sync(0xffffffffu, v, j);
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
__global__ void __launch_bounds__(kScoreThreads, 5) score_kernel(const ScoreArgs a) {
  constexpr int kN = kType == 2 ? 4 : 8, kWarps = kScoreThreads / 32, kU = 4;  // groups in flight per thread
  constexpr int kSize = kType == 2 ? 4 : 2;
  __shared__ ScoreSums sm_sums[kWarps];
  __shared__ uint64_t sm_keys[kWarps][32];
  __shared__ uint64_t sm_cand[kTop ? kScoreCand : 1];
  __shared__ uint32_t sm_share[kScoreThreads];
  __shared__ uint32_t sm_top[kWarps][32];
  __shared__ int sm_n, sm_shares, sm_last;
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
  constexpr float kLog2e = 1.4426950408889634f;
  // The thread's m, and Z and W in two halves each (even and odd logits).  For an ordinary m, y is one
  // fma, fma(x, log2 e, -M), M = m log2 e rounded; the rounding c = m log2 e - M shifts every y alike and
  // is taken out when m moves and at the end.  -infinity goes in as -65504 (fp16) or -1e30, far enough below kPlainLow for a weight of 0; a NaN turns
  // Z into one.  Other m (nothing but -infinity or NaN so far, masks of the type's lowest value, absurd
  // logits) take logit by logit.
  constexpr float kPlain = 1e6f, kPlainLow = kType == 0 ? -6e4f : -1e6f, kNothing = -1e30f;
  float m = -INFINITY, c = 0.f, bad = 0.f;
  uint64_t z2 = 0, w2 = 0, ml2 = 0;  // ml2: -M, twice
  float top = -INFINITY;  // largest logit of this thread's share (thread t: groups t, t + 256, ..., and the tail's)
  bool any = false;       // whether the share holds anything but NaN
  const uint64_t l2 = pack2(kLog2e, kLog2e);
  const auto move = [&](float big) {  // the share's maximum moves (seldom after the first groups)
    top = fmaxf(top, big);
    any |= big == big;
    if (big > m && big < INFINITY) {
      const float ml = big * kLog2e, cn = fabsf(big) <= kPlain ? fmaf(big, kLog2e, -ml) : 0.f;
      if (m > -INFINITY) {  // y falls by (big - m) log2 e, and its shift changes
        const float d = fmaxf((m - big) * kLog2e + (cn - c), -200.f), f = exp2f(d);
        w2 = mul2(pack2(f, f), fma2(pack2(d, d), z2, w2));
        z2 = mul2(pack2(f, f), z2);
      }
      m = big;
      c = cn;
      ml2 = pack2(-ml, -ml);
    }
  };
  const auto one = [&](float x) {  // any logit, any m
    if (x > top || !any) move(x);
    if (x != x) bad = 1.f;
    if (m > -INFINITY && x == x) {
      const float y = fmaxf((x - m) * kLog2e + c, -200.f), e = exp2f(y);  // (2^-200 is 0, and so is its product with y)
      z2 = add2(z2, pack2(e, 0.f));
      w2 = add2(w2, pack2(e * y, 0.f));
    }
  };
  const auto pair = [&](float x0, float x1) {
    const uint64_t y = fma2(pack2(x0, x1), l2, ml2);
    const float2 f = unpack2(y);
    float e0, e1;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e0) : "f"(f.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e1) : "f"(f.y));
    const uint64_t e = pack2(e0, e1);
    z2 = add2(z2, e);
    w2 = fma2(e, y, w2);
  };
  const auto take = [&](const uint4& raw) {
    const uint32_t r4[4] = {raw.x, raw.y, raw.z, raw.w};
    const float big = score_max<kType>(raw);
    if (big > top || !any) move(big);
    if (m >= kPlainLow && m <= kPlain) {
      if constexpr (kType == 2) {
        pair(max_nan(__uint_as_float(raw.x), kNothing), max_nan(__uint_as_float(raw.y), kNothing));
        pair(max_nan(__uint_as_float(raw.z), kNothing), max_nan(__uint_as_float(raw.w), kNothing));
      } else {
        const uint32_t low = kType == 1 ? 0xf149f149u : 0xfbfffbffu;  // about -1e30; -65504
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t c = max_pair_nan<kType == 1>(r4[i], low);
          pair(half_lo<kType == 1>(c), half_hi<kType == 1>(c));
        }
      }
    } else {
      float x[kN];
      score_unpack<kType>(raw, x);
#pragma unroll 1
      for (int i = 0; i < kN; ++i) one(i == 0 ? x[0] : i == 1 ? x[1] : i == 2 ? x[2] : i == 3 ? x[3] : i == 4 ? x[4 % kN] : i == 5 ? x[5 % kN] : i == 6 ? x[6 % kN] : x[7 % kN]);
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
    for (int u = 0; u < kU; ++u) take(w[u]);
  }
  for (; g < groups; g += kScoreThreads) take(group(g));
  for (int i = tail + tid; i < end; i += kScoreThreads) one(score_load<kType>(row, i));

  // ---------------------------------------------------------------- join the threads
  const float2 zz = unpack2(z2), ww = unpack2(w2);
  ScoreSums all = {m, zz.x + zz.y, ww.x + ww.y, bad};
  all.z *= exp2f(-c);  // 2^(y + c), and 2^(y + c) (y + c), without c
  all.w = fmaf(all.w, exp2f(-c), -c * all.z);
  if (all.z != all.z || top == INFINITY) all.bad = 1.f;
  if (all.bad != 0.f) all.z = all.w = 0.f;
  all = score_join_warp(all);
  if (lane == 0) sm_sums[warp] = all;
  uint64_t mine = 0;
  if (kTop) {
    // the maxima in order: the top_k-th bounds the answer from below (shares of NaN alone count as 0)
    sm_top[warp][lane] = score_sort32(any ? score_order(top) : 0u, lane);
  }
  __syncthreads();
  if (warp == 0) all = score_join_warp(lane < kWarps ? sm_sums[lane] : ScoreSums{-INFINITY, 0.f, 0.f, 0.f});
  if (kTop) {
#pragma unroll 1
    for (int h = kWarps / 2; h > 0; h /= 2) {
      if (warp < h) sm_top[warp][lane] = score_merge32(sm_top[warp][lane], sm_top[warp + h][lane], lane);
      __syncthreads();
    }
    const int want = min(a.top_k, max(0, end - begin));
    // (where fewer shares hold something it is 0: everything is a candidate)
    const uint32_t bound = want > 0 ? sm_top[0][want - 1] : ~0u;
    // the shares that reach it
    if ((any ? score_order(top) : 0u) >= bound) sm_share[atomicAdd(&sm_shares, 1)] = tid;
    __syncthreads();
    const int shares = sm_shares, per = (groups + kScoreThreads - 1) / kScoreThreads;
    const int n_tail = end - tail;
    // the groups of those shares, and the tail (once)
    const auto scan = [&](auto&& f) {
#pragma unroll 1
      for (int i = tid; i < shares * per; i += kScoreThreads) {
        const int gg = static_cast<int>(sm_share[i / per]) + (i % per) * kScoreThreads;
        if (gg < groups) f(group(gg), begin + gg * kN, kN);
      }
      for (int i = tid; i < n_tail; i += kScoreThreads) {
        uint4 w = make_uint4(0, 0, 0, 0);  // (only the first element counts)
        w.x = kType == 2 ? __float_as_uint(score_load<kType>(row, tail + i)) : static_cast<const uint16_t*>(static_cast<const void*>(row))[tail + i];
        f(w, tail + i, 1);
      }
    };
    scan([&](const uint4& w, int id, int n) {
      if (n == kN && bound != 0 && score_order(score_max<kType>(w)) < bound) return;
      float x[kN];
      score_unpack<kType>(w, x);
#pragma unroll
      for (int e = 0; e < kN; ++e)
        if (e < n && score_order(x[e]) >= bound) {
          const int at = atomicAdd(&sm_n, 1);
          if (at < kScoreCand) sm_cand[at] = score_key(x[e], id + e);
        }
    });
    __syncthreads();
    const int n = sm_n;
    if (n <= 32) {  // order them
      if (warp == 0) mine = score_sort32(lane < n ? sm_cand[lane] : uint64_t{0}, lane);
    } else if (n <= kScoreCand) {  // sorted lists of 32 per warp, merged
      for (int i = tid + n; i < kScoreCand; i += kScoreThreads) sm_cand[i] = 0;
      __syncthreads();
      uint64_t v = 0;
      for (int i = 32 * warp; i < n; i += kScoreThreads) v = score_merge32(v, score_sort32(sm_cand[i + lane], lane), lane);
      sm_keys[warp][lane] = v;
      __syncthreads();
      if (warp == 0) {
        for (int w = 1; w < min(kWarps, (n + 31) / 32); ++w) v = score_merge32(v, sm_keys[w][lane], lane);
        mine = v;
      }
    } else {  // too many (ties): the largest below the last one, top_k times
      uint64_t last = ~0ull;
#pragma unroll 1
      for (int k = 0; k < want; ++k) {
        uint64_t best = 0;
        scan([&](const uint4& w, int id, int n) {
          float x[kN];
          score_unpack<kType>(w, x);
#pragma unroll
          for (int e = 0; e < kN; ++e) {
            const uint64_t key = score_key(x[e], id + e);
            if (e < n && key < last && key > best) best = key;
          }
        });
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const uint64_t other = __shfl_xor_sync(0xffffffffu, best, o);
          best = best > other ? best : other;
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
    if (lane == 0) {
      sm_last = atom_add_acq_rel_gpu(a.count + r, 1) == a.split - 1;
      if (sm_last) a.count[r] = 0;
    }
  }
  __syncthreads();
  if (!sm_last) return;
  if (kTop) {  // the CTAs' candidates: lists w, w + 8, ... per warp, then the warps'
    const uint64_t* c = a.cand + r * a.split * kScoreMaxTop;
    uint64_t v = 0;
#pragma unroll 4
    for (int i = warp; i < a.split; i += kWarps) v = score_merge32(v, __ldcg(c + i * kScoreMaxTop + lane), lane);
    sm_keys[warp][lane] = v;
    __syncthreads();
#pragma unroll 1
    for (int h = kWarps / 2; h > 0; h /= 2) {
      if (warp < h) sm_keys[warp][lane] = score_merge32(sm_keys[warp][lane], sm_keys[warp + h][lane], lane);
      __syncthreads();
    }
  }
  if (warp == 0) {
    ScoreSums sums = {-INFINITY, 0.f, 0.f, 0.f};
    for (int i = lane; i < a.split; i += 32) {  // (at most two each; lanes joined in a fixed order)
      const float4 p = __ldcg(a.part + r * a.split + i);
      sums = score_join(sums, ScoreSums{p.x, p.y, p.z, p.w});
    }
    sums = score_join_warp(sums);
    score_write<kType>(a, r, row, sums, kTop ? sm_keys[0][lane] : 0, lane);
  }
}

}  // namespace opc
