// opc_score.cu -- C ABI of opc_token_logprobs (include/opc_b200.h).
#define OPC_WITHOUT_ERROR_WORD
#include <cuda_runtime.h>

#include <algorithm>

#include "../../include/opc_b200.h"
#include "opc_internal.h"
#include "opc_score.cuh"

using opc_host::cuda_fail;
using opc_host::fail;

namespace {

constexpr size_t kCounterBytes = opc::kScoreMaxRows * sizeof(int32_t);

int check_score(const char* who, int32_t rows, int32_t vocab, int32_t top_k) {
  if (rows < 0 || vocab < 1) return fail(OPC_ERR_INVALID, "%s: %d rows of %d logits", who, rows, vocab);
  if (top_k < 0 || top_k > opc::kScoreMaxTop || top_k > vocab)
    return fail(OPC_ERR_INVALID, "%s: top_k %d (at most %d, and at most the vocabulary of %d)", who, top_k, opc::kScoreMaxTop, vocab);
  return OPC_OK;
}

// How a call is divided: CTAs per row, logits of each, workspace bytes.
struct ScorePlan {
  int split, chunk;
  size_t bytes;
};

ScorePlan plan_score(int32_t rows, int32_t vocab, int sms) {
  // One CTA per row, unless the rows leave SMs idle: then up to two CTAs per SM, with no fewer than two
  // groups of 8 logits for each thread (128256 logits: one row 9.6 us instead of 20.3, 100 rows 18.7
  // instead of 20.8; 17 rows of 32000 9.5 and 9.1).
  ScorePlan p{1, vocab, kCounterBytes};
  if (rows > 0 && rows <= opc::kScoreMaxRows) {
    const int most = std::min<int>(opc::kScoreMaxSplit, vocab / (opc::kScoreThreads * 16));
    p.split = std::max(1, std::min(most, 2 * sms / rows));
    p.chunk = ((vocab + p.split - 1) / p.split + 7) / 8 * 8;
    p.split = (vocab + p.chunk - 1) / p.chunk;
  }
  if (p.split > 1) p.bytes += static_cast<size_t>(rows) * p.split * (sizeof(float4) + opc::kScoreMaxTop * sizeof(uint64_t));
  return p;
}

template <int kType, bool kVec>
auto score_of(bool top) {
  return top ? opc::score_kernel<kType, kVec, true> : opc::score_kernel<kType, kVec, false>;
}
template <int kType>
auto score_of(bool vec, bool top) {
  return vec ? score_of<kType, true>(top) : score_of<kType, false>(top);
}

}  // namespace

extern "C" {

size_t opc_token_logprobs_workspace_bytes(int32_t rows, int32_t vocab, int32_t top_k, int32_t device) {
  if (check_score("opc_token_logprobs_workspace_bytes", rows, vocab, top_k) != OPC_OK) return 0;
  int sms = 0;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  return plan_score(rows, vocab, sms).bytes;
}

int opc_token_logprobs(const void* logits, int64_t ld, int32_t dtype, int32_t rows, int32_t vocab,
                       const int32_t* targets, float* logprob, float* entropy, int32_t top_k, int32_t* top_ids,
                       float* top_logprobs, void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "opc_token_logprobs";
  const int rc = check_score(who, rows, vocab, top_k);
  if (rc != OPC_OK) return rc;
  if (dtype != OPC_F16 && dtype != OPC_BF16 && dtype != OPC_F32) return fail(OPC_ERR_UNSUPPORTED, "%s: element type %d", who, dtype);
  if ((targets != nullptr) != (logprob != nullptr)) return fail(OPC_ERR_INVALID, "%s: targets and logprob go together", who);
  if (rows == 0) return OPC_OK;
  if (top_k > 0 && (!top_ids || !top_logprobs)) return fail(OPC_ERR_INVALID, "%s: top_k %d without top_ids and top_logprobs", who, top_k);
  if (!logits || (reinterpret_cast<uintptr_t>(logits) & (dtype == OPC_F32 ? 3u : 1u)))
    return fail(OPC_ERR_INVALID, "%s: logits is NULL or not aligned to its elements", who);
  if (ld < vocab) return fail(OPC_ERR_INVALID, "%s: leading dimension %lld below the vocabulary of %d", who, static_cast<long long>(ld), vocab);
  opc_host::Device dev;
  const int rd = opc_host::current_device(&dev);
  if (rd != OPC_OK) return rd;
  const ScorePlan p = plan_score(rows, vocab, dev.sm_count);
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15u) || workspace_bytes < p.bytes)
    return fail(OPC_ERR_WORKSPACE, "%s: a 16-byte aligned workspace of %zu bytes is needed, got %zu", who, p.bytes, workspace_bytes);
  opc::ScoreArgs a;
  a.x = logits;
  a.ld = ld;
  a.rows = rows;
  a.vocab = vocab;
  a.top_k = top_k;
  a.targets = targets;
  a.logprob = logprob;
  a.entropy = entropy;
  a.top_ids = top_ids;
  a.top_logprobs = top_logprobs;
  a.err = dev.error_word;
  a.split = p.split;
  a.chunk = p.chunk;
  a.count = static_cast<int32_t*>(workspace);
  a.part = reinterpret_cast<float4*>(static_cast<char*>(workspace) + kCounterBytes);
  a.cand = reinterpret_cast<uint64_t*>(a.part + static_cast<size_t>(rows) * p.split);
  const bool vec = (reinterpret_cast<uintptr_t>(logits) & 15u) == 0 && ld % (dtype == OPC_F32 ? 4 : 8) == 0;
  auto kern = dtype == OPC_F32 ? score_of<2>(vec, top_k > 0) : dtype == OPC_BF16 ? score_of<1>(vec, top_k > 0) : score_of<0>(vec, top_k > 0);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows) * p.split);
  cfg.blockDim = dim3(opc::kScoreThreads);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];  // set-up overlaps the kernel before, which the kernel waits for
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, a);
  return e == cudaSuccess ? OPC_OK : cuda_fail(e, "opc_token_logprobs launch");
}

}  // extern "C"
