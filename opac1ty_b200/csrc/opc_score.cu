// opc_score.cu -- C ABI of opc_token_logprobs (include/opc_b200.h).
#define OPC_WITHOUT_ERROR_WORD
#include <cuda_runtime.h>

#include "../../include/opc_b200.h"
#include "opc_internal.h"
#include "opc_score.cuh"

using opc_host::cuda_fail;
using opc_host::fail;

namespace {

int check_score(const char* who, int32_t rows, int32_t vocab, int32_t top_k) {
  if (rows < 0 || vocab < 1) return fail(OPC_ERR_INVALID, "%s: %d rows of %d logits", who, rows, vocab);
  if (top_k < 0 || top_k > opc::kScoreMaxTop || top_k > vocab)
    return fail(OPC_ERR_INVALID, "%s: top_k %d (at most %d, and at most the vocabulary of %d)", who, top_k, opc::kScoreMaxTop, vocab);
  return OPC_OK;
}

}  // namespace

extern "C" {

size_t opc_token_logprobs_workspace_bytes(int32_t rows, int32_t vocab, int32_t top_k, int32_t device) {
  (void)device;
  if (check_score("opc_token_logprobs_workspace_bytes", rows, vocab, top_k) != OPC_OK) return 0;
  return 256;
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
  if (!workspace || workspace_bytes < 256) return fail(OPC_ERR_WORKSPACE, "%s: workspace of %zu bytes", who, workspace_bytes);
  opc::ScoreArgs a;
  a.x = logits;
  a.ld = ld;
  a.dtype = dtype;
  a.rows = rows;
  a.vocab = vocab;
  a.top_k = top_k;
  a.targets = targets;
  a.logprob = logprob;
  a.entropy = entropy;
  a.top_ids = top_ids;
  a.top_logprobs = top_logprobs;
  a.err = dev.error_word;
  opc::score_plain_kernel<<<rows, opc::kScoreThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? OPC_OK : cuda_fail(e, "opc_token_logprobs launch");
}

}  // extern "C"
