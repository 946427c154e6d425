// opc_kv.cu -- C ABI of the 4-bit paged cache (include/opc_b200.h): opc_kv_plan, opc_rope_turns,
// opc_kv_append, opc_kv_read, opc_kv_attention.
#define OPC_WITHOUT_ERROR_WORD
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <mutex>
#include <set>
#include <utility>

#include "../../include/opc_b200.h"
#include "opc_internal.h"
#include "opc_kv.cuh"
#include "opc_kv_attention.cuh"
#include "opc_kv_prompt.cuh"

namespace {

using opc_host::cuda_fail;
using opc_host::fail;

#define KV_CUDA(call, what)                            \
  do {                                                 \
    cudaError_t e_ = (call);                           \
    if (e_ != cudaSuccess) return cuda_fail(e_, what); \
  } while (0)

bool head_dim_ok(int hd) { return hd == 32 || hd == 64 || hd == 96 || hd == 128 || hd == 192 || hd == 256; }
bool page_size_ok(int p) { return p == 16 || p == 32 || p == 64 || p == 128 || p == 256; }
// Bytes of a cache; false where 64 bits do not hold them.
bool cache_bytes(int32_t n_pages, int32_t kv_heads, int64_t head_bytes, int64_t* total) {
  return !__builtin_mul_overflow(kv_heads * head_bytes, static_cast<int64_t>(n_pages), total);
}
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// The checks of a cache and a batch that every call makes.
int check_cache(const char* who, const opc_kv_cache* c) {
  if (!c) return fail(OPC_ERR_INVALID, "%s: cache is NULL", who);
  int64_t total = 0;
  if (c->kv_heads < 1 || c->kv_heads > 65535 || !head_dim_ok(c->head_dim) || !page_size_ok(c->page_size) || c->n_pages < 1 ||
      c->head_bytes != static_cast<int64_t>(c->page_size) * (c->head_dim + 8) ||
      !cache_bytes(c->n_pages, c->kv_heads, c->head_bytes, &total) || c->total_bytes != total)
    return fail(OPC_ERR_INVALID, "%s: the cache is not one that opc_kv_plan filled (kv_heads %d, head_dim %d, page_size %d, n_pages %d)",
                who, c->kv_heads, c->head_dim, c->page_size, c->n_pages);
  if (!c->pages || !aligned16(c->pages)) return fail(OPC_ERR_INVALID, "%s: cache.pages must be a 16-byte aligned device pointer", who);
  return OPC_OK;
}
int check_batch(const char* who, const opc_kv_batch* b) {
  if (!b) return fail(OPC_ERR_INVALID, "%s: batch is NULL", who);
  if (b->n_seqs < 0 || b->n_tokens < 0 || b->max_q < 0 || b->max_kv < 0 || b->max_pages < 0)
    return fail(OPC_ERR_INVALID, "%s: negative size in the batch (n_seqs %d, n_tokens %d, max_q %d, max_kv %d, max_pages %d)", who,
                b->n_seqs, b->n_tokens, b->max_q, b->max_kv, b->max_pages);
  if (b->n_seqs > 65535) return fail(OPC_ERR_INVALID, "%s: n_seqs %d above 65535", who, b->n_seqs);
  if (b->table_stride < b->max_pages)
    return fail(OPC_ERR_INVALID, "%s: table_stride %lld below max_pages %d", who, static_cast<long long>(b->table_stride), b->max_pages);
  if (b->n_seqs > 0 && b->n_tokens > 0 && (!b->q_start || !b->kv_len || (b->max_pages > 0 && !b->page_table)))
    return fail(OPC_ERR_INVALID, "%s: the batch's q_start, kv_len or page_table is NULL", who);
  return OPC_OK;
}
int check_type(const char* who, int32_t dtype) {
  if (dtype == OPC_F16 || dtype == OPC_BF16) return OPC_OK;
  return fail(OPC_ERR_UNSUPPORTED, "%s: element type %d (OPC_F16 and OPC_BF16 are supported)", who, dtype);
}
int check_matrix(const char* who, const char* name, const void* p, int64_t ld, int64_t cols) {
  if (!p) return fail(OPC_ERR_INVALID, "%s: %s is NULL", who, name);
  if (reinterpret_cast<uintptr_t>(p) & 1u) return fail(OPC_ERR_INVALID, "%s: %s is not aligned to its elements", who, name);
  if (ld < cols) return fail(OPC_ERR_INVALID, "%s: leading dimension %lld of %s below its %lld columns", who, static_cast<long long>(ld), name, static_cast<long long>(cols));
  return OPC_OK;
}
#define KV_CHECK(call)                 \
  do {                                 \
    const int rc_ = (call);            \
    if (rc_ != OPC_OK) return rc_;     \
  } while (0)

opc::KvGeom geom_of(const opc_kv_cache& c) {
  opc::KvGeom g;
  g.pages = static_cast<uint8_t*>(c.pages);
  g.head_bytes = c.head_bytes;
  g.kv_heads = c.kv_heads;
  g.hd = c.head_dim;
  g.page_size = c.page_size;
  g.page_shift = __builtin_ctz(static_cast<unsigned>(c.page_size));
  g.n_pages = c.n_pages;
  return g;
}
opc::KvRows rows_of(const opc_kv_batch& b, const opc_kv_cache& c, int* err) {
  opc::KvRows r;
  r.q_start = b.q_start;
  r.kv_len = b.kv_len;
  r.table = b.page_table;
  r.table_stride = b.table_stride;
  r.n_seqs = b.n_seqs;
  r.n_tokens = b.n_tokens;
  r.max_q = b.max_q;
  // (page counts are kept below 2^31 positions, so positions and their sums with tiles stay in 32 bits)
  r.max_pages = static_cast<int32_t>(std::min<int64_t>(b.max_pages, (INT32_MAX - 1024) / c.page_size));
  r.max_kv = std::min(b.max_kv, r.max_pages * c.page_size);
  r.err = err;
  return r;
}

// Lanes that take one head: head_dim / 8, rounded up to a power of two.
int lanes_per_head(int hd) {
  int n = 4;
  while (n < hd / 8) n *= 2;
  return n;
}

template <int kLpr, int kTok>
auto append_of(bool bf, bool vec) {
  return bf ? (vec ? opc::kv_append_kernel<kLpr, kTok, true, true> : opc::kv_append_kernel<kLpr, kTok, true, false>)
            : (vec ? opc::kv_append_kernel<kLpr, kTok, false, true> : opc::kv_append_kernel<kLpr, kTok, false, false>);
}
template <int kTok>
auto append_for(int lpr, bool bf, bool vec) {
  return lpr == 4 ? append_of<4, kTok>(bf, vec) : lpr == 8 ? append_of<8, kTok>(bf, vec)
       : lpr == 16 ? append_of<16, kTok>(bf, vec) : append_of<32, kTok>(bf, vec);
}
template <int kLpr>
auto read_of(bool bf, bool vec) {
  return bf ? (vec ? opc::kv_read_kernel<kLpr, true, true> : opc::kv_read_kernel<kLpr, true, false>)
            : (vec ? opc::kv_read_kernel<kLpr, false, true> : opc::kv_read_kernel<kLpr, false, false>);
}
auto read_for(int lpr, bool bf, bool vec) {
  return lpr == 4 ? read_of<4>(bf, vec) : lpr == 8 ? read_of<8>(bf, vec) : lpr == 16 ? read_of<16>(bf, vec) : read_of<32>(bf, vec);
}

// ------------------------------------------------------------------------------------------------
// Attention: how a call is divided
// ------------------------------------------------------------------------------------------------
struct AttentionPlan {
  int step_nt;          // row tiles of the step kernel, 0: not launched
  int step_q;           // the step kernel takes sequences of at most this many rows
  int step_grid;
  int64_t prompt_grid;  // 0: the prompt kernel is not launched
  int prompt_ctas;      // CTAs that may share their items' keys
  size_t bytes;         // workspace: the counters, then the records (of one kernel after the other)
};

constexpr size_t kCounterBytes = 4096;  // one per CTA of a launch

// The step kernel takes sequences of at most this many rows.
int step_rows(const opc_kv_cache& c, const opc_kv_batch& b, int group) {
  // Row tiles of 8 (query token, head) pairs: two where the accumulators leave registers for them.  (Heads
  // of 128, four rows of four heads over 4000 keys: 20 us in the step kernel, 35 in the prompt kernel;
  // 16 such sequences 39 and 96.)
  const int most = c.head_dim <= 128 ? 16 : 8;
  const int q = std::min(std::max(b.max_q, 0), most / group);
  // Where a sequence of few rows would leave rows of the batch to nobody, as with one sequence, the prompt
  // kernel takes what there is (five rows of four heads over 4000 keys: 47 us after a step kernel that
  // finds nothing to do, 36 without).
  return b.max_q > q && b.n_tokens > (b.n_seqs - 1LL) * b.max_q + q ? 0 : q;
}

// At most this many tile pairs, over all kv heads, are the prompt kernel's: the rows of all sequences, and one
// that is not full for each.
int64_t prompt_items(const opc_kv_cache& c, const opc_kv_batch& b, int group) {
  const int step_q = step_rows(c, b, group);
  if (b.max_q <= step_q) return 0;
  const int64_t rows = static_cast<int64_t>(opc::kv_p_qt(c.head_dim)) * opc::kKvPM;
  const int64_t pairs = (static_cast<int64_t>(b.max_q) * group + rows - 1) / rows;
  const int64_t all = std::min(pairs * b.n_seqs, static_cast<int64_t>(b.n_tokens) * group / rows +
                                                     std::min(b.n_seqs, b.n_tokens / (step_q + 1)));
  return std::max<int64_t>(1, all * c.kv_heads);
}

AttentionPlan plan_attention(const opc_kv_cache& c, const opc_kv_batch& b, int group, int sms) {
  AttentionPlan p{};
  p.step_q = step_rows(c, b, group);
  p.bytes = kCounterBytes;
  if (p.step_q > 0) {
    p.step_nt = p.step_q * group > 8 ? 2 : 1;
    p.step_grid = std::min<int>(sms * opc::kv_step_ctas(c.head_dim, p.step_nt), kCounterBytes / 4);
    p.bytes += static_cast<size_t>(p.step_grid) * 2 * (p.step_q * group) * (c.head_dim + 4) * 4;
  }
  if (b.max_q > p.step_q) {
    const int64_t rows = static_cast<int64_t>(opc::kv_p_qt(c.head_dim)) * opc::kKvPM;
    p.prompt_grid = prompt_items(c, b, group);
    // Fewer items than SMs share their keys, down to two tiles for each CTA.
    p.prompt_ctas = 1;
    if (b.max_kv > 3 * opc::kKvPN) {
      p.prompt_ctas = std::min<int>(sms, kCounterBytes / 4);
      p.prompt_grid = std::max<int64_t>(p.prompt_grid, p.prompt_ctas);
      p.bytes = std::max(p.bytes, kCounterBytes + static_cast<size_t>(p.prompt_ctas) * rows * (c.head_dim + 4) * 4);
    }
  }
  return p;
}

template <int kNT>
auto step_of(int hd) {
  if constexpr (kNT == 1) {
    if (hd == 192) return opc::kv_attention_step_kernel<192, 1>;
    if (hd == 256) return opc::kv_attention_step_kernel<256, 1>;
  }
  return hd == 32 ? opc::kv_attention_step_kernel<32, kNT> : hd == 64 ? opc::kv_attention_step_kernel<64, kNT>
       : hd == 96 ? opc::kv_attention_step_kernel<96, kNT> : opc::kv_attention_step_kernel<128, kNT>;
}

auto prompt_of(int hd) {
  return hd == 32 ? opc::kv_attention_prompt_kernel<32> : hd == 64 ? opc::kv_attention_prompt_kernel<64>
       : hd == 96 ? opc::kv_attention_prompt_kernel<96> : hd == 128 ? opc::kv_attention_prompt_kernel<128>
       : hd == 192 ? opc::kv_attention_prompt_kernel<192> : opc::kv_attention_prompt_kernel<256>;
}

// Launched with programmatic serialization: set-up overlaps the kernel before, which each of these
// kernels waits for before it reads anything.
template <typename... KArgs, typename... Args>
cudaError_t launch_pdl(void (*kern)(KArgs...), dim3 grid, int threads, int smem, cudaStream_t s, Args... args) {
  if (smem > 48 * 1024) {  // (once per kernel and device: the size is the kernel's own)
    static std::mutex mu;
    static std::set<std::pair<const void*, int>> done;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const std::pair<const void*, int> key(reinterpret_cast<const void*>(kern), dev);
    try {  // (no exception leaves a C entry)
      std::lock_guard<std::mutex> lk(mu);
      if (!done.count(key)) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
        done.insert(key);
      }
    } catch (...) {
      return cudaErrorMemoryAllocation;
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...);
}

}  // namespace

extern "C" {

int opc_kv_plan(int32_t kv_heads, int32_t head_dim, int32_t page_size, int32_t n_pages, opc_kv_cache* cache) {
  if (!cache) return fail(OPC_ERR_INVALID, "opc_kv_plan: cache is NULL");
  if (kv_heads < 1 || kv_heads > 65535 || n_pages < 1)
    return fail(OPC_ERR_INVALID, "opc_kv_plan: kv_heads %d, n_pages %d", kv_heads, n_pages);
  if (!head_dim_ok(head_dim)) return fail(OPC_ERR_UNSUPPORTED, "opc_kv_plan: head_dim %d (32, 64, 96, 128, 192 and 256 are supported)", head_dim);
  if (!page_size_ok(page_size)) return fail(OPC_ERR_UNSUPPORTED, "opc_kv_plan: page_size %d (16, 32, 64, 128 and 256 are supported)", page_size);
  const int64_t head_bytes = static_cast<int64_t>(page_size) * (head_dim + 8);
  int64_t total = 0;
  if (!cache_bytes(n_pages, kv_heads, head_bytes, &total))
    return fail(OPC_ERR_INVALID, "opc_kv_plan: %d pages of %d kv heads are more than 2^63 bytes", n_pages, kv_heads);
  cache->kv_heads = kv_heads;
  cache->head_dim = head_dim;
  cache->page_size = page_size;
  cache->n_pages = n_pages;
  cache->head_bytes = head_bytes;
  cache->total_bytes = total;
  cache->pages = nullptr;
  return OPC_OK;
}

int opc_rope_turns(const double* f, int32_t n, uint64_t* turns) {
  if (n < 0 || (n > 0 && (!f || !turns))) return fail(OPC_ERR_INVALID, "opc_rope_turns: NULL argument or n %d", n);
  for (int32_t i = 0; i < n; ++i) {
    if (!std::isfinite(f[i])) return fail(OPC_ERR_INVALID, "opc_rope_turns: frequency %d is not finite", i);
    // f / 2pi modulo 1 in the 64-bit mantissa of long double, as a fraction of 2^64
    long double t = static_cast<long double>(f[i]) / 6.283185307179586476925286766559L;
    t -= std::floor(t);
    const long double u = std::nearbyint(t * 18446744073709551616.0L);
    turns[i] = u >= 18446744073709551616.0L ? 0u : static_cast<uint64_t>(u);
  }
  return OPC_OK;
}

int opc_kv_append(const opc_kv_cache* cache, const opc_kv_batch* batch, int32_t heads, int32_t dtype,
                  const opc_rope* rope, const void* k, int64_t ldk, const void* v, int64_t ldv, const void* q,
                  int64_t ldq, void* q_out, int64_t ldqo, void* stream) {
  const char* who = "opc_kv_append";
  KV_CHECK(check_cache(who, cache));
  KV_CHECK(check_batch(who, batch));
  KV_CHECK(check_type(who, dtype));
  const int hd = cache->head_dim, kvh = cache->kv_heads;
  if (heads < 0 || heads > 65535) return fail(OPC_ERR_INVALID, "%s: heads %d", who, heads);
  if ((q != nullptr) != (q_out != nullptr)) return fail(OPC_ERR_INVALID, "%s: q and q_out go together", who);
  if (q && heads < 1) return fail(OPC_ERR_INVALID, "%s: q given with %d heads", who, heads);
  if (rope) {
    if (rope->rot_dim < 16 || rope->rot_dim % 16 || rope->rot_dim > hd)
      return fail(OPC_ERR_UNSUPPORTED, "%s: rot_dim %d (a multiple of 16 up to head_dim %d)", who, rope->rot_dim, hd);
    if (!rope->turns || (reinterpret_cast<uintptr_t>(rope->turns) & 7u))
      return fail(OPC_ERR_INVALID, "%s: rope.turns must be an 8-byte aligned device pointer", who);
  }
  if (batch->n_tokens == 0 || batch->n_seqs == 0) return OPC_OK;
  KV_CHECK(check_matrix(who, "k", k, ldk, static_cast<int64_t>(kvh) * hd));
  KV_CHECK(check_matrix(who, "v", v, ldv, static_cast<int64_t>(kvh) * hd));
  if (q) {
    KV_CHECK(check_matrix(who, "q", q, ldq, static_cast<int64_t>(heads) * hd));
    KV_CHECK(check_matrix(who, "q_out", q_out, ldqo, static_cast<int64_t>(heads) * hd));
  }
  opc_host::Device dev;
  KV_CHECK(opc_host::current_device(&dev));
  opc::KvAppendArgs a;
  a.C = geom_of(*cache);
  a.B = rows_of(*batch, *cache, dev.error_word);
  a.k = static_cast<const uint16_t*>(k);
  a.v = static_cast<const uint16_t*>(v);
  a.q = static_cast<const uint16_t*>(q);
  a.q_out = static_cast<uint16_t*>(q_out);
  a.ldk = ldk;
  a.ldv = ldv;
  a.ldq = ldq;
  a.ldqo = ldqo;
  a.heads = q ? heads : 0;
  a.rot_dim = rope ? rope->rot_dim : 0;
  a.interleaved = rope ? rope->interleaved != 0 : 0;
  a.turns = rope ? rope->turns : nullptr;
  const bool vec = aligned16(k) && aligned16(v) && ldk % 8 == 0 && ldv % 8 == 0 &&
                   (!q || (aligned16(q) && aligned16(q_out) && ldq % 8 == 0 && ldqo % 8 == 0));
  const int lpr = lanes_per_head(hd), groups = opc::kKvAppendThreads / lpr, all = 2 * kvh + a.heads;
  const bool bf = dtype == OPC_BF16;
  // few rows: a CTA per row and `groups` heads; many: four rows per CTA, which share its set-up (32/8 heads
  // of 128: 96 rows 3.7 and 9.5 us, 600 rows 8.9 and 11.0, 1200 rows 14.5 and 13.8, 5000 rows 51 and 36)
  const bool few = batch->n_tokens < 6 * dev.sm_count;
  const int tok = few ? 1 : 4;
  const dim3 grid((batch->n_tokens + tok - 1) / tok, few ? (all + groups - 1) / groups : 1);
  auto kern = few ? append_for<1>(lpr, bf, vec) : append_for<4>(lpr, bf, vec);
  KV_CUDA(launch_pdl(kern, grid, opc::kKvAppendThreads, 0, static_cast<cudaStream_t>(stream), a), "opc_kv_append launch");
  return OPC_OK;
}

int opc_kv_read(const opc_kv_cache* cache, const opc_kv_batch* batch, int32_t dtype, void* k, int64_t ldk, void* v,
                int64_t ldv, void* stream) {
  const char* who = "opc_kv_read";
  KV_CHECK(check_cache(who, cache));
  KV_CHECK(check_batch(who, batch));
  KV_CHECK(check_type(who, dtype));
  if (batch->n_tokens == 0 || batch->n_seqs == 0) return OPC_OK;
  const int64_t cols = static_cast<int64_t>(cache->kv_heads) * cache->head_dim;
  KV_CHECK(check_matrix(who, "k", k, ldk, cols));
  KV_CHECK(check_matrix(who, "v", v, ldv, cols));
  opc_host::Device dev;
  KV_CHECK(opc_host::current_device(&dev));
  opc::KvReadArgs a;
  a.C = geom_of(*cache);
  a.B = rows_of(*batch, *cache, dev.error_word);
  a.k = static_cast<uint16_t*>(k);
  a.v = static_cast<uint16_t*>(v);
  a.ldk = ldk;
  a.ldv = ldv;
  const bool vec = aligned16(k) && aligned16(v) && ldk % 8 == 0 && ldv % 8 == 0;
  auto kern = read_for(lanes_per_head(cache->head_dim), dtype == OPC_BF16, vec);
  KV_CUDA(launch_pdl(kern, dim3(batch->n_tokens), opc::kKvAppendThreads, 0, static_cast<cudaStream_t>(stream), a), "opc_kv_read launch");
  return OPC_OK;
}

size_t opc_kv_attention_workspace_bytes(const opc_kv_cache* cache, const opc_kv_batch* batch, int32_t heads,
                                        int32_t device) {
  if (!cache || !batch || heads < 1 || heads > 65535 || cache->kv_heads < 1 || heads % cache->kv_heads ||
      !head_dim_ok(cache->head_dim) || !page_size_ok(cache->page_size) || batch->n_seqs < 0 || batch->max_q < 0 ||
      batch->max_kv < 0)
    return 0;
  int sms = 0;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  return plan_attention(*cache, *batch, heads / cache->kv_heads, sms).bytes;
}

int opc_kv_attention(const opc_kv_cache* cache, const opc_kv_batch* batch, int32_t heads, int32_t dtype, float scale,
                     const void* q, int64_t ldq, void* out, int64_t ldo, float* lse, void* workspace,
                     size_t workspace_bytes, void* stream) {
  const char* who = "opc_kv_attention";
  KV_CHECK(check_cache(who, cache));
  KV_CHECK(check_batch(who, batch));
  KV_CHECK(check_type(who, dtype));
  if (heads < 1 || heads > 65535 || heads % cache->kv_heads)
    return fail(OPC_ERR_INVALID, "%s: %d heads over %d kv heads", who, heads, cache->kv_heads);
  if (!std::isfinite(scale)) return fail(OPC_ERR_INVALID, "%s: scale is not finite", who);
  if (batch->n_tokens == 0 || batch->n_seqs == 0) return OPC_OK;
  const int64_t cols = static_cast<int64_t>(heads) * cache->head_dim;
  KV_CHECK(check_matrix(who, "q", q, ldq, cols));
  KV_CHECK(check_matrix(who, "out", out, ldo, cols));
  const int group = heads / cache->kv_heads;
  const opc::KvRows rows = rows_of(*batch, *cache, nullptr);
  // (the step kernel counts its work in 32 bits: stages of keys, and what an item costs beside them)
  const int64_t stages = std::max(1, (rows.max_kv + opc::kKvStage - 1) / opc::kKvStage) + opc::kKvItemCost;
  if (static_cast<double>(batch->n_seqs) * cache->kv_heads * stages > UINT32_MAX)
    return fail(OPC_ERR_INVALID, "%s: %d sequences of up to %d keys over %d kv heads are too many for one call", who,
                batch->n_seqs, rows.max_kv, cache->kv_heads);
  // (rows are counted in 32 bits, tiles of them in a grid)
  if (static_cast<int64_t>(batch->n_tokens) * group > INT32_MAX - 1024 || prompt_items(*cache, *batch, group) > INT32_MAX)
    return fail(OPC_ERR_INVALID, "%s: %d tokens of %d heads over %d kv heads are too many for one call", who, batch->n_tokens, heads,
                cache->kv_heads);
  opc_host::Device dev;
  KV_CHECK(opc_host::current_device(&dev));
  AttentionPlan p = plan_attention(*cache, *batch, group, dev.sm_count);
  if (!workspace || !aligned16(workspace) || workspace_bytes < p.bytes)
    return fail(OPC_ERR_WORKSPACE, "%s: a 16-byte aligned workspace of %zu bytes is needed, got %zu", who, p.bytes, workspace_bytes);
  opc::KvAttnArgs a;
  a.C = geom_of(*cache);
  a.B = rows;
  a.B.err = dev.error_word;
  a.B.max_q = std::min(a.B.max_q, batch->n_tokens);
  a.q = static_cast<const uint16_t*>(q);
  a.out = static_cast<uint16_t*>(out);
  a.lse = lse;
  a.ldq = ldq;
  a.ldo = ldo;
  a.scale = scale;
  a.heads = heads;
  a.group = group;
  a.bf16 = dtype == OPC_BF16;
  a.vec = aligned16(q) && aligned16(out) && ldq % 8 == 0 && ldo % 8 == 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (p.step_nt) {
    a.lo_q = 1;
    a.hi_q = p.step_q;
    opc::KvSplit sp;
    sp.count = static_cast<int32_t*>(workspace);
    sp.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + kCounterBytes);
    sp.rows = p.step_q * group;
    auto kern = p.step_nt == 2 ? step_of<2>(cache->head_dim) : step_of<1>(cache->head_dim);
    KV_CUDA(launch_pdl(kern, dim3(p.step_grid), opc::kKvStepThreads, opc::kv_step_smem(cache->head_dim, p.step_nt), s, a, sp),
            "opc_kv_attention launch (steps)");
  }
  if (p.prompt_grid) {
    a.lo_q = p.step_q + 1;
    a.hi_q = a.B.max_q;
    opc::KvPromptSplit sp;
    sp.ctas = static_cast<uint32_t>(p.prompt_ctas);
    sp.count = static_cast<int32_t*>(workspace);
    sp.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + kCounterBytes);
    KV_CUDA(launch_pdl(prompt_of(cache->head_dim), dim3(static_cast<unsigned>(p.prompt_grid)), opc::kKvPThreads,
                       opc::kv_p_smem(cache->head_dim), s, a, sp),
            "opc_kv_attention launch (prompts)");
  }
  return OPC_OK;
}

}  // extern "C"
