// opc_i8.cu -- C ABI of the 8-bit products (opc_i8_*, include/opc_b200.h).
#define OPC_WITHOUT_ERROR_WORD
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>
#include <utility>

#include "../../include/opc_b200.h"
#include "opc_i8_gemm.cuh"
#include "opc_i8_rows.cuh"
#include "opc_internal.h"

using opc_host::cuda_fail;
using opc_host::fail;

namespace {

constexpr int kMaxWidth = 131071;           // 128 * 128 * 131071 < 2^31: no sum of products leaves 32 bits
constexpr int kMaxRows = INT32_MAX - 4095;  // rows rounded up to a tile stay below 2^31

int bytes_of(int32_t dtype) { return dtype == OPC_F32 ? 4 : 2; }
bool is_type(int32_t dtype) { return dtype == OPC_F16 || dtype == OPC_BF16 || dtype == OPC_F32; }

// A matrix of `rows` rows of n values at p with leading dimension ld: present and aligned to its elements.
int check_matrix(const char* who, const char* name, const void* p, int64_t ld, int32_t dtype, int32_t n) {
  if (!is_type(dtype)) return fail(OPC_ERR_UNSUPPORTED, "%s: element type %d of %s", who, dtype, name);
  if (!p || (reinterpret_cast<uintptr_t>(p) & (bytes_of(dtype) - 1u)))
    return fail(OPC_ERR_INVALID, "%s: %s is NULL or not aligned to its elements", who, name);
  if (ld < n) return fail(OPC_ERR_INVALID, "%s: leading dimension %lld of %s below %d", who, static_cast<long long>(ld), name, n);
  return OPC_OK;
}

int check_codes(const char* who, const char* name, const opc_i8_rows* m) {
  if (!m) return fail(OPC_ERR_INVALID, "%s: %s is NULL", who, name);
  if (m->rows < 0 || m->rows > kMaxRows || m->n < 1 || m->n > kMaxWidth)
    return fail(OPC_ERR_INVALID, "%s: %s is %d x %d (up to %d rows of 1 to %d values)", who, name, m->rows, m->n, kMaxRows, kMaxWidth);
  if (m->rows == 0) return OPC_OK;
  if (!m->codes || (reinterpret_cast<uintptr_t>(m->codes) & 15u) || m->ld < m->n || (m->ld & 15))
    return fail(OPC_ERR_INVALID, "%s: the codes of %s must start on 16 bytes in rows of a multiple of 16 bytes from %d on, got a leading dimension of %lld",
                who, name, m->n, static_cast<long long>(m->ld));
  if (!m->scales || (reinterpret_cast<uintptr_t>(m->scales) & 3u))
    return fail(OPC_ERR_INVALID, "%s: the scales of %s are NULL or not aligned", who, name);
  return OPC_OK;
}

// Whether every row starts on 16 bytes (a matrix that is not there: yes).
bool vec_ok(const void* p, int64_t ld, int32_t dtype, int32_t rows) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (!p || rows == 1 || (ld * bytes_of(dtype)) % 16 == 0);
}

// Whether `rows` rows of wa bytes, pa bytes apart from a on, and rows of wb bytes at b (as many as far apart, or one: pb 0)
// have no byte in common.
bool apart(const void* a, int64_t pa, int64_t wa, const void* b, int64_t pb, int64_t wb, int32_t rows) {
  using i128 = __int128;
  const i128 from_a = reinterpret_cast<uintptr_t>(a), from_b = reinterpret_cast<uintptr_t>(b);
  const i128 to_a = from_a + static_cast<i128>(rows - 1) * pa + wa, to_b = from_b + static_cast<i128>(pb ? rows - 1 : 0) * pb + wb;
  if (to_a <= from_b || to_b <= from_a) return true;
  if (rows == 1 || (pb && pb != pa)) return false;
  const i128 in = ((from_b - from_a) % pa + pa) % pa;  // where b's rows begin in a's
  return in >= wa && pa - in >= wb;
}

template <typename... KArgs, typename... Args>
cudaError_t launch(void (*kern)(KArgs...), unsigned ctas, int threads, void* stream, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(threads);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];  // the launch overlaps the end of the kernel before, which the kernel waits for
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

// One warp per row up to 1024 values; beyond, one CTA per row with 16 values a thread, or 8 where there
// are few rows and a row up to 8192 values (96 x 8192 bf16 norms 3.4 -> 3.2 us, 512 x 4096 fp32 ones 6.1 ->
// 5.8 us; but 28672 x 4096 quantized 97 -> 111 us), 32 from 16384 values on (shorter rows lose by it: 4097 x
// 14336 gated 62 -> 83 us; longer ones gain over being read twice: 4096 x 28672 gated 152 -> 143 us, normalized 322 ->
// 226; quantized alone they lose by it, 90 -> 108).  Rows of more
// than 32768 values, which no CTA's registers hold, are read twice.  (Clusters of CTAs that share a long row
// were slower than either: 4096 x 28672 gated 141 -> 188 us, 4096 x 40000 quantized 125 -> 181.)  Rows that do
// not all start on 16 bytes are moved value by value.
template <int kOp, int kTX, int kTU>
cudaError_t launch_rows(const opc::I8RowsArgs& a, bool vec, int sms, void* stream) {
  using opc::i8_rows_kernel;
  const int groups = (a.n + 7) / 8;
  if constexpr (kOp == opc::kI8Norm) {
    // Normalized rows beside their codes (tokens for layers of either kind): one kernel for every width, which reads
    // them twice.  In the others two more values to write for a place would take registers from every call (8191 x
    // 4096: 44 a thread would be 54, a CTA an SM less).
    if (a.plain)
      return launch(vec ? i8_rows_kernel<kOp, kTX, kTU, 0, false, true, true> : i8_rows_kernel<kOp, kTX, kTU, 0, false, false, true>, a.rows,
                    std::min(1024, (groups + 31) / 32 * 32), stream, a);
  }
  if (groups <= 128) {
    const int per = (groups + 31) / 32;
    auto k = !vec ? i8_rows_kernel<kOp, kTX, kTU, 4, true, false>
             : per == 1 ? i8_rows_kernel<kOp, kTX, kTU, 1, true, true>
             : per == 2 ? i8_rows_kernel<kOp, kTX, kTU, 2, true, true> : i8_rows_kernel<kOp, kTX, kTU, 4, true, true>;
    return launch(k, (a.rows + 3) / 4, 128, stream, a);
  }
  const int per = vec && groups <= 1024 && a.rows <= 4 * sms ? 1 : groups <= 2048 ? 2 : vec && groups <= 4096 ? 4 : 0;
  const int threads = per ? ((groups + per - 1) / per + 31) / 32 * 32 : 1024;
  auto k = !vec ? (per == 2 ? i8_rows_kernel<kOp, kTX, kTU, 2, false, false> : i8_rows_kernel<kOp, kTX, kTU, 0, false, false>)
           : per == 1 ? i8_rows_kernel<kOp, kTX, kTU, 1, false, true>
           : per == 2 ? i8_rows_kernel<kOp, kTX, kTU, 2, false, true>
           : per == 4 ? i8_rows_kernel<kOp, kTX, kTU, 4, false, true> : i8_rows_kernel<kOp, kTX, kTU, 0, false, true>;
  return launch(k, a.rows, threads, stream, a);
}

template <int kOp, int kTU>
cudaError_t launch_rows_x(int32_t x_type, const opc::I8RowsArgs& a, bool vec, int sms, void* stream) {
  if (x_type == OPC_F16) return launch_rows<kOp, opc::kI8F16, kTU == 4 ? opc::kI8F16 : kTU>(a, vec, sms, stream);
  if (x_type == OPC_BF16) return launch_rows<kOp, opc::kI8BF16, kTU == 4 ? opc::kI8BF16 : kTU>(a, vec, sms, stream);
  return launch_rows<kOp, opc::kI8F32, kTU == 4 ? opc::kI8F32 : kTU>(a, vec, sms, stream);
}
constexpr int kSame = 4;  // launch_rows_x: the second operand has the first one's type

// What the three quantizing calls share: the output's checks and arguments.
int start_rows(const char* who, const opc_i8_rows* out, void* values, int64_t ldv, int32_t v_dtype, opc::I8RowsArgs* a) {
  const int rc = check_codes(who, "the output", out);
  if (rc != OPC_OK || out->rows == 0) return rc;
  if (values) {
    const int rv = check_matrix(who, "values", values, ldv, v_dtype, out->n);
    if (rv != OPC_OK) return rv;
  }
  *a = {};
  a->rows = out->rows;
  a->n = out->n;
  a->codes = out->codes;
  a->ldc = out->ld;
  a->scales = out->scales;
  a->values = values;
  a->ldv = ldv;
  a->v_type = v_dtype;
  return OPC_OK;
}

// ---- the product's plan
// i8_plan, remembered by its sizes (a thread's last few; the choice costs about a microsecond).
opc::I8Plan plan_of(int32_t rows, int32_t M, int32_t K, const int (&clusters)[5]) {
  struct Known {
    int32_t rows, M, K;
    int clusters[5];
    opc::I8Plan plan;
  };
  thread_local Known known[8] = {};
  Known& k = known[(static_cast<uint32_t>(rows) * 31u + static_cast<uint32_t>(M) * 7u + static_cast<uint32_t>(K)) / 32u % 8u];
  if (k.rows != rows || k.M != M || k.K != K || !std::equal(clusters + 1, clusters + 5, k.clusters + 1)) {
    k.plan = opc::i8_plan(rows, M, K, clusters);
    k.rows = rows;
    k.M = M;
    k.K = K;
    std::copy(clusters + 1, clusters + 5, k.clusters + 1);
  }
  return k.plan;
}

// Rows of codes as a tensor of bytes, in boxes of 128 bytes x box rows, zeros beyond its edges.
int map_codes(const char* who, const opc_i8_rows* m, int box, CUtensorMap* map) {
  auto encode = opc_host::tensor_map_encoder();
  if (!encode) return fail(OPC_ERR_CUDA, "%s: cuTensorMapEncodeTiled unavailable", who);
  const cuuint64_t dim[2] = {static_cast<cuuint64_t>(m->n), static_cast<cuuint64_t>(m->rows)};
  const cuuint64_t stride[1] = {static_cast<cuuint64_t>(m->ld)};
  const cuuint32_t boxes[2] = {opc::kI8Block, static_cast<cuuint32_t>(box)}, step[2] = {1, 1};
  const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, m->codes, dim, stride, boxes, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? OPC_OK : fail(OPC_ERR_CUDA, "%s: cuTensorMapEncodeTiled failed (%d)", who, static_cast<int>(r));
}

void gemm_config(int ctas, int split, cudaLaunchConfig_t* cfg, cudaLaunchAttribute (&attr)[2]) {
  cfg->gridDim = dim3(ctas);
  cfg->blockDim = dim3(opc::kI8Threads);
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2 * split;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg->attrs = attr;
  cfg->numAttrs = 2;
}

// Once per device and kernel (number `which`): its shared memory, and how many clusters of 1 to 4 pairs
// run at once (0: none).
template <typename K>
cudaError_t gemm_setup(K k, int which, int (*clusters)[5]) {
  static std::atomic<uint32_t> known[64][3];  // 7 bits for each, and bit 31
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  uint32_t v = dev < 64 ? known[dev][which].load(std::memory_order_acquire) : 0u;
  if (!v) {
    e = cudaFuncSetAttribute(reinterpret_cast<const void*>(k), cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
    if (e != cudaSuccess) return e;
    v = 1u << 31;
    for (int split = 1, at = 0; split <= 4; ++split, at += 7) {
      cudaLaunchConfig_t cfg = {};
      cudaLaunchAttribute attr[2];
      gemm_config(2 * split, split, &cfg, attr);
      cfg.dynamicSmemBytes = 227 * 1024;
      int n = 0;
      if ((e = cudaOccupancyMaxActiveClusters(&n, k, &cfg)) != cudaSuccess) return e;
      v |= static_cast<uint32_t>(std::max(0, std::min(n, 127))) << at;
    }
    if (dev < 64) known[dev][which].store(v, std::memory_order_release);
  }
  for (int split = 1; split <= 4; ++split) (*clusters)[split] = static_cast<int>((v >> (7 * (split - 1))) & 127u);
  (*clusters)[1] = std::max(1, (*clusters)[1]);
  return cudaSuccess;
}

// ---- few tokens
struct GemvKernel {
  void (*kernel)(const int8_t*, int64_t, const int8_t*, int64_t, int32_t, opc::I8Out);
  int threads;
};
// 16 warps share K, or 8 where it is short (1024 -> 32768: 10.7 -> 8.3 us); each has one step of 128 values
// under way at a time, or two where there are few CTAs with long rows (14336 -> 4096: 13.4 -> 13.1 us,
// 4096 -> 4096 5.7 -> 5.2; but 4096 -> 28672 20.5 -> 22.9).
template <int kY, int kTok>
GemvKernel gemv_kernel_t(int32_t M, int32_t K, int sms) {
  if (K < 2048) return {opc::i8_gemv_kernel<kY, kTok, 8, 1>, 256};
  if (K >= 4096 && (M + 15) / 16 <= 2 * sms) return {opc::i8_gemv_kernel<kY, kTok, 16, 2>, 512};
  return {opc::i8_gemv_kernel<kY, kTok, 16, 1>, 512};
}
template <int kY>
GemvKernel gemv_kernel(int32_t rows, int32_t M, int32_t K, int sms) {
  return rows <= 8 ? gemv_kernel_t<kY, 1>(M, K, sms) : gemv_kernel_t<kY, 2>(M, K, sms);
}

int end_rows(const char* who, cudaError_t e) { return e == cudaSuccess ? OPC_OK : cuda_fail(e, who); }

}  // namespace

extern "C" {

int opc_i8_quantize(const void* x, int64_t ldx, int32_t dtype, const opc_i8_rows* out, void* values, int64_t ldv,
                    int32_t v_dtype, void* stream) {
  const char* who = "opc_i8_quantize";
  opc::I8RowsArgs a;
  int rc = start_rows(who, out, values, ldv, v_dtype, &a);
  if (rc != OPC_OK || out->rows == 0) return rc;
  if ((rc = check_matrix(who, "x", x, ldx, dtype, out->n)) != OPC_OK) return rc;
  a.x = x;
  a.ldx = ldx;
  const bool vec = vec_ok(x, ldx, dtype, out->rows) && vec_ok(values, ldv, v_dtype, out->rows);
  opc_host::Device dev;
  if ((rc = opc_host::current_device(&dev)) != OPC_OK) return rc;
  return end_rows(who, launch_rows_x<opc::kI8Quant, opc::kI8None>(dtype, a, vec, dev.sm_count, stream));
}

int opc_i8_add_rmsnorm(const void* h, int64_t ldh, int32_t h_dtype, const void* y, int64_t ldy, int32_t y_dtype,
                       const void* weight, int32_t w_dtype, float eps, void* h_out, int64_t ldho, const opc_i8_rows* out,
                       void* values, int64_t ldv, int32_t v_dtype, void* stream) {
  const char* who = "opc_i8_add_rmsnorm";
  opc::I8RowsArgs a;
  const bool unrounded = values && (v_dtype & OPC_I8_UNROUNDED);
  if (unrounded) v_dtype &= ~OPC_I8_UNROUNDED;
  int rc = start_rows(who, out, values, ldv, v_dtype, &a);
  if (rc != OPC_OK || out->rows == 0) return rc;
  if (unrounded) std::swap(a.values, a.plain);
  const int32_t n = out->n;
  if ((rc = check_matrix(who, "h", h, ldh, h_dtype, n)) != OPC_OK) return rc;
  if (y && (rc = check_matrix(who, "y", y, ldy, y_dtype, n)) != OPC_OK) return rc;
  if (y && y_dtype != h_dtype && h_dtype != OPC_F32)
    return fail(OPC_ERR_UNSUPPORTED, "%s: y of type %d beside h of type %d (the same, or h of type %d)", who, y_dtype, h_dtype, OPC_F32);
  if (weight && (rc = check_matrix(who, "weight", weight, n, w_dtype, n)) != OPC_OK) return rc;
  if (h_out && (rc = check_matrix(who, "h_out", h_out, ldho, h_dtype, n)) != OPC_OK) return rc;
  if (h_out) {  // written row by row while others are read: place for place over h or y, or apart from what is read
    const int64_t size = bytes_of(h_dtype), p = ldho * size, bytes = n * size, y_size = bytes_of(y_dtype);
    const auto same = [&](const void* q, int64_t ldq) { return h_out == q && (ldho == ldq || out->rows == 1); };
    if (!(same(h, ldh) || apart(h_out, p, bytes, h, ldh * size, bytes, out->rows)) ||
        (y && !((y_dtype == h_dtype && same(y, ldy)) || apart(h_out, p, bytes, y, ldy * y_size, n * y_size, out->rows))) ||
        (weight && !apart(h_out, p, bytes, weight, 0, static_cast<int64_t>(n) * bytes_of(w_dtype), out->rows)))
      return fail(OPC_ERR_INVALID, "%s: h_out overlaps h, y or the weight (it may be h, or y of its type, place for place)", who);
  }
  if (!(eps >= 1e-12f) || !std::isfinite(eps)) return fail(OPC_ERR_INVALID, "%s: eps %g (1e-12 or more)", who, static_cast<double>(eps));
  a.x = h;
  a.ldx = ldh;
  a.u = y;
  a.ldu = ldy;
  a.w = weight;
  a.w_type = w_dtype;
  a.h_out = h_out;
  a.ldh = ldho;
  a.eps = eps;
  a.inv_n = 1.0f / static_cast<float>(n);
  const int32_t rows = out->rows;
  const bool vec = vec_ok(h, ldh, h_dtype, rows) && vec_ok(y, ldy, y_dtype, rows) && vec_ok(weight, n, w_dtype, 1) &&
                   vec_ok(h_out, ldho, h_dtype, rows) && vec_ok(values, ldv, v_dtype, rows);
  opc_host::Device dev;
  if ((rc = opc_host::current_device(&dev)) != OPC_OK) return rc;
  cudaError_t e;
  if (!y) e = launch_rows_x<opc::kI8Norm, opc::kI8None>(h_dtype, a, vec, dev.sm_count, stream);
  else if (y_dtype == h_dtype) e = launch_rows_x<opc::kI8Norm, kSame>(h_dtype, a, vec, dev.sm_count, stream);
  else if (y_dtype == OPC_F16) e = launch_rows<opc::kI8Norm, opc::kI8F32, opc::kI8F16>(a, vec, dev.sm_count, stream);
  else e = launch_rows<opc::kI8Norm, opc::kI8F32, opc::kI8BF16>(a, vec, dev.sm_count, stream);
  return end_rows(who, e);
}

int opc_i8_silu_mul(const void* gate, int64_t ldg, const void* up, int64_t ldu, int32_t dtype, const opc_i8_rows* out,
                    void* values, int64_t ldv, int32_t v_dtype, void* stream) {
  const char* who = "opc_i8_silu_mul";
  opc::I8RowsArgs a;
  int rc = start_rows(who, out, values, ldv, v_dtype, &a);
  if (rc != OPC_OK || out->rows == 0) return rc;
  if ((rc = check_matrix(who, "gate", gate, ldg, dtype, out->n)) != OPC_OK) return rc;
  if ((rc = check_matrix(who, "up", up, ldu, dtype, out->n)) != OPC_OK) return rc;
  a.x = gate;
  a.ldx = ldg;
  a.u = up;
  a.ldu = ldu;
  const bool vec = vec_ok(gate, ldg, dtype, out->rows) && vec_ok(up, ldu, dtype, out->rows) && vec_ok(values, ldv, v_dtype, out->rows);
  opc_host::Device dev;
  if ((rc = opc_host::current_device(&dev)) != OPC_OK) return rc;
  return end_rows(who, launch_rows_x<opc::kI8Silu, kSame>(dtype, a, vec, dev.sm_count, stream));
}

int opc_i8_gemm(const opc_i8_rows* x, const opc_i8_rows* w, const void* bias, int32_t bias_dtype, void* y, int64_t ldy,
                int32_t y_dtype, void* stream) {
  const char* who = "opc_i8_gemm";
  int rc = check_codes(who, "x", x);
  if (rc != OPC_OK || (rc = check_codes(who, "w", w)) != OPC_OK) return rc;
  if (x->n != w->n) return fail(OPC_ERR_INVALID, "%s: x has rows of %d values, w of %d", who, x->n, w->n);
  if (w->rows < 1) return fail(OPC_ERR_INVALID, "%s: w has no rows", who);
  if (x->rows == 0) return OPC_OK;
  if ((rc = check_matrix(who, "y", y, ldy, y_dtype, w->rows)) != OPC_OK) return rc;
  if (bias && (rc = check_matrix(who, "bias", bias, w->rows, bias_dtype, w->rows)) != OPC_OK) return rc;
  opc_host::Device dev;
  if ((rc = opc_host::current_device(&dev)) != OPC_OK) return rc;
  const opc::I8Out o = {x->scales, w->scales, bias, y, ldy, x->rows, w->rows, bias_dtype};
  // Few tokens by mma.sync; beyond 8, which it reads twice as often, only where the weights are few (16 tokens,
  // 4096 -> 4096: 6.7 us instead of 9.0; 4096 -> 28672: 31.7 instead of 22.6).
  if (x->rows <= 8 || (x->rows <= 16 && static_cast<int64_t>(w->rows) * w->n <= 1 << 24)) {
    const GemvKernel g = y_dtype == OPC_F16 ? gemv_kernel<opc::kI8F16>(x->rows, w->rows, x->n, dev.sm_count)
                         : y_dtype == OPC_BF16 ? gemv_kernel<opc::kI8BF16>(x->rows, w->rows, x->n, dev.sm_count)
                                               : gemv_kernel<opc::kI8F32>(x->rows, w->rows, x->n, dev.sm_count);
    return end_rows(who, launch(g.kernel, (w->rows + 15) / 16, g.threads, stream, x->codes, x->ld, w->codes, w->ld, x->n, o));
  }
  auto k = y_dtype == OPC_F16 ? opc::i8_gemm_kernel<opc::kI8F16>
           : y_dtype == OPC_BF16 ? opc::i8_gemm_kernel<opc::kI8BF16> : opc::i8_gemm_kernel<opc::kI8F32>;
  int clusters[5];
  cudaError_t e = gemm_setup(k, y_dtype, &clusters);
  if (e != cudaSuccess) return cuda_fail(e, "opc_i8_gemm: setting up");
  const opc::I8Plan p = plan_of(x->rows, w->rows, x->n, clusters);
  if (!p.ctas) return fail(OPC_ERR_UNSUPPORTED, "%s: %d tokens times %d channels are too many tiles for one call", who, x->rows, w->rows);
  opc::I8GemmArgs a = {o, p.deal, dev.error_word};
  CUtensorMap tw, tx;
  if ((rc = map_codes(who, w, 128, &tw)) != OPC_OK || (rc = map_codes(who, x, p.deal.tile_n / 2, &tx)) != OPC_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  gemm_config(p.ctas, p.deal.split, &cfg, attr);
  cfg.dynamicSmemBytes = 1024 + static_cast<size_t>(opc::i8_stages(p.deal.tile_n, p.deal.sub)) * p.deal.sub * opc::i8_block_bytes(p.deal.tile_n) + 512;
  cfg.stream = static_cast<cudaStream_t>(stream);
  return end_rows(who, cudaLaunchKernelEx(&cfg, k, tw, tx, a));
}

}  // extern "C"
