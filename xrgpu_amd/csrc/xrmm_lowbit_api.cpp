// C ABI of the MX4 operators and the 8-bit paged cache: argument checks and dispatch.
#include <hip/hip_runtime.h>

#include <cmath>
#include <string>

#include "../../include/xrmm.h"
#include "xrmm_mx4.h"

namespace {

using xrmm::set_status;

int fail(const char* msg) { return set_status(XRMM_EINVAL, msg); }

int done(hipError_t e, const char* what) {
  return e == hipSuccess ? set_status(XRMM_OK, "") : set_status(XRMM_EDEVICE, std::string(what) + ": " + hipGetErrorString(e));
}

// -1: not a type of these operators
int type_of(int32_t d) {
  return d == XRMM_F32 ? xrmm::LT_F32 : d == XRMM_F16 ? xrmm::LT_F16 : d == XRMM_BF16 ? xrmm::LT_BF16 : -1;
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

constexpr int64_t kMaxK = int64_t(1) << 23;  // 64 rows of 16-bit values stay below 2^31 bytes

int mx4_geometry(xrmm::MxArgs& a, int64_t M, int64_t K, int64_t N, int32_t a_dtype, int32_t out_dtype) {
  if (K <= 0 || K > kMaxK) return fail("matmul_mx4: K must be positive and at most 2^23");
  if (N <= 0 || N > 0x7FFFFFFF) return fail("matmul_mx4: N must be positive and below 2^31");
  if (M < 0 || M > 0x7FFFFFFF) return fail("matmul_mx4: M must be non-negative and below 2^31");
  a = xrmm::MxArgs{};
  a.a_type = a_dtype == XRMM_U8 ? -1 : type_of(a_dtype);
  if (a_dtype != XRMM_U8 && a.a_type != xrmm::LT_F16 && a.a_type != xrmm::LT_BF16)
    return fail("matmul_mx4: A must be float16, bfloat16 or MX4 codes (uint8)");
  a.out = type_of(out_dtype);
  if (a.out < 0) return fail("matmul_mx4: the output must be float32, float16 or bfloat16");
  a.M = M;
  a.K = K;
  a.N = N;
  a.kb = (K + xrmm::MX_BLOCK - 1) / xrmm::MX_BLOCK;
  return XRMM_OK;
}

int cache_of(xrmm::KvCache& c, void* k, void* v, void* ks, void* vs, const void* table, const void* lengths,
             const void* starts, void* status, int64_t pages, int32_t page, int32_t heads, int32_t dim, int32_t cache_dtype,
             int32_t B, int32_t width, int64_t rows) {
  if (cache_dtype != XRMM_I8 && cache_dtype != XRMM_E4M3) return fail("kv8: the cache must be int8 or float8_e4m3fn");
  if (dim != 64 && dim != 96 && dim != 128 && dim != 256) return fail("kv8: head size must be 64, 96, 128 or 256");
  if (page < 16 || page > 256 || (page & (page - 1)) != 0) return fail("kv8: page size must be a power of two from 16 to 256");
  if (heads <= 0 || pages <= 0 || pages > 0x7FFFFFFF) return fail("kv8: the cache needs pages and heads");
  if (B < 0 || width < 0 || rows < 0 || rows > 0x7FFFFFFF) return fail("kv8: negative batch, table width or rows");
  if (static_cast<int64_t>(width) * page > 0x7FFFFF00) return fail("kv8: the table spans 2^31 tokens or more");
  if (B > 0 && starts == nullptr && rows % B != 0) return fail("kv8: rows of unequal counts need starts");
  if (B == 0 && rows != 0) return fail("kv8: rows without sequences");
  if (B > 0 && rows > 0 && (!k || !v || !ks || !vs || !table || !lengths)) return fail("null tensor pointer");
  if (!aligned(k, 16) || !aligned(v, 16)) return fail("kv8: the cache must be 16-byte aligned");
  if (!aligned(ks, 4) || !aligned(vs, 4) || !aligned(table, 4) || !aligned(lengths, 4) || !aligned(starts, 4) || !aligned(status, 4))
    return fail("kv8: scales, table, lengths, starts and status must be 4-byte aligned");
  c.k = static_cast<uint8_t*>(k);
  c.v = static_cast<uint8_t*>(v);
  c.ks = static_cast<float*>(ks);
  c.vs = static_cast<float*>(vs);
  c.table = static_cast<const int32_t*>(width > 0 ? table : lengths);
  c.lengths = static_cast<const int32_t*>(lengths);
  c.starts = static_cast<const int32_t*>(starts);
  c.status = static_cast<uint32_t*>(status);
  c.pages = pages;
  c.rows = rows;
  c.B = B;
  c.each = B > 0 ? static_cast<int32_t>(rows / B) : 0;
  c.width = width;
  c.Hkv = heads;
  c.D = dim;
  c.page = page;
  c.page_log2 = __builtin_ctz(static_cast<unsigned>(page));
  c.fp8 = cache_dtype == XRMM_E4M3;
  return XRMM_OK;
}

// Rows that one sequence may have: the caller's bound, or what the call holds.
int32_t most_rows(const xrmm::KvCache& c, int32_t max_new) {
  if (c.starts == nullptr) return c.each;
  const int32_t all = static_cast<int32_t>(c.rows);
  return max_new > 0 && max_new < all ? max_new : all;
}

}  // namespace

extern "C" {

int xrmm_mx4_quantize(const void* x, void* codes, void* scales, int64_t rows, int64_t K, int32_t dtype, void* stream) {
  xrmm::MxQuantArgs a{};
  a.dtype = type_of(dtype);
  if (a.dtype < 0) return fail("mx4_quantize: x must be float32, float16 or bfloat16");
  if (K <= 0 || K > kMaxK) return fail("mx4_quantize: K must be positive and at most 2^23");
  if (rows < 0 || rows > 0x7FFFFFFF) return fail("mx4_quantize: rows must be non-negative and below 2^31");
  if (rows > 0 && (!x || !codes || !scales)) return fail("null tensor pointer");
  if (!aligned(codes, 4) || !aligned(x, dtype == XRMM_F32 ? 4 : 2)) return fail("mx4_quantize: x and codes must be aligned");
  a.x = x;
  a.codes = static_cast<uint8_t*>(codes);
  a.scales = static_cast<uint8_t*>(scales);
  a.rows = rows;
  a.K = K;
  a.kb = (K + xrmm::MX_BLOCK - 1) / xrmm::MX_BLOCK;
  return done(xrmm::launch_mx4_quantize(a, static_cast<hipStream_t>(stream)), "mx4_quantize launch");
}

int64_t xrmm_matmul_mx4_workspace_bytes(int64_t M, int64_t K, int64_t N, int32_t a_dtype) {
  xrmm::MxArgs a;
  const int rc = mx4_geometry(a, M, K, N, a_dtype, XRMM_F32);
  set_status(XRMM_OK, "");
  return rc ? 0 : xrmm::mx4_workspace_bytes(M, K, N, a.a_type);
}

int xrmm_matmul_mx4(const void* A, const void* A_scales, int32_t a_dtype, const void* B, const void* scales,
                    const void* bias, void* Y, int32_t out_dtype, int64_t M, int64_t K, int64_t N, void* workspace,
                    int64_t workspace_bytes, void* stream) {
  xrmm::MxArgs a;
  if (int rc = mx4_geometry(a, M, K, N, a_dtype, out_dtype)) return rc;
  if ((a.a_type < 0) != (A_scales != nullptr) && M > 0) return fail("matmul_mx4: A_scales belong to MX4 codes, and only to them");
  if (M > 0 && (!A || !B || !scales || !Y)) return fail("null tensor pointer");
  if (!aligned(B, 16) || (a.a_type < 0 && !aligned(A, 16))) return fail("matmul_mx4: codes must be 16-byte aligned");
  const uintptr_t osz = out_dtype == XRMM_F32 ? 4 : 2;
  if (!aligned(A, 2) || !aligned(Y, osz) || !aligned(bias, osz)) return fail("matmul_mx4: A, bias and Y must be aligned to their elements");
  if (workspace != nullptr && !aligned(workspace, 256)) return fail("matmul_mx4: the workspace must be 256-byte aligned");
  a.A = A;
  a.As = static_cast<const uint8_t*>(A_scales);
  a.B = static_cast<const uint8_t*>(B);
  a.S = static_cast<const uint8_t*>(scales);
  a.bias = bias;
  a.Y = Y;
  a.ws = workspace;
  a.ws_bytes = workspace ? workspace_bytes : 0;
  return done(xrmm::launch_matmul_mx4(a, static_cast<hipStream_t>(stream)), "matmul_mx4 launch");
}

const char* xrmm_matmul_mx4_kernel(int64_t M, int64_t K, int64_t N, int32_t a_dtype) {
  xrmm::MxArgs a;
  if (mx4_geometry(a, M, K, N, a_dtype, XRMM_F32)) return nullptr;
  static const uint8_t probe[16] __attribute__((aligned(16))) = {};
  a.A = probe;
  set_status(XRMM_OK, "");
  return xrmm::mx4_kernel_name(a);
}

int xrmm_matmul_mx4_plan(int64_t M, int64_t K, int64_t N, int32_t a_dtype, int32_t have_workspace, int64_t* plan) {
  xrmm::MxArgs a;
  if (plan == nullptr) return fail("matmul_mx4_plan: null plan");
  if (int rc = mx4_geometry(a, M, K, N, a_dtype, XRMM_F32)) return rc;
  const xrmm::MxPlan p = xrmm::mx4_gemm_plan(M, K, N, a.a_type, have_workspace != 0);
  const int64_t v[6] = {64 * p.t, p.mt, p.nb, p.ns, p.splits, p.ws_bytes};
  for (int i = 0; i < 6; ++i) plan[i] = v[i];
  return set_status(XRMM_OK, "");
}

int xrmm_kv8_append(const void* k, const void* v, int64_t k_stride, int64_t v_stride, int32_t dtype, void* k_cache,
                    void* v_cache, void* k_scales, void* v_scales, int32_t cache_dtype, const void* block_table,
                    const void* lengths, const void* starts, void* status, int64_t rows, int32_t max_new, int32_t batch,
                    int32_t table_width, int64_t pages, int32_t page_size, int32_t kv_heads, int32_t head_dim, void* stream) {
  xrmm::KvAppendArgs a{};
  a.dtype = type_of(dtype);
  if (a.dtype < 0) return fail("kv8_append: k and v must be float32, float16 or bfloat16");
  if (int rc = cache_of(a.c, k_cache, v_cache, k_scales, v_scales, block_table, lengths, starts, status, pages, page_size,
                        kv_heads, head_dim, cache_dtype, batch, table_width, rows))
    return rc;
  if (rows > 0 && (!k || !v)) return fail("null tensor pointer");
  const int64_t row = static_cast<int64_t>(kv_heads) * head_dim;
  if (rows > 1 && (k_stride < row || v_stride < row)) return fail("kv8_append: token strides below kv_heads * head_dim");
  const uintptr_t sz = dtype == XRMM_F32 ? 4 : 2;
  if (!aligned(k, sz) || !aligned(v, sz)) return fail("kv8_append: k and v must be aligned to their elements");
  a.k = k;
  a.v = v;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.max_new = rows > 0 ? most_rows(a.c, max_new) : 0;
  return done(xrmm::launch_kv8_append(a, static_cast<hipStream_t>(stream)), "kv8_append launch");
}

namespace {

int attention_of(xrmm::KvAttnArgs& a, const void* q, int64_t q_stride, void* o, int32_t dtype, const void* k_cache,
                 const void* v_cache, const void* k_scales, const void* v_scales, int32_t cache_dtype,
                 const void* block_table, const void* lengths, const void* starts, void* status, int64_t rows,
                 int32_t max_new, int32_t batch, int32_t table_width, int64_t pages, int32_t page_size, int32_t q_heads,
                 int32_t kv_heads, int32_t head_dim, float scale, int32_t causal, int32_t window) {
  a = xrmm::KvAttnArgs{};
  a.dtype = type_of(dtype);
  if (a.dtype != xrmm::LT_F16 && a.dtype != xrmm::LT_BF16) return fail("kv8_attention: q must be float16 or bfloat16");
  if (int rc = cache_of(a.c, const_cast<void*>(k_cache), const_cast<void*>(v_cache), const_cast<void*>(k_scales),
                        const_cast<void*>(v_scales), block_table, lengths, starts, status, pages, page_size, kv_heads,
                        head_dim, cache_dtype, batch, table_width, rows))
    return rc;
  if (q_heads <= 0 || q_heads % kv_heads != 0) return fail("kv8_attention: query heads must be a multiple of the key heads");
  if (rows * q_heads > 0x7FFFFFFF) return fail("kv8_attention: 2^31 query rows or more");
  if (window < 0) return fail("kv8_attention: window must be non-negative");
  if (!std::isfinite(scale)) return fail("kv8_attention: scale must be finite");
  const int64_t row = static_cast<int64_t>(q_heads) * head_dim;
  if (rows > 1 && q_stride < row) return fail("kv8_attention: token stride below q_heads * head_dim");
  a.q = q;
  a.o = o;
  a.q_stride = q_stride;
  a.Hq = q_heads;
  a.max_new = rows > 0 ? most_rows(a.c, max_new) : 0;
  a.causal = causal != 0;
  a.window = window;
  a.scale = scale;
  return XRMM_OK;
}

}  // namespace

namespace {

// The arguments that decide a call's plan, with pointers that are never read.
int attention_geometry(xrmm::KvAttnArgs& a, int64_t rows, int32_t max_new, int32_t ragged, int32_t batch, int32_t table_width,
                       int32_t page_size, int32_t q_heads, int32_t kv_heads, int32_t head_dim, int32_t causal, int32_t window) {
  static const int32_t probe[4] __attribute__((aligned(16))) = {};
  return attention_of(a, probe, INT64_MAX, nullptr, XRMM_F16, probe, probe, probe, probe, XRMM_I8, probe, probe,
                      ragged ? probe : nullptr, nullptr, rows, max_new, batch, table_width, 1, page_size, q_heads, kv_heads,
                      head_dim, 1.f, causal, window);
}

}  // namespace

int64_t xrmm_kv8_attention_workspace_bytes(int64_t rows, int32_t max_new, int32_t ragged, int32_t batch, int32_t table_width,
                                           int32_t page_size, int32_t q_heads, int32_t kv_heads, int32_t head_dim,
                                           int32_t causal, int32_t window) {
  xrmm::KvAttnArgs a;
  const int rc = attention_geometry(a, rows, max_new, ragged, batch, table_width, page_size, q_heads, kv_heads, head_dim, causal, window);
  set_status(XRMM_OK, "");
  return rc ? 0 : xrmm::kv8_workspace_bytes(a);
}

const char* xrmm_kv8_attention_kernel(int64_t rows, int32_t max_new, int32_t ragged, int32_t batch, int32_t table_width,
                                      int32_t page_size, int32_t q_heads, int32_t kv_heads, int32_t head_dim, int32_t causal,
                                      int32_t window) {
  xrmm::KvAttnArgs a;
  if (attention_geometry(a, rows, max_new, ragged, batch, table_width, page_size, q_heads, kv_heads, head_dim, causal, window))
    return nullptr;
  set_status(XRMM_OK, "");
  return xrmm::kv8_kernel_name(a);
}

int xrmm_kv8_attention(const void* q, int64_t q_stride, void* output, int32_t dtype, const void* k_cache,
                       const void* v_cache, const void* k_scales, const void* v_scales, int32_t cache_dtype,
                       const void* block_table, const void* lengths, const void* starts, void* status, int64_t rows,
                       int32_t max_new, int32_t batch, int32_t table_width, int64_t pages, int32_t page_size,
                       int32_t q_heads, int32_t kv_heads, int32_t head_dim, float scale, int32_t causal, int32_t window,
                       void* workspace, int64_t workspace_bytes, void* stream) {
  xrmm::KvAttnArgs a;
  if (int rc = attention_of(a, q, q_stride, output, dtype, k_cache, v_cache, k_scales, v_scales, cache_dtype, block_table,
                            lengths, starts, status, rows, max_new, batch, table_width, pages, page_size, q_heads, kv_heads,
                            head_dim, scale, causal, window))
    return rc;
  if (rows > 0 && (!q || !output)) return fail("null tensor pointer");
  if (!aligned(q, 2) || !aligned(output, 2)) return fail("kv8_attention: q and the output must be aligned to their elements");
  if (workspace != nullptr && !aligned(workspace, 256)) return fail("kv8_attention: the workspace must be 256-byte aligned");
  a.ws = workspace;
  a.ws_bytes = workspace ? workspace_bytes : 0;
  return done(xrmm::launch_kv8_attention(a, static_cast<hipStream_t>(stream)), "kv8_attention launch");
}

namespace {

int shared_of(xrmm::KvAttnArgs& a, const void* shared_pages, int32_t shared_count) {
  if (shared_count < 0) return fail("kv8_shared_attention: negative count of shared pages");
  if (static_cast<int64_t>(shared_count) * a.c.page > 0x7FFFFF00) return fail("kv8_shared_attention: the shared pages span 2^31 tokens or more");
  if (shared_count > 0 && a.c.rows > 0 && !shared_pages) return fail("null tensor pointer");
  if (!aligned(shared_pages, 4)) return fail("kv8_shared_attention: the shared pages must be 4-byte aligned");
  a.shared = static_cast<const int32_t*>(shared_pages);
  a.shared_pages = shared_count;
  return XRMM_OK;
}

}  // namespace

int64_t xrmm_kv8_shared_attention_workspace_bytes(int64_t rows, int32_t max_new, int32_t ragged, int32_t batch, int32_t shared_count,
                                                  int32_t table_width, int32_t page_size, int32_t q_heads, int32_t kv_heads,
                                                  int32_t head_dim, int32_t causal, int32_t window) {
  static const int32_t probe[1] = {};
  xrmm::KvAttnArgs a;
  int rc = attention_geometry(a, rows, max_new, ragged, batch, table_width, page_size, q_heads, kv_heads, head_dim, causal, window);
  if (!rc) rc = shared_of(a, probe, shared_count);
  set_status(XRMM_OK, "");
  return rc ? 0 : xrmm::kv8_shared_workspace_bytes(a);
}

const char* xrmm_kv8_shared_attention_kernel(int64_t rows, int32_t max_new, int32_t ragged, int32_t batch, int32_t shared_count,
                                             int32_t table_width, int32_t page_size, int32_t q_heads, int32_t kv_heads,
                                             int32_t head_dim, int32_t causal, int32_t window) {
  static const int32_t probe[1] = {};
  xrmm::KvAttnArgs a;
  if (attention_geometry(a, rows, max_new, ragged, batch, table_width, page_size, q_heads, kv_heads, head_dim, causal, window) ||
      shared_of(a, probe, shared_count))
    return nullptr;
  set_status(XRMM_OK, "");
  return xrmm::kv8_shared_kernel_name(a);
}

int xrmm_kv8_shared_attention(const void* q, int64_t q_stride, void* output, int32_t dtype, const void* k_cache,
                              const void* v_cache, const void* k_scales, const void* v_scales, int32_t cache_dtype,
                              const void* shared_pages, int32_t shared_count, const void* block_table, const void* lengths,
                              const void* starts, void* status, int64_t rows, int32_t max_new, int32_t batch,
                              int32_t table_width, int64_t pages, int32_t page_size, int32_t q_heads, int32_t kv_heads,
                              int32_t head_dim, float scale, int32_t causal, int32_t window, void* workspace,
                              int64_t workspace_bytes, void* stream) {
  xrmm::KvAttnArgs a;
  // a table of no columns, where all positions are shared ones, may have no address
  if (int rc = attention_of(a, q, q_stride, output, dtype, k_cache, v_cache, k_scales, v_scales, cache_dtype,
                            table_width == 0 ? lengths : block_table, lengths, starts, status, rows, max_new, batch, table_width,
                            pages, page_size, q_heads, kv_heads, head_dim, scale, causal, window))
    return rc;
  if (int rc = shared_of(a, shared_pages, shared_count)) return rc;
  if (rows > 0 && (!q || !output)) return fail("null tensor pointer");
  if (!aligned(q, 2) || !aligned(output, 2)) return fail("kv8_shared_attention: q and the output must be aligned to their elements");
  if (workspace != nullptr && !aligned(workspace, 256)) return fail("kv8_shared_attention: the workspace must be 256-byte aligned");
  a.ws = workspace;
  a.ws_bytes = workspace ? workspace_bytes : 0;
  return done(xrmm::launch_kv8_shared_attention(a, static_cast<hipStream_t>(stream)), "kv8_shared_attention launch");
}

}  // extern "C"
