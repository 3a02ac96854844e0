// C ABI of rotary positions and of the draw of tokens: argument checks and dispatch.
#include <hip/hip_runtime.h>

#include <cmath>
#include <string>

#include "../../include/xrmm.h"
#include "xrmm_decode.h"

namespace {

using xrmm::set_status;

int fail(const char* msg) { return set_status(XRMM_EINVAL, msg); }

int done(hipError_t e, const char* what) {
  return e == hipSuccess ? set_status(XRMM_OK, "") : set_status(XRMM_EDEVICE, std::string(what) + ": " + hipGetErrorString(e));
}

int type_of(int32_t d) {
  return d == XRMM_F32 ? xrmm::LT_F32 : d == XRMM_F16 ? xrmm::LT_F16 : d == XRMM_BF16 ? xrmm::LT_BF16 : -1;
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// Rows of `width` bytes, `stride` bytes apart.
struct Rows {
  const void* p;
  int64_t stride, width;
};

// Whether no byte of one set of n rows is in the other, as far as equal strides or whole ranges show it.
bool apart(const Rows& a, const Rows& b, int64_t n) {
  if (a.width == 0 || b.width == 0 || n == 0) return true;
  const int64_t x = static_cast<int64_t>(reinterpret_cast<uintptr_t>(a.p)), y = static_cast<int64_t>(reinterpret_cast<uintptr_t>(b.p));
  if (x + (n - 1) * a.stride + a.width <= y || y + (n - 1) * b.stride + b.width <= x) return true;
  if (n > 1 && a.stride != b.stride) return false;
  if (n == 1) return false;  // their ranges meet
  const int64_t off = ((y - x) % a.stride + a.stride) % a.stride;  // where b's rows begin within a's
  return off >= a.width && off + b.width <= a.stride;
}

bool same(const Rows& a, const Rows& b, int64_t n) { return a.p == b.p && (n < 2 || a.stride == b.stride); }

constexpr int32_t kMaxVocab = 1 << 24;

int sample_geometry(xrmm::SampleArgs& a, int64_t rows, int64_t vocab, int32_t dtype) {
  a = xrmm::SampleArgs{};
  a.dtype = type_of(dtype);
  if (a.dtype < 0) return fail("sample: logits must be float32, float16 or bfloat16");
  if (rows < 0 || rows > 0x7FFFFFFF) return fail("sample: rows must be non-negative and below 2^31");
  if (vocab <= 0 || vocab > kMaxVocab) return fail("sample: a row must have 1 to 2^24 logits");
  a.rows = rows;
  a.V = static_cast<int32_t>(vocab);
  return XRMM_OK;
}

}  // namespace

extern "C" {

int xrmm_rope(const void* q, const void* k, void* q_out, void* k_out, int64_t q_stride, int64_t k_stride, int64_t q_out_stride,
              int64_t k_out_stride, int32_t dtype, const void* frequencies, int32_t rotary_dim, double magnitude,
              const void* positions, int32_t positions_dtype, const void* lengths, const void* starts, int64_t rows, int32_t batch,
              int32_t q_heads, int32_t k_heads, int32_t head_dim, int32_t interleaved, int32_t inverse, void* stream) {
  xrmm::RopeArgs a{};
  a.dtype = type_of(dtype);
  if (a.dtype < 0) return fail("rope: q and k must be float32, float16 or bfloat16");
  if (rows < 0 || rows > 0x7FFFFFFF) return fail("rope: rows must be non-negative and below 2^31");
  if (head_dim <= 0 || head_dim > 1024) return fail("rope: the head size must be 1 to 1024");
  if (rotary_dim <= 0 || rotary_dim % 2 != 0 || rotary_dim > head_dim) return fail("rope: the turned part must be even, positive and no more than the head");
  if (q_heads < 0 || k_heads < 0 || q_heads > (1 << 20) || k_heads > (1 << 20)) return fail("rope: heads must be non-negative and at most 2^20");
  if (!std::isfinite(magnitude)) return fail("rope: magnitude must be finite");
  if ((positions != nullptr) == (lengths != nullptr) && rows > 0) return fail("rope: give either positions or lengths");
  if (positions != nullptr && positions_dtype != XRMM_I32 && positions_dtype != XRMM_I64) return fail("rope: positions must be int32 or int64");
  if (positions != nullptr && starts != nullptr) return fail("rope: starts belong to lengths");
  if (batch < 0) return fail("rope: negative batch");
  if (lengths != nullptr && batch == 0 && rows != 0) return fail("rope: rows without sequences");
  if (lengths != nullptr && starts == nullptr && batch > 0 && rows % batch != 0) return fail("rope: rows of unequal counts need starts");
  const int64_t size = dtype == XRMM_F32 ? 4 : 2, qw = static_cast<int64_t>(q_heads) * head_dim, kw = static_cast<int64_t>(k_heads) * head_dim;
  if (rows > 1 && ((q_heads > 0 && (q_stride < qw || q_out_stride < qw)) || (k_heads > 0 && (k_stride < kw || k_out_stride < kw))))
    return fail("rope: token strides below heads * head_dim");
  if (rows <= 1 || q_heads == 0) q_stride = q_out_stride = qw;  // of no use
  if (rows <= 1 || k_heads == 0) k_stride = k_out_stride = kw;
  for (const int64_t stride : {q_stride, k_stride, q_out_stride, k_out_stride})
    if (rows > 1 && stride > INT64_MAX / 8 / rows) return fail("rope: token strides past any memory");  // ranges stay below 2^63 bytes
  if (rows > 0 && ((q_heads > 0 && (!q || !q_out)) || (k_heads > 0 && (!k || !k_out)) || !frequencies)) return fail("null tensor pointer");
  if (!aligned(q, size) || !aligned(k, size) || !aligned(q_out, size) || !aligned(k_out, size)) return fail("rope: tensors must be aligned to their elements");
  if (!aligned(frequencies, 8) || !aligned(positions, positions_dtype == XRMM_I64 ? 8 : 4) || !aligned(lengths, 4) || !aligned(starts, 4))
    return fail("rope: frequencies, positions, lengths and starts must be aligned to their elements");
  const Rows rq{q, q_stride * size, qw * size}, rk{k, k_stride * size, kw * size}, oq{q_out, q_out_stride * size, qw * size},
      ok{k_out, k_out_stride * size, kw * size};
  if (!(same(rq, oq, rows) || apart(rq, oq, rows)) || !(same(rk, ok, rows) || apart(rk, ok, rows)) || !apart(rq, ok, rows) ||
      !apart(rk, oq, rows) || !apart(oq, ok, rows))
    return fail("rope: an output may be its input's own memory, and else must not overlap inputs or the other output");
  a.q = q_heads > 0 ? q : nullptr;
  a.k = k_heads > 0 ? k : nullptr;
  a.oq = q_heads > 0 ? q_out : nullptr;
  a.ok = k_heads > 0 ? k_out : nullptr;
  a.q_stride = q_stride;
  a.k_stride = k_stride;
  a.oq_stride = q_out_stride;
  a.ok_stride = k_out_stride;
  a.freq = static_cast<const double*>(frequencies);
  a.positions = positions;
  a.wide_positions = positions_dtype == XRMM_I64;
  a.lengths = static_cast<const int32_t*>(lengths);
  a.starts = static_cast<const int32_t*>(starts);
  a.magnitude = magnitude;
  a.rows = rows;
  a.B = batch;
  a.each = batch > 0 ? static_cast<int32_t>(rows / batch) : 0;
  a.Hq = q_heads;
  a.Hk = k_heads;
  a.D = head_dim;
  a.R = rotary_dim;
  a.interleaved = interleaved != 0;
  a.inverse = inverse != 0;
  return done(xrmm::launch_rope(a, static_cast<hipStream_t>(stream)), "rope launch");
}

int64_t xrmm_sample_workspace_bytes(int64_t rows, int64_t vocab) {
  xrmm::SampleArgs a;
  const int rc = sample_geometry(a, rows, vocab, XRMM_F32);
  set_status(XRMM_OK, "");
  return rc ? 0 : xrmm::sample_workspace_bytes(rows, vocab);
}

int xrmm_sample(const void* logits, int64_t stride, int32_t dtype, const void* uniforms, const void* temperatures,
                const void* top_ks, const void* top_ps, const void* min_ps, double temperature, int32_t top_k, double top_p,
                double min_p, void* tokens, void* shares, int64_t rows, int64_t vocab, void* workspace, int64_t workspace_bytes,
                void* stream) {
  xrmm::SampleArgs a;
  if (int rc = sample_geometry(a, rows, vocab, dtype)) return rc;
  if (rows > 1 && stride < vocab) return fail("sample: row stride below the number of logits");
  if (!temperatures && !(temperature >= 0.0)) return fail("sample: temperature must be non-negative");
  if (!top_ks && top_k < 0) return fail("sample: top_k must be non-negative");
  if (!top_ps && !(top_p >= 0.0)) return fail("sample: top_p must be non-negative");
  if (!min_ps && !(min_p >= 0.0 && min_p <= 1.0)) return fail("sample: min_p must be from 0 to 1");
  if (rows > 0 && (!logits || !uniforms || !tokens || !shares)) return fail("null tensor pointer");
  if (!aligned(logits, dtype == XRMM_F32 ? 4 : 2)) return fail("sample: logits must be aligned to their elements");
  for (const void* p : {uniforms, temperatures, top_ks, top_ps, min_ps, static_cast<const void*>(tokens), static_cast<const void*>(shares)})
    if (!aligned(p, 4)) return fail("sample: the rows' numbers, settings and results must be 4-byte aligned");
  if (workspace != nullptr && !aligned(workspace, 256)) return fail("sample: the workspace must be 256-byte aligned");
  a.x = logits;
  a.stride = stride;
  a.u = static_cast<const float*>(uniforms);
  a.temperature = static_cast<const float*>(temperatures);
  a.top_k = static_cast<const int32_t*>(top_ks);
  a.top_p = static_cast<const float*>(top_ps);
  a.min_p = static_cast<const float*>(min_ps);
  a.temperature1 = temperature;
  a.top_k1 = top_k;
  a.top_p1 = top_p;
  a.min_p1 = min_p;
  a.tokens = static_cast<int32_t*>(tokens);
  a.shares = static_cast<float*>(shares);
  a.ws = workspace;
  a.ws_bytes = workspace ? workspace_bytes : 0;
  return done(xrmm::launch_sample(a, static_cast<hipStream_t>(stream)), "sample launch");
}

}  // extern "C"
