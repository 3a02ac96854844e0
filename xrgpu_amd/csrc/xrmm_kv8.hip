// The 8-bit paged cache: appending tokens, and the launches of attention over it.
#include "xrmm_kv8_attn.h"

namespace xrmm {

namespace {

// ---------------------------------------------------------------------------
// Append. A workgroup owns one page and head of K or V: it takes the largest magnitude of
// the tokens that enter the page, settles the page's scale, rounds the codes already there to
// it if it grew, and writes the new codes. No two workgroups touch one page and head.
//
// e(r) is the smallest integer with r <= qmax 2^e (at least -126; qmax 127 for int8, 448 for
// e4m3). A page whose first slot is among the new tokens, or whose scale is 0, gets the scale
// 2^e(max); another's scale is multiplied by 2^max(0, e(max / scale)). Scales that only grow by
// powers of two keep what is held within one step however often they grow (each growth at
// least halves the share of the roundings before it), and division by a power of two is exact.

template <bool FP8>
__device__ __forceinline__ int kv_exponent(float r) {  // finite r > 0
  constexpr float qmax = FP8 ? 448.f : 127.f;
  int e = static_cast<int>((__builtin_bit_cast(uint32_t, r) >> 23) & 255u) - 127 - (FP8 ? 8 : 6);
  e = e < -126 ? -126 : e;
  return r > qmax * __builtin_bit_cast(float, static_cast<uint32_t>(e + 127) << 23) ? e + 1 : e;
}

// Four values in [-qmax, qmax] -> four codes, to nearest, ties to even.
template <bool FP8>
__device__ __forceinline__ uint32_t kv_code4(float a, float b, float c, float d) {
  if constexpr (FP8) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true));
  } else {
    auto i = [](float x) { return static_cast<uint32_t>(static_cast<int>(__builtin_rintf(x))) & 255u; };
    return i(a) | (i(b) << 8) | (i(c) << 16) | (i(d) << 24);
  }
}

template <bool FP8>
__device__ __forceinline__ void kv_value4(uint32_t x, float (&v)[4]) {
  if constexpr (FP8) {
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(x), false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(x), true);
    v[0] = lo[0]; v[1] = lo[1]; v[2] = hi[0]; v[3] = hi[1];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = static_cast<float>(static_cast<int8_t>(x >> (8 * i)));
  }
}

constexpr int KVA_T = 256;
constexpr int KVA_H = 4;  // pieces of eight values that a thread keeps between the magnitudes and the codes (64 slots of 128 values)

// The tokens' addresses need neither page nor scale, so their loads leave before those are looked up, and a page of
// up to 8192 values is read once: 4100 tokens of 8 heads of 128 (bfloat16, e4m3) in 8.0 us, 14.0 with loads of
// four values, read twice, and a division for each. What is left is the chain lengths -> page -> scale -> codes of a
// workgroup that runs once.
template <typename T, bool FP8>
__global__ __launch_bounds__(KVA_T) void k_kv8_append(KvAppendArgs a, uint32_t touched) {
  constexpr float qmax = FP8 ? 448.f : 127.f;
  typedef T vec __attribute__((ext_vector_type(8), aligned(16)));
  typedef typename std::conditional<sizeof(T) == 2, uint16_t, uint32_t>::type U;
  typedef U uvec __attribute__((ext_vector_type(8)));
  const KvCache& c = a.c;
  const int tid = threadIdx.x;
  const bool isv = (blockIdx.x & 1u) != 0;
  uint32_t r = blockIdx.x >> 1;
  const int h = static_cast<int>(r % static_cast<uint32_t>(c.Hkv));
  r /= static_cast<uint32_t>(c.Hkv);
  const int b = static_cast<int>(r / touched), i = static_cast<int>(r % touched);
  int first, count;
  const bool rows = kv_rows(c, b, a.max_new, first, count);
  if (!rows && tid == 0 && c.status != nullptr) atomicMax(c.status, KV_BAD);
  const int64_t len = c.lengths[b], begin = len - count;  // positions begin .. len - 1 enter the cache
  if (count <= 0) return;
  const int64_t base = ((begin >> c.page_log2) + i) * c.page;  // first position of the page
  if (base >= len) return;
  const int from = begin > base ? static_cast<int>(begin - base) : 0;              // slots from .. to - 1 are new
  const int to = len - base < c.page ? static_cast<int>(len - base) : c.page;
  const int64_t stride = isv ? a.v_stride : a.k_stride;
  const T* x = static_cast<const T*>(isv ? a.v : a.k) + (first + base + from - begin) * stride + static_cast<int64_t>(h) * c.D;
  const bool whole = (reinterpret_cast<uintptr_t>(x) | static_cast<uintptr_t>(stride * sizeof(T))) % 16 == 0;
  const uint32_t pieces = static_cast<uint32_t>(c.D) >> 3, all = static_cast<uint32_t>(to - from) * pieces;
  const uint32_t inverse = (1u << 20) / pieces + 1u;  // p * inverse >> 20 = p / pieces for p < 2^20 / pieces (p < 2^13 here)
  auto piece = [&](uint32_t p) {
    const uint32_t row = (p * inverse) >> 20;
    return x + row * stride + (p - row * pieces) * 8u;
  };
  auto load = [&](uint32_t p) {
    const T* s = piece(p);
    vec v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = s[e];
    return v;
  };
  const uint32_t kept = !whole ? 0u : all < KVA_H * KVA_T ? all : KVA_H * KVA_T;  // pieces that registers hold
  vec held[KVA_H];
  // All pieces that the thread keeps; the code past the first stands apart, as single tokens do not reach it.
  auto each_held = [&](auto&& f) {
    if (tid < kept) f(0);
    if (__builtin_expect(kept > KVA_T, 0)) {
#pragma unroll
      for (int j = 1; j < KVA_H; ++j)
        if (tid + j * KVA_T < kept) f(j);
    }
  };
  each_held([&](int j) { held[j] = *reinterpret_cast<const vec*>(piece(tid + j * KVA_T)); });

  const int32_t page = base < 0 || base > 0x7FFFFFFF ? -1 : kv_page(c, b, static_cast<uint32_t>(base));
  if (page < 0) {
    if (tid == 0 && c.status != nullptr) atomicMax(c.status, KV_BAD);
    return;
  }
  const int64_t slot0 = (static_cast<int64_t>(page) * c.Hkv + h) * c.page;
  uint8_t* codes = (isv ? c.v : c.k) + slot0 * c.D;
  float* scale = (isv ? c.vs : c.ks) + static_cast<int64_t>(page) * c.Hkv + h;
  const float old = from == 0 ? 0.f : *scale;

  uvec tops8 = 0;  // the largest magnitudes' bits (above every finite one's for infinity and NaN), in x's own type
  auto raise = [&](const vec& v) { tops8 = __builtin_elementwise_max(tops8, __builtin_bit_cast(uvec, v) & static_cast<U>(static_cast<U>(~U(0)) >> 1)); };
  each_held([&](int j) { raise(held[j]); });
#pragma unroll 1
  for (uint32_t p = tid + kept; p < all; p += KVA_T) raise(load(p));
  U topu = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) topu = topu > tops8[e] ? topu : tops8[e];
  uint32_t top = __builtin_bit_cast(uint32_t, static_cast<float>(__builtin_bit_cast(T, topu)));
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint32_t m = static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), o, 64));
    top = top > m ? top : m;
  }
  __shared__ uint32_t tops[KVA_T / 64];
  if ((tid & 63) == 0) tops[tid >> 6] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < KVA_T / 64; ++w) top = top > tops[w] ? top : tops[w];

  const float amax = __builtin_bit_cast(float, top);
  const bool fresh = !(old != 0.f);
  int grow = 0;  // the held codes are divided by 2^grow
  float now;
  if (top >= 0x7F800000u) now = __builtin_nanf("");
  else if (fresh) now = top == 0u ? 0.f : two(kv_exponent<FP8>(amax));
  else if (!(old > 0.f) || old > 3.4028235e38f) now = old;  // a scale that is no scale stays
  else {
    const float ratio = amax / old;
    // a quotient past float32: the same one 2^160 smaller
    if (top != 0u) grow = ratio <= 3.4028235e38f ? kv_exponent<FP8>(ratio) : kv_exponent<FP8>(amax * two(-100) / (old * two(60))) + 160;
    grow = grow < 0 ? 0 : grow;
    now = ldexpf(old, grow);
  }
  if (grow > 0 && !fresh) {
    const float shrink = grow > 126 ? 0.f : two(-grow);
#pragma unroll 1
    for (uint32_t p = tid; p < static_cast<uint32_t>(from) * pieces / 2u; p += KVA_T) {
      u32x4* w = reinterpret_cast<u32x4*>(codes) + p;
      u32x4 y = *w;
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        float v[4];
        kv_value4<FP8>(y[d], v);
        y[d] = kv_code4<FP8>(v[0] * shrink, v[1] * shrink, v[2] * shrink, v[3] * shrink);
      }
      *w = y;
    }
  }
  const bool good = now > 0.f && now <= 3.4028235e38f;
  const uint32_t bits = __builtin_bit_cast(uint32_t, now);
  const bool power = (bits & 0x7FFFFFu) == 0u && bits >= 0x00800000u && bits <= 0x7E800000u;  // 2^-126 .. 2^126: so is its inverse
  auto store = [&](uint32_t p, const vec& v, auto&& scaled) {
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = fminf(fmaxf(scaled(static_cast<float>(v[e])), -qmax), qmax);
    u32x2 o;
    o[0] = kv_code4<FP8>(f[0], f[1], f[2], f[3]);
    o[1] = kv_code4<FP8>(f[4], f[5], f[6], f[7]);
    reinterpret_cast<u32x2*>(codes)[static_cast<uint32_t>(from) * pieces + p] = o;
  };
  if (power) {
    const float by = __builtin_bit_cast(float, 0x7F000000u - bits);
    auto times = [&](float f) { return f * by; };  // exact, as the division is
    each_held([&](int j) { store(tid + j * KVA_T, held[j], times); });
#pragma unroll 1
    for (uint32_t p = tid + kept; p < all; p += KVA_T) store(p, load(p), times);
  } else {  // another quantiser's scale, or none: short code rather than quick
#pragma unroll 1
    for (uint32_t p = tid; p < all; p += KVA_T) store(p, load(p), [&](float f) { return good ? f / now : 0.f; });
  }
  if (tid == 0) *scale = now;
}

}  // namespace

int64_t kv8_workspace_bytes(const KvAttnArgs& a) {
  return a.c.B == 0 || a.max_new == 0 ? 0 : attention_plan(a, true).ws_bytes;
}

const char* kv8_kernel_name(const KvAttnArgs& a) {
  return a.c.B > 0 && a.max_new > 0 && attention_plan(a, true).tile ? "kv8_tile" : "kv8_rows";
}

hipError_t launch_kv8_attention(const KvAttnArgs& a, hipStream_t st) {
  if (a.c.B == 0 || a.max_new == 0) return hipSuccess;
  KvPlan p = attention_plan(a, a.ws != nullptr);
  if (p.ws_bytes > a.ws_bytes) p = attention_plan(a, false);
  return attention_with<KV_PLAIN>(a, p, st);
}

hipError_t launch_kv8_append(const KvAppendArgs& a, hipStream_t st) {
  if (a.c.B == 0 || a.max_new == 0) return hipSuccess;
  // pages that a sequence's new tokens can lie in
  const int64_t touched = (a.max_new + a.c.page - 2) / a.c.page + 1;
  const int64_t grid = touched * a.c.B * a.c.Hkv * 2;
  if (!grid_counts(grid, KVA_T)) return hipErrorInvalidValue;
  const dim3 g(static_cast<uint32_t>(grid));
  const uint32_t t = static_cast<uint32_t>(touched);
  if (a.c.fp8) {
    if (a.dtype == LT_F32) k_kv8_append<float, true><<<g, KVA_T, 0, st>>>(a, t);
    else if (a.dtype == LT_F16) k_kv8_append<f16, true><<<g, KVA_T, 0, st>>>(a, t);
    else k_kv8_append<bf16, true><<<g, KVA_T, 0, st>>>(a, t);
  } else {
    if (a.dtype == LT_F32) k_kv8_append<float, false><<<g, KVA_T, 0, st>>>(a, t);
    else if (a.dtype == LT_F16) k_kv8_append<f16, false><<<g, KVA_T, 0, st>>>(a, t);
    else k_kv8_append<bf16, false><<<g, KVA_T, 0, st>>>(a, t);
  }
  return hipGetLastError();
}

}  // namespace xrmm
