// The 8-bit paged cache: appending tokens, and attention over it.
#include <atomic>
#include <type_traits>

#include "xrmm_lowbit.h"

namespace xrmm {

int device_cus();

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

__device__ __forceinline__ float two(int e) { return __builtin_bit_cast(float, static_cast<uint32_t>(e + 127) << 23); }

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

// ---------------------------------------------------------------------------
// Attention. Everything is computed transposed, so that no value changes lanes in the loop:
//
//   S^T = K Q^T   first operand K: lane (c, g) = (lane % 16, lane / 16) holds token c of 16 and the D / 4
//                 codes from g D / 4 on; second operand Q: the same d of row c
//   O^T = V^T P^T second operand P: S^T leaves lane (c, g) tokens 4 g .. + 3 of row c, which for two
//                 16-token tiles is the operand as it stands; first operand V^T: lane (c, g) holds the
//                 D / 16 codes from c D / 16 on of those eight tokens
//
// (the order of the summed index is free as long as both operands agree). A row's maximum, sum and
// rescaling factor belong to column c throughout. The codes are exact in binary16; a page's key scale
// multiplies its scores and its value scale its weights. Rows are the queries of one sequence that
// read one key head: row r is query r / G, head r % G of the group.

constexpr int KVT = 32;      // tokens of a step

// A token's softmax weight times its page's value scale enters binary16 as p vs 2^(KV_PE - e), where 2^e is a power of two
// above every value scale that the row has seen so far in magnitude: 2^KV_PE at most, so that small weights stay normal. A page
// that a row's mask hides does not count for it, so what the row cannot see does not change it. Only
// exponents are compared and shifted, so scales may be negative, and as small or as large as a float32 is. Binary16 is what
// the codes are exact in. Where a key head's rows of a sequence are one tile of 16, as in calls of single tokens, a weight is the sum of two
// binary16 terms (22 bits): the cache's bytes bound these calls, and the second term costs them 0 to 2 % (48 sequences of up to 8000 95.2 -> 96.4 us).
// Elsewhere instructions do, and a second term would cost 5 to 6 % by rows (32 tokens on 30000 71.6 -> 76.3) and 23 % by tiles (two chunks of
// 2000 on 4000 272 -> 335): a weight keeps eleven bits, which raises the error of float16 outputs against 64 bits from 2.1e-4 with
// float32 weights to 2.6e-4 (3.1e-4 in windows of few tokens), of bfloat16 ones not at all. The denominator sums the weights before they are rounded.
constexpr int KV_PE = 11;
constexpr int KV_NONE = -1000;  // e before any scale

// The smallest e with |scale| < 2^e; KV_NONE for 0 and for what is not finite.
__device__ __forceinline__ int kv_scale_exp(float scale) {
  const uint32_t m = __builtin_bit_cast(uint32_t, scale) & 0x7FFFFFFFu;
  return m - 1u < 0x7F7FFFFFu ? __builtin_amdgcn_frexp_expf(scale) : KV_NONE;
}

__device__ __forceinline__ float kv_shift(float x, int e) { return __builtin_ldexpf(x, e); }

// Four codes -> four binary16 values, exact.
template <bool FP8>
__device__ __forceinline__ f16x4 kv_half4(uint32_t x) {
  if constexpr (FP8) {
    const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.f, true);
    return f16x4{a[0], a[1], b[0], b[1]};
  } else {
    // bytes + 128 in the low bits of 1024.0, minus 1152
    const uint32_t y = x ^ 0x80808080u;
    const f16x2 off = {static_cast<f16>(-1152.f), static_cast<f16>(-1152.f)};
    const f16x2 a = as_h2(__builtin_amdgcn_perm(0x64646464u, y, 0x04010400u)) + off;
    const f16x2 b = as_h2(__builtin_amdgcn_perm(0x64646464u, y, 0x04030402u)) + off;
    return f16x4{a[0], a[1], b[0], b[1]};
  }
}

__device__ __forceinline__ f16x8 cat8(f16x4 a, f16x4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }

// Bytes [from, from + N) of a token's codes, N a multiple of two, in words.
template <int N>
struct KvBytes {
  uint32_t w[(N + 3) / 4];
};

template <int N>
__device__ __forceinline__ KvBytes<N> kv_bytes(const uint8_t* p) {
  KvBytes<N> r;
  if constexpr (N % 16 == 0) {
#pragma unroll
    for (int i = 0; i < N / 16; ++i) {
      const u32x4 x = ld16(p + 16 * i);
      r.w[4 * i] = x[0]; r.w[4 * i + 1] = x[1]; r.w[4 * i + 2] = x[2]; r.w[4 * i + 3] = x[3];
    }
  } else if constexpr (N % 8 == 0) {
#pragma unroll
    for (int i = 0; i < N / 8; ++i) {
      const u32x2 x = *reinterpret_cast<const u32x2*>(p + 8 * i);
      r.w[2 * i] = x[0]; r.w[2 * i + 1] = x[1];
    }
  } else if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) r.w[i] = *reinterpret_cast<const uint32_t*>(p + 4 * i);
  } else {  // 6
    static_assert(N == 6);
    const uint32_t a = *reinterpret_cast<const uint16_t*>(p), b = *reinterpret_cast<const uint16_t*>(p + 2);
    r.w[0] = a | (b << 16);
    r.w[1] = *reinterpret_cast<const uint16_t*>(p + 4);
  }
  return r;
}

// Few rows: the cache's bytes bound the call. A workgroup takes 16 rows of one sequence and key head and `chunk`
// tokens; its waves take turns at steps of 32 tokens, with the next step's codes in flight and the
// page after that looked up. Workgroups of one (sequence, head, rows) leave their
// unnormalised outputs, maxima and sums in the workspace, and the last to arrive joins them in
// token order. 48 sequences of up to 8000 tokens, 8 heads of 128, e4m3: 96 us (5.2 TB/s), unsplit; one of 65000, int8: 35 us, of
// which the join is about 8. The kernel's start shows in short calls: with queries loaded value by value a token on 4 took 9.5 us
// at head size 256 and 5.4 at 64, in pieces of 16 bytes (outputs of 8) 8.3 and 4.8.
constexpr int KVR_PASS = 8 * KVT;  // shares of tokens are multiples of it: a step of all waves, eight at most
constexpr int64_t KV_COUNTERS = 4096;      // bytes of arrival counters at the head of the workspace

template <int D>
constexpr int64_t kv_part_bytes() { return 16 * (D + 2) * 4; }  // [16][D] outputs, [16] (maximum, sum)

template <int D>
struct KvStep {
  int32_t pg[2];  // the two 16-token tiles lie in one page each
  float ks[2], vs[2];
  KvBytes<D / 4> k[2];
  KvBytes<D / 16> v[8];
};

template <int D, bool FP8, int W, bool TWO>
__global__ __launch_bounds__(64 * W, D > 128 || W == 8 ? 2 : 3) void k_kv8_rows(KvAttnArgs a, uint32_t row_tiles, uint32_t splits, uint32_t chunk) {
  constexpr int KD = D / 4, VD = D / 16;  // codes of a token that a lane holds
  const KvCache& c = a.c;
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t split = blockIdx.x % splits, unit = blockIdx.x / splits;
  const int tile = static_cast<int>(unit % row_tiles);
  const uint32_t bh = unit / row_tiles;
  const int h = static_cast<int>(bh % static_cast<uint32_t>(c.Hkv)), b = static_cast<int>(bh / static_cast<uint32_t>(c.Hkv));
  const int G = a.Hq / c.Hkv;
  int first, count;
  if (!kv_rows(c, b, a.max_new, first, count) && tid == 0 && c.status != nullptr) atomicMax(c.status, KV_BAD);
  const int nrows = count * G, r0 = tile * 16;
  if (r0 >= nrows) return;
  // positions past the table are left out: the walk over tokens ends with the table
  const int span = c.width << c.page_log2, all = c.lengths[b] > 0 ? c.lengths[b] : 0, past = all - count;
  const int len = all < span ? all : span;
  if (all > span && tid == 0 && c.status != nullptr) atomicMax(c.status, KV_BAD);

  // the tokens that any of the rows sees, and those that all of them see
  const int last = r0 + 16 < nrows ? r0 + 15 : nrows - 1, i0 = r0 / G, i1 = last / G;
  auto row_hi = [&](int i) { return a.causal && past + i + 1 < len ? past + i + 1 : len; };
  auto row_lo = [&](int i) { return a.window > 0 && past + i + 1 > a.window ? past + i + 1 - a.window : 0; };  // no difference below -2^31
  const int hi_all = row_hi(i1), lo_all = (row_lo(i0) < hi_all ? row_lo(i0) : hi_all) / KVT * KVT, full_lo = row_lo(i1), full_hi = row_hi(i0);
  const uint32_t parts = hi_all > lo_all ? (static_cast<uint32_t>(hi_all - lo_all) + chunk - 1) / chunk : 1u;  // at most `splits`
  if (split >= parts) return;
  const int tlo = lo_all + static_cast<int>(split * chunk);
  const int thi = splits > 1 && split + 1 < parts ? tlo + static_cast<int>(chunk) : hi_all;

  // the first token that a row sees: pages wholly before it may be gone (no branch around the lookup: it would be waited for)
  const int seen = row_lo(i0);
  auto find = [&](uint32_t t0, int32_t (&pg)[2]) {
#pragma unroll
    for (uint32_t u = 0; u < 2; ++u) {
      const uint32_t t = t0 + 16 * u;
      const int32_t p = kv_page(c, b, t);
      pg[u] = ((t < static_cast<uint32_t>(thi)) & (t + 16 > static_cast<uint32_t>(seen))) ? p : -2;
    }
  };
  auto load = [&](KvStep<D>& s, const int32_t (&pg)[2], uint32_t t0) {
#pragma unroll
    for (uint32_t u = 0; u < 2; ++u) {
      const uint32_t t = t0 + 16 * u;
      s.pg[u] = pg[u];
      const int64_t at = static_cast<int64_t>(pg[u] < 0 ? 0 : pg[u]) * c.Hkv + h;
      s.ks[u] = c.ks[at];
      s.vs[u] = c.vs[at];
      const int64_t slot = (at * c.page + (t & static_cast<uint32_t>(c.page - 1))) * D;
      s.k[u] = kv_bytes<KD>(c.k + slot + col * D + g * KD);
#pragma unroll
      for (int x = 0; x < 4; ++x) s.v[4 * u + x] = kv_bytes<VD>(c.v + slot + (4 * g + x) * D + col * VD);
    }
  };
  int32_t pg[2];
  KvStep<D> cur;
  const uint32_t tw = static_cast<uint32_t>(tlo + wave * KVT);
  find(tw, pg);
  load(cur, pg, tw);
  find(tw + W * KVT, pg);

  // this lane's row: its query as binary16 (scaled by a power of two for bfloat16), what it sees
  f16x8 q[KD / 8];
  float qs = a.scale * 1.44269504088896340736f;  // the factor of a score
  int lo, hi;
  {
    const int r = r0 + col;
    const bool ok = r < nrows;
    const int rr = ok ? r : nrows - 1, i = rr / G, hq = h * G + rr % G;
    const int64_t at = (first + i) * a.q_stride + static_cast<int64_t>(hq) * D + g * KD;
    hi = ok ? row_hi(i) : 0;
    lo = row_lo(i);
    // at any element's address; rows past the last read its row and see nothing
    typedef f16x8 f16x8_2 __attribute__((aligned(2)));
    const f16* src = static_cast<const f16*>(a.q) + at;
#pragma unroll
    for (int x = 0; x < KD / 8; ++x) q[x] = *reinterpret_cast<const f16x8_2*>(src + 8 * x);
    if (a.dtype != LT_F16) {
      uint32_t top = 0;
#pragma unroll
      for (int x = 0; x < KD / 8; ++x) {
        const u32x4 v = __builtin_bit_cast(u32x4, q[x]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t m0 = (v[e] << 16) & 0x7FFFFFFFu, m1 = v[e] & 0x7FFF0000u;
          top = top > m0 ? top : m0;
          top = top > m1 ? top : m1;
        }
      }
#pragma unroll
      for (int o = 16; o <= 32; o <<= 1) {
        const uint32_t m = static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), o, 64));
        top = top > m ? top : m;
      }
      // the largest magnitude comes to [2^14, 2^15): binary16 then holds what is 2^-28 of it exactly
      int e2 = static_cast<int>(top >> 23) - 127 - 14;
      if (top >= 0x7F800000u || top < 0x00800000u) e2 = 0;
      const float s1 = two(-(e2 / 2)), s2 = two(-(e2 - e2 / 2));
#pragma unroll
      for (int x = 0; x < KD / 8; ++x) {
        const bf16x8 v = __builtin_bit_cast(bf16x8, q[x]);
#pragma unroll
        for (int e = 0; e < 8; ++e) q[x][e] = static_cast<f16>(static_cast<float>(v[e]) * s1 * s2);
      }
      qs = qs * two(e2 / 2) * two(e2 - e2 / 2);
    }
  }

  f32x4 o[VD];
  float m = -__builtin_inff(), l = 0.f;
#pragma unroll
  for (int j = 0; j < VD; ++j) o[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  int ve = KV_NONE;  // this lane's row's sums are in units of 2^(ve - KV_PE)
  bool bad = false;

#pragma unroll 1
  for (int t0 = tlo + wave * KVT; t0 < thi; t0 += (W * KVT)) {
    KvStep<D> nxt;
    load(nxt, pg, static_cast<uint32_t>(t0) + W * KVT);
    find(static_cast<uint32_t>(t0) + 2 * (W * KVT), pg);
    bad |= cur.pg[0] == -1 || cur.pg[1] == -1;
    // scores
    f32x4 s[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      s[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int x = 0; x < KD / 8; ++x) {
        const f16x8 kf = cat8(kv_half4<FP8>(cur.k[u].w[2 * x]), kv_half4<FP8>(cur.k[u].w[2 * x + 1]));
        s[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, q[x], s[u], 0, 0, 0);
      }
    }
    const bool masked = t0 < full_lo || t0 + KVT > full_hi || cur.pg[0] < 0 || cur.pg[1] < 0;
    // a page's value scale above all that the row has seen: its sums go into that one's units
    const int was = ve;
    {
      int e[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) e[u] = kv_scale_exp(cur.vs[u]);
      if (masked) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
          if (cur.pg[u] < 0 || t0 + 16 * u >= hi || t0 + 16 * u + 16 <= lo) e[u] = KV_NONE;
      }
      const int top = e[0] > e[1] ? e[0] : e[1];
      ve = top > ve ? top : ve;
    }
    float top = -__builtin_inff();
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float v = s[u][e] * (qs * cur.ks[u]);
        if (masked) {
          const int tok = t0 + 16 * u + 4 * g + e;
          if (cur.pg[u] < 0 || tok < lo || tok >= hi) v = -__builtin_inff();
        }
        s[u][e] = v;
        top = fmaxf(top, v);
      }
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const float mn = fmaxf(m, top), base = mn == -__builtin_inff() ? 0.f : mn;
    const float f = __builtin_amdgcn_exp2f(m - base);
    m = mn;
    l *= f;
    const float fo = kv_shift(f, was - ve);
#pragma unroll
    for (int j = 0; j < VD; ++j) o[j] *= fo;
    f16x8 pf, pl;  // the weights; TWO: what binary16 leaves of them
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const float w = kv_shift(cur.vs[u], KV_PE - ve);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float v = s[u][e], p = __builtin_amdgcn_exp2f(v - base);
        l += p;
        // a masked token's weight is 0 whatever its page's scale holds
        const float x = v == -__builtin_inff() ? 0.f : p * w;
        pf[4 * u + e] = static_cast<f16>(x);
        if constexpr (TWO) pl[4 * u + e] = static_cast<f16>(x - static_cast<float>(pf[4 * u + e]));
      }
    }
    // values
    if (masked) {
#pragma unroll
      for (int x = 0; x < 8; ++x)
        if (cur.pg[x >> 2] < 0 || t0 + 16 * (x >> 2) + 4 * g + (x & 3) >= thi) {
#pragma unroll
          for (int y = 0; y < (VD + 3) / 4; ++y) cur.v[x].w[y] = 0u;  // no token: its codes may be anything
        }
    }
#pragma unroll
    for (int y = 0; y < (VD + 3) / 4; ++y) {
      // words of four d, eight tokens -> four fragments of eight tokens
      f16x4 t4[8];
#pragma unroll
      for (int x = 0; x < 8; ++x) t4[x] = kv_half4<FP8>(cur.v[x].w[y]);
#pragma unroll
      for (int z = 0; z < 4; ++z) {
        if (4 * y + z >= VD) break;
        const f16x8 vf = {t4[0][z], t4[1][z], t4[2][z], t4[3][z], t4[4][z], t4[5][z], t4[6][z], t4[7][z]};
        if constexpr (TWO) o[4 * y + z] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pl, o[4 * y + z], 0, 0, 0);
        o[4 * y + z] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf, o[4 * y + z], 0, 0, 0);
      }
    }
    cur = nxt;
  }
  if (bad && lane == 0 && c.status != nullptr) atomicMax(c.status, KV_BAD);

  // The waves' parts meet in LDS. Sums of rows: over the four lanes of a column, then the waves.
  constexpr int JT = VD < 8 ? VD : 8;  // output tiles of a round
  __shared__ float wm[W][16], wl[W][16];
  __shared__ f32x4 red[W][JT][64];
  __shared__ float row[16][D];
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  if (g == 0) {
    wm[wave][col] = m;
    wl[wave][col] = l;
  }
  __syncthreads();
  float top = wm[0][col];
#pragma unroll
  for (int w = 1; w < W; ++w) top = fmaxf(top, wm[w][col]);
  const float base = top == -__builtin_inff() ? 0.f : top;
  float sum = 0.f;
#pragma unroll
  for (int w = 0; w < W; ++w) sum += wl[w][col] * __builtin_amdgcn_exp2f(wm[w][col] - base);
  const float mine = __builtin_amdgcn_exp2f(m - base);
#pragma unroll
  for (int j0 = 0; j0 < VD; j0 += JT) {
    if (j0 > 0) __syncthreads();
#pragma unroll
    for (int j = 0; j < JT; ++j) {
      const f32x4 v = o[j0 + j] * mine;
      red[wave][j][lane] = f32x4{kv_shift(v[0], ve - KV_PE), kv_shift(v[1], ve - KV_PE), kv_shift(v[2], ve - KV_PE), kv_shift(v[3], ve - KV_PE)};
    }
    __syncthreads();
#pragma unroll 1
    for (int j = wave; j < JT; j += W) {  // the waves finish a tile each
      f32x4 v = red[0][j][lane];
#pragma unroll
      for (int w = 1; w < W; ++w) v += red[w][j][lane];
#pragma unroll
      for (int e = 0; e < 4; ++e) row[col][VD * (4 * g + e) + j0 + j] = v[e];
    }
  }
  // sums of this workgroup's tokens: the rows' outputs in `row`, maxima and sums where wave is 0 and g is 0
  __shared__ float rm[16], rl[16];
  if (tid < 16) {
    rm[tid] = top;
    rl[tid] = sum;
  }
  __syncthreads();
  const int rows = nrows - r0 < 16 ? nrows - r0 : 16, pieces = rows * (D / 4);  // pieces of four values
  auto put = [&](int p, f32x4 v, float lsum) {
    const int r = r0 + p / (D / 4);
    const float inv = lsum != 0.f ? 1.f / lsum : 0.f;
    const int64_t at = (static_cast<int64_t>(first + r / G) * a.Hq + h * G + r % G) * D + p % (D / 4) * 4;
    typedef u32x2 u32x2_2 __attribute__((aligned(2)));
    v *= inv;
    *reinterpret_cast<u32x2_2*>(static_cast<uint16_t*>(a.o) + at) =
        a.dtype == LT_F16 ? __builtin_bit_cast(u32x2, __builtin_convertvector(v, f16x4)) : __builtin_bit_cast(u32x2, __builtin_convertvector(v, bf16x4));
  };
  if (parts == 1) {
#pragma unroll 1
    for (int p = tid; p < pieces; p += 64 * W) put(p, *reinterpret_cast<const f32x4*>(&row[p / (D / 4)][p % (D / 4) * 4]), rl[p / (D / 4)]);
    return;
  }
  constexpr int COHERENT = 1 | 16;  // sc0 sc1: past the L2 of the XCD
  constexpr uint32_t PART = static_cast<uint32_t>(kv_part_bytes<D>());
  __shared__ int s_last;
  uint32_t* cnt = static_cast<uint32_t*>(a.ws);
  const rsrc_t rW = mk_rsrc(static_cast<uint8_t*>(a.ws) + KV_COUNTERS + static_cast<int64_t>(unit) * splits * PART, splits * PART);
#pragma unroll 1
  for (int p = tid; p < pieces; p += 64 * W)
    __builtin_amdgcn_raw_buffer_store_b128(*reinterpret_cast<const u32x4*>(&row[p / (D / 4)][p % (D / 4) * 4]), rW, split * PART + p * 16, 0, COHERENT);
  if (tid < rows) {
    const u32x2 ml = {__builtin_bit_cast(uint32_t, rm[tid]), __builtin_bit_cast(uint32_t, rl[tid])};
    __builtin_amdgcn_raw_buffer_store_b64(ml, rW, split * PART + 16 * D * 4 + tid * 8, 0, COHERENT);
  }
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (tid == 0) s_last = __hip_atomic_fetch_add(cnt + unit, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == parts - 1;
  __syncthreads();
  if (!s_last) return;
  if (tid == 0) __hip_atomic_store(cnt + unit, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  // The join: `groups` groups of threads take every groups-th part each, four parts' loads in flight, then meet in LDS.
  const int groups = pieces < 64 * W ? 64 * W / pieces : 1;
  f32x4* jo = &red[0][0][0];                                                 // [512]
  float *jm = reinterpret_cast<float*>(jo + 64 * W), *jl = jm + 64 * W;  // [512] each
  static_assert(sizeof(red) >= 64 * W * 24, "the join fits the waves' sums");
#pragma unroll 1
  for (int p0 = 0; p0 < pieces; p0 += 64 * W) {
    const int p = p0 + (groups > 1 ? tid % pieces : tid), grp = groups > 1 ? tid / pieces : 0;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    float vm = -__builtin_inff(), vl = 0.f;
    if (p < pieces && grp < groups) {
#pragma unroll 1
      for (uint32_t s = grp; s < parts; s += 4 * groups) {
        u32x4 x[4];
        f32x2 ml[4];
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
          const uint32_t at = s + i * groups < parts ? (s + i * groups) * PART : 0x80000000u;  // past the last: zeros
          x[i] = __builtin_amdgcn_raw_buffer_load_b128(rW, at + p * 16, 0, COHERENT);
          ml[i] = __builtin_bit_cast(f32x2, __builtin_amdgcn_raw_buffer_load_b64(rW, at + 16 * D * 4 + p / (D / 4) * 8, 0, COHERENT));
        }
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
          if (s + i * groups >= parts) break;
          const float pm = ml[i][0], mn = fmaxf(vm, pm), bs = mn == -__builtin_inff() ? 0.f : mn;
          const float f0 = __builtin_amdgcn_exp2f(vm - bs), f1 = __builtin_amdgcn_exp2f(pm - bs);
          v = v * f0 + __builtin_bit_cast(f32x4, x[i]) * f1;
          vl = vl * f0 + ml[i][1] * f1;
          vm = mn;
        }
      }
    }
    if (groups > 1) {
      jo[tid] = v;
      jm[tid] = vm;
      jl[tid] = vl;
      __syncthreads();
      if (grp == 0) {
        float bs = vm;
        for (int k = 1; k < groups; ++k) bs = fmaxf(bs, jm[tid + k * pieces]);
        bs = bs == -__builtin_inff() ? 0.f : bs;
        v = f32x4{0.f, 0.f, 0.f, 0.f};
        vl = 0.f;
        for (int k = 0; k < groups; ++k) {
          const float f = __builtin_amdgcn_exp2f(jm[tid + k * pieces] - bs);
          v += jo[tid + k * pieces] * f;
          vl += jl[tid + k * pieces] * f;
        }
      }
    }
    if (p < pieces && grp == 0) put(p, v, vl);
  }
}

// ---------------------------------------------------------------------------
// Many rows: products bound the call. A workgroup takes 128 rows (32 a wave) of one sequence and key head and walks over
// tiles of TT tokens: their codes become binary16 in LDS once for all rows, K as it lies (tokens by d), V transposed (d
// by tokens, the tokens of a piece in the order in which the scores leave the MFMA). The sums are those
// above with v_mfma_f32_32x32x16: a row's maximum, sum and factor belong to a lane, and P goes from one product
// into the next without leaving its lane. Pieces of 16 bytes are swizzled by their row, so that neither the
// fragments' rows nor the transposing stores meet in a bank.
//
// VALU instructions bound it, about 500 a wave and 64 tokens (codes to binary16, softmax); MFMAs run a fifth of the time. Two chunks
// of 2000 on 4000 tokens, 32 heads of 128 on 8: 262 to 272 us by the box; 32 tokens a tile with three workgroups a CU 476, eight waves 276.
//
// Two stages: while tile i computes, tile i + 1 goes from registers to LDS, tile i + 2 is loaded and the
// pages of tile i + 3 are looked up. One barrier a tile.
//
// A row's maximum may lag by up to 2^KV_LAG: the outputs are rescaled only when some row of the wave outgrows that
// (2^(KV_PE + KV_LAG) stays inside binary16). Workgroups of one key head follow each other on one XCD's L2 where heads and
// sequences make a multiple of eight; the rows that see the most tokens come first. Few workgroups
// and long contexts: tokens are split and joined as above.
constexpr int KVM_WAVES = 4, KVM_ROWS = 32 * KVM_WAVES, KVM_T = 64 * KVM_WAVES;
constexpr float KV_LAG = 4.f;

template <int D>
struct KvTile {
  static constexpr int TT = D > 128 ? 32 : 64;                     // tokens of a tile
  static constexpr int KP = D <= 64 ? 128 : D <= 128 ? 256 : 512;  // bytes of a token's K, of a d's V
  static constexpr int VP = TT * 2;
  static constexpr int STAGE = TT * KP + D * VP;
  static constexpr int KN = (TT * D / 16 + KVM_T - 1) / KVM_T, VN = (TT * D / 32 + KVM_T - 1) / KVM_T;  // pieces a thread moves
  static constexpr int64_t PART = KVM_ROWS * (D + 2) * 4;
};

// The slot of a token's K piece: a fragment reads one piece of eight consecutive tokens, a thread stores pieces 2 p and 2 p + 1
// of one, eight p after each other; both meet eight different columns of the banks.
__device__ __forceinline__ int kv_kslot(int t, int piece) { return piece ^ ((t ^ (piece >> 3)) & 7); }

template <int D>
__device__ __forceinline__ int kv_vslot(int d, int piece) {
  return KvTile<D>::TT == 64 ? piece ^ ((d ^ (d >> 3)) & 7) : piece ^ (((d >> 1) ^ (d >> 3)) & 3);
}

template <int D, bool FP8>
__global__ __launch_bounds__(KVM_T, D > 128 ? 1 : 2) void k_kv8_tile(KvAttnArgs a, uint32_t row_tiles, uint32_t splits, uint32_t chunk) {
  typedef KvTile<D> Ti;
  constexpr int TT = Ti::TT, KN = Ti::KN, VN = Ti::VN, JT = D / 32, GR = TT / 16;
  extern __shared__ __align__(16) unsigned char smem[];
  const KvCache& c = a.c;
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 31, hf = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t nbh = static_cast<uint32_t>(c.Hkv) * static_cast<uint32_t>(c.B), bh = blockIdx.x % nbh, rest = blockIdx.x / nbh;
  const uint32_t split = rest % splits;
  const int tile = static_cast<int>(row_tiles - 1 - rest / splits);
  const uint32_t unit = bh * row_tiles + static_cast<uint32_t>(tile);
  const int h = static_cast<int>(bh % static_cast<uint32_t>(c.Hkv)), b = static_cast<int>(bh / static_cast<uint32_t>(c.Hkv));
  const int G = a.Hq / c.Hkv;
  int first, count;
  if (!kv_rows(c, b, a.max_new, first, count) && tid == 0 && c.status != nullptr) atomicMax(c.status, KV_BAD);
  const int nrows = count * G, r0 = tile * KVM_ROWS;
  if (r0 >= nrows) return;
  const int span = c.width << c.page_log2, all = c.lengths[b] > 0 ? c.lengths[b] : 0, past = all - count;
  const int len = all < span ? all : span;
  if (all > span && tid == 0 && c.status != nullptr) atomicMax(c.status, KV_BAD);
  auto row_hi = [&](int i) { return a.causal && past + i + 1 < len ? past + i + 1 : len; };
  auto row_lo = [&](int i) { return a.window > 0 && past + i + 1 > a.window ? past + i + 1 - a.window : 0; };  // no difference below -2^31
  auto query = [&](int r) { return (r < nrows ? r : nrows - 1) / G; };  // of a row, the last one's past the end
  const int hi_all = row_hi(query(r0 + KVM_ROWS - 1)), lo_all = (row_lo(query(r0)) < hi_all ? row_lo(query(r0)) : hi_all) / TT * TT;
  const uint32_t parts = hi_all > lo_all ? (static_cast<uint32_t>(hi_all - lo_all) + chunk - 1) / chunk : 1u;
  if (split >= parts) return;
  const int tlo = lo_all + static_cast<int>(split * chunk);
  const int thi = splits > 1 && split + 1 < parts ? tlo + static_cast<int>(chunk) : hi_all;
  // this wave's rows: the tokens that any sees, and those that all see
  const int w0 = r0 + 32 * wave;
  const bool live = w0 < nrows;
  const int wlo = row_lo(query(w0)), whi = live ? row_hi(query(w0 + 31)) : 0, full_lo = row_lo(query(w0 + 31)), full_hi = row_hi(query(w0));

  // ---- moving a tile: K pieces of 16 codes of a token, V pieces of four tokens by eight d
  // Everything of a tile is loaded together, from pages looked up a tile before. Lane l looks up the page of the 16 tokens
  // l % GR and loads one scale of theirs, K's or (l & GR) V's; what a wave needs of them it reads from the lanes.
  uint32_t kc[KN][4], vc[VN][8];
  int32_t pgl;                 // this lane's page of the tile to be loaded next
  float scn;                   // this lane's scale of the loaded tile
  uint32_t none_n = 0;         // the loaded tile's 16-token groups in no page, a bit each
  bool bad = false;
  const int lg = lane & (GR - 1), seen = row_lo(query(r0));  // the first token that a row sees: pages wholly before it may be gone
  auto find = [&](int t0) {
    const int t = t0 + 16 * lg;
    const int32_t p = kv_page(c, b, t);
    pgl = ((t < thi) & (t + 16 > seen)) ? p : -2;
  };
  const uint32_t page_bytes = static_cast<uint32_t>(c.page) * D;  // of one head
  auto page_of = [&](int u) {  // of a group, page 0 where there is none
    const int32_t p = __builtin_amdgcn_readlane(pgl, u);
    return static_cast<uint32_t>(p < 0 ? 0 : p);
  };
  // where the first code of a group of 16 tokens lies
  auto group = [&](const uint8_t* base, int t0, int u) {
    const uint64_t at = static_cast<uint64_t>(page_of(u)) * static_cast<uint32_t>(c.Hkv) + static_cast<uint32_t>(h);
    return base + at * page_bytes + static_cast<uint32_t>((t0 + 16 * u) & (c.page - 1)) * D;
  };
  // The group of a thread's piece: one for the wave where its 64 pieces lie in 16 tokens, else chosen by lane.
  constexpr int KPT = D / 16, VPT = D / 32;  // K pieces of a token, V pieces (of four tokens) a token
  auto src_of = [&](const uint8_t* base, int t0, int x0, int per, int t, uint32_t off) {  // x0: the wave's first piece
    if (16 * per % 64 == 0) return group(base, t0, x0 / (16 * per)) + off;
    const uint8_t* g0 = group(base, t0, 0);
    const uint8_t* g1 = group(base, t0, 1);
    const uint8_t* g2 = group(base, t0, GR - 2);
    const uint8_t* g3 = group(base, t0, GR - 1);
    const uint8_t* r = (t & 16) != 0 ? g1 : g0;
    if (GR == 4 && (t & 32) != 0) r = (t & 16) != 0 ? g3 : g2;
    return r + off;
  };
  auto load = [&](int t0) {
    const int64_t at = static_cast<int64_t>(pgl < 0 ? 0 : pgl) * c.Hkv + h;
    scn = (lane & GR) != 0 ? c.vs[at] : c.ks[at];
    none_n = static_cast<uint32_t>(__ballot(pgl < 0)) & ((1u << GR) - 1u);
    bad |= pgl == -1;
#pragma unroll
    for (int i = 0; i < KN; ++i) {
      const int x = tid + KVM_T * i, t = x / KPT;
      const u32x4 v = ld16(src_of(c.k, t0, 64 * wave + KVM_T * i, KPT, t, static_cast<uint32_t>(t % 16 * D + x % KPT * 16)));
#pragma unroll
      for (int e = 0; e < 4; ++e) kc[i][e] = v[e];
    }
#pragma unroll
    for (int i = 0; i < VN; ++i) {
      const int x = tid + KVM_T * i, t = x / (4 * VPT) * 4;
      const uint8_t* src = src_of(c.v, t0, 64 * wave + KVM_T * i, VPT, t, static_cast<uint32_t>(t % 16 * D + x % (4 * VPT) * 8));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const u32x2 v = *reinterpret_cast<const u32x2*>(src + e * D);
        vc[i][2 * e] = v[0];
        vc[i][2 * e + 1] = v[1];
      }
    }
  };
  auto store = [&](int t0, int st) {
    unsigned char* ks = smem + st * Ti::STAGE;
    unsigned char* vs = ks + TT * Ti::KP;
#pragma unroll
    for (int i = 0; i < KN; ++i) {
      const int x = tid + KVM_T * i, t = x / (D / 16), p = x % (D / 16);
      if (KN * KVM_T > TT * (D / 16) && t >= TT) break;
      *reinterpret_cast<f16x8*>(ks + t * Ti::KP + kv_kslot(t, 2 * p) * 16) = cat8(kv_half4<FP8>(kc[i][0]), kv_half4<FP8>(kc[i][1]));
      *reinterpret_cast<f16x8*>(ks + t * Ti::KP + kv_kslot(t, 2 * p + 1) * 16) = cat8(kv_half4<FP8>(kc[i][2]), kv_half4<FP8>(kc[i][3]));
    }
#pragma unroll
    for (int i = 0; i < VN; ++i) {
      const int x = tid + KVM_T * i, q = x / (D / 8), d0 = x % (D / 8) * 8;
      if (VN * KVM_T > TT * D / 32 && q >= TT / 4) break;
      if (none_n != 0 || t0 + TT > thi) {  // tokens that are none: their codes may be anything
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if ((none_n >> (q >> 2) & 1u) != 0 || t0 + 4 * q + e >= thi) vc[i][2 * e] = vc[i][2 * e + 1] = 0u;
      }
      // tokens 4 q .. + 3 of a 32: piece 2 (q / 4) + q % 2, its half q / 2 % 2
      const int piece = q / 8 * 4 + (q % 8) / 4 * 2 + (q & 1), half = (q >> 1) & 1;
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const uint32_t r0 = vc[i][y], r1 = vc[i][2 + y], r2 = vc[i][4 + y], r3 = vc[i][6 + y];
        const uint32_t a0 = __builtin_amdgcn_perm(r1, r0, 0x05010400u), a1 = __builtin_amdgcn_perm(r1, r0, 0x07030602u);
        const uint32_t b0 = __builtin_amdgcn_perm(r3, r2, 0x05010400u), b1 = __builtin_amdgcn_perm(r3, r2, 0x07030602u);
        const uint32_t z[4] = {__builtin_amdgcn_perm(b0, a0, 0x05040100u), __builtin_amdgcn_perm(b0, a0, 0x07060302u),
                               __builtin_amdgcn_perm(b1, a1, 0x05040100u), __builtin_amdgcn_perm(b1, a1, 0x07060302u)};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int d = d0 + 4 * y + e;
          *reinterpret_cast<f16x4*>(vs + d * Ti::VP + kv_vslot<D>(d, piece) * 16 + half * 8) = kv_half4<FP8>(z[e]);
        }
      }
    }
  };

  // ---- the wave's queries as binary16 (scaled by a power of two for bfloat16): lane (row, half) holds d 16 x + 8 half .. + 7
  f16x8 q[D / 16];
  float qs = a.scale * 1.44269504088896340736f;  // the factor of a score
  int lo = 0, hi = 0;
  const int r = w0 + col;
  find(tlo);
  load(tlo);
  {
    const bool ok = r < nrows;
    const int i = query(r), hq = h * G + (ok ? r % G : 0);
    const uint16_t* src = static_cast<const uint16_t*>(a.q) + (first + i) * a.q_stride + static_cast<int64_t>(hq) * D + 8 * hf;
    const bool whole = ((reinterpret_cast<uintptr_t>(a.q) | static_cast<uintptr_t>(a.q_stride * 2)) & 15u) == 0;
    hi = ok ? row_hi(i) : 0;
    lo = row_lo(i);
#pragma unroll
    for (int x = 0; x < D / 16; ++x) {
      u32x4 v = {0u, 0u, 0u, 0u};
      if (ok) {
        if (whole) v = ld16(src + 16 * x);
        else
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = src[16 * x + 2 * e] | (static_cast<uint32_t>(src[16 * x + 2 * e + 1]) << 16);
      }
      q[x] = __builtin_bit_cast(f16x8, v);
    }
    if (a.dtype != LT_F16) {
      uint32_t top = 0;
#pragma unroll
      for (int x = 0; x < D / 16; ++x) {
        const u32x4 v = __builtin_bit_cast(u32x4, q[x]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t m0 = (v[e] << 16) & 0x7FFFFFFFu, m1 = v[e] & 0x7FFF0000u;
          top = top > m0 ? top : m0;
          top = top > m1 ? top : m1;
        }
      }
      const uint32_t m2 = static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 32, 64));
      top = top > m2 ? top : m2;
      // the largest magnitude comes to [2^14, 2^15): binary16 then holds what is 2^-28 of it exactly
      int e2 = static_cast<int>(top >> 23) - 127 - 14;
      if (top >= 0x7F800000u || top < 0x00800000u) e2 = 0;
      const float s1 = two(-(e2 / 2)), s2 = two(-(e2 - e2 / 2));
#pragma unroll
      for (int x = 0; x < D / 16; ++x) {
        const bf16x8 v = __builtin_bit_cast(bf16x8, q[x]);
#pragma unroll
        for (int e = 0; e < 8; ++e) q[x][e] = static_cast<f16>(static_cast<float>(v[e]) * s1 * s2);
      }
      qs = qs * two(e2 / 2) * two(e2 - e2 / 2);
    }
  }

  f32x16 o[JT];
#pragma unroll
  for (int j = 0; j < JT; ++j)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[j][e] = 0.f;
  float m = -__builtin_inff(), l = 0.f;
  int ve = KV_NONE;                  // this lane's row's sums are in units of 2^(ve - KV_PE)
  int most = KV_NONE, least = KV_NONE;  // at least, and at most, what ve is in every row of the wave
  float up = 0.f, down = 1.f;        // most - ve, and 2^-up
  // scale (as scn) and missing groups of the tile in LDS
  float scl;
  uint32_t none;
  auto take = [&] {
    scl = scn;
    none = none_n;
  };
  store(tlo, 0);
  take();
  find(tlo + TT);
  load(tlo + TT);
  find(tlo + 2 * TT);
  __syncthreads();

  int st = 0;
#pragma unroll 1
  for (int t0 = tlo; t0 < thi; t0 += TT, st ^= 1) {
    const unsigned char* ks = smem + st * Ti::STAGE;
    const unsigned char* vs = ks + TT * Ti::KP;
    auto move = [&] {  // the next tile to the other stage, the one after it to registers
      if (t0 + TT < thi) {
        store(t0 + TT, st ^ 1);
        take();
        load(t0 + 2 * TT);
        find(t0 + 3 * TT);
      }
    };
    if (t0 >= whi || t0 + TT <= wlo) {  // none of it is this wave's
      move();
      __syncthreads();
      continue;
    }
    const uint32_t no = none;
    const float sc = scl;
    const int was = ve;
    const bool open = no == 0 && t0 >= full_lo && t0 + TT <= full_hi;  // every row sees all of it
    // a value scale above all that a row has seen: its sums go into that one's units
    {
      const int el = kv_scale_exp(sc);
      int e[GR], top = KV_NONE;
#pragma unroll
      for (int u = 0; u < GR; ++u) {
        e[u] = __builtin_amdgcn_readlane(el, GR + u);
        top = e[u] > top ? e[u] : top;
      }
      if (!open || top > least) {
        if (open) {
          ve = top > ve ? top : ve;
          least = top;
        } else {
          top = KV_NONE;
#pragma unroll
          for (int u = 0; u < GR; ++u) {
            const int t = t0 + 16 * u;
            const bool have = (no >> u & 1u) == 0;
            top = have && t < whi && t + 16 > wlo && e[u] > top ? e[u] : top;
            ve = have && t < hi && t + 16 > lo && e[u] > ve ? e[u] : ve;
          }
        }
        most = top > most ? top : most;
        up = static_cast<float>(most - ve);
        down = kv_shift(1.f, ve - most);
      }
    }
    // Fragments are read ahead of their products: heads of 256 have one wave a SIMD, which waits for what it reads (1108 us read by read,
    // 978 four ahead of both products; two chunks of 2000 on 4000, 32 heads on 8). With 64 to 128 two ahead of K's: 280 for 286 at 96.
    f32x16 s[TT / 32];
    constexpr int KA = D > 128 ? 4 : 2;
    auto kfrag = [&](int x, int u) { return *reinterpret_cast<const f16x8*>(ks + (32 * u + col) * Ti::KP + kv_kslot(col, 2 * x + hf) * 16); };
    f16x8 kf[KA][TT / 32];
#pragma unroll
    for (int x = 0; x < KA; ++x)
#pragma unroll
      for (int u = 0; u < TT / 32; ++u) kf[x][u] = kfrag(x, u);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int x = 0; x < D / 16; ++x) {
#pragma unroll
      for (int u = 0; u < TT / 32; ++u) {
        s[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[x % KA][u], q[x], x == 0 ? f32x16{} : s[u], 0, 0, 0);
        if (x + KA < D / 16) kf[x % KA][u] = kfrag(x + KA, u);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    // A wave in between its products goes first, so that the SIMD's other one has the matrix cores meanwhile. It pays for heads of 64, whose
    // products are short (2048 tokens on themselves 51 -> 46.5 us); with 96, 128 and 256 it costs 0 to 3 %.
    if constexpr (D <= 64) __builtin_amdgcn_s_setprio(1);
    // lane-wise: V's factor of the weights, its logarithm and inverse, in units of 2^(most - KV_PE); or K's of the scores
    const float wl = kv_shift(sc, KV_PE - most), lwl = __builtin_amdgcn_logf(wl), rwl = __builtin_amdgcn_rcpf(wl);
    // factors of the usual kind, no masks: see below
    const bool usual = (lane & GR) != 0 ? wl >= 0x1p-8f && wl < 0x1p11f : sc >= 0.f && a.scale >= 0.f;
    const bool plain = (__ballot(!usual) & ((1u << (2 * GR)) - 1u)) == 0 && open;
    auto of = [&](float x, int u) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), u)); };
    move();
    {
      float top = -__builtin_inff();
      if (plain) {
        // no masks, key factors not negative: a group's largest score is its largest sum's
#pragma unroll
        for (int u = 0; u < GR; ++u) {
          float x = s[u / 2][8 * (u & 1)];
#pragma unroll
          for (int e = 1; e < 8; ++e) x = fmaxf(x, s[u / 2][8 * (u & 1) + e]);
          top = fmaxf(top, x * (qs * of(sc, u)));
        }
      } else {
#pragma unroll
        for (int u = 0; u < TT / 32; ++u)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int tok = 32 * u + 8 * (e >> 2) + 4 * hf + (e & 3);
            const bool out = (no >> (2 * u + (e >> 3)) & 1u) != 0 || t0 + tok < lo || t0 + tok >= hi;
            s[u][e] = out ? -__builtin_inff() : s[u][e] * (qs * of(sc, 2 * u + (e >> 3)));
            top = fmaxf(top, s[u][e]);
          }
      }
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      if (__any(top > m + KV_LAG || was < ve)) {
        const float mn = fmaxf(m, top), base = mn == -__builtin_inff() ? 0.f : mn;
        const float f = __builtin_amdgcn_exp2f(m - base);
        m = mn;
        l *= f;
        const float fo = kv_shift(f, was - ve);
#pragma unroll
        for (int j = 0; j < JT; ++j)
#pragma unroll
          for (int e = 0; e < 16; ++e) o[j][e] *= fo;
      }
      const float base = m == -__builtin_inff() ? 0.f : m, rise = up - base;
      float sums = 0.f;
      if constexpr (D <= 64) __builtin_amdgcn_s_setprio(0);
#pragma unroll
      for (int u = 0; u < TT / 32; ++u)
#pragma unroll
        for (int sl = 0; sl < 2; ++sl) {
          const int gu = 2 * u + sl;
          f16x8 pf;
          if (plain) {
            // the exponential with the value's factor in its exponent: one multiply-add and one exponential a weight
            const float kf = qs * of(sc, gu), lw = of(lwl, GR + gu) + rise;
            float sum = 0.f;
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
              const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][8 * sl + e], kf, lw));
              const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][8 * sl + e + 1], kf, lw));
              sum += p0 + p1;
              const f16x2 h2 = __builtin_convertvector((f32x2{p0, p1}), f16x2);
              pf[e] = h2[0];
              pf[e + 1] = h2[1];
            }
            sums += sum * of(rwl, GR + gu);
          } else {
            const float w = kv_shift(of(sc, GR + gu), KV_PE - ve);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float v = s[u][8 * sl + e], p = __builtin_amdgcn_exp2f(v - base);
              l += p;
              // a masked token's weight is 0 whatever its page's scale holds
              pf[e] = static_cast<f16>(v == -__builtin_inff() ? 0.f : p * w);
            }
          }
          auto vfrag = [&](int j) {
            const int d = 32 * j + col;
            return *reinterpret_cast<const f16x8*>(vs + d * Ti::VP + kv_vslot<D>(d, u * 4 + sl * 2 + hf) * 16);
          };
          if constexpr (D > 128) {
            constexpr int VA = 4;
            f16x8 vf[VA];
#pragma unroll
            for (int j = 0; j < VA; ++j) vf[j] = vfrag(j);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < JT; ++j) {
              o[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[j % VA], pf, o[j], 0, 0, 0);
              if (j + VA < JT) vf[j % VA] = vfrag(j + VA);
              __builtin_amdgcn_sched_barrier(0);
            }
          } else {
#pragma unroll
            for (int j = 0; j < JT; ++j) o[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vfrag(j), pf, o[j], 0, 0, 0);
          }
        }
      l += sums * down;
    }
    __syncthreads();
  }
  if (__any(bad) && lane == 0 && c.status != nullptr) atomicMax(c.status, KV_BAD);

  l += __shfl_xor(l, 32, 64);
  if (parts > 1) {
    constexpr int COHERENT = 1 | 16;  // sc0 sc1: past the L2 of the XCD
    constexpr uint32_t PART = static_cast<uint32_t>(Ti::PART), ML = KVM_ROWS * D * 4;
    int* s_last = reinterpret_cast<int*>(smem);
    uint32_t* cnt = static_cast<uint32_t*>(a.ws);
    const rsrc_t rW = mk_rsrc(static_cast<uint8_t*>(a.ws) + KV_COUNTERS + static_cast<int64_t>(unit) * splits * PART, splits * PART);
    const uint32_t at = (32 * wave + col) * (D * 4) + hf * 16, ml = ML + (32 * wave + col) * 8;
    if (r < nrows) {
#pragma unroll
      for (int j = 0; j < JT; ++j)
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const f32x4 v = {kv_shift(o[j][4 * y], ve - KV_PE), kv_shift(o[j][4 * y + 1], ve - KV_PE), kv_shift(o[j][4 * y + 2], ve - KV_PE), kv_shift(o[j][4 * y + 3], ve - KV_PE)};
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), rW, split * PART + at + j * 128 + y * 32, 0, COHERENT);
        }
      if (hf == 0) __builtin_amdgcn_raw_buffer_store_b64(u32x2{__builtin_bit_cast(uint32_t, m), __builtin_bit_cast(uint32_t, l)}, rW, split * PART + ml, 0, COHERENT);
    }
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (tid == 0) *s_last = __hip_atomic_fetch_add(cnt + unit, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == parts - 1;
    __syncthreads();
    if (!*s_last) return;
    __syncthreads();
    if (tid == 0) __hip_atomic_store(cnt + unit, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    m = -__builtin_inff();
    l = 0.f;
#pragma unroll
    for (int j = 0; j < JT; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[j][e] = 0.f;
    if (r < nrows) {
#pragma unroll 1
      for (uint32_t sp = 0; sp < parts; ++sp) {
        const f32x2 x = __builtin_bit_cast(f32x2, __builtin_amdgcn_raw_buffer_load_b64(rW, sp * PART + ml, 0, COHERENT));
        f32x4 v[JT][4];
#pragma unroll
        for (int j = 0; j < JT; ++j)
#pragma unroll
          for (int y = 0; y < 4; ++y)
            v[j][y] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rW, sp * PART + at + j * 128 + y * 32, 0, COHERENT));
        const float pm = x[0], mn = fmaxf(m, pm), base = mn == -__builtin_inff() ? 0.f : mn;
        const float f0 = __builtin_amdgcn_exp2f(m - base), f1 = __builtin_amdgcn_exp2f(pm - base);
        m = mn;
        l = l * f0 + x[1] * f1;
#pragma unroll
        for (int j = 0; j < JT; ++j)
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const f32x4 x4 = v[j][y];  // elements by name: this compiler may fold v[e >> 2][e & 3] over an array of vectors to element 0
            o[j][4 * y] = o[j][4 * y] * f0 + x4.x * f1;
            o[j][4 * y + 1] = o[j][4 * y + 1] * f0 + x4.y * f1;
            o[j][4 * y + 2] = o[j][4 * y + 2] * f0 + x4.z * f1;
            o[j][4 * y + 3] = o[j][4 * y + 3] * f0 + x4.w * f1;
          }
      }
    }
  }
  // 32 rows through the wave's part of LDS in the output's type, then whole pieces of 16 bytes
  const float inv = l != 0.f ? 1.f / l : 0.f;
  const int unit_e = parts > 1 ? 0 : ve - KV_PE;
  constexpr int PITCH = D * 2 + 16;
  unsigned char* strip = smem + wave * (32 * PITCH);
#pragma unroll
  for (int j = 0; j < JT; ++j)
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      u32x2 v;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float x0 = kv_shift(o[j][4 * y + 2 * e] * inv, unit_e), x1 = kv_shift(o[j][4 * y + 2 * e + 1] * inv, unit_e);
        v[e] = a.dtype == LT_F16 ? __builtin_bit_cast(uint32_t, f16x2{static_cast<f16>(x0), static_cast<f16>(x1)})
                                 : __builtin_bit_cast(uint32_t, bf16x2{static_cast<bf16>(x0), static_cast<bf16>(x1)});
      }
      *reinterpret_cast<u32x2*>(strip + col * PITCH + (32 * j + 8 * y + 4 * hf) * 2) = v;
    }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  const bool vec = (reinterpret_cast<uintptr_t>(a.o) & 15u) == 0;
#pragma unroll 1
  for (int x = lane; x < 32 * (D / 8); x += 64) {
    const int rr = w0 + x / (D / 8), p = x % (D / 8);
    if (rr >= nrows) continue;
    const unsigned char* src = strip + x / (D / 8) * PITCH + p * 16;
    uint16_t* dst = static_cast<uint16_t*>(a.o) + (static_cast<int64_t>(first + rr / G) * a.Hq + h * G + rr % G) * D + p * 8;
    if (vec) *reinterpret_cast<u32x4*>(dst) = *reinterpret_cast<const u32x4*>(src);
    else
      for (int e = 0; e < 8; ++e) dst[e] = reinterpret_cast<const uint16_t*>(src)[e];
  }
}

// Tokens are split only as far as the card has room for more workgroups at once: a start, a join and the code's own fetch
// cost more than even shares gain (one sequence of 65000: 129 us in shares of 256 tokens, 83 of 512, 57 of 1024, 39 of 2048,
// one a CU; 48 of up to 8000: 227 us in shares of 1024, 170 of 2048, 108 unsplit; 8 of 4000: 35 of 512, 25 of 1024, 32 of 2048).
// Up to 16 rows of a key head take k_kv8_rows, more whichever is estimated faster (us; measured at head size 128):
//   rows: for each round of the CUs 7, and the share's tokens at 75 a us; a join 5
//   tile: for each round of two workgroups a CU (heads of 256: one) 10, and the tokens at 36, 28, 24 or 18 a us with one to four
//         waves in use; a join 3 and 2 a part (its parts of 128 rows are read one after the other)
// 8 to 32 new tokens on 30000 with four heads a group: 41 to 79 us by rows, 89 to 184 by tiles; 32 sequences with 16 and 32 on 1000:
// 89 and 172 by rows, 43 and 56 by tiles.
struct KvPlan {
  bool tile;  // k_kv8_tile, else k_kv8_rows
  int waves;  // of k_kv8_rows
  int64_t row_tiles, splits, chunk, ws_bytes;
  double time;
};

KvPlan kind_plan(const KvAttnArgs& a, bool have_ws, bool tile) {
  const int64_t nrows = static_cast<int64_t>(a.max_new) * (a.Hq / a.c.Hkv), cus = device_cus() > 0 ? device_cus() : 256;
  const int64_t rows = tile ? KVM_ROWS : 16;
  KvPlan p{};
  p.tile = tile;
  p.row_tiles = (nrows + rows - 1) / rows;
  const int64_t units = p.row_tiles * a.c.Hkv * a.c.B;
  int64_t span = static_cast<int64_t>(a.c.width) << a.c.page_log2;
  if (a.window > 0) {  // what the rows' windows cover, from a multiple of a tile's tokens on
    const int64_t seen = static_cast<int64_t>(a.window) + (a.causal ? rows : a.max_new) + 64;
    span = span < seen ? span : seen;
  }
  span = span > 0 ? span : 1;
  const int64_t room = tile && a.c.D <= 128 ? 2 * cus : cus;
  const int live = nrows < KVM_ROWS ? static_cast<int>((nrows + 31) / 32) : 4;
  static constexpr double kTile[5] = {0, 36, 28, 24, 18};
  const double rate = tile ? kTile[live] : 75.0, start = tile ? 10.0 : 7.0, wide = a.c.D > 128 ? 2.0 : 1.0;
  const bool can = have_ws && units * 4 <= KV_COUNTERS && span > KVR_PASS && units < room;
  const int64_t most = can ? room / units : 1;
  for (int64_t want = tile ? 1 : most; want <= most; want = tile ? want + (want + 3) / 4 : want + 1) {
    int64_t chunk = want > 1 ? ((span + want - 1) / want + KVR_PASS - 1) / KVR_PASS * KVR_PASS : span;
    const int64_t parts = (span + chunk - 1) / chunk;
    const double time = static_cast<double>((units * parts + room - 1) / room) * (start + wide * static_cast<double>(chunk) / rate) +
                        (parts == 1 ? 0.0 : tile ? 3.0 + 2.0 * static_cast<double>(parts) : 5.0);
    if (p.splits == 0 || time < p.time) {
      p.splits = parts;
      p.chunk = chunk;
      p.time = time;
      p.ws_bytes = parts > 1 ? KV_COUNTERS + units * parts * rows * (a.c.D + 2) * 4 : 0;
    }
  }
  // Waves: two for a share of 64 tokens, four up to 256, and to 2048 where that keeps more than one workgroup a CU resident (us with
  // 8, 4 and 2 at 47 sequences of 12 tokens: 15.5, 10.1, 9.1; 100: 19.4, 12.8, 12.8; 400: 28, 21, 23; 1500: 51, 41, 60; 48
  // of up to 8000: 109, 131, 214; one of 65000: 40, 47, 72).
  p.waves = p.chunk <= 2 * KVT ? 2 : p.chunk <= 8 * KVT || (p.chunk <= 2048 && units * p.splits > cus) ? 4 : 8;
  return p;
}

KvPlan attention_plan(const KvAttnArgs& a, bool have_ws) {
  const KvPlan rows = kind_plan(a, have_ws, false);
  if (static_cast<int64_t>(a.max_new) * (a.Hq / a.c.Hkv) <= 16) return rows;
  const KvPlan tile = kind_plan(a, have_ws, true);
  return tile.time < rows.time ? tile : rows;
}

template <int D, bool FP8>
hipError_t attention_for(const KvAttnArgs& a, const KvPlan& p, hipStream_t st) {
  const int64_t n = p.row_tiles * p.splits * a.c.Hkv * a.c.B;
  if (n > 0x7FFFFFFF) return hipErrorInvalidValue;
  const dim3 grid(static_cast<uint32_t>(n));
  const uint32_t rt = static_cast<uint32_t>(p.row_tiles), sp = static_cast<uint32_t>(p.splits), ch = static_cast<uint32_t>(p.chunk);
  if (!p.tile) {
    auto rows = [&](auto two) {
      switch (p.waves) {
        case 2: k_kv8_rows<D, FP8, 2, decltype(two)::value><<<grid, 128, 0, st>>>(a, rt, sp, ch); break;
        case 4: k_kv8_rows<D, FP8, 4, decltype(two)::value><<<grid, 256, 0, st>>>(a, rt, sp, ch); break;
        default: k_kv8_rows<D, FP8, 8, decltype(two)::value><<<grid, 512, 0, st>>>(a, rt, sp, ch);
      }
    };
    if (p.row_tiles == 1) rows(std::true_type{});
    else rows(std::false_type{});
    return hipGetLastError();
  }
  constexpr int strips = KVM_WAVES * 32 * (D * 2 + 16), lds = 2 * KvTile<D>::STAGE > strips ? 2 * KvTile<D>::STAGE : strips;
  static std::atomic<int> done[kMaxDevices];
  if (lds > 65536) {
    const hipError_t e = raise_lds_cap(reinterpret_cast<const void*>(k_kv8_tile<D, FP8>), lds, done);
    if (e != hipSuccess) return e;
  }
  k_kv8_tile<D, FP8><<<grid, KVM_T, lds, st>>>(a, rt, sp, ch);
  return hipGetLastError();
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
  switch (a.c.D * 2 + (a.c.fp8 ? 1 : 0)) {
    case 128: return attention_for<64, false>(a, p, st);
    case 129: return attention_for<64, true>(a, p, st);
    case 192: return attention_for<96, false>(a, p, st);
    case 193: return attention_for<96, true>(a, p, st);
    case 256: return attention_for<128, false>(a, p, st);
    case 257: return attention_for<128, true>(a, p, st);
    case 512: return attention_for<256, false>(a, p, st);
    case 513: return attention_for<256, true>(a, p, st);
  }
  return hipErrorInvalidValue;
}

hipError_t launch_kv8_append(const KvAppendArgs& a, hipStream_t st) {
  if (a.c.B == 0 || a.max_new == 0) return hipSuccess;
  // pages that a sequence's new tokens can lie in
  const int64_t touched = (a.max_new + a.c.page - 2) / a.c.page + 1;
  const int64_t grid = touched * a.c.B * a.c.Hkv * 2;
  if (grid > 0x7FFFFFFF) return hipErrorInvalidValue;
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
