// The 8-bit paged cache: appending tokens, and attention over it.
#include "xrmm_lowbit.h"

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
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(x), false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(x), true);
    v[0] = lo[0]; v[1] = lo[1]; v[2] = hi[0]; v[3] = hi[1];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = static_cast<float>(static_cast<int8_t>(x >> (8 * i)));
  }
}

template <typename T>
__device__ __forceinline__ void kv_load4(const T* p, bool whole, float (&v)[4]) {
  typedef T vec __attribute__((ext_vector_type(4)));
  if (whole) {
    const vec x = *reinterpret_cast<const vec*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = static_cast<float>(x[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = static_cast<float>(p[i]);
  }
}

constexpr int KVA_T = 256;

template <typename T, bool FP8>
__global__ __launch_bounds__(KVA_T) void k_kv8_append(KvAppendArgs a, uint32_t touched) {
  constexpr float qmax = FP8 ? 448.f : 127.f;
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
  const int32_t page = base < 0 || base > 0x7FFFFFFF ? -1 : kv_page(c, b, static_cast<int>(base));
  if (page < 0) {
    if (tid == 0 && c.status != nullptr) atomicMax(c.status, KV_BAD);
    return;
  }
  const int from = begin > base ? static_cast<int>(begin - base) : 0;              // slots from .. to - 1 are new
  const int to = len - base < c.page ? static_cast<int>(len - base) : c.page;
  const int64_t stride = isv ? a.v_stride : a.k_stride;
  const T* x = static_cast<const T*>(isv ? a.v : a.k) + (first + base + from - begin) * stride + static_cast<int64_t>(h) * c.D;
  const int64_t slot0 = (static_cast<int64_t>(page) * c.Hkv + h) * c.page;
  uint8_t* codes = (isv ? c.v : c.k) + slot0 * c.D;
  float* scale = (isv ? c.vs : c.ks) + static_cast<int64_t>(page) * c.Hkv + h;
  const int pieces = c.D >> 2, all = (to - from) * pieces;  // pieces of four values
  const bool whole = (reinterpret_cast<uintptr_t>(x) | static_cast<uintptr_t>(stride * sizeof(T))) % (4 * sizeof(T)) == 0;

  uint32_t top = 0;  // the largest magnitude's bits (above every finite one's for infinity and NaN)
  for (int p = tid; p < all; p += KVA_T) {
    float v[4];
    kv_load4(x + (p / pieces) * stride + (p % pieces) * 4, whole, v);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t m = __builtin_bit_cast(uint32_t, v[e]) & 0x7FFFFFFFu;
      top = top > m ? top : m;
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint32_t m = static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), o, 64));
    top = top > m ? top : m;
  }
  __shared__ uint32_t tops[KVA_T / 64];
  if ((tid & 63) == 0) tops[tid >> 6] = top;
  const float old = from == 0 ? 0.f : *scale;
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
    for (int p = tid; p < from * pieces; p += KVA_T) {
      uint32_t* w = reinterpret_cast<uint32_t*>(codes) + p;
      float v[4];
      kv_value4<FP8>(*w, v);
      *w = kv_code4<FP8>(v[0] * shrink, v[1] * shrink, v[2] * shrink, v[3] * shrink);
    }
  }
  const bool good = now > 0.f && now <= 3.4028235e38f;
  for (int p = tid; p < all; p += KVA_T) {
    float v[4];
    kv_load4(x + (p / pieces) * stride + (p % pieces) * 4, whole, v);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = good ? fminf(fmaxf(v[e] / now, -qmax), qmax) : 0.f;
    reinterpret_cast<uint32_t*>(codes)[from * pieces + p] = kv_code4<FP8>(v[0], v[1], v[2], v[3]);
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
constexpr float KV_P = 1024.f;  // weights enter binary16 times this: small ones stay normal

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

constexpr int KVR_WAVES = 4;

template <int D, bool FP8, int NT>
__global__ __launch_bounds__(64 * KVR_WAVES) void k_kv8_rows(KvAttnArgs a, uint32_t row_tiles) {
  constexpr int KD = D / 4, VD = D / 16;  // codes of a token that a lane holds
  const KvCache& c = a.c;
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  uint32_t id = blockIdx.x;
  const int tile = static_cast<int>(id % row_tiles);
  id /= row_tiles;
  const int h = static_cast<int>(id % static_cast<uint32_t>(c.Hkv)), b = static_cast<int>(id / static_cast<uint32_t>(c.Hkv));
  const int G = a.Hq / c.Hkv;
  int first, count;
  if (!kv_rows(c, b, a.max_new, first, count) && tid == 0 && c.status != nullptr) atomicMax(c.status, KV_BAD);
  const int nrows = count * G, r0 = tile * 16 * NT;
  if (r0 >= nrows) return;
  // positions past the table are left out: the walk over tokens ends with the table
  const int span = c.width << c.page_log2, all = c.lengths[b], past = all - count;
  const int len = all < 0 ? 0 : all < span ? all : span;
  if (all > span && tid == 0 && c.status != nullptr) atomicMax(c.status, KV_BAD);

  // this lane's rows: their queries as binary16 (scaled by a power of two for bfloat16), what they see
  f16x8 q[NT][KD / 8];
  float qs[NT];  // the factor of a score
  int lo[NT], hi[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int r = r0 + 16 * t + col;
    const bool ok = r < nrows;
    const int i = ok ? r / G : 0, hq = h * G + (ok ? r % G : 0);
    const int64_t at = (first + i) * a.q_stride + static_cast<int64_t>(hq) * D + g * KD;
    const int p = past + i;
    hi[t] = !ok ? 0 : a.causal && p + 1 < len ? p + 1 : len;
    lo[t] = a.window > 0 && p - a.window + 1 > 0 ? p - a.window + 1 : 0;
    qs[t] = a.scale * 1.44269504088896340736f;
    if (a.dtype == LT_F16) {
#pragma unroll
      for (int e = 0; e < KD; ++e) q[t][e / 8][e % 8] = ok ? static_cast<const f16*>(a.q)[at + e] : static_cast<f16>(0.f);
    } else {
      float v[KD];
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < KD; ++e) {
        v[e] = ok ? static_cast<float>(static_cast<const bf16*>(a.q)[at + e]) : 0.f;
        const uint32_t m = __builtin_bit_cast(uint32_t, v[e]) & 0x7FFFFFFFu;
        top = top > m ? top : m;
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
      for (int e = 0; e < KD; ++e) q[t][e / 8][e % 8] = static_cast<f16>(v[e] * s1 * s2);
      qs[t] = qs[t] * two(e2 / 2) * two(e2 - e2 / 2);
    }
  }
  // the tokens that any of the rows sees, and those that all of them see
  const int i0 = r0 / G, i1 = (r0 + 16 * NT < nrows ? r0 + 16 * NT - 1 : nrows - 1) / G;
  auto row_hi = [&](int i) { return a.causal && past + i + 1 < len ? past + i + 1 : len; };
  auto row_lo = [&](int i) { return a.window > 0 && past + i - a.window + 1 > 0 ? past + i - a.window + 1 : 0; };
  const int tlo = row_lo(i0) / KVT * KVT, thi = row_hi(i1), full_lo = row_lo(i1), full_hi = row_hi(i0);

  f32x4 o[NT][VD];
  float m[NT], l[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    m[t] = -__builtin_inff();
    l[t] = 0.f;
#pragma unroll
    for (int j = 0; j < VD; ++j) o[t][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  float vref = 0.f;  // the value scale that the sums are in units of
  bool bad = false;

  for (int t0 = tlo + wave * KVT; t0 < thi; t0 += KVR_WAVES * KVT) {
    // the two 16-token tiles lie in one page each
    int32_t pg[2];
    float ks[2], vs[2];
    const uint8_t *kp[2], *vp[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int t = t0 + 16 * u;
      pg[u] = t < thi ? kv_page(c, b, t) : -2;
      bad |= pg[u] == -1;
      const int64_t at = static_cast<int64_t>(pg[u] < 0 ? 0 : pg[u]) * c.Hkv + h;
      ks[u] = c.ks[at];
      vs[u] = c.vs[at];
      const int64_t slot = at * c.page + (t & (c.page - 1));
      kp[u] = c.k + slot * D;
      vp[u] = c.v + slot * D;
    }
    // scores
    f32x4 s[NT][2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const KvBytes<KD> kc = kv_bytes<KD>(kp[u] + col * D + g * KD);
#pragma unroll
      for (int t = 0; t < NT; ++t) s[t][u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int x = 0; x < KD / 8; ++x) {
        const f16x8 kf = cat8(kv_half4<FP8>(kc.w[2 * x]), kv_half4<FP8>(kc.w[2 * x + 1]));
#pragma unroll
        for (int t = 0; t < NT; ++t) s[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, q[t][x], s[t][u], 0, 0, 0);
      }
    }
    // a page's value scale above all before it: the sums go into its units
#pragma unroll
    for (int u = 0; u < 2; ++u)
      if (pg[u] >= 0 && vs[u] > vref && vs[u] <= 3.4028235e38f) {
        const float f = vref / vs[u];
        vref = vs[u];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int j = 0; j < VD; ++j) o[t][j] *= f;
      }
    const float inv = vref > 0.f ? 1.f / vref : 0.f;
    const bool masked = t0 < full_lo || t0 + KVT > full_hi || pg[0] < 0 || pg[1] < 0;
    f16x8 pf[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float top = -__builtin_inff();
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float v = s[t][u][e] * (qs[t] * ks[u]);
          if (masked) {
            const int tok = t0 + 16 * u + 4 * g + e;
            if (pg[u] < 0 || tok < lo[t] || tok >= hi[t]) v = -__builtin_inff();
          }
          s[t][u][e] = v;
          top = fmaxf(top, v);
        }
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const float mn = fmaxf(m[t], top);
      const float base = mn == -__builtin_inff() ? 0.f : mn;
      const float f = __builtin_amdgcn_exp2f(m[t] - base);
      m[t] = mn;
      l[t] *= f;
#pragma unroll
      for (int j = 0; j < VD; ++j) o[t][j] *= f;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const float w = vs[u] * inv * KV_P;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float v = s[t][u][e], p = __builtin_amdgcn_exp2f(v - base);
          l[t] += p;
          // a masked token's weight is 0 whatever its page's scale holds
          pf[t][4 * u + e] = static_cast<f16>(v == -__builtin_inff() ? 0.f : p * w);
        }
      }
    }
    // values
    KvBytes<VD> vc[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      vc[x] = kv_bytes<VD>(vp[x >> 2] + (4 * g + (x & 3)) * D + col * VD);
      if (masked && (pg[x >> 2] < 0 || t0 + 16 * (x >> 2) + 4 * g + (x & 3) >= thi)) {
#pragma unroll
        for (int y = 0; y < (VD + 3) / 4; ++y) vc[x].w[y] = 0u;  // no token: its codes may be anything
      }
    }
#pragma unroll
    for (int y = 0; y < (VD + 3) / 4; ++y) {
      // words of four d, eight tokens -> four fragments of eight tokens
      f16x4 t4[8];
#pragma unroll
      for (int x = 0; x < 8; ++x) t4[x] = kv_half4<FP8>(vc[x].w[y]);
#pragma unroll
      for (int z = 0; z < 4; ++z) {
        if (4 * y + z >= VD) break;
        const f16x8 vf = {t4[0][z], t4[1][z], t4[2][z], t4[3][z], t4[4][z], t4[5][z], t4[6][z], t4[7][z]};
#pragma unroll
        for (int t = 0; t < NT; ++t) o[t][4 * y + z] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[t], o[t][4 * y + z], 0, 0, 0);
      }
    }
  }
  if (bad && lane == 0 && c.status != nullptr) atomicMax(c.status, KV_BAD);

  // The waves' parts meet in LDS. Sums of rows: over the four lanes of a column, then the waves.
  __shared__ float wm[KVR_WAVES][NT][16], wl[KVR_WAVES][NT][16];
  __shared__ f32x4 red[KVR_WAVES][4][64];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    l[t] += __shfl_xor(l[t], 16, 64);
    l[t] += __shfl_xor(l[t], 32, 64);
    if (g == 0) {
      wm[wave][t][col] = m[t];
      wl[wave][t][col] = l[t];
    }
  }
  __syncthreads();
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    float top = wm[0][t][col];
#pragma unroll
    for (int w = 1; w < KVR_WAVES; ++w) top = fmaxf(top, wm[w][t][col]);
    const float base = top == -__builtin_inff() ? 0.f : top;
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < KVR_WAVES; ++w) sum += wl[w][t][col] * __builtin_amdgcn_exp2f(wm[w][t][col] - base);
    const float mine = __builtin_amdgcn_exp2f(m[t] - base) * vref;
    const float inv = sum != 0.f ? 1.f / (sum * KV_P) : 0.f;
    const int r = r0 + 16 * t + col;
#pragma unroll
    for (int j0 = 0; j0 < VD; j0 += 4) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j0 + j < VD) red[wave][j][lane] = o[t][j0 + j] * mine;
      __syncthreads();
      // wave w finishes tile j0 + w
      const int j = j0 + wave;
      if (j < VD && r < nrows) {
        f32x4 v = red[0][wave][lane];
#pragma unroll
        for (int w = 1; w < KVR_WAVES; ++w) v += red[w][wave][lane];
        const int64_t at = (static_cast<int64_t>(first + r / G) * a.Hq + h * G + r % G) * D;
#pragma unroll
        for (int e = 0; e < 4; ++e) st_lt(a.o, at + VD * (4 * g + e) + j, v[e] * inv, a.dtype);
      }
      __syncthreads();
    }
  }
}

template <int D, bool FP8>
hipError_t rows_for(const KvAttnArgs& a, hipStream_t st) {
  constexpr int NT = 1;
  const int64_t G = a.Hq / a.c.Hkv, tiles = (a.max_new * G + 16 * NT - 1) / (16 * NT);
  const int64_t grid = tiles * a.c.Hkv * a.c.B;
  if (grid > 0x7FFFFFFF) return hipErrorInvalidValue;
  k_kv8_rows<D, FP8, NT><<<dim3(static_cast<uint32_t>(grid)), 64 * KVR_WAVES, 0, st>>>(a, static_cast<uint32_t>(tiles));
  return hipGetLastError();
}

}  // namespace

int64_t kv8_workspace_bytes(const KvAttnArgs&) { return 0; }

hipError_t launch_kv8_attention(const KvAttnArgs& a, hipStream_t st) {
  if (a.c.B == 0 || a.max_new == 0) return hipSuccess;
  switch (a.c.D * 2 + (a.c.fp8 ? 1 : 0)) {
    case 128: return rows_for<64, false>(a, st);
    case 129: return rows_for<64, true>(a, st);
    case 192: return rows_for<96, false>(a, st);
    case 193: return rows_for<96, true>(a, st);
    case 256: return rows_for<128, false>(a, st);
    case 257: return rows_for<128, true>(a, st);
    case 512: return rows_for<256, false>(a, st);
    case 513: return rows_for<256, true>(a, st);
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
