// Rotary positions: value pairs of each head, turned by position * frequency.
#include "xrmm_decode.h"

namespace xrmm {

namespace {

// Angles are products of 64 bits, taken to a quarter turn around a multiple of one there: position 10^6 at one radian a position
// leaves 10^-10 of a radian, where 32 bits would leave 0.06. Sine and cosine are their Taylor series, in 64 bits up to
// 10^-12, and rounded to float32 once with the magnitude; a token's are computed once for all of its heads. The turn itself is float32
// and rounded once to the storage type.
//
// The bytes bound it, and a few tokens the chain position -> angle -> values: queries and keys of 40 heads of 128 in one call
// take 17 us for 4100 tokens in bfloat16 (5.0 TB/s, a large copy's rate), 63 for 8192 in float32 (5.3), and 5 for a token. A workgroup takes a
// token, so that 96 of them lie on 96 CUs; a thread keeps its piece of a head (V values of one half and their
// partners, or V / 2 neighbouring pairs) and walks over the heads; the next piece is in flight while one is turned, the first
// before the angles are known.
constexpr int ROPE_T = 256;

// (cos, sin) of x = position * frequency, times m.
__device__ __forceinline__ f32x2 turn_of(double x, double m, bool inverse) {
  const double quarters = __builtin_rint(x * 0.63661977236758134308);  // x / (pi / 2)
  double r = __builtin_fma(quarters, -1.57079632679489655800, x);      // pi / 2 in two parts
  r = __builtin_fma(quarters, -6.12323399573676603587e-17, r);
  const double z = r * r;
  double s = 1.0 / 6227020800.0, c = 1.0 / 479001600.0;                // 1 / 13!, 1 / 12!
  s = __builtin_fma(-s, z, 1.0 / 39916800.0);
  c = __builtin_fma(-c, z, 1.0 / 3628800.0);
  s = __builtin_fma(-s, z, 1.0 / 362880.0);
  c = __builtin_fma(-c, z, 1.0 / 40320.0);
  s = __builtin_fma(-s, z, 1.0 / 5040.0);
  c = __builtin_fma(-c, z, 1.0 / 720.0);
  s = __builtin_fma(-s, z, 1.0 / 120.0);
  c = __builtin_fma(-c, z, 1.0 / 24.0);
  s = __builtin_fma(-s, z, 1.0 / 6.0);
  c = __builtin_fma(-c, z, 0.5);
  s = r * __builtin_fma(-s, z, 1.0) * m;
  c = __builtin_fma(-c, z, 1.0) * m;
  const int q = static_cast<int>(quarters - 4.0 * __builtin_floor(quarters * 0.25)) & 3;
  const double cs = q == 0 ? c : q == 1 ? -s : q == 2 ? -c : s, sn = q == 0 ? s : q == 1 ? c : q == 2 ? -s : -c;
  return f32x2{static_cast<float>(cs), static_cast<float>(inverse ? -sn : sn)};
}

template <typename T, int V, bool INTER>
__global__ __launch_bounds__(ROPE_T) void k_rope(RopeArgs a) {
  typedef T vec __attribute__((ext_vector_type(V), aligned(sizeof(T))));  // at any element's address
  extern __shared__ __align__(8) unsigned char smem[];
  f32x2* cs = reinterpret_cast<f32x2*>(smem);  // [R / 2]
  const int tid = threadIdx.x, half = a.R / 2, heads = a.Hq + a.Hk;
  const int64_t row = a.row0 + blockIdx.x;
  const bool moved = a.q != a.oq || (a.Hk > 0 && a.k != a.ok);  // else what passes is in place already

  // this thread's piece of a head, and the first of the heads that it visits
  const int turns = (INTER ? a.R : half) / V, pieces = turns + (moved ? (a.D - a.R + V - 1) / V : 0);
  const int lanes = pieces < ROPE_T ? ROPE_T / pieces : 1;     // threads at one piece
  const int first = pieces < ROPE_T ? tid / pieces : 0;
  struct Piece {
    vec x, y;
  };
  auto src = [&](int h) {
    const bool isk = h >= a.Hq;
    return static_cast<const T*>(isk ? a.k : a.q) + row * (isk ? a.k_stride : a.q_stride) + static_cast<int64_t>(isk ? h - a.Hq : h) * a.D;
  };
  auto dst = [&](int h) {
    const bool isk = h >= a.Hq;
    return static_cast<T*>(isk ? a.ok : a.oq) + row * (isk ? a.ok_stride : a.oq_stride) + static_cast<int64_t>(isk ? h - a.Hq : h) * a.D;
  };
  auto load = [&](int h, int c) {
    Piece p{};
    const T* s = src(h);
    if (c < turns) {
      p.x = *reinterpret_cast<const vec*>(s + c * V);
      if constexpr (!INTER) p.y = *reinterpret_cast<const vec*>(s + half + c * V);
    } else {
      const int at = a.R + (c - turns) * V;
      if (at + V <= a.D) p.x = *reinterpret_cast<const vec*>(s + at);
      else
#pragma unroll
        for (int e = 0; e < V; ++e) p.x[e] = at + e < a.D ? s[at + e] : T(0);
    }
    return p;
  };
  auto finish = [&](const Piece& p, int h, int c) {
    T* d = dst(h);
    if (c >= turns) {
      const int at = a.R + (c - turns) * V;
      if (at + V <= a.D) *reinterpret_cast<vec*>(d + at) = p.x;
      else
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (at + e < a.D) d[at + e] = p.x[e];
      return;
    }
    if constexpr (INTER) {
      const f32x2* w = cs + c * (V / 2);
      vec r;
#pragma unroll
      for (int e = 0; e < V; e += 2) {
        const f32x2 m = w[e / 2];
        const float x = static_cast<float>(p.x[e]), y = static_cast<float>(p.x[e + 1]);
        r[e] = static_cast<T>(__builtin_fmaf(x, m[0], -(y * m[1])));
        r[e + 1] = static_cast<T>(__builtin_fmaf(y, m[0], x * m[1]));
      }
      *reinterpret_cast<vec*>(d + c * V) = r;
    } else {
      const f32x2* w = cs + c * V;
      vec r0, r1;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const f32x2 m = w[e];
        const float x = static_cast<float>(p.x[e]), y = static_cast<float>(p.y[e]);
        r0[e] = static_cast<T>(__builtin_fmaf(x, m[0], -(y * m[1])));
        r1[e] = static_cast<T>(__builtin_fmaf(y, m[0], x * m[1]));
      }
      *reinterpret_cast<vec*>(d + c * V) = r0;
      *reinterpret_cast<vec*>(d + half + c * V) = r1;
    }
  };
  const int c0 = pieces < ROPE_T ? tid - first * pieces : tid;
  Piece cur{};
  const bool any = first < lanes && first < heads && c0 < pieces;
  if (any) cur = load(first, c0);

  double where;
  if (a.positions != nullptr) {
    where = a.wide_positions ? static_cast<double>(static_cast<const int64_t*>(a.positions)[row]) : static_cast<double>(static_cast<const int32_t*>(a.positions)[row]);
  } else if (a.starts == nullptr) {
    const int at = static_cast<int>(row), b = at / a.each;
    where = static_cast<double>(static_cast<int64_t>(a.lengths[b]) - a.each + (at - b * a.each));
  } else {
    // its sequence is the number of sequences that end at or before it, counted by each wave
    const int lane = tid & 63;
    int b = 0;
    for (int s = lane; s - lane < a.B; s += 64) b += __popcll(__ballot(s < a.B && a.starts[s < a.B ? s + 1 : 0] <= row));
    if (b >= a.B || a.starts[b] > row || a.starts[b + 1] <= row) return;  // no sequence's: left as it is
    where = static_cast<double>(static_cast<int64_t>(a.lengths[b]) - (static_cast<int64_t>(a.starts[b + 1]) - row));
  }
  for (int i = tid; i < half; i += ROPE_T) cs[i] = turn_of(where * a.freq[i], a.magnitude, a.inverse);
  __syncthreads();
  if (!any) return;
#pragma unroll 1
  for (int c = c0; c < pieces; c += ROPE_T) {  // once, unless a head has more pieces than threads
    int h = first;
    if (c != c0) cur = load(h, c);
#pragma unroll 1
    while (true) {
      const int next = h + lanes;
      Piece nxt{};
      if (next < heads) nxt = load(next, c);
      finish(cur, h, c);
      if (next >= heads) break;
      cur = nxt;
      h = next;
    }
  }
}

template <typename T, int V>
hipError_t rope_layout(const RopeArgs& a, hipStream_t st) {
  const size_t lds = static_cast<size_t>(a.R / 2) * sizeof(f32x2);
  RopeArgs x = a;
  for (; x.row0 < a.rows; x.row0 += kLaunchThreads / ROPE_T) {
    const int64_t left = a.rows - x.row0;
    const dim3 grid(static_cast<uint32_t>(left < kLaunchThreads / ROPE_T ? left : kLaunchThreads / ROPE_T));
    if (!a.interleaved) k_rope<T, V, false><<<grid, ROPE_T, lds, st>>>(x);
    else if constexpr (V > 1) k_rope<T, V, true><<<grid, ROPE_T, lds, st>>>(x);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <typename T>
hipError_t rope_type(const RopeArgs& a, hipStream_t st) {
  int v = 16 / static_cast<int>(sizeof(T));
  const int of = a.interleaved ? a.R : a.R / 2;
  while (of % v != 0) v /= 2;
  switch (v) {
    case 8:
      if constexpr (sizeof(T) == 2) return rope_layout<T, 8>(a, st);
      return hipErrorInvalidValue;
    case 4: return rope_layout<T, 4>(a, st);
    case 2: return rope_layout<T, 2>(a, st);
    default: return rope_layout<T, 1>(a, st);
  }
}

}  // namespace

hipError_t launch_rope(const RopeArgs& a, hipStream_t st) {
  if (a.rows == 0 || a.Hq + a.Hk == 0) return hipSuccess;
  switch (a.dtype) {
    case LT_F32: return rope_type<float>(a, st);
    case LT_F16: return rope_type<f16>(a, st);
    default: return rope_type<bf16>(a, st);
  }
}

}  // namespace xrmm
