// The draw of a token for each row of logits, by a given number.
#include "xrmm_decode.h"

namespace xrmm {

namespace {

// A logit x has the weight exp((x - max) / temperature), held as an integer in units of 2^-F of the largest: sums of integers have no
// order, so whatever adds them (lanes, waves, workgroups, atomics) a call gives one result, and borders are compared exactly. F = 62 -
// log2(vocabulary) keeps a row's sum below 2^63; at 2^17 tokens a weight is off by 2^-46 of the largest, below what a float32 u
// tells apart, and weights below 2^-46 of it (31 nats) are 0: such tokens are not drawn.
//
// Order: by logit, of equal ones (0 and -0 are) the lower index first: the composite (ordered bits of x, ~index), unique in a row. top_k, top_p
// and min_p each keep a prefix of that order. A row's thresholds come from a histogram over the distance to the maximum (64 bins a nat): the bins
// in which they can fall give a short list, and among its tokens each is found digit by digit of the composite.
constexpr int SB = 2048;      // bins
constexpr float SB_NAT = 64.f;  // bins a nat
constexpr int SLIST = 2048;   // tokens of the list; where more lie in the bins, the row itself is read in its place
constexpr int ST = 1024;      // threads of a row
constexpr int SW = ST / 64;

struct Draw {       // a row's settings
  double c;         // log2(e) / temperature
  float s;          // bins a unit of logit
  double top_p, least;  // least: in units of weights, or 0
  int k;            // 0: all
  bool greedy, p;
};

__device__ __forceinline__ Draw draw_of(const SampleArgs& a, int64_t row, int F) {
  Draw d;
  const double t = a.temperature ? static_cast<double>(a.temperature[row]) : a.temperature1;
  const double p = a.top_p ? static_cast<double>(a.top_p[row]) : a.top_p1;
  const double m = a.min_p ? static_cast<double>(a.min_p[row]) : a.min_p1;
  const int k = a.top_k ? a.top_k[row] : a.top_k1;
  d.greedy = !(t > 0.0);
  d.c = 1.44269504088896340736 / (d.greedy ? 1.0 : t);
  d.s = SB_NAT / static_cast<float>(d.greedy ? 1.0 : t);
  d.k = k > 0 && k < a.V ? k : 0;
  d.p = p < 1.0;
  d.top_p = p > 0.0 ? p : 0.0;
  d.least = m > 0.0 ? __builtin_ldexp(m < 1.0 ? m : 1.0, F) : 0.0;
  return d;
}

__device__ __forceinline__ uint32_t okey(float x) {  // ordered bits; -0 as 0
  const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.f);
  return u ^ (static_cast<int32_t>(u) < 0 ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float of_okey(uint32_t k) {
  return __builtin_bit_cast(float, k ^ (static_cast<int32_t>(k) < 0 ? 0x80000000u : 0xFFFFFFFFu));
}
__device__ __forceinline__ uint64_t composite(float x, uint32_t i) { return static_cast<uint64_t>(okey(x)) << 32 | (0xFFFFFFFFu - i); }

// 2^y in units of 2^-F, y <= 0: 2^n 2^f by the Taylor series of 2^f, |f| <= 1/2, whose rest after f^11 is 6 10^-15.
__device__ __forceinline__ double exp2_units(double y, int F) {
  const double n = __builtin_rint(y), r = (y - n) * 0.69314718055994530942;
  double p = 1.0 / 39916800.0;
  p = __builtin_fma(p, r, 1.0 / 3628800.0);
  p = __builtin_fma(p, r, 1.0 / 362880.0);
  p = __builtin_fma(p, r, 1.0 / 40320.0);
  p = __builtin_fma(p, r, 1.0 / 5040.0);
  p = __builtin_fma(p, r, 1.0 / 720.0);
  p = __builtin_fma(p, r, 1.0 / 120.0);
  p = __builtin_fma(p, r, 1.0 / 24.0);
  p = __builtin_fma(p, r, 1.0 / 6.0);
  p = __builtin_fma(p, r, 0.5);
  p = __builtin_fma(p, r, 1.0);
  p = __builtin_fma(p, r, 1.0);
  return __builtin_ldexp(p, static_cast<int>(n) + F);
}

struct Weigher {
  float top;   // the row's largest logit
  double topd, c;
  int F;
  __device__ __forceinline__ double units(float x) const {  // not yet rounded
    const double y = (static_cast<double>(x) - topd) * c;
    // a NaN is infinity less itself or times 0; the test keeps it and what rounds to 0 away
    return x == top ? __builtin_ldexp(1.0, F) : y > -static_cast<double>(F + 2) ? exp2_units(y, F) : 0.0;
  }
  __device__ __forceinline__ static uint64_t whole(double u) {  // to nearest; u <= 2^51
    return __builtin_bit_cast(uint64_t, u + 4503599627370496.0) & 0xFFFFFFFFFFFFFull;
  }
};

__device__ __forceinline__ int bin_of(float x, float top, float s) {
  return x == top ? 0 : static_cast<int>(fminf((top - x) * s, static_cast<float>(SB - 1)));
}

__device__ __forceinline__ uint64_t shfl_up64(uint64_t v, int o) {
  return static_cast<uint64_t>(static_cast<uint32_t>(__shfl_up(static_cast<int>(v >> 32), o, 64))) << 32 |
         static_cast<uint32_t>(__shfl_up(static_cast<int>(v), o, 64));
}
__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int o) {
  return static_cast<uint64_t>(static_cast<uint32_t>(__shfl_xor(static_cast<int>(v >> 32), o, 64))) << 32 |
         static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), o, 64));
}
__device__ __forceinline__ uint64_t wave_sum64(uint64_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += shfl_xor64(v, o);
  return v;
}
__device__ __forceinline__ uint64_t wave_scan64(uint64_t v, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint64_t u = shfl_up64(v, o);
    if (lane >= o) v += u;
  }
  return v;
}

// The number u's place in a sum s, rounded down: running sums of whole numbers pass u s where they pass it.
__device__ __forceinline__ uint64_t place_of(double u, uint64_t s) {
  const uint64_t q = u >= 1.0 ? ~0ull : u > 0.0 ? static_cast<uint64_t>(__builtin_ldexp(u, 64)) : 0ull;
  return __umul64hi(q, s);
}
// What top_p asks of a sum, one at least: a product of 64-bit floats, so that 0.9 of a hundred equal weights is ninety.
__device__ __forceinline__ uint64_t share_of(double p, uint64_t s) {
  const uint64_t n = static_cast<uint64_t>(__builtin_ceil(p * static_cast<double>(s)));
  return n < 1 ? 1 : n > s ? s : n;
}

template <typename T>
struct RowOf {
  static constexpr int VEC = 16 / sizeof(T);
  typedef T vec __attribute__((ext_vector_type(VEC), aligned(sizeof(T))));
  const T* x;
  // VEC values from i on; -infinity past `end` and for NaN
  __device__ __forceinline__ void load(float (&f)[VEC], int64_t i, int64_t end) const {
    if (i + VEC <= end) {
      const vec v = *reinterpret_cast<const vec*>(x + i);
#pragma unroll
      for (int e = 0; e < VEC; ++e) f[e] = static_cast<float>(v[e]);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) f[e] = i + e < end ? static_cast<float>(x[i + e]) : -__builtin_inff();
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) f[e] = f[e] == f[e] ? f[e] : -__builtin_inff();
  }
};

struct SampleLds {
  uint64_t mass[SB];
  uint32_t count[SB];
  uint64_t list[SLIST];
  uint64_t digits[256];
  uint64_t part[SW];
  uint64_t a64, b64;
  uint32_t n, a32, b32;
};

// The first bin whose running sum reaches `need` (its index to s.a32, the sum before it to s.a64; SB where none does),
// of masses or of counts. All threads.
template <bool MASS>
__device__ __forceinline__ void find_bin(SampleLds& s, uint64_t need) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  constexpr int N = SB / ST;
  uint64_t v[N], sum = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = MASS ? s.mass[tid * N + i] : s.count[tid * N + i];
    sum += v[i];
  }
  const uint64_t inc = wave_scan64(sum, lane);
  __syncthreads();
  if (lane == 63) s.part[wave] = inc;
  if (tid == 0) s.a32 = SB;
  __syncthreads();
  uint64_t before = inc - sum;
  for (int w = 0; w < wave; ++w) before += s.part[w];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (before < need && before + v[i] >= need) {
      s.a32 = tid * N + i;
      s.a64 = before;
    }
    before += v[i];
  }
  __syncthreads();
}

// The composite at which a running sum over the candidates, in descending order, reaches `need` (>= 1): of their weights, or of their
// number. `each(f)` calls f(composite, weight) for the candidates of each thread. 0 where all do not reach it; *rest: what is
// missing to `need` before the found one.
template <bool MASS, typename E>
__device__ __forceinline__ uint64_t find_composite(SampleLds& s, uint64_t need, E&& each) {
  const int tid = threadIdx.x, lane = tid & 63;
  uint64_t prefix = 0;
#pragma unroll 1
  for (int shift = 56; shift >= 0; shift -= 8) {
    __syncthreads();
    if (tid < 256) s.digits[tid] = 0;
    if (tid == 0) s.b32 = 256;
    __syncthreads();
    each([&](uint64_t comp, uint64_t w) {
      if (shift == 56 || comp >> (shift + 8) == prefix)
        atomicAdd(reinterpret_cast<unsigned long long*>(&s.digits[comp >> shift & 255]), static_cast<unsigned long long>(MASS ? w : 1));
    });
    __syncthreads();
    if (tid < 64) {  // digits 255 - 4 lane .. - 3, descending
      uint64_t v[4], sum = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) sum += v[i] = s.digits[255 - 4 * lane - i];
      uint64_t before = wave_scan64(sum, lane) - sum;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (before < need && before + v[i] >= need) {
          s.b32 = 255 - 4 * lane - i;
          s.b64 = need - before;
        }
        before += v[i];
      }
    }
    __syncthreads();
    const uint32_t digit = s.b32;
    if (digit == 256) return 0;
    prefix = prefix << 8 | digit;
    need = s.b64;
  }
  return prefix;
}

// One workgroup a row, all of it.
template <typename T>
__global__ __launch_bounds__(ST) void k_sample_row(SampleArgs a, int F) {
  typedef RowOf<T> R;
  constexpr int VEC = R::VEC;
  __shared__ SampleLds s;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x;
  const R r{static_cast<const T*>(a.x) + row * a.stride};
  const Draw d = draw_of(a, row, F);
  const int V = a.V;
  const float ninf = -__builtin_inff();

  // the largest logit, of the lowest index
  uint64_t best = 0;
  for (int i = tid * VEC; i < V; i += ST * VEC) {
    float f[VEC];
    r.load(f, i, V);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const uint64_t c = f[e] > ninf ? composite(f[e], i + e) : 0ull;
      best = c > best ? c : best;
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint64_t c = shfl_xor64(best, o);
    best = c > best ? c : best;
  }
  if (lane == 0) s.part[wave] = best;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < SW; ++w) best = s.part[w] > best ? s.part[w] : best;
  if (best == 0 || d.greedy) {
    if (tid == 0) {
      a.tokens[row] = best == 0 ? -1 : static_cast<int32_t>(0xFFFFFFFFu - static_cast<uint32_t>(best));
      a.shares[row] = best == 0 ? ninf : 0.f;
    }
    return;
  }
  const float top = of_okey(static_cast<uint32_t>(best >> 32));
  const Weigher weigh{top, static_cast<double>(top), d.c, F};

  uint64_t threshold = 0;  // composites from here on are kept
  if (d.k > 0 || d.p) {
    for (int i = tid; i < SB; i += ST) {
      s.mass[i] = 0;
      s.count[i] = 0;
    }
    if (tid == 0) s.n = 0;
    __syncthreads();
    for (int i = tid * VEC; i < V; i += ST * VEC) {
      float f[VEC];
      r.load(f, i, V);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        if (!(f[e] > ninf)) continue;
        const int b = bin_of(f[e], top, d.s);
        if (d.k > 0) atomicAdd(&s.count[b], 1u);
        if (d.p) atomicAdd(reinterpret_cast<unsigned long long*>(&s.mass[b]), static_cast<unsigned long long>(Weigher::whole(weigh.units(f[e]))));
      }
    }
    __syncthreads();
    // bins lo .. hi hold the thresholds; `above` tokens and `held` weight lie in those before lo
    int lo = 0, hi = SB - 1;
    uint64_t held_k = 0;
    if (d.k > 0) {
      find_bin<false>(s, static_cast<uint64_t>(d.k));
      hi = s.a32 < SB ? static_cast<int>(s.a32) : SB - 1;
      lo = hi;
    }
    if (d.p) {
      uint64_t all = 0;
      if (d.k > 0) {  // the weight before bin hi: top_p of it, at least, is wanted
        for (int i = lane; i < hi; i += 64) all += s.mass[i];
      } else {
        for (int i = lane; i < SB; i += 64) all += s.mass[i];
      }
      held_k = wave_sum64(all);
      find_bin<true>(s, share_of(d.top_p, held_k));
      const int b = s.a32 < SB ? static_cast<int>(s.a32) : SB - 1;
      lo = d.k > 0 && b > hi ? hi : b;
      if (d.k == 0) hi = lo;
    }
    uint64_t above = 0, held = 0;
    for (int i = lane; i < lo; i += 64) {
      above += s.count[i];
      held += s.mass[i];
    }
    above = wave_sum64(above);
    held = wave_sum64(held);
    // the list
    for (int i = tid * VEC; i < V; i += ST * VEC) {
      float f[VEC];
      r.load(f, i, V);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        if (!(f[e] > ninf)) continue;
        const int b = bin_of(f[e], top, d.s);
        if (b < lo || b > hi) continue;
        const uint32_t at = atomicAdd(&s.n, 1u);
        if (at < SLIST) s.list[at] = composite(f[e], i + e);
      }
    }
    __syncthreads();
    const uint32_t n = s.n;
    auto each = [&](auto&& f) {
      if (n <= SLIST) {
        for (uint32_t i = tid; i < n; i += ST) {
          const uint64_t c = s.list[i];
          f(c, Weigher::whole(weigh.units(of_okey(static_cast<uint32_t>(c >> 32)))));
        }
      } else {
        for (int i = tid * VEC; i < V; i += ST * VEC) {
          float x[VEC];
          r.load(x, i, V);
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            if (!(x[e] > ninf)) continue;
            const int b = bin_of(x[e], top, d.s);
            if (b >= lo && b <= hi) f(composite(x[e], i + e), Weigher::whole(weigh.units(x[e])));
          }
        }
      }
    };
    if (d.k > 0) threshold = find_composite<false>(s, static_cast<uint64_t>(d.k) - above, each);
    if (d.p) {
      uint64_t all = held_k;
      if (d.k > 0) {  // top_k's weight: what is held before the list, and the list's part of it
        __syncthreads();
        if (tid == 0) s.a64 = 0;
        __syncthreads();
        uint64_t mine = 0;
        each([&](uint64_t c, uint64_t w) { mine += c >= threshold ? w : 0ull; });
        mine = wave_sum64(mine);
        if (lane == 0) atomicAdd(reinterpret_cast<unsigned long long*>(&s.a64), static_cast<unsigned long long>(mine));
        __syncthreads();
        all = held + s.a64;
      }
      const uint64_t need = share_of(d.top_p, all);
      const uint64_t c = find_composite<true>(s, need > held ? need - held : 1, each);
      threshold = c > threshold ? c : threshold;
    }
  }

  // the draw: the running sum of the kept weights by index, narrowed to a wave's part at a time
  int begin = 0, end = V;
  uint64_t total = 0, target = 0;
  auto kept = [&](float x, uint32_t i) {
    if (!(x > ninf) || composite(x, i) < threshold) return uint64_t{0};
    const double u = weigh.units(x);
    return u >= d.least ? Weigher::whole(u) : uint64_t{0};
  };
  for (bool firsts = true;; firsts = false) {
    const int per = ((end - begin + SW - 1) / SW + 64 * VEC - 1) / (64 * VEC) * (64 * VEC);
    const int64_t from = begin + static_cast<int64_t>(wave) * per, to = from + per < end ? from + per : end;
    uint64_t mine = 0;
    for (int64_t i = from + lane * VEC; i < to; i += 64 * VEC) {
      float f[VEC];
      r.load(f, i, to);
#pragma unroll
      for (int e = 0; e < VEC; ++e) mine += kept(f[e], static_cast<uint32_t>(i + e));
    }
    mine = wave_sum64(mine);
    __syncthreads();
    if (lane == 0) s.part[wave] = mine;
    __syncthreads();
    uint64_t all = 0;
#pragma unroll
    for (int w = 0; w < SW; ++w) all += s.part[w];
    if (firsts) {
      total = all;
      target = place_of(static_cast<double>(a.u[row]), total);
    }
    int w = 0;
    uint64_t before = 0;
    while (w < SW - 1 && before + s.part[w] <= target) before += s.part[w++];
    target -= before;
    begin = begin + w * per;
    end = begin + per < end ? begin + per : end;
    if (per == 64 * VEC) break;
  }
  if (wave == 0) {
    float f[VEC];
    r.load(f, begin + lane * VEC, end);
    uint64_t k[VEC], mine = 0;
#pragma unroll
    for (int e = 0; e < VEC; ++e) mine += k[e] = kept(f[e], static_cast<uint32_t>(begin + lane * VEC + e));
    const uint64_t inc = wave_scan64(mine, lane);
    uint64_t before = inc - mine;
    if (before <= target && target < inc) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        if (before <= target && target < before + k[e]) {
          a.tokens[row] = begin + lane * VEC + e;
          a.shares[row] = static_cast<float>(log(weigh.units(f[e]) / static_cast<double>(total)));
        }
        before += k[e];
      }
    }
  }
}

template <typename T>
hipError_t sample_type(const SampleArgs& a, int F, hipStream_t st) {
  k_sample_row<T><<<dim3(static_cast<uint32_t>(a.rows)), ST, 0, st>>>(a, F);
  return hipGetLastError();
}

}  // namespace

int64_t sample_workspace_bytes(int64_t rows, int64_t V) { return 0; }

hipError_t launch_sample(const SampleArgs& a, hipStream_t st) {
  if (a.rows == 0) return hipSuccess;
  int log2v = 0;
  while ((int64_t{1} << log2v) < a.V) ++log2v;
  const int F = 62 - log2v < 51 ? 62 - log2v : 51;
  switch (a.dtype) {
    case LT_F32: return sample_type<float>(a, F, st);
    case LT_F16: return sample_type<f16>(a, F, st);
    default: return sample_type<bf16>(a, F, st);
  }
}

}  // namespace xrmm
