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
// and min_p each keep a prefix of that order. A row is read four times:
//   its largest logit
//   a histogram over the distance to it (64 bins a nat), which tells the bins in which each threshold lies: of counts for top_k, of
//     weights by float32's exponential for top_p, whose error is bounded and widens the bins
//   those bins' tokens into a list, and the exact weight of all before and behind them
//   the part in which the number falls.
// For top_k up to a quarter of the threads, the threads' own largest logits are counted in place of all: no fewer than top_k tokens reach
// the top_k-th of them, and hardly more, so the list holds all that may be kept.
//
// Vector instructions bound rows with top_p: 116 a token (256 rows of 50001), of which the 64-bit exponential is about 20; the others clean
// the logits, take their bins again in each pass, and choose and add whole weights.
//
// The histogram's bound on its error is two units of 2^-30 a token, so top_p's bins grow with the vocabulary. From 50000 logits on, the more the flatter,
// most rows with top_p of 0.95 or more list over SNEAR tokens (one row of 152000 24 -> 36 to 50 us), and from about 260000 some list over SLIST, with which
// a workgroup reads the row itself about ten times, a logit a thread (one row of 260000 with top_p 0.99 at temperature 1 2550 us for 44 at 1.5, 49 rows 4040 for
// 105): right, and slower than torch's elementary operations (310, 2960).
constexpr int SB = 2048;      // bins
constexpr float SB_NAT = 64.f;  // bins a nat
constexpr int SLIST = 2048;   // tokens of the list; where more lie in the bins, the row itself is read in its place
constexpr int SNEAR = 256;    // of a list this short, each token counts those before it; of a longer one digits are counted
constexpr int ST = 1024;      // threads of a row that one workgroup takes
constexpr int SP = 256;       // threads of a part of a row
constexpr int SAPPROX = 30;   // the histogram's weights are in units of 2^-30

struct Draw {       // a row's settings
  double c;         // log2(e) / temperature
  float s;          // bins a two of logits
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
  // 10^-30 to 10^30: the factors stay finite, and the largest float32, which stands for infinity, far from other logits
  const double heat = d.greedy ? 1.0 : t < 1e-30 ? 1e-30 : t < 1e30 ? t : 1e30;
  d.c = 1.44269504088896340736 / heat;
  d.s = 2.f * SB_NAT / static_cast<float>(heat);
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

// p r + c with c in scalar registers: the compiler's own choice copies c to vector registers for each product.
__device__ __forceinline__ double fma_s(double p, double r, double c) {
  double o;
  asm("v_fma_f64 %0, %1, %2, %3" : "=v"(o) : "v"(p), "v"(r), "s"(c));
  return o;
}

// What a logit weighs, in units of 2^-F of the largest, not yet rounded: 2^n 2^r for y = n + r, |r| <= 1/2, by the Taylor series of 2^r
// up to r^11, whose rest is 6 10^-15. Without branches, roundings to whole numbers by addition and powers of two by the exponent's bits.
// Below 2^-1000, -infinity among them, is 2^-1000, which rounds to none.
struct Weigher {
  float top;   // the row's largest logit
  double topd, c;
  int F;
  __device__ __forceinline__ Weigher(float t, double factor, int f) : top(t), topd(t), c(factor), F(f) {}
  __device__ __forceinline__ double units(float x) const {
    const double y = __builtin_fmax((static_cast<double>(x) - topd) * c, -1000.0);
    const double whole = y + 6755399441055744.0, r = y - (whole - 6755399441055744.0);  // 1.5 2^52: its low bits are the whole number
    // ln(2)^k / k!
    double p = 4.44553827187081e-10;
    p = fma_s(p, r, 7.054911620801121e-09);
    p = fma_s(p, r, 1.0178086009239696e-07);
    p = fma_s(p, r, 1.3215486790144305e-06);
    p = fma_s(p, r, 1.5252733804059838e-05);
    p = fma_s(p, r, 0.00015403530393381606);
    p = fma_s(p, r, 0.0013333558146428441);
    p = fma_s(p, r, 0.009618129107628477);
    p = fma_s(p, r, 0.055504108664821576);
    p = fma_s(p, r, 0.2402265069591007);
    p = fma_s(p, r, 0.6931471805599453);
    p = __builtin_fma(p, r, 1.0);
    const u32x2 bits = __builtin_bit_cast(u32x2, p);
    return __builtin_bit_cast(double, u32x2{bits[0], bits[1] + ((__builtin_bit_cast(u32x2, whole)[0] + static_cast<uint32_t>(F)) << 20)});
  }
  __device__ __forceinline__ static uint64_t whole(double u) {  // to nearest; u <= 2^51
    return __builtin_bit_cast(uint64_t, u + 4503599627370496.0) & 0xFFFFFFFFFFFFFull;
  }
};

// Half of top - x: no finite logits' overflows.
__device__ __forceinline__ float half_below(float x, float top) { return __builtin_fmaf(x, -0.5f, 0.5f * top); }

__device__ __forceinline__ int bin_of(float x, float top, float s) {
  return static_cast<int>(__builtin_amdgcn_fmed3f(half_below(x, top) * s, 0.f, static_cast<float>(SB - 1)));
}

// A lane's value of another lane by the data path of its row (CTRL), 0 where there is none.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t dpp64(uint64_t v) {
  const uint32_t lo = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xF, false));
  const uint32_t hi = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v >> 32), CTRL, ROWS, 0xF, false));
  return static_cast<uint64_t>(hi) << 32 | lo;
}
__device__ __forceinline__ uint64_t last_lane(uint64_t v) {
  return static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v >> 32), 63))) << 32 |
         static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), 63));
}
__device__ __forceinline__ uint64_t wave_scan64(uint64_t v) {  // inclusive
  v += dpp64<0x111, 0xF>(v);  // from 1, 2, 4 and 8 lanes before, in a row of 16
  v += dpp64<0x112, 0xF>(v);
  v += dpp64<0x114, 0xF>(v);
  v += dpp64<0x118, 0xF>(v);
  v += dpp64<0x142, 0xA>(v);  // the row's last lane to the next row
  return v + dpp64<0x143, 0xC>(v);  // lane 31 to the upper half
}
__device__ __forceinline__ uint64_t wave_sum64(uint64_t v) { return last_lane(wave_scan64(v)); }
__device__ __forceinline__ uint64_t wave_max64(uint64_t v) {
  auto with = [&](uint64_t u) { v = u > v ? u : v; };
  with(dpp64<0x111, 0xF>(v));
  with(dpp64<0x112, 0xF>(v));
  with(dpp64<0x114, 0xF>(v));
  with(dpp64<0x118, 0xF>(v));
  with(dpp64<0x142, 0xA>(v));
  with(dpp64<0x143, 0xC>(v));
  return last_lane(v);
}
__device__ __forceinline__ uint64_t row_sum64(uint64_t v) {  // of 16 lanes, in the last of them
  v += dpp64<0x111, 0xF>(v);
  v += dpp64<0x112, 0xF>(v);
  v += dpp64<0x114, 0xF>(v);
  return v + dpp64<0x118, 0xF>(v);
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

template <typename T, int N>
struct RowOf {
  static constexpr int VEC = N;
  typedef T vec __attribute__((ext_vector_type(VEC), aligned(sizeof(T))));
  const T* x;
  // NaN is -infinity, infinity the largest float32
  __device__ __forceinline__ static float value(T v) {
    const float x = static_cast<float>(v);
    return x == x ? fminf(x, 3.4028234663852886e38f) : -__builtin_inff();
  }
  // f(VEC values, index of the first) for `step` threads' vectors of from .. to - 1, this thread the `first` of them; AHEAD loads in flight.
  // The last vector ends with the stretch: what it repeats is -infinity. A row has VEC logits at least.
  template <int AHEAD, typename F>
  __device__ __forceinline__ void each(int from, int to, int first, int step, F&& f) const {
    const int stride = step * VEC, last = to - VEC;
    int i = from + first * VEC;
    vec v[AHEAD];
    auto load = [&](int at) {
      at = at < last ? at : last;
      return *reinterpret_cast<const vec*>(x + (at > 0 ? at : 0));
    };
#pragma unroll
    for (int n = 0; n < AHEAD; ++n) v[n] = load(i + n * stride);
#pragma unroll 1
    while (i < to) {
      const vec now = v[0];
#pragma unroll
      for (int n = 0; n + 1 < AHEAD; ++n) v[n] = v[n + 1];
      v[AHEAD - 1] = load(i + AHEAD * stride);
      float a[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) a[e] = value(now[e]);
      const int at = i < last ? i : last;
      if (__builtin_expect(at != i, 0)) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) a[e] = at + e >= i ? a[e] : -__builtin_inff();
      }
      f(a, at);
      i += stride;
    }
  }
  // f(logit, index), one by one in a short loop: for rows that list more than SLIST tokens
  template <typename F>
  __device__ __forceinline__ void slowly(int to, int first, int step, F&& f) const {
#pragma unroll 1
    for (int i = first; i < to; i += step) f(value(x[i]), i);
  }
};

struct HistLds {
  uint64_t mass[SB];
  uint32_t count[SB];
};

struct ListLds {
  uint64_t list[SLIST];    // composites
  uint64_t digits[256];    // also the weights of a short list
  uint64_t weight[256];    // of the row's parts
  uint64_t before[SNEAR];
  uint32_t kind[SNEAR];
};

struct BlockLds {
  uint64_t part[16];
  uint64_t a64, b64;
  uint32_t n, a32, b32;
  int last;
};

// Bins that decide: top_k's threshold lies in klo .. khi, with `above` tokens before klo; top_p's in plo .. phi. Both ranges are listed; tokens
// before `sure` are kept by both.
struct Cut {
  int klo, khi, plo, phi, sure;
  uint32_t above;
  __device__ __forceinline__ bool listed(int b) const { return (b >= klo && b <= khi) || (b >= plo && b <= phi); }
};

__device__ __forceinline__ bool few(const Draw& d, int threads) { return d.k > 0 && d.k <= threads / 4; }

// The sum of v over the workgroup, in all threads.
template <int NT>
__device__ __forceinline__ uint64_t block_sum64(BlockLds& s, uint64_t v) {
  const int tid = threadIdx.x;
  v = wave_sum64(v);
  __syncthreads();
  if ((tid & 63) == 0) s.part[tid >> 6] = v;
  __syncthreads();
  uint64_t all = 0;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) all += s.part[w];
  return all;
}

// The first bin whose running sum reaches `need`, of masses or of counts, and the sum before it; SB where none does. All threads.
template <bool MASS, int NT>
__device__ __forceinline__ int find_bin(BlockLds& s, const HistLds& hist, uint64_t need, uint64_t* before_it) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  constexpr int N = SB / NT;
  uint64_t v[N], sum = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = MASS ? hist.mass[tid * N + i] : hist.count[tid * N + i];
    sum += v[i];
  }
  const uint64_t inc = wave_scan64(sum);
  __syncthreads();
  if (lane == 63) s.part[wave] = inc;
  if (tid == 0) {
    s.a32 = SB;
    s.a64 = 0;
  }
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
  *before_it = s.a64;
  return static_cast<int>(s.a32);
}

// From the histogram of a row with top_k or top_p. All threads.
template <int NT>
__device__ __forceinline__ Cut cut_of(BlockLds& s, const HistLds& hist, const Draw& d, int V, int threads) {
  const int tid = threadIdx.x;
  Cut c{0, -1, 0, -1, 0, 0};
  uint64_t before;
  if (d.k > 0) {
    const int b = find_bin<false, NT>(s, hist, static_cast<uint64_t>(d.k), &before);
    if (few(d, threads)) {
      c.khi = b < SB ? b : SB - 1;
      c.phi = d.p ? c.khi : -1;
      return c;
    }
    if (b == SB) {  // fewer tokens than top_k: all are kept
      uint64_t n = 0;
      for (int i = tid; i < SB - 1; i += NT) n += hist.count[i];
      before = block_sum64<NT>(s, n);
    }
    c.klo = c.khi = c.sure = b < SB ? b : SB - 1;
    c.above = static_cast<uint32_t>(before);
  }
  if (d.p) {
    // top_k's weight is from that before its bin to that with it. A bin's weights are off by 2^-17 of themselves (float32's exponential,
    // of arguments up to 48) and half a unit each.
    const int end = d.k > 0 ? c.klo : SB;
    uint64_t m = 0;
    for (int i = tid; i < end; i += NT) m += hist.mass[i];
    m = block_sum64<NT>(s, m);
    const double least = d.top_p * static_cast<double>(m), most = d.top_p * static_cast<double>(m + (d.k > 0 ? hist.mass[c.klo] : 0));
    const double off = static_cast<double>(V) + 1.0;
    const double lo = least * (1.0 - 0x1p-16) - 2.0 * off, hi = most * (1.0 + 0x1p-16) + 2.0 * off;
    int l = 0, h = 0;
#pragma unroll 1
    for (int i = 0; i < 2; ++i) {
      l = h;
      h = find_bin<true, NT>(s, hist, i != 0 ? static_cast<uint64_t>(hi) + 1 : lo < 1.0 ? 1 : static_cast<uint64_t>(lo), &before);
    }
    c.phi = d.k > 0 ? (h < c.klo ? h : c.klo) : (h < SB ? h : SB - 1);
    c.plo = l < c.phi ? l : c.phi;
    c.sure = c.plo;
    if (d.k == 0) c.klo = SB;
  }
  __syncthreads();
  return c;
}

// The composite at which a running sum over the candidates, in descending order, reaches `need` (>= 1): of their weights, or of their
// number; 0 where all do not reach it. `each(f)` calls f(composite, weight) for the candidates of each thread. All threads.
template <bool MASS, typename E>
__device__ __forceinline__ uint64_t find_composite(BlockLds& s, ListLds& t, uint64_t need, E&& each) {
  const int tid = threadIdx.x, lane = tid & 63;
  uint64_t prefix = 0;
#pragma unroll 1
  for (int shift = 56; shift >= 0; shift -= 8) {
    __syncthreads();
    if (tid < 256) t.digits[tid] = 0;
    if (tid == 0) s.b32 = 256;
    __syncthreads();
    each([&](uint64_t comp, uint64_t w) {
      if (shift == 56 || comp >> (shift + 8) == prefix)
        atomicAdd(reinterpret_cast<unsigned long long*>(&t.digits[comp >> shift & 255]), static_cast<unsigned long long>(MASS ? w : 1));
    });
    __syncthreads();
    if (tid < 64) {  // digits 255 - 4 lane .. - 3, descending
      uint64_t v[4], sum = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) sum += v[i] = t.digits[255 - 4 * lane - i];
      uint64_t before = wave_scan64(sum) - sum;
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

// Of a short list: each token's number and weight of those before it, by 16 lanes a token (158 tokens 14.8 -> 0.7 us beside a thread for each).
// f(i, number, weight) in one lane for each token i; of j, `first` says whether it comes before i, t.kind[j] & 1 counts it and
// t.digits[j] is what it adds.
template <int NT, typename P, typename F>
__device__ __forceinline__ void each_before(const ListLds& t, uint32_t n, P&& first, F&& f) {
  const uint32_t lane = threadIdx.x & 15;
#pragma unroll 1
  for (uint32_t i0 = 0; i0 < n; i0 += NT / 16) {
    const uint32_t i = i0 + (threadIdx.x >> 4);
    const uint64_t c = t.list[i < n ? i : 0];
    uint64_t number = 0, weight = 0;
#pragma unroll 4
    for (uint32_t j = lane; j < n; j += 16) {
      const uint64_t cj = t.list[j], w = t.digits[j];
      const uint32_t k = t.kind[j];
      const bool is = first(cj, c);
      number += is ? k & 1u : 0u;
      weight += is ? w : 0;
    }
    number = row_sum64(number);
    weight = row_sum64(weight);
    if (lane == 15 && i < n) f(i, static_cast<uint32_t>(number), weight);
  }
}

// The composite from which on a row's tokens are kept. `n` tokens are listed, in t.list if no more than SLIST; `held` is the exact weight of the
// sure ones, `mid` of what top_k keeps behind top_p's bins for certain. All threads. Here of a short list.
template <int NT>
__device__ __forceinline__ uint64_t threshold_near(BlockLds& s, ListLds& t, const Draw& d, const Cut& cut, const Weigher& weigh, uint32_t n, uint64_t held,
                                                   uint64_t mid) {
  const int tid = threadIdx.x;
  uint64_t c = 0, w = 0, threshold = 0;
  bool in_k = false, in_p = false, before_k = false;
  if (tid < static_cast<int>(n)) {
    c = t.list[tid];
    const float x = of_okey(static_cast<uint32_t>(c >> 32));
    const int b = bin_of(x, weigh.top, d.s);
    w = Weigher::whole(weigh.units(x));
    in_k = b >= cut.klo && b <= cut.khi;
    in_p = b >= cut.plo && b <= cut.phi;
    before_k = b < cut.klo;
    t.digits[tid] = in_p ? w : 0;
    t.kind[tid] = in_k ? 1 : 0;
  }
  if (tid == 0) s.a64 = s.b64 = 0;
  __syncthreads();
  const uint32_t want_k = static_cast<uint32_t>(d.k) - cut.above;
  each_before<NT>(t, n, [](uint64_t x, uint64_t y) { return x > y; }, [&](uint32_t i, uint32_t number, uint64_t weight) {
    if (d.k > 0 && (t.kind[i] & 1u) != 0 && number + 1 == want_k) s.a64 = t.list[i];
    t.before[i] = weight;
  });
  __syncthreads();
  threshold = s.a64;  // 0 without top_k
  if (d.p) {
    const uint64_t all = held + mid + block_sum64<NT>(s, before_k || c >= threshold ? w : 0);
    const uint64_t need = share_of(d.top_p, all), want = need > held ? need - held : 1;
    if (in_p) {
      const uint64_t before = t.before[tid];
      if (before < want && before + w >= want) s.b64 = c;
    }
    __syncthreads();
    threshold = s.b64 > threshold ? s.b64 : threshold;
  }
  __syncthreads();
  return threshold;
}

// Of a longer one, or of the row where the list holds less than all: digit by digit. Apart, so that the other rows' code is short.
template <typename R, int NT>
__device__ __attribute__((noinline)) uint64_t threshold_far(BlockLds* sp, ListLds* tp, const R r, int V, const Draw d, const Cut cut, const Weigher weigh,
                                                            uint32_t n, uint64_t held, uint64_t mid) {
  BlockLds& s = *sp;
  ListLds& t = *tp;
  const int tid = threadIdx.x;
  // f(composite, weight, bin) for the listed tokens of bins from .. to
  auto each_of = [&](int from, int to, auto&& f) {
    auto one = [&](uint64_t c) {
      const float x = of_okey(static_cast<uint32_t>(c >> 32));
      const int b = bin_of(x, weigh.top, d.s);
      if (b >= from && b <= to && cut.listed(b)) f(c, Weigher::whole(weigh.units(x)), b);
    };
    if (n <= SLIST) {
#pragma unroll 1
      for (uint32_t i = tid; i < n; i += NT) one(t.list[i]);
    } else {
      r.slowly(V, tid, NT, [&](float x, int i) {
        if (x > -__builtin_inff()) one(composite(x, static_cast<uint32_t>(i)));
      });
    }
  };
  uint64_t threshold = 0;
  if (d.k > 0)
    threshold = find_composite<false>(s, t, static_cast<uint64_t>(d.k) - cut.above, [&](auto&& f) {
      each_of(cut.klo, cut.khi, [&](uint64_t c, uint64_t w, int) { f(c, w); });
    });
  if (d.p) {
    uint64_t mine = 0;
    each_of(0, SB, [&](uint64_t c, uint64_t w, int b) { mine += b < cut.klo || c >= threshold ? w : 0; });
    const uint64_t all = held + mid + block_sum64<NT>(s, mine), need = share_of(d.top_p, all);
    const uint64_t c = find_composite<true>(s, t, need > held ? need - held : 1, [&](auto&& f) {
      each_of(cut.plo, cut.phi, [&](uint64_t k, uint64_t w, int) { f(k, w); });
    });
    threshold = c > threshold ? c : threshold;
  }
  __syncthreads();
  return threshold;
}

template <typename R, int NT>
__device__ __forceinline__ uint64_t threshold_of(BlockLds& s, ListLds& t, const R& r, int V, const Draw& d, const Cut& cut, const Weigher& weigh, uint32_t n,
                                                 uint64_t held, uint64_t mid) {
  return n <= SNEAR ? threshold_near<NT>(s, t, d, cut, weigh, n, held, mid) : threshold_far<R, NT>(&s, &t, r, V, d, cut, weigh, n, held, mid);
}

// What a kept token weighs; 0 for one that is not.
struct Keep {
  Weigher weigh;
  double least;
  uint64_t threshold;
  __device__ __forceinline__ uint64_t operator()(float x, uint32_t i) const {
    if (!(x > -__builtin_inff()) || composite(x, i) < threshold) return 0;
    const double u = weigh.units(x);
    return u >= least ? Weigher::whole(u) : 0;
  }
};

// The thread that has a row's token writes it; one logarithm in a kernel's code.
struct Found {
  float x;
  int token;  // -1: another thread's
  uint64_t total;
  __device__ __forceinline__ void write(const SampleArgs& a, int64_t row, const Weigher& weigh) const {
    if (token < 0) return;
    a.tokens[row] = token;
    a.shares[row] = static_cast<float>(log(weigh.units(x) / static_cast<double>(total)));
  }
};

// The token at which the running sum of the kept weights over begin .. end - 1 passes `target`, narrowed to a wave's part at a time. All threads.
template <typename R, int NT>
__device__ __forceinline__ Found draw_in(BlockLds& s, const R& r, int begin, int end, const Keep& keep, uint64_t target, uint64_t total) {
  constexpr int VEC = R::VEC, NW = NT / 64;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
#pragma unroll 1
  while (true) {
    const int per = ((end - begin + NW - 1) / NW + 64 * VEC - 1) / (64 * VEC) * (64 * VEC);
    const int from = begin + wave * per, to = end - from < per ? end : from + per;
    float f[VEC];
    uint64_t k[VEC], mine = 0;
    int at = 0;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      f[e] = 0.f;
      k[e] = 0;
    }
    r.template each<1>(from, to, lane, 64, [&](const float (&x)[VEC], int i) {
      at = i;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        f[e] = x[e];
        mine += k[e] = keep(x[e], static_cast<uint32_t>(i + e));
      }
    });
    const uint64_t sum = wave_sum64(mine);
    __syncthreads();
    if (lane == 0) s.part[wave] = sum;
    __syncthreads();
    int w = 0;
    uint64_t before = 0;
    while (w < NW - 1 && before + s.part[w] <= target) before += s.part[w++];
    target -= before;
    if (per > 64 * VEC) {
      begin += w * per;
      end = end - begin < per ? end : begin + per;
      continue;
    }
    Found found{0.f, -1, total};
    if (w != wave) return found;  // one load a lane, still in its registers
    const uint64_t inc = wave_scan64(mine);
    before = inc - mine;
    if (before <= target && target < inc) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        if (before <= target && target < before + k[e]) {
          found.token = at + e;
          found.x = f[e];
        }
        before += k[e];
      }
    }
    return found;
  }
}

// The draw of a row from the kept weights of its parts (at most 256, in t.weight): the part, then the token in it. All threads.
template <typename R, int NT>
__device__ __forceinline__ Found draw_parts(BlockLds& s, ListLds& t, const SampleArgs& a, int64_t row, const R& r, const Keep& keep, int parts, int size) {
  const int tid = threadIdx.x, lane = tid & 63;
  uint64_t v[4], sum = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) sum += v[i] = lane * 4 + i < parts ? t.weight[lane * 4 + i] : 0;
  const uint64_t inc = wave_scan64(sum);
  const uint64_t total = last_lane(inc);
  const uint64_t target = place_of(static_cast<double>(a.u[row]), total);
  uint64_t before = inc - sum;
  if (tid < 64) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (before <= target && target < before + v[i]) {
        s.a32 = lane * 4 + i;
        s.a64 = target - before;
      }
      before += v[i];
    }
  }
  __syncthreads();
  const int from = static_cast<int>(s.a32) * size, to = a.V - from < size ? a.V : from + size;
  return draw_in<R, NT>(s, r, from, to, keep, s.a64, total);
}

// The listed tokens' kept weights to t.weight, by part. All threads.
template <typename R, int NT>
__device__ __forceinline__ void add_list(ListLds& t, const R& r, int V, const Draw& d, const Cut& cut, const Keep& keep, uint32_t n, int size) {
  const int tid = threadIdx.x;
  auto add = [&](float x, uint32_t i) {
    const uint64_t k = keep(x, i);
    if (k != 0) atomicAdd(reinterpret_cast<unsigned long long*>(&t.weight[i / static_cast<uint32_t>(size)]), static_cast<unsigned long long>(k));
  };
  if (n <= SLIST) {
#pragma unroll 1
    for (uint32_t i = tid; i < n; i += NT) {
      const uint64_t c = t.list[i];
      add(of_okey(static_cast<uint32_t>(c >> 32)), 0xFFFFFFFFu - static_cast<uint32_t>(c));
    }
    return;
  }
  r.slowly(V, tid, NT, [&](float x, int i) {
    if (x > -__builtin_inff() && cut.listed(bin_of(x, keep.weigh.top, d.s))) add(x, static_cast<uint32_t>(i));
  });
}

// The draw of a row whose kept tokens are all in a short list. All threads.
template <int NT>
__device__ __forceinline__ Found draw_list(BlockLds& s, ListLds& t, const SampleArgs& a, int64_t row, const Keep& keep, uint32_t n) {
  const int tid = threadIdx.x;
  uint64_t k = 0;
  if (tid < static_cast<int>(n)) {
    const uint64_t c = t.list[tid];
    k = keep(of_okey(static_cast<uint32_t>(c >> 32)), 0xFFFFFFFFu - static_cast<uint32_t>(c));
    t.digits[tid] = k;
  }
  const uint64_t total = block_sum64<NT>(s, k), target = place_of(static_cast<double>(a.u[row]), total);
  Found found{0.f, -1, total};
  each_before<NT>(t, n, [](uint64_t x, uint64_t y) { return static_cast<uint32_t>(x) > static_cast<uint32_t>(y); },  // a lower index
                  [&](uint32_t i, uint32_t, uint64_t before) {
                    if (before <= target && target < before + t.digits[i]) {
                      const uint64_t c = t.list[i];
                      found.token = static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(c));
                      found.x = of_okey(static_cast<uint32_t>(c >> 32));
                    }
                  });
  return found;
}

// This thread's largest logit of from .. to - 1 and the first index that has it (a thread's ascend); -infinity where there is none.
template <typename R, int NT>
__device__ __forceinline__ float thread_best(const R& r, int from, int to, uint32_t& at) {
  constexpr int VEC = R::VEC;
  float best = -__builtin_inff();
  at = 0;
  r.template each<4>(from, to, static_cast<int>(threadIdx.x), NT, [&](const float (&f)[VEC], int i) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      at = f[e] > best ? i + e : at;
      best = f[e] > best ? f[e] : best;
    }
  });
  return best;
}

// The workgroup's largest composite, in all threads; 0 where there is none.
template <int NT>
__device__ __forceinline__ uint64_t block_best(BlockLds& s, float x, uint32_t at) {
  uint64_t best = x > -__builtin_inff() ? composite(x, at) : 0;
  best = wave_max64(best);
  if ((threadIdx.x & 63) == 0) s.part[threadIdx.x >> 6] = best;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) best = s.part[w] > best ? s.part[w] : best;
  return best;
}

// from .. to - 1 into the histogram: counts of all of them (or of the threads' largest ones, `mine`), and weights by float32's exponential.
template <typename R, int NT>
__device__ __forceinline__ void count_in(HistLds& hist, const R& r, int from, int to, const Draw& d, const Weigher& weigh, bool few_k, float mine) {
  constexpr int VEC = R::VEC;
  if (few_k) {
    if (mine > -__builtin_inff()) atomicAdd(&hist.count[bin_of(mine, weigh.top, d.s)], 1u);
    return;
  }
  const float c = static_cast<float>(-2.0 * d.c);
  r.template each<4>(from, to, static_cast<int>(threadIdx.x), NT, [&](const float (&f)[VEC], int) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      if (!(f[e] > -__builtin_inff())) continue;  // rows that a grammar masks would meet in one bin
      const int b = bin_of(f[e], weigh.top, d.s);
      if (d.k > 0) atomicAdd(&hist.count[b], 1u);
      if (d.p) {
        const float y = half_below(f[e], weigh.top) * c;
        atomicAdd(reinterpret_cast<unsigned long long*>(&hist.mass[b]),
                  static_cast<unsigned long long>(static_cast<uint32_t>(__builtin_amdgcn_exp2f(y + static_cast<float>(SAPPROX)))));
      }
    }
  });
}

// from .. to - 1: listed tokens through `list(composite)`, and this thread's exact weights: of the sure ones, of those of them that min_p
// keeps, and of what lies behind top_p's bins and is top_k's for certain. `step`: threads that take a stretch together, `first` this one's place.
template <typename R, typename L>
__device__ __forceinline__ void split_in(const R& r, int from, int to, int first, int step, const Draw& d, const Cut& cut, const Weigher& weigh,
                                         uint64_t& held, uint64_t& kept, uint64_t& mid, L&& list) {
  constexpr int VEC = R::VEC;
  if (d.k == 0) {  // top_p alone: every token's weight counts
    uint64_t all = 0, sure = 0, listed = 0;
    r.template each<4>(from, to, first, step, [&](const float (&f)[VEC], int i) {
      bool any = false;
      uint64_t w[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const int b = bin_of(f[e], weigh.top, d.s);
        const double u = weigh.units(f[e]);
        w[e] = Weigher::whole(u);
        const uint64_t ws = b < cut.sure ? w[e] : 0;
        all += w[e];
        sure += ws;
        if (d.least > 0.0) kept += u >= d.least ? ws : 0;
        any |= b >= cut.plo && b <= cut.phi;
      }
      if (any) {  // few vectors
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const int b = bin_of(f[e], weigh.top, d.s);
          if (b >= cut.plo && b <= cut.phi && f[e] > -__builtin_inff()) {
            listed += w[e];
            list(composite(f[e], i + e));
          }
        }
      }
    });
    held = sure;
    if (!(d.least > 0.0)) kept = sure;
    mid = all - sure - listed;
    return;
  }
  r.template each<4>(from, to, first, step, [&](const float (&f)[VEC], int i) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const int b = bin_of(f[e], weigh.top, d.s);
      if (b > cut.khi || !(f[e] > -__builtin_inff())) continue;  // nearly all
      if (cut.listed(b)) list(composite(f[e], i + e));
      else {
        const double u = weigh.units(f[e]);
        const uint64_t w = Weigher::whole(u);
        if (b < cut.sure) {
          held += w;
          kept += u >= d.least ? w : 0;
        } else {
          mid += w;
        }
      }
    }
  });
}

// One workgroup a row, all of it; a wave's part is a stretch of the row.
template <typename T, int N>
__global__ __launch_bounds__(ST) void k_sample_row(SampleArgs a, int F) {
  typedef RowOf<T, N> R;
  constexpr int VEC = R::VEC;
  __shared__ BlockLds s;
  __shared__ HistLds hist;
  __shared__ ListLds t;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x;
  const R r{static_cast<const T*>(a.x) + row * a.stride};
  const Draw d = draw_of(a, row, F);
  const int V = a.V;
  const bool filter = d.k > 0 || d.p;
  if (filter && !d.greedy)
    for (int i = tid; i < SB; i += ST) {
      hist.mass[i] = 0;
      hist.count[i] = 0;
    }
  if (tid == 0) s.n = 0;
  uint32_t at;
  const float mine = thread_best<R, ST>(r, 0, V, at);
  const uint64_t best = block_best<ST>(s, mine, at);
  if (best == 0 || d.greedy) {
    if (tid == 0) {
      a.tokens[row] = best == 0 ? -1 : static_cast<int32_t>(0xFFFFFFFFu - static_cast<uint32_t>(best));
      a.shares[row] = best == 0 ? -__builtin_inff() : 0.f;
    }
    return;
  }
  const float top = of_okey(static_cast<uint32_t>(best >> 32));
  const Weigher weigh(top, d.c, F);
  Keep keep{weigh, d.least, 0};
  constexpr int parts = ST / 64;
  const int size = ((V + parts - 1) / parts + 64 * VEC - 1) / (64 * VEC) * (64 * VEC);
  const int from = wave * size < V ? wave * size : V, to = V - from < size ? V : from + size;
  if (!filter) {
    uint64_t kept = 0;
    r.template each<4>(from, to, lane, 64, [&](const float (&f)[VEC], int) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const double u = weigh.units(f[e]);
        kept += u >= d.least ? Weigher::whole(u) : 0;
      }
    });
    kept = wave_sum64(kept);
    if (lane == 0) t.weight[wave] = kept;
    draw_parts<R, ST>(s, t, a, row, r, keep, parts, size).write(a, row, weigh);
    return;
  }
  count_in<R, ST>(hist, r, 0, V, d, weigh, few(d, ST), mine);
  __syncthreads();
  const Cut cut = cut_of<ST>(s, hist, d, V, ST);
  uint64_t held = 0, kept = 0, mid = 0;
  split_in(r, from, to, lane, 64, d, cut, weigh, held, kept, mid, [&](uint64_t c) {
    const uint32_t n = atomicAdd(&s.n, 1u);
    if (n < SLIST) t.list[n] = c;
  });
  kept = wave_sum64(kept);
  if (lane == 0) t.weight[wave] = kept;
  if (d.p) {
    held = block_sum64<ST>(s, held);
    mid = block_sum64<ST>(s, mid);
  }
  __syncthreads();
  const uint32_t n = s.n;
  keep.threshold = threshold_of<R, ST>(s, t, r, V, d, cut, weigh, n, held, mid);
  Found found;
  if (cut.sure == 0 && n <= SNEAR) found = draw_list<ST>(s, t, a, row, keep, n);
  else {
    add_list<R, ST>(t, r, V, d, cut, keep, n, size);
    found = draw_parts<R, ST>(s, t, a, row, r, keep, parts, size);
  }
  found.write(a, row, weigh);
}

// ---------------------------------------------------------------------------
// Few rows: parts of a row by workgroups, in launches that end where the whole row has to be known. k_sample_top: the largest logit.
// k_sample_mass: the histogram, whose cut the last part to arrive takes; without top_k and top_p the parts' weights, and the draw.
// k_sample_draw: the list and the exact weights by part; the last part to arrive finds the threshold, the part in which the number
// falls, and the token in it. What parts leave for the last one goes past the L2 of its XCD.
struct SampleRow {        // at the head of the workspace, zero between calls
  uint64_t best;
  uint32_t arrived, pad;
};
struct SampleShare {      // a row's, behind the head
  uint64_t mass[SB];
  uint64_t list[SLIST];
  uint32_t count[SB];
  Cut cut;
  uint32_t n, pad;
};                        // and three weights of each part: kept, held, mid
constexpr int64_t SAMPLE_HEAD = 4096;
constexpr int SAMPLE_ROWS = static_cast<int>(SAMPLE_HEAD / sizeof(SampleRow));
static_assert(sizeof(SampleShare) % 8 == 0);

struct SamplePlan {
  int parts, size;        // of a row; size: logits of a part
  __host__ __device__ int64_t row_bytes() const { return (static_cast<int64_t>(sizeof(SampleShare)) + parts * 24 + 255) / 256 * 256; }
};

template <typename U>
__device__ __forceinline__ void put(U* p, U v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
template <typename U>
__device__ __forceinline__ U get(const U* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

__device__ __forceinline__ SampleRow* row_of(const SampleArgs& a, int64_t row) { return static_cast<SampleRow*>(a.ws) + row; }
__device__ __forceinline__ SampleShare* share_of_row(const SampleArgs& a, const SamplePlan& p, int64_t row) {
  return reinterpret_cast<SampleShare*>(static_cast<uint8_t*>(a.ws) + SAMPLE_HEAD + row * p.row_bytes());
}

// Whether this workgroup is the last of its row's parts. What it put before is seen by that one. All threads.
__device__ __forceinline__ bool last_part(BlockLds& s, SampleRow* w, int parts) {
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (threadIdx.x == 0) {
    s.last = __hip_atomic_fetch_add(&w->arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == static_cast<uint32_t>(parts) - 1u;
    if (s.last) put(&w->arrived, 0u);
  }
  __syncthreads();
  return s.last != 0;
}

template <typename T>
__global__ __launch_bounds__(SP) void k_sample_top(SampleArgs a, SamplePlan p, int F) {
  typedef RowOf<T, 16 / sizeof(T)> R;
  __shared__ BlockLds s;
  const int tid = threadIdx.x, part = static_cast<int>(blockIdx.x);
  const int64_t row = blockIdx.y;
  const R r{static_cast<const T*>(a.x) + row * a.stride};
  const int from = part * p.size, to = a.V - from < p.size ? a.V : from + p.size;
  SampleShare* w = share_of_row(a, p, row);
  for (int i = part * SP + tid; i < SB; i += p.parts * SP) {
    w->mass[i] = 0;
    w->count[i] = 0;
  }
  if (part == 0 && tid == 0) w->n = 0;
  uint32_t at;
  const float mine = thread_best<R, SP>(r, from, to, at);
  const uint64_t best = block_best<SP>(s, mine, at);
  if (tid == 0 && best != 0) __hip_atomic_fetch_max(&row_of(a, row)->best, best, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

template <typename T>
__global__ __launch_bounds__(SP) void k_sample_mass(SampleArgs a, SamplePlan p, int F) {
  typedef RowOf<T, 16 / sizeof(T)> R;
  constexpr int VEC = R::VEC;
  __shared__ BlockLds s;
  __shared__ union {
    HistLds hist;
    ListLds list;
  } u;
  const int tid = threadIdx.x, part = static_cast<int>(blockIdx.x);
  const int64_t row = blockIdx.y;
  const R r{static_cast<const T*>(a.x) + row * a.stride};
  const int from = part * p.size, to = a.V - from < p.size ? a.V : from + p.size;
  const Draw d = draw_of(a, row, F);
  SampleRow* w = row_of(a, row);
  SampleShare* sh = share_of_row(a, p, row);
  uint64_t* weights = reinterpret_cast<uint64_t*>(sh + 1);
  const uint64_t best = w->best;
  if (best == 0 || d.greedy) {
    if (!last_part(s, w, p.parts)) return;  // all parts have read `best`
    if (tid == 0) {
      a.tokens[row] = best == 0 ? -1 : static_cast<int32_t>(0xFFFFFFFFu - static_cast<uint32_t>(best));
      a.shares[row] = best == 0 ? -__builtin_inff() : 0.f;
      put(&w->best, uint64_t{0});
    }
    return;
  }
  const float top = of_okey(static_cast<uint32_t>(best >> 32));
  const Weigher weigh(top, d.c, F);
  if (d.k == 0 && !d.p) {
    const Keep keep{weigh, d.least, 0};
    uint64_t mine = 0;
    r.template each<4>(from, to, tid, SP, [&](const float (&f)[VEC], int) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const double u = weigh.units(f[e]);
        mine += u >= d.least ? Weigher::whole(u) : 0;
      }
    });
    mine = block_sum64<SP>(s, mine);
    if (tid == 0) put(weights + part, mine);
    if (!last_part(s, w, p.parts)) return;
    if (tid == 0) put(&w->best, uint64_t{0});
    if (tid < p.parts) u.list.weight[tid] = get(weights + tid);
    draw_parts<R, SP>(s, u.list, a, row, r, keep, p.parts, p.size).write(a, row, weigh);
    return;
  }
  const int threads = p.parts * SP;
  const bool few_k = few(d, threads);
  for (int i = tid; i < SB; i += SP) {
    u.hist.mass[i] = 0;
    u.hist.count[i] = 0;
  }
  float mine = 0.f;
  if (few_k) {
    uint32_t at;
    mine = thread_best<R, SP>(r, from, to, at);
  }
  __syncthreads();
  count_in<R, SP>(u.hist, r, from, to, d, weigh, few_k, mine);
  __syncthreads();
  for (int i = tid; i < SB; i += SP) {
    if (u.hist.count[i] != 0) __hip_atomic_fetch_add(&sh->count[i], u.hist.count[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (u.hist.mass[i] != 0) __hip_atomic_fetch_add(&sh->mass[i], u.hist.mass[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  if (!last_part(s, w, p.parts)) return;
  for (int i = tid; i < SB; i += SP) {
    u.hist.count[i] = d.k > 0 ? get(&sh->count[i]) : 0u;
    u.hist.mass[i] = d.p && !few_k ? get(&sh->mass[i]) : 0u;
  }
  __syncthreads();
  const Cut cut = cut_of<SP>(s, u.hist, d, a.V, threads);
  if (tid == 0) sh->cut = cut;  // for the next launch
}

template <typename T>
__global__ __launch_bounds__(SP) void k_sample_draw(SampleArgs a, SamplePlan p, int F) {
  typedef RowOf<T, 16 / sizeof(T)> R;
  __shared__ BlockLds s;
  __shared__ ListLds t;
  const int tid = threadIdx.x, part = static_cast<int>(blockIdx.x);
  const int64_t row = blockIdx.y;
  const R r{static_cast<const T*>(a.x) + row * a.stride};
  const int from = part * p.size, to = a.V - from < p.size ? a.V : from + p.size;
  const Draw d = draw_of(a, row, F);
  SampleRow* w = row_of(a, row);
  SampleShare* sh = share_of_row(a, p, row);
  uint64_t* weights = reinterpret_cast<uint64_t*>(sh + 1);
  const uint64_t best = w->best;
  if (best == 0) return;  // drawn, or nothing to draw
  const float top = of_okey(static_cast<uint32_t>(best >> 32));
  const Weigher weigh(top, d.c, F);
  const Cut cut = sh->cut;
  uint64_t held = 0, kept = 0, mid = 0;
  if (tid == 0) s.n = 0;
  __syncthreads();
  split_in(r, from, to, tid, SP, d, cut, weigh, held, kept, mid, [&](uint64_t c) {
    const uint32_t n = atomicAdd(&s.n, 1u);
    if (n < SLIST) t.list[n] = c;
  });
  kept = block_sum64<SP>(s, kept);
  if (tid == 0) put(weights + part, kept);
  if (d.p) {
    held = block_sum64<SP>(s, held);
    mid = block_sum64<SP>(s, mid);
    if (tid == 0) {
      put(weights + p.parts + part, held);
      put(weights + 2 * p.parts + part, mid);
    }
  }
  const uint32_t own = s.n;  // behind a barrier of the sums
  if (own > 0) {
    __syncthreads();
    if (tid == 0) s.a32 = __hip_atomic_fetch_add(&sh->n, own, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    const uint32_t base = s.a32;
    for (uint32_t i = tid; i < own && i < SLIST && base + i < SLIST; i += SP) put(&sh->list[base + i], t.list[i]);
  }
  if (!last_part(s, w, p.parts)) return;
  if (tid == 0) put(&w->best, uint64_t{0});
  // all that the parts left, in flight together
  const uint32_t n = get(&sh->n);
  const uint64_t head = get(&sh->list[tid]);
  const uint64_t w0 = tid < p.parts ? get(weights + tid) : 0, w1 = d.p && tid < p.parts ? get(weights + p.parts + tid) : 0,
                 w2 = d.p && tid < p.parts ? get(weights + 2 * p.parts + tid) : 0;
  t.list[tid] = head;
  for (uint32_t i = SP + tid; i < n && i < SLIST; i += SP) t.list[i] = get(&sh->list[i]);
  if (tid < p.parts) t.weight[tid] = w0;
  held = block_sum64<SP>(s, w1);
  mid = block_sum64<SP>(s, w2);
  __syncthreads();
  const Keep keep{weigh, d.least, threshold_of<R, SP>(s, t, r, a.V, d, cut, weigh, n, held, mid)};
  Found found;
  if (cut.sure == 0 && n <= SNEAR) found = draw_list<SP>(s, t, a, row, keep, n);
  else {
    add_list<R, SP>(t, r, a.V, d, cut, keep, n, p.size);
    found = draw_parts<R, SP>(s, t, a, row, r, keep, p.parts, p.size);
  }
  found.write(a, row, weigh);
}

// What a call's rows ask for: the numbers of estimated times below.
enum Kind { NO_FILTER, TOP_K, TOP_P };

Kind kind_of(const SampleArgs& a) {
  if (a.top_p != nullptr || a.top_p1 < 1.0) return TOP_P;
  return a.top_k != nullptr || (a.top_k1 > 0 && a.top_k1 < a.V) ? TOP_K : NO_FILTER;
}

// Rows by parts where that is estimated faster (us, measured on float32 logits, no filter / top_k 50 / top_p 0.95):
//   a workgroup a row: 7 + V / 2950, 10.5 + V / 5400, 12 + V / 1500 for each round of 256 (32000 logits: 16.6, 16.8, 33; 128000: 50, 34, 98)
//   by parts: 10.5, 22, 28 and the logits at 330, 500 and 170 thousand a us (1 x 128000: 11, 23, 34; 64 x 128000: 36, 38, 75)
// 64 parts a row and 512 workgroups at most, 1024 from 32 rows on (16 x 128000 with top_p 48 in 32 parts, 58 in 64; 64 x 128000 75
// in 16, 77 in 8).
bool sample_split(int64_t rows, int64_t V, Kind kind, SamplePlan& p) {
  static constexpr double kRow[3] = {7.0, 10.5, 12.0}, kRowRate[3] = {2950, 5400, 1500}, kStart[3] = {10.5, 22.0, 28.0}, kRate[3] = {330e3, 500e3, 170e3};
  if (rows < 1 || rows > SAMPLE_ROWS || V < 4096) return false;
  const double whole = kRow[kind] + static_cast<double>(V) / kRowRate[kind];
  const double parted = kStart[kind] + (kind == TOP_P && rows > 1 ? 6.0 : 0.0) + static_cast<double>(rows) * static_cast<double>(V) / kRate[kind];
  if (whole <= parted) return false;
  int64_t parts = (rows < 32 ? 512 : 1024) / rows;
  parts = parts < 64 ? parts : 64;
  const int64_t most = (V + 2047) / 2048;
  parts = parts < most ? parts : most;
  p.size = static_cast<int>(((V + parts - 1) / parts + 2047) / 2048 * 2048);
  p.parts = static_cast<int>((V + p.size - 1) / p.size);
  return p.parts > 1;
}

template <typename T>
hipError_t sample_type(SampleArgs a, int F, hipStream_t st) {
  SamplePlan p;
  if (a.ws != nullptr && sample_split(a.rows, a.V, kind_of(a), p) && a.ws_bytes >= SAMPLE_HEAD + a.rows * p.row_bytes()) {
    const dim3 grid(static_cast<uint32_t>(p.parts), static_cast<uint32_t>(a.rows));
    k_sample_top<T><<<grid, SP, 0, st>>>(a, p, F);
    k_sample_mass<T><<<grid, SP, 0, st>>>(a, p, F);
    if (kind_of(a) != NO_FILTER) k_sample_draw<T><<<grid, SP, 0, st>>>(a, p, F);
    return hipGetLastError();
  }
  constexpr int64_t most = kLaunchThreads / ST;
  while (true) {
    const dim3 grid(static_cast<uint32_t>(a.rows < most ? a.rows : most));
    if (a.V >= static_cast<int>(16 / sizeof(T))) k_sample_row<T, 16 / sizeof(T)><<<grid, ST, 0, st>>>(a, F);
    else k_sample_row<T, 1><<<grid, ST, 0, st>>>(a, F);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.rows <= most) return e;
    a.rows -= most;
    a.x = static_cast<const T*>(a.x) + most * a.stride;
    a.u += most;
    a.tokens += most;
    a.shares += most;
    if (a.temperature) a.temperature += most;
    if (a.top_p) a.top_p += most;
    if (a.min_p) a.min_p += most;
    if (a.top_k) a.top_k += most;
  }
}

}  // namespace

int64_t sample_workspace_bytes(int64_t rows, int64_t V) {  // whatever the call's settings
  int64_t most = 0;
  for (const Kind kind : {NO_FILTER, TOP_K, TOP_P}) {
    SamplePlan p;
    if (!sample_split(rows, V, kind, p)) continue;
    const int64_t n = SAMPLE_HEAD + rows * p.row_bytes();
    most = n > most ? n : most;
  }
  return most;
}

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
