// Attention of a batch whose sequences' first tokens lie in the same pages of the 8-bit cache.
#include <cstdlib>
#include <cstring>

#include "xrmm_kv8_attn.h"

namespace xrmm {

hipError_t launch_kv8_walk(const KvAttnArgs& a, const KvPlan& p, hipStream_t st);
hipError_t launch_kv8_prefix(const KvAttnArgs& a, const KvPlan& p, hipStream_t st);
hipError_t launch_kv8_own(const KvAttnArgs& a, const KvPlan& p, hipStream_t st);
hipError_t launch_kv8_both(const KvAttnArgs& a, const KvPlan& prefix, const KvPlan& own, hipStream_t st);

namespace {

// The parts of a row: weights exp2(maximum - the largest maximum), outputs added in a fixed order, divided by the sum. A thread has four
// values of a row and every fourth part, a wave's groups of 16 threads the four shares, and their loads in flight together; the shares meet across
// the wave. The parts' bytes and the start bound it: 11 us for 64 sequences of 32 heads of 128 in 33 parts (35 MB), 9.6 for 128 in 17 (36 MB), which
// is why part_plan counts the parts' bytes. Rows that `starts` leaves out are not written.
constexpr int KVJ_T = 256;

template <int D>
__global__ __launch_bounds__(KVJ_T) void k_kv8_join(KvAttnArgs a) {
  const int lane = threadIdx.x & 63, share = lane >> 4;
  const int64_t rows = a.c.rows * a.Hq, piece = (static_cast<int64_t>(blockIdx.x) * (KVJ_T / 64) + (threadIdx.x >> 6)) * 16 + (lane & 15);
  const int64_t out = piece / (D / 4);  // [row][head]; the same in a wave's shares
  const int d = static_cast<int>(piece % (D / 4)) * 4;
  const bool in = out < rows;
  const int row = in ? static_cast<int>(out / a.Hq) : 0, hq = in ? static_cast<int>(out % a.Hq) : 0, G = a.Hq / a.c.Hkv, h = hq / G;
  const int64_t at = static_cast<int64_t>(row) * G + hq % G;
  const KvPart<D> part(a, 0, h);
  float m = -__builtin_inff(), l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  constexpr int N = 8;
#pragma unroll 1
  for (int p0 = share; p0 < a.parts; p0 += 4 * N) {
    f32x4 x[N];
    f32x2 ml[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int64_t p = (p0 + 4 * i < a.parts ? p0 + 4 * i : p0) * rows + at;
      ml[i] = part.ml[p];
      x[i] = *reinterpret_cast<const f32x4*>(part.o + p * D + d);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      // no such part, or one that saw nothing and left no outputs; a query that is no number has a sum that is none
      if (p0 + 4 * i >= a.parts || (ml[i][0] == -__builtin_inff() && ml[i][1] == 0.f)) continue;
      const float mn = fmaxf(m, ml[i][0]), f0 = m == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(m - mn), f1 = __builtin_amdgcn_exp2f(ml[i][0] - mn);
      o = o * f0 + x[i] * f1;
      l = l * f0 + ml[i][1] * f1;
      m = mn;
    }
  }
#pragma unroll
  for (int s = 16; s <= 32; s <<= 1) {
    const float m1 = __shfl_xor(m, s, 64), l1 = __shfl_xor(l, s, 64);
    const f32x4 o1 = {__shfl_xor(o[0], s, 64), __shfl_xor(o[1], s, 64), __shfl_xor(o[2], s, 64), __shfl_xor(o[3], s, 64)};
    // the same operands in the same order in both lanes
    const bool low = (lane & s) == 0;
    const float ma = low ? m : m1, mb = low ? m1 : m, mn = fmaxf(ma, mb);
    const float fa = ma == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(ma - mn), fb = mb == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(mb - mn);
    o = (low ? o : o1) * fa + (low ? o1 : o) * fb;
    l = (low ? l : l1) * fa + (low ? l1 : l) * fb;
    m = mn;
  }
  int b, pos;
  if (!in || share != 0 || !kv_position(a, row, b, pos)) return;
  o *= l != 0.f ? 1.f / l : 0.f;
  typedef u32x2 u32x2_2 __attribute__((aligned(2)));
  *reinterpret_cast<u32x2_2*>(static_cast<uint16_t*>(a.o) + out * D + d) =
      a.dtype == LT_F16 ? __builtin_bit_cast(u32x2, __builtin_convertvector(o, f16x4)) : __builtin_bit_cast(u32x2, __builtin_convertvector(o, bf16x4));
}

hipError_t launch_join(const KvAttnArgs& a, hipStream_t st) {
  const int64_t n = (a.c.rows * a.Hq * (a.c.D / 4) + KVJ_T / 4 - 1) / (KVJ_T / 4);
  if (!grid_counts(n, KVJ_T)) return hipErrorInvalidValue;
  const dim3 grid(static_cast<uint32_t>(n));
  switch (a.c.D) {
    case 64: k_kv8_join<64><<<grid, KVJ_T, 0, st>>>(a); break;
    case 96: k_kv8_join<96><<<grid, KVJ_T, 0, st>>>(a); break;
    case 128: k_kv8_join<128><<<grid, KVJ_T, 0, st>>>(a); break;
    default: k_kv8_join<256><<<grid, KVJ_T, 0, st>>>(a);
  }
  return hipGetLastError();
}

// A launch that leaves parts: nrows rows of each of `seqs` sequences over `span` tokens, by the times of kind_plan and the bytes of its parts,
// written and read at 4 TB/s.
KvPlan part_plan(const KvAttnArgs& a, int64_t nrows, int64_t seqs, int64_t span, bool tile) {
  const int64_t cus = device_cus() > 0 ? device_cus() : 256, rows = tile ? KVM_ROWS : 16;
  KvPlan p{};
  p.tile = tile;
  p.row_tiles = (nrows + rows - 1) / rows;
  const int64_t units = p.row_tiles * a.c.Hkv * seqs, room = tile && a.c.D <= 128 ? 2 * cus : cus;
  const int live = nrows < KVM_ROWS ? static_cast<int>((nrows + 31) / 32) : 4;
  static constexpr double kTile[5] = {0, 36, 28, 24, 18};
  const double two = kv_two(a) && nrows > 16 ? tile ? 0.87 : 0.95 : 1.0;  // a weight's second term beside products, not beside bytes
  const double rate = (tile ? kTile[live] : 75.0) * two, start = tile ? 10.0 : 7.0, wide = a.c.D > 128 ? 2.0 : 1.0;
  const double part = 2.0 * static_cast<double>(nrows * seqs * a.c.Hkv) * (a.c.D + 2) * 4 / 4e6;  // us
  span = span > 0 ? span : 1;
  int64_t most = units < room ? room / units : 1;
  most = most < 64 ? most : 64;
  for (int64_t want = 1; want <= most; ++want) {
    const int64_t chunk = want > 1 ? ((span + want - 1) / want + KVR_PASS - 1) / KVR_PASS * KVR_PASS : (span + KVR_PASS - 1) / KVR_PASS * KVR_PASS;
    const int64_t parts = (span + chunk - 1) / chunk;
    const double time = static_cast<double>((units * parts + room - 1) / room) * (start + wide * static_cast<double>(chunk) / rate) + part * static_cast<double>(parts);
    if (p.splits == 0 || time < p.time) {
      p.splits = parts;
      p.chunk = chunk;
      p.time = time;
    }
  }
  p.waves = p.chunk <= 2 * KVT ? 2 : p.chunk <= 8 * KVT || (p.chunk <= 2048 && units * p.splits > cus) ? 4 : 8;
  return p;
}

// Whether own rows go into one launch with tiles of the shared tokens.
bool together(const KvAttnArgs& a, const KvPlan& own) { return !own.tile && own.row_tiles == 1 && a.c.D <= 128; }

struct SharedPlan {
  bool walk;  // the sequences one by one, over all of their tokens
  KvPlan all, prefix, own;
  int64_t ws_bytes;
};

// XRMM_KV8_SHARED names a way (as xrmm_kv8_shared_attention_kernel does) to take instead of the fastest one, where a call can go it.
SharedPlan shared_plan(const KvAttnArgs& a, bool have_ws) {
  const char* way = std::getenv("XRMM_KV8_SHARED");
  const bool walk = way != nullptr && std::strcmp(way, "kv8_walk") == 0, rows = way != nullptr && std::strcmp(way, "kv8_prefix_rows") == 0,
             tile = way != nullptr && std::strcmp(way, "kv8_prefix_tile") == 0;
  SharedPlan s{};
  const int64_t G = a.Hq / a.c.Hkv, tokens = static_cast<int64_t>(a.shared_pages) << a.c.page_log2;
  // the walk begins at a multiple of a tile's tokens before the sequences' own
  const int64_t own = 64 + (a.c.width > a.shared_pages ? static_cast<int64_t>(a.c.width - a.shared_pages) << a.c.page_log2 : 0);
  s.walk = true;
  s.all = attention_plan(a, have_ws);
  s.ws_bytes = s.all.ws_bytes;
  if (!have_ws || tokens == 0 || a.c.B < 2 || a.c.rows * G > 0x7FFFFFF0 || walk) return s;
  const int64_t nrows = static_cast<int64_t>(a.max_new) * G;
  auto faster = [](const KvPlan& x, const KvPlan& y, double more) { return y.time + more < x.time ? y : x; };
  s.own = part_plan(a, nrows, a.c.B, own, false);
  if (nrows > 16) s.own = faster(s.own, part_plan(a, nrows, a.c.B, own, true), 0.0);
  // Beside tiles the own rows cost about half of their time: with that counted, 64 rows a key head on 6400 shared tokens (8 heads of 128) go by
  // tiles, 23 us for 29 by rows.
  const double beside = together(a, s.own) ? 0.5 * s.own.time : s.own.time;
  s.prefix = part_plan(a, a.c.rows * G, 1, tokens, tile);
  if (!rows && !tile && a.c.rows * G > 16) s.prefix = faster(s.prefix, part_plan(a, a.c.rows * G, 1, tokens, true), beside - s.own.time);
  const double time = s.prefix.time + (s.prefix.tile ? beside : s.own.time) + 4.0;
  const int64_t bytes = KV_COUNTERS + (s.prefix.splits + s.own.splits) * a.c.rows * a.Hq * (a.c.D + 2) * 4;
  if ((rows || tile || time < s.all.time) && bytes <= int64_t{1} << 28) {
    s.walk = false;
    s.ws_bytes = bytes;
  }
  return s;
}

}  // namespace

int64_t kv8_shared_workspace_bytes(const KvAttnArgs& a) {
  return a.c.B == 0 || a.max_new == 0 ? 0 : shared_plan(a, true).ws_bytes;
}

const char* kv8_shared_kernel_name(const KvAttnArgs& a) {
  if (a.c.B == 0 || a.max_new == 0) return "kv8_walk";
  const SharedPlan p = shared_plan(a, true);
  return p.walk ? "kv8_walk" : p.prefix.tile ? "kv8_prefix_tile" : "kv8_prefix_rows";
}

hipError_t launch_kv8_shared_attention(const KvAttnArgs& a, hipStream_t st) {
  if (a.c.B == 0 || a.max_new == 0) return hipSuccess;
  SharedPlan p = shared_plan(a, a.ws != nullptr);
  if (p.ws_bytes > a.ws_bytes) p = shared_plan(a, false);
  if (p.walk) return launch_kv8_walk(a, p.all, st);
  KvAttnArgs x = a;
  x.parts = static_cast<int32_t>(p.prefix.splits + p.own.splits);
  x.parts_at = KV_COUNTERS;
  x.part0 = 0;
  if (p.prefix.tile && together(a, p.own)) {
    const hipError_t e = launch_kv8_both(x, p.prefix, p.own, st);
    return e == hipSuccess ? launch_join(x, st) : e;
  }
  hipError_t e = launch_kv8_prefix(x, p.prefix, st);
  x.part0 = static_cast<int32_t>(p.prefix.splits);
  if (e == hipSuccess) e = launch_kv8_own(x, p.own, st);
  return e == hipSuccess ? launch_join(x, st) : e;
}

}  // namespace xrmm
