// One of the walks of attention on shared pages (XRMM_KV_MODE: 1 walk, 2 prefix, 3 own, 4 the last two in one launch), in a translation
// unit each.
#include "xrmm_kv8_attn.h"

namespace xrmm {

#if XRMM_KV_MODE == 1
hipError_t launch_kv8_walk(const KvAttnArgs& a, const KvPlan& p, hipStream_t st) { return attention_with<KV_WALK>(a, p, st); }
#elif XRMM_KV_MODE == 2
hipError_t launch_kv8_prefix(const KvAttnArgs& a, const KvPlan& p, hipStream_t st) { return attention_with<KV_PREFIX>(a, p, st); }
#elif XRMM_KV_MODE == 4

namespace {

// Tiles over the shared tokens and single rows over the sequences' own, which need nothing of each other: the first are bound by instructions, the
// second by the cache's bytes. The short own workgroups come first, so that the long tiles fill the CUs behind them: 44 us for 64 sequences with
// 8192 shared tokens and 600 of their own (32 heads on 8 of 128, e4m3), 164 for 128 with 32768 and 301 (int8); weights of two terms (KV_PE), as rows of
// one tile have. With the kinds in turns by eights the last tiles begin late (4 us more, and 50). Heads of 256 leave no LDS for it.
template <int D, bool FP8>
__global__ __launch_bounds__(KVM_T, 2) void k_kv8_shared(KvAttnArgs a, uint32_t prefix_tiles, uint32_t prefix_splits, uint32_t prefix_chunk,
                                                         uint32_t prefix_blocks, uint32_t own_tiles, uint32_t own_splits, uint32_t own_chunk) {
  extern __shared__ __align__(16) unsigned char smem[];
  static_assert(sizeof(KvRowsLds<D, 4>) <= kv8_tile_lds<D>());
  const uint32_t own_blocks = gridDim.x - prefix_blocks;
  const bool prefix = blockIdx.x >= own_blocks;
  const uint32_t block = prefix ? blockIdx.x - own_blocks : blockIdx.x;
  if (prefix) kv8_tile<D, FP8, true, KV_PREFIX>(a, prefix_tiles, prefix_splits, prefix_chunk, block, smem);
  else {
    KvAttnArgs x = a;
    x.part0 = static_cast<int32_t>(prefix_splits);
    kv8_rows<D, FP8, 4, true, KV_OWN>(x, own_tiles, own_splits, own_chunk, block, *reinterpret_cast<KvRowsLds<D, 4>*>(smem));
  }
}

template <int D, bool FP8>
hipError_t shared_for(const KvAttnArgs& a, const KvPlan& p, const KvPlan& o, hipStream_t st) {
  const int64_t np = p.row_tiles * p.splits * a.c.Hkv, no = o.row_tiles * o.splits * a.c.Hkv * a.c.B;
  if (!grid_counts(np + no, KVM_T)) return hipErrorInvalidValue;
  constexpr int lds = kv8_tile_lds<D>();
  static std::atomic<int> done[kMaxDevices];
  if (lds > 65536) {
    const hipError_t e = raise_lds_cap(reinterpret_cast<const void*>(k_kv8_shared<D, FP8>), lds, done);
    if (e != hipSuccess) return e;
  }
  k_kv8_shared<D, FP8><<<dim3(static_cast<uint32_t>(np + no)), KVM_T, lds, st>>>(
      a, static_cast<uint32_t>(p.row_tiles), static_cast<uint32_t>(p.splits), static_cast<uint32_t>(p.chunk), static_cast<uint32_t>(np),
      static_cast<uint32_t>(o.row_tiles), static_cast<uint32_t>(o.splits), static_cast<uint32_t>(o.chunk));
  return hipGetLastError();
}

}  // namespace

hipError_t launch_kv8_both(const KvAttnArgs& a, const KvPlan& prefix, const KvPlan& own, hipStream_t st) {
  switch (a.c.D * 2 + (a.c.fp8 ? 1 : 0)) {
    case 128: return shared_for<64, false>(a, prefix, own, st);
    case 129: return shared_for<64, true>(a, prefix, own, st);
    case 192: return shared_for<96, false>(a, prefix, own, st);
    case 193: return shared_for<96, true>(a, prefix, own, st);
    case 256: return shared_for<128, false>(a, prefix, own, st);
    case 257: return shared_for<128, true>(a, prefix, own, st);
  }
  return hipErrorInvalidValue;
}

#else
hipError_t launch_kv8_own(const KvAttnArgs& a, const KvPlan& p, hipStream_t st) { return attention_with<KV_OWN>(a, p, st); }
#endif

}  // namespace xrmm
