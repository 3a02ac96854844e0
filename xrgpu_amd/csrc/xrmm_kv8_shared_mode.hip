// One of the walks of attention on shared pages (XRMM_KV_MODE: 1 walk, 2 prefix, 3 own), in a translation unit each.
#include "xrmm_kv8_attn.h"

namespace xrmm {

#if XRMM_KV_MODE == 1
hipError_t launch_kv8_walk(const KvAttnArgs& a, const KvPlan& p, hipStream_t st) { return attention_with<KV_WALK>(a, p, st); }
#elif XRMM_KV_MODE == 2
hipError_t launch_kv8_prefix(const KvAttnArgs& a, const KvPlan& p, hipStream_t st) { return attention_with<KV_PREFIX>(a, p, st); }
#else
hipError_t launch_kv8_own(const KvAttnArgs& a, const KvPlan& p, hipStream_t st) { return attention_with<KV_OWN>(a, p, st); }
#endif

}  // namespace xrmm
