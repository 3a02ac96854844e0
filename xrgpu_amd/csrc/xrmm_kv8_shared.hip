// Attention of a batch whose sequences' first tokens lie in the same pages of the 8-bit cache.
#include "xrmm_kv8_attn.h"

namespace xrmm {

int64_t kv8_shared_workspace_bytes(const KvAttnArgs& a) {
  return a.c.B == 0 || a.max_new == 0 ? 0 : attention_plan(a, true).ws_bytes;
}

hipError_t launch_kv8_shared_attention(const KvAttnArgs& a, hipStream_t st) { return attention_launch<KV_WALK>(a, st); }

}  // namespace xrmm
