// kv_attn_128.hip - kv_attn_impl.h's kernels for heads of up to 128 features
#include "kv_attn_impl.h"

namespace h3 {
void kv_attn_128(Ctx* c, const KvAttnArgs& P, const KvPlan& plan, bool two) { kv_attn_width<2>(c, P, plan, two); }
}  // namespace h3
