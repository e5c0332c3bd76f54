// kv_spans_128.hip - kv_attn_impl.h's kernels of kv_attention_spans for heads of up to 128 features
#include "kv_attn_impl.h"

namespace h3 {
void kv_spans_128(Ctx* c, const KvAttnArgs& P, const KvPlan& plan, bool two, bool shared) {
    if (shared) kv_attn_width<2, kKvShared>(c, P, plan, two);
    else kv_attn_width<2, kKvOwn>(c, P, plan, two);
}
}  // namespace h3
