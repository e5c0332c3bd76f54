// linear4_bf16.hip - linear4_impl.h's kernels for x of type H3S_BF16
#include "linear4_impl.h"

namespace h3 {
void l4_bf16(Ctx* c, const L4Args& P) { l4_type<H3S_BF16>(c, P); }
}  // namespace h3
