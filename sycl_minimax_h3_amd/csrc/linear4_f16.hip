// linear4_f16.hip - linear4_impl.h's kernels for x of type H3S_F16
#include "linear4_impl.h"

namespace h3 {
void l4_f16(Ctx* c, const L4Args& P) { l4_type<H3S_F16>(c, P); }
}  // namespace h3
