// linear4_f32.hip - linear4_impl.h's kernels for x of type H3S_F32
#include "linear4_impl.h"

namespace h3 {
void l4_f32(Ctx* c, const L4Args& P) { l4_type<H3S_F32>(c, P); }
}  // namespace h3
