// lin_chunk_f16.hip - lin_chunk_impl.h's kernels for inputs of type H3S_F16
#include "lin_chunk_impl.h"

namespace h3 {
void lin_chunk_f16(Ctx* c, const LinArgs& P, int kc, int nv, int64_t blocks, bool out) { lin_chunk_type<H3S_F16>(c, P, kc, nv, blocks, out); }
}  // namespace h3
