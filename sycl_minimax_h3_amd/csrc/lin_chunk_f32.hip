// lin_chunk_f32.hip - lin_chunk_impl.h's kernels for inputs of type H3S_F32
#include "lin_chunk_impl.h"

namespace h3 {
void lin_chunk_f32(Ctx* c, const LinArgs& P, int kc, bool wide, int64_t blocks, bool out) { lin_chunk_type<H3S_F32>(c, P, kc, wide, blocks, out); }
}  // namespace h3
