// lin.h - what the linear attention's translation units share (h3lm.h, lin_attention): the kernels' arguments.
#pragma once

#include "kv.h"

namespace h3 {

struct LinArgs {
    float* s;                                       // [slots, heads, dk, dv]
    int64_t slots;
    int heads, dk, dv;
    KvArgs kv;                                      // of it starts, seqs and rows
    const int32_t *source, *target;
    const float* decay;
    const void *q, *k, *v;
    int64_t q_stride, k_stride, v_stride;
    int q_each, k_each, v_each;                     // heads of the states that read one of theirs
    int dt;
    float scale;
    void* out;
    int out_dt;
    uint32_t least, most;                           // sequences of fewer or more rows are another launch's
    int slices, seg;                                // in pieces: ranges of v's features, tokens of a segment
    float* ws;                                      // the segments' sums, then their first states, one for each block of threads
    bool vec, s_vec;                                // rows of q, k, v and out, and states, that can be read and written 16 bytes at a time
};

int lin_attention(void* ctx, const h3_lin_state* state, const h3_lin_batch* batch, const float* decay, const void* q, int64_t q_stride,
                  int64_t q_heads, const void* k, int64_t k_stride, int64_t k_heads, const void* v, int64_t v_stride, int64_t v_heads,
                  int dt, float scale, void* out, int out_dt, void* work, uint64_t work_bytes);
int64_t lin_attention_work(void* ctx, const h3_lin_state* state, const h3_lin_batch* batch, int dt);

}  // namespace h3
