// kv.h - what the key/value cache's translation units share (h3lm.h): the arguments of the kernels and the host's checks.
#pragma once

#include "../../include/h3lm.h"
#include "common.h"

namespace h3 {

constexpr int kKvB = H3_KV_BLOCK;                               // tokens a block
inline int64_t kv_width(int64_t dim) { return (dim + 63) / 64 * 64; }   // a head's features as the codes hold them

// the cache and the batch as the kernels take them
struct KvArgs {
    int8_t *k, *v;
    float *ks, *vs;
    int64_t blocks;
    int heads, dim;
    const int32_t *table, *starts;
    int width, seqs, rows;
};

// the rows [r0, r0 + n) of sequence b, within the call's rows whatever `starts` says
__device__ __forceinline__ void kv_rows_of(const KvArgs& P, int b, int& r0, int& n) {
    const int a = P.starts[b], e = P.starts[b + 1];
    r0 = min(max(a, 0), P.rows);
    n = min(max(e, r0), P.rows) - r0;
}

// The blocks of 256 threads that one launch takes: a launch of 2^32 threads or more is cut without an error.
constexpr int64_t kKvMostBlocks = 0xffffff;

// Work laid out by the rows there are, for batches where `most` rows of every sequence would be far more: sequence b's items begin at
// floor(start * num / den) + each * b, and the last sequence that begins at or before item `at` has it. Found by the whole wavefront, 64
// sequences at a time (up to 63 sequences: one load, which the rows need anyway). Returns the item's number in its sequence b,
// whose rows are [r0, r0 + n); below 0 where the item is nobody's (rows before the first sequence). Whatever `starts` says, b is a
// sequence and the rows are within the call's.
__device__ __forceinline__ int kv_find(const KvArgs& P, int at, uint32_t num, uint32_t den, int each, int& b, int& r0, int& n) {
    const int lane = threadIdx.x & 63;
    int step = 1;                                                           // (fewer sequences than kKvMostBlocks: 64 step is an int)
    while (step * 64 < P.seqs) step *= 64;
    for (b = 0;; step /= 64) {
        const int c = b + lane * step;
        const int s = min(max(P.starts[min(c, P.seqs)], 0), P.rows);
        const int first = (int) ((uint32_t) s * num / den) + each * min(c, P.seqs);
        const int k = (int) __popcll(__ballot(c < P.seqs && first <= at) & ~1ull);   // (lane 0 is where none is)
        b += k * step;
        if (step > 1) continue;
        r0 = __builtin_amdgcn_readlane(s, k);
        n = min(max(k < 63 ? __builtin_amdgcn_readlane(s, k + 1) : P.starts[b + 1], r0), P.rows) - r0;
        return at - __builtin_amdgcn_readlane(first, k);
    }
}

// checks cache and batch and fills P: 0, or -1 with the reason
int kv_args(const std::string& fn, const h3_kv_cache* cache, const h3_kv_batch* batch, KvArgs& P);

int kv_write(void* ctx, const h3_kv_cache* cache, const h3_kv_batch* batch, const int32_t* past, const void* k, int64_t k_stride,
             const void* v, int64_t v_stride, int dt);
int kv_read(void* ctx, const h3_kv_cache* cache, const h3_kv_batch* batch, const int32_t* first, void* k, int64_t k_stride, void* v,
            int64_t v_stride, int dt);
int kv_attention(void* ctx, const h3_kv_cache* cache, const h3_kv_batch* batch, const int32_t* lengths, int64_t max_len, const void* q,
                 int64_t q_stride, int dt, int64_t q_heads, float scale, int64_t window, const uint8_t* mask, int64_t mask_stride,
                 void* out, int out_dt, float* lse, void* work, uint64_t work_bytes);
int64_t kv_attention_work(void* ctx, const h3_kv_cache* cache, const h3_kv_batch* batch, int64_t max_len, int64_t q_heads, int64_t window);
int kv_attention_spans(void* ctx, const h3_kv_cache* cache, const h3_kv_batch* batch, const h3_kv_shared* shared, const int32_t* lengths,
                       int64_t max_len, const void* q, int64_t q_stride, int dt, int64_t q_heads, float scale, int64_t window, int64_t sinks,
                       const uint8_t* mask, int64_t mask_stride, void* out, int out_dt, float* lse, void* work, uint64_t work_bytes);
int64_t kv_attention_spans_work(void* ctx, const h3_kv_cache* cache, const h3_kv_batch* batch, const h3_kv_shared* shared, int64_t max_len,
                                int64_t q_heads, int64_t window, int64_t sinks);
int linear4(void* ctx, const void* x, int dt, int64_t M, int64_t K, const uint8_t* codes, int64_t N, const void* scale, const void* mins,
            int scale_dt, int64_t group, const float* bias, void* out, int out_dt);

// element i of a float tensor of runtime type
__device__ __forceinline__ float load_any(const void* p, int dt, int64_t i) {
    if (dt == H3S_F32) return ((const float*) p)[i];
    const uint16_t u = ((const uint16_t*) p)[i];
    return dt == H3S_BF16 ? bf16_lo(u) : f16_lo(u);
}
__device__ __forceinline__ void store_any(void* p, int dt, int64_t i, float v) {
    if (dt == H3S_F32) ((float*) p)[i] = v;
    else if (dt == H3S_BF16) ((uint16_t*) p)[i] = (uint16_t) pack_bf16(v, 0.0f);
    else ((uint16_t*) p)[i] = (uint16_t) pack_f16(v, 0.0f);
}

}  // namespace h3
