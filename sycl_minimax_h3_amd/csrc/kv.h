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
