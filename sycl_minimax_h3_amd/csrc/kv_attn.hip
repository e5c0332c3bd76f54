// kv_attn.hip - kv_attention and kv_attention_work (h3lm.h) on the kernels of kv_attn_impl.h: the checks, the choice of the
// kernel and of the parts that the cache is split into, and the workspace.
#include <algorithm>
#include <cmath>

#include "kv_attn_impl.h"

namespace h3 {

// Rows: `most` tokens of a sequence times the heads that share a key/value head. Up to 32 (heads of up to 128 features) or 16 the four
// wavefronts of a block share 16 or 32 of them and the cache is read by all four (an answered token is bound by the cache's bytes);
// beyond, each has 16 or 32 rows of its own. With more rows shared, or wider heads, a wavefront holds so much that one runs on a SIMD: 16
// sequences of 4096 tokens, 8 heads, 64 rows: 65 us shared, 50 not; 32 rows 44 and 45; 32 rows of 256 features, 2048 tokens, 72 and 66.
// 32 rows of its own: where blocks of 128 rows still give each CU one and less than a quarter of their rows is none, and never for float32
// queries, whose two halves leave room for one wavefront a SIMD only (2048 tokens over 4096, 64 heads over 8 of 128: 16-bit 265 us
// with 32 rows, 356 with 16; float32 588 and 460; 64 sequences of 72 rows over 2048 tokens: 86 and 75).
// Places: a tile of rows each; as many as the rows of all sequences can lie in, where that is fewer than `most` rows of each take (one
// prompt of 8192 tokens among 1024 sequences of a token, 8 heads a key/value head: 1599 instead of 524288).
// Parts: of the same number of cache blocks for every sequence (at least eight, or four of a prompt's), as many as give each CU the two
// blocks of threads that it runs at once. (Parts beyond that, to even out sequences of different lengths, gave nothing: 64 sequences of up
// to 8192 tokens, 64 heads over 8 of 128, in 512, 1024 and 2048 blocks 133, 143 and 156 us, one of 131072 tokens 53, 57 and 62 us, and
// their merge 4, 7 and 11 us more. Longer parts: one sequence of 2000 tokens in parts of 8, 16 and 32 blocks 12.6, 15.5 and 18.5 us.)
static KvPlan kv_plan(const KvArgs& P, bool two, int64_t most, int64_t group, int64_t max_len, int64_t window, int cus) {
    KvPlan plan;
    const int64_t rows = std::min<int64_t>(most, P.rows) * group;
    auto even = [&](int64_t rt) { return (rows + rt - 1) / rt * P.seqs; };
    auto ragged = [&](int64_t rt) { return P.rows * group / rt + P.seqs; };
    plan.rows = rows > (P.dim <= 128 ? 32 : 16);
    plan.nq = plan.rows ? (two || rows <= 96 || std::min(even(128), ragged(128)) * P.heads < cus ? 1 : 2) : rows <= 16 ? 1 : 2;
    plan.rt = 16 * plan.nq * (plan.rows ? 4 : 1);
    plan.tiles = even(plan.rt) <= ragged(plan.rt) ? (rows + plan.rt - 1) / plan.rt : 0;
    plan.places = std::min(even(plan.rt), ragged(plan.rt));
    plan.blocks = plan.places * P.heads;
    int64_t keys = max_len > 0 ? std::min<int64_t>(max_len, (int64_t) P.width * kKvB) : (int64_t) P.width * kKvB;
    if (window > 0) keys = std::min(keys, std::min<int64_t>(window, INT32_MAX) + std::min<int64_t>(most, P.rows) + 2 * kKvB);
    const int64_t blocks = std::max<int64_t>((keys + kKvB - 1) / kKvB, 1), least = plan.rows ? 4 : 8;
    const int64_t want = std::max<int64_t>(1, std::min<int64_t>(2 * (int64_t) cus / std::max<int64_t>(plan.blocks, 1), 512));
    plan.per = (int) std::max(least, (blocks + want - 1) / want);
    plan.nsplit = (int) ((blocks + plan.per - 1) / plan.per);
    return plan;
}
// The launches of a call, one or two. Where some sequences can have many rows and others few (prompts beside answered tokens), those with up
// to 16 (or 32: larger groups) are a launch of the shared-rows kernel if that splits their caches further: a prompt of 2048 tokens
// beside a token over 131072, 64 heads over 8 of 128, 3469 us in one launch, 191 in two (129 and 49 by themselves); four prompts of 241 to 600
// tokens behind up to 900, for which the second finds nothing to do, 70 and 69.
static int kv_plans(const KvArgs& P, bool two, int64_t most, int64_t group, int64_t max_len, int64_t window, int cus, KvPlan (&plan)[2]) {
    plan[0] = kv_plan(P, two, most, group, max_len, window, cus);
    const int64_t few = (group <= 16 ? 16 : 32) / group;                         // tokens
    if (!plan[0].rows || few == 0 || (group > 16 && P.dim > 128) || std::min<int64_t>(most, P.rows) * P.seqs <= P.rows) return 1;
    plan[1] = kv_plan(P, two, few, group, max_len, window, cus);
    if (plan[1].nsplit <= plan[0].nsplit) return 1;
    plan[1].greatest = (uint32_t) (few * group);
    plan[0].least = plan[1].greatest + 1;
    return 2;
}
static int64_t kv_part_floats(const KvPlan& plan, int64_t W) { return plan.nsplit > 1 ? plan.blocks * plan.nsplit * plan.rt * (W + 2) : 0; }

static int attn_checks(const char* fn, const KvArgs& P, int64_t max_len, int64_t q_heads, int64_t window) {
    if (q_heads <= 0 || q_heads % P.heads != 0) return fail(std::string(fn) + ": the query heads must be a multiple of the key/value heads");
    if (q_heads > 65535) return fail(std::string(fn) + ": too many heads");
    if (max_len < 0 || window < 0) return fail(std::string(fn) + ": a negative length or window");
    if ((int64_t) P.rows * (q_heads / P.heads) > INT32_MAX) return fail(std::string(fn) + ": too many rows");
    return 0;
}

int64_t kv_attention_work(void* ctx, const h3_kv_cache* cache, const h3_kv_batch* batch, int64_t max_len, int64_t q_heads, int64_t window) try {
    const char* fn = "kv_attention_work";
    KvArgs P;
    if (kv_args(fn, cache, batch, P) || attn_checks(fn, P, max_len, q_heads, window)) return -1;
    Ctx* c = ctx_of(ctx, fn);
    if (!c) return -1;
    if (P.seqs == 0 || P.rows == 0 || batch->most == 0) return 0;
    // (the more of what 16-bit and float32 queries take)
    int64_t floats = 0;
    for (bool two : {false, true}) {
        KvPlan plan[2];
        int64_t sum = 0;
        for (int n = kv_plans(P, two, batch->most, q_heads / P.heads, max_len, window, c->cus, plan); n-- > 0;) sum += kv_part_floats(plan[n], kv_width(P.dim));
        floats = std::max(floats, sum);
    }
    return 4 * floats;
} catch (const std::exception& e) { return fail(e.what()); }

int kv_attention(void* ctx, const h3_kv_cache* cache, const h3_kv_batch* batch, const int32_t* lengths, int64_t max_len, const void* q,
                 int64_t q_stride, int dt, int64_t q_heads, float scale, int64_t window, const uint8_t* mask, int64_t mask_stride,
                 void* out, int out_dt, float* lse, void* work, uint64_t work_bytes) try {
    const char* fn = "kv_attention";
    KvAttnArgs A;
    if (kv_args(fn, cache, batch, A.kv) || attn_checks(fn, A.kv, max_len, q_heads, window)) return -1;
    if (!dt_ok(dt) || !dt_ok(out_dt)) return fail(std::string(fn) + ": unknown element type");
    if (!(scale >= 0.0f) || std::isinf(scale)) return fail(std::string(fn) + ": the scale must be a number above 0 (or 0: 1 / sqrt(dim))");
    if (mask && mask_stride < 0) return fail(std::string(fn) + ": a negative mask stride");
    if (A.kv.seqs == 0 || A.kv.rows == 0 || batch->most == 0) return 0;
    const int64_t dim = A.kv.dim;
    if (q_stride < q_heads * dim) return fail(std::string(fn) + ": the row stride is shorter than a row");
    if (!lengths || !q || !out) return fail(std::string(fn) + ": lengths, q and out are required");
    if (work && !aligned16(work)) return fail(std::string(fn) + ": the workspace must be 16-byte aligned");
    const int64_t group = q_heads / A.kv.heads;
    Ctx* c = ctx_of(ctx, fn);
    if (!c) return -1;
    const bool two = dt == H3S_F32;
    KvPlan plans[2];
    const int launches = kv_plans(A.kv, two, batch->most, group, max_len, window, c->cus, plans);
    const int64_t W = kv_width(dim);
    int64_t floats = 0;
    for (int i = 0; i < launches; ++i) {
        // (the merge has a block of threads a row)
        if (plans[i].blocks > kKvMostBlocks || plans[i].blocks * (plans[i].nsplit > 1 ? std::max(plans[i].nsplit, plans[i].rt) : 1) > kKvMostBlocks)
            return fail(std::string(fn) + ": too many blocks of work");
        floats += kv_part_floats(plans[i], W);
    }
    float* parts = nullptr;
    if (floats) {
        if (work) {
            if (work_bytes < (uint64_t) (4 * floats)) return fail(std::string(fn) + ": the workspace is smaller than kv_attention_work() says");
            parts = (float*) work;
        } else {
            hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
            if (hipStreamIsCapturing(c->stream, &st) != hipSuccess) (void) hipGetLastError();
            if (st != hipStreamCaptureStatusNone) return fail(std::string(fn) + ": a call recorded into a graph needs a workspace of its own");
            parts = c->scratch<float>(Ctx::KV_PART, (size_t) floats);
            if (!parts) return -1;
        }
    }
    A.lengths = lengths;
    A.q = q; A.q_stride = q_stride; A.q_dt = dt; A.group = (int) group; A.q_heads = (int) q_heads;
    A.scale = (float) ((scale > 0.0f ? (double) scale : 1.0 / std::sqrt((double) dim)) * 1.4426950408889634);
    A.window = (int) std::min<int64_t>(window, INT32_MAX / 2);
    A.mask = mask; A.mask_stride = mask_stride;
    A.out = out; A.out_dt = out_dt; A.lse = lse;
    A.q_vec = aligned16(q) && dim % 8 == 0 && (q_stride * elem_size(dt)) % 16 == 0;
    A.out_vec = aligned16(out) && dim % 4 == 0;
    A.mask_vec = mask && aligned16(mask) && mask_stride % 16 == 0;
    for (int i = 0; i < launches; ++i) {
        const KvPlan& plan = plans[i];
        A.tiles = (int) plan.tiles; A.places = (int) plan.places; A.nsplit = plan.nsplit; A.per = plan.per;
        A.least = plan.least; A.greatest = plan.greatest;
        A.po = parts;
        A.pml = parts ? parts + plan.blocks * plan.nsplit * plan.rt * W : nullptr;
        if (parts) parts += kv_part_floats(plan, W);
        switch (W / 64) {
            case 1: kv_attn_64(c, A, plan, two); break;
            case 2: kv_attn_128(c, A, plan, two); break;
            case 3: kv_attn_192(c, A, plan, two); break;
            default: kv_attn_256(c, A, plan, two); break;
        }
    }
    return launched(fn);
} catch (const std::exception& e) { return fail(e.what()); }

}  // namespace h3
