// kv_attn.hip - kv_attention and kv_attention_spans with the sizes of their workspaces (h3lm.h) on the kernels of kv_attn_impl.h: the checks,
// the choice of the kernel and of the parts that the cache is split into, and the workspace.
#include <algorithm>
#include <cmath>

#include "kv_attn_impl.h"

namespace h3 {

// What decides the plans beside the batch: the heads of a group, about the longest length, the window, and (kv_attention_spans) the first tokens
// that stay visible, the groups of sequences and about the longest of their shared tokens.
struct KvSight {
    int64_t group, max_len, window, sinks, groups, shared;
    bool spans() const { return sinks > 0 || groups > 0; }
    int64_t seen() const { return window > 0 ? window + sinks : INT64_MAX / 2; }   // tokens, by a row at most
};

// The rows' kernel of kv_attention_spans: its tiles and parts by an estimate of the time, in microseconds. Where the device is full, a cache block
// takes a tile of 128 rows 3.2 and one of 64 rows 2.2 (heads of 128, 16-bit queries; more features and float32 queries in proportion), a
// part's beginning and end about two more; a last round of at most a block of threads a CU goes faster by 0.7; parts are written and read at
// 5 TB/s, and joined by a launch (or taken up by the sequences' own: 0.6 each). About 80 rows of each of 18 sequences over 7000 tokens, 8
// heads of 96: 188 us in tiles and parts as kv_attention's, 98 so.
// tiles(rt): tiles of a head; join: 0 where the parts are taken up by another launch.
template <typename F>
static void kv_rows_plan(KvPlan& plan, F tiles, int64_t rows, int64_t heads, int64_t dim, int64_t blocks, bool two, int cus, double join, bool fine = false) {
    const int wc = (int) (kv_width(dim) / 64);
    const int64_t a_cu = wc == 1 ? 3 : wc == 2 ? 2 : 1, slots = a_cu * cus;
    plan.cost = 1e300;
    for (int nq = 1; nq <= (two || fine ? 1 : 2); ++nq) {
        const int64_t real = tiles(64 * nq) * heads;
        const double step = (nq == 2 ? 3.2 : 2.2) * (two ? 1.6 : fine ? 1.3 : 1.0) * (wc + 0.3) / 2.3 * (double) a_cu / 2;
        for (int64_t n = 1; n <= std::min<int64_t>(blocks, 64); ++n) {
            const int64_t per = (blocks + n - 1) / n, rest = real * n % slots;
            const double rounds = (double) (real * n / slots) + (rest == 0 ? 0.0 : rest <= cus && a_cu > 1 ? 0.7 : 1.0);
            const double parts = n > 1 || join == 0.0 ? (double) n * rows * heads * dim * 8.0 / 5e6 : 0.0;
            const double cost = rounds * (per + 2) * step + parts + (join == 0.0 ? 0.6 * n : n > 1 ? join : 0.0);
            if (cost < plan.cost) { plan.cost = cost; plan.nq = nq; plan.per = (int) per; }
        }
    }
    plan.rt = 64 * plan.nq;
    plan.nsplit = (int) ((blocks + plan.per - 1) / plan.per);
}

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
static KvPlan kv_plan(const KvArgs& P, bool two, int64_t most, const KvSight& sight, int cus, bool fine = false, bool tiles16 = false) {
    const int64_t group = sight.group, max_len = sight.max_len, window = sight.window;
    KvPlan plan;
    const int64_t rows = std::min<int64_t>(most, P.rows) * group;
    auto even = [&](int64_t rt) { return (rows + rt - 1) / rt * P.seqs; };
    auto ragged = [&](int64_t rt) { return P.rows * group / rt + P.seqs; };
    plan.rows = rows > (P.dim <= 128 ? 32 : 16);
    plan.fine = plan.rows && fine;
    int64_t keys = max_len > 0 ? std::min<int64_t>(max_len, (int64_t) P.width * kKvB) : (int64_t) P.width * kKvB;
    if (sight.groups) keys = std::max<int64_t>(keys - sight.shared, std::min<int64_t>(most, P.rows));
    if (window > 0) keys = std::min(keys, sight.seen() + std::min<int64_t>(most, P.rows) + 2 * kKvB);
    if (plan.rows && sight.spans()) {
        // (sequences have as many rows on average, and half a tile more, but none more tiles than the longest; a tile sees its window)
        const int64_t all = P.rows * group;
        auto tiles = [&](int64_t rt) { return std::max(std::min(all / rt + P.seqs / 2, (rows + rt - 1) / rt * P.seqs), (int64_t) P.seqs); };
        if (window > 0) keys = std::min<int64_t>(keys, sight.seen() + 128 / group + 2 * kKvB);
        kv_rows_plan(plan, tiles, all, P.heads, P.dim, std::max<int64_t>((keys + kKvB - 1) / kKvB, 1), two, cus, 6.0, fine);
        plan.tiles = even(plan.rt) <= ragged(plan.rt) ? (rows + plan.rt - 1) / plan.rt : 0;
        plan.places = std::min(even(plan.rt), ragged(plan.rt));
        plan.blocks = plan.places * P.heads;
        return plan;
    }
    plan.nq = plan.rows ? (two || fine || rows <= 96 || std::min(even(128), ragged(128)) * P.heads < cus ? 1 : 2) : rows <= 16 || tiles16 ? 1 : 2;
    plan.rt = 16 * plan.nq * (plan.rows ? 4 : 1);
    plan.tiles = even(plan.rt) <= ragged(plan.rt) ? (rows + plan.rt - 1) / plan.rt : 0;
    plan.places = std::min(even(plan.rt), ragged(plan.rt));
    plan.blocks = plan.places * P.heads;
    const int64_t blocks = std::max<int64_t>((keys + kKvB - 1) / kKvB, 1), least = plan.rows ? 4 : 8;
    const int64_t parted = tiles16 ? (int64_t) P.seqs * P.heads : plan.blocks;   // (few have a second tile)
    const int64_t want = std::max<int64_t>(1, std::min<int64_t>(2 * (int64_t) cus / std::max<int64_t>(parted, 1), 512));
    plan.per = (int) std::max(least, (blocks + want - 1) / want);
    // (with first or shared tokens: up to 12 blocks are one part, a third step of the wavefronts for the 4 us of a merge: four sequences of 612
    // tokens, 64 heads over 8 of 128, 15 to 11 us)
    if (sight.spans() && !plan.rows && blocks <= 12) plan.per = 12;
    plan.nsplit = (int) ((blocks + plan.per - 1) / plan.per);
    return plan;
}
// The launches of a call, one or two. Where some sequences can have many rows and others few (prompts beside answered tokens), those with up
// to 16 (or 32: larger groups) are a launch of the shared-rows kernel if that splits their caches further: a prompt of 2048 tokens
// beside a token over 131072, 64 heads over 8 of 128, 3469 us in one launch, 191 in two (129 and 49 by themselves); four prompts of 241 to 600
// tokens behind up to 900, for which the second finds nothing to do, 70 and 69.
// fine (16-bit queries, results that are not bfloat16): sequences of few rows have probabilities as two halves whatever stands beside them. Where
// none is longer than kKvHalves rows and the others have up to a tile (kKvBeside) on average, the rows' kernel has them so for all; else a
// second launch has all sequences of up to 32 rows (16 of wide heads), in tiles of 16 where most have no more, as tiles of 32 leave a SIMD one
// wavefront. float16 results, 64 heads over 8 of 128, by the rows' kernel with one half (11 bits) / with two / by two launches: 8 tokens beside seven
// answers over 8192 42, 47 and 59 us, behind a window of 1024 17, 18 and 30; 63 sequences of 4 tokens beside one of 8, over 8192, 236, 268 and
// 385; 15 of 4 beside one of 40, over 4096, 83, 93 and 108. Past the limits: 18 of 20 to 30 tokens over 7000 shared ones, 32 heads over 8 of 96, 101,
// 136 and 117; 53 of 12 to 31 over 5376, 8 over one of 80, 82, 112 and 73. bfloat16's last place does not show it.
constexpr int64_t kKvHalves = 512, kKvBeside = 64;   // rows: tokens times heads of a group
static int kv_plans(const KvArgs& P, bool two, bool fine, int64_t most, const KvSight& sight, int cus, KvPlan (&plan)[2]) {
    const int64_t group = sight.group, longest = std::min<int64_t>(most, P.rows), others = P.rows - longest;
    const bool ragged = longest * P.seqs > P.rows;
    const bool all = fine && ragged && longest * group <= kKvHalves && others * group <= kKvBeside * (P.seqs - 1);
    plan[0] = kv_plan(P, two, most, sight, cus, all);
    fine = fine && !all;                                                         // (from here on: the second launch is needed)
    const int64_t limit = fine ? (P.dim > 128 ? 16 : 32) : group <= 16 ? 16 : 32;
    const int64_t few = limit / group;                                           // tokens
    if (!plan[0].rows || few == 0 || (group > 16 && P.dim > 128) || !ragged) return 1;
    // (with first or shared tokens: where the sequences beside the longest have more rows on average, the rows' kernel takes those with few too)
    if (!fine && sight.spans() && others > 2 * few * (P.seqs - 1)) return 1;
    plan[1] = kv_plan(P, two, few, sight, cus, false, fine && group <= 16 && others * group <= 16 * (P.seqs - 1));
    if (!fine && plan[1].nsplit <= plan[0].nsplit) return 1;
    plan[1].greatest = (uint32_t) (few * group);
    plan[0].least = plan[1].greatest + 1;
    return 2;
}
// The launch of the shared tokens: all rows of a group are as one sequence's, and how many groups' rows there are is known, not each one's.
// fine: probabilities as two halves, as the few rows' kernel holds them for 16-bit queries; results of bfloat16 do not show it (48 tokens over 4096
// shared ones in six groups, 4 heads of 64: 16.8 us with one half, 17.1 so; 18 sequences of 30 tokens over 7000, 8 heads of 96, 78 and 104).
// Behind a window its parts are as long as what the rows can see (64 sequences over 8192 shared tokens, window 1024: 52 us in parts of all
// the shared blocks, 28 so).
static KvPlan kv_shared_plan(const KvArgs& P, bool two, bool fine, const KvSight& sight, int cus) {
    KvPlan plan;
    plan.shared = true;
    plan.fine = fine;
    const int64_t rows = P.rows * sight.group, each = (rows + sight.groups - 1) / sight.groups;
    auto places = [&](int64_t rt) { return rows / rt + sight.groups; };
    plan.rows = each > (P.dim <= 128 ? 32 : 16);
    const int64_t blocks = std::max<int64_t>((std::min(sight.shared, sight.seen() + 2 * kKvB) + kKvB - 1) / kKvB, 1);
    if (plan.rows) {
        kv_rows_plan(plan, [&](int64_t rt) { return std::max((rows + rt - 1) / rt, sight.groups); }, rows, P.heads, P.dim, blocks, two, cus, 0.0, fine);
        plan.tiles = 0;
        plan.places = places(plan.rt);
        plan.blocks = plan.places * P.heads;
    } else {
        plan.nq = each <= 16 ? 1 : 2;
        plan.rt = 16 * plan.nq;
        plan.tiles = 0;
        plan.places = places(plan.rt);
        plan.blocks = plan.places * P.heads;
        const int64_t want = std::max<int64_t>(1, std::min<int64_t>(2 * (int64_t) cus / std::max<int64_t>(plan.blocks, 1), 512));
        plan.per = (int) std::max<int64_t>(8, (blocks + want - 1) / want);
        plan.nsplit = (int) ((blocks + plan.per - 1) / plan.per);
    }
    return plan;
}
static int64_t kv_part_floats(const KvPlan& plan, int64_t W) {
    return plan.nsplit > 1 || plan.shared ? plan.blocks * plan.nsplit * plan.rt * (W + 2) : 0;
}

static int attn_checks(const char* fn, const KvArgs& P, int64_t max_len, int64_t q_heads, int64_t window) {
    if (q_heads <= 0 || q_heads % P.heads != 0) return fail(std::string(fn) + ": the query heads must be a multiple of the key/value heads");
    if (q_heads > 65535) return fail(std::string(fn) + ": too many heads");
    if (max_len < 0 || window < 0) return fail(std::string(fn) + ": a negative length or window");
    if ((int64_t) P.rows * (q_heads / P.heads) > INT32_MAX) return fail(std::string(fn) + ": too many rows");
    return 0;
}

// The sizes that a call with or without groups has; -1 with the reason
static int sight_of(const std::string& fn, const KvArgs& P, const h3_kv_shared* shared, int64_t max_len, int64_t q_heads, int64_t window, int64_t sinks,
                    KvSight& sight) {
    if (attn_checks(fn.c_str(), P, max_len, q_heads, window)) return -1;
    if (sinks < 0) return fail(fn + ": a negative number of first tokens");
    sight = KvSight{q_heads / P.heads, max_len, std::min<int64_t>(window, INT32_MAX), window > 0 ? std::min<int64_t>(sinks, INT32_MAX) : 0, 0, 0};
    if (!shared || shared->groups == 0) return 0;
    if (shared->groups < 0 || shared->most < 0) return fail(fn + ": a negative number of groups or shared tokens");
    if (shared->groups > kKvMostBlocks) return fail(fn + ": too many groups");   // (kv_group_of's steps of 64 stay within an int)
    if (!shared->first || !shared->tokens) return fail(fn + ": the groups' first sequences and shared tokens are required");
    sight.groups = shared->groups;
    sight.shared = shared->most > 0 ? std::min<int64_t>(shared->most, (int64_t) P.width * kKvB) : (int64_t) P.width * kKvB;
    return 0;
}
// All launches' plans: of the shared tokens first, where they have one. A launch and the reading of its sums cost 8 us or more; below so many bytes
// of all sequences' caches a CU it takes less to go through the shared ones again for each (they come from the caches of the device). Where
// sequences have many rows each, whose products bound them either way, the estimates decide: tiles of a group's rows are fuller (53
// sequences of up to 31 tokens over 5376 shared ones in 13 groups, 8 heads over one of 80: 67 us apart, 77 not; eight of up to 256 over 4096, 64
// heads over 8 of 128: 364 us apart, 355 not).
constexpr int64_t kKvApart = 192 << 10;
static int kv_all_plans(const KvArgs& P, bool two, bool fine, int64_t most, const KvSight& sight, int cus, KvPlan (&plan)[3]) {
    KvPlan own[2], behind[2], shared;
    KvSight all = sight;
    all.shared = 0;
    int n = kv_plans(P, two, fine, most, all, cus, own);
    const int64_t tokens = sight.max_len > 0 ? std::min<int64_t>(sight.max_len, (int64_t) P.width * kKvB) : (int64_t) P.width * kKvB;
    bool apart = sight.groups > 0 &&
                 std::min(std::max(tokens, sight.shared), sight.seen()) * P.seqs > cus * kKvApart / (2 * P.heads * kv_width(P.dim));
    if (apart) {
        const int m = kv_plans(P, two, fine, most, sight, cus, behind);
        // (probabilities as two halves where the sequences' own are: some have few rows)
        shared = kv_shared_plan(P, two, fine && (!behind[0].rows || behind[0].fine || m == 2), sight, cus);
        apart = !own[0].rows || shared.cost + behind[0].cost + 6.0 < own[0].cost;
        if (apart) {
            n = m;
            std::copy(behind, behind + m, own);
            plan[0] = shared;
        }
    }
    std::copy(own, own + n, plan + apart);
    return n + apart;
}

static int64_t attend_work(const char* fn, void* ctx, const h3_kv_cache* cache, const h3_kv_batch* batch, const h3_kv_shared* shared, int64_t max_len,
                           int64_t q_heads, int64_t window, int64_t sinks) {
    KvArgs P;
    KvSight sight;
    if (kv_args(fn, cache, batch, P) || sight_of(fn, P, shared, max_len, q_heads, window, sinks, sight)) return -1;
    Ctx* c = ctx_of(ctx, fn);
    if (!c) return -1;
    if (P.seqs == 0 || P.rows == 0 || batch->most == 0) return 0;
    // (the most of what float32 queries take, and 16-bit ones for 16-bit and float32 results)
    int64_t floats = 0;
    for (int type = 0; type < 3; ++type) {
        KvPlan plan[3];
        int64_t sum = 0;
        for (int n = kv_all_plans(P, type == 1, type == 2, batch->most, sight, c->cus, plan); n-- > 0;) sum += kv_part_floats(plan[n], kv_width(P.dim));
        floats = std::max(floats, sum);
    }
    return 4 * floats;
}

static int attend(const char* fn, void* ctx, const h3_kv_cache* cache, const h3_kv_batch* batch, const h3_kv_shared* shared, const int32_t* lengths,
                  int64_t max_len, const void* q, int64_t q_stride, int dt, int64_t q_heads, float scale, int64_t window, int64_t sinks,
                  const uint8_t* mask, int64_t mask_stride, void* out, int out_dt, float* lse, void* work, uint64_t work_bytes) {
    KvAttnArgs A{};
    KvSight sight;
    if (kv_args(fn, cache, batch, A.kv) || sight_of(fn, A.kv, shared, max_len, q_heads, window, sinks, sight)) return -1;
    if (!dt_ok(dt) || !dt_ok(out_dt)) return fail(std::string(fn) + ": unknown element type");
    if (!(scale >= 0.0f) || std::isinf(scale)) return fail(std::string(fn) + ": the scale must be a number above 0 (or 0: 1 / sqrt(dim))");
    if (mask && mask_stride < 0) return fail(std::string(fn) + ": a negative mask stride");
    if (A.kv.seqs == 0 || A.kv.rows == 0 || batch->most == 0) return 0;
    const int64_t dim = A.kv.dim;
    if (q_stride < q_heads * dim) return fail(std::string(fn) + ": the row stride is shorter than a row");
    if (!lengths || !q || !out) return fail(std::string(fn) + ": lengths, q and out are required");
    if (work && !aligned16(work)) return fail(std::string(fn) + ": the workspace must be 16-byte aligned");
    Ctx* c = ctx_of(ctx, fn);
    if (!c) return -1;
    const bool two = dt == H3S_F32, groups = sight.groups > 0;
    KvPlan plans[3];
    const int launches = kv_all_plans(A.kv, two, !two && out_dt != H3S_BF16, batch->most, sight, c->cus, plans);
    const int64_t W = kv_width(dim);
    int64_t floats = 0;
    for (int i = 0; i < launches; ++i) {
        // (the merge has a block of threads a row)
        const int64_t each = std::max<int64_t>(plans[i].nsplit, plans[i].nsplit > 1 ? plans[i].rt : 1);
        if (plans[i].blocks > kKvMostBlocks || plans[i].blocks * each > kKvMostBlocks) return fail(std::string(fn) + ": too many blocks of work");
        floats += kv_part_floats(plans[i], W);
    }
    float* parts = nullptr;
    if (floats) {
        if (work) {
            if (work_bytes < (uint64_t) (4 * floats)) return fail(std::string(fn) + ": the workspace is smaller than " + fn + "_work() says");
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
    A.q = q; A.q_stride = q_stride; A.q_dt = dt; A.group = (int) sight.group; A.q_heads = (int) q_heads;
    A.scale = (float) ((scale > 0.0f ? (double) scale : 1.0 / std::sqrt((double) dim)) * 1.4426950408889634);
    A.window = (int) std::min<int64_t>(window, INT32_MAX / 2);
    A.mask = mask; A.mask_stride = mask_stride;
    A.out = out; A.out_dt = out_dt; A.lse = lse;
    A.q_vec = aligned16(q) && dim % 8 == 0 && (q_stride * elem_size(dt)) % 16 == 0;
    A.out_vec = aligned16(out) && dim % 4 == 0;
    A.mask_vec = mask && aligned16(mask) && mask_stride % 16 == 0;
    A.sinks = (int) std::min<int64_t>(sight.sinks, INT32_MAX / 2);
    if (groups) { A.first = shared->first; A.shared = shared->tokens; A.groups = (int) sight.groups; }
    for (int i = 0; i < launches; ++i) {
        const KvPlan& plan = plans[i];
        A.tiles = (int) plan.tiles; A.places = (int) plan.places; A.nsplit = plan.nsplit; A.per = plan.per;
        A.least = plan.least; A.greatest = plan.greatest;
        A.po = parts;
        A.pml = parts ? parts + plan.blocks * plan.nsplit * plan.rt * W : nullptr;
        if (parts) parts += kv_part_floats(plan, W);
        const bool first = plan.shared;
        if (groups || A.sinks > 0) {
            switch (W / 64) {
                case 1: kv_spans_64(c, A, plan, two, first); break;
                case 2: kv_spans_128(c, A, plan, two, first); break;
                case 3: kv_spans_192(c, A, plan, two, first); break;
                default: kv_spans_256(c, A, plan, two, first); break;
            }
        } else {
            switch (W / 64) {
                case 1: kv_attn_64(c, A, plan, two); break;
                case 2: kv_attn_128(c, A, plan, two); break;
                case 3: kv_attn_192(c, A, plan, two); break;
                default: kv_attn_256(c, A, plan, two); break;
            }
        }
        if (first) { A.rt2 = plan.rt; A.nsplit2 = plan.nsplit; A.po2 = A.po; A.pml2 = A.pml; }
    }
    return launched(fn);
}

int64_t kv_attention_work(void* ctx, const h3_kv_cache* cache, const h3_kv_batch* batch, int64_t max_len, int64_t q_heads, int64_t window) try {
    return attend_work("kv_attention_work", ctx, cache, batch, nullptr, max_len, q_heads, window, 0);
} catch (const std::exception& e) { return fail(e.what()); }

int kv_attention(void* ctx, const h3_kv_cache* cache, const h3_kv_batch* batch, const int32_t* lengths, int64_t max_len, const void* q,
                 int64_t q_stride, int dt, int64_t q_heads, float scale, int64_t window, const uint8_t* mask, int64_t mask_stride,
                 void* out, int out_dt, float* lse, void* work, uint64_t work_bytes) try {
    return attend("kv_attention", ctx, cache, batch, nullptr, lengths, max_len, q, q_stride, dt, q_heads, scale, window, 0, mask, mask_stride, out, out_dt,
                  lse, work, work_bytes);
} catch (const std::exception& e) { return fail(e.what()); }

int64_t kv_attention_spans_work(void* ctx, const h3_kv_cache* cache, const h3_kv_batch* batch, const h3_kv_shared* shared, int64_t max_len,
                                int64_t q_heads, int64_t window, int64_t sinks) try {
    return attend_work("kv_attention_spans_work", ctx, cache, batch, shared, max_len, q_heads, window, sinks);
} catch (const std::exception& e) { return fail(e.what()); }

int kv_attention_spans(void* ctx, const h3_kv_cache* cache, const h3_kv_batch* batch, const h3_kv_shared* shared, const int32_t* lengths,
                       int64_t max_len, const void* q, int64_t q_stride, int dt, int64_t q_heads, float scale, int64_t window, int64_t sinks,
                       const uint8_t* mask, int64_t mask_stride, void* out, int out_dt, float* lse, void* work, uint64_t work_bytes) try {
    return attend("kv_attention_spans", ctx, cache, batch, shared, lengths, max_len, q, q_stride, dt, q_heads, scale, window, sinks, mask, mask_stride, out,
                  out_dt, lse, work, work_bytes);
} catch (const std::exception& e) { return fail(e.what()); }

}  // namespace h3
