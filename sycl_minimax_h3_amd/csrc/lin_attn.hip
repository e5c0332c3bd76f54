// lin_attn.hip - lin_attention and lin_attention_work (h3lm.h): the checks, the choice of the kernel, and the form for few tokens.
//
// Mathematics, for one head of one sequence: S = exp(-decay) S + k v^T and out = scale q S, token by token. A column of S meets only its
// own feature of v, so the features of v are split over blocks of threads without an exchange between them.
#include <algorithm>
#include <cmath>

#include "lin_chunk_impl.h"

namespace h3 {

constexpr int kLinCols = 32;                        // columns of S that a block of threads takes: 128 bytes of each row
constexpr int kLinToks = 8;                         // tokens whose rows lie in LDS at once

// Few tokens: a block of 256 threads holds 32 columns of a head's state in registers, rows r + 32 i and four columns a thread, over all
// tokens of the sequence. A token's sum over the rows of S is left as 32 parts in LDS and added up once for up to eight tokens. exp(-decay) is
// applied as S - (1 - exp(-decay)) S: a decay near 1 is held to 32 bits of its distance from 1, which is what far tokens' weights
// depend on. Bound by the state's bytes, read and written once (64 sequences, 64 heads of 128 x 128: 106 us, 5.1 TB/s, other states each pass).
template <int DKR, bool VEC>
__global__ __launch_bounds__(256) void lin_step_kernel(LinArgs P) {
    constexpr int K = 32 * DKR;
    __shared__ float sq[kLinToks][K], sk[kLinToks][K], sv[kLinToks][kLinCols];
    __shared__ float4 part[kLinToks][4][8];
    uint32_t id = blockIdx.x;
    const uint32_t slices = (uint32_t) (P.dv + kLinCols - 1) / kLinCols;
    const int c0 = (int) (id % slices) * kLinCols;
    id /= slices;
    const int h = (int) (id % (uint32_t) P.heads), b = (int) (id / (uint32_t) P.heads);
    int r0, n;
    kv_rows_of(P.kv, b, r0, n);
    if (n == 0 || (uint32_t) n < P.least || (uint32_t) n > P.most) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int c = c0 + 4 * (threadIdx.x & 7), r = threadIdx.x >> 3;
    const int64_t from = P.source[b], to = P.target[b];
    const int64_t head = (int64_t) P.dk * P.dv;
    float s[DKR][4];
    const bool begun = from >= 0 && from < P.slots;
    const float* sp = P.s + ((begun ? from : 0) * P.heads + h) * head;
#pragma unroll
    for (int i = 0; i < DKR; ++i) {
        const int row = r + 32 * i;
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][j] = 0.0f;
        if (!begun || row >= P.dk) continue;
        if constexpr (VEC) {
            if (c < P.dv) load_f32x(sp + (int64_t) row * P.dv + c, s[i], 4);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (c + j < P.dv) s[i][j] = sp[(int64_t) row * P.dv + c + j];
        }
    }
    const float less = expm1f(-P.decay[h]);          // exp(-decay) - 1
    const int64_t qo = (int64_t) (h / P.q_each) * P.dk, ko = (int64_t) (h / P.k_each) * P.dk, vo = (int64_t) (h / P.v_each) * P.dv + c0;
    for (int t0 = 0; t0 < n; t0 += kLinToks) {
        const int toks = min(n - t0, kLinToks);
        if (t0) __syncthreads();
        for (int i = threadIdx.x; i < toks * K; i += 256) {
            const int t = i / K, d = i % K;
            const int64_t row = (int64_t) r0 + t0 + t;
            sq[t][d] = d < P.dk ? load_any(P.q, P.dt, row * P.q_stride + qo + d) : 0.0f;
            sk[t][d] = d < P.dk ? load_any(P.k, P.dt, row * P.k_stride + ko + d) : 0.0f;
        }
        if ((int) threadIdx.x < toks * kLinCols) {
            const int t = threadIdx.x / kLinCols, d = threadIdx.x % kLinCols;
            sv[t][d] = c0 + d < P.dv ? load_any(P.v, P.dt, ((int64_t) r0 + t0 + t) * P.v_stride + vo + d) : 0.0f;
        }
        __syncthreads();
        for (int t = 0; t < toks; ++t) {
            const float4 v = *reinterpret_cast<const float4*>(&sv[t][4 * (threadIdx.x & 7)]);
            float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            const float vv[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int i = 0; i < DKR; ++i) {
                const float kd = sk[t][r + 32 * i], qd = sq[t][r + 32 * i];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    s[i][j] = __builtin_fmaf(kd, vv[j], __builtin_fmaf(s[i][j], less, s[i][j]));
                    y[j] = __builtin_fmaf(qd, s[i][j], y[j]);
                }
            }
            // over the wavefront's eight rows
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                y[j] += xor_lane<8>(y[j]);
                y[j] += xor_lane<16>(y[j]);
                y[j] += xor_lane<32>(y[j]);
            }
            if (lane < 8) part[t][wave][lane] = make_float4(y[0], y[1], y[2], y[3]);
        }
        __syncthreads();
        if ((int) threadIdx.x < toks * kLinCols) {
            const int t = threadIdx.x / kLinCols, d = threadIdx.x % kLinCols;
            const float* p = reinterpret_cast<const float*>(&part[t][0][0]) + d;
            const float y = (p[0] + p[32]) + (p[64] + p[96]);
            if (c0 + d < P.dv) store_any(P.out, P.out_dt, (((int64_t) r0 + t0 + t) * P.heads + h) * P.dv + c0 + d, y * P.scale);
        }
    }
    if (to < 0 || to >= P.slots) return;
    float* tp = P.s + (to * P.heads + h) * head;
#pragma unroll
    for (int i = 0; i < DKR; ++i) {
        const int row = r + 32 * i;
        if (row >= P.dk) continue;
        if constexpr (VEC) {
            if (c < P.dv) *reinterpret_cast<float4*>(tp + (int64_t) row * P.dv + c) = make_float4(s[i][0], s[i][1], s[i][2], s[i][3]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (c + j < P.dv) tp[(int64_t) row * P.dv + c + j] = s[i][j];
        }
    }
}

// The states at the segments' beginnings, where their own sums were: a thread has 16 bytes of a state through all segments of a sequence.
// (Blocks: a sixteen-row piece of a state in the chunk kernel's own layout, of a head, slice and sequence.) Bound by a walk's latency: 64
// heads of 128 x 128 in eight segments, 64 MB, 12 us.
template <int KC, int NW, int NV>
__global__ __launch_bounds__(64 * NW) void lin_scan_kernel(LinArgs P) {
    constexpr int FR = 2 * KC * NV, T = 64 * NW;
    uint32_t id = blockIdx.x;
    const int fr = (int) (id % FR), t = fr / NV, x = fr % NV;
    id /= FR;
    const int h = (int) (id % (uint32_t) P.heads);
    id /= (uint32_t) P.heads;
    const int slice = (int) (id % (uint32_t) P.slices), b = (int) (id / (uint32_t) P.slices);
    int r0, n;
    kv_rows_of(P.kv, b, r0, n);
    const int segs = (int) (((uint32_t) n + (uint32_t) P.seg - 1) / (uint32_t) P.seg);
    if (segs < 2 || (uint32_t) n < P.least || (uint32_t) n > P.most) return;
    const int lane = threadIdx.x & 63, l15 = lane & 15, g = lane >> 4, wave = threadIdx.x >> 6;
    const int c = slice * 16 * NW * NV + (wave * NV + x) * 16 + l15;
    const int64_t from = P.source[b];
    v4f_lin s = {0.0f, 0.0f, 0.0f, 0.0f};
    if (from >= 0 && from < P.slots && c < P.dv) {
        const float* sp0 = P.s + (from * P.heads + h) * ((int64_t) P.dk * P.dv);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = 16 * (t & ~1) + 8 * g + 4 * (t & 1) + i;
            if (d < P.dk) s[i] = sp0[(int64_t) d * P.dv + c];
        }
    }
    const float less = expm1f(-P.decay[h] * (float) P.seg);
    const int64_t place = r0 / P.seg + b, step = (int64_t) P.slices * P.heads * (FR * T * 4);
    float* ws = P.ws + ((place * P.slices + slice) * P.heads + h) * (FR * T * 4) + fr * (T * 4) + threadIdx.x * 4;
    // (eight segments' sums are on their way at once: one after another their latency is all there is)
    constexpr int A = 8;
    v4f_lin own[A];
    for (int j0 = 0; j0 < segs; j0 += A, ws += A * step) {
#pragma unroll
        for (int j = 0; j < A; ++j) own[j] = j0 + j + 1 < segs ? *reinterpret_cast<const v4f_lin*>(ws + j * step) : v4f_lin{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < A; ++j) {
            if (j0 + j >= segs) break;
            *reinterpret_cast<v4f_lin*>(ws + j * step) = s;
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] = __builtin_fmaf(s[i], less, s[i]) + own[j][i];
        }
    }
}

template <int KC, bool WIDE> static void lin_scan_run(Ctx* c, const LinArgs& P) {
    constexpr int NW = LinWaves<KC, WIDE>::NW, NV = LinWaves<KC, WIDE>::NV;
    lin_scan_kernel<KC, NW, NV><<<(unsigned) ((int64_t) P.kv.seqs * P.slices * P.heads * 2 * KC * NV), 64 * NW, 0, c->stream>>>(P);
}
template <int KC> static void lin_scan(Ctx* c, const LinArgs& P, bool wide) {
    if (wide) lin_scan_run<KC, true>(c, P);
    else lin_scan_run<KC, false>(c, P);
}

template <int DKR> static void lin_step(Ctx* c, const LinArgs& P, int64_t blocks) {
    if (P.s_vec) lin_step_kernel<DKR, true><<<(unsigned) blocks, 256, 0, c->stream>>>(P);
    else lin_step_kernel<DKR, false><<<(unsigned) blocks, 256, 0, c->stream>>>(P);
}

static int lin_checks(const std::string& fn, const h3_lin_state* state, const h3_lin_batch* batch, int dt) {
    if (!state || !batch) return fail(fn + ": the states and the batch are required");
    if (state->slots <= 0 || state->heads <= 0 || state->dk <= 0 || state->dv <= 0 || state->dk > 256 || state->dv > 256)
        return fail(fn + ": states have slots, heads and 1 to 256 features of keys and of values");
    if (state->slots > INT32_MAX || state->heads > 65535) return fail(fn + ": too many slots or heads");
    if (!state->s) return fail(fn + ": the states are required");
    if ((uintptr_t) state->s & 3) return fail(fn + ": the states must be 4-byte aligned");
    if (batch->seqs < 0 || batch->rows < 0 || batch->most < 0) return fail(fn + ": a negative size");
    if (batch->rows > INT32_MAX || batch->seqs >= INT32_MAX) return fail(fn + ": sizes past 32 bits");
    if (!dt_ok(dt)) return fail(fn + ": unknown element type");
    return 0;
}

// Which kernels take the call. Sequences of up to kLinFew tokens go token by token, others in pieces. 64 sequences of 64 heads of 128 x 128, of up to
// 1, 4, 6, 8 and 16 tokens, 0.7 of that on average, in a queue of passes over the same states: carried on 91, 96, 109, 120 and 163 us, in pieces
// 167, 172, 176, 178 and 187; begun, so that a state is only written, 48, 61, 72, 80 and 127, in pieces 86, 85, 86, 88 and 94. 16 of 16 heads
// of 256 x 256 carried on 25, 28, 31, 33 and 46, in pieces 35; begun 16, 19, 23, 26 and 40, in pieces 22: 6 is where these lose nothing yet, carried
// on 8 and more would pay. A launch for few tokens beside the others' takes 5 us and more: where the sequences beside the longest have more
// than kLinBeside tokens on average, or are up to four blocks of pieces a CU, all go in pieces (64 sequences of up to 8 tokens in two
// launches 96 us; eight of up to 39 37, in pieces 21; all begun).
constexpr int kLinFew = 6, kLinBeside = 4;
constexpr int64_t kLinLeast = 32, kLinSegs = 256;   // the least tokens of a segment, the most segments of an average sequence
struct LinPlan {
    bool step, chunk, split;
    int kc, slices;
    bool wide;
    int64_t seg, places, blocks, floats;
};
// A piece's time in microseconds (64 bfloat16 tokens of keys of up to 128 features, else 32) by the steps of 32 features of keys, in a block of
// threads with 128 or 64 features of values: a + b kc where it is alone on the device, and what each of the blocks of a CU takes of that where
// there are more (two run at once, if their LDS lets them). Measured over 512 tokens of 4, 256 and 512 heads of 128 features of values; keys of
// 128: bfloat16 5.9, 7.3 and 9.8 in blocks of 128, 4.3, 6.4 and 11.9 in twice as many of 64.
struct LinPiece { double a, b, each; };
static LinPiece lin_piece(int dt, int kc, bool wide) {
    if (dt == H3S_BF16) return kc <= 4 ? (wide ? LinPiece{3.3, 0.65, 0.82} : LinPiece{2.8, 0.33, 0.75}) : wide ? LinPiece{1.25, 0.3, 1.25} : LinPiece{1.5, 0.2, 0.75};
    if (dt == H3S_F16) return !wide ? LinPiece{1.65, 0.35, 0.75} : kc <= 4 ? LinPiece{2.0, 0.51, 0.82} : LinPiece{2.25, 0.36, 1.25};
    return !wide ? LinPiece{1.8, 0.54, kc <= 4 ? 0.75 : 1.15} : kc <= 4 ? LinPiece{2.6, 0.77, 0.82} : LinPiece{2.9, 0.53, 1.25};
}
// what a piece takes longer where a CU has so many blocks
static double lin_load(const LinPiece& t, double each) {
    return each <= 1.0 ? 1.0 + 0.2 * each : each <= 2.0 ? 1.2 + (2.0 * t.each - 1.2) * (each - 1.0) : t.each * each;
}
static LinPlan lin_plan(const h3_lin_state& state, const h3_lin_batch& batch, int dt, int cus) {
    LinPlan p{};
    const int64_t most = std::min(batch.most, batch.rows);
    p.chunk = most > kLinFew;
    p.step = !p.chunk || ((batch.seqs - 1) * state.heads * ((state.dv + 63) / 64) > 4 * (int64_t) cus &&
                          batch.rows - most <= kLinBeside * (batch.seqs - 1) && most * batch.seqs > batch.rows);
    p.kc = state.dk <= 32 ? 1 : state.dk > 64 && state.dk <= 96 ? 3 : (int) (state.dk + 63) / 64 * 2;
    // Segments, and a block's features of values, by an estimate of the time, of the average sequence (with a launch for few tokens: of as many
    // of the longest's length as there are rows for): the pieces one after another; a split one's own sums half as much again, and launches,
    // the states (written and read twice) at 4.5 TB/s and 0.3 a segment of the walk over them. (8192 tokens, 64 heads of 128: 1, 4, 8 and
    // 12 segments a head 770, 270, 220 and 240 us; four float32 prompts of up to 1500 tokens, 16 heads of 80 x 96, in segments of 256 and
    // 128 94 and 68. Three sequences of up to 362 tokens, 8 heads of 128 x 96: 36 us in blocks of 128 features, 25 of 64.)
    const int64_t piece = dt == H3S_BF16 && p.kc <= 4 ? 64 : 32, seqs = p.step ? std::max<int64_t>(batch.rows / most, 1) : batch.seqs;
    const int64_t length = std::max<int64_t>(std::min(most, batch.rows / seqs), 1), chains = seqs * state.heads;
    const int64_t pieces = (length + piece - 1) / piece, longest = (most + piece - 1) / piece;
    double best = 1e300;
    p.seg = most;
    for (const bool wide : {true, false}) {
        if (wide && state.dv <= 64) continue;
        const int64_t slices = wide ? (state.dv + 127) / 128 : (state.dv + 63) / 64;
        const LinPiece t = lin_piece(dt, p.kc, wide);
        for (int64_t n = 1; n <= std::min(pieces, kLinSegs); ++n) {
            const int64_t per = (pieces + n - 1) / n, segs = (pieces + per - 1) / per;
            // (Segments are of one length, and the CU with most of them is the last; of several sequences each has a shorter one more, and
            // they do not fill the CUs evenly. Whole sequences are not of one length: the longest goes on by itself.)
            const double blocks = (double) (chains * slices) * (segs > 1 && seqs > 1 ? segs + 0.5 : segs), each = blocks / cus;
            const double load = lin_load(t, segs > 1 && seqs > 1 ? std::ceil(each + 0.1) : segs > 1 && each > 1.0 ? std::ceil(each) : each);
            const double one = t.a + t.b * p.kc;
            const double states = (double) chains * segs * state.dk * state.dv * 16.0 / 4.5e6;
            const double cost = segs > 1 ? 1.5 * per * one * load + 11.0 + 0.3 * segs + states : one * std::max(pieces * load, longest * lin_load(t, std::min(each, 1.0)));
            if (cost < best) {
                best = cost;
                p.seg = segs > 1 ? std::max(per * piece, kLinLeast) : most;
                p.wide = wide;
                p.slices = (int) slices;
            }
        }
    }
    p.split = p.seg < most;
    if (!p.split) p.seg = most;
    p.places = p.split ? batch.rows / p.seg + batch.seqs : batch.seqs;
    p.blocks = p.places * p.slices * state.heads;
    p.floats = p.chunk && p.split ? p.blocks * (32 * p.kc) * (p.wide ? 128 : 64) : 0;
    return p;
}

// Whether a launch could take 2^32 threads or more, however the device's size splits the call; counted in 256 threads: a block of 64 features of
// values is one, of 128 two where keys have more than 128 features, and the walk has 2 or 4 kc of them a sequence and head.
static bool lin_too_many(const h3_lin_state& state, const h3_lin_batch& batch) {
    const LinPlan p = lin_plan(state, batch, H3S_BF16, 1);
    const int64_t steps = (state.dv + kLinCols - 1) / kLinCols, most = kKvMostBlocks / state.heads;
    const int64_t narrow = (state.dv + 63) / 64, wide = state.dv > 64 ? (state.dv + 127) / 128 * 2 : 0;
    const bool split = std::min(batch.most, batch.rows) > kLinLeast;
    const int64_t seg = std::max(kLinLeast, std::min({batch.most, batch.rows, batch.rows / batch.seqs}) / kLinSegs);   // the shortest
    const int64_t places = split ? batch.rows / seg + batch.seqs : batch.seqs;
    return (p.step && batch.seqs > most / steps) || (p.chunk && places > most / (p.kc > 4 ? std::max(narrow, wide) : narrow)) ||
           (p.chunk && split && batch.seqs > most / (2 * p.kc * std::max(narrow, wide)));
}

int64_t lin_attention_work(void* ctx, const h3_lin_state* state, const h3_lin_batch* batch, int dt) try {
    const char* fn = "lin_attention_work";
    if (lin_checks(fn, state, batch, dt)) return -1;
    const bool none = batch->seqs == 0 || batch->rows == 0 || batch->most == 0;
    if (!none && lin_too_many(*state, *batch)) return fail(std::string(fn) + ": too many blocks of work");
    Ctx* c = ctx_of(ctx, fn);
    if (!c) return -1;
    if (none) return 0;
    return 4 * lin_plan(*state, *batch, dt, c->cus).floats;
} catch (const std::exception& e) { return fail(e.what()); }

int lin_attention(void* ctx, const h3_lin_state* state, const h3_lin_batch* batch, const float* decay, const void* q, int64_t q_stride,
                  int64_t q_heads, const void* k, int64_t k_stride, int64_t k_heads, const void* v, int64_t v_stride, int64_t v_heads,
                  int dt, float scale, void* out, int out_dt, void* work, uint64_t work_bytes) try {
    const std::string fn = "lin_attention";
    if (lin_checks(fn, state, batch, dt)) return -1;
    if (!dt_ok(out_dt)) return fail(fn + ": unknown element type");
    const int64_t heads = state->heads, dk = state->dk, dv = state->dv;
    if (q_heads <= 0 || k_heads <= 0 || v_heads <= 0 || heads % q_heads || heads % k_heads || heads % v_heads)
        return fail(fn + ": the states' heads must be a multiple of q's, k's and v's");
    if (!(scale >= 0.0f) || std::isinf(scale)) return fail(fn + ": the scale must be a number above 0 (or 0: 1 / sqrt(dk))");
    if (batch->seqs == 0 || batch->rows == 0 || batch->most == 0) return 0;
    if (!batch->starts || !batch->source || !batch->target) return fail(fn + ": starts, source and target are required");
    if (q_stride < q_heads * dk || k_stride < k_heads * dk || v_stride < v_heads * dv) return fail(fn + ": a row stride is shorter than a row");
    if (!decay || !q || !k || !v || !out) return fail(fn + ": decay, q, k, v and out are required");
    if (work && !aligned16(work)) return fail(fn + ": the workspace must be 16-byte aligned");
    const int es = elem_size(dt);
    // (in pieces the rows of 64 tokens are reached by 32 bits of distance)
    auto vec = [&](const void* p, int64_t stride, int64_t dim) {
        return aligned16(p) && stride < (1 << 22) && stride * es % 16 == 0 && dim * es % 16 == 0;
    };
    LinArgs P{};
    P.s = state->s;
    P.slots = state->slots;
    P.heads = (int) heads; P.dk = (int) dk; P.dv = (int) dv;
    P.kv.starts = batch->starts; P.kv.seqs = (int) batch->seqs; P.kv.rows = (int) batch->rows;
    P.source = batch->source; P.target = batch->target; P.decay = decay;
    P.q = q; P.k = k; P.v = v;
    P.q_stride = q_stride; P.k_stride = k_stride; P.v_stride = v_stride;
    P.q_each = (int) (heads / q_heads); P.k_each = (int) (heads / k_heads); P.v_each = (int) (heads / v_heads);
    P.dt = dt; P.out = out; P.out_dt = out_dt;
    P.scale = scale > 0.0f ? scale : (float) (1.0 / std::sqrt((double) dk));
    P.least = 0; P.most = UINT32_MAX;
    P.s_vec = aligned16(P.s) && dv % 4 == 0;
    P.vec = vec(q, q_stride, dk) && vec(k, k_stride, dk) && vec(v, v_stride, dv) && aligned16(out) && heads * dv < (1 << 22);
    if (lin_too_many(*state, *batch)) return fail(fn + ": too many blocks of work");
    Ctx* c = ctx_of(ctx, fn.c_str());
    if (!c) return -1;
    const LinPlan plan = lin_plan(*state, *batch, dt, c->cus);
    const int64_t steps = batch->seqs * heads * ((dv + kLinCols - 1) / kLinCols);
    if (plan.floats) {
        if (work) {
            if (work_bytes < (uint64_t) (4 * plan.floats)) return fail(fn + ": the workspace is smaller than lin_attention_work() says");
            P.ws = (float*) work;
        } else {
            hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
            if (hipStreamIsCapturing(c->stream, &st) != hipSuccess) (void) hipGetLastError();
            if (st != hipStreamCaptureStatusNone) return fail(fn + ": a call recorded into a graph needs a workspace of its own");
            P.ws = c->scratch<float>(Ctx::LIN_STATE, (size_t) plan.floats);
            if (!P.ws) return -1;
        }
    }
    if (plan.step) {
        P.most = plan.chunk ? kLinFew : UINT32_MAX;
        switch (plan.kc) {
            case 1:
            case 2: lin_step<2>(c, P, steps); break;
            case 3:
            case 4: lin_step<4>(c, P, steps); break;
            case 6: lin_step<6>(c, P, steps); break;
            default: lin_step<8>(c, P, steps); break;
        }
    }
    if (plan.chunk) {
        P.least = plan.step ? kLinFew + 1 : 0;
        P.most = UINT32_MAX;
        P.slices = plan.slices;
        P.seg = (int) plan.seg;
        auto run = [&](bool outputs) {
            if (dt == H3S_BF16) lin_chunk_bf16(c, P, plan.kc, plan.wide, plan.blocks, outputs);
            else if (dt == H3S_F16) lin_chunk_f16(c, P, plan.kc, plan.wide, plan.blocks, outputs);
            else lin_chunk_f32(c, P, plan.kc, plan.wide, plan.blocks, outputs);
        };
        if (plan.split) {
            run(false);
            switch (plan.kc) {
                case 1: lin_scan<1>(c, P, plan.wide); break;
                case 2: lin_scan<2>(c, P, plan.wide); break;
                case 3: lin_scan<3>(c, P, plan.wide); break;
                case 4: lin_scan<4>(c, P, plan.wide); break;
                case 6: lin_scan<6>(c, P, plan.wide); break;
                default: lin_scan<8>(c, P, plan.wide); break;
            }
        }
        run(true);
    }
    return launched(fn.c_str());
} catch (const std::exception& e) { return fail(e.what()); }

}  // namespace h3
