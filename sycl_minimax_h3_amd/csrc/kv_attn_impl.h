// kv_attn_impl.h - the attention over the 8-bit key/value cache (h3lm.h, kv_attention).
//
// Mathematics, for one query row with scores s_j = q . k_j * scale over the tokens j it sees: p_j = 2^(s_j log2(e) - m), m the
// running maximum (less 15, kKvShift), l = sum p_j, o = sum p_j v_j / l, in one pass over the cache: where a block raises m, l and o are
// multiplied by 2^(m_old - m). Keys are codes times a block's scale, so s = (q . codes) * (k_scale * scale * log2 e): one factor a
// block. Values likewise: a block's sum of p_j codes_j is added to o with v_scale as the factor.
//
// Products on the matrix cores (16 x 16 x 32, half operands, float32 sums). The codes are whole numbers below 2^8, exact as
// half. Query rows are scaled by a power of two that takes their largest value to 2^14 .. 2^15, so half holds 16-bit types
// without loss down to 2^-29 of it; float32 rows are two halves (high and rest: 22 bits). Probabilities are 2^15 p, so that half keeps
// them down to p = 2^-29 at full precision. They are two halves too, but for many rows of 16-bit queries (kv_plans says which). (One half shows little in 16-bit
// results: 500 tokens, the error against 64 bits in float16 2.6e-4 of the result, 2.1e-4 with two; in bfloat16 1.69e-3 and 1.68e-3. It shows in
// float32 ones, 1.5e-4 and 2.5e-7. Two are 1-1.5 % of an answered token's time, whose bound is the cache's bytes - 64 sequences of up to 8192
// tokens 131.0 and 132.2 us, one of 300 8.4 and 8.8 - but double the values' products of prompts, and two wavefronts a SIMD have no registers
// for them.)
//
// Layout: S^T = K Q^T, with the keys as the first operand, leaves one query row a lane (lane % 16) and four keys a register
// group; the row statistics are the lane's own but for two exchanges (lanes 16 and 32 apart). The rows of K are taken in the order
// that makes those keys, as they stand, the second operand of O^T = V^T P^T: lane group g = lane / 16 holds the keys 16 g .. 16 g + 15
// of a block, which is also the 16 bytes of a V row that it loads. Probabilities never leave their registers.
//
// Work: a block of threads takes one key/value head of one sequence, a tile of its rows (tokens x the heads that share the
// key/value head) and a range of the cache blocks. Few rows (kv_attn_kernel): its four wavefronts share 16 NQ rows and take every
// fourth cache block (answered tokens; bound by the cache's bytes), joined through LDS. Many (kv_attn_rows_kernel): each has 16 NQ rows
// of its own (prompts).
// Where that leaves the device idle, the cache blocks are split over several blocks of threads, whose sums kv_merge_kernel
// joins in split order.
//
// First tokens that stay visible behind a window are a second range of the same walk. Tokens that sequences share are gone through by a launch
// of their own for all rows of a group (as if they were one sequence's: its cache is read once, and the rows fill the tiles), whose parts the
// sequences' own launch adds to its sums, or kv_join_kernel where it has parts too: (m, l, o) of two ranges join as those of two parts do.
// 64 sequences over 8192 shared tokens and up to 1024 of their own, 64 heads over 8 of 128: 45 us (0.38 PFLOP/s: one round of blocks of threads
// with 16 cache blocks each, whose beginning and end cost as much as two or three more) and 24 (the own tokens' bytes), where the caches' bytes
// one by one would take 235.
#pragma once

#include "kv.h"

namespace h3 {

typedef _Float16 v8h_kv __attribute__((ext_vector_type(8)));
typedef _Float16 v2h_kv __attribute__((ext_vector_type(2)));
typedef float v4f_kv __attribute__((ext_vector_type(4)));

// where m starts: below every score, and finite, so that m_old - m is never infinity minus infinity
constexpr float kKvUnset = -3e38f;
// Probabilities are held times 2^15: m is 15 below the running maximum. Where a block's largest score is 2^19 or more from zero (its steps
// 2^-4 and more) m is that score itself, and scores are rounded before m is taken off: the fused difference would be off by half a step of
// the score, past what half holds above 2^15 from 2^23 on, and without bound beyond.
constexpr float kKvShift = 15.0f, kKvFar = 524288.0f;

struct KvAttnArgs {
    KvArgs kv;
    const int32_t* lengths;
    const void* q;
    int64_t q_stride, mask_stride;
    int q_dt, group, q_heads;
    float scale;                                    // times log2(e)
    int window;                                     // 0: all
    const uint8_t* mask;
    void* out;
    int out_dt;
    float* lse;
    int tiles, places;                              // row tiles a sequence (0: laid out by the rows, see KvItem); row tiles of all sequences
    uint32_t least, greatest;                       // the sequences of fewer or more rows (tokens x heads of a group) are another launch's
    int nsplit, per;                                // parts, of `per` cache blocks each (the last: the rest)
    float *po, *pml;                                // the parts' sums [place, head, part, rows, W] and (m, l) [place, head, part, rows, 2]
    bool q_vec, out_vec, mask_vec;
    // of kv_attention_spans:
    int sinks;                                      // the first tokens that stay visible behind a window
    const int32_t *first, *shared;                  // [groups + 1]: a group's first sequence; [groups]: the tokens that it shares
    int groups;
    int rt2, nsplit2;                               // the rows of a block, and the parts, of the shared tokens' launch (0 parts: there is none)
    const float *po2, *pml2;                        // its parts
};

// What a launch goes through. kKvAll: all of a sequence's cache up to the row, or a window of it. kKvOwn: of that the first tokens too, and only
// what lies behind the tokens that a sequence shares. kKvShared: the shared tokens, for all rows of a group of sequences as if they were one's.
enum { kKvAll, kKvOwn, kKvShared };

// four codes as half: 2^10 + (code + 128) in the low bits of a half, less 2^10 + 128 (exact)
__device__ __forceinline__ void kv_half4(uint32_t u, v2h_kv& a, v2h_kv& b) {
    const uint32_t x = u ^ 0x80808080u;
    const v2h_kv off = {(_Float16) -1152.0f, (_Float16) -1152.0f};
    a = __builtin_bit_cast(v2h_kv, __builtin_amdgcn_perm(0x64646464u, x, 0x04010400u)) + off;
    b = __builtin_bit_cast(v2h_kv, __builtin_amdgcn_perm(0x64646464u, x, 0x04030402u)) + off;
}
__device__ __forceinline__ v8h_kv kv_half8(uint32_t u, uint32_t w) {
    v2h_kv a, b, c, d;
    kv_half4(u, a, b);
    kv_half4(w, c, d);
    return v8h_kv{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}
__device__ __forceinline__ v4f_kv kv_mma(const v8h_kv& a, const v8h_kv& b, const v4f_kv& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
// over the four lanes that share a query row (16 and 32 apart)
__device__ __forceinline__ float kv_max4(float x) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_int(x), __float_as_int(x), false, false);
    x = fmaxf(__int_as_float(r[0]), __int_as_float(r[1]));
    r = __builtin_amdgcn_permlane16_swap(__float_as_int(x), __float_as_int(x), false, false);
    return fmaxf(__int_as_float(r[0]), __int_as_float(r[1]));
}
__device__ __forceinline__ float kv_sum4(float x) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_int(x), __float_as_int(x), false, false);
    x = __int_as_float(r[0]) + __int_as_float(r[1]);
    r = __builtin_amdgcn_permlane16_swap(__float_as_int(x), __float_as_int(x), false, false);
    return __int_as_float(r[0]) + __int_as_float(r[1]);
}

// four consecutive features of an output row
__device__ __forceinline__ void kv_store4(const KvAttnArgs& P, int64_t at, int d, float a, float b, float c, float e) {
    const int dim = P.kv.dim;
    if (P.out_vec) {                                // dim a multiple of 4: all of them or none
        if (d >= dim) return;
        if (P.out_dt == H3S_F32) *reinterpret_cast<float4*>((float*) P.out + at + d) = make_float4(a, b, c, e);
        else if (P.out_dt == H3S_BF16) *reinterpret_cast<uint2*>((uint16_t*) P.out + at + d) = make_uint2(pack_bf16(a, b), pack_bf16(c, e));
        else *reinterpret_cast<uint2*>((uint16_t*) P.out + at + d) = make_uint2(pack_f16(a, b), pack_f16(c, e));
    } else {
        const float f[4] = {a, b, c, e};
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (d + i < dim) store_any(P.out, P.out_dt, at + d + i, f[i]);
    }
}
// the logarithm of the row's sum of exponentials from m and the sum of 2^(score - m)
__device__ __forceinline__ float kv_lse(float m, float l) {
    return l > 0.0f ? (m + __builtin_log2f(l)) * 0.69314718055994531f : l == 0.0f ? -__builtin_inff() : l;
}

// What a wavefront holds of its 16 NQ query rows: row lane % 16 of each tile
template <int WC, int NQ, bool TWO, bool PTWO, int MODE> struct KvRows {
    static constexpr int W = 64 * WC, DT = 4 * WC, PARTS = TWO ? 2 : 1, PP = PTWO ? 2 : 1;   // halves of a query, of a probability
    int pos[NQ], head[NQ];                          // the row's token (-1: no row), its query head
    int seq[MODE == kKvShared ? NQ : 1];            // its sequence
    int64_t tok[NQ];                                // its row of q and out (-1: none)
    float rowf[NQ], m[NQ], l[NQ];
    v8h_kv qf[NQ][WC][2][PARTS];
    v4f_kv o[NQ][DT];

    // rows rw .. of the R of a sequence with n rows from r0 on and len tokens, for key/value head h
    // (kKvShared: with the rows' tokens and sequences in `who`, from rw on)
    __device__ __forceinline__ void load(const KvAttnArgs& P, int h, int r0, int n, int len, uint32_t R, uint32_t rw, int l15, int g,
                                         const int2* who = nullptr) {
        const uint32_t group = P.group;
#pragma unroll
        for (int e = 0; e < NQ; ++e) {
            const bool valid = rw + 16 * e + l15 < R;
            const uint32_t r = valid ? rw + 16 * e + l15 : 0;
            const int j = (int) (r / group);
            head[e] = (int) (h * group + r % group);
            tok[e] = valid ? (int64_t) r0 + j : -1;
            if constexpr (MODE == kKvShared) {
                pos[e] = who[16 * e + l15].x;
                seq[e] = max(who[16 * e + l15].y, 0);
            } else {
                pos[e] = valid ? len - n + j : -1;
            }
            const int64_t row = ((int64_t) r0 + j) * P.q_stride + (int64_t) head[e] * P.kv.dim;
            float f[WC * 2][8];
            float top = 0.0f;
#pragma unroll
            for (int c = 0; c < WC; ++c)
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const int d = c * 64 + g * 16 + s * 8;
                    float* y = f[2 * c + s];
#pragma unroll
                    for (int i = 0; i < 8; ++i) y[i] = 0.0f;
                    if (valid && P.q_vec) {
                        if (d < P.kv.dim) {
                            if (P.q_dt == H3S_F32) load_f32x((const float*) P.q + row + d, y, 8);
                            else {
                                const uint4 u = *reinterpret_cast<const uint4*>((const uint16_t*) P.q + row + d);
                                if (P.q_dt == H3S_BF16) Vec<H3S_BF16>::unpack(u, y);
                                else Vec<H3S_F16>::unpack(u, y);
                            }
                        }
                    } else if (valid) {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (d + i < P.kv.dim) y[i] = load_any(P.q, P.q_dt, row + d + i);
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(y[i]));
                }
            top = kv_max4(top);
            // 2^k takes top to [2^14, 2^15) (a row of zeros, infinities or NaN: left as it is)
            const int k = top > 0.0f && top < __builtin_inff() ? 15 - __builtin_amdgcn_frexp_expf(top) : 0;
            rowf[e] = __builtin_ldexpf(P.scale, -k);
#pragma unroll
            for (int c = 0; c < WC; ++c)
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        float y = __builtin_ldexpf(f[2 * c + s][i], k);
                        pin(y);
                        const _Float16 hi = (_Float16) y;
                        qf[e][c][s][0][i] = hi;
                        if constexpr (TWO) qf[e][c][s][1][i] = (_Float16) (y - (float) hi);
                    }
            m[e] = kKvUnset;
            l[e] = 0.0f;
#pragma unroll
            for (int t = 0; t < DT; ++t) o[e][t] = v4f_kv{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }

    // the lane's keys of a cache block that the mask hides
    static __device__ __forceinline__ uint32_t masked(const KvAttnArgs& P, int b, int g, int key0) {
        uint32_t hidden = 0;
        const int k0 = key0 + g * 16;
        const uint8_t* mp = P.mask + (int64_t) b * P.mask_stride + k0;
        if (P.mask_vec && k0 + 16 <= P.mask_stride) {
            const uint4 u = *reinterpret_cast<const uint4*>(mp);
            const uint32_t w4[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int i = 0; i < 16; ++i) hidden |= ((w4[i >> 2] >> (8 * (i & 3))) & 0xffu) == 0 ? 1u << i : 0u;
        } else {
            for (int i = 0; i < 16; ++i)
                if (k0 + i >= P.mask_stride || mp[i] == 0) hidden |= 1u << i;
        }
        return hidden;
    }

    // kKvOwn, kKvShared: the mask's bytes of the lane's keys of a cache block (0: hidden), for the item's sequence or each row's. They are loaded before
    // the block's products and looked at behind them: where the scores want them, each block waits for them (53 sequences of up to 31 tokens
    // over 5376 shared ones in 13 groups, 8 heads over one of 80: 85 to 79 us).
    static constexpr int MASKS = MODE == kKvShared ? NQ : 1;
    __device__ __forceinline__ void mask_bytes(const KvAttnArgs& P, int b, int g, int key0, uint4 (&m)[MASKS]) const {
        if (MODE == kKvAll || !P.mask) return;
#pragma unroll
        for (int e = 0; e < MASKS; ++e) {
            const int k0 = key0 + g * 16;
            const uint8_t* mp = P.mask + (int64_t) (MODE == kKvShared ? seq[e] : b) * P.mask_stride + k0;
            if (P.mask_vec && k0 + 16 <= P.mask_stride) {
                m[e] = *reinterpret_cast<const uint4*>(mp);
            } else {
                uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (k0 + i < P.mask_stride) w[i >> 2] |= (uint32_t) mp[i] << (8 * (i & 3));
                m[e] = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
    }
    static __device__ __forceinline__ uint32_t none_of(const uint4& m) {
        // (a byte that is not 0 carries into its highest bit; the four bits' weights are summed by a dot product of bytes)
        auto some = [](uint32_t w) { return ((((w & 0x7f7f7f7fu) + 0x7f7f7f7fu) | w) >> 7) & 0x01010101u; };
        const uint32_t lo = __builtin_amdgcn_udot4(some(m.y), 0x80402010u, __builtin_amdgcn_udot4(some(m.x), 0x08040201u, 0, false), false);
        const uint32_t hi = __builtin_amdgcn_udot4(some(m.w), 0x80402010u, __builtin_amdgcn_udot4(some(m.z), 0x08040201u, 0, false), false);
        return (lo | hi << 8) ^ 0xffffu;
    }

    // One cache block's scores to probabilities: s (register t, i of lane group g: the key 16 g + 4 t + i of the block) to the operands
    // pf, times 2^15, and vsl, the factor of the block's values for each row. whole: every row sees every key.
    __device__ __forceinline__ void softmax(const KvAttnArgs& P, int b, int g, int key0, bool whole, float ks, float vs, v4f_kv (&s)[NQ][4],
                                            v8h_kv (&pf)[NQ][2][PP], float (&vsl)[NQ], const uint4 (&mask)[MASKS]) {
        uint32_t hidden = 0;                        // by the mask: bit 4 t + i
        if (MODE == kKvAll && !whole && P.mask) hidden = masked(P, b, g, key0);
        if (MODE == kKvOwn && !whole && P.mask) hidden = none_of(mask[0]);
#pragma unroll
        for (int e = 0; e < NQ; ++e) {
            uint32_t off = hidden;
            if (!whole) {
                if (MODE == kKvShared && P.mask) off = none_of(mask[MODE == kKvShared ? e : 0]);
                const int hi = pos[e] - key0 - g * 16;                  // the lane's keys 0 .. hi of 16 are not ahead of the row
                off |= hi >= 15 ? 0u : hi < 0 ? 0xffffu : 0xffffu & (0xfffeu << hi);
                if (P.window > 0) {
                    const int lo = hi - P.window + 1;                    // and lo .. are inside the window
                    uint32_t behind = lo <= 0 ? 0u : lo > 15 ? 0xffffu : (1u << lo) - 1;
                    if constexpr (MODE != kKvAll) {
                        const int first = P.sinks - key0 - g * 16;       // of them the first ones stay
                        behind &= first <= 0 ? 0xffffu : first > 15 ? 0u : 0xffffu << first;
                    }
                    off |= behind;
                }
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if ((off >> (4 * t + i)) & 1) s[e][t][i] = -__builtin_inff();
            }
            float top = -__builtin_inff();
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) top = fmaxf(top, s[e][t][i]);
            top = kv_max4(top);
            // Hidden scores are minus infinity, and a factor above 0 keeps them so. Where the row sees none of the block, the block has no
            // part in it whatever its scales are (NaN times minus infinity would be NaN).
            const bool seen = top > -__builtin_inff();
            float f = rowf[e] * ks;
            f = f < 1e-37f ? 1e-37f : f;
            f = seen ? f : 1.0f;
            vsl[e] = seen ? vs : 0.0f;
            const float big = top * f;
            const bool far = seen && fabsf(big) >= kKvFar;
            float from = big - kKvShift;
            if (__builtin_expect(__any(far), 0)) {
                from = far ? big : from;
                const float once = far ? f : 1.0f;
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[e][t][i] *= once;
                f = far ? 1.0f : f;
            }
            const float mn = fmaxf(m[e], from);
            if (__any(mn > m[e])) {
                const float alpha = __builtin_amdgcn_exp2f(m[e] - mn);
                l[e] *= alpha;
#pragma unroll
                for (int t = 0; t < DT; ++t) o[e][t] *= alpha;
                m[e] = mn;
            }
            float sum = 0.0f;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e][t][i], f, -m[e]));
                    sum += p;
                    const int at = 4 * (t & 1) + i;
                    const _Float16 hi = (_Float16) p;
                    pf[e][t >> 1][0][at] = hi;
                    if constexpr (PTWO) pf[e][t >> 1][1][at] = (_Float16) (p - (float) hi);
                }
            l[e] += sum;
        }
    }

    // V^T P^T of a feature tile, whose codes of the keys 8 .. of each 16 are a1
    __device__ __forceinline__ void products(const v8h_kv& a0, const v8h_kv& a1, const v8h_kv (&pf)[NQ][2][PP], v4f_kv (&y)[NQ]) const {
#pragma unroll
        for (int w = 0; w < PP; ++w) {
#pragma unroll
            for (int e = 0; e < NQ; ++e) y[e] = kv_mma(a0, pf[e][0][w], w ? y[e] : v4f_kv{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
            for (int e = 0; e < NQ; ++e) y[e] = kv_mma(a1, pf[e][1][w], y[e]);
        }
    }
    // O^T += v_scale of it, for the feature tile t
    __device__ __forceinline__ void add(int t, const v4f_kv (&y)[NQ], const float (&vsl)[NQ]) {
#pragma unroll
        for (int e = 0; e < NQ; ++e)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[e][t][i] = __builtin_fmaf(y[e][i], vsl[e], o[e][t][i]);
    }
};

// the first row of group c's sequences (of `groups`: behind the last), whatever `first` and `starts` say
__device__ __forceinline__ int kv_first_row(const KvAttnArgs& P, int first) {
    return min(max(P.kv.starts[min(max(first, 0), P.kv.seqs)], 0), P.kv.rows);
}
// The group that sequence b shares tokens in, or -1, its first sequence, the cache blocks that it shares and its rows [row, end); found by the
// whole wavefront, 64 groups at a time (as kv_find).
__device__ __forceinline__ int kv_group_of(const KvAttnArgs& P, int b, int& first, int& blocks, int& row, int& end) {
    const int lane = threadIdx.x & 63;
    int step = 1;
    while (step * 64 < P.groups + 1) step *= 64;
    for (int g = 0;; step /= 64) {
        const int c = g + lane * step, f = P.first[min(c, P.groups)], n = P.shared[min(c, P.groups - 1)];
        const int k = (int) __popcll(__ballot(c <= P.groups && f <= b) & ~1ull);
        g += k * step;
        if (step > 1) continue;
        first = __builtin_amdgcn_readlane(f, k);
        const int to = k < 63 ? __builtin_amdgcn_readlane(f, k + 1) : P.first[min(g + 1, P.groups)];
        blocks = min(max(__builtin_amdgcn_readlane(n, k), 0) / kKvB, P.kv.width);
        if (first > b || g >= P.groups || b >= to) return -1;
        first = max(first, 0);
        row = kv_first_row(P, first);
        end = kv_first_row(P, to);
        return g;
    }
}
// kv_find of groups in place of sequences: each is as one sequence of all its rows. Also its sequences [b, b1) and shared cache blocks.
__device__ __forceinline__ int kv_find_group(const KvAttnArgs& P, int at, uint32_t den, int& r0, int& n, int& b, int& b1, int& blocks) {
    const int lane = threadIdx.x & 63;
    int step = 1;
    while (step * 64 < P.groups) step *= 64;
    for (int g = 0;; step /= 64) {
        const int c = g + lane * step, f = P.first[min(c, P.groups)], t = P.shared[min(c, P.groups - 1)], s = kv_first_row(P, f);
        const int begin = (int) ((uint32_t) s * (uint32_t) P.group / den) + min(c, P.groups);
        const int k = (int) __popcll(__ballot(c < P.groups && begin <= at) & ~1ull);
        g += k * step;
        if (step > 1) continue;
        r0 = __builtin_amdgcn_readlane(s, k);
        b = min(max(__builtin_amdgcn_readlane(f, k), 0), P.kv.seqs);
        blocks = min(max(__builtin_amdgcn_readlane(t, k), 0) / kKvB, P.kv.width);
        const int next = k < 63 ? __builtin_amdgcn_readlane(f, k + 1) : P.first[min(g + 1, P.groups)];
        b1 = min(max(next, b), P.kv.seqs);
        n = max(k < 63 ? __builtin_amdgcn_readlane(s, k + 1) : kv_first_row(P, next), r0) - r0;
        return at - __builtin_amdgcn_readlane(begin, k);
    }
}

// Which rows, head, sequence and part of the cache a block of threads has. Sequences with about as many rows each have P.tiles tiles of RT
// rows; else each has its share: R of all sequences' rows lie in at most floor(R / RT) + 1 of the places from floor(its first / RT) + its number on.
template <int MODE> struct KvItem {
    int h, split, place, b, tile, r0, n, len;
    uint32_t R;
    int b1 = 0;                                                           // kKvShared: behind the group's last sequence
    int lo = 0, hi = 0, sink = 0, win = 0;                                // cache blocks: see spans()
    int first = 0, group = -1, row = 0, end_row = 0;                      // kKvOwn: the first sequence of its group, its group and that one's rows
    template <int RT> __device__ __forceinline__ void take(const KvAttnArgs& P) {
        uint32_t id = blockIdx.x;
        h = (int) (id % (uint32_t) P.kv.heads);
        id /= (uint32_t) P.kv.heads;
        split = (int) (id % (uint32_t) P.nsplit);
        rows<RT>(P, (int) (id / (uint32_t) P.nsplit));
    }
    // (a place that is no sequence's: a tile past every row)
    template <int RT> __device__ __forceinline__ void rows(const KvAttnArgs& P, int at) {
        place = at;
        if constexpr (MODE == kKvShared) {
            place = P.places - 1 - at;                                    // (the longest rows first; kv_shared_row counts from the groups' rows)
            tile = kv_find_group(P, place, RT, r0, n, b, b1, hi);
            R = tile < 0 || b1 <= b ? 0 : (uint32_t) n * P.group;
            b = min(b, P.kv.seqs - 1);
            len = 0;
            return;
        }
        if (P.tiles) {
            b = (int) ((uint32_t) at % (uint32_t) P.kv.seqs);
            tile = P.tiles - 1 - (int) ((uint32_t) at / (uint32_t) P.kv.seqs);    // the longest rows first
            kv_rows_of(P.kv, b, r0, n);
        } else {
            tile = kv_find(P.kv, P.places - 1 - at, P.group, RT, 1, b, r0, n);
        }
        R = (uint32_t) n * P.group;                                       // (rows * group is below 2^31)
        if (R < P.least || R > P.greatest) R = 0;
        len = min(max(P.lengths[b], 0), P.kv.width * kKvB);
        if constexpr (MODE == kKvOwn)
            if (P.groups) {
                group = kv_group_of(P, b, first, hi, row, end_row);
                if (group < 0) { first = b; hi = 0; }
                lo = P.nsplit2 ? hi : 0;
            }
    }
    // the cache blocks kb0 .. kb0 + count that any of the rows rt0 .. rt0 + rt can see
    __device__ __forceinline__ void range(const KvAttnArgs& P, uint32_t rt0, int rt, int& kb0, int& count) {
        const int base = len - n, bmin = base + (int) (rt0 / P.group), bmax = base + (int) ((min(R, rt0 + rt) - 1) / P.group);
        if constexpr (MODE != kKvAll) return spans(P, bmin, bmax, kb0, count);
        kb0 = P.window > 0 ? max(bmin - P.window + 1, 0) / kKvB : 0;
        count = bmax >= 0 ? max(bmax / kKvB + 1 - kb0, 0) : 0;
    }
    // The same of rows that are the tokens bmin .. bmax, as a count from 0: first the blocks of the first tokens, lo .. lo + sink, then those from
    // win on. (Shared tokens end at block hi, a sequence's own begin at block lo: hi too, or 0 where there is no launch of the shared ones.)
    __device__ __forceinline__ void spans(const KvAttnArgs& P, int bmin, int bmax, int& kb0, int& count) {
        int end = bmax >= 0 ? bmax / kKvB + 1 : 0;
        if constexpr (MODE == kKvShared) end = min(end, hi);
        win = max(P.window > 0 ? max(bmin - P.window + 1, 0) / kKvB : 0, lo);
        sink = P.window > 0 ? max(min(min((P.sinks + kKvB - 1) / kKvB, end), win) - lo, 0) : 0;
        kb0 = 0;
        count = sink + max(end - win, 0);
    }
    // the block that the walk's step i is
    __device__ __forceinline__ int block(int i) const { return MODE == kKvAll ? i : i < sink ? lo + i : win + (i - sink); }
    // the end of this part's blocks (from kb0 + split * per on); parts past the first that have none leave nothing
    __device__ __forceinline__ int end(const KvAttnArgs& P, int kb0, int count) const {
        return split + 1 == P.nsplit ? kb0 + count : kb0 + min(count, (split + 1) * P.per);
    }
    // the item's place among the parts' sums
    __device__ __forceinline__ int64_t part(const KvAttnArgs& P) const {
        return ((int64_t) place * P.kv.heads + h) * P.nsplit + split;
    }
};

// kKvShared: the tokens and sequences (-1: no row) of the tile's rows from rt0 on. A sequence's place is guessed as if all of the group had as many
// rows, and searched for where that is wrong.
template <int RT> __device__ __forceinline__ void kv_who(const KvAttnArgs& P, const KvItem<kKvShared>& it, uint32_t rt0, int2* who) {
    const uint32_t rr = rt0 + threadIdx.x;
    if (threadIdx.x >= RT) return;
    int2 w = make_int2(-1, -1);
    if (rr < it.R) {
        const int j = (int) (rr / (uint32_t) P.group), row = it.r0 + j;
        int b = it.b + (int) ((uint64_t) (uint32_t) j * (uint32_t) (it.b1 - it.b) / (uint32_t) it.n);
        int from = P.kv.starts[b], to = P.kv.starts[b + 1];
        if (row < from || row >= to) {
            int a = it.b, e = it.b1;                            // the last that begins at or before the row
            while (e - a > 1) {
                const int m = (a + e) >> 1;
                if (P.kv.starts[m] <= row) a = m;
                else e = m;
            }
            b = a;
            from = P.kv.starts[b];
            to = P.kv.starts[b + 1];
        }
        from = min(max(from, 0), P.kv.rows);
        to = min(max(to, from), P.kv.rows);
        if (row >= from && row < to) w = make_int2(min(max(P.lengths[b], 0), P.kv.width * kKvB) - (to - row), b);
    }
    who[threadIdx.x] = w;
}
// the least and greatest token of N rows
template <int N> __device__ __forceinline__ void kv_reach(const int2* who, int& posmin, int& posmax) {
    posmin = INT32_MAX;
    posmax = -1;
#pragma unroll
    for (int i = 0; i < (N + 63) / 64; ++i) {
        const int at = (threadIdx.x & 63) + 64 * i;
        const int2 w = who[N < 64 ? at % N : at];
        if (w.y >= 0) {
            posmin = min(posmin, w.x);
            posmax = max(posmax, w.x);
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        posmin = min(posmin, __shfl_xor(posmin, o));
        posmax = max(posmax, __shfl_xor(posmax, o));
    }
    posmin = __builtin_amdgcn_readfirstlane(posmin);
    posmax = __builtin_amdgcn_readfirstlane(posmax);
}
// a part that has no blocks
template <int RT> __device__ __forceinline__ void kv_nothing(const KvAttnArgs& P, const KvItem<kKvShared>& it) {
    if (threadIdx.x < RT) *reinterpret_cast<float2*>(P.pml + (it.part(P) * RT + threadIdx.x) * 2) = make_float2(kKvUnset, 0.0f);
}
// Whether a launch's sums are the results (with the shared tokens' parts), or parts of them
template <int MODE> __device__ __forceinline__ bool kv_direct(const KvAttnArgs& P) { return MODE != kKvShared && P.nsplit == 1; }

// kKvOwn: the first of the parts over shared tokens of row rr of the item's sequence, rt2 rows apart, or -1
__device__ __forceinline__ int64_t kv_shared_row(const KvAttnArgs& P, const KvItem<kKvOwn>& it, uint32_t rr) {
    if (it.group < 0 || P.nsplit2 == 0) return -1;
    const int row = it.r0 + (int) (rr / (uint32_t) P.group);
    if (row < it.row || row >= it.end_row) return -1;
    const uint32_t r2 = (uint32_t) (row - it.row) * (uint32_t) P.group + rr % (uint32_t) P.group, rt2 = (uint32_t) P.rt2;
    const int64_t place = (int) ((uint32_t) it.row * (uint32_t) P.group / rt2) + it.group + (int) (r2 / rt2);
    return (place * P.kv.heads + it.h) * P.nsplit2 * rt2 + r2 % rt2;
}
// (m, l) of the part s over shared tokens of a row
__device__ __forceinline__ float2 kv_shared_ml(const KvAttnArgs& P, int64_t row2, int s) {
    return s < P.nsplit2 ? *reinterpret_cast<const float2*>(P.pml2 + (row2 + (int64_t) s * P.rt2) * 2) : make_float2(kKvUnset, 0.0f);
}
// The weight of a part: 0 where nothing was seen, whose sums say nothing
__device__ __forceinline__ float kv_weight(const float2& ml, float top) { return ml.y == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(ml.x - top); }
// y += the sums of four parts times their weights, which the lanes first .. of 16 have in w; sums(i): a lane's in part i. Loaded together: one by
// one each waits for memory. (No weight: nothing seen, and there may be no sums.)
template <int WC, typename F> __device__ __forceinline__ void kv_take(float4 (&y)[WC], float w, int first, F sums) {
    float4 v[4][WC];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int t = 0; t < WC; ++t) v[i][t] = *reinterpret_cast<const float4*>(sums(i) + 64 * t);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float wi = __shfl(w, first + i, 16);
#pragma unroll
        for (int t = 0; t < WC; ++t) {
            y[t].x = wi == 0.0f ? y[t].x : __builtin_fmaf(v[i][t].x, wi, y[t].x);
            y[t].y = wi == 0.0f ? y[t].y : __builtin_fmaf(v[i][t].y, wi, y[t].y);
            y[t].z = wi == 0.0f ? y[t].z : __builtin_fmaf(v[i][t].z, wi, y[t].z);
            y[t].w = wi == 0.0f ? y[t].w : __builtin_fmaf(v[i][t].w, wi, y[t].w);
        }
    }
}

// Whether a key block is seen whole by rows that are the tokens posmin .. posmax
template <int MODE> __device__ __forceinline__ bool kv_whole(const KvAttnArgs& P, int key0, int posmin, int posmax) {
    return key0 + kKvB - 1 <= posmin && (P.window == 0 || key0 > posmax - P.window || (MODE != kKvAll && key0 + kKvB <= P.sinks)) && !P.mask;
}

// The walk over a sequence's blocks that are there. The wavefront holds 64 entries of the table, one a lane, so that a block's number is
// known without a wait for memory: read entry by entry, its latency stood before every block's loads (64 sequences of up to 8192 tokens
// 133.4 us, 130.7 so; 601 float32 tokens 33.8 and 33.1).
template <int MODE> struct KvPages {
    const int32_t *table, *shared;                  // kKvOwn: the sequence's row, and that of its group's first sequence for the blocks before hi
    int width, base, entry;
    __device__ __forceinline__ void take(const KvAttnArgs& P, const KvItem<MODE>& it) {
        table = P.kv.table + (int64_t) it.b * P.kv.width;
        if constexpr (MODE == kKvOwn) shared = P.kv.table + (int64_t) it.first * P.kv.width;
        width = P.kv.width;
        base = -64;
    }
    // the first block (of the walk) from kb on, in steps of BY, that is there (its page), or `last`
    template <int BY> __device__ __forceinline__ bool next(const KvAttnArgs& P, const KvItem<MODE>& it, int& kb, int& page, int last, int lane) {
        for (; kb < last; kb += BY) {
            if (kb - base >= 64) {
                base = kb;
                const int at = min(it.block(kb + lane), width - 1);
                if constexpr (MODE == kKvOwn) entry = (at < it.hi ? shared : table)[at];
                else entry = table[at];
            }
            page = __builtin_amdgcn_readlane(entry, kb - base);
            if (page >= 0 && page < P.kv.blocks) return true;
        }
        return false;
    }
};

// Few rows (up to 32 of a sequence and head): the four wavefronts of a block share 16 NQ rows and take every fourth cache block.
// Bound by the cache's bytes: the next block's codes are on their way while one is worked on (64 sequences of up to 8192 tokens, 8 heads of
// 128, 64 queries: 132 us, 4.9 TB/s; one of 131072 tokens 52.5 us, 5.1 TB/s, and the merge 4.8).
template <int WC, int NQ, bool TWO, int MODE = kKvAll>
__global__ __launch_bounds__(256) void kv_attn_kernel(KvAttnArgs P) {
    constexpr int W = 64 * WC, DT = 4 * WC, RT = 16 * NQ, KS = 4, PARTS = TWO ? 2 : 1;
    const int lane = threadIdx.x & 63, l15 = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int) (threadIdx.x >> 6));
    KvItem<MODE> it;
    it.template take<RT>(P);
    const int h = it.h, b = it.b;
    const uint32_t R = it.R, rw = (uint32_t) it.tile * RT, group = P.group;
    if (rw >= R) return;

    // the cache blocks that any of the rows can see, a part of them, every KS-th
    int posmin = it.len - it.n + (int) (rw / group), posmax = it.len - it.n + (int) ((min(R, rw + RT) - 1) / group);
    int kb0, count;
    __shared__ int2 who[MODE == kKvShared ? RT : 1];
    if constexpr (MODE == kKvShared) {
        // (without a window the rows' places decide nothing before the first scores: they are found behind the first loads)
        if (P.window > 0) {
            kv_who<RT>(P, it, rw, who);
            __syncthreads();
            kv_reach<RT>(who, posmin, posmax);
        } else {
            posmin = posmax = INT32_MAX;
        }
        it.spans(P, posmin, posmax, kb0, count);
        if (it.split && it.split * P.per >= count) return kv_nothing<RT>(P, it);
    } else {
        it.range(P, rw, RT, kb0, count);
        if (it.split && it.split * P.per >= count) return;
    }
    const int last = it.end(P, kb0, count);
    KvPages<MODE> pages;
    pages.take(P, it);
    uint4 kr[4][WC], vr[DT];
    const int koff = ((l15 >> 2) * 16 + (l15 & 3)) * W + g * 16, voff = l15 * 64 + g * 16;
    auto load_k = [&](int page) {
        const int8_t* p = P.kv.k + ((int64_t) page * P.kv.heads + h) * (kKvB * W) + koff;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int c = 0; c < WC; ++c) kr[t][c] = *reinterpret_cast<const uint4*>(p + t * 4 * W + c * 64);
    };
    auto load_v = [&](int page) {
        const int8_t* p = P.kv.v + ((int64_t) page * P.kv.heads + h) * (kKvB * W) + voff;
#pragma unroll
        for (int t = 0; t < DT; ++t) vr[t] = *reinterpret_cast<const uint4*>(p + t * 1024);
    };
    int kb = kb0 + it.split * P.per + wave, page = 0;
    float ks = 0.0f, vs = 0.0f;
    if (pages.template next<KS>(P, it, kb, page, last, lane)) {
        load_k(page);
        load_v(page);
        ks = P.kv.ks[(int64_t) page * P.kv.heads + h];
        vs = P.kv.vs[(int64_t) page * P.kv.heads + h];
    }
    if constexpr (MODE == kKvShared)
        if (P.window == 0) {
            kv_who<RT>(P, it, rw, who);
            __syncthreads();
            kv_reach<RT>(who, posmin, posmax);
        }
    KvRows<WC, NQ, TWO, true, MODE> q;              // (behind the first loads of the cache, which take longer)
    q.load(P, h, it.r0, it.n, it.len, R, rw, l15, g, who);
    while (kb < last) {
        int nkb = kb + KS, npage = 0;
        const bool more = pages.template next<KS>(P, it, nkb, npage, last, lane);
        const int key0 = it.block(kb) * kKvB;
        uint4 mask[MODE == kKvShared ? NQ : 1];
        q.mask_bytes(P, b, g, key0, mask);
        v4f_kv s[NQ][4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
            for (int e = 0; e < NQ; ++e) s[e][t] = v4f_kv{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < WC; ++c) {
                const v8h_kv a0 = kv_half8(kr[t][c].x, kr[t][c].y), a1 = kv_half8(kr[t][c].z, kr[t][c].w);
#pragma unroll
                for (int e = 0; e < NQ; ++e) {
#pragma unroll
                    for (int w = 0; w < PARTS; ++w) {
                        s[e][t] = kv_mma(a0, q.qf[e][c][0][w], s[e][t]);
                        s[e][t] = kv_mma(a1, q.qf[e][c][1][w], s[e][t]);
                    }
                }
            }
        }
        const float ks_now = ks, vs_now = vs;
        if (more) {
            load_k(npage);
            ks = P.kv.ks[(int64_t) npage * P.kv.heads + h];
            vs = P.kv.vs[(int64_t) npage * P.kv.heads + h];
        }
        const bool whole = kv_whole<MODE>(P, key0, posmin, posmax);
        v8h_kv pf[NQ][2][2];
        float vsl[NQ];
        q.softmax(P, b, g, key0, whole, ks_now, vs_now, s, pf, vsl, mask);
#pragma unroll
        for (int t = 0; t < DT; ++t) {
            v4f_kv y[NQ];
            q.products(kv_half8(vr[t].x, vr[t].y), kv_half8(vr[t].z, vr[t].w), pf, y);
            q.add(t, y, vsl);
        }
        if (more) load_v(npage);
        kb = nkb;
    }

    // the four wavefronts' sums, 16 rows at a time
    __shared__ float so[4][16][W + 4];
    __shared__ float sm[4][16], sl[4][16];
#pragma unroll
    for (int e = 0; e < NQ; ++e) {
        const float l = kv_sum4(q.l[e]);
        if (e) __syncthreads();
#pragma unroll
        for (int t = 0; t < DT; ++t)
            *reinterpret_cast<float4*>(&so[wave][l15][16 * t + 4 * g]) = make_float4(q.o[e][t][0], q.o[e][t][1], q.o[e][t][2], q.o[e][t][3]);
        if (g == 0) { sm[wave][l15] = q.m[e]; sl[wave][l15] = l; }
        __syncthreads();
        const int r = threadIdx.x >> 4, c = threadIdx.x & 15;
        const uint32_t rr = rw + 16 * e + r;
        if (rr < R) {
            const float mx = fmaxf(fmaxf(sm[0][r], sm[1][r]), fmaxf(sm[2][r], sm[3][r]));
            float wt[4], lt = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                wt[w] = __builtin_amdgcn_exp2f(sm[w][r] - mx);
                lt += sl[w][r] * wt[w];
            }
            const int64_t at = ((int64_t) it.r0 + rr / group) * P.q_heads + h * group + rr % group;
            const int64_t row = it.part(P) * RT + 16 * e + r;
            float top = mx;
            int64_t row2 = -1;
            if constexpr (MODE == kKvOwn) {
                row2 = kv_direct<MODE>(P) ? kv_shared_row(P, it, rr) : -1;
            }
            float4 more[WC];                                              // the parts over shared tokens: a lane has (m, l) of every 16th
#pragma unroll
            for (int t = 0; t < WC; ++t) more[t] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if constexpr (MODE == kKvOwn)
                if (row2 >= 0) {
                    float2 ml = kv_shared_ml(P, row2, c);
                    top = fmaxf(top, wave_max<16>(ml.x));
                    for (int s = 16; s < P.nsplit2; s += 16) top = fmaxf(top, wave_max<16>(kv_shared_ml(P, row2, s + c).x));
                    const float own = __builtin_amdgcn_exp2f(mx - top);
                    lt *= own;
#pragma unroll
                    for (int w = 0; w < 4; ++w) wt[w] *= own;
                    for (int s0 = 0; s0 < P.nsplit2; s0 += 16) {
                        if (s0) ml = kv_shared_ml(P, row2, s0 + c);
                        const float wl = kv_weight(ml, top);
                        lt += wave_sum<16>(ml.y * wl);
                        for (int s = s0; s < min(P.nsplit2, s0 + 16); s += 4)
                            kv_take<WC>(more, wl, s - s0, [&](int i) { return P.po2 + (row2 + (int64_t) min(s + i, P.nsplit2 - 1) * P.rt2) * W + 4 * c; });
                    }
                }
            const float inv = lt == 0.0f ? 0.0f : 1.0f / lt;
#pragma unroll
            for (int t = 0; t < WC; ++t) {
                const int d = 64 * t + 4 * c;
                float y[4] = {more[t].x, more[t].y, more[t].z, more[t].w};
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const float4 v = *reinterpret_cast<const float4*>(&so[w][r][d]);
                    y[0] = __builtin_fmaf(v.x, wt[w], y[0]);
                    y[1] = __builtin_fmaf(v.y, wt[w], y[1]);
                    y[2] = __builtin_fmaf(v.z, wt[w], y[2]);
                    y[3] = __builtin_fmaf(v.w, wt[w], y[3]);
                }
                if (kv_direct<MODE>(P)) kv_store4(P, at * P.kv.dim, d, y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv);
                else *reinterpret_cast<float4*>(P.po + row * W + d) = make_float4(y[0], y[1], y[2], y[3]);
            }
            if (c == 0) {
                if (!kv_direct<MODE>(P)) *reinterpret_cast<float2*>(P.pml + row * 2) = make_float2(mx, lt);
                else if (P.lse) P.lse[at] = kv_lse(top, lt);
            }
        }
    }
}

// A 16-byte place among the 16 of a lane group is mixed with the group and the feature chunk: 16 lanes that store side by side (four
// tokens' or one token's pieces) then lie on all banks. Reads stay 16 places of one group.
template <int WC> __device__ __forceinline__ int kv_mix(int g, int c) { return (4 * g) ^ (WC == 2 ? 2 * c : c); }

// Many rows: each of a block's four wavefronts has 16 NQ rows of its own, and all go through the same cache blocks. A block's codes
// are turned to half once, by all four, into LDS in the order of the products' operands (two stages, one barrier a cache block), where
// doing it in every wavefront took more vector instructions than the softmax. Bound by vector instructions beside the products (4096 tokens
// over 8192, 64 heads over 8 of 128: 947-1060 us by the card, 0.78-0.87 PFLOP/s, the matrix cores 34 % busy). Operands are read from LDS a
// step ahead of their products (960 us without, 16 sequences of 100 tokens of 256 features 203 to 181).
// (Heads of up to 64 features in tiles of 128 rows, three blocks a CU: where first or shared tokens are walked over too, 8 vector and 19 scalar
// registers go to memory, 2 vector ones in the launch of shared tokens; kv_attention's form has none.)
template <int WC, int NQ, bool TWO, int MODE = kKvAll, bool PTWO = TWO>
__global__ __launch_bounds__(256, WC == 1 ? 3 : WC == 2 && !TWO ? 2 : 1) void kv_attn_rows_kernel(KvAttnArgs P) {
    constexpr int W = 64 * WC, DT = 4 * WC, RT = 64 * NQ, PARTS = TWO ? 2 : 1;
    __shared__ v8h_kv sk[2][4][WC][2][64], sv[2][DT][2][64];              // [stage][key tile or feature tile][...][half][lane]
    const int lane = threadIdx.x & 63, l15 = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int) (threadIdx.x >> 6));
    KvItem<MODE> it;
    it.template take<RT>(P);
    const int h = it.h, b = it.b;
    const uint32_t R = it.R, rt0 = (uint32_t) it.tile * RT, rw = rt0 + wave * 16 * NQ, group = P.group;
    if (rt0 >= R) return;
    // the cache blocks that any of the block's rows can see, a part of them; the wavefront's own rows see posmin .. posmax
    const int base = it.len - it.n;
    int posmin = base + (int) (rw / group), posmax = rw < R ? base + (int) ((min(R, rw + 16 * NQ) - 1) / group) : -1;
    int kb0, count;
    __shared__ int2 who[MODE == kKvShared ? RT : 1];
    if constexpr (MODE == kKvShared) {
        if (P.window > 0) {                         // (as above)
            kv_who<RT>(P, it, rt0, who);
            __syncthreads();
            kv_reach<RT>(who, posmin, posmax);
        } else {
            posmin = posmax = INT32_MAX;
        }
        it.spans(P, posmin, posmax, kb0, count);
        if (it.split && it.split * P.per >= count) return kv_nothing<RT>(P, it);
    } else {
        it.range(P, rt0, RT, kb0, count);
        if (it.split && it.split * P.per >= count) return;
    }
    const int last = it.end(P, kb0, count);
    KvPages<MODE> pages;
    pages.take(P, it);
    // the thread's 16-byte pieces of a block's codes: piece t + 256 i
    uint4 kr[WC], vr[WC];
    float ks = 0.0f, vs = 0.0f;
    auto load = [&](int page) {
        const int64_t at = (int64_t) page * P.kv.heads + h;
        const uint4 *kp = reinterpret_cast<const uint4*>(P.kv.k + at * (kKvB * W)), *vp = reinterpret_cast<const uint4*>(P.kv.v + at * (kKvB * W));
#pragma unroll
        for (int i = 0; i < WC; ++i) {
            kr[i] = kp[threadIdx.x + 256 * i];
            vr[i] = vp[threadIdx.x + 256 * i];
        }
        ks = P.kv.ks[at];
        vs = P.kv.vs[at];
    };
    auto stage = [&](int st) {
#pragma unroll
        for (int i = 0; i < WC; ++i) {
            const int p = threadIdx.x + 256 * i;
            // keys: token p / 4 WC, the features 16 (p % 4 WC) ..; the token is row 4 (token / 16) + token % 4 of the key tile token / 4 % 4.
            const int key = p / (4 * WC), c = p % (4 * WC) / 4, kg = p % 4, at = 16 * kg + (((key >> 4) * 4 + (key & 3)) ^ kv_mix<WC>(kg, c));
            const int t = (key >> 2) & 3;
            sk[st][t][c][0][at] = kv_half8(kr[i].x, kr[i].y);
            sk[st][t][c][1][at] = kv_half8(kr[i].z, kr[i].w);
            // values: feature p / 4, the tokens 16 (p % 4) ..
            const int av = 16 * kg + (p / 4 % 16 ^ (4 * kg));
            sv[st][p / 64][0][av] = kv_half8(vr[i].x, vr[i].y);
            sv[st][p / 64][1][av] = kv_half8(vr[i].z, vr[i].w);
        }
    };
    int kb = kb0 + it.split * P.per, page = 0, st = 0;
    const bool any = pages.template next<1>(P, it, kb, page, last, lane);
    int nkb = kb, npage = 0;
    bool more = false;
    float ks_now = 0.0f, vs_now = 0.0f;
    if (any) load(page);
    if constexpr (MODE == kKvShared) {
        if (P.window == 0) {
            kv_who<RT>(P, it, rt0, who);
            __syncthreads();
        }
        kv_reach<16 * NQ>(who + wave * 16 * NQ, posmin, posmax);
    }
    KvRows<WC, NQ, TWO, PTWO, MODE> q;
    q.load(P, h, it.r0, it.n, it.len, R, rw, l15, g, who + (MODE == kKvShared ? wave * 16 * NQ : 0));
    if (any) {
        stage(0);
        ks_now = ks;
        vs_now = vs;
        nkb = kb + 1;
        more = pages.template next<1>(P, it, nkb, npage, last, lane);
        if (more) load(npage);
    }
    lds_barrier();
    while (kb < last) {
        const int key0 = it.block(kb) * kKvB;
        if (key0 <= posmax) {
            uint4 mask[MODE == kKvShared ? NQ : 1];
            q.mask_bytes(P, b, g, key0, mask);
            // a feature chunk's operands of all four key tiles are read while the one before is multiplied: four tiles' sums in turn
            // leave no product waiting for the last
            v4f_kv s[NQ][4];
            v8h_kv a[2][4];
            auto keys = [&](int i) {
#pragma unroll
                for (int t = 0; t < 4; ++t) a[i & 1][t] = sk[st][t][i / 2][i % 2][16 * g + (l15 ^ kv_mix<WC>(g, i / 2))];
            };
            keys(0);
#pragma unroll
            for (int i = 0; i < 2 * WC; ++i) {
                if (i + 1 < 2 * WC) keys(i + 1);
#pragma unroll
                for (int w = 0; w < PARTS; ++w)
#pragma unroll
                    for (int t = 0; t < 4; ++t)
#pragma unroll
                        for (int e = 0; e < NQ; ++e)
                            s[e][t] = kv_mma(a[i & 1][t], q.qf[e][i / 2][i % 2][w], i + w ? s[e][t] : v4f_kv{0.0f, 0.0f, 0.0f, 0.0f});
                __builtin_amdgcn_sched_barrier(0);
            }
            const bool whole = kv_whole<MODE>(P, key0, posmin, posmax);
            v8h_kv pf[NQ][2][PTWO ? 2 : 1];
            float vsl[NQ];
            q.softmax(P, b, g, key0, whole, ks_now, vs_now, s, pf, vsl, mask);
            // likewise a feature tile's operands, and the sums of the tile before are added to o meanwhile
            v8h_kv x[2][2];
            auto feats = [&](int t) {
                x[t & 1][0] = sv[st][t][0][16 * g + (l15 ^ (4 * g))];
                x[t & 1][1] = sv[st][t][1][16 * g + (l15 ^ (4 * g))];
            };
            v4f_kv y[2][NQ];
            feats(0);
#pragma unroll
            for (int t = 0; t < DT; ++t) {
                if (t + 1 < DT) feats(t + 1);
                q.products(x[t & 1][0], x[t & 1][1], pf, y[t & 1]);
                if (t) q.add(t - 1, y[(t & 1) ^ 1], vsl);
                __builtin_amdgcn_sched_barrier(0);
            }
            q.add(DT - 1, y[(DT - 1) & 1], vsl);
        }
        // the next block's codes, loaded a block ago, to the other stage, and the loads of the one after
        if (more) {
            stage(st ^ 1);
            ks_now = ks;
            vs_now = vs;
        }
        kb = nkb;
        if (more) {
            nkb = kb + 1;
            more = pages.template next<1>(P, it, nkb, npage, last, lane);
            if (more) load(npage);
        }
        lds_barrier();
        st ^= 1;
    }
#pragma unroll
    for (int e = 0; e < NQ; ++e) {
        float l = kv_sum4(q.l[e]);
        if (q.tok[e] < 0) continue;
        if constexpr (MODE == kKvOwn) {
            const int64_t row2 = kv_direct<MODE>(P) ? kv_shared_row(P, it, rw + 16 * e + l15) : -1;
            if (row2 >= 0) {
                float top = q.m[e];
#pragma unroll 4
                for (int s = 0; s < P.nsplit2; ++s) top = fmaxf(top, kv_shared_ml(P, row2, s).x);
                const float own = __builtin_amdgcn_exp2f(q.m[e] - top);
                q.m[e] = top;
                l *= own;
#pragma unroll
                for (int t = 0; t < DT; ++t) q.o[e][t] *= own;
                for (int s = 0; s < P.nsplit2; ++s) {
                    const float2 ml = kv_shared_ml(P, row2, s);
                    const float w = kv_weight(ml, top);
                    if (w == 0.0f) continue;
                    l = __builtin_fmaf(ml.y, w, l);
#pragma unroll
                    for (int t = 0; t < DT; ++t) {
                        const float4 v = *reinterpret_cast<const float4*>(P.po2 + (row2 + (int64_t) s * P.rt2) * W + 16 * t + 4 * g);
                        q.o[e][t][0] = __builtin_fmaf(v.x, w, q.o[e][t][0]);
                        q.o[e][t][1] = __builtin_fmaf(v.y, w, q.o[e][t][1]);
                        q.o[e][t][2] = __builtin_fmaf(v.z, w, q.o[e][t][2]);
                        q.o[e][t][3] = __builtin_fmaf(v.w, w, q.o[e][t][3]);
                    }
                }
            }
        }
        if (kv_direct<MODE>(P)) {
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            const int64_t at = q.tok[e] * P.q_heads + q.head[e];
#pragma unroll
            for (int t = 0; t < DT; ++t)
                kv_store4(P, at * P.kv.dim, 16 * t + 4 * g, q.o[e][t][0] * inv, q.o[e][t][1] * inv, q.o[e][t][2] * inv, q.o[e][t][3] * inv);
            if (P.lse && g == 0) P.lse[at] = kv_lse(q.m[e], l);
        } else {
            const int64_t row = it.part(P) * RT + (rw - rt0) + 16 * e + l15;
#pragma unroll
            for (int t = 0; t < DT; ++t)
                *reinterpret_cast<float4*>(P.po + row * W + 16 * t + 4 * g) = make_float4(q.o[e][t][0], q.o[e][t][1], q.o[e][t][2], q.o[e][t][3]);
            if (g == 0) *reinterpret_cast<float2*>(P.pml + row * 2) = make_float2(q.m[e], l);
        }
    }
}

// joins the parts of one row: one block of 256 threads a row, its wavefronts taking every fourth part, in that order
template <int WC, int RT>
__global__ __launch_bounds__(256) void kv_merge_kernel(KvAttnArgs P) {
    constexpr int W = 64 * WC;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t item = blockIdx.x / RT;
    const int r = (int) (blockIdx.x % RT);
    KvItem<kKvAll> it;
    it.h = (int) (item % P.kv.heads);
    it.template rows<RT>(P, (int) (item / P.kv.heads));
    const uint32_t rr = (uint32_t) it.tile * RT + r, group = P.group;
    if (rr >= it.R) return;
    int kb0, count;
    it.range(P, (uint32_t) it.tile * RT, RT, kb0, count);
    const int parts = min(max((count + P.per - 1) / P.per, 1), P.nsplit);
    const int64_t row0 = item * P.nsplit * RT + r;
    float mx = kKvUnset;
    for (int s = lane; s < parts; s += 64) mx = fmaxf(mx, P.pml[(row0 + (int64_t) s * RT) * 2]);
    mx = wave_max<64>(mx);
    float lt = 0.0f;
    for (int s = lane; s < parts; s += 64) {
        const float2 ml = *reinterpret_cast<const float2*>(P.pml + (row0 + (int64_t) s * RT) * 2);
        lt += ml.y * __builtin_amdgcn_exp2f(ml.x - mx);
    }
    lt = wave_sum<64>(lt);
    float y[WC];
#pragma unroll
    for (int t = 0; t < WC; ++t) y[t] = 0.0f;
#pragma unroll 4
    for (int s = wave; s < parts; s += 4) {
        const int64_t row = row0 + (int64_t) s * RT;
        const float w = __builtin_amdgcn_exp2f(P.pml[row * 2] - mx);
#pragma unroll
        for (int t = 0; t < WC; ++t) y[t] = __builtin_fmaf(P.po[row * W + 64 * t + lane], w, y[t]);
    }
    __shared__ float sy[4][W];
#pragma unroll
    for (int t = 0; t < WC; ++t) sy[wave][64 * t + lane] = y[t];
    __syncthreads();
    const int64_t at = ((int64_t) it.r0 + rr / group) * P.q_heads + it.h * group + rr % group;
    const float inv = lt == 0.0f ? 0.0f : 1.0f / lt;
    for (int d = threadIdx.x; d < P.kv.dim; d += 256)
        store_any(P.out, P.out_dt, at * P.kv.dim + d, ((sy[0][d] + sy[1][d]) + (sy[2][d] + sy[3][d])) * inv);
    if (P.lse && threadIdx.x == 0) P.lse[at] = kv_lse(mx, lt);
}

// Joins the parts of a row over its sequence's own blocks and, where its sequence shares tokens, over those. A block of 256 threads takes 16
// rows, 16 lanes each: a lane has four features of every 64 and (m, l) of every 16th part. (A block a row: 20 to 27 us for 12288 rows of two
// or three parts, most of it the blocks' beginnings; so 7.)
template <int WC, int RT>
__global__ __launch_bounds__(256) void kv_join_kernel(KvAttnArgs P) {
    constexpr int W = 64 * WC;
    const int c = threadIdx.x & 15, r = (int) (blockIdx.x % (RT / 16)) * 16 + (int) (threadIdx.x >> 4);
    const int64_t item = blockIdx.x / (RT / 16);
    KvItem<kKvOwn> it;
    it.h = (int) (item % P.kv.heads);
    it.template rows<RT>(P, (int) (item / P.kv.heads));
    const uint32_t rr = (uint32_t) it.tile * RT + r, group = P.group;
    if (rr >= it.R) return;                         // (16 lanes go together)
    int kb0, count;
    it.range(P, (uint32_t) it.tile * RT, RT, kb0, count);
    const int own = min(max((count + P.per - 1) / P.per, 1), P.nsplit);
    const int64_t row0 = item * P.nsplit * RT + r, row2 = kv_shared_row(P, it, rr);
    const int parts = own + (row2 >= 0 ? P.nsplit2 : 0);
    auto ml_of = [&](int s) {
        if (s >= parts) return make_float2(kKvUnset, 0.0f);
        return s < own ? *reinterpret_cast<const float2*>(P.pml + (row0 + (int64_t) s * RT) * 2) : kv_shared_ml(P, row2, s - own);
    };
    float2 ml = ml_of(c);
    float top = wave_max<16>(ml.x), lt = 0.0f;
    for (int s = 16; s < parts; s += 16) top = fmaxf(top, wave_max<16>(ml_of(s + c).x));
    float4 y[WC];
#pragma unroll
    for (int t = 0; t < WC; ++t) y[t] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int s0 = 0; s0 < parts; s0 += 16) {
        if (s0) ml = ml_of(s0 + c);
        const float wl = kv_weight(ml, top);
        lt += wave_sum<16>(ml.y * wl);
        for (int s = s0; s < min(parts, s0 + 16); s += 4)
            kv_take<WC>(y, wl, s - s0, [&](int i) {
                const int at = min(s + i, parts - 1);
                return (at < own ? P.po + (row0 + (int64_t) at * RT) * W : P.po2 + (row2 + (int64_t) (at - own) * P.rt2) * W) + 4 * c;
            });
    }
    const int64_t at = ((int64_t) it.r0 + rr / group) * P.q_heads + it.h * group + rr % group;
    const float inv = lt == 0.0f ? 0.0f : 1.0f / lt;
#pragma unroll
    for (int t = 0; t < WC; ++t) kv_store4(P, at * P.kv.dim, 64 * t + 4 * c, y[t].x * inv, y[t].y * inv, y[t].z * inv, y[t].w * inv);
    if (P.lse && c == 0) P.lse[at] = kv_lse(top, lt);
}

// which kernel takes the call, and in how many parts
struct KvPlan {
    bool rows;            // kv_attn_rows_kernel (else kv_attn_kernel)
    int nq, rt;           // its tiles of 16 rows a wavefront, and the rows a block of threads takes
    int64_t tiles, places;
    int nsplit, per;      // parts, and the cache blocks of each
    int64_t blocks;       // of threads, without the parts
    uint32_t least = 0, greatest = UINT32_MAX;
    bool shared = false;  // of the shared tokens
    double cost = 0.0;    // kv_attention_spans' rows: the estimate, in microseconds
    bool fine = false;    // kv_attn_rows_kernel with probabilities as two halves (float32 queries' are anyway)
};

template <int WC, int NQ, bool ROWS, int MODE>
static void kv_attn_run(Ctx* c, const KvAttnArgs& P, const KvPlan& plan, bool two) {
    const unsigned grid = (unsigned) (plan.blocks * plan.nsplit);
    constexpr int RT = (ROWS ? 64 : 16) * NQ;
    if constexpr (ROWS) {
        if (!two && !(NQ == 1 && plan.fine)) kv_attn_rows_kernel<WC, NQ, false, MODE><<<grid, 256, 0, c->stream>>>(P);
        if constexpr (NQ == 1) {
            if (two) kv_attn_rows_kernel<WC, 1, true, MODE><<<grid, 256, 0, c->stream>>>(P);
            else if (plan.fine) kv_attn_rows_kernel<WC, 1, false, MODE, true><<<grid, 256, 0, c->stream>>>(P);
        }
    } else {
        if (two) kv_attn_kernel<WC, NQ, true, MODE><<<grid, 256, 0, c->stream>>>(P);
        else kv_attn_kernel<WC, NQ, false, MODE><<<grid, 256, 0, c->stream>>>(P);
    }
    if (plan.nsplit > 1) {
        if constexpr (MODE == kKvOwn) kv_join_kernel<WC, RT><<<(unsigned) (plan.blocks * (RT / 16)), 256, 0, c->stream>>>(P);
        if constexpr (MODE == kKvAll) kv_merge_kernel<WC, RT><<<(unsigned) (plan.blocks * RT), 256, 0, c->stream>>>(P);
    }
}

// heads of up to 64 WC features (kv_attn_64.hip .. kv_attn_256.hip), the same of kv_attention_spans (kv_spans_64.hip .. kv_spans_256.hip)
void kv_attn_64(Ctx* c, const KvAttnArgs& P, const KvPlan& plan, bool two);
void kv_attn_128(Ctx* c, const KvAttnArgs& P, const KvPlan& plan, bool two);
void kv_attn_192(Ctx* c, const KvAttnArgs& P, const KvPlan& plan, bool two);
void kv_attn_256(Ctx* c, const KvAttnArgs& P, const KvPlan& plan, bool two);
void kv_spans_64(Ctx* c, const KvAttnArgs& P, const KvPlan& plan, bool two, bool shared);
void kv_spans_128(Ctx* c, const KvAttnArgs& P, const KvPlan& plan, bool two, bool shared);
void kv_spans_192(Ctx* c, const KvAttnArgs& P, const KvPlan& plan, bool two, bool shared);
void kv_spans_256(Ctx* c, const KvAttnArgs& P, const KvPlan& plan, bool two, bool shared);

template <int WC, int MODE = kKvAll>
static void kv_attn_width(Ctx* c, const KvAttnArgs& P, const KvPlan& plan, bool two) {
    if (plan.rows && plan.nq == 1) kv_attn_run<WC, 1, true, MODE>(c, P, plan, two);
    else if (plan.rows) kv_attn_run<WC, 2, true, MODE>(c, P, plan, two);
    else if (plan.nq == 1) kv_attn_run<WC, 1, false, MODE>(c, P, plan, two);
    else if constexpr (WC <= 2) kv_attn_run<WC, 2, false, MODE>(c, P, plan, two);
}

}  // namespace h3
