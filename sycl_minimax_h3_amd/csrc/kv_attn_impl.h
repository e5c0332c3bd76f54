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
// them down to p = 2^-29 at full precision. They are two halves too, but for many rows of 16-bit queries. (One half shows little in 16-bit
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
};

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
template <int WC, int NQ, bool TWO, bool PTWO> struct KvRows {
    static constexpr int W = 64 * WC, DT = 4 * WC, PARTS = TWO ? 2 : 1, PP = PTWO ? 2 : 1;   // halves of a query, of a probability
    int pos[NQ], head[NQ];                          // the row's token (-1: no row), its query head
    int64_t tok[NQ];                                // its row of q and out (-1: none)
    float rowf[NQ], m[NQ], l[NQ];
    v8h_kv qf[NQ][WC][2][PARTS];
    v4f_kv o[NQ][DT];

    // rows rw .. of the R of a sequence with n rows from r0 on and len tokens, for key/value head h
    __device__ __forceinline__ void load(const KvAttnArgs& P, int h, int r0, int n, int len, uint32_t R, uint32_t rw, int l15, int g) {
        const uint32_t group = P.group;
#pragma unroll
        for (int e = 0; e < NQ; ++e) {
            const bool valid = rw + 16 * e + l15 < R;
            const uint32_t r = valid ? rw + 16 * e + l15 : 0;
            const int j = (int) (r / group);
            head[e] = (int) (h * group + r % group);
            tok[e] = valid ? (int64_t) r0 + j : -1;
            pos[e] = valid ? len - n + j : -1;
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

    // One cache block's scores to probabilities: s (register t, i of lane group g: the key 16 g + 4 t + i of the block) to the operands
    // pf, times 2^15, and vsl, the factor of the block's values for each row. whole: every row sees every key.
    __device__ __forceinline__ void softmax(const KvAttnArgs& P, int b, int g, int key0, bool whole, float ks, float vs, v4f_kv (&s)[NQ][4],
                                            v8h_kv (&pf)[NQ][2][PP], float (&vsl)[NQ]) {
        uint32_t hidden = 0;                        // by the mask: bit 4 t + i
        if (!whole && P.mask) {
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
        }
#pragma unroll
        for (int e = 0; e < NQ; ++e) {
            uint32_t off = hidden;
            if (!whole) {
                const int hi = pos[e] - key0 - g * 16;                  // the lane's keys 0 .. hi of 16 are not ahead of the row
                off |= hi >= 15 ? 0u : hi < 0 ? 0xffffu : 0xffffu & (0xfffeu << hi);
                if (P.window > 0) {
                    const int lo = hi - P.window + 1;                    // and lo .. are inside the window
                    off |= lo <= 0 ? 0u : lo > 15 ? 0xffffu : (1u << lo) - 1;
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

// Which rows, head, sequence and part of the cache a block of threads has. Sequences with about as many rows each have P.tiles tiles of RT
// rows; else each has its share: R of all sequences' rows lie in at most floor(R / RT) + 1 of the places from floor(its first / RT) + its number on.
struct KvItem {
    int h, split, place, b, tile, r0, n, len;
    uint32_t R;
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
    }
    // the cache blocks kb0 .. kb0 + count that any of the rows rt0 .. rt0 + rt can see
    __device__ __forceinline__ void range(const KvAttnArgs& P, uint32_t rt0, int rt, int& kb0, int& count) const {
        const int base = len - n, bmin = base + (int) (rt0 / P.group), bmax = base + (int) ((min(R, rt0 + rt) - 1) / P.group);
        kb0 = P.window > 0 ? max(bmin - P.window + 1, 0) / kKvB : 0;
        count = bmax >= 0 ? max(bmax / kKvB + 1 - kb0, 0) : 0;
    }
    // the end of this part's blocks (from kb0 + split * per on); parts past the first that have none leave nothing
    __device__ __forceinline__ int end(const KvAttnArgs& P, int kb0, int count) const {
        return split + 1 == P.nsplit ? kb0 + count : kb0 + min(count, (split + 1) * P.per);
    }
    // the item's place among the parts' sums
    __device__ __forceinline__ int64_t part(const KvAttnArgs& P) const {
        return ((int64_t) place * P.kv.heads + h) * P.nsplit + split;
    }
};

// The walk over a sequence's blocks that are there. The wavefront holds 64 entries of the table, one a lane, so that a block's number is
// known without a wait for memory: read entry by entry, its latency stood before every block's loads (64 sequences of up to 8192 tokens
// 133.4 us, 130.7 so; 601 float32 tokens 33.8 and 33.1).
struct KvPages {
    const int32_t* table;
    int width, base, entry;
    __device__ __forceinline__ void take(const KvAttnArgs& P, int b) {
        table = P.kv.table + (int64_t) b * P.kv.width;
        width = P.kv.width;
        base = -64;
    }
    // the first block from kb on, in steps of BY, that is there (its page), or `last`
    template <int BY> __device__ __forceinline__ bool next(const KvAttnArgs& P, int& kb, int& page, int last, int lane) {
        for (; kb < last; kb += BY) {
            if (kb - base >= 64) {
                base = kb;
                entry = table[min(kb + lane, width - 1)];
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
template <int WC, int NQ, bool TWO>
__global__ __launch_bounds__(256) void kv_attn_kernel(KvAttnArgs P) {
    constexpr int W = 64 * WC, DT = 4 * WC, RT = 16 * NQ, KS = 4, PARTS = TWO ? 2 : 1;
    const int lane = threadIdx.x & 63, l15 = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int) (threadIdx.x >> 6));
    KvItem it;
    it.take<RT>(P);
    const int h = it.h, b = it.b;
    const uint32_t R = it.R, rw = (uint32_t) it.tile * RT, group = P.group;
    if (rw >= R) return;

    // the cache blocks that any of the rows can see, a part of them, every KS-th
    const int posmin = it.len - it.n + (int) (rw / group), posmax = it.len - it.n + (int) ((min(R, rw + RT) - 1) / group);
    int kb0, count;
    it.range(P, rw, RT, kb0, count);
    if (it.split && it.split * P.per >= count) return;
    const int last = it.end(P, kb0, count);
    KvPages pages;
    pages.take(P, b);
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
    if (pages.next<KS>(P, kb, page, last, lane)) {
        load_k(page);
        load_v(page);
        ks = P.kv.ks[(int64_t) page * P.kv.heads + h];
        vs = P.kv.vs[(int64_t) page * P.kv.heads + h];
    }
    KvRows<WC, NQ, TWO, true> q;                    // (behind the first loads of the cache, which take longer)
    q.load(P, h, it.r0, it.n, it.len, R, rw, l15, g);
    while (kb < last) {
        int nkb = kb + KS, npage = 0;
        const bool more = pages.next<KS>(P, nkb, npage, last, lane);
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
        const int key0 = kb * kKvB;
        const bool whole = key0 + kKvB - 1 <= posmin && (P.window == 0 || key0 > posmax - P.window) && !P.mask;
        v8h_kv pf[NQ][2][2];
        float vsl[NQ];
        q.softmax(P, b, g, key0, whole, ks_now, vs_now, s, pf, vsl);
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
            const float inv = lt == 0.0f ? 0.0f : 1.0f / lt;
#pragma unroll
            for (int t = 0; t < WC; ++t) {
                const int d = 64 * t + 4 * c;
                float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const float4 v = *reinterpret_cast<const float4*>(&so[w][r][d]);
                    y[0] = __builtin_fmaf(v.x, wt[w], y[0]);
                    y[1] = __builtin_fmaf(v.y, wt[w], y[1]);
                    y[2] = __builtin_fmaf(v.z, wt[w], y[2]);
                    y[3] = __builtin_fmaf(v.w, wt[w], y[3]);
                }
                if (P.nsplit == 1) kv_store4(P, at * P.kv.dim, d, y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv);
                else *reinterpret_cast<float4*>(P.po + row * W + d) = make_float4(y[0], y[1], y[2], y[3]);
            }
            if (c == 0) {
                if (P.nsplit > 1) *reinterpret_cast<float2*>(P.pml + row * 2) = make_float2(mx, lt);
                else if (P.lse) P.lse[at] = kv_lse(mx, lt);
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
template <int WC, int NQ, bool TWO>
__global__ __launch_bounds__(256, WC == 1 ? 3 : WC == 2 && !TWO ? 2 : 1) void kv_attn_rows_kernel(KvAttnArgs P) {
    constexpr int W = 64 * WC, DT = 4 * WC, RT = 64 * NQ, PARTS = TWO ? 2 : 1;
    __shared__ v8h_kv sk[2][4][WC][2][64], sv[2][DT][2][64];              // [stage][key tile or feature tile][...][half][lane]
    const int lane = threadIdx.x & 63, l15 = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int) (threadIdx.x >> 6));
    KvItem it;
    it.take<RT>(P);
    const int h = it.h, b = it.b;
    const uint32_t R = it.R, rt0 = (uint32_t) it.tile * RT, rw = rt0 + wave * 16 * NQ, group = P.group;
    if (rt0 >= R) return;
    // the cache blocks that any of the block's rows can see, a part of them; the wavefront's own rows see posmin .. posmax
    const int base = it.len - it.n;
    const int posmin = base + (int) (rw / group), posmax = rw < R ? base + (int) ((min(R, rw + 16 * NQ) - 1) / group) : -1;
    int kb0, count;
    it.range(P, rt0, RT, kb0, count);
    if (it.split && it.split * P.per >= count) return;
    const int last = it.end(P, kb0, count);
    KvPages pages;
    pages.take(P, b);
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
    const bool any = pages.next<1>(P, kb, page, last, lane);
    int nkb = kb, npage = 0;
    bool more = false;
    float ks_now = 0.0f, vs_now = 0.0f;
    if (any) load(page);
    KvRows<WC, NQ, TWO, TWO> q;
    q.load(P, h, it.r0, it.n, it.len, R, rw, l15, g);
    if (any) {
        stage(0);
        ks_now = ks;
        vs_now = vs;
        nkb = kb + 1;
        more = pages.next<1>(P, nkb, npage, last, lane);
        if (more) load(npage);
    }
    lds_barrier();
    while (kb < last) {
        const int key0 = kb * kKvB;
        if (key0 <= posmax) {
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
            const bool whole = key0 + kKvB - 1 <= posmin && (P.window == 0 || key0 > posmax - P.window) && !P.mask;
            v8h_kv pf[NQ][2][PARTS];
            float vsl[NQ];
            q.softmax(P, b, g, key0, whole, ks_now, vs_now, s, pf, vsl);
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
            more = pages.next<1>(P, nkb, npage, last, lane);
            if (more) load(npage);
        }
        lds_barrier();
        st ^= 1;
    }
#pragma unroll
    for (int e = 0; e < NQ; ++e) {
        const float l = kv_sum4(q.l[e]);
        if (q.tok[e] < 0) continue;
        if (P.nsplit == 1) {
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
    KvItem it;
    it.h = (int) (item % P.kv.heads);
    it.rows<RT>(P, (int) (item / P.kv.heads));
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

// which kernel takes the call, and in how many parts
struct KvPlan {
    bool rows;            // kv_attn_rows_kernel (else kv_attn_kernel)
    int nq, rt;           // its tiles of 16 rows a wavefront, and the rows a block of threads takes
    int64_t tiles, places;
    int nsplit, per;      // parts, and the cache blocks of each
    int64_t blocks;       // of threads, without the parts
    uint32_t least = 0, greatest = UINT32_MAX;
};

template <int WC, int NQ, bool ROWS>
static void kv_attn_run(Ctx* c, const KvAttnArgs& P, const KvPlan& plan, bool two) {
    const unsigned grid = (unsigned) (plan.blocks * plan.nsplit);
    constexpr int RT = (ROWS ? 64 : 16) * NQ;
    if constexpr (ROWS) {
        if (!two) kv_attn_rows_kernel<WC, NQ, false><<<grid, 256, 0, c->stream>>>(P);
        else if constexpr (NQ == 1) kv_attn_rows_kernel<WC, 1, true><<<grid, 256, 0, c->stream>>>(P);
    } else {
        if (two) kv_attn_kernel<WC, NQ, true><<<grid, 256, 0, c->stream>>>(P);
        else kv_attn_kernel<WC, NQ, false><<<grid, 256, 0, c->stream>>>(P);
    }
    if (plan.nsplit > 1) kv_merge_kernel<WC, RT><<<(unsigned) (plan.blocks * RT), 256, 0, c->stream>>>(P);
}

// heads of up to 64 WC features (kv_attn_64.hip .. kv_attn_256.hip)
void kv_attn_64(Ctx* c, const KvAttnArgs& P, const KvPlan& plan, bool two);
void kv_attn_128(Ctx* c, const KvAttnArgs& P, const KvPlan& plan, bool two);
void kv_attn_192(Ctx* c, const KvAttnArgs& P, const KvPlan& plan, bool two);
void kv_attn_256(Ctx* c, const KvAttnArgs& P, const KvPlan& plan, bool two);

template <int WC>
static void kv_attn_width(Ctx* c, const KvAttnArgs& P, const KvPlan& plan, bool two) {
    if (plan.rows && plan.nq == 1) kv_attn_run<WC, 1, true>(c, P, plan, two);
    else if (plan.rows) kv_attn_run<WC, 2, true>(c, P, plan, two);
    else if (plan.nq == 1) kv_attn_run<WC, 1, false>(c, P, plan, two);
    else if constexpr (WC <= 2) kv_attn_run<WC, 2, false>(c, P, plan, two);
}

}  // namespace h3
