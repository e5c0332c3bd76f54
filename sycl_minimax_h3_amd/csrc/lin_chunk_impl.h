// lin_chunk_impl.h - linear attention of many tokens (h3lm.h, lin_attention), in pieces of C tokens.
//
// Mathematics, for a piece of m tokens of one head that begins with the state S, with l = exp(-decay):
//     O = diag(l^(i+1)) Q S + (Q K^T . D) V,   D_ij = l^(i-j) for j <= i, else 0
//     S' = l^m S + K^T diag(l^(m-1-j)) V
// so that a token costs four products of a row with a matrix, three of them with matrices of the piece, instead of the state's update one
// token after another. Powers of l are exponentials of whole numbers of steps, each computed by itself, never as a quotient (l^i / l^j leaves
// float32 where the decay is strong).
//
// Number format: products on the matrix cores (16 x 16 x 32, bfloat16 operands, float32 sums). bfloat16 has float32's range, so
// nothing is scaled. An operand is a sum of bfloat16 parts: bfloat16 inputs are one, float16 ones two and float32 ones three (exact); the
// state and the piece's own products as operands are two for 16-bit inputs (17 bits, far below the rounding of a 16-bit result; 2.5e-6 of a
// float32 one) and three for float32; the decayed values that go into the state are three always, as the state is float32 and carried on.
// Products of parts that are below float32's last bit together are left out.
//
// Layout: the state is held in registers as the sum of its own update, S = K^T V: rows (keys' features) in the register groups, a column (a
// feature of v) a lane. As it stands that is the first operand of O^T = S^T Q^T, once in parts. Likewise P^T = K Q^T leaves its results as
// O^T += V^T P^T takes them. Which feature a row of a tile stands for is free, and is chosen such that the state's register groups are 8
// consecutive features, 16 bytes of a row of Q and K in LDS. V^T and K^T come out of LDS by the transposing read.
//
// Work: a block of four wavefronts has one head's piece after piece of a segment of a sequence, and 64 NV features of v, 16 NV a
// wavefront. Where heads and sequences are too few for the device, a sequence is split into segments: first each segment's own sums (this
// kernel without outputs), then the states at their beginnings (lin_scan_kernel), then the outputs.
#pragma once

#include "lin.h"

namespace h3 {

typedef __bf16 v8b_lin __attribute__((ext_vector_type(8)));
typedef __bf16 v2b_lin __attribute__((ext_vector_type(2)));
typedef float v2f_lin __attribute__((ext_vector_type(2)));
typedef float v4f_lin __attribute__((ext_vector_type(4)));
typedef short v4s_lin __attribute__((ext_vector_type(4)));

__device__ __forceinline__ v4f_lin lin_mma(const uint4& a, const uint4& b, const v4f_lin& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8b_lin, a), __builtin_bit_cast(v8b_lin, b), c, 0, 0, 0);
}
__device__ __forceinline__ uint32_t lin_pack(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f_lin) {a, b}, v2b_lin));
}
// Two values as N bfloat16 parts, the pairs packed. To the nearest where a rest is dropped (N = 2: 2^-18 of the value), exact for three:
// there the first two are cut, which keeps the largest float32 values in range.
template <int N> __device__ __forceinline__ void lin_split(float a, float b, uint32_t (&p)[N]) {
    if constexpr (N == 3) {
        const uint32_t ua = __float_as_uint(a) & 0xffff0000u, ub = __float_as_uint(b) & 0xffff0000u;
        const float ra = a - __uint_as_float(ua), rb = b - __uint_as_float(ub);
        const uint32_t va = __float_as_uint(ra) & 0xffff0000u, vb = __float_as_uint(rb) & 0xffff0000u;
        p[0] = (ua >> 16) | ub;
        p[1] = (va >> 16) | vb;
        p[2] = lin_pack(ra - __uint_as_float(va), rb - __uint_as_float(vb));
    } else {
        p[0] = lin_pack(a, b);
        if constexpr (N == 2) p[1] = lin_pack(a - bf16_lo(p[0]), b - bf16_hi(p[0]));
    }
}
// the segment that a block of threads has, of a sequence of `segs`
struct LinItem {
    int h, slice, place, b, seg, segs, r0, n;
    __device__ __forceinline__ bool take(const LinArgs& P) {
        uint32_t id = blockIdx.x;
        h = (int) (id % (uint32_t) P.heads);
        id /= (uint32_t) P.heads;
        slice = (int) (id % (uint32_t) P.slices);
        place = (int) (id / (uint32_t) P.slices);
        if (P.ws) {
            seg = kv_find(P.kv, place, 1, (uint32_t) P.seg, 1, b, r0, n);
            segs = (n + P.seg - 1) / P.seg;
        } else {                                                            // a segment is a sequence
            b = place;
            kv_rows_of(P.kv, b, r0, n);
            seg = 0;
            segs = n > 0;
        }
        return seg >= 0 && seg < segs && (uint32_t) n >= P.least && (uint32_t) n <= P.most;
    }
};

template <int DT, int KC, int NV> struct LinShape {
    static constexpr int NP = DT == H3S_BF16 ? 1 : DT == H3S_F16 ? 2 : 3;   // parts of an input
    static constexpr int NS = NP == 3 ? 3 : 2;                              // of the state and of a piece's products
    static constexpr int CT = NP == 1 && KC <= 4 ? 4 : 2, C = 16 * CT, U = CT / 2;
    static constexpr int DKP = 32 * KC, DVB = 64 * NV, FR = 2 * KC * NV;    // FR: 16-byte pieces of the state a thread holds
};

template <int DT, int KC, int NV, bool OUT>
__global__ __launch_bounds__(256) void lin_chunk_kernel(LinArgs P) {
    using Sh = LinShape<DT, KC, NV>;
    constexpr int NP = Sh::NP, NS = Sh::NS, CT = Sh::CT, C = Sh::C, U = Sh::U, DKP = Sh::DKP, DVB = Sh::DVB, FR = Sh::FR;
    constexpr int ES = DT == H3S_F32 ? 4 : 2, RAW = ES / 2;                 // 16-byte loads for 8 elements
    constexpr int KP = C * DKP / 2048, VP = C * DVB / 2048;                 // pieces of 8 elements a thread
    __shared__ uint4 sq[OUT ? NP : 1][OUT ? C * DKP / 8 : 1], sk[NP][C * DKP / 8], sv[NP][C * DVB / 8];
    __shared__ uint4 sp[OUT ? CT * U : 1][NS][64];
    __shared__ int first_bad[2];
    const int lane = threadIdx.x & 63, l15 = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int) (threadIdx.x >> 6));
    LinItem it;
    if (!it.take(P)) return;
    if (!OUT && it.seg + 1 == it.segs) return;                              // (nothing begins behind the last)
    const int h = it.h, t0 = it.seg * P.seg, count = min(P.seg, it.n - t0);
    const int64_t row0 = (int64_t) it.r0 + t0;
    const float decay = P.decay[h], rate = decay * -1.4426950408889634f;
    auto fade = [&](int steps) { return steps <= 0 ? 1.0f : __builtin_amdgcn_exp2f(rate * (float) steps); };
    const int col0 = it.slice * DVB, mycol = col0 + wave * 16 * NV;
    // feature of v (from mycol on) that row, or column, r of a tile of v stands for
    auto vcol = [&](int t, int r) { return NV == 2 ? 8 * (r >> 2) + 4 * t + (r & 3) : r; };

    // the state: register i of s[2 u + p][t]: keys' feature 32 u + 8 g + 4 p + i, v's feature vcol(t, l15)
    v4f_lin s[2 * KC][NV];
#pragma unroll
    for (int t = 0; t < 2 * KC; ++t)
#pragma unroll
        for (int x = 0; x < NV; ++x) s[t][x] = v4f_lin{0.0f, 0.0f, 0.0f, 0.0f};
    float* ws = P.ws + (int64_t) blockIdx.x * (FR * 1024) + threadIdx.x * 4;
    const int64_t head = (int64_t) P.dk * P.dv;
    if (OUT && it.segs > 1) {
#pragma unroll
        for (int t = 0; t < 2 * KC; ++t)
#pragma unroll
            for (int x = 0; x < NV; ++x) s[t][x] = *reinterpret_cast<const v4f_lin*>(ws + (t * NV + x) * 1024);
    } else if (OUT) {
        const int64_t from = P.source[it.b];
        if (from >= 0 && from < P.slots) {
            const float* sp0 = P.s + (from * P.heads + h) * head;
#pragma unroll
            for (int t = 0; t < 2 * KC; ++t)
#pragma unroll
                for (int x = 0; x < NV; ++x)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int d = 16 * (t & ~1) + 8 * g + 4 * (t & 1) + i, c = mycol + vcol(x, l15);
                        if (d < P.dk && c < P.dv) s[t][x][i] = sp0[(int64_t) d * P.dv + c];
                    }
        }
    }

    // 8 elements of a row from feature d on, as they lie in memory
    auto fetch = [&](uint4 (&raw)[RAW], const void* base, int64_t at, int d, int dim, bool vec, bool live) {
#pragma unroll
        for (int i = 0; i < RAW; ++i) {
            raw[i] = make_uint4(0, 0, 0, 0);
            const int e = d + i * (16 / ES);
            if (!live) continue;
            if (vec) {
                if (e < dim) raw[i] = *reinterpret_cast<const uint4*>((const char*) base + (at + e) * ES);
            } else if constexpr (ES == 4) {
                const uint32_t* p = (const uint32_t*) base + at;
                raw[i] = make_uint4(e < dim ? p[e] : 0, e + 1 < dim ? p[e + 1] : 0, e + 2 < dim ? p[e + 2] : 0, e + 3 < dim ? p[e + 3] : 0);
            } else {
                const uint16_t* p = (const uint16_t*) base + at;
                uint32_t w[4];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    w[j] = (e + 2 * j < dim ? p[e + 2 * j] : 0u) | (e + 2 * j + 1 < dim ? (uint32_t) p[e + 2 * j + 1] << 16 : 0u);
                raw[i] = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
    };
    // their bfloat16 parts
    auto parts = [&](const uint4 (&raw)[RAW], uint4 (&p)[NP]) {
        if constexpr (NP == 1) {
            p[0] = raw[0];
        } else {
            float f[8];
            if constexpr (NP == 2) Vec<H3S_F16>::unpack(raw[0], f);
            else {
                Vec<H3S_F32>::unpack(raw[0], f);
                Vec<H3S_F32>::unpack(raw[RAW - 1], f + 4);
            }
            uint32_t w[4][NP];
#pragma unroll
            for (int j = 0; j < 4; ++j) lin_split<NP>(f[2 * j], f[2 * j + 1], w[j]);
#pragma unroll
            for (int x = 0; x < NP; ++x) p[x] = make_uint4(w[0][x], w[1][x], w[2][x], w[3][x]);
        }
    };
    // 16-byte place of a token's slot: 8 tokens that are read side by side lie on all banks
    auto mix = [](int token) { return ((token & 1) << 2) | (token & 2) | ((token >> 2) & 1); };
    auto at_k = [&](int token, int slot) { return token * (DKP / 8) + (slot ^ mix(token)); };
    auto at_v = [&](int token, int slot) { return token * (DVB / 8) + (slot ^ mix(token)); };

    uint4 rq[OUT ? KP : 1][RAW], rk[KP][RAW], rv[VP][RAW];
    const int64_t qo = (int64_t) (h / P.q_each) * P.dk, ko = (int64_t) (h / P.k_each) * P.dk, vo = (int64_t) (h / P.v_each) * P.dv + col0;
    auto load = [&](int c0) {
#pragma unroll
        for (int i = 0; i < KP; ++i) {
            const int p = threadIdx.x + 256 * i, token = p / (DKP / 8), d = p % (DKP / 8) * 8;
            const bool live = c0 + token < count;
            if constexpr (OUT) fetch(rq[i], P.q, (row0 + c0 + token) * P.q_stride + qo, d, P.dk, P.q_vec, live);
            fetch(rk[i], P.k, (row0 + c0 + token) * P.k_stride + ko, d, P.dk, P.k_vec, live);
        }
#pragma unroll
        for (int i = 0; i < VP; ++i) {
            const int p = threadIdx.x + 256 * i, token = p / (DVB / 8), d = p % (DVB / 8) * 8;
            fetch(rv[i], P.v, (row0 + c0 + token) * P.v_stride + vo, d, P.dv - col0, P.v_vec, c0 + token < count);
        }
    };
    // Of a token with an infinity or NaN in v on, results are NaN, and earlier ones do not meet it: 0 times it would be NaN.
    auto finite = [&](const uint4 (&raw)[RAW]) {
        bool bad = false;
#pragma unroll
        for (int i = 0; i < RAW; ++i) {
            const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (DT == H3S_F32) bad |= (w[j] & 0x7f800000u) == 0x7f800000u;
                else {
                    constexpr uint32_t M = DT == H3S_BF16 ? 0x7f80u : 0x7c00u;
                    bad |= (w[j] & M) == M || (w[j] & (M << 16)) == M << 16;
                }
            }
        }
        return !bad;
    };
    auto stage = [&](int par) {
#pragma unroll
        for (int i = 0; i < KP; ++i) {
            const int p = threadIdx.x + 256 * i, token = p / (DKP / 8), slot = p % (DKP / 8);
            uint4 x[NP];
            if constexpr (OUT) {
                parts(rq[i], x);
#pragma unroll
                for (int y = 0; y < NP; ++y) sq[y][at_k(token, slot)] = x[y];
            }
            parts(rk[i], x);
#pragma unroll
            for (int y = 0; y < NP; ++y) sk[y][at_k(token, slot)] = x[y];
        }
#pragma unroll
        for (int i = 0; i < VP; ++i) {
            const int p = threadIdx.x + 256 * i, token = p / (DVB / 8), slot = p % (DVB / 8);
            uint4 x[NP];
            if (OUT && !finite(rv[i])) atomicMin(&first_bad[par], token);
            parts(rv[i], x);
#pragma unroll
            for (int y = 0; y < NP; ++y) sv[y][at_v(token, slot)] = x[y];
        }
    };
    // the transposing read: lane 4 r + m of a lane group gives 4 features of the row r, and lane c gets feature c of the four rows
    auto turned = [&](const uint4* area, int place16, int half) {
        const auto* p = (const __attribute__((address_space(3))) char*) area + place16 * 16 + half * 8;
        return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s_lin*) p));
    };
    const int tr = l15 >> 2, tm = l15 & 3;
    // operand of v: feature vcol(x, l15), the tokens 32 u + 4 g + 0..3 and 16 on
    auto v_operand = [&](int y, int u, int x) {
        uint2 a[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int token = 32 * u + 16 * e + 4 * g + tr, c = wave * 16 * NV + (NV == 2 ? 8 * tm + 4 * x : 4 * tm);
            a[e] = turned(sv[y], at_v(token, c >> 3), (c >> 2) & 1);
        }
        return make_uint4(a[0].x, a[0].y, a[1].x, a[1].y);
    };
    // operand of k: row r of the tile t stands for the feature 16 (t & ~1) + 8 (r / 4) + 4 (t & 1) + r % 4; tokens as v's
    auto kt_operand = [&](int y, int u, int t) {
        uint2 a[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int token = 32 * u + 16 * e + 4 * g + tr;
            a[e] = turned(sk[y], at_k(token, 2 * (t & ~1) + tm), t & 1);
        }
        return make_uint4(a[0].x, a[0].y, a[1].x, a[1].y);
    };

    // l^(m-1-j) for the lane's tokens j of a piece of m, and l^m - 1
    float wv[U][8], less = 0.0f;
    auto weights = [&](int m) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < 8; ++j) wv[u][j] = fade(m - 1 - (32 * u + 16 * (j >> 2) + 4 * g + (j & 3)));
        less = expm1f(-decay * (float) m);
    };
    weights(C);
    float li[OUT ? CT : 1];
    if constexpr (OUT) {
#pragma unroll
        for (int e = 0; e < CT; ++e) li[e] = fade(16 * e + l15 + 1) * P.scale;
        // the tiles right of the diagonal that share an operand with one on it
        for (int i = threadIdx.x; i < CT * U * NS * 64; i += 256) (&sp[0][0][0])[i] = make_uint4(0, 0, 0, 0);
        if (threadIdx.x < 2) first_bad[threadIdx.x] = INT32_MAX;
    }
    load(0);
    lds_barrier();
    int par = 0;
    for (int c0 = 0; c0 < count; c0 += C, par ^= 1) {
        stage(par);
        const int m = min(C, count - c0);
        lds_barrier();
        if (c0 + C < count) load(c0 + C);
        if constexpr (OUT) {
            if (threadIdx.x == 0) first_bad[par ^ 1] = INT32_MAX;
            const int bad = first_bad[par];
            // P^T = K Q^T . D of every fourth tile, as an operand
            for (int e = wave; e < CT * (CT + 1) / 2; e += 4) {
                const int ti = e >= 6 ? 3 : e >= 3 ? 2 : e >= 1 ? 1 : 0, tj = e - ti * (ti + 1) / 2;
                v4f_lin x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int u = 0; u < KC; ++u) {
                    uint4 a[NP], b[NP];
#pragma unroll
                    for (int y = 0; y < NP; ++y) {
                        a[y] = sk[y][at_k(16 * tj + l15, 4 * u + g)];
                        b[y] = sq[y][at_k(16 * ti + l15, 4 * u + g)];
                    }
#pragma unroll
                    for (int y = 0; y < NP; ++y)
#pragma unroll
                        for (int z = 0; z < NP; ++z)
                            if (NP < 3 || y + z < NP) x = lin_mma(a[y], b[z], x);
                }
                float f[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int steps = 16 * (ti - tj) + l15 - 4 * g - i;
                    f[i] = steps < 0 ? 0.0f : x[i] * (fade(steps) * P.scale);
                }
                uint32_t w[2][NS];
                lin_split<NS>(f[0], f[1], w[0]);
                lin_split<NS>(f[2], f[3], w[1]);
#pragma unroll
                for (int y = 0; y < NS; ++y)
                    reinterpret_cast<uint2*>(&sp[ti * U + (tj >> 1)][y][lane])[tj & 1] = make_uint2(w[0][y], w[1][y]);
            }
            // O^T = S^T Q^T, then the rows' decay
            v4f_lin o[CT][NV];
#pragma unroll
            for (int e = 0; e < CT; ++e)
#pragma unroll
                for (int x = 0; x < NV; ++x) o[e][x] = v4f_lin{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int u = 0; u < KC; ++u) {
                uint4 a[NV][NS];
#pragma unroll
                for (int x = 0; x < NV; ++x) {
                    uint32_t w[4][NS];
#pragma unroll
                    for (int j = 0; j < 4; ++j) lin_split<NS>(s[2 * u + (j >> 1)][x][2 * (j & 1)], s[2 * u + (j >> 1)][x][2 * (j & 1) + 1], w[j]);
#pragma unroll
                    for (int y = 0; y < NS; ++y) a[x][y] = make_uint4(w[0][y], w[1][y], w[2][y], w[3][y]);
                }
#pragma unroll
                for (int e = 0; e < CT; ++e) {
                    uint4 b[NP];
#pragma unroll
                    for (int y = 0; y < NP; ++y) b[y] = sq[y][at_k(16 * e + l15, 4 * u + g)];
#pragma unroll
                    for (int y = 0; y < NS; ++y)
#pragma unroll
                        for (int z = 0; z < NP; ++z)
                            if (y + z < NS)
#pragma unroll
                                for (int x = 0; x < NV; ++x) o[e][x] = lin_mma(a[x][y], b[z], o[e][x]);
                }
            }
#pragma unroll
            for (int e = 0; e < CT; ++e)
#pragma unroll
                for (int x = 0; x < NV; ++x) o[e][x] *= li[e];
            lds_barrier();
            // O^T += V^T P^T
#pragma unroll
            for (int u = 0; u < U; ++u) {
                uint4 a[NV][NP];
#pragma unroll
                for (int x = 0; x < NV; ++x)
#pragma unroll
                    for (int y = 0; y < NP; ++y) {
                        a[x][y] = v_operand(y, u, x);
                        if (__builtin_expect(bad < C, 0)) {
                            uint32_t w[4] = {a[x][y].x, a[x][y].y, a[x][y].z, a[x][y].w};
#pragma unroll
                            for (int j = 0; j < 8; ++j)
                                if (32 * u + 16 * (j >> 2) + 4 * g + (j & 3) >= bad) w[j >> 1] &= j & 1 ? 0xffffu : 0xffff0000u;
                            a[x][y] = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                    }
#pragma unroll
                for (int e = 2 * u; e < CT; ++e) {
                    uint4 b[NS];
#pragma unroll
                    for (int y = 0; y < NS; ++y) b[y] = sp[e * U + u][y][lane];
#pragma unroll
                    for (int y = 0; y < NP; ++y)
#pragma unroll
                        for (int z = 0; z < NS; ++z)
                            if (y + z < NS)
#pragma unroll
                                for (int x = 0; x < NV; ++x) o[e][x] = lin_mma(a[x][y], b[z], o[e][x]);
                }
            }
#pragma unroll
            for (int e = 0; e < CT; ++e) {
                const int i = 16 * e + l15;
                if (i >= m) continue;
                const int64_t at = ((row0 + c0 + i) * P.heads + h) * P.dv;
                if (__builtin_expect(i >= bad, 0))
#pragma unroll
                    for (int x = 0; x < NV; ++x) o[e][x] = v4f_lin{__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
#pragma unroll
                for (int x = 0; x < NV; ++x) {
                    const int c = mycol + vcol(x, 4 * g);
                    if (P.out_vec) {
                        if (c >= P.dv) continue;
                        if (P.out_dt == H3S_F32) *reinterpret_cast<v4f_lin*>((float*) P.out + at + c) = o[e][x];
                        else *reinterpret_cast<uint2*>((uint16_t*) P.out + at + c) =
                                 P.out_dt == H3S_BF16 ? make_uint2(pack_bf16(o[e][x][0], o[e][x][1]), pack_bf16(o[e][x][2], o[e][x][3]))
                                                      : make_uint2(pack_f16(o[e][x][0], o[e][x][1]), pack_f16(o[e][x][2], o[e][x][3]));
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (c + j < P.dv) store_any(P.out, P.out_dt, at + c + j, o[e][x][j]);
                    }
                }
            }
        }
        // S = l^m S + K^T (l^(m-1-j) V)
        if (m < C) weights(m);
#pragma unroll
        for (int t = 0; t < 2 * KC; ++t)
#pragma unroll
            for (int x = 0; x < NV; ++x)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[t][x][i] = __builtin_fmaf(s[t][x][i], less, s[t][x][i]);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            uint4 b[NV][3];
#pragma unroll
            for (int x = 0; x < NV; ++x) {
                float f[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) f[j] = 0.0f;
#pragma unroll
                for (int y = 0; y < NP; ++y) {
                    float e[8];
                    Vec<H3S_BF16>::unpack(v_operand(y, u, x), e);
#pragma unroll
                    for (int j = 0; j < 8; ++j) f[j] = y ? f[j] + e[j] : e[j];
                }
                uint32_t w[4][3];
#pragma unroll
                for (int j = 0; j < 4; ++j) lin_split<3>(f[2 * j] * wv[u][2 * j], f[2 * j + 1] * wv[u][2 * j + 1], w[j]);
#pragma unroll
                for (int y = 0; y < 3; ++y) b[x][y] = make_uint4(w[0][y], w[1][y], w[2][y], w[3][y]);
            }
#pragma unroll
            for (int t = 0; t < 2 * KC; ++t) {
                uint4 a[NP];
#pragma unroll
                for (int y = 0; y < NP; ++y) a[y] = kt_operand(y, u, t);
#pragma unroll
                for (int y = 0; y < NP; ++y)
#pragma unroll
                    for (int z = 0; z < 3; ++z)
                        if (y + z < 3)
#pragma unroll
                            for (int x = 0; x < NV; ++x) s[t][x] = lin_mma(a[y], b[x][z], s[t][x]);
            }
        }
        lds_barrier();
    }

    if constexpr (!OUT) {
#pragma unroll
        for (int t = 0; t < 2 * KC; ++t)
#pragma unroll
            for (int x = 0; x < NV; ++x) *reinterpret_cast<v4f_lin*>(ws + (t * NV + x) * 1024) = s[t][x];
    } else {
        const int64_t to = P.target[it.b];
        if (it.seg + 1 < it.segs || to < 0 || to >= P.slots) return;
        float* sp0 = P.s + (to * P.heads + h) * head;
#pragma unroll
        for (int t = 0; t < 2 * KC; ++t)
#pragma unroll
            for (int x = 0; x < NV; ++x)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int d = 16 * (t & ~1) + 8 * g + 4 * (t & 1) + i, c = mycol + vcol(x, l15);
                    if (d < P.dk && c < P.dv) sp0[(int64_t) d * P.dv + c] = s[t][x][i];
                }
    }
}

void lin_chunk_bf16(Ctx* c, const LinArgs& P, int kc, int nv, int64_t blocks, bool out);
void lin_chunk_f16(Ctx* c, const LinArgs& P, int kc, int nv, int64_t blocks, bool out);
void lin_chunk_f32(Ctx* c, const LinArgs& P, int kc, int nv, int64_t blocks, bool out);

template <int DT, int KC, int NV> static void lin_chunk_run(Ctx* c, const LinArgs& P, int64_t blocks, bool out) {
    if (out) lin_chunk_kernel<DT, KC, NV, true><<<(unsigned) blocks, 256, 0, c->stream>>>(P);
    else lin_chunk_kernel<DT, KC, NV, false><<<(unsigned) blocks, 256, 0, c->stream>>>(P);
}
template <int DT> static void lin_chunk_type(Ctx* c, const LinArgs& P, int kc, int nv, int64_t blocks, bool out) {
    if (kc == 2 && nv == 1) lin_chunk_run<DT, 2, 1>(c, P, blocks, out);
    else if (kc == 2) lin_chunk_run<DT, 2, 2>(c, P, blocks, out);
    else if (kc == 4 && nv == 1) lin_chunk_run<DT, 4, 1>(c, P, blocks, out);
    else if (kc == 4) lin_chunk_run<DT, 4, 2>(c, P, blocks, out);
    else if (kc == 6) lin_chunk_run<DT, 6, 1>(c, P, blocks, out);
    else lin_chunk_run<DT, 8, 1>(c, P, blocks, out);
}

}  // namespace h3
