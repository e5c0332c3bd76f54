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
// Work: a block of NW wavefronts has one head's piece after piece of a segment of a sequence, and 16 NW NV features of v, 16 NV a
// wavefront. Where heads and sequences are too few for the device, a sequence is split into segments: first each segment's own sums (this
// kernel without outputs), then the states at their beginnings (lin_scan_kernel), then the outputs.
//
// Bound (8192 tokens, 64 heads of 128 x 128, bfloat16, eight segments): the outputs, 150-180 us by the card's clock, by the issue of vector
// instructions beside the products: a wavefront's piece of 64 tokens is 194 products and some 800 others (powers of l, parts, addresses), which
// one SIMD's two wavefronts overlap little: the matrix cores are busy a third of the time. The segments' sums, 61-73 us, by k's and v's bytes
// (4.4-3.7 TB/s). float16 298 us in all, float32 442.
// Registers that go to memory, in the outputs of blocks of 128 features of values: float32 with 97 to 128 features of keys 3, rows off 16 bytes
// 19 (and bfloat16 2); the other rows off 16 bytes up to 16 scalar ones.
#pragma once

#include "lin.h"

namespace h3 {

typedef __bf16 v8b_lin __attribute__((ext_vector_type(8)));
typedef __bf16 v2b_lin __attribute__((ext_vector_type(2)));
typedef float v2f_lin __attribute__((ext_vector_type(2)));
typedef float v4f_lin __attribute__((ext_vector_type(4)));
typedef short v4s_lin __attribute__((ext_vector_type(4)));
typedef uint32_t v2u_lin __attribute__((ext_vector_type(2)));
typedef uint32_t v4u_lin __attribute__((ext_vector_type(4)));

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
        p[0] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
        p[1] = __builtin_amdgcn_perm(__float_as_uint(rb), __float_as_uint(ra), 0x07060302u);
        p[2] = lin_pack(ra - __uint_as_float(va), rb - __uint_as_float(vb));
    } else {
        p[0] = lin_pack(a, b);
        if constexpr (N == 2) p[1] = lin_pack(a - bf16_lo(p[0]), b - bf16_hi(p[0]));
    }
}
// a buffer resource over `bytes` from p on (a function: from a lambda that returns one, the kernel lost its host stub)
__device__ __forceinline__ __amdgpu_buffer_rsrc_t lin_rows(const char* p, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc((void*) p, (short) 0, bytes, 0x00020000);
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
            segs = (int) (((uint32_t) n + (uint32_t) P.seg - 1) / (uint32_t) P.seg);
        } else {                                                            // a segment is a sequence
            b = place;
            kv_rows_of(P.kv, b, r0, n);
            seg = 0;
            segs = n > 0;
        }
        return seg >= 0 && seg < segs && (uint32_t) n >= P.least && (uint32_t) n <= P.most;
    }
};

template <int DT, int KC, int NW, int NV> struct LinShape {
    static constexpr int NP = DT == H3S_BF16 ? 1 : DT == H3S_F16 ? 2 : 3;   // parts of an input
    static constexpr int NS = NP == 3 ? 3 : 2;                              // of the state and of a piece's products
    static constexpr int CT = NP == 1 && KC <= 4 ? 4 : 2, C = 16 * CT, U = CT / 2;
    // (in LDS a row is an even number of steps)
    static constexpr int T = 64 * NW, DKP = 64 * ((KC + 1) / 2), DVB = 16 * NW * NV;
};

template <int DT, int KC, int NW, int NV, bool OUT, bool VEC>
__global__ __launch_bounds__(64 * NW, (DT == H3S_F32 && KC > 4 && NW == 4 && OUT ? 1 : 2)) void lin_chunk_kernel(LinArgs P) {   // (1: LDS for one block)
    using Sh = LinShape<DT, KC, NW, NV>;
    constexpr int NP = Sh::NP, NS = Sh::NS, CT = Sh::CT, C = Sh::C, U = Sh::U, DKP = Sh::DKP, DVB = Sh::DVB, T = Sh::T;
    constexpr int ES = DT == H3S_F32 ? 4 : 2, RAW = ES / 2;                 // 16-byte loads for 8 elements
    constexpr int KN = C * DKP / 8, KP = (KN + T - 1) / T, VP = C * DVB / 8 / T;   // pieces of 8 elements, and those of a thread
    static_assert(VP * T * 8 == C * DVB, "a piece of v is whole pieces of the threads");
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

    // the state: register i of s[2 u + p][x]: keys' feature 32 u + 8 g + 4 p + i, v's feature mycol + 16 x + l15
    v4f_lin s[2 * KC][NV];
#pragma unroll
    for (int t = 0; t < 2 * KC; ++t)
#pragma unroll
        for (int x = 0; x < NV; ++x) s[t][x] = v4f_lin{0.0f, 0.0f, 0.0f, 0.0f};
    float* ws = P.ws + (int64_t) blockIdx.x * (32 * KC * DVB) + threadIdx.x * 4;
    const int64_t head = (int64_t) P.dk * P.dv;
    if (OUT && it.segs > 1) {
#pragma unroll
        for (int t = 0; t < 2 * KC; ++t)
#pragma unroll
            for (int x = 0; x < NV; ++x) s[t][x] = *reinterpret_cast<const v4f_lin*>(ws + (t * NV + x) * (4 * T));
    } else if (OUT) {
        const int64_t from = P.source[it.b];
        if (from >= 0 && from < P.slots) {
            const float* sp0 = P.s + (from * P.heads + h) * head + mycol + l15;
#pragma unroll
            for (int t = 0; t < 2 * KC; ++t)
#pragma unroll
                for (int x = 0; x < NV; ++x)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int d = 16 * (t & ~1) + 8 * g + 4 * (t & 1) + i;
                        if (d < P.dk && mycol + 16 * x + l15 < P.dv) s[t][x][i] = sp0[(int64_t) d * P.dv + 16 * x];
                    }
        }
    }

    // 8 elements of a row from feature d on, as they lie in memory, of a tensor whose row is not whole 16-byte pieces
    auto fetch = [&](uint4 (&raw)[RAW], const char* base, int64_t at, int d, int dim, bool live) {
#pragma unroll
        for (int i = 0; i < RAW; ++i) {
            raw[i] = make_uint4(0, 0, 0, 0);
            const int e = d + i * (16 / ES);
            if (!live || e >= dim) continue;
            if constexpr (ES == 4) {
                const uint32_t* p = (const uint32_t*) base + at;
                raw[i] = make_uint4(p[e], e + 1 < dim ? p[e + 1] : 0, e + 2 < dim ? p[e + 2] : 0, e + 3 < dim ? p[e + 3] : 0);
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
    // The same of whole pieces, through a buffer resource over the rows that there are: what lies behind them reads as zeros.
    // (at: bytes from the first row, 2^31 and more where there is no such feature; stays there with 64 rows' bytes, below 2^30, added)
    auto fetch16 = [&](uint4 (&raw)[RAW], const __amdgpu_buffer_rsrc_t& rows, const uint32_t (&at)[RAW], uint32_t on) {
#pragma unroll
        for (int i = 0; i < RAW; ++i) raw[i] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rows, (int) (at[i] + on), 0, 0));
    };
    auto distance = [&](uint32_t (&at)[RAW], uint32_t token, uint32_t stride, int d, int dim, bool live) {
#pragma unroll
        for (int i = 0; i < RAW; ++i) {
            const int e = d + i * (16 / ES);
            at[i] = live && e < dim ? (token * stride + e) * ES : 0x80000000u;
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
    // The 16-byte place of a token's slot (8 features): the slot's low bits are mixed with the token's, so that the lanes of an access that are
    // served together lie on as many of the 64 banks as they can. Those of a 16-byte read are 0-3, 12-15 and 20-27, and 4-11, 16-19 and
    // 28-31 (counted): rows of q and k, a token a lane and two neighbouring slots, so the slots' last bit goes with one of a token's last
    // two (8192 tokens of 64 heads: 7.5 to 2.8 million cycles of conflicts, 149.7 to 147.7 us). A transposing read of k meets eight tokens by
    // four slots, of v by two: other bits of the token's for v.
    auto mix_k = [](uint32_t rows, uint32_t token) {                        // rows: slots a token
        return rows % 16 == 0 ? ((token & 2) << 2) | (token & 4) | ((token >> 2) & 2) | (token & 1) : (token & 4) | ((token >> 2) & 2) | ((token >> 1) & 1);
    };
    auto mix_v = [](uint32_t rows, uint32_t token) {
        return rows % 16 == 0 ? ((token & 3) << 2) | ((token >> 1) & 2) | ((token >> 3) & 1) : ((token & 2) << 1) | ((token >> 1) & 2) | ((token >> 3) & 1);
    };
    auto at_k = [&](uint32_t token, uint32_t slot) { return token * (DKP / 8) + (slot ^ mix_k(DKP / 8, token)); };
    auto at_v = [&](uint32_t token, uint32_t slot) { return token * (DVB / 8) + (slot ^ mix_v(DVB / 8, token)); };

    // a thread's pieces of 8 elements are the same features of every KS-th (VS-th) token, where a row's pieces divide the threads: their places in
    // LDS then differ by constants, if those tokens are 16 or more apart (the mix goes by a token's lowest four bits)
    constexpr int KR = DKP / 8, VR = DVB / 8, KS = T % KR == 0 && T / KR % 16 == 0 ? T / KR : 0, VS = T / VR;
    static_assert(VS % 16 == 0, "the same mix for all of a thread's pieces");
    uint4 rq[OUT ? KP : 1][RAW], rk[KP][RAW], rv[VP][RAW];
    const char* const qp = (const char*) P.q + (row0 * P.q_stride + (int64_t) (h / P.q_each) * P.dk) * ES;
    const char* const kp = (const char*) P.k + (row0 * P.k_stride + (int64_t) (h / P.k_each) * P.dk) * ES;
    const char* const vp = (const char*) P.v + (row0 * P.v_stride + (int64_t) (h / P.v_each) * P.dv + col0) * ES;
    auto load = [&](int c0) {
        // (the tokens of a piece that is not whole stand at its end, behind zeros: what fades by a token's distance from the end is then
        // the same in every piece)
        const int left = min(C, count - c0), none = C - left;
        uint32_t me = threadIdx.x;
        asm volatile("" : "+v"(me));                                        // (distances are found again rather than kept)
        if constexpr (VEC) {
            const auto qr = lin_rows(qp + c0 * P.q_stride * ES, ((left - 1) * (int) P.q_stride + P.dk) * ES);
            const auto kr = lin_rows(kp + c0 * P.k_stride * ES, ((left - 1) * (int) P.k_stride + P.dk) * ES);
            const auto vr = lin_rows(vp + c0 * P.v_stride * ES, ((left - 1) * (int) P.v_stride + min(P.dv - col0, DVB)) * ES);
            const uint32_t qs = (uint32_t) P.q_stride, ks = (uint32_t) P.k_stride, vs = (uint32_t) P.v_stride;
            uint32_t at[RAW], bt[RAW];
            if constexpr (KS > 0) {
                const int d = me % KR * 8;
                const uint32_t token = me / KR - none;                      // (below 0: far behind the rows)
                distance(bt, token, ks, d, P.dk, true);
                if constexpr (OUT) distance(at, token, qs, d, P.dk, true);
#pragma unroll
                for (int i = 0; i < KP; ++i) {
                    if constexpr (OUT) fetch16(rq[i], qr, at, KS * i * qs * ES);
                    fetch16(rk[i], kr, bt, KS * i * ks * ES);
                }
            } else {
#pragma unroll
                for (int i = 0; i < KP; ++i) {
                    const int p = me + T * i, d = p % KR * 8;
                    const uint32_t token = p / KR - none;
                    const bool live = KN % T == 0 || p < KN;
                    distance(bt, token, ks, d, P.dk, live);
                    fetch16(rk[i], kr, bt, 0);
                    if constexpr (OUT) {
                        distance(at, token, qs, d, P.dk, live);
                        fetch16(rq[i], qr, at, 0);
                    }
                }
            }
            distance(at, me / VR - none, vs, me % VR * 8, P.dv - col0, true);
#pragma unroll
            for (int i = 0; i < VP; ++i) fetch16(rv[i], vr, at, VS * i * vs * ES);
        } else {
#pragma unroll
            for (int i = 0; i < KP; ++i) {
                const int p = me + T * i, token = p / KR - none, d = p % KR * 8;
                const bool live = token >= 0 && token < left;
                if constexpr (OUT) fetch(rq[i], qp, (c0 + token) * P.q_stride, d, P.dk, live);
                fetch(rk[i], kp, (c0 + token) * P.k_stride, d, P.dk, live);
            }
#pragma unroll
            for (int i = 0; i < VP; ++i) {
                const int p = me + T * i, token = p / VR - none, d = p % VR * 8;
                fetch(rv[i], vp, (c0 + token) * P.v_stride, d, P.dv - col0, token >= 0);
            }
        }
    };
    // Of a token with an infinity or NaN in v on, results are NaN, and earlier ones do not meet it: 0 times it would be NaN. (Two or one values
    // a word: an exponent of ones carries into the sign's place.)
    auto finite = [&](const uint4 (&raw)[RAW]) {
        constexpr uint32_t SIGN = DT == H3S_F32 ? 0x80000000u : 0x80008000u, ONE = DT == H3S_F32 ? 0x00800000u : DT == H3S_BF16 ? 0x00800080u : 0x04000400u;
        uint32_t any = 0;
#pragma unroll
        for (int i = 0; i < RAW; ++i)
            any |= ((raw[i].x & ~SIGN) + ONE) | ((raw[i].y & ~SIGN) + ONE) | ((raw[i].z & ~SIGN) + ONE) | ((raw[i].w & ~SIGN) + ONE);
        return (any & SIGN) == 0;
    };
    // (all of a thread's at once: the largest of each half word)
    auto all_finite = [&]() {
        if constexpr (DT == H3S_F32) {
            bool all = true;
#pragma unroll
            for (int i = 0; i < VP; ++i) all = all && finite(rv[i]);
            return all;
        } else {
            typedef uint16_t v2 __attribute__((ext_vector_type(2)));
            constexpr uint32_t E = DT == H3S_BF16 ? 0x7f80u : 0x7c00u;
            v2 top = {0, 0};
            auto one = [&](uint32_t w) { top = __builtin_elementwise_max(top, __builtin_bit_cast(v2, w & 0x7fff7fffu)); };
#pragma unroll
            for (int i = 0; i < VP; ++i) { one(rv[i][0].x); one(rv[i][0].y); one(rv[i][0].z); one(rv[i][0].w); }
            const uint32_t w = __builtin_bit_cast(uint32_t, top);
            return (w & 0xffffu) < E && (w >> 16) < E;
        }
    };
    const uint32_t k_to = at_k(threadIdx.x / KR, threadIdx.x % KR), v_to = at_v(threadIdx.x / VR, threadIdx.x % VR);
    auto stage = [&](int par) {
#pragma unroll
        for (int i = 0; i < KP; ++i) {
            const uint32_t p = threadIdx.x + T * i, to = KS ? k_to + KS * KR * i : at_k(p / KR, p % KR);
            if (KN % T != 0 && p >= KN) continue;
            uint4 x[NP];
            if constexpr (OUT) {
                parts(rq[i], x);
#pragma unroll
                for (int y = 0; y < NP; ++y) sq[y][to] = x[y];
            }
            parts(rk[i], x);
#pragma unroll
            for (int y = 0; y < NP; ++y) sk[y][to] = x[y];
        }
        if (OUT && __builtin_expect(!all_finite(), 0))
            for (int i = VP - 1; i >= 0; --i)
                if (!finite(rv[i])) atomicMin(&first_bad[par], (int) (threadIdx.x / VR + VS * i));
#pragma unroll
        for (int i = 0; i < VP; ++i) {
            uint4 x[NP];
            parts(rv[i], x);
#pragma unroll
            for (int y = 0; y < NP; ++y) sv[y][v_to + VS * VR * i] = x[y];
        }
    };
    // the transposing read: lane 4 r + m of a lane group gives 4 features of the row r, and lane c gets feature c of the four rows
    auto turned = [&](const uint4* area, uint32_t place16, uint32_t half) {
        const auto* p = (const __attribute__((address_space(3))) char*) area + place16 * 16 + half * 8;
        return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s_lin*) p));
    };
    const int tr = l15 >> 2, tm = l15 & 3;
    // (The places of the loops' operands: a slot's low bits meet those of the lane's place as an exclusive or, the rest is added.)
    constexpr uint32_t LOW = DKP / 8 % 16 == 0 ? 15 : 7;
    const uint32_t row_at = at_k(l15, g), turn_at = at_k(4 * g + tr, tm), v_at = at_v(4 * g + tr, 2 * NV * wave + (tm >> 1));
    // operand of q or k: token 16 e + l15, the features 32 u + 8 g + 0..7
    auto rows_of = [&](const uint4* area, uint32_t e, uint32_t u) { return area[(row_at ^ (4 * u & LOW)) + 16 * e * (DKP / 8) + (4 * u & ~LOW)]; };
    // operand of v: feature mycol + 16 x + l15, the tokens 32 u + 4 g + 0..3 and 16 on
    auto v_operand = [&](int y, int u, int x) {
        const uint32_t at = v_at ^ (2 * x);
        const uint2 a = turned(sv[y], at + 32 * u * (DVB / 8), tm & 1), b = turned(sv[y], at + (32 * u + 16) * (DVB / 8), tm & 1);
        return make_uint4(a.x, a.y, b.x, b.y);
    };
    // operand of k: row r of the tile t stands for the feature 16 (t & ~1) + 8 (r / 4) + 4 (t & 1) + r % 4; tokens as v's
    auto kt_operand = [&](int y, int u, int t) {
        const uint32_t slot = 4 * (t >> 1), at = (turn_at ^ (slot & LOW)) + (slot & ~LOW);
        const uint2 a = turned(sk[y], at + 32 * u * (DKP / 8), t & 1), b = turned(sk[y], at + (32 * u + 16) * (DKP / 8), t & 1);
        return make_uint4(a.x, a.y, b.x, b.y);
    };

    // Powers of l as products of a lane's own and the same for all lanes, each between 0 and 1: l^(i+1) of the lane's rows i = 16 e + l15 of a
    // piece, and l^(C-1-j) for its tokens j = 32 u + 16 e + 4 g + i. (Kept as few as they are: a few registers more and the loop's addresses
    // went to memory, with a wait for the loads in flight at each.)
    auto same = [](float x) { return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(x))); };
    const float less_whole = same(expm1f(-decay * (float) C));              // l^C - 1
    const float lp[4] = {1.0f, same(fade(1)), same(fade(2)), same(fade(3))}, lt[4] = {1.0f, same(fade(16)), same(fade(32)), same(fade(48))};
    const float row_fade = fade(l15 + 1) * P.scale, back_fade = fade(12 - 4 * g), left_fade = fade(13 + l15 - 4 * g) * P.scale;
    if constexpr (OUT) {
        // the tiles right of the diagonal that share an operand with one on it
        for (int i = threadIdx.x; i < CT * U * NS * 64; i += T) (&sp[0][0][0])[i] = make_uint4(0, 0, 0, 0);
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
        v4f_lin o[OUT ? CT : 1][NV];
        if constexpr (OUT) {
            if (threadIdx.x == 0) first_bad[par ^ 1] = INT32_MAX;
            // P^T = K Q^T . D of every NW-th tile, as an operand
            for (int e = wave; e < CT * (CT + 1) / 2; e += NW) {
                const int ti = e >= 6 ? 3 : e >= 3 ? 2 : e >= 1 ? 1 : 0, tj = e - ti * (ti + 1) / 2;
                v4f_lin z2[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
                for (int u = 0; u < KC; ++u) {
                    uint4 a[NP], b[NP];
#pragma unroll
                    for (int y = 0; y < NP; ++y) {
                        a[y] = rows_of(sk[y], tj, u);
                        b[y] = rows_of(sq[y], ti, u);
                    }
#pragma unroll
                    for (int y = 0; y < NP; ++y)
#pragma unroll
                        for (int z = 0; z < NP; ++z)
                            if (NP < 3 || y + z < NP) z2[u & 1] = lin_mma(a[y], b[z], z2[u & 1]);
                }
                const v4f_lin x = z2[0] + z2[1];
                float f[4];
                if (ti == tj) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int steps = l15 - 4 * g - i;
                        f[i] = steps < 0 ? 0.0f : x[i] * (fade(steps) * P.scale);
                    }
                } else {                                                    // 16 (ti - tj) + l15 - 4 g - i steps, all above 0
                    const float w = left_fade * (ti - tj == 1 ? 1.0f : ti - tj == 2 ? lt[1] : lt[2]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) f[i] = x[i] * (w * lp[3 - i]);
                }
                uint32_t w[2][NS];
                lin_split<NS>(f[0], f[1], w[0]);
                lin_split<NS>(f[2], f[3], w[1]);
#pragma unroll
                for (int y = 0; y < NS; ++y)
                    reinterpret_cast<uint2*>(&sp[ti * U + (tj >> 1)][y][lane])[tj & 1] = make_uint2(w[0][y], w[1][y]);
            }
            // O^T = S^T Q^T, then the rows' decay. (Here and below a step's operands are read and made during the products of the step before: the
            // two blocks of a CU go in step, so that one's vector instructions do not fill the other's products.)
            uint4 qb[2][CT][NP], sa[2][NV][NS];
            auto q_operands = [&](int u) {
#pragma unroll
                for (int e = 0; e < CT; ++e)
#pragma unroll
                    for (int y = 0; y < NP; ++y) qb[u & 1][e][y] = rows_of(sq[y], e, u);
            };
            auto s_operands = [&](int u) {
#pragma unroll
                for (int x = 0; x < NV; ++x) {
                    uint32_t w[4][NS];
#pragma unroll
                    for (int j = 0; j < 4; ++j) lin_split<NS>(s[2 * u + (j >> 1)][x][2 * (j & 1)], s[2 * u + (j >> 1)][x][2 * (j & 1) + 1], w[j]);
#pragma unroll
                    for (int y = 0; y < NS; ++y) sa[u & 1][x][y] = make_uint4(w[0][y], w[1][y], w[2][y], w[3][y]);
                }
            };
            q_operands(0);
            s_operands(0);
#pragma unroll
            for (int u = 0; u < KC; ++u) {
                if (u + 1 < KC) q_operands(u + 1);
                __builtin_amdgcn_sched_barrier(0);
                if (u + 1 < KC) s_operands(u + 1);
#pragma unroll
                for (int y = 0; y < NS; ++y)
#pragma unroll
                    for (int z = 0; z < NP; ++z)
                        if (y + z < NS)
#pragma unroll
                            for (int e = 0; e < CT; ++e)
#pragma unroll
                                for (int x = 0; x < NV; ++x)
                                    o[e][x] = lin_mma(sa[u & 1][x][y], qb[u & 1][e][z], u + y + z ? o[e][x] : v4f_lin{0.0f, 0.0f, 0.0f, 0.0f});
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int e = 0; e < CT; ++e) {
                float f = row_fade;
                pin(f);
                f = m == C ? f * lt[e] : fade(16 * e + l15 + 1 - (C - m)) * P.scale;
#pragma unroll
                for (int x = 0; x < NV; ++x)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[e][x][i] *= f;
            }
            lds_barrier();
        }
        // O^T += V^T P^T, and S = l^m S + K^T (l^(C-1-j) V)
        const float less = m == C ? less_whole : expm1f(-decay * (float) m);
        uint4 va[2][NV][NP], vb[2][NV][3];
        uint32_t vw[4][3];
        auto v_operands = [&](int u) {
#pragma unroll
            for (int x = 0; x < NV; ++x)
#pragma unroll
                for (int y = 0; y < NP; ++y) va[u & 1][x][y] = v_operand(y, u, x);
        };
        float vf[8];
        // tokens 2 j and 2 j + 1 of the lane's eight, faded, as parts: piece i = 4 x + j of 4 NV
        auto v_faded = [&](int u, int i) {
            const int x = i >> 2, j = i & 3;
            float f[2] = {0.0f, 0.0f};
            if (i == 0) {
                float w = back_fade;
                pin(w);                                                     // (else all products are kept)
#pragma unroll
                for (int k = 0; k < 4; ++k) vf[k] = w * lp[3 - k];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    vf[4 + k] = vf[k] * lt[2 * U - 2 - 2 * u];
                    vf[k] *= lt[2 * U - 1 - 2 * u];
                }
            }
#pragma unroll
            for (int y = 0; y < NP; ++y) {
                const uint4& a = va[u & 1][x][y];
                const uint32_t c = j == 0 ? a.x : j == 1 ? a.y : j == 2 ? a.z : a.w;
                f[0] = y ? f[0] + bf16_lo(c) : bf16_lo(c);
                f[1] = y ? f[1] + bf16_hi(c) : bf16_hi(c);
            }
            lin_split<3>(f[0] * vf[2 * j], f[1] * vf[2 * j + 1], vw[j]);
            if (j == 3)
#pragma unroll
                for (int y = 0; y < 3; ++y) vb[u & 1][x][y] = make_uint4(vw[0][y], vw[1][y], vw[2][y], vw[3][y]);
        };
        auto s_faded = [&](int t) {
#pragma unroll
            for (int x = 0; x < NV; ++x)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[t][x][i] = __builtin_fmaf(s[t][x][i], less, s[t][x][i]);
        };
        v_operands(0);
        if constexpr (OUT) {
            const int bad = __builtin_amdgcn_readfirstlane(first_bad[par]);
            constexpr int STEPS = U == 2 ? 6 : 2, EACH = (4 * NV + STEPS - 1) / STEPS;
            int at = 0, done = 0;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                uint4 pb[2][NS], a[NV][NP];
                auto p_operand = [&](int e) {
#pragma unroll
                    for (int y = 0; y < NS; ++y) pb[e & 1][y] = sp[e * U + u][y][lane];
                };
                p_operand(2 * u);
                if (u) v_operands(u);
#pragma unroll
                for (int x = 0; x < NV; ++x)
#pragma unroll
                    for (int y = 0; y < NP; ++y) a[x][y] = va[u & 1][x][y];
                if (__builtin_expect(bad < C, 0)) {
#pragma unroll
                    for (int x = 0; x < NV; ++x)
#pragma unroll
                        for (int y = 0; y < NP; ++y) {
                            uint32_t w[4] = {a[x][y].x, a[x][y].y, a[x][y].z, a[x][y].w};
#pragma unroll
                            for (int j = 0; j < 8; ++j)
                                if (32 * u + 16 * (j >> 2) + 4 * g + (j & 3) >= bad) w[j >> 1] &= j & 1 ? 0xffffu : 0xffff0000u;
                            a[x][y] = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                }
#pragma unroll
                for (int e = 2 * u; e < CT; ++e, ++at) {
                    if (e + 1 < CT) p_operand(e + 1);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int i = 0; i < EACH; ++i)
                        if (done < 4 * NV) v_faded(0, done++);
#pragma unroll
                    for (int y = 0; y < NP; ++y)
#pragma unroll
                        for (int z = 0; z < NS; ++z)
                            if (y + z < NS)
#pragma unroll
                                for (int x = 0; x < NV; ++x) o[e][x] = lin_mma(a[x][y], pb[e & 1][z], o[e][x]);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            if (__builtin_expect(bad < C, 0)) {
#pragma unroll
                for (int e = 0; e < CT; ++e)
                    if (16 * e + l15 >= bad)
#pragma unroll
                        for (int x = 0; x < NV; ++x) o[e][x] = v4f_lin{__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
            }
#pragma unroll
            for (int x = 0; x < NV; ++x) {
                const int c = mycol + 16 * x + 4 * g;
                if constexpr (VEC) {                                        // (stores behind the rows that there are go nowhere)
                    const int os = P.out_dt == H3S_F32 ? 4 : 2, wide = P.heads * P.dv;
                    const auto rows = lin_rows((const char*) P.out + ((row0 + c0) * wide + h * P.dv) * os, ((m - 1) * wide + P.dv) * os);
                    // (rows of zeros: below 0)
                    const uint32_t at = c < P.dv ? (uint32_t) (((l15 - (C - m)) * wide + c) * os) : 0x80000000u, on = 16 * wide * os;
                    if (P.out_dt == H3S_F32) {
#pragma unroll
                        for (int e = 0; e < CT; ++e) __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(v4u_lin, o[e][x]), rows, (int) (at + e * on), 0, 0);
                    } else if (P.out_dt == H3S_BF16) {
#pragma unroll
                        for (int e = 0; e < CT; ++e)
                            __builtin_amdgcn_raw_buffer_store_b64(v2u_lin{lin_pack(o[e][x][0], o[e][x][1]), lin_pack(o[e][x][2], o[e][x][3])}, rows, (int) (at + e * on), 0, 0);
                    } else {
#pragma unroll
                        for (int e = 0; e < CT; ++e)
                            __builtin_amdgcn_raw_buffer_store_b64(v2u_lin{pack_f16(o[e][x][0], o[e][x][1]), pack_f16(o[e][x][2], o[e][x][3])}, rows, (int) (at + e * on), 0, 0);
                    }
                } else {
#pragma unroll 1
                    for (int e = 0; e < CT; ++e) {
                        const int i = 16 * e + l15 - (C - m);
                        if (i < 0) continue;
                        const int64_t at = ((row0 + c0 + i) * P.heads + h) * P.dv;
                        v4f_lin y = o[0][x];
#pragma unroll
                        for (int f = 1; f < CT; ++f) y = e == f ? o[f][x] : y;
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (c + j < P.dv) store_any(P.out, P.out_dt, at + c + j, y[j]);
                    }
                }
            }
        }
        if constexpr (!OUT) {
#pragma unroll
            for (int i = 0; i < 4 * NV; ++i) v_faded(0, i);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            constexpr int G = NP == 1 ? 2 : 1, STEPS = 2 * KC / G, EACH = (4 * NV + STEPS - 1) / STEPS;   // G tiles a step
            uint4 ka[2][G][NP];
            auto k_operands = [&](int t) {
#pragma unroll
                for (int i = 0; i < G; ++i)
#pragma unroll
                    for (int y = 0; y < NP; ++y) ka[t / G & 1][i][y] = kt_operand(y, u, t + i);
            };
            k_operands(0);
            if (!OUT && u + 1 < U) v_operands(u + 1);
            if (u == 0)
#pragma unroll
                for (int i = 0; i < G; ++i) s_faded(i);
            int done = 0;
#pragma unroll
            for (int t = 0; t < 2 * KC; t += G) {
                if (t + G < 2 * KC) k_operands(t + G);
                __builtin_amdgcn_sched_barrier(0);
                if (u == 0 && t + G < 2 * KC)
#pragma unroll
                    for (int i = 0; i < G; ++i) s_faded(t + G + i);
                if (u + 1 < U)
#pragma unroll
                    for (int i = 0; i < EACH; ++i)
                        if (done < 4 * NV) v_faded(u + 1, done++);
#pragma unroll
                for (int y = 0; y < NP; ++y)
#pragma unroll
                    for (int z = 0; z < 3; ++z)
                        if (y + z < 3)
#pragma unroll
                            for (int i = 0; i < G; ++i)
#pragma unroll
                                for (int x = 0; x < NV; ++x) s[t + i][x] = lin_mma(ka[t / G & 1][i][y], vb[u & 1][x][z], s[t + i][x]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        lds_barrier();
    }

    if constexpr (!OUT) {
#pragma unroll
        for (int t = 0; t < 2 * KC; ++t)
#pragma unroll
            for (int x = 0; x < NV; ++x) *reinterpret_cast<v4f_lin*>(ws + (t * NV + x) * (4 * T)) = s[t][x];
    } else {
        const int64_t to = P.target[it.b];
        if (it.seg + 1 < it.segs || to < 0 || to >= P.slots) return;
        float* sp0 = P.s + (to * P.heads + h) * head + mycol + l15;
#pragma unroll
        for (int t = 0; t < 2 * KC; ++t)
#pragma unroll
            for (int x = 0; x < NV; ++x)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int d = 16 * (t & ~1) + 8 * g + 4 * (t & 1) + i;
                    if (d < P.dk && mycol + 16 * x + l15 < P.dv) sp0[(int64_t) d * P.dv + 16 * x] = s[t][x][i];
                }
    }
}

// How features of keys (32 KC, in steps of 32) and a block's of values (16 NW NV) go to wavefronts: two tiles of values a wavefront read an
// operand of q and k for twice the products, as long as the state leaves room for them (keys' features up to 128). (With the rows through
// buffer resources and the operands a step ahead: 356 to 240 us for 8192 tokens of 64 heads of 128.)
template <int KC, bool WIDE> struct LinWaves { static constexpr int NV = WIDE && KC <= 4 ? 2 : 1, NW = WIDE && KC > 4 ? 8 : 4; };

void lin_chunk_bf16(Ctx* c, const LinArgs& P, int kc, bool wide, int64_t blocks, bool out);
void lin_chunk_f16(Ctx* c, const LinArgs& P, int kc, bool wide, int64_t blocks, bool out);
void lin_chunk_f32(Ctx* c, const LinArgs& P, int kc, bool wide, int64_t blocks, bool out);

template <int DT, int KC, bool WIDE> static void lin_chunk_run(Ctx* c, const LinArgs& P, int64_t blocks, bool out) {
    constexpr int NW = LinWaves<KC, WIDE>::NW, NV = LinWaves<KC, WIDE>::NV;
    if (out && P.vec) lin_chunk_kernel<DT, KC, NW, NV, true, true><<<(unsigned) blocks, 64 * NW, 0, c->stream>>>(P);
    else if (out) lin_chunk_kernel<DT, KC, NW, NV, true, false><<<(unsigned) blocks, 64 * NW, 0, c->stream>>>(P);
    else if (P.vec) lin_chunk_kernel<DT, KC, NW, NV, false, true><<<(unsigned) blocks, 64 * NW, 0, c->stream>>>(P);
    else lin_chunk_kernel<DT, KC, NW, NV, false, false><<<(unsigned) blocks, 64 * NW, 0, c->stream>>>(P);
}
template <int DT, bool WIDE> static void lin_chunk_width(Ctx* c, const LinArgs& P, int kc, int64_t blocks, bool out) {
    switch (kc) {
        case 1: lin_chunk_run<DT, 1, WIDE>(c, P, blocks, out); break;
        case 2: lin_chunk_run<DT, 2, WIDE>(c, P, blocks, out); break;
        case 3: lin_chunk_run<DT, 3, WIDE>(c, P, blocks, out); break;
        case 4: lin_chunk_run<DT, 4, WIDE>(c, P, blocks, out); break;
        case 6: lin_chunk_run<DT, 6, WIDE>(c, P, blocks, out); break;
        default: lin_chunk_run<DT, 8, WIDE>(c, P, blocks, out); break;
    }
}
template <int DT> static void lin_chunk_type(Ctx* c, const LinArgs& P, int kc, bool wide, int64_t blocks, bool out) {
    if (wide) lin_chunk_width<DT, true>(c, P, kc, blocks, out);
    else lin_chunk_width<DT, false>(c, P, kc, blocks, out);
}

}  // namespace h3
