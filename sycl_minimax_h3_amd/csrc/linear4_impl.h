// linear4_impl.h - linear layers with 4-bit weights and group scales (h3lm.h, linear4).
//
// Mathematics: with w = s c - z in each group of inputs (z the group's minimum, or 8 s),
//     y = sum over groups of  s (sum x c) - z (sum x)  =  s (sum x (16 + c)) - (16 s + z) (sum x).
// A code put into the top four bits of the mantissa of a bfloat16 or half with the exponent of 16 is the number 16 + c, exactly:
// a shift and one and-or for two codes, with no conversion. The products sum x (16 + c) of a run of 32 inputs are one matrix
// instruction (16 x 16 x 32, float32 sums) with x as it stands (bfloat16, half; float32 as three bfloat16 parts). A run's sum of x is one
// more, with a first operand of ones in one row, shared by all columns of the wavefront; it leaves the sums of four runs as the
// first operand of a float32 instruction (16 x 16 x 4) whose second is the four 16 s + z: their products are one instruction for 128
// inputs. What is left for the vector units is one multiply-add by s a group and output.
//
// What that costs in digits: the two terms are roundings of numbers up to 24 / |c - 8| times their difference, more where x has one
// sign. Against float32 sums of x (c - 8) (5376 inputs, 16 rows, float32 out): uniform codes 1.3 times their error (3e-7 of the result), codes in a bell
// of deviation 2.5 around 8 2.2 times, those with x of mean 3 and deviation 1 20 times (5e-6), codes within one of 8 as well 66 times (1.7e-5).
// A 16-bit x is itself off by 2^-9 or 2^-12 of each value, so it keeps this form. float32 x takes sixteen times c - 8 as operands
// (whole numbers, exact in bfloat16; two instructions a code instead of one, for three products each) with z - 8 s against x's sums,
// and no sums without minima: half the error of float32 sums one by one in all four (before: 1.3 to 66 times). 300 rows 14336 -> 5376 286 to 308 us with minima, 243 to 228
// without; 8 rows 5376 -> 28672 70 to 82 and 56 to 55; one row 5376 -> 131072 101 to 117.
//
// Layout: a lane loads 16 bytes of a weight row, 32 codes; the four lanes of a row (16 apart) hold 128 consecutive inputs. A 4 x 4
// exchange between them (four lane swaps) leaves each with eight codes of each of four runs of 32 inputs, so that an instruction's 32
// inputs lie in one group.
//
// Work. One row (linear4_dot_kernel): the codes as above, multiplied by pairs on the vector units, with x in registers.
// Two to 16 rows (linear4_few_kernel): a wavefront takes 16 NT columns and every KW-th 128 inputs; the KW wavefronts of a block
// are joined through LDS in wavefront order. Bound by the codes' bytes: everything that a step needs is loaded a step ahead
// (16 rows, 28672 columns of 5376: 26.5 us, 3.1 TB/s).
// More rows (linear4_many_kernel): a block takes 16 MT rows x 128 columns (64 or 32 where that leaves CUs idle), in two groups of four
// wavefronts (four of two, eight of one) that take every other (fourth, eighth) 128 inputs; x goes through LDS, in the order of the
// instructions' operands, and each wavefront has 32 columns. Bound by vector instructions beside the products (300 rows 14336 -> 5376,
// groups of 32: 119-130 us, 0.36-0.39 PFLOP/s: a multiply-add for each register of a product, the codes, and 24 more product
// instructions beside each 32, for the sums of x and the minima).
#pragma once

#include "kv.h"

namespace h3 {

typedef __bf16 v8bf_l4 __attribute__((ext_vector_type(8)));
typedef _Float16 v8h_l4 __attribute__((ext_vector_type(8)));
typedef float v4f_l4 __attribute__((ext_vector_type(4)));

struct L4Args {
    const void* x;
    int64_t M, N;
    int K;                            // at most kL4MostK
    const uint8_t* codes;
    const void *scale, *mins;         // without minima: mins is scale (and not used)
    int scale_dt, has_mins;
    int group, groups;                // inputs a group; groups a row
    uint32_t magic;                   // 2^32 / (group / 32), rounded up (0: groups of 32)
    const float* bias;
    void* out;
    int out_dt;
};

constexpr int kL4MostK = 1 << 20;
// the group of the run r of 32 inputs: r / (group / 32) by a multiplication. With g = group / 32 and magic = (2^32 + e) / g, e < g, the
// product is r / g + r e / (2^32 g): the quotient is right where r e < 2^32, and r and g are at most 2^15
__device__ __forceinline__ int l4_group(const L4Args& P, int r) { return P.magic ? (int) __umulhi((uint32_t) r, P.magic) : r; }

template <int OP> __device__ __forceinline__ v4f_l4 l4_mma(const uint4& a, const uint4& b, const v4f_l4& c) {
    if constexpr (OP == H3S_F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h_l4, a), __builtin_bit_cast(v8h_l4, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf_l4, a), __builtin_bit_cast(v8bf_l4, b), c, 0, 0, 0);
}
// eight codes of a word as 16 + code, in the order 0 4 1 5 2 6 3 7. m and e: the codes' bits and the exponent, in registers (as literals
// the and and the or would be two instructions: one takes only one literal)
template <int OP> __device__ __forceinline__ void l4_constants(uint32_t& m, uint32_t& e) {
    m = OP == H3S_F16 ? 0x03C003C0u : 0x00780078u;
    e = OP == H3S_F16 ? 0x4C004C00u : 0x41804180u;
    asm volatile("" : "+s"(m));
    asm volatile("" : "+v"(e));
}
// float32 x (three PARTS): sixteen times code - 8, in the same order, exactly: a code less 8 is its four bits as a signed number once the
// highest is flipped, and those are the high half of a signed byte
template <int OP, int PARTS> __device__ __forceinline__ uint4 l4_codes(uint32_t w, uint32_t m, uint32_t e) {
    if constexpr (PARTS > 1) {
        const uint32_t even = ((w << 4) & 0xf0f0f0f0u) ^ 0x80808080u, odd = (w & 0xf0f0f0f0u) ^ 0x80808080u;
        auto pair = [](uint32_t u, int i) {
            const float a = (float) (int8_t) (u >> (8 * i)), b = (float) (int8_t) (u >> (8 * i + 16));
            return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
        };
        return make_uint4(pair(even, 0), pair(odd, 0), pair(even, 1), pair(odd, 1));
    } else if constexpr (OP == H3S_F16) return make_uint4(((w << 6) & m) | e, ((w << 2) & m) | e, ((w >> 2) & m) | e, ((w >> 6) & m) | e);
    else return make_uint4(((w << 3) & m) | e, ((w >> 1) & m) | e, ((w >> 5) & m) | e, ((w >> 9) & m) | e);
}
// what x's sum is taken off with: the weights' distance from s times the operands (float32 x without minima has none)
template <int PARTS> __device__ __forceinline__ float l4_off(float s, float least, bool mins) {
    if constexpr (PARTS > 1) return __builtin_fmaf(-8.0f, s, least);
    const float x = __builtin_fmaf(16.0f, s, least), y = 24.0f * s;
    return mins ? x : y;
}
// eight 16-bit values in that order
__device__ __forceinline__ uint4 l4_order(const uint4& u) {
    return make_uint4(__builtin_amdgcn_perm(u.z, u.x, 0x05040100u), __builtin_amdgcn_perm(u.z, u.x, 0x07060302u),
                      __builtin_amdgcn_perm(u.w, u.y, 0x05040100u), __builtin_amdgcn_perm(u.w, u.y, 0x07060302u));
}

// eight values of x as loaded, and as the parts of an instruction's operand
template <int DT> struct L4X {
    static constexpr int PARTS = 1;
    uint4 u;
    __device__ __forceinline__ void zero() { u = make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ void load(const void* x, int64_t at) { u = *reinterpret_cast<const uint4*>((const uint16_t*) x + at); }
    __device__ __forceinline__ void parts(uint4 (&f)[1]) const { f[0] = l4_order(u); }
};
template <> struct L4X<H3S_F32> {
    static constexpr int PARTS = 3;
    float4 a, b;
    __device__ __forceinline__ void zero() { a = b = make_float4(0.0f, 0.0f, 0.0f, 0.0f); }
    __device__ __forceinline__ void load(const void* x, int64_t at) {
        a = *reinterpret_cast<const float4*>((const float*) x + at);
        b = *reinterpret_cast<const float4*>((const float*) x + at + 4);
    }
    __device__ __forceinline__ void parts(uint4 (&f)[3]) const {
        float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int p = 0; p < 3; ++p) {
            const uint4 u = Vec<H3S_BF16>::pack(v);
            float r[8];
            Vec<H3S_BF16>::unpack(u, r);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = v[i] - r[i];
            f[p] = l4_order(u);
        }
    }
};

// How a 128-input step's scales of one column are loaded: 16-bit or float32 types with the step's scales in one load (they start
// on a boundary of their size), or any type one by one
enum { L4_S16 = 0, L4_S32 = 1, L4_SANY = 2 };

// a step's codes of one column, the run of 32 inputs j in word j
__device__ __forceinline__ void l4_exchange(const uint4& w, uint32_t (&c)[4]) {
    const auto p = __builtin_amdgcn_permlane32_swap(w.x, w.z, false, false);
    const auto q = __builtin_amdgcn_permlane32_swap(w.y, w.w, false, false);
    const auto r = __builtin_amdgcn_permlane16_swap(p[0], q[0], false, false);
    const auto s = __builtin_amdgcn_permlane16_swap(p[1], q[1], false, false);
    c[0] = r[0]; c[1] = r[1]; c[2] = s[0]; c[3] = s[1];
}

// The products of one step of 128 inputs: NT columns' codes and scales against MT x 16 rows. frag(a, j, f): the operand of the rows
// 16 a .. and the run j (zeros past the row's end); AHEAD: a run's operands are asked for before the products of the one
// before (from LDS: 300 rows 5376 -> 28672 247 to 211 us, 14336 -> 5376 127 to 120). Rows: place l of an operand is row 4 (l % 4) + l / 4,
// so that register i of lane group g sums row 4 i + g.
template <bool AHEAD, bool SUMS, int OP, int PARTS, int MT, int NT, int J, typename F>
__device__ __forceinline__ void l4_products(const uint4 (&sel)[4], uint32_t m, uint32_t e, const uint32_t (&c)[NT][4], const float (&sc)[NT][4 / J], const float (&off)[NT],
                                            F frag, v4f_l4 (&acc)[MT][NT]) {
    v4f_l4 sx[MT];
    uint4 x[2][MT][PARTS];
#pragma unroll
    for (int a = 0; a < MT; ++a) {
        sx[a] = v4f_l4{0.0f, 0.0f, 0.0f, 0.0f};
        if (AHEAD) frag(a, 0, x[0][a]);
    }
#pragma unroll
    for (int q = 0; q < 4 / J; ++q) {
        v4f_l4 y[MT][NT];
#pragma unroll
        for (int a = 0; a < MT; ++a)
#pragma unroll
            for (int b = 0; b < NT; ++b) y[a][b] = v4f_l4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = q * J; j < (q + 1) * J; ++j) {
            uint4 f[NT];
#pragma unroll
            for (int b = 0; b < NT; ++b) f[b] = l4_codes<OP, PARTS>(c[b][j], m, e);
            if (AHEAD && j < 3) {
#pragma unroll
                for (int a = 0; a < MT; ++a) frag(a, j + 1, x[(j & 1) ^ 1][a]);
            }
#pragma unroll
            for (int a = 0; a < MT; ++a) {
                uint4 (&xf)[PARTS] = x[AHEAD ? j & 1 : 0][a];
                if (!AHEAD) frag(a, j, xf);
#pragma unroll
                for (int p = 0; p < PARTS; ++p) {
                    if constexpr (SUMS) sx[a] = l4_mma<OP>(sel[j], xf[p], sx[a]);
#pragma unroll
                    for (int b = 0; b < NT; ++b) y[a][b] = l4_mma<OP>(xf[p], f[b], y[a][b]);
                }
            }
            if (AHEAD) __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int a = 0; a < MT; ++a)
#pragma unroll
            for (int b = 0; b < NT; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[a][b][i] = __builtin_fmaf(sc[b][q], y[a][b][i], acc[a][b][i]);
    }
    if constexpr (!SUMS) return;
#pragma unroll
    for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int b = 0; b < NT; ++b) acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x4f32(-sx[a][0], off[b], acc[a][b], 0, 0, 0);
}

// the first operands whose row 4 j is ones: the sums of x of run j then end in lane group j
template <int OP> __device__ __forceinline__ void l4_select(int l15, uint4 (&sel)[4]) {
    const uint32_t one = OP == H3S_F16 ? 0x3C003C00u : 0x3F803F80u;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t u = l15 == 4 * j ? one : 0;
        sel[j] = make_uint4(u, u, u, u);
    }
}

// (loaded whether there is one or not: a load in a branch would have every wavefront wait for all its loads where the branch ends)
__device__ __forceinline__ float l4_bias(const L4Args& P, int64_t n) {
    const float* p = P.bias ? P.bias + min(n, P.N - 1) : (const float*) P.codes;
    return *p;
}
__device__ __forceinline__ void l4_store(const L4Args& P, int64_t m0, int64_t n, int g, const v4f_l4& y, float read) {
    const float bias = P.bias ? read : 0.0f;
    if (n >= P.N) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t m = m0 + 4 * i + g;
        if (m < P.M) store_any(P.out, P.out_dt, m * P.N + n, y[i] + bias);
    }
}

// ---- one row of x: multiply-adds of pairs of codes -----------------------------------------------------------------------------

// c + a.lo b.lo + a.hi b.hi
template <int OP> __device__ __forceinline__ float l4_dot(uint32_t a, uint32_t b, float c) {
    typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    if constexpr (OP == H3S_F16) return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, a), __builtin_bit_cast(h2, b), c, false);
    else return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf2, a), __builtin_bit_cast(bf2, b), c, false);
}

// Wavefronts of a block, at most: three on a SIMD, as many as there are with 168 registers each. (Eleven: 6144 inputs in two chunks a wavefront
// instead of one, 28672 columns 27 to 31 us where twelve take 21 to 25; 24576 inputs past the kernel, 8192 columns 34 to 67 instead of 29 to
// 41; 5376 inputs the same. Against: float32, 12288 inputs -> 8192 columns 38 to 51 us here, 29 to 44 in linear4_few_kernel; with 28672 columns
// 74 to 102 and 99 to 151.)
constexpr int kL4DotWaves = 12;

// A row of weights is cut into chunks of 512 inputs; a wavefront has U of them (every KW-th), with x's values for them in registers, and
// walks down the rows: 16 lanes take a row's chunk, 32 codes each, four rows at a time. So its loads are runs of 256 bytes, the scale of a
// lane's codes is one 2-byte load beside its neighbours', and no operand goes through LDS. (As matrix instructions' operands - 16
// rows a load, 64 bytes of each, a scale gathered from 16 rows - the same loads alone took 94 us where the codes come in 62.) Per tile of
// 16 rows the wavefronts' sums are joined through LDS, in wavefront order; the loads go on across tiles, DP row steps ahead. Bound by the
// codes' bytes: 131072 columns of 5376 67-72 us by the card, 5.0-5.4 TB/s. (One row of x only: with two 28672 columns took 32 us, with
// four 43, where linear4_few_kernel takes 24.)
template <int DT, int U, bool MINS>
__global__ __launch_bounds__(64 * kL4DotWaves) void linear4_dot_kernel(L4Args P) {
    constexpr int OP = DT == H3S_F16 ? H3S_F16 : H3S_BF16, PARTS = L4X<DT>::PARTS, DP = U == 1 ? 4 : U == 2 ? 3 : 2;
    const int lane = threadIdx.x & 63, l = lane & 15, q = lane >> 4, KW = (int) (blockDim.x >> 6);
    const int wave = __builtin_amdgcn_readfirstlane((int) (threadIdx.x >> 6));
    const int tiles = (int) ((P.N + 15) / 16), grid = (int) gridDim.x;
    const int ses = P.scale_dt == H3S_F32 ? 4 : 2;
    // the lane's inputs k .. k + 31 of each chunk (past the row's end: its last ones, against zeros)
    uint32_t kofs[U], gofs[U];
    bool in[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int k = (wave + u * KW) * 512 + l * 32;
        in[u] = k < P.K;
        kofs[u] = (uint32_t) (min(k, P.K - 32) / 2);
        gofs[u] = (uint32_t) (l4_group(P, min(k, P.K - 32) / 32) * ses);
    }
    uint4 w[DP][U];
    uint32_t sr[DP][U], zr[DP][U];
    int ltile = blockIdx.x, lrs = 0;
    // (never skipped, so that the loads in flight are counted; past the last tile: the last rows again)
    auto load = [&](int d) {
        const int64_t rb = min((int64_t) ltile * 16 + lrs * 4, P.N - 1);
        const int qe = (int) min<int64_t>(q, P.N - 1 - rb);
        const uint8_t* cp = P.codes + rb * (P.K / 2);
        const char *sp = (const char*) P.scale + rb * P.groups * ses, *zp = (const char*) P.mins + rb * P.groups * ses;
        const uint32_t co = (uint32_t) (qe * (P.K / 2)), so = (uint32_t) (qe * P.groups * ses);
#pragma unroll
        for (int u = 0; u < U; ++u) w[d][u] = *reinterpret_cast<const uint4*>(cp + (co + kofs[u]));
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (ses == 4) {
                sr[d][u] = *reinterpret_cast<const uint32_t*>(sp + (so + gofs[u]));
                if constexpr (MINS) zr[d][u] = *reinterpret_cast<const uint32_t*>(zp + (so + gofs[u]));
            } else {
                sr[d][u] = *reinterpret_cast<const uint16_t*>(sp + (so + gofs[u]));
                if constexpr (MINS) zr[d][u] = *reinterpret_cast<const uint16_t*>(zp + (so + gofs[u]));
            }
        }
        if (++lrs == 4) {
            lrs = 0;
            ltile = min(ltile + grid, tiles - 1);
        }
    };
#pragma unroll
    for (int d = 0; d < DP; ++d) load(d);
    // x as operands: the pairs in the order of l4_codes, and the sum of each lane's 32 values
    uint32_t x[U][PARTS][16];
    float sx[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const char* xp = (const char*) P.x + 2 * kofs[u] * (DT == H3S_F32 ? 4 : 2);
        sx[u] = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            L4X<DT> v;
            v.load(xp, 8 * e);
            if (!in[u]) v.zero();
            uint4 f[PARTS];
            v.parts(f);
#pragma unroll
            for (int p = 0; p < PARTS; ++p) {
                x[u][p][4 * e] = f[p].x; x[u][p][4 * e + 1] = f[p].y; x[u][p][4 * e + 2] = f[p].z; x[u][p][4 * e + 3] = f[p].w;
                float y[8];
                Vec<OP>::unpack(f[p], y);
#pragma unroll
                for (int i = 0; i < 8; ++i) sx[u] += y[i];
            }
        }
    }
    uint32_t cm, ce;
    l4_constants<OP>(cm, ce);
    const bool bf = P.scale_dt == H3S_BF16, wide = ses == 4;
    auto number = [&](uint32_t r) {
        const float a = bf16_lo(r), b = f16_lo(r), c = __uint_as_float(r);
        return wide ? c : bf ? a : b;
    };
    __shared__ float part[2][16][kL4DotWaves + 1];
    int turn = 0, rs = 0, tile = blockIdx.x;
    while (tile < tiles) {
#pragma unroll
        for (int d = 0; d < DP; ++d) {
            float acc = 0.0f;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint32_t c[4] = {w[d][u].x, w[d][u].y, w[d][u].z, w[d][u].w};
                float y = 0.0f;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint4 f = l4_codes<OP, PARTS>(c[e], cm, ce);
#pragma unroll
                    for (int p = 0; p < PARTS; ++p) {
                        y = l4_dot<OP>(x[u][p][4 * e], f.x, y);
                        y = l4_dot<OP>(x[u][p][4 * e + 1], f.y, y);
                        y = l4_dot<OP>(x[u][p][4 * e + 2], f.z, y);
                        y = l4_dot<OP>(x[u][p][4 * e + 3], f.w, y);
                    }
                }
                const float s = number(sr[d][u]);
                acc = __builtin_fmaf(PARTS > 1 ? 0.0625f * s : s, y, acc);
                if constexpr (MINS || PARTS == 1) acc = __builtin_fmaf(-l4_off<PARTS>(s, MINS ? number(zr[d][u]) : 0.0f, MINS), sx[u], acc);
            }
            load(d);
            acc = wave_sum<16>(acc);
            if (l == 0) part[turn & 1][rs * 4 + q][wave] = acc;
            if (++rs == 4) {
                // (the area is written again two tiles later, behind the next tile's barrier)
                lds_barrier();
                const int64_t col = (int64_t) tile * 16 + threadIdx.x;
                if (threadIdx.x < 16 && tile < tiles && col < P.N) {
                    float y = part[turn & 1][threadIdx.x][0];
                    for (int v = 1; v < KW; ++v) y += part[turn & 1][threadIdx.x][v];
                    store_any(P.out, P.out_dt, col, y + (P.bias ? P.bias[col] : 0.0f));
                }
                ++turn;
                rs = 0;
                tile += grid;
            }
        }
    }
}

// ---- up to 16 rows ------------------------------------------------------------------------------------------------------------

// The scales and minima of four steps of one column: lane group g loads those of step first + g (one gather for four steps: a gather
// from 16 rows of weights costs about as much as 16 x 64 bytes of codes), and a step's are passed on from its group.
template <int J, int SM, int PARTS> struct L4Q {
    static constexpr int CNT = 4 / J, RAW = SM == L4_S16 ? (CNT + 1) / 2 : CNT;
    uint32_t s[RAW], z[RAW];
    // scale, mins: the tile's first column's; off: the bytes from there to the lane's column; r: the first run of the lane's step
    __device__ __forceinline__ void load(const L4Args& P, const char* scale, const char* mins, uint32_t off, int r) {
        if constexpr (SM == L4_SANY) {
            const int most = P.K / 32 - 1, es = P.scale_dt == H3S_F32 ? 4 : 2;
#pragma unroll
            for (int c = 0; c < CNT; ++c) {
                const uint32_t at = off + (uint32_t) (l4_group(P, min(r + J * c, most)) * es);
                s[c] = es == 4 ? *reinterpret_cast<const uint32_t*>(scale + at) : *reinterpret_cast<const uint16_t*>(scale + at);
                z[c] = es == 4 ? *reinterpret_cast<const uint32_t*>(mins + at) : *reinterpret_cast<const uint16_t*>(mins + at);
            }
        } else {
            const uint32_t at = off + (uint32_t) (J == 1 ? r : J == 2 ? r / 2 : l4_group(P, r)) * (SM == L4_S32 ? 4 : 2);
            take(scale + at, s);
            take(mins + at, z);
        }
    }
    __device__ __forceinline__ void take(const char* p, uint32_t (&u)[RAW]) const {
        if constexpr (RAW == 4) { const uint4 v = *reinterpret_cast<const uint4*>(p); u[0] = v.x; u[1] = v.y; u[2] = v.z; u[3] = v.w; }
        else if constexpr (RAW == 2) { const uint2 v = *reinterpret_cast<const uint2*>(p); u[0] = v.x; u[1] = v.y; }
        else if constexpr (SM == L4_S16 && CNT == 1) u[0] = *reinterpret_cast<const uint16_t*>(p);
        else u[0] = *reinterpret_cast<const uint32_t*>(p);
    }
    // those of the step of lane group `from` (lane: 4 (16 from + lane % 16)), for every lane
    __device__ __forceinline__ void pass(const L4Args& P, int lane, int g, float (&sc)[CNT], float& off) const {
        uint32_t a[RAW], b[RAW];
#pragma unroll
        for (int i = 0; i < RAW; ++i) {
            a[i] = (uint32_t) __builtin_amdgcn_ds_bpermute(lane, (int) s[i]);
            b[i] = (uint32_t) __builtin_amdgcn_ds_bpermute(lane, (int) z[i]);
        }
        float zc[CNT];
#pragma unroll
        for (int c = 0; c < CNT; ++c) {
            sc[c] = number(P, a, c);
            zc[c] = number(P, b, c);
        }
        float own = sc[0], least = zc[0];
        if constexpr (CNT == 2) { own = g < 2 ? sc[0] : sc[1]; least = g < 2 ? zc[0] : zc[1]; }
        else if constexpr (CNT == 4) { own = g < 2 ? (g ? sc[1] : sc[0]) : (g == 2 ? sc[2] : sc[3]); least = g < 2 ? (g ? zc[1] : zc[0]) : (g == 2 ? zc[2] : zc[3]); }
        off = l4_off<PARTS>(own, least, P.has_mins != 0);
        if constexpr (PARTS > 1) {
#pragma unroll
            for (int c = 0; c < CNT; ++c) sc[c] *= 0.0625f;
        }
    }
    __device__ __forceinline__ float number(const L4Args& P, const uint32_t* u, int c) const {
        const uint32_t v = SM == L4_S16 && CNT > 1 ? (c & 1 ? u[c >> 1] >> 16 : u[c >> 1] & 0xffffu) : u[c];
        const float x = __uint_as_float(v), a = bf16_lo(v), b = f16_lo(v);
        if (SM == L4_S32) return x;
        const float h = P.scale_dt == H3S_BF16 ? a : b;
        return SM == L4_SANY && P.scale_dt == H3S_F32 ? x : h;
    }
};

constexpr int kL4FewWaves = 12;       // wavefronts of a block, at most

// J: runs of 32 inputs to one scale (4: groups are multiples of 128 inputs, 2: of 64, 1: of 32).
// A block walks the tiles of 16 NT columns that are its own. Its KW wavefronts have 4 quads x 4 steps of 128 inputs each, one run of
// memory in a weight row, and are joined through LDS at the end of a tile; the loads go on across tiles.
// XR (16-bit x, one quad: up to 12 x 512 inputs): a wavefront's operands of x stay in registers. Otherwise they are loaded in the step that uses
// them (from the L2).
template <int DT, int NT, int J, int SM, bool SUMS, bool XR>
__global__ __launch_bounds__(64 * kL4FewWaves) void linear4_few_kernel(L4Args P, int quads) {
    constexpr int OP = DT == H3S_F16 ? H3S_F16 : H3S_BF16, PARTS = L4X<DT>::PARTS, XES = DT == H3S_F32 ? 4 : 2, DP = XR ? 4 : 2;
    const int lane = threadIdx.x & 63, l15 = lane & 15, g = lane >> 4, KW = (int) (blockDim.x >> 6);
    const int wave = __builtin_amdgcn_readfirstlane((int) (threadIdx.x >> 6));
    const int steps = (P.K + 127) / 128, first = wave * quads * 4, grid = (int) gridDim.x;
    const int tiles = (int) ((P.N + 16 * NT - 1) / (16 * NT));
    const int row = min((l15 & 3) * 4 + (l15 >> 2), (int) P.M - 1);              // (places without a row: the last again, not stored)
    const int ses = SM == L4_S32 || (SM == L4_SANY && P.scale_dt == H3S_F32) ? 4 : 2;
    // the operand of run j of a step (zeros past the row's end)
    auto load_x = [&](int step, int j, L4X<DT>& x) {
        const int k = step * 128 + 32 * j + 8 * g;
        x.load((const char*) P.x + (uint32_t) (row * P.K + min(k, P.K - 8)) * XES, 0);
        if (SM == L4_SANY && k >= P.K) x.zero();
    };
    uint4 w[DP][NT];                                                              // DP steps in flight
    L4Q<J, SM, PARTS> now[NT], next[NT];
    // where the loads of the codes are (the scales': one quad ahead of the step in hand): a tile's first column, the lane's bytes from there
    struct At {
        const uint8_t* codes;
        const char *scale, *mins;
        uint32_t coff[NT], soff[NT];
    };
    auto enter = [&](int tile, At& a) {
        const int64_t n0 = (int64_t) tile * (16 * NT);
        a.codes = P.codes + n0 * (P.K / 2);
        a.scale = (const char*) P.scale + n0 * P.groups * ses;
        a.mins = (const char*) P.mins + n0 * P.groups * ses;
        const int left = (int) min<int64_t>(P.N - 1 - n0, 16 * NT);               // (columns past the last: the last again, not stored)
#pragma unroll
        for (int b = 0; b < NT; ++b) {
            const int n = min(16 * b + l15, left);
            a.coff[b] = (uint32_t) (n * (P.K / 2) + 16 * g);
            a.soff[b] = (uint32_t) (n * P.groups * ses);
        }
    };
    // (Loads are never skipped: with the same ones in every round the compiler counts those in flight; where there is nothing to load it is
    // the last step or the last tile again.)
    auto load_w = [&](const At& a, int step, uint4 (&wd)[NT]) {
        const int st = min(step, steps - 1);
#pragma unroll
        for (int b = 0; b < NT; ++b) {
            uint32_t at = a.coff[b];
            if (SM == L4_SANY) at = min(at, a.coff[b] - 16 * g + (uint32_t) (P.K / 2 - 16 - st * 64));    // (within the row)
            wd[b] = *reinterpret_cast<const uint4*>(a.codes + st * 64 + at);
        }
    };
    auto load_s = [&](const At& a, int step) {
#pragma unroll
        for (int b = 0; b < NT; ++b) next[b].load(P, a.scale, a.mins, a.soff[b], min(step + g, steps - 1) * 4);
    };
    int tile = blockIdx.x, quad = 0, turn = 0;
    At here, then;                                                                // this quad's tile and the next quad's
    enter(tile, here);
    load_s(here, first);
#pragma unroll
    for (int r = 0; r < DP; ++r) load_w(here, first + r, w[r]);
    L4X<DT> xr[XR ? 4 : 1][4];
    if constexpr (XR) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                load_x(min(first + r, steps - 1), j, xr[r][j]);
                xr[r][j].u = l4_order(xr[r][j].u);
            }
    }
    uint4 sel[4];
    l4_select<OP>(l15, sel);
    uint32_t cm, ce;
    l4_constants<OP>(cm, ce);
    __shared__ v4f_l4 part[2][NT][kL4FewWaves][64];
    v4f_l4 acc[1][NT];
#pragma unroll
    for (int b = 0; b < NT; ++b) acc[0][b] = v4f_l4{0.0f, 0.0f, 0.0f, 0.0f};
    while (tile < tiles) {
        const bool end = quad + 1 == quads;
        const int ntile = end ? min(tile + grid, tiles - 1) : tile, nfirst = end ? first : first + 4 * (quad + 1);
        enter(ntile, then);
#pragma unroll
        for (int b = 0; b < NT; ++b) now[b] = next[b];
        load_s(then, nfirst);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int step = first + 4 * quad + r;
            if constexpr (!XR) {
#pragma unroll
                for (int j = 0; j < 4; ++j) load_x(min(step, steps - 1), j, xr[0][j]);
            }
            uint32_t c[NT][4];
            float sc[NT][4 / J], off[NT];
#pragma unroll
            for (int b = 0; b < NT; ++b) {
                l4_exchange(w[r % DP][b], c[b]);
                now[b].pass(P, 4 * (16 * r + l15), g, sc[b], off[b]);
                if (SM == L4_SANY && step * 128 + 128 > P.K) {
#pragma unroll
                    for (int q = 0; q < 4 / J; ++q) sc[b][q] = step * 128 + 32 * J * q < P.K ? sc[b][q] : 0.0f;
                    off[b] = step * 128 + 32 * g < P.K ? off[b] : 0.0f;
                }
            }
            if (r + DP < 4) load_w(here, step + DP, w[r % DP]);
            else load_w(then, nfirst + r + DP - 4, w[r % DP]);
            if (step < steps) {
                l4_products<false, SUMS, OP, PARTS, 1, NT, J>(sel, cm, ce, c, sc, off, [&](int, int j, uint4(&f)[PARTS]) {
                    if constexpr (XR) f[0] = xr[r][j].u;
                    else xr[0][j].parts(f);
                }, acc);
            }
        }
        here = then;
        ++quad;
        if (end) {
            // the wavefronts' sums, in wavefront order, by one of them in turn; the others go on (the area is used again two tiles later,
            // behind the next tile's barrier)
#pragma unroll
            for (int b = 0; b < NT; ++b) {
                part[turn & 1][b][wave][lane] = acc[0][b];
                acc[0][b] = v4f_l4{0.0f, 0.0f, 0.0f, 0.0f};
            }
            lds_barrier();
            if (wave == turn % KW) {
#pragma unroll
                for (int b = 0; b < NT; ++b) {
                    const int64_t n = (int64_t) tile * (16 * NT) + 16 * b + l15;
                    v4f_l4 y = part[turn & 1][b][0][lane];
                    for (int v = 1; v < KW; ++v) y += part[turn & 1][b][v][lane];
                    l4_store(P, 0, n, g, y, l4_bias(P, n));
                }
            }
            ++turn;
            quad = 0;
            tile += grid;
        }
    }
}

// CG: wavefronts side by side, of 32 columns each; the block's 8 / CG groups of them take every (8 / CG)th step of 128 inputs
template <int DT, int MT, int CG, int J, int SM, bool SUMS>
__global__ __launch_bounds__(512, 2) void linear4_many_kernel(L4Args P) {
    constexpr int NT = 2, OP = DT == H3S_F16 ? H3S_F16 : H3S_BF16, PARTS = L4X<DT>::PARTS;
    constexpr int KG = 8 / CG, COLS = 16 * NT * CG;
    constexpr int PIECES = 16 * MT * 16 / (64 * CG);                              // 8-input pieces of x a thread stages
    __shared__ uint4 xs[KG][2][MT][4][PARTS][64];                                 // [K group][stage][rows][run][part][lane]
    const int lane = threadIdx.x & 63, l15 = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int) (threadIdx.x >> 6)), kg = wave / CG;
    // blocks eight apart run on one XCD: the row tiles of a column block lie there one after another and share its codes
    const int64_t mt = (P.M + 16 * MT - 1) / (16 * MT), id = blockIdx.x;
    const int64_t nb = id / (8 * mt) * 8 + id % 8, n0 = nb * COLS + wave % CG * (16 * NT), m0 = id / 8 % mt * (16 * MT);
    if (nb * COLS >= P.N) return;
    const int steps = (P.K + 127) / 128;
    const int ses = SM == L4_S32 || (SM == L4_SANY && P.scale_dt == H3S_F32) ? 4 : 2;
    const int64_t from = min(n0, P.N - 1);                                        // (a wavefront past the columns: the last one, not stored)
    const uint8_t* cbase = P.codes + from * (P.K / 2);
    const char *sbase = (const char*) P.scale + from * P.groups * ses, *zbase = (const char*) P.mins + from * P.groups * ses;
    uint32_t coff[NT], soff[NT];
    v4f_l4 acc[MT][NT];
#pragma unroll
    for (int b = 0; b < NT; ++b) {
        const int n = (int) min<int64_t>(16 * b + l15, P.N - 1 - from);
        coff[b] = (uint32_t) (n * (P.K / 2) + 16 * g);
        soff[b] = (uint32_t) (n * P.groups * ses);
#pragma unroll
        for (int a = 0; a < MT; ++a) acc[a][b] = v4f_l4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    uint4 sel[4];
    l4_select<OP>(l15, sel);
    uint32_t cm, ce;
    l4_constants<OP>(cm, ce);
    // x: piece t + 64 CG p of the K group's step is 8 inputs (16 pieces a row)
    constexpr int XES = DT == H3S_F32 ? 4 : 2;
    const int t = threadIdx.x % (64 * CG);
    L4X<DT> xr[PIECES];
    const char* xbase = (const char*) P.x + m0 * P.K * XES;
    uint32_t xoff[PIECES];
#pragma unroll
    for (int p = 0; p < PIECES; ++p) xoff[p] = (uint32_t) ((int) min<int64_t>((t + 64 * CG * p) / 16, P.M - 1 - m0) * P.K + t % 16 * 8) * XES;
    uint4 w[NT];
    L4Q<J, SM, PARTS> now[NT], next[NT];                                          // the scales of four of the K group's steps
    auto load_x = [&](int step) {
        const char* xp = xbase + (int64_t) step * 128 * XES;
        const bool out = SM == L4_SANY && step * 128 + t % 16 * 8 >= P.K;
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            xr[p].load(xp + (out ? xoff[p] - t % 16 * 8 * XES : xoff[p]), 0);
            if (out) xr[p].zero();
        }
    };
    auto store_x = [&](int stage) {
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int at = t + 64 * CG * p, r = at / 16, k8 = at % 16;                // place: row 4 (l % 4) + l / 4 at l,
                                                                                  // its low bits by the lane group (banks)
            uint4 f[PARTS];
            xr[p].parts(f);
#pragma unroll
            for (int q = 0; q < PARTS; ++q) xs[kg][stage][r / 16][k8 / 4][q][k8 % 4 * 16 + (r % 4) * 4 + (r % 16 / 4 ^ k8 % 4)] = f[q];
        }
    };
    auto load_w = [&](int step) {
        const uint8_t* cp = cbase + step * 64;
#pragma unroll
        for (int b = 0; b < NT; ++b) {
            uint32_t at = coff[b];
            if (SM == L4_SANY) at = min(at, coff[b] - 16 * g + (uint32_t) (P.K / 2 - 16 - step * 64));   // (within the row)
            w[b] = *reinterpret_cast<const uint4*>(cp + at);
        }
    };
    auto load_s = [&](int step) {
#pragma unroll
        for (int b = 0; b < NT; ++b) next[b].load(P, sbase, zbase, soff[b], min(step + KG * g, steps - 1) * 4);
    };
    // all K groups make the same number of rounds (their last may have no step)
    // (Loads are never skipped, see linear4_few_kernel: past the end it is the last step again.)
    load_s(kg);
    load_x(min(kg, steps - 1));
    load_w(min(kg, steps - 1));
    store_x(0);
    load_x(min(kg + KG, steps - 1));
    lds_barrier();
    for (int first = 0; first < steps; first += 4 * KG) {
#pragma unroll
        for (int b = 0; b < NT; ++b) now[b] = next[b];
        load_s(first + 4 * KG + kg);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int step = first + KG * r + kg;
            if (step < steps) {
                uint32_t c[NT][4];
                float sc[NT][4 / J], off[NT];
#pragma unroll
                for (int b = 0; b < NT; ++b) {
                    l4_exchange(w[b], c[b]);
                    now[b].pass(P, 4 * (16 * r + l15), g, sc[b], off[b]);
                    if (SM == L4_SANY && step * 128 + 128 > P.K) {
#pragma unroll
                        for (int q = 0; q < 4 / J; ++q) sc[b][q] = step * 128 + 32 * J * q < P.K ? sc[b][q] : 0.0f;
                        off[b] = step * 128 + 32 * g < P.K ? off[b] : 0.0f;
                    }
                }
                load_w(min(step + KG, steps - 1));
                l4_products<PARTS == 1, SUMS, OP, PARTS, MT, NT, J>(sel, cm, ce, c, sc, off, [&](int a, int j, uint4(&f)[PARTS]) {
#pragma unroll
                    for (int q = 0; q < PARTS; ++q) f[q] = xs[kg][r & 1][a][j][q][lane ^ g];
                }, acc);
                store_x((r & 1) ^ 1);
                load_x(min(step + 2 * KG, steps - 1));
            }
            lds_barrier();
        }
    }
    // the groups' sums to the first's, in their order
    v4f_l4* part = reinterpret_cast<v4f_l4*>(&xs[0][0][0][0][0][0]);
    static_assert(sizeof(xs) >= (size_t) (KG - 1) * CG * MT * NT * 64 * 16, "the sums fit x's stages");
    if (kg) {
#pragma unroll
        for (int a = 0; a < MT; ++a)
#pragma unroll
            for (int b = 0; b < NT; ++b) part[(((wave - CG) * MT + a) * NT + b) * 64 + lane] = acc[a][b];
    }
    __syncthreads();
    if (kg == 0) {
        float bias[NT];
#pragma unroll
        for (int b = 0; b < NT; ++b) bias[b] = l4_bias(P, n0 + 16 * b + l15);
#pragma unroll
        for (int a = 0; a < MT; ++a)
#pragma unroll
            for (int b = 0; b < NT; ++b) {
                v4f_l4 y = acc[a][b];
#pragma unroll
                for (int k = 0; k + 1 < KG; ++k) y += part[(((k * CG + wave) * MT + a) * NT + b) * 64 + lane];
                l4_store(P, m0 + 16 * a, n0 + 16 * b + l15, g, y, bias[b]);
            }
    }
}

template <int DT, int NT, int J, int SM, bool SUMS, bool XR>
static void l4_few_run(Ctx* c, const L4Args& P, int quads, int kw) {
    // a block walks as many tiles as any other, or one less
    const int64_t tiles = (P.N + 16 * NT - 1) / (16 * NT), turns = (tiles + c->cus - 1) / c->cus;
    linear4_few_kernel<DT, NT, J, SM, SUMS, XR><<<(unsigned) ((tiles + turns - 1) / turns), 64 * kw, 0, c->stream>>>(P, quads);
}
template <int DT, int J, int SM, bool SUMS>
static void l4_few(Ctx* c, const L4Args& P) {
    // the fewest quads of steps a wavefront that 12 wavefronts can share the inputs in
    const int steps = (P.K + 127) / 128, quads = (steps + 4 * kL4FewWaves - 1) / (4 * kL4FewWaves), kw = (steps + 4 * quads - 1) / (4 * quads);
    if constexpr (DT != H3S_F32) {
        if (quads == 1) return l4_few_run<DT, 1, J, SM, SUMS, true>(c, P, quads, kw);
    }
    l4_few_run<DT, 2, J, SM, SUMS, false>(c, P, quads, kw);
}
// the blocks of tiles of `rows` rows and 32 cg columns; those of a column tile go to one XCD of eight, so an eighth of them is a whole number
static int64_t l4_blocks(const L4Args& P, int rows, int cg) {
    return (P.M + rows - 1) / rows * (((P.N + 32 * cg - 1) / (32 * cg) + 7) / 8 * 8);
}
template <int DT, int MT, int CG, int J, int SM, bool SUMS>
static void l4_many_run(Ctx* c, const L4Args& P) {
    linear4_many_kernel<DT, MT, CG, J, SM, SUMS><<<(unsigned) l4_blocks(P, 16 * MT, CG), 512, 0, c->stream>>>(P);
}
// Half as many columns a block, and twice the groups along the inputs, while the blocks still run at once (as far as x's stages fit LDS):
// 5376 -> 5376, 32 rows 38 to 18 us, 128 rows 52 to 34; 14336 -> 5376, 32 rows 92 to 33 us, 128 rows 126 to 72.
template <int DT, int MT, int J, int SM, bool SUMS>
static void l4_many(Ctx* c, const L4Args& P) {
    if constexpr (MT == 2) {
        if (l4_blocks(P, 32, 1) <= c->cus) return l4_many_run<DT, MT, 1, J, SM, SUMS>(c, P);
    }
    if (l4_blocks(P, 16 * MT, 2) <= c->cus) l4_many_run<DT, MT, 2, J, SM, SUMS>(c, P);
    else l4_many_run<DT, MT, 4, J, SM, SUMS>(c, P);
}
template <int DT, int J, int SM, bool SUMS>
static void l4_run(Ctx* c, const L4Args& P) {
    if constexpr (DT == H3S_F32) {
        // (three parts: x's stages of 32 rows and more than two groups do not fit LDS, those of 16 rows do: 32 rows 5376 -> 5376 56 to
        // 26 us, 14336 -> 5376 140 to 58)
        if (P.M <= 16) l4_few<DT, J, SM, SUMS>(c, P);
        else if (l4_blocks(P, 16, 2) <= c->cus) l4_many_run<DT, 1, 2, J, SM, SUMS>(c, P);
        else l4_many_run<DT, 2, 4, J, SM, SUMS>(c, P);
    } else {
        // Up to 16 rows as one operand, unless x's operands do not fit the wavefronts' registers there and few columns leave the inputs to
        // split (14336 -> 5376: 16 rows 41 us, in tiles of 32 rows 32). Tiles of 32 rows up to 32 rows, and beyond while the device runs
        // all blocks of 64 columns of them at once (64 rows: 5376 -> 5376 34 to 22 us, 14336 -> 5376 75 to 47).
        if (P.M <= 4 || (P.M <= 16 && (P.K <= 512 * kL4FewWaves || l4_blocks(P, 32, 1) > c->cus))) l4_few<DT, J, SM, SUMS>(c, P);
        else if (P.M <= 32 || l4_blocks(P, 32, 2) <= c->cus) l4_many<DT, 2, J, SM, SUMS>(c, P);
        else l4_many<DT, 4, J, SM, SUMS>(c, P);
    }
}
template <int DT, int U>
static void l4_dot_run(Ctx* c, const L4Args& P) {
    const int64_t tiles = (P.N + 15) / 16, turns = (tiles + 2 * c->cus - 1) / (2 * c->cus);
    const unsigned grid = (unsigned) ((tiles + turns - 1) / turns);
    const int chunks = (P.K + 511) / 512, kw = (chunks + U - 1) / U;
    if (P.has_mins) linear4_dot_kernel<DT, U, true><<<grid, 64 * kw, 0, c->stream>>>(P);
    else linear4_dot_kernel<DT, U, false><<<grid, 64 * kw, 0, c->stream>>>(P);
}
// whether the call has one row, whose values for a wavefront's chunks fit its registers (the last run starts it)
template <int DT> static bool l4_dot_takes(Ctx* c, const L4Args& P) {
    const int chunks = (P.K + 511) / 512;
    if (P.M > 1) return false;
    if (chunks <= kL4DotWaves) l4_dot_run<DT, 1>(c, P);
    else if (chunks <= 2 * kL4DotWaves) l4_dot_run<DT, 2>(c, P);
    else if (chunks <= 4 * kL4DotWaves && L4X<DT>::PARTS == 1) l4_dot_run<DT, L4X<DT>::PARTS == 1 ? 4 : 1>(c, P);
    else return false;
    return true;
}
// x's sums are needed but for float32 x without minima, whose operands are the weights less their scale
template <int DT, int J, int SM>
static void l4_sums(Ctx* c, const L4Args& P) {
    if constexpr (DT == H3S_F32) {
        if (!P.has_mins) return l4_run<DT, J, SM, false>(c, P);
    }
    l4_run<DT, J, SM, true>(c, P);
}
template <int DT>
static void l4_type(Ctx* c, const L4Args& P) {
    if (l4_dot_takes<DT>(c, P)) return;
    // a step of 128 inputs has 4, 2 or 1 scales: one load where every column's lie on a boundary of their size
    const int64_t cnt = P.group % 128 == 0 ? 1 : P.group == 64 ? 2 : P.group == 32 ? 4 : 0;
    const bool vec = cnt && P.groups % cnt == 0 && ((uintptr_t) P.scale | (uintptr_t) P.mins) % (uintptr_t) (cnt * elem_size(P.scale_dt)) == 0;
    if (!vec) l4_sums<DT, 1, L4_SANY>(c, P);
    else if (P.scale_dt == H3S_F32) {
        if (cnt == 1) l4_sums<DT, 4, L4_S32>(c, P);
        else if (cnt == 2) l4_sums<DT, 2, L4_S32>(c, P);
        else l4_sums<DT, 1, L4_S32>(c, P);
    } else {
        if (cnt == 1) l4_sums<DT, 4, L4_S16>(c, P);
        else if (cnt == 2) l4_sums<DT, 2, L4_S16>(c, P);
        else l4_sums<DT, 1, L4_S16>(c, P);
    }
}
void l4_bf16(Ctx* c, const L4Args& P);
void l4_f16(Ctx* c, const L4Args& P);
void l4_f32(Ctx* c, const L4Args& P);

}  // namespace h3
