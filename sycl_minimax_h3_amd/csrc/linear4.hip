// linear4.hip - linear layers with 4-bit weights and group scales (h3lm.h, linear4).
//
// Mathematics: with w = s c - z in each group of inputs (z the group's minimum, or 8 s),
//     y = sum over groups of  s (sum x c) - z (sum x)  =  s (sum x (16 + c)) - (16 s + z) (sum x).
// A code put into the top four bits of the mantissa of a bfloat16 or half with the exponent of 16 is the number 16 + c, exactly:
// a shift and one and-or for two codes, with no conversion. The products sum x (16 + c) of 32 inputs are one matrix instruction
// (16 x 16 x 32, float32 sums) with x as it stands (bfloat16, half; float32 as three bfloat16 parts), and sum x is one more with ones,
// shared by all columns of the wavefront. (16 against c of 0 .. 15: the two terms are at most five times the difference of typical
// codes, so float32 sums lose little over two bits.)
//
// Layout: a lane loads 16 bytes of a weight row, 32 codes; the four lanes of a row (16 apart) hold 128 consecutive inputs. A 4 x 4
// exchange between them (four lane swaps) leaves each with eight codes of each of four runs of 32 inputs, so that an instruction's 32
// inputs lie in one group. Rows of x are spread so that up to four rows cost one scale product a group.
//
// Work: a wavefront takes 16 NT columns and every KW-th run of 128 inputs, against 16 MT rows; the KW wavefronts of a block
// share the columns and are joined through LDS in wavefront order. Bound by the codes' bytes for few rows.
#include <algorithm>

#include "kv.h"

namespace h3 {

typedef short v8s_l4 __attribute__((ext_vector_type(8)));
typedef __bf16 v8bf_l4 __attribute__((ext_vector_type(8)));
typedef _Float16 v8h_l4 __attribute__((ext_vector_type(8)));
typedef float v4f_l4 __attribute__((ext_vector_type(4)));

struct L4Args {
    const void* x;
    int64_t M, K, N;
    const uint8_t* codes;
    const void *scale, *mins;
    int scale_dt;
    int64_t group, groups;            // inputs a group; groups a row
    const float* bias;
    void* out;
    int out_dt;
    bool svec;                        // a run's scales in one load
};

template <int DT> __device__ __forceinline__ v4f_l4 l4_mma(const uint4& a, const uint4& b, const v4f_l4& c) {
    if constexpr (DT == H3S_F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h_l4, a), __builtin_bit_cast(v8h_l4, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf_l4, a), __builtin_bit_cast(v8bf_l4, b), c, 0, 0, 0);
}
// eight codes of a word as 16 + code, in the order 0 4 1 5 2 6 3 7
template <int DT> __device__ __forceinline__ uint4 l4_codes(uint32_t w) {
    if constexpr (DT == H3S_F16) {
        constexpr uint32_t m = 0x03C003C0u, e = 0x4C004C00u;
        return make_uint4(((w << 6) & m) | e, ((w << 2) & m) | e, ((w >> 2) & m) | e, ((w >> 6) & m) | e);
    } else {
        constexpr uint32_t m = 0x00780078u, e = 0x41804180u;
        return make_uint4(((w << 3) & m) | e, ((w >> 1) & m) | e, ((w >> 5) & m) | e, ((w >> 9) & m) | e);
    }
}
// eight 16-bit values in that order
__device__ __forceinline__ uint4 l4_order(const uint4& u) {
    return make_uint4(__builtin_amdgcn_perm(u.z, u.x, 0x05040100u), __builtin_amdgcn_perm(u.z, u.x, 0x07060302u),
                      __builtin_amdgcn_perm(u.w, u.y, 0x05040100u), __builtin_amdgcn_perm(u.w, u.y, 0x07060302u));
}
// eight values of x from input k on (the caller: within the row)
template <int DT, int PARTS> __device__ __forceinline__ void l4_x(const void* x, int64_t at, uint4 (&f)[PARTS]) {
    if constexpr (DT != H3S_F32) {
        f[0] = l4_order(*reinterpret_cast<const uint4*>((const uint16_t*) x + at));
    } else {
        float v[8];
        load_f32x((const float*) x + at, v, 8);
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
            const uint4 u = Vec<H3S_BF16>::pack(v);
            float r[8];
            Vec<H3S_BF16>::unpack(u, r);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = v[i] - r[i];
            f[p] = l4_order(u);
        }
    }
}

// the scales (or minima) of a run of 128 inputs from input kk on, one for each 32 J of them, of the row that starts at element
// `row`; vec: they are consecutive and lie on a boundary of their size
template <int J> __device__ __forceinline__ void l4_scales(const L4Args& P, const void* p, int64_t row, int64_t kk, float* f) {
    constexpr int CNT = 4 / J;
    if (P.svec) {
        const int64_t i = row + kk / P.group;
        if (P.scale_dt == H3S_F32) {
#pragma unroll
            for (int c = 0; c < CNT; ++c) f[c] = ((const float*) p)[i + c];
        } else {
            uint32_t u[2] = {0, 0};
            if constexpr (CNT == 4) { const uint2 v = *reinterpret_cast<const uint2*>((const uint16_t*) p + i); u[0] = v.x; u[1] = v.y; }
            else if constexpr (CNT == 2) u[0] = *reinterpret_cast<const uint32_t*>((const uint16_t*) p + i);
            else u[0] = ((const uint16_t*) p)[i];
#pragma unroll
            for (int c = 0; c < CNT; ++c) {
                const uint32_t h = (u[c >> 1] >> (16 * (c & 1))) & 0xffffu;
                f[c] = P.scale_dt == H3S_BF16 ? bf16_lo(h) : f16_lo(h);
            }
        }
    } else {
#pragma unroll
        for (int c = 0; c < CNT; ++c) {
            const int64_t k = kk + 32 * J * c;
            f[c] = k < P.K ? load_any(p, P.scale_dt, row + k / P.group) : 0.0f;
        }
    }
}

// J: runs of 32 inputs to one scale product (4: groups are multiples of 128 inputs, 2: of 64, 1: of 32)
template <int DT, int MT, int NT, int KW, int NI, int J>
__global__ __launch_bounds__(64 * KW) void linear4_kernel(L4Args P) {
    constexpr int PARTS = DT == H3S_F32 ? 3 : 1, OP = DT == H3S_F16 ? H3S_F16 : H3S_BF16, CNT = 4 / J;
    const int lane = threadIdx.x & 63, l15 = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int) (threadIdx.x >> 6));
    const int64_t n0 = (int64_t) blockIdx.x * (16 * NT), m0 = (int64_t) blockIdx.y * (16 * MT);
    // the row of x in place l15 of the first operand: sums of rows 4 i + g end in register i of lane group g
    const int mrow = (l15 & 3) * 4 + (l15 >> 2);
    v4f_l4 acc[MT][NT];
#pragma unroll
    for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int b = 0; b < NT; ++b) acc[a][b] = v4f_l4{0.0f, 0.0f, 0.0f, 0.0f};
    const uint32_t one = OP == H3S_F16 ? 0x3C003C00u : 0x3F803F80u;
    const uint4 ones = make_uint4(one, one, one, one);
    const int64_t steps = (P.K + 127) / 128;
    const uint8_t* crow[NT];
    int64_t srow[NT];
#pragma unroll
    for (int b = 0; b < NT; ++b) {
        const int64_t n = min(n0 + 16 * b + l15, P.N - 1);          // (columns past the last: its own again, not stored)
        crow[b] = P.codes + n * (P.K / 2);
        srow[b] = n * P.groups;
    }
    auto load_codes = [&](int64_t step, uint4 (&w)[NT]) {
        const int64_t k = step * 128 + g * 32;
#pragma unroll
        for (int b = 0; b < NT; ++b) w[b] = k < P.K ? *reinterpret_cast<const uint4*>(crow[b] + k / 2) : make_uint4(0, 0, 0, 0);
    };
    uint4 w[NT];
    if (wave < steps) load_codes(wave, w);
    for (int64_t step = wave; step < steps; step += KW) {
        const int64_t kk = step * 128;
        uint32_t c[NT][4];
#pragma unroll
        for (int b = 0; b < NT; ++b) {
            // run j of 32 inputs to word j: the 4 x 4 words of the four lanes of a row exchanged
            auto p = __builtin_amdgcn_permlane32_swap(w[b].x, w[b].z, false, false);
            auto q = __builtin_amdgcn_permlane32_swap(w[b].y, w[b].w, false, false);
            auto r = __builtin_amdgcn_permlane16_swap(p[0], q[0], false, false);
            auto s = __builtin_amdgcn_permlane16_swap(p[1], q[1], false, false);
            c[b][0] = r[0]; c[b][1] = r[1]; c[b][2] = s[0]; c[b][3] = s[1];
        }
        if (step + KW < steps) load_codes(step + KW, w);
        float sc[NT][CNT], off[NT][CNT];
#pragma unroll
        for (int b = 0; b < NT; ++b) {
            l4_scales<J>(P, P.scale, srow[b], kk, sc[b]);
            if (P.mins) {
                l4_scales<J>(P, P.mins, srow[b], kk, off[b]);
#pragma unroll
                for (int i = 0; i < CNT; ++i) off[b][i] = __builtin_fmaf(16.0f, sc[b][i], off[b][i]);
            } else {
#pragma unroll
                for (int i = 0; i < CNT; ++i) off[b][i] = 24.0f * sc[b][i];
            }
        }
#pragma unroll
        for (int q = 0; q < CNT; ++q) {
            v4f_l4 y[MT][NT], sx[MT];
#pragma unroll
            for (int a = 0; a < MT; ++a) {
                sx[a] = v4f_l4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int b = 0; b < NT; ++b) y[a][b] = v4f_l4{0.0f, 0.0f, 0.0f, 0.0f};
            }
#pragma unroll
            for (int j = q * J; j < (q + 1) * J; ++j) {
                if (kk + 32 * j >= P.K) break;
                uint4 f[NT];
#pragma unroll
                for (int b = 0; b < NT; ++b) f[b] = l4_codes<OP>(c[b][j]);
#pragma unroll
                for (int a = 0; a < MT; ++a) {
                    const int64_t row = m0 + 16 * a + mrow;
                    uint4 xf[PARTS];
#pragma unroll
                    for (int p = 0; p < PARTS; ++p) xf[p] = make_uint4(0, 0, 0, 0);
                    if (row < P.M) l4_x<DT, PARTS>(P.x, row * P.K + kk + 32 * j + 8 * g, xf);
#pragma unroll
                    for (int p = 0; p < PARTS; ++p) {
                        sx[a] = l4_mma<OP>(xf[p], ones, sx[a]);
#pragma unroll
                        for (int b = 0; b < NT; ++b) y[a][b] = l4_mma<OP>(xf[p], f[b], y[a][b]);
                    }
                }
            }
#pragma unroll
            for (int a = 0; a < MT; ++a)
#pragma unroll
                for (int b = 0; b < NT; ++b)
#pragma unroll
                    for (int i = 0; i < NI; ++i) {
                        const float d = __builtin_fmaf(sc[b][q], y[a][b][i], -off[b][q] * sx[a][i]);
                        acc[a][b][i] = acc[a][b][i] + d;
                    }
        }
    }
    // the wavefronts' sums, in wavefront order
    __shared__ v4f_l4 part[KW][64];
#pragma unroll
    for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int b = 0; b < NT; ++b) {
            if (a || b) __syncthreads();
            part[wave][lane] = acc[a][b];
            __syncthreads();
            if (wave == (a * NT + b) % KW) {
                v4f_l4 y = part[0][lane];
#pragma unroll
                for (int v = 1; v < KW; ++v) y += part[v][lane];
                const int64_t n = n0 + 16 * b + l15;
                if (n < P.N) {
                    const float bias = P.bias ? P.bias[n] : 0.0f;
#pragma unroll
                    for (int i = 0; i < NI; ++i) {
                        const int64_t m = m0 + 16 * a + 4 * i + g;
                        if (m < P.M) store_any(P.out, P.out_dt, m * P.N + n, y[i] + bias);
                    }
                }
            }
        }
}

template <int DT, int MT, int NT, int KW, int NI>
static void l4_run(Ctx* c, const L4Args& P) {
    const dim3 grid((unsigned) ((P.N + 16 * NT - 1) / (16 * NT)), (unsigned) ((P.M + 16 * MT - 1) / (16 * MT)));
    if (P.group % 128 == 0) linear4_kernel<DT, MT, NT, KW, NI, 4><<<grid, 64 * KW, 0, c->stream>>>(P);
    else if (P.group % 64 == 0) linear4_kernel<DT, MT, NT, KW, NI, 2><<<grid, 64 * KW, 0, c->stream>>>(P);
    else linear4_kernel<DT, MT, NT, KW, NI, 1><<<grid, 64 * KW, 0, c->stream>>>(P);
}
template <int DT>
static void l4_rows(Ctx* c, const L4Args& P) {
    if (P.M <= 4) l4_run<DT, 1, 2, 8, 1>(c, P);
    else if (P.M <= 16) l4_run<DT, 1, 2, 8, 4>(c, P);
    else if (P.M <= 32) l4_run<DT, 2, 2, 8, 4>(c, P);
    else l4_run<DT, 4, 2, 4, 4>(c, P);
}

int linear4(void* ctx, const void* x, int dt, int64_t M, int64_t K, const uint8_t* codes, int64_t N, const void* scale, const void* mins,
            int scale_dt, int64_t group, const float* bias, void* out, int out_dt) try {
    const char* fn = "linear4";
    if (!dt_ok(dt) || !dt_ok(out_dt) || !dt_ok(scale_dt)) return fail(std::string(fn) + ": unknown element type");
    if (M < 0 || N < 0 || K < 0) return fail(std::string(fn) + ": a negative size");
    if (M == 0 || N == 0) return 0;
    if (group <= 0 || group % 32 != 0 || K % group != 0 || K == 0)
        return fail(std::string(fn) + ": the group size must be a multiple of 32 that divides the inputs (" + std::to_string(group) + " of " + std::to_string(K) + ")");
    if (!x || !codes || !scale || !out) return fail(std::string(fn) + ": x, codes, scale and out are required");
    if (!aligned16(x) || !aligned16(codes)) return fail(std::string(fn) + ": x and codes must be 16-byte aligned");
    if ((N + 31) / 32 > 0x7fffffff || (M + 15) / 16 > 65535) return fail(std::string(fn) + ": too many rows or columns");
    Ctx* c = ctx_of(ctx, fn);
    if (!c) return -1;
    L4Args P{x, M, K, N, codes, scale, mins, scale_dt, group, K / group, bias, out, out_dt, false};
    // a run of 128 inputs has 128 / group scales (1, 2 or 4): one load where every row's lie on such a boundary
    const int64_t cnt = group % 128 == 0 ? 1 : group % 64 == 0 ? 2 : 4;
    const uintptr_t span = (uintptr_t) (cnt * elem_size(scale_dt));
    P.svec = P.groups % cnt == 0 && (group == 32 || group == 64 || group % 128 == 0) && (uintptr_t) scale % span == 0 && (!mins || (uintptr_t) mins % span == 0);
    switch (dt) {
        case H3S_BF16: l4_rows<H3S_BF16>(c, P); break;
        case H3S_F16: l4_rows<H3S_F16>(c, P); break;
        default: l4_rows<H3S_F32>(c, P); break;
    }
    return launched(fn);
} catch (const std::exception& e) { return fail(e.what()); }

}  // namespace h3
