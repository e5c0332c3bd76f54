// kv_cache.hip - the 8-bit key/value cache's own operators (h3lm.h): kv_write (new tokens into their blocks) and kv_read
// (tokens out of them as values), and the table of function pointers that reaches all of h3lm.h.
//
// Mathematics: a block is 64 tokens of one head, keys or values, with one scale s = max|x| / 127 over all of it, so a code is
// off by at most s / 2. A block that tokens join later keeps its scale unless a larger token comes: then s' = max|x| / 127 of
// the newcomers, and the old codes are rounded again at s' (c' = rint(c s / s')). One block of threads owns one cache block of
// one head and side, so it finds the maximum, rescales and writes with no other writer and no atomics.
#include <algorithm>

#include "kv.h"

namespace h3 {

int kv_args(const std::string& fn, const h3_kv_cache* cache, const h3_kv_batch* batch, KvArgs& P) {
    if (!cache || !batch) return fail(fn + ": the cache and the batch are required");
    const h3_kv_cache& c = *cache;
    const h3_kv_batch& q = *batch;
    if (c.blocks <= 0 || c.heads <= 0 || c.dim <= 0 || c.dim > 256) return fail(fn + ": a cache has blocks, heads and 1 to 256 features a head");
    if (c.blocks > INT32_MAX || c.heads > 65535) return fail(fn + ": too many blocks or heads");
    if (q.seqs < 0 || q.rows < 0 || q.width < 0 || q.most < 0) return fail(fn + ": a negative size");
    if (q.rows > INT32_MAX || q.seqs >= INT32_MAX || q.width > (INT32_MAX - 64) / kKvB) return fail(fn + ": sizes past 32 bits");
    if (!c.k || !c.v || !c.k_scale || !c.v_scale) return fail(fn + ": the cache's codes and scales are required");
    if (!aligned16(c.k) || !aligned16(c.v)) return fail(fn + ": the cache's codes must be 16-byte aligned");
    if (q.seqs > 0 && (!q.starts || (q.width > 0 && !q.table))) return fail(fn + ": the table and the starts are required");
    P = KvArgs{c.k, c.v, c.k_scale, c.v_scale, c.blocks, (int) c.heads, (int) c.dim, q.table, q.starts, (int) q.width, (int) q.seqs, (int) q.rows};
    return 0;
}

// the maximum over a block of 256 threads, on every thread (with a barrier); a NaN anywhere gives NaN
__device__ __forceinline__ float block_max(float m, bool nan) {
    __shared__ float red[4];
    __shared__ int bad[4];
    m = wave_max<64>(m);
    const int any = __any(nan);
    if ((threadIdx.x & 63) == 0) { red[threadIdx.x >> 6] = m; bad[threadIdx.x >> 6] = any; }
    __syncthreads();
    m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    return (bad[0] | bad[1] | bad[2] | bad[3]) ? __builtin_nanf("") : m;
}

// four consecutive elements of a row from feature d on, zeros from `dim` on; vec: in one load (dim a multiple of 4, so they are all in
// or all out)
__device__ __forceinline__ void load4(const void* p, int dt, int64_t row, int d, int dim, bool vec, float* f) {
    if (vec) {
        if (d >= dim) {
            f[0] = f[1] = f[2] = f[3] = 0.0f;
        } else if (dt == H3S_F32) {
            load_f32x((const float*) p + row + d, f, 4);
        } else {
            const uint2 u = *reinterpret_cast<const uint2*>((const uint16_t*) p + row + d);
            float g[8];
            if (dt == H3S_BF16) Vec<H3S_BF16>::unpack(make_uint4(u.x, u.y, 0, 0), g);
            else Vec<H3S_F16>::unpack(make_uint4(u.x, u.y, 0, 0), g);
            f[0] = g[0]; f[1] = g[1]; f[2] = g[2]; f[3] = g[3];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = d + i < dim ? load_any(p, dt, row + d + i) : 0.0f;
    }
}
__device__ __forceinline__ void store4(void* p, int dt, int64_t row, int d, int dim, bool vec, const float* f) {
    if (vec) {
        if (d >= dim) return;
        if (dt == H3S_F32) *reinterpret_cast<float4*>((float*) p + row + d) = make_float4(f[0], f[1], f[2], f[3]);
        else *reinterpret_cast<uint2*>((uint16_t*) p + row + d) =
                 dt == H3S_BF16 ? make_uint2(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3])) : make_uint2(pack_f16(f[0], f[1]), pack_f16(f[2], f[3]));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (d + i < dim) store_any(p, dt, row + d + i, f[i]);
    }
}

// four old codes at the new scale, those where `keep` has a bit; zeros elsewhere
__device__ __forceinline__ uint32_t rescaled(uint32_t u, float ratio, uint32_t keep) {
    float c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float v = __builtin_rintf((float) (int8_t) (u >> (8 * i)) * ratio);
        // (a ratio that is not finite belongs to a scale that is not: the code then says nothing, and any is as good)
        c[i] = (keep >> i) & 1 ? fminf(fmaxf(v, -127.0f), 127.0f) : 0.0f;
    }
    return pack_i8x4(c[0], c[1], c[2], c[3]);
}

struct KvWriteArgs {
    KvArgs kv;
    const int32_t* past;
    const void *xk, *xv;
    int64_t k_stride, v_stride;
    int dt, nb;              // nb: blocks a sequence may touch (0: laid out by the rows, see kv_place)
    int k_vec, v_vec;        // rows four elements at a time
};
// (Chosen between, never indexed by the side: an index into the kernel's arguments became a scalar load whose base and offset
// were no multiples of 4 by themselves, and scalar loads drop the two low bits of each.)

// A block of threads: one head and side of the i-th cache block that sequence b's rows [r0, r0 + n) lie in. Where sequences have about
// as many rows each, a sequence has nb of them; else its share of the rows: n rows lie in at most floor(n / 64) + 2 blocks.
struct KvPlace { int side, h, i, b, r0, n; };
__device__ __forceinline__ KvPlace kv_place(const KvArgs& P, int nb) {
    KvPlace o;
    uint32_t id = blockIdx.x;
    o.side = (int) (id & 1);
    id >>= 1;
    o.h = (int) (id % (uint32_t) P.heads);
    id /= (uint32_t) P.heads;
    if (nb) {
        o.i = (int) (id % (uint32_t) nb);
        o.b = (int) (id / (uint32_t) nb);
        kv_rows_of(P, o.b, o.r0, o.n);
    } else {
        o.i = kv_find(P, (int) id, 1, kKvB, 2, o.b, o.r0, o.n);
    }
    return o;
}

constexpr int kKvRow = kKvB / 4 + 1;      // words of a feature's 64 tokens in LDS, one more than they are (banks)

// One block of threads: one cache block of one head, keys (side 0) or values (side 1). Thread t holds the pieces t + 256 p, p < WC, of
// four tokens x four features, W / 4 pieces side by side: its loads of the rows and its stores of keys are whole runs of them, and a
// piece's codes are four words either way round. Values go through LDS into a feature's tokens. Bound by latency for single tokens (the
// sequence's place, the rows, a maximum over the block, one store: 4.5 us; 64 sequences' 7.8) and by the rows' bytes for prompts (four of
// 5734 tokens in all 12.8 us).
template <int WC>
__global__ __launch_bounds__(256) void kv_write_kernel(KvWriteArgs A) {
    constexpr int W = 64 * WC;
    const KvArgs& P = A.kv;
    __shared__ uint32_t codes[W * kKvRow];
    const auto [side, h, i, b, r0, n] = kv_place(P, A.nb);
    const int64_t past = max(A.past[b], 0), end = min(past + n, (int64_t) P.width * kKvB);
    const int64_t j = past / kKvB + i;                                      // the sequence's block
    if (i < 0 || end <= past || j * kKvB >= end) return;                    // (no new token: the block is not touched)
    const int page = P.table[(int64_t) b * P.width + j];
    const int kept = (int) max(past - j * kKvB, (int64_t) 0);               // its tokens [0, kept) were there
    const int last = (int) min(end - j * kKvB, (int64_t) kKvB);             // and [kept, last) are new
    const int64_t row0 = r0 + (j * kKvB - past);                            // the row of its token 0 (with kept > 0: before r0)
    const int t = threadIdx.x;
    const void* x = side ? A.xv : A.xk;
    const int64_t stride = side ? A.v_stride : A.k_stride;
    const bool vec = (side ? A.v_vec : A.k_vec) != 0;

    float f[WC][4][4];                                                      // [piece][token][feature]
    float m = 0.0f;
    bool nan = false;
#pragma unroll
    for (int p = 0; p < WC; ++p) {
        const int tok = (t + 256 * p) / (W / 4) * 4, d = (t + 256 * p) % (W / 4) * 4;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (tok + k >= kept && tok + k < last) {
                load4(x, A.dt, (row0 + tok + k) * stride + (int64_t) h * P.dim, d, P.dim, vec, f[p][k]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) f[p][k][e] = 0.0f;
            }
        }
    }
    if (page < 0 || page >= P.blocks) return;                               // (after the rows' loads, which need not wait for it)
    const int64_t tile = (int64_t) page * P.heads + h;
    float* scale = (side ? P.vs : P.ks) + tile;
    const float was = kept ? *scale : 0.0f;
#pragma unroll
    for (int p = 0; p < WC; ++p)
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                m = fmaxf(m, fabsf(f[p][k][e]));
                nan = nan || f[p][k][e] != f[p][k][e];
            }
    m = block_max(m, nan);                                                  // (a barrier: every thread has read the old scale)
    float s = m / 127.0f;
    // (a NaN on either side wins)
    s = s != s ? s : was > s || was != was ? was : s;
    s = s < 1e-30f ? 1e-30f : s;
    const bool moved = kept && s != was;                                    // (NaN: rescaled, to no effect)
    const float ratio = was / s, inv = 1.0f / s;                            // (quant_code: x / s as the IEEE division gives it)
    if (t == 0) *scale = s;

    int8_t* base = (side ? P.v : P.k) + tile * kKvB * W;
#pragma unroll
    for (int p = 0; p < WC; ++p) {
        const int tok = (t + 256 * p) / (W / 4) * 4, d = (t + 256 * p) % (W / 4) * 4;
        if (side == 0 && tok + 4 <= kept && !moved) continue;               // (old tokens only, unchanged)
        float c[4][4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) c[k][e] = fmaxf(quant_code(f[p][k][e], s, inv), -127.0f);
        if (side == 0) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                uint32_t* dst = reinterpret_cast<uint32_t*>(base + (int64_t) (tok + k) * W + d);
                if (tok + k >= kept) *dst = pack_i8x4(c[k][0], c[k][1], c[k][2], c[k][3]);
                else if (moved) *dst = rescaled(*dst, ratio, 15u);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) codes[(d + e) * kKvRow + tok / 4] = pack_i8x4(c[0][e], c[1][e], c[2][e], c[3][e]);
        }
    }
    if (side == 0) return;
    __syncthreads();
    // values: 16-byte pieces of 16 tokens of one feature; pieces of old tokens only are left alone unless the scale moved
#pragma unroll
    for (int p = 0; p < WC; ++p) {
        const int piece = t + 256 * p, d = piece / 4, k0 = (piece % 4) * 16;
        const int old = min(max(kept - k0, 0), 16);
        if (old == 16 && !moved) continue;
        uint4* dst = reinterpret_cast<uint4*>(base + (int64_t) d * kKvB + k0);
        uint4 u = make_uint4(0, 0, 0, 0);
        if (old) u = *dst;
        uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int o = min(max(old - 4 * q, 0), 4);                      // old tokens in this word
            if (moved) w[q] = rescaled(w[q], ratio, (1u << o) - 1);
            const uint32_t mask = o == 4 ? 0xffffffffu : (1u << (8 * o)) - 1;
            w[q] = (w[q] & mask) | (codes[d * kKvRow + k0 / 4 + q] & ~mask);
        }
        *dst = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

struct KvReadArgs {
    KvArgs kv;
    const int32_t* first;
    void *xk, *xv;
    int64_t k_stride, v_stride;
    int dt, nb;
    int k_vec, v_vec;
};

// One block of threads: the tokens that a read takes out of one cache block of one head and side (pieces as in kv_write_kernel). Bound as
// there: one token 4.9 us, the four prompts 10.4.
template <int WC>
__global__ __launch_bounds__(256) void kv_read_kernel(KvReadArgs A) {
    constexpr int W = 64 * WC;
    const KvArgs& P = A.kv;
    __shared__ uint32_t codes[W * kKvRow];
    const auto [side, h, i, b, r0, n] = kv_place(P, A.nb);
    const int64_t first = max(A.first[b], 0), end = first + n;
    const int64_t j = first / kKvB + i;
    if (i < 0 || j * kKvB >= end) return;
    const int page = j < P.width ? P.table[(int64_t) b * P.width + j] : -1;
    const bool there = page >= 0 && page < P.blocks;
    const int from = (int) max(first - j * kKvB, (int64_t) 0), to = (int) min(end - j * kKvB, (int64_t) kKvB);
    const int64_t row0 = r0 + (j * kKvB - first), tile = (int64_t) (there ? page : 0) * P.heads + h;
    const float s = there ? (side ? P.vs : P.ks)[tile] : 0.0f;
    const int8_t* base = (side ? P.v : P.k) + tile * kKvB * W;
    const int t = threadIdx.x;
    void* x = side ? A.xv : A.xk;
    const int64_t stride = side ? A.v_stride : A.k_stride;
    const bool vec = (side ? A.v_vec : A.k_vec) != 0;
    uint32_t w[WC][4];                                                      // a piece's codes: by token for keys, by feature for values
    if (side == 1) {
#pragma unroll
        for (int p = 0; p < WC; ++p) {
            const int piece = t + 256 * p, d = piece / 4, k0 = (piece % 4) * 16;
            uint4 u = make_uint4(0, 0, 0, 0);
            if (there && k0 < to && k0 + 16 > from) u = *reinterpret_cast<const uint4*>(base + (int64_t) d * kKvB + k0);
            uint32_t* dst = codes + d * kKvRow + k0 / 4;
            dst[0] = u.x; dst[1] = u.y; dst[2] = u.z; dst[3] = u.w;
        }
        __syncthreads();
    }
#pragma unroll
    for (int p = 0; p < WC; ++p) {
        const int tok = (t + 256 * p) / (W / 4) * 4, d = (t + 256 * p) % (W / 4) * 4;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            w[p][k] = 0;
            if (side == 1) w[p][k] = codes[(d + k) * kKvRow + tok / 4];
            else if (there && tok + k >= from && tok + k < to) w[p][k] = *reinterpret_cast<const uint32_t*>(base + (int64_t) (tok + k) * W + d);
        }
    }
#pragma unroll
    for (int p = 0; p < WC; ++p) {
        const int tok = (t + 256 * p) / (W / 4) * 4, d = (t + 256 * p) % (W / 4) * 4;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (tok + k < from || tok + k >= to) continue;
            float f[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) f[e] = there ? (float) (int8_t) (side ? w[p][e] >> (8 * k) : w[p][k] >> (8 * e)) * s : 0.0f;
            store4(x, A.dt, (row0 + tok + k) * stride + (int64_t) h * P.dim, d, P.dim, vec, f);
        }
    }
}

// what kv_write and kv_read check alike, and their grid: `most` rows of a sequence can lie in nb blocks, all rows in rows / 64 + 2 seqs
// (one sequence of 16400 rows among 1024 of one: 1281 cache blocks in 2304 places instead of 263168)
static int row_checks(const std::string& fn, const KvArgs& P, const h3_kv_batch& q, const int32_t* at, const char* at_name, const void* k,
                      int64_t k_stride, const void* v, int64_t v_stride, int dt, int* nb, unsigned* grid) {
    const int64_t feats = (int64_t) P.heads * P.dim;
    if (!dt_ok(dt)) return fail(fn + ": unknown element type");
    if (!at || !k || !v) return fail(fn + ": k, v and " + at_name + " are required");
    if (k_stride < feats || v_stride < feats) return fail(fn + ": a row stride is shorter than a row");
    const int64_t each = (std::min<int64_t>(q.most, P.rows) + kKvB - 2) / kKvB + 1, all = P.rows / kKvB + 2 * (int64_t) P.seqs;
    *nb = each * P.seqs <= all ? (int) each : 0;
    const int64_t places = *nb ? each * P.seqs : all;
    if (places > kKvMostBlocks / 2 / P.heads) return fail(fn + ": too many blocks of work");
    *grid = (unsigned) (places * P.heads * 2);
    return 0;
}
// whether rows of k or v can be taken four elements at a time
static bool rows_vec(const void* p, int64_t stride, int dim, int dt) {
    const int piece = 4 * elem_size(dt);
    return (uintptr_t) p % piece == 0 && dim % 4 == 0 && stride % 4 == 0;
}

int kv_write(void* ctx, const h3_kv_cache* cache, const h3_kv_batch* batch, const int32_t* past, const void* k, int64_t k_stride,
             const void* v, int64_t v_stride, int dt) try {
    const char* fn = "kv_write";
    KvWriteArgs A;
    if (kv_args(fn, cache, batch, A.kv)) return -1;
    if (A.kv.seqs == 0 || A.kv.rows == 0 || batch->most == 0 || A.kv.width == 0) return 0;
    unsigned grid;
    if (row_checks(fn, A.kv, *batch, past, "past", k, k_stride, v, v_stride, dt, &A.nb, &grid)) return -1;
    Ctx* c = ctx_of(ctx, fn);
    if (!c) return -1;
    A.past = past;
    A.xk = k; A.xv = v;
    A.k_stride = k_stride; A.v_stride = v_stride;
    A.dt = dt;
    A.k_vec = rows_vec(k, k_stride, A.kv.dim, dt);
    A.v_vec = rows_vec(v, v_stride, A.kv.dim, dt);
    switch (kv_width(A.kv.dim) / 64) {
        case 1: kv_write_kernel<1><<<grid, 256, 0, c->stream>>>(A); break;
        case 2: kv_write_kernel<2><<<grid, 256, 0, c->stream>>>(A); break;
        case 3: kv_write_kernel<3><<<grid, 256, 0, c->stream>>>(A); break;
        default: kv_write_kernel<4><<<grid, 256, 0, c->stream>>>(A); break;
    }
    return launched(fn);
} catch (const std::exception& e) { return fail(e.what()); }

int kv_read(void* ctx, const h3_kv_cache* cache, const h3_kv_batch* batch, const int32_t* first, void* k, int64_t k_stride, void* v,
            int64_t v_stride, int dt) try {
    const char* fn = "kv_read";
    KvReadArgs A;
    if (kv_args(fn, cache, batch, A.kv)) return -1;
    if (A.kv.seqs == 0 || A.kv.rows == 0 || batch->most == 0) return 0;
    unsigned grid;
    if (row_checks(fn, A.kv, *batch, first, "first", k, k_stride, v, v_stride, dt, &A.nb, &grid)) return -1;
    Ctx* c = ctx_of(ctx, fn);
    if (!c) return -1;
    A.first = first;
    A.xk = k; A.xv = v;
    A.k_stride = k_stride; A.v_stride = v_stride;
    A.dt = dt;
    A.k_vec = rows_vec(k, k_stride, A.kv.dim, dt);
    A.v_vec = rows_vec(v, v_stride, A.kv.dim, dt);
    switch (kv_width(A.kv.dim) / 64) {
        case 1: kv_read_kernel<1><<<grid, 256, 0, c->stream>>>(A); break;
        case 2: kv_read_kernel<2><<<grid, 256, 0, c->stream>>>(A); break;
        case 3: kv_read_kernel<3><<<grid, 256, 0, c->stream>>>(A); break;
        default: kv_read_kernel<4><<<grid, 256, 0, c->stream>>>(A); break;
    }
    return launched(fn);
} catch (const std::exception& e) { return fail(e.what()); }

}  // namespace h3

// (host only: a constant of function addresses would otherwise be emitted into the device code as well)
#ifndef __HIP_DEVICE_COMPILE__
extern "C" __attribute__((visibility("default"))) const h3_lm_api h3lm = {
    (int64_t) sizeof(h3_lm_api), h3::kv_write, h3::kv_read, h3::kv_attention, h3::kv_attention_work, h3::linear4,
};
#endif
