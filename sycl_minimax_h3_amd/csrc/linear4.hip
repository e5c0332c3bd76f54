// linear4.hip - linear4 (h3lm.h): the checks and the choice of the kernel (linear4_impl.h).
#include <algorithm>

#include "linear4_impl.h"

namespace h3 {

int linear4(void* ctx, const void* x, int dt, int64_t M, int64_t K, const uint8_t* codes, int64_t N, const void* scale, const void* mins,
            int scale_dt, int64_t group, const float* bias, void* out, int out_dt) try {
    const char* fn = "linear4";
    if (!dt_ok(dt) || !dt_ok(out_dt) || !dt_ok(scale_dt)) return fail(std::string(fn) + ": unknown element type");
    if (M < 0 || N < 0 || K < 0) return fail(std::string(fn) + ": a negative size");
    if (M == 0 || N == 0) return 0;
    if (group <= 0 || group % 32 != 0 || K % group != 0 || K == 0)
        return fail(std::string(fn) + ": the group size must be a multiple of 32 that divides the inputs (" + std::to_string(group) + " of " + std::to_string(K) + ")");
    if (K > kL4MostK) return fail(std::string(fn) + ": at most " + std::to_string(kL4MostK) + " inputs");
    if (!x || !codes || !scale || !out) return fail(std::string(fn) + ": x, codes, scale and out are required");
    if (!aligned16(x) || !aligned16(codes)) return fail(std::string(fn) + ": x and codes must be 16-byte aligned");
    // A launch of 2^32 threads or more is cut without an error: rows past what one takes (in the smallest tiles that long calls have, 32
    // rows x 128 columns a block of 512 threads) are launches of their own.
    const int64_t most = 0x7fffff, across = ((N + 127) / 128 + 7) / 8 * 8;
    if (M > ((int64_t) 1 << 31) || across > most) return fail(std::string(fn) + ": too many rows or columns");
    const int64_t chunk = most / across * 32;
    Ctx* c = ctx_of(ctx, fn);
    if (!c) return -1;
    const uint64_t runs = (uint64_t) group / 32;
    L4Args P{x, M, N, (int) K, codes, scale, mins ? mins : scale, scale_dt, mins != nullptr, (int) group, (int) (K / group),
             runs == 1 ? 0u : (uint32_t) (((1ull << 32) + runs - 1) / runs), bias, out, out_dt};
    for (int64_t m = 0; m < M; m += chunk) {
        P.x = (const char*) x + m * K * elem_size(dt);
        P.out = (char*) out + m * N * elem_size(out_dt);
        P.M = std::min(chunk, M - m);
        if (dt == H3S_BF16) l4_bf16(c, P);
        else if (dt == H3S_F16) l4_f16(c, P);
        else l4_f32(c, P);
    }
    return launched(fn);
} catch (const std::exception& e) { return fail(e.what()); }

}  // namespace h3
