/* h3lm.h - the operators of libh3hip.so that run a language model token by token: an 8-bit key/value cache, the attention
 * that reads it, and linear layers with 4-bit weights. They stand beside h3hip.h's causal attention and linear layers (the
 * text encoder's whole-sequence forms) and follow its conventions: device pointers of the context's GPU, asynchronous on the
 * context's stream in call order, 0 or -1 with the reason in h3s_last_error(), arguments checked before any work is queued,
 * empty shapes do nothing. No counterpart in the reference.
 *
 * The library's function names are the reference's header and its additions (h3hip.h) and stay that set; these operators are
 * reached through one exported table of function pointers, `h3lm`:
 *
 *     #include "h3lm.h"
 *     h3lm.kv_write(ctx, &cache, &batch, past, k, k_stride, v, v_stride, H3S_BF16);
 *
 * A call whose work would take 2^32 threads of the device or more is refused ("too many blocks of work").
 *
 * All of them can be recorded into a HIP graph (kv_attention with a workspace of the caller's, below). The values behind
 * device pointers - block tables, starts, lengths - are read on the device when the work runs, so a recorded graph is replayed
 * on new ones. No value there makes a kernel read or write outside its buffers: entries out of range are treated as stated.
 */
#ifndef H3LM_H
#define H3LM_H

#include "h3hip.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { H3_KV_BLOCK = 64 };   /* tokens in a block of the cache */

/* One layer's key/value cache: a pool of `blocks` blocks of 64 tokens, for `heads` key/value heads of `dim` features (1 to
 * 256), held as 8-bit codes with one scale for each block and head (value = code * scale). With w = dim up to the next
 * multiple of 64: */
typedef struct {
    int8_t* k;        /* [blocks, heads, 64, w]: a token's features side by side; 16-byte aligned */
    int8_t* v;        /* [blocks, heads, w, 64]: a feature's tokens side by side; 16-byte aligned */
    float* k_scale;   /* [blocks, heads] */
    float* v_scale;   /* [blocks, heads] */
    int64_t blocks, heads, dim;
} h3_kv_cache;

/* The sequences of one call. Token p of sequence b lies in block table[b * width + p / 64], at p % 64; an entry outside
 * 0 .. blocks - 1 is a block that is not there (its tokens are neither written nor seen). Sequence b's tokens of this call
 * are the rows starts[b] .. starts[b + 1] - 1 of the row operands (starts ascending, within 0 .. rows; what lies outside is
 * cut off); rows behind starts[seqs] are neither read nor written. `most`: at least the most rows of any sequence (a
 * sequence's rows from `most` on may be left out). */
typedef struct {
    const int32_t* table;    /* [seqs, width] */
    const int32_t* starts;   /* [seqs + 1] */
    int64_t seqs, width, rows, most;
} h3_kv_batch;

typedef struct {
    int64_t size;            /* bytes of this table: a later library's is longer */

    /* New tokens into the cache: row starts[b] + j of k and v (heads * dim features of type dt, rows at element strides
     * k_stride and v_stride) becomes token past[b] + j of sequence b. For each block and head touched,
     *     s' = max(s, max|x| / 127, 1e-30) over the block's new tokens (s: its scale if tokens before past[b] lie in it, else 0)
     *     new codes rint(x / s') in -127 .. 127; where s' > s the old codes become rint(c * (s / s'))
     * in float32 with IEEE division; codes behind the last token are zero. So a block's old tokens lose precision when a larger
     * one joins them, and writing tokens one by one may give other codes than writing them together. An infinity or NaN in a new
     * token makes its block's scale infinite or NaN, and the block's tokens read as such. Tokens past the table's end are
     * dropped; a past below 0 counts as 0. No two sequences may write into one block; blocks they share may only be read. */
    int (*kv_write)(void* ctx, const h3_kv_cache* cache, const h3_kv_batch* batch, const int32_t* past, const void* k,
                    int64_t k_stride, const void* v, int64_t v_stride, int dt);

    /* Tokens out of the cache as values: row starts[b] + j of k and v (heads * dim features of type dt) receives token
     * first[b] + j of sequence b, zeros where that is not in the cache's blocks (a first below 0 counts
     * as 0). code * scale in float32, rounded to dt. */
    int (*kv_read)(void* ctx, const h3_kv_cache* cache, const h3_kv_batch* batch, const int32_t* first, void* k,
                   int64_t k_stride, void* v, int64_t v_stride, int dt);

    /* Attention of each sequence's newest tokens over its cached ones, those tokens themselves among them: with lengths[b]
     * tokens in the cache (kv_write's past[b] plus the rows), row starts[b] + j is token p = lengths[b] - rows of b + j, and sees
     * the tokens 0 .. p, of them the last `window` (0: all), of them those whose byte mask[b * mask_stride + token] is not zero
     * (mask NULL: all; tokens from mask_stride on are hidden). softmax(q . k * scale) v with query head h reading key/value head
     * h / (q_heads / heads); scale 0: 1 / sqrt(dim), else above 0. q [rows, q_heads * dim] of type dt at element stride q_stride; out
     * [rows, q_heads * dim] of type out_dt; lse NULL or float32 [rows, q_heads], the logarithm of the row's sum of exponentials. A row
     * that sees nothing gets zeros (lse -infinity). Hidden tokens have no effect, whatever their codes, scales and mask say.
     * Products, softmax and sums are float32 (q to 11 bits of each value for 16-bit types, which is all they have, 22 for float32;
     * probabilities to 22, and to 11 for 16-bit q where a sequence has more than 32 rows times heads of a group, or 16 with dim above
     * 128), rounded once to out_dt.
     * Lengths count as at least 0 and at most the table's 64 * width tokens. out may not overlap q.
     * max_len: about the longest of the lengths (0: the table's width); it only decides how the work is split. Sequences with many
     * rows and with few may be mixed: each takes the kernel for its number of rows.
     * work: a device workspace of at least kv_attention_work(...) bytes, 16-byte aligned, in use until the call's work is done;
     * NULL: the context's own scratch. A call recorded into a graph has to bring its own (two graphs, or a graph and eager calls,
     * would share the context's): -1 otherwise, unless it needs none. */
    int (*kv_attention)(void* ctx, const h3_kv_cache* cache, const h3_kv_batch* batch, const int32_t* lengths, int64_t max_len,
                        const void* q, int64_t q_stride, int dt, int64_t q_heads, float scale, int64_t window, const uint8_t* mask,
                        int64_t mask_stride, void* out, int out_dt, float* lse, void* work, uint64_t work_bytes);
    /* The bytes that kv_attention needs for these arguments (0: none), or -1. */
    int64_t (*kv_attention_work)(void* ctx, const h3_kv_cache* cache, const h3_kv_batch* batch, int64_t max_len, int64_t q_heads,
                                 int64_t window);

    /* A linear layer with 4-bit weights: out [M, N] of type out_dt = x W^T + bias, x [M, K] of type dt. codes [N, K / 2]: byte i of
     * a row holds the codes of inputs 2 i (low four bits) and 2 i + 1. With g = k / group and scale [N, K / group] of type scale_dt:
     *     W[n, k] = scale[n, g] * (code - 8)            mins NULL
     *     W[n, k] = scale[n, g] * code - mins[n, g]     mins [N, K / group] of type scale_dt
     * group: a multiple of 32 that divides K, and K at most 2^20. Float32 sums; bias float32 [N] or NULL, added before the one rounding. codes and x
     * 16-byte aligned, rows whole 16-byte pieces (K a multiple of 32 makes them so). out may not overlap x. No workspace.
     * 16-bit x: the sums run over x * (16 + code), with 24 times x's sum (16 times, and the minima) taken off again. float32's rounding then counts
     * against those: up to 2e-5 of the result where x has one sign and the codes lie within one of 8, 3e-7 for uniform codes. float32 x: the sums run
     * over x * (code - 8) in all of x's digits (values below 2^-110 have fewer). Either way an infinity or NaN in a row of x makes that row of
     * out infinite or NaN (and no other row), and so may values whose sums times 31 leave float32. */
    int (*linear4)(void* ctx, const void* x, int dt, int64_t M, int64_t K, const uint8_t* codes, int64_t N, const void* scale,
                   const void* mins, int scale_dt, int64_t group, const float* bias, void* out, int out_dt);
} h3_lm_api;

extern const h3_lm_api h3lm;

#ifdef __cplusplus
}
#endif
#endif
